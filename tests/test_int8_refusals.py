"""CPU tests: what the 8-bit integer and MoE gradient entries refuse, before any CUDA call."""
import ctypes

import pytest

P = 0x10000      # an address that is only compared, never read


@pytest.fixture(scope="module")
def capi(built_lib):
    from layerstormgemmkernels_b200 import capi as _capi
    return _capi


def gemm(capi, **kw):
    d = dict(M=4, N=8, K=64, A=P, lda=64, B=P, ldb=64, D=P, scale_A=P, scale_B=P, output_dtype=0)
    d.update(kw)
    return capi.Int8GemmParams(**d)


@pytest.mark.parametrize("kw,error,text", [
    (dict(M=-1), ValueError, "negative"), (dict(K=0), ValueError, "1 <= K"), (dict(K=131057, lda=131072, ldb=131072), ValueError, "1 <= K"),
    (dict(lda=48), ValueError, "smaller than K"), (dict(ldb=48), ValueError, "smaller than K"), (dict(A=None), ValueError, "null"),
    (dict(scale_A=None), ValueError, "null"), (dict(scale_B=None), ValueError, "null"), (dict(D=None), ValueError, "null"),
    (dict(A=P + 8), RuntimeError, "16-byte"), (dict(B=P + 1), RuntimeError, "16-byte"), (dict(lda=72), RuntimeError, "16-byte"),
    (dict(ldb=65), RuntimeError, "16-byte"), (dict(D=P + 1), RuntimeError, "aligned"), (dict(D=P + 2, output_dtype=1), RuntimeError, "aligned"),
    (dict(scale_A=P + 2), RuntimeError, "aligned"), (dict(scale_B=P + 1), RuntimeError, "aligned"),
    (dict(output_dtype=3), RuntimeError, "bf16, fp16 or f32")])
def test_gemm_refusals(capi, kw, error, text):
    with pytest.raises(error, match=text):
        capi.check(capi.lib.lsg_int8_gemm(ctypes.byref(gemm(capi, **kw)), None))


def test_gemm_nothing_to_do(capi):
    assert capi.lib.lsg_int8_gemm(ctypes.byref(gemm(capi, M=0, A=None)), None) == 0
    assert capi.lib.lsg_int8_gemm(ctypes.byref(gemm(capi, N=0, B=None)), None) == 0
    with pytest.raises(ValueError, match="null"):
        capi.check(capi.lib.lsg_int8_gemm(None, None))


def test_gemm_from_bf16_refusals(capi):
    need = capi.lib.lsg_int8_gemm_from_bf16_workspace_bytes(40, 64)
    assert need == 40 * 64 + 256 and capi.lib.lsg_int8_gemm_from_bf16_workspace_bytes(0, 64) == 0
    assert capi.lib.lsg_int8_gemm_from_bf16_workspace_bytes(30, 100) == 3584 + 256   # rows of 112 bytes
    assert capi.lib.lsg_int8_gemm_from_bf16_workspace_bytes(1, 100) == 0             # quantized inside the mat-vec

    def call(dtype=0, ws=P, size=need, M=40, **kw):
        kw["M"] = M
        capi.check(capi.lib.lsg_int8_gemm_from_bf16(ctypes.byref(gemm(capi, **kw)), dtype, ws, size, None))
    for kw, error, text in ((dict(dtype=1), RuntimeError, "bf16 or fp16"), (dict(ws=None), RuntimeError, "workspace"),
                            (dict(size=need - 1), RuntimeError, "workspace"), (dict(ws=P + 16), RuntimeError, "256-byte"),
                            (dict(lda=63), ValueError, "stride"), (dict(K=0), ValueError, "1 <= K"), (dict(A=None), ValueError, "null"),
                            (dict(ldb=72), RuntimeError, "16-byte"), (dict(A=P + 1), RuntimeError, "aligned")):
        with pytest.raises(error, match=text):
            call(**kw)


def test_quantizer_refusals(capi):
    def quant(x=P, ldx=64, dtype=0, codes=P, ldq=64, scales=P, rows=4, K=64):
        capi.check(capi.lib.lsg_dynamic_int8_quant(x, ldx, dtype, codes, ldq, scales, rows, K, None))
    for kw, error, text in ((dict(dtype=1), RuntimeError, "bf16 or fp16"), (dict(rows=-1), ValueError, "negative"),
                            (dict(rows=1 << 31), ValueError, "rows"), (dict(ldx=63), ValueError, "stride"),
                            (dict(ldq=48), ValueError, "stride"), (dict(ldq=72), RuntimeError, "16-byte"),
                            (dict(codes=P + 4), RuntimeError, "16-byte"), (dict(x=P + 1), RuntimeError, "aligned"),
                            (dict(scales=P + 2), RuntimeError, "aligned"), (dict(x=None), ValueError, "null"),
                            (dict(scales=None), ValueError, "null")):
        with pytest.raises(error, match=text):
            quant(**kw)
    quant(rows=0, x=None)
    with pytest.raises(ValueError, match="stride"):
        capi.check(capi.lib.lsg_silu_mul_int8_quant(P, 64, P, 32, 0, P, 64, P, 4, 64, None))
    with pytest.raises(RuntimeError, match="f32"):
        capi.check(capi.lib.lsg_silu_mul_int8_quant(P, 64, P, 64, 5, P, 64, P, 4, 64, None))
    with pytest.raises(ValueError, match="top_k"):
        capi.check(capi.lib.lsg_moe_permute_int8(P, 64, 0, P, 4, 0, 64, P, 64, P, None))
    with pytest.raises(ValueError, match="pairs"):
        capi.check(capi.lib.lsg_moe_permute_int8(P, 64, 0, P, 1 << 30, 4, 64, P, 64, P, None))


def test_grouped_refusals(capi):
    def call(T=8, **kw):
        d = dict(num_experts=2, N=8, K=64, A_base=P, lda=64, B_base=P, ldb=64, D_base=P, scale_A_base=P, scale_B_base=P,
                 expert_offsets=P, output_dtype=0)
        d.update(kw)
        capi.check(capi.lib.lsg_int8_grouped_gemm(ctypes.byref(capi.Int8GroupedGemmParams(**d)), T, None))
    for kw, error, text in ((dict(num_experts=1025), ValueError, "1024"), (dict(N=-1), ValueError, "negative"), (dict(T=-1), ValueError, "negative"),
                            (dict(expert_offsets=None), ValueError, "null"), (dict(lda=72), RuntimeError, "16-byte"),
                            (dict(num_experts=1024, N=1 << 22), ValueError, "weight rows"), (dict(output_dtype=9), RuntimeError, "bf16")):
        with pytest.raises(error, match=text):
            call(**kw)
    call(T=0)
    call(num_experts=0)


def test_ffn_refusals(capi):
    need = capi.lib.lsg_int8_moe_ffn_workspace_bytes(4, 2, 64, 32)
    assert need > 0 and capi.lib.lsg_int8_moe_ffn_workspace_bytes(0, 2, 64, 32) == 0

    def call(ws=P, size=need, **kw):
        d = dict(num_tokens=4, top_k=2, num_experts=2, H=64, I=32, hidden=P, ld_hidden=64, input_dtype=0, expert_offsets=P,
                 inv_perm=P, gate_up=P, gate_up_scales=P, down=P, down_scales=P, D=P, output_dtype=0)
        d.update(kw)
        capi.check(capi.lib.lsg_int8_moe_ffn(ctypes.byref(capi.Int8MoeFfnParams(**d)), ws, size, None))
    for kw, error, text in ((dict(H=72), ValueError, "multiples of 16"), (dict(I=40), ValueError, "multiples of 16"),
                            (dict(I=0), ValueError, "multiples of 16"), (dict(top_k=0), ValueError, "top_k"),
                            (dict(num_tokens=-1), ValueError, "negative"), (dict(num_experts=2000), ValueError, "1024"),
                            (dict(input_dtype=1), RuntimeError, "bf16 or fp16"), (dict(output_dtype=7), RuntimeError, "bf16"),
                            (dict(ws=None), RuntimeError, "workspace"), (dict(size=need - 1), RuntimeError, "workspace"),
                            (dict(ws=P + 64), RuntimeError, "256-byte"), (dict(inv_perm=None), ValueError, "null"),
                            (dict(gate_up=P + 4), RuntimeError, "16-byte"), (dict(down=None), ValueError, "null"),
                            (dict(ld_hidden=60), ValueError, "stride")):
        with pytest.raises(error, match=text):
            call(**kw)
    call(num_tokens=0)


def test_moe_gradient_refusals(capi):
    L = capi.lib
    for fn, args, error, text in (
            (L.lsg_moe_permute_backward, (P, 3, P, 8, 4, 2, 64, P, None), RuntimeError, "dtype"),
            (L.lsg_moe_permute_backward, (P, 0, P, 8, 4, 17, 64, P, None), ValueError, "top_k"),
            (L.lsg_moe_permute_backward, (P, 0, P, -1, 4, 2, 64, P, None), ValueError, "negative"),
            (L.lsg_moe_permute_backward, (P, 0, None, 8, 4, 2, 64, P, None), ValueError, "null"),
            (L.lsg_moe_permute_backward, (P, 0, P, 8, 1 << 30, 4, 64, P, None), ValueError, "pairs"),
            (L.lsg_moe_unpermute_backward, (P, P, 0, P, P, None, 0, 9, 4, 2, 64, P, P, None), ValueError, "more rows"),
            (L.lsg_moe_unpermute_backward, (P, P, 0, P, P, P, 0, 8, 4, 2, 64, P, P, None), ValueError, "num_experts"),
            (L.lsg_moe_unpermute_backward, (P, None, 0, P, P, None, 0, 8, 4, 2, 64, P, P, None), ValueError, "null"),
            (L.lsg_moe_unpermute_backward, (P, P, 0, P, P, None, 0, 8, 4, 2, -64, P, P, None), ValueError, "negative"),
            (L.lsg_moe_permute_backward, (P + 2, 1, P, 8, 4, 2, 64, P, None), RuntimeError, "aligned"),
            (L.lsg_moe_unpermute_backward, (P, P + 1, 0, P, P, None, 0, 8, 4, 2, 64, P, P, None), RuntimeError, "aligned"),
            (L.lsg_moe_route_backward, (P, P, P, 4, 2000, 2, P, None), ValueError, "E <= 1024"),
            (L.lsg_moe_route_backward, (P, P, P, 4, 2, 3, P, None), ValueError, "top_k"),
            (L.lsg_moe_route_backward, (P, P, None, 4, 8, 2, P, None), ValueError, "null"),
            (L.lsg_moe_permute_dtype, (P, 9, P, 8, 4, 2, 64, P, None), RuntimeError, "dtype"),
            (L.lsg_moe_unpermute_dtype, (P, 1, P, P, 8, 4, 0, 64, P, None), ValueError, "top_k")):
        with pytest.raises(error, match=text):
            capi.check(fn(*args))
    assert L.lsg_moe_permute_backward(None, 0, None, 0, 0, 2, 64, None, None) == 0
    assert L.lsg_moe_route_backward(None, None, None, 0, 8, 2, None, None) == 0


def test_operators_refuse_cpu_tensors(capi):
    import torch
    from layerstormgemmkernels_b200 import ops
    from layerstormgemmkernels_b200.torch_ext import build_ext
    build_ext.build_ops()
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    q = torch.zeros(8, 64, dtype=torch.int8)
    s = torch.ones(8)
    inv = torch.zeros(8, dtype=torch.int32)
    for bad in (lambda: ops.dynamic_int8_quant(x), lambda: ops.weight_int8_quant(x), lambda: ops.silu_mul_int8_quant(x, x),
                lambda: ops.int8_gemm(q, q, s, s, 8, 8, 64, "bf16"), lambda: ops.int8_gemm_from_bf16(x, q, s),
                lambda: ops.moe_permute_int8(x, inv, 2), lambda: ops.moe_permute_backward(x, inv, 2),
                lambda: ops.moe_unpermute_backward(x, x, inv, s.view(4, 2)),
                lambda: ops.moe_route_backward(inv.view(4, 2), s.view(4, 2), s.view(4, 2), 8)):
        with pytest.raises(RuntimeError, match="CUDA"):
            bad()


def test_unpermute_output_type_refusals(capi):
    f = capi.lib.lsg_moe_unpermute_to
    for args, error, text in (((P, 0, P, P, 8, 4, 2, 64, P, 2, None), RuntimeError, "rows' type"),
                              ((P, 1, P, P, 8, 4, 2, 64, P, 9, None), RuntimeError, "rows' type"),
                              ((P, 1, P, P, 8, 4, 17, 64, P, 0, None), ValueError, "top_k"),
                              ((P + 2, 1, P, P, 8, 4, 2, 64, P, 0, None), RuntimeError, "aligned"),
                              ((P, 1, P, P, 8, 4, 2, 64, P + 1, 0, None), RuntimeError, "aligned"),
                              ((P, 1, None, P, 8, 4, 2, 64, P, 0, None), ValueError, "null"),
                              ((P, 1, P, P, -1, 4, 2, 64, P, 0, None), ValueError, "negative")):
        with pytest.raises(error, match=text):
            capi.check(f(*args))
    assert f(None, 1, None, None, 0, 0, 2, 64, None, 0, None) == 0


def test_bf16_rows_that_the_row_entries_refuse(capi):
    """Rows off the boundaries that the bf16 entries read on; rows without values are nothing to do."""
    L = capi.lib
    for fn, args, error, text in ((L.lsg_moe_unpermute, (P + 2, P, P, 4, 2, 64, P, None), RuntimeError, "4-byte"),
                                  (L.lsg_moe_unpermute, (P, P, P, 4, 2, 6, P + 2, None), RuntimeError, "4-byte"),
                                  (L.lsg_moe_unpermute, (P, P, P, 4, 2, -2, P, None), ValueError, "negative"),
                                  (L.lsg_moe_permute, (P + 8, P, 8, 2, 64, P, None), RuntimeError, "16-byte"),
                                  (L.lsg_moe_permute, (P, P, 8, 2, -8, P, None), ValueError, "negative")):
        with pytest.raises(error, match=text):
            capi.check(fn(*args))
    assert L.lsg_moe_permute(P, P, 8, 2, 0, P, None) == 0 and L.lsg_moe_unpermute(P, P, P, 4, 2, 0, P, None) == 0


def test_row_operators_refuse_cpu_tensors(capi):
    import torch
    from layerstormgemmkernels_b200 import ops
    inv, w = torch.zeros(8, dtype=torch.int32), torch.ones(4, 2)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        for bad in (lambda: ops.moe_permute(torch.zeros(4, 64, dtype=dtype), inv, 2),
                    lambda: ops.moe_unpermute(torch.zeros(8, 64, dtype=dtype), inv, w)):
            with pytest.raises(RuntimeError, match="rows must be contiguous BF16"):
                bad()
