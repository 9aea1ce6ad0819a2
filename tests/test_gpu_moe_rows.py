"""GPU tests of the ways of rows to the experts and back: what the combination rounds, and rows that start
anywhere.

Tolerances, with u = 2^-24: a sum of k products in fp32 is off by at most (k + 1) u times the sum of the
magnitudes, and storing it adds half a step of the type (bf16 2^-8, fp16 2^-11 of the value; fp16 below
its normal range 2^-25)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
HALF_STEP = {BF16: 2.0 ** -8, FP16: 2.0 ** -11, FP32: U}
NAME = {BF16: "bf16", FP16: "fp16", FP32: "fp32"}


@pytest.fixture(scope="module")
def ops():
    from layerstormgemmkernels_b200 import ops as _ops
    return _ops


def routed(ops, T, E, k, seed):
    g = torch.Generator().manual_seed(seed)
    idx, w = ops.moe_route(torch.randn(T, E, generator=g).cuda(), k)
    if T > 4:
        idx[1] = -1                      # a token that no expert takes
        idx[2, 0] = E                    # an expert that is not there
    offs, perm, inv = ops.moe_permutation(idx, E)
    return g, w, offs, perm, inv


def check_sum(out, y, inv, w):
    iv, (T, k) = inv.cpu().long().view(w.shape), w.shape
    part = torch.where((iv >= 0).unsqueeze(-1), y.cpu().double()[iv.clamp_min(0)], torch.zeros(1, dtype=torch.float64))
    part = part * w.cpu().double().unsqueeze(-1)
    want = part.sum(1)
    tol = (k + 1) * U * part.abs().sum(1) * (1 + 2.0 ** -7) + HALF_STEP[out.dtype] * want.abs() + (2.0 ** -25 if out.dtype == FP16 else 0)
    assert bool(((out.cpu().double() - want).abs() <= tol).all())


# -----------------------------------------------------------------------------------------
# One rounding from fp32 rows to a 16-bit output
# -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("to", [BF16, FP16])
@pytest.mark.parametrize("T,E,k,H", [(1, 4, 1, 4), (1, 128, 8, 2048), (5, 4, 4, 33), (7, 6, 3, 1), (33, 60, 4, 1001), (130, 8, 2, 4096),
                                     (64, 16, 16, 260), (2100, 16, 6, 512)])
def test_fp32_rows_leave_with_one_rounding(ops, T, E, k, H, to):
    """The fp32 combination's bits, rounded once; rows that start 4 bytes off too."""
    g, w, offs, perm, inv = routed(ops, T, E, k, T + H)
    flat = torch.randn(T * k * H + 1, generator=g).cuda()
    for y in (flat[:-1].view(T * k, H), flat[1:].view(T * k, H)):
        out = ops.moe_unpermute(y, inv, w, NAME[to])
        assert out.dtype == to and torch.equal(out, ops.moe_unpermute(y, inv, w).to(to))
        check_sum(out, y, inv, w)
        assert torch.equal(ops.moe_unpermute(y, inv, w, "fp32"), ops.moe_unpermute(y, inv, w))


def test_experts_rows_in_fp32(ops):
    """Experts' rows in fp32 and a bf16 output: off by one rounding, at most half a step of bf16, from the
    combination in 64 bits of the rows that the block formed."""
    g = torch.Generator().manual_seed(3)
    T, E, k, H, I = 50, 8, 2, 512, 256
    hidden = torch.randn(T, H, generator=g).to(BF16).cuda()
    gate_up, gus = ops.weight_int8_quant((torch.randn(E, 2 * I, H, generator=g) * 0.05).to(BF16).cuda())
    down, ds = ops.weight_int8_quant((torch.randn(E, H, I, generator=g) * 0.05).to(BF16).cuda())
    idx, w = ops.moe_route(torch.randn(T, E, generator=g).cuda(), k)
    offs, _, inv = ops.moe_permutation(idx, E)
    rows = ops.int8_moe_ffn(hidden, offs, inv, k, gate_up, gus, down, ds, "fp32")
    check_sum(ops.moe_unpermute(rows, inv, w, "bf16"), rows, inv, w)


def test_output_types_that_are_refused(ops):
    y, inv, w = torch.randn(8, 16, device="cuda"), torch.arange(8, dtype=torch.int32, device="cuda"), torch.ones(4, 2, device="cuda")
    for bad in (lambda: ops.moe_unpermute(y.half(), inv, w, "bf16"), lambda: ops.moe_unpermute(y.bfloat16(), inv, w, "fp32"),
                lambda: ops.moe_unpermute(y, inv, w, "int8")):
        with pytest.raises(RuntimeError):
            bad()


# -----------------------------------------------------------------------------------------
# Rows of every type from any address; what no type takes
# -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("T,E,k,H", [(1, 4, 1, 2), (5, 4, 4, 34), (33, 60, 4, 1002), (40, 8, 2, 2048), (17, 30, 12, 264)])
def test_rows_from_any_address(ops, T, E, k, H, dtype):
    """Rows that start one to eight values off an aligned buffer give the bits of an aligned copy."""
    g, w, offs, perm, inv = routed(ops, T, E, k, T + H)
    xs, ys = torch.randn(T * H + 8, generator=g).to(dtype).cuda(), torch.randn(T * k * H + 8, generator=g).to(dtype).cuda()
    for off in (0, 1, 2, 3, 4, 8):
        x, y = xs[off:off + T * H].view(T, H), ys[off:off + T * k * H].view(T * k, H)
        n = int(offs[-1])
        assert torch.equal(ops.moe_permute(x, perm, k)[:n], x[(perm[:n] // k).long()])
        out = ops.moe_unpermute(y, inv, w)
        assert torch.equal(out, ops.moe_unpermute(y.clone(), inv, w))
        check_sum(out, y, inv, w)
        assert torch.equal(out, ops.moe_unpermute(y, inv.view(T, k), w))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_rows_without_values_or_tokens(ops, dtype):
    perm, w = torch.arange(6, dtype=torch.int32, device="cuda"), torch.ones(3, 2, device="cuda")
    assert ops.moe_permute(torch.zeros(3, 0, dtype=dtype, device="cuda"), perm, 2).shape == (6, 0)
    assert ops.moe_unpermute(torch.zeros(6, 0, dtype=dtype, device="cuda"), perm, w).shape == (3, 0)
    assert ops.moe_permute(torch.zeros(0, 8, dtype=dtype, device="cuda"), perm[:0], 2).shape == (0, 8)
    assert ops.moe_unpermute(torch.zeros(0, 8, dtype=dtype, device="cuda"), perm[:0], w[:0]).shape == (0, 8)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_rows_refused(ops, dtype):
    """Every type alike: layouts, index and weight types and sizes that the kernels do not read."""
    x, y = torch.zeros(4, 16, dtype=dtype, device="cuda"), torch.zeros(8, 16, dtype=dtype, device="cuda")
    inv, w = torch.arange(8, dtype=torch.int32, device="cuda"), torch.ones(4, 2, device="cuda")
    for bad in (lambda: ops.moe_permute(x.t(), inv, 2), lambda: ops.moe_permute(x[:, :8], inv, 2), lambda: ops.moe_permute(x, inv.long(), 2),
                lambda: ops.moe_permute(x, inv.cpu(), 2), lambda: ops.moe_permute(x, inv[::2], 2),
                lambda: ops.moe_unpermute(y.t(), inv, w), lambda: ops.moe_unpermute(y[:, :8], inv, w),
                lambda: ops.moe_unpermute(y, inv.long(), w), lambda: ops.moe_unpermute(y, inv[:7], w),
                lambda: ops.moe_unpermute(y, inv, w.half()), lambda: ops.moe_unpermute(y, inv, w.to(dtype).double()),
                lambda: ops.moe_unpermute(y, inv, torch.ones(2, 4, device="cuda").t()), lambda: ops.moe_unpermute(y, inv.cpu(), w),
                lambda: ops.moe_unpermute(y, inv, w.cpu())):
        with pytest.raises(RuntimeError, match="must be"):
            bad()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("T,k,H", [(1, 1, 2), (6, 4, 34), (9, 8, 2048), (40, 12, 264), (5, 3, 33)])
def test_indices_outside_the_rows(ops, T, k, H, dtype):
    """An index that names no row, or no token's pair, on either side: such a pair adds nothing, such a row
    is not written."""
    g = torch.Generator().manual_seed(T * k + H)
    rows = T * k - (1 if T > 1 else 0)                      # y one row short of the pairs
    inv = torch.randperm(T * k, generator=g).int()
    far = torch.tensor([rows, rows + 1, 2 ** 31 - 1, 2 ** 30, -1, -2 ** 31], dtype=torch.int64).int()
    inv[::3] = far[torch.arange(len(inv[::3])) % 6]
    w = torch.rand(T, k, generator=g) + 0.1
    y = torch.randn(rows, H, generator=g).to(dtype)
    out = ops.moe_unpermute(y.cuda(), inv.cuda(), w.cuda())
    check_sum(out, y, torch.where((inv >= 0) & (inv < rows), inv, torch.full_like(inv, -1)), w)
    x = torch.randn(T, H, generator=g).to(dtype)
    perm = torch.arange(T * k, dtype=torch.int32)
    perm[::2] = torch.tensor([T * k, T * k + 7, 2 ** 31 - 1, -1, -k, -2 ** 31], dtype=torch.int64).int()[torch.arange(len(perm[::2])) % 6]
    good = (perm >= 0) & (perm < T * k)
    got = ops.moe_permute(x.cuda(), perm.cuda(), k).cpu()
    assert torch.equal(got[good], x[(perm[good] // k).long()])


def test_more_than_sixteen_slots(ops):
    """bf16 rows in pairs have any number of slots; other rows at most 16 on the way back."""
    g = torch.Generator().manual_seed(1)
    T, k, H = 7, 20, 66
    inv, w = torch.randperm(T * k, generator=g).int().cuda(), torch.rand(T, k, generator=g).cuda()
    y = torch.randn(T * k, H, generator=g)
    check_sum(ops.moe_unpermute(y.to(BF16).cuda(), inv, w), y.to(BF16), inv, w)
    x = torch.randn(T, H, generator=g).cuda()
    for dtype in (BF16, FP16, FP32):
        assert torch.equal(ops.moe_permute(x.to(dtype), inv, k), x.to(dtype)[(inv // k).long()])
    for bad in (y.cuda(), y.half().cuda(), y[:, 1:].to(BF16).contiguous().cuda()):
        with pytest.raises(ValueError, match="top_k"):
            ops.moe_unpermute(bad, inv, w)
