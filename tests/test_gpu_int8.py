"""GPU tests of the 8-bit integer family against its definition in 64 bits: the per-row quantizers
(codes and scales exact), the dense and grouped products, the expert block, views, graphs and streams.

Tolerances: a code of dynamic_int8_quant is a whole number fixed by the definition, so equal.  A
product is an exact int32 sum (exact in float64 too) and three fp32 roundings (2^-24 each) and the
output's own rounding (bf16 2^-8, fp16 2^-11, half of torch.finfo(t).eps)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 0.0}


@pytest.fixture(scope="module")
def ops():
    from layerstormgemmkernels_b200 import ops as _ops
    return _ops


def ref_codes(x):
    """The definition with whole-number quotients: 127 x / a in float64, half-way cases to even (the
    float64 quotient of a bf16 or fp16 pair is never rounded onto or across a half-way point)."""
    x = x.double()
    a = x.abs().amax(-1, keepdim=True)
    q = torch.where(a > 0, (x * 127.0 / a), torch.zeros_like(x)).round()
    return q, (a.squeeze(-1).float() / 127.0)


def check_product(D, acc, sa, sb, kind):
    ref = acc * sa.double().unsqueeze(1) * sb.double().unsqueeze(0)
    err = (D.double() - ref).abs()
    tol = (HALF_STEP[kind] + 4 * 2.0 ** -24) * ref.abs() + (2.0 ** -24 if kind == "fp16" else 0.0)
    assert bool((err <= tol).all()), float((err - tol).max())


def rand_codes(g, rows, K):
    w = torch.randint(-127, 128, (rows, (K + 15) // 16 * 16), generator=g, dtype=torch.int8)
    return w.cuda()[:, :K]


# -----------------------------------------------------------------------------------------
# Quantizers
# -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("M,K", [(1, 1), (3, 7), (5, 8), (1, 16), (2, 100), (7, 2048), (3, 2056), (4, 4096), (33, 8200),
                                 (2, 14336), (2, 16384), (2, 16392), (1, 40000), (300, 768)])
def test_dynamic_quant(ops, dtype, M, K):
    g = torch.Generator().manual_seed(M * K)
    x = torch.randn(M, K, generator=g).to(dtype)
    codes, scales = ops.dynamic_int8_quant(x.cuda())
    q, s = ref_codes(x)
    assert codes.shape == (M, K) and codes.dtype == torch.int8 and (M == 1 or codes.stride(0) % 16 == 0)
    assert torch.equal(codes.cpu().double(), q)
    assert torch.equal(scales.cpu(), s)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_dynamic_quant_half_way_and_extremes(ops, dtype):
    """Every half-way quotient of a row whose maximum is 127 or 254, x = a / 2 (63.5), all powers of two
    as the maximum, the smallest subnormals, the largest finite values, zeros, negative zeros."""
    rows = []
    half = torch.arange(-253, 254, dtype=torch.float64) / 2
    for top in (127.0, 254.0, 127.0 * 2.0 ** -10):
        r = torch.zeros(1024, dtype=torch.float64)
        r[:507] = half * top / 127.0
        r[600] = top
        rows.append(r)
    lo, hi = (-133, 127) if dtype == BF16 else (-24, 15)
    g = torch.Generator().manual_seed(3)
    for e in range(lo, hi + 1, 4):
        m = 1.0 + torch.randint(0, 128, (1,), generator=g).item() / 128
        a = m * 2.0 ** e
        r = torch.rand(1024, generator=g, dtype=torch.float64).mul(2).sub(1) * a
        r[0], r[1], r[2] = a, -a / 2, a / 2
        rows.append(r)
    big = torch.finfo(dtype).max
    rows.append(torch.linspace(-big, big, 1024, dtype=torch.float64))
    rows.append(torch.zeros(1024, dtype=torch.float64))
    rows.append(torch.full((1024,), -0.0, dtype=torch.float64))
    x = torch.stack(rows).to(dtype)
    for v in (x, x[:, :1000], x[:, 1:1000]):     # whole pieces, a shorter row, an odd start
        codes, scales = ops.dynamic_int8_quant(v.cuda() if v is x else x.cuda()[:, v.storage_offset():][:, :v.size(1)])
        q, s = ref_codes(v)
        assert torch.equal(codes.cpu().double(), q)
        assert torch.equal(scales.cpu(), s)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("K", [1000, 1001])
def test_dynamic_quant_not_finite(ops, bad, K):
    x = torch.randn(4, K, generator=torch.Generator().manual_seed(1)).to(BF16)
    x[1, 17] = bad
    x[2, K - 1] = bad
    codes, scales = ops.dynamic_int8_quant(x.cuda())
    q, s = ref_codes(x[[0, 3]])
    assert torch.equal(codes.cpu()[[0, 3]].double(), q) and torch.equal(scales.cpu()[[0, 3]], s)
    assert bool(scales.cpu()[1:3].isnan().all()) and not bool(codes.cpu()[1:3].any())
    w = rand_codes(torch.Generator().manual_seed(2), 24, K)
    D = ops.int8_gemm(codes, w, scales, torch.ones(24, device="cuda"), 4, 24, K, "bf16").cpu()
    assert bool(D[1:3].isnan().all()) and bool(D[[0, 3]].isfinite().all())


def test_dynamic_quant_views_and_empty(ops):
    base = torch.randn(20, 600, generator=torch.Generator().manual_seed(5)).to(BF16).cuda()
    for v in (base[::2], base[:, 100:356], base[3:4, 7:300], base[:, 3:203], base[::3, 64:]):
        codes, scales = ops.dynamic_int8_quant(v)
        q, s = ref_codes(v.cpu())
        assert torch.equal(codes.cpu().double(), q) and torch.equal(scales.cpu(), s)
    codes, scales = ops.dynamic_int8_quant(base[:0])
    assert codes.shape == (0, 600) and scales.shape == (0,)
    codes, scales = ops.dynamic_int8_quant(base[:, :0])
    assert codes.shape == (20, 0) and not bool(scales.any())


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_weight_quant(ops, dtype):
    g = torch.Generator().manual_seed(8)
    w = (torch.randn(3, 40, 96, generator=g) * 0.02).to(dtype)
    q, s = ref_codes(w.view(120, 96))
    codes, scales = ops.weight_int8_quant(w.cuda())
    assert torch.equal(codes.cpu().double().view(120, 96), q) and torch.equal(scales.cpu().view(120), s)
    codes, scales = ops.weight_int8_quant(w[1].contiguous().cuda())
    assert torch.equal(codes.cpu().double(), q[40:80]) and torch.equal(scales.cpu(), s[40:80])


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("M,K", [(1, 16), (3, 77), (9, 768), (5, 2056), (4, 14336), (2, 16400)])
def test_silu_mul_quant(ops, dtype, M, K):
    """silu(g) * u in fp32 is at most 2^-20 (relative) off: expf and the quotient two ulp each, an addition
    and a product half an ulp, 5 * 2^-23.  A code is the nearest integer to a quotient of at most 127
    with the errors of value and maximum, so |code - quotient| <= 0.5 + 127 * 2^-19."""
    g = torch.Generator().manual_seed(M + K)
    both = (torch.randn(M, 2 * K, generator=g) * 2).to(dtype)
    gate, up = both[:, :K], both[:, K:]
    h = gate.double() * torch.sigmoid(gate.double()) * up.double()
    a = h.abs().amax(1)
    dev = both.cuda()
    for gt, ut in ((gate.contiguous().cuda(), up.contiguous().cuda()), (dev[:, :K], dev[:, K:])):
        codes, scales = ops.silu_mul_int8_quant(gt, ut)
        assert bool(((scales.cpu().double() - a / 127).abs() <= a / 127 * 2.0 ** -19).all())
        off = (codes.cpu().double() - h * 127 / a.unsqueeze(1)).abs().max()
        assert off <= 0.5 + 127 * 2.0 ** -19, off


def test_silu_mul_far_gates(ops):
    """Gates whose exponential overflows or vanishes: silu(-100) u and silu(100) u; an infinite row."""
    gate = torch.tensor([[-100.0, -1000.0, 100.0, 3.0] * 8, [-100.0, -200.0, -90.0, -80.0] * 8, [math.inf, 1, 1, 1] * 8])
    up = torch.ones_like(gate)
    codes, scales = ops.silu_mul_int8_quant(gate.to(BF16).cuda(), up.to(BF16).cuda())
    codes, scales = codes.cpu(), scales.cpu()
    assert codes[0, :4].tolist() == [0, 0, 127, 4]       # 3 sigmoid(3) * 1.27 = 3.63
    assert float(scales[0]) == pytest.approx(100 / 127, rel=2.0 ** -19)
    assert codes[1, 3] == -127 and bool(scales[2].isnan()) and not bool(codes[2].any())


# -----------------------------------------------------------------------------------------
# Products
# -----------------------------------------------------------------------------------------
DENSE = [(1, 1, 1), (1, 7, 16), (1, 128, 4096), (2, 1000, 1008), (3, 257, 333), (4, 64, 64), (3, 40, 1), (9, 17, 7), (20, 300, 15), (260, 9500, 40), (5, 129, 2048), (8, 1024, 14336),
         (9, 300, 4096), (16, 515, 1040), (17, 4099, 512), (31, 128, 144), (33, 96, 4000), (64, 640, 2064), (65, 1, 4096),
         (77, 2048, 7168), (127, 255, 100), (128, 256, 128), (129, 257, 2304), (200, 3000, 1024), (256, 512, 4096),
         (257, 1025, 513), (300, 4096, 1024), (511, 130, 2000), (1000, 777, 1552), (1024, 2048, 2048),
         (300, 9601, 136), (513, 4099, 400), (1001, 4352, 1040), (1500, 6000, 2320)]      # CTA pairs


@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("M,N,K", DENSE)
def test_gemm(ops, M, N, K, kind):
    g = torch.Generator().manual_seed(M + 3 * N + 7 * K)
    A, B = rand_codes(g, M, K), rand_codes(g, N, K)
    top = 1.0 / (127.0 * math.sqrt(K))
    sa = (torch.rand(M, generator=g) + 0.1).cuda() * top
    sb = (torch.rand(N, generator=g) + 0.1).cuda() / 64
    D = ops.int8_gemm(A, B, sa, sb, M, N, K, kind)
    acc = A.double() @ B.double().t()
    check_product(D, acc, sa, sb, kind)


# Sizes whose estimates choose tiles of 16 to 256 tokens, in single CTAs, in pairs and with K cut among two,
# four and eight CTAs; the rows and channels end inside a tile.
FORMS = [(15, 14337, 272), (16, 6000, 2048), (18, 13, 2050), (19, 2001, 2064), (17, 6003, 4096), (20, 130, 30), (31, 14336, 48),
         (45, 1008, 4100), (33, 4099, 4096), (47, 14333, 528), (49, 14336, 1040), (63, 14335, 2048), (79, 14336, 520),
         (81, 14339, 528), (95, 14336, 1040), (99, 2005, 4096), (97, 14336, 530), (113, 14337, 1056), (130, 2000, 4090),
         (129, 14336, 528), (161, 2003, 4096), (190, 14331, 528), (223, 14336, 544), (250, 14336, 513), (1780, 130, 4096),
         (3001, 129, 2048), (2100, 600, 144)]


@pytest.mark.parametrize("M,N,K", FORMS)
def test_gemm_forms_of_tiles(ops, M, N, K):
    g = torch.Generator().manual_seed(M + N + K)
    A, B = rand_codes(g, M, K), rand_codes(g, N, K)
    sa, sb = (torch.rand(M, generator=g) + 0.1).cuda(), (torch.rand(N, generator=g) + 0.1).cuda()
    D = ops.int8_gemm(A, B, sa, sb, M, N, K, "fp32")
    check_product(D, A.double() @ B.double().t(), sa, sb, "fp32")


@pytest.mark.parametrize("M", [1, 4, 16, 40, 300])
def test_gemm_extreme_codes_and_longest_k(ops, M):
    """-128 in every place at the longest K: sums of 128 * 128 * 131056 = 2^31 - 2^18."""
    K, N = 131056, 130
    A = torch.full((M, K), -128, dtype=torch.int8, device="cuda")
    B = torch.full((N, K), -128, dtype=torch.int8, device="cuda")
    B[1] = 127
    B[2] = 0
    one = torch.ones(M, device="cuda")
    D = ops.int8_gemm(A, B, one, torch.ones(N, device="cuda"), M, N, K, "fp32")
    want = torch.full((N,), float(128 * 128 * K), dtype=torch.float64)
    want[1], want[2] = -128.0 * 127 * K, 0.0
    assert torch.equal(D.cpu().double(), want.float().double().expand(M, N))


@pytest.mark.parametrize("M", [1, 3, 20, 150])
def test_gemm_views_and_what_lies_behind_k(ops, M):
    """Rows further apart than K; bytes behind K must not count."""
    g = torch.Generator().manual_seed(M)
    K, N = 1003, 200
    A = torch.randint(-128, 128, (2 * M, 1056), generator=g, dtype=torch.int8).cuda()[::2, 16:16 + K]
    B = torch.randint(-128, 128, (N, 1024), generator=g, dtype=torch.int8).cuda()[:, :K]
    sa, sb = torch.rand(M, generator=g).cuda(), torch.rand(N, generator=g).cuda()
    check_product(ops.int8_gemm(A, B, sa, sb, M, N, K, "fp32"), A.double() @ B.double().t(), sa, sb, "fp32")


@pytest.mark.parametrize("M", [0, 1, 8, 40, 200])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_gemm_from_bf16_is_the_two_calls(ops, M, dtype):
    g = torch.Generator().manual_seed(M)
    N, K = 300, 2000
    x = torch.randn(M, 2 * K, generator=g).to(dtype).cuda()
    w, ws = ops.weight_int8_quant((torch.randn(N, K, generator=g) * 0.02).to(BF16).cuda())
    for v in (x[:, :K].contiguous(), x[:, :K], x[:, 3:3 + K]):
        for kind in ("bf16", "fp16", "fp32"):
            got = ops.int8_gemm_from_bf16(v, w, ws, kind)
            codes, scales = ops.dynamic_int8_quant(v)
            assert torch.equal(got, ops.int8_gemm(codes, w, scales, ws, M, N, K, kind))


def test_gemm_from_bf16_rows_not_finite_and_zero(ops):
    x = torch.randn(3, 512, generator=torch.Generator().manual_seed(2)).to(BF16).cuda()
    x[0] = 0
    x[1, 5] = math.inf
    w = rand_codes(torch.Generator().manual_seed(2), 40, 512)
    D = ops.int8_gemm_from_bf16(x, w, torch.ones(40, device="cuda"))
    assert not bool(D[0].any()) and bool(D[1].isnan().all()) and bool(D[2].isfinite().all())


# -----------------------------------------------------------------------------------------
# Rows grouped by expert
# -----------------------------------------------------------------------------------------
def offsets_of(counts):
    o = torch.zeros(len(counts) + 1, dtype=torch.int32)
    o[1:] = torch.tensor(counts, dtype=torch.int32).cumsum(0)
    return o


GROUPS = [[1], [0], [3, 0, 0, 5], [0, 0, 9], [8, 8, 8], [1] * 40, [130, 0, 1, 257, 64], [0] * 33 + [17], [300, 2],
          [16, 17, 31, 32, 33, 0, 127, 128, 129], [2, 1, 0, 0, 7] * 13, [700, 1, 0, 1300], [257, 900, 600]]


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("counts", GROUPS, ids=lambda c: f"{len(c)}x{sum(c)}")
@pytest.mark.parametrize("N,K", [(192, 256), (77, 1040), (3600, 80)])
def test_grouped_gemm(ops, counts, N, K, kind):
    E, used = len(counts), sum(counts)
    T = used + 5                                # rows behind the last expert's stay as they are
    g = torch.Generator().manual_seed(used + N)
    A = rand_codes(g, T, K)
    B = torch.randint(-127, 128, (E, N, K), generator=g, dtype=torch.int8).cuda()
    sa, sb = torch.rand(T, generator=g).cuda(), torch.rand(E, N, generator=g).cuda()
    offs = offsets_of(counts)
    D = torch.full((T, N), 7.0, dtype={"bf16": BF16, "fp32": FP32}[kind], device="cuda")
    assert ops.int8_grouped_gemm(A, B, D, sa, sb, offs.cuda(), N, K, kind) is D
    assert bool((D[used:] == 7.0).all())
    for e in range(E):
        a, b = int(offs[e]), int(offs[e + 1])
        check_product(D[a:b], A[a:b].double() @ B[e].double().t(), sa[a:b], sb[e], kind)


def test_grouped_offsets_past_the_rows(ops):
    """Offsets that run past the caller's rows are taken as the row count."""
    g = torch.Generator().manual_seed(4)
    A, B = rand_codes(g, 40, 128), torch.randint(-127, 128, (3, 64, 128), generator=g, dtype=torch.int8).cuda()
    one, sb = torch.ones(40, device="cuda"), torch.ones(3, 64, device="cuda")
    D = torch.zeros(40, 64, device="cuda")
    ops.int8_grouped_gemm(A, B, D, one, sb, torch.tensor([0, 10, 50, 60], dtype=torch.int32, device="cuda"), 64, 128, "fp32")
    assert torch.equal(D[:10].double(), A[:10].double() @ B[0].double().t())
    assert torch.equal(D[10:].double(), A[10:].double() @ B[1].double().t())


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("T,E,k,H", [(1, 8, 2, 64), (5, 4, 4, 100), (33, 60, 4, 2048), (300, 128, 8, 520), (7, 3, 1, 33)])
def test_permute_int8(ops, T, E, k, H, dtype):
    g = torch.Generator().manual_seed(T + H)
    idx = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).int().cuda()
    if T > 3:
        idx[1] = -1                              # a token without a row
        idx[2, 0] = E                            # and a pair without one
    offs, perm, inv = ops.moe_permutation(idx, E)
    hidden = torch.randn(T, H, generator=g).to(dtype).cuda()
    codes, scales = ops.moe_permute_int8(hidden, inv, k)
    used = int(offs[-1])
    q, s = ref_codes(hidden.cpu())
    token = (perm[:used].cpu() // k).long()
    assert torch.equal(codes.cpu()[:used].double(), q[token]) and torch.equal(scales.cpu()[:used], s[token])
    assert used == int(((idx >= 0) & (idx < E)).sum())


def experts(g, E, H, I):
    gate_up = torch.randint(-127, 128, (E, 2 * I, H), generator=g, dtype=torch.int8).cuda()
    down = torch.randint(-127, 128, (E, H, I), generator=g, dtype=torch.int8).cuda()
    gus = ((torch.rand(E, 2 * I, generator=g) + 0.5) * 0.02 / 70).cuda()
    ds = ((torch.rand(E, H, generator=g) + 0.5) * 0.02 / 70).cuda()
    return gate_up, gus, down, ds


@pytest.mark.parametrize("T,E,k,H,I", [(1, 8, 2, 64, 32), (1, 128, 8, 256, 96), (9, 4, 4, 512, 144), (40, 16, 4, 128, 256),
                                       (64, 128, 8, 256, 192), (200, 8, 2, 1024, 528), (700, 8, 2, 256, 128),
                                       (3, 2, 1, 2048, 768), (129, 3, 3, 48, 272), (600, 3, 2, 144, 1600)])
@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_moe_ffn(ops, T, E, k, H, I, kind):
    """Route, sort, experts, combine: the block gives the bits of its four steps, and the steps are
    right by the tests above; the whole is compared with 64 bits by norm: fp32 values that differ by
    2^-20 change a code for at most one value in 127 * 2^-19 of them, so next to nothing beside the
    output's rounding."""
    g = torch.Generator().manual_seed(T + I)
    hidden = torch.randn(T, H, generator=g).to(BF16).cuda()
    gate_up, gus, down, ds = experts(g, E, H, I)
    idx, w = ops.moe_route(torch.randn(T, E, generator=g).cuda(), k)
    if T > 3:
        idx[2, 0] = -1
        idx[3] = E
    offs, perm, inv = ops.moe_permutation(idx, E)
    used = int(offs[-1])
    rows = ops.int8_moe_ffn(hidden, offs, inv, k, gate_up, gus, down, ds, kind)

    codes, scales = ops.moe_permute_int8(hidden, inv, k)
    gu = torch.zeros(T * k, 2 * I, device="cuda")
    ops.int8_grouped_gemm(codes, gate_up, gu, scales, gus, offs, 2 * I, H, "fp32")
    act, act_scales = ops.silu_mul_int8_quant(gu[:, :I], gu[:, I:])
    D = torch.zeros_like(rows)
    ops.int8_grouped_gemm(act, down, D, act_scales, ds, offs, H, I, kind)
    assert torch.equal(rows[:used], D[:used])

    out = ops.moe_unpermute(rows, inv, w)
    q, s = ref_codes(hidden.cpu())
    want = torch.zeros(T, H, dtype=torch.float64)
    for t in range(T):
        for j in range(k):
            e = int(idx[t, j])
            if e < 0 or e >= E:
                continue
            p = (gate_up[e].cpu().double() @ q[t]) * s[t].double() * gus[e].cpu().double()
            h = p[:I] * torch.sigmoid(p[:I]) * p[I:]
            a = h.abs().max()
            want[t] += float(w[t, j]) * (down[e].cpu().double() @ (h * 127 / a).round()) * (a / 127) * ds[e].cpu().double()
    rel = float((out.cpu().double() - want).norm() / want.norm())
    # bf16 rows and output: two roundings of 2^-8 at most; a row in fp32 leaves what codes and sums move
    assert rel <= (2 * 2.0 ** -8 if kind == "bf16" else 2.0 ** -10), rel
    if T > 3:
        assert not bool(out[3].any())


def four_steps(ops, hidden, offs, inv, k, gate_up, gus, down, ds, kind, fill):
    """int8_moe_ffn from its four public steps; rows without an expert hold `fill`."""
    rows, I, H = hidden.size(0) * k, down.size(2), hidden.size(1)
    codes, scales = ops.moe_permute_int8(hidden, inv, k)
    gu = torch.zeros(rows, 2 * I, device="cuda")
    ops.int8_grouped_gemm(codes, gate_up, gu, scales, gus, offs, 2 * I, H, "fp32")
    act, act_scales = ops.silu_mul_int8_quant(gu[:, :I], gu[:, I:])
    D = torch.full((rows, H), fill, device="cuda", dtype={"bf16": BF16, "fp16": FP16, "fp32": FP32}[kind])
    return ops.int8_grouped_gemm(act, down, D, act_scales, ds, offs, H, I, kind)


@pytest.mark.parametrize("kind,dtype", [("bf16", BF16), ("fp16", FP16), ("fp32", BF16)])
@pytest.mark.parametrize("T,E,k,H,I", [(1, 1, 1, 16, 16), (1, 3, 1, 1040, 16), (1, 128, 8, 2048, 768), (1, 7, 3, 48, 5456),
                                       (2, 5, 4, 528, 1040), (3, 4, 2, 1024, 2032), (4, 1024, 2, 272, 512), (8, 6, 1, 2048, 2048),
                                       (1, 4, 2, 16384, 48), (7, 2, 1, 16, 1024), (2, 300, 4, 1008, 80), (8, 2, 1, 2064, 16),
                                       (9, 4, 1, 64, 64), (1, 9, 8, 64, 2064)])
def test_moe_ffn_few_rows(ops, T, E, k, H, I, kind, dtype):
    """Up to eight rows, on both sides of the sizes that the streaming form takes: the bits of the four
    steps, from hidden rows that start on any 2 bytes, with an infinite and a zero token among them, and
    again (a fresh run changes nothing)."""
    g = torch.Generator().manual_seed(T + E + H + I)
    base = torch.randn(T + 2, H + 7, generator=g).to(dtype).cuda()
    hidden = base[1:T + 1, 3:H + 3]
    if T > 3:
        hidden[1, H // 2] = math.inf
        hidden[2] = 0
    gate_up, gus, down, ds = experts(g, E, H, I)
    idx = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).int().cuda()
    for at in (hidden, hidden.contiguous()):
        offs, perm, inv = ops.moe_permutation(idx, E)
        rows = ops.int8_moe_ffn(at, offs, inv, k, gate_up, gus, down, ds, kind)
        D = four_steps(ops, at, offs, inv, k, gate_up, gus, down, ds, kind, 0.0)
        used = int(offs[-1])
        assert used == T * k and torch.equal(rows.nan_to_num(7.0, 8.0, 9.0), D.nan_to_num(7.0, 8.0, 9.0))
        assert bool(rows.isnan().any()) == (T > 3)
        assert torch.equal(rows.nan_to_num(7.0), ops.int8_moe_ffn(at, offs, inv, k, gate_up, gus, down, ds, kind).nan_to_num(7.0))


@pytest.mark.parametrize("gone", [(), (0,), (1, 3), (0, 1, 2, 3)])
def test_moe_ffn_few_rows_without_an_expert(ops, gone):
    """Pairs that no expert here takes (padding, another rank's) leave the rows behind the last one out;
    the combination skips them."""
    g = torch.Generator().manual_seed(5)
    T, E, k, H, I = 4, 6, 2, 256, 96
    hidden = torch.randn(T, H, generator=g).to(BF16).cuda()
    gate_up, gus, down, ds = experts(g, E, H, I)
    idx, w = ops.moe_route(torch.randn(T, E, generator=g).cuda(), k)
    whole_offs, _, whole_inv = ops.moe_permutation(idx, E)
    whole = ops.moe_unpermute(ops.int8_moe_ffn(hidden, whole_offs, whole_inv, k, gate_up, gus, down, ds), whole_inv, w)
    for t in gone:
        idx[t] = E if t % 2 else -1
    offs, perm, inv = ops.moe_permutation(idx, E)
    rows = ops.int8_moe_ffn(hidden, offs, inv, k, gate_up, gus, down, ds)
    out = ops.moe_unpermute(rows, inv, w)
    for t in range(T):
        if t in gone:
            assert not bool(out[t].any())
        else:
            assert torch.equal(out[t], whole[t])


def test_dense_and_grouped_agree(ops):
    """One expert with all rows is the dense product, bit for bit."""
    g = torch.Generator().manual_seed(11)
    for M in (1, 6, 30, 140):
        A, B = rand_codes(g, M, 768), rand_codes(g, 320, 768)
        sa, sb = torch.rand(M, generator=g).cuda(), torch.rand(320, generator=g).cuda()
        D = torch.empty(M, 320, device="cuda")
        ops.int8_grouped_gemm(A, B.view(1, 320, 768), D, sa, sb.view(1, 320), torch.tensor([0, M], dtype=torch.int32, device="cuda"),
                              320, 768, "fp32")
        assert torch.equal(D, ops.int8_gemm(A, B, sa, sb, M, 320, 768, "fp32"))


# -----------------------------------------------------------------------------------------
# Graphs and streams
# -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("T", [1, 24, 300])
def test_graph_replay_sees_new_inputs(ops, T):
    g = torch.Generator().manual_seed(T)
    E, k, H, I = 8, 2, 256, 128
    gate_up, gus, down, ds = experts(g, E, H, I)
    w, ws = ops.weight_int8_quant((torch.randn(400, H, generator=g) * 0.02).to(BF16).cuda())
    hidden = torch.randn(T, H, generator=g).to(BF16).cuda()
    logits = torch.randn(T, E, generator=g).cuda()

    def step():
        idx, wt = ops.moe_route(logits, k)
        offs, _, inv = ops.moe_permutation(idx, E)
        rows = ops.int8_moe_ffn(hidden, offs, inv, k, gate_up, gus, down, ds)
        return ops.moe_unpermute(rows, inv, wt), ops.int8_gemm_from_bf16(hidden, w, ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                           # two captured steps of the same inputs
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs))
    for round in range(2):
        hidden.copy_(torch.randn(T, H, generator=g).to(BF16))
        logits.copy_(torch.randn(T, E, generator=g))
        want = step()
        for graph, outs in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


@pytest.mark.parametrize("M", [2, 40, 500])
def test_two_streams_at_once(ops, M):
    g = torch.Generator().manual_seed(M)
    N, K = 1024, 2048
    w, ws = ops.weight_int8_quant((torch.randn(N, K, generator=g) * 0.02).to(BF16).cuda())
    xs = [torch.randn(M, K, generator=g).to(BF16).cuda() for _ in range(2)]
    want = [ops.int8_gemm_from_bf16(x, w, ws) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(ops.int8_gemm_from_bf16(xs[i], w, ws))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(d, want[i]) for d in got[i])


@pytest.mark.parametrize("M", [1, 2, 8, 60, 300])
def test_weights_made_right_before(ops, M):
    """The weight is quantized by the launch in front of the product, into memory that held the weight of
    the call before: nothing of the product may read it earlier than that launch has ended."""
    g = torch.Generator().manual_seed(M)
    N, K = 9600, 512
    x = torch.randn(M, K, generator=g).to(BF16).cuda()
    hidden_codes, hidden_scales = ops.dynamic_int8_quant(x)
    src = [(torch.randn(N, K, generator=g) * 0.02).to(BF16).cuda() for _ in range(3)]
    want = []
    for w in src:
        codes, scales = ops.weight_int8_quant(w)
        torch.cuda.synchronize()
        want.append(ops.int8_gemm_from_bf16(x, codes, scales))
        torch.cuda.synchronize()
        del codes, scales
    got = []
    for i in range(12):
        codes, scales = ops.weight_int8_quant(src[i % 3])
        got.append(ops.int8_gemm(hidden_codes, codes, hidden_scales, scales, M, N, K, "bf16"))
        codes, scales = ops.weight_int8_quant(src[i % 3])
        got.append(ops.int8_gemm_from_bf16(x, codes, scales))
        del codes, scales
    torch.cuda.synchronize()
    for i, d in enumerate(got):
        assert torch.equal(d, want[(i // 2) % 3]), i


@pytest.mark.parametrize("T,k", [(1, 8), (2, 4), (3, 2), (5, 2)])
def test_experts_one_layer_behind_the_other(ops, T, k):
    """Layers in one pair of weight buffers: offsets, scales and weights are written right in front of each
    call, whose result is the next one's input; with a wait between all launches every layer's bits are the same.
    (silu(g) * u is about quadratic in its input: without a norm the last layers' values fall below bf16's range, so
    what counts is the first ones'.)"""
    g = torch.Generator().manual_seed(T)
    E, H, I = 16, 1024, 512
    layers = [experts(g, E, H, I) for _ in range(3)]
    x = torch.randn(T, H, generator=g).to(BF16).cuda()
    logits = [torch.randn(T, E, generator=g).cuda() for _ in range(3)]
    now = [torch.empty_like(t) for t in layers[0]]

    def run(wait):
        h, every = x.clone(), []
        for n in range(9):
            idx, w = ops.moe_route(logits[(n + n // 3) % 3], k)
            offs, _, inv = ops.moe_permutation(idx, E)
            for t, src in zip(now, layers[n % 3]):
                t.copy_(src)
            wait()
            rows = ops.int8_moe_ffn(h, offs, inv, k, *now)
            wait()
            h = ops.moe_unpermute(rows, inv, w)
            wait()
            every += [rows, h]
        return every

    want = run(torch.cuda.synchronize)
    assert all(bool(d.isfinite().all()) for d in want) and all(bool(d.any()) for d in want[:6])
    for _ in range(4):
        assert all(torch.equal(a, b) for a, b in zip(run(lambda: None), want))


@pytest.mark.parametrize("T", [3, 400])
def test_experts_on_two_streams(ops, T):
    g = torch.Generator().manual_seed(T)
    E, k, H, I = 8, 2, 512, 256
    gate_up, gus, down, ds = experts(g, E, H, I)
    sets = []
    for _ in range(2):
        hidden = torch.randn(T, H, generator=g).to(BF16).cuda()
        idx, _ = ops.moe_route(torch.randn(T, E, generator=g).cuda(), k)
        offs, _, inv = ops.moe_permutation(idx, E)
        sets.append((hidden, offs, inv))
    want = [ops.int8_moe_ffn(h, o, i, k, gate_up, gus, down, ds) for h, o, i in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(10):
        for j, st in enumerate(streams):
            with torch.cuda.stream(st):
                h, o, i = sets[j]
                got[j].append(ops.int8_moe_ffn(h, o, i, k, gate_up, gus, down, ds))
    torch.cuda.synchronize()
    for j in range(2):
        assert all(torch.equal(d, want[j]) for d in got[j])


def test_offsets_that_fall(ops):
    """Offsets are taken as a rising sequence inside [0, T]: what falls or lies outside makes experts empty
    and never reaches past the rows."""
    g = torch.Generator().manual_seed(21)
    A, B = rand_codes(g, 64, 256), torch.randint(-127, 128, (4, 96, 256), generator=g, dtype=torch.int8).cuda()
    one, sb = torch.ones(64, device="cuda"), torch.ones(4, 96, device="cuda")
    D = torch.full((64, 96), -1.0, device="cuda")
    ops.int8_grouped_gemm(A, B, D, one, sb, torch.tensor([-3, 20, 5, 30, 1 << 30], dtype=torch.int32, device="cuda"), 96, 256, "fp32")
    for e, (a, b) in enumerate(((0, 20), (20, 20), (20, 30), (30, 64))):
        assert torch.equal(D[a:b].double(), A[a:b].double() @ B[e].double().t())


@pytest.mark.parametrize("E", [1, 300, 1024])
def test_many_experts(ops, E):
    g = torch.Generator().manual_seed(E)
    counts = torch.randint(0, 4, (E,), generator=g).tolist()
    counts[E // 2] = 37
    T, N, K = sum(counts), 64, 128
    A, B = rand_codes(g, T, K), torch.randint(-127, 128, (E, N, K), generator=g, dtype=torch.int8).cuda()
    sa, sb = torch.rand(T, generator=g).cuda(), torch.rand(E, N, generator=g).cuda()
    offs = offsets_of(counts)
    D = torch.empty(T, N, device="cuda")
    ops.int8_grouped_gemm(A, B, D, sa, sb, offs.cuda(), N, K, "fp32")
    expert = torch.repeat_interleave(torch.arange(E), torch.tensor(counts)).cuda()
    acc = torch.bmm(B[expert].double(), A.double().unsqueeze(-1)).squeeze(-1)
    ref = acc * sa.double().unsqueeze(1) * sb.double()[expert]
    assert bool(((D.double() - ref).abs() <= 4 * 2.0 ** -24 * ref.abs()).all())


def test_refused_on_cuda(ops):
    x = torch.randn(4, 64).to(BF16).cuda()
    w = torch.zeros(8, 64, dtype=torch.int8, device="cuda")
    one = torch.ones(8, device="cuda")
    codes, scales = ops.dynamic_int8_quant(x)
    for bad in (lambda: ops.dynamic_int8_quant(x.float()), lambda: ops.dynamic_int8_quant(x.t()),
                lambda: ops.dynamic_int8_quant(x[0].expand(4, 64)), lambda: ops.dynamic_int8_quant(x.cpu()),
                lambda: ops.int8_gemm(codes, w, scales, one, 4, 9, 64, "bf16"),
                lambda: ops.int8_gemm(codes, w, scales[:3], one, 4, 8, 64, "bf16"),
                lambda: ops.int8_gemm(codes, w, scales, one.half(), 4, 8, 64, "bf16"),
                lambda: ops.int8_gemm(codes, w, scales, one, 4, 8, 64, "int8"),
                lambda: ops.int8_gemm(codes[:, 1:], w[:, 1:], scales, one, 4, 8, 63, "bf16"),      # rows off 16 bytes
                lambda: ops.int8_gemm(codes[:, :0], w[:, :0], scales, one, 4, 8, 0, "bf16"),
                lambda: ops.int8_gemm_from_bf16(x, w[:, :48], one), lambda: ops.int8_gemm_from_bf16(x.float(), w, one),
                lambda: ops.silu_mul_int8_quant(x, x[:, :32]), lambda: ops.moe_permute_int8(x, one.int(), 3),
                lambda: ops.weight_int8_quant(torch.zeros(2, 3, 20, dtype=BF16, device="cuda"))):
        with pytest.raises(RuntimeError):
            bad()


@pytest.mark.parametrize("top", [-20.0, -86.0, -87.4, -88.5, -89.0, -91.0])
def test_silu_mul_of_gates_far_below_zero(ops, top):
    """Rows whose gates are all far below zero, with values of `up` that bring silu(g) * u back to the size of
    ordinary activations: nothing of them is lost.  e^(-|g| / 2) is off by two ulp at most and counts twice
    (8 * 2^-24); the products with it, the sum, the reciprocal and the two products behind it add 2^-24 each:
    14 * 2^-24 in all, below 2^-20."""
    g = torch.Generator().manual_seed(7)
    gate = top - torch.rand(3, 512, generator=g)
    up = torch.randn(3, 512, generator=g) * math.exp(-top - 10)
    h = gate.double() * torch.sigmoid(gate.double()) * up.double()
    a = h.abs().amax(1)
    codes, scales = ops.silu_mul_int8_quant(gate.cuda(), up.cuda())
    assert bool(((scales.cpu().double() - a / 127).abs() <= a / 127 * 2.0 ** -19).all())
    off = (codes.cpu().double() - h * 127 / a.unsqueeze(1)).abs().max()
    assert off <= 0.5 + 127 * 2.0 ** -19, off
