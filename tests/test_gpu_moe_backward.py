"""GPU tests of the MoE routing steps in fp16 and fp32, of pairs without a row, and of the gradients of
the three steps, against the formulas in 64 bits and against differences.

Tolerances, with u = 2^-24: a sum of n products in fp32 is off by at most (n + 1) u times the sum of
the magnitudes, in whatever order; storing in bf16, fp16 adds half a step of the type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: U}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
SIZES = [(1, 4, 1, 8), (1, 128, 8, 2048), (5, 4, 4, 33), (7, 6, 3, 1), (33, 60, 4, 1001), (130, 8, 2, 4096), (64, 16, 16, 264),
         (300, 128, 8, 512)]


@pytest.fixture(scope="module")
def ops():
    from layerstormgemmkernels_b200 import ops as _ops
    return _ops


def routed(ops, T, E, k, seed, drop=True):
    g = torch.Generator().manual_seed(seed)
    idx, w = ops.moe_route(torch.randn(T, E, generator=g).cuda(), k)
    if drop and T > 4:
        idx[1] = -1                      # a token that no expert takes
        idx[2, 0] = E                    # an expert that is not there
        idx[4, k - 1] = -7
    offs, perm, inv = ops.moe_permutation(idx, E)
    return g, idx, w, offs, perm, inv


@pytest.mark.parametrize("T,E,k", [(5, 4, 4), (33, 60, 4), (128, 8, 8), (130, 8, 8), (4096, 16, 2)])
def test_permutation_of_pairs_without_a_row(ops, T, E, k):
    """Both routes (one CTA, and chunks): inv is -1 for such a pair, perm is 0 behind the last row."""
    _, idx, _, offs, perm, inv = routed(ops, T, E, k, T)
    flat = idx.flatten().cpu()
    valid = (flat >= 0) & (flat < E)
    n = int(valid.sum())
    order = torch.sort(torch.where(valid, flat, torch.full_like(flat, 1 << 20)), stable=True).indices[:n].int()
    assert int(offs[-1]) == n and torch.equal(perm.cpu()[:n], order) and not bool(perm.cpu()[n:].any())
    want = torch.full((T * k,), -1, dtype=torch.int32)
    want[order.long()] = torch.arange(n, dtype=torch.int32)
    assert torch.equal(inv.cpu(), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,E,k,H", SIZES)
def test_there_and_back(ops, T, E, k, H, dtype):
    g, idx, w, offs, perm, inv = routed(ops, T, E, k, T + H)
    n = int(offs[-1])
    x = torch.randn(T, H, generator=g).to(dtype)
    rows = ops.moe_permute(x.cuda(), perm, k)
    assert torch.equal(rows.cpu()[:n], x[(perm.cpu()[:n] // k).long()])
    y = torch.randn(T * k, H, generator=g).to(dtype)
    out = ops.moe_unpermute(y.cuda(), inv, w).cpu().double()
    iv = inv.cpu().long().view(T, k)
    part = torch.where((iv >= 0).unsqueeze(-1), y.double()[iv.clamp_min(0)], torch.zeros(1, dtype=torch.float64)) * w.cpu().double().unsqueeze(-1)
    want = part.sum(1)
    assert bool(((out - want).abs() <= (k + 1) * U * part.abs().sum(1) + HALF_STEP[dtype] * want.abs() * (1 + 2.0 ** -7) + 2.0 ** -25).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,E,k,H", SIZES)
def test_gradients(ops, T, E, k, H, dtype):
    g, idx, w, offs, perm, inv = routed(ops, T, E, k, 3 * T + H)
    n, iv = int(offs[-1]), inv.cpu().long().view(T, k)
    has = (iv >= 0).unsqueeze(-1)
    y = torch.randn(T * k, H, generator=g).to(dtype)
    gout = torch.randn(T, H, generator=g).to(dtype)
    grad_y, grad_w = ops.moe_unpermute_backward(gout.cuda(), y.cuda(), inv, w, offs)
    assert grad_y.dtype == dtype and not bool(grad_y[n:].any())
    wd, gd = w.cpu().double(), gout.double()
    want = torch.zeros(T * k, H, dtype=torch.float64)
    for t in range(T):
        for s in range(k):
            if iv[t, s] >= 0:
                want[iv[t, s]] = wd[t, s] * gd[t]
    small = 2.0 ** -25 if dtype == torch.float16 else 0.0      # below fp16's normal range
    assert bool(((grad_y.cpu().double() - want).abs() <= (HALF_STEP[dtype] + 2 * U) * want.abs() + small).all())
    prod = torch.where(has, y.double()[iv.clamp_min(0)], torch.zeros(1, dtype=torch.float64)) * gd.unsqueeze(1)
    assert bool(((grad_w.cpu().double() - prod.sum(-1)).abs() <= (H + 1) * U * prod.abs().sum(-1)).all())
    # without the offsets the rows that have a pair are the same
    other, other_w = ops.moe_unpermute_backward(gout.cuda(), y.cuda(), inv, w)
    assert torch.equal(other[:n], grad_y[:n]) and torch.equal(other_w, grad_w)

    grow = torch.randn(T * k, H, generator=g).to(dtype)
    grad_h = ops.moe_permute_backward(grow.cuda(), inv, k)
    part = torch.where(has, grow.double()[iv.clamp_min(0)], torch.zeros(1, dtype=torch.float64))
    want = part.sum(1)
    assert bool(((grad_h.cpu().double() - want).abs() <= (k + 1) * U * part.abs().sum(1) + HALF_STEP[dtype] * want.abs() * (1 + 2.0 ** -7) + small).all())

    grad_logits = ops.moe_route_backward(idx, w, grad_w, E)
    gw = grad_w.cpu().double()
    d = wd * (gw - (wd * gw).sum(-1, keepdim=True))
    want = torch.zeros(T, E + 1, dtype=torch.float64)
    ix = idx.cpu().long()
    want.scatter_add_(1, torch.where((ix >= 0) & (ix < E), ix, torch.full_like(ix, E)), d)
    tol = (k + 4) * U * (wd * (gw.abs() + (wd * gw).abs().sum(-1, keepdim=True))).amax(-1, keepdim=True)
    assert bool(((grad_logits.cpu().double() - want[:, :E]).abs() <= tol + 2.0 ** -140).all())


def test_same_expert_named_twice(ops):
    """A caller's own indices may name an expert twice: its logit gets both slots' gradients."""
    idx = torch.tensor([[3, 3, 1], [0, 2, 0]], dtype=torch.int32, device="cuda")
    w = torch.tensor([[0.5, 0.25, 0.25], [0.125, 0.5, 0.375]], device="cuda")
    gw = torch.tensor([[1.0, -2.0, 4.0], [8.0, 1.0, -3.0]], device="cuda")
    got = ops.moe_route_backward(idx, w, gw, 5).cpu()
    d = (w * (gw - (w * gw).sum(-1, keepdim=True))).cpu()
    want = torch.zeros(2, 5)
    want[0, 3], want[0, 1] = d[0, 0] + d[0, 1], d[0, 2]
    want[1, 0], want[1, 2] = d[1, 0] + d[1, 2], d[1, 1]
    assert torch.equal(got, want)            # sums of few-bit numbers: exact


def test_router_gradient_against_differences(ops):
    """Route, sort, experts (here a fixed matrix each), combine, and a loss: the logits' gradient by the
    operators against central differences of the same formula in float64 (error of the difference
    quotient about h^2, 1e-6; of the fp32 gradient below 1e-5 of its largest value)."""
    T, E, k, H = 6, 8, 3, 40
    g = torch.Generator().manual_seed(1)
    logits = torch.randn(T, E, generator=g)
    x, c = torch.randn(T, H, generator=g), torch.randn(T, H, generator=g)
    mats = torch.randn(E, H, H, generator=g).double() / H ** 0.5

    def loss(l, x):
        w, idx = torch.softmax(l, -1).topk(k)
        w = w / w.sum(-1, keepdim=True)
        out = torch.stack([sum(w[t, s] * (mats[idx[t, s]] @ x[t]) for s in range(k)) for t in range(T)])
        return (out * c.double()).sum()

    idx, w = ops.moe_route(logits.cuda(), k)
    offs, perm, inv = ops.moe_permutation(idx, E)
    rows = ops.moe_permute(x.cuda(), perm, k)
    expert = idx.flatten()[perm.long()].long().cpu()
    y = torch.einsum("rij,rj->ri", mats[expert], rows.cpu().double()).float().cuda()
    grad_y, grad_w = ops.moe_unpermute_backward(c.cuda(), y, inv, w, offs)
    grad_logits = ops.moe_route_backward(idx, w, grad_w, E).cpu().double()
    grad_rows = torch.einsum("rij,ri->rj", mats[expert], grad_y.cpu().double()).float().cuda()
    grad_x = ops.moe_permute_backward(grad_rows, inv, k).cpu().double()
    h = 1e-3
    for t, e in ((0, int(idx[0, 0])), (1, int(idx[1, 2])), (2, 0), (3, int(idx[3, 1])), (5, 7)):
        up, dn = logits.double().clone(), logits.double().clone()
        up[t, e] += h
        dn[t, e] -= h
        diff = float(loss(up, x.double()) - loss(dn, x.double())) / (2 * h)
        assert abs(diff - float(grad_logits[t, e])) <= 1e-5 * max(1.0, float(grad_logits.abs().max()))
    for t, j in ((0, 0), (2, 7), (5, 39)):
        up, dn = x.double().clone(), x.double().clone()
        up[t, j] += h
        dn[t, j] -= h
        diff = float(loss(logits.double(), up) - loss(logits.double(), dn)) / (2 * h)
        assert abs(diff - float(grad_x[t, j])) <= 1e-5 * max(1.0, float(grad_x.abs().max()))


@pytest.mark.parametrize("dtype", DTYPES)
def test_empty(ops, dtype):
    e = torch.empty(0, 16, dtype=dtype, device="cuda")
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    assert ops.moe_permute_backward(e, none, 2).shape == (0, 16)
    gy, gw = ops.moe_unpermute_backward(e, e, none, torch.empty(0, 2, device="cuda"))
    assert gy.shape == (0, 16) and gw.shape == (0, 2)
    assert ops.moe_route_backward(none.view(0, 2), torch.empty(0, 2, device="cuda"), torch.empty(0, 2, device="cuda"), 4).shape == (0, 4)
    # every pair without a row
    inv = torch.full((6,), -1, dtype=torch.int32, device="cuda")
    y = torch.randn(6, 16, device="cuda").to(dtype)
    gy, gw = ops.moe_unpermute_backward(y[:3], y, inv, torch.ones(3, 2, device="cuda"), torch.zeros(5, dtype=torch.int32, device="cuda"))
    assert not bool(gw.any()) and not bool(gy.any())
    assert not bool(ops.moe_permute_backward(y, inv, 2).any())
    assert not bool(ops.moe_unpermute(y, inv, torch.ones(3, 2, device="cuda")).any())


def test_not_finite_stays_in_its_rows(ops):
    """A NaN in one row of y or of the gradient reaches what the formulas say it reaches, no more."""
    T, E, k, H = 40, 8, 2, 520
    g, idx, w, offs, perm, inv = routed(ops, T, E, k, 9, drop=False)
    y, gout = torch.randn(T * k, H, generator=g).cuda(), torch.randn(T, H, generator=g).cuda()
    y[5, 3] = float("nan")
    gout[7, 100] = float("inf")
    grad_y, grad_w = ops.moe_unpermute_backward(gout, y, inv, w, offs)
    bad = torch.zeros(T * k, dtype=torch.bool)
    bad[int(perm[5])] = True
    bad[7 * k:8 * k] = True
    assert torch.equal(~grad_w.flatten().isfinite().cpu(), bad)
    assert int((~grad_y.isfinite()).sum()) == k


def test_backward_in_a_graph_and_twice(ops):
    """Captured and replayed on new inputs; the same inputs give the same bits."""
    T, E, k, H = 100, 16, 4, 1000
    g, idx, w, offs, perm, inv = routed(ops, T, E, k, 5)
    y, gout, grow = (torch.randn(n, H, generator=g).to(torch.bfloat16).cuda() for n in (T * k, T, T * k))

    def step():
        gy, gw = ops.moe_unpermute_backward(gout, y, inv, w, offs)
        return gy, gw, ops.moe_route_backward(idx, w, gw, E), ops.moe_permute_backward(grow, inv, k)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for _ in range(2):
        for t in (y, gout, grow):
            t.copy_(torch.randn(t.shape, generator=g).to(torch.bfloat16))
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_refused_on_cuda(ops):
    y, gout = torch.randn(8, 16, device="cuda"), torch.randn(4, 16, device="cuda")
    inv, w = torch.arange(8, dtype=torch.int32, device="cuda"), torch.ones(4, 2, device="cuda")
    for bad in (lambda: ops.moe_unpermute_backward(gout.half(), y, inv, w), lambda: ops.moe_unpermute_backward(gout[:, :8], y, inv, w),
                lambda: ops.moe_unpermute_backward(gout, y, inv[:7], w), lambda: ops.moe_unpermute_backward(gout, y, inv.long(), w),
                lambda: ops.moe_unpermute_backward(gout, y.t(), inv, w), lambda: ops.moe_unpermute_backward(gout, torch.zeros(9, 16, device="cuda"), inv, w),
                lambda: ops.moe_permute_backward(y, inv, 3), lambda: ops.moe_permute_backward(y.double(), inv, 2),
                lambda: ops.moe_route_backward(inv.view(4, 2), w, w[:3], 8), lambda: ops.moe_route_backward(inv.view(4, 2), w, w, 1),
                lambda: ops.moe_permute(y.double(), inv, 2), lambda: ops.moe_unpermute(y.half(), inv, w.half())):
        with pytest.raises(RuntimeError):
            bad()
