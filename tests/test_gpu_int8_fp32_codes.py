"""GPU tests of the codes of fp32 values, through silu(g) * u of gates of 32 (silu(32) is 32 in fp32, and
32 u is exact): the nearest integer to 127 x / a with half-way cases to even, whatever the row.

The quotient in float64 is never rounded onto or across half-way: 254 x and (2 k + 1) a are whole multiples of a
common unit of at least 2^-33 of the quotient, and float64 keeps 2^-46 of 127."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from layerstormgemmkernels_b200 import ops as _ops
    return _ops


def next_to_half_way(rows, seed, scale=1.0):
    """fp32 [rows, 3 * 127 + 3]: a row's maximum, and the three values nearest to each (k + 1/2) / 127 of it."""
    g = np.random.default_rng(seed)
    a = (g.random(rows) + 1).astype(np.float32) * np.float32(scale)
    a[0], a[1] = np.float32(381 * scale), np.float32(127 * scale)
    mid = (a[:, None].astype(np.float64) * (np.arange(127) + 0.5) / 127).astype(np.float32)
    x = np.concatenate([mid, np.nextafter(mid, np.float32(0)), np.nextafter(mid, np.float32(np.inf))], 1)
    x *= g.choice([-1, 1], x.shape).astype(np.float32)
    return torch.from_numpy(np.concatenate([a[:, None], x, -a[:, None], np.zeros_like(a[:, None])], 1))


def exact(x):
    x = x.double()
    a = x.abs().amax(1, keepdim=True)
    return (x * 127.0 / a).round(), a.squeeze(1).float() / 127.0


@pytest.mark.parametrize("scale", [1.0, 2.0 ** -90, 2.0 ** -112, 2.0 ** 100])
@pytest.mark.parametrize("copies", [1, 2, 6, 45])         # rows of a piece a thread, of two, and longer than 16384 values
def test_quantizer(ops, copies, scale):
    x = next_to_half_way(200 if copies < 45 else 20, copies, scale).repeat(1, copies)
    assert torch.equal((x / 32) * 32, x)
    for K in (x.size(1), x.size(1) - 5):               # whole pieces of eight values, and value by value
        v = x[:, :K].contiguous()
        codes, scales = ops.silu_mul_int8_quant(torch.full_like(v, 32.0).cuda(), (v / 32).cuda())
        q, s = exact(v)
        assert torch.equal(scales.cpu(), s) and torch.equal(codes.cpu().double(), q)


def test_half_way_from_bf16(ops):
    """127 * 3 and 24 * 0.0625 are bf16 products: the quotient 127 * 1.5 / 381 is one half, its code 0."""
    gate, up = torch.tensor([[127.0, 24.0] * 8]), torch.tensor([[3.0, 0.0625] * 8])
    codes, scales = ops.silu_mul_int8_quant(gate.to(BF16).cuda(), up.to(BF16).cuda())
    assert codes.cpu()[0].tolist() == [127, 0] * 8 and float(scales) == 3.0


@pytest.mark.parametrize("T", [1, 3, 9, 40, 1200])
def test_expert_block(ops, T):
    """One expert that leaves 32 u_i in value i (gate rows of scale 32, up rows of scale u_i over one input of code
    127 and scale 1 / 127) and hands every code on by itself: the streaming form and the four launches."""
    I = H = 384
    x = next_to_half_way(3, T)[2]
    u = torch.cat([x, torch.zeros(I - x.numel())]) / 32
    hidden = torch.zeros(T, H, dtype=BF16)
    hidden[:, 0] = 1.0
    gate_up = torch.zeros(1, 2 * I, H, dtype=torch.int8)
    gate_up[0, :, 0] = 1                               # sum 127, times 1 / 127 in fp32
    one = (torch.tensor(1.0) / 127) * 127
    assert float(one) == 1.0
    gus = torch.cat([torch.full((I,), 32.0), u])[None]
    down, ds = torch.eye(I, dtype=torch.int8)[None].contiguous(), torch.ones(1, H)
    offs, inv = torch.tensor([0, T], dtype=torch.int32), torch.arange(T, dtype=torch.int32)
    rows = ops.int8_moe_ffn(hidden.cuda(), offs.cuda(), inv.cuda(), 1, gate_up.cuda(), gus.cuda(), down.cuda(), ds.cuda(), "fp32").cpu()
    q, s = exact(32 * u[None])
    assert torch.equal(rows, (q.float() * s[:, None]).expand(T, H))
