"""GPU tests of the int8 tensor-core kernel when a wait runs out: the kernel records it, waits for what it has
under way and returns, and the next call gives the bits of the one before.

The longest K makes it happen without a fault: the 1024 K blocks of a tile take 340 cycles each at least (16 KB of
weights at 48 bytes a cycle), 0.17 ms, and 0.1 ms for tiles of 256 tokens that four CTAs share; a limit of one cycle
gives a wait up after its first 17 looks of at most 2 us each."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
K = 131056


@pytest.fixture(scope="module")
def ops():
    from layerstormgemmkernels_b200 import ops as _ops
    return _ops


def codes(rows, k, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-127, 128, (rows, k), generator=g, dtype=torch.int8, device="cuda")


def gives_up_and_goes_on(call):
    """The call with a limit that runs out between two calls without."""
    from layerstormgemmkernels_b200 import capi
    want = call()
    assert capi.device_status() == 0
    for _ in range(3):
        capi.check(capi.lib.lsg_set_wait_limit_cycles(1))
        try:
            call()
            assert capi.device_status() != 0        # synchronizes: the kernel has returned
        finally:
            capi.check(capi.lib.lsg_set_wait_limit_cycles(0))
        assert torch.equal(call(), want)
        assert capi.device_status() == 0


@pytest.mark.parametrize("rows,N", [(16, 512), (48, 1024), (300, 9600)])        # single CTAs; pairs
def test_rows_of_experts(ops, rows, N):
    A, B = codes(rows, K, 1), codes(N, K, 2)
    sa, sb = torch.ones(rows, device="cuda"), torch.ones(1, N, device="cuda")
    offs = torch.tensor([0, rows], dtype=torch.int32, device="cuda")

    def call():
        return ops.int8_grouped_gemm(A, B.view(1, N, K), torch.zeros(rows, N, device="cuda"), sa, sb, offs, N, K, "fp32")
    gives_up_and_goes_on(call)


@pytest.mark.parametrize("M,N", [(500, 2000), (300, 4000), (1000, 4000)])      # K cut among four and two CTAs; pairs
def test_dense_behind_the_quantizer(ops, M, N):
    """Weights are under way before the quantizer has ended."""
    x = torch.randn(M, K, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").to(BF16)
    w, ws = codes(N, K, 4), torch.ones(N, device="cuda")
    gives_up_and_goes_on(lambda: ops.int8_gemm_from_bf16(x, w, ws, "fp32"))


@pytest.mark.parametrize("rows,I", [(40, 64), (300, 4800)])
def test_gate_and_up(ops, rows, I):
    hidden = torch.randn(rows, K, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda").to(BF16)
    gate_up, down = codes(2 * I, K, 6).view(1, 2 * I, K), codes(K, I, 7).view(1, K, I)
    gus, ds = torch.full((1, 2 * I), 1e-6, device="cuda"), torch.ones(1, K, device="cuda")
    offs = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    inv = torch.arange(rows, dtype=torch.int32, device="cuda")
    gives_up_and_goes_on(lambda: ops.int8_moe_ffn(hidden, offs, inv, 1, gate_up, gus, down, ds, "fp32"))


def test_streaming_forms_with_a_short_limit(ops):
    """One row, and one token's experts: their waits are for copies of a few KB and end long before any limit.
    Whatever a limit of one cycle does, the call returns and the next ones give the same bits."""
    from layerstormgemmkernels_b200 import capi
    x = torch.randn(1, 8192, generator=torch.Generator(device="cuda").manual_seed(8), device="cuda").to(BF16)
    w, ws = codes(16384, 8192, 9), torch.ones(16384, device="cuda")
    gate_up, down = codes(8 * 2048, 8192, 10).view(8, 2048, 8192), codes(8 * 8192, 1024, 11).view(8, 8192, 1024)
    gus, ds = torch.full((8, 2048), 1e-5, device="cuda"), torch.ones(8, 8192, device="cuda")
    offs = torch.arange(9, dtype=torch.int32, device="cuda").clamp_max(8)
    inv = torch.arange(8, dtype=torch.int32, device="cuda")

    def call():
        return torch.cat([ops.int8_gemm_from_bf16(x, w, ws, "fp32").flatten(),
                          ops.int8_moe_ffn(x, offs, inv, 8, gate_up, gus, down, ds, "fp32").flatten()])
    want = call()
    for _ in range(10):
        capi.check(capi.lib.lsg_set_wait_limit_cycles(1))
        try:
            got = call()
            if capi.device_status() == 0:
                assert torch.equal(got, want)
        finally:
            capi.check(capi.lib.lsg_set_wait_limit_cycles(0))
        assert torch.equal(call(), want) and capi.device_status() == 0
