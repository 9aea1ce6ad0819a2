"""CPU model of the codes of fp32 values: the nearest integer to 127 x / a, half-way cases to even, from one fused
multiply-add and, where that came next to half-way, from two products and their rounding errors."""
import numpy as np

from tests.test_int8_rounding import exact_code, rounded_up

F32 = np.float32
DOUBT = -0.5 + 1.0625 * 2.0 ** -16


def f32(v):
    return v.astype(F32).astype(np.float64)


def settled(x, a):
    """The kernel's steps for x >= 0; x, a of 24 bits as float64, in which their products are exact."""
    c = rounded_up(127.0 / a)
    n = np.rint(x * c)
    w, h = 254.0 / 256, (2 * n - 1) / 256
    p, q = f32(w * x), f32(h * a)
    s = f32(f32(p - q) + f32(f32(w * x - p) - f32(h * a - q)))
    down = (s < 0) | ((s == 0) & (n % 2 == 1))
    return np.where((f32(x * c - n) < DOUBT) & down, n - 1, n)


def pairs(seed):
    """Rows' maxima of 24 bits and every value next to (k + 1/2) a / 127, at each step of one unit of x around it."""
    g = np.random.default_rng(seed)
    a = g.integers(1 << 23, 1 << 24, 4000)
    a[:100] = 127 << g.integers(0, 18, 100)
    a[100:200] = 381 << g.integers(0, 16, 100)
    a[200:300] = (g.integers(1 << 15, 1 << 16, 100) * 127) | 1
    k = np.arange(127)
    for shift in (0, 3, 6):                           # x of 24 bits below a, or with its last bits three, six places down
        big = a.astype(object) << shift
        x = np.array([[((2 * int(kk) + 1) * int(b)) // 254 for kk in k] for b in big])
        for step in (-1, 0, 1, 2):
            xx = np.maximum(x + step, 0)
            keep = (xx < (1 << 24)) & (xx <= np.array(big, dtype=np.int64)[:, None])
            yield xx, np.array(big, dtype=np.int64)[:, None], keep


def test_codes_next_to_half_way():
    for x, a, keep in pairs(1):
        want = exact_code(x, a)
        assert np.array_equal(np.where(keep, settled(x.astype(float), a.astype(float)), 0), np.where(keep, want, 0))


def test_the_fused_operation_alone_would_not_do():
    a, x = np.array([381.0]), np.array([1.5])
    assert np.rint(x * rounded_up(127.0 / a)) == 1 and settled(x, a) == 0        # the quotient is 1 / 2


def test_random_values():
    g = np.random.default_rng(2)
    a = g.integers(1 << 23, 1 << 24, (2000, 1))
    x = g.integers(0, 1 << 24, (2000, 500)) % (a + 1)
    assert np.array_equal(settled(x.astype(float), a.astype(float)), exact_code(x, a))
