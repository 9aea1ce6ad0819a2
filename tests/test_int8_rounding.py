"""CPU models of the rounding that the int8 quantizers rely on, over every pair of significands: the code of
127 x / a, nearest with half-way cases to even, from one fused multiply-add (bf16) and from a corrected
quotient (fp16).  Products of these operands are exact in float64, so float64 stands for the exact value."""
import numpy as np

F32 = np.float32


def exact_code(x, a):
    """Integers x, a > 0 (any common unit): rne(127 x / a) by whole-number arithmetic."""
    q, r = np.divmod(127 * x, a)
    return q + ((2 * r > a) | ((2 * r == a) & (q % 2 == 1)))


def rounded_up(v):
    c = v.astype(F32)
    return np.where(c.astype(np.float64) < v, np.nextafter(c, F32(np.inf)), c).astype(np.float64)


def test_one_fma_is_the_code_for_bf16():
    a = np.arange(128, 256, dtype=np.int64)[:, None]
    x = np.arange(0, 256, dtype=np.int64)[None, :]
    for d in range(0, 10):                       # a is 2^d times larger than its significand says
        big = a << d
        keep = x <= big
        c = rounded_up(127.0 / big)
        code = np.rint(x * c)                    # what adding 1.5 * 2^23 in one fused operation leaves
        assert np.array_equal(np.where(keep, code, 0), np.where(keep, exact_code(x, big), 0))


def test_nearest_reciprocal_would_not_do():
    """127 / a rounded to nearest instead of up: x = a / 2 (63.5) falls to 63 for some a."""
    a = np.arange(128, 256, dtype=np.int64) * 2
    c = (127.0 / a).astype(F32).astype(np.float64)
    assert np.any(np.rint(a / 2 * c) != exact_code(a // 2, a))


def test_corrected_quotient_is_the_code_for_fp16():
    a = np.arange(1024, 2048, dtype=np.int64)[:, None]
    x = np.arange(0, 2048, dtype=np.int64)[None, :]
    for d in range(0, 10):
        big = a << d
        rcp = (1.0 / big).astype(F32).astype(np.float64)
        y = (127 * x).astype(np.float64)
        t = (y * rcp).astype(F32).astype(np.float64)
        rest = (y - t * big).astype(F32).astype(np.float64)
        q = (t + rest * rcp).astype(F32).astype(np.float64)
        keep = x <= big
        assert np.array_equal(np.where(keep, np.rint(q), 0), np.where(keep, exact_code(x, big), 0))
