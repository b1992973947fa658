"""attention_paged.cu's weighted probabilities in f16 numbers with a power of two of their own per row and block, step by step
in numpy: the references move as the kernel moves them, and the sums keep their accuracy whatever the scales are."""
import numpy as np
import pytest

TOP, START, MOST_E = 15, 8, 126


def f32(x):
    return np.asarray(x, dtype=np.float64).astype(np.float32)


def exponent(x):
    """Unbiased exponent bits of f32 numbers (-127 for zero and below 2^-126)."""
    return ((np.asarray(x, np.float32).view(np.uint32) >> 23) & 0xff).astype(np.int64) - 127


def pow2(n):
    return np.where(n < -126, 0.0, np.exp2(np.maximum(n, -126).astype(np.float64)))


def two_f16(w):
    """A weight as the sum of two f16 numbers: the first its leading 11 bits, the second what is left."""
    y = (w.view(np.uint32) & np.uint32(0xffffe000)).view(np.float32)
    return y.astype(np.float16).astype(np.float64) + (w - y).astype(np.float16).astype(np.float64)


def one_f16(w):
    return w.astype(np.float16).astype(np.float64)


def row(x, s, codes, hold):
    """One row: scores x [T] (log2), scales s [T, NB] f16, codes [T, NB] -> sums [NB] times 2^-M, M, l; and the range of the
    largest held weight over the steps after the first."""
    T, NB = s.shape
    M, L, E, O = np.float32(-3.4028235e38), np.float64(0), np.full(NB, MOST_E), np.zeros(NB)
    largest = np.zeros(NB)  # of the weights so far, in the present unit
    with np.errstate(over="ignore", invalid="ignore"):
        for t in range(0, T, 16):
            xs, ss = f32(x[t:t + 16]), s[t:t + 16].astype(np.float32)
            p = f32(np.exp2(xs.astype(np.float64) - M))
            w = f32(f32(ss.astype(np.float64) * p[:, None]) * np.exp2(E.astype(np.float64)))
            if np.nanmax(np.abs(w)) > 2.0 ** TOP or p.max() > 2.0 ** TOP:
                m = max(M, np.ceil(xs.max()))
                n = int(min(np.float64(m) - np.float64(M), 300))
                M = np.float32(m)
                L *= pow2(np.int64(-n))
                p = f32(np.exp2(xs.astype(np.float64) - M))
                big = exponent(np.abs(f32(ss.astype(np.float64) * p[:, None])).max(0))
                old = E + n
                E = np.minimum(np.minimum(old, MOST_E), START - big)
                f = pow2(E - old)
                O, largest = O * f, largest * f
                w = f32(f32(ss.astype(np.float64) * p[:, None]) * np.exp2(E.astype(np.float64)))
                assert np.abs(w).max() < 2.0 ** (START + 1) and p.max() <= 1
            assert np.isfinite(w).all() and np.abs(w).max() <= 2.0 ** TOP and p.max() <= 2.0 ** TOP
            L += p.astype(np.float64).sum()
            O += (hold(w) * codes[t:t + 16]).sum(0)
            largest = np.maximum(largest, np.abs(w).max(0))
    assert (largest[np.abs(s.astype(np.float64)).max(0) > 0] >= 2.0 ** START).all()
    return O * np.exp2(-E.astype(np.float64)), float(M), float(L)


@pytest.mark.parametrize("hold,rel", [(two_f16, 2.0 ** -22), (one_f16, 2.0 ** -11)])
@pytest.mark.parametrize("spread", [0, 10, 18, 24])
@pytest.mark.parametrize("how", ["blocks", "tokens", "growing", "one", "far"])
def test_weights_keep_their_accuracy(hold, rel, spread, how):
    rng = np.random.default_rng(spread)
    T, NB = 1024, 4
    x = rng.standard_normal(T) * 2
    size = np.zeros((T, NB))
    if how == "blocks":
        size += np.array([0, -spread, -spread / 2, 3])
    elif how == "tokens":
        size -= rng.integers(0, spread + 1, (T, NB))
    elif how == "growing":
        size += np.linspace(-spread, 0, T)[:, None] * np.array([1, 0.5, 0, -1]) - np.array([0, 0, 0, spread])
        x += np.linspace(0, 30, T)
    elif how == "one":  # a token that weighs nothing and is 2^spread times the others
        size -= spread
        size[333] = 0
        x[333] = -70
    else:  # scores near the end of f32: equal ones, whatever their size
        x = np.full(T, -3e37)
        size -= rng.integers(0, spread + 1, (T, NB))
    s = ((rng.random((T, NB)) + 0.5) * np.exp2(size) * np.where(rng.random((T, NB)) < 0.5, -1, 1)).astype(np.float16)
    s[:40, 2] = 0  # a block that begins with zeros
    codes = rng.integers(-8, 8, (T, NB))
    got, M, l = row(x, s, codes, hold)
    xs = f32(x).astype(np.float64)
    p = np.exp2(xs - xs.max())
    want = (p[:, None] * s.astype(np.float64) * codes).sum(0) / p.sum()
    weight = (p[:, None] * np.abs(s.astype(np.float64))).sum(0) / p.sum()
    # every weight is off by rel of itself (and three f32 roundings and the scores' in p) or by 2^-24 where the largest
    # is at least 2^8; codes are at most 8
    largest = (p[:, None] * np.abs(s.astype(np.float64))).max(0) / p.sum()
    bound = 8 * ((rel + 8 * 2.0 ** -24) * weight + T * 2.0 ** -32 * largest)
    assert (np.abs(got / l - want) <= bound).all(), np.abs(got / l - want) / bound
