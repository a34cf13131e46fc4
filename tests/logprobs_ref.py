"""Log probabilities, entropy and order of rows of logits in 64 bits, and what the kernel's may be off by
(test infrastructure).

The kernel's differences (x - m) c are fp32: 3 roundings, and their exponentials within 2^-23; sums of
exponentials are fp32 over a lane's 32 and 64-bit beyond.  A running sum is rescaled when its maximum moves: at most a wave's 16 passes over
131072 logits, six steps across its lanes, three waves, six steps across parts, each by an exponential of its own
within the same error, 34 in all with a term's first.  The maximum's own term is exactly 1 and kept apart, so the error
lies in the other terms' share of the sum.  So are sums of e times its exponent."""
import numpy as np

ULP = 2.0 ** -24


def order(x, k):
    """The k largest of a row: NaN first, +0 above -0, the lowest index first."""
    x = np.asarray(x, np.float32)
    b = x.view(np.uint32).astype(np.uint64)
    up = np.where(np.isnan(x), np.uint64(2 ** 32 - 1), np.where(b >> np.uint64(31), b ^ np.uint64(2 ** 32 - 1), b | np.uint64(2 ** 31)))
    return np.lexsort((np.arange(len(x)), -up.astype(np.int64)))[:k]


def row(x, temperature):
    """(logp of every token, entropy, bound on logp's error beside its rounding, the same on the entropy's)."""
    x = np.asarray(x, np.float64)
    t = float(np.float32(temperature))
    if np.isnan(x).any() or not np.isfinite(x.max()):
        return np.full(len(x), np.nan), np.nan, 0.0, 0.0
    d = (x - x.max()) / t
    e = np.exp(d)
    s = e.sum()
    rest = e.copy()
    rest[x.argmax()] = 0
    logp = d - np.log1p(rest.sum())
    p, gap = e / s, np.where(np.isfinite(d), -d, 0)
    entropy = np.log1p(rest.sum()) + (p * gap).sum()
    one = 3 * ULP * gap + (34 * 2 + 32) * ULP
    off = (rest / s * one).sum()
    return logp, entropy, off, off + (p * gap * (one + 2 * ULP)).sum() + off * (p * gap).sum()
