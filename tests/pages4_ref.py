"""A 64-bit statement of the 4-bit paged cache's values (test infrastructure), from include/jev.h:
per token, KV head and side a power 2^e, per 32 elements a step u and a zero point z, codes n."""
import numpy as np

GROUP = 32


def quantise(x):
    """(codes n, steps u, zero points z, powers e) of finite fp32 rows x [..., dim]."""
    x = np.asarray(x, np.float32)
    g = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    hi, lo = np.maximum(g.max(-1), 0), np.maximum(-g.min(-1), 0)
    span = 2.0 * (np.float32(0.5) * hi + np.float32(0.5) * lo).astype(np.float64)  # fp32, where twice it may be past fp32
    m, ex = np.frexp(span.max(-1))
    e = np.maximum(ex - np.where(m <= 225.0 / 256.0, 8, 7), -126)
    unit = np.ldexp(1.0, e)[..., None]
    u = np.maximum(1, sum((span > 15.0 * k * unit) for k in range(15)))
    z = np.rint(lo / (u * unit))
    n = np.clip(np.rint(g / (u * unit)[..., None]) + z[..., None], 0, 15)
    return n, u, z, e


def values(x):
    """The fp32 values that rows x read as."""
    x = np.asarray(x, np.float32)
    ok = np.isfinite(x).all(-1)
    n, u, z, e = quantise(np.where(ok[..., None], x, 0))
    y = ((n - z[..., None]) * u[..., None]).reshape(x.shape) * np.ldexp(1.0, e)[..., None]
    return np.where(ok[..., None], y, np.nan).astype(np.float32)


class Side:
    """One layer's stored keys, or values, of one request; `other` is the other side, whose NaN are these'."""

    def __init__(self, heads, dim):
        self.read, self.other = np.zeros((0, heads, dim), np.float32), None

    def store(self, past, x):
        self.read = np.concatenate([self.read[:past], np.zeros((past - len(self.read[:past]), *self.read.shape[1:]), np.float32), values(x)])

    def values(self, length):
        y = self.read[:length]
        if self.other is None:
            return y
        bad = np.isnan(self.other.read[:length]).any(-1)
        return np.where(bad[..., None], np.float32(np.nan), y)


class Cache(dict):
    """What Rig.kv is, for the 4-bit cache: (request, layer, "k" or "v") -> Side."""

    def __init__(self, heads, dim):
        super().__init__()
        self.shape = heads, dim

    def setdefault(self, key, _):
        r, layer, name = key
        if key not in self:
            pair = self[r, layer, "k"], self[r, layer, "v"] = Side(*self.shape), Side(*self.shape)
            pair[0].other, pair[1].other = pair[1], pair[0]
        return self[key]
