"""A 64-bit statement of the paged 8-bit cache (test infrastructure): allocation, rotation,
block scales and codes, attention, from their definitions in include/jev.h."""
import math

import numpy as np

import npref

BLOCK = 16


def pages(n, page):
    return -(-n // page)


class Table:
    """The allocator: which pages every request has, and a plan's outputs."""

    def __init__(self, n_pages, page, max_requests, max_context):
        self.n_pages, self.page, self.max_requests, self.max_context = n_pages, page, max_requests, max_context
        self.length = [0] * max_requests
        self.own = [[] for _ in range(max_requests)]

    def plan(self, request, past, fresh, n_tokens):
        """(status, outputs by name); status 0, 1 (EINVAL) or 3 (ENOMEM), the library's numbers."""
        n, width = len(request), pages(self.max_context, self.page)
        out = {"table": np.full((n, width), -1), "slot": np.full(n_tokens, -1), "position": np.full(n_tokens, -1),
               "row": np.full(n_tokens, -1), "start": np.zeros(n + 1, int)}
        ok = len(set(request)) == n and all(0 <= r < self.max_requests for r in request)
        if ok:
            past = [self.length[r] for r in request] if past is None else past
            ok = all(0 <= p <= self.length[r] and f >= 0 and p + f <= self.max_context for r, p, f in zip(request, past, fresh))
        if not ok or sum(fresh) > n_tokens:
            return 1, out
        kept = [self.own[r][:pages(p, self.page)] for r, p in zip(request, past)]
        own = [list(o) for o in self.own]
        for r, k in zip(request, kept):
            own[r] = k
        free = sorted(set(range(self.n_pages)) - {x for o in own for x in o})
        need = sum(pages(p + f, self.page) - len(k) for p, f, k in zip(past, fresh, kept))
        if need > len(free):
            return 3, out
        self.own, t = own, 0
        for b, (r, p, f) in enumerate(zip(request, past, fresh)):
            more = pages(p + f, self.page) - len(own[r])
            own[r] += free[:more]
            free = free[more:]
            self.length[r] = p + f
            out["table"][b, :len(own[r])] = own[r]
            out["start"][b + 1] = t + f
            for i in range(f):
                out["position"][t], out["row"][t] = p + i, b
                out["slot"][t] = own[r][(p + i) // self.page] * self.page + (p + i) % self.page
                t += 1
        return 0, out


def rotate(cfg, x, pos, half, query):
    """x [tokens, heads, dim] rotated for its positions, in 64 bits."""
    rd, n = cfg.rope_dim, cfg.rope_dim // 2
    x = np.array(x, np.float64)
    if rd:
        freqs, mag = npref.rope_tables(cfg)
        angle = np.asarray(pos, np.float64)[:, None] * freqs
        c, s = (np.cos(angle) * mag)[:, None], (np.sin(angle) * mag)[:, None]
        a, b = (slice(0, n), slice(n, rd)) if half else (slice(0, rd, 2), slice(1, rd, 2))
        x0, x1 = x[..., a].copy(), x[..., b].copy()
        x[..., a], x[..., b] = x0 * c - x1 * s, x0 * s + x1 * c
    return x * npref.position_scale(cfg, pos)[:, None, None] if query else x


class Cache:
    """One layer's stored values of one request: [position][head][dim] codes and their blocks' scales."""

    def __init__(self, heads, dim):
        self.code, self.scale = np.zeros((0, heads, dim)), np.zeros((0, heads), np.float32)

    def store(self, past, x):
        """x [fresh, heads, dim] at positions past .. (fp32 values)."""
        x = np.asarray(x, np.float32)
        end = past + len(x)
        rows, blocks = pages(end, BLOCK) * BLOCK, pages(end, BLOCK)
        code, scale = np.zeros((rows, *self.code.shape[1:])), np.zeros((blocks, self.scale.shape[1]), np.float32)
        keep = pages(past, BLOCK)
        code[:past], scale[:keep] = self.code[:past], self.scale[:keep]
        for b in range(past // BLOCK, blocks if len(x) else 0):
            lo, hi = max(past, b * BLOCK), min(end, (b + 1) * BLOCK)
            for h in range(scale.shape[1]):
                v = x[lo - past:hi - past, h]
                new = np.float32(np.nan) if not np.isfinite(v).all() else np.float32(np.abs(v).max() / np.float32(127))
                old = scale[b, h] if lo > b * BLOCK else np.float32(0)
                s = old if np.isnan(old) else new if np.isnan(new) or new > old else old
                scale[b, h] = s
                if s > 0:
                    code[b * BLOCK:lo, h] = np.rint(code[b * BLOCK:lo, h] * np.float64(old) / np.float64(s))
                    code[lo:hi, h] = np.clip(np.rint(v.astype(np.float64) / np.float64(s)), -127, 127)
                else:
                    code[b * BLOCK:hi, h] = 0
        self.code, self.scale = code, scale

    def values(self, length):
        """fp32 [length, heads, dim]."""
        s = np.repeat(self.scale, BLOCK, axis=0)[:length]
        return self.code[:length].astype(np.float32) * s[:, :, None]


def attend(q, k, v, past):
    """q [fresh, heads, dim] at positions past .. over k, v [past + fresh, kv heads, dim]; also a bound on
    what fp16 pairs and fp32 sums may be off by (see tests/test_gpu_pages.py)."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    f, heads, d = q.shape
    g = heads // k.shape[1]
    out, off = np.empty_like(q), np.empty((f, heads))
    for h in range(heads):
        kh, vh = k[:, h // g], v[:, h // g]
        s = q[:, h] @ kh.T / math.sqrt(d)
        a = np.abs(q[:, h]) @ np.abs(kh).T / math.sqrt(d)
        seen = np.arange(len(kh)) <= past + np.arange(f)[:, None]
        s = np.where(seen, s, -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        out[:, h] = p @ np.where(seen.any(0)[:, None], vh, 0)
        # a score: q within 2^-21 of its pair, d products summed in fp32 and two roundings of their scale;
        # its exponential: the score's error twice (numerator, sum) and a few roundings; the sums over keys
        e = np.where(seen, a, 0).max(-1) * (2.0 ** -21 + (d + 4) * 2.0 ** -24) + 2.0 ** -21 + np.abs(np.where(seen, s, 0)).max(-1) * 2.0 ** -23
        off[:, h] = np.where(seen, np.abs(vh).max(-1), 0).max(-1) * (2 * np.expm1(e) + 2.0 ** -19 + len(kh) * 2.0 ** -24)
    return out, off
