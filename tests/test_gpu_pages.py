"""The paged 8-bit cache on the GPU against its 64-bit statement (tests/pages_ref.py).

Plans and stored values are compared bit for bit: rotation and codes are 64-bit up to one
rounding, so the stored value is determined.  Attention is held to a bound by arithmetic
(pages_ref.attend): a query row enters as an fp16 pair (each half to nearest: 2^-22 relative,
with the pair's own floor 2^-21), a score is a sum of head_dim fp32 products (2^-24 each), an
exponential's relative error is its argument's absolute one, the weight's pair 2^-21, and the
sums over n keys n 2^-24."""
import ctypes

import numpy as np
import pytest

import jev
import pages_ref as R

pytestmark = pytest.mark.gpu


def cfg(heads=4, kv=2, dim=128, layers=1, rope=0, **kw):
    return jev.ModelConfig(n_layers=layers, n_heads=heads, n_kv_heads=kv, head_dim=dim, rope_dim=rope, **kw)


class Rig:
    """A KvPages and its statement, driven together."""

    def __init__(self, config, n_pages, page=16, requests=8, context=4096, tokens=4096, half=False):
        import torch

        self.t, self.c, self.half = torch, config, half
        self.p = jev.KvPages(config, n_pages, page, requests, context, tokens, half)
        self.table = R.Table(n_pages, page, requests, context)
        self.kv = {}

    def dev(self, a, dtype=None):
        return self.t.as_tensor(np.ascontiguousarray(a), dtype=dtype, device="cuda")

    def ints(self, a):
        return self.dev(a, self.t.int32)

    def plan(self, request, fresh, past=None, pad=0, outputs=True):
        """The plan's outputs, checked; the library's error, if it refuses."""
        n, tokens = len(request), max(0, sum(fresh)) + pad
        tokens = min(tokens, self.p.max_tokens)
        out = {"table": self.t.full((n, R.pages(self.table.max_context, self.table.page)), -7, dtype=self.t.int32, device="cuda"),
               "start": self.t.full((n + 1,), -7, dtype=self.t.int32, device="cuda")}
        for name in ("slot", "position", "row"):
            out[name] = self.t.full((tokens,), -7, dtype=self.t.int32, device="cuda")
        before = list(self.table.length)
        self.args = self.ints(request), None if past is None else self.ints(past), self.ints(fresh)
        self.p.plan_device(self.args[0].data_ptr(), 0 if past is None else self.args[1].data_ptr(), self.args[2].data_ptr(), n, tokens,
                           **({k: v.data_ptr() for k, v in out.items()} if outputs else {}))
        status, want = self.table.plan(list(request), past, list(fresh), tokens)
        if status:
            with pytest.raises(jev.JevError) as e:
                self.p.sync()
            assert e.value.code == status
        else:
            self.p.sync()
        if outputs:
            for k, v in want.items():
                np.testing.assert_array_equal(out[k].cpu().numpy(), v, err_msg=k)
        self.batch = [] if status else [(r, before[r] if past is None else past[b], fresh[b]) for b, r in enumerate(request)]
        self.tokens, self.slots = tokens, want["slot"]
        return status

    def store(self, q=None, k=None, v=None, layer=0, lead=0, gap=0):
        """Stores k and v, returns the rotated q; checks both.  `gap` floats between rows, `lead` before the first."""
        c, total = self.c, sum(f for _, _, f in self.batch)

        def laid(x, width):
            if x is None:
                return None, 0
            a = np.full(lead + self.tokens * (width + gap), np.nan, np.float32)
            rows = a[lead:].reshape(self.tokens, width + gap)
            rows[:len(x), :width] = x.reshape(len(x), width)
            t = self.dev(a)
            return t, t.data_ptr() + 4 * lead

        (tq, pq), (tk, pk), (tv, pv) = laid(q, c.qdim), laid(k, c.kvdim), laid(v, c.kvdim)
        out = self.t.full((lead + self.tokens * c.qdim,), -7.0, device="cuda")
        self.p.store_device(layer, pq, c.qdim + gap, pk, pv, c.kvdim + gap, out.data_ptr() + 4 * lead if q is not None else 0)
        self.p.sync()
        pos = np.concatenate([np.arange(p, p + f) for _, p, f in self.batch]) if self.batch else np.zeros(0)
        if q is not None:
            got = out.cpu().numpy()[lead:].reshape(self.tokens, c.n_heads, c.head_dim)
            want = R.rotate(c, q, pos, self.half, True)
            # one rounding to fp32 (2^-24 relative); 64-bit sines and cosines are off by an ulp or two of 64 bits
            assert np.all(np.abs(got[:total] - want) <= np.abs(want) * 2.0 ** -24 * 1.0001 + np.abs(q).max(initial=0) * 1e-15 + 1e-44)
            assert np.all(got[total:] == -7)
        if k is not None:
            at = 0
            kr = R.rotate(c, k, pos, self.half, False).astype(np.float32)
            for r, p, f in self.batch:
                for name, x in (("k", kr), ("v", v)):
                    self.kv.setdefault((r, layer, name), R.Cache(c.n_kv_heads, c.head_dim)).store(p, x[at:at + f])
                at += f
        return out[lead:].reshape(self.tokens, c.n_heads, c.head_dim) if q is not None else None

    def check_values(self, layer=0):
        """Every stored value of the batch's requests."""
        page = self.table.page
        for r, p, f in self.batch:
            n = p + f
            if n == 0:
                continue
            slots = self.ints([self.table.own[r][i // page] * page + i % page for i in range(n)])
            k, v = (self.t.full((n, self.c.n_kv_heads, self.c.head_dim), -7.0, device="cuda") for _ in "kv")
            self.p.read_device(layer, slots.data_ptr(), n, k.data_ptr(), v.data_ptr())
            self.p.sync()
            for name, got in (("k", k), ("v", v)):
                np.testing.assert_array_equal(got.cpu().numpy(), self.kv[r, layer, name].values(n), err_msg=f"{name} of request {r}")

    def attend(self, q, layer=0, check=True):
        c, total = self.c, sum(f for _, _, f in self.batch)
        x = np.zeros((self.tokens, c.n_heads, c.head_dim), np.float32)
        x[:total] = q
        dq = self.dev(x)
        out = self.t.full_like(dq, -7.0)
        self.p.attend_device(layer, dq.data_ptr(), out.data_ptr())
        self.p.sync()
        got, at = out.cpu().numpy(), 0
        assert np.all(got[total:] == -7)  # rows behind the last request stay as they were
        for r, p, f in self.batch if check else []:
            if f:
                with np.errstate(all="ignore"):
                    want, off = R.attend(q[at:at + f], self.kv[r, layer, "k"].values(p + f), self.kv[r, layer, "v"].values(p + f), p)
                bad = ~(np.abs(got[at:at + f] - want) <= off[:, :, None])
                assert not bad.any(), (r, p, f, np.argwhere(bad)[:3], np.abs(got[at:at + f] - want).max(), off.max())
            at += f
        return got[:total]

    def fill(self, rs, request, fresh, past=None, spread=1.0, layer=0, check=False):
        """Plans and stores normal values."""
        self.plan(request, fresh, past, outputs=False)
        n = sum(fresh)
        k, v = (rs.randn(n, self.c.n_kv_heads, self.c.head_dim).astype(np.float32) * np.float32(spread) for _ in "kv")
        self.store(None, k, v, layer)
        if check:
            self.check_values(layer)


@pytest.fixture
def rs():
    return np.random.RandomState(7)


# ---------------------------------------------------------------- plan


@pytest.mark.parametrize("page,n_pages,requests,context", [(16, 70, 6, 300), (64, 33, 9, 700), (256, 20, 3, 2000), (32, 4000, 1500, 90), (16, 9000, 4096, 33)])
def test_plans_follow_the_allocator(gpu, rs, page, n_pages, requests, context):
    """Steps of growing, cut back, released and idle requests, until the pool runs out, against the statement."""
    rig = Rig(cfg(heads=1, kv=1, dim=64), n_pages, page, requests, context, tokens=30000)
    refused = 0
    for step in range(14):
        n = rs.randint(1, requests + 1)
        request = rs.permutation(requests)[:n]
        length = np.array([rig.table.length[r] for r in request])
        past = None if step % 3 == 0 else rs.randint(0, length + 1)
        kept = length if past is None else past
        fresh = np.minimum(rs.choice([0, 1, 1, 17, context], n), context - kept)
        if fresh.sum() > 30000:
            fresh = np.minimum(fresh, 1)
        refused += rig.plan([int(r) for r in request], [int(f) for f in fresh], None if past is None else [int(p) for p in past],
                            pad=int(rs.choice([0, 5]))) != 0
    assert step == 13 and (refused > 0) == (page in (16, 64, 256) and n_pages < 100)


def test_plan_forms_and_edges(gpu):
    rig = Rig(cfg(heads=1, kv=1, dim=64, rope=64), 64, 16, 4, 512, tokens=600)
    assert rig.plan([2], [1]) == 0                       # one token
    assert rig.plan([0, 1, 3], [0, 0, 0]) == 0           # nothing
    assert rig.plan([], []) == 0
    assert rig.plan([3, 0], [512, 1], pad=11) == 0       # a whole context: the lists take a launch of their own
    assert rig.plan([3], [1]) == 1                       # past the context
    assert rig.plan([3], [0], [0]) == 0                  # released
    assert rig.plan([0, 1, 2, 3], [500, 400, 100, 1], [0, 0, 0, 0]) == 1  # more than 600 rows
    assert rig.plan([0, 1], [512, 64]) == 1              # past the context again, another request
    assert rig.plan([1], [511]) == 0
    assert rig.plan([0], [500]) == 3                     # 32 pages more, and 30 are free
    assert rig.plan([0], [470]) == 0                     # all of them but one
    assert rig.plan([1], [400], [0]) == 0


@pytest.mark.parametrize("request_,past,fresh", [([4], None, [1]), ([-1], None, [1]), ([1, 1], None, [1, 1]), ([0], [2], [1]), ([0], [-1], [1]),
                                                 ([0], None, [-1]), ([0, 1], None, [2 ** 31 - 1, 5]), ([0], [1], [2 ** 31 - 1])])
def test_refused_plans_change_nothing(gpu, request_, past, fresh):
    rig = Rig(cfg(heads=1, kv=1, dim=64), 40, 16, 4, 512, tokens=64)
    assert rig.plan([0, 2], [1, 20]) == 0
    assert rig.plan(request_, fresh, past, pad=0) == 1
    # the calls after it do nothing
    out = rig.t.full((64, 64), -7.0, device="cuda")
    rig.p.store_device(0, out.data_ptr(), 64, out.data_ptr(), out.data_ptr(), 64, out.data_ptr())
    q = rig.t.zeros((64, 64), device="cuda")
    rig.p.attend_device(0, q.data_ptr(), out.data_ptr())
    rig.t.cuda.synchronize()
    assert bool((out == -7).all())
    assert rig.plan([2, 0], [3, 17]) == 0


# ---------------------------------------------------------------- rotation


@pytest.mark.parametrize("dim,rope", [(128, 128), (128, 96), (128, 20), (128, 2), (64, 64), (64, 44), (64, 4)])
@pytest.mark.parametrize("half", [False, True])
def test_rotation(gpu, rs, dim, rope, half):
    rig = Rig(cfg(6, 2, dim, rope=rope, rope_freq_base=10000.0), 300, 16, 3, 4096, half=half)
    rig.plan([1, 0, 2], [37, 1, 700], pad=3)
    for lead, gap in ((0, 0), (0, 4), (1, 0), (3, 5)):  # vector and single accesses
        rig.store(rs.randn(738, 6, dim).astype(np.float32), lead=lead, gap=gap)


def test_rotation_in_place(gpu, rs):
    rig = Rig(cfg(4, 1, 128, rope=128), 20, 16, 2, 160)
    rig.plan([0], [33])
    q = rs.randn(33, 4, 128).astype(np.float32)
    x = rig.dev(q)
    rig.p.store_device(0, x.data_ptr(), 512, 0, 0, 0, x.data_ptr())
    y = rig.store(q)
    assert bool((x == y).all())


@pytest.mark.parametrize("kw", [dict(rope_scale_factor=4.0), dict(rope_scale_factor=16.0, rope_scaling_yarn=1, rope_original_context=256),
                                dict(rope_scale_factor=2.0, rope_scaling_yarn=1, rope_original_context=64, yarn_mscale=1.0, yarn_mscale_all_dim=0.5,
                                     attention_temperature_scale=0.25, rope_attn_factor=1.5, yarn_ext_factor=0.75)])
def test_scaled_positions(gpu, rs, kw):
    rig = Rig(cfg(4, 2, 128, rope=128, rope_freq_base=1e6, **kw), 200, 16, 2, 2000)
    rig.plan([0, 1], [1500, 3], pad=1)
    x = rs.randn(1503, 4, 128).astype(np.float32)
    rig.store(x, x[:, :2], x[:, 2:])
    rig.check_values()


def test_far_positions_keep_their_angle(gpu, rs):
    rig = Rig(cfg(1, 1, 64, rope=64), 65538, 256, 1, 1 << 24, tokens=1 << 22)
    request = rig.ints([0])
    for n in (1 << 22, 1 << 22, 1 << 22, 9):  # (the statement's own tables would take minutes here)
        fresh = rig.ints([n])
        rig.p.plan_device(request.data_ptr(), 0, fresh.data_ptr(), 1, n)
        rig.p.sync()
    rig.batch, rig.tokens = [(0, 3 << 22, 9)], 9
    q = rs.randn(9, 1, 64).astype(np.float32)
    out = rig.t.empty((9, 1, 64), device="cuda")
    x = rig.dev(q)
    rig.p.store_device(0, x.data_ptr(), 64, 0, 0, 0, out.data_ptr())
    rig.p.sync()
    want = R.rotate(rig.c, q, (3 << 22) + np.arange(9), False, True)
    # the library's 64-bit frequency may be an ulp off numpy's: 2^-52 of an angle of 2^23.6 radians
    assert np.all(np.abs(out.cpu().numpy() - want) <= np.abs(want) * 2.0 ** -24 + np.abs(q).max() * 2.0 ** -27)


# ---------------------------------------------------------------- store


@pytest.mark.parametrize("dim,page,rope,half", [(128, 16, 128, False), (128, 64, 32, True), (64, 32, 0, False), (64, 256, 60, True)])
def test_stored_values(gpu, rs, dim, page, rope, half):
    """Steps of uneven sizes whose values grow and shrink: blocks begun, filled, rescaled."""
    rig = Rig(cfg(4, 2, dim, rope=rope), 40 + 4000 // page, page, 5, 900, half=half)
    for fresh in ([1, 5, 16, 0, 33], [1, 1, 1, 1, 1], [15, 11, 1, 200, 0], [1, 1, 16, 17, 31]):
        rig.plan([3, 0, 4, 1, 2], fresh, outputs=False)
        n = sum(fresh)
        k, v = (rs.randn(n, 2, dim).astype(np.float32) * np.exp2(rs.randint(-9, 10, (n, 1, 1))).astype(np.float32) for _ in "kv")
        rig.store(rs.randn(n, 4, dim).astype(np.float32), k, v, lead=int(rs.randint(2)), gap=int(rs.choice([0, 4, 3])))
        rig.check_values()


def test_special_values(gpu, rs):
    """Zeros, exact halves, the largest and smallest numbers, infinities and NaN; a block stays NaN until it is begun anew."""
    rig = Rig(cfg(2, 2, 64), 40, 16, 2, 320)
    x = rs.randn(112, 2, 64).astype(np.float32)
    x[0:16] = 0
    x[16:32] = rs.randint(-254, 255, (16, 2, 64)) / 2.0  # a scale of 1: halves
    x[16, :, 0] = 127
    x[32:48] *= 1e37
    x[48:64] *= 1e-39
    x[64:80] = 2.0 ** -149
    x[81, 0, 3] = np.nan
    x[96, 1, 60] = np.inf
    rig.plan([1], [112])
    rig.store(None, x, x[::-1].copy())
    rig.check_values()
    rig.fill(rs, [1], [4], [86], check=True)   # into the NaN block
    rig.fill(rs, [1], [40], [80], check=True)  # the block begun anew


def test_cut_back_requests_share_the_pool(gpu, rs):
    """Pages given back and taken by another request; a cut block keeps its scale."""
    rig = Rig(cfg(2, 1, 128), 14, 16, 3, 192)  # all 14 pages in the end: 61, 70 and 67 tokens
    rig.fill(rs, [0, 1], [100, 60], check=True)
    rig.fill(rs, [0, 2], [3, 66], [37, 0], spread=0.1, check=True)
    rig.fill(rs, [1, 0, 2], [1, 30, 1], check=True)
    rig.fill(rs, [1], [60], [0], check=True)


def test_layers_are_apart(gpu, rs):
    rig = Rig(cfg(2, 1, 64, layers=3), 6, 32, 2, 96)
    rig.plan([1, 0], [40, 7])
    for layer in (2, 0, 1):
        k, v = (rs.randn(47, 1, 64).astype(np.float32) * (layer + 1) for _ in "kv")
        rig.store(None, k, v, layer)
    for layer in range(3):
        rig.check_values(layer)
        rig.attend(rs.randn(47, 2, 64).astype(np.float32), layer)


def test_reading_outside_the_pool(gpu, rs):
    rig = Rig(cfg(1, 1, 64), 3, 16, 1, 48)
    rig.fill(rs, [0], [48])
    slots = rig.ints([-1, 48, 2 ** 31 - 1, -2 ** 31, 47])
    k = rig.t.full((5, 64), -7.0, device="cuda")
    v = k.clone()
    rig.p.read_device(0, slots.data_ptr(), 5, k.data_ptr(), v.data_ptr())
    rig.p.sync()
    assert bool((k[:4] == 0).all()) and bool((v[:4] == 0).all()) and bool((k[4] != 0).any())


# ---------------------------------------------------------------- attention


@pytest.mark.parametrize("heads,kv,dim", [(4, 1, 128), (8, 8, 64), (7, 1, 64), (32, 2, 128), (20, 1, 128), (48, 1, 64), (6, 2, 128)])
@pytest.mark.parametrize("page", [16, 128])
def test_single_tokens(gpu, rs, heads, kv, dim, page):
    """One token a request over lengths about every border."""
    past = [0, 1, 14, 15, 16, 62, 63, 64, 65, 127, 255, 256, 257, 300, 511, 513, 700, 1025]
    rig = Rig(cfg(heads, kv, dim), 600 if page == 16 else 120, page, len(past), 1100, 8000)
    rig.fill(rs, list(range(len(past))), past)
    ids = [int(i) for i in rs.permutation(len(past))]
    rig.fill(rs, ids, [1] * len(past))
    rig.attend(rs.randn(len(past), heads, dim).astype(np.float32))


@pytest.mark.parametrize("heads,kv,dim", [(4, 1, 128), (3, 3, 64), (10, 2, 128), (16, 1, 64), (40, 2, 128)])
def test_prompts(gpu, rs, heads, kv, dim):
    """Ragged batches: nothing, single tokens, a few, more than a tile of any width, behind pasts of any length."""
    past = [0, 5, 0, 63, 300, 129, 0, 17]
    fresh = [1, 130, 0, 2, 33, 64, 301, 4]
    rig = Rig(cfg(heads, kv, dim), 200, 16, 8, 500)
    rig.fill(rs, list(range(8)), past)
    rig.plan([6, 1, 2, 0, 7, 4, 5, 3], [fresh[i] for i in (6, 1, 2, 0, 7, 4, 5, 3)], pad=5)
    n = sum(fresh)
    rig.store(None, rs.randn(n, kv, dim).astype(np.float32), rs.randn(n, kv, dim).astype(np.float32))
    rig.attend(rs.randn(n, heads, dim).astype(np.float32))


def test_long_contexts(gpu, rs):
    for past in (5000, 40000):
        rig = Rig(cfg(4, 1, 64), 2600, 16, 1, 41000, 41000)
        rig.fill(rs, [0], [past])
        rig.fill(rs, [0], [1])
        rig.attend(rs.randn(1, 4, 64).astype(np.float32))
        rig.fill(rs, [0], [70])
        rig.attend(rs.randn(70, 4, 64).astype(np.float32))


@pytest.mark.parametrize("fresh", [1, 90])
def test_scales_far_apart(gpu, rs, fresh):
    """Queries and values far from one: the pairs stay inside fp16's range by powers of two."""
    rig = Rig(cfg(4, 2, 128), 40, 16, 1, 600)
    n = 400 + fresh
    k = rs.randn(n, 2, 128).astype(np.float32) * np.float32(1e-18)
    v = rs.randn(n, 2, 128).astype(np.float32) * np.exp2(np.repeat(rs.randint(-100, 100, -(-n // 16)), 16)[:n, None, None]).astype(np.float32)
    rig.plan([0], [400])
    rig.store(None, k[:400], v[:400])
    rig.plan([0], [fresh])
    rig.store(None, k[400:], v[400:])
    rig.attend(rs.randn(fresh, 4, 128).astype(np.float32) * np.float32(1e18))
    rig.attend(rs.randn(fresh, 4, 128).astype(np.float32) * np.float32(1e-30))
    rig.attend(np.zeros((fresh, 4, 128), np.float32))


@pytest.mark.parametrize("fresh", [3, 90])
def test_masked_places_may_hold_anything(gpu, rs, fresh):
    """NaN in blocks past a query's own position leaves it alone; a query that sees one is NaN; one query's NaN stays its own."""
    rig = Rig(cfg(4, 2, 64), 40, 16, 1, 600)
    rig.fill(rs, [0], [32])
    rig.plan([0], [fresh])
    k, v = (rs.randn(fresh, 2, 64).astype(np.float32) for _ in "kv")
    rig.store(None, k, v)
    q = rs.randn(fresh, 4, 64).astype(np.float32)
    q[1, 2] = np.nan
    q[0, 1, 5] = np.inf
    want = rig.attend(q, check=False)
    assert np.isnan(want[1, 2]).all() and np.isnan(want[0, 1]).all() and np.isfinite(np.delete(want, [0, 1], 0)).all()
    assert np.isfinite(want[1, [0, 1, 3]]).all()
    if fresh > 16:
        k[80, 0, 0] = np.nan
        v[81, 1, 0] = np.inf
        rig.plan([0], [fresh], [32])
        rig.store(None, k, v)
        got = rig.attend(q, check=False)
        np.testing.assert_array_equal(got[:80 - 80 % 16], want[:80 - 80 % 16])
        assert np.isnan(got[80:, :2]).all() and np.isnan(got[81:, 2:]).all()


def test_single_tokens_do_not_depend_on_the_batch(gpu, rs):
    past = [3, 700, 64, 2000, 130]
    rig = Rig(cfg(8, 2, 128), 300, 16, 6, 2100)
    rig.fill(rs, [0, 1, 2, 3, 4], past)
    rig.plan([0, 1, 2, 3, 4], [1] * 5)
    q, k, v = (rs.randn(5, h, 128).astype(np.float32) for h in (8, 2, 2))
    rig.store(None, k, v)
    together = rig.attend(q)
    for i in range(5):
        rig.plan([i], [1], [past[i]], outputs=False)
        rig.store(None, k[i:i + 1], v[i:i + 1])
        np.testing.assert_array_equal(rig.attend(q[i:i + 1])[0], together[i])
    rig.fill(rs, [5], [900])  # beside a prompt
    rig.plan([5, 3], [800, 1], [100, past[3]])
    x = [np.concatenate([rs.randn(800, h, 128).astype(np.float32), y[3:4]]) for h, y in ((8, q), (2, k), (2, v))]
    rig.store(None, x[1], x[2])
    np.testing.assert_array_equal(rig.attend(x[0])[800], together[3])


@pytest.mark.parametrize("fresh", [1, 60])
def test_parts_of_an_earlier_call_are_not_seen(gpu, rs, fresh):
    """Split tiles' partial results, whose places every call uses again, with other queries each time."""
    rig = Rig(cfg(8, 2, 128), 1300, 16, 3, 9100, 20000)
    rig.fill(rs, [0, 1, 2], [9000, 3000, 1030])
    rig.fill(rs, [0, 1, 2], [fresh] * 3)
    q = [rs.randn(3 * fresh, 8, 128).astype(np.float32) * s for s in (1, 3, 0.1)]
    first = [rig.attend(x) for x in q]
    dq = [rig.dev(x) for x in q]
    out = [rig.t.empty_like(dq[0]) for _ in range(60)]
    rig.t.cuda.synchronize()
    for i in range(60):
        rig.p.attend_device(0, dq[i % 3].data_ptr(), out[i].data_ptr())
    rig.p.sync()
    for i in range(60):
        np.testing.assert_array_equal(out[i].cpu().numpy(), first[i % 3])


def test_two_caches_at_once(gpu, rs):
    """Handles have their own streams and workspaces."""
    rigs = [Rig(cfg(8, 2, 128), 200, 16, 4, 800) for _ in range(2)]
    q = [rs.randn(4, 8, 128).astype(np.float32) for _ in rigs]
    alone = []
    for rig, x in zip(rigs, q):
        rig.fill(rs, [0, 1, 2, 3], [500, 3, 700, 64])
        rig.fill(rs, [0, 1, 2, 3], [1] * 4)
        alone.append(rig.attend(x))
    dq = [rig.dev(x) for rig, x in zip(rigs, q)]
    out = [[rig.t.empty_like(x) for _ in range(20)] for rig, x in zip(rigs, dq)]
    rigs[0].t.cuda.synchronize()
    for i in range(20):
        for rig, x, o in zip(rigs, dq, out):
            rig.p.attend_device(0, x.data_ptr(), o[i].data_ptr())
    for rig, o, want in zip(rigs, out, alone):
        rig.p.sync()
        for y in o:
            np.testing.assert_array_equal(y.cpu().numpy(), want)


def test_a_step_is_captured_and_replayed(gpu, rs):
    """plan, store and attend in a HIP graph, replayed with other lengths, queries and values in the same arrays."""
    hip = ctypes.CDLL("libamdhip64.so.7")  # the runtime that the library has loaded
    rig = Rig(cfg(8, 2, 128, rope=128), 120, 16, 3, 700)
    ref = Rig(cfg(8, 2, 128, rope=128), 120, 16, 3, 700)
    seed = rs.randint(1 << 30)
    for r in (rig, ref):
        r.fill(np.random.RandomState(seed), [0, 1, 2], [70, 15, 400])
    n, t = 40, rig.t
    request, fresh = rig.ints([2, 0, 1]), rig.ints([1, 1, 1])
    q, out, rot = t.zeros((n, 8, 128), device="cuda"), t.full((n, 8, 128), -7.0, device="cuda"), t.zeros((n, 8, 128), device="cuda")
    k, v = t.zeros((n, 2, 128), device="cuda"), t.zeros((n, 2, 128), device="cuda")
    t.cuda.synchronize()
    stream, graph, ex = ctypes.c_void_p(rig.p.stream), ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 2) == 0  # relaxed: other threads' calls are their own
    rig.p.plan_device(request.data_ptr(), 0, fresh.data_ptr(), 3, n)
    rig.p.store_device(0, q.data_ptr(), 1024, k.data_ptr(), v.data_ptr(), 256, rot.data_ptr())
    rig.p.attend_device(0, rot.data_ptr(), out.data_ptr())
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(ex), graph, None, None, 0) == 0
    for more in ([1, 1, 1], [1, 30, 0], [1, 1, 1], [0, 2, 38], [0, 0, 0], [1, 1, 1]):
        total = sum(more)
        xs = [rs.randn(total, h, 128).astype(np.float32) for h in (8, 2, 2)]
        for dst, x in zip((q, k, v), xs):
            dst[:total] = rig.dev(x)
        fresh.copy_(rig.ints(more))
        out.fill_(-7.0)
        t.cuda.synchronize()
        assert hip.hipGraphLaunch(ex, stream) == 0
        rig.p.sync()
        ref.plan([2, 0, 1], more, outputs=False, pad=n - total)
        got = out.cpu().numpy()
        assert np.all(got[total:] == -7)
        y = ref.store(*xs)
        np.testing.assert_array_equal(got[:total], ref.attend(y.cpu().numpy()[:total]))
    rig.t.cuda.synchronize()
    assert hip.hipGraphExecDestroy(ex) == 0 and hip.hipGraphDestroy(graph) == 0


def test_many_steps_in_a_row(gpu, rs):
    """A prompt, then tokens one by one, each step over what the last one left."""
    rig = Rig(cfg(4, 2, 64, rope=64), 64, 32, 2, 512)
    for fresh in [(57, 3)] + [(1, 1)] * 9 + [(20, 0), (1, 1), (0, 33), (1, 1)]:
        rig.plan([0, 1], list(fresh), outputs=False)
        n = sum(fresh)
        y = rig.store(rs.randn(n, 4, 64).astype(np.float32), rs.randn(n, 2, 64).astype(np.float32), rs.randn(n, 2, 64).astype(np.float32))
        rig.attend(y.cpu().numpy()[:n])
    rig.check_values()


@pytest.mark.parametrize("eager", [([0], [1]), (list(range(12)), [1] * 12), ([0], [40]), ([], [])])
@pytest.mark.parametrize("replayed", [([1, 2, 0, 3], [1, 1, 1, 1]), ([2, 3], [30, 1]), ([2], [9])])
def test_calls_for_a_smaller_plan_than_the_replayed_one(gpu, rs, eager, replayed):
    """A graph's plan, replayed after a plan call of other sizes: the calls after it do all of it or nothing."""
    hip = ctypes.CDLL("libamdhip64.so.7")
    rig = Rig(cfg(8, 2, 64, rope=64), 80, 16, 12, 300)
    rig.fill(rs, list(range(12)), [50, 20, 70, 16] + [5] * 8)
    t, n, stream = rig.t, sum(replayed[1]), ctypes.c_void_p(rig.p.stream)
    request, fresh = rig.ints(replayed[0]), rig.ints(replayed[1])
    graph, ex = ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    rig.p.plan_device(request.data_ptr(), 0, fresh.data_ptr(), len(replayed[0]), n)
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(ex), graph, None, None, 0) == 0
    rig.plan(eager[0], eager[1], outputs=False)
    assert hip.hipGraphLaunch(ex, stream) == 0
    rig.p.sync()
    assert rig.table.plan(list(replayed[0]), None, list(replayed[1]), n)[0] == 0
    # 64 rows are there, so a call that went too far would show and not fault
    q, k, v = (t.as_tensor(rs.randn(64, h, 64).astype(np.float32), device="cuda") for h in (8, 2, 2))
    rot, out = t.full((64, 8, 64), -7.0, device="cuda"), t.full((64, 8, 64), -7.0, device="cuda")
    # requests of more than 16 rows (4 tokens here) get wide tiles, where a plan call has more tokens than requests
    fits = [n <= sum(eager[1]) and len(replayed[0]) <= len(eager[0])]
    fits.append(fits[0] and (max(replayed[1]) <= 4 or sum(eager[1]) > len(eager[0])))
    for ok, got, call in ((fits[0], rot, lambda: rig.p.store_device(0, q.data_ptr(), 512, k.data_ptr(), v.data_ptr(), 128, rot.data_ptr())),
                          (fits[1], out, lambda: rig.p.attend_device(0, q.data_ptr(), out.data_ptr()))):
        call()
        if ok:
            rig.p.sync()
        else:
            with pytest.raises(jev.JevError) as e:
                rig.p.sync()
            assert e.value.code == 6
        y = got.cpu().numpy()
        assert np.all(y[n if ok else 0:] == -7) and (not ok or not np.any(y[:n] == -7))
    rig.plan([1], [3], outputs=False)  # and the next plan is as any other
    xs = [rs.randn(3, h, 64).astype(np.float32) for h in (8, 2, 2)]
    rig.store(*xs)
    t.cuda.synchronize()
    assert hip.hipGraphExecDestroy(ex) == 0 and hip.hipGraphDestroy(graph) == 0


@pytest.mark.parametrize("fresh", [1, 40])
def test_pages_past_32_bit_offsets(gpu, rs, fresh):
    """A pool whose codes lie past 2^32 bytes, after a plan of the most tokens there can be: its tiles' keys
    are 2^37, and a part's share of them is past 32 bits."""
    n = 1 << 22
    rig = Rig(cfg(8, 8, 128), (n >> 8) + 8, 256, 2, n, n)  # 1024 bytes a token: request 0 takes the first 2^32
    request, count = rig.ints([0]), rig.ints([n])
    rig.p.plan_device(request.data_ptr(), 0, count.data_ptr(), 1, n)
    rig.p.sync()
    rig.table.own[0], rig.table.length[0] = list(range(n >> 8)), n
    rig.fill(rs, [1], [300], check=True)
    assert min(rig.table.own[1]) == n >> 8
    rig.plan([1], [fresh], outputs=False)
    x = [rs.randn(fresh, 8, 128).astype(np.float32) for _ in "qkv"]
    rig.store(*x)
    rig.check_values()
    rig.attend(x[0])


def test_more_tiles_than_workgroups(gpu, rs):
    """As many requests as there can be, some in parts: the workgroups of the 16-row tiles take turns."""
    rig = Rig(cfg(2, 1, 64), 9000, 16, 4096, 3000, 40000)
    lens = rs.randint(0, 9, 4096)
    lens[rs.permutation(4096)[:9]] = rs.randint(1024, 2999, 9)
    for part in np.array_split(np.arange(4096), 2):
        rig.fill(rs, [int(r) for r in part], [int(x) for x in lens[part]])
    rig.fill(rs, list(range(4096)), [1] * 4096)
    rig.attend(rs.randn(4096, 2, 64).astype(np.float32))


@pytest.mark.parametrize("fresh", [[1, 1], [70, 3]])
def test_attention_and_reading_at_any_alignment(gpu, rs, fresh):
    rig = Rig(cfg(8, 2, 128), 200, 32, 2, 3000)
    rig.fill(rs, [0, 1], [1500, 40])
    rig.fill(rs, [0, 1], fresh)
    t, n = rig.t, sum(fresh)
    q = rs.randn(n, 8, 128).astype(np.float32)
    want = rig.attend(q)
    slots = rig.ints([rig.table.own[0][i // 32] * 32 + i % 32 for i in range(37)])
    kv = rig.kv[0, 0, "k"].values(37), rig.kv[0, 0, "v"].values(37)
    for lead in (1, 2, 3):
        x, out = (t.full((lead + n * 1024 + 4,), -7.0, device="cuda") for _ in "qo")
        k, v = (t.full((lead + 37 * 256 + 4,), -7.0, device="cuda") for _ in "kv")
        x[lead:lead + n * 1024] = rig.dev(q).reshape(-1)
        t.cuda.synchronize()
        rig.p.attend_device(0, x.data_ptr() + 4 * lead, out.data_ptr() + 4 * lead)
        rig.p.read_device(0, slots.data_ptr(), 37, k.data_ptr() + 4 * lead, v.data_ptr() + 4 * lead)
        rig.p.sync()
        for y, w in ((out, want), (k, kv[0]), (v, kv[1])):
            y = y.cpu().numpy()
            np.testing.assert_array_equal(y[lead:-4], np.ravel(w))
            assert np.all(y[:lead] == -7) and np.all(y[-4:] == -7)


def test_parts_of_very_long_contexts(gpu, rs):
    """Past 131072 tokens a part is a share of the length."""
    rig = Rig(cfg(2, 1, 64), 9000, 16, 1, 143000, 143000)
    rig.fill(rs, [0], [142001])
    rig.fill(rs, [0], [1])
    rig.attend(rs.randn(1, 2, 64).astype(np.float32))
    rig.fill(rs, [0], [40])
    rig.attend(rs.randn(40, 2, 64).astype(np.float32))
