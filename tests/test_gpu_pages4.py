"""The 4-bit paged cache on the GPU against its 64-bit statement (tests/pages4_ref.py).

Stored values are compared bit for bit: rotation is 64-bit up to one rounding, and steps and
codes are whole numbers by exact comparisons, so what is read is determined.  Attention is
held to the bounds of the 8-bit cache's tests (tests/pages_ref.py's `attend`): a query row is
an fp16 pair here too (its scale takes one more rounding, 2^-24), codes times steps are exact
in fp16, a weight is a pair truncated at 2^-21."""
import ctypes

import numpy as np
import pytest

import jev
import pages4_ref as R4
import pages_ref as R
from test_gpu_pages import Rig, cfg

pytestmark = pytest.mark.gpu


# A context of which no call is small enough to go without wide tiles.
ROOMY = 1 << 20


class Rig4(Rig):
    def __init__(self, config, n_pages, page=16, requests=8, context=4096, tokens=4096, half=False):
        import torch

        self.t, self.c, self.half = torch, config, half
        self.p = jev.KvPages(config, n_pages, page, requests, context, tokens, half, bits=4)
        self.table = R.Table(n_pages, page, requests, context)
        self.kv = R4.Cache(config.n_kv_heads, config.head_dim)

    def place(self, r, i):
        page = self.table.page
        return self.table.own[r][i // page] * page + i % page


@pytest.fixture
def rs():
    return np.random.RandomState(27)


# ---------------------------------------------------------------- store and read


@pytest.mark.parametrize("dim,page,rope,half", [(128, 16, 128, False), (128, 64, 32, True), (128, 256, 20, True), (64, 32, 0, False), (64, 256, 60, True),
                                                (64, 16, 64, False)])
def test_stored_values(gpu, rs, dim, page, rope, half):
    """Steps of uneven sizes, rows of any magnitude: blocks begun and filled, vector and single accesses."""
    rig = Rig4(cfg(4, 2, dim, rope=rope), 40 + 4000 // page, page, 5, 900, half=half)
    for fresh in ([1, 5, 16, 0, 33], [1, 1, 1, 1, 1], [15, 11, 1, 200, 0], [1, 1, 16, 17, 31]):
        rig.plan([3, 0, 4, 1, 2], fresh, outputs=False)
        n = sum(fresh)
        k, v = (rs.randn(n, 2, dim).astype(np.float32) * np.exp2(rs.randint(-9, 10, (n, 1, 1))).astype(np.float32) for _ in "kv")
        k *= np.exp2(rs.randint(-3, 4, (1, 2, dim))).astype(np.float32)
        rig.store(rs.randn(n, 4, dim).astype(np.float32), k, v, lead=int(rs.randint(2)), gap=int(rs.choice([0, 4, 3])))
        rig.check_values()


def special(rs, dim):
    """Rows whose steps and codes lie on borders: zeros, one sign, exact halves, the largest and smallest numbers."""
    x = rs.randn(144, 2, dim).astype(np.float32)
    x[0:8] = 0
    x[8:16, :, :32] = 0
    x[16:32] = rs.randint(-14, 15, (16, 2, dim)) / 2.0  # halves
    x[16:32, :, ::32], x[16:32, :, 1::32] = 8, -7
    x[32:40] *= 1e37
    x[40:44] = 3.4e38 * np.sign(x[40:44])  # a span past fp32's range
    x[44:48] *= 1e-39
    x[48:52] = 2.0 ** -149
    x[52:56] *= 2.0 ** -126
    x[56:64] = np.abs(x[56:64])
    x[64:72] = -np.abs(x[64:72])
    x[72:80] = 225.0
    x[80:88] = rs.randint(-112, 114, (8, 2, dim))
    x[80:88, :, 5], x[80:88, :, 6] = 112.5, -112.5  # a span of exactly 225
    x[88:96, :, 5], x[88:96, :, 6] = np.nextafter(np.float32(113), np.float32(200)), -112
    for i in range(96, 111):  # group spans of exactly 15 u, and a bit more
        x[i] = rs.randint(-1, 2, (2, dim))
        x[i, :, 0], x[i, :, 33], x[i, :, 34] = 225, (i - 95) * 15 - 3, -3
    x[111] = x[110]
    x[111, :, 33] = np.nextafter(x[110, :, 33], np.float32(999))
    x[112:128] = np.ldexp(1.0, rs.randint(-60, 60, (16, 2, dim))) * np.sign(x[112:128])
    x[128] = 1.0
    x[129] = -0.0
    return x


@pytest.mark.parametrize("dim", [64, 128])
def test_special_values(gpu, rs, dim):
    rig = Rig4(cfg(2, 2, dim), 40, 16, 2, 320)
    x = special(rs, dim)
    rig.plan([1], [len(x)])
    rig.store(None, x, x[::-1].copy())
    rig.check_values()


@pytest.mark.parametrize("dim", [64, 128])
def test_a_value_that_is_not_finite_is_its_tokens_alone(gpu, rs, dim):
    """K or V of one head: that token and head read as NaN, both sides; others, and the other head, as they are."""
    rig = Rig4(cfg(2, 2, dim), 40, 16, 2, 320)
    k, v = (rs.randn(50, 2, dim).astype(np.float32) for _ in "kv")
    k[7, 0, 3], v[20, 1, dim - 1], k[33, 1, 40], v[33, 0, 0] = np.nan, np.inf, -np.inf, np.nan
    rig.plan([1], [50])
    rig.store(None, k, v)
    rig.check_values()
    assert sum(np.isnan(rig.kv[1, 0, "k"].values(50)).any(-1).ravel()) == 4
    rig.fill(rs, [1], [20], [33], check=True)  # over it again


def test_cut_back_requests_share_the_pool(gpu, rs):
    rig = Rig4(cfg(2, 1, 128), 14, 16, 3, 192)  # all 14 pages in the end: 61, 70 and 67 tokens
    rig.fill(rs, [0, 1], [100, 60], check=True)
    rig.fill(rs, [0, 2], [3, 66], [37, 0], spread=0.1, check=True)
    rig.fill(rs, [1, 0, 2], [1, 30, 1], check=True)
    rig.fill(rs, [1], [60], [0], check=True)


def test_layers_are_apart(gpu, rs):
    rig = Rig4(cfg(2, 1, 64, layers=3), 6, 32, 2, 96)
    rig.plan([1, 0], [40, 7])
    for layer in (2, 0, 1):
        k, v = (rs.randn(47, 1, 64).astype(np.float32) * (layer + 1) for _ in "kv")
        rig.store(None, k, v, layer)
    for layer in range(3):
        rig.check_values(layer)
        rig.attend(rs.randn(47, 2, 64).astype(np.float32), layer)


def test_reading_outside_the_pool_and_before_a_store(gpu, rs):
    rig = Rig4(cfg(1, 1, 64), 3, 16, 1, 48)
    slots = rig.ints([-1, 48, 2 ** 31 - 1, -2 ** 31, 47])
    k = rig.t.full((5, 64), -7.0, device="cuda")
    v = k.clone()
    rig.p.read_device(0, slots.data_ptr(), 5, k.data_ptr(), v.data_ptr())
    rig.p.sync()
    assert bool((k == 0).all()) and bool((v == 0).all())  # a new pool holds zeros
    rig.fill(rs, [0], [48])
    rig.p.read_device(0, slots.data_ptr(), 5, k.data_ptr(), v.data_ptr())
    rig.p.sync()
    assert bool((k[:4] == 0).all()) and bool((v[:4] == 0).all()) and bool((k[4] != 0).any())


def test_a_token_reads_the_same_whatever_is_stored_beside_it(gpu, rs):
    """One prompt, or the same tokens one by one: the same values, and the same attention of the last."""
    rigs = [Rig4(cfg(8, 2, 128, rope=128), 20, 16, 1, 200) for _ in range(2)]
    q, k, v = (rs.randn(40, h, 128).astype(np.float32) for h in (8, 2, 2))
    got = []
    for rig, steps in zip(rigs, ([40], [1] * 40)):
        at = 0
        for n in steps:
            rig.plan([0], [n], outputs=False)
            y = rig.store(q[at:at + n], k[at:at + n], v[at:at + n])
            at += n
        rig.check_values()
        if len(steps) == 1:
            rig.plan([0], [1], [39], outputs=False)
            y = rig.store(q[39:], k[39:], v[39:])
        got.append(rig.attend(y.cpu().numpy()[-1:]))
    np.testing.assert_array_equal(got[0], got[1])


# ---------------------------------------------------------------- attention


@pytest.mark.parametrize("heads,kv,dim", [(4, 1, 128), (8, 8, 64), (7, 1, 64), (32, 2, 128), (20, 1, 128), (48, 1, 64), (6, 2, 128), (9, 1, 128)])
@pytest.mark.parametrize("page", [16, 128])
def test_single_tokens(gpu, rs, heads, kv, dim, page):
    """One token a request over lengths about every border."""
    past = [0, 1, 14, 15, 16, 62, 63, 64, 65, 127, 255, 256, 257, 300, 511, 513, 700, 1025]
    rig = Rig4(cfg(heads, kv, dim), 600 if page == 16 else 120, page, len(past), 1100, 8000)
    rig.fill(rs, list(range(len(past))), past)
    ids = [int(i) for i in rs.permutation(len(past))]
    rig.fill(rs, ids, [1] * len(past))
    rig.attend(rs.randn(len(past), heads, dim).astype(np.float32))


@pytest.mark.parametrize("heads,kv,dim", [(4, 1, 128), (3, 3, 64), (10, 2, 128), (16, 1, 64), (40, 2, 128), (8, 2, 64)])
@pytest.mark.parametrize("context", [500, ROOMY])
def test_prompts(gpu, rs, heads, kv, dim, context):
    """Ragged batches: nothing, single tokens, a few, more than a tile of any width, behind pasts of any length."""
    past = [0, 5, 0, 63, 300, 129, 0, 17]
    fresh = [1, 130, 0, 2, 33, 64, 301, 4]
    rig = Rig4(cfg(heads, kv, dim), 200, 16, 8, context)
    rig.fill(rs, list(range(8)), past)
    rig.plan([6, 1, 2, 0, 7, 4, 5, 3], [fresh[i] for i in (6, 1, 2, 0, 7, 4, 5, 3)], pad=5)
    n = sum(fresh)
    rig.store(None, rs.randn(n, kv, dim).astype(np.float32), rs.randn(n, kv, dim).astype(np.float32))
    rig.attend(rs.randn(n, heads, dim).astype(np.float32))


@pytest.mark.parametrize("fresh", range(1, 10))
def test_a_few_tokens(gpu, rs, fresh):
    """Two to 36 rows of a KV head: tiles of eight rows and of sixteen, several of them."""
    for heads, dim in ((8, 128), (4, 64)):
        rig = Rig4(cfg(heads, 2, dim), 300, 32, 3, 1500)
        rig.fill(rs, [0, 1, 2], [1200, 64, 0])
        rig.fill(rs, [2, 0, 1], [fresh] * 3)
        rig.attend(rs.randn(3 * fresh, heads, dim).astype(np.float32))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("context", [41000, ROOMY])
def test_long_contexts(gpu, rs, context, dim):
    """Parts of five lengths and more: rows of one token, two, three, and of several tiles."""
    for past in (5000, 40000):
        rig = Rig4(cfg(4, 1, dim), 2600, 16, 1, context, 41000)
        rig.fill(rs, [0], [past])
        for fresh in (1, 2, 3, 30, 70):
            rig.fill(rs, [0], [fresh])
            rig.attend(rs.randn(fresh, 4, dim).astype(np.float32))


@pytest.mark.parametrize("context", [143000, ROOMY])
def test_parts_of_very_long_contexts(gpu, rs, context):
    rig = Rig4(cfg(2, 1, 64), 9000, 16, 1, context, 143000)
    rig.fill(rs, [0], [142001])
    rig.fill(rs, [0], [1])
    rig.attend(rs.randn(1, 2, 64).astype(np.float32))
    for fresh in (40, 200):
        rig.fill(rs, [0], [fresh])
        rig.attend(rs.randn(fresh, 2, 64).astype(np.float32))


@pytest.mark.parametrize("fresh,context", [(1, 600), (90, 600), (150, 600), (150, ROOMY)])
def test_scales_far_apart(gpu, rs, fresh, context):
    """Queries and values far from one: the pairs stay inside fp16's range by powers of two."""
    rig = Rig4(cfg(4, 2, 128), 40, 16, 1, context)
    n = 400 + fresh
    k = rs.randn(n, 2, 128).astype(np.float32) * np.float32(1e-18)
    v = rs.randn(n, 2, 128).astype(np.float32) * np.exp2(rs.randint(-100, 100, (n, 1, 1))).astype(np.float32)
    rig.plan([0], [400])
    rig.store(None, k[:400], v[:400])
    rig.plan([0], [fresh])
    rig.store(None, k[400:], v[400:])
    rig.attend(rs.randn(fresh, 4, 128).astype(np.float32) * np.float32(1e18))
    rig.attend(rs.randn(fresh, 4, 128).astype(np.float32) * np.float32(1e-30))
    rig.attend(np.zeros((fresh, 4, 128), np.float32))


@pytest.mark.parametrize("context", [3000, ROOMY])
def test_many_tokens_of_one_among_idle_requests(gpu, rs, context):
    """No more tokens than requests, nearly all of them one request's: tiles of sixteen rows whose keys are split, or,
    where the context may be long, are not."""
    rig = Rig4(cfg(8, 2, 128), 300, 16, 64, context)
    rig.fill(rs, list(range(64)), [2500] + [16] * 63)
    rig.plan(list(range(64)), [60] + [0] * 61 + [1, 3])
    rig.store(None, *(rs.randn(64, 2, 128).astype(np.float32) for _ in "kv"))
    rig.attend(rs.randn(64, 8, 128).astype(np.float32))


@pytest.mark.parametrize("n", [30, 203, 206])
def test_drafts_of_few_and_of_many_requests(gpu, rs, n):
    """Five tiles of sixteen rows a request: up to 1024 of them a KV head, and wide tiles where there are more; beside a
    prompt, a single token, a few, and nothing."""
    rig = Rig4(cfg(8, 2, 64), 4000, 16, n + 4, 1500, 40000)
    past = [int(x) for x in rs.randint(0, 200, n + 4)]
    past[5], past[-1] = 1040, 30  # (in two parts)
    rig.fill(rs, list(range(n + 4)), past)
    fresh = [17 + i % 4 for i in range(n)] + [1, 300, 0, 3]
    rig.plan(list(range(n + 4)), fresh)
    total = sum(fresh)
    rig.store(None, *(rs.randn(total, 2, 64).astype(np.float32) for _ in "kv"))
    rig.attend(rs.randn(total, 8, 64).astype(np.float32))


@pytest.mark.parametrize("scale", [1e-37, 1e-25, 1e25])
@pytest.mark.parametrize("context", [200, ROOMY])
def test_queries_and_keys_at_the_ends_of_the_range(gpu, rs, scale, context):
    """Small queries over large keys and the other way round: their product is what counts."""
    rig = Rig4(cfg(8, 2, 64), 40, 16, 1, context)
    k, v = (rs.randn(90, 2, 64).astype(np.float32) for _ in "kv")
    rig.plan([0], [90])
    rig.store(None, k * np.float32(scale), v)
    rig.attend(rs.randn(90, 8, 64).astype(np.float32) * np.float32(1.0 / np.float32(scale)))


@pytest.mark.parametrize("fresh,context", [(2, 600), (4, 600), (90, 600), (150, 600), (150, ROOMY)])
def test_masked_places_may_hold_anything(gpu, rs, fresh, context):
    """NaN past a query's own position leaves it alone; a query that sees one is NaN; one query's NaN stays its own."""
    rig = Rig4(cfg(4, 2, 64), 40, 16, 1, context)
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
    at = fresh * 7 // 8  # not the first
    for bad_k, bad_v in (((at, 0, 0), None), (None, (at, 0, 63)), ((at, 0, 5), (at, 0, 6))):
        kb, vb = k.copy(), v * np.float32(1e30)  # beside values whose power is near the largest
        for x, i in ((kb, bad_k), (vb, bad_v)):
            if i:
                x[i] = np.nan
        rig.plan([0], [fresh], [32])
        rig.store(None, k, v * np.float32(1e30))
        clean = rig.attend(q, check=False)
        rig.plan([0], [fresh], [32])
        rig.store(None, kb, vb)
        got = rig.attend(q, check=False)
        np.testing.assert_array_equal(got[:at], clean[:at])
        assert np.isnan(got[at:, :2]).all()
        np.testing.assert_array_equal(got[at:, 2:], clean[at:, 2:])


@pytest.mark.parametrize("context", [2100, ROOMY])
def test_single_tokens_do_not_depend_on_the_batch(gpu, rs, context):
    past = [3, 700, 64, 2000, 130]
    rig = Rig4(cfg(8, 2, 128), 300, 16, 6, context)
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


@pytest.mark.parametrize("fresh", [2, 3, 4])
@pytest.mark.parametrize("context", [2500, ROOMY])
def test_a_few_tokens_do_not_depend_on_the_batch(gpu, rs, fresh, context):
    """Alone, beside a prompt, beside many drafts: up to sixteen rows of a KV head have the same bits."""
    for dim in (64, 128):
        rig = Rig4(cfg(8, 2, dim), 1000, 16, 210, context, 8000)
        rig.fill(rs, [0], [2100])
        x = [rs.randn(fresh, h, dim).astype(np.float32) for h in (8, 2, 2)]
        rig.plan([0], [fresh])
        rig.store(None, *x[1:])
        alone = rig.attend(x[0])
        for ids, more in (([1], [800]), (list(range(1, 210)), [17] * 209), ([5], [1])):
            rig.plan([0] + ids, [fresh] + more, [2100] + [0] * len(ids))
            y = [np.concatenate([a, rs.randn(sum(more), *a.shape[1:]).astype(np.float32)]) for a in x]
            rig.store(None, *y[1:])
            np.testing.assert_array_equal(rig.attend(y[0], check=False)[:fresh], alone)


@pytest.mark.parametrize("fresh,context", [(1, 9100), (4, 9100), (60, 9100), (80, 9100), (60, ROOMY), (80, ROOMY)])
def test_parts_of_an_earlier_call_are_not_seen(gpu, rs, fresh, context):
    rig = Rig4(cfg(8, 2, 128), 1300, 16, 3, context, 20000)
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
    """A 4-bit and an 8-bit cache: handles have their own streams and workspaces."""
    rigs = [Rig4(cfg(8, 2, 128), 200, 16, 4, 800), Rig(cfg(8, 2, 128), 200, 16, 4, 800)]
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
    rig, ref = (Rig4(cfg(8, 2, 128, rope=128), 120, 16, 3, 700) for _ in range(2))
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
    for more in ([1, 1, 1], [1, 30, 0], [1, 1, 1], [0, 2, 38], [0, 0, 0], [1, 1, 1], [3, 4, 5]):
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


def test_a_graph_replayed_with_few_and_many_drafts(gpu, rs):
    """A captured plan and attention whose replays have 16-row tiles of all requests, wide ones, none, and both."""
    hip = ctypes.CDLL("libamdhip64.so.7")
    R_, n = 220, 5000
    rig, ref = (Rig4(cfg(8, 2, 64), 1200, 16, R_, 400, n) for _ in range(2))
    past = [int(x) for x in rs.randint(0, 30, R_)]
    seed = rs.randint(1 << 30)
    for r in (rig, ref):
        r.fill(np.random.RandomState(seed), list(range(R_)), past)
    t = rig.t
    request, kept, fresh = rig.ints(list(range(R_))), rig.ints(past), rig.ints([1] * R_)
    q, out = t.zeros((n, 8, 64), device="cuda"), t.full((n, 8, 64), -7.0, device="cuda")
    k, v = t.zeros((n, 2, 64), device="cuda"), t.zeros((n, 2, 64), device="cuda")
    t.cuda.synchronize()
    stream, graph, ex = ctypes.c_void_p(rig.p.stream), ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 2) == 0  # relaxed: other threads' calls are their own
    rig.p.plan_device(request.data_ptr(), kept.data_ptr(), fresh.data_ptr(), R_, n)
    rig.p.store_device(0, 0, 0, k.data_ptr(), v.data_ptr(), 128, 0)
    rig.p.attend_device(0, q.data_ptr(), out.data_ptr())
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(ex), graph, None, None, 0) == 0
    for more in ([20] * R_, [20] * 30 + [0] * 190, [1] * R_, [0] * R_, [300] + [3] * 100 + [18] * 119, [20] * R_):
        total = sum(more)
        xs = [rs.randn(total, h, 64).astype(np.float32) for h in (8, 2, 2)]
        for dst, x in zip((q, k, v), xs):
            dst[:total] = rig.dev(x)
        fresh.copy_(rig.ints(more))
        out.fill_(-7.0)
        t.cuda.synchronize()
        assert hip.hipGraphLaunch(ex, stream) == 0
        rig.p.sync()
        ref.plan(list(range(R_)), more, past, outputs=False, pad=n - total)
        got = out.cpu().numpy()
        assert np.all(got[total:] == -7)
        ref.store(None, *xs[1:])
        np.testing.assert_array_equal(got[:total], ref.attend(xs[0]))
    rig.t.cuda.synchronize()
    assert hip.hipGraphExecDestroy(ex) == 0 and hip.hipGraphDestroy(graph) == 0


@pytest.mark.parametrize("fresh,context", [([1, 1], 3000), ([30, 3], 3000), ([70, 3], 3000), ([70, 3], ROOMY)])
def test_attention_and_reading_at_any_alignment(gpu, rs, fresh, context):
    rig = Rig4(cfg(8, 2, 128), 200, 32, 2, context)
    rig.fill(rs, [0, 1], [1500, 40])
    rig.fill(rs, [0, 1], fresh)
    t, n = rig.t, sum(fresh)
    q = rs.randn(n, 8, 128).astype(np.float32)
    want = rig.attend(q)
    slots = rig.ints([rig.place(0, i) for i in range(37)])
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


@pytest.mark.parametrize("fresh", [1, 40, 300])
def test_pages_past_32_bit_offsets(gpu, rs, fresh):
    """A pool whose codes lie past 2^32 bytes."""
    n = 1 << 22
    rig = Rig4(cfg(8, 8, 128), (n >> 8) + 8, 256, 2, n, n)  # 1104 bytes a token: request 0 takes the first 2^32
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
    rig = Rig4(cfg(2, 1, 64), 9000, 16, 4096, 3000, 40000)
    lens = rs.randint(0, 9, 4096)
    lens[rs.permutation(4096)[:9]] = rs.randint(1024, 2999, 9)
    for part in np.array_split(np.arange(4096), 2):
        rig.fill(rs, [int(r) for r in part], [int(x) for x in lens[part]])
    rig.fill(rs, list(range(4096)), [1] * 4096)
    rig.attend(rs.randn(4096, 2, 64).astype(np.float32))


@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (32, 2, 64), (20, 1, 128)])
@pytest.mark.parametrize("fresh,context", [(1, 200), (40, 200), (70, 200), (70, ROOMY)])
def test_queries_keep_their_bits(gpu, rs, heads, kv, dim, fresh, context):
    """Queries of one element: a score is one product, so its error is the query's alone: its pair (2^-21, lo's own
    rounding among it), the softmax's scale on it (2^-24, and its logarithm's factor), the exponent's rounding."""
    rig = Rig4(cfg(heads, kv, dim), 100, 16, 40, context, 3000)
    n = 20 if fresh == 1 else 2
    rig.fill(rs, list(range(n)), [60] * n)
    rig.plan(list(range(n)), [fresh] * n)
    k, v = (rs.randn(n * fresh, kv, dim).astype(np.float32) for _ in "kv")
    rig.store(None, k, v)
    q = np.zeros((n * fresh, heads, dim), np.float32)
    at = rs.randint(0, dim, q.shape[:2])
    np.put_along_axis(q, at[..., None], rs.randn(*at.shape, 1).astype(np.float32) * 40, -1)
    got, i = rig.attend(q), 0
    for r, p, f in rig.batch:
        k, v = (rig.kv[r, 0, x].values(p + f).astype(np.float64) for x in "kv")
        want, _ = R.attend(q[i:i + f], k, v, p)
        g = heads // kv
        score = np.abs(np.einsum("fhd,nhd->fhn", q[i:i + f], np.repeat(k, g, 1))).max(-1) / np.sqrt(dim)
        off = np.repeat(np.abs(v).max((0, 2)), g) * (2 * np.expm1(score * (2.0 ** -21 + 3 * 2.0 ** -24) + 2.0 ** -20) + 2.0 ** -19 + len(k) * 2.0 ** -24)
        assert np.all(np.abs(got[i:i + f] - want) <= off[..., None]), (r, np.abs(got[i:i + f] - want).max(), off.min())
        i += f


# ---------------------------------------------------------------- values far apart


def attended(rig, r, q, past):
    """Exact attention and its bound (tests/test_gpu_pages_range.py has the arithmetic; here a weight's floor is
    2^-32 of the heaviest weight times power, for each of its codes times steps)."""
    k, v = (rig.kv[r, 0, x].values(past + len(q)).astype(np.float64) for x in "kv")
    _, _, _, e = R4.quantise(v.astype(np.float32))
    power = np.ldexp(1.0, e)
    heads, d = q.shape[1:]
    g, n = heads // k.shape[1], len(k)
    out, off = np.empty(q.shape), np.empty(q.shape)
    seen = np.arange(n) <= past + np.arange(len(q))[:, None]
    for h in range(heads):
        kh, vh, ph, x = k[:, h // g], v[:, h // g], power[:, h // g], q[:, h].astype(np.float64)
        s = np.where(seen, x @ kh.T / np.sqrt(d), -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        a = np.abs(x) @ np.abs(kh).T / np.sqrt(d)
        err = np.expm1(a * (2.0 ** -21 + (d + 4) * 2.0 ** -24) + np.abs(np.where(seen, s, 0)) * 2.0 ** -22 + 2.0 ** -18) + 2.0 ** -19
        out[:, h] = p @ vh
        pe = p * err
        moved = (pe @ np.abs(vh) + pe.sum(-1, keepdims=True) * np.abs(out[:, h])) / (1 - pe.sum(-1, keepdims=True))
        off[:, h] = (moved + p @ np.abs(vh) * (n * 2.0 ** -24 + 2.0 ** -20) +
                     2.0 ** -32 * (p * ph).max(-1, keepdims=True) * (seen @ (np.abs(vh) / ph[:, None])) + 2.0 ** -140)
    return out, off


def check(rig, r, q, got, past):
    want, off = attended(rig, r, q, past)
    bad = ~(np.abs(got - want) <= off)
    assert not bad.any(), (np.argwhere(bad)[:3].tolist(), np.nanmax(np.abs(got - want) / off))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("begin", [16, 21, 48, 89])
@pytest.mark.parametrize("large", [1e6, 1e15, 1e30])
@pytest.mark.parametrize("context", [200, ROOMY])
def test_later_tokens_leave_earlier_ones_alone(gpu, rs, dim, begin, large, context):
    """A prompt whose tokens from one on, inside a block too, have far larger keys and values: the ones before have
    the bits that they have without them."""
    rig = Rig4(cfg(8, 2, dim), 20, 16, 1, context)
    q, k, v = (rs.randn(90, h, dim).astype(np.float32) for h in (8, 2, 2))
    for side in (1, 0):
        got = []
        for by in (1.0, large):
            x = [k.copy(), v.copy()]
            x[side][begin:] *= np.float32(by)
            rig.plan([0], [90], [0])
            rig.store(None, *x)
            got.append(rig.attend(q, check=False)[:begin])
            check(rig, 0, q[:begin], got[-1], 0)
        np.testing.assert_array_equal(got[1], got[0])


@pytest.mark.parametrize("fresh,context", [(1, 700), (3, 700), (90, 700), (90, ROOMY)])
@pytest.mark.parametrize("where", [(0, 16), (5, 6), (48, 64), (480, 493)])
@pytest.mark.parametrize("ratio", [2.0 ** 14, 2.0 ** 24, 2.0 ** 34, 2.0 ** 110])
@pytest.mark.parametrize("score", [0.0, 12.0, 200.0])
def test_values_far_apart(gpu, rs, fresh, context, where, ratio, score):
    """Tokens of far larger values that the softmax gives little weight, or none, before, among and beside those
    that a query attends."""
    rig = Rig4(cfg(8, 2, 128), 80, 16, 1, context)
    n, at = 496 + fresh, slice(*where)
    k, v = rs.randn(n, 2, 128).astype(np.float32) * np.float32(0.3), rs.randn(n, 2, 128).astype(np.float32)
    k[at, :, 0] = -score * np.sqrt(128) / 8
    v[at] *= np.float32(ratio)
    rig.plan([0], [496])
    rig.store(None, k[:496], v[:496])
    rig.plan([0], [fresh])
    rig.store(None, k[496:], v[496:])
    q = rs.randn(fresh, 8, 128).astype(np.float32) * np.float32(0.5)
    q[:, :, 0] = 8
    check(rig, 0, q, rig.attend(q, check=False), 496)


@pytest.mark.parametrize("fresh,context", [(1, 1200), (40, 1200), (80, 1200), (80, ROOMY)])
@pytest.mark.parametrize("ratio", [2.0 ** -60, 2.0 ** -20, 1.0, 2.0 ** 40, 2.0 ** 100])
def test_any_magnitudes(gpu, rs, fresh, context, ratio):
    """Every token's key and value row of its own magnitude, zeros among them; attended values at either end of fp32."""
    rig = Rig4(cfg(8, 2, 64), 200, 16, 1, context)
    n = 1000 + fresh
    k = rs.randn(n, 2, 64).astype(np.float32) * np.exp2(rs.uniform(-12, 0.5, (n, 2, 1))).astype(np.float32)
    v = rs.randn(n, 2, 64).astype(np.float32) * np.exp2(rs.uniform(-30, 8, (n, 2, 1))).astype(np.float32) * np.float32(ratio)
    v[rs.permutation(n)[:50]] = 0
    k[rs.permutation(n)[:50]] = 0
    rig.plan([0], [1000])
    rig.store(None, k[:1000], v[:1000])
    rig.plan([0], [fresh])
    rig.store(None, k[1000:], v[1000:])
    q = rs.randn(fresh, 8, 64).astype(np.float32) * 3
    check(rig, 0, q, rig.attend(q, check=False), 1000)


@pytest.mark.parametrize("context", [100, ROOMY])
def test_values_of_zeros_only(gpu, rs, context):
    rig = Rig4(cfg(4, 1, 64), 20, 16, 1, context)
    for fresh in (1, 50, 80):
        rig.plan([0], [fresh], [0])
        rig.store(None, rs.randn(fresh, 1, 64).astype(np.float32), np.zeros((fresh, 1, 64), np.float32))
        assert np.all(rig.attend(rs.randn(fresh, 4, 64).astype(np.float32), check=False) == 0)
