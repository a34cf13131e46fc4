"""The paged attention over values whose magnitudes lie far apart, from block to block and
against fp32's range: keys that a query cannot see, or gives no weight, cost its result nothing.

The bound, per output: with p the exact weights, a weight is off by E relative, of which
  * its score's error: q within 2^-21 of its fp16 pair, head_dim products summed in fp32
    (2^-24 each) and a few roundings of scales, all of sum |q| |k|; the exponent's roundings,
    2^-22 of |score| and 2^-18 (an argument of up to 2^5 beside the score, twice);
  * 2^-19: the pair's truncation (2^-21), its exponential and the scale on it.
An error of p_i moves the output by p_i E_i (|v_i| + |out|).  The fp32 sums over n keys are off
by n 2^-24 sum p |v| (and 2^-20 of it: rescaling and merging).  A weight smaller than the pair's
last bit, 2^-24 where the heaviest p * (V scale) is at least 2^8, loses at most that bit for
each of its codes: 2^-32 max(p * scale) sum |code|."""
import numpy as np
import pytest

import jev
import pages_ref as R
from test_gpu_pages import Rig, cfg

pytestmark = pytest.mark.gpu


def attended(rig, r, q, past, layer=0):
    """Exact attention of q [fresh, heads, dim] over request r's stored values, and its bound."""
    k, vc = rig.kv[r, layer, "k"], rig.kv[r, layer, "v"]
    n = past + len(q)
    heads, d = q.shape[1:]
    g = heads // k.code.shape[1]
    keys = k.values(n).astype(np.float64)
    scale = np.repeat(vc.scale, R.BLOCK, axis=0)[:n].astype(np.float64)
    code = vc.code[:n]
    out, off = np.empty(q.shape), np.empty(q.shape)
    seen = np.arange(n) <= past + np.arange(len(q))[:, None]
    for h in range(heads):
        kh, sh, ch = keys[:, h // g], scale[:, h // g], code[:, h // g]
        x = q[:, h].astype(np.float64)
        s = np.where(seen, x @ kh.T / np.sqrt(d), -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        a = np.abs(x) @ np.abs(kh).T / np.sqrt(d)
        e = np.expm1(a * (2.0 ** -21 + (d + 4) * 2.0 ** -24) + np.abs(np.where(seen, s, 0)) * 2.0 ** -22 + 2.0 ** -18) + 2.0 ** -19
        pv, pe = p * sh, p * e
        out[:, h] = pv @ ch
        size = pv @ np.abs(ch)
        moved = ((pe * sh) @ np.abs(ch) + pe.sum(-1, keepdims=True) * np.abs(out[:, h])) / (1 - pe.sum(-1, keepdims=True))
        off[:, h] = moved + size * (n * 2.0 ** -24 + 2.0 ** -20) + 2.0 ** -32 * pv.max(-1, keepdims=True) * (seen @ np.abs(ch)) + 2.0 ** -140
    return out, off


def check(rig, r, q, got, past):
    want, off = attended(rig, r, q, past)
    bad = ~(np.abs(got - want) <= off)
    worst = np.nanmax(np.abs(got - want) / off)
    assert not np.count_nonzero(bad), (np.argwhere(bad)[:3].tolist(), worst)


@pytest.fixture
def rs():
    return np.random.RandomState(17)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("begin", [16, 32, 48])
@pytest.mark.parametrize("large", [1e6, 1e15, 1e30])
def test_later_tokens_leave_earlier_ones_alone(gpu, rs, dim, begin, large):
    """A prompt whose tokens from a block's begin on have far larger values: the ones before have the bits that
    they have without them."""
    rig = Rig(cfg(8, 2, dim), 20, 16, 1, 200)
    q, k, v = (rs.randn(90, h, dim).astype(np.float32) for h in (8, 2, 2))
    got = []
    for by in (1.0, large):
        x = v.copy()
        x[begin:] *= np.float32(by)
        rig.plan([0], [90], [0])
        rig.store(None, k, x)
        got.append(rig.attend(q, check=False)[:begin])
        check(rig, 0, q[:begin], got[-1], 0)
    np.testing.assert_array_equal(got[1], got[0])


def keys_at(rs, n, heads, dim, score, at):
    """Keys whose scores with queries of `queries` are about `score` lower at the places `at`."""
    k = rs.randn(n, heads, dim).astype(np.float32) * np.float32(0.3)
    k[at, :, 0] = -score * np.sqrt(dim) / 8
    return k


def queries(rs, n, heads, dim):
    q = rs.randn(n, heads, dim).astype(np.float32) * np.float32(0.5)
    q[:, :, 0] = 8
    return q


@pytest.mark.parametrize("fresh", [1, 90])
@pytest.mark.parametrize("where", [(0, 16), (48, 64), (112, 128), (480, 496)])
@pytest.mark.parametrize("ratio", [2.0 ** 14, 2.0 ** 24, 2.0 ** 34, 2.0 ** 110])
@pytest.mark.parametrize("score", [0.0, 12.0, 200.0])
def test_values_far_apart(gpu, rs, fresh, where, ratio, score):
    """A block of far larger values that the softmax gives little weight, or none, before, among and after the
    blocks that a query attends."""
    rig = Rig(cfg(8, 2, 128), 80, 16, 1, 700)
    n, at = 496 + fresh, slice(*where)
    k, v = keys_at(rs, n, 2, 128, score, at), rs.randn(n, 2, 128).astype(np.float32)
    v[at] *= np.float32(ratio)
    rig.plan([0], [496])
    rig.store(None, k[:496], v[:496])
    rig.plan([0], [fresh])
    rig.store(None, k[496:], v[496:])
    q = queries(rs, fresh, 8, 128)
    check(rig, 0, q, rig.attend(q, check=False), 496)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("large", [1e6, 1e15, 1e30])
def test_values_that_grow_along_a_prompt(gpu, rs, dim, large):
    """Every row of a prompt whose first tokens, or last ones, have far larger values."""
    rig = Rig(cfg(8, 2, dim), 20, 16, 1, 200)
    for at in (slice(0, 16), slice(5, 40), slice(40, 90)):
        q, k, v = (rs.randn(90, h, dim).astype(np.float32) for h in (8, 2, 2))
        v[at] *= np.float32(large)
        rig.plan([0], [90], [0])
        rig.store(None, k, v)
        check(rig, 0, q, rig.attend(q, check=False), 0)


@pytest.mark.parametrize("dim,fresh", [(64, 1), (128, 1), (64, 70), (128, 70)])
def test_values_far_apart_in_other_parts(gpu, rs, dim, fresh):
    """The same where the large values are another part's, and every block's magnitude is its own."""
    rig = Rig(cfg(4, 1, dim), 400, 16, 1, 5200, 5200)
    n = 5000 + fresh
    block = np.arange(n) // 16
    loud = rs.randint(0, 2, block[-1] + 1)[block] * (np.arange(n) % 1024 < 600)
    k = keys_at(rs, n, 1, dim, np.where(loud, rs.choice([0, 7, 60, 300], block[-1] + 1)[block], 0)[:, None], slice(None))
    v = rs.randn(n, 1, dim).astype(np.float32) * np.exp2(np.where(loud, rs.randint(0, 100, block[-1] + 1)[block], -3)).astype(np.float32)[:, None, None]
    rig.plan([0], [5000])
    rig.store(None, k[:5000], v[:5000])
    rig.plan([0], [fresh])
    rig.store(None, k[5000:], v[5000:])
    q = queries(rs, fresh, 4, dim)
    check(rig, 0, q, rig.attend(q, check=False), 5000)


@pytest.mark.parametrize("fresh", [1, 90])
@pytest.mark.parametrize("scale", [2.0 ** -140, 2.0 ** -126, 2.0 ** -100, 0.0])
def test_the_smallest_values(gpu, rs, fresh, scale):
    """Values about fp32's smallest numbers, alone and beside ordinary ones of little weight; zeros with all of it."""
    rig = Rig(cfg(4, 2, 64), 40, 16, 1, 400)
    n, at = 300 + fresh, slice(64, 96)
    for large in (scale, 1.0):
        k, v = keys_at(rs, n, 2, 64, 60.0, at), rs.randn(n, 2, 64).astype(np.float32) * np.float32(scale)
        v[at] = rs.randn(32, 2, 64) * large
        rig.plan([0], [300], [0])
        rig.store(None, k[:300], v[:300])
        rig.plan([0], [fresh])
        rig.store(None, k[300:], v[300:])
        q = queries(rs, fresh, 4, 64)
        check(rig, 0, q, rig.attend(q, check=False), 300)


@pytest.mark.parametrize("fresh", [1, 90])
@pytest.mark.parametrize("n", [200, 1900])
@pytest.mark.parametrize("large", [1e36, 3e38])
def test_the_largest_values(gpu, rs, fresh, n, large):
    """Values about fp32's largest numbers: their sum over the keys is past it, their mean is not."""
    rig = Rig(cfg(8, 2, 128), 140, 16, 1, 2000)
    n += fresh
    k, v = (rs.randn(n, 2, 128).astype(np.float32) * np.float32(0.1) for _ in "kv")
    v = (rs.uniform(0.5, 1, (n, 2, 128)) * large).astype(np.float32)
    rig.plan([0], [n - fresh])
    rig.store(None, k[:-fresh], v[:-fresh])
    rig.plan([0], [fresh])
    rig.store(None, k[-fresh:], v[-fresh:])
    q = rs.randn(fresh, 8, 128).astype(np.float32)
    check(rig, 0, q, rig.attend(q, check=False), n - fresh)


@pytest.mark.parametrize("fresh", [1, 40])
def test_tokens_that_were_not_stored_are_zeros_in_a_new_pool(gpu, rs, fresh):
    """A layer's blocks that nothing was stored into: read and attended as zeros."""
    rig = Rig(cfg(4, 2, 64), 40, 16, 1, 400)
    rig.plan([0], [100])
    for name in "kv":
        rig.kv[0, 0, name] = R.Cache(2, 64)
        rig.kv[0, 0, name].store(0, np.zeros((100, 2, 64)))
    rig.check_values()
    q = rs.randn(100, 4, 64).astype(np.float32)
    assert not rig.attend(q).any()
    rig.plan([0], [fresh])
    rig.store(None, *(rs.randn(fresh, 2, 64).astype(np.float32) for _ in "kv"))
    rig.check_values()
    q = rs.randn(fresh, 4, 64).astype(np.float32)
    check(rig, 0, q, rig.attend(q, check=False), 100)


@pytest.mark.parametrize("fresh", [1, 90])
@pytest.mark.parametrize("large,small", [("k", "q"), ("q", "k")])
@pytest.mark.parametrize("by", [1e30, 3e37])
def test_queries_and_keys_at_the_ends_of_the_range(gpu, rs, fresh, large, small, by):
    """Scores of about one from a factor near fp32's smallest numbers and one near its largest."""
    rig = Rig(cfg(8, 2, 128), 40, 16, 1, 500)
    n = 400 + fresh
    x = {"q": rs.randn(fresh, 8, 128), "k": rs.randn(n, 2, 128), "v": rs.randn(n, 2, 128)}
    x[large] *= by
    x[small] /= by
    x = {name: y.astype(np.float32) for name, y in x.items()}
    rig.plan([0], [400])
    rig.store(None, x["k"][:400], x["v"][:400])
    rig.plan([0], [fresh])
    rig.store(None, x["k"][400:], x["v"][400:])
    check(rig, 0, x["q"], rig.attend(x["q"], check=False), 400)


@pytest.mark.parametrize("fresh", [1, 90])
@pytest.mark.parametrize("past", [40, 1500])
def test_scores_past_the_range_are_no_numbers(gpu, rs, fresh, past):
    """All scores past fp32's least number: NaN, not zeros.  Where one key has a score within the range, its value."""
    rig = Rig(cfg(4, 2, 64), 140, 16, 1, 2000)
    n = past + fresh
    k, v = np.full((n, 2, 64), -1e20, np.float32), rs.randn(n, 2, 64).astype(np.float32)
    k[16:32, 1] = 0
    v[16:32, 1] = 127 * 2.0 ** -5
    rig.plan([0], [past])
    rig.store(None, k[:past], v[:past])
    rig.plan([0], [fresh])
    rig.store(None, k[past:], v[past:])
    got = rig.attend(np.full((fresh, 4, 64), 1e20, np.float32), check=False)
    assert np.isnan(got[:, :2]).all()
    # sixteen equal weights of one value: a rounding each of their sum's parts
    np.testing.assert_allclose(got[:, 2:], 127 * 2.0 ** -5, rtol=2.0 ** -20)
