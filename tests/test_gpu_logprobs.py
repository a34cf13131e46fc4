"""Log probabilities on the GPU against their statement in 64 bits (tests/logprobs_ref.py has the bounds)."""
import ctypes

import numpy as np
import pytest

import jev
import logprobs_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture
def rs():
    return np.random.RandomState(31)


class Rig:
    def __init__(self, vocab, rows):
        import torch

        self.t, self.vocab, self.p = torch, vocab, jev.LogProbs(vocab, rows)

    def run(self, x, given=None, top=0, temperature=1.0, pad=0, lead=0):
        """The call's outputs as arrays; rows `pad` floats apart, `lead` before the first."""
        t, rows = self.t, len(x)
        given = np.zeros((rows, 0), np.int32) if given is None else np.asarray(given, np.int32)
        n = given.shape[1]
        a = np.full(lead + rows * (self.vocab + pad), 3e38, np.float32)  # what lies between the rows would be the largest
        a[lead:].reshape(rows, -1)[:, :self.vocab] = x
        dx, dg = t.as_tensor(a, device="cuda"), t.as_tensor(given, device="cuda")
        out = [t.full((lead + rows * w + 3,), -7, dtype=d, device="cuda") for w, d in
               ((n, t.float32), (1, t.float32), (top, t.int32), (top, t.float32))]
        at = [o.data_ptr() + 4 * lead for o in out]
        t.cuda.synchronize()
        self.p.logprobs_device(dx.data_ptr() + 4 * lead, self.vocab + pad, rows, dg.data_ptr(), n, top, temperature, *at)
        self.p.sync()
        res = []
        for o, w in zip(out, (n, 1, top, top)):
            y = o.cpu().numpy()
            assert np.all(y[:lead] == -7) and np.all(y[lead + rows * w:] == -7)
            res.append(y[lead:lead + rows * w].reshape(rows, w))
        return jev.TokenLogProbs(res[0], res[1][:, 0], res[2], res[3])

    def check(self, x, given=None, top=0, temperature=1.0, **kw):
        x = np.asarray(x, np.float32)
        got = self.run(x, given, top, temperature, **kw)
        for r in range(len(x)):
            logp, entropy, off, off_h = R.row(x[r], temperature)
            want = R.order(x[r], top)
            np.testing.assert_array_equal(got.top[r], want)
            ids = want if given is None else np.concatenate([want, given[r]])
            y = got.top_logp[r] if given is None else np.concatenate([got.top_logp[r], got.logp[r]])
            w = logp[ids]
            with np.errstate(invalid="ignore", over="ignore"):
                same = (y == w.astype(np.float32)) | (np.isnan(y) & np.isnan(w))  # infinities (past fp32's range too) and NaN
                assert np.all(same | (np.abs(y - w) <= off + np.abs(w) * R.ULP * 1.001 + 1e-45)), (r, y, w, off)
                assert (np.isnan(entropy) and np.isnan(got.entropy[r])) or abs(got.entropy[r] - entropy) <= off_h + entropy * R.ULP * 1.001 + 1e-45, (
                    r, got.entropy[r], entropy, off_h)
        return got


@pytest.mark.parametrize("vocab", [1, 2, 3, 31, 33, 255, 257, 1000, 2047, 2049, 4095, 4097, 8191, 32000, 50021, 131072, 131075])
@pytest.mark.parametrize("top", [0, 1, 5, 32])
def test_rows_of_any_width(gpu, rs, vocab, top):
    top = min(top, vocab)
    rig = Rig(vocab, 5)
    for rows, temperature in ((1, 1.0), (5, 0.75)):
        x = rs.randn(rows, vocab) * rs.uniform(0.5, 6, (rows, 1))
        rig.check(x, rs.randint(0, vocab, (rows, 4)), top, temperature)


@pytest.mark.parametrize("rows", [1, 2, 31, 33, 64, 700, 1023, 1025, 2049, 5000])
def test_any_number_of_rows(gpu, rs, rows):
    """Rows in many parts, in two, and whole."""
    rig = Rig(9000, rows)
    rig.check(rs.randn(rows, 9000).astype(np.float32) * 3, rs.randint(0, 9000, (rows, 2)), 7)


@pytest.mark.parametrize("pad,lead", [(0, 0), (1, 0), (3, 1), (64, 2), (5, 3)])
def test_any_alignment_and_stride(gpu, rs, pad, lead):
    rig = Rig(12345, 6)
    x, given = rs.randn(6, 12345).astype(np.float32) * 4, rs.randint(0, 12345, (6, 3))
    want = rig.check(x, given, 9)
    got = rig.check(x, given, 9, pad=pad, lead=lead)
    for a, b in zip(want, got):
        np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("temperature", [1e-3, 0.1, 0.7, 1.0, 1.5, 50.0, 1e6])
def test_temperatures(gpu, rs, temperature):
    rig = Rig(20000, 4)
    rig.check(rs.randn(4, 20000) * 3, rs.randint(0, 20000, (4, 9)), 20, temperature)


@pytest.mark.parametrize("gap", [1.0, 10.0, 16.0, 20.0, 40.0, 80.0])
def test_nearly_certain_tokens(gpu, rs, gap):
    """What is left to the others is small: its logarithm keeps its bits."""
    rig = Rig(30000, 3)
    x = rs.randn(3, 30000).astype(np.float32)
    at = rs.randint(0, 30000, 3)
    x[np.arange(3), at] = x.max(1) + np.float32(gap)
    got = rig.check(x, at[:, None], 3)
    assert np.all(got.top[:, 0] == at) and np.all(got.logp[:, 0] < 0) and np.all(got.entropy > 0)


def test_masked_logits(gpu, rs):
    """-inf where tokens are ruled out: some, whole parts of a row, all but one, all."""
    rig = Rig(20000, 8)
    x = rs.randn(8, 20000).astype(np.float32)
    x[0, rs.permutation(20000)[:9000]] = -np.inf
    x[1, :10000] = -np.inf
    x[2, 5000:] = -np.inf
    x[3] = -np.inf
    x[3, 17777] = 0.25
    x[4] = -np.inf
    x[5, 1:] = -np.inf
    x[6, :-1] = -np.inf
    x[7] = -np.inf
    x[7, ::4000] = 1.0
    given = np.array([[0, 19999, 17777]] * 8)
    got = rig.check(x, given, 32)
    assert np.isnan(got.logp[4]).all() and got.logp[3, 2] == 0 and got.entropy[3] == 0 and got.logp[3, 0] == -np.inf


def test_values_that_are_not_finite(gpu, rs):
    rig = Rig(9000, 7)
    x = rs.randn(7, 9000).astype(np.float32)
    x[0, 4321] = np.nan
    x[1, 8999] = np.inf
    x[2, 0], x[2, 7000] = np.nan, np.inf
    x[3, :] = np.nan
    x[4, rs.permutation(9000)[:40]] = np.inf
    x[5, rs.permutation(9000)[:40]] = np.nan
    x[5, rs.permutation(9000)[:40]] = -np.inf
    x[6, 100] = -np.nan
    x[6, 1:50] = -np.inf
    got = rig.check(x, np.array([[4321, 0]] * 7), 32)
    assert np.isnan(got.entropy).all() and np.isnan(got.logp).all()


def test_large_and_small_logits(gpu, rs):
    rig = Rig(5000, 6)
    x = rs.randn(6, 5000).astype(np.float32)
    x[0] *= 1e30
    x[1] *= 1e-30
    x[2] *= 1e-42
    x[3] = 3.4e38 * np.sign(x[3])
    x[4] = 0
    x[5] = 1e8 + x[5]
    rig.check(x, rs.randint(0, 5000, (6, 4)), 10)


@pytest.mark.parametrize("k", [1, 2, 31, 32])
def test_ties_and_orders(gpu, rs, k):
    """Equal logits go to the lowest index, whatever order the row is in; +0 is above -0."""
    n = 40000
    rig = Rig(n, 12)
    x = np.zeros((12, n), np.float32)
    x[1] = rs.randint(0, 5, n)
    x[2] = np.arange(n)
    x[3] = -np.arange(n)
    x[4] = np.where(rs.rand(n) < 0.5, 0.0, -0.0)
    x[5] = np.arange(n) // 100
    x[6] = (np.arange(n) % 128 == 5) * (1 + rs.rand(n))      # one lane's logits are the largest
    x[7] = np.where(np.arange(n) % 256 < 4 * k, rs.rand(n), -1)  # as many lanes' as are asked for
    x[8] = rs.randint(0, 3, n) * np.float32(1e-45)
    x[9] = np.sort(rs.randn(n))
    x[10, rs.permutation(n)[:20]] = 7
    x[11] = -np.inf
    x[11, -10:] = 1
    rig.check(x, None, k)


def test_outputs_that_are_not_wanted(gpu, rs):
    rig = Rig(6000, 3)
    t = rig.t
    x = rs.randn(3, 6000).astype(np.float32)
    want = rig.run(x, np.array([[5], [6], [7]]), 4)
    dx, dg = t.as_tensor(x, device="cuda"), t.as_tensor(np.array([[5], [6], [7]], np.int32), device="cuda")
    e, i, l, g = t.empty(3, device="cuda"), t.empty((3, 4), dtype=t.int32, device="cuda"), t.empty((3, 4), device="cuda"), t.empty((3, 1), device="cuda")
    t.cuda.synchronize()
    a = (dx.data_ptr(), 6000, 3)
    rig.p.logprobs_device(*a, entropy=e.data_ptr())
    rig.p.logprobs_device(*a, n_top=4, top=i.data_ptr())
    rig.p.logprobs_device(*a, n_top=4, top_logp=l.data_ptr())
    rig.p.logprobs_device(*a, dg.data_ptr(), 1, logp=g.data_ptr())
    rig.p.logprobs_device(*a[:2], 0, entropy=e.data_ptr())
    rig.p.sync()
    for got, w in ((e, want.entropy), (i, want.top), (l, want.top_logp), (g, want.logp)):
        np.testing.assert_array_equal(got.cpu().numpy(), w)


def test_given_tokens_outside_the_vocabulary(gpu, rs):
    """And many of them, some named twice."""
    rig = Rig(4500, 3)
    x = rs.randn(3, 4500).astype(np.float32)
    ids = rs.randint(0, 4500, (3, 1000))
    ids[:, 500:] = ids[:, :500]
    got = rig.check(x, ids)
    np.testing.assert_array_equal(got.logp[:, 500:], got.logp[:, :500])
    bad = rig.run(x, np.array([[-1, 4500, 2 ** 31 - 1, -2 ** 31, 9]] * 3))
    assert np.isnan(bad.logp[:, :4]).all() and np.isfinite(bad.logp[:, 4]).all()


def test_calls_in_a_row_and_two_handles(gpu, rs):
    """Partial results, whose places every call uses again; another handle's calls beside them."""
    t = Rig(30000, 40).t
    rigs = [Rig(30000, 40), Rig(30000, 40)]
    xs = [rs.randn(n, 30000).astype(np.float32) * s for n, s in ((40, 1), (3, 4), (17, 2))]
    want = [rigs[0].check(x, None, 6) for x in xs]
    dx = [t.as_tensor(x, device="cuda") for x in xs]
    outs = [[(t.empty((len(x), 6), dtype=t.int32, device="cuda"), t.empty((len(x), 6), device="cuda"), t.empty(len(x), device="cuda"))
             for x in xs * 20] for _ in rigs]
    t.cuda.synchronize()
    for i in range(60):
        for rig, out in zip(rigs, outs):
            ids, lp, e = out[i]
            rig.p.logprobs_device(dx[i % 3].data_ptr(), 30000, len(xs[i % 3]), n_top=6, entropy=e.data_ptr(), top=ids.data_ptr(), top_logp=lp.data_ptr())
    for rig, out in zip(rigs, outs):
        rig.p.sync()
        for i, (ids, lp, e) in enumerate(out):
            np.testing.assert_array_equal(ids.cpu().numpy(), want[i % 3].top)
            np.testing.assert_array_equal(lp.cpu().numpy(), want[i % 3].top_logp)
            np.testing.assert_array_equal(e.cpu().numpy(), want[i % 3].entropy)


def test_a_call_is_captured_and_replayed(gpu, rs):
    hip = ctypes.CDLL("libamdhip64.so.7")  # the runtime that the library has loaded
    rig = Rig(40000, 8)
    t = rig.t
    dx, dg = t.zeros((8, 40000), device="cuda"), t.zeros((8, 2), dtype=t.int32, device="cuda")
    out = [t.empty((8, 2), device="cuda"), t.empty(8, device="cuda"), t.empty((8, 5), dtype=t.int32, device="cuda"), t.empty((8, 5), device="cuda")]
    t.cuda.synchronize()
    stream, graph, ex = ctypes.c_void_p(rig.p.stream), ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    rig.p.logprobs_device(dx.data_ptr(), 40000, 8, dg.data_ptr(), 2, 5, 1.5, *(o.data_ptr() for o in out))
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(ex), graph, None, None, 0) == 0
    for _ in range(4):
        x, given = rs.randn(8, 40000).astype(np.float32) * 3, rs.randint(0, 40000, (8, 2)).astype(np.int32)
        dx.copy_(t.as_tensor(x))
        dg.copy_(t.as_tensor(given))
        t.cuda.synchronize()
        assert hip.hipGraphLaunch(ex, stream) == 0
        rig.p.sync()
        for o, w in zip(out, rig.check(x, given, 5, 1.5)):
            np.testing.assert_array_equal(o.cpu().numpy(), w)
    assert hip.hipGraphExecDestroy(ex) == 0 and hip.hipGraphDestroy(graph) == 0


def test_rows_past_32_bit_offsets(gpu, rs):
    """Rows that begin past 2^32 bytes."""
    rig = Rig(1000, 3)
    t = rig.t
    ld = 1 << 29  # floats
    dx = t.empty(2 * ld + 1000, device="cuda")
    x = rs.randn(3, 1000).astype(np.float32)
    for r in range(3):
        dx[r * ld:r * ld + 1000] = t.as_tensor(x[r], device="cuda")
    top, e = t.empty((3, 8), dtype=t.int32, device="cuda"), t.empty(3, device="cuda")
    t.cuda.synchronize()
    rig.p.logprobs_device(dx.data_ptr(), ld, 3, n_top=8, entropy=e.data_ptr(), top=top.data_ptr())
    rig.p.sync()
    want = rig.check(x, None, 8)
    np.testing.assert_array_equal(top.cpu().numpy(), want.top)
    np.testing.assert_array_equal(e.cpu().numpy(), want.entropy)
