"""A served step end to end over the 8- and 4-bit paged caches: store and attention under a model's
layers, then log probabilities of its logits, against the same step's full logits in 64 bits."""
import numpy as np
import pytest

import jev
import logprobs_ref as R
from test_gpu_model import cancel_while_running

pytestmark = pytest.mark.gpu


def config(**kw):
    return jev.ModelConfig(**{**dict(n_layers=3, hidden=512, n_heads=8, n_kv_heads=2, head_dim=128, ffn=1024, vocab=3000), **kw})


@pytest.fixture(scope="module", params=["Q8_0", "Q5_1", "Q4_0"])
def model(request):
    return jev.SynthModel(config(), jev.TYPE_NAMES[request.param]).open(0)


def same(got, logits, given, top, temperature):
    """Log probabilities of a step against its logits (of the same kernels, so the same bits)."""
    for r, x in enumerate(logits):
        logp, entropy, off, off_h = R.row(x, temperature)
        ids = R.order(x, top)
        np.testing.assert_array_equal(got.top[r], ids)
        for y, w in ((got.top_logp[r], logp[ids]), (got.logp[r], logp[given[r]])):
            assert np.all(np.abs(y - w) <= off + np.abs(w) * R.ULP * 1.001)
        assert abs(got.entropy[r] - entropy) <= off_h + entropy * R.ULP * 1.001


@pytest.mark.parametrize("bits", [8, 4])
def test_a_step_answers_with_log_probabilities(gpu, model, bits):
    """Prompts, then single tokens: at each request's last token, the same as from forward_pages' logits."""
    rs = np.random.RandomState(5)
    pages = [jev.KvPages(model.config, 100, 16, 4, 400, 600, bits=bits) for _ in range(2)]
    lens = [0, 0, 0]
    for step in ([100, 1, 37], [1, 1, 1], [1, 20, 3]):
        toks = [rs.randint(0, 3000, n).tolist() for n in step]
        given = rs.randint(0, 3000, (3, 4))
        logits = model.forward_pages(pages[0], [2, 0, 1], toks, past=lens)
        got = model.forward_pages_logprobs(pages[1], [2, 0, 1], toks, given, 5, 0.8, past=lens)
        same(got, logits, given, 5, 0.8)
        lens = [a + b for a, b in zip(lens, step)]
    one = rs.randint(0, 3000, 1).tolist()  # a request alone: the one-token path
    logits = model.forward_pages(pages[0], [0], [one], past=[lens[1]])
    same(model.forward_pages_logprobs(pages[1], [0], [one], [[7]], 3, past=[lens[1]]), logits, [[7]], 3, 1.0)


def near(x):
    """What two paths' log probabilities of logits x may differ by: 1e-3 of the logits' norm each, twice (see
    tests/test_gpu_pages_steps.py)."""
    return 2 * 1e-3 * np.linalg.norm(x)


@pytest.mark.parametrize("bits", [8, 4])
def test_every_token_of_a_step(gpu, model, bits):
    """More rows than the head takes at a time.  Each request's last row has the bits of the step that asks for
    those alone; in 4 bits, where no later token changes an earlier one's codes, a row is its prompt's beginning's."""
    rs = np.random.RandomState(6)
    pages = jev.KvPages(model.config, 100, 16, 2, 700, 700, bits=bits)
    toks = [rs.randint(0, 3000, n).tolist() for n in (515, 30)]
    given = rs.randint(0, 3000, (545, 2))
    got = model.forward_pages_logprobs(pages, [1, 0], toks, given, 6, past=[0, 0], every=True)
    last = model.forward_pages_logprobs(pages, [1, 0], toks, given[[514, 544]], 6, past=[0, 0])
    for x, y in zip(got, last):
        np.testing.assert_array_equal(x[[514, 544]], y)
    for r in (1, 200, 255, 256, 272, 273, 515, 516, 530) if bits == 4 else ():
        b, t = (0, r) if r < 515 else (1, r - 515)
        x = model.forward_pages(pages, [1 - b], [toks[b][:t + 1]], past=[0])[0]
        logp, entropy, _, _ = R.row(x, 1.0)
        assert np.all(np.abs(got.logp[r] - logp[given[r]]) <= near(x)) and np.all(np.abs(got.top_logp[r] - logp[got.top[r]]) <= near(x))
    for x, y in zip(model.forward_pages_logprobs(pages, [1, 0], toks, given, 6, past=[0, 0], every=True), got):
        np.testing.assert_array_equal(x, y)


def test_no_row_is_scored_alone(gpu):
    """One row more than 255 times the head's 256: the last row has the bits of its request's own step (a head of one
    row would be the one-token path's)."""
    rs = np.random.RandomState(12)
    m = jev.SynthModel(config(n_layers=1), jev.TYPE_Q8_0).open(0)
    counts = [15] * 255 + [16] * 3841
    assert sum(counts) == 255 * 256 + 1
    toks = [rs.randint(0, 3000, n).tolist() for n in counts]
    pages = jev.KvPages(m.config, 4100, 16, 4096, 16, 66000, bits=4)
    given = rs.randint(0, 3000, (65281, 20))
    got = m.forward_pages_logprobs(pages, list(range(4096)), toks, given, 20, past=[0] * 4096, every=True)
    alone = m.forward_pages_logprobs(pages, [4095], toks[-1:], given[-16:], 20, past=[0], every=True)
    for x, y in zip(got, alone):
        np.testing.assert_array_equal(x[-16:], y)


@pytest.mark.parametrize("bits", [8, 4])
def test_prompts_are_scored(gpu, model, bits):
    """paged_logprobs over several steps: each prompt as alone, and its tokens' log probabilities from logits."""
    rs = np.random.RandomState(8)
    prompts = [rs.randint(0, 3000, n).tolist() for n in (2, 90, 17, 200, 64, 3)]
    pages = jev.KvPages(model.config, 16, 16, 3, 250, 240, bits=bits)
    got = jev.paged_logprobs(model, pages, prompts, top=4, temperature=1.3)
    assert [len(x.logp) for x in got] == [len(p) - 1 for p in prompts]
    for p, x in zip(prompts, got):
        assert x.logp.shape == (len(p) - 1, 1) and x.top.shape == (len(p) - 1, 4)
        logits = model.forward_pages(pages, [0], [p[:-1]], past=[0])
        logp, _, _, _ = R.row(logits[0], 1.3)
        assert abs(x.logp[-1, 0] - logp[p[-1]]) <= near(logits[0]) and abs(x.top_logp[-1, 0] - logp.max()) <= near(logits[0])
    pages.release(range(3))
    assert len(jev.paged_greedy(model, pages, prompts[:2], 3)) == 2  # all pages are free again


def test_greedy_over_four_bits(gpu, model):
    """paged_greedy's continuations over a 4-bit cache are the step loop's own, whatever the schedule."""
    rs = np.random.RandomState(9)
    prompts = [rs.randint(0, 3000, n).tolist() for n in (20, 3, 45, 9)]
    wide = jev.KvPages(model.config, 60, 16, 4, 100, 200, bits=4)
    tight = jev.KvPages(model.config, 6, 16, 2, 100, 60, bits=4)
    a, b = (jev.paged_greedy(model, p, prompts, 6) for p in (wide, tight))
    assert [x[0] for x in a] == [x[0] for x in b] and all(len(x) == 6 for x in a)


def test_four_bits_are_near_the_context_cache(gpu):
    """The logits after a prompt: 4-bit rows are off by some 8 to 12 % each, averaged by the softmax."""
    m = jev.SynthModel(config(), jev.TYPE_Q8_0).open(0)
    toks = jev.random_tokens(200, 3000, 4)
    want = m.forward(toks)
    rel = []
    for bits in (8, 4):
        pages = jev.KvPages(m.config, 20, 16, 1, 300, 300, bits=bits)
        got = m.forward_pages(pages, [0], [list(toks)], past=[0])[0]
        rel.append(np.linalg.norm(got - want) / np.linalg.norm(want))
    assert rel[0] < rel[1] < 0.5, rel


def test_a_cancelled_score(gpu):
    """jev_cancel reaches a scored step; the step after it is whole."""
    m = jev.SynthModel(config(n_layers=8, vocab=131072, hidden=1024), jev.TYPE_Q8_0).open(0)
    pages = jev.KvPages(m.config, 300, 16, 1, 4096, 4096, bits=4)
    toks = jev.random_tokens(4096, 131072, 4)
    given = [[1]] * 4096
    want = m.forward_pages_logprobs(pages, [0], [toks], given, 3, past=[0], every=True)
    for _ in range(20):
        try:
            cancel_while_running(m, lambda: m.forward_pages_logprobs(pages, [0], [toks], given, 3, past=[0], every=True))
        except jev.CancelledError:
            break
    else:
        pytest.fail("no cancel reached a step in flight in 20 attempts")
    got = m.forward_pages_logprobs(pages, [0], [toks], given, 3, past=[0], every=True)
    for a, b in zip(got, want):
        np.testing.assert_array_equal(a, b)
