"""Steps over a paged cache that are cancelled, and a schedule's continuations to their ends, on the GPU."""
import numpy as np
import pytest

import jev
from helpers import tiny_config
from test_gpu_model import cancel_while_running

pytestmark = pytest.mark.gpu


def test_a_cancelled_step_is_taken_again(gpu):
    """jev_cancel reaches a step in flight; the next one names what each request keeps and gives the same bits."""
    cfg = tiny_config()
    tokens = [[int(t) for t in jev.random_tokens(n, cfg.vocab, 31 + n)] for n in (3900, 50)]
    with jev.SynthModel(cfg, jev.TYPE_Q8_0).open(0) as m, jev.KvPages(cfg, 300, 16, 2, 4100, 4100) as p:
        m.forward_pages(p, [1, 0], [[1, 2, 3], [4]], past=[0, 0], outputs=False)
        want = m.forward_pages(p, [0, 1], tokens, past=[1, 3])
        m.cancel()  # aimed at no call
        for _ in range(20):
            try:
                cancel_while_running(m, lambda: m.forward_pages(p, [0, 1], tokens, past=[1, 3]))
            except jev.CancelledError:
                break
        else:
            pytest.fail("no cancel reached a step in flight in 20 attempts")
        np.testing.assert_array_equal(m.forward_pages(p, [0, 1], tokens, past=[1, 3]), want)
        assert m.cached_token_count == 0


def test_every_prompt_gets_its_own_continuation(gpu):
    """paged_greedy's tokens against the loop of steps with one other request beside it, to the end.  A row that
    runs alone takes the one-token kernels, whose logits may differ by 1e-3 of their norm (a code's border, see
    test_gpu_pages_model.py): the first other token, if any, has a logit within that of the largest, twice."""
    cfg = tiny_config()
    rs = np.random.RandomState(8)
    prompts = [[int(t) for t in rs.randint(0, cfg.vocab, n)] for n in (40, 3, 90, 17, 64, 2)]
    with jev.SynthModel(cfg, jev.TYPE_Q8_0).open(0) as m, jev.KvPages(cfg, 30, 16, 4, 200, 150) as p:
        got = jev.paged_greedy(m, p, prompts, 12)
        assert [len(g) for g in got] == [12] * 6
        for prompt, g in zip(prompts, got):
            p.release(range(4))
            logits = m.forward_pages(p, [0, 1], [prompt, [1, 2]])[0]
            for token in g:
                best = jev.index_of_max(logits)
                if token != best:
                    assert logits[best] - logits[token] <= 2 * 1e-3 * np.linalg.norm(logits)
                logits = m.forward_pages(p, [0, 1], [[token], [3]])[0]
