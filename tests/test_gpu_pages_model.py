"""The model over a paged 8-bit cache: jev_forward_pages and paged_greedy on the GPU."""
import numpy as np
import pytest

import jev
import npref
import pages_ref as R
from helpers import rel_l2, tiny_config

pytestmark = pytest.mark.gpu


def stepped(cfg, W, steps):
    """Each step's tokens through the model in 64 bits, its keys and values held as the cache holds them."""
    caches = [{n: R.Cache(cfg.n_kv_heads, cfg.head_dim) for n in "kv"} for _ in range(cfg.n_layers)]
    past, out = 0, []
    for tokens in steps:
        n, H, hd = len(tokens), cfg.n_heads, cfg.head_dim
        pos = np.arange(past, past + n)
        h = W["token_embd.weight"][tokens].copy()
        for l in range(cfg.n_layers):
            p = f"blk.{l}."
            x = npref.rmsnorm(h, W[p + "attn_norm.weight"], cfg.rms_eps)
            q = R.rotate(cfg, (x @ W[p + "attn_q.weight"].T).reshape(n, H, hd), pos, False, True)
            k = R.rotate(cfg, (x @ W[p + "attn_k.weight"].T).reshape(n, -1, hd), pos, False, False)
            v = (x @ W[p + "attn_v.weight"].T).reshape(n, -1, hd)
            caches[l]["k"].store(past, k)
            caches[l]["v"].store(past, v)
            a, _ = R.attend(q, caches[l]["k"].values(past + n), caches[l]["v"].values(past + n), past)
            h = h + a.reshape(n, H * hd) @ W[p + "attn_output.weight"].T
            x = npref.rmsnorm(h, W[p + "ffn_norm.weight"], cfg.rms_eps)
            g = x @ W[p + "ffn_gate.weight"].T
            h = h + (g / (1 + np.exp(-g)) * (x @ W[p + "ffn_up.weight"].T)) @ W[p + "ffn_down.weight"].T
        past += n
        out.append(npref.rmsnorm(h[-1:], W["output_norm.weight"], cfg.rms_eps)[0] @ W["token_embd.weight"].T)
    return out


CONFIGS = [(jev.TYPE_Q8_0, {}), (jev.TYPE_Q5_1, dict(n_heads=6, rope_dim=64)),
           (jev.TYPE_Q4_0, dict(n_kv_heads=4, rope_scaling_yarn=1, rope_original_context=32, rope_scale_factor=4.0, attention_temperature_scale=0.1))]


@pytest.mark.parametrize("kind,kw", CONFIGS)
def test_logits_follow_the_statement(gpu, kind, kw):
    """Prompts and single tokens of several requests.  The model's own error is 2^-20 or so; a key or value
    that lies within it of a code's border (one in ten thousand) takes the next code, 1/127 of its block's
    largest: some 1e-4 of the logits, far below what leaving the cache's rounding out would give (checked)."""
    cfg = tiny_config(**kw)
    synth = jev.SynthModel(cfg, kind)
    W = npref.dequantized(synth)
    rs = np.random.RandomState(5)
    steps = {r: [rs.randint(0, cfg.vocab, n) for n in ns] for r, ns in {2: (37, 1, 1, 20), 0: (1, 1, 16, 1), 1: (70, 5, 1, 1)}.items()}
    want = {r: stepped(cfg, W, s) for r, s in steps.items()}
    pages = jev.KvPages(cfg, 40, 16, 3, 200, 200)
    with synth.open(0) as m:
        for i in range(4):
            got = m.forward_pages(pages, [2, 0, 1], [steps[r][i] for r in (2, 0, 1)])
            for g, r in zip(got, (2, 0, 1)):
                assert rel_l2(want[r][i], g) <= 1e-3, (i, r, rel_l2(want[r][i], g))
        own = m.forward(np.concatenate(steps[1]))
        assert rel_l2(want[1][3], own) > 2e-3  # the 8-bit cache is seen
        # one request alone, one token: the one-token path
        got = m.forward_pages(pages, [1], [steps[1][3]], past=[76])
        assert rel_l2(want[1][3], got[0]) <= 1e-3


def test_a_request_alone_has_the_same_bits(gpu):
    cfg = tiny_config()
    rs = np.random.RandomState(6)
    with jev.SynthModel(cfg, jev.TYPE_Q8_0).open(0) as m, jev.KvPages(cfg, 40, 16, 3, 200, 200) as a, jev.KvPages(cfg, 40, 32, 3, 200, 200) as b:
        prompts = [rs.randint(0, cfg.vocab, n) for n in (2, 33, 90)]
        for p in (a, b):
            p.release([0, 1, 2])
        every = range(cfg.vocab)  # by rows: the full-vocabulary head of one output is the one-token kernel
        together = m.forward_pages(a, [0, 1, 2], prompts, past=[0, 0, 0], vocab_rows=every)
        rows = m.forward_pages(a, [1, 0, 2], [[5, 6], [7, 8], [9]], vocab_rows=[3, 1])
        for i, nxt in enumerate(([7, 8], [5, 6])):
            np.testing.assert_array_equal(m.forward_pages(b, [2], [prompts[i]], past=[0], vocab_rows=every)[0], together[i])
            np.testing.assert_array_equal(m.forward_pages(b, [2], [nxt], vocab_rows=[3, 1])[0], rows[1 - i])
        assert m.cached_token_count == 0  # the context's own cache is left alone


def test_steps_are_refused_on_the_device_and_go_on(gpu):
    cfg = tiny_config()
    with jev.SynthModel(cfg, jev.TYPE_Q8_0).open(0) as m, jev.KvPages(cfg, 3, 16, 2, 200, 200) as p:
        first = m.forward_pages(p, [0], [[1, 2, 3]])
        for bad, code in (((([0], [[4] * 46])), 3), (([0], [[4] * 198]), 1)):
            with pytest.raises(jev.JevError) as e:
                m.forward_pages(p, *bad)
            assert e.value.code == code
        with pytest.raises(jev.JevError):
            m.forward_pages(p, [0], [[4]], past=[4])  # more than it has
        np.testing.assert_array_equal(m.forward_pages(p, [0], [[1, 2, 3]], past=[0]), first)
        assert m.forward_pages(p, [0], [[4] * 45], outputs=False) is None
        p.release([0])
        m.forward_pages(p, [1], [[4] * 48], outputs=False)


def test_paged_greedy_is_the_step_by_step_loop(gpu):
    """A busy schedule gives every prompt what it gets alone (prompts of two tokens and more; a lone row's
    single-token steps take the one-token path, so a second request keeps running beside it)."""
    cfg = tiny_config()
    rs = np.random.RandomState(8)
    prompts = [[int(t) for t in rs.randint(0, cfg.vocab, n)] for n in (40, 3, 90, 17, 64, 2)]
    with jev.SynthModel(cfg, jev.TYPE_Q8_0).open(0) as m, jev.KvPages(cfg, 30, 16, 4, 200, 150) as p:
        got = jev.paged_greedy(m, p, prompts, 12)
        assert [len(g) for g in got] == [12] * 6
        for i, prompt in enumerate(prompts):
            p.release(range(4))
            logits = m.forward_pages(p, [0, 1], [prompt, [1, 2]])
            want = []
            for _ in range(12):
                want.append(jev.index_of_max(logits[0]))
                logits = m.forward_pages(p, [0, 1], [[want[-1]], [3]])
            k = next((j for j in range(12) if got[i][j] != want[j]), 12)
            # the last prompts' tails run alone: the one-token path, equal up to a near tie
            assert k == 12 or i in (4, 5), (i, k)
        stopped = jev.paged_greedy(m, p, prompts, 12, stop_tokens=[got[0][4]])
        assert stopped[0] == got[0][:got[0].index(got[0][4]) + 1]
