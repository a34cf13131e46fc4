"""Log probabilities without a device: what is refused before one is touched, what is launched
(tests/fake_hip.py), and the statement's own properties."""
import ctypes

import numpy as np
import pytest

import fake_hip
import jev
import logprobs_ref as R
from jev import _lib as L


@pytest.mark.parametrize("vocab,rows", [(0, 1), (-1, 1), ((1 << 28) + 1, 1), (1000, 0), (1000, -5), (1000, (1 << 24) + 1)])
def test_create_refuses_before_touching_a_device(vocab, rows):
    with pytest.raises(jev.ArgumentError):
        jev.LogProbs(vocab, rows)


def test_null_handles_are_refused():
    lib = jev.lib()
    lib.jev_logprobs_destroy(None)
    assert lib.jev_logprobs_stream(None) is None
    h = ctypes.c_void_p()
    assert lib.jev_logprobs_create(10, 10, 0, None) == L.JEV_EINVAL
    assert lib.jev_logprobs_device(None, 0, 10, 0, 0, 0, 0, 1.0, 0, 0, 0, 0) == L.JEV_EINVAL
    assert lib.jev_logprobs_sync(None) == L.JEV_EINVAL
    p = ctypes.POINTER(ctypes.c_int32)()
    assert lib.jev_forward_pages_logprobs(None, None, p, p, p, 1, p, 1, 0, p, 0, 1, 1.0, None, None, p, None) == L.JEV_EINVAL


def test_calls_refuse_bad_arguments():
    got = fake_hip.run("""
lp = jev.LogProbs(100, 8)
def no(*a, **kw):
    try:
        lp.logprobs_device(*a, **kw)
    except jev.ArgumentError:
        return not launches()
    return False
def yes(*a, **kw):
    lp.logprobs_device(*a, **kw)
    return len(launches())
launches()
nan, inf = float("nan"), float("inf")
result = [
    no(64, 99, 1, entropy=64), no(64, 100, 9, entropy=64), no(64, 100, -1, entropy=64), no(0, 100, 1, entropy=64), no(64, 100, 1),
    no(64, 100, 1, 0, 2, logp=64), no(64, 100, 1, 64, 2), no(64, 100, 1, 64, -1, logp=64), no(64, 100, 1, n_top=3), no(64, 100, 1, n_top=33, top=64),
    no(64, 100, 1, n_top=-1, top=64, entropy=64), no(64, 100, 1, temperature=0.0, entropy=64), no(64, 100, 1, temperature=-1.0, entropy=64),
    no(64, 100, 1, temperature=nan, entropy=64), no(64, 100, 1, temperature=inf, entropy=64), no(64, 100, 1, temperature=1e-39, entropy=64),
    no(64, 100, 1, temperature=3e38 * 1.1, entropy=64),
    yes(64, 100, 0, entropy=64) == 0, yes(64, 100, 8, entropy=64) == 1, yes(64, 1 << 40, 8, n_top=32, top_logp=64) == 1, yes(0, 100, 0, entropy=64) == 0,
]
small = jev.LogProbs(3, 8)
try:
    small.logprobs_device(64, 3, 1, n_top=4, top=64)
    result.append(False)
except jev.ArgumentError:
    result.append(True)
""")
    assert all(got), got


def test_the_grid_follows_the_rows():
    """One row of a large vocabulary over many workgroups, many rows one each; never more partial results than there is room for."""
    got = fake_hip.run("""
result = []
for vocab in (100, 50021, 131072, 1 << 28):
    lp = jev.LogProbs(vocab, 100000)
    for rows in (1, 2, 12, 64, 1000, 1024, 1025, 2047, 5000, 100000):
        lp.logprobs_device(64, vocab, rows, entropy=64)
        result.append([vocab, rows, launches()[0][1][0]])
""")
    for vocab, rows, grid in got:
        parts = grid // rows
        assert grid == rows * parts and parts <= 16 and (parts == 1 or grid <= 1024)
        assert parts == 1 or (parts - 1) * 8192 < vocab
        if rows == 1 and vocab == 131072:
            assert parts == 16


def test_scores_refuse_bad_arguments_without_a_step():
    got = fake_hip.run("""
cfg = jev.ModelConfig(n_layers=1, hidden=256, n_heads=4, n_kv_heads=2, head_dim=128, ffn=512, vocab=512)
m = jev.SynthModel(cfg, jev.TYPE_Q8_0).open(0)
p = jev.KvPages(cfg, 20, 16, 3, 200, 100, bits=4)
def no(f, *a, **kw):
    launches()
    try:
        f(*a, **kw)
    except jev.ArgumentError:
        return not launches()
    return False
s = m.forward_pages_logprobs
result = [
    no(s, p, [0], [[1, 2]], [[512]]), no(s, p, [0], [[1, 2]], [[-1]]), no(s, p, [0], [[1, 2]], [[1]], top=33), no(s, p, [0], [[1, 2]], [[1]], top=-1),
    no(s, p, [0], [[1, 2]], [[1]], temperature=0.0), no(s, p, [0], [[1, 2]], [[1], [2]]), no(s, p, [0], [[1, 2]], [[1]], every=True),
    no(s, p, [0], [[1, 2]], [1]), no(s, p, [0, 0], [[1], [2]], [[1], [2]]), no(s, p, [3], [[1]], [[1]]), no(s, p, [0], [[]], [[1]]),
    no(s, p, [0], [[512]], [[1]]), no(s, p, [0], [[1] * 101], [[1]]),
    no(jev.paged_logprobs, m, p, [[1]]), no(jev.paged_logprobs, m, p, [[1, 2], []]), no(jev.paged_logprobs, m, p, [[1] * 102]),
]
""")
    assert all(got), got


def test_scored_rows_go_through_the_head_in_like_groups():
    """257 rows are not 256 and one: a single row would take the one-token head."""
    got = fake_hip.run("""
cfg = jev.ModelConfig(n_layers=1, hidden=256, n_heads=4, n_kv_heads=2, head_dim=128, ffn=512, vocab=512)
m = jev.SynthModel(cfg, jev.TYPE_Q8_0).open(0)
p = jev.KvPages(cfg, 200, 16, 3, 2000, 1000, bits=4)
result = []
for n in (1, 2, 256, 257, 513, 1000):
    launches()
    m.forward_pages_logprobs(p, [0], [[1] * n], [[2]] * n, past=[0], every=True)
    result.append([n, [g[0] for name, g, _, _ in launches() if "logprobs" in name]])
""")
    for n, grids in got:
        groups = -(-n // 256)
        assert len(grids) == groups and sum(grids) == n and (n == 1 or min(grids) >= 2)


def test_the_order():
    x = np.array([0.0, -0.0, 1.0, np.nan, -np.inf, 1.0, np.inf, 0.0], np.float32)
    assert list(R.order(x, 8)) == [3, 6, 2, 5, 0, 7, 1, 4]
