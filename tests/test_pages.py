"""The paged cache's host side without a device: what it refuses before it touches one, and what
a cache allocates and launches (tests/fake_hip.py)."""
import ctypes

import numpy as np
import pytest

import fake_hip
import jev
import pages_ref as R
from jev import _lib as L


@pytest.mark.parametrize("model,kw", [
    (dict(n_heads=32, n_kv_heads=7), {}), (dict(head_dim=96), {}), (dict(head_dim=256), {}), (dict(rope_dim=130), {}), (dict(rope_dim=3), {}),
    (dict(rope_dim=-2), {}), (dict(n_layers=0), {}), (dict(n_heads=2048, n_kv_heads=8), {}), (dict(rope_freq_base=0.0), {}),
    (dict(rope_scale_factor=0.0), {}), (dict(rope_scale_factor=float("nan")), {}),
    ({}, dict(page_tokens=8)), ({}, dict(page_tokens=48)), ({}, dict(page_tokens=512)), ({}, dict(n_pages=0)), ({}, dict(n_pages=1 << 27)),
    ({}, dict(max_requests=0)), ({}, dict(max_requests=4097)), ({}, dict(max_context=0)), ({}, dict(max_context=(1 << 24) + 1)),
    (dict(n_heads=1024, n_kv_heads=1), dict(max_tokens=(1 << 18) + 1)), ({}, dict(max_tokens=0)), ({}, dict(max_tokens=(1 << 22) + 1)), ({}, dict(rope_half=2))])
def test_create_refuses_before_touching_a_device(model, kw):
    c = L.PagesConfig(**{**dict(n_pages=10, page_tokens=16, max_requests=2, max_context=100, max_tokens=100, rope_half=0), **kw})
    h = ctypes.c_void_p()
    rc = jev.lib().jev_pages_create(ctypes.byref(jev.ModelConfig(**model).to_c()), ctypes.byref(c), 0, ctypes.byref(h))
    assert rc in (L.JEV_EINVAL, L.JEV_EDATA) and not h.value and jev.lib().jev_last_error()


def test_null_handles_are_refused():
    lib = jev.lib()
    lib.jev_pages_destroy(None)
    assert lib.jev_pages_stream(None) is None
    for rc in (lib.jev_pages_create(None, None, 0, None), lib.jev_pages_plan_device(None, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0),
               lib.jev_pages_store_device(None, 0, 0, 0, 0, 0, 0, 0), lib.jev_pages_attend_device(None, 0, 0, 0),
               lib.jev_pages_read_device(None, 0, 0, 0, 0, 0), lib.jev_pages_release(None, None, 0), lib.jev_pages_sync(None)):
        assert rc == L.JEV_EINVAL


def test_calls_refuse_bad_arguments():
    got = fake_hip.run("""
cfg = jev.ModelConfig(n_layers=2, n_heads=4, n_kv_heads=2, head_dim=128)
p = jev.KvPages(cfg, 20, 16, 3, 200, 100)
def no(f, *a):
    try:
        f(*a)
    except jev.ArgumentError:
        return not launches()
    return False
launches()
result = [
    no(p.plan_device, 64, 0, 64, 4, 10), no(p.plan_device, 64, 0, 64, -1, 10), no(p.plan_device, 64, 0, 64, 2, 101), no(p.plan_device, 64, 0, 64, 2, -1),
    no(p.plan_device, 0, 0, 64, 2, 10), no(p.plan_device, 64, 0, 0, 2, 10),
    no(p.store_device, 2, 64, 512, 64, 64, 256, 64), no(p.store_device, -1, 64, 512, 64, 64, 256, 64), no(p.store_device, 0, 64, 511, 64, 64, 256, 128),
    no(p.store_device, 0, 64, 512, 64, 64, 255, 128), no(p.store_device, 0, 64, 512, 64, 0, 256, 128), no(p.store_device, 0, 64, 512, 0, 64, 256, 128),
    no(p.store_device, 0, 0, 512, 64, 64, 256, 128), no(p.store_device, 0, 64, 512, 64, 64, 256, 0), no(p.store_device, 0, 0, 0, 0, 0, 0, 0),
    no(p.store_device, 0, 64, 640, 64, 64, 256, 64),
    no(p.attend_device, 2, 64, 128), no(p.attend_device, 0, 0, 128), no(p.attend_device, 0, 64, 0), no(p.attend_device, 0, 64, 64),
    no(p.read_device, 0, 64, -1, 64, 64), no(p.read_device, 2, 64, 1, 64, 64), no(p.read_device, 0, 0, 1, 64, 64), no(p.read_device, 0, 64, 1, 0, 64),
    no(p.release, [0, 1, 2, 3]),
]
""")
    assert all(got), got


def test_forward_pages_refuses():
    got = fake_hip.run("""
m = model(heads=4, kv=2)
def pages(**kw):
    half = kw.pop("half", False)
    c = dict(n_layers=1, n_heads=4, n_kv_heads=2, head_dim=128)
    c.update(kw)
    return jev.KvPages(jev.ModelConfig(**c), 20, 16, 3, 200, 100, half)
p = pages()
def no(q, *a, **kw):
    try:
        m.forward_pages(q, *a, **kw)
    except jev.ArgumentError:
        return not launches()
    return False
launches()
t = [1, 2, 3]
result = [no(q, [0], [t]) for q in (pages(n_layers=2), pages(n_heads=8), pages(n_kv_heads=4), pages(head_dim=64, rope_dim=64), pages(half=True),
                                    pages(rope_freq_base=1e4), pages(rope_dim=64), pages(attention_temperature_scale=0.5))]
result += [no(p, [], []), no(p, [3], [t]), no(p, [-1], [t]), no(p, [1, 1], [t, t]), no(p, [0], [[]]), no(p, [0, 1], [t]), no(p, [0], [t], past=[-1]),
           no(p, [0], [t], past=[0, 0]), no(p, [0], [[512]]), no(p, [0], [[-1]]), no(p, [0], [t * 34]), no(p, [0], [t], vocab_rows=[512]),
           no(p, [0], [t], vocab_rows=[])]
m.forward_pages(p, [2, 0], [t, [4]], vocab_rows=[5, 6])
names = [n for n, *_ in launches()]
result.append(sum("pages_plan" in n for n in names) == 1 and sum("pages_store" in n for n in names) == 1 and not any("attn_" in n for n in names))
""")
    assert all(got), got


def test_a_cache_that_finds_no_room_leaves_nothing():
    got = fake_hip.run("""
cfg = jev.ModelConfig(n_layers=2, n_heads=4, n_kv_heads=2, head_dim=128)
jev.KvPages(cfg, 64, 16, 4, 200, 100).close()
result, live = [], F.fake_live()
need = 0
for left in range(0, 2500000, 130001):
    room(left)
    try:
        jev.KvPages(cfg, 64, 16, 4, 200, 100).close()
        result.append([True, F.fake_live() - live])
    except jev.JevError as e:
        result.append([e.code, F.fake_live() - live])
""")
    assert [L.JEV_ENOMEM, 0] in got and [True, 0] in got and all(x[1] == 0 and x[0] in (True, L.JEV_ENOMEM) for x in got)


def test_nothing_is_allocated_after_create():
    got = fake_hip.run("""
cfg = jev.ModelConfig(n_layers=2, n_heads=4, n_kv_heads=2, head_dim=128)
p = jev.KvPages(cfg, 64, 16, 4, 800, 900)
live = F.fake_live()
room(0)
for n, t in ((1, 1), (4, 900), (4, 4), (0, 0)):
    p.plan_device(64, 0, 64, n, t, 64, 64, 64, 64, 64)
    p.store_device(1, 64, 512, 64, 64, 256, 128)
    p.attend_device(1, 64, 128)
    p.read_device(1, 64, 5, 64, 64)
    p.release([0, 1])
result = [F.fake_live() - live, F.fake_refused()]
""")
    assert got == [0, 0]


def test_the_statement_of_codes():
    """tests/pages_ref.py's own blocks: scales only grow, codes follow, a cut block keeps its scale."""
    c = R.Cache(1, 4)
    c.store(0, np.full((3, 1, 4), 1.0))
    c.store(3, np.full((1, 1, 4), 254.0))
    assert c.scale[0, 0] == 2 and c.code[0, 0, 0] == 0 and c.code[3, 0, 0] == 127  # half a step: to even
    c.store(1, np.full((20, 1, 4), -127.0))
    assert c.scale[0, 0] == 2 and c.scale[1, 0] == 1 and list(c.code[[1, 15, 16], 0, 0]) == [-64, -64, -127]
    c.store(18, np.full((1, 1, 4), np.nan))
    assert np.isnan(c.scale[1, 0]) and np.isnan(c.values(19)[17]).all() and np.isfinite(c.values(16)).all()


class FakeModel:
    """Next token = a function of everything a request holds."""

    def __init__(self, vocab):
        self.vocab, self.held, self.steps = vocab, {}, []

    def forward_pages(self, pages, requests, tokens, past):
        assert len(set(requests)) == len(requests) and sum(map(len, tokens)) <= pages.max_tokens
        out = np.zeros((len(requests), self.vocab), np.float32)
        for b, (r, t, p) in enumerate(zip(requests, tokens, past)):
            self.held[r] = self.held.get(r, [])[:p] + list(t)
            assert len(self.held[r]) == p + len(t) <= pages.max_context
            out[b, sum((i + 1) * x for i, x in enumerate(self.held[r])) % self.vocab] = 1
        assert sum(R.pages(len(self.held[r]), pages.page_tokens) for r in self.held) <= pages.n_pages
        self.steps.append(len(requests))
        return out


class FakePages:
    def __init__(self, model, n_pages, page, requests, context, tokens):
        self.model, self.n_pages, self.page_tokens, self.max_requests = model, n_pages, page, requests
        self.max_context, self.max_tokens = context, tokens

    def release(self, requests):
        for r in requests:
            self.model.held.pop(r, None)


@pytest.mark.parametrize("n_pages,requests,tokens", [(100, 8, 400), (9, 8, 60), (100, 2, 60), (6, 1, 50)])
def test_paged_greedy_schedules(n_pages, requests, tokens):
    rs = np.random.RandomState(3)
    prompts = [[int(x) for x in rs.randint(0, 50, n)] for n in (1, 30, 7, 49, 16, 17, 2)]
    m = FakeModel(50)
    got = jev.paged_greedy(m, FakePages(m, n_pages, 16, requests, 80, tokens), prompts, 9, stop_tokens=[11])
    for p, g in zip(prompts, got):
        held, want = list(p), []
        while len(want) < 9 and 11 not in want:
            want.append(sum((i + 1) * x for i, x in enumerate(held)) % 50)
            held.append(want[-1])
        assert g == want
    assert not m.held and (max(m.steps) > 1) == (requests > 1)


def test_paged_greedy_refuses_what_cannot_fit():
    m = FakeModel(50)
    p = FakePages(m, 6, 16, 4, 80, 50)
    for prompts, new in (([[1] * 51], 2), ([[1] * 40], 42), ([[]], 2), ([[1]], 0), ([[1]] * 3 + [[1] * 50], 48)):
        with pytest.raises(jev.ArgumentError):
            jev.paged_greedy(m, p, prompts, new)


@pytest.mark.parametrize("counts,cls", [([1, 1], "PROF_DECODE_ATTN"), ([3, 1], "PROF_ATTN")])
def test_attention_over_pages_is_stamped(counts, cls):
    """The per-kernel profiler times it like every other attention launch (1 ms each there), and counts its work."""
    log, read = fake_hip.run(f"""
m = model(heads=4, kv=2)
p = jev.KvPages(jev.ModelConfig(n_layers=1, n_heads=4, n_kv_heads=2, head_dim=128), 20, 16, 3, 200, 100)
L = jev.lib()
jev._lib.check(L.jev_profile_enable(m._h, 1))
launches()
m.forward_pages(p, [0, 2], [[1] * n for n in {counts}], past=[20, 0])
n, ms, flops = ctypes.c_int64(), ctypes.c_double(), ctypes.c_double()
jev._lib.check(L.jev_profile_read(m._h, jev._lib.{cls}, ctypes.byref(n), ctypes.byref(ms), ctypes.byref(flops), None))
result = [[(k, a, b) for k, g, a, b in launches() if "pages_attend" in k], [n.value, ms.value, flops.value]]
""")
    assert len(log) == 1 and log[0][1] and log[0][2] and log[0][1] != log[0][2]
    pairs = sum(p + i + 1 for p, n in zip((20, 0), counts) for i in range(n))
    assert read == [1, 1.0, 4.0 * 128 * 4 * pairs]
