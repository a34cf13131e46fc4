"""The 4-bit paged cache's host side without a device: what creating it refuses, what it allocates
and launches (tests/fake_hip.py); its statement's own properties."""
import ctypes

import numpy as np
import pytest

import fake_hip
import jev
import pages4_ref as R4
from jev import _lib as L


@pytest.mark.parametrize("bits", [0, 1, 2, 3, 5, 6, 16, -4, -8])
def test_create_refuses_other_widths(bits):
    c = L.PagesConfig(10, 16, 2, 100, 100, 0)
    h = ctypes.c_void_p()
    rc = jev.lib().jev_pages_create_bits(ctypes.byref(jev.ModelConfig().to_c()), ctypes.byref(c), bits, 0, ctypes.byref(h))
    assert rc == L.JEV_EINVAL and not h.value and b"8 or 4" in jev.lib().jev_last_error()
    with pytest.raises(jev.ArgumentError):
        jev.KvPages(jev.ModelConfig(), 10, bits=bits)


@pytest.mark.parametrize("model,kw", [(dict(head_dim=96), {}), (dict(n_heads=32, n_kv_heads=7), {}), ({}, dict(page_tokens=8)), ({}, dict(n_pages=0))])
def test_create_refuses_what_the_8_bit_cache_does(model, kw):
    c = L.PagesConfig(**{**dict(n_pages=10, page_tokens=16, max_requests=2, max_context=100, max_tokens=100, rope_half=0), **kw})
    h = ctypes.c_void_p()
    rc = jev.lib().jev_pages_create_bits(ctypes.byref(jev.ModelConfig(**model).to_c()), ctypes.byref(c), 4, 0, ctypes.byref(h))
    assert rc in (L.JEV_EINVAL, L.JEV_EDATA) and not h.value


def test_null_arguments_are_refused():
    h = ctypes.c_void_p()
    c = L.PagesConfig(10, 16, 2, 100, 100, 0)
    m = jev.ModelConfig().to_c()
    for args in ((None, ctypes.byref(c), 4, 0, ctypes.byref(h)), (ctypes.byref(m), None, 4, 0, ctypes.byref(h)), (ctypes.byref(m), ctypes.byref(c), 4, 0, None)):
        assert jev.lib().jev_pages_create_bits(*args) == L.JEV_EINVAL


def test_a_pool_takes_its_bytes():
    """138 bytes a token and KV head of 128, 70 of 64; 8 bits: 256.5 and 128.5."""
    got = fake_hip.run("""
def live(bits, dim, pages):
    p = jev.KvPages(jev.ModelConfig(n_layers=3, n_heads=4, n_kv_heads=2, head_dim=dim, rope_dim=dim), pages, 32, 4, 300, 200, bits=bits)
    n = F.fake_live()
    p.close()
    return n
result = [live(bits, dim, 8192) - live(bits, dim, 4096) for bits in (4, 8) for dim in (64, 128)]
""")
    tokens, rows = 4096 * 32, 3 * 2  # of the further pages; layers x KV heads
    for n, a_row in zip(got, (70, 138, 128.5, 256.5)):
        assert n >= tokens * rows * a_row
        assert n - tokens * rows * a_row < 60 * tokens * rows  # partial results and lists


def test_calls_refuse_bad_arguments():
    got = fake_hip.run("""
cfg = jev.ModelConfig(n_layers=2, n_heads=4, n_kv_heads=2, head_dim=128)
p = jev.KvPages(cfg, 20, 16, 3, 200, 100, bits=4)
def no(f, *a):
    try:
        f(*a)
    except jev.ArgumentError:
        return not launches()
    return False
launches()
result = [
    no(p.plan_device, 64, 0, 64, 4, 10), no(p.plan_device, 64, 0, 64, 2, 101), no(p.plan_device, 0, 0, 64, 2, 10),
    no(p.store_device, 2, 64, 512, 64, 64, 256, 64), no(p.store_device, 0, 64, 511, 64, 64, 256, 128), no(p.store_device, 0, 64, 512, 64, 0, 256, 128),
    no(p.store_device, 0, 0, 0, 0, 0, 0, 0), no(p.store_device, 0, 64, 640, 64, 64, 256, 64),
    no(p.attend_device, 2, 64, 128), no(p.attend_device, 0, 0, 128), no(p.attend_device, 0, 64, 64),
    no(p.read_device, 0, 64, -1, 64, 64), no(p.read_device, 2, 64, 1, 64, 64), no(p.read_device, 0, 0, 1, 64, 64),
    no(p.release, [0, 1, 2, 3]),
]
""")
    assert all(got)


def test_calls_launch_the_4_bit_kernels():
    got = fake_hip.run("""
result = []
for bits in (4, 8):
    p = jev.KvPages(jev.ModelConfig(n_layers=1, n_heads=4, n_kv_heads=2, head_dim=64, rope_dim=64), 64, 16, 4, 256, 256, bits=bits)
    for n, t in ((0, 0), (1, 1), (2, 40)):
        p.plan_device(64, 0, 64, n, t)
        launches()
        p.store_device(0, 64, 256, 64, 64, 128, 128)
        p.attend_device(0, 64, 128)
        p.read_device(0, 64, 3, 64, 64)
        result.append([("pages4" in name, min(g)) for name, g, _, _ in launches()])
""")
    assert [len(x) for x in got] == [3] * 6
    assert all(four and g >= 1 for x in got[:3] for four, g in x) and not any(four for x in got[3:] for four, _ in x)


def test_values_are_within_half_a_step():
    rs = np.random.RandomState(3)
    x = rs.randn(3000, 2, 128).astype(np.float32) * np.exp2(rs.randint(-120, 120, (3000, 1, 1))).astype(np.float32) * (0.5 + rs.randn(1, 2, 128) ** 2).astype(np.float32)
    x[:20] = np.abs(x[:20])
    n, u, z, e = R4.quantise(x)
    assert u.min() >= 1 and u.max() <= 15 and z.max() <= 15 and n.max() <= 15
    step = np.repeat(np.ldexp(1.0, e)[..., None] * u, 32, -1)
    err = np.abs(R4.values(x).astype(np.float64) - x)
    assert np.all(err <= step * (0.5 + 2.0 ** -20))  # (a span is rounded to fp32)
    assert np.sqrt((err ** 2).sum() / (x.astype(np.float64) ** 2).sum()) < 0.14
