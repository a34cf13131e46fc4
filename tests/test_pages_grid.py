"""How many workgroups the paged attention launches, without a device (tests/fake_hip.py):
what the call's requests can need, not what the pool has room for."""
import fake_hip


def test_the_attention_grid_follows_the_call():
    got = fake_hip.run("""
cfg = jev.ModelConfig(n_layers=1, n_heads=8, n_kv_heads=2, head_dim=128)
def grids(pages, requests, context):
    p = jev.KvPages(cfg, pages, 16, requests, context, 4096)
    out = []
    for n, t in ((1, 1), (3, 3), (0, 0), (2, 90)):
        p.plan_device(64, 0, 64, n, t)
        launches()
        p.attend_device(0, 64, 128)
        out.append([g[0] for name, g, _, _ in launches() if "pages_attend" in name])
    p.close()
    return out
result = [grids(pages, requests, context) for pages, requests in ((1 << 10, 4), (1 << 17, 4), (1 << 17, 4096)) for context in (300, 8192, 20000, 1 << 20)]
""")
    kv = 2
    for i, g in enumerate(got):
        most = [1, 8, 16, 65][i % 4]  # parts of the longest request: of 1024 keys, 2048 past 16384, at most 65
        assert [len(x) for x in g] == [1] * 4
        one, three, none, prompts = (x[0] for x in g)
        assert kv <= one <= kv * (most + 2) and kv * 3 <= three <= kv * 3 * (most + 2) and none == kv
        # two requests of 45 tokens: wide tiles over the workgroups there are, and the 16-row form of either
        assert prompts <= kv * (2 * most + 90 * 4 // 16 + 2) + kv * (90 * 4 // 128 + 2 + 512 // kv)
    assert got[4] == got[8]


def test_a_decode_step_of_twelve_rows_plans_in_one_launch():
    """Its angles among the lists: 12 tokens of 64 pairs, as the model has; 24 are quicker with two."""
    got = fake_hip.run("""
p = jev.KvPages(jev.ModelConfig(n_layers=1, n_heads=32, n_kv_heads=8, head_dim=128, rope_dim=128), 4096, 16, 64, 1024, 4096)
result = []
for n in (1, 12, 16, 24):
    launches()
    p.plan_device(64, 64, 64, n, n)
    result.append(len(launches()))
""")
    assert got == [1, 1, 1, 2]


def test_a_batch_of_no_requests_is_launched():
    """Rows to spare and nothing in them: a grid all the same."""
    got = fake_hip.run("""
p = jev.KvPages(jev.ModelConfig(n_layers=1, n_heads=4, n_kv_heads=4, head_dim=64, rope_dim=64), 64, 16, 4, 256, 256)
result = []
for t in (0, 1, 5):
    p.plan_device(0, 0, 0, 0, t)
    p.store_device(0, 64, 256, 64, 64, 256, 128)
    p.attend_device(0, 64, 128)
    result += [min(g) for _, g, _, _ in launches()]
""")
    assert min(got) >= 1 and len(got) >= 9
