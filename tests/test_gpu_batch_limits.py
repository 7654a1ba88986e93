"""The batch operators at the sizes where they change their ways: thousands of
sequences, tables far wider than the sequences, rows cut by clusters of CTAs
and rows whose keys do not fit in shared memory."""
import pytest
import torch

import batch_ref as ref

pytestmark = pytest.mark.gpu


def cache_of(c):
    from genllm_b200.batch import PagedBatch
    return PagedBatch(c.k_pool, c.v_pool, c.table, c.lens)


def widen(c, pages):
    """The same sequences with `pages` entries in each table row."""
    table = torch.full((c.table.shape[0], pages, 2), -1, dtype=torch.int32, device="cuda")
    table[:, :c.table.shape[1]] = c.table
    c.table = table
    return c


def long_case(n, hkv=1, d=64, group=2, seed=0, dtype=torch.bfloat16):
    """One sequence of n tokens, made on the GPU."""
    g = torch.Generator("cuda").manual_seed(seed)
    pages = -(-(n + 1) // 16)
    randn = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)  # noqa: E731
    ids = torch.stack([torch.randperm(pages, generator=g, device="cuda") for _ in range(2)], -1).int()
    return ref.Case(randn(pages, 16, hkv, d), randn(pages, 16, hkv, d), ids[None].contiguous(),
                    torch.tensor([n], dtype=torch.int32, device="cuda"), randn(1, hkv * group, d), randn(1, hkv, d),
                    randn(1, hkv, d))


def test_decode_of_4096_sequences():
    from genllm_b200.batch import batch_decode
    lens = [(37 * i) % 50 - 2 for i in range(4096)]
    c = ref.make_case([max(-1, n) for n in lens], 1, 1, 64, torch.float16, seed=1)
    out = torch.zeros_like(c.q)
    batch_decode(cache_of(c), c.q, c.k_new, c.v_new, out=out)
    rows = torch.arange(0, 4096, 13)
    sub = ref.Case(c.k_pool, c.v_pool, c.table[rows.cuda()], c.lens[rows.cuda()], c.q[rows.cuda()], c.k_new[rows.cuda()],
                   c.v_new[rows.cuda()])
    want = ref.decode(sub)
    ref.check_close(out[rows.cuda()], want["out"], want["slack"])
    assert bool((out[c.lens < 0] == 0).all())


@pytest.mark.parametrize("hq,hkv", [(1, 1), (256, 256), (17, 17)])
def test_decode_of_one_long_sequence(hq, hkv):
    from genllm_b200.batch import batch_decode
    c = long_case(30001 if hkv == 1 else 500, hkv, 64, hq // hkv, seed=2)
    want = ref.decode(c)
    w = torch.zeros(1, hkv, c.table.shape[1] * 16, device="cuda")
    out = batch_decode(cache_of(c), c.q, c.k_new, c.v_new, weights_out=w)
    ref.check_close(out, want["out"], want["slack"])
    ref.check_close(w[0, :, :int(c.lens[0]) + 1], want["weights"][0], want["weight_slack"][0])


def test_a_table_far_wider_than_the_sequences():
    from genllm_b200.batch import batch_decode, page_bounds, select_pages
    c = widen(ref.make_case([100, 0, 700], 8, 4, 128, torch.bfloat16, seed=3), 70000)
    want = ref.decode(c)
    cache = cache_of(c)
    bound = page_bounds(cache)
    pages = select_pages(cache, c.q, bound, 9, first=1, last=1)
    assert torch.equal(pages.cpu(), ref.select(c, bound, 9, 1, 1, 1))
    out = batch_decode(cache, c.q, c.k_new, c.v_new)
    ref.check_close(out, want["out"], want["slack"])
    assert cache.check_device_errors() == 0


def exact_order(c, bound, pages, head, group):
    """Pages of sequence 0 by falling score, equal ones by index."""
    rows = bound[c.table[0, :pages, 0].long(), head].double()
    u = torch.stack([torch.where(q >= 0, q * rows[:, 1], q * rows[:, 0]).sum(-1)
                     for q in c.q[0, head * group:(head + 1) * group].double()]).amax(0)
    return u.sort(descending=True, stable=True).indices


@pytest.mark.parametrize("n,wide,flat", [(300000, 0, False), (300000, 0, True), (90000, 140000, False), (90000, 140000, True)])
def test_select_over_clusters_and_beyond_shared_memory(n, wide, flat):
    """18751 pages (a cluster a row), and a table of 140000 (keys in the
    workspace); flat: many pages of equal scores at the cut."""
    from genllm_b200.batch import PageSelect, page_bounds
    c = long_case(n, hkv=2, seed=4)
    if flat:
        c.q[:, 0:2] = 0  # head 0: all scores 0
        c.k_pool[: c.k_pool.shape[0] // 2] = c.k_pool[:1]  # half the pages alike
    if wide:
        widen(c, wide)
    cache = cache_of(c)
    bound = page_bounds(cache)
    got = PageSelect(cache, c.q, bound, 777, first=0, last=0, extra=1).run()
    pages = -(-(n + 1) // 16)
    for h in range(2):
        want = exact_order(c, bound, pages, h, 2)[:777].sort().values.int()
        assert torch.equal(got[0, h], want)


@pytest.mark.parametrize("n,keep,wide", [(200001, 60000, 0), (90000, 1, 25000), (90000, 89999, 25000), (5000, 2500, 25000)])
def test_evict_over_clusters_and_beyond_shared_memory(n, keep, wide):
    from genllm_b200.batch import CacheEvict
    c = long_case(n, hkv=2, seed=5)
    if wide:
        widen(c, wide)
    g = torch.Generator("cuda").manual_seed(6)
    w = torch.rand((1, 2, 16 * c.table.shape[1]), generator=g, device="cuda")
    w[0, 1] = (w[0, 1] * 3).floor()  # three values: the cut falls among equal ones
    recent = min(keep, 100)
    rank = w[..., :n].clone()
    rank[..., n - recent:] = float("inf")
    order = rank.sort(dim=-1, descending=True, stable=True).indices[..., :keep]
    old_k, old_v, old_w = c.k_pool.clone(), c.v_pool.clone(), w.clone()
    positions = torch.zeros(w.shape, dtype=torch.int32, device="cuda")
    cache = cache_of(c)
    lens = CacheEvict(cache, w, c.lens.clone(), keep=keep, recent=recent, positions_out=positions).run()
    assert lens.tolist() == [keep] and cache.check_device_errors() == 0
    t = torch.arange(keep, device="cuda")
    for h in range(2):
        kept = order[0, h].sort().values
        held = positions[0, h, :keep].long()
        assert torch.equal(held.sort().values, kept)
        stays = kept[kept < keep]
        assert torch.equal(held[stays], stays)
        moved = torch.ones(keep, dtype=torch.bool, device="cuda")
        moved[stays] = False
        assert torch.equal(held[moved], kept[kept >= keep])  # the i-th hole holds the i-th kept slot behind
        assert torch.equal(w[0, h, :keep], old_w[0, h, held])
        for pool, old, which in ((c.k_pool, old_k, 0), (c.v_pool, old_v, 1)):
            ids = c.table[0, :, which].long()
            assert torch.equal(pool[ids[t // 16], t % 16, h], old[ids[held // 16], held % 16, h])
