"""gkv_batch_page_bounds and gkv_batch_select_pages against their definitions."""
import pytest
import torch

import batch_ref as ref

pytestmark = pytest.mark.gpu

RAGGED = [0, 1, 15, 16, 17, -1, 33, 100, 700]


def cache_of(c):
    from genllm_b200.batch import PagedBatch
    return PagedBatch(c.k_pool, c.v_pool, c.table, c.lens)


def same(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hkv,d", [(8, 128), (1, 64), (3, 256), (11, 64)])
def test_bounds(hkv, d, dtype):
    from genllm_b200.batch import page_bounds
    c = ref.make_case(RAGGED, hkv, hkv, d, dtype, seed=d)
    cache = cache_of(c)
    into = torch.full((c.k_pool.shape[0], hkv, 2, d), 9.0, dtype=dtype, device="cuda")
    want = ref.bounds(c, into)
    assert same(page_bounds(cache, into), want)
    # The page each sequence's next token goes to, from its tokens so far and that one.
    for b, n in enumerate(c.lens.tolist()):
        if n >= 0:
            c.k_pool[int(c.table[b, n // 16, 0]), n % 16] = c.k_new[b]
    want = ref.bounds(c, into, start=c.lens, extra=1)
    assert same(page_bounds(cache, into, start=c.lens, extra=1), want)
    assert cache.check_device_errors() == 0


def test_bounds_from_the_middle_and_nan():
    from genllm_b200.batch import page_bounds
    c = ref.make_case([300, 40, 7], 4, 4, 128, torch.bfloat16, seed=2)
    c.k_pool[int(c.table[0, 9, 0]), 5, 2, 17] = float("nan")
    c.k_pool[int(c.table[1, 1, 0]), 1, 0, 3] = -float("inf")
    start = torch.tensor([130, -7, 100], dtype=torch.int32, device="cuda")  # negative: from 0; behind the end: nothing
    into = torch.zeros((c.k_pool.shape[0], 4, 2, 128), dtype=torch.bfloat16, device="cuda")
    got = page_bounds(cache_of(c), into.clone(), start=start)
    want = ref.bounds(c, into, start=start.clamp(min=0))
    nan = torch.isnan(want)
    assert bool(nan.any()) and torch.equal(torch.isnan(got), nan) and torch.equal(got[~nan], want[~nan])


@pytest.mark.parametrize("n_pages,first,last,extra", [(1, 0, 0, 0), (4, 1, 1, 1), (7, 3, 4, 0), (16, 0, 2, 1), (200, 1, 1, 1)])
@pytest.mark.parametrize("hq,hkv,d,dtype", [(16, 8, 128, torch.bfloat16), (7, 1, 64, torch.float16),
                                            (48, 3, 256, torch.bfloat16), (11, 11, 64, torch.bfloat16)])
def test_select(hq, hkv, d, dtype, n_pages, first, last, extra):
    from genllm_b200.batch import page_bounds, select_pages
    c = ref.make_case(RAGGED + [1003], hq, hkv, d, dtype, seed=n_pages)
    cache = cache_of(c)
    bound = page_bounds(cache)
    want = ref.select(c, bound, n_pages, first, last, extra)
    pages = torch.full((len(RAGGED) + 1, hkv, n_pages), 77, dtype=torch.int32, device="cuda")
    got = select_pages(cache, c.q, bound, n_pages, first=first, last=last, extra=extra, pages=pages).cpu()
    want[RAGGED.index(-1)] = 77  # a skipped sequence's list stays as it was
    assert torch.equal(got, want)
    assert cache.check_device_errors() == 0


def test_select_ties_nan_and_forced_pages():
    from genllm_b200.batch import page_bounds, select_pages
    c = ref.make_case([320], 4, 2, 64, torch.bfloat16, seed=4)
    for lp in (3, 7, 8, 12, 13):  # equal pages: the lower ones are taken
        c.k_pool[int(c.table[0, lp, 0])] = c.q[0].abs().amax()
    c.q = c.q.abs()
    c.k_pool[int(c.table[0, 15, 0]), 2, 1, 5] = float("nan")
    c.k_pool[int(c.table[0, 16, 0]), 2, 1, 5] = float("inf")
    cache = cache_of(c)
    bound = page_bounds(cache)
    for n_pages, first, last in ((2, 0, 0), (3, 0, 1), (4, 2, 1), (1, 0, 1), (1, 1, 0)):
        got = select_pages(cache, c.q, bound, n_pages, first=first, last=last, extra=0).cpu()
        assert torch.equal(got, ref.select(c, bound, n_pages, first, last, 0))
    assert 15 in select_pages(cache, c.q, bound, 2, first=0, last=0, extra=0)[0, 1].tolist()


def test_bounds_of_forced_pages_are_not_looked_at():
    from genllm_b200.batch import page_bounds, select_pages
    c = ref.make_case([700, 90], 8, 4, 128, torch.bfloat16, seed=9)
    cache = cache_of(c)
    bound = page_bounds(cache)
    want = ref.select(c, bound, 6, 2, 1, 1)
    for b, n in ((0, 700), (1, 90)):
        for lp in (0, 1, n // 16):
            bound[int(c.table[b, lp, 0])] = float("nan") if b else float("inf")
    assert torch.equal(select_pages(cache, c.q, bound, 6, first=2, last=1, extra=1).cpu(), want)


def test_select_zero_queries():
    """All scores equal: the lowest pages."""
    from genllm_b200.batch import page_bounds, select_pages
    c = ref.make_case([500], 8, 4, 128, torch.float16, seed=5)
    c.q.zero_()
    cache = cache_of(c)
    got = select_pages(cache, c.q, page_bounds(cache), 5, first=0, last=1, extra=0).cpu()
    assert got[0].tolist() == [[0, 1, 2, 3, 31]] * 4


def test_select_long():
    """More pages than a block has threads; two runs agree."""
    from genllm_b200.batch import PageSelect, page_bounds
    c = ref.make_case([40000], 8, 2, 64, torch.bfloat16, seed=6)
    cache = cache_of(c)
    bound = page_bounds(cache)
    op = PageSelect(cache, c.q, bound, 300, first=2, last=3, extra=1)
    a = op.run().clone()
    assert torch.equal(a, op.run())
    lo, hi = (bound[c.table[0, :2501, 0].long()][:, :, i].double() for i in range(2))
    for h in range(2):
        u = torch.stack([torch.where(x >= 0, x * hi[:, h], x * lo[:, h]).sum(-1) for x in c.q[0, 4 * h:4 * h + 4].double()]).amax(0)
        u[:2] = u[-3:] = float("inf")
        assert torch.equal(a[0, h].long().cpu(), u.sort(descending=True, stable=True).indices[:300].sort().values.cpu())


def test_bad_pages_are_flagged():
    from genllm_b200.batch import page_bounds, select_pages
    c = ref.make_case([100, 50], 4, 2, 64, torch.bfloat16, seed=7)
    cache = cache_of(c)
    bound = page_bounds(cache)
    c.table[0, 2, 0] = c.k_pool.shape[0] + 4
    page_bounds(cache, bound)
    assert cache.check_device_errors() == 1
    select_pages(cache, c.q, bound, 3, first=0, last=0, extra=0)
    assert cache.check_device_errors() == 1
    c.lens[1] = 2000000000
    page_bounds(cache, bound, extra=1)
    assert cache.check_device_errors() & 4


def test_a_sparse_step_equals_a_dense_one_when_all_pages_are_taken():
    from genllm_b200.batch import batch_decode, page_bounds, select_pages
    c = ref.make_case([100, 250, 3], 16, 8, 128, torch.bfloat16, seed=8)
    cache = cache_of(c)
    pages = select_pages(cache, c.q, page_bounds(cache), 40)
    out = batch_decode(cache, c.q, c.k_new, c.v_new, pages=pages)
    want = ref.decode(c)
    ref.check_close(out, want["out"], want["slack"])
