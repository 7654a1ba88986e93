"""Calls that the batch operators' documentation allows: other streams, fresh
outputs, one graph for several operators, layouts of a single sequence."""
import pytest
import torch

import batch_ref as ref

pytestmark = pytest.mark.gpu


def cache_of(c):
    from genllm_b200.batch import PagedBatch
    return PagedBatch(c.k_pool, c.v_pool, c.table, c.lens)


def same(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


def run_beside_a_busy_stream(bind):
    """Binds on a stream with much work queued and runs on an idle one."""
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(100_000_000)
    op = bind()
    op.run(stream=side)
    torch.cuda.synchronize()
    return op


def test_select_bound_on_a_busy_stream():
    from genllm_b200.batch import PageSelect, page_bounds
    c = ref.make_case([700, 90], 8, 4, 64, torch.bfloat16, seed=1)
    cache = cache_of(c)
    bound = page_bounds(cache)
    op = run_beside_a_busy_stream(lambda: PageSelect(cache, c.q, bound, 6))
    assert torch.equal(op.pages.cpu(), ref.select(c, bound, 6, 1, 1, 1))


def test_evict_bound_on_a_busy_stream():
    from genllm_b200.batch import CacheEvict
    c = ref.make_case([300, 40], 2, 2, 64, torch.bfloat16, seed=2)
    w = torch.rand((2, 2, 16 * c.table.shape[1]), device="cuda")
    want = ref.evict(c, w, c.lens.clone(), 64, 8)
    seen = c.lens.clone()
    op = run_beside_a_busy_stream(lambda: CacheEvict(cache_of(c), w, seen, keep=64, recent=8))
    assert torch.equal(op.lens_out, want[0]) and torch.equal(op.positions_out, want[2]) and same(c.k_pool, want[3])
