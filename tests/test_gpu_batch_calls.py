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


def test_decode_bound_on_a_busy_stream():
    from genllm_b200.batch import BatchDecode
    c = ref.make_case([700, 90, -1], 8, 4, 64, torch.bfloat16, seed=3)
    want = ref.decode(c)
    op = run_beside_a_busy_stream(lambda: BatchDecode(cache_of(c), c.q, c.k_new, c.v_new))
    ref.check_close(op.out[:2], want["out"][:2], want["slack"][:2])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_of_skipped_sequences_in_a_new_output(dtype):
    """Outputs that the call makes hold zeros and -inf there, as of a sequence without tokens."""
    from genllm_b200.batch import BatchDecode, batch_decode
    c = ref.make_case([40, -1, 300, -1], 8, 4, 128, dtype, seed=4)
    cache = cache_of(c)
    skipped = c.lens < 0
    for _ in range(3):
        junk = [torch.full_like(c.q, 7.0), torch.full((4, 8), 7.0, device="cuda")]
        del junk  # memory that new tensors of these sizes are likely to get
        op = BatchDecode(cache, c.q, lse=True)
        out = op.run()
        assert bool((out[skipped] == 0).all()) and bool((op.lse[skipped] == -float("inf")).all())
        del op, out
        junk = torch.full_like(c.q, 7.0)
        del junk
        assert bool((batch_decode(cache, c.q)[skipped] == 0).all())


def test_one_sequence_of_one_head_at_odd_strides():
    """The strides of a single row are never used, whatever they are."""
    from genllm_b200.batch import BatchDecode, CacheEvict, PageSelect, PagedBatch, page_bounds

    def odd(t, stride):
        into = torch.as_strided(torch.zeros(t.numel() + 64, dtype=t.dtype, device="cuda"), t.shape, stride)
        return into.copy_(t)

    c = ref.make_case([11], 1, 1, 64, torch.bfloat16, seed=6, width=1)
    c.q, c.k_new, c.v_new = odd(c.q, (3, 5, 1)), odd(c.k_new, (9, 1, 1)), odd(c.v_new, (1003, 7, 1))
    c.table = odd(c.table, (5, 3, 1))
    cache = PagedBatch(c.k_pool, c.v_pool, c.table, c.lens)
    want = ref.decode(c)
    op = BatchDecode(cache, c.q, c.k_new, c.v_new)
    ref.check_close(op.run(), want["out"], want["slack"])
    bound = page_bounds(cache)
    assert PageSelect(cache, c.q, bound, 1, first=0, last=0).run().tolist() == [[[0]]]
    w = torch.rand(1, 1, 16, device="cuda")
    assert CacheEvict(cache, w, c.lens.clone(), keep=5).run().tolist() == [5]
    assert cache.check_device_errors() == 0
