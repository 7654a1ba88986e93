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


def test_bounds_of_full_pages_that_sequences_share():
    from genllm_b200.batch import page_bounds, select_pages
    c = ref.make_case([90, 70, 64], 8, 4, 64, torch.float16, seed=7)
    c.table[1:, :4] = c.table[0, :4]  # 64 tokens in common, the rest each its own
    cache = cache_of(c)
    into = torch.zeros((c.k_pool.shape[0], 4, 2, 64), dtype=torch.float16, device="cuda")
    want = ref.bounds(c, into)
    got = page_bounds(cache, into)
    assert same(got, want)
    assert torch.equal(select_pages(cache, c.q, got, 3, extra=0).cpu(), ref.select(c, got, 3, 1, 1, 0))


def test_bounds_follow_an_eviction():
    """Rows move between pages: selection behind it takes the bounds of the cut cache."""
    from genllm_b200.batch import CacheEvict, page_bounds, select_pages
    c = ref.make_case([500, 130], 8, 2, 128, torch.bfloat16, seed=8)
    cache = cache_of(c)
    bound = page_bounds(cache)
    w = torch.rand((2, 2, 16 * c.table.shape[1]), device="cuda")
    want = ref.evict(c, w, c.lens.clone(), 100, 10)
    CacheEvict(cache, w, c.lens.clone(), keep=100, recent=10, lens_out=c.lens).run()
    page_bounds(cache, bound)
    assert same(c.k_pool, want[3]) and same(bound, ref.bounds(c, bound))
    pages = select_pages(cache, c.q, bound, 4, extra=0)
    assert torch.equal(pages.cpu(), ref.select(c, bound, 4, 1, 1, 0))


def test_decodes_and_an_eviction_in_one_graph():
    """Two layers' steps, the cut of the second and a step behind it, captured
    together: each kernel starts early beside the one before it."""
    from genllm_b200.batch import BatchDecode, CacheEvict
    lens = [90, 200, -1]
    layers = [ref.make_case(lens, 8, 4, 64, torch.bfloat16, seed=40 + i, spare=4) for i in range(2)]
    a, b = layers
    w = torch.rand((3, 4, 16 * b.table.shape[1]), device="cuda")
    totals = torch.zeros_like(w)
    seen = b.lens + 1
    # What the graph is to leave, a step at a time.
    wants = [ref.decode(x) for x in layers]
    sim = ref.Case(b.k_pool.clone(), b.v_pool.clone(), b.table, b.lens + (b.lens >= 0).int(), b.q, b.k_new, b.v_new)
    for s, n in enumerate(lens):
        if n >= 0:
            for pool, new, which in ((sim.k_pool, b.k_new, 0), (sim.v_pool, b.v_new, 1)):
                pool[int(b.table[s, n // 16, which]), n % 16] = new[s]
    cut = ref.evict(sim, w, seen, 60, 4)
    sim.k_pool, sim.v_pool, sim.lens = cut[3], cut[4], cut[0]
    after = ref.decode(sim)
    caches = [cache_of(x) for x in layers]
    steps = [BatchDecode(x, y.q, y.k_new, y.v_new) for x, y in zip(caches, layers)]
    evict = CacheEvict(caches[1], w, seen, keep=60, recent=4, lens_out=b.lens)
    again = BatchDecode(caches[1], b.q, b.k_new, b.v_new, weights_out=totals)
    old = [[t.clone() for t in (x.k_pool, x.v_pool, x.lens)] for x in layers] + [[w.clone()]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for s in steps:
            s.run()
        b.lens.add_((b.lens >= 0).int())
        evict.run()
        again.run()
    live = torch.tensor([0, 1])
    for _ in range(3):
        for x, was in zip(layers, old):
            for t, o in zip((x.k_pool, x.v_pool, x.lens), was):
                t.copy_(o)
        w.copy_(old[2][0])
        graph.replay()
        for s, want in zip(steps, wants):
            ref.check_close(s.out[live], want["out"][live], want["slack"][live])
        assert torch.equal(b.lens, cut[0]) and torch.equal(w, cut[1]) and torch.equal(evict.positions_out, cut[2])
        ref.check_close(again.out[live], after["out"][live], after["slack"][live])
        for s in (0, 1):
            n = int(b.lens[s])
            page, slot = b.table[s, n // 16].tolist(), n % 16
            cut[3][page[0], slot], cut[4][page[1], slot] = b.k_new[s], b.v_new[s]
            ref.check_close(totals[s, :, :n + 1], after["weights"][s], after["weight_slack"][s])
        assert same(b.k_pool, cut[3]) and same(b.v_pool, cut[4])
    assert caches[1].check_device_errors() == 0
