"""gkv_batch_evict against its definition, and runs of the batch operators together."""
import math

import pytest
import torch

import batch_ref as ref

pytestmark = pytest.mark.gpu

LENS = [0, 1, 40, 64, -1, 300, 1500]


def cache_of(c):
    from genllm_b200.batch import PagedBatch
    return PagedBatch(c.k_pool, c.v_pool, c.table, c.lens)


def same(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


def check(c, w, seen, keep, recent, tracked=None, positions=None, in_place=False):
    from genllm_b200.batch import CacheEvict
    want = ref.evict(c, w, seen, keep, recent, tracked, positions)
    cache = cache_of(c)
    if in_place:
        options = dict(lens_out=c.lens)
    else:
        first_positions = positions if positions is not None else torch.zeros(w.shape, dtype=torch.int32, device="cuda")
        options = dict(weights_out=w.clone(), positions_out=first_positions.clone())
    old = w.clone()
    op = CacheEvict(cache, w, seen, keep=keep, recent=recent, tracked=tracked, positions=positions, **options)
    lens = op.run()
    assert cache.check_device_errors() == 0
    assert torch.equal(lens, want[0])
    assert torch.equal(op.weights_out.view(torch.int32), want[1].view(torch.int32))
    assert torch.equal(op.positions_out, want[2])
    assert same(c.k_pool, want[3]) and same(c.v_pool, want[4])
    if not in_place:
        assert torch.equal(w.view(torch.int32), old.view(torch.int32))
    return op


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("keep,recent", [(0, 0), (1, 0), (1, 1), (17, 5), (64, 64), (128, 0), (1499, 30), (5000, 10)])
@pytest.mark.parametrize("hkv,d,dtype", [(2, 64, torch.float16), (3, 128, torch.bfloat16), (1, 256, torch.bfloat16)])
def test_first_eviction(hkv, d, dtype, keep, recent, in_place):
    c = ref.make_case(LENS, hkv, hkv, d, dtype, seed=keep)
    g = torch.Generator("cuda").manual_seed(keep)
    w = torch.rand((len(LENS), hkv, 16 * c.table.shape[1]), generator=g, device="cuda") ** 4
    check(c, w, c.lens.clamp(min=0) + 3, keep, recent, in_place=in_place)


def test_tracked_positions():
    """Slots kept before hold tokens of any age; those appended since are in order."""
    lens = [100, 333, 50]
    c = ref.make_case(lens, 2, 2, 64, torch.bfloat16, seed=1)
    g = torch.Generator().manual_seed(2)
    width = 16 * c.table.shape[1] + 5
    tracked, seen = torch.tensor([64, 300, 50], dtype=torch.int32), torch.tensor([500, 1000, 60], dtype=torch.int32)
    positions = torch.zeros(3, 2, width, dtype=torch.int32)
    for b in range(3):
        for h in range(2):
            old = int(seen[b]) - (lens[b] - int(tracked[b]))
            positions[b, h, :tracked[b]] = torch.randperm(old, generator=g)[:tracked[b]].int()
    w = torch.rand(3, 2, width, generator=g).cuda()
    check(c, w, seen.cuda(), 40, 25, tracked.cuda(), positions.cuda())


def test_equal_weights_infinities_and_nan():
    c = ref.make_case([200], 4, 4, 64, torch.float16, seed=3)
    w = torch.zeros(1, 4, 16 * c.table.shape[1], device="cuda")
    w[0, 1, ::2] = -0.0
    w[0, 2] = torch.randint(0, 3, w[0, 2].shape, device="cuda").float()
    w[0, 3, :200] = torch.randn(200, device="cuda")
    w[0, 3, 100], w[0, 3, 150], w[0, 3, 151], w[0, 3, 10] = math.nan, math.inf, -math.inf, -math.nan
    check(c, w, c.lens.clone(), 30, 7)
    c = ref.make_case([200], 4, 4, 64, torch.float16, seed=3)
    check(c, w, c.lens.clone(), 1, 0)


def test_long_rows_and_repeats():
    c = ref.make_case([20000, 9000], 2, 2, 64, torch.bfloat16, seed=4)
    w = torch.rand((2, 2, 16 * c.table.shape[1]), device="cuda")
    check(c, w, c.lens.clone(), 8192, 100)


def test_bad_pages_are_flagged():
    from genllm_b200.batch import CacheEvict
    c = ref.make_case([100], 2, 2, 64, torch.bfloat16, seed=5)
    w = torch.rand((1, 2, 16 * c.table.shape[1]), device="cuda")
    cache = cache_of(c)
    c.table[0, 5, 1] = 1 << 20
    CacheEvict(cache, w, c.lens.clone(), keep=20).run()
    assert cache.check_device_errors() == 1
    c.lens[0] = 1 << 30
    c.table[0, 5, 1] = 0
    CacheEvict(cache, w, c.lens.clone(), keep=20).run()
    assert cache.check_device_errors() & 4


def test_captured_eviction():
    from genllm_b200.batch import CacheEvict
    c = ref.make_case([500, 90], 2, 2, 64, torch.bfloat16, seed=6)
    w = torch.rand((2, 2, 16 * c.table.shape[1]), device="cuda")
    seen = c.lens.clone()
    want = ref.evict(c, w, seen, 70, 8)
    op = CacheEvict(cache_of(c), w, seen, keep=70, recent=8, lens_out=c.lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op.run()
    graph.replay()
    assert torch.equal(c.lens, want[0]) and same(c.k_pool, want[3]) and same(c.v_pool, want[4])
    assert torch.equal(w, want[1])


def test_decode_with_totals_then_eviction_over_many_steps():
    """A serving loop on a budget: append and attend, total the attention, cut
    back every 16 steps; the cache holds the tokens an ideal one would."""
    from genllm_b200.batch import BatchDecode, CacheEvict, PagedBatch
    hq, hkv, d, keep, recent = 8, 2, 64, 48, 12
    lens = [0, 30, 60]
    c = ref.make_case(lens, hq, hkv, d, torch.bfloat16, seed=9, width=5, spare=1)
    batch, width = 3, 5 * 16
    # Room for keep + 16 tokens in every row.
    total = batch * 5
    pools = [torch.zeros(total, 16, hkv, d, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    g = torch.Generator("cuda").manual_seed(10)
    table = torch.stack([torch.randperm(total, generator=g, device="cuda").view(batch, 5) for _ in range(2)], -1).int()
    for b, n in enumerate(lens):
        for t in range(n):
            for w, (mine, theirs) in enumerate(((pools[0], c.k_pool), (pools[1], c.v_pool))):
                mine[int(table[b, t // 16, w]), t % 16] = theirs[int(c.table[b, t // 16, w]), t % 16]
    c.k_pool, c.v_pool, c.table = pools[0], pools[1], table
    cache = PagedBatch(c.k_pool, c.v_pool, c.table, c.lens)
    weights = torch.zeros(batch, hkv, width, device="cuda")
    positions = torch.zeros(batch, hkv, width, dtype=torch.int32, device="cuda")
    tracked, seen = torch.zeros(batch, dtype=torch.int32, device="cuda"), c.lens.clone()
    step = BatchDecode(cache, c.q, c.k_new, c.v_new, weights=weights, weights_out=weights, decay=0.95)
    cut = CacheEvict(cache, weights, seen, keep=keep, recent=recent, tracked=tracked, positions=positions, lens_out=c.lens)
    for i in range(40):
        for t in (c.q, c.k_new, c.v_new):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda").to(t.dtype))
        want = ref.decode(c)
        step.run()
        ref.check_close(step.out, want["out"], want["slack"], f"step {i}")
        c.lens += 1
        seen += 1
        if i % 16 == 15:
            expect = ref.evict(c, weights, seen, keep, recent, tracked, positions)
            cut.run()
            tracked.copy_(c.lens)
            assert torch.equal(c.lens, expect[0]) and torch.equal(weights, expect[1]) and torch.equal(positions, expect[2])
            assert same(c.k_pool, expect[3]) and same(c.v_pool, expect[4])
            for b in range(batch):
                kept = positions[b, :, :int(c.lens[b])]
                for h in range(hkv):  # the most recent tokens are all there
                    assert set(range(max(0, int(seen[b]) - recent), int(seen[b]))) <= set(kept[h].tolist())
    assert cache.check_device_errors() == 0


def test_managed_prompt_then_sparse_steps():
    """A prompt through the manager's chunk path, then sparse and dense steps over the layer's own pages."""
    from genllm_b200.batch import BatchDecode, PageBounds, PagedBatch, PageSelect
    from genllm_b200.paged_attention import PagedAttentionManager, paged_attention
    g = torch.Generator("cuda").manual_seed(3)
    hq, hkv, d, prompt = 16, 8, 128, 300
    randn = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    m = PagedAttentionManager(0)
    m.init_layer(0, hkv, d)
    m.reserve_layer(0, 40)
    paged_attention(m, 0, randn(1, hq, prompt, d), randn(1, hkv, prompt, d), randn(1, hkv, prompt, d))
    m.append_kv_pages(0, 40)  # room for the steps to come
    k_ids, v_ids = m.page_table(0)
    k_pool, v_pool = m.pool_tensors(0)
    table = torch.tensor([list(zip(k_ids, v_ids))], dtype=torch.int32, device="cuda")
    c = ref.Case(k_pool, v_pool, table, torch.tensor([prompt], dtype=torch.int32, device="cuda"), randn(1, hq, d),
                 randn(1, hkv, d), randn(1, hkv, d))
    cache = PagedBatch(c.k_pool, c.v_pool, c.table, c.lens)
    bound = PageBounds(cache, torch.zeros(40, hkv, 2, d, dtype=torch.bfloat16, device="cuda")).run()
    select = PageSelect(cache, c.q, bound, 6, first=1, last=2)
    step = BatchDecode(cache, c.q, c.k_new, c.v_new, pages=select.pages)
    refresh = PageBounds(cache, bound, start=c.lens, extra=1)
    for _ in range(20):
        for t in (c.q, c.k_new, c.v_new):
            t.copy_(randn(*t.shape))
        pages = ref.select(c, bound, 6, 1, 2, 1)
        want = ref.decode(c, pages=pages)
        want_bounds = bound.clone()
        select.run()
        step.run()
        refresh.run()
        assert torch.equal(select.pages.cpu(), pages)
        ref.check_close(step.out, want["out"], want["slack"])
        assert same(bound, ref.bounds(c, want_bounds, start=c.lens, extra=1))
        c.lens += 1
    want = ref.decode(c)
    dense = BatchDecode(cache, c.q, c.k_new, c.v_new)
    ref.check_close(dense.run(), want["out"], want["slack"])
    assert cache.check_device_errors() == 0


def test_a_managed_layer_evicted_and_decoded_on():
    """A manager's layer cut back by the batch operators, its freed pages back
    in the pool, then more tokens through the manager's own decode."""
    from genllm_b200.batch import BatchDecode, CacheEvict, PagedBatch
    from genllm_b200.paged_attention import PagedAttentionManager, paged_attention
    g = torch.Generator("cuda").manual_seed(4)
    hq, hkv, d, prompt, keep = 16, 8, 128, 500, 100
    randn = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    m = PagedAttentionManager(0)
    m.init_layer(0, hkv, d)
    m.reserve_layer(0, 40)
    paged_attention(m, 0, randn(1, hq, prompt, d), randn(1, hkv, prompt, d), randn(1, hkv, prompt, d))
    k_ids, v_ids = m.page_table(0)
    k_pool, v_pool = m.pool_tensors(0)
    table = torch.tensor([list(zip(k_ids, v_ids))], dtype=torch.int32, device="cuda")
    c = ref.Case(k_pool, v_pool, table, torch.tensor([prompt], dtype=torch.int32, device="cuda"), randn(1, hq, d),
                 randn(1, hkv, d), randn(1, hkv, d))
    cache = PagedBatch(c.k_pool, c.v_pool, c.table, c.lens)
    weights = torch.zeros(1, hkv, 16 * table.shape[1], device="cuda")
    for _ in range(5):  # totals over the cached tokens alone
        c.q.copy_(randn(1, hq, d))
        BatchDecode(cache, c.q, weights=weights, weights_out=weights).run()
    want = ref.evict(c, weights, c.lens.clone(), keep, 20)
    CacheEvict(cache, weights, c.lens.clone(), keep=keep, recent=20, lens_out=c.lens).run()
    left = -(-keep // 16)
    m.set_page_table(0, k_ids[:left], v_ids[:left], keep)
    for which, ids in ((0, k_ids), (1, v_ids)):
        for i in reversed(ids[left:]):
            m.pool(0, which).free(i)
    assert same(c.k_pool, want[3]) and same(c.v_pool, want[4])
    for step in range(20):
        q, k, v = randn(1, hq, 1, d), randn(1, hkv, 1, d), randn(1, hkv, 1, d)
        n = m.get_layer(0).num_cached
        ids = m.page_table(0)
        c.table = torch.tensor([list(zip(*ids))], dtype=torch.int32, device="cuda")
        c.lens.fill_(n)
        c.q, c.k_new, c.v_new = q[:, :, 0], k[:, :, 0], v[:, :, 0]
        expect = ref.decode(c)
        out = paged_attention(m, 0, q, k, v)
        torch.cuda.synchronize()
        err = (out[0, :, 0].double() - expect["out"][0]).abs()
        # the op's own bounds: 2e-3 absolute, and one rounding to bf16
        assert float((err - 2 ** -8 * expect["out"][0].abs()).max()) <= 2e-3, step
    assert m.get_layer(0).num_cached == keep + 20 and m.check_device_errors(0) == 0


def test_batch_and_managed_steps_in_turn_without_waiting():
    """A token through the batch decode, the next through the manager's own
    decode, which streams pages ahead of its predecessor's end: each sees what
    the other wrote, with the host waiting for neither."""
    from genllm_b200.batch import BatchDecode, PagedBatch
    from genllm_b200.paged_attention import PagedAttentionManager, paged_attention
    g = torch.Generator("cuda").manual_seed(5)
    hq, hkv, d, prompt, steps = 16, 8, 128, 1000, 60
    randn = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    m = PagedAttentionManager(0)
    m.init_layer(0, hkv, d)
    m.reserve_layer(0, 80)
    K, V = randn(1, hkv, prompt, d), randn(1, hkv, prompt, d)
    paged_attention(m, 0, randn(1, hq, prompt, d), K, V)
    new = [(randn(1, hq, 1, d), randn(1, hkv, 1, d), randn(1, hkv, 1, d)) for _ in range(steps)]
    k_pool, v_pool = m.pool_tensors(0)
    table = torch.zeros(1, 80, 2, dtype=torch.int32, device="cuda")
    lens = torch.tensor([prompt], dtype=torch.int32, device="cuda")
    cache = PagedBatch(k_pool, v_pool, table, lens)
    outs, ops = [], []
    torch.cuda.synchronize()
    for i, (q, k, v) in enumerate(new):
        if i % 2:
            outs.append(paged_attention(m, 0, q, k, v)[0, :, 0])
        else:
            m.append_kv_pages(0, 1)  # the host's count; the batch decode writes the row
            ids = torch.tensor(list(zip(*m.page_table(0))), dtype=torch.int32)
            table[0, :len(ids)].copy_(ids.pin_memory(), non_blocking=True)
            ops.append(BatchDecode(cache, q[:, :, 0], k[:, :, 0], v[:, :, 0]))
            outs.append(ops[-1].run()[0])
        lens += 1
    torch.cuda.synchronize()
    keys = torch.cat([K[0]] + [k[0] for _, k, _ in new], 1).double()
    values = torch.cat([V[0]] + [v[0] for _, _, v in new], 1).double()
    for i, (q, _, _) in enumerate(new):
        n = prompt + i + 1
        s = torch.einsum("hgd,hnd->hgn", q[0, :, 0].double().view(hkv, 2, d), keys[:, :n]) * d ** -0.5
        want = (s.softmax(-1) @ values[:, :n]).reshape(hq, d)
        err = (outs[i].double() - want).abs() - 2 ** -8 * want.abs()
        assert float(err.max()) <= 2e-3, i  # the decode op's own bound beside one rounding
    assert cache.check_device_errors() == 0 and m.check_device_errors(0) == 0


def test_two_operators_in_one_captured_step():
    """Two layers' decodes and an eviction in one graph, replayed between eager calls of the same operators."""
    from genllm_b200.batch import BatchDecode, CacheEvict, PagedBatch
    cases = [ref.make_case([90, 200], 8, 4, 64, torch.bfloat16, seed=40 + i, spare=40) for i in range(2)]
    caches = [PagedBatch(c.k_pool, c.v_pool, c.table, c.lens) for c in cases]
    steps = [BatchDecode(x, c.q, c.k_new, c.v_new) for x, c in zip(caches, cases)]
    w = torch.rand((2, 4, 16 * cases[1].table.shape[1]), device="cuda")
    cut = CacheEvict(caches[1], w, cases[1].lens.clone(), keep=60, recent=4, positions_out=torch.zeros(w.shape, dtype=torch.int32, device="cuda"))
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        for s in steps:
            s.run()
    for i in range(6):
        wants = [ref.decode(c) for c in cases]
        if i % 2:
            for s in steps:
                s.run()
        else:
            graph.replay()
        for s, want in zip(steps, wants):
            ref.check_close(s.out, want["out"], want["slack"])
        for c in cases:
            c.lens += 1
        if i == 3:
            want = ref.evict(cases[1], w, cases[1].lens.clone(), 60, 4)
            CacheEvict(caches[1], w, cases[1].lens.clone(), keep=60, recent=4, lens_out=cases[1].lens).run()
            assert same(cases[1].k_pool, want[3]) and torch.equal(cases[1].lens, want[0])
    del cut
