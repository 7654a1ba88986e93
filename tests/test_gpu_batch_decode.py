"""gkv_batch_decode against the 64-bit definition (batch_ref.decode)."""
import pytest
import torch

import batch_ref as ref

pytestmark = pytest.mark.gpu


def run(c, append=True, dtype=None, **options):
    from genllm_b200.batch import PagedBatch, batch_decode
    cache = PagedBatch(c.k_pool, c.v_pool, c.table, c.lens)
    out = torch.full(tuple(c.q.shape), 7.0, dtype=dtype or c.q.dtype, device=c.q.device)
    lse = torch.full(tuple(c.q.shape[:2]), 7.0, device=c.q.device)
    args = (c.k_new, c.v_new) if append else ()
    batch_decode(cache, c.q, *args, out=out, lse=lse, **options)
    assert cache.check_device_errors() == 0
    return out, lse


def check(c, out, lse, want, rows=None):
    live = (c.lens >= 0).cpu()
    ref.check_close(out[live], want["out"][live], want["slack"][live], "out")
    fine = torch.isfinite(want["lse"][live])
    got = lse[live].double()
    assert torch.equal(torch.isfinite(got), fine)
    over = (got - want["lse"][live]).abs() - want["lse_slack"][live]
    assert not fine.any() or float(over[fine].max()) <= 0
    assert bool((out[~live] == 7.0).all()) and bool((lse[~live] == 7.0).all())  # skipped rows stay as they were


RAGGED = [0, 1, 15, 16, 17, -1, 33, 100, 255, 256, 257, 700]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hkv", [(8, 8), (4, 1), (14, 2), (9, 3), (32, 2), (5, 5), (22, 11), (40, 8)])
def test_ragged(hq, hkv, d, dtype):
    c = ref.make_case(RAGGED, hq, hkv, d, dtype, seed=hq + d)
    want = ref.decode(c)
    before_k, before_v = c.k_pool.clone(), c.v_pool.clone()
    out, lse = run(c)
    check(c, out, lse, want)
    # Only the new tokens' slots changed, to the rows given.
    for pool, before, new, which in ((c.k_pool, before_k, c.k_new, 0), (c.v_pool, before_v, c.v_new, 1)):
        for b, n in enumerate(c.lens.tolist()):
            if n >= 0:
                before[int(c.table[b, n // 16, which]), n % 16] = new[b]
        assert torch.equal(pool.view(torch.int16), before.view(torch.int16))


@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (8, 1, 64), (16, 1, 128), (4, 4, 256)])
@pytest.mark.parametrize("lens", [[5000], [0], [1], [4097, 3, 2500], [20000, 0, 17]])
def test_split_lengths(lens, hq, hkv, d):
    c = ref.make_case(lens, hq, hkv, d, torch.bfloat16, seed=sum(lens))
    out, lse = run(c)
    check(c, out, lse, ref.decode(c))


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_without_append(out_dtype):
    c = ref.make_case(RAGGED, 16, 8, 128, torch.bfloat16, seed=3)
    pools = c.k_pool.clone(), c.v_pool.clone()
    out, lse = run(c, append=False, dtype=out_dtype)
    check(c, out, lse, ref.decode(c, append=False))
    zero = RAGGED.index(0)
    assert bool((out[zero] == 0).all()) and bool((lse[zero] == -float("inf")).all())
    for a, b in zip(pools, (c.k_pool, c.v_pool)):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))


def test_many_short_sequences():
    lens = [(7 * i) % 40 - 1 for i in range(700)]
    c = ref.make_case(lens, 4, 2, 64, torch.float16, seed=11)
    out, lse = run(c)
    check(c, out, lse, ref.decode(c))


def test_strided_inputs_and_table():
    c = ref.make_case([40, 7, 300], 12, 4, 128, torch.bfloat16, seed=5)
    want = ref.decode(c)
    big = torch.zeros(3, 2, 12 + 4 + 4, 128, dtype=torch.bfloat16, device="cuda")
    big[:, 1, :12], big[:, 1, 12:16], big[:, 1, 16:] = c.q, c.k_new, c.v_new
    table = torch.zeros(3, c.table.shape[1] + 5, 2, dtype=torch.int32, device="cuda")
    table[:, :c.table.shape[1]] = c.table
    c.q, c.k_new, c.v_new, c.table = big[:, 1, :12], big[:, 1, 12:16], big[:, 1, 16:], table[:, :c.table.shape[1]]
    assert not c.q.is_contiguous()
    out, lse = run(c)
    check(c, out, lse, want)


def test_large_scores_and_scale():
    """One token per sequence holds all the weight: the maximum moves late."""
    c = ref.make_case([600, 90], 16, 8, 128, torch.bfloat16, seed=6)
    for b, t in ((0, 599), (1, 40)):
        page = int(c.table[b, t // 16, 0])
        c.k_pool[page, t % 16] = c.q[b, ::2] * 4
    out, lse = run(c, scale=0.5)
    check(c, out, lse, ref.decode(c, scale=0.5))


def test_infinite_and_nan_rows():
    """-inf scores carry no weight, NaN keys reach their head alone."""
    c = ref.make_case([64, 50, 20], 8, 4, 64, torch.float16, seed=7)
    c.q = c.q.abs() + 0.1
    c.k_pool[int(c.table[0, 1, 0]), 3, 1] = -float("inf")
    c.k_pool[int(c.table[1, 0, 0]), 2, 2] = float("nan")
    c.k_pool[int(c.table[2, 0, 0]), :, 0] = -float("inf")
    c.k_pool[int(c.table[2, 1, 0]), :4, 0] = -float("inf")
    c.k_new[2, 0] = -float("inf")  # nothing but -inf for this head: not a number, as the definition has it
    out, lse = run(c)
    o = out.double()
    want = ref.decode(c)
    assert torch.equal(torch.isnan(o), torch.isnan(want["out"]))
    assert bool(torch.isnan(o[1, 4:6]).all()) and bool(torch.isnan(o[2, 0:2]).all())
    ok = ~torch.isnan(want["out"])
    ref.check_close(out[ok], want["out"][ok], want["slack"][ok])


@pytest.mark.parametrize("n_list", [1, 5, 64])
@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (7, 1, 64), (6, 3, 256)])
def test_page_lists(hq, hkv, d, n_list):
    lens = [0, 5, 16, 200, 1500, -1, 31]
    c = ref.make_case(lens, hq, hkv, d, torch.bfloat16, seed=8)
    g = torch.Generator().manual_seed(9)
    pages = torch.full((len(lens), hkv, n_list), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        live = -(-(max(n, 0) + 1) // 16)
        for h in range(hkv):
            pick = torch.randperm(live, generator=g)[:n_list].int()
            pages[b, h, :len(pick)] = pick
            if h % 3 == 2:
                pages[b, h, 0] = -1
            if b == 3 and h == 0:
                pages[b, h] = -1  # nothing is listed: zeros
            if b == 4 and n_list >= 5:
                pages[b, h, 1] = 1 << 20
    pages = pages.cuda()
    want = ref.decode(c, pages=pages)
    out, lse = run(c, pages=pages)
    check(c, out, lse, want)
    assert bool((out[3, :hq // hkv] == 0).all())
    # The new token is appended whether or not its page is listed.
    for b, n in enumerate(lens):
        if n >= 0:
            assert torch.equal(c.k_pool[int(c.table[b, n // 16, 0]), n % 16], c.k_new[b])


@pytest.mark.parametrize("decay,in_place,append", [(1.0, False, True), (0.9, True, True), (0.0, False, False)])
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (7, 1, 64), (10, 5, 256), (32, 2, 64)])
def test_totals(hq, hkv, d, decay, in_place, append):
    from genllm_b200.batch import PagedBatch, BatchDecode
    lens = [0, 1, 16, 33, 900, -1, 4000]
    c = ref.make_case(lens, hq, hkv, d, torch.bfloat16, seed=12)
    want = ref.decode(c, append=append)
    w = torch.rand(len(lens), hkv, 16 * c.table.shape[1] + 3, device="cuda")
    before = w.clone()
    w_out = w if in_place else torch.full_like(w, 5.0)
    rest = w_out.clone()
    cache = PagedBatch(c.k_pool, c.v_pool, c.table, c.lens)
    new = (c.k_new, c.v_new) if append else ()
    BatchDecode(cache, c.q, *new, weights=w, weights_out=w_out, decay=decay).run()
    assert cache.check_device_errors() == 0
    for b, n in enumerate(lens):
        m = 0 if n < 0 else n + append
        assert torch.equal(w_out[b, :, m:], rest[b, :, m:])
        if m == 0:
            continue
        old = before[b, :, :m].double()
        old[:, n:] = 0
        exact = decay * old + want["weights"][b]
        slack = want["weight_slack"][b] + 3 * 2.0 ** -24 * (decay * old + want["weights"][b])
        ref.check_close(w_out[b, :, :m], exact, slack, f"totals of {n}")


@pytest.mark.parametrize("hq,hkv,d", [(8, 1, 64), (32, 2, 64), (14, 2, 128), (12, 3, 64), (20, 4, 128), (4, 1, 256), (32, 2, 256)])
@pytest.mark.parametrize("lens", [[9000], [16 * 592], [16 * 1184 - 1], [300, 20000, 0, 15], [31, 5000, 47, 5000, 1],
                                  [2000] * 9, [16 * 37] * 32])
def test_workers_of_a_block_share_a_sequence(hq, hkv, d, lens):
    """Few kv heads: several workers of a block hold parts of one sequence."""
    c = ref.make_case(lens, hq, hkv, d, torch.bfloat16, seed=40)
    out, lse = run(c)
    check(c, out, lse, ref.decode(c))
    again, lse_again = run(c)
    assert torch.equal(out.view(torch.int16), again.view(torch.int16)) and torch.equal(lse, lse_again)


@pytest.mark.parametrize("hq,hkv,d", [(8, 1, 64), (14, 2, 128), (20, 4, 128), (4, 1, 256)])
def test_parts_without_a_key(hq, hkv, d):
    """Lists of which long runs name no page: whole parts, and whole blocks' parts, attend nothing."""
    c = ref.make_case([9000, 20000, 40], hq, hkv, d, torch.bfloat16, seed=41)
    n = c.table.shape[1]
    pages = torch.arange(n, dtype=torch.int32, device="cuda").expand(3, hkv, n).contiguous()
    pages[0, :, :300] = -1
    pages[1, 0, 20:1200] = -1
    pages[1, hkv - 1, 700:] = -1
    pages[2] = -1
    out, lse = run(c, pages=pages)
    check(c, out, lse, ref.decode(c, pages=pages))


def test_totals_without_a_total_so_far():
    from genllm_b200.batch import PagedBatch, batch_decode
    c = ref.make_case([50], 4, 2, 64, torch.bfloat16)
    w = torch.empty(1, 2, 64, device="cuda")
    batch_decode(PagedBatch(c.k_pool, c.v_pool, c.table, c.lens), c.q, c.k_new, c.v_new, weights_out=w)
    assert torch.allclose(w[..., :51].sum(-1), torch.full((1, 2), 2.0, device="cuda"), atol=1e-4)


def test_bits_repeat():
    c = ref.make_case([3000, 17, 800, 0], 16, 4, 128, torch.bfloat16, seed=13)
    a, la = run(c)
    for _ in range(3):
        b, lb = run(c)
        assert torch.equal(a.view(torch.int16), b.view(torch.int16)) and torch.equal(la, lb)


def test_bad_pages_and_lengths_are_flagged():
    """Checked in the kernel: the page is skipped, the word is set, the stream goes on."""
    from genllm_b200.batch import PagedBatch, batch_decode
    c = ref.make_case([100, 40, 33], 8, 4, 64, torch.bfloat16, seed=14)
    want = ref.decode(c)
    c.table[1, 1, 1] = c.k_pool.shape[0]
    c.table[0, 6, 0] = -5  # the page that would receive the new token
    cache = PagedBatch(c.k_pool, c.v_pool, c.table, c.lens)
    out = batch_decode(cache, c.q, c.k_new, c.v_new)
    assert cache.check_device_errors() == 1
    assert cache.check_device_errors() == 0
    ref.check_close(out[2], want["out"][2], want["slack"][2])
    c = ref.make_case([100, 40], 8, 4, 64, torch.bfloat16, seed=15)
    c.lens[0] = 1 << 30
    c.lens[1] = 16 * c.table.shape[1]  # full: no slot for the new token
    pools = c.k_pool.clone()
    cache = PagedBatch(c.k_pool, c.v_pool, c.table, c.lens)
    batch_decode(cache, c.q, c.k_new, c.v_new)
    assert cache.check_device_errors() & 4
    assert torch.equal(pools.view(torch.int16), c.k_pool.view(torch.int16))


@pytest.mark.parametrize("lens", [[40], [5000, 40]])
def test_totals_of_a_sequence_of_bad_pages(lens):
    """No page can be read: no attention, so the totals only decay."""
    from genllm_b200.batch import PagedBatch, batch_decode
    c = ref.make_case(lens, 8, 4, 64, torch.bfloat16, seed=17)
    c.table[0] = -1
    w = torch.rand(len(lens), 4, 16 * c.table.shape[1], device="cuda")
    before = w.clone()
    cache = PagedBatch(c.k_pool, c.v_pool, c.table, c.lens)
    lse = torch.zeros(len(lens), 8, device="cuda")
    out = batch_decode(cache, c.q, c.k_new, c.v_new, lse=lse, weights=w, weights_out=w, decay=0.5)
    assert cache.check_device_errors() == 1
    n = lens[0]
    assert bool((out[0] == 0).all()) and bool((lse[0] == -float("inf")).all())
    assert torch.equal(w[0, :, :n], 0.5 * before[0, :, :n]) and bool((w[0, :, n] == 0).all())
    assert torch.equal(w[0, :, n + 1:], before[0, :, n + 1:])


def test_captured_steps_follow_the_lengths():
    """One capture, replayed while the lengths and the table move."""
    from genllm_b200.batch import PagedBatch, BatchDecode
    lens = [0, 14, 200, -1]
    c = ref.make_case(lens, 16, 8, 128, torch.bfloat16, seed=16, spare=40)
    cache = PagedBatch(c.k_pool, c.v_pool, c.table, c.lens)
    step = BatchDecode(cache, c.q, c.k_new, c.v_new, lse=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step.run()
    g = torch.Generator("cuda").manual_seed(1)
    for _ in range(30):
        for t in (c.q, c.k_new, c.v_new):
            t.copy_(torch.randn(t.shape, generator=g, device="cuda").to(t.dtype))
        want = ref.decode(c)
        graph.replay()
        live = (c.lens >= 0).cpu()
        ref.check_close(step.out[live], want["out"][live], want["slack"][live])
        c.lens += (c.lens >= 0).int()
    assert cache.check_device_errors() == 0


def test_two_streams_at_once():
    from genllm_b200.batch import PagedBatch, BatchDecode
    cases = [ref.make_case([2000 + 100 * i, 30], 16, 8, 128, torch.bfloat16, seed=20 + i) for i in range(2)]
    wants = [ref.decode(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in range(2)]
    steps = [BatchDecode(PagedBatch(c.k_pool, c.v_pool, c.table, c.lens), c.q, c.k_new, c.v_new) for c in cases]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for step, s in zip(steps, streams):
            step.run(stream=s)
    torch.cuda.synchronize()
    for step, w in zip(steps, wants):
        ref.check_close(step.out, w["out"], w["slack"])


def test_shared_prefix_pages():
    """Sequences may read the same pages."""
    c = ref.make_case([64, 64, 64], 8, 8, 64, torch.float16, seed=30)
    c.table[1:, :4] = c.table[0, :4]
    want = ref.decode(c)
    out, lse = run(c)
    check(c, out, lse, want)


def test_offsets_behind_32_bits():
    """Pages whose bytes and elements lie behind 2^32."""
    hkv, d = 8, 128
    pages = (1 << 32) // (16 * hkv * d) + 40  # elements pass 2^32
    k_pool = torch.empty(pages, 16, hkv, d, dtype=torch.bfloat16, device="cuda")
    v_pool = torch.empty_like(k_pool)
    c = ref.make_case([100, 60], 16, hkv, d, torch.bfloat16, seed=31)
    want = ref.decode(c)
    n = c.k_pool.shape[0]
    k_pool[pages - n:], v_pool[pages - n:] = c.k_pool, c.v_pool
    c.table = torch.where(c.table >= 0, c.table + (pages - n), c.table)
    c.k_pool, c.v_pool = k_pool, v_pool
    out, lse = run(c)
    check(c, out, lse, want)
    assert torch.equal(k_pool[int(c.table[0, 6, 0]), 4], c.k_new[0])
