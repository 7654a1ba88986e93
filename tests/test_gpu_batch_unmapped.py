"""Pages that are not in the pool, and lengths beyond the table row: what the
batch operators leave behind when they skip them."""
import pytest
import torch

import batch_ref as ref

pytestmark = pytest.mark.gpu


def cache_of(c):
    from genllm_b200.batch import PagedBatch
    return PagedBatch(c.k_pool, c.v_pool, c.table, c.lens)


def listed(c, bound, n_pages, first, last, extra, mapped):
    """The definition for sequence 0: forced pages, then mapped ones by score, then the others by index."""
    hkv, group = c.k_pool.shape[2], c.q.shape[1] // c.k_pool.shape[2]
    live = -(-(int(c.lens[0]) + extra) // 16)
    lists = torch.full((1, hkv, n_pages), -1, dtype=torch.int32)
    for h in range(hkv):
        rank = []
        for lp in range(live):
            if lp < first or lp >= live - last:
                rank.append((0, 0.0, lp))
            elif lp in mapped:
                lo, hi = bound[int(c.table[0, lp, 0]), h].double()
                rank.append((1, -max(float(torch.where(x >= 0, x * hi, x * lo).sum())
                                     for x in c.q[0, h * group:(h + 1) * group].double()), lp))
            else:
                rank.append((2, 0.0, lp))
        took = sorted(x[2] for x in sorted(rank)[:n_pages])
        lists[0, h, :len(took)] = torch.tensor(took, dtype=torch.int32)
    return lists


# A row by one CTA of 512 threads, by one of 1024, by a cluster, with its keys in the workspace.
@pytest.mark.parametrize("wide", [0, 5000, 20000, 140000])
@pytest.mark.parametrize("first,last", [(0, 0), (2, 1)])
@pytest.mark.parametrize("pages,mapped,n_pages", [(20, (1, 4, 9, 13, 18), 8), (20, (), 8), (20, (0, 1, 19), 19),
                                                  (100, (3, 50, 51, 77), 40), (100, (), 99), (300, (0, 299), 70)])
def test_a_cut_among_unmapped_pages(pages, mapped, n_pages, first, last, wide):
    from genllm_b200.batch import page_bounds, select_pages
    c = ref.make_case([16 * pages - 1], 4, 2, 64, torch.bfloat16, seed=pages + n_pages)
    bound = page_bounds(cache_of(c))
    keep = torch.zeros(pages, dtype=torch.bool, device="cuda")
    keep[list(mapped)] = True
    c.table[0, :pages][~keep] = -1
    if wide:
        table = torch.full((1, wide, 2), -1, dtype=torch.int32, device="cuda")
        table[:, :pages] = c.table
        c.table = table
    cache = cache_of(c)
    got = torch.full((1, 2, n_pages), 77, dtype=torch.int32, device="cuda")
    select_pages(cache, c.q, bound, n_pages, first=first, last=last, extra=1, pages=got)
    assert cache.check_device_errors() == 1
    assert torch.equal(got.cpu(), listed(c, bound, n_pages, first, last, 1, set(mapped)))


def evicted(c, w, seen, keep, recent, bad):
    """The definition where some pages cannot be read or written: a slot whose
    move is skipped keeps its own token, weight and position. All arrays."""
    batch, hkv, width = w.shape
    w_out, k_pool, v_pool = w.clone(), c.k_pool.clone(), c.v_pool.clone()
    p_out = torch.zeros(w.shape, dtype=torch.int32)
    cap = 16 * c.table.shape[1]
    lens = torch.zeros(batch, dtype=torch.int32)
    for b, length in enumerate(c.lens.tolist()):
        n = min(length, cap)
        left = min(n, keep)
        lens[b] = left
        pos = [int(seen[b]) - (length - t) for t in range(n)]
        for h in range(hkv):
            x = w[b, h].tolist()
            rank = sorted(range(n), key=lambda t: (0, 0.0, t) if pos[t] >= int(seen[b]) - recent else (1, -x[t], t))[:left]
            source = list(range(left))
            for to, of in zip(sorted(set(range(left)) - set(rank)), sorted(t for t in rank if t >= left)):
                if (b, to // 16) in bad or (b, of // 16) in bad:
                    continue
                source[to] = of
                for pool, old, which in ((k_pool, c.k_pool, 0), (v_pool, c.v_pool, 1)):
                    pool[int(c.table[b, to // 16, which]), to % 16, h] = old[int(c.table[b, of // 16, which]), of % 16, h]
            w_out[b, h, :left] = w[b, h, torch.tensor(source, device=w.device)]
            p_out[b, h, :left] = torch.tensor([pos[t] for t in source], dtype=torch.int32)
    return lens, w_out, p_out, k_pool, v_pool


def same(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("bad", [[(0, 1, 0), (0, 5, 1)], [(0, 0, 1), (1, 20, 0), (1, 3, 0)], [(1, i, 1) for i in range(12, 25)]])
def test_a_move_that_is_skipped_leaves_its_slot(bad, in_place):
    from genllm_b200.batch import CacheEvict
    c = ref.make_case([100, 395], 2, 2, 64, torch.bfloat16, seed=21)
    for b, lp, which in bad:
        c.table[b, lp, which] = (1 << 20) if which else -3
    g = torch.Generator("cuda").manual_seed(22)
    w = torch.rand((2, 2, 16 * c.table.shape[1]), generator=g, device="cuda")
    seen = c.lens + 7
    want = evicted(c, w, seen, 60, 9, {(b, lp) for b, lp, _ in bad})
    cache = cache_of(c)
    options = dict(lens_out=c.lens) if in_place else dict(weights_out=w.clone())
    op = CacheEvict(cache, w, seen, keep=60, recent=9, **options)
    assert torch.equal(op.run().cpu(), want[0])
    assert cache.check_device_errors() == 1
    assert torch.equal(op.weights_out, want[1]) and torch.equal(op.positions_out.cpu(), want[2])
    assert same(c.k_pool, want[3]) and same(c.v_pool, want[4])


def test_positions_of_a_length_beyond_the_table_row():
    """Slot t holds position seen - (lens - t) whatever the row holds of them."""
    from genllm_b200.batch import CacheEvict
    c = ref.make_case([111, 300], 2, 2, 64, torch.float16, seed=23)
    c.lens[0] += 20  # 131 tokens, 112 of them in the row's 7 pages
    c.table = c.table[:, :7].contiguous()
    c.lens[1] = 90
    c.k_pool.nan_to_num_(), c.v_pool.nan_to_num_()
    w = torch.rand((2, 2, 16 * 7), device="cuda")
    seen = c.lens + 4
    want = evicted(c, w, seen, 50, 30, set())
    cache = cache_of(c)
    op = CacheEvict(cache, w, seen, keep=50, recent=30)
    assert torch.equal(op.run().cpu(), want[0])
    assert cache.check_device_errors() == 4
    assert torch.equal(op.weights_out, want[1]) and torch.equal(op.positions_out.cpu(), want[2])
    assert same(c.k_pool, want[3]) and same(c.v_pool, want[4])
