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


@pytest.mark.parametrize("wide", [0, 20000, 140000])  # a row by one CTA, by a cluster, with its keys in the workspace
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
