"""How many bits of the attention weights reach the outputs of the batch decode."""
import math

import pytest
import torch

import batch_ref as ref

pytestmark = pytest.mark.gpu


def one_score_each(lens, gaps, dtype, hkv=8, d=64):
    """Sequences whose token 0 scores gaps[b] nats above all others (scale 1,
    exact in the type); its value is 0, the others' are 1 to 4."""
    c = ref.make_case(lens, hkv, hkv, d, dtype, seed=len(lens), spare=0)
    c.q.zero_()
    c.q[..., 0] = 1
    g = torch.Generator("cuda").manual_seed(1)
    c.k_pool.zero_()
    c.v_pool.copy_(torch.randint(1, 5, c.v_pool.shape, generator=g, device="cuda"))
    for b, gap in enumerate(gaps):
        k_id, v_id = c.table[b, 0].tolist()
        c.k_pool[k_id, 0, :, 0] = gap
        c.v_pool[v_id, 0] = 0
    return c


def shares(c, gaps):
    """The outputs by the formula, in 64 bits, and the sums of the values behind token 0."""
    out, sums = torch.zeros(c.q.shape, dtype=torch.float64, device="cuda"), torch.zeros(c.q.shape, dtype=torch.float64, device="cuda")
    for b, gap in enumerate(gaps):
        n = int(c.lens[b])
        t = torch.arange(n, device="cuda")
        sums[b] = c.v_pool[c.table[b].long()[t // 16, 1], t % 16].double().sum(0)
        out[b] = sums[b] * math.exp(-gap) / (1 + (n - 1) * math.exp(-gap))
    return out, sums


# Scores are exact products; in log2 units they carry two roundings (the scale's
# and their own) and the difference to the maximum one more: 3 x 2^-24 of gap x
# log2 e, which as a relative error of the weight is 3 x 2^-24 of the gap in nats.
# The exponential is good to 2^-22, the sums of n weights and the reciprocal's
# product to (n + 8) x 2^-24. (All relative to the output.)
def relative(gap, n):
    return (3 * gap + 4 + n + 8) * 2.0 ** -24


@pytest.mark.parametrize("gap", [4.5, 11.75, 13.0, 16.0, 17.5])
def test_small_weights_in_f16(gap):
    """Whole sequences a worker, the leading token's value 0: the output is what
    the weights far below the maximum hold. Of 2^15 times a weight two f16 terms
    keep 22 bits, or steps of 2^-24: half a step is 2^-40 of the largest weight."""
    from genllm_b200.batch import PagedBatch, batch_decode
    n = 64
    lens, gaps = [n] * 300, [gap] * 300
    c = one_score_each(lens, gaps, torch.float16)
    got = batch_decode(PagedBatch(c.k_pool, c.v_pool, c.table, c.lens), c.q, scale=1.0,
                       out=torch.zeros(c.q.shape, device="cuda")).double()
    want, sums = shares(c, gaps)
    slack = want * (relative(gap, n) + 2.0 ** -22) + sums * 2.0 ** -40
    assert float(((got - want).abs() - slack).max()) <= 0, float(((got - want).abs() / want).max())


def test_weights_in_bf16_keep_their_bits():
    """An f32 output shows the weights' 24 bits: three bf16 terms hold them all."""
    from genllm_b200.batch import PagedBatch, batch_decode
    n = 8
    gaps = [0.5 + i / 64 for i in range(64)]
    c = one_score_each([n] * 64, gaps, torch.bfloat16)
    assert c.k_pool[:, 0, 0, 0].float().unique().numel() > 32
    gaps = [float(c.k_pool[int(c.table[b, 0, 0]), 0, 0, 0]) for b in range(64)]  # as bf16 holds them
    got = batch_decode(PagedBatch(c.k_pool, c.v_pool, c.table, c.lens), c.q, scale=1.0,
                       out=torch.zeros(c.q.shape, device="cuda")).double()
    want, _ = shares(c, gaps)
    slack = want * torch.tensor([relative(gap, n) for gap in gaps], device="cuda").view(-1, 1, 1)
    assert float(((got - want).abs() - slack).max()) <= 0, float(((got - want).abs() / want).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hkv,group,d", [(1, 1, 64), (8, 4, 128), (2, 16, 256)])
def test_every_page_of_a_long_row_is_in_the_output(hkv, group, d, dtype):
    """Equal scores, page j's values 1 in dimension j mod D alone: an output is a
    count over n, which holds one rounding of 1/n and one of the product."""
    from genllm_b200.batch import PagedBatch, batch_decode
    n = 30001
    pages = -(-n // 16)
    g = torch.Generator("cuda").manual_seed(2)
    table = torch.stack([torch.randperm(pages, generator=g, device="cuda") for _ in range(2)], -1).int()[None].contiguous()
    k_pool = torch.randn(pages, 16, hkv, d, generator=g, device="cuda").to(dtype)
    v_pool = torch.zeros(pages, 16, hkv, d, dtype=dtype, device="cuda")
    lp = torch.arange(pages, device="cuda")
    v_pool[table[0, :, 1].long(), :, :, lp % d] = 1
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    q = torch.zeros(1, hkv * group, d, dtype=dtype, device="cuda")
    got = batch_decode(PagedBatch(k_pool, v_pool, table, lens), q, out=torch.zeros(q.shape, device="cuda")).double()
    rows = torch.full((pages,), 16.0, dtype=torch.float64, device="cuda")
    rows[-1] = n - 16 * (pages - 1)
    want = torch.zeros(d, dtype=torch.float64, device="cuda").index_add_(0, lp % d, rows) / n
    assert float(((got - want).abs() - 3 * 2.0 ** -24 * want).max()) <= 0
