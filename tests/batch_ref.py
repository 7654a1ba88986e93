"""Plain 64-bit implementations of the batch operators and the cases they are
tested on. Tolerances are derived here, from the kernels' roundings."""
import math
from dataclasses import dataclass

import torch

PAGE = 16


@dataclass
class Case:
    k_pool: torch.Tensor
    v_pool: torch.Tensor
    table: torch.Tensor
    lens: torch.Tensor
    q: torch.Tensor
    k_new: torch.Tensor
    v_new: torch.Tensor


def make_case(lens, hq, hkv, d, dtype, seed=0, device="cuda", spare=1, poison=True, width=None):
    """Sequences of the given lengths with room for `spare` more tokens, their
    pages scattered over pools whose unused slots hold NaN."""
    g = torch.Generator().manual_seed(seed)
    per_row = [max(0, -(-(max(n, 0) + spare) // PAGE)) for n in lens]
    width = width or max(1, max(per_row))
    total = sum(per_row)
    pool = total + 3
    table = torch.full((len(lens), width, 2), -1, dtype=torch.int32)
    ids = [torch.randperm(pool, generator=g), torch.randperm(pool, generator=g)]
    at = 0
    pools = [torch.full((pool, PAGE, hkv, d), float("nan")) if poison else torch.zeros(pool, PAGE, hkv, d)
             for _ in range(2)]
    for b, n in enumerate(lens):
        for w in range(2):
            mine = ids[w][at:at + per_row[b]]
            table[b, :per_row[b], w] = mine.int()
            rows = torch.randn((per_row[b] * PAGE, hkv, d), generator=g)
            rows[max(n, 0):] = float("nan") if poison else 0.0
            pools[w][mine] = rows.view(per_row[b], PAGE, hkv, d)
        at += per_row[b]
    rand = lambda *s: torch.randn(s, generator=g).to(dtype).to(device)  # noqa: E731
    return Case(pools[0].to(dtype).to(device), pools[1].to(dtype).to(device), table.to(device),
                torch.tensor(lens, dtype=torch.int32, device=device), rand(len(lens), hq, d), rand(len(lens), hkv, d),
                rand(len(lens), hkv, d))


def rows_of(c: Case, b, append):
    """(K, V) of sequence b's tokens, [n, Hkv, D] in 64 bits."""
    n = int(c.lens[b])
    t = torch.arange(n, device=c.lens.device)
    ids = c.table[b].long()[t // PAGE]
    k, v = c.k_pool[ids[:, 0], t % PAGE].double(), c.v_pool[ids[:, 1], t % PAGE].double()
    if append:
        k, v = torch.cat([k, c.k_new[b, None].double()]), torch.cat([v, c.v_new[b, None].double()])
    return k, v


def decode(c: Case, append=True, scale=None, pages=None):
    """out, lse [B, Hq], weights (list of [Hkv, n], summed over the group) and
    the error allowed per output before its last rounding."""
    batch, hq, d = c.q.shape
    hkv = c.k_pool.shape[2]
    group = hq // hkv
    scale = d ** -0.5 if scale is None else scale
    dev = c.q.device
    out = torch.zeros(batch, hq, d, dtype=torch.float64, device=dev)
    slack = torch.zeros_like(out)
    lse = torch.full((batch, hq), -math.inf, dtype=torch.float64, device=dev)
    lse_slack = torch.zeros_like(lse)
    weights, weight_slack = [], []
    p_split = 2.0 ** -16 if c.q.dtype == torch.bfloat16 else 2.0 ** -22
    for b in range(batch):
        if int(c.lens[b]) < 0:
            weights.append(None), weight_slack.append(None)
            continue
        k, v = rows_of(c, b, append)
        n = k.shape[0]
        total, allowed = torch.zeros(hkv, n, dtype=torch.float64, device=dev), torch.zeros(hkv, n, dtype=torch.float64, device=dev)
        for h in range(hkv):
            use = torch.arange(n, device=dev)
            if pages is not None:
                in_use = -(-n // PAGE)
                listed = [int(x) for x in pages[b, h, :min(pages.shape[2], in_use)].tolist() if 0 <= int(x) < in_use]
                use = torch.cat([use[x * PAGE:(x + 1) * PAGE] for x in listed] + [use[:0]])
            if use.numel() == 0:
                continue
            for g in range(h * group, (h + 1) * group):
                q = c.q[b, g].double()
                s = scale * (k[use, h] @ q)
                p = s.softmax(-1)
                out[b, g] = p @ v[use, h]
                lse[b, g] = s.logsumexp(-1)
                if pages is None:
                    total[h] += p
                # fp32: the dot product (D roundings of its running sum), its scaling, the
                # exponential's argument and value; the sums over the tokens; P's two 16-bit terms
                # (and, in f16, what lies below their smallest step).
                dot = abs(scale) * (k[use, h].abs() @ q.abs())
                most = lambda x: float(x[torch.isfinite(x)].max()) if bool(torch.isfinite(x).any()) else 0.0  # noqa: E731
                e_s = (d + 4) * 2.0 ** -24 * most(dot) + 4 * 2.0 ** -24 * most(s.abs())
                rel = 2 * e_s + 2.0 ** -21 + (len(use) + 8) * 2.0 ** -24
                weigh = p @ v[use, h].abs()
                slack[b, g] = (rel + p_split) * weigh + 2.0 ** -24 * v[use, h].abs().sum(0) + 2.0 ** -126
                lse_slack[b, g] = e_s + rel + 2.0 ** -22 * abs(float(lse[b, g]))
                if pages is None:
                    allowed[h] += (2 * rel + 2.0 ** -21 * (1 + abs(float(lse[b, g])))) * p + 2.0 ** -100
        weights.append(total), weight_slack.append(allowed)
    return dict(out=out, slack=slack, lse=lse, lse_slack=lse_slack, weights=weights, weight_slack=weight_slack)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def check_close(got, want, slack, what=""):
    """|got - want| within the computation's slack and one rounding to got's type."""
    g = got.double()
    assert g.shape == want.shape
    assert torch.equal(torch.isnan(g), torch.isnan(want)), f"{what}: NaN in other places"
    fine = torch.isfinite(want)
    assert torch.equal(g[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), f"{what}: infinities"
    # bf16 outputs flush what is subnormal, f16 ones step evenly below their smallest normal value.
    tiny = torch.finfo(got.dtype).tiny * (1.0 if got.dtype == torch.bfloat16 else torch.finfo(got.dtype).eps)
    bound = slack + half_step(got.dtype) * (want.abs() + slack) + tiny
    over = ((g - want).abs() - bound)[fine]
    assert over.numel() == 0 or float(over.max()) <= 0, f"{what}: {float((g - want).abs()[fine].max()):.3g} off, " \
        f"{float(over.max()):.3g} above the bound"


def bounds(c: Case, into, start=None, extra=0):
    into = into.clone()
    for b, n in enumerate(c.lens.tolist()):
        if n < 0:
            continue
        n += extra
        first = 0 if start is None else int(start[b]) // PAGE
        for lp in range(first, -(-n // PAGE)):
            page = int(c.table[b, lp, 0])
            rows = c.k_pool[page, :min(PAGE, n - lp * PAGE)].double()
            into[page, :, 0], into[page, :, 1] = rows.amin(0).to(into.dtype), rows.amax(0).to(into.dtype)
    return into


def select(c: Case, bound, n_pages, first, last, extra):
    batch, hq, d = c.q.shape
    hkv = c.k_pool.shape[2]
    group = hq // hkv
    pages = torch.full((batch, hkv, n_pages), -1, dtype=torch.int32)
    for b, n in enumerate(c.lens.tolist()):
        if n < 0:
            continue
        live = -(-(n + extra) // PAGE)
        for h in range(hkv):
            rank = []
            for lp in range(live):
                if lp < first or lp >= live - last:
                    rank.append((-3, 0.0, lp))
                    continue
                lo, hi = bound[int(c.table[b, lp, 0]), h].double()
                u = [(torch.where(x >= 0, x * hi, x * lo)).sum().item() for x in c.q[b, h * group:(h + 1) * group].double()]
                rank.append((-2, 0.0, lp) if any(math.isnan(x) for x in u) else (0, -max(u), lp))
            took = sorted(x[2] for x in sorted(rank)[:n_pages])
            pages[b, h, :len(took)] = torch.tensor(took, dtype=torch.int32)
    return pages


def evict(c: Case, weights, seen, keep, recent, tracked=None, positions=None):
    """(lens, weights, positions, K pool, V pool) afterwards; weights and
    positions below the new length only (the rest as it was / 0)."""
    batch, hkv, _ = weights.shape
    lens, w_out = c.lens.clone(), weights.clone()
    p_out = positions.clone() if positions is not None else torch.zeros(weights.shape, dtype=torch.int32, device=weights.device)
    k_pool, v_pool = c.k_pool.clone(), c.v_pool.clone()
    for b, n in enumerate(c.lens.tolist()):
        if n < 0:
            continue
        left, s = min(n, keep), int(seen[b])
        lens[b] = left
        for h in range(hkv):
            known = int(tracked[b]) if tracked is not None else 0
            pos = [int(positions[b, h, t]) if t < known else s - (n - t) for t in range(n)]
            rank = []
            for t, w in enumerate(weights[b, h, :n].tolist()):
                order = 0 if pos[t] >= s - recent else 1 if math.isnan(w) else 2
                rank.append((order, -w if order == 2 else 0.0, t))
            kept = sorted(x[2] for x in sorted(rank)[:left])
            holes = [t for t in range(left) if t not in set(kept)]
            moved = [t for t in kept if t >= left]
            source = list(range(left))
            for to, of in zip(holes, moved):
                source[to] = of
                for pool, old, which in ((k_pool, c.k_pool, 0), (v_pool, c.v_pool, 1)):
                    pool[int(c.table[b, to // PAGE, which]), to % PAGE, h] = \
                        old[int(c.table[b, of // PAGE, which]), of % PAGE, h]
            w_out[b, h, :left] = weights[b, h][torch.tensor(source, dtype=torch.long, device=weights.device)] if left else w_out[b, h, :0]
            p_out[b, h, :left] = torch.tensor([pos[t] for t in source], dtype=torch.int32, device=weights.device)
    return lens, w_out, p_out, k_pool, v_pool
