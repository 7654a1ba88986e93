"""Cases of the batched paged-cache operators: one new token for each of many sequences over one paged KV cache.

The operators, with what they stand for in a serving loop:

* decode: append each sequence's new K/V row to its page and attend it over the sequence's cache; with ``weights`` also add
  the attention every cached token received to a running (decayed) total, which eviction ranks tokens by;
* bounds: the smallest and largest key of every page, per head and dimension, after a prompt or a step;
* sparse: pick each KV head's best pages by those bounds, attend the new token over the picked pages only, refresh the
  bounds of the page it went to;
* evict: keep the heaviest and the most recent tokens of every KV head and move the kept rows that lie behind the new
  length into the slots that became free.

``own`` False computes the plain forms below with elementary torch operations in 32 bits (the page scores in 64: a page's
place in an order hangs on their last bits); True makes the framework's calls on the same inputs.
"""
import math
import random

import torch

own = False

PAGE = 16
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # One user's next token, short context (the single-layer decode shape of the benchmark): latency counts.
        dict(name="decode 1x1024", kind="decode", batch=1, short=1024, long=1024, heads=16, kv_heads=8, dim=128, dtype="bf16",
             append=True, padded=0),
        # One user's next token, long context.
        dict(name="decode 1x32768", kind="decode", batch=1, short=32768, long=32768, heads=32, kv_heads=8, dim=128,
             dtype="bf16", append=True, padded=0),
        # A serving batch of ragged lengths, its last rows unused (a captured step of fixed batch size).
        dict(name="decode ragged 64", kind="decode", batch=64, short=16, long=8192, heads=32, kv_heads=8, dim=128,
             dtype="bf16", append=True, padded=3),
        # Small heads, an odd group of query heads, half precision, sequences from one token on, nothing appended.
        dict(name="decode f16 d64 ragged 33", kind="decode", batch=33, short=1, long=2048, heads=14, kv_heads=2, dim=64,
             dtype="f16", append=False, padded=0),
        # The attention totals behind eviction: one long context, and a ragged batch.
        dict(name="weights 1x32768", kind="weights", batch=1, short=32768, long=32768, heads=32, kv_heads=8, dim=128,
             dtype="bf16", decay=1.0),
        dict(name="weights ragged 16", kind="weights", batch=16, short=100, long=32768, heads=16, kv_heads=8, dim=128,
             dtype="bf16", decay=0.99),
        # Bounds of a prompt that was just prefilled, and of a batch of prompts.
        dict(name="bounds 1x8192", kind="bounds", batch=1, short=8192, long=8192, kv_heads=8, dim=128, dtype="bf16"),
        dict(name="bounds f16 d64 ragged 24", kind="bounds", batch=24, short=33, long=32768, kv_heads=4, dim=64, dtype="f16"),
        # A step over the best 1024 tokens' pages of a long context, and over the best 2048 of a ragged batch of longer ones.
        dict(name="sparse 1x32768", kind="sparse", batch=1, short=32768, long=32768, heads=32, kv_heads=8, dim=128,
             dtype="bf16", pages=64, first=1, last=2),
        dict(name="sparse ragged 8", kind="sparse", batch=8, short=1000, long=131072, heads=32, kv_heads=8, dim=128,
             dtype="bf16", pages=128, first=1, last=4),
        # Halving one long cache, and the steady state of a batch that is cut back to its budget every 256 tokens.
        dict(name="evict 1x32768", kind="evict", batch=1, short=32768, long=32768, kv_heads=8, dim=128, dtype="bf16",
             keep=16384, recent=1024, tracked=False),
        dict(name="evict 32x4352", kind="evict", batch=32, short=4352, long=4352, kv_heads=8, dim=128, dtype="bf16",
             keep=4096, recent=512, tracked=True),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "weights", "bounds", "sparse", "sparse", "evict"])
    heads, kv_heads = rng.choice([(16, 8), (32, 8), (14, 2), (8, 8), (8, 1), (40, 8), (12, 3), (32, 2), (24, 12), (20, 4)])
    case = dict(kind=kind, batch=_log_uniform(rng, 1, 64), heads=heads, kv_heads=kv_heads, dim=rng.choice([64, 128]),
                dtype=rng.choice(["bf16", "f16"]))
    # The longest sequence: at most 2^17 tokens and no more rows in all than the largest listed case of the kind.
    rows = {"decode": 1 << 19, "weights": 1 << 19, "bounds": 1 << 18, "sparse": 1 << 20, "evict": 1 << 19}[kind]
    top = max(32, min(1 << 17, rows // (case["batch"] * kv_heads)))
    case["long"] = _log_uniform(rng, 16, top)
    case["short"] = _log_uniform(rng, 1, case["long"])
    if kind == "decode":
        case.update(append=rng.random() < 0.7, padded=rng.choice([0, 0, min(2, case["batch"] - 1)]))
    elif kind == "weights":
        case.update(decay=rng.choice([1.0, 0.9, 0.995]))
    elif kind == "sparse":
        pages = _log_uniform(rng, 4, 256)
        case.update(pages=pages, first=rng.randint(0, 2), last=rng.randint(1, 2))
    elif kind == "evict":
        keep = _log_uniform(rng, 8, max(16, case["long"]))
        case.update(keep=keep, recent=rng.randint(0, keep // 2), tracked=rng.random() < 0.5)
    if kind in ("bounds", "evict"):
        del case["heads"]
    return case


def _lengths(case):
    """The cached tokens of each sequence, evenly spread over the logarithm from short to long; the same for every seed."""
    b, lo, hi = case["batch"], case["short"], case["long"]
    return [min(hi, max(lo, round(lo * (hi / lo) ** ((i + 0.5) / b)))) for i in range(b)]


def _inputs(case, seed):
    """The cache and the step's inputs, from the seed alone."""
    g = torch.Generator("cuda").manual_seed(seed)
    order = random.Random(seed)
    kind, hkv, dim, dtype = case["kind"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    lens = _lengths(case)
    order.shuffle(lens)
    batch = len(lens)
    # Room for one more token in every row; the pages of all rows are scattered over the pools, K and V apart.
    per_row = [(n + PAGE) // PAGE for n in lens]
    width, total = max(per_row), sum(per_row)
    pool = total + 8
    col = torch.arange(width, device="cuda")
    have = col < torch.tensor(per_row, device="cuda")[:, None]
    table = torch.full((batch, width, 2), -1, dtype=torch.int32, device="cuda")
    for which in range(2):
        table[..., which][have] = torch.randperm(pool, generator=g, device="cuda")[:total].int()

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    s = dict(case=case, k_pool=normal(pool, PAGE, hkv, dim), v_pool=normal(pool, PAGE, hkv, dim), table=table)
    for i in range(case.get("padded", 0)):
        lens[batch - 1 - i] = -1
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if kind in ("decode", "weights", "sparse"):
        s["q"] = normal(batch, case["heads"], dim)
        s["out"] = torch.zeros(batch, case["heads"], dim, dtype=dtype, device="cuda")
        if case.get("append", True):
            s["k_new"], s["v_new"] = normal(batch, hkv, dim), normal(batch, hkv, dim)
    if kind == "decode":
        s["lse"] = torch.zeros(batch, case["heads"], dtype=torch.float32, device="cuda")
    if kind in ("bounds", "sparse"):
        s["bounds"] = torch.zeros(pool, hkv, 2, dim, dtype=dtype, device="cuda")
    if kind == "sparse":
        # Kept by the steps before this one: the bounds of whole pages.
        s["bounds"][:, :, 0], s["bounds"][:, :, 1] = s["k_pool"].amin(1), s["k_pool"].amax(1)
    if kind in ("weights", "evict"):
        # Received attention is heavy-tailed.
        shape = (batch, hkv, width * PAGE)
        s["weights"] = torch.empty(shape, device="cuda").exponential_(generator=g).pow_(3)
        s["weights_out"] = torch.zeros(shape, device="cuda")
    if kind == "evict":
        # `seen` tokens in all; the first `tracked` slots were kept by an eviction before and hold tokens of any age.
        kept = [min(n, case["keep"]) if case["tracked"] else 0 for n in lens]
        seen = [n + (3 * k) // 2 for n, k in zip(lens, kept)]
        s["tracked"] = torch.tensor(kept, dtype=torch.int32, device="cuda")
        s["seen"] = torch.tensor(seen, dtype=torch.int32, device="cuda")
        old = s["seen"] - s["lens"] + s["tracked"]  # tokens seen when the tracked slots were kept
        most = max(1, max(x - n + k for x, n, k in zip(seen, lens, kept)))
        age = torch.rand((batch, hkv, most), generator=g, device="cuda")
        age.masked_fill_(torch.arange(most, device="cuda") >= old[:, None, None], 2.0)
        spread = age.argsort(-1).int()[..., : max(1, max(kept))]
        s["positions"] = torch.zeros((batch, hkv, width * PAGE), dtype=torch.int32, device="cuda")
        s["positions"][..., : spread.shape[-1]] = spread
        s["positions_out"] = torch.zeros_like(s["positions"])
        s["lens_out"] = torch.zeros_like(s["lens"])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:  # the plan that a program keeps: its buffers bound once, as its steps run on the same ones
        from genllm_b200 import batch as gb
        cache = gb.PagedBatch(s["k_pool"], s["v_pool"], s["table"], s["lens"])
        kind = case["kind"]
        if kind == "decode":
            s["plan"] = gb.BatchDecode(cache, s["q"], s.get("k_new"), s.get("v_new"), out=s["out"], lse=s["lse"])
        elif kind == "weights":
            s["plan"] = gb.BatchDecode(cache, s["q"], s["k_new"], s["v_new"], out=s["out"], weights=s["weights"],
                                       weights_out=s["weights_out"], decay=case["decay"])
        elif kind == "bounds":
            s["plan"] = gb.PageBounds(cache, s["bounds"])
        elif kind == "sparse":
            s["select"] = gb.PageSelect(cache, s["q"], s["bounds"], case["pages"], first=case["first"], last=case["last"],
                                        extra=1)
            s["plan"] = gb.BatchDecode(cache, s["q"], s["k_new"], s["v_new"], out=s["out"], pages=s["select"].pages)
            s["refresh"] = gb.PageBounds(cache, s["bounds"], start=s["lens"], extra=1)
        else:
            s["plan"] = gb.CacheEvict(cache, s["weights"], s["seen"], keep=case["keep"], recent=case["recent"],
                                      tracked=s["tracked"], positions=s["positions"], weights_out=s["weights_out"],
                                      positions_out=s["positions_out"], lens_out=s["lens_out"])
    return s


def run(s):
    kind = s["case"]["kind"]
    if not own:
        return _PLAIN[kind](s)
    if kind == "decode":
        s["plan"].run()
        return dict(out=s["out"], lse=s["lse"], k_pool=s["k_pool"], v_pool=s["v_pool"])
    if kind == "weights":
        s["plan"].run()
        return dict(out=s["out"], weights=s["weights_out"], k_pool=s["k_pool"], v_pool=s["v_pool"])
    if kind == "bounds":
        s["plan"].run()
        return dict(bounds=s["bounds"])
    if kind == "sparse":
        pages = s["select"].run()
        s["plan"].run()
        s["refresh"].run()
        return dict(pages=pages, out=s["out"], bounds=s["bounds"], k_pool=s["k_pool"], v_pool=s["v_pool"])
    s["plan"].run()
    return dict(lens=s["lens_out"], weights=s["weights_out"], positions=s["positions_out"], k_pool=s["k_pool"],
                v_pool=s["v_pool"])


# ---- plain forms ---------------------------------------------------------------------------------------------------


def _append(s):
    """Write the new rows to their slots; the rows' attended lengths."""
    if "k_new" not in s:
        return s["lens"]
    row = (s["lens"] >= 0).nonzero()[:, 0]
    at = s["lens"][row].long()
    entry = s["table"][row, at // PAGE].long()
    s["k_pool"][entry[:, 0], at % PAGE] = s["k_new"][row]
    s["v_pool"][entry[:, 1], at % PAGE] = s["v_new"][row]
    return torch.where(s["lens"] >= 0, s["lens"] + 1, s["lens"])


def _attend(q, k, v, valid):
    """Attention of q [B, Hkv, G, D] over k, v [B, Hkv, N, D] where valid [B, 1 or Hkv, N]: output, log-sum-exp, weights."""
    score = (q @ k.transpose(-1, -2)) * q.shape[-1] ** -0.5
    score = score.masked_fill(~valid[:, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = top.masked_fill(top == -math.inf, 0.0)
    p = (score - top).exp()
    total = p.sum(-1, keepdim=True)
    p = p / total.masked_fill(total == 0, 1.0)
    return p @ v, (total.log() + top)[..., 0], p


def _step(s, n):
    """The new token over the whole cache: outputs into the state's buffers, weights [B, Hkv, G, N]."""
    batch, width = s["table"].shape[:2]
    hkv, dim = s["k_pool"].shape[2:]
    valid = torch.arange(width * PAGE, device="cuda") < n[:, None]
    page = s["table"].clamp(min=0).long()
    k, v = (pool[page[..., i]].view(batch, width * PAGE, hkv, dim).float() for i, pool in enumerate((s["k_pool"], s["v_pool"])))
    k, v = (x.masked_fill_(~valid[..., None, None], 0.0).transpose(1, 2) for x in (k, v))
    q = s["q"].float().view(batch, hkv, -1, dim)
    out, lse, p = _attend(q, k, v, valid[:, None])
    live = (n >= 0)[:, None]
    s["out"].copy_(torch.where(live[..., None], out.reshape(s["out"].shape), s["out"].float()))
    if "lse" in s:
        s["lse"].copy_(torch.where(live, lse.reshape(batch, -1), s["lse"]))
    return p


def _plain_decode(s):
    _step(s, _append(s))
    return dict(out=s["out"], lse=s["lse"], k_pool=s["k_pool"], v_pool=s["v_pool"])


def _plain_weights(s):
    n = _append(s)
    p = _step(s, n).sum(2)
    t = torch.arange(p.shape[-1], device="cuda")
    before = torch.where(t < s["lens"][:, None, None], s["weights"], 0.0)
    s["weights_out"].copy_(torch.where(t < n[:, None, None], s["case"]["decay"] * before + p, s["weights_out"]))
    return dict(out=s["out"], weights=s["weights_out"], k_pool=s["k_pool"], v_pool=s["v_pool"])


def _refresh(s, start, n):
    """The bounds of every page that holds one of the tokens [start, n)."""
    batch, width = s["table"].shape[:2]
    col = torch.arange(width, device="cuda")
    row, lp = ((col >= start[:, None] // PAGE) & (col * PAGE < n[:, None])).nonzero(as_tuple=True)
    page = s["table"][row, lp, 0].long()
    rows = s["k_pool"][page].float()
    gone = (torch.arange(PAGE, device="cuda") >= (n[row] - lp * PAGE)[:, None])[..., None, None]
    s["bounds"][page, :, 0] = rows.masked_fill(gone, math.inf).amin(1).to(rows.dtype).to(s["bounds"].dtype)
    s["bounds"][page, :, 1] = rows.masked_fill(gone, -math.inf).amax(1).to(s["bounds"].dtype)


def _plain_bounds(s):
    _refresh(s, torch.zeros_like(s["lens"]), s["lens"])
    return dict(bounds=s["bounds"])


def _select(s, n):
    """The picked logical pages [B, Hkv, pages] in rising order, -1 behind them: the first and last ones, then the best."""
    case = s["case"]
    batch, width = s["table"].shape[:2]
    hkv, dim = s["k_pool"].shape[2:]
    live = (n + PAGE - 1) // PAGE
    bound = s["bounds"][s["table"][..., 0].clamp(min=0).long()].permute(0, 2, 3, 1, 4).double()  # [B, Hkv, 2, W, D]
    q = s["q"].double().view(batch, hkv, -1, dim)
    score = (bound[:, :, 0] @ q.clamp(max=0.0).transpose(-1, -2) + bound[:, :, 1] @ q.clamp(min=0.0).transpose(-1, -2)).amax(-1)
    col = torch.arange(width, device="cuda")
    there = (col < live[:, None])[:, None]
    kept = ((col < case["first"]) | (col >= live[:, None] - case["last"]))[:, None]
    score = score.masked_fill(kept, math.inf).masked_fill(~there, -math.inf)
    best = score.sort(dim=-1, descending=True, stable=True).indices[..., : case["pages"]]
    best = best.masked_fill(best >= live[:, None, None], width)
    best = best.sort(-1).values.int()
    pages = torch.full((batch, hkv, case["pages"]), -1, dtype=torch.int32, device="cuda")
    pages[..., : best.shape[-1]] = torch.where(best < live[:, None, None], best, -1)
    return pages


def _plain_sparse(s):
    lens = s["lens"]
    n = lens + 1
    pages = _select(s, n)
    _append(s)
    batch, hkv, count = pages.shape
    dim = s["q"].shape[-1]
    row = torch.arange(batch, device="cuda")[:, None, None]
    head = torch.arange(hkv, device="cuda")[None, :, None]
    lp = pages.clamp(min=0).long()
    entry = s["table"][row, lp].clamp(min=0).long()
    k, v = (pool.transpose(1, 2)[entry[..., i], head].reshape(batch, hkv, count * PAGE, dim).float()
            for i, pool in enumerate((s["k_pool"], s["v_pool"])))
    at = lp[..., None] * PAGE + torch.arange(PAGE, device="cuda")
    valid = ((at < n[:, None, None, None]) & (pages >= 0)[..., None]).view(batch, hkv, count * PAGE)
    k, v = (x.masked_fill(~valid[..., None], 0.0) for x in (k, v))
    out, _, _ = _attend(s["q"].float().view(batch, hkv, -1, dim), k, v, valid)
    s["out"].copy_(out.reshape(s["out"].shape))
    _refresh(s, lens, n)
    return dict(pages=pages, out=s["out"], bounds=s["bounds"], k_pool=s["k_pool"], v_pool=s["v_pool"])


def _plain_evict(s):
    case = s["case"]
    n, seen = (s[x][:, None, None] for x in ("lens", "seen"))
    width = s["weights"].shape[-1]
    t = torch.arange(width, device="cuda", dtype=torch.int32)
    position = torch.where(t < s["tracked"][:, None, None], s["positions"], seen - n + t)
    rank = s["weights"].masked_fill(position >= seen - case["recent"], math.inf).masked_fill(t >= n, -math.inf)
    order = rank.sort(dim=-1, descending=True, stable=True).indices
    left = n.clamp(max=case["keep"])
    kept = torch.zeros_like(rank, dtype=torch.bool).scatter_(-1, order, (t < left).expand_as(rank))
    hole, moved = ~kept & (t < left), kept & (t >= left)
    # The i-th hole takes the i-th kept row behind the new length.
    source = t.long().expand_as(rank).clone()
    source[hole] = t.long().expand_as(rank)[moved]
    stays = t < left
    s["weights_out"].copy_(torch.where(stays, s["weights"].gather(-1, source), s["weights_out"]))
    s["positions_out"].copy_(torch.where(stays, position.expand_as(rank).gather(-1, source), s["positions_out"]))
    s["lens_out"].copy_(left.view(-1))
    row, head, to = hole.nonzero(as_tuple=True)
    of = source[hole]
    for i, pool in enumerate((s["k_pool"], s["v_pool"])):
        page = s["table"][..., i].long()
        pool[page[row, to // PAGE], to % PAGE, head] = pool[page[row, of // PAGE], of % PAGE, head]
    return dict(lens=s["lens_out"], weights=s["weights_out"], positions=s["positions_out"], k_pool=s["k_pool"],
                v_pool=s["v_pool"])


_PLAIN = dict(decode=_plain_decode, weights=_plain_weights, bounds=_plain_bounds, sparse=_plain_sparse, evict=_plain_evict)


# ---- the definition in 64 bits, one sequence at a time ----------------------------------------------------------------


def exact(case, seed):
    """What is computed (outputs, log-sum-exps, attention totals); what is only moved or picked has None in its place."""
    kind = case["kind"]
    if kind in ("bounds", "evict"):
        return None
    s = _inputs(case, seed)
    hkv, dim = case["kv_heads"], case["dim"]
    group = case["heads"] // hkv
    out, lse = s["out"].double(), torch.zeros(case["batch"], case["heads"], dtype=torch.float64, device="cuda")
    total = s["weights_out"].double() if kind == "weights" else None
    new = "k_new" in s
    for b, length in enumerate(s["lens"].tolist()):
        if length < 0:
            continue
        rows = torch.arange(length, device="cuda")
        ids = s["table"][b].long()[rows // PAGE]
        key, value = s["k_pool"][ids[:, 0], rows % PAGE].double(), s["v_pool"][ids[:, 1], rows % PAGE].double()
        if new:
            key, value = torch.cat([key, s["k_new"][b, None].double()]), torch.cat([value, s["v_new"][b, None].double()])
        n = key.shape[0]
        for h in range(hkv):
            q = s["q"][b, h * group:(h + 1) * group].double()
            use = torch.arange(n, device="cuda")
            if kind == "sparse":
                pages = -(-n // PAGE)
                low, high = (s["bounds"][s["table"][b, :pages, 0].long(), h, i].double() for i in range(2))
                score = torch.stack([torch.maximum(low * x, high * x).sum(-1) for x in q]).amax(0)
                score[: case["first"]] = math.inf
                score[max(0, pages - case["last"]):] = math.inf
                pick = torch.zeros(pages, dtype=torch.bool, device="cuda")
                pick[score.argsort(descending=True, stable=True)[: case["pages"]]] = True
                use = use[pick[use // PAGE]]
            at = slice(h * group, (h + 1) * group)
            if use.numel() == 0:
                lse[b, at] = -math.inf
                continue
            z = q @ key[use, h].T / math.sqrt(dim)
            lse[b, at] = z.logsumexp(-1)
            p = z.softmax(-1)
            out[b, at] = p @ value[use, h]
            if kind == "weights":
                total[b, h, :n] = p.sum(0)
                total[b, h, :length] += case["decay"] * s["weights"][b, h, :length].double()
    if kind == "decode":
        return dict(out=out, lse=lse, k_pool=None, v_pool=None)
    if kind == "weights":
        return dict(out=out, weights=total, k_pool=None, v_pool=None)
    return dict(pages=None, out=out, bounds=None, k_pool=None, v_pool=None)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------


def work(case):
    kind, hkv, dim = case["kind"], case["kv_heads"], case["dim"]
    heads, row = case.get("heads", hkv), 2 * dim  # bytes of one head's row
    lens = _lengths(case)
    if case.get("padded"):
        # Which rows are padding goes by the seed: the mean over all of them.
        lens = [n * (1 - case["padded"] / len(lens)) for n in lens]
    batch, tokens = len(lens), sum(lens)
    pages = sum(-(-n // PAGE) for n in lens)
    step = batch * heads * row * 2 + (batch * hkv * row * 4 if case.get("append", True) else 0)  # q, out; new rows in and out
    if kind in ("decode", "weights"):
        moved = tokens * hkv * row * 2 + pages * 8 + step
        if kind == "weights":
            moved += tokens * hkv * 8
        return dict(bytes=moved, flops=4 * tokens * heads * dim)
    if kind == "bounds":
        return dict(bytes=tokens * hkv * row + pages * (hkv * row * 2 + 4), flops=2 * tokens * hkv * dim)
    if kind == "sparse":
        picked = sum(min(case["pages"], -(-(n + 1) // PAGE)) for n in lens)
        moved = pages * (hkv * row * 2 + 4) + picked * hkv * (PAGE * row * 2 + 4) + step + batch * hkv * row * (PAGE + 2)
        return dict(bytes=moved, flops=2 * pages * heads * dim + 4 * picked * PAGE * heads * dim)
    # evict: every weight and tracked position in; the kept ones out; a kept row behind the new length is read and written.
    moved = 0.0
    for n in lens:
        left = min(n, case["keep"])
        recent = min(case["recent"], left)
        chance = (left - recent) / max(1, n - recent)  # that a row which is not recent is kept
        back = recent + max(0, n - recent - left) * chance if n - recent >= left else n - left
        rows = back if n > left else 0
        moved += hkv * (4 * n + 8 * left + (4 * left if case["tracked"] else 0) + rows * row * 2 * 2)
    return dict(bytes=moved, flops=tokens * hkv)
