"""Decode over shared prefixes, attention weights of cached tokens and eviction by
them: plain forms, calls and cases.

``kind`` of a case:

``shared``  one query token a sequence against the FP8 cache, where the
            sequences of a group share their first pages: the group's prefix is
            attended once for all of its sequences
``track``   the decode step that also adds, for every cached token and kv head,
            the attention weight that the step's queries gave it
``window``  the same weights for the last queries of prompts, without an output
``evict``   the heaviest tokens of each (sequence, kv head) and its last ones
            are chosen by those weights, and their rows move together in the
            sequence's pages

The FP8 cache is ``k_cache``, ``v_cache`` e4m3 [pages, BS, H, 128] with a scale
per row, ``k_scale``, ``v_scale`` fp32 [pages, BS, H]; token t of a sequence is
row t % BS of page tables[t // BS].  Weights are fp32 [pages, H, BS]: a
token's entry is the sum, over the q heads that read its kv head and over the
queries, of softmax(q . k * k_scale * scale) at that token.
"""

import math

import torch

own = False

DEV = "cuda"
D = 128
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
HEADS = ((32, 8), (16, 8), (64, 8), (40, 8), (8, 1), (12, 4))


def listed():
    return [
        # An assistant's system prompt and tool list of 8k tokens under 64
        # conversations, at the 8B layer's heads.
        dict(name="shared_64x8k", kind="shared", batch=64, groups=1, least_prefix=8192,
             most_prefix=8192, least_tail=512, most_tail=512, hq=32, hk=8, block=256, width=0,
             dtype="bf16"),
        # Several applications' prompts in one batch, of different popularity
        # and length, conversations of any length.
        dict(name="shared_groups", kind="shared", batch=128, groups=8, least_prefix=512,
             most_prefix=6144, least_tail=16, most_tail=2048, hq=32, hk=8, block=256, width=0,
             dtype="fp16"),
        # Four samples of one prompt on a small model, under a graph's table.
        dict(name="shared_b4", kind="shared", batch=4, groups=1, least_prefix=1024,
             most_prefix=1024, least_tail=60, most_tail=60, hq=16, hk=8, block=256, width=32,
             dtype="fp16"),
        # The headline decode of the 8B layer, keeping its tokens' weights.
        dict(name="track_64x4k", kind="track", batch=64, least=4096, most=4096, hq=32, hk=8,
             block=256, width=0, dtype="bf16"),
        # Lengths spread over three orders of magnitude.
        dict(name="track_ragged", kind="track", batch=96, least=16, most=8192, hq=32, hk=8,
             block=256, width=0, dtype="fp16"),
        # One interactive user on a small model.
        dict(name="track_b1", kind="track", batch=1, least=700, most=700, hq=16, hk=8, block=256,
             width=16, dtype="fp16"),
        # One long prompt's last 32 queries.
        dict(name="window_32k", kind="window", least=32768, most=32768, seqs=1, window=32, hq=32,
             hk=8, block=256, add=False, dtype="bf16"),
        # A batch of prompts of any lengths, the shortest ones below the window.
        dict(name="window_8", kind="window", least=20, most=8192, seqs=8, window=64, hq=32, hk=8,
             block=256, add=False, dtype="fp16"),
        # A short turn of 16 tokens, added to what the cache's tokens have.
        dict(name="window_turn", kind="window", least=600, most=600, seqs=1, window=16, hq=16, hk=8,
             block=256, add=True, dtype="fp16"),
        # Long prompts cut to an eighth after their prefill.
        dict(name="evict_8x32k", kind="evict", batch=8, least=32768, most=32768, budget=4096,
             recent=32, start=0, hk=8, block=256),
        # A batch at its budget gives a page of each sequence back.
        dict(name="evict_64", kind="evict", batch=64, least=4352, most=4352, budget=4096,
             recent=1024, start=256, hk=8, block=256),
        # One short conversation, little over its budget.
        dict(name="evict_one", kind="evict", batch=1, least=300, most=300, budget=256, recent=64,
             start=4, hk=8, block=256),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("shared", "track", "window", "evict"))
    hq, hk = rng.choice(HEADS)
    case = dict(kind=kind, hk=hk, block=rng.choice((256, 256, 512)))
    block = case["block"]
    if kind != "evict":
        case.update(hq=hq, dtype=rng.choice(("fp16", "bf16")))
    if kind == "shared":
        batch = _log(rng, 1, 128)
        groups = _log(rng, 1, max(1, batch // 2))
        most = _log(rng, block, max(block, min(8192, 65536 // groups)))
        tail = _log(rng, 1, max(1, 65536 // batch // 4))
        return dict(case, batch=batch, groups=groups,
                    least_prefix=rng.choice((0, block, most)), most_prefix=most,
                    least_tail=rng.choice((1, tail)), most_tail=tail,
                    width=rng.choice((0, 0, 2 * (-(-(most + tail) // block)))))
    if kind == "track":
        batch = _log(rng, 1, 128)
        most = _log(rng, 1, min(65536, 262144 // batch))
        return dict(case, batch=batch, least=rng.choice((1, most)), most=most,
                    width=rng.choice((0, 0, 2 * (-(-most // block)))))
    if kind == "window":
        seqs = _log(rng, 1, 16)
        most = _log(rng, 1, 32768 // seqs)
        return dict(case, seqs=seqs, least=rng.choice((1, most)), most=most,
                    window=_log(rng, 1, 64), add=rng.random() < 0.5)
    batch = _log(rng, 1, 64)
    most = _log(rng, 2, min(65536, 262144 // batch))
    budget = max(1, int(most * rng.choice((0.125, 0.5, 0.95))))
    recent = int(budget * rng.choice((0.0, 0.1, 0.5)))
    return dict(case, batch=batch, least=rng.choice((1, most)), most=most, budget=budget,
                recent=recent, start=rng.choice((0, min(4, budget - recent))))


# ------------------------------------------------------------ plain forms --

def _gather(s, tables, lens):
    """Slots [rows, tokens] of the tables' tokens, and which of them exist."""
    block = s["block"]
    t = torch.arange(int(tables.shape[1]) * block, device=DEV)
    slots = tables.clamp_min(0).long()[:, t // block] * block + t % block
    return slots, t[None] < lens[:, None]


def _rows(cache, scale, slots):
    """The rows of these slots as fp32 [rows, H, tokens, 128]."""
    heads = cache.shape[2]
    x = cache.view(-1, heads, D)[slots.flatten()].float()
    x = x * scale.view(-1, heads)[slots.flatten()][..., None]
    return x.view(*slots.shape, heads, D).permute(0, 2, 1, 3)


def _weigh(q, k, seen, scale):
    """softmax over the seen keys: q [rows, H, n, 128], k [rows, H, keys, 128]."""
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(scale)
    p.masked_fill_(~seen, -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(top.masked_fill_(top == -math.inf, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    return p.div_(total.masked_fill_(total == 0, 1.0))


def _plain_decode(s, weights):
    """The decode of sequences, whether they share pages or not."""
    q, kc, vc = s["q"], s["cache"][0], s["cache"][1]
    b, hq, _ = q.shape
    hk = kc.shape[2]
    out = torch.empty_like(q)
    tables = s["tables"][:, :s["pages"]]
    step = max(1, 2 ** 19 // (s["pages"] * s["block"]))
    for i in range(0, b, step):
        part = slice(i, i + step)
        slots, live = _gather(s, tables[part], s["lens"][part])
        k, v = (_rows(s["cache"][j], s["cache"][2 + j], slots) for j in (0, 1))
        p = _weigh(q[part].float().view(-1, hk, hq // hk, D), k, live[:, None, None], s["scale"])
        out[part] = torch.matmul(p, v).view(-1, hq, D).to(q.dtype)
        if weights is not None:
            _record(s, weights, p.sum(2), slots, live, s["lens"][part] - 1)
    return out


def _record(s, weights, sums, slots, live, newest):
    """Adds sums [rows, H, tokens]; the entry of token `newest` and later is set."""
    block = s["block"]
    row, token = live.nonzero(as_tuple=True)
    slot = slots[row, token]
    at = (slot // block, slice(None), slot % block)
    old = weights[at] * (token < newest[row]).float()[:, None]
    weights[at] = old + sums.permute(0, 2, 1)[row, token]


def _plain_window(s):
    q, cu_q, cu_k = s["q"], s["cu_q"].long(), s["cu_k"].long()
    total, hq, _ = q.shape
    hk = s["cache"][0].shape[2]
    seqs, most = len(cu_q) - 1, s["max_q"]
    lq, lk = cu_q.diff(), cu_k.diff()
    i = torch.arange(most, device=DEV)
    for n in range(seqs):
        one = slice(n, n + 1)
        slots, live = _gather(s, s["tables"][one], lk[one])
        k = _rows(s["cache"][0], s["cache"][2], slots)
        rows = q[(cu_q[n] + i).clamp_max(total - 1)].float().view(most, hk, hq // hk, D)
        rows = rows.permute(1, 2, 0, 3)[None]
        sees = torch.where(i < lq[n], lk[n] - lq[n] + i + 1, 0)
        seen = torch.arange(k.shape[2], device=DEV) < sees[:, None]
        seen = seen.repeat(hq // hk, 1)
        p = _weigh(rows.flatten(2, 3), k, seen[None, None], s["scale"])
        newest = lk[one] if s["add"] else torch.zeros_like(lk[one])
        _record(s, s["weights"], p.sum(2), slots, live, newest)
    return s["weights"]


def _plain_evict(s):
    lens, budget, start = s["lens"].long(), s["budget"], s["start"]
    slots, live = _gather(s, s["tables"], lens)
    block, (b, tokens) = s["block"], slots.shape
    w = s["weights"][slots // block, :, slots % block].permute(0, 2, 1)
    heads = w.shape[1]
    t = torch.arange(tokens, device=DEV)
    # kept whatever their weight: the first ones, and the last ones in the
    # places that remain
    last = min(s["recent"], max(0, budget - start))
    fixed = (t < start) | (t >= lens[:, None] - last)
    order = torch.where(torch.isnan(w), -math.inf, w).sort(dim=-1, descending=True, stable=True)[1]
    rank = (live.long() * (1 + fixed.long()))[:, None].expand(b, heads, tokens).gather(-1, order)
    order = order.gather(-1, rank.sort(dim=-1, descending=True, stable=True)[1])
    n = lens.clamp_max(budget)
    most = min(budget, tokens)
    place = torch.arange(most, device=DEV)
    chosen = torch.where(place < n[:, None, None], order[..., :most], tokens).sort(-1)[0]
    kept = torch.full((b, heads, budget), -1, dtype=torch.int32, device=DEV)
    kept[..., :most] = torch.where(chosen < tokens, chosen, -1).to(torch.int32)
    row, head, i = (kept >= 0).nonzero(as_tuple=True)
    src = slots[row, kept[row, head, i].long()]
    dst = slots[row, i]
    for x in s["cache"]:
        x = (x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x).flatten(0, 1)
        x[dst, head] = x[src, head]
    return {"kept": kept, "lens": n.to(torch.int32), **dict(zip("kvab", s["cache"]))}


# ------------------------------------------------------------------ calls --

def run(s):
    kind = s["kind"]
    if not own:
        if kind == "shared":
            return _plain_decode(s, None)
        if kind == "track":
            return {"out": _plain_decode(s, s["weights"]), "weights": s["weights"]}
        return _plain_window(s) if kind == "window" else _plain_evict(s)
    import microserve_amd as M
    if kind == "shared":
        return M.fp8_shared_prefix_decode_attention(
            s["q"], *s["cache"], s["lens"], s["tables"], s["scale"], s["cu_groups"],
            s["prefix_lens"], max_prefix_len=s["max_prefix"])
    if kind == "track":
        out = M.fp8_decode_attention_weights(s["q"], *s["cache"], s["lens"], s["tables"],
                                             s["scale"], s["weights"])
        return {"out": out, "weights": s["weights"]}
    if kind == "window":
        return M.fp8_window_attention_weights(
            s["q"], s["cache"][0], s["cache"][2], s["tables"], s["cu_q"], s["cu_k"], s["max_q"],
            s["scale"], s["weights"], accumulate=s["add"], max_seqlen_k=s["max_k"])
    kept, lens = M.select_kv_tokens(s["weights"], s["lens"], s["tables"], s["budget"],
                                    recent=s["recent"], start=s["start"])
    M.evict_kv_tokens(*s["cache"], kept, lens, s["tables"])
    return {"kept": kept, "lens": lens, **dict(zip("kvab", s["cache"]))}


# ----------------------------------------------------------------- inputs --

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _spread(n, least, most):
    """n whole numbers from least to most, even over the logarithm, the largest
    last."""
    if n == 1 or least == most:
        return [most] * n
    lo, hi = math.log(least + 1), math.log(most + 1)
    return [int(round(math.exp(lo + (hi - lo) * i / (n - 1)))) - 1 for i in range(n)]


def _deal(g, values):
    order = torch.randperm(len(values), generator=g, device=DEV).tolist()
    return [values[i] for i in order]


def _cache(g, pages, heads, block):
    """A filled pool: K rows with a few channels several times the others, as
    the rotary embedding's low frequencies leave them."""
    gain = 1.0 + 7.0 * (torch.rand(heads, D, generator=g, device=DEV) < 0.04)
    values, scales = [], []
    for x in (gain, torch.ones_like(gain)):
        x = _normal(g, pages, block, heads, D).mul_(x)
        scale = x.abs().amax(-1).clamp_min(1e-8) / 448.0
        values.append(x.div_(scale[..., None]).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn))
        scales.append(scale)
    return (*values, *scales)


def _weights(g, pages, heads, block):
    """Accumulated weights as a few steps leave them: most small, a few large,
    some that no query has looked at."""
    w = 1e-3 * torch.exp(2.0 * _normal(g, pages, heads, block))
    return w * (torch.rand(w.shape, generator=g, device=DEV) < 0.9)


def _tables(g, own_pages, shared, block, width):
    """Rows of permuted pages: sequence i has the pages of its list in `shared`
    (numbers below `count`), then own_pages[i] of its own."""
    rows, lists = len(own_pages), [x for x in shared]
    count = 1 + max((p for x in lists for p in x), default=-1)
    pool = max(1, count + sum(own_pages))
    order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
    most = max(1, max(len(x) + n for x, n in zip(lists, own_pages)))
    at = torch.full((rows, max(width, most)), -1, dtype=torch.int64)
    for i, (x, n) in enumerate(zip(lists, own_pages)):
        at[i, :len(x) + n] = torch.tensor([*x, *range(count, count + n)], dtype=torch.int64)
        count += n
    at = at.to(DEV)
    return torch.where(at >= 0, order[at.clamp_min(0)], -1), pool, most


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _sizes(batch, groups):
    """Sequences of each group: the g-th is g + 1 times as popular as the first."""
    left = batch - groups
    sizes = [1 + left * 2 * (g + 1) // (groups * (groups + 1)) for g in range(groups)]
    sizes[-1] += batch - sum(sizes)
    return sizes


def _prefixes(case):
    block = case["block"]
    lens = _spread(case["groups"], case["least_prefix"], case["most_prefix"])
    return [n // block * block for n in lens]


def prepare(case, seed):
    g, kind, block, hk = _gen(seed), case["kind"], case["block"], case["hk"]
    s = dict(kind=kind, block=block, scale=D ** -0.5)
    if kind == "shared":
        sizes, prefixes = _sizes(case["batch"], case["groups"]), _deal(g, _prefixes(case))
        tails = _deal(g, _spread(case["batch"], case["least_tail"], case["most_tail"]))
        shared, lens, first, at = [], [], 0, 0
        for n, p in zip(sizes, prefixes):
            shared += [list(range(first, first + p // block))] * n
            lens += [p + x for x in tails[at:at + n]]
            first, at = first + p // block, at + n
        own_pages = [-(-n // block) - len(x) for n, x in zip(lens, shared)]
        tables, pool, pages = _tables(g, own_pages, shared, block, case["width"])
        cu = [0]
        for n in sizes:
            cu.append(cu[-1] + n)
        s.update(cu_groups=_ints(cu), prefix_lens=_ints(prefixes), max_prefix=max(prefixes))
    elif kind == "window":
        lens = _deal(g, _spread(case["seqs"], case["least"], case["most"]))
        tables, pool, pages = _tables(g, [-(-n // block) for n in lens], [[]] * len(lens), block, 0)
        cu_q, cu_k = [0], [0]
        for n in lens:
            cu_q.append(cu_q[-1] + min(n, case["window"]))
            cu_k.append(cu_k[-1] + n)
        s.update(cu_q=_ints(cu_q), cu_k=_ints(cu_k), add=case["add"], max_k=max(lens),
                 max_q=min(max(lens), case["window"]),
                 q=_normal(g, cu_q[-1], case["hq"], D).to(TYPES[case["dtype"]]))
    else:
        lens = _deal(g, _spread(case["batch"], case["least"], case["most"]))
        tables, pool, pages = _tables(g, [-(-n // block) for n in lens], [[]] * len(lens), block,
                                      case.get("width", 0))
    if kind in ("shared", "track"):
        s["q"] = _normal(g, case["batch"], case["hq"], D).to(TYPES[case["dtype"]])
    if kind == "evict":
        s.update({x: case[x] for x in ("budget", "recent", "start")})
    if kind != "shared":
        s["weights"] = _weights(g, pool, hk, block)
    s.update(tables=tables, pages=pages, lens=_ints(lens), cache=_cache(g, pool, hk, block))
    return s


# ---------------------------------------------------------------- amounts --

def work(case):
    kind, hk = case["kind"], case["hk"]
    row = 2 * (D + 4)  # a token's K and V of one kv head, with their scales
    if kind == "shared":
        prefixes = _prefixes(case)
        sizes = _sizes(case["batch"], case["groups"])
        tails = sum(_spread(case["batch"], case["least_tail"], case["most_tail"]))
        # (prefixes are dealt to the groups: their mean size)
        seen = tails + sum(prefixes) * sum(sizes) / len(sizes)
        return {"bytes": (tails + sum(prefixes)) * hk * row + case["batch"] * case["hq"] * 4 * D,
                "flops": 4 * seen * case["hq"] * D}
    if kind == "track":
        tokens = sum(_spread(case["batch"], case["least"], case["most"]))
        return {"bytes": tokens * hk * (row + 8) + case["batch"] * case["hq"] * 4 * D,
                "flops": 4 * tokens * case["hq"] * D}
    if kind == "window":
        lens = _spread(case["seqs"], case["least"], case["most"])
        new = [min(n, case["window"]) for n in lens]
        pairs = sum(w * (n - (w - 1) / 2) for n, w in zip(lens, new))
        return {"bytes": sum(lens) * hk * (row / 2 + (8 if case["add"] else 4))
                + sum(new) * case["hq"] * 2 * D, "flops": 2 * pairs * case["hq"] * D}
    # every weight that competes is read, and each kept row behind the first
    # one that goes is read and written
    lens = _spread(case["batch"], case["least"], case["most"])
    moved = sum(max(0, case["budget"] - case["start"]) for n in lens if n > case["budget"])
    kept = len(lens) * case["budget"]
    return {"bytes": hk * (4 * sum(lens) + 2 * row * moved + 4 * kept), "flops": 0}


# ---------------------------------------------------- the definition, in 64 --

def _sequence(s, i, n):
    """K and V [H, n, 128] of sequence i in 64 bits."""
    pages = s["tables"][i, :-(-n // s["block"])].long()
    k, v = (s["cache"][j][pages].double() * s["cache"][2 + j][pages].double()[..., None]
            for j in (0, 1))
    return tuple(x.flatten(0, 1)[:n].transpose(0, 1).contiguous() for x in (k, v))


def _attention(q, k, scale, sees):
    """Weights [H, n * group, keys] of rows q [n, Hq, 128], query i seeing the
    first sees[i] keys."""
    n, hq, _ = q.shape
    hk, lk, _ = k.shape
    x = q.double().view(n, hk, hq // hk, D).transpose(0, 1).reshape(hk, -1, D)
    score = torch.bmm(x, k.transpose(1, 2).contiguous()) * scale
    dark = torch.arange(lk, device=DEV)[None] >= sees[:, None]
    score.masked_fill_(dark.repeat_interleave(hq // hk, 0)[None], -math.inf)
    return torch.softmax(score, -1)


def exact(case, seed):
    kind = case["kind"]
    if kind == "evict":
        return None  # rows are chosen and moved: nothing is computed
    s = prepare(case, seed)
    block = s["block"]
    weights = s["weights"].double() if kind != "shared" else None

    def put(i, sums, add):
        for p in range(-(-sums.shape[1] // block)):
            part = sums[:, p * block:(p + 1) * block]
            place = weights[int(s["tables"][i, p]), :, :part.shape[1]]
            place.copy_(part + add(p * block, place))

    if kind == "window":
        cu_q, cu_k = s["cu_q"].tolist(), s["cu_k"].tolist()
        for i in range(len(cu_q) - 1):
            lk, q = cu_k[i + 1] - cu_k[i], s["q"][cu_q[i]:cu_q[i + 1]]
            k, _ = _sequence(s, i, lk)
            sees = lk - len(q) + 1 + torch.arange(len(q), device=DEV)
            sums = _attention(q, k, s["scale"], sees).sum(1)
            put(i, sums, lambda _, old: old if s["add"] else 0.0)
        return weights
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for i, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        k, v = _sequence(s, i, n)
        p = _attention(s["q"][i:i + 1], k, s["scale"], torch.tensor([n], device=DEV))
        out[i] = torch.bmm(p, v).reshape(-1, D)
        if weights is not None:
            def add(first, old, n=n):  # the newest token's entry is set
                return old * (first + torch.arange(old.shape[1], device=DEV) < n - 1)
            put(i, p.sum(1), add)
    return out if kind == "shared" else {"out": out, "weights": weights}
