"""Long contexts over a paged key/value cache, as cases that can be timed: attention that adds up how much every position was looked at,
evicting the positions that were looked at least, rotary positions in other layouts, on part of a head and scaled; and what a
program reads off the logits at the end: log probabilities of given tokens.

``listed()`` are fixed cases, ``draw(rng)`` gives others of the same ranges.  ``prepare`` builds what a program holds before
the call, ``run`` is one pass through an operator: elementary torch operations where ``own`` is false, the package's entry
points where it is true.  ``exact`` computes the same from the definitions in 64 bits."""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda:0"
DIM = 128   # width of a head
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def _weigh(name, batch, nodes, context, ragged, q_heads, kv_heads, page):
    return {"name": name, "kind": "weigh", "batch": batch, "nodes": nodes, "context": context, "ragged": ragged, "q_heads": q_heads,
            "kv_heads": kv_heads, "page": page}


def _evict(name, batch, layers, context, ragged, keep, recent, shared, kv_heads, page):
    return {"name": name, "kind": "evict", "batch": batch, "layers": layers, "context": context, "ragged": ragged, "keep": keep, "recent": recent,
            "shared": shared, "kv_heads": kv_heads, "page": page}


def _rope(name, batch, nodes, context, pairs, layout, scaled, dtype, q_heads, kv_heads, page):
    return {"name": name, "kind": "rope", "batch": batch, "nodes": nodes, "context": context, "pairs": pairs, "layout": layout, "scaled": scaled,
            "dtype": dtype, "q_heads": q_heads, "kv_heads": kv_heads, "page": page}


def _logprobs(name, rows, vocab, dtype, top, masked, pad):
    return {"name": name, "kind": "logprobs", "rows": rows, "vocab": vocab, "dtype": dtype, "top": top, "masked": masked, "pad": pad}


def listed():
    return [
        # one sequence, one token, a short context: what the attention of a single decoding step costs
        _weigh("weigh_b1_n1_ctx100", 1, 1, 100, False, 32, 8, 16),
        # sixteen sequences decoding together at a 4096-token context, every step counted
        _weigh("weigh_b16_n1_ctx4096", 16, 1, 4096, False, 32, 8, 64),
        # the last chunks of prompts of very different lengths vote on what stays, the narrower model
        _weigh("weigh_b13_n27_ragged7000", 13, 27, 7000, True, 16, 4, 64),
        # large chunks of long prompts
        _weigh("weigh_b4_n64_ctx32768", 4, 64, 32768, False, 32, 8, 128),
        # a prompt is cut to half its length after it has been read, in all layers of the decoder
        _evict("evict_b1_ctx4096_keep2048", 1, 32, 4096, False, 2048, 128, False, 8, 64),
        # sixteen sequences that keep to a budget: each time a page's worth of new tokens has come, as many positions go
        _evict("evict_b16_ctx2112_keep2048", 16, 6, 2112, False, 2048, 64, False, 8, 64),
        # sequences in pairs that share the pages of a prompt are cut apart, to odd lengths
        _evict("evict_b4_shared_ragged", 4, 16, 1500, True, 701, 33, True, 4, 32),
        # one token of one sequence, neighbouring dims as pairs; chunks of a batch, half of every head rotated, frequencies scaled for a longer context
        _rope("rope_b1_n1_interleaved", 1, 1, 4000, 64, "interleaved", False, "float32", 32, 8, 64),
        _rope("rope_b16_n64_part_scaled", 16, 64, 500, 32, "halves", True, "bfloat16", 32, 8, 64),
        # the chosen token of one sequence with its alternatives; a short batch under a grammar that masks most of the vocabulary, in a padded
        # buffer; a chunk of a prompt that is scored
        _logprobs("logprobs_r1_v128256_top20", 1, 128256, "float32", 20, 0.0, 0),
        _logprobs("logprobs_r77_v32001_masked", 77, 32001, "bfloat16", 5, 0.7, 63),
        _logprobs("logprobs_r1024_v128256_top5", 1024, 128256, "float32", 5, 0.0, 0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges above."""
    case = _drawn(rng)
    del case["name"]
    return case


def _drawn(rng):
    kind = rng.choice(["weigh"] * 3 + ["evict"] * 3 + ["rope"] + ["logprobs"] * 3)
    kv_heads = rng.choice([4, 8])
    page = rng.choice([16, 32, 64, 128])
    if kind == "weigh":
        batch, nodes, group = _log_int(rng, 1, 32), _log_int(rng, 1, 64), rng.choice([1, 2, 4, 4, 8])
        room = 4 * 64 * 32 * 32768 // (batch * nodes * kv_heads * group)
        return _weigh("", batch, nodes, _log_int(rng, 16, max(16, min(32768, 40 * 8 * 4096 // (batch * kv_heads), room))), rng.random() < 0.5,
                      kv_heads * group, kv_heads, page)
    if kind == "evict":
        batch, layers = _log_int(rng, 1, 16), _log_int(rng, 1, 32)
        context = _log_int(rng, 64, max(64, min(20000, 32 * 8 * 4096 // (batch * layers * kv_heads))))
        keep = rng.randint(1, context)
        return _evict("", batch, layers, context, rng.random() < 0.5, keep, rng.choice([0, rng.randint(0, keep), rng.randint(0, min(keep, 128))]),
                      rng.random() < 0.3, kv_heads, page)
    if kind == "rope":
        return _rope("", _log_int(rng, 1, 16), _log_int(rng, 1, 64), _log_int(rng, 16, 1000), rng.choice([64, 64, 32, 16, rng.randint(1, 64)]),
                     rng.choice(["halves", "interleaved"]), rng.random() < 0.5, rng.choice(["float32", "bfloat16"]),
                     kv_heads * rng.choice([1, 2, 4, 8]), kv_heads, page)
    vocab = _log_int(rng, 500, 128256)
    return _logprobs("", _log_int(rng, 1, max(1, min(8192, 1024 * 128256 // vocab))), vocab, rng.choice(sorted(DTYPES)), rng.choice([0, 1, 5, 20, 32]),
                     rng.choice([0.0, 0.0, 0.7]), rng.choice([0, 0, 1, 64]))


# ---- inputs ------------------------------------------------------------------------------------------------------------------


def _lengths(case):
    """Context length of every sequence; does not depend on the seed, so that the work of a case does not."""
    n = case["batch"]
    if not case.get("ragged"):
        return [case["context"]] * n
    r = random.Random(7 * n + case["context"])
    return [case["context"]] + [_log_int(r, 1, case["context"]) for _ in range(n - 1)]


def _shared(case):
    """How many pages of every sequence are those of the one before it."""
    lens = _lengths(case)
    return [min(lens[r - 1], lens[r]) // case["page"] if case.get("shared") and r % 2 else 0 for r in range(len(lens))]


def _generator(seed):
    return torch.Generator(DEV).manual_seed(seed)


def _pool(case, layers, pages, gen):
    """Keys and values [layers, pages, heads, page, 128] in bf16; keys of a few channels are larger, as in trained models."""
    shape = (layers, pages, case["kv_heads"], case["page"], DIM)
    k, v = torch.empty(shape, dtype=torch.bfloat16, device=DEV), torch.empty(shape, dtype=torch.bfloat16, device=DEV)
    gain = torch.ones(DIM, device=DEV)
    gain[::17] = 3.0
    for i in range(layers):
        k[i] = torch.randn(shape[1:], generator=gen, device=DEV) * gain
        v[i] = torch.randn(shape[1:], generator=gen, device=DEV)
    return k, v


def _cache(case, layers, extra, spare, seed, gen):
    """Sequences on pages scattered over the pool, with room for `extra` tokens behind the context; `spare` free pages.  Table, counts and lengths
    are parts of one tensor, so that a pass that changes them can put them back at once."""
    page, lens = case["page"], _lengths(case)
    rows = len(lens)
    held = [-(-(n + extra) // page) for n in lens]
    shared = _shared(case)
    pages = sum(held) - sum(shared) + spare + 3
    width = max(held) + 1
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    ints = torch.zeros(rows * width + pages + rows, dtype=torch.int32)
    table, refs = ints[:rows * width].view(rows, width), ints[rows * width:rows * width + pages]
    table.fill_(-1)
    ints[rows * width + pages:] = torch.tensor(lens, dtype=torch.int32)
    at = 0
    for r, h in enumerate(held):
        table[r, :shared[r]] = table[r - 1, :shared[r]]
        table[r, shared[r]:h] = order[at:at + h - shared[r]]
        at += h - shared[r]
        refs[table[r, :h].long()] += 1
    ints = ints.to(DEV)
    k, v = _pool(case, layers, pages, gen)
    st = {"case": case, "k": k, "v": v, "ints": ints, "table": ints[:rows * width].view(rows, width), "refs": ints[rows * width:rows * width + pages],
          "lens": ints[rows * width + pages:]}
    if own:
        from tyloquant_b200 import PagedCache
        st["cache"] = PagedCache(k, v, st["table"], st["lens"], st["refs"])
    return st


def _masks(rng, batch, nodes):
    """Chains (chunks of a prompt) and random trees, whose nodes see themselves and what is above them."""
    masks = []
    for b in range(batch):
        m = []
        for i in range(nodes):
            up = i - 1 if b % 2 == 0 else rng.randrange(max(0, i - 8), i) if i else -1
            m.append((m[up] if i else 0) | 1 << i)
        masks.append([x - (1 << 64) if x >> 63 else x for x in m])
    return torch.tensor(masks, dtype=torch.int64, device=DEV)


def _frequencies(case):
    """theta^(-j/P); scaled: low frequencies divided by four, high ones kept, a ramp between them; and the factor on the rotated values."""
    p = case["pairs"]
    f = 500000.0 ** (-torch.arange(p, dtype=torch.float64, device=DEV) / p)
    if not case["scaled"]:
        return f, 1.0
    ramp = torch.clamp(torch.arange(p, dtype=torch.float64, device=DEV) / p * 2 - 0.5, 0, 1)
    return f * (1 - ramp + ramp / 4), 0.1 * math.log(4.0) + 1


def prepare(case, seed):
    rng, gen = random.Random(seed), _generator(seed)
    kind = case["kind"]
    if kind == "weigh":
        st = _cache(case, 1, case["nodes"], 0, seed, gen)
        st["masks"] = _masks(rng, case["batch"], case["nodes"])
        st["q"] = torch.randn((case["batch"], case["nodes"], case["q_heads"], DIM), generator=gen, device=DEV).to(torch.bfloat16)
        st["weights"] = torch.rand((1, case["batch"], case["kv_heads"], st["table"].shape[1] * case["page"]), generator=gen, device=DEV) * 1e-3
        return st
    if kind == "evict":
        st = _cache(case, case["layers"], 0, case["batch"] * -(-case["keep"] // case["page"]) if case["shared"] else 0, seed, gen)
        shape = (case["layers"], case["batch"], case["kv_heads"], st["table"].shape[1] * case["page"])
        # accumulated weights span orders of magnitude; a few positions were never looked at
        st["fresh"] = torch.exp(2 * torch.randn(shape, generator=gen, device=DEV)) * (torch.rand(shape, generator=gen, device=DEV) > 0.05)
        st["weights"] = st["fresh"].clone()
        st["before"] = st["ints"].clone()
        st["keep"] = torch.tensor([max(1, case["keep"] - 3 * r) for r in range(case["batch"])] if case["ragged"] else [case["keep"]] * case["batch"],
                                  dtype=torch.int32, device=DEV)
        return st
    if kind == "rope":
        st = _cache(case, 1, case["nodes"], 0, seed, gen)
        # positions run on from what the sequence had before some of it was evicted
        st["depths"] = (torch.arange(case["nodes"])[None] + torch.tensor([[rng.randrange(20000)] for _ in range(case["batch"])])).to(DEV, torch.int32)
        heads = case["q_heads"] + 2 * case["kv_heads"]
        st["qkv"] = torch.randn((case["batch"], case["nodes"], heads * DIM), generator=gen, device=DEV).to(DTYPES[case["dtype"]])
        st["freqs"], st["factor"] = _frequencies(case)
        return st
    rows, vocab = case["rows"], case["vocab"]
    logits = (torch.randn((rows, vocab + case["pad"]), generator=gen, device=DEV) * 2.5).to(DTYPES[case["dtype"]])[:, :vocab]
    tokens = torch.randint(vocab, (rows,), generator=gen, device=DEV)
    if case["masked"]:
        for r in range(rows):   # row by row: the mask of a whole chunk would be as large as the logits
            logits[r].masked_fill_(torch.rand(vocab, generator=gen, device=DEV) < case["masked"], -math.inf)
    guess = logits.argmax(1)
    likely = torch.rand(rows, generator=gen, device=DEV) < 0.5   # half of the tokens are the model's own
    tokens = torch.where(likely, guess, tokens)
    tokens[torch.rand(rows, generator=gen, device=DEV) < 1 / 16] = -1   # padding
    return {"case": case, "logits": logits, "tokens": tokens.int()}


# ---- one pass ----------------------------------------------------------------------------------------------------------------


def _gather(pool, table):
    """Pages of one layer in the order of the table: [batch, heads, tokens, 128]."""
    x = pool[table.clamp(min=0).long()]
    b, p, h, t, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(b, h, p * t, d)


def _weigh_plain(st):
    case, lens, masks, q = st["case"], st["lens"].long(), st["masks"], st["q"].float()
    b, n, hq, _ = q.shape
    hk = case["kv_heads"]
    k, v = _gather(st["k"][0], st["table"]).float(), _gather(st["v"][0], st["table"]).float()
    pos = torch.arange(k.shape[2], device=DEV)
    node = pos[None, None, :] - lens[:, None, None]   # [batch, 1, tokens]
    bit = (masks[:, :, None] >> node.clamp(0, 63)) & 1
    see = (node < 0) | ((node < n) & (bit == 1))      # [batch, nodes, tokens]
    see &= st["table"].repeat_interleave(case["page"], 1)[:, None, :] >= 0
    v = torch.where(see.any(1)[:, None, :, None], v, 0.0)
    g = hq // hk
    q = q.reshape(b, n, hk, g, DIM).permute(0, 2, 1, 3, 4).reshape(b, hk, n * g, DIM)
    s = (q @ k.transpose(2, 3)) * (1.0 / math.sqrt(DIM))
    s = s.reshape(b, hk, n, g, -1).masked_fill(~see[:, None, :, None, :], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = (p.reshape(b, hk, n * g, -1) @ v).reshape(b, hk, n, g, DIM)
    mass = p.sum((2, 3))
    old = st["weights"][0]
    st["weights"][0] = torch.where((node < 0), old + mass, torch.where(node < n, mass, old))
    return out.permute(0, 2, 1, 3, 4).reshape(b, n, hq, DIM).to(torch.bfloat16), st["weights"]


def _evict_plain(st):
    case, table, refs, lens, weights = st["case"], st["table"], st["refs"], st["lens"], st["weights"]
    page, keep = case["page"], st["keep"].long()
    layers, rows, heads, cap = weights.shape
    width = table.shape[1]
    n = lens.long()
    go = n > keep
    k = torch.where(go, keep, n)
    recent = k.clamp(max=case["recent"])
    b = k - recent
    # pages: what is shared below the new length is exchanged for the lowest free pages, what lies behind it goes back
    entry = torch.arange(width, device=DEV)[None]
    inside = entry < (-(-k // page))[:, None]
    have = table >= 0
    swap = go[:, None] & inside & have & (refs[table.clamp(min=0).long()] > 1)
    free = torch.argsort((refs > 0).to(torch.int8), stable=True)
    lack = (swap.sum() - (refs <= 0).sum()).clamp(min=0)
    act = go & (lack == 0)
    rank = (torch.cumsum(swap.reshape(-1), 0) - 1).clamp(min=0).reshape(rows, width)
    old = table.clone()
    new = torch.where(swap, free[rank].int(), table)
    new = torch.where(go[:, None] & ~inside, -1, new)
    new = torch.where(act[:, None], new, table)
    count = torch.zeros(refs.numel() + 1, dtype=torch.int32, device=DEV)
    one = torch.ones(rows * width, dtype=torch.int32, device=DEV)
    left = torch.where(act[:, None] & have & (new != old), old, refs.numel()).reshape(-1).long()
    came = torch.where(act[:, None] & swap, new, refs.numel()).reshape(-1).long()
    refs += (count.index_add(0, came, one) - count.index_add(0, left, one))[:-1]
    table.copy_(new)
    # which of the older slots stay
    slot = torch.arange(cap, device=DEV)
    older = slot < (n - recent)[:, None]                                          # [rows, cap]
    key = torch.where(older[None, :, None] & ~weights.isnan(), weights, -math.inf)
    place = torch.argsort(torch.argsort(key, dim=-1, descending=True, stable=True), dim=-1)   # of each slot among them
    kept = (place < b[None, :, None, None]) & older[None, :, None]
    below = slot < b[:, None]
    hole = below[None, :, None] & ~kept
    move = kept & ~below[None, :, None]
    holes, moves = torch.argsort((~hole).to(torch.int8), dim=-1, stable=True), torch.argsort((~move).to(torch.int8), dim=-1, stable=True)
    some = torch.arange(cap, device=DEV) < hole.sum(-1, keepdim=True)
    source = torch.where((slot >= b[:, None]) & (slot < k[:, None]), slot + (n - k)[:, None], slot)[None, :, None].expand(layers, rows, heads, cap).clone()
    source.scatter_(-1, torch.where(some, holes, cap - 1), torch.where(some, moves, source.gather(-1, torch.full_like(holes, cap - 1))))
    most = int(case["keep"])
    at = torch.arange(most, device=DEV)
    source = source[..., :most]
    todo = act[:, None] & (at < k[:, None])                                       # [rows, most]
    weights[..., :most] = torch.where(todo[None, :, None], weights.gather(-1, source), weights[..., :most])
    from_page = old.long()[torch.arange(rows, device=DEV)[None, :, None, None], source // page]
    to_page = new.long().gather(1, (at // page)[None].expand(rows, most))
    layer = torch.arange(layers, device=DEV)[:, None, None, None]
    head = torch.arange(heads, device=DEV)[None, None, :, None]
    todo = todo[None, :, None].expand(layers, rows, heads, most)
    to = (layer.expand_as(source)[todo], to_page[None, :, None].expand_as(source)[todo], head.expand_as(source)[todo], (at % page).expand_as(source)[todo])
    come = (to[0], from_page[todo], to[2], (source % page)[todo])
    for pool in (st["k"], st["v"]):
        pool[to] = pool[come]
    lens.copy_(torch.where(act, k, n))
    return torch.where(act, n - k, 0).int(), lack.int().reshape(1)


def _rope_plain(st):
    case, lens, depths, qkv = st["case"], st["lens"].long(), st["depths"], st["qkv"].float()
    b, n, _ = qkv.shape
    hq, hk, page, p = case["q_heads"], case["kv_heads"], case["page"], case["pairs"]
    x = qkv.reshape(b, n, hq + 2 * hk, DIM)
    angle = (lens[:, None] + depths).double()[:, :, None] * st["freqs"]
    cos, sin = (torch.cos(angle) * st["factor"]).float()[:, :, None], (torch.sin(angle) * st["factor"]).float()[:, :, None]
    part = x[:, :, :hq + hk, :2 * p]
    lo, hi = (part[..., :p], part[..., p:]) if case["layout"] == "halves" else (part[..., 0::2], part[..., 1::2])
    lo, hi = lo * cos - hi * sin, hi * cos + lo * sin
    part = torch.cat([lo, hi], -1) if case["layout"] == "halves" else torch.stack([lo, hi], -1).reshape(b, n, hq + hk, 2 * p)
    turned = torch.cat([part, x[:, :, :hq + hk, 2 * p:]], -1).to(torch.bfloat16)
    slot = lens[:, None] + torch.arange(n, device=DEV)
    pages, at = st["table"].gather(1, slot // page).long(), slot % page
    st["k"][0][pages, :, at] = turned[:, :, hq:]
    st["v"][0][pages, :, at] = x[:, :, hq + hk:].to(torch.bfloat16)
    return turned[:, :, :hq].contiguous(), st["k"], st["v"]


def _logprobs_plain(st):
    z, tokens, k = st["logits"].float(), st["tokens"].long(), st["case"]["top"]
    top = z.amax(-1, keepdim=True)
    d = z - top
    e = torch.exp(d)
    total = e.sum(-1)
    lse = top[:, 0] + torch.log(total)
    entropy = torch.log(total) - torch.where(e > 0, e * d, 0.0).sum(-1) / total
    there = tokens >= 0
    zt = z.gather(1, tokens.clamp(min=0)[:, None])
    before = torch.arange(z.shape[1], device=DEV)[None] < tokens[:, None]
    rank = ((z > zt) | ((z == zt) & before)).sum(-1) + 1
    best, token = torch.sort(z, dim=-1, descending=True, stable=True)
    return (torch.where(there, zt[:, 0] - lse, 0.0), entropy, torch.where(there, rank, 0).int(), best[:, :k] - lse[:, None], token[:, :k].int())


def run(state):
    kind, case = state["case"]["kind"], state["case"]
    if kind == "evict":   # the sequences as they are before each eviction
        state["ints"].copy_(state["before"])
        state["weights"].copy_(state["fresh"])
        if own:
            dropped, lack = state["cache"].evict(state["weights"], state["keep"], recent=case["recent"])
        else:
            dropped, lack = _evict_plain(state)
        return dropped, lack, state["table"], state["lens"], state["refs"], state["weights"], state["k"], state["v"]
    if not own:
        return {"weigh": _weigh_plain, "rope": _rope_plain, "logprobs": _logprobs_plain}[kind](state)
    if kind == "weigh":
        return state["cache"].attend(0, state["q"], state["masks"], weights=state["weights"]), state["weights"]
    if kind == "rope":
        q = state["cache"].write(0, state["qkv"], state["depths"], state["freqs"], layout=case["layout"], factor=state["factor"])
        return q, state["k"], state["v"]
    from tyloquant_b200 import token_logprobs
    return tuple(token_logprobs(state["logits"], state["tokens"], top=case["top"]))


def work(case):
    kind = case["kind"]
    if kind == "weigh":
        tokens = sum(n + case["nodes"] for n in _lengths(case))
        rows = case["batch"] * case["nodes"] * case["q_heads"]
        seen = sum(n * case["nodes"] for n in _lengths(case)) * case["q_heads"]
        return {"bytes": tokens * case["kv_heads"] * (DIM * 4 + 8) + rows * DIM * 4 + case["batch"] * case["nodes"] * 8, "flops": 4 * seen * DIM}
    if kind == "evict":   # weights are read; what has to move is as many as an even spread of the heaviest positions makes
        moved = read = 0.0
        lens, shared = _lengths(case), _shared(case)
        for r, n in enumerate(lens):
            k = max(1, case["keep"] - 3 * r) if case["ragged"] else case["keep"]
            if n <= k:
                continue
            recent = min(case["recent"], k)
            stay = (k - recent) / (n - recent) if n > recent else 0
            both = max(shared[r:r + 2]) if r % 2 == 0 else shared[r]   # what stays on pages that another sequence has too is copied
            read += n
            moved += recent + (k - recent) * (1 - stay) + min(both * case["page"], k - recent) * stay
        return {"bytes": int(case["layers"] * case["kv_heads"] * (read * 4 + moved * (DIM * 8 + 8))), "flops": 0}
    if kind == "rope":
        n = case["batch"] * case["nodes"]
        heads = case["q_heads"] + 2 * case["kv_heads"]
        return {"bytes": n * (heads * DIM * (2 + DTYPES[case["dtype"]].itemsize) + 4), "flops": 6 * n * (heads - case["kv_heads"]) * case["pairs"]}
    return {"bytes": case["rows"] * (case["vocab"] * DTYPES[case["dtype"]].itemsize + 16 + 8 * case["top"]), "flops": 5 * case["rows"] * case["vocab"]}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------------


def _exact_weigh(st):
    case, page, n = st["case"], st["case"]["page"], st["case"]["nodes"]
    group = case["q_heads"] // case["kv_heads"]
    table, masks = st["table"].cpu().tolist(), st["masks"].cpu().tolist()
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    weights = st["weights"].double()
    for b, length in enumerate(st["lens"].cpu().tolist()):
        total = length + n
        ids = torch.tensor(table[b][:-(-total // page)], device=DEV)
        bits = torch.tensor([[(m >> j) & 1 for j in range(n)] for m in masks[b]], device=DEV).bool()
        weights[0, b, :, length:total] = 0
        for h in range(case["kv_heads"]):
            k = st["k"][0, ids, h].reshape(-1, DIM)[:total].double()
            v = st["v"][0, ids, h].reshape(-1, DIM)[:total].double()
            for j in range(group):
                s = st["q"][b, :, h * group + j].double() @ k.T / math.sqrt(DIM)
                s[:, length:].masked_fill_(~bits, -math.inf)
                p = torch.softmax(s, -1)
                out[b, :, h * group + j] = p @ v
                weights[0, b, h, :total] += p.sum(0)
    return out, weights


def _exact_rope(st):
    case, lens, depths = st["case"], st["lens"].cpu().tolist(), st["depths"].cpu().tolist()
    hq, hk, page, table, p = case["q_heads"], case["kv_heads"], case["page"], st["table"].cpu().tolist(), case["pairs"]
    x = st["qkv"].reshape(case["batch"], case["nodes"], hq + 2 * hk, DIM).double()
    k, v, out = st["k"].double(), st["v"].double(), torch.zeros(x[:, :, :hq].shape, dtype=torch.float64, device=DEV)
    first = torch.arange(p, device=DEV) * (1 if case["layout"] == "halves" else 2)
    second = first + (p if case["layout"] == "halves" else 1)
    for b in range(case["batch"]):
        for i in range(case["nodes"]):
            turn = torch.polar(torch.full_like(st["freqs"], st["factor"]), (lens[b] + depths[b][i]) * st["freqs"])
            z = x[b, i, :hq + hk].clone()
            w = torch.complex(z[:, first], z[:, second]) * turn
            z[:, first], z[:, second] = w.real, w.imag
            pg, at = divmod(lens[b] + i, page)
            out[b, i], k[0, table[b][pg], :, at], v[0, table[b][pg], :, at] = z[:hq], z[hq:], x[b, i, hq + hk:]
    return out, k, v


def _exact_logprobs(st):
    case, tokens = st["case"], st["tokens"].cpu().tolist()
    k = case["top"]
    logprob, entropy, rank, best, token = [], [], [], [], []
    for r in range(case["rows"]):
        z = st["logits"][r].double()
        p = torch.log_softmax(z, 0)
        entropy.append(torch.special.entr(torch.exp(p)).sum())
        t = tokens[r]
        logprob.append(p[t] if t >= 0 else torch.zeros_like(p[0]))
        rank.append((z > z[t]).sum() + (z[:t] == z[t]).sum() + 1 if t >= 0 else torch.zeros((), dtype=torch.int64, device=DEV))
        if k:
            line = torch.topk(z, k).values[-1]
            some = torch.nonzero(z > line)[:, 0] if line == -math.inf else torch.nonzero(z >= line)[:, 0]
            if line == -math.inf:
                some = torch.cat([some, torch.nonzero(z == line)[:k, 0]])
            order = some[torch.sort(z[some], descending=True, stable=True).indices[:k]]
            best.append(p[order])
            token.append(order)
    empty = torch.zeros((case["rows"], 0), device=DEV)
    return (torch.stack(logprob), torch.stack(entropy), torch.stack(rank), torch.stack(best) if k else empty.double(), torch.stack(token) if k else empty.long())


def exact(case, seed):
    if case["kind"] == "evict":   # keys, values and weights are moved, nothing is computed
        return None
    return {"weigh": _exact_weigh, "rope": _exact_rope, "logprobs": _exact_logprobs}[case["kind"]](prepare(case, seed))
