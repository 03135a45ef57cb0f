"""The work of a decoder whose sequences share pages of one key/value cache, as cases that can be timed: rotary embedding and cache
write of a tree of drafted tokens, attention of that tree over the cache, keeping the accepted branch, reserving and forking
pages for beams, and the selection of the beams themselves.

``listed()`` are fixed cases, ``draw(rng)`` gives others of the same ranges.  ``prepare`` builds what a program holds before
the call, ``run`` is one pass through an operator: elementary torch operations where ``own`` is false, the package's entry
points where it is true.  ``exact`` computes the same from the definitions in 64 bits."""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda:0"
DIM = 128   # width of a head


def _attend(name, batch, nodes, context, ragged, q_heads, kv_heads, page):
    return {"name": name, "kind": "attend", "batch": batch, "nodes": nodes, "context": context, "ragged": ragged, "q_heads": q_heads,
            "kv_heads": kv_heads, "page": page}


def _write(name, batch, nodes, context, q_heads, kv_heads, page):
    return {"name": name, "kind": "write", "batch": batch, "nodes": nodes, "context": context, "q_heads": q_heads, "kv_heads": kv_heads, "page": page}


def _accept(name, batch, nodes, accepted, context, layers, kv_heads, page):
    return {"name": name, "kind": "accept", "batch": batch, "nodes": nodes, "accepted": accepted, "context": context, "layers": layers,
            "kv_heads": kv_heads, "page": page}


def _fork(name, groups, beams, survivors, context, layers, kv_heads, page):
    return {"name": name, "kind": "fork", "groups": groups, "beams": beams, "survivors": survivors, "context": context, "layers": layers,
            "kv_heads": kv_heads, "page": page}


def _beams(name, groups, beams, k, vocab, done):
    return {"name": name, "kind": "beams", "groups": groups, "beams": beams, "k": k, "vocab": vocab, "done": done}


def listed():
    return [
        # one sequence, one token, a short context: what the attention of a single decoding step costs
        _attend("attend_b1_n1_ctx100", 1, 1, 100, False, 32, 8, 16),
        # sixteen sequences decoding together at a 4096-token context
        _attend("attend_b16_n1_ctx4096", 16, 1, 4096, False, 32, 8, 64),
        # trees of 27 drafted tokens on sequences of very different lengths, the narrower model
        _attend("attend_b13_n27_ragged7000", 13, 27, 7000, True, 16, 4, 64),
        # large trees (or chunks of a prompt) on long contexts
        _attend("attend_b4_n64_ctx32768", 4, 64, 32768, False, 32, 8, 128),
        # the step's own queries, keys and values: one token of one sequence; large trees of a batch
        _write("write_b1_n1", 1, 1, 4000, 32, 8, 64),
        _write("write_b16_n64", 16, 64, 500, 32, 8, 64),
        # after a verification: the accepted branch of a small tree, the branches of a batch of larger ones (the work does not
        # depend on the contexts, which are short here for the sake of the memory that all layers take)
        _accept("accept_b1_n8", 1, 8, 4, 200, 32, 8, 64),
        _accept("accept_b16_n48", 16, 48, 13, 100, 16, 8, 32),
        # a step of beam search moves to its surviving beams: one request, sixteen
        _fork("fork_g1_b4", 1, 4, 2, 230, 32, 8, 64),
        _fork("fork_g16_b4", 16, 4, 2, 100, 6, 8, 64),
        # the selection: one request with four beams; sixteen with eight, twice as many candidates kept as beams, some beams done
        _beams("beams_g1_b4_v128256", 1, 4, 4, 128256, 0.0),
        _beams("beams_g16_b8_v128256", 16, 8, 16, 128256, 0.1),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges above; attention more often than the others."""
    case = _drawn(rng)
    del case["name"]
    return case


def _drawn(rng):
    kind = rng.choice(["attend"] * 4 + ["write"] + ["accept"] * 2 + ["fork"] * 2 + ["beams"] * 2)
    kv_heads = rng.choice([4, 8])
    page = rng.choice([16, 32, 64, 128])
    if kind == "attend":
        batch, nodes, group = _log_int(rng, 1, 32), _log_int(rng, 1, 64), rng.choice([1, 2, 4, 4, 8])
        room = 4 * 64 * 32 * 32768 // (batch * nodes * kv_heads * group)
        return _attend("", batch, nodes, _log_int(rng, 16, max(16, min(32768, 40 * 8 * 4096 // (batch * kv_heads), room))), rng.random() < 0.5,
                       kv_heads * group, kv_heads, page)
    if kind == "write":
        return _write("", _log_int(rng, 1, 16), _log_int(rng, 1, 64), _log_int(rng, 16, 1000), kv_heads * rng.choice([1, 2, 4, 8]), kv_heads, page)
    if kind == "accept":
        nodes = _log_int(rng, 2, 64)
        return _accept("", _log_int(rng, 1, 16), nodes, rng.randint(1, max(1, nodes // 2)), _log_int(rng, 16, 100), _log_int(rng, 2, 16), kv_heads, page)
    if kind == "fork":
        beams = rng.randint(2, 8)
        return _fork("", _log_int(rng, 1, 64 // beams), beams, rng.randint(1, beams), _log_int(rng, 16, 200), _log_int(rng, 2, 6), kv_heads, page)
    beams = rng.randint(1, 8)
    return _beams("", _log_int(rng, 1, 16), beams, beams * rng.choice([1, 2]), _log_int(rng, 1000, 128256), rng.choice([0.0, 0.0, 0.2]))


# ---- inputs ------------------------------------------------------------------------------------------------------------------


def _lengths(case):
    """Context length of every sequence; does not depend on the seed, so that the work of a case does not."""
    n = case["batch"]
    if not case.get("ragged"):
        return [case["context"]] * n
    r = random.Random(7 * n + case["context"])
    return [case["context"]] + [_log_int(r, 1, case["context"]) for _ in range(n - 1)]


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


def _state(case, layers, k, v, table, lens, refs):
    st = {"case": case, "k": k, "v": v, "table": table.to(DEV), "lens": torch.tensor(lens, dtype=torch.int32, device=DEV), "refs": refs.to(DEV)}
    if own:
        from tyloquant_b200 import PagedCache
        st["cache"] = PagedCache(k, v, st["table"], st["lens"], st["refs"])
    return st


def _private_pages(case, layers, lens, extra, seed, gen):
    """Every sequence on pages of its own, scattered over the pool: room for `extra` tokens behind the context."""
    page = case["page"]
    held = [-(-(n + extra) // page) for n in lens]
    pages = sum(held) + 3
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((len(lens), max(held) + 1), -1, dtype=torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    at = 0
    for r, h in enumerate(held):
        table[r, :h] = order[at:at + h]
        refs[order[at:at + h].long()] = 1
        at += h
    k, v = _pool(case, layers, pages, gen)
    return _state(case, layers, k, v, table, lens, refs)


def _trees(rng, batch, nodes):
    """Random trees: node 0 is the root, the parent of another one of the eight nodes before it."""
    return [[-1] + [rng.randrange(max(0, i - 8), i) for i in range(1, nodes)] for _ in range(batch)]


def _masks_depths(parents):
    masks, depths = [], []
    for tree in parents:
        m, d = [], []
        for i, p in enumerate(tree):
            m.append((m[p] if i else 0) | 1 << i)
            d.append(d[p] + 1 if i else 0)
        masks.append([x - (1 << 64) if x >> 63 else x for x in m])
        depths.append(d)
    return torch.tensor(masks, dtype=torch.int64, device=DEV), torch.tensor(depths, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    rng, gen = random.Random(seed), _generator(seed)
    kind = case["kind"]
    if kind == "attend":
        st = _private_pages(case, 1, _lengths(case), case["nodes"], seed, gen)
        st["masks"], _ = _masks_depths(_trees(rng, case["batch"], case["nodes"]))
        st["q"] = torch.randn((case["batch"], case["nodes"], case["q_heads"], DIM), generator=gen, device=DEV).to(torch.bfloat16)
        return st
    if kind == "write":
        st = _private_pages(case, 1, _lengths(case), case["nodes"], seed, gen)
        _, st["depths"] = _masks_depths(_trees(rng, case["batch"], case["nodes"]))
        st["qkv"] = torch.randn((case["batch"], case["nodes"], (case["q_heads"] + 2 * case["kv_heads"]) * DIM), generator=gen, device=DEV)
        st["freqs"] = 500000.0 ** (-torch.arange(DIM // 2, dtype=torch.float64, device=DEV) * 2 / DIM)
        return st
    if kind == "accept":
        st = _private_pages(case, case["layers"], _lengths(case), case["nodes"], seed, gen)
        nodes, take = case["nodes"], case["accepted"]
        parents = _trees(rng, case["batch"], nodes)
        ids = [[rng.randrange(128000) for _ in t] for t in parents]
        targets = [[rng.randrange(128000) for _ in t] for t in parents]
        for p, i, t in zip(parents, ids, targets):   # the branch that the model agrees with; node 1 is never on it, so every accepted node has to move
            branch = [0] + sorted(rng.sample(range(2, nodes), min(take, nodes - 1) - 1)) if nodes > 2 and take > 1 else [0]
            for a, b in zip(branch, branch[1:]):
                p[b], t[a] = a, i[b]
        for name, x in (("parents", parents), ("ids", ids), ("targets", targets)):
            st[name] = torch.tensor(x, dtype=torch.int32, device=DEV)
        return st
    if kind == "fork":
        page, beams = case["page"], case["beams"]
        lens = [case["context"] + 7 * g for g in range(case["groups"]) for _ in range(beams)]
        shared = [case["context"] // page] * case["groups"]
        width = max(lens) // page + 2
        pages = sum(shared) + sum(-(-n // page) - shared[i // beams] for i, n in enumerate(lens)) + 2 * len(lens) + 3
        order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        table = torch.full((len(lens), width), -1, dtype=torch.int32)
        refs = torch.zeros(pages, dtype=torch.int32)
        at = 0
        for g in range(case["groups"]):   # the prompt's full pages are shared, what follows is each beam's own
            head = order[at:at + shared[g]]
            at += shared[g]
            for b in range(beams):
                r = g * beams + b
                tail = -(-lens[r] // page) - shared[g]
                table[r, :shared[g]] = head
                table[r, shared[g]:shared[g] + tail] = order[at:at + tail]
                refs[order[at:at + tail].long()] = 1
                at += tail
            refs[head.long()] = beams
        parents = []
        for g in range(case["groups"]):
            alive = rng.sample(range(beams), case["survivors"])
            parents += [g * beams + b for b in alive + [rng.choice(alive) for _ in range(beams - len(alive))]]
        k, v = _pool(case, case["layers"], pages, gen)
        st = _state(case, case["layers"], k, v, table, lens, refs)
        st["parents"] = torch.tensor(parents, dtype=torch.int32, device=DEV)
        st["ones"] = torch.ones(len(lens), dtype=torch.int32, device=DEV)
        return st
    rows = (case["groups"], case["beams"])
    return {"case": case, "logits": torch.randn((*rows, case["vocab"]), generator=gen, device=DEV) * 2.5,
            "scores": -5.0 - 2.0 * torch.rand(rows, generator=gen, device=DEV),
            "done": (torch.rand(rows, generator=gen, device=DEV) < case["done"]).to(torch.int32)}


# ---- one pass ----------------------------------------------------------------------------------------------------------------


def _gather(pool, table):
    """Pages of one layer in the order of the table: [batch, heads, tokens, 128]."""
    x = pool[table.clamp(min=0).long()]
    b, p, h, t, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(b, h, p * t, d)


def _attend_plain(st):
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
    out = (p.reshape(b, hk, n * g, -1) @ v).reshape(b, hk, n, g, DIM) / torch.where(total == 0, 1.0, total)
    return out.permute(0, 2, 1, 3, 4).reshape(b, n, hq, DIM).to(torch.bfloat16)


def _write_plain(st):
    case, lens, depths, qkv = st["case"], st["lens"].long(), st["depths"], st["qkv"]
    b, n, _ = qkv.shape
    hq, hk, page = case["q_heads"], case["kv_heads"], case["page"]
    x = qkv.reshape(b, n, hq + 2 * hk, DIM)
    angle = (lens[:, None] + depths).double()[:, :, None] * st["freqs"]
    cos, sin = torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]
    lo, hi = x[:, :, :hq + hk, :DIM // 2], x[:, :, :hq + hk, DIM // 2:]
    turned = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1).to(torch.bfloat16)
    slot = lens[:, None] + torch.arange(n, device=DEV)
    pages, at = st["table"].gather(1, slot // page).long(), slot % page
    st["k"][0][pages, :, at] = turned[:, :, hq:]
    st["v"][0][pages, :, at] = x[:, :, hq + hk:].to(torch.bfloat16)
    return turned[:, :, :hq].contiguous(), st["k"], st["v"]


def _accept_plain(st):
    case, lens, parents, ids, targets = st["case"], st["lens"].long(), st["parents"], st["ids"], st["targets"]
    b, n = ids.shape
    node = torch.arange(n, device=DEV)
    cur, live = torch.zeros(b, 1, dtype=torch.long, device=DEV), torch.ones(b, 1, dtype=torch.bool, device=DEV)
    path, count = [cur], torch.ones(b, 1, dtype=torch.long, device=DEV)
    for _ in range(n - 1):
        fits = live & (node > cur) & (parents == cur) & (ids == targets.gather(1, cur))
        live = fits.any(1, keepdim=True)
        cur = torch.where(live, torch.where(fits, node, n).amin(1, keepdim=True), cur)
        path.append(torch.where(live, cur, -1))
        count = count + live
    path = torch.cat(path, 1)
    to = lens[:, None] + node
    come = torch.where(path >= 0, lens[:, None] + path, to)   # a slot behind the branch keeps what it has
    page = case["page"]
    tp, ta, cp, ca = st["table"].gather(1, to // page).long(), to % page, st["table"].gather(1, come // page).long(), come % page
    for pool in (st["k"], st["v"]):
        pool[:, tp, :, ta] = pool[:, cp, :, ca]
    lens_out = (lens[:, None] + count)[:, 0].int()
    return count[:, 0].int(), targets.gather(1, cur)[:, 0], path.int(), lens_out, st["k"], st["v"]


def _extend_plain(st):
    """Pages for one more token of every sequence: free pages in ascending order to the sequences in ascending order."""
    table, refs, page = st["table"], st["refs"], st["case"]["page"]
    at = (st["lens"].long() // page)[:, None]   # the page of the next token
    miss = table.gather(1, at) < 0
    rank = torch.cumsum(miss[:, 0], 0)[:, None] - 1
    free = torch.argsort((refs > 0).to(torch.int8), stable=True)
    lack = (miss.sum() - (refs <= 0).sum()).clamp(min=0)
    give = miss & (lack == 0)
    new = free[rank.clamp(min=0)]
    table.scatter_(1, at, torch.where(give, new.int(), table.gather(1, at)))
    refs.index_add_(0, new[:, 0], give[:, 0].int())
    return lack.int().reshape(1)


def _fork_plain(st):
    """Sequence r goes on as sequence parents[r]: whole pages are shared, a page that is partly filled is copied for all but the first."""
    case, table, lens, refs = st["case"], st["table"], st["lens"].long(), st["refs"]
    page, parents = case["page"], st["parents"].long()
    rows, width = table.shape
    n_pages = refs.numel()
    new_len = lens[parents]
    held = (torch.arange(width, device=DEV)[None] * page < new_len[:, None])
    new = torch.where(held, table[parents], -1)
    last = ((new_len - 1).clamp(min=0) // page)[:, None]
    last_id = new.gather(1, last)
    part = (new_len % page > 0)[:, None]
    twin = ((last_id == last_id.T) & part & part.T).tril(-1).any(1)
    count = torch.zeros(n_pages + 1, dtype=torch.int32, device=DEV)
    one = torch.ones(rows * width, dtype=torch.int32, device=DEV)
    old_pages = torch.where(table < 0, n_pages, table).reshape(-1).long()
    gone = refs - count.index_add(0, old_pages, one)[:-1]
    new_once = torch.where(twin[:, None] & (torch.arange(width, device=DEV)[None] == last), -1, new)
    after = gone + count.index_add(0, torch.where(new_once < 0, n_pages, new_once).reshape(-1).long(), one)[:-1]
    lack = (twin.sum() - (after <= 0).sum()).clamp(min=0)
    free = torch.argsort((after > 0).to(torch.int8), stable=True)
    fresh = free[(torch.cumsum(twin, 0) - 1).clamp(min=0)]
    ok = lack == 0
    copied = (twin & ok).nonzero()[:, 0]
    src, dst = last_id[copied, 0].long(), fresh[copied]
    filled = torch.arange(page, device=DEV)[None, :] < (new_len[copied] % page)[:, None]
    for pool in (st["k"], st["v"]):
        pool[:, dst] = torch.where(filled[None, :, None, :, None], pool[:, src], pool[:, dst])
    new.scatter_(1, last, torch.where(twin[:, None], fresh[:, None].int(), last_id))
    after = after.index_add(0, fresh, twin.int())
    table.copy_(torch.where(ok, new, table))
    refs.copy_(torch.where(ok, after, refs))
    st["lens"].copy_(torch.where(ok, new_len, lens))
    return lack.int().reshape(1)


def _beams_plain(st):
    logits, scores, done, k = st["logits"], st["scores"].double(), st["done"] > 0, st["case"]["k"]
    g, w, vocab = logits.shape
    z = logits.double()
    top = z.amax(-1, keepdim=True)
    lse = top + torch.log(torch.exp(z - top).sum(-1, keepdim=True))
    best, token = torch.sort(logits, dim=-1, descending=True, stable=True)   # a beam's candidates: by logit, equal ones by token
    best, token = best[..., :k], token[..., :k]
    cand = scores[..., None] + (best.double() - lse)
    eos = torch.arange(k, device=DEV) == 0   # a beam that is done goes on as itself, its only candidate
    cand = torch.where(done[..., None], torch.where(eos, scores[..., None], -math.inf), cand)
    token = torch.where(done[..., None], torch.where(eos, 2, -1), token)
    parent = (torch.arange(g, device=DEV)[:, None, None] * w + torch.arange(w, device=DEV)[None, :, None]).expand(g, w, k)
    parent = torch.where(done[..., None] & ~eos, -1, parent)
    behind = (parent < 0).reshape(g, -1)
    order = torch.argsort(behind.to(torch.int8), dim=-1, stable=True)
    flat = cand.reshape(g, -1).gather(1, order)
    score, at = torch.sort(flat, dim=-1, descending=True, stable=True)
    at = order.gather(1, at[:, :k])
    return score[:, :k].float(), parent.reshape(g, -1).gather(1, at).int(), token.reshape(g, -1).gather(1, at).int()


def run(state):
    kind = state["case"]["kind"]
    if own:
        if kind == "beams":
            from tyloquant_b200 import beam_select
            return beam_select(state["logits"], state["scores"], state["case"]["k"], done=state["done"], eos=2)
        cache = state["cache"]
        if kind == "attend":
            return cache.attend(0, state["q"], state["masks"])
        if kind == "write":
            return cache.write(0, state["qkv"], state["depths"], state["freqs"]), state["k"], state["v"]
        if kind == "accept":
            count, token, path, lens = cache.accept(state["ids"], state["parents"], state["targets"])
            return count, token, path, lens, state["k"], state["v"]
        lack = cache.extend(state["ones"])
        return lack, cache.fork(state["parents"]), state["table"], state["lens"], state["refs"], state["k"], state["v"]
    if kind == "fork":
        lack = _extend_plain(state)
        return lack, _fork_plain(state), state["table"], state["lens"], state["refs"], state["k"], state["v"]
    return {"attend": _attend_plain, "write": _write_plain, "accept": _accept_plain, "beams": _beams_plain}[kind](state)


def work(case):
    kind = case["kind"]
    if kind == "attend":
        tokens = sum(n + case["nodes"] for n in _lengths(case))
        rows = case["batch"] * case["nodes"] * case["q_heads"]
        seen = sum(n * case["nodes"] for n in _lengths(case)) * case["q_heads"]
        return {"bytes": tokens * case["kv_heads"] * DIM * 4 + rows * DIM * 4 + case["batch"] * case["nodes"] * 8, "flops": 4 * seen * DIM}
    if kind == "write":
        n = case["batch"] * case["nodes"]
        heads = case["q_heads"] + 2 * case["kv_heads"]
        return {"bytes": n * (heads * DIM * 6 + 4), "flops": 6 * n * (heads - case["kv_heads"]) * DIM // 2}
    if kind == "accept":
        n = case["batch"] * case["nodes"]
        take = min(case["accepted"], case["nodes"] - 1)
        moved = case["batch"] * max(0, take - 1) * case["layers"] * case["kv_heads"]
        return {"bytes": moved * DIM * 8 + n * 16, "flops": 0}
    if kind == "fork":
        copied = (case["beams"] - case["survivors"]) * sum((case["context"] + 7 * g) % case["page"] for g in range(case["groups"]))
        held = case["beams"] * sum(-(-(case["context"] + 7 * g) // case["page"]) for g in range(case["groups"]))
        return {"bytes": copied * case["layers"] * case["kv_heads"] * DIM * 8 + held * 16, "flops": 0}
    rows = case["groups"] * case["beams"]
    return {"bytes": rows * (case["vocab"] * 4 + 8) + case["groups"] * case["k"] * 12, "flops": 3 * rows * case["vocab"]}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------------


def _exact_attend(st):
    case, page, n = st["case"], st["case"]["page"], st["case"]["nodes"]
    group = case["q_heads"] // case["kv_heads"]
    table, masks = st["table"].cpu().tolist(), st["masks"].cpu().tolist()
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    for b, length in enumerate(st["lens"].cpu().tolist()):
        total = length + n
        ids = torch.tensor(table[b][:-(-total // page)], device=DEV)
        bits = torch.tensor([[(m >> j) & 1 for j in range(n)] for m in masks[b]], device=DEV).bool()
        for h in range(case["kv_heads"]):
            k = st["k"][0, ids, h].reshape(-1, DIM)[:total].double()
            v = st["v"][0, ids, h].reshape(-1, DIM)[:total].double()
            for j in range(group):
                s = st["q"][b, :, h * group + j].double() @ k.T / math.sqrt(DIM)
                s[:, length:].masked_fill_(~bits, -math.inf)
                out[b, :, h * group + j] = torch.softmax(s, -1) @ v
    return out


def _exact_write(st):
    case, lens, depths = st["case"], st["lens"].cpu().tolist(), st["depths"].cpu().tolist()
    hq, hk, page, table = case["q_heads"], case["kv_heads"], case["page"], st["table"].cpu().tolist()
    x = st["qkv"].reshape(case["batch"], case["nodes"], hq + 2 * hk, DIM).double()
    k, v, out = st["k"].double(), st["v"].double(), torch.zeros(x[:, :, :hq].shape, dtype=torch.float64, device=DEV)
    for b in range(case["batch"]):
        for i in range(case["nodes"]):
            turn = torch.polar(torch.ones_like(st["freqs"]), (lens[b] + depths[b][i]) * st["freqs"])
            z = torch.complex(x[b, i, :hq + hk, :DIM // 2], x[b, i, :hq + hk, DIM // 2:]) * turn
            z = torch.cat([z.real, z.imag], -1)
            p, at = divmod(lens[b] + i, page)
            out[b, i], k[0, table[b][p], :, at], v[0, table[b][p], :, at] = z[:hq], z[hq:], x[b, i, hq + hk:]
    return out, k, v


def _exact_accept(st):
    case, page, table = st["case"], st["case"]["page"], st["table"].cpu().tolist()
    lens, ids, parents, targets = (st[x].cpu().tolist() for x in ("lens", "ids", "parents", "targets"))
    k, v = st["k"].clone(), st["v"].clone()
    counts, tokens, paths = [], [], []
    for b in range(case["batch"]):
        path = [0]
        while True:
            nxt = [c for c in range(path[-1] + 1, case["nodes"]) if parents[b][c] == path[-1] and ids[b][c] == targets[b][path[-1]]]
            if not nxt:
                break
            path.append(nxt[0])
        for i, node in enumerate(path):
            (tp, ta), (cp, ca) = divmod(lens[b] + i, page), divmod(lens[b] + node, page)
            k[:, table[b][tp], :, ta], v[:, table[b][tp], :, ta] = st["k"][:, table[b][cp], :, ca], st["v"][:, table[b][cp], :, ca]
        counts.append(len(path))
        tokens.append(targets[b][path[-1]])
        paths.append(path + [-1] * (case["nodes"] - len(path)))
    new = [n + c for n, c in zip(lens, counts)]
    return tuple(torch.tensor(x, device=DEV) for x in (counts, tokens, paths, new)) + (k, v)


def _exact_fork(st):
    page = st["case"]["page"]
    table, lens, refs, parents = (st[x].cpu().tolist() for x in ("table", "lens", "refs", "parents"))
    k, v = st["k"].clone(), st["v"].clone()
    for r, n in enumerate(lens):   # a page for the next token
        if table[r][n // page] < 0:
            p = refs.index(0)
            table[r][n // page], refs[p] = p, 1
    new, new_lens = [], [lens[p] for p in parents]
    for row in table:
        for p in row:
            if p >= 0:
                refs[p] -= 1
    for r, p in enumerate(parents):
        used = -(-new_lens[r] // page)
        new.append(table[p][:used] + [-1] * (len(table[p]) - used))
    seen, again = set(), []
    for r, n in enumerate(new_lens):
        for i, p in enumerate(new[r]):
            if p < 0:
                continue
            if n % page and i == n // page and p in seen:
                again.append((r, i, p, n % page))
                continue
            if n % page and i == n // page:
                seen.add(p)
            refs[p] += 1
    for r, i, p, n in again:
        q = refs.index(0)
        refs[q], new[r][i] = 1, q
        k[:, q, :, :n], v[:, q, :, :n] = st["k"][:, p, :, :n], st["v"][:, p, :, :n]
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    return zero, zero, torch.tensor(new, device=DEV), torch.tensor(new_lens, device=DEV), torch.tensor(refs, device=DEV), k, v


def _exact_beams(st):
    logits, scores, done, k = (st["logits"].cpu().numpy(), st["scores"].cpu().numpy().astype(np.float64), st["done"].cpu().numpy(), st["case"]["k"])
    g, w, _ = logits.shape
    score, parent, token = np.full((g, k), -np.inf), np.full((g, k), -1), np.full((g, k), -1)
    for i in range(g):
        cand = []
        for j in range(w):
            if done[i, j]:
                cand.append((-scores[i, j], j, 0.0, 2))
                continue
            z = logits[i, j].astype(np.float64)
            lse = np.logaddexp.reduce(z)
            cut = np.partition(z, len(z) - k)[len(z) - k]
            cand += [(-(scores[i, j] + (z[t] - lse)), j, -z[t], int(t)) for t in np.flatnonzero(z >= cut)]
        for c, (s, j, _, t) in enumerate(sorted(cand)[:k]):
            score[i, c], parent[i, c], token[i, c] = -s, i * w + j, t
    return tuple(torch.from_numpy(x).to(DEV) for x in (score, parent, token))


def exact(case, seed):
    st = prepare(case, seed)
    return {"attend": _exact_attend, "write": _exact_write, "accept": _exact_accept, "fork": _exact_fork, "beams": _exact_beams}[case["kind"]](st)
