"""Plain restatements of the operators on a paged cache, in numpy and 64 bits."""

import numpy as np


def _len(st, r):
    return min(max(int(st["lens"][r]), 0), st["table"].shape[1] * st["k"].shape[3])


def state(rng, lens, *, extra=0, page=16, kv_heads=2, layers=1, spare=3, width=None, shuffle=True):
    """Sequences on pages of their own, room for `extra` tokens behind each; what no sequence has written is NaN."""
    held = [-(-(n + extra) // page) for n in lens]
    pages = sum(held) + spare
    order = rng.permutation(pages) if shuffle else np.arange(pages)
    table = np.full((len(lens), (max(held) + 1) if width is None else width), -1, dtype=np.int32)
    refs = np.zeros(pages, dtype=np.int32)
    k = np.full((layers, pages, kv_heads, page, 128), np.nan, dtype=np.float32)
    v = np.full_like(k, np.nan)
    at = 0
    for r, h in enumerate(held):
        table[r, :h] = order[at:at + h]
        refs[table[r, :h]] = 1
        at += h
        for t in range(lens[r] + extra):
            k[:, table[r, t // page], :, t % page] = rng.standard_normal((layers, kv_heads, 128))
            v[:, table[r, t // page], :, t % page] = rng.standard_normal((layers, kv_heads, 128))
    return {"k": k, "v": v, "table": table, "lens": np.array(lens, dtype=np.int32), "refs": refs}


def masks_depths(parents):
    masks, depths = np.zeros(parents.shape, dtype=np.uint64), np.zeros(parents.shape, dtype=np.int32)
    for r, row in enumerate(parents):
        for i, p in enumerate(row):
            if i == 0:
                masks[r, 0] = 1 if p == -1 else 0
            elif 0 <= p < i and masks[r, p]:
                masks[r, i] = masks[r, p] | np.uint64(1 << i)
                depths[r, i] = depths[r, p] + 1
    return masks, depths


def attend(st, layer, q, masks, scale):
    """-> (out, weight): the outputs and, for tolerances, the sum of the probabilities times |v|."""
    rows, nodes, hq, _ = q.shape
    page, hk, pages = st["k"].shape[3], st["k"].shape[2], st["k"].shape[1]
    out, weight = np.zeros(q.shape), np.zeros(q.shape)
    for r in range(rows):
        n = _len(st, r)
        total = min(n + nodes, st["table"].shape[1] * page)
        ids = [int(st["table"][r, t // page]) for t in range(total)]
        ok = np.array([0 <= p < pages for p in ids], dtype=bool)
        for i in range(nodes):
            see = ok.copy()
            for t in range(n, total):
                see[t] &= bool((int(masks[r, i]) >> (t - n)) & 1)
            at = np.flatnonzero(see)
            if not len(at):
                continue
            pg, sl = np.array([ids[t] for t in at]), at % page
            for h in range(hq):
                kk = st["k"][layer, pg, h // (hq // hk), sl].astype(np.float64)
                vv = st["v"][layer, pg, h // (hq // hk), sl].astype(np.float64)
                with np.errstate(all="ignore"):
                    s = (kk @ q[r, i, h].astype(np.float64)) * scale
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    out[r, i, h], weight[r, i, h] = p @ vv, p @ np.abs(vv)
    return out, weight


def write(st, layer, qkv, depths, freqs, hq):
    """Changes st; returns the rotated queries in 64 bits and the unrounded keys and values [rows, nodes, heads, 128]."""
    rows, nodes, _ = qkv.shape
    page, hk, pages = st["k"].shape[3], st["k"].shape[2], st["k"].shape[1]
    x = qkv.reshape(rows, nodes, hq + 2 * hk, 128).astype(np.float64)
    pos = np.array([[_len(st, r) + depths[r, i] for i in range(nodes)] for r in range(rows)], dtype=np.float64)
    ang = (pos[:, :, None] * freqs)[:, :, None]
    lo, hi = x[:, :, :hq + hk, :64], x[:, :, :hq + hk, 64:]
    turned = np.concatenate([lo * np.cos(ang) - hi * np.sin(ang), hi * np.cos(ang) + lo * np.sin(ang)], -1)
    k, v = turned[:, :, hq:], x[:, :, hq + hk:]
    for r in range(rows):
        for i in range(nodes):
            t = _len(st, r) + i
            p = int(st["table"][r, t // page]) if t // page < st["table"].shape[1] else -1
            if 0 <= p < pages:
                st["k"][layer, p, :, t % page], st["v"][layer, p, :, t % page] = k[r, i], v[r, i]
    return turned[:, :, :hq], k, v


def accept(st, ids, parents, targets):
    """Changes k and v of st; returns count, token, path, new lengths."""
    rows, nodes = ids.shape
    page, pages = st["k"].shape[3], st["k"].shape[1]
    count, token, path = np.zeros(rows, np.int32), np.full(rows, -1, np.int32), np.full((rows, nodes), -1, np.int32)
    new = np.array([_len(st, r) for r in range(rows)], np.int32)
    old_k, old_v = st["k"].copy(), st["v"].copy()

    def slot(r, t):
        p = int(st["table"][r, t // page]) if t // page < st["table"].shape[1] else -1
        return (p, t % page) if 0 <= p < pages else None

    for r in range(rows):
        if parents[r, 0] != -1:
            continue
        branch = [0]
        while True:
            nxt = [c for c in range(branch[-1] + 1, nodes) if parents[r, c] == branch[-1] and ids[r, c] == targets[r, branch[-1]]]
            if not nxt:
                break
            branch.append(nxt[0])
        for i, b in enumerate(branch):
            to, come = slot(r, new[r] + i), slot(r, new[r] + b)
            if to and come:
                st["k"][:, to[0], :, to[1]], st["v"][:, to[0], :, to[1]] = old_k[:, come[0], :, come[1]], old_v[:, come[0], :, come[1]]
        count[r], token[r] = len(branch), targets[r, branch[-1]]
        path[r, :len(branch)] = branch
        new[r] += len(branch)
    return count, token, path, new


def extend(st, tokens):
    """Changes st; returns the status."""
    page, width, pages = st["k"].shape[3], st["table"].shape[1], st["k"].shape[1]
    want, lack = [], 0
    for r, n in enumerate(tokens):
        if n <= 0:
            continue
        last = -(-(_len(st, r) + int(n)) // page)
        lack += max(0, last - width)
        want += [(r, i) for i in range(_len(st, r) // page, min(last, width)) if not 0 <= st["table"][r, i] < pages]
    free = np.flatnonzero(st["refs"] <= 0)
    lack += max(0, len(want) - len(free))
    if lack:
        return lack
    for (r, i), p in zip(want, free):
        st["table"][r, i], st["refs"][p] = p, 1
    return 0


def fork(st, parents):
    """Changes st; returns the status."""
    page, pages = st["k"].shape[3], st["k"].shape[1]
    rows, width = st["table"].shape
    if any(p < -1 or p >= rows for p in parents):
        return -1
    refs, table, lens = st["refs"].copy(), np.full_like(st["table"], -1), np.zeros(rows, np.int32)
    for p in st["table"].reshape(-1):
        if 0 <= p < pages:
            refs[p] -= 1
    seen, twins = set(), []
    for r, p in enumerate(parents):
        if p < 0:
            continue
        lens[r] = _len(st, p)
        used = -(-int(lens[r]) // page)
        table[r, :used] = [x if 0 <= x < pages else -1 for x in st["table"][p, :used]]
        for i in range(used):
            x = table[r, i]
            if x < 0:
                continue
            if i == lens[r] // page and x in seen:
                twins.append((r, i, int(x), int(lens[r]) % page))
                continue
            if i == lens[r] // page:
                seen.add(x)
            refs[x] += 1
    free = np.flatnonzero(refs <= 0)
    if len(free) < len(twins):
        return len(twins) - len(free)
    old_k, old_v = st["k"].copy(), st["v"].copy()
    for (r, i, x, n), p in zip(twins, free):
        table[r, i] = p
        refs[p] += 1
        st["k"][:, p, :, :n], st["v"][:, p, :, :n] = old_k[:, x, :, :n], old_v[:, x, :, :n]
    st["table"][:], st["lens"][:], st["refs"][:] = table, lens, refs
    return 0


def beam_candidates(logits, scores, done, eos, k):
    """All candidates of every group, best first: lists of (score, row, token)."""
    g, w, vocab = logits.shape
    out = []
    for i in range(g):
        cand = []
        for b in range(w):
            if done is not None and done[i, b]:
                cand.append((-float(scores[i, b]), b, 0.0, eos))
                continue
            z = logits[i, b].astype(np.float64)
            with np.errstate(all="ignore"):
                lse = z.max() + np.log(np.exp(z - z.max()).sum())
                s = float(scores[i, b]) + (z - lse)
            s = np.where(np.isnan(s), -np.inf, s)
            y = np.where(np.isnan(z), -np.inf, z)
            order = np.lexsort((np.arange(vocab), -y))[:k]   # a beam's candidates: by logit, equal ones by token
            cand += [(-s[t], b, -y[t], int(t)) for t in order]
        cand.sort()
        out.append([(-s, i * w + b, t) for s, b, _, t in cand])
    return out
