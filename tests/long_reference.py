"""Plain restatements of the operators for long contexts, in numpy and 64 bits; the states are those of paged_reference."""

import numpy as np

import paged_reference as R


def sees(st, r, masks_row, nodes):
    """-> (positions there are, [nodes, positions] what every node sees, [positions] with a page)."""
    page, pages, width = st["k"].shape[3], st["k"].shape[1], st["table"].shape[1]
    n = R._len(st, r)
    total = min(n + nodes, width * page)
    ok = np.array([0 <= int(st["table"][r, t // page]) < pages for t in range(total)], dtype=bool)
    see = np.repeat(ok[None], nodes, 0)
    for i in range(nodes):
        for t in range(n, total):
            see[i, t] &= bool((int(masks_row[i]) >> (t - n)) & 1)
    return total, see, ok


def weigh(st, layer, q, masks, scale, weights):
    """The weights [layers, rows, kv_heads, positions] after the call, and the largest sum of |q k| of every (row, kv head)."""
    rows, nodes, hq, _ = q.shape
    page, hk = st["k"].shape[3], st["k"].shape[2]
    out, size = weights.astype(np.float64), np.zeros((rows, hk))
    for r in range(rows):
        n = R._len(st, r)
        total, see, ok = sees(st, r, masks[r], nodes)
        ids = np.where(ok, st["table"][r, np.arange(total) // page], 0)
        for h in range(hk):
            k = np.where(ok[:, None], st["k"][layer, ids, h, np.arange(total) % page], 0.0).astype(np.float64)
            mass = np.zeros(total)
            for i in range(nodes):
                for g in range(hq // hk):
                    x = q[r, i, h * (hq // hk) + g].astype(np.float64)
                    with np.errstate(all="ignore"):
                        s = (k @ x) * scale
                        size[r, h] = max(size[r, h], np.nan_to_num(np.where(see[i], np.abs(k) @ np.abs(x), 0), posinf=0).max(initial=0))
                        s = s[see[i]]
                        if not len(s):
                            continue
                        p = np.exp(s - s.max())
                        p = np.where(s == -np.inf, 0.0, p / p.sum())   # nothing for a score of minus infinity
                    mass[see[i]] += p
            out[layer, r, h, :n] += np.where(ok[:n], mass[:n], 0.0)
            out[layer, r, h, n:total] = mass[n:]
    return out, size


def evict(st, weights, keep, recent):
    """Changes st and weights; returns (dropped, status)."""
    page, pages = st["k"].shape[3], st["k"].shape[1]
    layers, rows, heads, _ = weights.shape
    width = st["table"].shape[1]
    lens = [R._len(st, r) for r in range(rows)]
    cut = [r for r in range(rows) if 0 <= keep[r] < lens[r]]
    old = st["table"].copy()
    swaps = [(r, i) for r in cut for i in range(width) if i * page < keep[r] and 0 <= old[r, i] < pages and st["refs"][old[r, i]] > 1]
    free = np.flatnonzero(st["refs"] <= 0)
    dropped = np.zeros(rows, np.int32)
    if len(free) < len(swaps):
        return dropped, len(swaps) - len(free)
    for (r, i), p in zip(swaps, free):
        st["refs"][old[r, i]] -= 1
        st["table"][r, i], st["refs"][p] = p, 1
    for r in cut:
        for i in range(width):
            if i * page >= keep[r]:
                if 0 <= old[r, i] < pages:
                    st["refs"][old[r, i]] -= 1
                st["table"][r, i] = -1
    was = {"k": st["k"].copy(), "v": st["v"].copy()}
    for r in cut:
        n, k = lens[r], int(keep[r])
        late = min(recent, k)
        b = k - late
        dropped[r], st["lens"][r] = n - k, k
        for layer in range(layers):
            for h in range(heads):
                w = weights[layer, r, h].copy()
                y = np.where(np.isnan(w[:n - late]), -np.inf, w[:n - late])
                stay = sorted(np.lexsort((np.arange(n - late), -y))[:b].tolist())
                holes = [s for s in range(b) if s not in set(stay)]
                source = list(range(b))
                for hole, s in zip(holes, [s for s in stay if s >= b]):
                    source[hole] = s
                source += range(n - late, n)
                for to, come in enumerate(source):
                    weights[layer, r, h, to] = w[come]
                    a, c = old[r, come // page], st["table"][r, to // page]
                    if 0 <= a < pages and 0 <= c < pages:
                        for x in ("k", "v"):
                            st[x][layer, c, h, to % page] = was[x][layer, a, h, come % page]
    return dropped, 0


def rope(st, layer, qkv, depths, freqs, hq, layout, factor):
    """Changes st; returns the rotated queries, unrounded, and the keys and values [rows, nodes, heads, 128]."""
    rows, nodes, _ = qkv.shape
    page, hk, pages = st["k"].shape[3], st["k"].shape[2], st["k"].shape[1]
    x = qkv.reshape(rows, nodes, hq + 2 * hk, 128).astype(np.float64)
    p = len(freqs)
    a = np.arange(p) if layout == "halves" else 2 * np.arange(p)
    b = a + (p if layout == "halves" else 1)
    pos = np.array([[R._len(st, r) + int(depths[r, i]) for i in range(nodes)] for r in range(rows)], dtype=np.float64)
    ang = (pos[:, :, None] * freqs)[:, :, None]
    turned = x[:, :, :hq + hk].copy()
    turned[..., a] = factor * (x[:, :, :hq + hk][..., a] * np.cos(ang) - x[:, :, :hq + hk][..., b] * np.sin(ang))
    turned[..., b] = factor * (x[:, :, :hq + hk][..., b] * np.cos(ang) + x[:, :, :hq + hk][..., a] * np.sin(ang))
    k, v = turned[:, :, hq:], x[:, :, hq + hk:]
    for r in range(rows):
        for i in range(nodes):
            t = R._len(st, r) + i
            page_no = int(st["table"][r, t // page]) if t // page < st["table"].shape[1] else -1
            if 0 <= page_no < pages:
                st["k"][layer, page_no, :, t % page], st["v"][layer, page_no, :, t % page] = k[r, i], v[r, i]
    return turned[:, :, :hq], k, v


def logprobs(logits, tokens, top):
    """-> logprob, entropy, rank, top_logprobs, top_tokens, and the average distance from the largest logit (for tolerances)."""
    rows, vocab = logits.shape
    lp, en, rank, tl, tt, far = np.zeros(rows), np.zeros(rows), np.zeros(rows, int), np.zeros((rows, top)), np.zeros((rows, top), int), np.zeros(rows)
    for r in range(rows):
        z, t = logits[r].astype(np.float64), int(tokens[r])
        there = 0 <= t < vocab
        if np.isnan(z).any() or z.max() in (np.inf, -np.inf):
            lp[r], en[r], tl[r], tt[r] = np.nan if there else 0.0, np.nan, np.nan, -1
            continue
        with np.errstate(all="ignore"):
            d = z - z.max()
            p = np.exp(d)
            s = p.sum()
            x = np.where(p > 0, p * d, 0.0).sum() / s
        en[r], far[r] = np.log(s) - x, -x
        order = np.lexsort((np.arange(vocab), -z))
        if there:
            lp[r], rank[r] = d[t] - np.log(s), int(np.flatnonzero(order == t)[0]) + 1
        tt[r], tl[r] = order[:top], d[order[:top]] - np.log(s)
    return lp, en, rank, tl, tt, far
