"""The dense decoder over a paged cache: its steps against those over the decoder's own cache, drafted trees against single steps, beam
search against a search that runs every beam on its own.

Two passes over the same tokens differ by the kernels that a batch takes (products within 3.6e-4), by bf16 queries in place of float32
ones, by bf16 probabilities and by the rounding of attention outputs and activations to bf16; a block stays within 3e-3 of a
float32 restatement (as over the decoder's own cache), the logits of two blocks within 1e-2 of each other."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tyloquant_b200 import MfqbError, PagedCache  # noqa: E402
from tyloquant_b200 import decoder as D  # noqa: E402
from test_nint_gpu import rel_l2  # noqa: E402

CFG = dict(hidden=512, n_q_heads=4, n_kv_heads=2, ffn=768, vocab=1000, layers=2)
DEV = "cuda:0"


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _cache(rows, pages=60, page=16, width=10):
    return PagedCache.empty(layers=CFG["layers"], kv_heads=CFG["n_kv_heads"], page=page, pages=pages, rows=rows, width=width)


def _decoder(max_batch, max_ctx=0, **over):
    return D.random_decoder(**{**CFG, **over}, max_ctx=max_ctx, max_batch=max_batch, seed=21)[0]


def _sequence(cache, r, which):
    """Keys or values of one sequence, [layers, tokens, heads, 128]."""
    pages = cache.table[r][cache.table[r] >= 0].long()
    x = getattr(cache, which)[:, pages].permute(0, 1, 3, 2, 4).flatten(1, 2)
    return x[:, :int(cache.lens[r])].float().cpu().numpy()


def _chain(rows, nodes):
    return _i32([[-1] + list(range(nodes - 1))] * rows)


def _prompt(dec, cache, ids):
    """ids [rows, n]: the prompt as a chain that is kept whole; returns the logits [rows, n, vocab]."""
    rows, n = ids.shape
    parents = _chain(rows, n)
    assert int(cache.extend(n)) == 0
    dec.verify(ids, parents)
    logits = dec.read_logits(rows * n).view(rows, n, -1)
    accepted = torch.cat([ids[:, 1:], ids[:, :1]], 1).contiguous()
    count, _, _, _ = cache.accept(ids, parents, accepted, lens_out=cache.lens)
    assert count.tolist() == [n] * rows
    return logits


@pytest.mark.parametrize("rows", [1, 3, 6])
def test_steps_over_pages_agree_with_the_own_cache(rows):
    dec = _decoder(8, max_ctx=96)
    dec.fill_cache(0)
    rng = np.random.default_rng(rows)
    tokens = [_i32(rng.integers(0, 1000, rows)) for _ in range(40)]
    want = []
    for t in tokens:
        full = torch.zeros(rows, dtype=torch.int32, device=DEV)
        full.copy_(t)
        dec.step(full)
        want.append(dec.read_logits(rows))
    cache = _cache(rows)
    dec.set_cache(cache)
    for i, t in enumerate(tokens):
        assert int(cache.extend(1)) == 0
        dec.step(t)
        assert rel_l2(dec.read_logits(rows).cpu().numpy(), want[i].cpu().numpy()) <= 1e-2, i
    assert cache.lens.tolist() == [40] * rows
    dec.set_cache(None)   # its own cache is as it was left
    dec.step(tokens[0])
    dec.free()


def test_a_prompt_in_one_pass_agrees_with_steps():
    rows, n = 3, 37
    ids = _i32(np.random.default_rng(0).integers(0, 1000, (rows, n)))
    dec = _decoder(rows * 64)
    one, many = _cache(rows), _cache(rows)
    dec.set_cache(one)
    want = []
    for i in range(n):
        assert int(one.extend(1)) == 0
        dec.step(ids[:, i].contiguous())
        want.append(dec.read_logits(rows))
    dec.set_cache(many)
    got = _prompt(dec, many, ids)
    for i in range(n):
        assert rel_l2(got[:, i].cpu().numpy(), want[i].cpu().numpy()) <= 1e-2, i
    assert torch.equal(one.lens, many.lens)
    for r in range(rows):
        for which in "kv":
            assert rel_l2(_sequence(one, r, which), _sequence(many, r, which)) <= 1e-2
    dec.free()


@pytest.mark.parametrize("heads,kv", [(6, 2), (8, 1), (16, 1), (2, 2)])
def test_head_groups_that_the_own_cache_does_not_take_too(heads, kv):
    """Three and sixteen query heads per KV head, over pages alone: a prompt in one pass against steps."""
    rows, n = 2, 20
    ids = _i32(np.random.default_rng(heads).integers(0, 1000, (rows, n)))
    dec = D.random_decoder(hidden=heads * 128, n_q_heads=heads, n_kv_heads=kv, ffn=512, vocab=1000, layers=1, max_ctx=0, max_batch=rows * n, seed=5, distinct_layers=1)[0]
    caches = [PagedCache.empty(layers=1, kv_heads=kv, page=16, pages=8, rows=rows, width=4) for _ in range(2)]
    dec.set_cache(caches[0])
    want = []
    for i in range(n):
        assert int(caches[0].extend(1)) == 0
        dec.step(ids[:, i].contiguous())
        want.append(dec.read_logits(rows))
    dec.set_cache(caches[1])
    got = _prompt(dec, caches[1], ids)
    for i in range(n):
        assert rel_l2(got[:, i].cpu().numpy(), want[i].cpu().numpy()) <= 1e-2, i
    dec.free()


def test_drafted_trees_give_what_single_steps_give():
    """Every node's logits are those of a decoder that has taken the tokens above it one by one; the accepted branch leaves the cache as if
    it had been decoded."""
    rows, nodes = 2, 9
    rng = np.random.default_rng(1)
    prompt = _i32(rng.integers(0, 1000, (rows, 21)))
    dec = _decoder(rows * 32)
    cache = _cache(rows)
    dec.set_cache(cache)
    _prompt(dec, cache, prompt)
    parents = [[-1, 0, 0, 1, 2, 2, 4, 3, 6], [-1, 0, 1, 1, 0, 4, 5, 2, 7]]
    ids = rng.integers(0, 1000, (rows, nodes))

    def above(r, i):
        out = []
        while i >= 0:
            out.append(i)
            i = parents[r][i]
        return out[::-1]

    assert int(cache.extend(nodes)) == 0
    dec.verify(_i32(ids), _i32(parents))
    got = dec.read_logits(rows * nodes).view(rows, nodes, -1)
    alone = _cache(rows)
    for i in range(nodes):
        steps = [above(r, i) for r in range(rows)]
        for r in range(rows):
            alone.table.fill_(-1)
            alone.lens.zero_()
            alone.refs.zero_()
            dec.set_cache(alone)
            _prompt(dec, alone, prompt)
            for node in steps[r]:
                assert int(alone.extend(1)) == 0
                dec.step(_i32([ids[0][node] if r == 0 else 0, ids[1][node] if r == 1 else 0]))
            want = dec.read_logits(rows)[r]
            assert rel_l2(got[r, i].cpu().numpy(), want.cpu().numpy()) <= 1e-2, (r, i)
    # accept: targets made to agree with one branch of each tree
    dec.set_cache(cache)
    targets = np.full((rows, nodes), -1)
    for r, branch in enumerate(([0, 2, 4, 6, 8], [0, 1, 2, 7])):
        for a, b in zip(branch, branch[1:]):
            targets[r, a] = ids[r][b]
    count, _, path, _ = cache.accept(_i32(ids), _i32(parents), _i32(targets), lens_out=cache.lens)
    assert count.tolist() == [5, 4] and cache.lens.tolist() == [26, 25]
    alone.table.fill_(-1)
    alone.lens.zero_()
    alone.refs.zero_()
    dec.set_cache(alone)
    _prompt(dec, alone, prompt)
    for node0, node1 in zip([0, 2, 4, 6], [0, 1, 2, 7]):
        assert int(alone.extend(1)) == 0
        dec.step(_i32([ids[0][node0], ids[1][node1]]))
    for r, n in enumerate((25, 25)):   # the last accepted node of the first tree was not stepped
        for which in "kv":
            a, b = _sequence(cache, r, which)[:, :n], _sequence(alone, r, which)
            assert a.shape == b.shape and rel_l2(a, b) <= 1e-2, (r, which)
    dec.free()


def _search(dec, prompt, beams, steps, eos):
    """Beam search that keeps no cache: every beam's tokens are run from the start; float64 log softmax."""
    live = [([], 0.0, False)]
    for _ in range(steps):
        cand = []
        for b, (toks, score, over) in enumerate(live):
            if over:
                cand.append((-score, b, 0.0, toks, None))
                continue
            cache = _cache(1)
            dec.set_cache(cache)
            ids = torch.cat([prompt, _i32([toks])], 1) if toks else prompt
            z = _prompt(dec, cache, ids.contiguous())[0, -1].double().cpu().numpy()
            lse = z.max() + np.log(np.exp(z - z.max()).sum())
            for t in np.argsort(-z, kind="stable")[:beams]:
                cand.append((-(score + z[t] - lse), b, -z[t], toks + [int(t)], int(t)))
        cand.sort(key=lambda c: c[:3])
        live = [(toks, -s, t is None or t == eos) for s, _, _, toks, t in cand[:beams]]
    return live


def test_beam_search_agrees_with_beams_run_on_their_own():
    beams, steps = 4, 9
    prompt = _i32(np.random.default_rng(2).integers(0, 1000, (1, 18)))
    dec = _decoder(68)
    want = _search(dec, prompt, beams, steps, eos=-1)
    cache = _cache(beams, pages=30)
    dec.set_cache(cache)
    ids = prompt.repeat(beams, 1)
    ids[1:] = 0
    parents = _chain(beams, 17)
    parents[1:] = -2   # one sequence has the prompt, up to its last token
    assert int(cache.extend(_i32([17] + [0] * (beams - 1)))) == 0
    dec.verify(ids[:, :17].contiguous(), parents)
    accepted = torch.cat([ids[:, 1:17], ids[:, :1]], 1).contiguous()
    cache.accept(ids[:, :17].contiguous(), parents, accepted, lens_out=cache.lens)
    assert int(cache.fork(_i32([0] * beams))) == 0
    scores = torch.tensor([0.0] + [-np.inf] * (beams - 1), dtype=torch.float32, device=DEV)
    done = torch.zeros(beams, dtype=torch.int32, device=DEV)
    tokens = prompt[:, -1].repeat(beams).contiguous()
    history = [[] for _ in range(beams)]
    for _ in range(steps):
        tokens, from_, status = dec.beam_step(tokens, scores, done, beams, eos=-1)
        assert status.tolist() == [0, 0]
        history = [history[p] + [t] for p, t in zip(from_.tolist(), tokens.tolist())]
    # scores agree within what the two ways' logits may differ by; the sequences where the search's own scores are further apart
    got = scores.double().cpu().numpy()
    assert np.abs(got - [w[1] for w in want]).max() <= 0.05
    for h, g in zip(history, got):
        near = [w for w in want if abs(w[1] - g) <= 0.05]
        assert any(h == w[0] for w in near) or len(near) > 1 or abs(g - want[-1][1]) <= 0.1, (h, g, want)
    assert cache.lens.tolist() == [17 + steps] * beams
    used = cache.table[cache.table >= 0]
    assert torch.equal(cache.refs, torch.bincount(used, minlength=30).int())
    dec.free()


def test_beams_that_end_and_pages_that_run_out():
    beams = 2
    dec = _decoder(16)
    cache = _cache(4, pages=5, width=4)   # two groups of two beams
    dec.set_cache(cache)
    ids = _i32(np.random.default_rng(3).integers(0, 1000, (4, 15)))
    _prompt(dec, cache, ids[:, :4].contiguous())   # four pages are taken
    scores, done = torch.zeros(4, device=DEV), torch.zeros(4, dtype=torch.int32, device=DEV)
    tokens = ids[:, 4].contiguous()
    dec.set_cache(cache)
    ends = 0
    for step in range(11):   # 15 tokens: within the pages
        tokens, from_, status = dec.beam_step(tokens, scores, done, beams, eos=int(tokens[0]) if step == 3 else -1)
        if status.tolist() != [0, 0]:
            break
        ends = max(ends, int(done.sum()))
    assert status.tolist()[0] == 0 or int(cache.lens.max()) % 16 == 0
    before = [x.clone() for x in (tokens, scores, done, cache.lens)]
    cache.lens.fill_(16)   # the next token needs a page for every sequence, one is free
    again, from_, status = dec.beam_step(before[0], scores, done, beams, eos=-1)
    assert status.tolist()[0] > 0 and status.tolist()[1] == 0
    assert torch.equal(again, before[0]) and from_.tolist() == [0, 1, 2, 3] and cache.lens.tolist() == [16] * 4
    assert torch.equal(scores, before[1]) and torch.equal(done, before[2])
    dec.free()


def test_a_captured_beam_step_replays():
    """Bit for bit, with 4-bit weights throughout: two to four rows of 6-bit weights take a kernel whose sums differ in the last bit from call to
    call."""
    beams = 4
    dec = _decoder(16, ffn_profile=(4, 24, 6))
    caches, outs = [], []
    prompt = _i32(np.random.default_rng(4).integers(0, 1000, (4, 4)))
    for captured in (False, True):
        cache = _cache(beams, pages=40)
        dec.set_cache(cache)
        _prompt(dec, cache, prompt)
        scores, done, tokens = torch.zeros(4, device=DEV), torch.zeros(4, dtype=torch.int32, device=DEV), _i32([1, 2, 3, 4])
        got, _, _ = dec.beam_step(tokens, scores, done, beams, eos=5)   # one call first
        tokens.copy_(got)
        torch.cuda.synchronize()
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                got, _, status = dec.beam_step(tokens, scores, done, beams, eos=5)
                tokens.copy_(got)
        for _ in range(30):
            if captured:
                graph.replay()
            else:
                got, _, status = dec.beam_step(tokens, scores, done, beams, eos=5)
                tokens.copy_(got)
            assert status.tolist() == [0, 0]
        caches.append(cache)
        outs.append((tokens.clone(), scores.clone(), done.clone()))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert torch.equal(caches[0].table, caches[1].table) and torch.equal(caches[0].k, caches[1].k)
    dec.free()


def test_what_the_decoder_refuses():
    dec = _decoder(8)
    cache = _cache(3)
    with pytest.raises(MfqbError, match="no cache of its own"):
        dec.step(_i32([1, 2, 3]))
    with pytest.raises(ValueError, match="set_cache"):
        dec.verify(_i32([[1]] * 3), _i32([[-1]] * 3))
    with pytest.raises(MfqbError, match="layers"):
        dec.set_cache(PagedCache.empty(layers=1, kv_heads=2, page=16, pages=4, rows=2, width=2))
    with pytest.raises(MfqbError, match="sequences"):
        dec.set_cache(_cache(9))
    dec.set_cache(cache)
    with pytest.raises(MfqbError, match="3 sequences"):
        dec.step(_i32([1, 2]))
    with pytest.raises(MfqbError, match="rows outside"):
        dec.verify(_i32([[1] * 3] * 3), _i32([[-1, 0, 1]] * 3))   # 9 rows, the decoder takes 8
    with pytest.raises(ValueError, match="parents"):
        dec.verify(_i32([[1, 2]] * 3), _i32([[-1]] * 3))
    scores, done = torch.zeros(3, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)
    with pytest.raises(MfqbError, match="groups"):
        dec.beam_step(_i32([1, 2, 3]), scores, done, 2, eos=-1)
    with pytest.raises(ValueError, match="scores"):
        dec.beam_step(_i32([1, 2, 3]), scores.double(), done, 3, eos=-1)
    with pytest.raises(MfqbError, match="cache"):
        dec.fill_cache(4)
    dec.free()
