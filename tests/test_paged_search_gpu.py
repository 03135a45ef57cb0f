"""Beam search over pages: beams that have ended, steps that cannot be made, a search against beams run on their own."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import paged_reference as R  # noqa: E402
from test_nint_gpu import rel_l2  # noqa: E402
from test_paged_decoder_gpu import DEV, _cache, _chain, _decoder, _i32, _prompt, _sequence  # noqa: E402

BITWISE = dict(ffn_profile=(4, 24, 6))   # no kernel whose sums differ in the last bit from call to call


def _state(cache, *more):
    return [x.clone() for x in (cache.k, cache.v, cache.table, cache.lens, cache.refs, *more)]


def _restore(cache, saved, *more):
    for x, y in zip((cache.k, cache.v, cache.table, cache.lens, cache.refs, *more), saved):
        x.copy_(y)


def _counts(cache):
    return torch.bincount(cache.table[cache.table >= 0], minlength=cache.pages).int()


def test_a_step_that_lacks_pages_changes_nothing():
    """Neither lengths nor pages that the caller has reserved behind them: the step is done again when there is room."""
    dec = _decoder(64)
    cache = _cache(2, pages=6, width=5)
    dec.set_cache(cache)
    _prompt(dec, cache, _i32(np.random.default_rng(5).integers(0, 1000, (2, 16))))
    assert int(cache.extend(_i32([40, 0]))) == 0   # three more pages for the first sequence; the second needs one
    cache.refs[cache.refs == 0] = 1                # and somebody else holds the last
    scores, done, tokens = torch.tensor([-1.0, -2.0], device=DEV), _i32([0, 0]), _i32([3, 4])
    before = _state(cache, scores, done)
    got, parents, status = dec.beam_step(tokens, scores, done, 2, eos=-1)
    assert status.tolist() == [1, 0] and got.tolist() == [3, 4] and parents.tolist() == [0, 1]
    for x, y in zip((cache.table, cache.lens, cache.refs, scores, done), before[2:]):
        assert torch.equal(x, y)
    cache.refs[(cache.refs == 1) & (_counts(cache) == 0)] = 0
    got, parents, status = dec.beam_step(tokens, scores, done, 2, eos=-1)
    assert status.tolist() == [0, 0] and cache.lens.tolist() == [17, 17]
    assert torch.equal(cache.refs, _counts(cache))
    dec.free()


def test_a_fork_that_lacks_pages_changes_nothing():
    """Both beams go on from the first, the pages of the second are held elsewhere too: there is none for the copy."""
    dec = _decoder(64)
    cache = _cache(4, pages=8, width=4)
    dec.set_cache(cache)
    _prompt(dec, cache, _i32(np.random.default_rng(5).integers(0, 1000, (4, 16))))
    assert int(cache.extend(4)) == 0   # two pages each, none is left
    cache.lens.copy_(_i32([20, 31, 19, 20]))
    cache.refs[cache.table[1, :2].long()] += 1
    scores, done, tokens = torch.tensor([0.0, -1e4, -2.0, -3.0], device=DEV), _i32([0, 0, 1, 1]), _i32([3, 4, 5, 6])
    before = _state(cache, scores, done)
    for _ in range(2):
        got, parents, status = dec.beam_step(tokens, scores, done, 2, eos=-1)
        assert status.tolist() == [0, 1] and got.tolist() == [3, 4, 5, 6] and parents.tolist() == [0, 1, 2, 3]
        for x, y in zip((cache.table, cache.lens, cache.refs, scores, done), before[2:]):
            assert torch.equal(x, y)
    cache.refs[cache.table[1, :2].long()] -= 1   # its other holder lets go
    got, parents, status = dec.beam_step(tokens, scores, done, 2, eos=-1)
    assert status.tolist() == [0, 0] and parents.tolist() == [0, 0, 2, 3] and cache.lens.tolist() == [21, 21, 19, 20]
    assert torch.equal(cache.refs, _counts(cache))
    dec.free()


def test_a_group_that_has_ended_takes_no_pages():
    """A finished group at the end of its table, beside a living one that takes the last pages of the pool: its lengths, pages and scores stay,
    and the living group goes on as it does beside a group that has room."""
    dec = _decoder(64, **BITWISE)
    got = []
    for width, pages, length in ((2, 7, 32), (4, 40, 32)):
        cache = _cache(4, pages=pages, width=width)
        dec.set_cache(cache)
        _prompt(dec, cache, _i32(np.random.default_rng(6).integers(0, 1000, (4, 12))))
        assert int(cache.extend(_i32([length - 12] * 2 + [0, 0]))) == 0
        cache.lens[:2] = length          # the first group's tables are full where they are two wide
        assert int(cache.extend(_i32([0, 0, 4, 4]))) == 0
        scores, done, tokens = torch.tensor([-3.0, -4.0, 0.0, -0.5], device=DEV), _i32([1, 1, 0, 0]), _i32([9, 9, 1, 2])
        table, k, v = cache.table[:2].clone(), cache.k.clone(), cache.v.clone()
        mine = table[:, :2].reshape(-1).long()
        steps = []
        for step in range(8):
            tokens, parents, status = dec.beam_step(tokens, scores, done, 2, eos=-1)
            if width == 2 and step == 4:
                # past its first page the living group needs a page a beam and has one: that, and nothing else, stops it
                assert int((cache.refs == 0).sum()) <= 1
            if status.tolist() != [0, 0]:
                break
            steps.append((tokens[2:].tolist(), parents[2:].tolist(), scores[2:].tolist()))
            assert cache.lens.tolist() == [length] * 2 + [12 + step + 1] * 2
            assert scores[:2].tolist() == [-3.0, -4.0] and done.tolist() == [1, 1, 0, 0]
            assert tokens[:2].tolist() == [0, 0] and parents[:2].tolist() == [0, 1]   # eos -1 is handed on as token 0
            assert torch.equal(cache.table[:2, :2], table[:, :2]) and torch.equal(cache.k[:, mine], k[:, mine]) and torch.equal(cache.v[:, mine], v[:, mine])
        got.append(steps)
    assert len(got[0]) >= 4 and len(got[1]) == 8
    for a, b in zip(*got):
        assert a[0] == b[0] and a[1] == b[1] and np.allclose(a[2], b[2], atol=0.05)
    dec.free()


def test_a_beam_that_ends_stays_as_it_is():
    """The token that a step selects first is made the end: that beam is done from then on, with its score, its length and that token, as long as it is
    among the best; a captured step does the same."""
    beams = 3
    dec = _decoder(64, **BITWISE)
    cache = _cache(2 * beams, pages=80)
    dec.set_cache(cache)
    _prompt(dec, cache, _i32(np.random.default_rng(7).integers(0, 1000, (2 * beams, 9))))
    scores, done, tokens = torch.tensor([0.0, -9.0, -9.5] * 2, device=DEV), _i32([0] * 6), _i32([1, 2, 3, 4, 5, 6])
    saved = _state(cache, scores, done)
    dry, dry_from, _ = dec.beam_step(tokens, scores, done, beams, eos=-1)
    dry_scores = scores.clone()
    assert not done.any()
    eos = int(dry[0])
    _restore(cache, saved, scores, done)
    tokens, parents, status = dec.beam_step(tokens, scores, done, beams, eos=eos)
    assert torch.equal(tokens, dry) and torch.equal(parents, dry_from) and torch.equal(scores, dry_scores) and status.tolist() == [0, 0]
    assert torch.equal(done, (dry == eos).int()) and int(done[0]) == 1
    assert cache.lens.tolist() == [10] * 6   # the last token of each beam before this step
    graph, stayed = None, 0
    for step in range(12):
        old_scores, old_done, old_lens = scores.tolist(), done.tolist(), cache.lens.tolist()
        old_pages = [cache.table[r, :-(-n // 16)].tolist() for r, n in enumerate(old_lens)]
        if step == 6:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                tokens, parents, status = dec.beam_step(tokens_in := tokens, scores, done, beams, eos=eos)
        if graph is not None:
            if step > 6:
                tokens_in.copy_(tokens)
            graph.replay()
        else:
            tokens, parents, status = dec.beam_step(tokens, scores, done, beams, eos=eos)
        assert status.tolist() == [0, 0]
        for r, p in enumerate(parents.tolist()):
            assert r // beams == p // beams
            if old_done[p]:
                stayed += 1
                assert int(done[r]) == 1 and int(tokens[r]) == eos and float(scores[r]) == old_scores[p] and int(cache.lens[r]) == old_lens[p]
                n = old_lens[p] // 16   # whole pages are the same ones
                assert cache.table[r, :n].tolist() == old_pages[p][:n]
            else:
                assert int(done[r]) == int(int(tokens[r]) == eos) and float(scores[r]) < old_scores[p] and int(cache.lens[r]) == old_lens[p] + 1
        assert parents[:beams].tolist().count(0) >= 1 or not old_done[0]   # the best beam, done, is never lost
        assert torch.equal(cache.refs, _counts(cache))
        # what is held is what the lengths need
        assert [(row >= 0).sum().item() for row in cache.table] == [-(-n // 16) for n in cache.lens.tolist()]
    assert stayed >= 12
    dec.free()


def test_every_row_has_a_beam_to_go_on_from():
    """Scores of minus infinity and NaN, beams that are done: a group never has fewer candidates than beams."""
    beams = 3
    dec = _decoder(64, **BITWISE)
    cache = _cache(3 * beams, pages=80)
    dec.set_cache(cache)
    _prompt(dec, cache, _i32(np.random.default_rng(10).integers(0, 1000, (3 * beams, 5))))
    scores = torch.tensor([-np.inf] * 3 + [np.nan, -np.inf, -1.0] + [-np.inf, np.nan, -2.0], dtype=torch.float32, device=DEV)
    done, tokens = _i32([0, 0, 0, 0, 1, 1, 1, 1, 1]), _i32(list(range(9)))
    for _ in range(4):
        tokens, parents, status = dec.beam_step(tokens, scores, done, beams, eos=-1)
        assert status.tolist() == [0, 0]
        assert [p // beams for p in parents.tolist()] == [r // beams for r in range(9)] and not torch.isnan(scores).any()
        assert done[:3].tolist() == [0] * 3 and done[6:].tolist() == [1] * 3 and int(done[3]) == 1
        assert float(scores[3]) == -1.0 and float(scores[6]) == -2.0 and (scores[:3] == -np.inf).all()
        assert torch.equal(cache.refs, _counts(cache))
    assert cache.lens[:3].tolist() == [9] * 3 and cache.lens[6:].tolist() == [5] * 3
    dec.free()


def test_tokens_that_go_round_in_place():
    """The tokens that one step writes are the next one's input, with nothing between the two; against steps that are waited for."""
    beams, runs = 4, []
    dec = _decoder(64, **BITWISE)
    for wait in (True, False):
        cache = _cache(beams, pages=40)
        dec.set_cache(cache)
        _prompt(dec, cache, _i32(np.random.default_rng(8).integers(0, 1000, (beams, 5))))
        scores, done, tokens = torch.zeros(beams, device=DEV), _i32([0] * beams), _i32([1, 2, 3, 4])
        history = []
        for _ in range(30):
            tokens, parents, _ = dec.beam_step(tokens, scores, done, beams, eos=-1)
            if wait:
                torch.cuda.synchronize()
                tokens = tokens.clone()
            history.append((tokens, parents))
        runs.append((torch.stack([torch.stack(h) for h in history]), scores, cache.k))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    dec.free()


def test_one_beam_is_the_greedy_step():
    dec = _decoder(64, **BITWISE)
    caches = [_cache(1), _cache(1)]
    prompt = _i32(np.random.default_rng(9).integers(0, 1000, (1, 7)))
    for c in caches:
        dec.set_cache(c)
        _prompt(dec, c, prompt)
    token = [_i32([11]), _i32([11])]
    scores, done = torch.zeros(1, device=DEV), _i32([0])
    for _ in range(20):
        dec.set_cache(caches[0])
        assert int(caches[0].extend(1)) == 0
        token[0] = dec.step(token[0])
        dec.set_cache(caches[1])
        token[1], parents, status = dec.beam_step(token[1], scores, done, 1, eos=-1)
        assert torch.equal(token[0], token[1]) and parents.tolist() == [0] and status.tolist() == [0, 0]
    assert caches[0].lens.tolist() == caches[1].lens.tolist() == [27]
    dec.free()


def test_every_step_of_a_search():
    """Rows, tokens and scores of each step are those that 64 bits select from the step's own logits; the logits of every beam, and at the end its keys
    and values token by token, are those of its tokens run on their own."""
    beams, steps = 4, 10
    dec = _decoder(96)
    prompt = _i32(np.random.default_rng(100).integers(0, 1000, (1, 18)))
    cache = _cache(beams, pages=30)
    dec.set_cache(cache)
    ids, chain = prompt.repeat(beams, 1), _chain(beams, 17)
    chain[1:] = -2   # one sequence has the prompt, up to its last token
    assert int(cache.extend(_i32([17] + [0] * (beams - 1)))) == 0
    dec.verify(ids[:, :17].contiguous(), chain)
    cache.accept(ids[:, :17].contiguous(), chain, torch.cat([ids[:, 1:17], ids[:, :1]], 1).contiguous(), lens_out=cache.lens)
    assert int(cache.fork(_i32([0] * beams))) == 0
    scores = torch.tensor([0.0] + [-np.inf] * (beams - 1), dtype=torch.float32, device=DEV)
    done, tokens, history, moved = _i32([0] * beams), prompt[:, -1].repeat(beams).contiguous(), [[]] * beams, 0
    logits, asked = [], []
    for _ in range(steps):
        before = scores.cpu().numpy().copy()
        tokens, parents, status = dec.beam_step(tokens, scores, done, beams, eos=-1)
        assert status.tolist() == [0, 0]
        z = dec.read_logits(beams)
        logits.append(z.cpu().numpy())
        asked.append(history)
        cand = R.beam_candidates(logits[-1][None], before[None], None, -1, beams)[0][:beams]
        assert [(p, t) for _, p, t in cand] == list(zip(parents.tolist(), tokens.tolist()))
        # a float32 rounding, and the log of a sum of float32 exponentials with 2^-21 each
        assert all(abs(s - c[0]) <= 2.0 ** -24 * abs(c[0]) + 2.0 ** -20 for s, c in zip(scores.tolist(), cand))
        moved += parents.tolist() != list(range(beams))
        history = [history[p] + [t] for p, t in zip(parents.tolist(), tokens.tolist())]
    assert moved >= 3 and torch.equal(cache.refs, _counts(cache))
    held = [(history[r], _sequence(cache, r, "k"), _sequence(cache, r, "v")) for r in range(beams)]
    for z, beams_then in zip(logits, asked):
        for b, toks in enumerate(beams_then):
            alone = _cache(1)
            dec.set_cache(alone)
            want = _prompt(dec, alone, torch.cat([prompt, _i32([toks])], 1).contiguous() if toks else prompt)[0, -1]
            assert rel_l2(z[b], want.cpu().numpy()) <= 1e-2, (b, toks)
    for toks, k, v in held:   # the last token is not in the cache yet
        alone = _cache(1)
        dec.set_cache(alone)
        _prompt(dec, alone, torch.cat([prompt, _i32([toks[:-1]])], 1).contiguous())
        for got, which in ((k, "k"), (v, "v")):
            want = _sequence(alone, 0, which)
            assert got.shape == want.shape
            assert all(rel_l2(got[layer, t], want[layer, t]) <= 1e-2 for layer in range(got.shape[0]) for t in range(got.shape[1]))
    dec.free()
