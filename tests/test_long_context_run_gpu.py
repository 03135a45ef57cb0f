"""The operators for long contexts together, as a decoder uses them: passes that add up weights, eviction, going on behind it, log probabilities;
their calls on other streams, in graphs, and over memory whose offsets pass 32 bits."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import long_reference as L  # noqa: E402
import paged_reference as R  # noqa: E402
from test_long_context_gpu import _bf, _cache, _i32, _masks, _random_trees, _round_state, _weights  # noqa: E402
from test_paged_decoder_gpu import CFG, _decoder, _prompt  # noqa: E402
from test_paged_decoder_gpu import _cache as _empty_cache  # noqa: E402
from test_nint_gpu import rel_l2  # noqa: E402
from tyloquant_b200 import MfqbError, PagedCache, rope_frequencies, token_logprobs  # noqa: E402

DEV = "cuda:0"


def _host(cache):
    return {n: getattr(cache, n).float().cpu().numpy() if n in "kv" else getattr(cache, n).cpu().numpy().copy() for n in ("k", "v", "table", "lens", "refs")}


def _clone(cache):
    return PagedCache(*(getattr(cache, n).clone() for n in ("k", "v", "table", "lens", "refs")))


def test_a_decoder_that_keeps_to_a_budget():
    """Every query's probabilities sum to one; a cut cache is the restatement's, and steps over either agree as two passes over the same tokens do (the
    decoder's products of few rows may add their parts in the order of arrival: two plain steps from one state differ in the last bit of some logits;
    1e-2 as for all passes); keys come at the positions that the sequence has, not at its slots; log probabilities of the steps' logits."""
    rows, n, group = 3, 37, CFG["n_q_heads"] // CFG["n_kv_heads"]
    ids = _i32(np.random.default_rng(0).integers(0, 1000, (rows, n)))
    dec, cache = _decoder(rows * 64), _empty_cache(rows)
    weights, dropped = cache.new_weights(), torch.zeros(rows, dtype=torch.int32, device=DEV)
    dec.set_cache(cache, weights=weights, dropped=dropped)
    logits = _prompt(dec, cache, ids)
    lp = token_logprobs(logits[:, :-1].reshape(-1, 1000), ids[:, 1:].reshape(-1).contiguous(), top=4)
    want = torch.log_softmax(logits[:, :-1].reshape(-1, 1000).double(), -1)
    assert (lp.logprob.double() - want.gather(1, ids[:, 1:].reshape(-1, 1).long())[:, 0]).abs().max() <= 1e-5
    for i in range(4):
        assert int(cache.extend(1)) == 0
        dec.step(_i32([i, i + 7, 900 - i]))
    total = weights.double().sum(-1).cpu().numpy()
    assert np.allclose(total, group * (n + 4), rtol=1e-4), total   # bf16 plays no part in it
    whole = _clone(cache)                       # not cut
    st, host_w = _host(cache), weights.cpu().numpy().copy()
    gone, status = cache.evict(weights, _i32([20, 41, -1]), recent=6)
    want_gone, want_status = L.evict(st, host_w, [20, 41, -1], 6)
    assert int(status) == want_status == 0 and gone.tolist() == want_gone.tolist() == [21, 0, 0]
    assert np.array_equal(weights.cpu().numpy(), host_w) and np.array_equal(cache.k.float().cpu().numpy(), st["k"])
    dropped += gone
    other = PagedCache(_bf(st["k"]).to(DEV), _bf(st["v"]).to(DEV), *(torch.from_numpy(st[x].copy()).to(DEV) for x in ("table", "lens", "refs")))
    assert int(cache.extend(1)) == 0 and int(other.extend(1)) == 0 and int(whole.extend(1)) == 0
    token = _i32([5, 6, 7])
    dec.step(token)
    first = dec.read_logits(rows).clone()
    dec.set_cache(other, dropped=dropped)
    dec.step(token)
    assert rel_l2(first.cpu().numpy(), dec.read_logits(rows).cpu().numpy()) <= 1e-2
    dec.set_cache(whole)
    dec.step(token)

    def key(c, r):   # of layer 0, which is the token's and its position's alone
        t = int(c.lens[r]) - 1
        return c.k[0, int(c.table[r, t // c.page]), :, t % c.page]

    for r in range(rows):
        assert torch.equal(key(cache, r), key(whole, r)), r
    dec.set_cache(cache, weights=weights, dropped=dropped)
    with pytest.raises(MfqbError, match="weights are attached"):
        dec.beam_step(token, torch.zeros(rows, device=DEV), torch.zeros(rows, dtype=torch.int32, device=DEV), 1, 2)
    dec.free()


def test_a_captured_budget_follows_its_sequences():
    """A step, and an eviction of whatever is over the budget, as one graph: replays go by the lengths as they are."""
    rows, budget = 2, 24
    dec, cache = _decoder(rows * 8), _empty_cache(rows)
    weights, dropped, token, ones = cache.new_weights(), torch.zeros(rows, dtype=torch.int32, device=DEV), _i32([3, 4]), _i32([1, 1])
    keep = _i32([budget, budget + 3])
    dec.set_cache(cache, weights=weights, dropped=dropped)

    def step():
        cache.extend(ones)
        dec.step(token, token)
        gone, status = cache.evict(weights, keep, recent=8)
        dropped.add_(gone)
        return token_logprobs(dec.read_logits(rows), token, top=3), status

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lp, status = step()
    for i in range(60):
        graph.replay()
    torch.cuda.synchronize()
    assert int(status) == 0 and cache.lens.tolist() == [budget, budget + 3]
    assert (cache.lens + dropped).tolist() == [61, 61]
    assert lp.rank.tolist() == [1, 1] and torch.equal(lp.top_tokens[:, 0], token)   # the step's own token is the best one
    used = set(cache.table[cache.table >= 0].tolist())
    assert len(used) == 4 and int(cache.refs.sum()) == 4
    dec.free()


def test_calls_on_another_stream_and_two_at_once():
    """Two caches on two streams while both are busy, against the same calls one after the other."""
    rng = np.random.default_rng(1)
    states = [_round_state(R.state(rng, [900, 30, 2000], extra=9, page=32, kv_heads=2, layers=2)) for _ in range(2)]
    ws = [_weights(rng, st) for st in states]
    masks, _ = R.masks_depths(_random_trees(rng, 3, 9))
    q = _bf(rng.standard_normal((3, 9, 16, 128))).to(DEV)
    logits = torch.from_numpy(rng.standard_normal((2, 70000), dtype=np.float32)).to(DEV)

    def calls(cache, w):
        out = [cache.attend(layer, q, _masks(masks), weights=w) for layer in (0, 1)]
        gone, _ = cache.evict(w, 500, recent=100)
        x = cache.write(0, torch.ones(3, 9, 20 * 128, device=DEV, dtype=torch.bfloat16), _i32(np.zeros((3, 9))) + gone[:, None], rope_frequencies(device=DEV, dims=64))
        return [*out, gone, x, w, cache.k, cache.v, *token_logprobs(logits, _i32([5, 6]), top=8)]

    want = [calls(_cache(st), torch.from_numpy(w.copy()).to(DEV)) for st, w in zip(states, ws)]
    caches, weights = [_cache(st) for st in states], [torch.from_numpy(w.copy()).to(DEV) for w in ws]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for s, c, w in zip(streams, caches, weights):
        with torch.cuda.stream(s):
            got.append(calls(c, w))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        for x, y in zip(a, b):
            assert torch.equal(x.float().nan_to_num(7.0), y.float().nan_to_num(7.0))


@pytest.mark.parametrize("nodes,hq", [(1, 8), (9, 16), (40, 8), (64, 32)])
def test_weights_repeat_bit_for_bit(nodes, hq):
    rng = np.random.default_rng(nodes)
    st = _round_state(R.state(rng, [3000, 0, 77, 500], extra=nodes, page=64, kv_heads=2))
    masks, _ = R.masks_depths(_random_trees(rng, 4, nodes))
    cache, q = _cache(st), _bf(rng.standard_normal((4, nodes, hq, 128))).to(DEV)
    runs = []
    for _ in range(3):
        w = cache.new_weights()
        for _ in range(2):
            cache.attend(0, q, _masks(masks), weights=w)
        runs.append(w)
    assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])


def test_weights_past_32_bits():
    """2^31 weights and more: a table of 2^21 positions for the last of 64 sequences, whose keys the weights come from (their scores would not
    fit), and its eviction, whose keys do not fit shared memory."""
    rng = np.random.default_rng(2)
    rows, heads, page, width = 64, 8, 1024, 2048
    st = R.state(rng, [0] * (rows - 1) + [700], extra=3, page=page, kv_heads=heads, layers=2, width=width)
    st = _round_state(st)
    cache = _cache(st)
    weights = cache.new_weights()
    assert weights.numel() >= 2 ** 31
    q = _bf(rng.standard_normal((rows, 3, heads, 128)))
    masks, _ = R.masks_depths(_random_trees(rng, rows, 3))
    cache.attend(1, q.to(DEV), _masks(masks), weights=weights)
    small = {n: (x[-1:] if n in ("table", "lens") else x) for n, x in st.items()}
    small["table"] = small["table"][:, :1].copy()
    want, size = L.weigh(small, 1, q[-1:].float().numpy(), masks[-1:], 128 ** -0.5, np.zeros((2, 1, heads, page), np.float32))
    got = weights[1, -1, :, :page].cpu().numpy()
    assert np.abs(got - want[1, 0]).max() <= 3e-3 * want.max() and np.abs(got - want[1, 0]).sum() <= 1e-3 * want.sum()
    assert weights[1, -1].count_nonzero() == (got != 0).sum() and not weights[0].any()
    host = got.copy()[None, None]
    dropped, status = cache.evict(weights, 300, recent=50)
    both = np.concatenate([np.zeros_like(host), host])
    L.evict(small, both, [300], 50)
    assert int(status) == 0 and dropped.tolist() == [0] * (rows - 1) + [400]
    assert np.array_equal(weights[:, -1, :, :page].cpu().numpy(), both[:, 0])
    assert np.array_equal(cache.k.float().cpu().numpy(), small["k"].astype(np.float32), equal_nan=True)


def test_logits_past_32_bits():
    """Rows whose offsets pass 2^31 values."""
    rows, vocab = 36000, 65536
    logits = torch.empty((rows, vocab), dtype=torch.bfloat16, device=DEV)
    for i in range(0, rows, 4000):
        logits[i:i + 4000].normal_(generator=torch.Generator(DEV).manual_seed(i))
    tokens = torch.arange(rows, dtype=torch.int32, device=DEV) % vocab
    got = token_logprobs(logits, tokens, top=2)
    for r in (0, 32767, 32768, 35999):
        z = logits[r].double()
        p = torch.log_softmax(z, 0)
        assert abs(float(got.logprob[r]) - float(p[r])) <= 1e-5 * abs(float(p[r]))
        assert int(got.rank[r]) == int((z > z[r]).sum() + (z[:r] == z[r]).sum()) + 1
        assert int(got.top_tokens[r, 0]) == int((z == z.max()).nonzero()[0, 0])


def test_arguments_that_are_refused():
    st = R.state(np.random.default_rng(0), [20, 30], extra=2, page=16, kv_heads=2)
    cache = _cache(st)
    w, q = cache.new_weights(), torch.zeros(2, 2, 4, 128, dtype=torch.bfloat16, device=DEV)
    m = torch.ones(2, 2, dtype=torch.int64, device=DEV)
    for bad in (w[:, :1], w.double(), w.cpu(), w[..., :-1], w.transpose(0, 1)):
        with pytest.raises(ValueError, match="weights"):
            cache.attend(0, q, m, weights=bad)
        with pytest.raises(ValueError, match="weights"):
            cache.evict(bad, 5)
    wide = torch.zeros(*w.shape[:-1], 2 * w.shape[-1], device=DEV)[..., ::2]
    with pytest.raises(ValueError, match="contiguous"):
        cache.evict(wide, 5)
    with pytest.raises(ValueError, match="keep"):
        cache.evict(w, torch.zeros(3, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="keep"):
        cache.evict(w, torch.zeros(2, dtype=torch.int64, device=DEV))
    with pytest.raises(MfqbError, match="negative"):
        cache.evict(w, 5, recent=-1)
    x, d, f = torch.zeros(2, 2, 8 * 128, device=DEV), torch.zeros(2, 2, dtype=torch.int32, device=DEV), rope_frequencies(device=DEV)
    for args, kw in (((0, x.half(), d, f), {}), ((0, x, d, f.float()), {}), ((0, x, d, torch.zeros(65, dtype=torch.float64, device=DEV)), {}),
                     ((0, x, d, f.view(2, 32)), {}), ((0, x, d, f), dict(layout="thirds"))):
        with pytest.raises(ValueError):
            cache.write(*args, **kw)
    with pytest.raises(MfqbError, match="factor"):
        cache.write(0, x, d, f, factor=float("nan"))
    dec = _decoder(4)
    with pytest.raises(ValueError, match="go with a cache"):
        dec.set_cache(None, weights=w)
    own = _empty_cache(2)
    with pytest.raises(ValueError, match="weights"):
        dec.set_cache(own, weights=w)
    with pytest.raises(ValueError, match="dropped"):
        dec.set_cache(own, dropped=torch.zeros(3, dtype=torch.int32, device=DEV))
    dec.free()


def test_pools_past_32_bits():
    """The same sequences on the last pages of pools of more than 2^31 values and 2^32 bytes: the same weights, eviction and writes as on the first ones."""
    rng = np.random.default_rng(3)
    heads, page, pages = 4, 64, 40000
    st = _round_state(R.state(rng, [700, 300], extra=40, page=page, kv_heads=heads, layers=2, spare=2))
    few = st["refs"].size
    near = _cache(st)
    big = [torch.zeros((2, pages, heads, page, 128), dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    assert big[0].numel() > 2 ** 31
    for x, name in zip(big, "kv"):
        x[:, pages - few:] = getattr(near, name)
    refs = torch.ones(pages, dtype=torch.int32, device=DEV)
    refs[pages - few:] = near.refs
    far = PagedCache(*big, torch.where(near.table >= 0, near.table + (pages - few), -1), near.lens.clone(), refs)
    got = []
    for cache in (near, far):
        w = cache.new_weights()
        for nodes, hq in ((1, 8), (40, 16)):
            r = np.random.default_rng(nodes)
            masks, _ = R.masks_depths(_random_trees(r, 2, nodes))
            for layer in (0, 1):
                cache.attend(layer, _bf(r.standard_normal((2, nodes, hq, 128))).to(DEV), _masks(masks), weights=w)
        gone, status = cache.evict(w, 200, recent=30)
        x = torch.from_numpy(np.random.default_rng(9).standard_normal((2, 3, 16 * 128), dtype=np.float32)).to(DEV)
        q = cache.write(1, x, _i32(np.arange(3)[None]) + gone[:, None], rope_frequencies(device=DEV, dims=96), layout="interleaved")
        got.append((w, gone, status, cache.lens, q, cache.k[:, -few:], cache.v[:, -few:]))
    for a, b in zip(*got):
        assert torch.equal(a.float().nan_to_num(5.0), b.float().nan_to_num(5.0))
