"""Attention that adds up its weights, eviction by them, and rotary positions in other layouts against plain restatements in 64 bits.

Tolerances.  A weight is exp(scale s) / sum of such.  A float32 score of 128 exact products is off by at most 128 * 2^-23 * sum |q k| (a rounding
or a cut per addition, the tensor core's too), which moves the numerator and the sum by the factor exp of scale times that; the exponentials
of the approximate unit are off by 2^-22 and by the rounding of an argument below 2^7, 2^-17; the sum of n terms by n * 2^-24, the
sum over the rows likewise.  Rotated values: sines and cosines in float32 are off by 2^-23, the products and their difference by
2^-23 of |x| + |y|, and the result is rounded to bf16, by 2^-8 of itself."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import long_reference as L  # noqa: E402
import paged_reference as R  # noqa: E402
from tyloquant_b200 import PagedCache, rope_frequencies, rope_yarn_factor  # noqa: E402
from tyloquant_b200 import token_logprobs  # noqa: E402

DEV = "cuda:0"


def _bf(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(torch.bfloat16)


def _round_state(st):
    st["k"], st["v"] = _bf(st["k"]).float().numpy(), _bf(st["v"]).float().numpy()
    return st


def _cache(st):
    return PagedCache(_bf(st["k"]).to(DEV), _bf(st["v"]).to(DEV), *(torch.from_numpy(st[n].copy()).to(DEV) for n in ("table", "lens", "refs")))


def _gpu(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to(DEV)


def _i32(x):
    return _gpu(np.asarray(x, dtype=np.int32))


def _masks(x):
    return torch.from_numpy(np.ascontiguousarray(x).view(np.int64)).to(DEV)


def _random_trees(rng, rows, nodes):
    return np.array([[-1] + [int(rng.integers(max(0, i - 8), i)) for i in range(1, nodes)] for _ in range(rows)])


def _check_weigh(rng, st, q, masks, scale=128 ** -0.5, layer=0, calls=1):
    q = _bf(q).float().numpy()
    cache = _cache(st)
    before = rng.random(tuple(cache.new_weights().shape)).astype(np.float32)
    weights = _gpu(before)
    plain = cache.attend(layer, _bf(q).to(DEV), _masks(masks), scale=scale)
    want = before
    for _ in range(calls):
        out = cache.attend(layer, _bf(q).to(DEV), _masks(masks), scale=scale, weights=weights)
        want, size = L.weigh(st, layer, q, masks, scale, want)
    assert torch.equal(out.view(torch.int16), plain.view(torch.int16)), "the attention itself changes"
    got = weights.cpu().numpy()
    with np.errstate(invalid="ignore"):
        added = np.abs(want - before) + np.abs(want)   # at least what has been added
    rel = 2 * scale * 128 * 2.0 ** -23 * size.max() + 2.0 ** -16 + want.shape[3] * 2.0 ** -24 + q.shape[1] * q.shape[2] * 2.0 ** -24
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    same = fine & (want == before)
    assert np.array_equal(got[same], before[same]), "entries that no call adds to"
    assert (np.abs(got - want)[fine] <= (calls * rel * added)[fine]).all(), (np.abs(got - want) / np.maximum(added, 1e-30))[fine].max()
    return got


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("hq,hk", [(2, 2), (4, 2), (8, 1), (12, 4), (5, 1), (16, 1)])
def test_weights_by_heads_and_pages(hq, hk, page):
    rng = np.random.default_rng(hq * 100 + hk + page)
    st = _round_state(R.state(rng, [0, 1, 15, 130, 257], extra=7, page=page, kv_heads=hk, layers=2))
    masks, _ = R.masks_depths(_random_trees(rng, 5, 7))
    for layer in (0, 1):
        _check_weigh(rng, st, rng.standard_normal((5, 7, hq, 128)), masks, layer=layer)


@pytest.mark.parametrize("nodes,hq,hk", [(1, 4, 1), (8, 4, 1), (9, 4, 1), (16, 4, 1), (17, 4, 1), (32, 4, 1), (33, 4, 1), (64, 4, 1), (33, 8, 1), (64, 16, 1), (43, 3, 1)])
def test_weights_by_rows(nodes, hq, hk):
    """Around 32, 64, 128 and 256 rows of a kv head, up to 1024; contexts that are split, and tables that are not."""
    rng = np.random.default_rng(nodes * hq)
    for lens, width in (([700, 3, 257], None), ([192 - nodes // 2, 0, 100], 4)):
        st = _round_state(R.state(rng, lens, extra=nodes, page=64, kv_heads=hk, width=width))
        masks, _ = R.masks_depths(_random_trees(rng, 3, nodes))
        _check_weigh(rng, st, 2.0 * rng.standard_normal((3, nodes, hq, 128)), masks)


@pytest.mark.parametrize("nodes", [2, 40])
@pytest.mark.parametrize("context", [1, 63, 127, 128, 129, 255, 256, 257, 1000, 2049])
def test_weights_by_context(context, nodes):
    rng = np.random.default_rng(context)
    for lens in ([context], [context, 0, 5], [5, context, context]):
        st = _round_state(R.state(rng, lens, extra=nodes, page=64, kv_heads=2))
        masks, _ = R.masks_depths(_random_trees(rng, len(lens), nodes))
        _check_weigh(rng, st, rng.standard_normal((len(lens), nodes, 8, 128)), masks)


@pytest.mark.parametrize("nodes", [3, 40])
def test_weights_of_rows_that_see_nothing_and_pages_that_are_not_there(nodes):
    rng = np.random.default_rng(nodes)
    st = _round_state(R.state(rng, [40, 0, 300, 77], extra=nodes, page=16, kv_heads=2))
    masks, _ = R.masks_depths(_random_trees(rng, 4, nodes))
    masks[0, 1] = masks[1] = 0       # a node of no use; a sequence of none at all
    st["table"][2, 3], st["table"][2, 5], st["table"][3, 4] = -1, 10 ** 6, -7
    _check_weigh(rng, st, rng.standard_normal((4, nodes, 4, 128)), masks, calls=2)


@pytest.mark.parametrize("nodes", [3, 40])
def test_weights_of_scores_that_are_no_numbers(nodes):
    """NaN where a row's scores have one, and only where it sees; nothing for a score of minus infinity; unseen nodes do not matter."""
    rng = np.random.default_rng(nodes)
    st = _round_state(R.state(rng, [300, 30, 40, 20], extra=nodes, page=16, kv_heads=1))
    masks, _ = R.masks_depths(_random_trees(rng, 4, nodes))
    q = np.abs(rng.standard_normal((4, nodes, 4, 128)))

    def at(r, t):
        return 0, st["table"][r, t // 16], 0, t % 16

    st["k"][at(0, 200)] = -np.inf              # every score of the position is minus infinity
    st["k"][at(1, 30 + nodes - 1)] = np.inf    # the last node's: plus infinity for those that see it
    st["k"][at(2, 7)] = np.nan
    for t in range(20 + nodes):
        st["k"][at(3, t)] = -np.inf            # nothing above minus infinity
    got = _check_weigh(rng, st, q, masks)
    assert np.isnan(got[0, 1, 0, :30]).all() and np.isnan(got[0, 2, 0, :40]).all() and not np.isnan(got[0, 0]).any() and not np.isnan(got[0, 3]).any()


def test_weights_of_many_sequences_and_long_contexts():
    rng = np.random.default_rng(6)
    lens = [int(x) for x in rng.integers(0, 300, 70)]
    st = _round_state(R.state(rng, lens, extra=3, page=16, kv_heads=2))
    masks, _ = R.masks_depths(_random_trees(rng, 70, 3))
    _check_weigh(rng, st, rng.standard_normal((70, 3, 4, 128)), masks)
    st = _round_state(R.state(rng, [9000, 40, 5000], extra=2, page=128, kv_heads=1))
    masks, _ = R.masks_depths(_random_trees(rng, 3, 2))
    for hq in (4, 16):
        _check_weigh(rng, st, 2.0 * rng.standard_normal((3, 2, hq, 128)), masks)


# ---- eviction ----------------------------------------------------------------------------------------------------------------


def _weights(rng, st, kind="spread"):
    shape = (st["k"].shape[0], len(st["lens"]), st["k"].shape[2], st["table"].shape[1] * st["k"].shape[3])
    w = np.exp(3 * rng.standard_normal(shape)).astype(np.float32)
    if kind == "ties":
        w = np.round(np.log2(w)).astype(np.float32) - 2      # few values, some of them negative, zeros of both signs
        w[w == 0] *= rng.choice([-1.0, 1.0], int((w == 0).sum()))
    elif kind == "equal":
        w[:] = 0.25
    elif kind == "wild":
        w[rng.random(shape) < 0.2] = np.nan
        w[rng.random(shape) < 0.2] = np.inf
        w[rng.random(shape) < 0.2] = -np.inf
        w[rng.random(shape) < 0.1] = 3e38
        w[rng.random(shape) < 0.1] = 1e-42
    elif kind == "rising":
        w = np.broadcast_to(np.arange(shape[-1], dtype=np.float32) * 1e-3, shape).copy()
    return w


def _check_evict(st, w, keep, recent):
    cache, weights = _cache(st), _gpu(w)
    want_w = w.copy()
    dropped, status = cache.evict(weights, keep if isinstance(keep, int) else _i32(keep), recent=recent)
    want, lack = L.evict(st, want_w, [keep] * len(st["lens"]) if isinstance(keep, int) else keep, recent)
    assert int(status) == lack and np.array_equal(dropped.cpu().numpy(), want)
    for name in ("table", "lens", "refs"):
        assert np.array_equal(getattr(cache, name).cpu().numpy(), st[name]), name
    assert np.array_equal(weights.cpu().numpy().view(np.uint32), want_w.view(np.uint32))
    for name in ("k", "v"):
        assert np.array_equal(getattr(cache, name).float().cpu().numpy(), st[name].astype(np.float32), equal_nan=True), name
    return cache


@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "wild", "rising"])
@pytest.mark.parametrize("page,heads,layers", [(16, 2, 3), (64, 1, 2), (256, 3, 1)])
def test_eviction_by_weights_and_pages(page, heads, layers, kind):
    rng = np.random.default_rng(page + heads)
    for keep, recent in ((50, 10), (50, 50), (50, 400), (33, 0), (1, 1), (1, 0), (0, 5), (300, 7)):
        st = _round_state(R.state(rng, [0, 1, 51, 50, 200, 333], page=page, kv_heads=heads, layers=layers, extra=3))
        _check_evict(st, _weights(rng, st, kind), keep, recent)


@pytest.mark.parametrize("n,keep,recent", [(2047, 1000, 100), (2048, 1024, 0), (2049, 1025, 64), (5000, 4990, 129), (5000, 2500, 2500), (6001, 700, 128), (4096, 1, 0)])
@pytest.mark.parametrize("kind", ["spread", "ties", "equal"])
def test_eviction_around_the_steps(n, keep, recent, kind):
    """Lengths around the kernel's steps of 2048 slots, a few dropped and nearly all, latest rows that overlap their new places."""
    rng = np.random.default_rng(n + keep)
    st = _round_state(R.state(rng, [n, 10], page=64, kv_heads=1))
    _check_evict(st, _weights(rng, st, kind), keep, recent)


def test_eviction_of_a_table_whose_keys_do_not_fit_shared_memory():
    rng = np.random.default_rng(3)
    for kind in ("spread", "ties"):
        st = _round_state(R.state(rng, [3000, 100, 2500], page=1024, kv_heads=2, width=60))
        _check_evict(st, _weights(rng, st, kind), [1500, 90, 2400], 40)


def test_eviction_of_many_heads_without_a_cluster():
    rng = np.random.default_rng(4)
    st = _round_state(R.state(rng, [int(x) for x in rng.integers(1, 90, 60)], page=16, kv_heads=5, layers=1))
    _check_evict(st, _weights(rng, st), [int(x) for x in rng.integers(-2, 60, 60)], 5)


def _share(rng, st, pairs):
    """Sequence b takes the first `count` pages of sequence a in place of its own."""
    for a, b, count in pairs:
        for i in range(count):
            st["refs"][st["table"][b, i]] -= 1
            st["table"][b, i] = st["table"][a, i]
            st["refs"][st["table"][a, i]] += 1


@pytest.mark.parametrize("spare", [0, 1, 4, 40])
def test_eviction_from_shared_pages(spare):
    """What other sequences see stays; pages that two cut sequences share are exchanged in both, or nothing changes at all."""
    rng = np.random.default_rng(spare)
    for keep in ([60, 50, -1, 70, 10], [-1, 20, 90, 33, 0], [64, 64, 64, 64, 64]):
        st = _round_state(R.state(rng, [100, 90, 100, 80, 85], page=16, kv_heads=2, layers=2, spare=spare))
        _share(rng, st, [(0, 1, 5), (2, 3, 3), (2, 4, 2)])
        _check_evict(st, _weights(rng, st), keep, 8)


def test_eviction_without_pages_and_with_odd_counts():
    """Entries without a page have nothing to move; a free page's count may be negative and becomes one when the page is given out."""
    rng = np.random.default_rng(8)
    st = _round_state(R.state(rng, [100, 90, 70], page=16, kv_heads=2, layers=2, spare=6))
    _share(rng, st, [(0, 1, 3)])
    st["refs"][st["refs"] == 0] = -2
    st["table"][0, 4], st["table"][1, 1], st["table"][2, 0] = -1, 10 ** 6, -9
    st["lens"][2] = 10 ** 6     # taken as what the table can hold
    _check_evict(st, _weights(rng, st), [40, 41, 20], 11)


# ---- rotary positions --------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("layout", ["halves", "interleaved"])
@pytest.mark.parametrize("pairs", [64, 48, 32, 20, 1, 2, 3, 7, 33, 63])
def test_rotary_layouts(pairs, layout, dtype):
    rng = np.random.default_rng(pairs)
    lens, nodes, hq, hk = [0, 15, 33, 500, 61], 5, 6, 2
    for factor in (1.0, rope_yarn_factor(8.0)):
        st = _round_state(R.state(rng, lens, extra=nodes, page=16, kv_heads=hk, layers=2))
        st["table"][4, 61 // 16 + 1:] = -1     # some nodes have no page
        freqs = rope_frequencies(device=DEV, dims=2 * pairs)
        depths = rng.integers(0, 100000, (5, nodes)).astype(np.int32)
        qkv = 3.0 * rng.standard_normal((5, nodes, (hq + 2 * hk) * 128)).astype(np.float32)
        if dtype == "bfloat16":
            qkv = _bf(qkv).float().numpy()
        cache = _cache(st)
        q = cache.write(1, _gpu(qkv).to(getattr(torch, dtype)), _i32(depths), freqs, layout=layout, factor=factor)
        want, _, _ = L.rope(st, 1, qkv, depths, freqs.cpu().numpy(), hq, layout, factor)
        for got, ref in ((q.float().cpu().numpy(), want), (cache.k.float().cpu().numpy(), st["k"]), (cache.v.float().cpu().numpy(), st["v"])):
            assert np.array_equal(np.isnan(got), np.isnan(ref))
            top = 2 * factor * np.abs(qkv).max()
            assert np.nanmax(np.abs(got - ref) - 2.0 ** -8 * np.abs(ref)) <= 2.0 ** -21 * top
        x = qkv.reshape(5, nodes, -1, 128)[:, :, :hq, 2 * pairs:]
        assert np.array_equal(q[..., 2 * pairs:].float().cpu().numpy(), _bf(x).float().numpy()), "dims that pass"


def test_rotary_default_is_the_same_in_both_calls():
    """What turns whole heads in halves gives the same bits as bfloat16 or with a factor as the plain call does."""
    rng = np.random.default_rng(1)
    st = _round_state(R.state(rng, [5, 700], extra=3, page=16, kv_heads=2))
    x = _bf(rng.standard_normal((2, 3, 8 * 128))).to(DEV)
    a, b = _cache(st), _cache(st)
    depths, freqs = _i32([[0, 1, 2]] * 2), rope_frequencies(device=DEV)
    qa, qb = a.write(0, x.float(), depths, freqs), b.write(0, x, depths, freqs)
    assert torch.equal(qa.view(torch.int16), qb.view(torch.int16)) and torch.equal(a.k.view(torch.int16), b.k.view(torch.int16))
    assert torch.equal(a.v.view(torch.int16), b.v.view(torch.int16))


def test_rotary_values_that_are_no_numbers():
    """An infinity stays in its pair; dims that pass keep theirs."""
    st = R.state(np.random.default_rng(0), [4], extra=1, page=16, kv_heads=1)
    x = np.ones((1, 1, 3 * 128), np.float32)
    x[0, 0, 3], x[0, 0, 100], x[0, 0, 130] = np.inf, -np.inf, np.nan
    for layout in ("halves", "interleaved"):
        q = _cache(st).write(0, _gpu(x), _i32([[7]]), rope_frequencies(device=DEV, dims=96), layout=layout)[0, 0, 0].float().cpu().numpy()
        other = 51 if layout == "halves" else 2
        assert q[100] == -np.inf and np.isfinite(np.delete(q, [3, other, 100])).all() and not np.isfinite(q[3])
