"""The operators on a paged cache against plain restatements in 64 bits: attention of drafted trees, cache write, accepted branches,
reserved and forked pages, beam selection, and a run of them as a decoder uses them.

Tolerances.  A bf16 result is off by at most half a step, 2^-8 of its size.  Attention rounds each probability to bf16 too, 2^-8 of
it, and may do so in the sum of the products and in the sum that normalises it: the average moves by at most 2 * 2^-8 times the
average of |v|.  Float32 scores of 128 terms and the exponentials add less than 2^-12 of that average
(|score| <= 60 in these tests: 128 * 2^-24 * 60 * log2(e))."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import paged_reference as R  # noqa: E402
from oracle import mfq_oracle as O  # noqa: E402
from tyloquant_b200 import PagedCache, beam_select, rope_frequencies, tree_masks  # noqa: E402

DEV = "cuda:0"


def _bf(x):
    """Rounded to bf16, infinities and NaN as they are."""
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).to(torch.bfloat16)


def _round_state(st):
    st["k"], st["v"] = _bf(st["k"]).float().numpy(), _bf(st["v"]).float().numpy()
    return st


def _cache(st):
    return PagedCache(_bf(st["k"]).to(DEV), _bf(st["v"]).to(DEV), *(torch.from_numpy(st[n].copy()).to(DEV) for n in ("table", "lens", "refs")))


def _i32(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).to(DEV)


def _u64(x):
    return torch.from_numpy(np.ascontiguousarray(x).view(np.int64)).to(DEV)


def _same_pool(pool, want):
    assert np.array_equal(pool.float().cpu().numpy(), want.astype(np.float32), equal_nan=True)


def _random_trees(rng, rows, nodes):
    return np.array([[-1] + [int(rng.integers(max(0, i - 8), i)) for i in range(1, nodes)] for _ in range(rows)])


def _check_attend(st, q, masks, scale=128 ** -0.5, layer=0, cache=None, same=True):
    q = _bf(q).float().numpy()
    cache = cache or _cache(st)
    got = cache.attend(layer, _bf(q).to(DEV), _u64(masks), scale=scale).float().cpu().numpy()
    want, weight = R.attend(st, layer, q, masks, scale)
    fine = np.isfinite(want)
    assert np.array_equal(np.isfinite(got), fine)
    if same:
        assert np.array_equal(np.isnan(got), np.isnan(want)), "NaN in other places"
        assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)].astype(np.float32))
    bound = 2.0 ** -8 * np.abs(want) + (2.0 ** -7 + 2.0 ** -12) * weight
    off = np.abs(got[fine] - want[fine])
    assert (off <= bound[fine]).all(), (off - bound[fine]).max()
    return got


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("hq,hk", [(2, 2), (4, 2), (8, 1), (12, 4), (5, 1), (16, 1)])
def test_attention_by_heads_and_pages(hq, hk, page):
    rng = np.random.default_rng(hq * 100 + hk + page)
    nodes = 7
    st = _round_state(R.state(rng, [0, 1, 15, 130, 257], extra=nodes, page=page, kv_heads=hk, layers=2))
    masks, _ = R.masks_depths(_random_trees(rng, 5, nodes))
    for layer in (0, 1):
        _check_attend(st, rng.standard_normal((5, nodes, hq, 128)), masks, layer=layer)


@pytest.mark.parametrize("nodes", [1, 2, 3, 17, 32, 33, 48, 63, 64])
def test_attention_by_nodes(nodes):
    rng = np.random.default_rng(nodes)
    st = _round_state(R.state(rng, [0, 3, 127, 128, 129, 500], extra=nodes, page=32, kv_heads=2))
    masks, _ = R.masks_depths(_random_trees(rng, 6, nodes))
    _check_attend(st, 3.0 * rng.standard_normal((6, nodes, 8, 128)), masks)


@pytest.mark.parametrize("context", [1, 63, 64, 65, 126, 127, 128, 200, 255, 256, 257, 1000, 2049])
def test_attention_by_context(context):
    """Contexts around the tiles, alone and beside short ones: splits over the context and their merge."""
    rng = np.random.default_rng(context)
    for lens in ([context], [context, 0, 5], [5, context, context]):
        st = _round_state(R.state(rng, lens, extra=4, page=64, kv_heads=2))
        masks, _ = R.masks_depths(_random_trees(rng, len(lens), 4))
        _check_attend(st, rng.standard_normal((len(lens), 4, 8, 128)), masks)


def test_attention_of_long_contexts():
    rng = np.random.default_rng(5)
    st = _round_state(R.state(rng, [9000, 40, 5000], extra=2, page=128, kv_heads=1))
    masks, _ = R.masks_depths(_random_trees(rng, 3, 2))
    _check_attend(st, 2.0 * rng.standard_normal((3, 2, 4, 128)), masks)


def test_attention_of_many_sequences():
    rng = np.random.default_rng(6)
    lens = [int(x) for x in rng.integers(0, 300, 70)]
    st = _round_state(R.state(rng, lens, extra=3, page=16, kv_heads=2))
    masks, _ = R.masks_depths(_random_trees(rng, 70, 3))
    _check_attend(st, rng.standard_normal((70, 3, 4, 128)), masks)


@pytest.mark.parametrize("hq,hk,nodes", [(16, 1, 64), (16, 1, 9), (8, 1, 17), (32, 8, 64), (3, 1, 43), (3, 1, 11), (3, 1, 22)])
def test_attention_by_rows(hq, hk, nodes):
    """Around 32, 64, 128 and 256 rows of a kv head, up to 1024; contexts that are split, and tables of up to 256 positions, which are not."""
    rng = np.random.default_rng(hq * nodes)
    for lens, width in (([700, 3, 257], None), ([192 - nodes // 2, 0, 100], 4)):
        st = _round_state(R.state(rng, lens, extra=nodes, page=64, kv_heads=hk, width=width))
        masks, _ = R.masks_depths(_random_trees(rng, 3, nodes))
        _check_attend(st, 2.0 * rng.standard_normal((3, nodes, hq, 128)), masks)


@pytest.mark.parametrize("value,which", [(np.nan, "k"), (np.nan, "v"), (np.inf, "k"), (-np.inf, "k"), (np.inf, "v")])
def test_what_is_seen_counts(value, which):
    """Infinities and NaN in the context, in one part of a split one, and scores that are all minus infinity.  (An infinite value is infinity or
    NaN in its dimension: a part that does not hold it multiplies it by zero.)"""
    rng = np.random.default_rng(30)
    st = _round_state(R.state(rng, [900, 40, 1], extra=2, page=64, kv_heads=2))
    for r, t in ((0, 333), (1, 7), (2, 0)):
        st[which][0, st["table"][r, t // 64], :, t % 64, 5] = value
    q = rng.standard_normal((3, 2, 4, 128))
    q[..., 5] = 1.0   # an infinite key's score has its sign
    masks = np.array([[1, 3], [1, 3], [0, 0]], np.uint64)   # the third sequence sees its one token alone
    _check_attend(st, q, masks, same=which == "k")


def test_caches_on_two_streams():
    rng = np.random.default_rng(31)
    sts = [_round_state(R.state(rng, lens, extra=20, page=32, kv_heads=2)) for lens in ([3000, 10, 500], [90, 2000, 1])]
    masks, _ = R.masks_depths(_random_trees(rng, 3, 20))
    caches, m = [_cache(st) for st in sts], _u64(masks)
    qs = [_bf(rng.standard_normal((3, 20, 8, 128))).to(DEV) for _ in sts]
    want = [c.attend(0, q, m).clone() for c, q in zip(caches, qs)]
    streams = [torch.cuda.Stream() for _ in sts]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(caches[i].attend(0, qs[i], m))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_rising_scores_and_scales():
    """Scores that grow along the context (every tile raises the maximum), shrink along it, and lie far from zero."""
    rng = np.random.default_rng(7)
    for sign in (1.0, -1.0):
        st = R.state(rng, [700, 300], extra=3, page=64, kv_heads=1)
        for r, n in enumerate((700, 300)):
            for t in range(n + 3):
                st["k"][0, st["table"][r, t // 64], 0, t % 64] = sign * t / 64.0
        st = _round_state(st)
        masks, _ = R.masks_depths(_random_trees(rng, 2, 3))
        q = np.abs(rng.standard_normal((2, 3, 2, 128)))
        _check_attend(st, q, masks, scale=0.04)
        _check_attend(st, -q, masks, scale=0.04)


def test_masks_that_leave_nothing_or_gaps():
    """Arbitrary masks: nothing, only others, every second node; over an empty context a row sees nothing and is zero."""
    rng = np.random.default_rng(8)
    nodes = 40
    st = _round_state(R.state(rng, [0, 0, 90, 128], extra=nodes, page=16, kv_heads=2))
    masks = np.zeros((4, nodes), np.uint64)
    masks[1, ::2] = rng.integers(0, 1 << 40, 20).astype(np.uint64)
    masks[2] = np.uint64(0x5555555555)
    masks[3, 5] = np.uint64(1 << 39)
    q = rng.standard_normal((4, nodes, 4, 128))
    got = _check_attend(st, q, masks)
    assert not got[0].any() and not got[1, 1::2].any()
    # bits behind the last node mean nothing
    assert np.array_equal(_check_attend(st, q, masks | np.uint64(0xFF << 40)), got)


@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_what_is_not_seen_has_no_effect(value):
    """NaN and infinities in nodes of other branches, behind the last node and on other pages; where they are seen they count."""
    rng = np.random.default_rng(9)
    nodes = 9
    st = _round_state(R.state(rng, [0, 60, 250], extra=nodes, page=16, kv_heads=2))
    parents = np.array([[-1, 0, 0, 1, 2, 1, 4, 6, 3]] * 3)
    masks, _ = R.masks_depths(parents)
    q = rng.standard_normal((3, nodes, 4, 128))
    clean = _check_attend(st, q, masks)
    for r in range(3):
        for which, node, dims in (("v", 2, slice(3, 5)), ("k", 5, slice(0, 128)), ("v", 8, slice(100, 101))):
            t = int(st["lens"][r]) + node
            st[which][0, st["table"][r, t // 16], :, t % 16, dims] = value
    got = _check_attend(st, q, masks)
    for node in (0, 1, 3):   # neither under 2, nor 5, nor 8
        assert np.array_equal(got[:, node], clean[:, node])


def test_pages_outside_the_pool_are_not_read():
    rng = np.random.default_rng(10)
    st = _round_state(R.state(rng, [100, 40, 300], extra=5, page=16, kv_heads=2))
    for r, i, p in ((0, 2, -1), (0, 3, 10 ** 6), (1, 2, -(1 << 31)), (2, 0, len(st["refs"])), (2, 17, (1 << 31) - 1), (2, 19, -5)):
        st["table"][r, i] = p
    masks, _ = R.masks_depths(_random_trees(rng, 3, 5))
    _check_attend(st, rng.standard_normal((3, 5, 4, 128)), masks)
    st["table"][:] = -1   # nothing anywhere
    assert not _check_attend(st, rng.standard_normal((3, 5, 4, 128)), masks).any()


def test_lengths_outside_the_table():
    rng = np.random.default_rng(11)
    st = _round_state(R.state(rng, [64, 30, 64], page=16, kv_heads=1, width=4))
    st["lens"][:] = [1000, -5, (1 << 31) - 1]
    masks, _ = R.masks_depths(_random_trees(rng, 3, 6))
    _check_attend(st, rng.standard_normal((3, 6, 2, 128)), masks)


def test_offsets_past_32_bits():
    """A pool of more than 2^32 bytes: pages at its end."""
    pages, page, hk = 5000, 512, 4
    k = torch.zeros(1, pages, hk, page, 128, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros_like(k)
    g = torch.Generator(DEV).manual_seed(1)
    ids = [pages - 1, 1, pages - 2]
    for p in ids:
        k[0, p] = torch.randn(hk, page, 128, generator=g, device=DEV)
        v[0, p] = torch.randn(hk, page, 128, generator=g, device=DEV)
    small = {"k": k[:, ids].float().cpu().numpy(), "v": v[:, ids].float().cpu().numpy(), "table": np.array([[0, 1, 2]], np.int32), "lens": np.array([1300], np.int32)}
    cache = PagedCache(k, v, _i32([ids]), _i32([1300]), torch.ones(pages, dtype=torch.int32, device=DEV))
    rng = np.random.default_rng(12)
    masks, _ = R.masks_depths(_random_trees(rng, 1, 4))
    _check_attend(small, rng.standard_normal((1, 4, 8, 128)), masks, cache=cache)


def test_writes_and_moves_past_32_bits():
    """The same pool sizes for what writes: cache write, accepted branch and fork on the last pages of a pool of more than 2^32 bytes."""
    layers, pages, page, hk, hq = 2, 9000, 256, 2, 4
    k = torch.zeros(layers, pages, hk, page, 128, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros_like(k)
    assert k.numel() * 2 > 1 << 31 and k.numel() > 1 << 30
    last = pages - 1
    refs = torch.ones(pages, dtype=torch.int32, device=DEV)
    refs[last - 1] = 0
    cache = PagedCache(k, v, _i32([[last, -1], [-1, -1]]), _i32([10, 0]), refs)
    rng = np.random.default_rng(40)
    small = {"k": np.zeros((layers, 2, hk, page, 128), np.float32), "v": np.zeros((layers, 2, hk, page, 128), np.float32), "table": np.array([[1, -1], [-1, -1]], np.int32),
             "lens": np.array([10, 0], np.int32), "refs": np.array([0, 1], np.int32)}
    depths = np.array([[0, 1, 1, 2, 2]] * 2)
    freqs = rope_frequencies(device=DEV)
    for layer in range(layers):
        qkv = rng.standard_normal((2, 5, (hq + 2 * hk) * 128)).astype(np.float32)
        cache.write(layer, torch.from_numpy(qkv).to(DEV), _i32(depths), freqs)
        R.write(small, layer, qkv, depths, freqs.cpu().numpy(), hq)
    two = lambda pool: pool[:, last - 1:].float().cpu().numpy()   # the last two pages
    for got, want in ((two(k), small["k"]), (two(v), small["v"])):
        assert (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 12 * 2.0 ** -20).all()
    small["k"], small["v"] = two(k), two(v)
    parents, ids, targets = np.array([[-1, 0, 0, 2, 3]] * 2), np.array([[0, 7, 1, 1, 1]] * 2), np.ones((2, 5))
    cache.accept(_i32(ids), _i32(parents), _i32(targets), lens_out=cache.lens)
    small["lens"] = R.accept(small, ids, parents, targets)[3]
    assert np.array_equal(two(k), small["k"]) and np.array_equal(two(v), small["v"])
    cache.lens[1] = small["lens"][1] = 0
    assert int(cache.fork(_i32([0, 0]))) == R.fork(small, [0, 0]) == 0
    assert cache.table.tolist() == [[last, -1], [last - 1, -1]] and cache.lens.tolist() == [14, 14]
    assert np.array_equal(two(k), small["k"]) and np.array_equal(two(v), small["v"])
    assert not k[:, :last - 1].any() and not v[:, :last - 1].any()


@pytest.mark.parametrize("rows,nodes,hq,hk", [(1, 1, 4, 2), (3, 5, 8, 1), (2, 64, 6, 2), (20, 9, 32, 8)])
def test_write(rows, nodes, hq, hk):
    rng = np.random.default_rng(nodes)
    lens = [int(x) for x in rng.integers(0, 200, rows)]
    lens[0] = 0
    st = _round_state(R.state(rng, lens, extra=nodes, page=16, kv_heads=hk, layers=2))
    st["table"][-1, (lens[-1] + nodes - 1) // 16] = -1 if rows > 1 else st["table"][-1, (lens[-1] + nodes - 1) // 16]   # a page that is missing
    cache = _cache(st)
    _, depths = R.masks_depths(_random_trees(rng, rows, nodes))
    qkv = rng.standard_normal((rows, nodes, (hq + 2 * hk) * 128)).astype(np.float32)
    freqs = rope_frequencies(10000.0, DEV)
    q = cache.write(1, torch.from_numpy(qkv).to(DEV), _i32(depths), freqs).float().cpu().numpy()
    want, _, _ = R.write(st, 1, qkv, depths, freqs.cpu().numpy(), hq)
    # half a bf16 step, and float32 products of values below 6: 2^-20 of them
    assert (np.abs(q - want) <= 2.0 ** -8 * np.abs(want) + 12 * 2.0 ** -20).all()
    for got, ref in ((cache.k, st["k"]), (cache.v, st["v"])):
        got = got.float().cpu().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(ref))
        assert (np.abs(got - ref)[~np.isnan(ref)] <= 2.0 ** -8 * np.abs(ref)[~np.isnan(ref)] + 12 * 2.0 ** -20).all()
    assert np.array_equal(cache.lens.cpu().numpy(), st["lens"])


def test_angles_of_far_positions():
    """2^26 + 13 positions: a float32 angle would be off by whole radians."""
    width, page = 1 << 17, 1024
    st = {"k": np.zeros((1, 2, 1, page, 128), np.float32), "v": np.zeros((1, 2, 1, page, 128), np.float32), "table": np.full((1, width), -1, np.int32),
          "lens": np.array([(1 << 26) + 13], np.int32), "refs": np.ones(2, np.int32)}
    st["table"][0, 1 << 16] = 1
    cache = _cache(st)
    rng = np.random.default_rng(1)
    qkv = rng.standard_normal((1, 3, 4 * 128)).astype(np.float32)
    freqs = rope_frequencies(500000.0, DEV)
    q = cache.write(0, torch.from_numpy(qkv).to(DEV), _i32([[0, 1, 2]]), freqs).float().cpu().numpy()
    want, _, _ = R.write(st, 0, qkv, np.array([[0, 1, 2]]), freqs.cpu().numpy(), 2)
    assert (np.abs(q - want) <= 2.0 ** -8 * np.abs(want) + 12 * 2.0 ** -20).all()
    k = cache.k.float().cpu().numpy()
    assert (np.abs(k - st["k"]) <= 2.0 ** -8 * np.abs(st["k"]) + 12 * 2.0 ** -20).all()


def test_tree_masks():
    rng = np.random.default_rng(2)
    for rows, nodes in ((1, 1), (3, 2), (5, 31), (2, 33), (40, 64)):
        parents = _random_trees(rng, rows, nodes)
        if nodes > 5:
            parents[0] = np.arange(nodes) - 1        # a chain
            parents[1, 3], parents[1, 4] = 3, 7      # not an earlier node: unused, with what hangs below
            parents[1, 5] = -1                       # a second root
        if rows > 2:
            parents[2, 0] = 0                        # the row is unused
        masks, depths = tree_masks(_i32(parents))
        want, want_depths = R.masks_depths(parents)
        assert np.array_equal(masks.cpu().numpy().view(np.uint64), want) and np.array_equal(depths.cpu().numpy(), want_depths)


@pytest.mark.parametrize("rows,nodes,page", [(1, 1, 16), (4, 2, 16), (6, 12, 16), (3, 64, 32), (5, 40, 128)])
def test_accept(rows, nodes, page):
    rng = np.random.default_rng(rows * nodes)
    lens = [int(x) for x in rng.integers(0, 100, rows)]
    st = _round_state(R.state(rng, lens, extra=nodes, page=page, kv_heads=3, layers=2))
    parents = _random_trees(rng, rows, nodes)
    ids, targets = rng.integers(0, 3, (rows, nodes)), rng.integers(0, 3, (rows, nodes))   # few tokens: long branches, several fitting children
    if nodes == 64:
        parents[0] = np.arange(64) - 1
        ids[0], targets[0] = 1, 1        # all of a chain: nothing moves
        parents[1] = [-1] + [0] * 63     # a root with 63 children, the last one fits
        ids[1], targets[1] = 2, 1
        ids[1, 63] = 1
    if rows > 3:
        parents[3, 0] = 5                # an unused row
    cache = _cache(st)
    count, token, path, lens_out = cache.accept(_i32(ids), _i32(parents), _i32(targets))
    want = R.accept(st, ids, parents, targets)
    for got, ref in zip((count, token, path, lens_out), want):
        assert np.array_equal(got.cpu().numpy(), ref)
    _same_pool(cache.k, st["k"])
    _same_pool(cache.v, st["v"])
    assert np.array_equal(cache.lens.cpu().numpy(), lens)
    cache.accept(_i32(ids), _i32(parents), _i32(targets), lens_out=cache.lens)   # in place
    assert np.array_equal(cache.lens.cpu().numpy(), want[3])


def test_accept_on_pages_that_are_missing():
    rng = np.random.default_rng(3)
    st = _round_state(R.state(rng, [14, 30], extra=8, page=16, kv_heads=1))
    st["table"][0, 1], st["table"][1, 1] = -1, 10 ** 6
    parents, ids, targets = np.array([[-1, 0, 0, 2, 3, 4, 5, 6]] * 2), np.array([[0, 9, 1, 1, 1, 1, 1, 1]] * 2), np.ones((2, 8))
    cache = _cache(st)
    got = cache.accept(_i32(ids), _i32(parents), _i32(targets))
    want = R.accept(st, ids, parents, targets)
    for a, b in zip(got, want):
        assert np.array_equal(a.cpu().numpy(), b)
    _same_pool(cache.k, st["k"])


def _same_cache(cache, st):
    for name in ("table", "lens", "refs"):
        assert np.array_equal(getattr(cache, name).cpu().numpy(), st[name]), name
    _same_pool(cache.k, st["k"])
    _same_pool(cache.v, st["v"])


@pytest.mark.parametrize("page", [16, 128])
def test_pages_of_random_forks(page):
    """Many steps of reserving and forking, with sequences that end, full pages, empty sequences and a pool that runs out."""
    rng = np.random.default_rng(page)
    rows = 7
    st = _round_state(R.state(rng, [3, page, page + 1, 2 * page, 0, 5 * page - 1, 17], page=page, kv_heads=2, layers=2, width=8, spare=2))
    cache = _cache(st)
    lacks = 0
    for step in range(60):
        if step % 3 == 2:
            parents = rng.integers(0, rows, rows)
            parents[rng.random(rows) < 0.05] = -1
            want = R.fork(st, parents)
            got = int(cache.fork(_i32(parents)))
        else:
            tokens = rng.integers(-1, 2 * page // 3, rows)
            want = R.extend(st, tokens)
            got = int(cache.extend(_i32(tokens)))
            if want == 0 and step % 3 == 0:   # the tokens arrive
                add = np.minimum(np.maximum(tokens, 0), 1 + page // 4)
                for r in range(rows):
                    for t in range(int(st["lens"][r]), int(st["lens"][r] + add[r])):
                        p = st["table"][r, t // page]
                        st["k"][:, p, :, t % page], st["v"][:, p, :, t % page] = (_bf(rng.standard_normal((2, 2, 128))).float().numpy() for _ in range(2))
                cache.k.copy_(_bf(st["k"]))
                cache.v.copy_(_bf(st["v"]))
                st["lens"] += add.astype(np.int32)
                cache.lens.copy_(torch.from_numpy(st["lens"]))
        assert got == want, step
        lacks += want > 0
        _same_cache(cache, st)
        assert (st["refs"] == np.bincount(st["table"][st["table"] >= 0], minlength=len(st["refs"]))).all()
    assert lacks > 3   # the pool did run out


def test_forks_that_are_refused_or_do_not_fit():
    rng = np.random.default_rng(4)
    st = _round_state(R.state(rng, [20, 33, 5], page=16, kv_heads=1, spare=0))
    cache = _cache(st)
    for parents in ([0, 3, 1], [0, -2, 1], [(1 << 31) - 1, 0, 0]):
        assert int(cache.fork(_i32(parents))) == -1
        _same_cache(cache, st)
    assert int(cache.fork(_i32([0, 1, 0]))) == R.fork(st, [0, 1, 0]) == 0   # the page that sequence 2 gives back is the one it gets
    _same_cache(cache, st)
    assert int(cache.fork(_i32([1, 1, 1]))) == R.fork(st, [1, 1, 1])
    _same_cache(cache, st)
    assert int(cache.fork(_i32([-1, -1, -1]))) == R.fork(st, [-1, -1, -1]) == 0
    _same_cache(cache, st)
    assert not st["refs"].any()
    for tokens in ([1, 0, 1000], [1 << 30, 1, 1], [16 * len(st["refs"]), 1, 0]):
        want = R.extend(st, tokens)
        assert int(cache.extend(_i32(tokens))) == want > 0
        _same_cache(cache, st)


def test_a_large_pool_and_many_sequences():
    """More pages than a thread block looks at in a round, free ones scattered; 1024 sequences; more pages wanted than threads."""
    rng = np.random.default_rng(13)
    pages, rows, width = 20000, 1024, 16
    refs = (rng.random(pages) < 0.8).astype(np.int32)
    table, lens = np.full((rows, width), -1, np.int32), rng.integers(0, 2, rows).astype(np.int32) * 5
    used = np.flatnonzero(refs)[:rows]
    table[lens > 0, 0] = used[lens > 0]
    st = {"k": np.zeros((1, pages, 1, 16, 128), np.float32), "v": np.zeros((1, pages, 1, 16, 128), np.float32), "table": table, "lens": lens, "refs": refs}
    cache = _cache(st)
    tokens = np.full(rows, 30)
    assert int(cache.extend(_i32(tokens))) == R.extend(st, tokens) == 0   # some 2000 pages
    parents = rng.integers(0, rows, rows)
    parents[::3] = np.flatnonzero(lens)[0]
    assert int(cache.fork(_i32(parents))) == R.fork(st, parents) == 0
    for name in ("table", "lens", "refs"):
        assert np.array_equal(getattr(cache, name).cpu().numpy(), st[name]), name


def _check_beams(logits, scores, k, done=None, eos=-1, exact_ids=True):
    got = beam_select(torch.from_numpy(logits).to(DEV), torch.from_numpy(scores).to(DEV), k, None if done is None else _i32(done), eos)
    s, rows, tokens = (x.cpu().numpy() for x in got)
    want = R.beam_candidates(logits, scores, done, eos, k)
    for g, cand in enumerate(want):
        cand = cand[:k] + [(-np.inf, -1, -1)] * (k - len(cand))
        ref = np.array([c[0] for c in cand])
        fine = np.isfinite(ref)
        # a float32 rounding, and the log of a sum of float32 exponentials with 2^-21 each
        assert (np.abs(s[g][fine] - ref[fine]) <= 2.0 ** -24 * np.abs(ref[fine]) + 2.0 ** -20).all()
        assert np.array_equal(s[g][~fine], ref[~fine])
        same = (rows[g] == [c[1] for c in cand]) & (tokens[g] == [c[2] for c in cand])
        if exact_ids:
            assert same.all(), (g, cand, rows[g], tokens[g])
        else:   # candidates of different beams whose scores are nearer than the sums' error may change places
            pick = {(c[1], c[2]): c[0] for c in want[g]}
            for i in np.flatnonzero(~same):
                assert abs(pick[(rows[g][i], tokens[g][i])] - ref[i]) <= 2.0 ** -19
    return s, rows, tokens


@pytest.mark.parametrize("vocab", [1, 5, 999, 8192, 8193, 32001, 50000, 262145])
@pytest.mark.parametrize("groups,beams,k", [(1, 1, 1), (3, 4, 8), (2, 33, 40)])
def test_beam_selection(groups, beams, k, vocab):
    if vocab * groups * beams > 4 << 20:
        groups, beams = 1, 8
    rng = np.random.default_rng(vocab + k)
    logits = (3.0 * rng.standard_normal((groups, beams, vocab))).astype(np.float32)
    scores = -10.0 * rng.random((groups, beams)).astype(np.float32)
    _check_beams(logits, scores, min(k, vocab), exact_ids=False)
    done = (rng.random((groups, beams)) < 0.3).astype(np.int32)
    _check_beams(logits, scores, min(k, vocab), done, eos=7, exact_ids=False)


def test_the_largest_selections():
    """128 beams, 128 candidates, a million tokens: the merge's lists do not fit shared memory, or not all at once."""
    rng = np.random.default_rng(20)
    for groups, beams, vocab, k in ((1, 128, 20000, 64), (1, 2, 1 << 20, 128), (1, 64, 1 << 17, 128), (1, 64, 600000, 128), (2, 40, 3000, 3)):
        logits = rng.standard_normal((groups, beams, vocab), dtype=np.float32) * 2
        _check_beams(logits, -rng.random((groups, beams), dtype=np.float32), k, exact_ids=False)


def test_rows_with_few_live_tokens():
    """A vocabulary of which most is masked out: more than a list's worth of equal minus infinities, with and without enough others."""
    rng = np.random.default_rng(21)
    for live in (0, 3, 40, 3000):
        logits = np.full((2, 2, 30000), -np.inf, np.float32)
        at = rng.permutation(30000)[:live]
        logits[:, :, at] = rng.standard_normal((2, 2, live)).astype(np.float32)
        _check_beams(logits, np.array([[0.0, -1.0], [-2.0, 0.0]], np.float32), 20)


@pytest.mark.parametrize("k", [1, 16, 64, 128])
@pytest.mark.parametrize("masked", [float("-inf"), float(torch.finfo(torch.float32).min), -1e4])
def test_rows_that_a_mask_has_left_little_of(masked, k):
    """One value for what is masked: with few others, with others in every slice; slices that begin with something below it or a NaN; its
    count around a list's length; all of a slice's first tokens live, which fill the selection or not."""
    rng = np.random.default_rng(22)
    logits = np.full((4, 2, 20003), masked, np.float32)
    logits[0, 0, rng.permutation(20003)[:5]] = 1.0
    at = rng.permutation(20003)[:700]
    logits[0, 1, at] = rng.standard_normal(700).astype(np.float32)
    below = -np.inf if masked > -np.inf else np.nan
    logits[1, 0, [0, 1, 8192, 8300, 16384]] = below
    logits[1, 0, 9000:9003] = 2.0
    logits[1, 1, :200] = below
    logits[1, 1, 300:] = below
    logits[2, 0, 1030:8192] = below
    logits[2, 0, 8192 + 1020:] = below
    logits[2, 1] = rng.standard_normal(20003).astype(np.float32)
    logits[2, 1, ::2] = masked
    logits[3, 0, :100] = rng.standard_normal(100).astype(np.float32)
    logits[3, 1, 60:8192] = 3.0
    _check_beams(logits, -rng.random((4, 2)).astype(np.float32), k, exact_ids=False)


@pytest.mark.parametrize("k", [1, 7, 33, 128])
def test_the_best_all_in_one_thread(k):
    """A slice whose largest logits a single thread holds, one whose first tokens are the largest, in rising and falling order."""
    rng = np.random.default_rng(23)
    logits = rng.standard_normal((2, 2, 8192 + 900)).astype(np.float32)
    mine = (np.arange(8)[:, None] * 1024 + 4 * 37 + np.arange(4)).ravel()
    logits[0, 0, mine] += 20.0
    logits[0, 1, mine[:9]] = 20.0
    logits[1, 0] = np.sort(logits[1, 0])[::-1]
    logits[1, 1] = np.sort(logits[1, 1])
    _check_beams(logits, -rng.random((2, 2)).astype(np.float32), k, exact_ids=False)


def test_equal_candidates_go_to_the_lower_beam_and_token():
    """Equal beams on rows of every alignment, equal logits, a row of one value, more equal logits than a thread holds."""
    for vocab in (997, 1000, 20001):
        row = np.round(np.random.default_rng(vocab).standard_normal(vocab) * 2).astype(np.float32)
        logits = np.stack([row] * 6).reshape(2, 3, vocab)
        _check_beams(logits, np.zeros((2, 3), np.float32), 16)
        _check_beams(np.zeros((1, 2, vocab), np.float32), np.zeros((1, 2), np.float32), 128)
    logits = np.full((1, 1, 40000), -1.0, np.float32)
    logits[0, 0, 5::3] = 2.0
    _check_beams(logits, np.zeros((1, 1), np.float32), 128)
    logits[0, 0, ::2] = np.float32(-0.0)
    logits[0, 0, 1::2] = 0.0
    _check_beams(logits, np.zeros((1, 1), np.float32), 100)


def test_infinities_and_nan_in_a_selection():
    rng = np.random.default_rng(14)
    logits = rng.standard_normal((4, 3, 9001)).astype(np.float32)
    logits[0, 0, 8500] = np.nan
    logits[0, 1, 3] = np.inf
    logits[1, 0] = -np.inf
    logits[1, 1, 100:] = -np.inf
    logits[2] = np.nan
    logits[3, :, :8192] = -np.inf
    logits[3, 1, 5] = np.nan
    scores = np.zeros((4, 3), np.float32)
    scores[3, 2] = -np.inf
    _check_beams(logits, scores, 12)
    first = np.array([[0.0, -np.inf, -np.inf]] * 4, np.float32)   # the first step of a search: one live beam
    _check_beams(rng.standard_normal((4, 3, 500)).astype(np.float32), first, 6)


def test_beams_that_are_done():
    rng = np.random.default_rng(15)
    logits, scores = rng.standard_normal((2, 4, 100)).astype(np.float32), -rng.random((2, 4)).astype(np.float32)
    done = np.array([[1, 1, 1, 1], [0, 1, 0, 0]], np.int32)
    logits[done > 0] = np.nan   # is not read
    s, rows, tokens = _check_beams(logits, scores, 8, done, eos=42)
    assert (rows[0, 4:] == -1).all() and (tokens[0, :4] == 42).all()


def test_a_draft_then_beams_on_one_cache():
    """As a program uses them: a prompt's keys are written node by node as a chain, a tree is drafted and attended, the accepted branch
    stays, the sequence is forked into beams, and every beam attends its next token."""
    rng = np.random.default_rng(16)
    hq, hk, page = 8, 2, 16
    cache = PagedCache.empty(layers=2, kv_heads=hk, page=page, pages=40, rows=4, width=8)
    st = {n: getattr(cache, n).float().cpu().numpy() if n in "kv" else getattr(cache, n).cpu().numpy() for n in ("k", "v", "table", "lens", "refs")}
    freqs = rope_frequencies(device=DEV)

    def forward(parents, layer):
        qkv = rng.standard_normal((4, parents.shape[1], (hq + 2 * hk) * 128)).astype(np.float32)
        masks, depths = tree_masks(_i32(parents))
        q = cache.write(layer, torch.from_numpy(qkv).to(DEV), depths, freqs)
        want_masks, want_depths = R.masks_depths(parents)
        R.write(st, layer, qkv, want_depths, freqs.cpu().numpy(), hq)
        used = np.array([int(m).bit_count() > 0 for m in want_masks[:, 0]])
        st["k"], st["v"] = (getattr(cache, n).float().cpu().numpy() for n in "kv")   # one rounding apart, checked above
        got = cache.attend(layer, q, masks).float().cpu().numpy()
        want, weight = R.attend(st, layer, q.float().cpu().numpy(), want_masks, 128 ** -0.5)
        assert (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + (2.0 ** -7 + 2.0 ** -12) * weight).all()
        assert not got[~used].any()

    prompt = np.array([np.arange(21) - 1] + [np.full(21, -2)] * 3)   # sequence 0 alone
    assert int(cache.extend(_i32([40, 0, 0, 0]))) == R.extend(st, [40, 0, 0, 0]) == 0
    for layer in (0, 1):
        forward(prompt, layer)
    ids = np.arange(84).reshape(4, 21)
    targets = np.roll(ids, -1, axis=1)
    count, token, _, _ = cache.accept(_i32(ids), _i32(prompt), _i32(targets), lens_out=cache.lens)
    assert count.tolist() == [21, 0, 0, 0] and token.tolist() == [0, -1, -1, -1]
    st["lens"][:] = R.accept(st, ids, prompt, targets)[3]
    tree = np.array([[-1, 0, 0, 1, 2, 2, 5]] + [[-2] * 7] * 3)
    for layer in (0, 1):
        forward(tree, layer)
    ids = np.array([[0, 1, 2, 3, 4, 5, 6]] * 4)
    targets = np.array([[2, 0, 5, 0, 0, 6, 9]] * 4)
    _, token, path, _ = cache.accept(_i32(ids), _i32(tree), _i32(targets), lens_out=cache.lens)
    assert path[0].tolist() == [0, 2, 5, 6, -1, -1, -1] and int(token[0]) == 9
    st["lens"][:] = R.accept(st, ids, tree, targets)[3]
    assert int(cache.fork(_i32([0, 0, 0, 0]))) == R.fork(st, [0, 0, 0, 0]) == 0
    _same_cache(cache, st)
    logits = rng.standard_normal((1, 4, 1000)).astype(np.float32)
    _, rows, _ = beam_select(torch.from_numpy(logits).to(DEV), torch.tensor([[0.0, -1.0, -2.0, -1.5]], device=DEV), 4)
    assert int(cache.extend(1)) == R.extend(st, [1] * 4) == 0
    for layer in (0, 1):
        forward(np.full((4, 1), -1), layer)
    cache.lens += 1
    st["lens"] += 1
    assert int(cache.fork(rows[0])) == R.fork(st, rows[0].cpu().numpy()) == 0
    _same_cache(cache, st)


def test_a_captured_step_replays():
    """Reserve, write, attend, select and fork in one graph, replayed: the lengths and tables it meets differ from replay to replay."""
    rng = np.random.default_rng(17)
    hq, hk = 4, 2

    def make():
        c = PagedCache.empty(layers=1, kv_heads=hk, page=16, pages=64, rows=4, width=8)
        c.fork(torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=DEV))
        return c

    qkv, logits = torch.zeros(4, 1, (hq + 2 * hk) * 128, device=DEV), torch.zeros(1, 4, 500, device=DEV)
    scores, freqs = torch.zeros(1, 4, device=DEV), rope_frequencies(device=DEV)
    parents = torch.full((4, 1), -1, dtype=torch.int32, device=DEV)

    def step(c):
        lack = c.extend(torch.ones(4, dtype=torch.int32, device=DEV))
        masks, depths = tree_masks(parents)
        out = c.attend(0, c.write(0, qkv, depths, freqs), masks)
        c.lens.add_(1)
        s, rows, tokens = beam_select(logits, scores, 4)
        return lack, c.fork(rows[0]), out, s, rows, tokens

    a, b = make(), make()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step(make())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(b)
    for _ in range(40):
        qkv.copy_(torch.from_numpy(rng.standard_normal(qkv.shape).astype(np.float32)))
        logits.copy_(torch.from_numpy(3 * rng.standard_normal(logits.shape).astype(np.float32)))
        want = step(a)
        graph.replay()
        for x, y in zip(want, outs):
            assert torch.equal(x, y)
        assert int(want[0]) == 0 and int(want[1]) == 0
        assert torch.equal(a.table, b.table) and torch.equal(a.lens, b.lens) and torch.equal(a.k, b.k)


def test_refused_tensors():
    cache = PagedCache.empty(layers=1, kv_heads=2, page=16, pages=4, rows=2, width=2)
    q, m = torch.zeros(2, 1, 4, 128, dtype=torch.bfloat16, device=DEV), torch.ones(2, 1, dtype=torch.int64, device=DEV)
    for bad_q, bad_m in ((q.float(), m), (q[:1], m), (q, m.int()), (q.cpu(), m), (q, m.cpu())):
        with pytest.raises(ValueError):
            cache.attend(0, bad_q, bad_m)
    with pytest.raises(RuntimeError, match="layer"):
        cache.attend(1, q, m)
    with pytest.raises(RuntimeError, match="query heads"):
        cache.attend(0, q[:, :, :3].contiguous(), m)
    with pytest.raises(ValueError, match="contiguous"):
        cache.attend(0, q, m, out=torch.empty(2, 1, 128, 4, dtype=torch.bfloat16, device=DEV).transpose(2, 3))
    with pytest.raises(ValueError, match="table"):
        PagedCache(cache.k, cache.v, cache.table.long(), cache.lens, cache.refs)
    with pytest.raises(RuntimeError, match="power of two"):
        PagedCache.empty(layers=1, kv_heads=2, page=24, pages=4, rows=2, width=2)
    # strides of other orders are taken
    wide = torch.randn(2, 1, 8, 128, device=DEV).to(torch.bfloat16)
    cache.lens.fill_(0)
    assert int(cache.extend(1)) == 0
    assert torch.equal(cache.attend(0, wide[:, :, ::2], m), cache.attend(0, wide[:, :, ::2].contiguous(), m))
