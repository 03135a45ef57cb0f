"""Pools of more than 2^31 values and 2^32 bytes each of keys and values, with the sequences on their last pages: element offsets that
32 bits do not hold.  (Offsets in pieces of 16 bytes would need pools of 2^34 values each: not reached here.)"""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import paged_reference as R  # noqa: E402
from test_paged_cache_gpu import DEV, _check_attend, _i32, _random_trees  # noqa: E402
from tyloquant_b200 import PagedCache, rope_frequencies  # noqa: E402


def _pools(*shape):
    k = torch.zeros(*shape, 128, dtype=torch.bfloat16, device=DEV)
    assert k.numel() > 1 << 31 and 2 * k.numel() > 1 << 32
    return k, torch.zeros_like(k)


def test_attention_at_the_end_of_a_large_pool():
    pages, page, hk = 9000, 512, 4
    k, v = _pools(1, pages, hk, page)
    g = torch.Generator(DEV).manual_seed(1)
    ids = [pages - 1, 1, pages - 2]
    for p in ids:
        k[0, p] = torch.randn(hk, page, 128, generator=g, device=DEV)
        v[0, p] = torch.randn(hk, page, 128, generator=g, device=DEV)
    v[0, pages - 2, :, 1302 - 1024, 7] = np.inf   # of a node: added by the row that sees it, from the pool
    small = {"k": k[:, ids].float().cpu().numpy(), "v": v[:, ids].float().cpu().numpy(), "table": np.array([[0, 1, 2]], np.int32), "lens": np.array([1300], np.int32)}
    cache = PagedCache(k, v, _i32([ids]), _i32([1300]), torch.ones(pages, dtype=torch.int32, device=DEV))
    rng = np.random.default_rng(12)
    parents = np.array([[-1, 0, 0, 1]])
    masks, _ = R.masks_depths(parents)
    _check_attend(small, rng.standard_normal((1, 4, 8, 128)), masks, cache=cache)
    masks, _ = R.masks_depths(_random_trees(rng, 1, 40))
    small["v"][:] = v[:, ids].float().cpu().numpy()
    _check_attend(small, rng.standard_normal((1, 40, 16, 128)), masks, cache=cache)


def test_writes_branches_and_forks_at_the_end_of_a_large_pool():
    layers, pages, page, hk, hq = 2, 18000, 256, 2, 4
    k, v = _pools(layers, pages, hk, page)
    last = pages - 1
    refs = torch.ones(pages, dtype=torch.int32, device=DEV)
    refs[last - 1] = 0
    cache = PagedCache(k, v, _i32([[last, -1], [-1, -1]]), _i32([10, 0]), refs)
    rng = np.random.default_rng(40)
    small = {"k": np.zeros((layers, 2, hk, page, 128), np.float32), "v": np.zeros((layers, 2, hk, page, 128), np.float32), "table": np.array([[1, -1], [-1, -1]], np.int32),
             "lens": np.array([10, 0], np.int32), "refs": np.array([0, 1], np.int32)}
    depths, freqs = np.array([[0, 1, 1, 2, 2]] * 2), rope_frequencies(device=DEV)
    for layer in range(layers):
        qkv = rng.standard_normal((2, 5, (hq + 2 * hk) * 128)).astype(np.float32)
        cache.write(layer, torch.from_numpy(qkv).to(DEV), _i32(depths), freqs)
        R.write(small, layer, qkv, depths, freqs.cpu().numpy(), hq)
    two = lambda pool: pool[:, last - 1:].float().cpu().numpy()   # the last two pages
    for got, want in ((two(k), small["k"]), (two(v), small["v"])):
        # half a bf16 step, and float32 products of values below 6: 2^-20 of them
        assert (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 12 * 2.0 ** -20).all() and got[1, 1, :, 10:15].any()
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
