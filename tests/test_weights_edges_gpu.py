"""Sums of attention weights where the lanes of a warp differ: tiles of which some positions are context and others nodes, each seen by
other nodes; bounds as of test_long_context_gpu."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import paged_reference as R  # noqa: E402
import long_reference as L  # noqa: E402
from test_long_context_gpu import _bf, _cache, _check_weigh, _masks, _random_trees, _round_state  # noqa: E402


@pytest.mark.parametrize("hq", [3, 5, 16])
@pytest.mark.parametrize("context", [1, 97, 113, 127, 255, 257 + 30])
def test_tiles_in_which_every_position_is_seen_by_other_nodes(context, hq):
    """More than 64 rows: sums from the keys; up to 64 in a table of one item: sums by the attention's own warps, whose last positions are a part of a warp."""
    rng = np.random.default_rng(context * 20 + hq)
    for nodes, width in ((64, None), (23, None), (3, 16)):
        if width is not None and context + nodes > width * 16:
            continue
        st = _round_state(R.state(rng, [context, 5], extra=nodes, page=16, kv_heads=1, width=width))
        masks, _ = R.masks_depths(_random_trees(rng, 2, nodes))
        masks |= np.uint64(1) << rng.integers(0, nodes, masks.shape).astype(np.uint64)   # not trees alone: any node
        first = _check_weigh(rng, st, rng.standard_normal((2, nodes, hq, 128)), masks, calls=2)
        assert first.shape[3] == st["table"].shape[1] * 16


@pytest.mark.parametrize("nodes", [1, 4, 16, 17, 40, 64])
@pytest.mark.parametrize("width", [8, 30])
def test_weights_of_large_scores(nodes, width):
    """Scores near 1000 that are whole numbers, so that float32 holds each exactly, in units 2^-4.  An exponent is off by its rounding, 2^-21 below 2^4, the unit by
    2^-22, the sum of n terms by n 2^-24, that over the rows likewise.  From the keys (more than 64 rows) a row's maximum and sum are one float32 of 2^10 to
    2^11, which is off by 2^-14: a weight by ln 2 times that, where scores of that size that are no whole numbers are off by as much themselves."""
    rng = np.random.default_rng(nodes)
    hq, context, scale = 4, 40, 2.0 ** -4
    st = R.state(rng, [context, 17], extra=nodes, page=16, kv_heads=1, width=width)
    real = ~np.isnan(st["k"])
    st["k"] = np.where(real, 125.0 + rng.integers(-1, 2, st["k"].shape), np.nan).astype(np.float32)
    st = _round_state(st)
    masks, _ = R.masks_depths(_random_trees(rng, 2, nodes))
    q = np.ones((2, nodes, hq, 128), np.float32)
    q[..., :20] += rng.integers(-1, 2, (2, nodes, hq, 20))
    cache = _cache(st)
    w = cache.new_weights()
    cache.attend(0, _bf(q).to("cuda:0"), _masks(masks), scale=scale, weights=w)
    want, size = L.weigh(st, 0, q, masks, scale, np.zeros(tuple(w.shape), np.float32))
    assert 700 < scale * size.max() < 1400
    rel = 2.0 ** -20 + (context + nodes + nodes * hq) * 2.0 ** -24 + (np.log(2) * 2.0 ** -14 if nodes * hq > 64 else 0.0)
    got = w.cpu().numpy()
    assert (np.abs(got - want) <= rel * want).all(), (np.abs(got - want) / np.maximum(want, 1e-30)).max() / rel
