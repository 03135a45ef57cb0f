"""Sums of attention weights where the lanes of a warp differ: tiles of which some positions are context and others nodes, each seen by
other nodes; bounds as of test_long_context_gpu."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import paged_reference as R  # noqa: E402
from test_long_context_gpu import _check_weigh, _random_trees, _round_state  # noqa: E402


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
