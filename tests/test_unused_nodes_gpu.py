"""Trees of different sizes in one pass of a decoder that adds up weights: nodes that are not there, and sequences without a tree, add nothing.
Probabilities of a query sum to one; two passes over the same tokens agree within 1e-2 as in test_paged_decoder_gpu."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_nint_gpu import rel_l2  # noqa: E402
from test_paged_decoder_gpu import CFG, _cache, _decoder, _i32, _prompt  # noqa: E402
from tyloquant_b200 import PagedCache  # noqa: E402

DEV = "cuda:0"


def _clone(cache):
    return PagedCache(*(getattr(cache, n).clone() for n in ("k", "v", "table", "lens", "refs")))


@pytest.mark.parametrize("width", [10, 40])
@pytest.mark.parametrize("nodes", [5, 20, 40, 64])
def test_unused_nodes_add_nothing(nodes, width):
    """Sums by the attention itself, beside its merge, and from the keys; short tables and split ones."""
    rows, n, group = 4, 45, CFG["n_q_heads"] // CFG["n_kv_heads"]
    rng = np.random.default_rng(nodes)
    dec, cache = _decoder(rows * 64), _cache(rows, pages=120, width=width)
    dec.set_cache(cache)
    _prompt(dec, cache, _i32(rng.integers(0, 1000, (rows, n))))
    some = max(2, nodes // 3)
    parents = np.array([[-1] + [int(rng.integers(max(0, i - 4), i)) for i in range(1, nodes)] for _ in range(rows)])
    parents[1, some:] = -1                                # as many as fit its tree; what follows are no nodes
    parents[2, :] = -2                                    # no tree at all
    parents[3, 1] = 7                                     # a node that is none, and what hangs below it
    used = [nodes, some, 0]
    inside = {0}
    for i in range(2, nodes):
        if int(parents[3, i]) in inside:
            inside.add(i)
    used.append(len(inside))
    ids = _i32(rng.integers(0, 1000, (rows, nodes)))
    assert int(cache.extend(nodes)) == 0
    alone = _clone(cache)
    before = torch.rand(tuple(cache.new_weights().shape), generator=torch.Generator(DEV).manual_seed(1), device=DEV)
    weights = before.clone()
    dec.set_cache(cache, weights=weights)
    dec.verify(ids, _i32(parents))
    assert torch.equal(weights[:, 2, :, :n], before[:, 2, :, :n]) and not weights[:, 2, :, n:n + nodes].any()
    for r in range(rows):
        added = (weights[:, r, :, :n + nodes].double().sum(-1) - before[:, r, :, :n].double().sum(-1)).cpu().numpy()
        assert np.abs(added - group * used[r]).max() <= 1e-4 * (group * nodes + n), (r, added, used)
        assert torch.equal(weights[:, r, :, n + nodes:], before[:, r, :, n + nodes:])
    assert not weights[:, 1, :, n + some:n + nodes].any()
    # the second sequence's tree in a pass of its own size
    few = alone.new_weights()
    dec.set_cache(alone, weights=few)
    dec.verify(ids[:, :some].contiguous(), _i32(parents[:, :some]))
    got = weights[:, 1].double()
    got[..., :n] -= before[:, 1, :, :n].double()
    assert rel_l2(got[..., :n + some].cpu().numpy(), few[:, 1, :, :n + some].double().cpu().numpy()) <= 1e-2
    dec.free()


def test_steps_count_every_sequence():
    rows, group = 3, CFG["n_q_heads"] // CFG["n_kv_heads"]
    dec, cache = _decoder(8), _cache(rows)
    weights = cache.new_weights()
    dec.set_cache(cache, weights=weights)
    for i in range(5):
        assert int(cache.extend(1)) == 0
        dec.step(_i32([i, 7 + i, 100 + i]))
    assert (weights.double().sum(-1) - 5 * group).abs().max() <= 1e-4 * 5 * group
    dec.free()
