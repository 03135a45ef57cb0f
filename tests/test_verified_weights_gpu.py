"""Trees of drafted tokens over a cache whose weights are added up: the branch that is kept takes its weights along, and an eviction
goes by them."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import long_reference as L  # noqa: E402
import paged_reference as R  # noqa: E402
from test_long_context_gpu import _bf, _cache, _gpu, _i32, _masks, _random_trees, _round_state  # noqa: E402
from test_paged_decoder_gpu import CFG, _decoder, _prompt  # noqa: E402
from test_paged_decoder_gpu import _cache as _empty_cache  # noqa: E402

DEV = "cuda:0"


def _moved(st, weights, path, lens):
    """weights after the branches `path` of trees behind `lens`, as accept leaves them."""
    out, cap = weights.copy(), weights.shape[3]
    for r, branch in enumerate(path):
        for i, b in enumerate(x for x in branch if x >= 0):
            if lens[r] + b < cap:
                out[:, r, :, lens[r] + i] = weights[:, r, :, lens[r] + b]
    return out


@pytest.mark.parametrize("rows,nodes,heads,layers", [(1, 1, 1, 1), (1, 9, 3, 40), (5, 12, 2, 3), (3, 64, 8, 2), (40, 7, 4, 1)])
def test_an_accepted_branch_takes_its_weights_along(rows, nodes, heads, layers):
    """Keys, values, lengths and outputs are those of the call without weights; all other weights stay; ends of tables, pages that are not there."""
    rng = np.random.default_rng(rows * nodes)
    lens = [int(x) for x in rng.integers(0, 60, rows)]
    if rows > 2:
        lens[2] = 128 - nodes // 2   # the tree runs over the end of the table
    st = _round_state(R.state(rng, [min(n, 128 - nodes) for n in lens], extra=nodes, page=16, kv_heads=heads, layers=layers, width=8))
    st["lens"][:] = lens
    if rows > 3:
        st["table"][3, lens[3] // 16] = -1
        st["table"][4, (lens[4] + nodes) // 16] = 10 ** 6
    parents = _random_trees(rng, rows, nodes)
    ids, targets = rng.integers(0, 3, (rows, nodes)), rng.integers(0, 3, (rows, nodes))
    if nodes == 64:
        parents[0], ids[0], targets[0] = np.arange(64) - 1, 1, 1                 # all of a chain: nothing moves
        parents[1], ids[1], targets[1] = [-1] + [0] * 63, [2] * 63 + [1], 1      # the last of 63 children
    if rows > 4:
        parents[1, 0] = 5   # an unused row
    a, b = _cache(st), _cache(st)
    before = rng.standard_normal(tuple(a.new_weights().shape)).astype(np.float32)
    w = _gpu(before)
    plain = a.accept(_i32(ids), _i32(parents), _i32(targets))
    got = b.accept(_i32(ids), _i32(parents), _i32(targets), weights=w)
    for x, y in zip(plain, got):
        assert torch.equal(x, y)
    assert torch.equal(a.k.view(torch.int16), b.k.view(torch.int16)) and torch.equal(a.v.view(torch.int16), b.v.view(torch.int16))
    want = _moved(st, before, got[2].tolist(), lens)
    assert np.array_equal(w.cpu().numpy(), want)
    assert rows == 1 or not np.array_equal(want, before)
    c, again = _cache(st), _gpu(before)
    c.accept(_i32(ids), _i32(parents), _i32(targets), lens_out=c.lens, weights=again)   # lengths in place
    assert torch.equal(again, w) and torch.equal(c.lens, got[3])


def test_a_branch_and_its_weights_in_a_graph():
    rng = np.random.default_rng(5)
    st = _round_state(R.state(rng, [20, 3], extra=16, page=16, kv_heads=2, layers=2))
    cache = _cache(st)
    before = rng.standard_normal(tuple(cache.new_weights().shape)).astype(np.float32)
    w = _gpu(before)
    parents = np.array([[-1, 0, 0, 1, 2, 2, 4, 3], [-1, 0, 1, 1, 0, 4, 5, 2]])
    ids, targets = _i32(np.ones((2, 8))), _i32(np.zeros((2, 8)))
    parents = _i32(parents)
    cache.accept(ids, parents, targets, weights=w)   # nothing agrees
    assert torch.equal(w, _gpu(before))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.accept(ids, parents, targets, weights=w)
    ids[0, 1] = ids[0, 4] = 0
    targets.copy_(_i32([[1, 0, 0, 0, 1, 0, 0, 0], [1, 0, 0, 0, 0, 0, 0, 0]]))
    graph.replay()
    torch.cuda.synchronize()
    assert out[0].tolist()[0] > 1
    assert np.array_equal(w.cpu().numpy(), _moved(st, before, out[2].tolist(), [20, 3]))


def test_a_verified_tree_then_its_branch_then_an_eviction():
    """A decoder verifies a tree that is partly rejected, twice, and the cache is cut: positions of the branch go by what its own nodes were given."""
    rows, nodes = 2, 9
    rng = np.random.default_rng(1)
    prompt = _i32(rng.integers(0, 1000, (rows, 21)))
    dec, cache = _decoder(rows * 32), _empty_cache(rows)
    weights, dropped = cache.new_weights(), torch.zeros(rows, dtype=torch.int32, device=DEV)
    dec.set_cache(cache, weights=weights, dropped=dropped)
    _prompt(dec, cache, prompt)
    parents = [[-1, 0, 0, 1, 2, 2, 4, 3, 6], [-1, 0, 1, 1, 0, 4, 5, 2, 7]]
    branches = [0, 2, 4, 6, 8], [0, 1, 2, 7, 8]
    group = CFG["n_q_heads"] // CFG["n_kv_heads"]
    for step in range(2):
        lens = cache.lens.tolist()
        ids = rng.integers(0, 1000, (rows, nodes))
        assert int(cache.extend(nodes)) == 0
        dec.verify(_i32(ids), _i32(parents))
        seen = weights.cpu().numpy().copy()
        for r in range(rows):   # the root is seen by all nodes, a leaf by itself alone
            assert (seen[:, r, :, lens[r]] > seen[:, r, :, lens[r] + 5]).all()
        targets = np.full((rows, nodes), -1)
        for r, branch in enumerate(branches):
            for a, b in zip(branch, branch[1:]):
                targets[r, a] = ids[r][b]
        count, _, path, _ = cache.accept(_i32(ids), _i32(parents), _i32(targets), lens_out=cache.lens, weights=weights)
        assert count.tolist() == [5, 5] and path[0, :5].tolist() == branches[0]
        got = weights.cpu().numpy()
        for r in range(rows):
            assert np.array_equal(got[:, r, :, lens[r]:lens[r] + 5], seen[:, r][:, :, [lens[r] + b for b in branches[r]]])
            assert np.array_equal(got[:, r, :, :lens[r]], seen[:, r, :, :lens[r]])
    st = {n: getattr(cache, n).float().cpu().numpy() if n in "kv" else getattr(cache, n).cpu().numpy().copy() for n in ("k", "v", "table", "lens", "refs")}
    host = weights.cpu().numpy().copy()
    gone, status = cache.evict(weights, 24, recent=3)
    want, lack = L.evict(st, host, [24, 24], 3)
    assert int(status) == lack == 0 and gone.tolist() == want.tolist() == [7, 7]
    assert np.array_equal(weights.cpu().numpy(), host) and np.array_equal(cache.k.float().cpu().numpy(), st["k"])
    dropped += gone
    assert int(cache.extend(1)) == 0
    total = weights[:, :, :, :24].double().sum(-1)
    dec.step(_i32([5, 6]))
    assert ((weights[:, :, :, :25].double().sum(-1) - total - group).abs() <= 1e-4 * (total + group)).all()
    dec.free()


def test_weights_that_are_refused():
    st = R.state(np.random.default_rng(0), [20, 30], extra=2, page=16, kv_heads=2)
    cache = _cache(st)
    x = _i32(np.zeros((2, 2)))
    w = cache.new_weights()
    for bad in (w[:, :1], w.double(), w.cpu(), w[..., :-1], w.transpose(0, 1)):
        with pytest.raises(ValueError, match="weights"):
            cache.accept(x, x, x, weights=bad)
