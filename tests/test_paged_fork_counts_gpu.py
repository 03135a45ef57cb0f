"""Counts of pages at the edges of what the contract allows: a count of 0 or less is a free page, whatever it is."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import paged_reference as R  # noqa: E402
from test_paged_cache_gpu import DEV, _cache, _i32, _round_state  # noqa: E402


@pytest.mark.parametrize("spare", [3, 9000])   # plans in shared memory, and beside the pool
@pytest.mark.parametrize("free", [-1, -7, -(1 << 31)])
def test_a_page_that_a_fork_gives_out_is_counted_once(free, spare):
    """Free pages with negative counts: the page of a copy is held by one entry and not given out again."""
    st = _round_state(R.state(np.random.default_rng(1), [20, 5, 0], page=16, kv_heads=1, width=4, spare=spare, shuffle=False))
    st["refs"][3:] = free   # pages 0 and 1 are the first sequence's, 2 the second's
    cache = _cache(st)
    assert int(cache.fork(_i32([0, 0, 0]))) == 0
    # the second sequence's page goes back and is the lowest free one
    assert cache.table.tolist() == [[0, 1, -1, -1], [0, 2, -1, -1], [0, 3, -1, -1]]
    assert cache.refs[:4].tolist() == [3, 1, 1, 1] and (cache.refs[4:] == free).all()
    for p in (2, 3):
        assert torch.equal(cache.k[:, p, :, :4], cache.k[:, 1, :, :4]) and torch.equal(cache.v[:, p, :, :4], cache.v[:, 1, :, :4])
    assert int(cache.extend(_i32([13, 0, 0]))) == 0   # the next page is another one
    assert cache.table[0].tolist() == [0, 1, 4, -1] and cache.refs[:5].tolist() == [3, 1, 1, 1, 1]
    assert int(cache.fork(_i32([0, 1, -1]))) == 0     # and what is given back can be given out again
    assert cache.table.tolist() == [[0, 1, -1, -1], [0, 2, -1, -1], [-1] * 4] and cache.refs[:5].tolist() == [2, 1, 1, 0, 0]
    assert cache.lens.tolist() == [20, 20, 0] and cache.table.device == torch.device(DEV)
