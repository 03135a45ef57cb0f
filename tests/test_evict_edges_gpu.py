"""Evictions whose free slots or moving rows are more than a list holds: lists are filled again, in the middle of a step; keys in shared memory
and not, pages of which much stays but has to be copied, more rows kept as the latest than go."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import paged_reference as R  # noqa: E402
from test_long_context_gpu import _check_evict, _round_state, _share, _weights  # noqa: E402


def _light_first(rng, st, w):
    """Nearly all that stays lies behind the new length."""
    n = int(st["lens"][0])
    w[:, 0, :, :n // 2] *= 1e-6
    w[:, 0, :, n // 2:n] += 1.0
    return w


@pytest.mark.parametrize("kind", ["spread", "ties", "light_first"])
@pytest.mark.parametrize("width", [None, 50])
def test_lists_that_are_filled_again(width, kind):
    """12000 positions cut to 6000: some 3000 free slots below the new length, nearly 6000 in the last case."""
    rng = np.random.default_rng(11)
    page = 64 if width is None else 1024   # 51200 positions: keys do not fit shared memory
    for keep, recent in ((6000, 0), (6000, 5), (5000, 2100)):
        st = _round_state(R.state(rng, [12000, 10], page=page, kv_heads=1, width=width))
        w = _weights(rng, st, "spread" if kind == "light_first" else kind)
        _check_evict(st, _light_first(rng, st, w) if kind == "light_first" else w, keep, recent)


@pytest.mark.parametrize("n,keep", [(4097, 2049), (8192, 4096), (8191, 2050)])
def test_lists_that_are_just_full(n, keep):
    """2048 and one more; holes and movers in alternate slots, and all of a step."""
    rng = np.random.default_rng(n)
    for pattern in ("alternate", "late"):
        st = _round_state(R.state(rng, [n], page=64, kv_heads=2))
        w = rng.random((1, 1, 2, st["table"].shape[1] * 64)).astype(np.float32)
        if pattern == "alternate":
            w[..., 1::2] += 10.0
        else:
            w[..., n - keep:] += 10.0
        _check_evict(st, w, keep, 0)


def test_shared_pages_with_more_kept_slots_than_a_list_holds():
    rng = np.random.default_rng(4)
    st = _round_state(R.state(rng, [7000, 7000], page=64, kv_heads=1, spare=220))
    _share(rng, st, [(0, 1, 100)])
    w = _weights(rng, st)
    w[..., :5000] += 100.0   # what is heavy lies on the shared pages
    _check_evict(st, w, [5500, 4700], 64)


@pytest.mark.parametrize("n,keep,recent", [(1000, 999, 999), (1000, 999, 512), (1000, 990, 500), (3000, 2999, 2999), (700, 650, 60), (2049, 2048, 64), (2049, 2048, 2000)])
def test_fewer_go_than_are_kept_as_the_latest(n, keep, recent):
    """A budget that is kept token by token; a window of the latest alone."""
    rng = np.random.default_rng(n + recent)
    st = _round_state(R.state(rng, [n, n - 300, 5], page=16, kv_heads=2, layers=2))
    _share(rng, st, [(0, 1, 3)])
    _check_evict(st, _weights(rng, st), [keep, keep - 300, 5], recent)
