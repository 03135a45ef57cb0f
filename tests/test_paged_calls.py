"""Calls on a paged cache that are made right or refused on the host (no GPU needed)."""

import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from test_paged_cache import A, _says, _view  # noqa: E402
from tyloquant_b200._capi import lib  # noqa: E402


def test_outputs_over_inputs_are_refused():
    """Values of nodes that are no numbers are added after rows were written, with the queries read again."""
    v, n = C.byref(_view()), C.c_uint64()
    assert lib.mfqb_tree_attention_work(v, 4, 2, C.byref(n)) == 0
    size = 3 * 2 * 4 * 256   # q and out: 3 sequences, 2 nodes, 4 heads
    for out in (A, A + 16, A + size - 16, A - size + 16):
        _says(1, "overlap", lib.mfqb_tree_attention(v, 0, A, 4, 2, A + (1 << 24), 1.0, out, A + (1 << 25), n.value, None))
    x_size = 3 * 2 * (4 + 4) * 512   # qkv: 4 query heads, 2 + 2 of keys and values
    for out in (A, A + 16, A + x_size - 16, A - size + 16):
        _says(1, "overlap", lib.mfqb_cache_write(v, 0, A, 4, 2, A + (1 << 24), A + (1 << 25), out, None))
