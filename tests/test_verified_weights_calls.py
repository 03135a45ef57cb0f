"""Calls that keep a branch with its weights and are refused on the host (no GPU needed)."""

import ctypes as C

import pytest

pytest.importorskip("torch")

from test_paged_cache import A, _says, _view  # noqa: E402
from tyloquant_b200._capi import lib  # noqa: E402


def test_accepting_with_weights_refuses():
    v = C.byref(_view())

    def call(view=v, nodes=2, weights=A, **null):
        names = ("ids", "parents", "targets", "count", "token", "path", "lens_out")
        p = [None if null.get(n) else A for n in names]
        return lib.mfqb_tree_accept_weigh(view, p[0], p[1], p[2], nodes, *p[3:], weights, None)

    _says(1, "weights", call(weights=None))
    _says(1, "weights", call(weights=A + 2))
    for name in ("ids", "parents", "targets", "count", "token", "path", "lens_out"):
        _says(1, "mfqb_tree_accept_weigh: null", call(**{name: True}))
    for nodes in (0, 65):
        _says(3, "nodes", call(nodes=nodes))
    bad = _view(page=24)
    _says(3, "power of two", call(view=C.byref(bad)))
