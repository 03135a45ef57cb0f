"""What the entry points on a paged cache refuse before anything reaches a GPU, and the Python checks (no GPU needed)."""

import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import paged_reference as R  # noqa: E402
from tyloquant_b200 import PagedCache, _capi, beam_select, tree_masks  # noqa: E402
from tyloquant_b200._capi import CacheView, lib  # noqa: E402

A = 1 << 20   # stands for an aligned address; the calls below are refused before it is used


def _view(**over):
    f = dict(k=A, v=A, table=A, lens=A, refs=A, layers=2, kv_heads=2, page=16, pages=8, rows=3, width=4)
    f.update(over)
    return CacheView(*(f[n] for n, _ in CacheView._fields_))


def _says(code, text, got):
    assert got == code, lib.mfqb_last_error()
    assert text in lib.mfqb_last_error().decode()


BAD_VIEWS = [(dict(k=0), 1, "null pointer"), (dict(refs=0), 1, "null pointer"), (dict(k=A + 2), 1, "aligned"), (dict(page=24), 3, "power of two"),
             (dict(page=8), 3, "power of two"), (dict(page=2048), 3, "power of two"), (dict(rows=0), 3, "sequences"), (dict(rows=1025), 3, "sequences"),
             (dict(pages=0), 1, "positive"), (dict(layers=0), 1, "positive"), (dict(kv_heads=0), 1, "positive"), (dict(width=0), 3, "positions"),
             (dict(page=1024, width=(1 << 20) + 1), 3, "positions"), (dict(width=1 << 25, rows=64), 3, "positions")]


@pytest.mark.parametrize("over,code,text", BAD_VIEWS)
def test_views_that_are_refused(over, code, text):
    v, n = C.byref(_view(**over)), C.c_uint64()
    calls = [lib.mfqb_cache_extend(v, A, A, None), lib.mfqb_cache_fork_work(v, C.byref(n)), lib.mfqb_cache_fork(v, A, A, A, 1 << 40, None),
             lib.mfqb_cache_write(v, 0, A, 4, 1, A, A, A, None), lib.mfqb_tree_attention_work(v, 4, 1, C.byref(n)),
             lib.mfqb_tree_attention(v, 0, A, 4, 1, A, 1.0, A, A, 1 << 40, None), lib.mfqb_tree_accept(v, A, A, A, 1, A, A, A, A, None)]
    for got in calls:
        _says(code, text, got)


def test_arguments_that_are_refused():
    v, n = C.byref(_view()), C.c_uint64()
    _says(1, "null cache", lib.mfqb_cache_extend(None, A, A, None))
    _says(1, "null argument", lib.mfqb_cache_extend(v, None, A, None))
    assert lib.mfqb_cache_fork_work(v, C.byref(n)) == 0
    _says(1, "work must", lib.mfqb_cache_fork(v, A, A, A, n.value - 1, None))
    _says(1, "work must", lib.mfqb_cache_fork(v, A, A, A + 8, n.value, None))
    for nodes in (0, 65):
        _says(3, "nodes", lib.mfqb_cache_write(v, 0, A, 4, nodes, A, A, A, None))
        _says(3, "nodes", lib.mfqb_tree_attention(v, 0, A, 4, nodes, A, 1.0, A, A, 1 << 40, None))
        _says(3, "nodes", lib.mfqb_tree_accept(v, A, A, A, nodes, A, A, A, A, None))
        _says(3, "nodes", lib.mfqb_tree_masks(A, 3, nodes, A, A, None))
    _says(1, "do not fit", lib.mfqb_tree_attention(C.byref(_view(width=1)), 0, A, 4, 17, A, 1.0, A, A, 1 << 40, None))
    _says(3, "sequences", lib.mfqb_tree_masks(A, 1025, 4, A, A, None))
    for layer in (-1, 2):
        _says(1, "layer", lib.mfqb_cache_write(v, layer, A, 4, 1, A, A, A, None))
        _says(1, "layer", lib.mfqb_tree_attention(v, layer, A, 4, 1, A, 1.0, A, A, 1 << 40, None))
    for heads in (0, 3, 34):
        _says(3, "query heads", lib.mfqb_tree_attention(v, 0, A, heads, 1, A, 1.0, A, A, 1 << 40, None))
    _says(1, "aligned", lib.mfqb_tree_attention(v, 0, A + 2, 4, 1, A, 1.0, A, A, 1 << 40, None))
    _says(1, "aligned", lib.mfqb_cache_write(v, 0, A + 4, 4, 1, A, A, A, None))
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        _says(1, "scale", lib.mfqb_tree_attention(v, 0, A, 4, 1, A, scale, A, A, 1 << 40, None))
    _says(1, "aligned", lib.mfqb_tree_attention(v, 0, A, 4, 1, A + 4, 1.0, A, A, 1 << 40, None))
    _says(1, "aligned", lib.mfqb_cache_write(v, 0, A, 4, 1, A, A + 4, A, None))
    _says(1, "aligned", lib.mfqb_tree_masks(A, 3, 4, A + 4, A, None))
    assert lib.mfqb_tree_attention_work(v, 4, 1, C.byref(n)) == 0
    _says(1, "work must", lib.mfqb_tree_attention(v, 0, A, 4, 1, A, 1.0, A, A, n.value - 1, None))


def test_selections_that_are_refused():
    n = C.c_uint64()
    for groups, beams, vocab, k, code, text in ((0, 4, 100, 4, 3, "beams"), (1, 129, 100, 4, 3, "beams"), (1 << 10, 64, 100, 4, 3, "beams"), (1, 4, 0, 1, 3, "tokens"),
                                                (1, 4, (1 << 20) + 1, 1, 3, "tokens"), (1, 4, 100, 0, 1, "k must"), (1, 4, 1000, 129, 1, "k must"), (1, 4, 5, 6, 1, "k must"),
                                                (1, 100, 1000, 82, 3, "beams times k")):
        _says(code, text, lib.mfqb_beam_select_work(groups, beams, vocab, k, C.byref(n)))
        _says(code, text, lib.mfqb_beam_select(A, groups, beams, vocab, A, None, 0, k, A, A, A, A, 1 << 40, None))
    assert lib.mfqb_beam_select_work(2, 4, 100, 4, C.byref(n)) == 0
    _says(1, "work must", lib.mfqb_beam_select(A, 2, 4, 100, A, None, 0, 4, A, A, A, A, n.value - 1, None))
    _says(1, "null argument", lib.mfqb_beam_select(None, 2, 4, 100, A, None, 0, 4, A, A, A, A, n.value, None))


def test_python_checks():
    t = torch.zeros(2, 3, 2, 16, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="k must be"):
        PagedCache(t, t, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="parents must be"):
        tree_masks(torch.zeros(1, 1, dtype=torch.int32))
    with pytest.raises(ValueError, match="logits must be"):
        beam_select(torch.zeros(1, 1, 10), torch.zeros(1, 1), 1)
    assert _capi.CacheView.rows.offset == 56   # the C struct's layout


def test_the_restatements_agree_with_each_other():
    """A forked sequence attends like its parent did; an accepted branch like its nodes did."""
    rng = np.random.default_rng(0)
    st = R.state(rng, [21, 32, 0], extra=6, width=6, spare=6)
    q = rng.standard_normal((3, 6, 4, 128))
    parents = np.array([[-1, 0, 0, 1, 3, 2]] * 3)
    masks, depths = R.masks_depths(parents)
    assert masks[0].tolist() == [1, 3, 5, 11, 27, 37] and depths[0].tolist() == [0, 1, 1, 2, 3, 2]
    before, _ = R.attend(st, 0, q, masks, 0.1)
    ids, targets = np.arange(18).reshape(3, 6), np.full((3, 6), -7)
    targets[:, 0], targets[:, 1], targets[:, 3] = ids[:, 1], ids[:, 3], ids[:, 4]
    count, token, path, lens = R.accept(st, ids, parents, targets)
    assert count.tolist() == [4] * 3 and token.tolist() == [-7] * 3 and path[0].tolist() == [0, 1, 3, 4, -1, -1]
    st["lens"][:] = lens - 1
    last, _ = R.attend(st, 0, q[:, 4:5], np.ones((3, 1), np.uint64), 0.1)
    assert np.allclose(last[:, 0], before[:, 4])
    st["lens"][:] = lens
    assert R.fork(st, [0, 0, 1]) == 0
    assert (st["refs"] == np.bincount(st["table"][st["table"] >= 0], minlength=len(st["refs"]))).all()
    st["lens"] -= 1
    again, _ = R.attend(st, 0, q[[0, 0, 1], 4:5], np.ones((3, 1), np.uint64), 0.1)
    assert np.allclose(again[:, 0], before[[0, 0, 1], 4])
