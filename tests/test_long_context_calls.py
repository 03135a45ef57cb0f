"""Calls of the operators for long contexts that are refused on the host, and scaled rotary frequencies (no GPU needed)."""

import ctypes as C
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_paged_cache import A, _says, _view  # noqa: E402
from tyloquant_b200 import rope_frequencies, rope_yarn_factor  # noqa: E402
from tyloquant_b200._capi import lib  # noqa: E402

B, D, W = A + (1 << 24), A + (1 << 25), A + (1 << 26)


def test_weighing_attention_refuses():
    v, n = C.byref(_view()), C.c_uint64()
    assert lib.mfqb_tree_attention_weigh_work(v, 4, 2, C.byref(n)) == 0
    plain = C.c_uint64()
    assert lib.mfqb_tree_attention_work(v, 4, 2, C.byref(plain)) == 0 and n.value > plain.value

    def call(layer=0, q=A, heads=4, nodes=2, masks=B, scale=1.0, out=D, weights=W, work=W + (1 << 24), size=n.value):
        return lib.mfqb_tree_attention_weigh(v, layer, q, heads, nodes, masks, scale, out, weights, work, size, None)

    _says(1, "weights", call(weights=None))
    _says(1, "weights", call(weights=W + 2))
    _says(1, "null", call(q=None))
    _says(1, "layer", call(layer=9))
    _says(1, "scale", call(scale=0.0))
    _says(1, "work", call(size=n.value - 1))
    _says(1, "work", call(work=W + 8))
    _says(3, "query heads", call(heads=3))
    _says(3, "nodes", call(nodes=65))
    _says(1, "overlap", call(weights=A))
    _says(1, "overlap", call(weights=D + 16))
    _says(1, "overlap", call(weights=W + (1 << 24)))
    _says(1, "overlap", call(out=A))
    _says(1, "null", lib.mfqb_tree_attention_weigh_work(v, 4, 2, None))


def test_eviction_refuses():
    v, n = C.byref(_view()), C.c_uint64()
    assert lib.mfqb_cache_evict_work(v, C.byref(n)) == 0 and n.value > 0

    def call(weights=W, keep=A, recent=0, dropped=B, status=D, work=D + (1 << 20), size=n.value):
        return lib.mfqb_cache_evict(v, weights, keep, recent, dropped, status, work, size, None)

    for name in ("weights", "keep", "dropped", "status", "work"):
        _says(1, "null", call(**{name: None}))
    _says(1, "must not be negative", call(recent=-1))
    _says(1, "work", call(size=n.value - 1))
    _says(1, "work", call(work=D + 8))
    _says(1, "null", lib.mfqb_cache_evict_work(v, None))
    bad = _view()
    bad.page = 24
    _says(3, "power of two", lib.mfqb_cache_evict(C.byref(bad), W, A, 0, B, D, D + (1 << 20), n.value, None))


def test_rotary_write_refuses():
    v = C.byref(_view())

    def call(layer=0, qkv=A, dtype=0, heads=4, nodes=2, depths=B, freqs=B + (1 << 20), pairs=64, layout=0, factor=1.0, out=D):
        return lib.mfqb_cache_write_rope(v, layer, qkv, dtype, heads, nodes, depths, freqs, pairs, layout, factor, out, None)

    for name in ("qkv", "depths", "freqs", "out"):
        _says(1, "null", call(**{name: None}))
    _says(1, "type of qkv", call(dtype=2))
    _says(1, "aligned", call(qkv=A + 8))
    _says(1, "aligned", call(freqs=B + (1 << 20) + 4))
    _says(1, "layer", call(layer=-1))
    _says(1, "query heads", call(heads=0))
    for pairs in (0, 65):
        _says(3, "pairs", call(pairs=pairs))
    _says(1, "layout", call(layout=2))
    for factor in (0.0, -1.0, math.nan, math.inf):
        _says(1, "factor", call(factor=factor))
    _says(1, "overlap", call(out=A))
    _says(1, "overlap", call(out=A + 2 * 3 * 2 * 8 * 128 - 16, dtype=1))   # bf16: half as many bytes
    _says(3, "nodes", call(nodes=0))


def test_logprobs_refuse():
    def call(logits=A, dtype=0, rows=4, vocab=100, stride=100, tokens=B, top=5, lp=D, en=D, rank=D, tl=D, tt=D):
        return lib.mfqb_token_logprobs(logits, dtype, rows, vocab, stride, tokens, top, lp, en, rank, tl, tt, None)

    for name in ("logits", "tokens", "lp", "en", "rank", "tl", "tt"):
        _says(1, "null", call(**{name: None}))
    _says(1, "type", call(dtype=3))
    _says(1, "aligned", call(logits=A + 2))
    for rows in (0, -3, (1 << 24) + 1):
        _says(1, "rows", call(rows=rows))
    for vocab in (0, (1 << 20) + 1):
        _says(3, "vocabulary", call(vocab=vocab, stride=1 << 21))
    _says(1, "every", call(stride=99))
    for top in (-1, 33):
        _says(3, "alternatives", call(top=top))
    _says(3, "alternatives", call(top=5, vocab=4))


def test_scaled_frequencies():
    """Against the definitions, written out with numpy."""
    for dims in (128, 64, 10):
        j = np.arange(dims // 2)
        f = 10000.0 ** (-2.0 * j / dims)
        for got, want in ((rope_frequencies(10000.0, "cpu", dims=dims), f), (rope_frequencies(10000.0, "cpu", dims=dims, scaling="linear", factor=4.0), f / 4)):
            assert got.dtype == torch.float64 and np.allclose(got.numpy(), want, rtol=1e-14)
        length, s, low, high = 8192, 8.0, 1.0, 4.0
        wave = 2 * math.pi / f
        mix = (length / wave - low) / (high - low)
        want = np.where(wave < length / high, f, np.where(wave > length / low, f / s, (1 - mix) * f / s + mix * f))
        assert np.allclose(rope_frequencies(10000.0, "cpu", dims=dims, scaling="bands", factor=s, original=length).numpy(), want, rtol=1e-13)
        ends = [dims * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(10000.0)) for turns in (32.0, 1.0)]
        first, last = max(math.floor(ends[0]), 0), min(math.ceil(ends[1]), dims - 1)
        ramp = np.clip((j - first) / (last - first), 0, 1)
        assert np.allclose(rope_frequencies(10000.0, "cpu", dims=dims, scaling="yarn", factor=s, original=length).numpy(), f / s * ramp + f * (1 - ramp), rtol=1e-13)
    assert rope_yarn_factor(1.0) == 1.0 and abs(rope_yarn_factor(4.0) - (0.1 * math.log(4.0) + 1)) < 1e-15


def test_frequencies_refuse():
    for bad in (dict(dims=0), dict(dims=7), dict(dims=130), dict(scaling="cubic"), dict(scaling="linear", factor=0.5), dict(scaling="linear", factor=math.nan),
                dict(scaling="bands", factor=2.0), dict(scaling="yarn", factor=2.0, original=0), dict(scaling="bands", factor=2.0, original=100, low=5.0),
                dict(scaling="linear", factor=math.inf)):
        with pytest.raises(ValueError):
            rope_frequencies(10000.0, "cpu", **bad)
    for bad in (0.5, math.nan, math.inf):
        with pytest.raises(ValueError):
            rope_yarn_factor(bad)
