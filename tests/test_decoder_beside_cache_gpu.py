"""What a decoder has attached beside its cache, weights and counts of dropped positions: refusals and what they leave."""

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_paged_decoder_gpu import _cache, _decoder, _i32  # noqa: E402
from tyloquant_b200 import MfqbError  # noqa: E402

DEV = "cuda:0"


def test_a_beam_step_says_what_is_in_its_way():
    dec, cache = _decoder(8), _cache(2)
    weights, dropped = cache.new_weights(), _i32([0, 0])
    beam = _i32([1, 2]), torch.zeros(2, device=DEV), _i32([0, 0]), 1, 2
    for beside, text in ((dict(dropped=dropped), "dropped positions are attached"), (dict(weights=weights), "weights are attached"),
                         (dict(weights=weights, dropped=dropped), "weights are attached")):
        dec.set_cache(cache, **beside)
        with pytest.raises(MfqbError, match=text):
            dec.beam_step(*beam)
        assert cache.lens.tolist() == [0, 0] and not cache.refs.any()
    dec.set_cache(cache)
    _, _, status = dec.beam_step(*beam)
    assert status.tolist() == [0, 0] and cache.lens.tolist() == [1, 1]
    dec.free()


def test_weights_that_are_refused_change_nothing():
    """The decoder goes on over the cache and the weights that it had."""
    rows = 2
    dec, cache, other = _decoder(8), _cache(rows), _cache(rows)
    weights = cache.new_weights()
    dec.set_cache(cache, weights=weights)
    assert int(cache.extend(2)) == 0
    dec.step(_i32([1, 2]))
    odd = torch.zeros(weights.numel() + 1, device=DEV)[1:].view(weights.shape)   # contiguous, but no 16-byte boundary
    for bad, text in ((odd, "16-byte"), (weights[:1], "weights"), (weights.double(), "weights")):
        with pytest.raises(ValueError, match=text):
            dec.set_cache(other, weights=bad)
    with pytest.raises(ValueError, match="dropped"):
        dec.set_cache(other, weights=weights, dropped=_i32([0, 0, 0]))
    dec.step(_i32([3, 4]))
    assert cache.lens.tolist() == [2, 2] and other.lens.tolist() == [0, 0]
    assert (weights.double().sum(-1) - 2 * 2).abs().max() <= 1e-3   # two queries a KV head, two steps
    dec.free()


def test_no_memory_for_weights_leaves_no_pages(monkeypatch):
    """The native call fails: nothing is attached any more, as where there is no memory for a cache."""
    from tyloquant_b200 import decoder as D

    class Lib:
        def __getattr__(self, name):
            return getattr(lib, name)

        def mfqb_decoder_set_weights(self, *args):
            return lib.mfqb_decoder_set_weights(None, None, None)

    lib, dec, cache = D.lib, _decoder(8), _cache(2)
    monkeypatch.setattr(D, "lib", Lib())
    with pytest.raises(MfqbError):
        dec.set_cache(cache, weights=cache.new_weights())
    monkeypatch.setattr(D, "lib", lib)
    with pytest.raises(MfqbError, match="none is attached"):
        dec.step(_i32([1, 2]))
    dec.free()
