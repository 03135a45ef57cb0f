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
