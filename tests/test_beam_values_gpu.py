"""Beams whose logits are no numbers: what becomes of their candidates and of the other beams."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_paged_cache_gpu import DEV, _check_beams  # noqa: E402
from tyloquant_b200 import beam_select  # noqa: E402


@pytest.mark.parametrize("value", [np.nan, np.inf])
@pytest.mark.parametrize("vocab", [500, 20000])
def test_a_logit_that_is_no_number_takes_its_beam_out(value, vocab):
    """All candidates of the beam have the score minus infinity, those with finite logits too; the other beam is chosen as if it were alone.  A masked
    token, minus infinity, takes nothing out."""
    rng = np.random.default_rng(vocab)
    logits = rng.standard_normal((1, 2, vocab)).astype(np.float32)
    logits[0, 1, vocab // 2:vocab // 2 + 100] = -np.inf
    alone = [x.cpu().numpy() for x in beam_select(torch.from_numpy(logits[:, 1:]).to(DEV), torch.tensor([[-2.0]], device=DEV), 6)]
    logits[0, 0, vocab // 3] = value
    scores, rows, tokens = _check_beams(logits, np.array([[0.0, -2.0]], np.float32), 6)
    assert (rows == 1).all() and np.array_equal(scores, alone[0]) and np.array_equal(tokens, alone[2]) and np.isfinite(scores).all()
    done = np.array([[0, 1]], np.int32)   # the other one has ended: its only candidate first, then the first beam's by logit
    scores, rows, tokens = _check_beams(logits, np.array([[0.0, -2.0]], np.float32), 6, done, eos=9)
    assert scores[0, 0] == -2.0 and tokens[0, 0] == 9 and (rows[0, 1:] == 0).all() and (scores[0, 1:] == -np.inf).all()
    y = np.where(np.isnan(logits[0, 0]), -np.inf, logits[0, 0])
    assert tokens[0, 1:].tolist() == np.lexsort((np.arange(vocab), -y))[:5].tolist()
