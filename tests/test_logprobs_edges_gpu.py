"""Log probabilities of rows that are split over several CTAs and start or end inside a 16-byte vector: the first CTA has the row's
beginning, the last one its end; bounds as of test_logprobs_gpu."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_logprobs_gpu import DEV, _check  # noqa: E402


def _apart(z, skip, pad, dtype):
    """The rows as parts of wider ones, between infinities."""
    wide = torch.full((z.shape[0], skip + z.shape[1] + pad), torch.inf, device=DEV, dtype=dtype)
    part = wide[:, skip:skip + z.shape[1]]
    part.copy_(torch.from_numpy(z))
    return part


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [50257, 70001, 128257])
@pytest.mark.parametrize("skip,pad", [(0, 0), (1, 0), (3, 2), (5, 4)])
def test_split_rows_at_any_element(skip, pad, vocab, dtype):
    """Tokens in the first and the last vector, in the middle, and none."""
    rng = np.random.default_rng(vocab + skip)
    for rows in (1, 3, 70):
        z = _apart(2.5 * rng.standard_normal((rows, vocab), dtype=np.float32), skip, pad, dtype)
        ends = [0, 1, vocab - 1, vocab - 2, 7, vocab // 2, -1, vocab]
        tokens = [ends[(r + skip) % len(ends)] for r in range(rows)]
        _check(z, tokens, 20)
        if rows == 1:
            for t in ends:
                _check(z, [t], 3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [70001, 128257])
def test_split_rows_of_which_a_mask_leaves_little(vocab, dtype):
    """One CTA's slice alone, its neighbours' nothing; single logits at the ends; fewer than are asked for; masked tokens and their ranks."""
    rng = np.random.default_rng(vocab)
    rows = []
    for first, last in ((0, 9000), (vocab - 9000, vocab), (vocab // 2, vocab // 2 + 50), (0, 1), (vocab - 1, vocab), (vocab // 4 - 3, vocab // 4 + 3)):
        row = np.full(vocab, -np.inf, np.float32)
        row[first:last] = rng.standard_normal(last - first)
        rows.append(row)
    rows.append(np.full(vocab, -3.3e38, np.float32))   # all masked by a finite value
    rows[-1][vocab - 5:] = 0.0
    z = np.array(rows)
    for skip in (0, 1, 3):
        x = _apart(z, skip, 2, dtype)
        for tokens in ([5, vocab - 1, vocab // 2 + 7, 0, vocab - 1, vocab // 4, vocab - 3], [vocab - 1, 0, 1, 1, 0, vocab - 2, 0], [2, 2, 2, 2, 2, 2, 2]):
            _check(x, tokens, 32)


@pytest.mark.parametrize("vocab", [70001, 128257])
def test_split_rows_of_equal_logits(vocab):
    """What is asked for lies in the first CTA's slice, or is spread over all of them, with ties."""
    rng = np.random.default_rng(vocab)
    z = np.array([np.zeros(vocab), rng.integers(0, 3, vocab), np.where(np.arange(vocab) % 9001 == 17, 2.0, 1.0), np.arange(vocab) / 64.0, -np.arange(vocab) / 64.0], dtype=np.float32)
    for skip in (0, 2):
        x = _apart(z, skip, 1, torch.float32)
        for top in (1, 5, 32):
            _check(x, [0, vocab - 1, 9018, 3, vocab - 1], top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(1, 32767), (1, 32769), (2, 65535), (2, 65537), (150, 66001), (149, 33001), (40, 80011), (38, 79993), (37, 80011)])
def test_around_the_numbers_of_ctas(rows, vocab, dtype):
    """One, two, four and eight CTAs a row, by bytes, rows and logits of a slice."""
    rng = np.random.default_rng(vocab)
    z = _apart(2.5 * rng.standard_normal((rows, vocab), dtype=np.float32), 1, 2, dtype)
    _check(z, [(0, vocab - 1, vocab // 3, -1)[r % 4] for r in range(rows)], 7)
