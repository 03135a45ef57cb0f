"""Log probabilities of given tokens against a plain restatement in 64 bits.

Tolerances.  Each of the vocab / 512 terms that a thread adds in turn, and each of some 64 joins, rounds by 2^-24 of the sum; an exponential of the approximate
unit is off by 2^-22 and by the rounding of its argument, 2^-23 of the logit's distance d from the largest (its average over the distribution is
`far`).  So log sums are off by e = (vocab / 512 + 64) 2^-24 + 2^-21 + far 2^-22, a log probability by that and half a step of itself and of z - max;
the entropy, log sum + average distance, by e + far e + (vocab / 512 + 64) 2^-24 far, and half a step."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import long_reference as L  # noqa: E402
from tyloquant_b200 import token_logprobs  # noqa: E402

DEV = "cuda:0"


def _check(logits, tokens, top):
    """logits: a CUDA tensor [rows, vocab]."""
    rows, vocab = logits.shape
    got = [x.cpu().numpy() for x in token_logprobs(logits, torch.tensor(tokens, dtype=torch.int32, device=DEV), top=top)]
    lp, en, rank, tl, tt, far = L.logprobs(logits.float().cpu().numpy(), tokens, top)
    n = (vocab / 512 + 64) * 2.0 ** -24
    e = n + 2.0 ** -21 + far * 2.0 ** -22
    z = np.nan_to_num(np.abs(logits.float().cpu().numpy().astype(np.float64)), posinf=0).max(1)

    def near(a, b, tol):
        with np.errstate(invalid="ignore"):
            exact = (a == b) | (np.isnan(a) & np.isnan(b))   # infinities and NaN
            assert (exact | (np.abs(a - b) <= tol)).all(), np.nanmax(np.abs(a - b) - tol)

    with np.errstate(invalid="ignore"):
        near(got[0], lp, e + 2.0 ** -23 * (np.abs(lp) + np.log(vocab)))
        near(got[1], en, e + far * (e + n) + 2.0 ** -22 * (far + np.log(vocab)))
        near(got[3], tl, (e + 2.0 ** -23 * np.log(vocab))[:, None] + 2.0 ** -23 * np.abs(tl))
    assert np.array_equal(got[2], rank) and np.array_equal(got[4], tt)
    del z
    return got


def _tokens(rng, rows, vocab):
    t = rng.integers(0, vocab, rows)
    t[rng.random(rows) < 0.1] = -1
    return t.tolist()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [1, 2, 7, 31, 32, 33, 500, 4097, 32001, 128256])
def test_by_vocabulary(vocab, dtype):
    rng = np.random.default_rng(vocab)
    for rows in (1, 3):
        z = torch.from_numpy(2.5 * rng.standard_normal((rows, vocab), dtype=np.float32)).to(DEV, dtype)
        for top in sorted({0, 1, min(5, vocab), min(32, vocab)}):
            _check(z, _tokens(rng, rows, vocab), top)


@pytest.mark.parametrize("rows", [1, 2, 5, 18, 19, 37, 74, 148, 296, 600])
def test_by_rows(rows):
    """Few rows are split over clusters of two CTAs, and longer ones of up to eight."""
    rng = np.random.default_rng(rows)
    for vocab in (33000, 70000, 130000) if rows <= 74 else (33000,):
        z = torch.from_numpy(2.5 * rng.standard_normal((rows, vocab), dtype=np.float32)).to(DEV)
        _check(z, _tokens(rng, rows, vocab), 20)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("pad,skip", [(1, 0), (3, 1), (8, 5), (0, 0)])
def test_rows_that_lie_apart(pad, skip, dtype):
    """Rows that start at any element, as parts of wider ones; what lies between them does not count."""
    rng = np.random.default_rng(pad)
    wide = torch.full((6, 5003 + pad + skip), torch.inf, device=DEV, dtype=dtype)
    z = wide[:, skip:skip + 5003]
    z.copy_(torch.from_numpy(rng.standard_normal((6, 5003))))
    _check(z, [0, 5002, 1, 7, -1, 5003], 17)
    _check(z.t().contiguous().t(), [0, 5002, 1, 7, -1, 5003], 17)


@pytest.mark.parametrize("vocab", [40, 3000, 70000])
def test_equal_logits(vocab):
    """All equal; few different values; all the best ones in one thread's vectors; rising and falling rows."""
    rng = np.random.default_rng(vocab)
    rows = [np.zeros(vocab), np.full(vocab, -3.4028234e38), rng.integers(0, 3, vocab), np.arange(vocab) / 64.0, -np.arange(vocab) / 64.0,
            np.where(np.arange(vocab) // 4 % 512 == 3, 5.0 + rng.random(vocab), 0.0), np.where(np.arange(vocab) // 4 % 512 < 30, 5.0, rng.random(vocab)),
            np.where(np.arange(vocab) % 2, 0.0, -0.0)]
    z = torch.from_numpy(np.array(rows, dtype=np.float32)).to(DEV)
    for top in (1, 5, 32):
        _check(z, rng.integers(0, vocab, len(rows)).tolist(), top)
    _check(torch.cat([z] * 40), rng.integers(0, vocab, 40 * len(rows)).tolist(), 32)   # a CTA a row


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [1, 7, 40, 500, 8001])
def test_many_short_rows(vocab, dtype):
    """CTAs of 128 threads; a sixth of the rows all equal, a sixth of few values."""
    rng = np.random.default_rng(vocab)
    z = 2.5 * rng.standard_normal((600, vocab), dtype=np.float32)
    z[::6] = 1.5
    z[1::6] = np.round(z[1::6])
    _check(torch.from_numpy(z).to(DEV, dtype), _tokens(rng, 600, vocab), min(32, vocab))


def test_masked_logits_and_rows_without_a_log_sum():
    rng = np.random.default_rng(0)
    vocab = 9001
    z = rng.standard_normal((10, vocab)).astype(np.float32)
    z[0, 5:] = -np.inf
    z[1] = -np.inf
    z[2, 100] = np.nan
    z[3, 100] = np.inf
    z[4, :] = -np.inf
    z[4, 8000] = 3.0
    z[5, rng.random(vocab) < 0.9] = -np.inf
    z[6] = -3.4028234e38
    z[6, 17] = -np.inf
    z[7, 100] = 3e38
    z[8] *= 1e4
    z[9, 1:] = -3.4028234e38
    for tokens in ([3, 3, 3, 3, 8000, 3, 3, 3, 3, 0], [7, 100, 100, 100, 3, 4, 17, 100, 0, 9], [-1, -1, -1, -1, 9001, 2 ** 30, -5, -1, -1, -1]):
        for top in (0, 1, 32):
            got = _check(torch.from_numpy(z).to(DEV), tokens, top)
            for r in (1, 2, 3):
                assert np.isnan(got[1][r]) and got[2][r] == 0 and (got[4][r] == -1).all()
    assert got[2][4] == 0 and got[0][0] == 0.0


def test_no_rows_and_refusals():
    z = torch.zeros((0, 50), device=DEV)
    assert token_logprobs(z, torch.zeros(0, dtype=torch.int32, device=DEV), top=3).top_tokens.shape == (0, 3)
    z, t = torch.zeros((2, 50), device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    for bad in (lambda: token_logprobs(z[0], t), lambda: token_logprobs(z.double(), t), lambda: token_logprobs(z, t[:1]), lambda: token_logprobs(z, t.long()),
                lambda: token_logprobs(z.cpu(), t), lambda: token_logprobs(z, t.cpu())):
        with pytest.raises(ValueError):
            bad()
    from tyloquant_b200 import MfqbError
    for top in (-1, 33, 51):
        with pytest.raises((MfqbError, RuntimeError)):
            token_logprobs(z, t, top=top)


def test_repeats_bit_for_bit_and_in_a_graph():
    rng = np.random.default_rng(2)
    z = torch.from_numpy(rng.standard_normal((3, 60000), dtype=np.float32)).to(DEV)
    t = torch.tensor([5, 6, 59999], dtype=torch.int32, device=DEV)
    first = token_logprobs(z, t, top=9)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = token_logprobs(z, t, top=9)
    z.copy_(z.flip(0))
    t.copy_(t.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(first, out):
        assert torch.equal(a, b.flip(0))
