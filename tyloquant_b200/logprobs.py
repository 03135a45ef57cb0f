"""What a program reads off the logits besides the next token: log probabilities of given tokens, with entropy, rank and the best
alternatives.  torch only provides device memory and streams."""

from __future__ import annotations

from typing import NamedTuple

from . import _fast
from ._capi import BF16, F16, F32
from .cache import _call, _need
from .linear import _torch


class TokenLogprobs(NamedTuple):
    logprob: object       # float32 [rows]
    entropy: object       # float32 [rows]
    rank: object          # int32 [rows]
    top_logprobs: object  # float32 [rows, top]
    top_tokens: object    # int32 [rows, top]


def token_logprobs(logits, tokens, top: int = 0) -> TokenLogprobs:
    """Per row of ``logits`` (float32, bfloat16 or float16 [rows, vocab]; rows may lie apart): the log probability of ``tokens`` (int32 [rows]), the
    entropy of the distribution in nats, the token's rank (1 = the best; equal logits: the lower number first) and the ``top`` best
    tokens (at most 32) with their log probabilities, best first.  A token outside [0, vocab) is none (padding): log probability 0, rank 0.  What is
    masked out is minus infinity.  A row with a NaN or plus infinity, or with nothing above minus infinity, has NaN for log
    probabilities and entropy, rank 0 and tokens -1.

    Asynchronous on the current stream of the logits' device; can be captured into a CUDA graph after a first call of the same type."""
    torch = _torch()
    if logits.dim() != 2 or not logits.is_cuda:
        raise ValueError("logits must be a CUDA tensor [rows, vocab]")
    dtype = F32 if logits.dtype is torch.float32 else BF16 if logits.dtype is torch.bfloat16 else F16 if logits.dtype is torch.float16 else None
    if dtype is None:
        raise ValueError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    rows, vocab = logits.shape
    dev = logits.get_device()
    z = logits if logits.stride(1) == 1 and logits.stride(0) >= vocab else logits.contiguous()
    t = _need(tokens, torch.int32, (rows,), dev, "tokens")
    top = int(top)
    # the host's part of a call is mostly these; sizes in positions and the type of a tensor at hand are the cheapest forms
    logprob = z.new_empty(rows) if dtype == F32 else z.new_empty(rows, dtype=torch.float32)
    entropy, rank = torch.empty_like(logprob), torch.empty_like(t)
    top_logprobs, top_tokens = logprob.new_empty(rows, max(top, 0)), t.new_empty(rows, max(top, 0))
    if rows:
        _call(_fast.token_logprobs, dev, z.data_ptr(), dtype, rows, vocab, z.stride(0), t.data_ptr(), top, logprob.data_ptr(), entropy.data_ptr(),
              rank.data_ptr(), top_logprobs.data_ptr(), top_tokens.data_ptr())
    return TokenLogprobs(logprob, entropy, rank, top_logprobs, top_tokens)
