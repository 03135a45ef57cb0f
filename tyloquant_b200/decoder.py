"""Dense decoder step over the C ABI (mirrors ``QuantLinear`` / ``FFN`` / ``FullBlock::forward`` /
``Model::next_token`` of the reference runtime, cpp_runtime/mfq_decode.cpp:9116-9407, 10456-10602,
12210-12400, 13993-14145, for Llama-shaped blocks).  torch only provides device memory and streams."""

from __future__ import annotations

import ctypes as C

import numpy as np

from ._capi import DecoderConfig, check, lib
from .linear import QuantWeight, _stream_ptr, _torch


class Decoder:
    """One rank's share of a decoder: borrowed weight handles, KV cache, one greedy step per call."""

    def __init__(self, *, hidden, n_q_heads, n_kv_heads, ffn, vocab, layers, max_ctx, max_batch,
                 rope_theta=500000.0, rms_eps=1e-5, rank=0, world=1, comm=None, device=0):
        self.cfg = DecoderConfig(hidden, n_q_heads, n_kv_heads, 128, ffn, vocab, layers, max_ctx, max_batch, rope_theta, rms_eps)
        self.rank, self.world, self.device = rank, world, device
        self._comm = comm
        self._keep = []   # the weights are borrowed by the native object: keep them alive here
        self._cache, self._beside = None, None
        self._h = C.c_void_p()
        check(lib.mfqb_decoder_create(C.byref(self.cfg), rank, world, comm._h if comm is not None else None, device, C.byref(self._h)))

    def set_layer(self, layer: int, qkv: QuantWeight, o: QuantWeight, gate_up: QuantWeight, down: QuantWeight) -> None:
        check(lib.mfqb_decoder_set_layer(self._h, layer, qkv._h, o._h, gate_up._h, down._h))
        self._keep += [qkv, o, gate_up, down]

    def vocab_shard(self):
        b, n = C.c_int(), C.c_int()
        check(lib.mfqb_decoder_vocab_shard(self._h, C.byref(b), C.byref(n)))
        return b.value, n.value

    def set_head(self, lm_head: QuantWeight, embedding) -> None:
        torch = _torch()
        if embedding.dtype != torch.bfloat16 or not embedding.is_cuda or not embedding.is_contiguous():
            raise ValueError("embedding must be a contiguous bfloat16 CUDA tensor [vocab, hidden]")
        check(lib.mfqb_decoder_set_head(self._h, lm_head._h, embedding.data_ptr()))
        self._keep += [lm_head, embedding]

    def fill_cache(self, ctx_len: int, seed: int = 0) -> None:
        check(lib.mfqb_decoder_fill_cache(self._h, ctx_len, seed, _stream_ptr(self.device)))

    def step(self, ids_in, ids_out=None):
        torch = _torch()
        if ids_in.dtype != torch.int32 or ids_in.get_device() != self.device:
            raise ValueError(f"ids_in must be an int32 tensor [batch] on cuda:{self.device}")
        ids_in = ids_in.contiguous()
        if ids_out is None:
            ids_out = torch.empty_like(ids_in)
        elif ids_out.dtype != torch.int32 or ids_out.get_device() != self.device or ids_out.numel() < ids_in.numel() or not ids_out.is_contiguous():
            raise ValueError(f"ids_out must be a contiguous int32 tensor with room for {ids_in.numel()} tokens on cuda:{self.device}")
        check(lib.mfqb_decoder_step(self._h, ids_in.data_ptr(), ids_in.numel(), ids_out.data_ptr(), _stream_ptr(self.device)))
        return ids_out

    def layer(self, layer: int, h_in):
        torch = _torch()
        h_in = h_in.contiguous().float()
        out = torch.empty_like(h_in)
        check(lib.mfqb_decoder_layer(self._h, layer, h_in.data_ptr(), h_in.shape[0], out.data_ptr(), _stream_ptr(self.device)))
        return out

    def read_cache(self, layer: int, row: int, which: int, ctx: int):
        torch = _torch()
        nkv = self.cfg.n_kv_heads // self.world
        out = torch.empty((nkv, ctx, 128), dtype=torch.bfloat16, device=f"cuda:{self.device}")
        check(lib.mfqb_decoder_read_cache(self._h, layer, row, which, ctx, out.data_ptr(), _stream_ptr(self.device)))
        return out

    def read_logits(self, rows: int):
        """float32 [rows, vocabulary rows of this rank]: the logits of the last step."""
        torch = _torch()
        begin, n = C.c_int(), C.c_int()
        check(lib.mfqb_decoder_vocab_shard(self._h, C.byref(begin), C.byref(n)))
        out = torch.empty((rows, n.value), dtype=torch.float32, device=f"cuda:{self.device}")
        check(lib.mfqb_decoder_read_logits(self._h, rows, out.data_ptr(), _stream_ptr(self.device)))
        return out

    def set_cache(self, cache, weights=None, dropped=None) -> None:
        """Runs over a :class:`PagedCache` from here on (``None``: over the decoder's own cache again); a row per sequence.  ``max_ctx=0`` at
        creation leaves the decoder without a cache of its own.  The decoder keeps the cache alive while it is attached; a graph that was
        captured over it needs it as long as it is replayed.

        ``weights`` (``cache.new_weights()``): every pass adds up in them how much each position was looked at, for ``cache.evict``.  ``dropped`` (int32
        [rows]): what has been evicted of every sequence so far, added to its positions; add to it what ``evict`` returns.  Both are kept
        alive like the cache; ``beam_step`` is refused with either.  After ``verify`` give the weights to ``cache.accept`` too, which moves the kept
        branch's; what the queries of rejected nodes have added to the context's positions stays.  Unused nodes add nothing.  The passes' work memory, which
        stays with the decoder, holds scores then: up to 512 MB (see ``PagedCache.attend``)."""
        from .cache import _need
        torch = _torch()
        if cache is None and (weights is not None or dropped is not None):
            raise ValueError("weights and dropped go with a cache")
        if weights is not None:
            cache._weights(weights)
            if weights.data_ptr() % 16:
                raise ValueError("weights must be 16-byte aligned")
        if dropped is not None and _need(dropped, torch.int32, (cache.rows,), self.device, "dropped") is not dropped:
            raise ValueError("dropped must be contiguous")
        check(lib.mfqb_decoder_set_cache(self._h, None if cache is None else C.byref(cache._view)))
        self._cache, self._beside = cache, (weights, dropped)   # borrowed by the native object
        if weights is not None or dropped is not None:
            try:
                check(lib.mfqb_decoder_set_weights(self._h, None if weights is None else weights.data_ptr(), None if dropped is None else dropped.data_ptr()))
            except Exception:   # no memory for what its passes need: no pages without what was asked for beside them
                lib.mfqb_decoder_set_cache(self._h, None)
                self._cache, self._beside = None, None
                raise

    def _rows(self, t, shape, dtype, what):
        from .cache import _need
        if self._cache is None:
            raise ValueError("the decoder runs over its own cache: set_cache first")
        return _need(t, dtype, shape, self.device, what)

    def verify(self, ids, parents):
        """The drafted trees of all sequences in one pass (``ids``, ``parents`` int32 [rows, nodes], see ``tree_masks``): returns the model's own
        greedy token at every node.  Reserve ``nodes`` tokens first (``cache.extend``); ``cache.accept`` keeps the branch that agrees (give it
        the weights where some are attached)."""
        torch = _torch()
        if ids.dim() != 2:
            raise ValueError("ids must be an int32 tensor [rows, nodes]")
        rows = self._cache.rows if self._cache is not None else 0
        shape = (rows, ids.shape[1])
        i, p = self._rows(ids, shape, torch.int32, "ids"), self._rows(parents, shape, torch.int32, "parents")
        out = torch.empty_like(i)
        check(lib.mfqb_decoder_verify(self._h, i.data_ptr(), p.data_ptr(), ids.shape[1], out.data_ptr(), _stream_ptr(self.device)))
        return out

    def beam_step(self, ids, scores, done, beams: int, eos: int):
        """One step of beam search over groups of ``beams`` sequences: ``ids`` int32 [rows], ``scores`` float32 and ``done`` int32 [rows], which are
        changed in place, like the cache.  Returns (tokens [rows], the sequences they go on from [rows], status [2]: of the
        cache's extend and fork)."""
        torch = _torch()
        rows = self._cache.rows if self._cache is not None else 0
        i = self._rows(ids, (rows,), torch.int32, "ids")
        for t, dtype, what in ((scores, torch.float32, "scores"), (done, torch.int32, "done")):
            if self._rows(t, (rows,), dtype, what) is not t:
                raise ValueError(f"{what} must be contiguous")
        tokens, parents, status = torch.empty_like(i), torch.empty_like(i), i.new_empty(2)
        check(lib.mfqb_decoder_beam_step(self._h, i.data_ptr(), beams, scores.data_ptr(), done.data_ptr(), eos, tokens.data_ptr(), parents.data_ptr(),
                                         status.data_ptr(), _stream_ptr(self.device)))
        return tokens, parents, status

    def free(self) -> None:
        if self._h:
            lib.mfqb_decoder_free(self._h)
            self._h = C.c_void_p()
        self._keep = []

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def random_decoder(*, hidden, n_q_heads, n_kv_heads, ffn, vocab, layers, max_ctx, max_batch, rank=0, world=1, comm=None,
                   device=0, seed=5000, attn_profile=(4, 24, 6), ffn_profile=(6, 24, 7), distinct_layers=2, keep_blobs=False):
    """A random-init decoder in this rank's tensor-parallel shapes: attention projections in
    ``attn_profile``, FFN and lm_head in ``ffn_profile`` (bits, group size, sub-scale bits).
    ``distinct_layers`` layers are packed from their own seeded blobs; the others are device copies of
    those (every layer still streams its own memory).  Returns (decoder, blobs) -- blobs of the packed
    layers when ``keep_blobs`` (for parity checks against the oracle)."""
    from . import encode
    torch = _torch()
    d = f"cuda:{device}"
    dec = Decoder(hidden=hidden, n_q_heads=n_q_heads, n_kv_heads=n_kv_heads, ffn=ffn, vocab=vocab, layers=layers, max_ctx=max_ctx,
                  max_batch=max_batch, rank=rank, world=world, comm=comm, device=device)
    nq, nkv, f = n_q_heads // world, n_kv_heads // world, ffn // world
    shapes = {"qkv": ((nq + 2 * nkv) * 128, hidden, attn_profile), "o": (hidden, nq * 128, attn_profile),
              "gate_up": (2 * f, hidden, ffn_profile), "down": (hidden, f, ffn_profile)}
    base, blobs = [], []
    for li in range(min(distinct_layers, layers)):
        ws, bl = {}, {}
        for j, (name, (n, k, (bits, gs, sb))) in enumerate(shapes.items()):
            blob = encode.random_nint_blob(n, k, bits, gs, sb, seed=seed + 100 * li + 10 * j + rank * 7919, device=d)
            ws[name] = QuantWeight.from_blob(f"NINT{bits}", blob, device=device)
            if keep_blobs:
                bl[name] = blob
        base.append(ws)
        blobs.append(bl)
    for li in range(layers):
        src = base[li % len(base)]
        ws = src if li < len(base) else {k: v.clone() for k, v in src.items()}
        dec.set_layer(li, ws["qkv"], ws["o"], ws["gate_up"], ws["down"])
    vb, vn = dec.vocab_shard()
    bits, gs, sb = ffn_profile
    head_blob = encode.random_nint_blob(vn, hidden, bits, gs, sb, seed=seed + 9000 + rank * 7919, device=d)
    lm_head = QuantWeight.from_blob(f"NINT{bits}", head_blob, device=device)
    gen = torch.Generator(d).manual_seed(seed + 1)   # the embedding is replicated: same seed on every rank
    emb = torch.randn((vocab, hidden), device=d, generator=gen).to(torch.bfloat16)
    dec.set_head(lm_head, emb)
    if keep_blobs:
        blobs.append({"lm_head": head_blob, "embedding": emb})
    return dec, blobs
