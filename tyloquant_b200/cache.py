"""A key/value cache in pages that sequences share, and the operators of a decoder over it: writing a step's keys and values, attention
of drafted tokens, keeping the accepted branch, forking sequences; and the selection of beams.  torch only provides device
memory and streams.

All calls are asynchronous on the current stream of the cache's device, allocate nothing outside torch's allocator and can be
captured into a CUDA graph."""

from __future__ import annotations

import ctypes as C
import functools

from . import _fast
from ._capi import CacheView, check, lib
from .linear import _torch

HEAD_DIM = 128
MAX_NODES = 64


def _need(t, dtype, shape, device: int, what: str):
    """`t` as a contiguous tensor; raises unless it has this type and shape and is on this GPU."""
    if t.dtype is dtype and t.get_device() == device and t.shape == shape:
        return t if t.is_contiguous() else t.contiguous()
    raise ValueError(f"{what} must be a {str(dtype).replace('torch.', '')} tensor {list(shape)} on cuda:{device}, got {t.dtype} {list(t.shape)} on {t.device}")


def _call(fn, device: int, *args) -> None:
    """One library call on the current stream of a device, which is made current where it is not."""
    cuda = _torch()._C
    if cuda._cuda_getDevice() == device:
        status = fn(*args, cuda._cuda_getCurrentRawStream(device))
    else:
        with _torch().cuda.device(device):
            status = fn(*args, cuda._cuda_getCurrentRawStream(device))
    if status:
        check(status)


def rope_frequencies(theta: float = 500000.0, device="cuda"):
    """float64 [64]: theta^(-2j/128), what ``PagedCache.write`` takes."""
    torch = _torch()
    return float(theta) ** (-torch.arange(HEAD_DIM // 2, dtype=torch.float64, device=device) * 2 / HEAD_DIM)


def tree_masks(parents):
    """``parents`` int32 [rows, nodes] (-1 for the root, node 0; an earlier node for every other one) -> (masks int64 [rows, nodes], bit j =
    node j is the node itself or above it; depths int32 [rows, nodes]).  Nodes with any other entry, and what hangs below them,
    are unused: mask and depth 0."""
    torch = _torch()
    if parents.dim() != 2 or not parents.is_cuda:
        raise ValueError("parents must be an int32 CUDA tensor [rows, nodes]")
    dev = parents.get_device()
    p = _need(parents, torch.int32, parents.shape, dev, "parents")
    masks, depths = p.new_empty(p.shape, dtype=torch.int64), torch.empty_like(p)
    _call(_fast.tree_masks, dev, p.data_ptr(), p.shape[0], p.shape[1], masks.data_ptr(), depths.data_ptr())
    return masks, depths


class PagedCache:
    """Keys and values ``k``, ``v`` bf16 [layers, pages, kv_heads, page, 128], ``table`` int32 [rows, width], ``lens`` int32 [rows],
    ``refs`` int32 [pages], all contiguous on one device; the tensors stay the caller's and are changed in place, never exchanged.

    The object holds a workspace beside them: like them it has to live as long as calls on it are under way on other streams
    than that it was made on, and as long as a graph that has captured its calls is replayed."""

    def __setattr__(self, name, value):
        if name in ("k", "v", "table", "lens", "refs") and getattr(self, name, value) is not value:
            raise AttributeError(f"{name} of a cache is not exchanged, the library holds its address: change it in place")
        object.__setattr__(self, name, value)

    def __init__(self, k, v, table, lens, refs):
        torch = _torch()
        if k.dim() != 5 or k.shape[4] != HEAD_DIM or not k.is_cuda:
            raise ValueError("k must be a bfloat16 CUDA tensor [layers, pages, kv_heads, page, 128]")
        if table.dim() != 2:
            raise ValueError("table must be an int32 tensor [rows, width]")
        layers, pages, heads, page, _ = k.shape
        rows, width = table.shape
        for t, dtype, shape, what in ((k, torch.bfloat16, k.shape, "k"), (v, torch.bfloat16, k.shape, "v"), (table, torch.int32, (rows, width), "table"),
                                      (lens, torch.int32, (rows,), "lens"), (refs, torch.int32, (pages,), "refs")):
            if _need(t, dtype, shape, k.get_device(), what) is not t:
                raise ValueError(f"{what} must be contiguous")
        self.k, self.v, self.table, self.lens, self.refs = k, v, table, lens, refs
        self.layers, self.pages, self.kv_heads, self.page, self.rows, self.width = layers, pages, heads, page, rows, width
        self.device = k.get_device()
        self._view = CacheView(k.data_ptr(), v.data_ptr(), table.data_ptr(), lens.data_ptr(), refs.data_ptr(), layers, heads, page, pages, rows, width)
        self._ptr = C.addressof(self._view)
        size = C.c_uint64()
        with torch.cuda.device(self.device):
            check(lib.mfqb_cache_fork_work(C.byref(self._view), C.byref(size)))   # refuses a shape that the library does not take
        self._fork_work = lens.new_empty((size.value + 3) // 4)   # calls on one cache are in order: they can share it
        self._attend_work = {}

    @classmethod
    def empty(cls, *, layers: int, kv_heads: int, page: int, pages: int, rows: int, width: int, device: int = 0):
        """A cache of ``pages`` free pages for ``rows`` empty sequences of up to ``width`` pages each."""
        torch = _torch()
        d = f"cuda:{device}"
        shape = (layers, pages, kv_heads, page, HEAD_DIM)
        return cls(torch.zeros(shape, dtype=torch.bfloat16, device=d), torch.zeros(shape, dtype=torch.bfloat16, device=d),
                   torch.full((rows, width), -1, dtype=torch.int32, device=d), torch.zeros(rows, dtype=torch.int32, device=d),
                   torch.zeros(pages, dtype=torch.int32, device=d))

    def _int32(self, t, shape, what):
        return _need(t, _torch().int32, shape, self.device, what)

    def extend(self, tokens):
        """Reserves pages for ``tokens[r]`` more tokens of every sequence (int32 [rows], or one number for all).  Returns int32 [1] on the
        device: 0, or how many pages were missing (then nothing has changed)."""
        torch = _torch()
        if isinstance(tokens, int):
            tokens = torch.full((self.rows,), tokens, dtype=torch.int32, device=self.k.device)
        t = self._int32(tokens, (self.rows,), "tokens")
        status = self.lens.new_empty(1)
        _call(_fast.cache_extend, self.device, self._ptr, t.data_ptr(), status.data_ptr())
        return status

    def fork(self, parents):
        """Sequence r goes on as sequence ``parents[r]`` (int32 [rows]; -1 ends it).  Full pages are shared, partly filled ones copied for all but
        the first that goes on with them; pages reserved behind the lengths go back.  Returns int32 [1] on the device: 0, how many
        pages were missing, or -1 for an entry outside [-1, rows); where it is not 0 nothing has changed."""
        p = self._int32(parents, (self.rows,), "parents")
        status = self.lens.new_empty(1)
        work = self._fork_work
        _call(_fast.cache_fork, self.device, self._ptr, p.data_ptr(), status.data_ptr(), work.data_ptr(), work.numel() * 4)
        return status

    def write(self, layer: int, qkv, depths, freqs):
        """Rotary embedding and cache write of the nodes of every sequence: ``qkv`` float32 [rows, nodes, (q_heads + 2 kv_heads) * 128], positions
        ``lens + depths`` (int32 [rows, nodes]), ``freqs`` float64 [64].  Keys and values of node i go to slot lens + i; returns the
        rotated queries, bf16 [rows, nodes, q_heads, 128]."""
        torch = _torch()
        if qkv.dim() != 3 or qkv.shape[0] != self.rows or qkv.shape[2] % HEAD_DIM or qkv.shape[2] // HEAD_DIM <= 2 * self.kv_heads:
            raise ValueError(f"qkv must be [{self.rows}, nodes, (q_heads + {2 * self.kv_heads}) * 128], got {list(qkv.shape)}")
        nodes, hq = qkv.shape[1], qkv.shape[2] // HEAD_DIM - 2 * self.kv_heads
        x = _need(qkv, torch.float32, qkv.shape, self.device, "qkv")
        d = self._int32(depths, (self.rows, nodes), "depths")
        f = _need(freqs, torch.float64, (HEAD_DIM // 2,), self.device, "freqs")
        q = x.new_empty((self.rows, nodes, hq, HEAD_DIM), dtype=torch.bfloat16)
        _call(_fast.cache_write, self.device, self._ptr, layer, x.data_ptr(), hq, nodes, d.data_ptr(), f.data_ptr(), q.data_ptr())
        return q

    def attend(self, layer: int, q, masks, scale: float | None = None, out=None):
        """Attention of the nodes over the cache: ``q`` bf16 [rows, nodes, q_heads, 128], ``masks`` int64 [rows, nodes] (``tree_masks``); node i sees
        the positions below its sequence's length and the nodes whose bits are set.  Returns bf16 like ``q``; zeros where a node sees
        nothing.  ``scale`` is 1 / sqrt(128) unless given."""
        torch = _torch()
        if q.dim() != 4 or q.shape[0] != self.rows or q.shape[3] != HEAD_DIM:
            raise ValueError(f"q must be [{self.rows}, nodes, q_heads, 128], got {list(q.shape)}")
        _, nodes, hq, _ = q.shape
        x = _need(q, torch.bfloat16, q.shape, self.device, "q")
        m = _need(masks, torch.int64, (self.rows, nodes), self.device, "masks")
        if out is None:
            out = torch.empty_like(x)
        elif _need(out, torch.bfloat16, q.shape, self.device, "out") is not out:
            raise ValueError("out must be contiguous")
        size = self._attend_work.get((hq, nodes))
        if size is None:
            n = C.c_uint64()
            with torch.cuda.device(self.device):
                check(lib.mfqb_tree_attention_work(C.byref(self._view), hq, nodes, C.byref(n)))
            size = self._attend_work[(hq, nodes)] = (n.value + 15) // 16 * 16
        work = x.new_empty(size // 2)
        _call(_fast.tree_attention, self.device, self._ptr, layer, x.data_ptr(), hq, nodes, m.data_ptr(), HEAD_DIM ** -0.5 if scale is None else scale,
              out.data_ptr(), work.data_ptr(), size)
        return out

    def accept(self, ids, parents, targets, lens_out=None):
        """Keeps the branch of every tree that the model agrees with: from the root on the lowest child whose drafted token ``ids`` is the model's
        own ``targets`` of the node above (all int32 [rows, nodes]); its keys and values move to the slots behind ``lens``.  Returns
        (count [rows], next token [rows], path [rows, nodes], new lengths [rows]); the cache's own lengths change only where they
        are given as ``lens_out``."""
        if ids.dim() != 2:
            raise ValueError(f"ids must be an int32 tensor [{self.rows}, nodes]")
        torch, nodes = _torch(), ids.shape[1]
        shape = (self.rows, nodes)
        i, p, t = self._int32(ids, shape, "ids"), self._int32(parents, shape, "parents"), self._int32(targets, shape, "targets")
        if lens_out is None:
            lens_out = torch.empty_like(self.lens)
        elif self._int32(lens_out, (self.rows,), "lens_out") is not lens_out:
            raise ValueError("lens_out must be contiguous")
        count, token, path = torch.empty_like(self.lens), torch.empty_like(self.lens), torch.empty_like(i)
        _call(_fast.tree_accept, self.device, self._ptr, i.data_ptr(), p.data_ptr(), t.data_ptr(), nodes, count.data_ptr(), token.data_ptr(), path.data_ptr(),
              lens_out.data_ptr())
        return count, token, path, lens_out


@functools.lru_cache(maxsize=64)
def _beam_work(groups: int, beams: int, vocab: int, k: int) -> int:
    n = C.c_uint64()
    check(lib.mfqb_beam_select_work(groups, beams, vocab, k, C.byref(n)))
    return (n.value + 15) // 16 * 16


def beam_select(logits, scores, k: int, done=None, eos: int = -1):
    """The ``k`` best continuations of every group by ``scores + log_softmax(logits)``, largest first: ``logits`` float32 [groups, beams, vocab],
    ``scores`` float32 [groups, beams], ``done`` int32 [groups, beams] (a beam with a non-zero entry goes on as itself with token
    ``eos``).  Returns (scores float32 [groups, k], rows int32 [groups, k] = group * beams + beam, tokens int32 [groups, k]);
    equal candidates: the lower beam, then the larger logit, then the lower token.  A NaN or plus infinity among a beam's logits makes all
    its candidates' scores minus infinity; what is masked out is minus infinity."""
    torch = _torch()
    if logits.dim() != 3 or not logits.is_cuda:
        raise ValueError("logits must be a float32 CUDA tensor [groups, beams, vocab]")
    g, w, vocab = logits.shape
    dev = logits.get_device()
    z = _need(logits, torch.float32, logits.shape, dev, "logits")
    sc = _need(scores, torch.float32, (g, w), dev, "scores")
    dn = None if done is None else _need(done, torch.int32, (g, w), dev, "done")
    size = _beam_work(g, w, vocab, k)
    work = z.new_empty(size // 4)
    out, rows = z.new_empty((g, k)), z.new_empty((g, k), dtype=torch.int32)
    tokens = torch.empty_like(rows)
    _call(_fast.beam_select, dev, z.data_ptr(), g, w, vocab, sc.data_ptr(), None if dn is None else dn.data_ptr(), eos, k, out.data_ptr(), rows.data_ptr(),
          tokens.data_ptr(), work.data_ptr(), size)
    return out, rows, tokens
