"""Calls on a paged cache that are made right or refused on the host (no GPU needed)."""

import contextlib
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from test_paged_cache import A, _says, _view  # noqa: E402
from tyloquant_b200 import cache as M  # noqa: E402
from tyloquant_b200._capi import lib  # noqa: E402


def test_outputs_over_inputs_are_refused():
    """Values of nodes that are no numbers are added after rows were written, with the queries read again."""
    v, n = C.byref(_view()), C.c_uint64()
    assert lib.mfqb_tree_attention_work(v, 4, 2, C.byref(n)) == 0
    size = 3 * 2 * 4 * 256   # q and out: 3 sequences, 2 nodes, 4 heads
    for out in (A, A + 16, A + size - 16, A - size + 16):
        _says(1, "overlap", lib.mfqb_tree_attention(v, 0, A, 4, 2, A + (1 << 24), 1.0, out, A + (1 << 25), n.value, None))
    x_size = 3 * 2 * (4 + 4) * 512   # qkv: 4 query heads, 2 + 2 of keys and values
    for out in (A, A + 16, A + x_size - 16, A - size + 16):
        _says(1, "overlap", lib.mfqb_cache_write(v, 0, A, 4, 2, A + (1 << 24), A + (1 << 25), out, None))


class _OtherDevice:
    """torch with device 0 current, and a stream number for each device."""

    def __init__(self):
        self.now, self._C = 0, self
        self.cuda = self

    def _cuda_getDevice(self):
        return self.now

    def _cuda_getCurrentRawStream(self, device):
        return 1000 + device

    @contextlib.contextmanager
    def device(self, device):
        old, self.now = self.now, device
        yield
        self.now = old


def test_calls_while_another_device_is_current(monkeypatch):
    """The call is made with the cache's device current and on that device's stream, and the old one is current again behind it."""
    fake = _OtherDevice()
    monkeypatch.setattr(M, "_torch", lambda: fake)
    seen = []

    def fn(*args):
        seen.append((fake.now, args))
        return 0

    M._call(fn, 0, "a", 1)
    M._call(fn, 1, "b", 2)
    assert seen == [(0, ("a", 1, 1000)), (1, ("b", 2, 1001))] and fake.now == 0
