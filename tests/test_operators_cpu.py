"""What the embedding and windowed-attention calls refuse before anything could run, without a GPU."""

import ctypes as C

import pytest
import torch

import mcsparse_b200 as mc
from mcsparse_b200 import capi
from mcsparse_b200.capi import lib

INVALID, REFUSED = capi.MCSPARSE_STATUS_INVALID_VALUE, capi.MCSPARSE_STATUS_NOT_SUPPORTED


class Stub:
    """A handle nobody created, on a stream of the CPU: the library answers NOT_INITIALIZED once Python's checks have passed."""
    h = None
    pointer_mode = capi.MCSPARSE_POINTER_MODE_HOST

    class stream:
        device_index = -1  # what a CPU tensor reports


def test_window_descriptor():
    d = C.c_void_p()

    def create(window=8, sinks=0, hq=4, hk=2, dim=64, scale=0.125, kind=capi.MACA_R_16BF, out=C.byref(d)):
        return lib.mcsparseB200CreateWindow(out, window, sinks, hq, hk, dim, scale, kind)

    assert create(out=None) == INVALID
    for bad in (dict(window=0), dict(window=-1), dict(sinks=-1), dict(hq=0), dict(hk=0), dict(hk=3), dict(dim=0), dict(scale=float("nan")),
                dict(scale=float("inf"))):
        assert create(**bad) == INVALID, bad
    for bad in (dict(dim=129), dict(kind=capi.MACA_R_64F), dict(kind=capi.MACA_R_8I)):
        assert create(**bad) == REFUSED, bad
    assert create(window=1 << 62, sinks=1 << 62) == 0
    assert lib.mcsparseB200DestroyWindow(d) == 0 and lib.mcsparseB200DestroyWindow(None) == 0
    with pytest.raises(mc.McsparseError):
        mc.Window(0, 0, 1, 1, 64, torch.bfloat16)
    with pytest.raises(ValueError):
        mc.Window(1, 0, 1, 1, 64, torch.int64)


def test_null_handle():
    size = C.c_size_t()
    one = C.c_float(1.0)
    w = mc.Window(4, 1, 2, 1, 64, torch.float16)
    h = C.byref(capi.Heads(256, 128, 64))
    c = C.byref(capi.Cache(256, 128, 64, 64))
    never = capi.MCSPARSE_STATUS_NOT_INITIALIZED
    assert lib.mcsparseB200EmbeddingLookup(None, C.byref(one), 1, 256, 2, 0, None, None) == never
    assert lib.mcsparseB200EmbeddingGradient_bufferSize(None, 1, 2, None, None, C.byref(size)) == never
    assert lib.mcsparseB200EmbeddingGradient(None, C.byref(one), 1, 256, 2, 0, None, C.byref(one), None, 256) == never
    assert lib.mcsparseB200WindowAttention(None, w.d, 1, None, None, 1, 1, h, h, h, h, None) == never
    assert lib.mcsparseB200WindowAttentionBackward_bufferSize(None, w.d, 1, 1, 1, C.byref(size)) == never
    assert lib.mcsparseB200WindowAttentionBackward(None, w.d, 1, None, None, 1, 1, h, h, h, h, 256, h, h, h, h, 256) == never
    assert lib.mcsparseB200WindowAttentionDecode_bufferSize(None, w.d, 1, 1, 1, C.byref(size)) == never
    assert lib.mcsparseB200WindowAttentionDecode(None, w.d, 1, 256, h, c, c, 1, 1, None, 1, h, None, 256) == never


def test_tensors_are_checked_before_the_call():
    w = mc.Window(4, 1, 2, 1, 64, torch.float16)
    q, k = torch.zeros(5, 2, 64, dtype=torch.float16), torch.zeros(5, 1, 64, dtype=torch.float16)
    with pytest.raises(mc.McsparseError):  # nothing to object to but the handle
        mc.window_attention(Stub, w, q, k, k, q.clone())
    for bad in (lambda: mc.window_attention(Stub, w, q.float(), k, k, q), lambda: mc.window_attention(Stub, w, q, q, k, q),
                lambda: mc.window_attention(Stub, w, q, k, k[:4], q), lambda: mc.window_attention(Stub, w, q, k, k, q[..., :32]),
                lambda: mc.window_attention(Stub, w, q.transpose(1, 2).contiguous().transpose(1, 2), k, k, q),
                lambda: mc.window_attention(Stub, w, q, k, k, q, torch.zeros(5, 2)),
                lambda: mc.window_attention(Stub, w, q, k, k, q, q_offsets=torch.zeros(2)),
                lambda: mc.window_attention(Stub, w, q, k, k, q, q_offsets=torch.zeros(2, dtype=torch.int32), k_offsets=torch.zeros(3, dtype=torch.int32)),
                lambda: mc.window_attention_decode(Stub, w, q, k[None], k[None], torch.zeros(5, dtype=torch.int32), q, buffer=torch.zeros(1)),
                lambda: mc.window_attention_decode(Stub, w, q, k, k, torch.zeros(5, dtype=torch.int32), q)):
        with pytest.raises(ValueError):
            bad()
    ids = torch.zeros(3, dtype=torch.int64)
    table, y = mc.DnMat(torch.zeros(4, 8), 4, 8, 8), mc.DnMat(torch.zeros(3, 8), 3, 8, 8)
    with pytest.raises(mc.McsparseError):
        mc.embedding_lookup(Stub, ids, table, y)
    for bad in (lambda: mc.embedding_lookup(Stub, ids.double(), table, y), lambda: mc.embedding_lookup(Stub, ids[None], table, y),
                lambda: mc.embedding_lookup(Stub, torch.zeros(6, dtype=torch.int64)[::2], table, y)):
        with pytest.raises(ValueError):
            bad()
    grad = lambda buffer, **kw: mc.embedding_gradient(Stub, ids, y, table, buffer, **kw)
    with pytest.raises(mc.McsparseError):  # the buffer's size is asked first
        grad(torch.zeros(64, dtype=torch.uint8))


def test_gradient_buffers_and_scalars(monkeypatch):
    from mcsparse_b200 import operators
    monkeypatch.setattr(operators, "embedding_gradient_buffer_size", lambda *a: 64)
    monkeypatch.setattr(operators, "_GRADIENT_SIZES", {})

    class Device(Stub):
        pointer_mode = capi.MCSPARSE_POINTER_MODE_DEVICE

    ids = torch.zeros(3, dtype=torch.int64)
    table, y = mc.DnMat(torch.zeros(4, 8), 4, 8, 8), mc.DnMat(torch.zeros(3, 8), 3, 8, 8)
    room, one = torch.zeros(64, dtype=torch.uint8), torch.ones(1)
    for handle, scalars in ((Stub, {}), (Device, dict(alpha=one, beta=one))):
        for buffer in (None, room[:63], room.float(), torch.zeros(128, dtype=torch.uint8)[::2]):
            with pytest.raises(ValueError):
                mc.embedding_gradient(handle, ids, y, table, buffer, **scalars)
        with pytest.raises(mc.McsparseError):  # nothing to object to but the handle
            mc.embedding_gradient(handle, ids, y, table, room, **scalars)
    for bad in (1.0, one.double(), torch.ones(2)):  # a scalar of the host, of another type or size
        with pytest.raises(ValueError):
            mc.embedding_gradient(Device, ids, y, table, room, alpha=bad, beta=one)

    class Elsewhere(Device):
        class stream:
            device_index = 0

    with pytest.raises(ValueError):  # a scalar on another device than the handle's
        operators._scalar(Elsewhere, one)
