"""Products with matrices that are never stored, over the C API: embedding rows and their gradient, windowed attention.

Thin calls into ``capi.lib`` like :mod:`mcsparse_b200.host`: torch supplies device memory and streams, all arithmetic
happens in libmcsparse.so. Every call is asynchronous on the handle's stream; tensors that live on another device than the
handle's, or that have another type or shape than the call needs, are refused with ``ValueError`` before anything runs.
"""

import ctypes as C
import math
import struct
import threading

import torch

from . import capi
from .capi import check, lib
from .host import _DTYPE

_INDEX = {torch.int32: capi.MCSPARSE_INDEX_32I, torch.int64: capi.MCSPARSE_INDEX_64I}
_HEADS, _CACHE = C.sizeof(capi.Heads), C.sizeof(capi.Cache)
_pack4, _pack8, _pack_decode = (struct.Struct(f"{n}q").pack_into for n in (12, 24, 14))


class _Block(threading.local):
    """Room for the mcsparseB200Heads_t / mcsparseB200Cache_t of one call, side by side and addressed by their parts: the library
    copies them before the call returns."""

    def __init__(self):
        self.memory = (C.c_int64 * 24)()
        self.at = C.addressof(self.memory)


_block = _Block()
_GRADIENT_SIZES = {}  # buffer sizes asked for so far, by device, tokens and table


def _scalar(handle, value):
    """A float as a C argument: a host scalar, or a one-element fp32 device tensor in device pointer mode."""
    if handle.pointer_mode == capi.MCSPARSE_POINTER_MODE_DEVICE:
        if not (isinstance(value, torch.Tensor) and value.dtype == torch.float32 and value.numel() == 1
                and value.get_device() == handle.stream.device_index):
            raise ValueError("device pointer mode: alpha and beta are one-element float32 tensors on the handle's device")
        return value.data_ptr()
    return C.byref(C.c_float(value))


def _on_device(handle, *tensors):
    device = handle.stream.device_index
    for t in tensors:
        if t.get_device() != device:
            raise ValueError(f"tensor on {t.device}, handle on device {device}")


def _indices(handle, indices):
    kind = _INDEX.get(indices.dtype)
    if kind is None:
        raise ValueError(f"indices must be int32 or int64, got {indices.dtype}")
    if indices.dim() != 1 or not indices.is_contiguous():
        raise ValueError("indices must be one contiguous row")
    return kind


def embedding_lookup(handle, indices, E, Y, alpha=1.0, base=0):
    """Y[t] = alpha * E[indices[t] - base]; a row of zeros for an index outside the table. E, Y: ``DnMat`` in row order."""
    kind = _indices(handle, indices)
    _on_device(handle, indices, E.values, Y.values)
    check(lib.mcsparseB200EmbeddingLookup(handle.h, _scalar(handle, alpha), indices.numel(), indices.data_ptr(), kind, base, E.d, Y.d),
          "mcsparseB200EmbeddingLookup")


def embedding_gradient_buffer_size(handle, indices, dY, dE):
    size = C.c_size_t()
    check(lib.mcsparseB200EmbeddingGradient_bufferSize(handle.h, indices.numel(), _indices(handle, indices), dY.d, dE.d,
                                                       C.byref(size)), "mcsparseB200EmbeddingGradient_bufferSize")
    return size.value


def _buffer(buffer, need):
    """Address of the caller's work buffer, once it is large enough."""
    if buffer is None or buffer.dtype != torch.uint8 or not buffer.is_contiguous() or buffer.numel() < need:
        raise ValueError(f"the work buffer must be {need} contiguous bytes (uint8) or more")
    return buffer.data_ptr()


def embedding_gradient(handle, indices, dY, dE, buffer, alpha=1.0, beta=0.0, base=0):
    """dE = alpha * S^T dY + beta * dE, S the 0/1 matrix of the indices. Indices outside the table contribute nothing."""
    key = handle.stream.device_index, indices.numel(), dE.rows, dE.cols
    need = _GRADIENT_SIZES.get(key)
    if need is None:
        if len(_GRADIENT_SIZES) >= 1024:
            _GRADIENT_SIZES.clear()
        need = _GRADIENT_SIZES[key] = embedding_gradient_buffer_size(handle, indices, dY, dE)
    kind, work = _indices(handle, indices), _buffer(buffer, need)
    _on_device(handle, indices, dY.values, dE.values, buffer)
    check(lib.mcsparseB200EmbeddingGradient(handle.h, _scalar(handle, alpha), indices.numel(), indices.data_ptr(), kind, base, dY.d,
                                            _scalar(handle, beta), dE.d, work), "mcsparseB200EmbeddingGradient")


class Window:
    """mcsparseB200WindowDescr_t: the pattern (window, sinks) and the heads of a windowed attention.

    ``scale`` defaults to 1 / sqrt(head_dim)."""

    def __init__(self, window, sinks, q_heads, kv_heads, head_dim, dtype, scale=None):
        self.window, self.sinks = int(window), int(sinks)
        self.q_heads, self.kv_heads, self.head_dim = int(q_heads), int(kv_heads), int(head_dim)
        self.dtype = dtype
        self.scale = 1.0 / math.sqrt(head_dim) if scale is None and head_dim > 0 else float(scale or 0.0)
        self.d = None
        self._sizes = {}  # buffer sizes asked for so far
        if dtype not in _DTYPE:
            raise ValueError(f"no value type for {dtype}")
        d = C.c_void_p()
        check(lib.mcsparseB200CreateWindow(C.byref(d), self.window, self.sinks, self.q_heads, self.kv_heads, self.head_dim,
                                           self.scale, _DTYPE[dtype]), "mcsparseB200CreateWindow")
        self.d = d

    def __del__(self):
        if getattr(self, "d", None) is not None and lib is not None:  # lib is None at interpreter shutdown
            lib.mcsparseB200DestroyWindow(self.d)
            self.d = None

    def _size(self, handle, name, *sizes):
        """What the library's `name` call reports for these sizes."""
        key = (handle.stream.device_index, name, *sizes)
        need = self._sizes.get(key)
        if need is None:
            size = C.c_size_t()
            check(getattr(lib, name)(handle.h, self.d, *sizes, C.byref(size)), name)
            if len(self._sizes) >= 1024:
                self._sizes.clear()
            need = self._sizes[key] = size.value
        return need


def _heads(device, t, tokens, heads, window, what):
    """Address and strides of a tokens x heads x head_dim tensor with consecutive values in its last dimension."""
    if t.dtype is not window.dtype or t.shape != (tokens, heads, window.head_dim) or t.get_device() != device:
        raise ValueError(f"{what}: {t.dtype} {tuple(t.shape)} on {t.device}, expected {window.dtype} "
                         f"{(tokens, heads, window.head_dim)} on the handle's device")
    stride = t.stride()
    if stride[2] != 1 and window.head_dim > 1:
        raise ValueError(f"{what}: the last dimension must be consecutive")
    return t.data_ptr(), stride[0], stride[1]


def _offsets(device, q_offsets, k_offsets):
    """Sequences, and the addresses of their offsets."""
    if q_offsets is None:
        if k_offsets is not None:
            raise ValueError("k_offsets without q_offsets")
        return 1, None, None
    if k_offsets is None:
        k_offsets = q_offsets
    for t in (q_offsets, k_offsets) if k_offsets is not q_offsets else (q_offsets,):
        if t.dtype is not torch.int32 or t.dim() != 1 or t.shape[0] < 1 or not t.is_contiguous() or t.get_device() != device:
            raise ValueError("offsets must be a contiguous int32 row of sequences + 1 entries on the handle's device")
    n = q_offsets.shape[0]
    if k_offsets.shape[0] != n:
        raise ValueError("q_offsets and k_offsets must describe the same number of sequences")
    return n - 1, q_offsets.data_ptr(), k_offsets.data_ptr()


def _lse(device, lse, shape):
    if lse is None:
        return None
    if lse.dtype is not torch.float32 or lse.shape != shape or not lse.is_contiguous() or lse.get_device() != device:
        raise ValueError(f"lse must be a contiguous float32 tensor of {shape} on the handle's device")
    return lse.data_ptr()


def window_attention(handle, window, q, k, v, out, lse=None, q_offsets=None, k_offsets=None):
    """out = softmax(scale * q k^T on the window's pattern) v over a ragged batch (see mcsparseB200WindowAttention).

    q, out: queries x q_heads x head_dim; k, v: keys x kv_heads x head_dim, any token and head strides. q_offsets,
    k_offsets: int32 offsets of the sequences (k_offsets defaults to q_offsets; neither: one sequence). lse: q_heads x queries."""
    device = handle.stream.device_index
    tq, tk, hq, hk = q.shape[0], k.shape[0], window.q_heads, window.kv_heads
    _pack4(_block.memory, 0, *_heads(device, q, tq, hq, window, "q"), *_heads(device, k, tk, hk, window, "k"),
           *_heads(device, v, tk, hk, window, "v"), *_heads(device, out, tq, hq, window, "out"))
    batch, qo, ko = _offsets(device, q_offsets, k_offsets)
    p = _block.at
    check(lib.mcsparseB200WindowAttention(handle.h, window.d, batch, qo, ko, tq, tk, p, p + _HEADS, p + 2 * _HEADS, p + 3 * _HEADS,
                                          _lse(device, lse, (hq, tq))), "mcsparseB200WindowAttention")


def window_attention_backward_buffer_size(handle, window, batch, total_q, total_k):
    return window._size(handle, "mcsparseB200WindowAttentionBackward_bufferSize", batch, total_q, total_k)


def window_attention_backward(handle, window, q, k, v, out, lse, dout, dq, dk, dv, buffer, q_offsets=None, k_offsets=None):
    """Gradients dq, dk, dv of :func:`window_attention`; ``out`` and ``lse`` are what it wrote."""
    device = handle.stream.device_index
    tq, tk, hq, hk = q.shape[0], k.shape[0], window.q_heads, window.kv_heads
    _pack8(_block.memory, 0, *_heads(device, q, tq, hq, window, "q"), *_heads(device, k, tk, hk, window, "k"),
           *_heads(device, v, tk, hk, window, "v"), *_heads(device, out, tq, hq, window, "out"),
           *_heads(device, dout, tq, hq, window, "dout"), *_heads(device, dq, tq, hq, window, "dq"),
           *_heads(device, dk, tk, hk, window, "dk"), *_heads(device, dv, tk, hk, window, "dv"))
    batch, qo, ko = _offsets(device, q_offsets, k_offsets)
    if lse is None:
        raise ValueError("the backward pass needs lse")
    work = _buffer(buffer, window_attention_backward_buffer_size(handle, window, batch, tq, tk))
    _on_device(handle, buffer)
    p = _block.at
    check(lib.mcsparseB200WindowAttentionBackward(
        handle.h, window.d, batch, qo, ko, tq, tk, p, p + _HEADS, p + 2 * _HEADS, p + 3 * _HEADS, _lse(device, lse, (hq, tq)),
        p + 4 * _HEADS, p + 5 * _HEADS, p + 6 * _HEADS, p + 7 * _HEADS, work), "mcsparseB200WindowAttentionBackward")


def window_attention_decode_buffer_size(handle, window, batch, max_pages, page_size=1):
    """Bytes for sequences of at most max_pages * page_size tokens."""
    return window._size(handle, "mcsparseB200WindowAttentionDecode_bufferSize", batch, max_pages, page_size)


def _cache(device, t, window, what):
    shape = t.shape
    if (t.dtype is not window.dtype or len(shape) != 4 or shape[2] != window.kv_heads or shape[3] != window.head_dim
            or t.get_device() != device):
        raise ValueError(f"{what}: {t.dtype} {tuple(shape)} on {t.device}, expected {window.dtype} (pages, page size, "
                         f"{window.kv_heads}, {window.head_dim}) on the handle's device")
    stride = t.stride()
    if stride[3] != 1 and window.head_dim > 1:
        raise ValueError(f"{what}: the last dimension must be consecutive")
    return t.data_ptr(), stride[0], stride[1], stride[2]


def window_attention_decode(handle, window, q, k_cache, v_cache, lengths, out, lse=None, buffer=None, page_table=None):
    """One query per sequence, the newest of ``lengths[b]`` tokens in a cache (see mcsparseB200WindowAttentionDecode).

    q, out: batch x q_heads x head_dim; k_cache, v_cache: pages x page size x kv_heads x head_dim; page_table: int32,
    batch x pages of a sequence (None: page b is all of sequence b); lse: batch x q_heads."""
    device = handle.stream.device_index
    batch, hq = q.shape[0], window.q_heads
    _pack_decode(_block.memory, 0, *_heads(device, q, batch, hq, window, "q"), *_heads(device, out, batch, hq, window, "out"),
                 *_cache(device, k_cache, window, "k_cache"), *_cache(device, v_cache, window, "v_cache"))
    pages, page_size = k_cache.shape[:2]
    if v_cache.shape != k_cache.shape:
        raise ValueError("k_cache and v_cache must hold the same pages")
    if lengths.dtype is not torch.int32 or lengths.shape != (batch,) or not lengths.is_contiguous() or lengths.get_device() != device:
        raise ValueError("lengths must be a contiguous int32 row on the handle's device, one per sequence")
    if page_table is None:
        table, max_pages = None, 1
        if pages < batch:
            raise ValueError("without a page table the cache holds a page for every sequence")
    else:
        if (page_table.dtype is not torch.int32 or page_table.dim() != 2 or page_table.shape[0] != batch or not page_table.is_contiguous()
                or page_table.get_device() != device):
            raise ValueError("page_table must be a contiguous int32 tensor of batch x pages on the handle's device")
        table, max_pages = page_table.data_ptr(), page_table.shape[1]
    work = _buffer(buffer, window_attention_decode_buffer_size(handle, window, batch, max_pages, page_size))
    _on_device(handle, buffer)
    p = _block.at
    check(lib.mcsparseB200WindowAttentionDecode(handle.h, window.d, batch, lengths.data_ptr(), p, p + 2 * _HEADS, p + 2 * _HEADS + _CACHE,
                                                pages, page_size, table, max_pages, p + _HEADS, _lse(device, lse, (batch, hq)), work),
          "mcsparseB200WindowAttentionDecode")
