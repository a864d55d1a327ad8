"""Products with matrices that are never stored, over the C API: embedding rows and their gradient, windowed attention.

Thin calls into ``capi.lib`` like :mod:`mcsparse_b200.host`: torch supplies device memory and streams, all arithmetic
happens in libmcsparse.so. Every call is asynchronous on the handle's stream; tensors that live on another device than the
handle's, or that have another type or shape than the call needs, are refused with ``ValueError`` before anything runs.
"""

import ctypes as C
import math

import torch

from . import capi
from .capi import check, lib
from .host import _DTYPE, _ptr, _scalar


def _index_type(indices):
    if indices.dtype == torch.int64:
        return capi.MCSPARSE_INDEX_64I
    if indices.dtype == torch.int32:
        return capi.MCSPARSE_INDEX_32I
    raise ValueError(f"indices must be int32 or int64, got {indices.dtype}")


def _float_scalar(handle, value):
    """A float as a C argument: a host scalar, or a one-element fp32 device tensor in device pointer mode."""
    if handle.pointer_mode == capi.MCSPARSE_POINTER_MODE_DEVICE:
        if not (isinstance(value, torch.Tensor) and value.dtype == torch.float32 and value.numel() == 1 and value.is_cuda):
            raise ValueError("device pointer mode: alpha and beta are one-element float32 device tensors")
        return _ptr(value), value
    v = _scalar(value, torch.float32)
    return C.cast(C.byref(v), C.c_void_p), v


def _same_device(handle, *tensors):
    device = handle.stream.device
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"tensor on {t.device}, handle on {device}")


def _indices(handle, indices):
    _same_device(handle, indices)
    if indices.dim() != 1 or not (indices.is_contiguous() or indices.numel() <= 1):
        raise ValueError("indices must be one contiguous row")
    return _index_type(indices)


def embedding_lookup(handle, indices, E, Y, alpha=1.0, base=0):
    """Y[t] = alpha * E[indices[t] - base]; a row of zeros for an index outside the table. E, Y: ``DnMat`` in row order."""
    kind = _indices(handle, indices)
    _same_device(handle, E.values, Y.values)
    pa, keep = _float_scalar(handle, alpha)
    check(lib.mcsparseB200EmbeddingLookup(handle.h, pa, indices.numel(), _ptr(indices), kind, base, E.d, Y.d),
          "mcsparseB200EmbeddingLookup")
    del keep


def embedding_gradient_buffer_size(handle, indices, dY, dE):
    size = C.c_size_t()
    check(lib.mcsparseB200EmbeddingGradient_bufferSize(handle.h, indices.numel(), _index_type(indices), dY.d, dE.d,
                                                       C.byref(size)), "mcsparseB200EmbeddingGradient_bufferSize")
    return size.value


def _buffer(handle, buffer, need):
    """The caller's work buffer, checked: its device, type and size."""
    _same_device(handle, buffer)
    if buffer.dtype != torch.uint8 or not buffer.is_contiguous() or buffer.numel() < need:
        raise ValueError(f"the work buffer must be {need} contiguous bytes (uint8) or more")
    return _ptr(buffer)


def embedding_gradient(handle, indices, dY, dE, buffer, alpha=1.0, beta=0.0, base=0):
    """dE = alpha * S^T dY + beta * dE, S the 0/1 matrix of the indices. Indices outside the table contribute nothing."""
    kind = _indices(handle, indices)
    _same_device(handle, dY.values, dE.values)
    work = _buffer(handle, buffer, embedding_gradient_buffer_size(handle, indices, dY, dE))
    pa, keep_a = _float_scalar(handle, alpha)
    pb, keep_b = _float_scalar(handle, beta)
    check(lib.mcsparseB200EmbeddingGradient(handle.h, pa, indices.numel(), _ptr(indices), kind, base, dY.d, pb, dE.d, work),
          "mcsparseB200EmbeddingGradient")
    del keep_a, keep_b


class Window:
    """mcsparseB200WindowDescr_t: the pattern (window, sinks) and the heads of a windowed attention.

    ``scale`` defaults to 1 / sqrt(head_dim)."""

    def __init__(self, window, sinks, q_heads, kv_heads, head_dim, dtype, scale=None):
        self.window, self.sinks = int(window), int(sinks)
        self.q_heads, self.kv_heads, self.head_dim = int(q_heads), int(kv_heads), int(head_dim)
        self.dtype = dtype
        self.scale = 1.0 / math.sqrt(head_dim) if scale is None and head_dim > 0 else float(scale or 0.0)
        self.d = None
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


def _heads(handle, t, tokens, heads, window, what):
    """mcsparseB200Heads_t of a tokens x heads x head_dim tensor with consecutive values in its last dimension."""
    _same_device(handle, t)
    if t.dtype != window.dtype or tuple(t.shape) != (tokens, heads, window.head_dim):
        raise ValueError(f"{what}: {t.dtype} {tuple(t.shape)}, expected {window.dtype} {(tokens, heads, window.head_dim)}")
    if window.head_dim > 1 and t.stride(2) != 1:
        raise ValueError(f"{what}: the last dimension must be consecutive")
    return capi.Heads(_ptr(t).value, t.stride(0), t.stride(1))


def _offsets(handle, offsets, what):
    if offsets is None:
        return None
    _same_device(handle, offsets)
    if offsets.dtype != torch.int32 or offsets.dim() != 1 or offsets.numel() < 1 or not offsets.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 row of sequences + 1 offsets")
    return offsets


def _batch(handle, q_offsets, k_offsets):
    q_offsets, k_offsets = _offsets(handle, q_offsets, "q_offsets"), _offsets(handle, k_offsets, "k_offsets")
    if k_offsets is None:
        k_offsets = q_offsets
    if q_offsets is None and k_offsets is not None:
        raise ValueError("k_offsets without q_offsets")
    if q_offsets is None:
        return 1, None, None
    if q_offsets.numel() != k_offsets.numel():
        raise ValueError("q_offsets and k_offsets must describe the same number of sequences")
    return q_offsets.numel() - 1, _ptr(q_offsets), _ptr(k_offsets)


def _lse(handle, lse, shape):
    if lse is None:
        return None
    _same_device(handle, lse)
    if lse.dtype != torch.float32 or tuple(lse.shape) != shape or not lse.is_contiguous():
        raise ValueError(f"lse must be a contiguous float32 tensor of {shape}")
    return _ptr(lse)


def window_attention(handle, window, q, k, v, out, lse=None, q_offsets=None, k_offsets=None):
    """out = softmax(scale * q k^T on the window's pattern) v over a ragged batch (see mcsparseB200WindowAttention).

    q, out: queries x q_heads x head_dim; k, v: keys x kv_heads x head_dim, any token and head strides. q_offsets,
    k_offsets: int32 offsets of the sequences (k_offsets defaults to q_offsets; neither: one sequence). lse: q_heads x queries."""
    batch, qo, ko = _batch(handle, q_offsets, k_offsets)
    tq, tk = q.shape[0], k.shape[0]
    tensors = [_heads(handle, t, n, h, window, name) for t, n, h, name in (
        (q, tq, window.q_heads, "q"), (k, tk, window.kv_heads, "k"), (v, tk, window.kv_heads, "v"), (out, tq, window.q_heads, "out"))]
    check(lib.mcsparseB200WindowAttention(handle.h, window.d, batch, qo, ko, tq, tk, *(C.byref(t) for t in tensors),
                                          _lse(handle, lse, (window.q_heads, tq))), "mcsparseB200WindowAttention")


def window_attention_backward_buffer_size(handle, window, batch, total_q, total_k):
    size = C.c_size_t()
    check(lib.mcsparseB200WindowAttentionBackward_bufferSize(handle.h, window.d, batch, total_q, total_k, C.byref(size)),
          "mcsparseB200WindowAttentionBackward_bufferSize")
    return size.value


def window_attention_backward(handle, window, q, k, v, out, lse, dout, dq, dk, dv, buffer, q_offsets=None, k_offsets=None):
    """Gradients dq, dk, dv of :func:`window_attention`; ``out`` and ``lse`` are what it wrote."""
    batch, qo, ko = _batch(handle, q_offsets, k_offsets)
    tq, tk = q.shape[0], k.shape[0]
    hq, hk = window.q_heads, window.kv_heads
    t = [_heads(handle, x, n, h, window, name) for x, n, h, name in (
        (q, tq, hq, "q"), (k, tk, hk, "k"), (v, tk, hk, "v"), (out, tq, hq, "out"), (dout, tq, hq, "dout"), (dq, tq, hq, "dq"),
        (dk, tk, hk, "dk"), (dv, tk, hk, "dv"))]
    if lse is None:
        raise ValueError("the backward pass needs lse")
    p = [C.byref(x) for x in t]
    work = _buffer(handle, buffer, window_attention_backward_buffer_size(handle, window, batch, tq, tk))
    check(lib.mcsparseB200WindowAttentionBackward(handle.h, window.d, batch, qo, ko, tq, tk, *p[:4], _lse(handle, lse, (hq, tq)),
                                                  *p[4:], work), "mcsparseB200WindowAttentionBackward")


def window_attention_decode_buffer_size(handle, window, batch, max_pages, page_size=1):
    """Bytes for sequences of at most max_pages * page_size tokens."""
    size = C.c_size_t()
    check(lib.mcsparseB200WindowAttentionDecode_bufferSize(handle.h, window.d, batch, max_pages, page_size, C.byref(size)),
          "mcsparseB200WindowAttentionDecode_bufferSize")
    return size.value


def _cache(handle, t, window, what):
    _same_device(handle, t)
    if t.dtype != window.dtype or t.dim() != 4 or tuple(t.shape[2:]) != (window.kv_heads, window.head_dim):
        raise ValueError(f"{what}: {t.dtype} {tuple(t.shape)}, expected {window.dtype} (pages, page size, "
                         f"{window.kv_heads}, {window.head_dim})")
    if window.head_dim > 1 and t.stride(3) != 1:
        raise ValueError(f"{what}: the last dimension must be consecutive")
    return capi.Cache(_ptr(t).value, t.stride(0), t.stride(1), t.stride(2))


def window_attention_decode(handle, window, q, k_cache, v_cache, lengths, out, lse=None, buffer=None, page_table=None):
    """One query per sequence, the newest of ``lengths[b]`` tokens in a cache (see mcsparseB200WindowAttentionDecode).

    q, out: batch x q_heads x head_dim; k_cache, v_cache: pages x page size x kv_heads x head_dim; page_table: int32,
    batch x pages of a sequence (None: page b is all of sequence b); lse: batch x q_heads."""
    batch = q.shape[0]
    tq = [_heads(handle, t, batch, window.q_heads, window, name) for t, name in ((q, "q"), (out, "out"))]
    kc, vc = _cache(handle, k_cache, window, "k_cache"), _cache(handle, v_cache, window, "v_cache")
    if k_cache.shape[:2] != v_cache.shape[:2]:
        raise ValueError("k_cache and v_cache must hold the same pages")
    pages, page_size = k_cache.shape[:2]
    _same_device(handle, lengths, page_table)
    if lengths.dtype != torch.int32 or tuple(lengths.shape) != (batch,) or not lengths.is_contiguous():
        raise ValueError("lengths must be a contiguous int32 row, one per sequence")
    if page_table is None:
        max_pages = 1
        if pages < batch:
            raise ValueError("without a page table the cache holds a page for every sequence")
    else:
        if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != batch or not page_table.is_contiguous():
            raise ValueError("page_table must be a contiguous int32 tensor of batch x pages")
        max_pages = page_table.shape[1]
    if buffer is None:
        raise ValueError("a work buffer is needed (window_attention_decode_buffer_size)")
    work = _buffer(handle, buffer, window_attention_decode_buffer_size(handle, window, batch, max_pages, page_size))
    check(lib.mcsparseB200WindowAttentionDecode(handle.h, window.d, batch, _ptr(lengths), C.byref(tq[0]), C.byref(kc), C.byref(vc),
                                                pages, page_size, None if page_table is None else _ptr(page_table), max_pages,
                                                C.byref(tq[1]), _lse(handle, lse, (batch, window.q_heads)), work),
          "mcsparseB200WindowAttentionDecode")
