"""The paged 8-bit KV cache, attention over it and sampling
(``rce_qmm_kv_*``, ``rce_qmm_sample_dev`` in include/rce_qmm.h): what a
program that steps many sequences with ``mm_batched_dev`` needs between the
projections and after the head.  Everything works on device addresses and is
asynchronous on the given stream (None: the context's); there is no CPU path.
"""
from __future__ import annotations

import ctypes

import numpy as np

from ._lib import QmmError, check, lib
from .qmm import Context, DeviceBuffer, _ptr

__all__ = ["KvCache", "KvBatch", "Rope", "kv_append_dev", "kv_read_dev", "kv_attention_dev", "sample_dev"]


class _Cache(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "v", "k_scale", "v_scale")] + \
               [(n, ctypes.c_size_t) for n in ("n_pages", "page_tokens", "n_kv_heads", "d_head")]


class _Batch(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("row_offsets", "seq_lens", "pages")] + \
               [(n, ctypes.c_size_t) for n in ("n_seqs", "n_rows", "max_pages")]


class _Rope(ctypes.Structure):
    _fields_ = [("cs", ctypes.c_void_p), ("dim", ctypes.c_size_t), ("n_pos", ctypes.c_size_t)]


class _Sampling(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("u", "temperature", "top_k", "top_p", "min_p")]


class KvCache:
    """A pool of pages (rce_qmm_kv_cache): device addresses of the key and
    value codes and their scales, in the layout the header gives."""

    def __init__(self, n_pages: int, page_tokens: int, n_kv_heads: int, d_head: int, k: int = 0, v: int = 0,
                 k_scale: int = 0, v_scale: int = 0):
        self.c = _Cache(k or None, v or None, k_scale or None, v_scale or None, n_pages, page_tokens, n_kv_heads, d_head)
        self.buffers: tuple = ()

    @classmethod
    def allocate(cls, ctx: Context, n_pages: int, page_tokens: int, n_kv_heads: int, d_head: int) -> "KvCache":
        """A pool in device memory of its own (contents undefined), freed by
        ``free`` or with the object."""
        c = cls(n_pages, page_tokens, n_kv_heads, d_head)
        codes, scales = c.sizes()
        c.buffers = tuple(DeviceBuffer(ctx, n) for n in (codes, codes, 4 * scales, 4 * scales))
        c.c.k, c.c.v, c.c.k_scale, c.c.v_scale = (b.ptr for b in c.buffers)
        return c

    def sizes(self) -> tuple[int, int]:
        """(bytes of the key codes, and of the value codes; scales of each)."""
        b, n = ctypes.c_size_t(), ctypes.c_size_t()
        check(lib().rce_qmm_kv_sizes(ctypes.byref(self.c), ctypes.byref(b), ctypes.byref(n)))
        return b.value, n.value

    def free(self) -> None:
        for b in self.buffers:
            b.free()
        self.buffers = ()


class KvBatch:
    """The rows of a call and their sequences (rce_qmm_kv_batch): device
    addresses of row_offsets [n_seqs + 1], seq_lens [n_seqs] and pages
    [n_seqs][max_pages], all int32."""

    def __init__(self, row_offsets: int, seq_lens: int, pages: int, n_seqs: int, n_rows: int, max_pages: int):
        self.c = _Batch(row_offsets or None, seq_lens or None, pages or None, n_seqs, n_rows, max_pages)


class Rope:
    """A rotation table on the device (rce_qmm_rope)."""

    def __init__(self, cs: int, dim: int, n_pos: int):
        self.c = _Rope(cs or None, dim, n_pos)
        self.buffer: DeviceBuffer | None = None

    @staticmethod
    def table(freq_base: float, dim: int, n_pos: int) -> np.ndarray:
        """The decoder's table [n_pos, dim / 2, 2] (rce_qmm_rope_table)."""
        if dim % 2 or dim < 0 or n_pos < 0:
            raise QmmError(2, "dim must be even, n_pos not negative")
        out = np.empty((n_pos, dim // 2, 2), np.float32)
        check(lib().rce_qmm_rope_table(freq_base, dim, n_pos, _ptr(out)))
        return out

    @classmethod
    def upload(cls, ctx: Context, freq_base: float, dim: int, n_pos: int) -> "Rope":
        b = DeviceBuffer.from_numpy(ctx, cls.table(freq_base, dim, n_pos))
        r = cls(b.ptr, dim, n_pos)
        r.buffer = b
        return r


def _p(a: int | None) -> ctypes.c_void_p:
    return ctypes.c_void_p(a or None)


def _ref(x):
    return ctypes.byref(x.c) if x is not None else None


def kv_append_dev(ctx: Context, cache: KvCache, batch: KvBatch, k_dev: int, v_dev: int, dtype, k_stride: int,
                  v_stride: int, rope: Rope | None = None, stream: int | None = None) -> None:
    """Quantize and append the batch's rows of keys (rotated) and values
    (rce_qmm_kv_append_dev); strides in values from row to row."""
    check(lib().rce_qmm_kv_append_dev(ctx.handle, _ref(cache), _ref(batch), _p(k_dev), k_stride, _p(v_dev), v_stride,
                                      int(dtype), _ref(rope), _p(stream)))


def kv_read_dev(ctx: Context, cache: KvCache, batch: KvBatch, k_out: int | None, v_out: int | None, dtype,
                stream: int | None = None) -> None:
    """The cached values of the batch's rows (rce_qmm_kv_read_dev)."""
    check(lib().rce_qmm_kv_read_dev(ctx.handle, _ref(cache), _ref(batch), _p(k_out), _p(v_out), int(dtype), _p(stream)))


def kv_attention_dev(ctx: Context, cache: KvCache, batch: KvBatch, q_dev: int, q_dtype, q_stride: int, n_q_heads: int,
                     out_dev: int, out_dtype, scale: float, rope: Rope | None = None, window: int = 0,
                     out_stride: int | None = None, stream: int | None = None) -> None:
    """Causal attention of the batch's query rows over the cache
    (rce_qmm_kv_attention_dev); out_stride None: rows without gaps."""
    check(lib().rce_qmm_kv_attention_dev(ctx.handle, _ref(cache), _ref(batch), _p(q_dev), int(q_dtype), q_stride, n_q_heads,
                                         _ref(rope), scale, window, _p(out_dev), int(out_dtype),
                                         n_q_heads * cache.c.d_head if out_stride is None else out_stride, _p(stream)))


def sample_dev(ctx: Context, logits_dev: int, dtype, n_rows: int, vocab: int, row_stride: int, u_dev: int, ids_dev: int,
               probs_dev: int | None = None, temperature_dev: int | None = None, top_k_dev: int | None = None,
               top_p_dev: int | None = None, min_p_dev: int | None = None, stream: int | None = None) -> None:
    """One token per row from its logits and its uniform number
    (rce_qmm_sample_dev); a filter without an array is off."""
    s = _Sampling(u_dev or None, temperature_dev or None, top_k_dev or None, top_p_dev or None, min_p_dev or None)
    check(lib().rce_qmm_sample_dev(ctx.handle, _p(logits_dev), int(dtype), n_rows, vocab, row_stride, ctypes.byref(s),
                                   _p(ids_dev), _p(probs_dev), _p(stream)))
