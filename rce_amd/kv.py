"""The paged 8-bit KV cache, attention over it and sampling
(``rce_qmm_kv_*``, ``rce_qmm_sample_dev`` in include/rce_qmm.h): what a
program that steps many sequences with ``mm_batched_dev`` needs between the
projections and after the head.  Everything works on device addresses and is
asynchronous on the given stream (None: the context's); there is no CPU path.
"""
from __future__ import annotations

import ctypes
import struct

import numpy as np

from ._lib import QmmError, check, lib
from .qmm import Context, DeviceBuffer, _ptr

__all__ = ["KvCache", "KvBatch", "Rope", "kv_append_dev", "kv_read_dev", "kv_attention_dev", "sample_dev"]


# The header's structs as bytes: made once per object, passed as they are (a
# decode step makes several calls of a few microseconds each).
_CACHE = struct.Struct("@PPPPNNNN")
_BATCH = struct.Struct("@PPPNNN")
_ROPE = struct.Struct("@PNN")
_SAMPLING = struct.Struct("@PPPPP")


def _pack(fmt: struct.Struct, *values: int) -> bytes:
    try:
        return fmt.pack(*values)
    except struct.error as e:
        raise QmmError(2, f"an address or a size is out of range: {e}") from None


class KvCache:
    """A pool of pages (rce_qmm_kv_cache): device addresses of the key and
    value codes and their scales, in the layout the header gives."""

    __slots__ = ("raw", "d_head", "buffers")

    def __init__(self, n_pages: int, page_tokens: int, n_kv_heads: int, d_head: int, k: int = 0, v: int = 0,
                 k_scale: int = 0, v_scale: int = 0):
        self.raw = _pack(_CACHE, k, v, k_scale, v_scale, n_pages, page_tokens, n_kv_heads, d_head)
        self.d_head = d_head
        self.buffers: tuple = ()

    @classmethod
    def allocate(cls, ctx: Context, n_pages: int, page_tokens: int, n_kv_heads: int, d_head: int) -> "KvCache":
        """A pool in device memory of its own (contents undefined), freed by
        ``free`` or with the object."""
        shape = (n_pages, page_tokens, n_kv_heads, d_head)
        codes, scales = cls(*shape).sizes()
        buffers = tuple(DeviceBuffer(ctx, n) for n in (codes, codes, 4 * scales, 4 * scales))
        c = cls(*shape, *(b.ptr for b in buffers))
        c.buffers = buffers
        return c

    def sizes(self) -> tuple[int, int]:
        """(bytes of the key codes, and of the value codes; scales of each)."""
        b, n = ctypes.c_size_t(), ctypes.c_size_t()
        check(lib().rce_qmm_kv_sizes(self.raw, ctypes.byref(b), ctypes.byref(n)))
        return b.value, n.value

    def free(self) -> None:
        """Free a pool that ``allocate`` made: later calls with it are refused
        (a null cache buffer)."""
        if self.buffers:
            self.raw = _pack(_CACHE, 0, 0, 0, 0, *_CACHE.unpack(self.raw)[4:])
        for b in self.buffers:
            b.free()
        self.buffers = ()


class KvBatch:
    """The rows of a call and their sequences (rce_qmm_kv_batch): device
    addresses of row_offsets [n_seqs + 1], seq_lens [n_seqs] and pages
    [n_seqs][max_pages], all int32."""

    __slots__ = ("raw",)

    def __init__(self, row_offsets: int, seq_lens: int, pages: int, n_seqs: int, n_rows: int, max_pages: int):
        self.raw = _pack(_BATCH, row_offsets, seq_lens, pages, n_seqs, n_rows, max_pages)


class Rope:
    """A rotation table on the device (rce_qmm_rope)."""

    __slots__ = ("raw", "buffer")

    def __init__(self, cs: int, dim: int, n_pos: int):
        self.raw = _pack(_ROPE, cs, dim, n_pos)
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


def _raw(x) -> bytes | None:
    return None if x is None else x.raw


def kv_append_dev(ctx: Context, cache: KvCache, batch: KvBatch, k_dev: int, v_dev: int, dtype, k_stride: int,
                  v_stride: int, rope: Rope | None = None, stream: int | None = None) -> None:
    """Quantize and append the batch's rows of keys (rotated) and values
    (rce_qmm_kv_append_dev); strides in values from row to row."""
    st = lib().rce_qmm_kv_append_dev(ctx.handle, _raw(cache), _raw(batch), k_dev, k_stride, v_dev, v_stride, dtype,
                                     _raw(rope), stream)
    if st:
        check(st)


def kv_read_dev(ctx: Context, cache: KvCache, batch: KvBatch, k_out: int | None, v_out: int | None, dtype,
                stream: int | None = None) -> None:
    """The cached values of the batch's rows (rce_qmm_kv_read_dev)."""
    st = lib().rce_qmm_kv_read_dev(ctx.handle, _raw(cache), _raw(batch), k_out, v_out, dtype, stream)
    if st:
        check(st)


def kv_attention_dev(ctx: Context, cache: KvCache, batch: KvBatch, q_dev: int, q_dtype, q_stride: int, n_q_heads: int,
                     out_dev: int, out_dtype, scale: float, rope: Rope | None = None, window: int = 0,
                     out_stride: int | None = None, stream: int | None = None) -> None:
    """Causal attention of the batch's query rows over the cache
    (rce_qmm_kv_attention_dev); out_stride None: rows without gaps."""
    if out_stride is None and cache is not None:
        out_stride = n_q_heads * cache.d_head
    st = lib().rce_qmm_kv_attention_dev(ctx.handle, _raw(cache), _raw(batch), q_dev, q_dtype, q_stride, n_q_heads, _raw(rope),
                                        scale, window, out_dev, out_dtype, out_stride or 0, stream)
    if st:
        check(st)


def sample_dev(ctx: Context, logits_dev: int, dtype, n_rows: int, vocab: int, row_stride: int, u_dev: int, ids_dev: int,
               probs_dev: int | None = None, temperature_dev: int | None = None, top_k_dev: int | None = None,
               top_p_dev: int | None = None, min_p_dev: int | None = None, stream: int | None = None) -> None:
    """One token per row from its logits and its uniform number
    (rce_qmm_sample_dev); a filter without an array is off."""
    s = _pack(_SAMPLING, u_dev or 0, temperature_dev or 0, top_k_dev or 0, top_p_dev or 0, min_p_dev or 0)
    st = lib().rce_qmm_sample_dev(ctx.handle, logits_dev, dtype, n_rows, vocab, row_stride, s, ids_dev, probs_dev, stream)
    if st:
        check(st)
