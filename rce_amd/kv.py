"""The paged 8-bit KV cache, its pages, norms and rotation of heads, attention
and sampling (``rce_qmm_kv_*``, ``rce_qmm_qk_norm_rope_dev``,
``rce_qmm_sample_dev`` in include/rce_qmm.h): what a program that steps many
sequences with ``mm_batched_dev`` needs between the projections and after the
head.  Everything works on device addresses and is
asynchronous on the given stream (None: the context's); there is no CPU path.
"""
from __future__ import annotations

import ctypes
import struct

import numpy as np

from ._lib import QmmError, check, lib
from .qmm import Context, DeviceBuffer, _ptr

__all__ = ["KvCache", "KvBatch", "KvTable", "Rope", "Heads", "kv_append_dev", "kv_read_dev", "kv_attention_dev",
           "kv_attention_sinks_dev", "qk_norm_rope_dev", "kv_copy_dev", "kv_fork_dev", "kv_release_dev",
           "kv_reserve_dev", "kv_compact_dev", "sample_dev"]


# The header's structs as bytes: made once per object, passed as they are (a
# decode step makes several calls of a few microseconds each).
_CACHE = struct.Struct("@PPPPNNNN")
_BATCH = struct.Struct("@PPPNNN")
_ROPE = struct.Struct("@PNN")
_SAMPLING = struct.Struct("@PPPPP")
_TABLE = struct.Struct("@PNN")
_HEADS = struct.Struct("@PNPNPN")
_SCALING = struct.Struct("@ffPNff")


def _range(e: struct.error) -> QmmError:
    return QmmError(2, f"an address or a size is out of range: {e}")


def _pack(fmt: struct.Struct, *values: int) -> bytes:
    try:
        return fmt.pack(*values)
    except struct.error as e:
        raise _range(e) from None


class KvCache:
    """A pool of pages (rce_qmm_kv_cache): device addresses of the key and
    value codes and their scales, in the layout the header gives."""

    __slots__ = ("raw", "d_head", "buffers")

    def __init__(self, n_pages: int, page_tokens: int, n_kv_heads: int, d_head: int, k: int = 0, v: int = 0,
                 k_scale: int = 0, v_scale: int = 0):
        try:
            self.raw = _CACHE.pack(k, v, k_scale, v_scale, n_pages, page_tokens, n_kv_heads, d_head)
        except struct.error as e:
            raise _range(e) from None
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
        try:
            self.raw = _BATCH.pack(row_offsets, seq_lens, pages, n_seqs, n_rows, max_pages)
        except struct.error as e:
            raise _range(e) from None


class Rope:
    """A rotation table on the device (rce_qmm_rope)."""

    __slots__ = ("raw", "buffer")

    def __init__(self, cs: int, dim: int, n_pos: int):
        try:
            self.raw = _ROPE.pack(cs, dim, n_pos)
        except struct.error as e:
            raise _range(e) from None
        self.buffer: DeviceBuffer | None = None

    @staticmethod
    def table(freq_base: float, dim: int, n_pos: int) -> np.ndarray:
        """The decoder's table [n_pos, dim / 2, 2] (rce_qmm_rope_table)."""
        if dim % 2 or dim < 0 or n_pos < 0:
            raise QmmError(2, "dim must be even, n_pos not negative")
        out = np.empty((n_pos, dim // 2, 2), np.float32)
        check(lib().rce_qmm_rope_table(freq_base, dim, n_pos, _ptr(out)))
        return out

    @staticmethod
    def scaled_table(freq_base: float, dim: int, n_pos: int, factor: float = 1.0, divisors=None, orig_context: int = 0,
                     beta_fast: float = 32.0, beta_slow: float = 1.0, magnitude: float = 1.0) -> np.ndarray:
        """A table [n_pos, dim / 2, 2] for long contexts, by angles in 64
        bits (rce_qmm_rope_table_scaled): frequencies divided by `divisors`
        (one per pair) and by `factor`, with `orig_context` the slow pairs'
        only, between beta_fast and beta_slow turns over it."""
        if dim % 2 or dim < 0 or n_pos < 0:
            raise QmmError(2, "dim must be even, n_pos not negative")
        if divisors is not None:
            divisors = np.ascontiguousarray(divisors, np.float32)
            if divisors.shape != (dim // 2,):
                raise QmmError(2, "divisors must be one value per pair")
        out = np.empty((n_pos, dim // 2, 2), np.float32)
        how = _pack(_SCALING, factor, magnitude, 0 if divisors is None else divisors.ctypes.data, orig_context, beta_fast, beta_slow)
        check(lib().rce_qmm_rope_table_scaled(freq_base, dim, n_pos, how, _ptr(out)))
        return out

    @classmethod
    def upload(cls, ctx: Context, freq_base: float, dim: int, n_pos: int, **scaling) -> "Rope":
        """The decoder's table on the device, or with any of
        ``scaled_table``'s arguments that one."""
        make = cls.scaled_table if scaling else cls.table
        b = DeviceBuffer.from_numpy(ctx, make(freq_base, dim, n_pos, **scaling))
        r = cls(b.ptr, dim, n_pos)
        r.buffer = b
        return r


class KvTable:
    """Sequences' page tables (rce_qmm_kv_table): device address of pages
    [n_seqs][max_pages] int32, -1 where there is no page."""

    __slots__ = ("raw",)

    def __init__(self, pages: int, n_seqs: int, max_pages: int):
        try:
            self.raw = _TABLE.pack(pages, n_seqs, max_pages)
        except struct.error as e:
            raise _range(e) from None


class Heads:
    """Query or key heads of ``qk_norm_rope_dev`` (rce_qmm_heads): device
    addresses, strides in values from row to row; weight 0: ones."""

    __slots__ = ("raw",)

    def __init__(self, in_dev: int, in_stride: int, n_heads: int, out_dev: int, out_stride: int, weight: int = 0):
        try:
            self.raw = _HEADS.pack(in_dev, in_stride, out_dev, out_stride, weight, n_heads)
        except struct.error as e:
            raise _range(e) from None


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


def kv_attention_sinks_dev(ctx: Context, cache: KvCache, batch: KvBatch, q_dev: int, q_dtype, q_stride: int, n_q_heads: int,
                           out_dev: int, out_dtype, scale: float, window: int, sinks: int, rope: Rope | None = None,
                           out_stride: int | None = None, stream: int | None = None) -> None:
    """``kv_attention_dev`` with a window and `sinks` first positions that
    every row sees (rce_qmm_kv_attention_sinks_dev)."""
    if out_stride is None and cache is not None:
        out_stride = n_q_heads * cache.d_head
    st = lib().rce_qmm_kv_attention_sinks_dev(ctx.handle, cache and cache.raw, batch and batch.raw, q_dev, q_dtype, q_stride,
                                              n_q_heads, rope and rope.raw, scale, window, sinks, out_dev, out_dtype, out_stride or 0, stream)
    if st:
        check(st)


def qk_norm_rope_dev(ctx: Context, batch: KvBatch, q: Heads | None, k: Heads | None, d_head: int, in_dtype, out_dtype,
                     eps: float | None = None, rope: Rope | None = None, interleaved: bool = False,
                     stream: int | None = None) -> None:
    """Norms (eps None: none) and rotation of query and key heads in one
    pass (rce_qmm_qk_norm_rope_dev)."""
    st = lib().rce_qmm_qk_norm_rope_dev(ctx.handle, batch and batch.raw, q and q.raw, k and k.raw, d_head, in_dtype, out_dtype,
                                        -1.0 if eps is None else eps, rope and rope.raw, interleaved, stream)
    if st:
        check(st)


def kv_copy_dev(ctx: Context, src: KvCache, dst: KvCache, src_ids_dev: int, dst_ids_dev: int, n: int,
                stream: int | None = None) -> None:
    """Pages of one pool to pages of another, or of itself (rce_qmm_kv_copy_dev)."""
    st = lib().rce_qmm_kv_copy_dev(ctx.handle, src and src.raw, dst and dst.raw, src_ids_dev, dst_ids_dev, n, stream)
    if st:
        check(st)


def kv_fork_dev(ctx: Context, cache: KvCache, src: KvTable, dst: KvTable, parents_dev: int, refs_dev: int,
                stream: int | None = None) -> None:
    """Every sequence of `dst` gets its parent's pages in `src`
    (rce_qmm_kv_fork_dev)."""
    st = lib().rce_qmm_kv_fork_dev(ctx.handle, cache and cache.raw, src and src.raw, dst and dst.raw, parents_dev, refs_dev, stream)
    if st:
        check(st)


def kv_release_dev(ctx: Context, cache: KvCache, table: KvTable, refs_dev: int, from_dev: int | None = None,
                   to_dev: int | None = None, stream: int | None = None) -> None:
    """Give up the pages wholly in positions from .. to - 1 of each sequence
    (rce_qmm_kv_release_dev; None: all)."""
    st = lib().rce_qmm_kv_release_dev(ctx.handle, cache and cache.raw, table and table.raw, from_dev, to_dev, refs_dev, stream)
    if st:
        check(st)


def kv_reserve_dev(ctx: Context, cache: KvCache, batch: KvBatch, refs_dev: int, missing_dev: int | None = None,
                   stream: int | None = None) -> None:
    """Pages of their own for the batch's rows, written into its tables
    (rce_qmm_kv_reserve_dev)."""
    st = lib().rce_qmm_kv_reserve_dev(ctx.handle, cache and cache.raw, batch and batch.raw, refs_dev, missing_dev, stream)
    if st:
        check(st)


def kv_compact_dev(ctx: Context, cache: KvCache, table: KvTable, refs_dev: int, new_ids_dev: int,
                   n_used_dev: int | None = None, stream: int | None = None) -> None:
    """The used pages to the front of the pool (rce_qmm_kv_compact_dev)."""
    st = lib().rce_qmm_kv_compact_dev(ctx.handle, cache and cache.raw, table and table.raw, refs_dev, new_ids_dev, n_used_dev, stream)
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
