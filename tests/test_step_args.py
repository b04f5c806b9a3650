"""What the entry points of routing, head norms with rotation, page tables
and attention with sinks refuse, on the host (nothing here reaches a device),
and the scaled rotation tables."""
import math
import struct

import numpy as np
import pytest

import rce_amd
from rce_amd import GgufDtype as G
from rce_amd import _lib
from test_kv_args import BAD, BAD_BATCHES, BAD_CACHES, DTYPE, NULL, FakeContext, batch, cache, refused

M = 1 << 20


def sinks(c, b, rope=None, q=8 * M, qt=G.F32, qs=256, n_q=4, out=9 * M, ot=G.F32, scale=0.125, window=9, n=4, os=256):
    rce_amd.kv_attention_sinks_dev(FakeContext(), c, b, q, qt, qs, n_q, out, ot, scale, window, n, rope=rope, out_stride=os)


def reserve(c, b, refs=8 * M, missing=9 * M):
    rce_amd.kv_reserve_dev(FakeContext(), c, b, refs, missing)


@pytest.mark.parametrize("call", [sinks, reserve])
def test_caches_and_batches(call):
    for kw, st in BAD_CACHES:
        refused(st, call, cache(**kw), batch())
    for kw, st in BAD_BATCHES:
        refused(st, call, cache(), batch(**kw))
    refused(NULL, call, None, batch())
    refused(NULL, call, cache(), None)


def test_sinks():
    for kw, st in ((dict(q=0), NULL), (dict(out=0), NULL), (dict(qs=255), BAD), (dict(os=255), BAD), (dict(n_q=3), BAD),
                   (dict(scale=-1.0), BAD), (dict(scale=float("nan")), BAD), (dict(qt=G.Q8_0), DTYPE), (dict(ot=G.Q8_0), DTYPE),
                   (dict(q=M + 2), BAD), (dict(out=M + 1), BAD), (dict(rope=rce_amd.Rope(M, 64, 63)), BAD)):
        refused(st, sinks, cache(), batch(), **kw)
    refused(BAD, sinks, cache(), batch(max_pages=0))
    sinks(cache(), batch(n_rows=0), q=0, out=0, n=(1 << 64) - 1)


# ---- page tables ---------------------------------------------------------------------

def table(pages=8 * M, n_seqs=3, max_pages=5):
    return rce_amd.KvTable(pages, n_seqs, max_pages)


def fork(c, a, b, parents=9 * M, refs=10 * M):
    rce_amd.kv_fork_dev(FakeContext(), c, a, b, parents, refs)


def release(c, t, refs=9 * M, **kw):
    rce_amd.kv_release_dev(FakeContext(), c, t, refs, **kw)


def compact(c, t, refs=9 * M, new_ids=10 * M, n_used=None):
    rce_amd.kv_compact_dev(FakeContext(), c, t, refs, new_ids, n_used)


def copy(a, b, src=9 * M, dst=10 * M, n=2):
    rce_amd.kv_copy_dev(FakeContext(), a, b, src, dst, n)


SHAPES = [(kw, st) for kw, st in BAD_CACHES if st == BAD and not {"k", "v", "k_scale", "v_scale"} & set(kw)]
BAD_TABLES = [(dict(pages=0), NULL), (dict(pages=M + 2), BAD), (dict(n_seqs=M + 1), BAD), (dict(max_pages=1 << 31), BAD),
              (dict(n_seqs=M, max_pages=2048), BAD), (dict(max_pages=(1 << 64) - 1), BAD)]


def test_tables():
    for f in (lambda t: fork(cache(), t, table()), lambda t: fork(cache(), table(), t), lambda t: release(cache(), t),
              lambda t: compact(cache(), t)):
        for kw, st in BAD_TABLES:
            refused(st, f, table(**kw))
        refused(NULL, f, None)
    for f in (lambda c: fork(c, table(), table()), lambda c: release(c, table()), lambda c: compact(c, table()), lambda c: copy(c, cache()),
              lambda c: copy(cache(), c)):
        for kw, st in SHAPES:
            refused(st, f, cache(**kw))
        refused(NULL, f, None)
    for kw, st in ((dict(parents=0), NULL), (dict(refs=0), NULL), (dict(parents=M + 1), BAD), (dict(refs=M + 2), BAD)):
        refused(st, fork, cache(), table(), table(), **kw)
    for kw, st in ((dict(refs=0), NULL), (dict(refs=M + 2), BAD), (dict(from_dev=M + 1), BAD), (dict(to_dev=M + 2), BAD)):
        refused(st, release, cache(), table(), **kw)
    for kw, st in ((dict(refs=0), NULL), (dict(refs=M + 2), BAD), (dict(missing=M + 2), BAD)):
        refused(st, reserve, cache(), batch(), **kw)
    for kw, st in ((dict(refs=0), NULL), (dict(new_ids=0), NULL), (dict(new_ids=M + 1), BAD), (dict(n_used=M + 2), BAD)):
        refused(st, compact, cache(), table(), **kw)
    refused(BAD, compact, cache(n_pages=(1 << 23) + 1, n_kv_heads=1), table())


def test_copies():
    for kw in (dict(page_tokens=64), dict(n_kv_heads=4), dict(d_head=128)):
        refused(BAD, copy, cache(), cache(**kw))
    for kw, st in ((dict(k=0), NULL), (dict(v_scale=0), NULL), (dict(v=M + 8), BAD)):
        refused(st, copy, cache(), cache(**kw))
        refused(st, copy, cache(**kw), cache())
        refused(st, compact, cache(**kw), table())
    for kw, st in ((dict(src=0), NULL), (dict(dst=0), NULL), (dict(src=M + 2), BAD), (dict(dst=M + 1), BAD), (dict(n=1 << 31), BAD)):
        refused(st, copy, cache(), cache(), **kw)


def test_empty_table_calls_do_nothing():
    for kw in (dict(n_seqs=0), dict(max_pages=0), dict(n_seqs=0, pages=0)):
        fork(cache(), table(), table(**kw), parents=0, refs=0)
        release(cache(), table(**kw), refs=0)
    copy(cache(), cache(n_pages=9), n=0, src=0, dst=0)
    reserve(cache(), batch(n_seqs=0), refs=0)
    reserve(cache(), batch(n_rows=0, row_offsets=0, seq_lens=0, pages=0), missing=None)


def test_null_contexts():
    L = _lib.lib()
    c, t, b = cache().raw, table().raw, batch().raw
    assert L.rce_qmm_kv_fork_dev(None, c, t, t, M, M, None) == NULL
    assert L.rce_qmm_kv_release_dev(None, c, t, None, None, M, None) == NULL
    assert L.rce_qmm_kv_reserve_dev(None, c, b, M, None, None) == NULL
    assert L.rce_qmm_kv_compact_dev(None, c, t, M, M, None, None) == NULL
    assert L.rce_qmm_kv_copy_dev(None, c, c, M, M, 1, None) == NULL
    assert L.rce_qmm_qk_norm_rope_dev(None, b, None, None, 64, 0, 0, 1e-6, None, 0, None) == NULL
    assert L.rce_qmm_moe_route_dev(None, M, 0, 1, 8, 8, rce_amd.MoeRouting(2).raw, M, M, None) == NULL
    assert L.rce_qmm_moe_route_dev(FakeContext().handle, M, 0, 1, 8, 8, None, M, M, None) == NULL


# ---- norms and rotation of heads ---------------------------------------------------------

def heads(**kw):
    a = dict(in_dev=8 * M, in_stride=256, n_heads=4, out_dev=9 * M, out_stride=256)
    a.update(kw)
    return rce_amd.Heads(**a)


def norm(q, k=None, b=None, d=64, it=G.F32, ot=G.F32, eps=1e-6, rope=None):
    rce_amd.qk_norm_rope_dev(FakeContext(), batch() if b is None else b, q, k, d, it, ot, eps, rope=rope)


def test_heads():
    wide = heads(in_stride=4096, out_stride=4096)
    for kw, st in ((dict(d=0), BAD), (dict(d=63), BAD), (dict(d=1026), BAD), (dict(it=G.Q8_0), DTYPE), (dict(ot=77), DTYPE),
                   (dict(eps=float("nan")), BAD), (dict(eps=float("inf")), BAD), (dict(rope=rce_amd.Rope(0, 64, 64)), NULL),
                   (dict(rope=rce_amd.Rope(M, 66, 64)), BAD), (dict(rope=rce_amd.Rope(M, 7, 64)), BAD),
                   (dict(rope=rce_amd.Rope(M + 2, 8, 64)), BAD), (dict(b=batch(row_offsets=0)), NULL), (dict(b=batch(seq_lens=0)), NULL),
                   (dict(b=batch(row_offsets=M + 2)), BAD), (dict(b=batch(n_seqs=M + 1)), BAD), (dict(b=batch(n_rows=(1 << 27) + 1)), BAD)):
        refused(st, norm, wide, **kw)
    for kw, st in ((dict(in_dev=0), NULL), (dict(out_dev=0), NULL), (dict(in_stride=255), BAD), (dict(out_stride=255), BAD),
                   (dict(in_dev=M + 2), BAD), (dict(out_dev=M + 1), BAD), (dict(weight=M + 2), BAD), (dict(n_heads=1 << 40), BAD),
                   (dict(out_dev=8 * M, out_stride=260), BAD)):
        refused(st, norm, heads(**kw))
        refused(st, norm, None, heads(**kw))
    refused(BAD, norm, heads(out_dev=8 * M), ot=G.F16)  # in place with another size
    refused(BAD, norm, heads(n_heads=M, in_stride=64 * M, out_stride=64 * M), b=batch(n_rows=65))
    with pytest.raises(rce_amd.QmmError):
        rce_amd.qk_norm_rope_dev(FakeContext(), None, heads(), None, 64, G.F32, G.F32)


def test_empty_head_calls_do_nothing():
    norm(None)
    norm(heads(n_heads=0, in_dev=0, out_dev=0))
    for kw in (dict(n_rows=0), dict(n_seqs=0, row_offsets=0, seq_lens=0)):
        norm(heads(in_dev=0), b=batch(**kw))


# ---- routing -----------------------------------------------------------------------------

def route(lg=M, dtype=G.F32, n=2, e=16, stride=16, ids=2 * M, w=3 * M, top_k=2, **kw):
    rce_amd.moe_route_dev(FakeContext(), lg, dtype, n, e, stride, rce_amd.MoeRouting(top_k, **kw), ids, w)


def test_routing():
    for kw, st in ((dict(lg=0), NULL), (dict(ids=0), NULL), (dict(w=0), NULL), (dict(lg=M + 2), BAD), (dict(ids=M + 2), BAD),
                   (dict(w=M + 1), BAD), (dict(bias_dev=M + 2), BAD), (dict(stride=15), BAD), (dict(e=0), BAD), (dict(e=1025, stride=1025), BAD),
                   (dict(n=(1 << 24) + 1), BAD), (dict(top_k=0), BAD), (dict(top_k=-1), BAD), (dict(top_k=17), BAD), (dict(e=256, stride=256, top_k=65), BAD),
                   (dict(dtype=G.Q4_0), DTYPE), (dict(n_group=3), BAD), (dict(n_group=4, topk_group=0), BAD),
                   (dict(n_group=4, topk_group=5), BAD), (dict(n_group=8, topk_group=1, top_k=3), BAD),
                   (dict(n_group=4, topk_group=2, group_top=0), BAD), (dict(n_group=4, topk_group=2, group_top=3), BAD),
                   (dict(e=130, stride=130, n_group=65, topk_group=3), BAD), (dict(scale=float("nan")), BAD), (dict(scale=float("inf")), BAD), (dict(scale=1e300), BAD)):
        refused(st, route, **kw)
    bad = bytearray(rce_amd.MoeRouting(2).raw)
    bad[0:4] = (2).to_bytes(4, "little")  # no such scores
    assert _lib.lib().rce_qmm_moe_route_dev(FakeContext().handle, M, 0, 1, 8, 8, bytes(bad), M, M, None) == BAD
    route(n=0, lg=0, ids=0, w=0)
    with pytest.raises(rce_amd.QmmError):
        rce_amd.MoeRouting(1 << 65)


# ---- scaled rotation tables ------------------------------------------------------------------

def angles(base, dim, n_pos, factor=1.0, divisors=None, orig=0, fast=32.0, slow=1.0):
    """Angles [n_pos, dim / 2] in the widest floats at hand."""
    L = np.longdouble
    i = np.arange(dim // 2).astype(L)
    f = L(base) ** (-2 * i / L(dim))
    if divisors is not None:
        f = f / np.asarray(divisors, np.float32).astype(L)
    keep = np.zeros(dim // 2, L)
    if orig:
        pair = lambda t: dim * math.log(orig / (t * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        low, high = max(0, math.floor(pair(fast))), min(dim - 1, math.ceil(pair(slow)))
        keep = 1 - np.clip((i - low) / max(0.001, high - low), 0, 1)
    f = f * keep + f / L(np.float32(factor)) * (1 - keep)
    return np.arange(n_pos).astype(L)[:, None] * f


@pytest.mark.parametrize("base,dim,n_pos,kw", [
    (10000.0, 128, 70, {}), (10000.0, 2, 9, {}), (500000.0, 64, 131073, dict(factor=8.0)),
    (10000.0, 128, 40000, dict(factor=16.0, orig_context=4096)), (1e6, 96, 3000, dict(factor=4.0, orig_context=32768, beta_fast=24.0, beta_slow=2.0)),
    (500000.0, 128, 9000, dict(divisors=True)), (10000.0, 64, 500, dict(factor=4.0, magnitude=0.1 * math.log(4.0) + 1.0)),
    (10000.0, 32, 50, dict(factor=2.5, orig_context=10))])
def test_scaled_tables(base, dim, n_pos, kw):
    """Angles below 2^18 in 64 bits are within 2^18 * 2^-50 of theirs (the power, two quotients, the blend
    and the product: under 8 roundings), far below a rounding to binary32."""
    kw = dict(kw)
    if kw.get("divisors"):
        kw["divisors"] = np.linspace(1, 8, dim // 2, dtype=np.float32)
    got = rce_amd.Rope.scaled_table(base, dim, n_pos, **kw)
    th = angles(base, dim, n_pos, kw.get("factor", 1.0), kw.get("divisors"), kw.get("orig_context", 0), kw.get("beta_fast", 32.0), kw.get("beta_slow", 1.0))
    m = np.float64(np.float32(kw.get("magnitude", 1.0)))
    want = np.stack([np.cos(th), np.sin(th)], -1).astype(np.float64) * m
    assert got.shape == (n_pos, dim // 2, 2) and got.dtype == np.float32
    assert np.all(np.abs(got - want) <= 2.0 ** -24 * np.abs(want) + 2.0 ** -31)


def test_scaled_tables_refused():
    t = rce_amd.Rope.scaled_table
    for kw in (dict(factor=0.0), dict(factor=-1.0), dict(factor=float("inf")), dict(factor=float("nan")), dict(magnitude=0.0),
               dict(divisors=[1.0, 0.0]), dict(divisors=[1.0, float("nan")]), dict(divisors=[1.0]), dict(orig_context=8, beta_fast=0.0),
               dict(orig_context=8, beta_slow=float("inf")), dict(orig_context=1 << 70), dict(factor=1e300)):
        refused(BAD, t, 10000.0, 4, 3, **kw)
    for args in ((0.0, 4, 3), (float("inf"), 4, 3), (float("nan"), 4, 3), (1e4, 3, 3), (1e4, -2, 3), (1e4, 4, -1)):
        refused(BAD, t, *args)
    refused(BAD, t, 0.5, 4, 3, orig_context=8)
    L = _lib.lib()
    assert L.rce_qmm_rope_table_scaled(1e4, 4, 3, None, M) == NULL
    assert L.rce_qmm_rope_table_scaled(1e4, 4, 3, struct.pack("@ffPNff", 1.0, 1.0, 0, 0, 32.0, 1.0), None) == NULL
    assert t(1e4, 0, 5).shape == (5, 0, 2) and t(1e4, 4, 0).shape == (0, 2, 2)
