"""The calls of routing, heads, pages and sinks on other streams than their
context's and on other contexts: the same bits; rows further apart than 2^31
values."""
import numpy as np
import pytest

import kv_case as kc
import rce_amd
import serve_case as sc
from kv_case import F32
from rce_amd import GgufDtype as G

pytestmark = pytest.mark.gpu


def everything(c, up, stream):
    """All calls once, one after the other on one stream; their results."""
    rng = np.random.default_rng(50)
    heads, per, d, page, n, max_pages, n_pages, e = 2, 2, 64, 16, 3, 60, 190, 128
    n_q = heads * per
    news = np.array([5, 1, 700])
    lens = np.array([300, 900, 760])
    rows = int(news.sum())
    off, ln = up(np.concatenate([[0], np.cumsum(news)]).astype(np.int32)), up(lens.astype(np.int32))
    pool = kc.Pool(n_pages, page, heads, d, rng)
    bufs = [up(getattr(pool, name)) for name in ("k", "v", "k_scale", "v_scale")]
    cache = rce_amd.KvCache(n_pages, page, heads, d, *(b.ptr for b in bufs[:2]), *(b.ptr for b in bufs[2:]))
    first = np.full((n, max_pages), -1, np.int32)
    ids = rng.permutation(n_pages)[:60]
    first[0, :19], first[1, :30], first[2, :4] = ids[:19], ids[10:40], ids[40:44]
    refs = up(np.bincount(first[first >= 0], minlength=n_pages).astype(np.int32))
    a, b = up(first), up(np.full((n, max_pages), -1, np.int32))
    ta, tb = (rce_amd.KvTable(x.ptr, n, max_pages) for x in (a, b))
    parents, missing, new_ids, used = up(np.array([0, 1, 2], np.int32)), up(np.zeros(n, np.int32)), up(np.zeros(n_pages, np.int32)), up(np.zeros(1, np.int32))
    width = (n_q + 2 * heads) * d
    x = up(rng.standard_normal((rows, width)).astype(F32))
    qk, out = up(np.zeros((rows, (n_q + heads) * d), F32)), up(np.zeros((rows, n_q * d), F32))
    w = up((1 + 0.1 * rng.standard_normal(d)).astype(F32))
    cs = up(rce_amd.Rope.table(10000.0, d, max_pages * page))
    lg, bias = up(rng.standard_normal((rows, e)).astype(F32)), up((0.1 * rng.standard_normal(e)).astype(F32))
    eid, ew = up(np.zeros((rows, 8), np.int32)), up(np.zeros((rows, 8), F32))
    src, dst = up(np.array([3], np.int32)), up(np.array([3], np.int32))
    kw = {"stream": stream}
    batch = rce_amd.KvBatch(off.ptr, ln.ptr, b.ptr, n, rows, max_pages)
    h = lambda at, count, col: rce_amd.Heads(x.ptr + 4 * at * d, width, count, qk.ptr + 4 * col * d, (n_q + heads) * d, w.ptr)  # noqa: E731
    rce_amd.qk_norm_rope_dev(c, batch, h(0, n_q, 0), h(n_q, heads, n_q), d, G.F32, G.F32, 1e-5, rope=rce_amd.Rope(cs.ptr, d, max_pages * page), **kw)
    rce_amd.kv_fork_dev(c, cache, ta, tb, parents.ptr, refs.ptr, **kw)
    rce_amd.kv_reserve_dev(c, cache, batch, refs.ptr, missing.ptr, **kw)
    rce_amd.kv_append_dev(c, cache, batch, qk.ptr + 4 * n_q * d, x.ptr + 4 * (n_q + heads) * d, G.F32, (n_q + heads) * d, width, **kw)
    rce_amd.kv_release_dev(c, cache, ta, refs.ptr, **kw)
    rce_amd.kv_compact_dev(c, cache, tb, refs.ptr, new_ids.ptr, used.ptr, **kw)
    rce_amd.kv_copy_dev(c, cache, cache, src.ptr, dst.ptr, 0, **kw)
    rce_amd.kv_attention_sinks_dev(c, cache, batch, qk.ptr, G.F32, (n_q + heads) * d, n_q, out.ptr, G.F32, 0.125, 400, 20, **kw)
    rce_amd.moe_route_dev(c, lg.ptr, G.F32, rows, e, e, rce_amd.MoeRouting(8, sigmoid=True, bias_dev=bias.ptr, n_group=4, topk_group=2, group_top=2),
                          eid.ptr, ew.ptr, **kw)
    return [qk, out, eid, ew, refs, a, b, missing, new_ids, used, *bufs]


def test_same_bits_on_streams_and_contexts(ctx):
    results = []
    with rce_amd.Context(0) as other:
        for c, stream in ((ctx, None), (ctx, other.stream), (other, None), (other, ctx.stream), (other, 0)):
            held = []

            def up(arr):
                held.append(rce_amd.DeviceBuffer.from_numpy(ctx, arr))
                return held[-1]
            outs = everything(c, up, stream)
            ctx.synchronize()
            other.synchronize()
            results.append([b.download(np.uint8, b.nbytes) for b in outs])
            for b in held:
                b.free()
    assert np.isfinite(results[0][1].view(F32)).all() and results[0][1].any()
    for r in results[1:]:
        for p, q in zip(results[0], r):
            assert np.array_equal(p, q)


def test_calls_at_once_on_two_contexts():
    """Two contexts' reservations, compactions and attention queued together: neither sees the other's plan."""
    with rce_amd.Context(0) as c0, rce_amd.Context(0) as c1:
        held = []

        def up(arr):
            held.append(rce_amd.DeviceBuffer.from_numpy(c0, arr))
            return held[-1]
        alone = everything(c0, up, None)
        c0.synchronize()
        want = [b.download(np.uint8, b.nbytes) for b in alone]
        for _ in range(3):
            both = [everything(c, up, None) for c in (c0, c1)]
            c0.synchronize()
            c1.synchronize()
            for outs in both:
                for b, w in zip(outs, want):
                    assert np.array_equal(b.download(np.uint8, b.nbytes), w)
        for b in held:
            b.free()


@pytest.mark.parametrize("d", [64, 66])
def test_rows_of_heads_far_apart(ctx, d):
    """in and out strides of 2^30 values and more."""
    rng = np.random.default_rng(d)
    stride, rows = (1 << 30) + 8, 3
    x = kc.to_bits(rng.standard_normal((rows, d)), G.F16)
    big = rce_amd.DeviceBuffer(ctx, 2 * (2 * stride + d))
    L = rce_amd._lib.lib()
    for r in range(rows):
        rce_amd._lib.check(L.rce_qmm_memcpy_h2d(ctx.handle, big.ptr + 2 * r * stride, x[r].ctypes.data, 2 * d))
    up = lambda a: rce_amd.DeviceBuffer.from_numpy(ctx, a)  # noqa: E731
    off, ln, cs = up(np.array([0, 3], np.int32)), up(np.array([9], np.int32)), rce_amd.Rope.table(10000.0, d, 9)
    table = up(cs)
    h = rce_amd.Heads(big.ptr, stride, 1, big.ptr, stride)
    rce_amd.qk_norm_rope_dev(ctx, rce_amd.KvBatch(off.ptr, ln.ptr, 0, 1, rows, 0), None, h, d, G.F16, G.F16, 1e-6, rope=rce_amd.Rope(table.ptr, d, 9))
    ctx.synchronize()
    for r in range(rows):
        got = np.empty(d, np.float16)
        rce_amd._lib.check(L.rce_qmm_memcpy_d2h(ctx.handle, got.ctypes.data, big.ptr + 2 * r * stride, 2 * d))
        y, b = sc.norm_rope(x[r:r + 1].astype(F32), None, 1e-6, cs, 6 + r, False)
        assert np.all(np.abs(got - y[0]) <= b[0] + 2.0 ** -11 * (np.abs(y[0]) + b[0]) + 2.0 ** -25)
    for b in (big, off, ln, table):
        b.free()
