"""Attention where blocks serve the ends and beginnings of several sequences, at
every head size; pools whose codes pass 32-bit offsets; batches of single
tokens beside a long prompt."""
import numpy as np
import pytest

import kv_case as kc
import rce_amd
from kv_case import F32
from rce_amd import GgufDtype as G
from test_gpu_kv import Attn, check_attention, fused

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out_dtype,window", [(G.F32, 0), (G.F16, 0), (G.BF16, 27000)])
@pytest.mark.parametrize("d", [64, 128, 192, 256])
def test_long_tokens_in_line_of_every_head_size(ctx, d, out_dtype, window):
    """Five sequences of the same pages, six times over: 36 units and 13500 tiles per head, 53 cells
    of the line a block."""
    print(f"line d={d} {out_dtype.name} window={window}", flush=True)
    rng = np.random.default_rng(d)
    lens, news, page, heads, per, times = [30000, 27001, 29999, 64, 28500], [1, 1, 2, 1, 9], 512, 2, 2, 6
    one, n_pages = kc.make_batch(rng, [max(lens)], [1], page)
    pool = kc.Pool(n_pages, page, heads, d, rng)
    few = kc.Batch(lens, news, np.repeat(one.pages, len(lens), 0), page)
    batch = kc.Batch(lens * times, news * times, np.repeat(one.pages, len(lens) * times, 0), page)
    rows = few.n_rows

    def q_edit(x):
        x[rows:] = np.tile(x[:rows], (times - 1, 1))
    a = Attn(ctx, pool, batch, heads * per, G.F16, out_dtype, rope=d, window=window, q_edit=q_edit)
    a.call()
    ctx.synchronize()
    got = kc.widen(a.bits(), out_dtype).reshape(times, rows, heads * per, d).astype(np.float64)
    want, bound = kc.attention(pool, few, a.q[:rows], a.cs, a.scale, window, out_dtype == G.F32)
    a.free()
    far = np.abs(got - want) - (bound + kc.out_eps(out_dtype) * (np.abs(want) + bound) + 2.0 ** -25)
    assert far.max() <= 0, (far.max(), bound.max())


def test_codes_past_32_bit_offsets(ctx):
    """A pool of 1100 pages of 4 MiB (keys, and values): rows appended to its last pages, read back
    and attended to by single tokens and by a prompt."""
    n_big, page, heads, d, dtype = 1100, 4096, 8, 128, G.F16
    print("pool of 4.6 GB", flush=True)
    rng = np.random.default_rng(3)
    lens = [4200, 90]
    batch, n_pages = kc.make_batch(rng, lens, lens, page)
    pool = kc.Pool(n_pages, page, heads, d, rng)
    up = lambda b: np.where(b.pages >= 0, n_big - 1 - b.pages, b.pages).astype(np.int32)  # noqa: E731
    cache = rce_amd.KvCache.allocate(ctx, n_big, page, heads, d)
    raw, stride, ka, va, k, v = fused(rng, batch.n_rows, heads, d, dtype)
    cs = kc.rope_cs(d, batch.cap)
    x, pages, table = (rce_amd.DeviceBuffer.from_numpy(ctx, b) for b in (raw, up(batch), cs))
    rope = rce_amd.Rope(table.ptr, d, batch.cap)

    def device(b):
        arrays = [rce_amd.DeviceBuffer.from_numpy(ctx, y) for y in (b.offsets, np.asarray(b.lens, np.int32))]
        return rce_amd.KvBatch(arrays[0].ptr, arrays[1].ptr, pages.ptr, len(lens), b.n_rows, b.pages.shape[1]), arrays
    db, keep = device(batch)
    rce_amd.kv_append_dev(ctx, cache, db, x.ptr + ka * 2, x.ptr + va * 2, dtype, stride, stride, rope=rope)
    ctx.synchronize()
    kc.append(pool, batch, k, v, cs)
    out = [rce_amd.DeviceBuffer(ctx, batch.n_rows * heads * d * 4) for _ in range(2)]
    rce_amd.kv_read_dev(ctx, cache, db, out[0].ptr, out[1].ptr, G.F32)
    ctx.synchronize()
    got = [o.download(F32, batch.n_rows * heads * d).reshape(batch.n_rows, heads, d) for o in out]
    for r, s, pos in batch.rows():
        for g, name in zip(got, "kv"):
            assert np.array_equal(g[r], pool.values(name, batch.page_of(s, pos, n_pages), pos).astype(F32)), (name, r)
    for news in ([1, 1], [70, 90]):
        print(f"attention of {news} rows", flush=True)
        b = kc.Batch(lens, news, batch.pages, page)
        db, more = device(b)
        q = kc.to_bits(rng.standard_normal((b.n_rows, heads * d)).astype(F32), G.F16)
        qb = rce_amd.DeviceBuffer.from_numpy(ctx, q)
        rce_amd.kv_attention_dev(ctx, cache, db, qb.ptr, G.F16, heads * d, heads, out[0].ptr, G.F32, 0.088, rope=rope)
        ctx.synchronize()
        y = out[0].download(F32, b.n_rows * heads * d).reshape(b.n_rows, heads, d)
        want, bound = kc.attention(pool, b, q.astype(F32).reshape(b.n_rows, heads, d), cs, float(F32(0.088)), 0, True)
        assert np.all(np.abs(y - want) <= bound + 2.0 ** -24 * (np.abs(want) + bound))
        for z in (qb, *more):
            z.free()
    for z in (x, pages, table, *keep, *out):
        z.free()
    cache.free()


@pytest.mark.parametrize("out_dtype", [G.F32, G.F16])
@pytest.mark.parametrize("per,new,page", [(1, 1600, 4096), (4, 449, 64), (4, 449, 2048), (2, 900, 4096)])
def test_single_tokens_beside_a_long_prompt(ctx, per, new, page, out_dtype):
    """The prompt among so many single tokens that a sequence has few rows on average, in tables of
    a page each, short and long; empty sequences and rows behind the last one."""
    n, heads = 90, 8
    rng = np.random.default_rng(new)
    lens = [int(x) for x in rng.integers(1, 300, n)]
    news = [1] * n
    lens[n // 2], news[n // 2] = new + 60, new
    lens[5] = news[5] = news[9] = 0
    check_attention(ctx, 64, heads, per, page, lens, news, G.F16, out_dtype, rope=64, window=200, n_rows=sum(news) + 7)
