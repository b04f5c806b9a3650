"""The paged 8-bit KV cache on the GPU: append and read bit for bit against
the rule, attention against 64 bits within the error its arithmetic allows,
at ragged lengths, odd strides, every head size, masks that leave rows empty,
bad pages and non-finite values."""
import numpy as np
import pytest

import kv_case as kc
import rce_amd
from bench import Hip
from kv_case import F32
from rce_amd import GgufDtype as G

pytestmark = pytest.mark.gpu


def same_pool(a, b):
    for n in ("k", "v"):
        assert np.array_equal(getattr(a, n), getattr(b, n)), n
    for n in ("k_scale", "v_scale"):
        x, y = getattr(a, n), getattr(b, n)
        assert np.array_equal(np.isnan(x), np.isnan(y)) and np.array_equal(x[~np.isnan(x)], y[~np.isnan(y)]), n


def fused(rng, rows, heads, d, dtype, gap=0, lead=0, spread=True):
    """Keys and values as slices of one buffer [rows][lead + 2 heads d + gap]:
    (bytes, stride, k offset, v offset, k values, v values)."""
    w = lead + 2 * heads * d + gap
    x = rng.standard_normal((rows, w)).astype(F32)
    if spread:
        x *= np.exp(rng.standard_normal((rows, 1))).astype(F32)
    raw = kc.to_bits(x, dtype)
    val = kc.widen(raw, dtype)
    k = val[:, lead:lead + heads * d].reshape(rows, heads, d)
    v = val[:, lead + heads * d:lead + 2 * heads * d].reshape(rows, heads, d)
    return raw, w, lead, lead + heads * d, k, v


def run_append(ctx, dev, raw, stride, k_at, v_at, dtype, stream=None):
    size = raw.dtype.itemsize
    x = rce_amd.DeviceBuffer.from_numpy(ctx, raw)
    rce_amd.kv_append_dev(ctx, dev.cache, dev.b, x.ptr + k_at * size, x.ptr + v_at * size, dtype, stride, stride,
                          rope=dev.rope, stream=stream)
    ctx.synchronize()
    x.free()


def check_append(ctx, d, heads, page, dtype, rope, lens, news, gap=0, lead=0, seed=1, n_rows=None, edit=None, pages=None):
    print(f"append d={d} heads={heads} page={page} {dtype.name} rope={rope} lens={lens} news={news} gap={gap}", flush=True)
    rng = np.random.default_rng(seed)
    batch, n_pages = kc.make_batch(rng, lens, news, page, n_rows=n_rows)
    if pages:
        pages(batch, n_pages)
    pool = kc.Pool(n_pages, page, heads, d, rng)
    cs = kc.rope_cs(rope, batch.cap)
    raw, stride, ka, va, k, v = fused(rng, batch.n_rows, heads, d, dtype, gap, lead)
    if edit:
        edit(raw, k, v)
    dev = kc.Device(ctx, pool, batch, cs)
    run_append(ctx, dev, raw, stride, ka, va, dtype)
    got, want = dev.download(), pool.copy()
    kc.append(want, batch, k, v, cs)
    same_pool(got, want)
    dev.free()
    return got, want, batch


@pytest.mark.parametrize("dtype", [G.F32, G.F16, G.BF16])
@pytest.mark.parametrize("d,rope", [(64, 64), (128, 128), (192, 96), (256, 0), (128, 6), (64, 34), (128, 8)])
def test_append_types_and_sizes(ctx, d, rope, dtype):
    check_append(ctx, d, 3, 32, dtype, rope, [1, 17, 40, 33, 64], [1, 1, 23, 33, 9])


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("gap,lead", [(0, 0), (1, 3), (4, 8)])
def test_append_strides_and_pages(ctx, page, gap, lead):
    check_append(ctx, 128, 2, page, G.F32, 128, [5, 300, 128], [5, 30, 1], gap, lead)
    check_append(ctx, 64, 1, page, G.F16, 32, [16], [16], gap, lead)


def test_append_rows_left_out(ctx):
    """Rows of negative positions, positions past the table, pages outside the
    pool, sequences without rows or length, rows behind the last sequence."""
    check_append(ctx, 64, 2, 16, G.F32, 64, [3, 40, 0, 20], [7, 2, 0, 20], n_rows=33)

    def pages(b, n):
        b.pages[0, 1] = n
        b.pages[1, 0] = -1
        b.pages[1, 1] = 2 ** 31 - 1
    check_append(ctx, 64, 2, 16, G.F16, 64, [40, 40], [40, 30], pages=pages)

    def short(b, n):
        b.pages = b.pages[:, :2].copy()
        b.lens[0] = 2 ** 31 - 1
    check_append(ctx, 64, 1, 16, G.F32, 0, [50, 40], [5, 20], pages=short)


def test_append_non_finite_zero_and_tiny(ctx):
    def edit(raw, k, v):
        for x in (k, v):  # views of raw
            x[0, 0, 3] = np.nan
            x[9, 1, 5] = np.inf
            x[2] = 0
        k[20:36, 0] = 0
        v[20:36, 1] = F32(1e-42)
        k[36:, :] *= F32(1e-30)
        v[36:, :] *= F32(1e30)
    got, _, _ = check_append(ctx, 64, 2, 16, G.F32, 0, [16, 20, 52], [16, 4, 32], edit=edit)
    assert np.isnan(got.k_scale).any() and np.isinf(got.v_scale).any()


@pytest.mark.parametrize("d,heads,page,dtype", [(64, 4, 16, G.F32), (128, 2, 64, G.F16)])
def test_append_token_by_token(ctx, d, heads, page, dtype):
    """Single tokens, some growing their block's scale, and a chunk in between."""
    rng = np.random.default_rng(7)
    steps = [1] * 5 + [9] + [1] * 20 + [3]
    total = sum(steps)
    full, n_pages = kc.make_batch(rng, [total, total], [total, total], page)
    pool = kc.Pool(n_pages, page, heads, d, rng)
    cs = kc.rope_cs(d, full.cap)
    want = pool.copy()
    dev, at = kc.Device(ctx, pool, full, cs), 0
    for m in steps:
        at += m
        b = kc.Batch([at, at], [m, m], full.pages, page)
        for buf, a in zip(dev.bufs[4:6], (b.offsets, np.asarray(b.lens, np.int32))):
            buf.upload(a)
        dev.rows(b.n_rows)
        raw, stride, ka, va, k, v = fused(rng, b.n_rows, heads, d, dtype)
        run_append(ctx, dev, raw, stride, ka, va, dtype)
        kc.append(want, b, k, v, cs)
        same_pool(dev.download(), want)
    dev.free()


@pytest.mark.parametrize("dtype", [G.F32, G.F16, G.BF16])
@pytest.mark.parametrize("d", [64, 128, 192, 256])
def test_read(ctx, d, dtype):
    print(f"read d={d} {dtype.name}", flush=True)
    rng = np.random.default_rng(d)
    batch, n_pages = kc.make_batch(rng, [37, 3, 70], [20, 5, 64], 32, n_rows=95)
    batch.pages[2, 1] = n_pages + 5
    pool = kc.Pool(n_pages, 32, 2, d, rng)
    dev = kc.Device(ctx, pool, batch)
    t = kc.np_type(dtype)
    fill = np.full(95 * 2 * d, 0x3C3C, np.uint16).view(np.float16).astype(F32)
    start = kc.to_bits(fill, dtype)
    out = [rce_amd.DeviceBuffer.from_numpy(ctx, start) for _ in range(2)]
    rce_amd.kv_read_dev(ctx, dev.cache, dev.b, out[0].ptr, out[1].ptr, dtype)
    ctx.synchronize()
    for name, o in zip("kv", out):
        got = o.download(t, 95 * 2 * d).reshape(95, 2, d)
        want = start.reshape(95, 2, d).copy()
        for r, s, pos in batch.rows():
            page = batch.page_of(s, pos, n_pages)
            if page is not None:
                want[r] = kc.to_bits(pool.values(name, page, pos).astype(F32), dtype)
        assert np.array_equal(got.view(np.uint8), want.view(np.uint8)), name
    rce_amd.kv_read_dev(ctx, dev.cache, dev.b, None, out[0].ptr, dtype)  # one of the two alone
    ctx.synchronize()
    assert np.array_equal(out[0].download(t, 95 * 2 * d).view(np.uint8), out[1].download(t, 95 * 2 * d).view(np.uint8))
    for b in out:
        b.free()
    dev.free()


@pytest.mark.parametrize("dtype", [G.F16, G.BF16])
def test_read_rounds_the_f32_product(ctx, dtype):
    """A million values: about one in 30000 tells the product rounded to f32 and
    then to 16 bits from the product rounded once."""
    rng = np.random.default_rng(2)
    rows = 4096
    batch, n_pages = kc.make_batch(rng, [rows], [rows], 64)
    pool = kc.Pool(n_pages, 64, 2, 128, rng)
    dev = kc.Device(ctx, pool, batch)
    out = [rce_amd.DeviceBuffer(ctx, rows * 256 * 2) for _ in range(2)]
    rce_amd.kv_read_dev(ctx, dev.cache, dev.b, out[0].ptr, out[1].ptr, dtype)
    ctx.synchronize()
    pg = batch.pages[0]
    k = pool.k[pg].astype(F32) * pool.k_scale[pg][..., None, None]  # [pages, heads, blocks, 16, d]
    v = pool.v[pg].transpose(0, 1, 2, 4, 3).astype(F32) * pool.v_scale[pg][..., None, None]
    for o, x in zip(out, (k, v)):
        want = kc.to_bits(x.transpose(0, 2, 3, 1, 4).reshape(-1), dtype)
        assert np.array_equal(o.download(kc.np_type(dtype), rows * 256).view(np.uint16), want.view(np.uint16))
        o.free()
    dev.free()


# ---- attention --------------------------------------------------------------------

class Attn:
    """One attention call, its inputs kept on the device."""

    def __init__(self, ctx, pool, batch, n_q, q_dtype, out_dtype, rope=0, window=0, scale=None, gap=0, seed=3, q_edit=None):
        rng = np.random.default_rng(seed)
        self.ctx, self.pool, self.batch, self.n_q, self.window = ctx, pool, batch, n_q, window
        self.q_dtype, self.out_dtype, self.gap = q_dtype, out_dtype, gap
        d = pool.d
        self.scale = float(F32(1 / np.sqrt(d) if scale is None else scale))
        self.cs = kc.rope_cs(rope, batch.cap)
        self.stride = n_q * d + gap
        x = rng.standard_normal((batch.n_rows, self.stride)).astype(F32)
        if q_edit:
            q_edit(x)
        self.raw = kc.to_bits(x, q_dtype)
        self.q = kc.widen(self.raw, q_dtype)[:, :n_q * d].reshape(batch.n_rows, n_q, d)
        self.dev = kc.Device(ctx, pool, batch, self.cs)
        self.x = rce_amd.DeviceBuffer.from_numpy(ctx, self.raw)
        self.t = kc.np_type(out_dtype)
        self.fill = kc.to_bits(np.full(batch.n_rows * self.stride, 7.0, F32), out_dtype)
        self.out = rce_amd.DeviceBuffer.from_numpy(ctx, self.fill)

    def call(self, stream=None, ctx=None):
        rce_amd.kv_attention_dev(ctx or self.ctx, self.dev.cache, self.dev.b, self.x.ptr, self.q_dtype, self.stride, self.n_q,
                                 self.out.ptr, self.out_dtype, self.scale, rope=self.dev.rope, window=self.window,
                                 out_stride=self.stride, stream=stream)

    def bits(self):
        return self.out.download(self.t, self.batch.n_rows * self.stride)

    def check(self):
        self.call()
        self.ctx.synchronize()
        bits = self.bits().reshape(self.batch.n_rows, self.stride)
        d = self.pool.d
        got = kc.widen(bits, self.out_dtype).astype(np.float64)
        want, bound = kc.attention(self.pool, self.batch, self.q, self.cs, self.scale, self.window, self.out_dtype == G.F32)
        rows = int(self.batch.offsets[-1])
        assert np.all(got[:, self.n_q * d:] == 7.0) and np.all(got[rows:] == 7.0), "written outside the rows"
        g, w, b = got[:rows, :self.n_q * d].reshape(rows, self.n_q, d), want[:rows], bound[:rows]
        assert np.array_equal(np.isnan(g), np.isnan(w)), "NaN pattern"
        ok = ~np.isnan(w)
        far = np.abs(g - w)[ok] - (b + kc.out_eps(self.out_dtype) * (np.abs(w) + b) + 2.0 ** -25)[ok]
        assert far.size == 0 or far.max() <= 0, f"off by {np.abs(g - w)[ok].max():.3g}, allowed {b[ok].max():.3g}"
        return bits

    def free(self):
        for b in (self.x, self.out):
            b.free()
        self.dev.free()


def check_attention(ctx, d, heads, per, page, lens, news, q_dtype=G.F32, out_dtype=G.F32, rope=0, window=0, seed=5, edit=None,
                    n_rows=None, **kw):
    print(f"attention d={d} heads={heads}x{per} page={page} lens={lens} news={news} {q_dtype.name}->{out_dtype.name} "
          f"rope={rope} window={window}", flush=True)
    rng = np.random.default_rng(seed)
    batch, n_pages = kc.make_batch(rng, lens, news, page, n_rows=n_rows)
    pool = kc.Pool(n_pages, page, heads, d, rng)
    if edit:
        edit(pool, batch)
    a = Attn(ctx, pool, batch, heads * per, q_dtype, out_dtype, rope, window, **kw)
    bits = a.check()
    a.free()
    return bits


@pytest.mark.parametrize("q_dtype,out_dtype", [(G.F32, G.F32), (G.F16, G.F16), (G.BF16, G.BF16), (G.F32, G.F16), (G.F16, G.F32)])
@pytest.mark.parametrize("d", [64, 128, 192, 256])
def test_attention_types_and_sizes(ctx, d, q_dtype, out_dtype):
    check_attention(ctx, d, 2, 3, 32, [1, 16, 63, 64, 65, 200], [1, 1, 2, 1, 30, 17], q_dtype, out_dtype, rope=d // 2)


@pytest.mark.parametrize("per", [1, 2, 4, 5, 8, 16, 20, 33])
def test_attention_head_layouts(ctx, per):
    check_attention(ctx, 64, 2, per, 16, [70, 9, 130], [1, 3, 1], G.F16, G.F16, rope=64)
    check_attention(ctx, 64, 1, per, 16, [70, 9, 130], [1, 9, 40], G.F32, G.F32)


@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 150, 10 ** 9, 2 ** 40])
def test_attention_windows(ctx, window):
    check_attention(ctx, 64, 2, 2, 16, [1, 200, 333, 64], [1, 1, 100, 64], window=window, rope=64)
    check_attention(ctx, 128, 1, 4, 64, [1, 200, 333, 64], [1, 1, 100, 64], G.F16, G.F16, window=window)


@pytest.mark.parametrize("page", [16, 128, 512])
@pytest.mark.parametrize("out_dtype", [G.F32, G.F16])
def test_attention_long_sequences_split(ctx, page, out_dtype):
    """Key ranges over several blocks, joined in a second launch, beside short ones."""
    check_attention(ctx, 64, 2, 4, page, [5000, 3, 1200, 0, 2049], [1, 1, 2, 0, 1], G.F32, out_dtype, rope=32)
    check_attention(ctx, 128, 1, 2, page, [3000], [20], G.F16, out_dtype)
    check_attention(ctx, 256, 1, 1, page, [1500], [1], G.F16, out_dtype, window=900)


@pytest.mark.parametrize("out_dtype,window", [(G.F32, 0), (G.F16, 0), (G.F16, 30001)])
def test_attention_long_ragged_sequences_in_line(ctx, out_dtype, window):
    """Blocks that serve the end of one sequence and the beginning of the next."""
    check_attention(ctx, 64, 8, 2, 64, [60000, 100, 40000, 0, 33333, 64, 31000], [1, 1, 2, 0, 1, 1, 9], G.F32, out_dtype,
                    rope=64, window=window)


@pytest.mark.parametrize("out_dtype", [G.F32, G.F16])
def test_attention_long_tokens_in_line_beside_prompts(ctx, out_dtype):
    """Both parts of a call split, one of them as a line: one join for both."""
    check_attention(ctx, 64, 8, 2, 128, [30000, 900, 28001, 33333, 64, 31000, 29999], [1, 150, 2, 1, 64, 1, 1], G.F16, out_dtype,
                    rope=64, n_rows=225)


def test_attention_in_line_of_many_units(ctx):
    """More sequences than a wave has lanes, several of them in a block."""
    rng = np.random.default_rng(8)
    lens = [int(n) for n in rng.integers(0, 30000, 70)]
    lens[5] = lens[66] = 0
    check_attention(ctx, 64, 1, 1, 256, lens, [min(n, 1) for n in lens], G.F16, G.F16)


def test_attention_of_sequences_that_share_their_pages(ctx):
    """16384 sequences of the same pages: block number times a block's cells passes 31 bits.
    Four queries in turn, so that every row has its expected value."""
    rng = np.random.default_rng(14)
    n, length, page, heads, d = 16384, 33000, 1024, 8, 64
    one, n_pages = kc.make_batch(rng, [length], [4], page)
    pool = kc.Pool(n_pages, page, heads, d, rng)
    four = kc.Batch([length] * 4, [1] * 4, np.repeat(one.pages, 4, 0), page)
    batch = kc.Batch([length] * n, [1] * n, np.repeat(one.pages, n, 0), page)
    q = kc.to_bits(rng.standard_normal((4, heads * d)).astype(F32), G.F16)
    dev = kc.Device(ctx, pool, batch)
    x = rce_amd.DeviceBuffer.from_numpy(ctx, np.tile(q, (n // 4, 1)))
    out = rce_amd.DeviceBuffer(ctx, n * heads * d * 2)
    rce_amd.kv_attention_dev(ctx, dev.cache, dev.b, x.ptr, G.F16, heads * d, heads, out.ptr, G.F16, 0.125)
    ctx.synchronize()
    got = out.download(np.float16, n * heads * d).reshape(n // 4, 4, heads, d).astype(np.float64)
    want, bound = kc.attention(pool, four, q.astype(F32).reshape(4, heads, d), None, 0.125, 0, False)
    assert np.all(np.abs(got - want) <= bound + kc.out_eps(G.F16) * (np.abs(want) + bound) + 2.0 ** -25)
    for b in (x, out):
        b.free()
    dev.free()


def test_attention_many_sequences(ctx):
    """More sequences than a wave has lanes, empty ones among them."""
    rng = np.random.default_rng(11)
    lens = [int(n) for n in rng.integers(0, 90, 150)]
    news = [min(n, int(rng.integers(0, 4))) for n in lens]
    check_attention(ctx, 64, 2, 2, 16, lens, news, G.F16, G.F16, rope=64)
    lens[70] = 900
    news[70] = 1
    check_attention(ctx, 64, 2, 2, 16, lens, news, G.F32, G.F32)


@pytest.mark.parametrize("news", [[64, 64, 64], [300, 17, 1], [129, 0, 200]])
@pytest.mark.parametrize("out_dtype", [G.F32, G.F16])
def test_attention_prompts(ctx, news, out_dtype):
    check_attention(ctx, 128, 2, 4, 64, news, news, out_dtype, out_dtype, rope=128)
    check_attention(ctx, 64, 1, 3, 16, [n + 100 for n in news], news, out_dtype, out_dtype, window=77)


@pytest.mark.parametrize("d,rope", [(64, 34), (64, 64), (128, 6), (128, 64), (192, 192), (192, 0), (256, 128), (256, 256)])
@pytest.mark.parametrize("q_dtype,out_dtype", [(G.F32, G.F32), (G.F16, G.F16), (G.BF16, G.BF16), (G.BF16, G.F32)])
def test_attention_prompts_of_every_head_size(ctx, d, rope, q_dtype, out_dtype):
    """Units of 128 query rows: one short of full, full, one more; single rows beside them."""
    check_attention(ctx, d, 2, 3, 32, [43, 128, 170, 90], [43, 33, 1, 90], q_dtype, out_dtype, rope=rope)


@pytest.mark.parametrize("length,new", [(0, 0), (1, 1), (700, 1), (700, 5), (300, 300), (7000, 20), (20000, 1), (20000, 90)])
def test_attention_of_one_sequence_in_a_padded_batch(ctx, length, new):
    for t in (G.F32, G.F16):
        check_attention(ctx, 64, 2, 2, 64, [length], [new], t, t, rope=64, n_rows=new + 40)


@pytest.mark.parametrize("page", [16, 64, 1024])
@pytest.mark.parametrize("out_dtype", [G.F32, G.F16])
def test_attention_prompts_after_long_contexts(ctx, page, out_dtype):
    """Split key ranges of 128-row units, beside single tokens whose ranges are split too."""
    check_attention(ctx, 128, 1, 4, page, [3000, 700, 2500], [40, 1, 70], G.F16, out_dtype, rope=128)
    check_attention(ctx, 64, 2, 2, page, [5000, 0, 900], [50, 0, 100], G.F32, out_dtype, window=2000)
    check_attention(ctx, 256, 1, 1, page, [2000], [129], G.F16, out_dtype, rope=256)


@pytest.mark.parametrize("window", [1, 15, 64, 65, 200])
@pytest.mark.parametrize("out_dtype", [G.F32, G.F16])
def test_attention_prompts_with_windows(ctx, window, out_dtype):
    check_attention(ctx, 64, 1, 5, 16, [300, 64, 130], [300, 64, 7], G.F32, out_dtype, rope=64, window=window)
    check_attention(ctx, 192, 1, 2, 128, [150, 280], [70, 140], G.F16, out_dtype, window=window)


@pytest.mark.parametrize("gap", [1, 2, 8])
def test_attention_prompts_of_odd_strides_and_row_counts(ctx, gap):
    for t in (G.F32, G.F16, G.BF16):
        check_attention(ctx, 64, 2, 3, 16, [70, 9, 33], [70, 3, 33], t, t, gap=gap, rope=64, n_rows=120)


@pytest.mark.parametrize("out_dtype", [G.F32, G.F16])
@pytest.mark.parametrize("d", [64, 256])
def test_attention_prompts_of_growing_scores(ctx, out_dtype, d):
    """Each block's scores pass the earlier ones' by much, or its values' scale does:
    the running maximum and the running scale move at every tile; and the reverse."""
    for name in ("k", "v"):
        for flip in (False, True):
            def edit(pool, b):
                for s in range(len(b.lens)):
                    n = max(1, (b.lens[s] + 15) // 16)
                    for blk in range(n):
                        f = 10.0 ** (4.0 * (n - 1 - blk if flip else blk) / n - 2)
                        page = b.pages[s, blk * 16 // pool.page]
                        getattr(pool, name + "_scale")[page, :, blk % pool.b] *= F32(f)
            check_attention(ctx, d, 1, 2, 32, [400, 90], [200, 90], G.F32, out_dtype, edit=edit)


def test_attention_rows_left_out(ctx):
    """Negative positions, positions past the table, rows behind the last
    sequence, pages outside the pool (their positions unseen), a row that
    sees nothing at all."""
    check_attention(ctx, 64, 2, 2, 16, [3, 40, 0, 20], [7, 2, 0, 20], n_rows=33, rope=64)

    def bad(pool, b):
        b.pages[0, 1] = pool.n_pages
        b.pages[1, :] = -1
        b.pages[2, 0] = -5
    check_attention(ctx, 64, 2, 2, 16, [60, 40, 90], [60, 3, 1], edit=bad)
    check_attention(ctx, 64, 2, 2, 16, [60, 40, 90], [60, 3, 90], G.F16, G.F16, edit=bad, window=10)

    def short(pool, b):
        b.pages = b.pages[:, :2].copy()
    check_attention(ctx, 64, 1, 4, 16, [50, 40, 32], [30, 20, 1], edit=short)
    check_attention(ctx, 128, 1, 1, 16, [100, 40, 32], [100, 20, 1], G.F16, G.F16, edit=short)


@pytest.mark.parametrize("window", [0, 1, 40])
@pytest.mark.parametrize("per", [1, 3])
def test_attention_prompts_with_rows_before_the_first_position(ctx, per, window):
    """A unit's 16 rows begin at negative positions and end at valid ones."""
    check_attention(ctx, 64, 1, per, 16, [100, 3, 64], [130, 150, 70], G.F32, G.F32, rope=64, window=window)
    check_attention(ctx, 128, 1, per, 16, [100, 3, 64], [130, 150, 70], G.F16, G.F16, window=window)


@pytest.mark.parametrize("out_dtype", [G.F32, G.F16])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_attention_non_finite_blocks(ctx, bad, out_dtype):
    """A non-finite scale reaches the rows that see its block and no others."""
    def edit(pool, b):
        for s, blk, name in ((0, 2, "k"), (1, 0, "v"), (2, 5, "v"), (3, 3, "k")):
            page = b.pages[s, blk * 16 // pool.page]
            at = blk % pool.b
            getattr(pool, name + "_scale")[page, 0, at] = bad
            codes = getattr(pool, name)
            codes[page, 0, at] = 0  # as an append leaves it
    check_attention(ctx, 64, 2, 2, 32, [64, 40, 120, 100], [64, 3, 60, 1], G.F32, out_dtype, edit=edit)
    check_attention(ctx, 64, 2, 2, 32, [64, 40, 120, 100], [64, 3, 60, 1], G.F32, out_dtype, edit=edit, window=9)


@pytest.mark.parametrize("out_dtype", [G.F32, G.F16])
def test_attention_values_far_apart(ctx, out_dtype):
    """Scales of neighbouring blocks far apart, zero ones, queries of very
    different size, large and zero score scales."""
    def edit(pool, b):
        r = np.random.default_rng(4)
        pool.v_scale[:] = (10.0 ** r.uniform(-6, 2, pool.v_scale.shape)).astype(F32)
        pool.k_scale[r.random(pool.k_scale.shape) < 0.2] = 0
        pool.v_scale[r.random(pool.v_scale.shape) < 0.2] = 0

    def q_edit(x):
        x *= (10.0 ** np.linspace(-3, 1, len(x))[:, None]).astype(F32)
        x[0] = 0
        x[-1, :64] = np.nan
        x[-2, 64] = np.inf
    check_attention(ctx, 64, 2, 2, 32, [64, 40, 200], [64, 3, 60], G.F32, out_dtype, edit=edit, q_edit=q_edit)
    check_attention(ctx, 64, 2, 2, 32, [64, 40, 200], [64, 3, 60], G.F32, out_dtype, scale=0.0)
    check_attention(ctx, 64, 2, 2, 32, [64, 40, 200], [64, 3, 60], G.F32, out_dtype, scale=2.0)


@pytest.mark.parametrize("lens,news", [([400, 90], [200, 90]), ([1500, 90], [1, 2])])
@pytest.mark.parametrize("exp", [-126, -118, -100])
def test_attention_of_tiny_values(ctx, exp, lens, news):
    """Value scales down to 2^-126: as the same call with scales near 1, to a power of two (weights
    are rounded to 2^-11, or 2^-18 of the largest where the scales are at their least)."""
    def edit(to):
        def f(pool, b):
            r = np.random.default_rng(6)
            pool.v_scale[:] = (r.uniform(1.0, 1.9, pool.v_scale.shape) * 2.0 ** to).astype(F32)
        return f
    got, want = (check_attention(ctx, 64, 1, 2, 32, lens, news, G.F32, G.F32, edit=edit(e)).astype(np.float64) * 2.0 ** -e
                 for e in (exp, 0))
    assert np.isfinite(got).all() and np.abs(got - want).max() <= 2.0 ** -10 * np.abs(want).max()


def test_attention_strides_and_unwritten_pages(ctx):
    check_attention(ctx, 64, 2, 2, 16, [70, 9], [1, 3], gap=5)
    check_attention(ctx, 128, 2, 1, 16, [70, 9], [1, 3], G.F16, G.F16, gap=1)

    def poison(pool, b):  # blocks past a sequence's end hold anything
        for s, n in enumerate(b.lens):
            for p in range((n + 15) // 16 * 16, b.cap, 16):
                page = b.page_of(s, p, pool.n_pages)
                if page is not None:
                    pool.k_scale[page, :, p % pool.page // 16] = np.nan
                    pool.v_scale[page, :, p % pool.page // 16] = np.inf
    check_attention(ctx, 64, 2, 2, 64, [70, 9, 33], [1, 3, 33], edit=poison)


def long_attn(ctx, seed=3):
    rng = np.random.default_rng(9)
    batch, n_pages = kc.make_batch(rng, [2500, 300, 40], [1, 3, 40], 32)
    pool = kc.Pool(n_pages, 32, 2, 128, rng)
    return Attn(ctx, pool, batch, 8, G.F16, G.F16, rope=128, seed=seed)


def test_attention_same_bits_again_on_streams_and_contexts(ctx):
    a = long_attn(ctx)
    want = a.check()
    hip = Hip()
    with rce_amd.Context(0) as other:
        for stream, c in ((None, ctx), (other.stream, ctx), (None, other), (0, other)):
            a.out.upload(a.fill)
            a.call(stream=stream, ctx=c)
            ctx.synchronize()
            other.synchronize()
            assert np.array_equal(a.bits().view(np.uint8).reshape(-1), want.view(np.uint8).reshape(-1))
    del hip
    a.free()


def test_recorded_step_replayed_as_positions_advance():
    """Append and attention of single tokens recorded once; the batch's arrays
    and the inputs change between replays, other calls run in between, and every replay
    equals the eager calls."""
    rng = np.random.default_rng(12)
    heads, d, page, n = 2, 64, 16, 3
    with rce_amd.Context(0) as c:
        start = [5, 30, 700]
        batch, n_pages = kc.make_batch(rng, [x + 20 for x in start], [1] * n, page)
        pool = kc.Pool(n_pages, page, heads, d, rng)
        batch.lens = [x + 1 for x in start]
        a = Attn(c, pool, batch, 4, G.F32, G.F32, rope=d)
        w = 2 * heads * d
        kv = rce_amd.DeviceBuffer(c, n * w * 4)

        def step():
            rce_amd.kv_append_dev(c, a.dev.cache, a.dev.b, kv.ptr, kv.ptr + heads * d * 4, G.F32, w, w, rope=a.dev.rope)
            a.call()
        hip = Hip()
        g, ex = hip.capture(c.stream, step)
        host = pool.copy()
        other = long_attn(c)
        for i in range(4):
            lens = [x + 1 + i for x in start]
            b = kc.Batch(lens, [1] * n, batch.pages, page)
            x = rng.standard_normal((n, w)).astype(F32)
            kv.upload(x)
            a.dev.bufs[5].upload(np.asarray(lens, np.int32))
            other.call()
            c.synchronize()
            hip.launch(ex, c.stream)
            c.synchronize()
            kc.append(host, b, x[:, :heads * d].reshape(n, heads, d), x[:, heads * d:].reshape(n, heads, d), a.cs)
            same_pool(a.dev.download(), host)
            got = a.bits().copy()
            a.pool, a.batch = host, b
            assert np.array_equal(a.check().view(np.uint32).reshape(-1), got.view(np.uint32).reshape(-1))
        hip.destroy(g, ex)
        other.free(); a.free(); kv.free()
