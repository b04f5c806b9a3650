"""rce_qmm_kv_attention_sinks_dev against 64 bits within the bound that
serve_case.attention restates: windows and sinks around tile borders, every
head size and type, single tokens, drafts, chunks and prompts, middles freed,
what is hidden full of NaN, ranges split over blocks and units in a line."""
import numpy as np
import pytest

import kv_case as kc
import rce_amd
import serve_case as sc
from bench import Hip
from kv_case import F32
from rce_amd import GgufDtype as G

pytestmark = pytest.mark.gpu


def free_middles(batch, window, sinks):
    """The pages that no row sees name none."""
    for s, (n, m) in enumerate(zip(batch.lens, batch.news)):
        low = max(0, n - m - window + 1)
        for i in range(batch.pages.shape[1]):
            if i * batch.page >= sinks and (i + 1) * batch.page <= low:
                batch.pages[s, i] = -1


def spoil(pool, batch):
    """Every page that no table names, and page 0 of them first, holds NaN and infinite scales."""
    used = set(batch.pages.ravel().tolist())
    for p in range(pool.n_pages):
        if p not in used:
            pool.k_scale[p], pool.v_scale[p] = np.nan, np.inf
            pool.k[p], pool.v[p] = 127, -127


class Run:
    def __init__(self, ctx, rng, lens, news, page, heads, per, d, it, ot, rope=0, free=None, extra_rows=0, q_gap=0, edit=None):
        self.ctx, self.it, self.ot, self.d, self.n_q = ctx, it, ot, d, heads * per
        self.batch, n_pages = kc.make_batch(rng, lens, news, page, n_rows=sum(news) + extra_rows)
        if free:
            free_middles(self.batch, *free)
        self.pool = kc.Pool(n_pages, page, heads, d, rng)
        spoil(self.pool, self.batch)
        if edit:
            edit(self.pool, self.batch)
        self.cs = kc.rope_cs(rope, self.batch.cap)
        self.dev = kc.Device(ctx, self.pool, self.batch, self.cs)
        rows = self.batch.n_rows
        self.q_stride = self.n_q * d + q_gap
        self.q = kc.to_bits(rng.standard_normal((rows, self.q_stride)), it)
        self.qb = rce_amd.DeviceBuffer.from_numpy(ctx, self.q)
        self.blank = kc.to_bits(np.full((rows, self.n_q * d), 7.0), ot)
        self.ob = rce_amd.DeviceBuffer.from_numpy(ctx, self.blank)
        self.scale = float(F32(d ** -0.5))

    def call(self, window, sinks, stream=None):
        rce_amd.kv_attention_sinks_dev(self.ctx, self.dev.cache, self.dev.b, self.qb.ptr, self.it, self.q_stride, self.n_q, self.ob.ptr, self.ot,
                                       self.scale, window, sinks, rope=self.dev.rope, stream=stream)

    def out(self):
        return self.ob.download(kc.np_type(self.ot), self.blank.size).reshape(-1, self.n_q, self.d)

    def check(self, window, sinks, rows=None):
        self.ob.upload(self.blank)
        self.call(window, sinks)
        self.ctx.synchronize()
        o = self.out()
        x = kc.widen(self.q, self.it)[:, :self.n_q * self.d].reshape(-1, self.n_q, self.d)
        want = sc.attention(self.pool, self.batch, x, self.cs, self.scale, window, sinks, self.ot == G.F32, rows)
        eps = kc.out_eps(self.ot)
        # binary16 below 2^-14 stands in steps of 2^-24 (a value of 3e-8 becomes 0 or 6e-8): half of one, where eps |y| is less
        step = 2.0 ** -25 if self.ot == G.F16 else 0.0
        for r, (y, b) in want.items():
            err = np.abs(kc.widen(o[r], self.ot).astype(np.float64) - y)
            assert np.all(err <= b + np.maximum(eps * (np.abs(y) + b), step)), (r, window, sinks, float(np.max(err)))
        n = int(self.batch.offsets[-1])
        assert np.array_equal(o[n:].view(np.uint8), self.blank.reshape(o.shape)[n:].view(np.uint8))

    def free(self):
        self.qb.free(); self.ob.free(); self.dev.free()


@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("it,ot", [(G.F32, G.F32), (G.F16, G.F16), (G.BF16, G.BF16), (G.F32, G.F16)])
def test_modes(ctx, d, it, ot):
    """One token, drafts and a prompt's chunk in one call of each kind."""
    rng = np.random.default_rng(d)
    for lens, news in (([1, 300, 77, 513, 64, 65], [1] * 6), ([5, 400, 130], [5, 3, 7]), ([290, 61, 200], [150, 61, 3]), ([350], [350])):
        print(f"sinks d={d} {it}->{ot} {lens} {news}", flush=True)
        r = Run(ctx, rng, lens, news, 16, 2, 2, d, it, ot, rope=d if len(lens) % 2 else 0)
        for window, sinks in ((1, 1), (40, 4), (64, 64), (100, 70)):
            r.check(window, sinks)
        r.free()


@pytest.mark.parametrize("page", [16, 64, 128, 4096])
@pytest.mark.parametrize("news", [1, 6, 90])
def test_windows_and_sinks(ctx, page, news):
    rng = np.random.default_rng(page + news)
    r = Run(ctx, rng, [700, 96, 333], [news, news, min(news, 12)], page, 1, 4, 64, G.F16, G.F16, rope=32)
    for window in (1, 2, 63, 64, 65, 128, 200, 699, 700, 5000):
        for sinks in (0, 1, 4, 63, 64, 65, 127, 300, 1000):
            print(f"sinks page={page} new={news} window={window} sinks={sinks}", flush=True)
            r.check(window, sinks, rows={0, news // 2, news - 1, news, 2 * news - 1, 2 * news})
    r.free()


@pytest.mark.parametrize("news", [1, 5, 130])
@pytest.mark.parametrize("window,sinks", [(64, 4), (100, 20), (30, 64), (1, 1), (250, 130)])
def test_freed_middles(ctx, news, window, sinks):
    """Pages between the sinks and the window freed; in their place, and in page 0, what must not be seen."""
    print(f"sinks freed new={news} window={window} sinks={sinks}", flush=True)
    rng = np.random.default_rng(window)
    r = Run(ctx, rng, [900, 450, 1200], [news, news, 1], 16, 2, 2, 64, G.F16, G.F16, free=(window, sinks))
    r.check(window, sinks)
    r.free()


def test_rows_left_out(ctx):
    """Rows before position 0 and behind the table give zeros; rows behind the last sequence keep theirs; an empty sequence."""
    rng = np.random.default_rng(1)
    for news in ([4, 0, 3, 30], [40, 0, 3, 60]):
        r = Run(ctx, rng, [40, 1, 300, 80], news, 16, 1, 2, 64, G.F16, G.F16, extra_rows=3)
        r.batch.lens = [2, 0, 300, 400]  # the last one's rows end behind its table of 304
        r.dev.bufs[5].upload(np.asarray(r.batch.lens, np.int32))
        r.check(20, 5)
        r.free()


def test_missing_pages_and_spoilt_ones(ctx):
    """A sink's page missing, the window's missing, both: the rest, or zeros."""
    rng = np.random.default_rng(2)
    for news in (1, 70):
        r = Run(ctx, rng, [400, 400, 400, 200], [news] * 4, 16, 1, 2, 64, G.F32, G.F32)
        r.batch.pages[0, 0] = -1
        r.batch.pages[1, 1:] = 1 << 30
        r.batch.pages[2] = -7
        r.dev.bufs[6].upload(r.batch.pages)
        r.check(40, 8)
        r.free()


@pytest.mark.parametrize("d,it,ot", [(64, G.F16, G.F16), (128, G.BF16, G.BF16), (128, G.F32, G.F16), (192, G.F16, G.F16), (256, G.F32, G.F16),
                                     (64, G.F32, G.F32)])
def test_scores_and_scales_that_move(ctx, d, it, ot):
    """Prompts whose blocks' scores or value scales grow or fall along the keys, by little in each tile and by much, or lie
    apart at random, some of them 0: tiles that every row sees need a new maximum or none, a larger scale or a far smaller one."""
    for n in range(7):
        def edit(pool, batch):
            rng = np.random.default_rng(n)
            for s, length in enumerate(batch.lens):
                blocks = -(-length // 16)
                for blk in range(blocks):
                    at = batch.pages[s, blk * 16 // pool.page], slice(None), blk % pool.b
                    f = 10.0 ** (4.0 * (blocks - 1 - blk if n & 1 else blk) / blocks - 2)
                    if n < 2:
                        pool.k_scale[at] *= F32(f)
                    elif n < 4:
                        pool.v_scale[at] *= F32(f)
                    elif n == 4:
                        pool.k_scale[at] *= F32(rng.choice([0.1, 1, 30]))
                    elif n == 5:
                        pool.v_scale[at] = 0 if rng.random() < 0.2 else 10.0 ** rng.uniform(-6, 2)
                    else:
                        pool.k_scale[at] *= F32(rng.choice([0, 1, 3]))
                        pool.v_scale[at] *= F32(2.0 ** rng.integers(-14, 14))
        print(f"sinks moving {n} d={d} {it}->{ot}", flush=True)
        r = Run(ctx, np.random.default_rng(d + n), [700, 290], [300, 290], 32, 1, 2, d, it, ot, edit=edit)
        r.check(330, 20)
        r.free()


def test_no_sinks_is_the_window_alone(ctx):
    """Bit for bit; and a window of 0 is none."""
    rng = np.random.default_rng(3)
    for news in (1, 9, 200):
        r = Run(ctx, rng, [1500, 300], [news, news], 32, 2, 4, 64, G.F16, G.F16, rope=64)
        for window, sinks in ((100, 0), (0, 0), (0, 50)):
            r.call(window, sinks)
            r.ctx.synchronize()
            a = r.out()
            rce_amd.kv_attention_dev(ctx, r.dev.cache, r.dev.b, r.qb.ptr, r.it, r.q_stride, r.n_q, r.ob.ptr, r.ot, r.scale, rope=r.dev.rope, window=window)
            ctx.synchronize()
            assert np.array_equal(a.view(np.uint8), r.out().view(np.uint8))
        r.free()


def per_key(pool, batch, q, scale, window, sinks, f32_out, row):
    """(out, bound) [n_q, d] of a row, the bound from each key's own error.

    A key's weight is w_j (1 + a_j), |a_j| <= h_j = e^(s_j) - 1: s_j holds the score's error -- the query's whole numbers', 0.51 steps of two
    limbs and one step of three (the f32 product in front of the rounding has steps of a half there), times scale sum|k_j|, and
    2^-21 |score| for some eight roundings of its factors -- and 2^-21 for the exponential and the products after it.  A rescale by e^(m - m'),
    at most one a tile, adds 2^-22 and 2^-24 of the difference; the differences add up to twice the largest score at most.  With
    a_ the mean of a, out' - out = sum w_j a_j (v_j - out) / (1 + a_).  The products' weights alone are rounded to binary16
    (2^-11; two terms, 2^-20 with the factors' roundings), or in its steps of 2^-24 below 2^-14: 2^-25 of 512 for the
    largest scale, 2^-34 max |v| a key; sums of n terms add n 2^-23."""
    n_q, d = q.shape
    qmax = 127.0 * (65536 if f32_out else 256)
    s = int(np.searchsorted(batch.offsets, row, side="right")) - 1
    pos = batch.lens[s] - (int(batch.offsets[s + 1]) - row)
    j = np.arange(pos + 1)
    j = j[(j > pos - window) | (j < sinks)]
    g = batch.pages[s, j // pool.page]
    b, i = j % pool.page // kc.BLOCK, j % kc.BLOCK
    K = pool.k[g, :, b, i].astype(np.float64) * pool.k_scale[g, :, b].astype(np.float64)[..., None]
    V = pool.v[g, :, b, :, i].astype(np.float64) * pool.v_scale[g, :, b].astype(np.float64)[..., None]
    out, bound = np.zeros((n_q, d)), np.zeros((n_q, d))
    for h in range(n_q):
        k, v, x = K[:, h // (n_q // pool.heads)], V[:, h // (n_q // pool.heads)], q[h].astype(np.float64)
        sc = k @ x * scale
        w = np.exp(sc - sc.max())
        w /= w.sum()
        out[h] = w @ v
        step = np.abs(x).max() / qmax
        e = scale * np.abs(k).sum(1) * step * (1.0 if f32_out else 0.51) + 2.0 ** -21 * np.abs(sc) + 2.0 ** -21
        e += (len(j) / 64 + 2) * 2.0 ** -22 + 2.0 ** -23 * np.abs(sc).max()
        eta = np.expm1(e)
        mean = w @ eta
        assert mean < 0.5
        bound[h] = (w * eta) @ np.abs(v - out[h]) / (1 - mean)
        bound[h] += ((2.0 ** -20 if f32_out else 2.0 ** -11) + len(j) * 2.0 ** -23) * (w @ np.abs(v)) * (1 + 2 * mean)
        bound[h] += 2.0 ** -34 * len(j) * np.abs(v).max()
    return out, bound


@pytest.mark.parametrize("d,it,ot", [(64, G.F16, G.F16), (128, G.BF16, G.BF16), (128, G.F32, G.F16), (256, G.F32, G.F16), (256, G.F16, G.F32),
                                     (64, G.F32, G.F32)])
@pytest.mark.parametrize("how", ["grow", "fall", "apart", "few"])
@pytest.mark.parametrize("news", [1, 7, 290])
def test_scores_that_move_by_each_keys_error(ctx, d, it, ot, how, news):
    """Blocks of keys whose scores grow or fall along the row, or lie apart at random, within bounds that results of a wrong weight or a
    rescale left out do not keep: most are a few roundings of the result."""
    print(f"sinks moving by key {how} new={news} d={d} {it}->{ot}", flush=True)

    def edit(pool, batch):
        rng = np.random.default_rng(d)
        for s, length in enumerate(batch.lens):
            blocks = -(-length // 16)
            for blk in range(blocks):
                at = batch.pages[s, blk * 16 // pool.page], slice(None), blk % pool.b
                part = blk / blocks
                f = {"grow": 10.0 ** (2 * part - 1), "fall": 10.0 ** (1 - 2 * part), "apart": rng.choice([0.1, 1, 10]),
                     "few": rng.choice([0, 0.3, 1, 3])}[how]
                pool.k_scale[at] *= F32(f)
    r = Run(ctx, np.random.default_rng(d + news), [700, 290], [news, news], 32, 1, 2, d, it, ot, edit=edit)
    window, sinks = 330, 20
    r.ob.upload(r.blank)
    r.call(window, sinks)
    ctx.synchronize()
    o = kc.widen(r.out(), ot).astype(np.float64)
    x = kc.widen(r.q, it)[:, :r.n_q * d].reshape(-1, r.n_q, d)
    eps, step = kc.out_eps(ot), 2.0 ** -25 if ot == G.F16 else 0.0
    for row in sorted({0, news // 3, news // 2, news - 1, news, news + news // 2, 2 * news - 1}):
        y, b = per_key(r.pool, r.batch, x[row], r.scale, window, sinks, ot == G.F32, row)
        err = np.abs(o[row] - y)
        assert np.all(err <= b + np.maximum(eps * (np.abs(y) + b), step)), (row, float(np.max(err / b)))
    r.free()


def test_a_window_alone_against_64_bits(ctx):
    """Both entry points without sinks, or without a window, each on cleared results and within the bound."""
    rng = np.random.default_rng(3)
    for news in (1, 9, 200):
        r = Run(ctx, rng, [1500, 300], [news, news], 32, 2, 4, 64, G.F16, G.F16, rope=64)
        for window, sinks in ((100, 0), (0, 0), (0, 50)):
            r.check(window, sinks, rows={0, news - 1, news, 2 * news - 1})
            a = r.out()
            r.ob.upload(r.blank)
            rce_amd.kv_attention_dev(ctx, r.dev.cache, r.dev.b, r.qb.ptr, r.it, r.q_stride, r.n_q, r.ob.ptr, r.ot, r.scale, rope=r.dev.rope, window=window)
            ctx.synchronize()
            assert np.array_equal(a.view(np.uint8), r.out().view(np.uint8))
        r.free()


@pytest.mark.parametrize("ot", [G.F32, G.F16])
@pytest.mark.parametrize("news", [1, 4, 60])
def test_split_ranges(ctx, news, ot):
    """A long window and many sinks: ranges over blocks, joined; a range that ends inside the sinks."""
    rng = np.random.default_rng(4)
    r = Run(ctx, rng, [9000, 30, 4000], [news, min(news, 30), 1], 64, 1, 2, 64, ot, ot, free=(5000, 1500))
    for window, sinks in ((5000, 1500), (4000, 1400), (100, 1500), (5000, 1)):
        r.check(window, sinks, rows={0, news - 1, news, int(r.batch.offsets[-1]) - 1})
    r.free()


def test_units_in_a_line(ctx):
    """Enough tiles that units are cut as one line over the blocks."""
    rng = np.random.default_rng(5)
    n = 50
    lens = rng.integers(2000, 4000, n)
    r = Run(ctx, rng, lens, [1] * n, 64, 8, 1, 64, G.F16, G.F16, free=(3000, 200))
    r.check(3000, 200, rows=set(range(0, n, 7)) | {n - 1})
    r.check(3500, 1, rows={3, n - 2})
    r.free()


def test_long_prompt_among_tokens(ctx):
    rng = np.random.default_rng(6)
    n = 20
    r = Run(ctx, rng, [300] * n + [5000], [1] * n + [5000], 64, 1, 2, 64, G.F16, G.F16)
    rows = {0, n - 1, n, n + 63, n + 64, n + 500, n + 4200, n + 4999}
    r.check(700, 100, rows=rows)
    r.check(64, 4, rows=rows)
    r.check(4000, 4, rows=rows)
    r.free()


@pytest.mark.parametrize("lens,news,page", [([237, 250], [10, 12], 128), ([256], [200], 64), ([1020, 1000], [1, 1], 1024), ([1024, 500], [3, 3], 512)])
def test_tables_as_long_as_the_keys(ctx, lens, news, page):
    """Windows and sinks that together pass what the table spans: units of no more tiles than positions, none split where
    the call has no join."""
    rng = np.random.default_rng(len(lens) + page)
    r = Run(ctx, rng, lens, news, page, 1, 8, 64, G.F16, G.F16, rope=64)
    for window, sinks in ((983, 4), (200, 200), (5000, 64), (150, 17), (lens[0], lens[0])):
        r.check(window, sinks, rows={0, news[0] - 1, news[0], sum(news) - 1})
    r.free()


def test_strides_of_queries(ctx):
    rng = np.random.default_rng(7)
    for gap in (1, 64):
        r = Run(ctx, rng, [500, 90], [2, 50], 16, 2, 3, 64, G.F16, G.F32, rope=48, q_gap=gap)
        r.check(77, 9)
        r.free()


def test_equal_scores_count_each_key_once(ctx):
    """With q = 0 a row is the mean of what it sees: sinks that the window holds too are not seen twice."""
    rng = np.random.default_rng(8)
    r = Run(ctx, rng, [10, 70, 130], [1, 1, 1], 16, 1, 1, 64, G.F32, G.F32)
    r.q[:] = 0
    r.qb.upload(r.q)
    for window, sinks in ((8, 8), (64, 64), (65, 20), (130, 130)):
        r.check(window, sinks)
    r.free()


def test_again_and_recorded(ctx):
    """The same bits again, and from a recorded call between others while the sequences grow."""
    rng = np.random.default_rng(9)
    with rce_amd.Context(0) as c:
        r = Run(c, rng, [6000, 300, 2500], [1, 1, 1], 64, 2, 4, 64, G.F16, G.F16, rope=64)
        b = Run(c, rng, [3000, 3000], [40, 1], 64, 2, 4, 64, G.F16, G.F16)
        hip = Hip()
        g, ex = hip.capture(c.stream, lambda: r.call(2000, 300))
        for i in range(3):
            lens = [6000 - 500 * i, 200 + 50 * i, 2500 - i]
            r.batch.lens = lens
            r.dev.bufs[5].upload(np.asarray(lens, np.int32))
            b.call(2500, 500)
            hip.launch(ex, c.stream)
            c.synchronize()
            once = r.out()
            r.check(2000, 300)
            assert np.array_equal(once.view(np.uint8), r.out().view(np.uint8))
        hip.destroy(g, ex)
        r.free(); b.free()
