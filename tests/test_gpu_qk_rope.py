"""rce_qmm_qk_norm_rope_dev against the formula in 64 bits within the bound
that serve_case.norm_rope derives: head sizes, pairs, rotated parts, types,
strides and alignments, ragged batches, rows left as they were, in place."""
import numpy as np
import pytest

import kv_case as kc
import rce_amd
import serve_case as sc
from bench import Hip
from kv_case import F32
from rce_amd import GgufDtype as G

pytestmark = pytest.mark.gpu


class Call:
    """Rows of a fused projection [q heads | k heads | more], results in buffers of their own."""

    def __init__(self, ctx, rng, lens, news, n_q, n_k, d, it, ot, rope=0, n_pos=None, eps=1e-6, weights=True, interleaved=False, gap=0, shift=0,
                 more_rows=0, size=1.0, base=10000.0):
        self.ctx, self.d, self.it, self.ot, self.eps, self.interleaved = ctx, d, it, ot, eps, interleaved
        self.n = (n_q, n_k)
        self.offsets = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        self.lens = np.asarray(lens, np.int32)
        self.rows = int(self.offsets[-1]) + more_rows
        self.stride = (n_q + 2 * n_k) * d + gap
        self.shift = shift  # values in front of the first row, in and out
        x = rng.standard_normal((self.rows, self.stride)) * size * rng.uniform(0.1, 10, (self.rows, 1))
        self.bits = kc.to_bits(x, it)
        self.weights = [(1 + 0.3 * rng.standard_normal(d)).astype(F32) if weights else None for _ in range(2)]
        n_pos = max(1, int(self.lens.max())) if n_pos is None else n_pos
        self.cs = rce_amd.Rope.table(base, rope, n_pos) if rope else None
        self.n_pos = n_pos
        up = lambda a: rce_amd.DeviceBuffer.from_numpy(ctx, a)  # noqa: E731
        head = np.zeros(shift, self.bits.dtype)
        self.x = up(np.concatenate([head, self.bits.ravel()]))
        self.at = [up(self.offsets), up(self.lens)]
        self.w = [None if w is None else up(np.concatenate([np.zeros(shift % 4, F32), w])) for w in self.weights]
        self.rope = None
        if self.cs is not None:
            self.table = up(self.cs)
            self.rope = rce_amd.Rope(self.table.ptr, rope, n_pos)
        self.out_stride = [m * d + gap for m in self.n]
        self.fill = np.frombuffer(b"\xa5" * 4, np.uint32).view(kc.np_type(ot))[0]
        self.out = [up(np.full(shift + self.rows * max(1, s), self.fill, kc.np_type(ot))) for s in self.out_stride]

    def batch(self):
        return rce_amd.KvBatch(self.at[0].ptr, self.at[1].ptr, 0, len(self.lens), self.rows, 0)

    def heads(self, i, in_place=False):
        size = np.dtype(self.bits.dtype).itemsize
        p = self.x.ptr + size * (self.shift + (self.n[0] * self.d if i else 0))
        o = self.out[i].ptr + np.dtype(kc.np_type(self.ot)).itemsize * self.shift
        w = 0 if self.w[i] is None else self.w[i].ptr + 4 * (self.shift % 4)
        if in_place:
            return rce_amd.Heads(p, self.stride, self.n[i], p, self.stride, w)
        return rce_amd.Heads(p, self.stride, self.n[i], o, self.out_stride[i], w)

    def run(self, **kw):
        rce_amd.qk_norm_rope_dev(self.ctx, self.batch(), self.heads(0, **kw), self.heads(1, **kw), self.d, self.it, self.ot, self.eps,
                                 rope=self.rope, interleaved=self.interleaved)

    def got(self, i):
        """[rows, heads, d] and what lies between the rows."""
        s = self.out_stride[i]
        o = self.out[i].download(kc.np_type(self.ot), self.shift + self.rows * max(1, s))
        assert np.array_equal(o[:self.shift].view(np.uint8), np.full(self.shift, self.fill, o.dtype).view(np.uint8))
        o = o[self.shift:].reshape(self.rows, -1)[:, :s]
        return o[:, :self.n[i] * self.d].reshape(self.rows, self.n[i], self.d), o[:, self.n[i] * self.d:]

    def want(self, i):
        """{row: (out, bound)} of the rows that have a position."""
        x = kc.widen(self.bits, self.it)
        a = 0 if i == 0 else self.n[0] * self.d
        res = {}
        for s, n in enumerate(self.lens):
            for r in range(self.offsets[s], self.offsets[s + 1]):
                pos = max(int(n), 0) - (int(self.offsets[s + 1]) - r)
                if pos < 0 or (self.cs is not None and pos >= self.n_pos):
                    continue
                with np.errstate(over="ignore", invalid="ignore"):
                    res[r] = sc.norm_rope(x[r, a:a + self.n[i] * self.d].reshape(self.n[i], self.d), self.weights[i], self.eps, self.cs, pos, self.interleaved)
        return res

    def compare(self):
        half, tiny = sc.half_step(self.ot)
        for i in range(2):
            if not self.n[i]:
                continue
            o, between = self.got(i)
            assert np.all(between.view(np.uint8) == 0xA5)
            want = self.want(i)
            for r in range(self.rows):
                if r not in want:
                    assert np.all(o[r].view(np.uint8) == 0xA5), r
                    continue
                y, b = want[r]
                with np.errstate(invalid="ignore"):
                    err = np.abs(kc.widen(o[r], self.ot).astype(np.float64) - y)
                assert np.all(err <= b + half * (np.abs(y) + b) + tiny), (r, i, np.max(err - b - half * np.abs(y)))

    def free(self):
        for b in [self.x, *self.at, *self.out, *[w for w in self.w if w is not None]] + ([self.table] if self.rope else []):
            b.free()


def case(ctx, seed, *args, **kw):
    c = Call(ctx, np.random.default_rng(seed), *args, **kw)
    c.run()
    ctx.synchronize()
    c.compare()
    c.free()


TYPES = [(G.F32, G.F32), (G.F16, G.F16), (G.BF16, G.BF16), (G.F32, G.F16), (G.F32, G.BF16), (G.F16, G.F32), (G.BF16, G.F16)]


@pytest.mark.parametrize("d", [2, 6, 16, 32, 48, 64, 80, 96, 112, 128, 130, 192, 256, 512, 1008, 1024])
@pytest.mark.parametrize("interleaved", [False, True])
def test_heads(ctx, d, interleaved):
    for i, (it, ot) in enumerate(TYPES):
        print(f"qk d={d} {it}->{ot} interleaved={interleaved}", flush=True)
        rope = (d, d // 2 // 2 * 2, 0, d // 4 // 16 * 16, d)[i % 5]
        case(ctx, d + i, [9, 300, 40], [3, 1, 17], (3, 8, 1)[i % 3], (1, 2, 5)[i % 3], d, it, ot, rope=rope, interleaved=interleaved)


@pytest.mark.parametrize("rope", [0, 2, 8, 16, 24, 32, 64, 96, 126, 128])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("eps", [None, 1e-5])
def test_rotated_part(ctx, rope, interleaved, eps):
    case(ctx, rope, [700, 33], [5, 33], 4, 2, 128, G.F32, G.F32, rope=rope, interleaved=interleaved, eps=eps, weights=eps is not None)


@pytest.mark.parametrize("gap,shift", [(0, 1), (1, 0), (8, 8), (5, 3), (8, 4), (16, 2)])
@pytest.mark.parametrize("it,ot", TYPES[:4])
def test_strides_and_alignment(ctx, gap, shift, it, ot):
    case(ctx, gap, [80, 5, 64], [2, 5, 30], 5, 3, 64, it, ot, rope=64, gap=gap, shift=shift)


def test_weights_of_ones_and_one_kind(ctx):
    case(ctx, 1, [40], [40], 4, 4, 64, G.F16, G.F16, rope=64, weights=False)
    case(ctx, 2, [40], [40], 0, 4, 64, G.F16, G.F16, rope=64)
    case(ctx, 3, [40], [40], 4, 0, 64, G.F16, G.F16, rope=64)
    case(ctx, 4, [40], [40], 0, 4, 66, G.F16, G.F16, rope=64)


def test_null_kinds(ctx):
    c = Call(ctx, np.random.default_rng(5), [9], [9], 2, 3, 64, G.F32, G.F32, rope=64)
    rce_amd.qk_norm_rope_dev(ctx, c.batch(), None, c.heads(1), 64, G.F32, G.F32, c.eps, rope=c.rope)
    rce_amd.qk_norm_rope_dev(ctx, c.batch(), c.heads(0), None, 64, G.F32, G.F32, c.eps, rope=c.rope)
    ctx.synchronize()
    c.compare()
    c.free()


@pytest.mark.parametrize("d", [64, 66])
def test_rows_left_as_they_were(ctx, d):
    """Rows of no sequence, at negative positions and behind the table; empty sequences; a sequence with no positions."""
    case(ctx, d, [5, 0, 3, 200, 50, 1], [7, 2, 0, 4, 50, 1], 2, 1, d, G.F16, G.F32, rope=32, n_pos=48, more_rows=3)
    case(ctx, d, [5, 0, 3, -4, 1], [7, 2, 0, 4, 1], 2, 1, d, G.F16, G.F32, more_rows=2)


@pytest.mark.parametrize("n_seqs", [63, 64, 65, 129, 4096, 4097, 5000])
def test_many_sequences(ctx, n_seqs):
    """The search for a row's sequence: 64 ends a step, empty sequences among them."""
    rng = np.random.default_rng(n_seqs)
    news = rng.choice([0, 0, 1, 1, 2], n_seqs)
    news[-1] = 1
    lens = news + rng.integers(0, 100, n_seqs)
    case(ctx, n_seqs, lens, news, 1, 1, 32, G.F16, G.F32, rope=32)


@pytest.mark.parametrize("size", [1e-30, 1e-12, 1e12, 1e17])
def test_small_and_large(ctx, size):
    case(ctx, 7, [30], [30], 2, 2, 64, G.F32, G.F32, rope=64, size=size, eps=1e-30 if size < 1 else 1e-6)


@pytest.mark.parametrize("d,rope", [(16, 16), (64, 64), (192, 64), (1024, 0), (66, 66), (130, 0)])
@pytest.mark.parametrize("eps", [0.0, 1e-38, 1e-42])
@pytest.mark.parametrize("it", [G.F32, G.BF16])
def test_mean_squares_below_binary32(ctx, d, rope, eps, it):
    """Heads whose mean square, or every square, is a subnormal number or none of binary32, between heads of ordinary
    size, and heads of subnormal values.  (The smallest are 0 in BF16: 0 / 0 without an eps.)"""
    c = Call(ctx, np.random.default_rng(d), [40], [40], 5, 3, d, it, G.F32, rope=rope, eps=eps)
    sizes = np.array([1, 1e-18, 1e-19, 1e-20, 3e-16, 1e-23, 1e-30, 1e-37, 1e-39, 1e-41])
    x = kc.widen(c.bits, it).astype(np.float64)
    heads = x[:, :8 * d].reshape(c.rows, 8, d)
    heads *= sizes[np.arange(c.rows * 8).reshape(c.rows, 8) % len(sizes)][..., None]
    c.bits = kc.to_bits(x.astype(F32), it)
    c.x.upload(c.bits.ravel())
    c.run()
    ctx.synchronize()
    half, tiny = sc.half_step(G.F32)
    for i in range(2):
        o, _ = c.got(i)
        for r, (y, b) in c.want(i).items():
            nothing = np.isnan(y).all(1)
            assert eps == 0 or not nothing.any()
            assert np.isnan(o[r][nothing]).all()
            with np.errstate(invalid="ignore"):
                err = np.abs(o[r].astype(np.float64) - y)
            assert np.all((err <= b + half * (np.abs(y) + b) + tiny)[~nothing]), (r, i)
    c.free()


@pytest.mark.parametrize("d", [64, 66])
@pytest.mark.parametrize("eps", [1e-38, 1e-42])
def test_zeros_with_a_small_eps(ctx, d, eps):
    c = Call(ctx, np.random.default_rng(d), [6], [6], 3, 1, d, G.F32, G.F32, rope=64, eps=eps)
    bits = c.bits.copy()
    bits[::2, :3 * d] = 0
    c.bits = bits
    c.x.upload(bits.ravel())
    c.run()
    ctx.synchronize()
    c.compare()
    assert np.all(c.got(0)[0][::2] == 0)
    c.free()


def test_zeros_and_what_is_not_finite(ctx):
    """A head of zeros stays zeros; a NaN or infinity spoils its own head alone."""
    c = Call(ctx, np.random.default_rng(8), [6], [6], 3, 1, 64, G.F32, G.F32, rope=64)
    bits = c.bits.copy()
    bits[0, :64] = 0
    bits[1, 64 + 5] = np.nan
    bits[2, 128 + 63] = np.inf
    c.x.upload(bits.ravel())
    c.run()
    ctx.synchronize()
    o, _ = c.got(0)
    assert np.all(o[0, 0] == 0)
    assert np.all(np.isnan(o[1, 1])) and np.isnan(o[2, 2, 63]) and np.isnan(o[2, 2, 31])
    good = np.ones((6, 3), bool)
    good[0, 0] = good[1, 1] = good[2, 2] = False
    want = c.want(0)
    for r in range(6):
        y, b = want[r]
        assert np.all((np.abs(o[r] - y) <= b + 2.0 ** -24 * np.abs(y))[good[r]])
    c.free()


@pytest.mark.parametrize("it", [G.F32, G.F16, G.BF16])
@pytest.mark.parametrize("d,rope,interleaved", [(128, 128, False), (128, 64, True), (66, 34, False), (66, 66, True)])
def test_in_place(ctx, it, d, rope, interleaved):
    """The same bits as beside, values behind the keys untouched."""
    c = Call(ctx, np.random.default_rng(9), [400, 30], [3, 30], 5, 2, d, it, it, rope=rope, interleaved=interleaved, gap=2 if d == 66 else 0)
    c.run()
    ctx.synchronize()
    beside = [c.got(i)[0] for i in range(2)]
    c.run(in_place=True)
    ctx.synchronize()
    x = c.x.download(c.bits.dtype, c.rows * c.stride).reshape(c.rows, c.stride)
    assert np.array_equal(x[:, :5 * d].reshape(c.rows, 5, d).view(np.uint8), beside[0].view(np.uint8))
    assert np.array_equal(x[:, 5 * d:7 * d].reshape(c.rows, 2, d).view(np.uint8), beside[1].view(np.uint8))
    assert np.array_equal(x[:, 7 * d:].view(np.uint8), c.bits[:, 7 * d:].view(np.uint8))
    c.free()


def test_far_positions(ctx):
    """A scaled table's far end, and positions beyond 2^17."""
    rng = np.random.default_rng(10)
    c = Call(ctx, rng, [200000, 131073], [2, 5], 2, 1, 64, G.F16, G.F32, rope=64)
    c.cs = rce_amd.Rope.scaled_table(10000.0, 64, 200000, factor=16.0, orig_context=8192, magnitude=1.2)
    c.table.upload(c.cs)
    c.run()
    ctx.synchronize()
    c.compare()
    c.free()


def test_in_front_of_the_cache(ctx):
    """Without a norm and in f32 it is the append's rotation, to the roundings of it."""
    c = Call(ctx, np.random.default_rng(11), [90], [20], 2, 2, 64, G.F32, G.F32, rope=64, eps=None, weights=False)
    c.run()
    ctx.synchronize()
    o, _ = c.got(1)
    k = c.bits[:, 128:256].reshape(20, 2, 64)
    for r in range(20):
        assert np.array_equal(o[r].view(np.uint32), kc.rotate(k[r], c.cs, 70 + r).view(np.uint32))
    c.free()


def test_recorded(ctx):
    c = Call(ctx, np.random.default_rng(12), [50, 20], [4, 20], 4, 2, 128, G.F16, G.F16, rope=128)
    hip = Hip()
    g, ex = hip.capture(ctx.stream, c.run)
    for i in range(3):
        c.lens = np.array([50 - 7 * i, 20 + i], np.int32)
        c.n_pos = 50
        c.at[1].upload(c.lens)
        for o, s in zip(c.out, c.out_stride):
            o.upload(np.full(c.rows * s, c.fill, kc.np_type(c.ot)))
        case(ctx, 13, [9], [9], 1, 1, 64, G.F32, G.F32, rope=64)
        hip.launch(ex, ctx.stream)
        ctx.synchronize()
        c.compare()
    hip.destroy(g, ex)
    c.free()
