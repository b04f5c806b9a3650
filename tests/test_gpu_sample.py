"""rce_qmm_sample_dev against sampling in 64 bits: the same tokens, and their
probabilities to an f32 rounding, over sizes, types, filters alone and
together, ties, rows without weight and numbers at the ends of [0, 1)."""
import numpy as np
import pytest

import kv_case as kc
import rce_amd
from bench import Hip
from kv_case import F32
from rce_amd import GgufDtype as G

pytestmark = pytest.mark.gpu


class Call:
    def __init__(self, ctx, logits, dtype, u, stride=None, **par):
        """logits [rows, vocab] f32; par: arrays or numbers per filter."""
        self.ctx, self.dtype = ctx, dtype
        self.n, self.v = logits.shape
        self.stride = stride or self.v
        full = np.full((self.n, self.stride), 1e30, F32)  # what stands between the rows would win
        full[:, :self.v] = logits
        raw = kc.to_bits(full, dtype)
        self.x = kc.widen(raw, dtype)[:, :self.v]
        self.u = np.broadcast_to(np.asarray(u, F32), (self.n,)).copy()
        self.par = {k: np.broadcast_to(np.asarray(a, np.int32 if k == "top_k" else F32), (self.n,)).copy() for k, a in par.items()}
        up = lambda a: rce_amd.DeviceBuffer.from_numpy(ctx, a)  # noqa: E731
        self.lg, self.ub = up(raw), up(self.u)
        self.pb = {k: up(a) for k, a in self.par.items()}
        self.ids = up(np.full(self.n + 1, -77, np.int32))
        self.probs = up(np.full(self.n + 1, -77, F32))

    def call(self, stream=None, probs=True):
        rce_amd.sample_dev(self.ctx, self.lg.ptr, self.dtype, self.n, self.v, self.stride, self.ub.ptr, self.ids.ptr,
                           probs_dev=self.probs.ptr if probs else None, stream=stream,
                           **{k + "_dev": b.ptr for k, b in self.pb.items()})

    def result(self):
        return self.ids.download(np.int32, self.n + 1), self.probs.download(F32, self.n + 1)

    def expect(self):
        names = {"temperature": "temp"}
        return [kc.sample(self.x[r], self.u[r], **{names.get(k, k): a[r] for k, a in self.par.items()}) for r in range(self.n)]

    def check(self):
        self.call()
        self.ctx.synchronize()
        ids, probs = self.result()
        assert ids[-1] == -77 and probs[-1] == -77
        for r, (i, p) in enumerate(self.expect()):
            assert ids[r] == i, (r, int(ids[r]), i, {k: a[r] for k, a in self.par.items()}, self.u[r])
            # one rounding to f32, the sums' own (2^-37 of the largest weight and vocab terms) far below it
            assert abs(probs[r] - p) <= 2.0 ** -23 * p, (r, probs[r], p)
        self.free()

    def free(self):
        for b in (self.lg, self.ub, self.ids, self.probs, *self.pb.values()):
            b.free()


def rows(seed, n, v, size=2.5):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((n, v)) * size * rng.uniform(0.2, 1.5, (n, 1))
    x[np.arange(n), rng.integers(0, v, n)] += rng.uniform(0, 12, n)
    return x.astype(F32), rng.random(n).astype(F32)


FILTERS = [{}, {"temperature": 0.7}, {"top_k": 40}, {"top_p": 0.9}, {"min_p": 0.05},
           {"temperature": 1.3, "top_k": 50, "top_p": 0.95, "min_p": 0.02}, {"top_k": 5, "top_p": 0.3},
           {"top_p": 0.999, "temperature": 2.0}, {"temperature": 0.0, "top_k": 3}, {"temperature": 50.0, "top_k": 700},
           {"top_k": 2 ** 31 - 1, "top_p": 1.5, "min_p": -1.0}, {"top_p": 0.0}, {"min_p": 2.0}, {"top_k": 1}, {"top_k": -4}]


@pytest.mark.parametrize("par", FILTERS, ids=str)
@pytest.mark.parametrize("v", [1, 2, 63, 1000, 4097, 32000])
def test_filters_and_sizes(ctx, v, par):
    print(f"sample v={v} {par}", flush=True)
    x, u = rows(v, 7, v)
    Call(ctx, x, G.F32, u, **par).check()


@pytest.mark.parametrize("dtype", [G.F32, G.F16, G.BF16])
@pytest.mark.parametrize("v,n", [(128000, 5), (151937, 2), (32003, 70), (9, 300)])
def test_types_rows_of_own_settings_and_strides(ctx, dtype, v, n):
    """16-bit logits have many equal values: ties at every threshold."""
    print(f"sample {dtype.name} v={v} n={n}", flush=True)
    x, u = rows(n, n, v)
    rng = np.random.default_rng(v)
    par = {"temperature": rng.choice([0.0, 0.3, 1.0, 1.7], n), "top_k": rng.choice([0, 1, 20, 500, v], n),
           "top_p": rng.choice([0.1, 0.5, 0.95, 1.0], n), "min_p": rng.choice([0.0, 0.01, 0.2], n)}
    Call(ctx, x, dtype, u, stride=v + 13, **par).check()
    Call(ctx, x, dtype, u, **par).check()


@pytest.mark.parametrize("n", [1, 3, 40, 129])
def test_long_rows(ctx, n):
    """Rows that several blocks share (a block each where they are many): nothing cut, cut
    within a few elements, within many, both filters with many left, as flat and as peaked
    rows have it."""
    print(f"sample long rows n={n}", flush=True)
    v = 40009 if n > 40 else 133337
    x, u = rows(n, n, v)
    x[::3] *= F32(0.15)
    rng = np.random.default_rng(n)
    for par in ({}, {"top_p": 0.9}, {"top_k": 3000}, {"top_k": 40}, {"top_k": 20000, "top_p": 0.8}, {"min_p": 0.3, "top_p": 0.95},
                {"top_k": v - 1, "temperature": 0.05}, {"temperature": 0.0}, {"top_p": 1e-6}):
        Call(ctx, x, G.F32, u, **par).check()
        if n > 3:
            break
    par = {"temperature": rng.choice([0.0, 0.2, 1.0, 1.7], n), "top_k": rng.choice([0, 1, 20, 1500, v], n),
           "top_p": rng.choice([0.1, 0.5, 0.95, 1.0], n), "min_p": rng.choice([0.0, 0.01, 0.2], n)}
    Call(ctx, x, G.F32, u, **par).check()


def test_long_rows_recorded_and_replayed():
    """The kernels of split rows share a buffer of the context's: replays between other calls of
    both kinds equal the expected tokens every time."""
    with rce_amd.Context(0) as c:
        x, u = rows(21, 5, 90001)
        a = Call(c, x, G.F32, u, top_p=0.9, temperature=0.8)
        y, w = rows(22, 3, 50001)
        b = Call(c, y, G.F32, w, top_k=30, top_p=0.9)
        hip = Hip()
        g, ex = hip.capture(c.stream, a.call)
        for i in range(4):
            u = np.roll(u, 1)
            a.u = u
            a.ub.upload(u)
            a.ids.upload(np.full(6, -77, np.int32))
            b.call()
            c.synchronize()
            hip.launch(ex, c.stream)
            b.call()
            c.synchronize()
            for call in (a, b):
                ids, probs = call.result()
                for r, (t, p) in enumerate(call.expect()):
                    assert ids[r] == t and abs(probs[r] - p) <= 2.0 ** -23 * p
        hip.destroy(g, ex)
        a.free()
        b.free()


@pytest.mark.parametrize("par", [{}, {"top_k": 2000}, {"top_p": 0.37}, {"top_p": 0.6, "top_k": 50000}, {"min_p": 1.0}], ids=str)
def test_long_rows_of_equal_and_missing_logits(ctx, par):
    x, u = rows(11, 6, 70001)
    x[0] = 1.5
    x[1] = -np.inf
    x[2, :] = np.nan
    x[2, 70000] = -3
    x[3, ::7] = x[3].max()
    x[4, 60000:] = -np.inf
    x[4, 13] = np.inf
    x[5, 5:69000] = -3.4e38
    Call(ctx, x, G.F32, u, **par).check()


def test_ties(ctx):
    """Equal logits: the lower ids are kept, sums of equal weights are exact."""
    x = np.zeros((8, 1000), F32)
    u = np.array([0, 0.25, 0.5, 0.999, 0.001, 0.75, 0.1249, 0.125], F32)
    Call(ctx, x, G.F32, u).check()
    Call(ctx, x, G.F32, u, top_k=8).check()
    Call(ctx, x, G.F32, u, top_p=0.25).check()
    Call(ctx, x, G.F32, u, top_k=64, top_p=0.5, min_p=1.0).check()
    x[:, 500:510] = 1
    x[:, 3] = -0.0
    Call(ctx, x, G.F32, u, top_k=12).check()
    Call(ctx, x, G.F32, u, top_k=7, top_p=0.6).check()
    Call(ctx, x, G.F32, u, min_p=1.0).check()
    Call(ctx, x, G.F32, u, temperature=0.0).check()
    x = np.repeat(np.arange(125, dtype=F32)[None] * 0.01, 8, 0).repeat(8, 1)  # eight of each
    for k in (1, 3, 8, 9, 12, 999):
        Call(ctx, x, G.F32, u, top_k=k).check()
    for p in (0.01, 0.3, 0.8):
        Call(ctx, x, G.F32, u, top_p=p, top_k=500).check()


def test_infinities_and_nan(ctx):
    x, u = rows(3, 9, 300)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, :] = np.nan
    x[2, 299] = -3
    x[3, 5] = x[3, 200] = np.inf
    x[4, ::2] = -np.inf
    x[5, 0] = np.nan
    x[6] = -3.4e38
    x[7, 7] = 3.4e38
    x[8, :] = -np.inf
    x[8, 17] = -3.4028235e38
    for par in ({}, {"top_k": 4}, {"top_p": 0.5}, {"temperature": 0.0}, {"temperature": 1e-30}, {"min_p": 0.1, "top_k": 299},
                {"temperature": 3e38}):
        Call(ctx, x, G.F32, u, **par).check()
    # more infinite logits than are kept; the whole range of f32
    y = x[:3].copy()
    y[:] = -3
    y[:, 20:30] = np.inf
    for par in ({"top_k": 3}, {"top_p": 0.25}, {"top_k": 7, "top_p": 0.5}):
        Call(ctx, y, G.F32, [0.0, 0.5, 0.99], **par).check()
    y = np.linspace(-3.4e38, 3.4e38, 300, dtype=F32)[None].repeat(3, 0)
    for par in ({"top_k": 30}, {"top_p": 0.25}, {"top_k": 70, "top_p": 0.5}):
        Call(ctx, y, G.F32, [0.0, 0.5, 0.99], temperature=3e38, **par).check()
        Call(ctx, (y / F32(1e38)) * F32(1e-44), G.F32, [0.0, 0.5, 0.99], temperature=1e-44, **par).check()
    # an infinite temperature: every finite logit alike
    y = np.where(np.isinf(x), 0, x)[4:6].copy()
    Call(ctx, y, G.F32, u[4:6], temperature=np.inf).check()


def test_numbers_at_the_ends(ctx):
    x, _ = rows(5, 6, 5000)
    top = np.nextafter(F32(1), F32(0))
    for par in ({}, {"top_p": 0.7}, {"top_k": 3, "temperature": 0.5}):
        Call(ctx, x, G.F32, [0, top, 1e-40, 0.5, 2.0 ** -24, 1 - 2.0 ** -10], **par).check()
        # outside [0, 1): the nearest end
        a, b = Call(ctx, x, G.F32, [-1, 1, np.nan, 7, -np.inf, np.inf], **par), \
            Call(ctx, x, G.F32, [0, top, 0, top, 0, top], **par)
        for c in (a, b):
            c.call()
        ctx.synchronize()
        assert np.array_equal(a.result()[0], b.result()[0])
        a.free(); b.free()


def test_flat_rows_reach_every_part(ctx):
    """Nearly flat rows: the draw falls into any part of the vocabulary, and the
    nucleus is most of it."""
    rng = np.random.default_rng(8)
    x = (rng.standard_normal((64, 50001)) * 0.01).astype(F32)
    u = (np.arange(64) / 64 + 0.003).astype(F32)
    Call(ctx, x, G.F32, u).check()
    Call(ctx, x, G.F32, u, top_p=0.9).check()
    Call(ctx, x, G.F32, u, top_k=40000, top_p=0.99).check()


def test_recorded_and_other_streams(ctx):
    x, u = rows(21, 5, 32000)
    with rce_amd.Context(0) as c:
        call = Call(c, x, G.F32, u, top_k=50, top_p=0.9)
        hip = Hip()
        g, ex = hip.capture(c.stream, call.call)
        for i in range(4):
            y, v = rows(30 + i, 5, 32000)
            call.lg.upload(y)
            call.ub.upload(v)
            call.x, call.u = y, v
            c.synchronize()
            hip.launch(ex, c.stream)
            c.synchronize()
            ids, probs = call.result()
            want = call.expect()
            assert list(ids[:5]) == [w[0] for w in want]
            call.call(stream=ctx.stream, probs=False)
            ctx.synchronize()
            again = call.result()
            assert np.array_equal(again[0], ids) and np.array_equal(again[1], probs)
        hip.destroy(g, ex)
        call.free()
