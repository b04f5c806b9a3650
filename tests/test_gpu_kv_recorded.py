"""A whole serving step (projections, append, attention, output projection, head,
sampling) recorded once and replayed as the sequences grow, with eager calls of
other sizes on the same context in between: every replay leaves what the eager
step leaves in a pool of its own, bit for bit."""
import numpy as np
import pytest

import kv_case as kc
import oracle as O
import rce_amd
from bench import Hip
from kv_case import F32
from rce_amd import GgufDtype as G
from rce_amd import Mode

pytestmark = pytest.mark.gpu


class Step:
    """One token for each sequence, in a pool of its own."""

    def __init__(self, c, w, shape, pool, batch, cs, par):
        self.c, self.w, self.shape = c, w, shape
        dm, heads, per, d, vocab, n = shape
        self.dev = kc.Device(c, pool, batch, cs)
        self.dev.rows(n)
        alloc = lambda k: rce_amd.DeviceBuffer(c, 4 * n * k)  # noqa: E731
        self.x, self.qkv, self.att = alloc(dm), alloc((heads * per + 2 * heads) * d), alloc(heads * per * d)
        self.y, self.lg, self.ids, self.u = alloc(dm), alloc(vocab), alloc(1), alloc(1)
        self.temp, self.topk, self.topp = (rce_amd.DeviceBuffer.from_numpy(c, p) for p in par)

    def run(self):
        dm, heads, per, d, vocab, n = self.shape
        n_q, width = heads * per, (heads * per + 2 * heads) * d
        rce_amd.mm_batched_dev(self.c, self.x.ptr, G.F32, n, self.w["qkv"], self.qkv.ptr, Mode.EXACT)
        k_at = self.qkv.ptr + n_q * d * 4
        rce_amd.kv_append_dev(self.c, self.dev.cache, self.dev.b, k_at, k_at + heads * d * 4, G.F32, width, width, rope=self.dev.rope)
        rce_amd.kv_attention_dev(self.c, self.dev.cache, self.dev.b, self.qkv.ptr, G.F32, width, n_q, self.att.ptr, G.F32,
                                 d ** -0.5, rope=self.dev.rope)
        rce_amd.mm_batched_dev(self.c, self.att.ptr, G.F32, n, self.w["wo"], self.y.ptr, Mode.EXACT)
        rce_amd.mm_batched_dev(self.c, self.y.ptr, G.F32, n, self.w["head"], self.lg.ptr, Mode.EXACT)
        rce_amd.sample_dev(self.c, self.lg.ptr, G.F32, n, vocab, vocab, self.u.ptr, self.ids.ptr, temperature_dev=self.temp.ptr,
                           top_k_dev=self.topk.ptr, top_p_dev=self.topp.ptr)

    def put(self, x, u, lens):
        self.x.upload(x)
        self.u.upload(u)
        self.dev.bufs[5].upload(lens)
        self.ids.upload(np.full(len(u), -9, np.int32))

    def state(self):
        dm, heads, per, d, vocab, n = self.shape
        p = self.dev.download()
        return [self.qkv.download(np.uint32, n * (heads * per + 2 * heads) * d), self.att.download(np.uint32, n * heads * per * d),
                self.lg.download(np.uint32, n * vocab), self.ids.download(np.int32, n), p.k, p.v, p.k_scale.view(np.uint32),
                p.v_scale.view(np.uint32)]

    def free(self):
        for b in (self.x, self.qkv, self.att, self.y, self.lg, self.ids, self.u, self.temp, self.topk, self.topp):
            b.free()
        self.dev.free()


@pytest.mark.parametrize("vocab", [500, 40000])
def test_recorded_step(vocab):
    """Vocabularies whose rows fit a block's LDS, and whose rows several blocks share."""
    print(f"recorded step vocab={vocab}", flush=True)
    rng = np.random.default_rng(vocab)
    dm, heads, per, d, page, n, steps = 256, 2, 2, 64, 16, 3, 5
    n_q = heads * per
    width = (n_q + 2 * heads) * d
    with rce_amd.Context(0) as c:
        make = lambda r, k: (O.quantize((rng.standard_normal((r, k)) * 0.06).astype(F32), O.Q8_0), r, k)  # noqa: E731
        raw = {"qkv": make(width, dm), "wo": make(dm, n_q * d), "head": make(vocab, dm)}
        w = {k: rce_amd.QuantWeight.from_owned_bytes(c, b, O.Q8_0, r, k_) for k, (b, r, k_) in raw.items()}
        embd = rng.standard_normal((vocab, dm)).astype(F32)
        lens = np.array([4, 1200, 77], np.int32)  # split keys among them
        full, n_pages = kc.make_batch(rng, [int(x) + steps + 1 for x in lens], [1] * n, page)
        pool = kc.Pool(n_pages, page, heads, d, rng)
        cs = kc.rope_cs(d, full.cap)
        par = np.array([0.8, 1.0, 0.5], F32), np.array([0, 20, 3], np.int32), np.array([0.9, 1, 0.7], F32)
        shape = (dm, heads, per, d, vocab, n)
        a, b = (Step(c, w, shape, pool, full, cs, par) for _ in range(2))
        other = Step(c, w, shape, pool, full, cs, par)
        tokens = rng.integers(0, vocab, n)
        hip = Hip()
        g, ex = hip.capture(c.stream, a.run)  # records, runs nothing
        big = rce_amd.DeviceBuffer.from_numpy(c, np.zeros(64 * 2 * dm, F32))  # 64 rows in, 64 out
        for i in range(steps):
            lens = lens + 1
            x, u = embd[tokens], rng.random(n).astype(F32)
            for s in (a, b):
                s.put(x, u, lens)
            other.put(x[::-1].copy(), u, lens - 1)
            other.run()
            rce_amd.mm_batched_dev(c, big.ptr, G.F32, 64, w["wo"], big.ptr + 4 * 64 * dm, Mode.EXACT)
            c.synchronize()
            hip.launch(ex, c.stream)
            other.run()
            c.synchronize()
            b.run()
            c.synchronize()
            got, want = a.state(), b.state()
            for name, p, q in zip(("qkv", "attention", "logits", "ids", "k", "v", "k_scale", "v_scale"), got, want):
                assert np.array_equal(p, q), (i, name)
            assert np.all((got[3] >= 0) & (got[3] < vocab))
            tokens = got[3]
        hip.destroy(g, ex)
        for s in (a, b, other):
            s.free()
        big.free()
        for q in w.values():
            q.close()
