"""A serving step of a model with experts, norms of its heads and long chats
as a program runs it: projections, norms and rotation, pages reserved, append,
attention over a window and sinks, pages behind the window released, output
projection, routing, grouped experts, head and sampling; a sequence forked on
the way, the pool compacted.  Every stage against its own restatement on what
the stage before it gave; the same step recorded and replayed."""
import numpy as np
import pytest

import kv_case as kc
import oracle as O
import rce_amd
import serve_case as sc
from bench import Hip
from kv_case import F32
from rce_amd import GgufDtype as G
from rce_amd import Mode

pytestmark = pytest.mark.gpu

DM, HEADS, PER, D, VOCAB, PAGE, EXPERTS, TOP, DFF = 256, 2, 2, 64, 300, 16, 16, 3, 128
N_Q, WIDTH = HEADS * PER, (HEADS * PER + 2 * HEADS) * D
WINDOW, SINKS, EPS, N, MAX_PAGES, N_PAGES = 24, 4, 1e-6, 4, 8, 26


class Model:
    def __init__(self, ctx, rng):
        self.ctx = ctx
        make = lambda r, c: O.quantize((rng.standard_normal((r, c)) * 0.06).astype(F32), O.Q8_0)  # noqa: E731
        self.raw = {"qkv": (WIDTH, DM), "wo": (DM, N_Q * D), "router": (EXPERTS, DM), "head": (VOCAB, DM)}
        self.raw = {k: (make(r, c), r, c) for k, (r, c) in self.raw.items()}
        self.w = {k: rce_amd.QuantWeight.from_owned_bytes(ctx, b, O.Q8_0, r, c) for k, (b, r, c) in self.raw.items()}
        self.experts = [[make(r, c) for _ in range(EXPERTS)] for r, c in ((DFF, DM), (DFF, DM), (DM, DFF))]
        self.we = [[rce_amd.QuantWeight.from_owned_bytes(ctx, b, O.Q8_0, r, c) for b in bs]
                   for bs, (r, c) in zip(self.experts, ((DFF, DM), (DFF, DM), (DM, DFF)))]
        self.norms = [(1 + 0.2 * rng.standard_normal(D)).astype(F32) for _ in range(2)]
        self.bias = (0.1 * rng.standard_normal(EXPERTS)).astype(F32)
        self.embd = rng.standard_normal((VOCAB, DM)).astype(F32)
        self.cs = rce_amd.Rope.scaled_table(10000.0, D, MAX_PAGES * PAGE, factor=4.0, orig_context=32)
        up = lambda a: rce_amd.DeviceBuffer.from_numpy(ctx, a)  # noqa: E731
        self.dev = [up(a) for a in (*self.norms, self.bias, self.cs)]

    def free(self):
        for w in [*self.w.values(), *(w for ws in self.we for w in ws)]:
            w.close()
        for b in self.dev:
            b.free()


class Step:
    """The device state of a program: a pool, tables and counts, and the buffers of up to `rows` rows."""

    def __init__(self, model, pool, rows):
        self.m, self.ctx, self.pool = model, model.ctx, pool
        up = lambda a: rce_amd.DeviceBuffer.from_numpy(self.ctx, a)  # noqa: E731
        alloc = lambda k: up(np.zeros(rows * k, F32))  # noqa: E731
        self.bufs = [up(getattr(pool, n)) for n in ("k", "v", "k_scale", "v_scale")]
        k, v, ks, vs = (b.ptr for b in self.bufs)
        self.cache = rce_amd.KvCache(N_PAGES, PAGE, HEADS, D, k=k, v=v, k_scale=ks, v_scale=vs)
        self.x, self.qkv, self.qk, self.att, self.y, self.lg = (alloc(c) for c in (DM, WIDTH, (N_Q + HEADS) * D, N_Q * D, DM, EXPERTS))
        self.ew, self.out, self.head = alloc(TOP), alloc(DM), alloc(VOCAB)
        self.eid = up(np.zeros(rows * TOP, np.int32))
        self.ids, self.u = up(np.zeros(rows, np.int32)), alloc(1)
        self.pages, self.refs = up(np.full((N, MAX_PAGES), -1, np.int32)), up(np.zeros(N_PAGES, np.int32))
        self.missing, self.lo, self.hi = (up(np.zeros(N, np.int32)) for _ in range(3))
        self.off, self.lens = up(np.zeros(N + 1, np.int32)), up(np.zeros(N, np.int32))
        self.table = rce_amd.KvTable(self.pages.ptr, N, MAX_PAGES)
        self.n = 0

    def put(self, x, u, offsets, lens):
        self.n = int(offsets[-1])
        for b, a in ((self.x, x), (self.u, u), (self.off, offsets.astype(np.int32)), (self.lens, lens.astype(np.int32)),
                     (self.lo, np.full(N, SINKS, np.int32)), (self.hi, np.maximum(lens - WINDOW + 1, 0).astype(np.int32))):
            b.upload(a)
        self.batch = rce_amd.KvBatch(self.off.ptr, self.lens.ptr, self.pages.ptr, N, self.n, MAX_PAGES)

    def run(self):
        c, m, n = self.ctx, self.m, self.n
        qn, kn, bias, cs = (b.ptr for b in m.dev)
        rce_amd.mm_batched_dev(c, self.x.ptr, G.F32, n, m.w["qkv"], self.qkv.ptr, Mode.EXACT)
        k_at, k_out = self.qkv.ptr + N_Q * D * 4, self.qk.ptr + N_Q * D * 4
        width = (N_Q + HEADS) * D
        rce_amd.qk_norm_rope_dev(c, self.batch, rce_amd.Heads(self.qkv.ptr, WIDTH, N_Q, self.qk.ptr, width, qn),
                                 rce_amd.Heads(k_at, WIDTH, HEADS, k_out, width, kn), D, G.F32, G.F32, EPS,
                                 rope=rce_amd.Rope(cs, D, MAX_PAGES * PAGE), interleaved=True)
        rce_amd.kv_reserve_dev(c, self.cache, self.batch, self.refs.ptr, self.missing.ptr)
        rce_amd.kv_append_dev(c, self.cache, self.batch, k_out, k_at + HEADS * D * 4, G.F32, width, WIDTH)
        rce_amd.kv_attention_sinks_dev(c, self.cache, self.batch, self.qk.ptr, G.F32, width, N_Q, self.att.ptr, G.F32, D ** -0.5, WINDOW, SINKS)
        rce_amd.kv_release_dev(c, self.cache, self.table, self.refs.ptr, self.lo.ptr, self.hi.ptr)
        rce_amd.mm_batched_dev(c, self.att.ptr, G.F32, n, m.w["wo"], self.y.ptr, Mode.EXACT)
        rce_amd.mm_batched_dev(c, self.y.ptr, G.F32, n, m.w["router"], self.lg.ptr, Mode.EXACT)
        rce_amd.moe_route_dev(c, self.lg.ptr, G.F32, n, EXPERTS, EXPERTS,
                              rce_amd.MoeRouting(TOP, sigmoid=True, bias_dev=bias, n_group=4, topk_group=2, group_top=2, scale=1.5),
                              self.eid.ptr, self.ew.ptr)
        rce_amd.moe_swiglu_dev(c, *m.we, self.y.ptr, n, self.eid.ptr, self.ew.ptr, TOP, self.out.ptr, Mode.F16_MFMA)
        rce_amd.mm_batched_dev(c, self.out.ptr, G.F32, n, m.w["head"], self.head.ptr, Mode.EXACT)
        rce_amd.sample_dev(c, self.head.ptr, G.F32, n, VOCAB, VOCAB, self.u.ptr, self.ids.ptr)

    def get(self, b, dtype, *shape):
        return b.download(dtype, int(np.prod(shape))).reshape(shape)

    def state(self):
        n = self.n
        return [self.get(b, np.uint32, n, k) for b, k in ((self.qkv, WIDTH), (self.qk, (N_Q + HEADS) * D), (self.att, N_Q * D), (self.lg, EXPERTS),
                                                          (self.eid, TOP), (self.ew, TOP), (self.out, DM), (self.head, VOCAB), (self.ids, 1))] + \
            [b.download(np.uint8, b.nbytes) for b in self.bufs] + [self.get(self.pages, np.int32, N, MAX_PAGES), self.get(self.refs, np.int32, N_PAGES)]

    def free(self):
        for b in vars(self).values():
            if isinstance(b, rce_amd.DeviceBuffer):
                b.free()
        for b in self.bufs:
            b.free()


def check(s, m, host, tables, x, u, offsets, lens):
    """Every stage of the step that `s` ran on what the stage before it gave; host, tables: the pool and tables before it."""
    n = s.n
    qkv = s.get(s.qkv, F32, n, WIDTH)
    mul = lambda a, k: O.mm_batched(a, m.raw[k][0], O.Q8_0, m.raw[k][1], m.raw[k][2]).reshape(n, -1)  # noqa: E731
    assert np.array_equal(qkv, mul(x, "qkv"))
    qk = s.get(s.qk, F32, n, N_Q + HEADS, D)
    for r in range(n):
        seq = int(np.searchsorted(offsets[1:], r, side="right"))
        pos = int(lens[seq] - (offsets[seq + 1] - r))
        for a, b, w in ((0, N_Q, m.norms[0]), (N_Q, N_Q + HEADS, m.norms[1])):
            y, bound = sc.norm_rope(qkv[r, a * D:b * D].reshape(-1, D), w, EPS, m.cs, pos, True)
            assert np.all(np.abs(qk[r, a:b] - y) <= bound + sc.U * np.abs(y))
    missing = tables.reserve(offsets.tolist(), lens.tolist())
    assert not any(missing) and not s.get(s.missing, np.int32, N).any()
    tables.apply(host)
    b = kc.Batch(lens.tolist(), np.diff(offsets).tolist(), tables.pages, PAGE)
    kc.append(host, b, qk[:, N_Q:], qkv[:, (N_Q + HEADS) * D:].reshape(n, HEADS, D), None)
    for name, buf in zip(("k", "v", "k_scale", "v_scale"), s.bufs):
        want = getattr(host, name)
        assert np.array_equal(buf.download(want.dtype, want.size).reshape(want.shape).view(np.uint8), want.view(np.uint8)), name
    att = s.get(s.att, F32, n, N_Q, D)
    for r, (y, bound) in sc.attention(host, b, qk[:, :N_Q], None, float(F32(D ** -0.5)), WINDOW, SINKS, True).items():
        assert np.all(np.abs(att[r] - y) <= bound + sc.U * np.abs(y))
    tables.release([SINKS] * N, np.maximum(lens - WINDOW + 1, 0).tolist())
    assert np.array_equal(s.get(s.pages, np.int32, N, MAX_PAGES), tables.pages) and np.array_equal(s.get(s.refs, np.int32, N_PAGES), tables.refs)
    y = mul(att.reshape(n, -1), "wo")
    lg = s.get(s.lg, F32, n, EXPERTS)
    assert np.array_equal(lg, mul(y, "router"))
    eid, ew = s.get(s.eid, np.int32, n, TOP), s.get(s.ew, F32, n, TOP)
    want_id, want_w = sc.route(lg, TOP, sigmoid=True, bias=m.bias, groups=4, kept=2, group_top=2, scale=1.5)
    assert np.array_equal(eid, want_id) and np.all(np.abs(ew - want_w) <= 2.0 ** -23 * want_w)
    out = s.get(s.out, F32, n, DM)
    ref = O.moe_swiglu_ffn(y, *m.experts, O.Q8_0, DFF, eid, ew).reshape(n, DM)
    assert np.linalg.norm(out - ref) <= 3e-3 * np.linalg.norm(ref)  # the mode's bound
    head = s.get(s.head, F32, n, VOCAB)
    assert np.array_equal(head, mul(out, "head"))
    ids = s.get(s.ids, np.int32, n)
    for r in range(n):
        assert ids[r] == kc.sample(head[r], u[r])[0]
    return ids


def test_step(ctx):
    rng = np.random.default_rng(41)
    m = Model(ctx, rng)
    host = kc.Pool(N_PAGES, PAGE, HEADS, D, rng)
    s = Step(m, host, 64)
    tables = sc.Tables(np.full((N, MAX_PAGES), -1), np.zeros(N_PAGES), PAGE)
    lens = np.zeros(N, int)
    tokens = None
    for step in range(9):
        news = np.array([21, 3, 35, 0]) if step == 0 else np.array([1, 1, 1, 1 if step > 2 else 0])
        if step == 3:  # the first prompt gets a second answer
            parents = rce_amd.DeviceBuffer.from_numpy(ctx, np.array([-1, -1, -1, 0], np.int32))
            rce_amd.kv_fork_dev(ctx, s.cache, s.table, s.table, parents.ptr, s.refs.ptr)
            ctx.synchronize()
            parents.free()
            tables.fork(tables.pages, [-1, -1, -1, 0])
            lens[3] = lens[0]
        if step == 6:  # the second one ends, the pool moves together
            lo = rce_amd.DeviceBuffer.from_numpy(ctx, np.array([1 << 20, 0, 1 << 20, 1 << 20], np.int32))
            ids = rce_amd.DeviceBuffer(ctx, 4 * N_PAGES)
            rce_amd.kv_release_dev(ctx, s.cache, s.table, s.refs.ptr, from_dev=lo.ptr)
            rce_amd.kv_compact_dev(ctx, s.cache, s.table, s.refs.ptr, ids.ptr)
            ctx.synchronize()
            tables.release([1 << 20, 0, 1 << 20, 1 << 20])
            want, _ = tables.compact()
            tables.apply(host)
            assert np.array_equal(ids.download(np.int32, N_PAGES), want)
            lo.free(); ids.free()
            lens[1] = 0
        lens = lens + news
        offsets = np.concatenate([[0], np.cumsum(news)])
        n = int(offsets[-1])
        if step == 3:
            tokens = np.append(tokens, rng.integers(0, VOCAB))  # the second answer begins with another token
        x = m.embd[rng.integers(0, VOCAB, n) if tokens is None else tokens]
        u = rng.random(n).astype(F32)
        s.put(x, u, offsets, lens)
        s.run()
        ctx.synchronize()
        drawn = check(s, m, host, tables, x, u, offsets, lens)
        tokens = drawn[offsets[1:][news > 0] - 1] if step == 0 else drawn
    s.free()
    m.free()


def test_recorded_step():
    """One token of each of four sequences, recorded once; replays between eager steps of another state on the same
    context leave what the eager step leaves, bit for bit."""
    rng = np.random.default_rng(42)
    with rce_amd.Context(0) as c:
        m = Model(c, rng)
        pool = kc.Pool(N_PAGES, PAGE, HEADS, D, rng)
        a, b, other = (Step(m, pool.copy(), 64) for _ in range(3))
        lens = np.array([20, 3, 35, 15])
        off = np.concatenate([[0], np.cumsum(lens)])
        x, u = m.embd[rng.integers(0, VOCAB, off[-1])], rng.random(off[-1]).astype(F32)
        for s in (a, b, other):
            for i in range(0, 4):  # the prompts, one after the other: 64 rows at most
                o = np.concatenate([np.zeros(i + 1, int), np.full(N - i, lens[i])])
                done = np.where(np.arange(N) <= i, lens, 0)
                s.put(x[off[i]:off[i + 1]], u[off[i]:off[i + 1]], o, done)
                s.run()
        c.synchronize()
        tokens, one = rng.integers(0, VOCAB, N), np.arange(N + 1)
        hip = Hip()
        a.put(m.embd[tokens], u[:N], one, lens + 1)
        g, ex = hip.capture(c.stream, a.run)
        for i in range(5):
            lens = lens + 1
            x, u = m.embd[tokens], rng.random(N).astype(F32)
            for s in (a, b):
                s.put(x, u, one, lens)
            other.put(x[::-1].copy(), u, one, lens)
            other.run()
            c.synchronize()
            hip.launch(ex, c.stream)
            other.run()
            c.synchronize()
            b.run()
            c.synchronize()
            for p, q in zip(a.state(), b.state()):
                assert np.array_equal(p, q), i
            tokens = a.get(a.ids, np.int32, N)
        hip.destroy(g, ex)
        for s in (a, b, other):
            s.free()
        m.free()
