"""A serving step as a program runs it: projections of several sequences by
mm_batched_dev, append, attention, output projection and head, sampling, the
drawn tokens' embeddings into the next step; every stage against its own
restatement on the stage's actual inputs."""
import numpy as np
import pytest

import kv_case as kc
import oracle as O
import rce_amd
from kv_case import F32
from rce_amd import GgufDtype as G
from rce_amd import Mode

pytestmark = pytest.mark.gpu


def test_step(ctx):
    rng = np.random.default_rng(31)
    dm, heads, per, d, vocab, page, n = 256, 2, 2, 64, 500, 16, 3
    n_q = heads * per
    width = (n_q + 2 * heads) * d
    make = lambda r, c: O.quantize((rng.standard_normal((r, c)) * 0.06).astype(F32), O.Q8_0)  # noqa: E731
    raw = {"qkv": (make(width, dm), width, dm), "wo": (make(dm, n_q * d), dm, n_q * d), "head": (make(vocab, dm), vocab, dm)}
    w = {k: rce_amd.QuantWeight.from_owned_bytes(ctx, b, O.Q8_0, r, c) for k, (b, r, c) in raw.items()}
    embd = rng.standard_normal((vocab, dm)).astype(F32)
    news = [7, 1, 18]  # the prompts, then single tokens
    steps = 6
    full, n_pages = kc.make_batch(rng, [m + steps for m in news], news, page)
    pool = kc.Pool(n_pages, page, heads, d, rng)
    cs = kc.rope_cs(d, full.cap)
    rows_max = sum(news)
    dev = kc.Device(ctx, pool, full, cs)
    alloc = lambda nbytes: rce_amd.DeviceBuffer(ctx, nbytes)  # noqa: E731
    x, qkv, att, y, lg = (alloc(4 * rows_max * c) for c in (dm, width, n_q * d, dm, vocab))
    ids, u, temp, topk, topp = (alloc(4 * n) for _ in range(5))
    temp.upload(np.full(n, 0.8, F32)); topk.upload(np.array([0, 20, 3], np.int32)); topp.upload(np.array([0.9, 1, 0.7], F32))
    scale = float(F32(d ** -0.5))
    host, lens = pool.copy(), [0] * n
    tokens = rng.integers(0, vocab, rows_max)
    for step in range(steps):
        counts = news if step == 0 else [1] * n
        lens = [a + m for a, m in zip(lens, counts)]
        b = kc.Batch(lens, counts, full.pages, page)
        rows = b.n_rows
        dev.bufs[4].upload(b.offsets)
        dev.bufs[5].upload(np.asarray(lens, np.int32))
        dev.rows(rows)
        xin = embd[tokens]
        x.upload(xin)
        uu = rng.random(n).astype(F32)
        u.upload(uu)
        # the whole step on the device
        rce_amd.mm_batched_dev(ctx, x.ptr, G.F32, rows, w["qkv"], qkv.ptr, Mode.EXACT)
        k_at = qkv.ptr + n_q * d * 4
        rce_amd.kv_append_dev(ctx, dev.cache, dev.b, k_at, k_at + heads * d * 4, G.F32, width, width, rope=dev.rope)
        rce_amd.kv_attention_dev(ctx, dev.cache, dev.b, qkv.ptr, G.F32, width, n_q, att.ptr, G.F32, scale, rope=dev.rope)
        rce_amd.mm_batched_dev(ctx, att.ptr, G.F32, rows, w["wo"], y.ptr, Mode.EXACT)
        rce_amd.mm_batched_dev(ctx, y.ptr, G.F32, rows, w["head"], lg.ptr, Mode.EXACT)
        # the last row of each sequence: one call a sequence where the rows are not evenly spaced
        if step == 0:
            for s in range(n):
                rce_amd.sample_dev(ctx, lg.ptr + 4 * vocab * (int(b.offsets[s + 1]) - 1), G.F32, 1, vocab, vocab, u.ptr + 4 * s,
                                   ids.ptr + 4 * s, temperature_dev=temp.ptr + 4 * s, top_k_dev=topk.ptr + 4 * s,
                                   top_p_dev=topp.ptr + 4 * s)
        else:
            rce_amd.sample_dev(ctx, lg.ptr, G.F32, n, vocab, vocab, u.ptr, ids.ptr, temperature_dev=temp.ptr,
                               top_k_dev=topk.ptr, top_p_dev=topp.ptr)
        ctx.synchronize()
        # each stage on what the one before it gave
        got = qkv.download(F32, rows * width).reshape(rows, width)
        assert np.array_equal(got, O.mm_batched(xin, raw["qkv"][0], O.Q8_0, width, dm).reshape(rows, width))
        cut = lambda a, c: got[:, a:a + c * d].reshape(rows, c, d)  # noqa: E731
        kc.append(host, b, cut(n_q * d, heads), cut((n_q + heads) * d, heads), cs)
        state = dev.download()
        for name in ("k", "v", "k_scale", "v_scale"):
            assert np.array_equal(getattr(state, name), getattr(host, name)), name
        a = att.download(F32, rows * n_q * d).reshape(rows, n_q, d)
        want, bound = kc.attention(host, b, cut(0, n_q), cs, scale, 0, True)
        assert np.all(np.abs(a - want) <= bound + 2.0 ** -24 * np.abs(want))
        yy = O.mm_batched(a.reshape(rows, -1), raw["wo"][0], O.Q8_0, dm, n_q * d).reshape(rows, dm)
        logits = O.mm_batched(yy, raw["head"][0], O.Q8_0, vocab, dm).reshape(rows, vocab)
        assert np.array_equal(lg.download(F32, rows * vocab).reshape(rows, vocab), logits)
        drawn = ids.download(np.int32, n)
        for s in range(n):
            assert drawn[s] == kc.sample(logits[b.offsets[s + 1] - 1], uu[s], 0.8, (0, 20, 3)[s], F32((0.9, 1, 0.7)[s]))[0]
        tokens = drawn
    for q in (x, qkv, att, y, lg, ids, u, temp, topk, topp):
        q.free()
    dev.free()
