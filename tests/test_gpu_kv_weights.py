"""Attention's softmax weights where they are small or meet values of very
different size: weights far below the largest count in their sum, and what a
row does not see has no part in its precision."""
import numpy as np
import pytest

import kv_case as kc
import rce_amd
from kv_case import F32
from rce_amd import GgufDtype as G
from test_gpu_kv import Attn, check_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out_dtype", [G.F32, G.F16, G.BF16])
@pytest.mark.parametrize("new,n", [(1, 512), (40, 64), (600, 16)])
def test_many_small_weights_count_in_the_sum(ctx, new, n, out_dtype):
    """Key 0 outweighs each of 65536 others by 2^22.6, all together by 2^6.6; only its value is not
    zero, so every result is that value times its weight.  One value scale in four is 2^11.9 larger.
    Sequences of the same pages, so many that their keys are not split over blocks.

    Allowed, relative: the result's rounding; the weight's (2^-11 in one binary16 term, 2^-21
    in two); half an ulp of a sum below 2 for each of the 1024 tiles; 2^-16 for the roundings of the scores
    (of 22.6, in binary32 and from a query of 15 bits: below 2^-11 of weights that make 2^-6.6)
    and the sums of 16 terms."""
    length, page, heads, d = 65536, 1024, 8, 64
    print(f"small weights new={new} n={n} {out_dtype.name}", flush=True)
    rng = np.random.default_rng(1)
    one, n_pages = kc.make_batch(rng, [length], [new], page)
    batch = kc.Batch([length] * n, [new] * n, np.repeat(one.pages, n, 0), page)
    pool = kc.Pool(n_pages, page, heads, d, rng)
    pool.k[:] = 0
    pool.v[:] = 0
    p0 = batch.pages[0, 0]
    pool.k[p0, :, 0, 0, 0] = 127
    pool.v[p0, :, 0, :, 0] = 100
    pool.k_scale[:] = F32(22.6 * np.log(2) / 127)
    pool.v_scale[:] = 1
    pool.v_scale[:, :, 1::4] = F32(2.0 ** 11.9)

    def q_edit(x):
        x[:] = 0
        x[:, ::d] = 1
    a = Attn(ctx, pool, batch, heads, G.F32, out_dtype, scale=1.0, q_edit=q_edit)
    a.call()
    ctx.synchronize()
    got = kc.widen(a.bits(), out_dtype).reshape(n, new, heads, d).astype(np.float64)
    top = np.exp(float(pool.k_scale[p0, 0, 0]) * 127)
    others = length - new + np.arange(new)
    want = (100 * top / (top + others))[:, None, None]
    allowed = kc.out_eps(out_dtype) + (2.0 ** -21 if out_dtype == G.F32 else 2.0 ** -11) + 1024 * 2.0 ** -24 + 2.0 ** -16
    off = np.abs(got / want - 1).max()
    a.free()
    assert off <= allowed, (off, allowed)


@pytest.mark.parametrize("out_dtype", [G.F32, G.BF16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 9])
def test_values_of_unseen_blocks_cost_no_precision(ctx, d, window, out_dtype):
    """Each block's values are 2^30 times the last one's, or (rows that see at most 9 positions) the
    next one's: rows of one unit see values of very different size, and every row is as exact as what
    it sees allows."""
    for flip in (False, True)[:2 if window else 1]:
        def edit(pool, b):
            for s, length in enumerate(b.lens):
                for blk in range(-(-length // 16)):
                    page = b.pages[s, blk * 16 // pool.page]
                    pool.v_scale[page, :, blk % pool.b] *= F32(2.0 ** (30 * ((3 - blk) if flip else blk)))
        check_attention(ctx, d, 1, 1, 32, [60, 37], [20, 5], G.F32, out_dtype, edit=edit, window=window)
        check_attention(ctx, d, 2, 1, 32, [64], [64], G.F32, out_dtype, edit=edit, window=window)
        check_attention(ctx, d, 1, 4, 16, [50, 64], [50, 40], G.F32, out_dtype, edit=edit, window=window)


@pytest.mark.parametrize("out_dtype", [G.F16, G.BF16])
@pytest.mark.parametrize("d", [64, 128, 192, 256])
def test_single_tokens_to_16_bits_have_two_terms_per_weight(ctx, d, out_dtype):
    """Queries that are exact in 15 bits and small scores, so that the bound of F32 results holds;
    results near 0 (many of those over all dimensions) tell a weight's rounding to 2^-11 from one to 2^-21."""
    rng = np.random.default_rng(d)
    batch, n_pages = kc.make_batch(rng, [20, 17, 2500, 40], [1, 2, 1, 3], 32)
    pool = kc.Pool(n_pages, 32, 2, d, rng)

    def q_edit(x):
        x[:] = np.rint(x * 30).clip(-127, 127)
        x[:, ::d] = 127
    a = Attn(ctx, pool, batch, 6, G.F16, out_dtype, scale=2.0 ** -10, q_edit=q_edit)
    a.call()
    ctx.synchronize()
    rows = batch.n_rows
    got = kc.widen(a.bits(), out_dtype).reshape(rows, 6, d).astype(np.float64)
    want, bound = kc.attention(pool, batch, a.q, None, a.scale, 0, True)
    a.free()
    far = np.abs(got - want) - (bound + kc.out_eps(out_dtype) * (np.abs(want) + bound) + 2.0 ** -25)
    assert far.max() <= 0, (far.max(), bound.max())
