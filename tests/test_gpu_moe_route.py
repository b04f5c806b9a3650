"""rce_qmm_moe_route_dev against the rule in 64 bits (serve_case.route): the
same experts, weights to a rounding; rows that leave nothing to choose,
infinities, equal logits, groups of every size, strides, replays."""
import numpy as np
import pytest

import kv_case as kc
import rce_amd
import serve_case as sc
from bench import Hip
from kv_case import F32
from rce_amd import GgufDtype as G

pytestmark = pytest.mark.gpu

# the sums and quotients of 64 bits: within 2^-40 of the weight for 1024 experts
WEIGHT = 2.0 ** -24 + 2.0 ** -40


def run(ctx, logits, dtype, how, stride=None, bias=None):
    """(ids, weights) of rows of bits, padded to `stride` with NaN."""
    n, e = logits.shape
    stride = stride or e
    pad = np.full((n, stride), 0x7FC0 if dtype == G.BF16 else np.nan, logits.dtype)
    pad[:, :e] = logits
    up = lambda a: rce_amd.DeviceBuffer.from_numpy(ctx, a)  # noqa: E731
    k = how["top_k"]
    lg, ids, w = up(pad), up(np.full((n + 1, k), -7, np.int32)), up(np.full((n + 1, k), np.nan, F32))
    b = None if bias is None else up(bias)
    routing = rce_amd.MoeRouting(k, sigmoid=how.get("sigmoid", False), bias_dev=0 if b is None else b.ptr, n_group=how.get("groups", 1),
                                 topk_group=how.get("kept", 1), group_top=how.get("group_top", 1),
                                 normalize=how.get("normalize", True), scale=how.get("scale", 1.0))
    rce_amd.moe_route_dev(ctx, lg.ptr, dtype, n, e, stride, routing, ids.ptr, w.ptr)
    ctx.synchronize()
    got = ids.download(np.int32, (n + 1) * k).reshape(n + 1, k), w.download(F32, (n + 1) * k).reshape(n + 1, k)
    assert np.all(got[0][n] == -7) and np.all(np.isnan(got[1][n]))  # nothing behind the last token
    for x in (lg, ids, w, b):
        if x is not None:
            x.free()
    return got[0][:n], got[1][:n]


def check(ctx, logits, dtype, how, **kw):
    bits = kc.to_bits(logits, dtype)
    with np.errstate(over="ignore"):
        ids, w = run(ctx, bits, dtype, how, **kw)
        want_ids, want = sc.route(kc.widen(bits, dtype), bias=kw.get("bias"), **how)
    assert np.array_equal(ids, want_ids), np.argwhere(ids != want_ids)[:5]
    assert np.all(np.abs(w - want) <= WEIGHT * np.abs(want) + 2.0 ** -150)


HOWS = [dict(top_k=1), dict(top_k=2, normalize=False), dict(top_k=2, sigmoid=True, scale=2.5), dict(top_k=4, sigmoid=True, normalize=False)]


@pytest.mark.parametrize("dtype", [G.F32, G.F16, G.BF16])
@pytest.mark.parametrize("experts", [4, 7, 8, 9, 16, 33, 60, 64, 65, 128, 160, 256, 300, 512, 1000, 1024])
def test_experts(ctx, experts, dtype):
    print(f"route experts={experts} dtype={dtype}", flush=True)
    rng = np.random.default_rng(experts)
    for i, how in enumerate(HOWS):
        n = (1, 3, 37, 130)[i]
        lg = (rng.standard_normal((n, experts)) * 2).astype(F32)
        bias = (rng.standard_normal(experts) * 0.3).astype(F32) if i % 2 else None
        check(ctx, lg, dtype, how, bias=bias, stride=experts + (0, 1, 5, 64)[i])


@pytest.mark.parametrize("experts,top_k", [(8, 8), (5, 5), (16, 16), (64, 17), (64, 64), (40, 33), (256, 64), (1024, 64)])
@pytest.mark.parametrize("bias", [False, True])
def test_many_chosen(ctx, experts, top_k, bias):
    rng = np.random.default_rng(top_k)
    lg = rng.standard_normal((9, experts)).astype(F32)
    check(ctx, lg, G.F32, dict(top_k=top_k, sigmoid=bias), bias=rng.standard_normal(experts).astype(F32) if bias else None)


@pytest.mark.parametrize("experts,groups,kept,top_k", [(8, 2, 1, 2), (8, 8, 3, 3), (256, 8, 4, 8), (160, 8, 3, 6), (64, 64, 5, 5), (60, 3, 2, 7),
                                                       (512, 16, 1, 8), (1024, 32, 31, 4), (12, 4, 4, 2), (130, 13, 6, 2), (1024, 2, 1, 64)])
@pytest.mark.parametrize("group_top", [1, 2])
@pytest.mark.parametrize("sigmoid,bias", [(False, False), (True, False), (True, True), (False, True)])
def test_groups(ctx, experts, groups, kept, top_k, group_top, sigmoid, bias):
    rng = np.random.default_rng(experts + groups + group_top)
    lg = (rng.standard_normal((21, experts)) * 1.5).astype(F32)
    b = (rng.standard_normal(experts) * 0.2).astype(F32) if bias else None
    for dtype in (G.F32, G.BF16):
        check(ctx, lg, dtype, dict(top_k=top_k, sigmoid=sigmoid, groups=groups, kept=kept, group_top=group_top), bias=b)


def odd_rows(rng, e):
    """Rows with nothing to choose, little to choose, and no order among some."""
    x = rng.standard_normal((14, e)).astype(F32)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, 1:] = -np.inf
    x[3, :-1] = np.nan
    x[4] = 0
    x[4, ::2] = -0.0
    x[5] = np.inf
    x[6, e // 2] = np.inf
    x[6, 0] = -np.inf
    x[7] = 3.25
    x[8] *= 1e30
    x[9] *= 1e-42  # subnormal
    x[10, :] = -1e4
    x[10, e // 3] = -1e4 + 1
    x[11, ::3] = -np.inf
    x[11, 1::3] = np.nan
    x[12] = np.where(np.arange(e) % 2, np.finfo(F32).max, np.finfo(F32).min)
    x[13] = np.round(x[13])  # many equals
    return x


@pytest.mark.parametrize("experts,how", [(8, dict(top_k=2)), (8, dict(top_k=8, sigmoid=True)), (33, dict(top_k=5, normalize=False)), (64, dict(top_k=20)),
                                         (256, dict(top_k=8, sigmoid=True)), (200, dict(top_k=8, groups=8, kept=3)),
                                         (256, dict(top_k=8, groups=8, kept=4, group_top=2, sigmoid=True)), (24, dict(top_k=9, groups=6, kept=3, group_top=2))])
@pytest.mark.parametrize("bias", [None, "some", "odd"])
def test_odd_rows(ctx, experts, how, bias):
    """(-1e4 and the like are beyond binary16: the rows become infinities there, which is a case of its own)"""
    print(f"route odd rows experts={experts} {how} bias={bias}", flush=True)
    rng = np.random.default_rng(experts)
    lg = odd_rows(rng, experts)
    b = None
    if bias:
        b = (rng.standard_normal(experts) * 0.5).astype(F32)
        if bias == "odd":
            b[:5] = np.nan, -np.inf, np.inf, 1e30, -1e30
    for dtype in (G.F32, G.BF16, G.F16):
        with np.errstate(over="ignore"):
            check(ctx, lg, dtype, how, bias=b)


MANY = 10003  # tokens of a call from which several share a wave, and an odd rest


@pytest.mark.parametrize("experts,how", [(9, dict(top_k=2)), (60, dict(top_k=4, sigmoid=True)), (64, dict(top_k=16)), (64, dict(top_k=6, groups=8, kept=3)),
                                         (100, dict(top_k=5, normalize=False)), (128, dict(top_k=8, groups=4, kept=2, group_top=2, sigmoid=True)),
                                         (160, dict(top_k=6, groups=10, kept=4)), (160, dict(top_k=6, groups=8, kept=3, group_top=2)), (256, dict(top_k=8, sigmoid=True)),
                                         (256, dict(top_k=8, groups=8, kept=4, group_top=2, sigmoid=True)), (256, dict(top_k=1, groups=2, kept=1, group_top=2)),
                                         (256, dict(top_k=12, groups=16, kept=5, normalize=False)), (250, dict(top_k=3)), (200, dict(top_k=2, groups=5, kept=2))])
@pytest.mark.parametrize("bias", [None, "some", "odd", "wide"])
def test_many_tokens(ctx, experts, how, bias):
    """Rows of all sorts among ordinary ones; strides that are whole words, and not; biases far beyond the scores."""
    print(f"route many experts={experts} {how} bias={bias}", flush=True)
    rng = np.random.default_rng(experts)
    lg = (rng.standard_normal((MANY, experts)) * 2).astype(F32)
    lg[100:114], lg[-14:] = odd_rows(rng, experts), odd_rows(rng, experts)
    lg[500:700] = np.round(lg[500:700] * 4) / 4  # equals in every row
    b = None
    if bias:
        b = (rng.standard_normal(experts) * (3 if bias == "wide" else 0.3)).astype(F32)
        if bias == "odd":
            b[:5] = np.nan, -np.inf, np.inf, 1e30, -1e30
    at = np.concatenate([np.arange(90, 120), rng.integers(0, MANY, 100), np.arange(500, 540), np.arange(MANY - 20, MANY)])
    for i, dtype in enumerate((G.F32, G.BF16, G.F16)):
        bits = kc.to_bits(lg, dtype)
        ids, w = run(ctx, bits, dtype, how, stride=experts + (3, 0, 4)[i], bias=b)
        want_ids, want = sc.route(kc.widen(bits[at], dtype), bias=b, **how)
        assert np.array_equal(ids[at], want_ids), np.argwhere(ids[at] != want_ids)[:5]
        assert np.all(np.abs(w[at] - want) <= WEIGHT * np.abs(want) + 2.0 ** -150)


def test_scores_next_to_each_other(ctx):
    """Scores that 32 bits hold as equals, a bias apart: 1 - 2^-26 against 1 - 2^-27 by the sigmoid, and by the
    softmax two logits that differ by 2^-23 under a bias of 1000."""
    lg = np.array([[18.0215, 18.7150, 0, 0, 0, 0, 0, 0], [18.7150, 18.0215, 0, 0, 0, 0, 0, 0]], F32)
    check(ctx, lg, G.F32, dict(top_k=1, sigmoid=True), bias=np.zeros(8, F32))
    lg = np.array([[0.5, 0.5 + 2.0 ** -23, 0, 0], [0.5 + 2.0 ** -23, 0.5, 0, 0]], F32)
    check(ctx, lg, G.F32, dict(top_k=1), bias=np.array([1000, 1000, 0, 0], F32))
    # among many tokens, and of many experts: the first two a step of the last bit apart, either way round
    for e, n in ((16, 10002), (100, 9), (256, 10002), (256, 9)):
        rng = np.random.default_rng(e)
        lg = (rng.standard_normal((n, e)) * 0.3).astype(F32)
        up, down = F32(3), np.nextafter(F32(3), F32(0))
        lg[::2, e // 2], lg[::2, e // 3] = up, down
        lg[1::2, e // 2], lg[1::2, e // 3] = down, up
        for bias in (None, np.full(e, 0.5, F32)):
            at = np.arange(0, n, max(1, n // 40))
            for how in (dict(top_k=2, sigmoid=True), dict(top_k=1)):
                ids, _ = run(ctx, lg, G.F32, how, bias=bias)
                assert np.array_equal(ids[at], sc.route(lg[at], bias=bias, **how)[0])


def near_groups(rng, n, e, groups, size, sigmoid):
    """(logits [n, e], bias [e], the two groups): two groups of which each counts by a bias of +b and one of -b, their sums
    1e-7 to 1e-5 apart one way or the other (a logit's rounding moves a sum by 2^-24 at most); all other experts far below."""
    g0, g1 = sorted(rng.choice(groups, 2, replace=False))
    at = [g0 * size, g0 * size + size - 1, g1 * size, g1 * size + size - 1]
    lg = np.full((n, e), -30.0, F32)
    apart = 10.0 ** rng.uniform(-7, -5, n) * rng.choice([-1, 1], n)
    if sigmoid:
        s = rng.uniform(0.3, 0.7, (n, 3))
        s = np.column_stack([s, s[:, 0] + s[:, 1] - s[:, 2] + apart])
        s = np.where((s[:, 3:] > 0.05) & (s[:, 3:] < 0.95), s, np.array([0.4, 0.6, 0.55, 0.45]) + apart[:, None] * [0, 0, 0, 1])
        lg[:, at] = np.log(s / (1 - s))
    else:
        a = rng.uniform(0.1, 0.9, (n, 2)) * np.column_stack([0.5 + apart / 2, 0.5 - apart / 2])
        lg[:, at] = np.log(np.column_stack([a[:, 0], 0.5 + apart / 2 - a[:, 0], a[:, 1], 0.5 - apart / 2 - a[:, 1]]))
    return lg, at


@pytest.mark.parametrize("experts,groups", [(4, 2), (16, 4), (64, 8), (128, 4), (256, 8), (256, 2), (512, 16), (1024, 32)])
@pytest.mark.parametrize("sigmoid", [True, False])
@pytest.mark.parametrize("size", [2.0, 16.0, 100.0, 1000.0, 3e4])
def test_groups_whose_biases_cancel(ctx, experts, groups, sigmoid, size):
    """A group counts by two experts of opposite large biases: the sum is small, what 32 bits lose of each addend is not.  Few
    tokens, and the same rows in a call of many."""
    print(f"route cancelling experts={experts} groups={groups} sigmoid={sigmoid} size={size}", flush=True)
    rng = np.random.default_rng(experts + int(size))
    per = experts // groups
    lg, at = near_groups(rng, 200, experts, groups, per, sigmoid)
    bias = np.full(experts, -4 * size, F32)
    bias[at] = size, -size, size, -size
    how = dict(top_k=2, sigmoid=sigmoid, groups=groups, kept=1, group_top=2)
    check(ctx, lg, G.F32, how, bias=bias)
    many = np.tile(lg, (33, 1))  # 6600 tokens
    ids, _ = run(ctx, many, G.F32, how, bias=bias)
    assert np.array_equal(ids, np.tile(sc.route(lg, bias=bias, **how)[0], (33, 1)))


def test_a_group_lost_to_its_neighbour(ctx):
    """64 bits: 0.67821895 against 0.67821878; sums of what 32 bits hold of the addends: 0.67821789 against 0.67821980."""
    lg = np.array([[-0.96945596, -0.39202467, 0.28211886, -2.1097460]], F32)
    check(ctx, lg, G.F32, dict(top_k=2, sigmoid=True, groups=2, kept=1, group_top=2), bias=np.array([16, -16, 16, -16], F32))


def test_group_sums_beyond_32_bits(ctx):
    """Two biases whose sum passes binary32, up or down, beside groups that are as far out, nearer, or hold no expert."""
    big = 3e38
    for b in ([big, big, big, 3.1e38, 1, 1, 0, 0], [-big, -big, -3.1e38, -big, np.nan, np.nan, -np.inf, -np.inf],
              [-big, -big, np.nan, -np.inf, -big, -3.1e38, np.nan, np.nan], [np.inf, 0, big, big, np.inf, 1, np.nan, np.inf]):
        rng = np.random.default_rng(11)
        lg = rng.standard_normal((20, 8)).astype(F32)
        for perm in ([0, 1, 2, 3, 4, 5, 6, 7], [6, 7, 0, 1, 4, 5, 2, 3], [2, 3, 6, 7, 0, 1, 4, 5]):
            for kept, k in ((1, 1), (1, 2), (2, 3), (3, 6)):
                with np.errstate(over="ignore"):
                    check(ctx, lg, G.F32, dict(top_k=k, sigmoid=True, groups=4, kept=kept, group_top=2), bias=np.array(b, F32)[perm])


def test_a_wide_call(ctx):
    """Rows further apart than 2^31 values, and more tokens than a launch's first blocks."""
    n, e, stride = 3, 8, (1 << 30) + 8
    rng = np.random.default_rng(0)
    lg = rng.standard_normal((n, e)).astype(F32)
    big = rce_amd.DeviceBuffer(ctx, 2 * (2 * stride + e))
    bits = kc.to_bits(lg, G.F16)
    for r in range(n):
        rce_amd._lib.check(rce_amd._lib.lib().rce_qmm_memcpy_h2d(ctx.handle, big.ptr + 2 * r * stride, bits[r].ctypes.data, 2 * e))
    ids, w = (rce_amd.DeviceBuffer(ctx, 4 * n * 2) for _ in range(2))
    rce_amd.moe_route_dev(ctx, big.ptr, G.F16, n, e, stride, rce_amd.MoeRouting(2), ids.ptr, w.ptr)
    ctx.synchronize()
    want, _ = sc.route(kc.widen(bits, G.F16), 2)
    assert np.array_equal(ids.download(np.int32, n * 2).reshape(n, 2), want)
    for b in (big, ids, w):
        b.free()
    lg = rng.standard_normal((70001, 8)).astype(F32)
    ids, w = run(ctx, lg, G.F32, dict(top_k=2))
    at = rng.integers(0, len(lg), 300)
    want, ww = sc.route(lg[at], 2)
    assert np.array_equal(ids[at], want) and np.all(np.abs(w[at] - ww) <= WEIGHT * ww)


def test_same_as_the_host_router(ctx):
    """rce_qmm_moe_router's softmax in f32: the same experts for logits apart, weights to its arithmetic."""
    rng = np.random.default_rng(3)
    lg = rng.standard_normal((256, 8)).astype(F32)
    for normalize in (True, False):
        ids, w = run(ctx, lg, G.F32, dict(top_k=2, normalize=normalize))
        hi, hw = rce_amd.moe_router(lg, 2, normalize)
        assert np.array_equal(ids, hi)
        assert np.all(np.abs(w - hw) <= 16 * 2.0 ** -24 * hw)  # 8 exponentials, their sum, two quotients


def test_recorded(ctx):
    rng = np.random.default_rng(4)
    n, e, k = 50, 256, 8
    hip = Hip()
    up = lambda a: rce_amd.DeviceBuffer.from_numpy(ctx, a)  # noqa: E731
    lg, bias = up(np.zeros((n, e), F32)), (rng.standard_normal(e) * 0.2).astype(F32)
    b, ids, w = up(bias), up(np.zeros((n, k), np.int32)), up(np.zeros((n, k), F32))
    how = rce_amd.MoeRouting(k, sigmoid=True, bias_dev=b.ptr, n_group=8, topk_group=4, group_top=2)
    g, ex = hip.capture(ctx.stream, lambda: rce_amd.moe_route_dev(ctx, lg.ptr, G.F32, n, e, e, how, ids.ptr, w.ptr))
    for _ in range(3):
        x = rng.standard_normal((n, e)).astype(F32)
        lg.upload(x)
        run(ctx, x[:, :8].copy(), G.F32, dict(top_k=2))
        hip.launch(ex, ctx.stream)
        ctx.synchronize()
        want, ww = sc.route(x, k, sigmoid=True, bias=bias, groups=8, kept=4, group_top=2)
        assert np.array_equal(ids.download(np.int32, n * k).reshape(n, k), want)
        assert np.all(np.abs(w.download(F32, n * k).reshape(n, k) - ww) <= WEIGHT * ww)
    hip.destroy(g, ex)
    for x in (lg, b, ids, w):
        x.free()
