"""Sampling from vocabularies above 2^18, whose runs have several steps and whose
weights have fewer bits."""
import numpy as np
import pytest

import kv_case as kc
from kv_case import F32
from rce_amd import GgufDtype as G
from test_gpu_sample import Call, rows

pytestmark = pytest.mark.gpu


def check(call):
    """The oracle's tokens; of a probability w / total the rounding to f32, and what weights as whole
    numbers of 2^-S leave of it: half a unit in w and in each of the vocabulary's."""
    call.call()
    call.ctx.synchronize()
    ids, probs = call.result()
    unit = 2.0 ** -min(50, 62 - int(np.ceil(np.log2(call.v))))
    for r, (i, p) in enumerate(call.expect()):
        assert ids[r] == i, (r, int(ids[r]), i, {k: a[r] for k, a in call.par.items()}, call.u[r])
        if i < 0 or p == 1.0:
            assert probs[r] == F32(p)
            continue
        t = float(call.par["temperature"][r]) if "temperature" in call.par else 1.0
        w = np.exp((float(call.x[r, i]) - float(call.x[r].max())) / t)
        allowed = p * (2.0 ** -23 + unit / 2 * (1 / w + call.v * p / w))
        assert abs(probs[r] - p) <= allowed, (r, probs[r], p, allowed)
    call.free()


FILTERS = [{}, {"top_p": 0.9}, {"top_k": 40}, {"top_k": 1000, "top_p": 0.95}, {"top_k": 5000}, {"top_k": 300000, "top_p": 0.8},
           {"min_p": 0.01, "temperature": 0.7}, {"temperature": 0.0}]


@pytest.mark.parametrize("par", FILTERS, ids=str)
@pytest.mark.parametrize("v,dtype", [(262144, G.F32), (262145, G.F32), (262145, G.BF16), (1500013, G.F32), (1500013, G.F16)])
def test_large_vocabularies(ctx, v, dtype, par):
    print(f"sample v={v} {dtype.name} {par}", flush=True)
    x, u = rows(v, 4, v)
    x[2] *= F32(0.02)  # flat: any run, and the last one
    x[3] *= F32(0.02)
    u[3] = np.nextafter(F32(1), F32(0))
    check(Call(ctx, x, dtype, u, stride=v + 7, **par))


def test_the_largest_vocabulary(ctx):
    """2^24 logits, flat: the draws fall into every quarter."""
    v = 1 << 24
    rng = np.random.default_rng(4)
    x = (rng.standard_normal((4, v), F32) * F32(0.01))
    check(Call(ctx, x, G.F16, [0.1, 0.3, 0.6, np.nextafter(F32(1), F32(0))]))


def test_many_rows(ctx):
    """More rows than a call splits: a block per row."""
    v, n = 262145, 130
    x, u = rows(5, n, v)
    x[::5] *= F32(0.02)
    rng = np.random.default_rng(6)
    par = {"top_k": rng.choice([0, 30, 3000], n), "top_p": rng.choice([0.6, 1.0], n)}
    check(Call(ctx, x, G.F16, u, stride=v + 2, **par))
