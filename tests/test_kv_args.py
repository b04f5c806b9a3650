"""What the kv and sampling entry points refuse, on the host: nothing here
reaches a device (no argument check looks at the context or follows a device
address), and the tables and sizes a program computes."""
import ctypes

import numpy as np
import pytest

import kv_case as kc
import rce_amd
from rce_amd import _lib
from rce_amd import GgufDtype as G

NULL, BAD, DTYPE = 1, 2, 3


class FakeContext:
    """Not a context: refusals come before its first use."""

    def __init__(self):
        self.room = ctypes.create_string_buffer(4096)
        self.handle = ctypes.c_void_p(ctypes.addressof(self.room))


def cache(**kw):
    a = dict(n_pages=4, page_tokens=32, n_kv_heads=2, d_head=64, k=1 << 20, v=2 << 20, k_scale=3 << 20, v_scale=4 << 20)
    a.update(kw)
    return rce_amd.KvCache(**a)


def batch(**kw):
    a = dict(row_offsets=5 << 20, seq_lens=6 << 20, pages=7 << 20, n_seqs=2, n_rows=3, max_pages=2)
    a.update(kw)
    return rce_amd.KvBatch(**a)


def refused(status, f, *args, **kw):
    with pytest.raises(rce_amd.QmmError) as e:
        f(*args, **kw)
    assert e.value.status == status, e.value


BAD_CACHES = [(dict(page_tokens=8), BAD), (dict(page_tokens=48), BAD), (dict(page_tokens=8192), BAD), (dict(page_tokens=0), BAD),
              (dict(d_head=80), BAD), (dict(d_head=0), BAD), (dict(d_head=512), BAD), (dict(n_kv_heads=0), BAD),
              (dict(n_kv_heads=1 << 40), BAD), (dict(n_pages=0), BAD), (dict(n_pages=1 << 31), BAD), (dict(n_pages=1 << 20, page_tokens=4096, n_kv_heads=16), BAD), (dict(k=0), NULL),
              (dict(v=0), NULL), (dict(k_scale=0), NULL), (dict(v_scale=0), NULL), (dict(k=(1 << 20) + 8), BAD),
              (dict(v=(1 << 20) + 1), BAD), (dict(k_scale=(1 << 20) + 2), BAD), (dict(v_scale=(1 << 20) + 1), BAD)]
BAD_BATCHES = [(dict(row_offsets=0), NULL), (dict(seq_lens=0), NULL), (dict(pages=0), NULL), (dict(pages=(1 << 20) + 2), BAD),
               (dict(n_seqs=(1 << 20) + 1), BAD), (dict(n_rows=(1 << 27) + 1), BAD), (dict(max_pages=1 << 30), BAD),
               (dict(max_pages=(1 << 64) - 1), BAD), (dict(n_rows=(1 << 64) - 1), BAD)]


def append(c, b, rope=None, k=8 << 20, v=9 << 20, dtype=G.F32, ks=128, vs=128):
    rce_amd.kv_append_dev(FakeContext(), c, b, k, v, dtype, ks, vs, rope=rope)


def read(c, b, k=8 << 20, v=9 << 20, dtype=G.F32):
    rce_amd.kv_read_dev(FakeContext(), c, b, k, v, dtype)


def attend(c, b, rope=None, q=8 << 20, qt=G.F32, qs=256, n_q=4, out=9 << 20, ot=G.F32, scale=0.125, window=0, os=256):
    rce_amd.kv_attention_dev(FakeContext(), c, b, q, qt, qs, n_q, out, ot, scale, rope=rope, window=window, out_stride=os)


@pytest.mark.parametrize("call", [append, read, attend])
def test_caches_and_batches(call):
    for kw, st in BAD_CACHES:
        refused(st, call, cache(**kw), batch())
    for kw, st in BAD_BATCHES:
        refused(st, call, cache(), batch(**kw))
    refused(NULL, call, None, batch())
    refused(NULL, call, cache(), None)


@pytest.mark.parametrize("call", [append, attend])
def test_rotation_tables(call):
    for rope, st in ((rce_amd.Rope(0, 64, 64), NULL), (rce_amd.Rope(1 << 20, 63, 64), BAD), (rce_amd.Rope(1 << 20, 66, 64), BAD),
                     (rce_amd.Rope(1 << 20, 64, 63), BAD), (rce_amd.Rope((1 << 20) + 2, 64, 64), BAD)):
        refused(st, call, cache(), batch(), rope=rope)


def test_rows():
    for kw, st in ((dict(k=0), NULL), (dict(v=0), NULL), (dict(ks=127), BAD), (dict(vs=0), BAD), (dict(k=(1 << 20) + 2), BAD),
                   (dict(dtype=G.Q8_0), DTYPE), (dict(dtype=77), DTYPE), (dict(ks=1 << 50), BAD)):
        refused(st, append, cache(), batch(), **kw)
    for kw, st in ((dict(dtype=G.Q4_0), DTYPE), (dict(k=(1 << 20) + 1), BAD), (dict(v=(1 << 20) + 2), BAD)):
        refused(st, read, cache(), batch(), **kw)
    for kw, st in ((dict(q=0), NULL), (dict(out=0), NULL), (dict(qs=255), BAD), (dict(os=255), BAD), (dict(n_q=3), BAD),
                   (dict(n_q=0), BAD), (dict(n_q=1 << 40), BAD), (dict(scale=-1.0), BAD), (dict(scale=float("nan")), BAD),
                   (dict(scale=float("inf")), BAD), (dict(qt=G.Q8_0), DTYPE), (dict(ot=G.Q8_0), DTYPE),
                   (dict(q=(1 << 20) + 2), BAD), (dict(out=(1 << 20) + 1), BAD)):
        refused(st, attend, cache(), batch(), **kw)
    refused(BAD, attend, cache(), batch(max_pages=0))
    big = dict(n_kv_heads=65536)
    refused(BAD, append, cache(**big), batch(n_rows=1 << 27), ks=1 << 22, vs=1 << 22)
    refused(BAD, read, cache(**big), batch(n_rows=1 << 27))
    refused(BAD, attend, cache(**big), batch(n_rows=1 << 27), n_q=65536, qs=1 << 22, os=1 << 22)


def test_empty_calls_do_nothing():
    for b in (batch(n_rows=0), batch(n_seqs=0), batch(n_rows=0, row_offsets=0, seq_lens=0, pages=0)):
        append(cache(), b, k=0, v=0)
        read(cache(), b)
        attend(cache(), b, q=0, out=0)
    read(cache(), batch(), k=0, v=0)
    append(cache(), batch(max_pages=0, pages=0))
    rce_amd.sample_dev(FakeContext(), 0, G.F32, 0, 10, 10, 0, 0)


def test_sampling():
    def call(lg=1 << 20, dtype=G.F32, n=2, v=10, stride=10, u=2 << 20, ids=3 << 20, **kw):
        rce_amd.sample_dev(FakeContext(), lg, dtype, n, v, stride, u, ids, **kw)
    for kw, st in ((dict(lg=0), NULL), (dict(u=0), NULL), (dict(ids=0), NULL), (dict(v=0), BAD), (dict(v=(1 << 24) + 1), BAD),
                   (dict(stride=9), BAD), (dict(n=(1 << 20) + 1), BAD), (dict(dtype=G.Q8_0), DTYPE), (dict(lg=(1 << 20) + 2), BAD),
                   (dict(u=(1 << 20) + 2), BAD), (dict(ids=(1 << 20) + 1), BAD), (dict(probs_dev=(1 << 20) + 1), BAD),
                   (dict(top_p_dev=(1 << 20) + 2), BAD), (dict(top_k_dev=(1 << 20) + 2), BAD)):
        refused(st, call, **kw)
    L = _lib.lib()
    assert L.rce_qmm_sample_dev(None, 1 << 20, 0, 1, 10, 10, None, 1 << 20, None, None) == NULL


def test_null_contexts():
    L = _lib.lib()
    assert L.rce_qmm_kv_append_dev(None, None, None, None, 0, None, 0, 0, None, None) == NULL
    assert L.rce_qmm_kv_read_dev(None, None, None, None, None, 0, None) == NULL
    assert L.rce_qmm_kv_attention_dev(None, None, None, None, 0, 0, 0, None, 0.0, 0, None, 0, 0, None) == NULL
    assert L.rce_qmm_kv_sizes(None, None, None) == NULL


def test_sizes():
    assert cache().sizes() == (4 * 2 * 32 * 64, 4 * 2 * 2)
    assert cache(n_pages=1 << 20, page_tokens=64, n_kv_heads=8, d_head=128).sizes() == (1 << 36, 1 << 25)
    refused(BAD, cache(page_tokens=24).sizes)


def test_rope_table():
    t = rce_amd.Rope.table(10000.0, 8, 5)
    assert t.shape == (5, 4, 2) and t.dtype == np.float32
    theta = np.arange(5)[:, None] * 10000.0 ** (-np.arange(4) / 4)
    # the angle in f32 carries the errors of logf, expf and three products
    assert np.abs(t[..., 0] - np.cos(theta)).max() < 5 * 2.0 ** -21 and np.abs(t[..., 1] - np.sin(theta)).max() < 5 * 2.0 ** -21
    assert rce_amd.Rope.table(10000.0, 0, 5).shape == (5, 0, 2)
    for a in ((10000.0, 7, 5), (0.0, 8, 5), (float("nan"), 8, 5), (1e4, 65538, 1)):
        refused(BAD, rce_amd.Rope.table, *a)


def test_oracle_attention_is_the_plain_sum():
    """The oracle's own check: one key gives its value, a window of one the newest."""
    rng = np.random.default_rng(0)
    b, n = kc.make_batch(rng, [1, 40], [1, 5], 16)
    pool = kc.Pool(n, 16, 2, 64, rng)
    q = rng.standard_normal((6, 4, 64)).astype(np.float32)
    out, _ = kc.attention(pool, b, q, None, 0.125, 1, True)
    for r, s, pos in b.rows():
        v = pool.values("v", b.page_of(s, pos, n), pos)
        assert np.allclose(out[r], np.repeat(v, 2, 0), rtol=1e-12)
