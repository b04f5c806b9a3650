"""The paged 8-bit KV cache restated in numpy: the append's rule bit for bit
in binary32, attention in 64 bits with the error its arithmetic allows, and
sampling in 64 bits.  Test infrastructure only."""
import math

import numpy as np

import rce_amd
from rce_amd import GgufDtype as G

F32, F64 = np.float32, np.float64
BLOCK = 16


def to_bits(x, dtype):
    """f32 values as the bytes of `dtype` (round to nearest even)."""
    x = np.ascontiguousarray(x, F32)
    if dtype == G.F32:
        return x
    if dtype == G.F16:
        return x.astype(np.float16)
    u = x.view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def widen(b, dtype):
    if dtype == G.F32:
        return b
    if dtype == G.F16:
        return b.astype(F32)
    return (b.astype(np.uint32) << 16).view(F32)


def np_type(dtype):
    return {G.F32: np.float32, G.F16: np.float16, G.BF16: np.uint16}[dtype]


class Pool:
    """Host copy of a pool, in the header's layout."""

    def __init__(self, n_pages, page, heads, d, rng=None):
        self.n_pages, self.page, self.heads, self.d, self.b = n_pages, page, heads, d, page // BLOCK
        rng = rng or np.random.default_rng(0)
        s = (n_pages, heads, self.b)
        self.k = np.clip(np.rint(rng.standard_normal(s + (BLOCK, d)) * 40), -127, 127).astype(np.int8)
        self.v = np.clip(np.rint(rng.standard_normal(s + (d, BLOCK)) * 40), -127, 127).astype(np.int8)
        self.k_scale = (rng.uniform(0.5, 1.5, s) * 0.03).astype(F32)
        self.v_scale = (rng.uniform(0.3, 1.7, s) * 0.03).astype(F32)

    def copy(self):
        p = Pool.__new__(Pool)
        p.__dict__.update(self.__dict__)
        for n in ("k", "v", "k_scale", "v_scale"):
            setattr(p, n, getattr(self, n).copy())
        return p

    def values(self, name, page, pos):
        """[heads, d] values of one position, in f64."""
        b, i = pos % self.page // BLOCK, pos % BLOCK
        c = self.k[page, :, b, i] if name == "k" else self.v[page, :, b, :, i]
        s = getattr(self, name + "_scale")[page, :, b]
        with np.errstate(invalid="ignore"):
            return c.astype(F64) * s.astype(F64)[:, None]


class Batch:
    def __init__(self, lens, news, pages, page, n_rows=None):
        self.lens, self.news = list(lens), list(news)
        self.offsets = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        self.pages = np.asarray(pages, np.int32).reshape(len(lens), -1)
        self.page = page
        self.n_rows = int(self.offsets[-1]) if n_rows is None else n_rows

    @property
    def cap(self):
        return self.pages.shape[1] * self.page

    def rows(self):
        """(row, sequence, position) of every row that belongs to a sequence."""
        for s, (n, m) in enumerate(zip(self.lens, self.news)):
            for i in range(m):
                yield int(self.offsets[s]) + i, s, max(n, 0) - m + i

    def page_of(self, s, pos, n_pages):
        if pos < 0 or pos >= self.cap:
            return None
        p = int(self.pages[s, pos // self.page])
        return p if 0 <= p < n_pages else None


def make_batch(rng, lens, news, page, spare=2, n_rows=None):
    """Random distinct pages for sequences of these lengths."""
    counts = [max(1, -(-n // page)) for n in lens]
    n_pages = sum(counts) + spare
    ids = rng.permutation(n_pages)
    pages = np.full((len(lens), max(counts)), -1, np.int32)
    at = 0
    for s, c in enumerate(counts):
        pages[s, :c] = ids[at:at + c]
        at += c
    return Batch(lens, news, pages, page, n_rows), n_pages


def rope_cs(dim, n_pos, base=10000.0):
    return rce_amd.Rope.table(base, dim, n_pos) if dim else None


def rotate(x, cs, pos):
    """x [heads, d] f32, one rounding per operation."""
    if cs is None:
        return x
    h = cs.shape[1]
    c, s = cs[pos, :, 0], cs[pos, :, 1]
    a, b = x[:, :h], x[:, h:2 * h]
    return np.concatenate([a * c - b * s, a * s + b * c, x[:, 2 * h:]], 1)


def append(pool, batch, k, v, cs):
    """The header's append rule on a host pool; k, v [rows, heads, d] f32."""
    todo = {}
    for r, s, pos in batch.rows():
        page = batch.page_of(s, pos, pool.n_pages)
        if page is not None:
            todo.setdefault((page, pos % pool.page // BLOCK), []).append((pos % BLOCK, r, pos))
    with np.errstate(all="ignore"):
        for (page, b), rows in todo.items():
            o = min(i for i, _, _ in rows)
            for name, src in (("k", k), ("v", v)):
                sc = getattr(pool, name + "_scale")
                codes = pool.k[page, :, b] if name == "k" else pool.v[page, :, b].transpose(0, 2, 1)  # views
                x = np.stack([rotate(src[r], cs, p) if name == "k" else src[r] for _, r, p in rows], 1)
                for h in range(pool.heads):
                    old = sc[page, h, b] if o else F32(0)
                    d = np.abs(x[h]).max() / F32(127)  # NaN passes through max
                    if d < F32(2.0 ** -126):
                        d = F32(0)
                    new = F32(np.nan) if np.isnan(d) or np.isnan(old) else max(old, d)
                    some = new > 0 and np.isfinite(new)
                    inv = F32(1) / new if some else F32(0)
                    ratio = old / new if some else F32(0)
                    if o and (not some or new != old):
                        codes[h, :o] = np.rint(codes[h, :o].astype(F32) * ratio).astype(np.int8)
                    q = np.rint(x[h] * inv)
                    q = np.clip(np.where(np.isnan(q), 0, q), -127, 127).astype(np.int8)
                    for j, (i, _, _) in enumerate(rows):
                        codes[h, i] = q[j]
                    sc[page, h, b] = new


def attention(pool, batch, q, cs, scale, window, f32_out):
    """(out, bound) [rows, n_q, d] in f64 for q [rows, n_q, d] f32 values.

    The bound: a score's error is at most scale * sum|k| * max|q| / (2 QMAX)
    (whole-number q), 2^-21 |s| for the roundings of its products and of its
    base-2 form, and as much again through the subtracted maximum; a weight's
    relative error is twice that, 2^-22 from the exponential, and its binary16
    rounding (2^-12 here, one term; 2^-21, two terms) or 2^-38 of the row's largest
    weight times the ratio of the tile's scales; the sums of n terms
    add n 2^-23.  All against sum p |v|."""
    n_q, d = q.shape[1], q.shape[2]
    per = n_q // pool.heads
    qmax = 127.0 * (65536 if f32_out else 256)
    out = np.zeros(q.shape, F64)
    bound = np.zeros(q.shape, F64)
    for r, s, pos in batch.rows():
        if pos < 0 or pos >= batch.cap:
            continue
        seen = [(p, batch.page_of(s, p, pool.n_pages)) for p in range(max(0, pos - window + 1) if window else 0, pos + 1)]
        seen = [(p, g) for p, g in seen if g is not None]
        if not seen:
            continue
        P, Gs = np.array([p for p, _ in seen]), np.array([g for _, g in seen])
        b, i = P % pool.page // BLOCK, P % BLOCK
        with np.errstate(all="ignore"):
            K = pool.k[Gs, :, b, i].astype(F64) * pool.k_scale[Gs, :, b].astype(F64)[..., None]
            V = pool.v[Gs, :, b, :, i].astype(F64) * pool.v_scale[Gs, :, b].astype(F64)[..., None]
            x = rotate(q[r], cs, pos).astype(F64)
            for h in range(n_q):
                k, v = K[:, h // per], V[:, h // per]
                sc = k @ x[h] * scale
                w = np.exp(sc - sc.max())
                w /= w.sum()
                out[r, h] = w @ v
                ds = scale * np.abs(k).sum(1).max() * np.abs(x[h]).max() / (2 * qmax) + 2 * np.abs(sc).max() * 2.0 ** -21
                rel = 4 * ds + 2.0 ** -22 + (2.0 ** -21 if f32_out else 2.0 ** -12) + len(P) * 2.0 ** -23
                tail = 2.0 ** -38 * len(P) * np.abs(v).max() * 4
                bound[r, h] = rel * (w @ np.abs(v)) * 2 + tail
    return out, bound


def out_eps(dtype):
    return {G.F32: 2.0 ** -24, G.F16: 2.0 ** -11, G.BF16: 2.0 ** -8}[dtype]


def sample(logits, u, temp=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(id, probability) of one row, logits f32 values."""
    x = np.where(np.isnan(logits), -np.inf, logits.astype(F64)) + 0.0
    n = len(x)
    best = int(np.argmax(x))
    if x[best] == -np.inf:
        return -1, 0.0
    if not temp > 0:
        return best, 1.0
    with np.errstate(all="ignore"):
        w = np.exp((x - x[best]) / F64(temp))
    w = np.where(x == x[best], 1.0, np.where(x == -np.inf, 0.0, np.nan_to_num(w)))
    order = np.argsort(-x, kind="stable")
    if 0 < top_k < n:
        order = order[:top_k]
    ws = w[order]
    if top_p < 1:
        before = np.concatenate([[0.0], np.cumsum(ws)[:-1]])
        keep = before < F64(top_p) * math.fsum(ws)
        keep[0] = True
        order = order[keep]
    if min_p > 0:
        keep = w[order] >= F64(min_p)
        keep[0] = True
        order = order[keep]
    order = np.sort(order)
    c = np.cumsum(w[order])
    at = order[min(len(order) - 1, int(np.searchsorted(c, F64(u) * c[-1], side="right")))]
    return int(at), w[at] / c[-1]


# ---- the device side ------------------------------------------------------------

class Device:
    """A pool and a batch on the device."""

    def __init__(self, ctx, pool, batch, cs=None):
        self.ctx, self.pool, self.batch = ctx, pool, batch
        up = lambda a: rce_amd.DeviceBuffer.from_numpy(ctx, a)  # noqa: E731
        self.bufs = [up(pool.k), up(pool.v), up(pool.k_scale), up(pool.v_scale), up(batch.offsets),
                     up(np.asarray(batch.lens, np.int32)), up(batch.pages)]
        k, v, ks, vs, off, ln, pg = (b.ptr for b in self.bufs)
        self.cache = rce_amd.KvCache(pool.n_pages, pool.page, pool.heads, pool.d, k=k, v=v, k_scale=ks, v_scale=vs)
        self.at = (off, ln, pg)
        self.rows(batch.n_rows)
        self.rope = None
        if cs is not None:
            self.bufs.append(up(cs))
            self.rope = rce_amd.Rope(self.bufs[-1].ptr, cs.shape[1] * 2, cs.shape[0])

    def rows(self, n):
        """The batch with n rows."""
        self.b = rce_amd.KvBatch(*self.at, len(self.batch.lens), n, self.batch.pages.shape[1])

    def download(self):
        p = self.pool.copy()
        for n, b in zip(("k", "v", "k_scale", "v_scale"), self.bufs):
            a = getattr(p, n)
            setattr(p, n, b.download(a.dtype, a.size).reshape(a.shape))
        return p

    def free(self):
        for b in self.bufs:
            b.free()
