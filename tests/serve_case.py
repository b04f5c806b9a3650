"""The serving step's routing, head norms with rotation, page tables and
attention with sinks restated on the host: choices as plain lists, numbers in
64 bits with the error that the kernels' arithmetic allows.  Test
infrastructure only."""
import numpy as np

from kv_case import BLOCK, F32, F64, rotate

U = 2.0 ** -24  # a rounding to binary32


def half_step(dtype):
    """Relative error of one rounding to a type, and of one among its subnormal numbers."""
    from rce_amd import GgufDtype as G
    return {G.F32: (U, 2.0 ** -150), G.F16: (2.0 ** -11, 2.0 ** -25), G.BF16: (2.0 ** -8, 2.0 ** -134)}[dtype]


# ---- routing ----------------------------------------------------------------------

def route(logits, top_k, sigmoid=False, bias=None, groups=1, kept=1, group_top=1, normalize=True, scale=1.0):
    """(ids, weights) of rows of f32 logits, one after the other."""
    n, e = logits.shape
    ids, weights = np.zeros((n, top_k), np.int32), np.zeros((n, top_k), F64)
    size = e // groups
    with np.errstate(all="ignore"):
        for t in range(n):
            x = np.where(np.isnan(logits[t]), -np.inf, logits[t].astype(F64)) + 0.0
            if sigmoid:
                score = 1 / (1 + np.exp(-x))
            else:
                w = np.where(x == x.max(), 1.0, np.exp(x - x.max()))
                score = w / w.sum()
            value = score if bias is None else score + bias.astype(F64)
            dead = (x == -np.inf) | np.isnan(value) | (value == -np.inf)
            key = np.where(dead, -np.inf, x if bias is None else value)
            value = np.where(dead, -np.inf, x if bias is None and group_top == 1 else value)
            chosen = list(range(groups))
            if kept < groups:
                def worth(g):
                    best = sorted((v for v in value[g * size:(g + 1) * size] if v > -np.inf), reverse=True)[:group_top]
                    return sum(best) if best else -np.inf
                worths = [worth(g) for g in range(groups)]
                chosen = sorted(range(groups), key=lambda g: (-worths[g], g))[:kept]
            order = sorted((i for i in range(e) if i // size in chosen), key=lambda i: (-key[i], i))[:top_k]
            w = np.array([0.0 if key[i] == -np.inf else score[i] for i in order])
            if normalize:
                w = w / w.sum() if w.sum() > 0 else w * 0
            ids[t], weights[t] = order, w * F64(F32(scale))
    return ids, weights


# ---- norms and rotation -----------------------------------------------------------

def norm_rope(x, weight, eps, cs, pos, interleaved):
    """(out, bound) of heads x [heads, d] (f32 values) at a position.

    The sum of squares' 24 roundings, its division's and eps's halve in the
    root; with the root's, the reciprocal's and two products' a value is
    within 18 U, and a pair's two products and their sum add 2 U: 24 U of the
    pair's |a c| + |b s| holds them."""
    y = x.astype(F64)
    if eps is not None:
        y = y / np.sqrt((y * y).mean(1, keepdims=True) + F64(F32(eps))) * (1.0 if weight is None else weight.astype(F64))
    out, size = y.copy(), np.abs(y)
    if cs is not None:
        h = cs.shape[1]
        c, s = cs[pos, :, 0].astype(F64), cs[pos, :, 1].astype(F64)
        a, b = (slice(0, 2 * h, 2), slice(1, 2 * h, 2)) if interleaved else (slice(0, h), slice(h, 2 * h))
        out[:, a], out[:, b] = y[:, a] * c - y[:, b] * s, y[:, a] * s + y[:, b] * c
        size[:, a], size[:, b] = (np.abs(y[:, a] * c) + np.abs(y[:, b] * s), np.abs(y[:, a] * s) + np.abs(y[:, b] * c))
    return out, 24 * U * size


# ---- page tables ------------------------------------------------------------------

class Tables:
    """Tables and counts; copies, what was copied: (from, to, blocks)."""

    def __init__(self, pages, refs, page):
        self.pages = [[int(p) for p in row] for row in pages]
        self.refs = [int(r) for r in refs]
        self.page = page
        self.copies = []

    def named(self, p):
        return 0 <= p < len(self.refs)

    def fork(self, to, parents):
        """Rows of `to` (tables with the same counts) from this one's."""
        for i, parent in enumerate(parents):
            if not 0 <= parent < len(self.pages):
                continue
            for j in range(len(to[i])):
                p = self.pages[parent][j] if j < len(self.pages[parent]) else -1
                if self.named(p):
                    self.refs[p] += 1
                to[i][j] = p if self.named(p) else -1

    def release(self, lo=None, hi=None):
        for s, row in enumerate(self.pages):
            for j, p in enumerate(row):
                if (lo is None or j * self.page >= lo[s]) and (hi is None or (j + 1) * self.page <= hi[s]):
                    if self.named(p):
                        self.refs[p] -= 1
                    row[j] = -1

    def reserve(self, offsets, lens):
        """Counts of missing pages; offsets, lens as in a batch."""
        start = list(self.refs)
        items = []
        for s, row in enumerate(self.pages):
            new, n = offsets[s + 1] - offsets[s], max(lens[s], 0)
            lo, hi = max(0, n - new), min(n, len(row) * self.page)
            items += [(s, j, lo) for j in range(lo // self.page, (hi - 1) // self.page + 1)] if hi > lo else []
        asks = {}
        for s, j, _ in items:
            p = self.pages[s][j]
            if self.named(p) and start[p] > 1:
                asks.setdefault(p, []).append((s, j))
        keeps = {a[0] for p, a in asks.items() if len(a) == start[p]}
        asking = {x for a in asks.values() for x in a} - keeps
        free = [p for p, r in enumerate(start) if r == 0]
        missing = [0] * len(self.pages)
        for s, j, lo in items:
            p = self.pages[s][j]
            shared = (s, j) in asking
            if self.named(p) and not shared:
                continue
            if shared:
                self.refs[p] -= 1
            to = free.pop(0) if free else -1
            if to < 0:
                missing[s] += 1
            else:
                self.refs[to] = 1
                if shared and j == lo // self.page and lo % self.page:
                    self.copies.append((p, to, -(-(lo % self.page) // BLOCK)))
            self.pages[s][j] = to
        return missing

    def compact(self):
        """(new ids, pages used)."""
        used = [p for p, r in enumerate(self.refs) if r]
        n = len(used)
        holes = [p for p in range(n) if not self.refs[p]]
        to = dict(zip([p for p in used if p >= n], holes))
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
            self.copies.append((a, b, self.page // BLOCK))
        ids = [-1] * len(self.refs)
        for p in used:
            ids[p] = to.get(p, p)
        self.pages = [[ids[p] if self.named(p) else p for p in row] for row in self.pages]
        return ids, n

    def apply(self, pool):
        """The copies on a host pool, all from what was there before."""
        was = pool.copy()
        for a, b, blocks in self.copies:
            for n in ("k", "v", "k_scale", "v_scale"):
                getattr(pool, n)[b, :, :blocks] = getattr(was, n)[a, :, :blocks]
        self.copies = []


# ---- attention with sinks -----------------------------------------------------------

def attention(pool, batch, q, cs, scale, window, sinks, f32_out, rows=None):
    """{row: (out, bound)} [n_q, d] for q [rows, n_q, d] f32 values: the
    sum over a window and first positions, its bound as kv_case.attention
    derives it (a score's error scale * sum|k| * max|q| / (2 QMAX) and 2^-21 of
    it twice, the weights' and sums' roundings, all against sum p |v|)."""
    n_q, d = q.shape[1], q.shape[2]
    per = n_q // pool.heads
    qmax = 127.0 * (65536 if f32_out else 256)
    got = {}
    for r, s, pos in batch.rows():
        if rows is not None and r not in rows:
            continue
        got[r] = np.zeros((n_q, d)), np.zeros((n_q, d))
        if pos < 0 or pos >= batch.cap:
            continue
        j = np.arange(pos + 1)
        if window:
            j = j[(j > pos - window) | (j < sinks)]
        g = batch.pages[s, j // pool.page]
        ok = (g >= 0) & (g < pool.n_pages)
        j, g = j[ok], g[ok]
        if not len(j):
            continue
        b, i = j % pool.page // BLOCK, j % BLOCK
        with np.errstate(all="ignore"):
            K = pool.k[g, :, b, i].astype(F64) * pool.k_scale[g, :, b].astype(F64)[..., None]
            V = pool.v[g, :, b, :, i].astype(F64) * pool.v_scale[g, :, b].astype(F64)[..., None]
            x = rotate(q[r], cs, pos).astype(F64)
            for h in range(n_q):
                k, v = K[:, h // per], V[:, h // per]
                sc = k @ x[h] * scale
                w = np.exp(sc - sc.max())
                w /= w.sum()
                ds = scale * np.abs(k).sum(1).max() * np.abs(x[h]).max() / (2 * qmax) + 2 * np.abs(sc).max() * 2.0 ** -21
                rel = 4 * ds + 2.0 ** -22 + (2.0 ** -21 if f32_out else 2.0 ** -12) + len(j) * 2.0 ** -23
                got[r][0][h] = w @ v
                got[r][1][h] = rel * (w @ np.abs(v)) * 2 + 2.0 ** -38 * len(j) * np.abs(v).max() * 4
    return got
