"""The page calls against plain lists (serve_case.Tables): tables, counts and
every byte of the pool after forks, reservations with copies, releases and
compactions; pools that run out, large batches, recorded calls."""
import numpy as np
import pytest

import kv_case as kc
import rce_amd
import serve_case as sc
from bench import Hip
from kv_case import F32

pytestmark = pytest.mark.gpu

PARTS = ("k", "v", "k_scale", "v_scale")


class Pages:
    """A pool, tables and counts on the device and as lists."""

    def __init__(self, ctx, rng, n_pages, page, heads, d, n_seqs, max_pages):
        self.ctx, self.shape = ctx, (n_seqs, max_pages)
        self.pool = kc.Pool(n_pages, page, heads, d, rng)
        self.host = sc.Tables(np.full((n_seqs, max_pages), -1), np.zeros(n_pages), page)
        up = lambda a: rce_amd.DeviceBuffer.from_numpy(ctx, a)  # noqa: E731
        self.bufs = [up(getattr(self.pool, n)) for n in PARTS]
        k, v, ks, vs = (b.ptr for b in self.bufs)
        self.cache = rce_amd.KvCache(n_pages, page, heads, d, k=k, v=v, k_scale=ks, v_scale=vs)
        self.pages, self.refs = up(np.full(self.shape, -1, np.int32)), up(np.zeros(n_pages, np.int32))
        self.table = rce_amd.KvTable(self.pages.ptr, *self.shape)
        self.missing = up(np.full(n_seqs, 99, np.int32))
        self.extra = [self.pages, self.refs, self.missing]

    def put(self, rows, refs=None):
        """Tables, and the counts that they make."""
        rows = np.asarray(rows, np.int32)
        if refs is None:
            refs = np.bincount(rows[(rows >= 0) & (rows < len(self.host.refs))], minlength=len(self.host.refs))
        self.host = sc.Tables(rows, refs, self.host.page)
        self.pages.upload(rows)
        self.refs.upload(np.asarray(refs, np.int32))

    def arr(self, a):
        b = rce_amd.DeviceBuffer.from_numpy(self.ctx, np.asarray(a, np.int32))
        self.extra.append(b)
        return b.ptr

    def batch(self, news, lens, pages=None):
        off = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        n_seqs, max_pages = self.shape
        return off, rce_amd.KvBatch(self.arr(off), self.arr(lens), self.pages.ptr if pages is None else pages, n_seqs, int(off[-1]), max_pages)

    def reserve(self, news, lens):
        off, b = self.batch(news, lens)
        rce_amd.kv_reserve_dev(self.ctx, self.cache, b, self.refs.ptr, self.missing.ptr)
        want = self.host.reserve(off.tolist(), list(lens))
        self.host.apply(self.pool)
        self.check()
        assert np.array_equal(self.missing.download(np.int32, self.shape[0]), want)
        return want

    def release(self, lo=None, hi=None):
        rce_amd.kv_release_dev(self.ctx, self.cache, self.table, self.refs.ptr, None if lo is None else self.arr(lo), None if hi is None else self.arr(hi))
        self.host.release(lo, hi)
        self.check()

    def check(self):
        self.ctx.synchronize()
        assert np.array_equal(self.pages.download(np.int32, np.prod(self.shape)).reshape(self.shape), np.array(self.host.pages).reshape(self.shape))
        assert np.array_equal(self.refs.download(np.int32, len(self.host.refs)), self.host.refs)
        for n, b in zip(PARTS, self.bufs):
            a = getattr(self.pool, n)
            assert np.array_equal(b.download(a.dtype, a.size).reshape(a.shape).view(np.uint8), a.view(np.uint8)), n

    def free(self):
        for b in self.bufs + self.extra:
            b.free()


@pytest.mark.parametrize("page,heads,d", [(16, 1, 64), (16, 8, 128), (32, 2, 192), (64, 3, 64), (256, 1, 256), (4096, 1, 64)])
def test_sequences_come_and_go(ctx, page, heads, d):
    """Prompts, tokens across page borders, forks, rejected drafts, ends; the pool never runs out."""
    print(f"pages page={page} heads={heads} d={d}", flush=True)
    rng = np.random.default_rng(page + heads)
    n, max_pages = 6, 4
    p = Pages(ctx, rng, n * max_pages + 3, page, heads, d, n, max_pages)
    lens = np.zeros(n, int)
    for step in range(14):
        news = np.where(lens == 0, rng.integers(0, 2 * page, n), rng.integers(0, page // 2 + 2, n))
        news = np.minimum(news, max_pages * page - lens)
        lens += news
        p.reserve(news, lens)
        if step % 3 == 1:  # two sequences end, two others go on twice
            a = rng.permutation(n)
            lo = np.where(np.isin(np.arange(n), a[:2]), 0, 1 << 30)
            p.release(lo=lo)
            parents = np.full(n, -1)
            parents[a[:2]] = a[2:4]
            rce_amd.kv_fork_dev(ctx, p.cache, p.table, p.table, p.arr(parents), p.refs.ptr)
            p.host.fork(p.host.pages, parents.tolist())
            p.check()
            lens[a[:2]] = lens[a[2:4]]
        if step % 4 == 2:  # drafts taken back
            lens = np.maximum(lens - rng.integers(0, page, n), 0)
            p.release(lo=lens)
        if step % 5 == 4:
            ids, used = rce_amd.DeviceBuffer(ctx, 4 * p.pool.n_pages), rce_amd.DeviceBuffer(ctx, 4)
            rce_amd.kv_compact_dev(ctx, p.cache, p.table, p.refs.ptr, ids.ptr, used.ptr)
            want, n_used = p.host.compact()
            p.host.apply(p.pool)
            p.check()
            assert np.array_equal(ids.download(np.int32, p.pool.n_pages), want) and used.download(np.int32, 1)[0] == n_used
            ids.free(); used.free()
    p.release()
    assert not any(p.host.refs)
    p.free()


def test_who_keeps_a_shared_page(ctx):
    """All three holders write: the first keeps it; two of three write: both leave; one that does not write holds it."""
    p = Pages(ctx, np.random.default_rng(1), 12, 16, 2, 64, 4, 2)
    p.put([[7, -1], [7, -1], [7, -1], [3, -1]])
    assert p.reserve([1, 1, 1, 1], [5, 9, 16, 4]) == [0, 0, 0, 0]
    assert p.host.pages[0][0] == 7 and p.host.refs[7] == 1
    p.put([[7, -1], [7, -1], [7, -1], [3, -1]])
    p.reserve([1, 0, 1, 0], [5, 9, 16, 4])
    assert p.host.refs[7] == 1 and p.host.pages[1][0] == 7
    # shared by tables that this call does not see
    p.put([[7, 8], [7, -1], [-1, -1], [-1, -1]], refs=[0] * 7 + [5, 2] + [0] * 3)
    p.reserve([17, 1, 0, 0], [32, 3, 0, 0])
    # one sequence names a page twice
    p.put([[7, 7], [-1, -1], [-1, -1], [-1, -1]])
    p.reserve([20, 0, 0, 0], [30, 0, 0, 0])
    assert p.host.pages[0][0] == 7
    p.free()


@pytest.mark.parametrize("lo", [0, 1, 15, 16, 17, 40, 63])
def test_what_is_copied(ctx, lo):
    """The blocks that start in front of the first row, of every head and part, and no others."""
    p = Pages(ctx, np.random.default_rng(lo), 8, 64, 3, 64, 2, 2)
    p.put([[5, -1], [5, -1]])
    p.reserve([1, 1], [lo + 1, lo + 1])
    p.put([[5, 2], [5, 2]])
    p.reserve([64, 64], [lo + 64, lo + 64])
    p.free()


@pytest.mark.parametrize("heads,d", [(1, 64), (8, 256)])
def test_what_is_copied_in_front_of_many_pages(ctx, heads, d):
    """A shared page at a long chunk's beginning: more items than a round, copied by the plan or behind it."""
    p = Pages(ctx, np.random.default_rng(heads), 1300, 16, heads, d, 2, 1200)
    rows = np.full((2, 1200), -1)
    rows[0, :3], rows[1, :3] = (5, 700, 9), (5, 700, 11)
    p.put(rows)
    p.reserve([1100 * 16, 0], [40 + 1100 * 16, 40])
    p.put(rows)
    p.reserve([1100 * 16, 20], [23 + 1100 * 16, 43])
    p.free()


def test_a_pool_that_runs_out(ctx):
    """Pages go to the first that ask; what misses is counted, its entries name none, a shared page is lost there."""
    p = Pages(ctx, np.random.default_rng(2), 5, 16, 1, 64, 4, 3)
    p.put([[0, -1, -1], [0, -1, -1], [-1, -1, -1], [4, -1, -1]])
    assert p.reserve([3, 20, 40, 1], [5, 30, 40, 17]) == [0, 0, 2, 1]
    p.put([[0, 1, 2], [3, 4, 0], [-1, -1, -1], [-1, -1, -1]])
    assert p.reserve([0, 1, 16, 1], [48, 40, 16, 1]) == [0, 1, 1, 1]
    assert p.host.pages[1][2] == -1 and p.host.refs[0] == 1
    p.free()


def test_entries_that_name_no_page(ctx):
    """Ids outside the pool anywhere in a table, rows without positions, rows behind the table."""
    p = Pages(ctx, np.random.default_rng(3), 9, 16, 1, 64, 4, 2)
    p.put([[1 << 30, -5], [9, 3], [-(1 << 31), (1 << 31) - 1], [4, 4]])
    p.reserve([3, 20, 0, 0], [3, 30, 0, 0])
    p.put([[1 << 30, -5], [9, 3], [-(1 << 31), (1 << 31) - 1], [4, 8]])
    p.reserve([5, 2, 1, 40], [3, 0, -7, 60])  # rows at -2 .. 2; none; none; 20 .. 59 of 32
    p.put([[1 << 30, 2], [9, 3], [-(1 << 31), (1 << 31) - 1], [4, 8]])
    p.release(lo=[0, 16, -5, 1], hi=[33, 31, 16, 32])
    parents = [3, 7, -1, 0]
    other = rce_amd.DeviceBuffer.from_numpy(ctx, np.full((4, 3), 77, np.int32))
    rce_amd.kv_fork_dev(ctx, p.cache, p.table, rce_amd.KvTable(other.ptr, 4, 3), p.arr(parents), p.refs.ptr)
    to = [[77] * 3 for _ in range(4)]
    p.host.fork(to, parents)
    p.check()
    assert np.array_equal(other.download(np.int32, 12).reshape(4, 3), to)
    one = rce_amd.DeviceBuffer.from_numpy(ctx, np.full((4, 1), 77, np.int32))
    rce_amd.kv_fork_dev(ctx, p.cache, p.table, rce_amd.KvTable(one.ptr, 4, 1), p.arr(parents), p.refs.ptr)
    to = [[77] for _ in range(4)]
    p.host.fork(to, parents)
    p.check()
    assert np.array_equal(one.download(np.int32, 4).reshape(4, 1), to)
    other.free(); one.free()
    p.free()


def test_no_rows(ctx):
    """Counts of missing pages become 0; nothing else moves."""
    p = Pages(ctx, np.random.default_rng(4), 4, 16, 1, 64, 3, 2)
    p.put([[0, -1], [0, 1], [2, -1]])
    assert p.reserve([0, 0, 0], [5, 20, 3]) == [0, 0, 0]
    p.missing.upload(np.full(3, 5, np.int32))
    rce_amd.kv_reserve_dev(ctx, p.cache, rce_amd.KvBatch(0, 0, 0, 3, 0, 2), p.refs.ptr, p.missing.ptr)
    p.check()
    assert not p.missing.download(np.int32, 3).any()
    p.free()


def test_without_counts_of_missing(ctx):
    p = Pages(ctx, np.random.default_rng(5), 2, 16, 1, 64, 2, 2)
    off, b = p.batch([20, 20], [20, 20])
    rce_amd.kv_reserve_dev(ctx, p.cache, b, p.refs.ptr)
    p.host.reserve(off.tolist(), [20, 20])
    p.check()
    p.free()


@pytest.mark.parametrize("n_seqs,max_pages,n_pages", [(1, 3000, 5000), (1023, 3, 4100), (1024, 3, 9000), (1025, 3, 4096), (3000, 2, 6500), (2500, 5, 30000)])
def test_large_batches(ctx, n_seqs, max_pages, n_pages):
    """More sequences, more pages and more free pages than one round of the plan takes; shared ones far apart."""
    print(f"pages n_seqs={n_seqs} max_pages={max_pages} n_pages={n_pages}", flush=True)
    rng = np.random.default_rng(n_seqs)
    p = Pages(ctx, rng, n_pages, 16, 1, 64, n_seqs, max_pages)
    for _ in range(2):
        rows = np.full((n_seqs, max_pages), -1)
        held = rng.integers(0, max_pages + 1, n_seqs)
        ids = rng.permutation(n_pages)[: n_pages // 3]
        for s, h in enumerate(held):
            rows[s, :h] = rng.choice(ids, h)  # shared at random
        p.put(rows)
        lens = np.minimum(held * 16 + rng.integers(0, 20, n_seqs), max_pages * 16)
        news = np.minimum(rng.integers(0, 40, n_seqs), lens)
        if n_seqs == 1:
            lens, news = np.array([48000]), np.array([47000])
        p.reserve(news, lens)
    p.free()


@pytest.mark.parametrize("n_pages,share", [(1, 0.0), (1, 1.0), (7, 0.5), (4096, 0.5), (4097, 0.9), (9001, 0.1), (20000, 0.97)])
def test_compact(ctx, n_pages, share):
    rng = np.random.default_rng(n_pages)
    p = Pages(ctx, rng, n_pages, 16, 1, 64, 5, 40)
    refs = np.where(rng.random(n_pages) < share, rng.integers(1, 5, n_pages), 0)  # other tables name most of them
    rows = rng.integers(0, n_pages, (5, 40))
    rows = np.where((refs[rows] > 0) & (rng.random((5, 40)) < 0.8), rows, rng.choice([-1, n_pages, 1 << 29], (5, 40)))
    p.put(rows, refs)
    ids, used = (rce_amd.DeviceBuffer.from_numpy(ctx, np.full(n, 77, np.int32)) for n in (n_pages + 1, 2))
    rce_amd.kv_compact_dev(ctx, p.cache, p.table, p.refs.ptr, ids.ptr, used.ptr)
    want, n = p.host.compact()
    p.host.apply(p.pool)
    p.check()
    assert np.array_equal(ids.download(np.int32, n_pages + 1), want + [77])
    assert used.download(np.int32, 2).tolist() == [n, 77]
    # again: nothing is left to move; without a table, without the count
    rce_amd.kv_compact_dev(ctx, p.cache, rce_amd.KvTable(0, 0, 0), p.refs.ptr, ids.ptr)
    p.check()
    assert np.array_equal(ids.download(np.int32, n_pages), [i if i < n else -1 for i in range(n_pages)])
    ids.free(); used.free()
    p.free()


@pytest.mark.parametrize("page,heads,d", [(16, 1, 64), (64, 5, 192), (4096, 2, 64), (128, 8, 128)])
def test_copies_between_pools(ctx, page, heads, d):
    rng = np.random.default_rng(page)
    a, b = (Pages(ctx, rng, n, page, heads, d, 1, 1) for n in (6, 9))
    src, dst = [5, 0, 0, 6, 2, -1, 3], [1, 8, 4, 0, 9, 2, 3]
    rce_amd.kv_copy_dev(ctx, a.cache, b.cache, a.arr(src), a.arr(dst), len(src))
    for s, t in zip(src, dst):
        if 0 <= s < 6 and 0 <= t < 9:
            for n in PARTS:
                getattr(b.pool, n)[t] = getattr(a.pool, n)[s]
    a.check(); b.check()
    rce_amd.kv_copy_dev(ctx, b.cache, b.cache, a.arr([1, 3]), a.arr([0, 7]), 2)
    for n in PARTS:
        getattr(b.pool, n)[[0, 7]] = getattr(b.pool, n)[[1, 3]]
    b.check()
    a.free(); b.free()


def test_a_pool_beyond_32_bits(ctx):
    """Pages whose codes lie behind 4 GiB: copied by a reservation, a compaction and by hand."""
    n, page, d = 70000, 1024, 64
    with rce_amd.Context(0) as c:
        cache = rce_amd.KvCache.allocate(c, n, page, 1, d)
        k, v, ks, vs = cache.buffers
        size = page * d
        rng = np.random.default_rng(6)
        one = rng.integers(-127, 128, size).astype(np.int8)
        L = rce_amd._lib.lib()
        put = lambda b, at, a: rce_amd._lib.check(L.rce_qmm_memcpy_h2d(c.handle, b.ptr + at, a.ctypes.data, a.nbytes))  # noqa: E731

        def get(b, at, nbytes):
            a = np.empty(nbytes, np.int8)
            rce_amd._lib.check(L.rce_qmm_memcpy_d2h(c.handle, a.ctypes.data, b.ptr + at, nbytes))
            return a
        far = n - 2
        put(k, far * size, one)
        put(v, far * size, one[::-1].copy())
        up = lambda a: rce_amd.DeviceBuffer.from_numpy(c, np.asarray(a, np.int32))  # noqa: E731
        refs = np.ones(n, np.int32)
        refs[far], refs[n - 1], refs[3] = 2, 0, 0
        refs[far - 1] = 0
        r, pages, off, lens = up(refs), up([[far], [far]]), up([0, 1, 2]), up([page, page])
        refs[3] = 1
        r.upload(refs)
        rce_amd.kv_reserve_dev(c, cache, rce_amd.KvBatch(off.ptr, lens.ptr, pages.ptr, 2, 2, 1), r.ptr)
        c.synchronize()
        assert pages.download(np.int32, 2).tolist() == [far, far - 1]
        assert np.array_equal(get(k, (far - 1) * size, size), one) and np.array_equal(get(v, (far - 1) * size, size), one[::-1])
        a, b = up([far - 1]), up([n - 1])
        rce_amd.kv_copy_dev(c, cache, cache, a.ptr, b.ptr, 1)
        c.synchronize()
        assert np.array_equal(get(k, (n - 1) * size, size), one) and np.array_equal(get(v, (n - 1) * size, size), one[::-1])
        refs = np.zeros(n, np.int32)
        refs[far] = 2
        r.upload(refs)
        pages.upload(np.array([far, far], np.int32))
        ids = up(np.zeros(n))
        rce_amd.kv_compact_dev(c, cache, rce_amd.KvTable(pages.ptr, 2, 1), r.ptr, ids.ptr)
        c.synchronize()
        assert pages.download(np.int32, 2).tolist() == [0, 0]
        assert np.array_equal(get(k, 0, size), one) and np.array_equal(get(v, 0, size), one[::-1])
        for x in (r, pages, off, lens, a, b, ids):
            x.free()
        cache.free()


def test_recorded(ctx):
    """Fork, release, reserve and compact recorded as one graph: every replay against the lists, other calls on the
    context's buffer in between."""
    rng = np.random.default_rng(7)
    n, page, max_pages = 5, 16, 6
    with rce_amd.Context(0) as c:
        p = Pages(c, rng, 40, page, 2, 64, n, max_pages)
        other = Pages(c, rng, 30, page, 1, 64, 9, 3)
        up = lambda a: rce_amd.DeviceBuffer.from_numpy(c, np.asarray(a, np.int32))  # noqa: E731
        lens = np.array([3, 20, 16, 33, 47])
        p.reserve(lens, lens)
        parents, ends, off, ln = up([0, 0, 2, 2, 4]), up(np.zeros(n)), up(np.arange(n + 1)), up(lens)
        to, ids = up(np.full((n, max_pages), -1)), up(np.zeros(40))
        tt = rce_amd.KvTable(to.ptr, n, max_pages)
        same = up(np.arange(n))

        def step():  # the beams go on in the second table, and back into the first
            rce_amd.kv_fork_dev(c, p.cache, p.table, tt, parents.ptr, p.refs.ptr)
            rce_amd.kv_release_dev(c, p.cache, p.table, p.refs.ptr)
            rce_amd.kv_fork_dev(c, p.cache, tt, p.table, same.ptr, p.refs.ptr)
            rce_amd.kv_release_dev(c, p.cache, tt, p.refs.ptr)
            rce_amd.kv_reserve_dev(c, p.cache, rce_amd.KvBatch(off.ptr, ln.ptr, p.pages.ptr, n, n, max_pages), p.refs.ptr, p.missing.ptr)
            rce_amd.kv_compact_dev(c, p.cache, p.table, p.refs.ptr, ids.ptr)
        hip = Hip()
        g, ex = hip.capture(c.stream, step)
        for i in range(4):
            pick = rng.integers(0, n, n)
            lens = lens[pick] + 1
            parents.upload(pick.astype(np.int32))
            ln.upload(lens.astype(np.int32))
            other.release()
            other.reserve(rng.integers(0, 40, 9), np.full(9, 40))
            hip.launch(ex, c.stream)
            c.synchronize()
            rows = [list(r) for r in p.host.pages]
            p.host.fork(p.host.pages, [])
            p.host.pages = rows
            new = [[-1] * max_pages for _ in range(n)]
            p.host.fork(new, pick.tolist())
            p.host.release()
            p.host.pages = new
            p.host.reserve(list(range(n + 1)), lens.tolist())
            p.host.apply(p.pool)
            p.host.compact()
            p.host.apply(p.pool)
            p.check()
        hip.destroy(g, ex)
        for b in (parents, ends, off, ln, to, ids, same):
            b.free()
        p.free(); other.free()
