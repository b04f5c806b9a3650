// kv_pages.hip -- copying, forking, reserving, releasing and compacting the
// pages of the paged KV cache (include/rce_qmm.h).
//
// refs[p] counts the table entries that name page p; 0: it is free.  What is
// chosen (free pages, what keeps a shared page, what moves where) depends on
// the tables and counts alone: integer atomics in any order, and ranks.
#include "kv_pages.h"

#include <algorithm>

namespace rce_qmm {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ int seen(const int32_t *p) {  // what other waves' atomics left
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// A barrier behind which the block's waves see each other's accesses to memory by `seen` and atomics: waves of one block share an
// L2, so that it is enough for them to have arrived there.  (A fence for the whole GPU writes back what the L2 holds of the kernels before:
// behind a copy of 300 MB it cost 3 us.)
__device__ __forceinline__ void arrived() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// ---- tables -----------------------------------------------------------------

__global__ __launch_bounds__(256) void k_kv_fork(KvTable from, KvTable to, const int32_t *parents, KvRefs R) {
    const unsigned at = blockIdx.x * 256 + threadIdx.x;
    if (at >= to.entries()) return;
    const unsigned s = at / (unsigned)to.max_pages, i = at - s * (unsigned)to.max_pages;
    const int parent = parents[s];
    if ((unsigned)parent >= (unsigned)from.n_seqs) return;
    int p = i < (unsigned)from.max_pages ? from.pages[(size_t)parent * from.max_pages + i] : -1;
    if ((unsigned)p < (unsigned)R.n_pages) atomicAdd(R.refs + p, 1);
    else p = -1;
    to.pages[at] = p;
}

__global__ __launch_bounds__(256) void k_kv_release(KvTable t, int page_tokens, const int32_t *from, const int32_t *to, KvRefs R) {
    const unsigned at = blockIdx.x * 256 + threadIdx.x;
    if (at >= t.entries()) return;
    const unsigned s = at / (unsigned)t.max_pages, i = at - s * (unsigned)t.max_pages;
    const int64_t lo = (int64_t)i * page_tokens;
    if ((from && lo < from[s]) || (to && lo + page_tokens > to[s])) return;
    const int p = t.pages[at];
    if ((unsigned)p < (unsigned)R.n_pages) atomicSub(R.refs + p, 1);
    t.pages[at] = -1;
}

// ---- reserve -------------------------------------------------------------------

// The pages that a call's rows touch are its items, in the order of (sequence, position): one block
// plans them all.  An item without a page needs one; an item whose page others name too asks to leave
// it.  Where all that name a page ask, the first of them keeps it.  Free pages are those whose count is 0, in
// order, looked for EACH * PLAN counts at a time.
//
// A call of up to PLAN items (a token of every sequence) keeps them in registers and finds who asks for the same page in a
// table in LDS.  One of up to HOLD * PLAN items without a shared page (prompts) is held as well.  Others go over the items once per
// step, and count on the pages' own counts: an item that asks takes one off; where that leaves none, the least item number - CODE that is
// written there keeps the page.
//
// What bounds it: the chain of loads (lengths, entries, counts), barriers of 16 waves.  Behind the first AHEAD looks each look for free pages is a
// load and two barriers more, 1 us for 4096 counts: 64 tokens that each need a page, with the free ones at the pool's end: 4.0 us in a pool of 16384 pages,
// 16 of 65536, 64 of 262144, 256 of 2^20.
constexpr int PLAN = 1024;       // threads
constexpr int CODE = 1 << 30;    // items are fewer than 2^24
constexpr int EACH = 4;          // counts that a thread looks at for free pages, and items of a thread's step
constexpr int RING = 2 * EACH * PLAN;
constexpr int HOLD = 8;          // items that a thread holds
constexpr int AHEAD = 4;         // looks' counts that are loaded first of all: behind other kernels each load comes from HBM
constexpr int SLOTS = 2 * PLAN;  // of the table in LDS

struct Front {  // the first `blocks` blocks of page src to page dst, every head
    int src, dst, blocks, pad;
};
struct Room {
    int n_fronts, pad[3];
    Front fronts[1 << 20];   // one per sequence at most
    uint8_t wants[1 << 24];  // per item: 0 nothing, 1 a page, 2 to leave a shared one
};

// Prefix sum over the block (before this thread) and its total; `part`: LDS of 16 ints, free again after it.
__device__ __forceinline__ int block_scan(int v, int *part, int &total) {
    const int wave = threadIdx.x >> 6, incl = wave_scan(v);
    if ((threadIdx.x & 63) == 63) part[wave] = incl;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < PLAN / 64; w++) {
        const int p = part[w];
        before += w < wave ? p : 0;
        total += p;
    }
    __syncthreads();
    return before + incl - v;
}

// Ranks among N * PLAN values in the order of (wave, e, lane): value e of this thread is number 64 (N wave + e) + lane.
// of[e]: the true ones before it; the total is the same in all threads.
template <int N>
__device__ __forceinline__ int ranks(const bool (&is)[N], int *part, int (&of)[N]) {
    const int wave = threadIdx.x >> 6;
    int n = 0;
#pragma unroll
    for (int e = 0; e < N; e++) {
        const uint64_t m = __ballot(is[e]);
        of[e] = n + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
        n += __popcll(m);
    }
    if ((threadIdx.x & 63) == 0) part[wave] = n;
    __syncthreads();
    int before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < PLAN / 64; w++) {
        const int p = part[w];
        before += w < wave ? p : 0;
        total += p;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < N; e++) of[e] += before;
    return total;
}
template <int N>
__device__ __forceinline__ int numbered(int e) { return 64 * (N * (threadIdx.x >> 6) + e) + (threadIdx.x & 63); }

// A front's head h and kind (0 keys, 1 values): thread i of n.
__device__ __forceinline__ void copy_front(const KvPool &P, int d, const Front &f, int h, int kind, int i, int n) {
    const size_t a = ((size_t)f.src * P.heads + h) << P.lg_b, b = ((size_t)f.dst * P.heads + h) << P.lg_b;
    int8_t *codes = kind ? P.v : P.k;
    const u32x4 *from = reinterpret_cast<const u32x4 *>(codes + a * (KV_BLOCK * d));
    u32x4 *to = reinterpret_cast<u32x4 *>(codes + b * (KV_BLOCK * d));
#pragma unroll 4
    for (int j = i; j < f.blocks * d; j += n) to[j] = from[j];
    float *scale = kind ? P.v_scale : P.k_scale;
    for (int j = i; j < f.blocks; j += n) scale[b + j] = scale[a + j];
}

// d: 0, or the head size where the block copies the fronts itself.
__global__ __launch_bounds__(PLAN) void k_kv_reserve(KvRows B, int lg_page, int32_t *pages, KvRefs R, int32_t *missing, Room *room, KvPool P, int d) {
    __shared__ int part[PLAN / 64], start[PLAN + 1], slot0[PLAN], front0[PLAN], lost[PLAN], ring[RING];
    __shared__ int n_fronts;
    int *const key = ring, *const asked = ring + SLOTS, *const first_ask = ring + 2 * SLOTS;  // before the ring is used
    static_assert(3 * SLOTS <= RING, "the table fits the ring");
    const int tid = threadIdx.x;
    if (!B.n_rows || !B.cap) {  // no items; the batch's arrays may be null
        if (missing)
            for (int s = tid; s < B.n_seqs; s += PLAN) missing[s] = 0;
        return;
    }
    auto entry = [&](int s, int slot) { return pages + (size_t)s * B.max_pages + slot; };

    // the first counts, on their way while the items are found
    int ahead[AHEAD][EACH];
#pragma unroll
    for (int a = 0; a < AHEAD; a++)
#pragma unroll
        for (int e = 0; e < EACH; e++) ahead[a][e] = R.refs[min(EACH * PLAN * a + numbered<EACH>(e), R.n_pages - 1)];
    int head = 0, have = 0, looked = 0;  // the ring's first free page, its free pages, counts looked at
    auto look = [&](const int (&counts)[EACH]) {
        bool free[EACH];
        int of[EACH];
#pragma unroll
        for (int e = 0; e < EACH; e++) free[e] = looked + numbered<EACH>(e) < R.n_pages && counts[e] == 0;
        const int more = ranks<EACH>(free, part, of);
#pragma unroll
        for (int e = 0; e < EACH; e++)
            if (free[e] && have + of[e] < RING) ring[(head + have + of[e]) & (RING - 1)] = looked + numbered<EACH>(e);
        have += more;
        looked += min(EACH * PLAN, R.n_pages - looked);
        __syncthreads();
    };
    auto look_for = [&](int wanted) {  // the same in every thread
#pragma unroll
        for (int a = 0; a < AHEAD; a++)
            if (looked == EACH * PLAN * a && have < wanted && looked < R.n_pages) look(ahead[a]);
        while (have < wanted && looked < R.n_pages) {
            int counts[EACH];
#pragma unroll
            for (int e = 0; e < EACH; e++) counts[e] = seen(R.refs + min(looked + numbered<EACH>(e), R.n_pages - 1));
            look(counts);
        }
    };
    // a free page for an item (rank: items of this step that need one before it), or none; its page p is left behind if it has one
    auto give = [&](int s, int slot, int rank, int p, bool leaves) {
        const int to = rank < have ? ring[(head + rank) & (RING - 1)] : -1;
        *entry(s, slot) = to;
        if (to < 0) return false;
        R.refs[to] = 1;
        // what stands in front of the call's rows in the page it leaves
        const int q = s & (PLAN - 1);
        if (leaves && slot == slot0[q] && front0[q]) room->fronts[atomicAdd(&n_fronts, 1)] = {p, to, front0[q], 0};
        return true;
    };
    // items of the sequences c .. c + PLAN - 1, and where they start
    auto list = [&](int c) {
        int n = 0, items;
        if (c + tid < B.n_seqs) {
            const KvSeq q = kv_seq(B, c + tid);
            const int lo = q.lo(), hi = q.hi(B);
            slot0[tid] = lo >> lg_page;
            front0[tid] = ((lo & ((1 << lg_page) - 1)) + KV_BLOCK - 1) / KV_BLOCK;
            n = hi > lo ? ((hi - 1) >> lg_page) - slot0[tid] + 1 : 0;
        }
        start[tid] = block_scan(n, part, items);
        if (tid == 0) start[PLAN] = items;
        __syncthreads();
        return items;
    };
    auto sequence = [&](int i) {  // the last one that starts at or before item i
        int s = 0;
#pragma unroll
        for (int o = PLAN / 2; o; o /= 2)
            if (start[s + o] <= i) s += o;
        return s;
    };

    auto copy = [&] {  // the fronts, or their number for the next kernel
        if (!d) {
            __syncthreads();
            if (tid == 0) room->n_fronts = n_fronts;
            return;
        }
        arrived();
        for (int u = tid >> 6; u < n_fronts * P.heads * 2; u += PLAN / 64) {
            const int *p = &room->fronts[(u >> 1) / P.heads].src;
            copy_front(P, d, {seen(p), seen(p + 1), seen(p + 2), 0}, (u >> 1) % P.heads, u & 1, tid & 63, 64);
        }
    };

    if (tid == 0) n_fronts = 0;
    lost[tid] = 0;
#pragma unroll
    for (int i = 0; i < SLOTS / PLAN; i++) {
        key[tid + PLAN * i] = -1;
        asked[tid + PLAN * i] = 0;
        first_ask[tid + PLAN * i] = PLAN;
    }
    int items = list(0);
    if (B.n_seqs <= PLAN && items <= PLAN) {
        const bool is = tid < items;
        const int s = sequence(min(tid, max(items - 1, 0))), slot = slot0[s] + tid - start[s];
        const int p = is ? *entry(s, slot) : 0;
        const bool named = (unsigned)p < (unsigned)R.n_pages;
        const int refs = is && named ? R.refs[p] : 0;
        bool need = is && !named, leaves = is && named && refs > 1;
        if (__syncthreads_or(leaves)) {
            int h = (int)(((uint32_t)p * 2654435769u) >> 21);  // of 2048
            static_assert(SLOTS == 2048, "11 bits");
            if (leaves) {
                for (;;) {  // at most PLAN of the SLOTS are taken: an empty one comes
                    const int k = atomicCAS(key + h, -1, p);
                    if (k == -1 || k == p) break;
                    h = (h + 1) & (SLOTS - 1);
                }
                atomicAdd(asked + h, 1);
                atomicMin(first_ask + h, tid);
            }
            __syncthreads();
            if (leaves && asked[h] == refs && first_ask[h] == tid) leaves = false;
            need |= leaves;
        }
        int total;
        const int rank = block_scan(need, part, total);
        look_for(total);
        if (need) {
            if (leaves) atomicSub(R.refs + p, 1);
            if (!give(s, slot, rank, p, leaves)) atomicAdd(lost + s, 1);
        }
        copy();
        if (missing && tid < B.n_seqs) missing[tid] = lost[tid];
        return;
    }

    if (B.n_seqs <= PLAN && items <= HOLD * PLAN) {  // HOLD items a thread, no shared page among them
        int s[HOLD], slot[HOLD], p[HOLD], of[HOLD];
        bool need[HOLD], shared = false;
#pragma unroll
        for (int e = 0; e < HOLD; e++) {
            const int at = min(numbered<HOLD>(e), items - 1);
            s[e] = sequence(at);
            slot[e] = slot0[s[e]] + at - start[s[e]];
        }
#pragma unroll
        for (int e = 0; e < HOLD; e++) p[e] = *entry(s[e], slot[e]);
#pragma unroll
        for (int e = 0; e < HOLD; e++) {
            const bool named = (unsigned)p[e] < (unsigned)R.n_pages;
            need[e] = numbered<HOLD>(e) < items && !named;
            if (named) shared |= R.refs[p[e]] > 1;  // (behind the last item: its own again)
        }
        if (!__syncthreads_or(shared)) {
            look_for(ranks<HOLD>(need, part, of));
#pragma unroll
            for (int e = 0; e < HOLD; e++)
                if (need[e] && !give(s[e], slot[e], of[e], -1, false)) atomicAdd(lost + s[e], 1);
            copy();
            if (missing && tid < B.n_seqs) missing[tid] = lost[tid];
            return;
        }
    }

    if (missing)
        for (int s = tid; s < B.n_seqs; s += PLAN) missing[s] = 0;
    // f(number of the first, items' sequences and places, how many) for EACH consecutive items of every thread; every thread calls it
    int chunk = 0;
    auto each = [&](auto f) {
        int before = 0;
        for (int c = 0; c < B.n_seqs; c += PLAN) {
            if (c != chunk) {
                __syncthreads();
                items = list(c);
                chunk = c;
            }
            for (int i0 = 0; i0 < items; i0 += EACH * PLAN) {
                int s[EACH], slot[EACH];
                const int i = i0 + EACH * tid, n = min(EACH, max(0, items - i));
                int q = sequence(min(i, items - 1));
#pragma unroll
                for (int e = 0; e < EACH; e++) {
                    const int at = min(i + e, items - 1);
                    while (start[q + 1] <= at) q++;  // start[PLAN] is above all
                    s[e] = c + q;
                    slot[e] = slot0[q] + at - start[q];
                }
                f(before + i, s, slot, n);
            }
            before += items;
        }
    };

    bool shared = false;
    each([&](int item, const int (&s)[EACH], const int (&slot)[EACH], int n) {
        int p[EACH], refs[EACH];
#pragma unroll
        for (int e = 0; e < EACH; e++) p[e] = *entry(s[e], slot[e]);
#pragma unroll
        for (int e = 0; e < EACH; e++) refs[e] = (unsigned)p[e] < (unsigned)R.n_pages ? R.refs[p[e]] : 0;
#pragma unroll
        for (int e = 0; e < EACH; e++)
            if (e < n) {
                const int want = (unsigned)p[e] >= (unsigned)R.n_pages ? 1 : refs[e] > 1 ? 2 : 0;
                room->wants[item + e] = (uint8_t)want;
                shared |= want == 2;
            }
    });
    if (__syncthreads_or(shared)) {
        each([&](int item, const int (&s)[EACH], const int (&slot)[EACH], int n) {
            for (int e = 0; e < n; e++)
                if (room->wants[item + e] == 2) atomicSub(R.refs + *entry(s[e], slot[e]), 1);
        });
        arrived();
        each([&](int item, const int (&s)[EACH], const int (&slot)[EACH], int n) {
            for (int e = 0; e < n; e++) {
                if (room->wants[item + e] != 2) continue;
                int32_t *r = R.refs + *entry(s[e], slot[e]);
                if (seen(r) <= 0) atomicMin(r, item + e - CODE);
            }
        });
    }
    arrived();
    each([&](int item, const int (&s)[EACH], const int (&slot)[EACH], int n) {
        int p[EACH], count = 0;
        bool need[EACH], leaves[EACH];
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            const int want = e < n ? room->wants[item + e] : 0;
            leaves[e] = want == 2;
            need[e] = want == 1;
            p[e] = -1;
            if (leaves[e]) {
                p[e] = *entry(s[e], slot[e]);
                leaves[e] = need[e] = seen(R.refs + p[e]) != item + e - CODE;
                if (!need[e]) __hip_atomic_store(R.refs + p[e], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            count += need[e];
        }
        int total, rank = block_scan(count, part, total);
        look_for(total);
#pragma unroll
        for (int e = 0; e < EACH; e++)
            if (need[e] && !give(s[e], slot[e], rank++, p[e], leaves[e]) && missing) atomicAdd(missing + s[e], 1);
        const int used = min(have, total);
        head = (head + used) & (RING - 1);
        have -= used;
        __syncthreads();  // the ring's places are read
    });
    copy();
}

// A block takes a front's head and kind (keys, values), every block of the grid the next ones.
__global__ __launch_bounds__(256) void k_kv_copy_fronts(KvPool P, int d, const Room *room) {
    const int n = room->n_fronts * P.heads * 2;
    for (int u = blockIdx.x; u < n; u += gridDim.x)
        copy_front(P, d, room->fronts[(u >> 1) / P.heads], (u >> 1) % P.heads, u & 1, threadIdx.x, 256);
}

// ---- whole pages ------------------------------------------------------------

// Pages src[i] of one pool to dst[i] of another (or the same), i < *count (null: n): a block takes PIECE bytes of a page's
// keys or values, every block of the grid the next ones.
// Past the L2s, which the page's readers would not find it in anyway (333 MB in 63 -> 61 us).
// The first `renaming` blocks give the entries of t their pages' new ids instead.
constexpr int PIECE = 16384;
__global__ __launch_bounds__(256) void k_kv_copy(KvPool A, KvPool B, size_t page_bytes, int pieces, const int32_t *src, const int32_t *dst,
                                                 const int32_t *count, int n, KvTable t, const int32_t *new_ids, unsigned renaming) {
    if (blockIdx.x < renaming) {
        for (unsigned i = blockIdx.x * 256 + threadIdx.x; i < t.entries(); i += renaming * 256) {
            const int p = t.pages[i];
            if ((unsigned)p < (unsigned)A.n_pages) t.pages[i] = new_ids[p];
        }
        return;
    }
    const size_t units = (size_t)(count ? *count : n) * 2 * pieces;
    for (size_t u = blockIdx.x - renaming; u < units; u += gridDim.x - renaming) {
        const size_t m = u / (2 * pieces);
        const int rest = (int)(u - m * 2 * pieces), kind = rest & 1, piece = rest >> 1;
        const int a = src[m], b = dst[m];
        if ((unsigned)a >= (unsigned)A.n_pages || (unsigned)b >= (unsigned)B.n_pages) continue;
        const int8_t *from = (kind ? A.v : A.k) + (size_t)a * page_bytes + (size_t)piece * PIECE;
        int8_t *to = (kind ? B.v : B.k) + (size_t)b * page_bytes + (size_t)piece * PIECE;
        const int bytes = (int)min((size_t)PIECE, page_bytes - (size_t)piece * PIECE), end = bytes / 16;
        u32x4 v[4];
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = reinterpret_cast<const u32x4 *>(from)[min((int)threadIdx.x + 256 * j, end - 1)];
#pragma unroll
        for (int j = 0; j < 4; j++)
            if ((int)threadIdx.x + 256 * j < end) __builtin_nontemporal_store(v[j], reinterpret_cast<u32x4 *>(to) + threadIdx.x + 256 * j);
        if (piece == 0) {
            const int scales = A.heads << A.lg_b;
            const float *fs = (kind ? A.v_scale : A.k_scale) + (size_t)a * scales;
            float *ts = (kind ? B.v_scale : B.k_scale) + (size_t)b * scales;
            for (int i = threadIdx.x; i < scales; i += 256) ts[i] = fs[i];
        }
    }
}

// The used pages behind the first n_used ones move, in order, to the free pages among those.
struct Moves {
    int count, pad[3];
    int32_t src[KV_COMPACT_PAGES / 2], dst[KV_COMPACT_PAGES / 2];
};
// One block: the used pages are counted; then each page's place among the used ones says what it is to do, LOOK counts a thread and
// step: the free ones among the first n are listed, and the used ones behind them take them in order.
constexpr int LOOK = 16;
__device__ __forceinline__ void look_at(const KvRefs &R, int from, int (&r)[LOOK]) {
#pragma unroll
    for (int e = 0; e < LOOK; e++) r[e] = R.refs[min(from + numbered<LOOK>(e), R.n_pages - 1)];
#pragma unroll
    for (int e = 0; e < LOOK; e++) r[e] = from + numbered<LOOK>(e) < R.n_pages ? r[e] : 0;
}
__global__ __launch_bounds__(PLAN) void k_kv_compact(KvRefs R, int32_t *new_ids, int32_t *n_used, Moves *moves) {
    __shared__ int part[PLAN / 64], list[LOOK * PLAN / 2];  // where ref holds all counts, what is free below n: half of them at most
    const int tid = threadIdx.x;
    __shared__ int before_n;  // used pages among the first n
    int ref[LOOK], of[LOOK], n = 0;
    bool is[LOOK];
    for (int p0 = 0; p0 < R.n_pages; p0 += LOOK * PLAN) {
        look_at(R, p0, ref);
#pragma unroll
        for (int e = 0; e < LOOK; e++) is[e] = ref[e] != 0;
        n += ranks<LOOK>(is, part, of);
    }
    const bool once = R.n_pages <= LOOK * PLAN;  // ref, is and of hold all
    int used = 0;                                // before this step
    for (int p0 = 0; p0 < R.n_pages; p0 += LOOK * PLAN) {
        int total = n;
        if (!once) {
            look_at(R, p0, ref);
#pragma unroll
            for (int e = 0; e < LOOK; e++) is[e] = ref[e] != 0;
            total = ranks<LOOK>(is, part, of);
        }
        // what is not used before n, in order: the pages before it less the used ones
#pragma unroll
        for (int e = 0; e < LOOK; e++) {
            const int p = p0 + numbered<LOOK>(e), u = used + of[e];
            if (p == n) before_n = u;
            if (p >= n) continue;
            if (!is[e]) {
                moves->dst[p - u] = p;
                if (once) list[p - u] = p;
            }
            new_ids[p] = is[e] ? p : -1;
        }
        if (once) __syncthreads();
        else arrived();
        int to[LOOK];
#pragma unroll
        for (int e = 0; e < LOOK; e++) {
            const int r = used + of[e] - before_n;
            to[e] = p0 + numbered<LOOK>(e) < n || !is[e] ? -1 : once ? list[r] : seen(moves->dst + r);
        }
#pragma unroll
        for (int e = 0; e < LOOK; e++) {
            const int p = p0 + numbered<LOOK>(e);
            if (p < n || p >= R.n_pages) continue;
            if (is[e]) {
                moves->src[used + of[e] - before_n] = p;
                R.refs[to[e]] = ref[e];
                R.refs[p] = 0;
            }
            new_ids[p] = to[e];
        }
        used += total;
    }
    if (tid == 0) {
        moves->count = n < R.n_pages ? n - before_n : 0;
        if (n_used) *n_used = n;
    }
}

dim3 over_entries(const KvTable &t) { return dim3((unsigned)((t.entries() + 255) / 256)); }
constexpr size_t OWN_COPY = (size_t)128 << 10;  // bytes that the planning block copies itself: 4 beams of 4 heads of 64, whole pass with fork and release 17.1 -> 13.8 us
constexpr size_t COPY_BLOCKS = 4096, RENAME_BLOCKS = 256;
// Whole reservations with blocks of up to 256 : 512 : 1024 : 2048 : 4096 for the fronts (us, 8 heads of 128, half a page of 128 positions each): 128 fronts
// 13.9 : 10.3 : 8.7 : 8.9 : 9.2, 512 fronts 51 : 33 : 24 : 21 : 20; with nothing to copy the launch costs 2 us of 7, whatever their number.
constexpr size_t FRONT_BLOCKS = 2048;

void copy_pages(const KvPool &from, const KvPool &to, int d_head, const int32_t *src, const int32_t *dst, const int32_t *count, int n,
                const KvTable &t, const int32_t *new_ids, hipStream_t s) {
    const size_t bytes = ((size_t)from.heads << from.lg_b) * KV_BLOCK * d_head, pieces = (bytes + PIECE - 1) / PIECE;
    const size_t renaming = std::min(RENAME_BLOCKS, (t.entries() + 255) / 256);
    const dim3 g((unsigned)(std::min(COPY_BLOCKS, std::max((size_t)1, (size_t)n * 2 * pieces)) + renaming));
    hipLaunchKernelGGL(k_kv_copy, g, dim3(256), 0, s, from, to, bytes, (int)pieces, src, dst, count, n, t, new_ids, (unsigned)renaming);
}

}  // namespace

size_t kv_pages_bytes() { return std::max(sizeof(Room), sizeof(Moves)); }

hipError_t launch_kv_copy(const KvPool &from, const KvPool &to, int d_head, const int32_t *src, const int32_t *dst, int n, hipStream_t s) {
    copy_pages(from, to, d_head, src, dst, nullptr, n, {nullptr, 0, 0}, nullptr, s);
    return hipGetLastError();
}

hipError_t launch_kv_fork(const KvTable &from, const KvTable &to, const int32_t *parents, const KvRefs &refs, hipStream_t s) {
    hipLaunchKernelGGL(k_kv_fork, over_entries(to), dim3(256), 0, s, from, to, parents, refs);
    return hipGetLastError();
}

hipError_t launch_kv_release(const KvTable &t, int page_tokens, const int32_t *from, const int32_t *to, const KvRefs &refs, hipStream_t s) {
    hipLaunchKernelGGL(k_kv_release, over_entries(t), dim3(256), 0, s, t, page_tokens, from, to, refs);
    return hipGetLastError();
}

hipError_t launch_kv_reserve(const KvPool &pool, const KvRows &rows, int d_head, int32_t *pages, int32_t *refs, int32_t *missing,
                             void *room, hipStream_t s) {
    Room *r = static_cast<Room *>(room);
    // what the fronts come to at most: a page per sequence
    const bool small = ((size_t)rows.n_seqs * pool.heads * 2 << pool.lg_b) * KV_BLOCK * d_head <= OWN_COPY;
    hipLaunchKernelGGL(k_kv_reserve, dim3(1), dim3(PLAN), 0, s, rows, pool.lg_b + 4, pages, KvRefs{refs, pool.n_pages}, missing, r, pool,
                       small ? d_head : 0);
    if (!rows.n_rows || !rows.cap || small) return hipGetLastError();
    const dim3 g((unsigned)std::min(FRONT_BLOCKS, (size_t)rows.n_seqs * pool.heads * 2));
    hipLaunchKernelGGL(k_kv_copy_fronts, g, dim3(256), 0, s, pool, d_head, r);
    return hipGetLastError();
}

hipError_t launch_kv_compact(const KvPool &pool, int d_head, const KvTable &t, int32_t *refs, int32_t *new_ids, int32_t *n_used,
                             void *room, hipStream_t s) {
    Moves *m = static_cast<Moves *>(room);
    hipLaunchKernelGGL(k_kv_compact, dim3(1), dim3(PLAN), 0, s, KvRefs{refs, pool.n_pages}, new_ids, n_used, m);
    copy_pages(pool, pool, d_head, m->src, m->dst, &m->count, pool.n_pages / 2, t, new_ids, s);
    return hipGetLastError();
}

}  // namespace rce_qmm
