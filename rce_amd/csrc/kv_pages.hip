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
// it.  Where all that name a page ask (its count falls to 0), the first of them keeps it: its number - CODE
// is then the least that is written to the count.
constexpr int PLAN = 1024;       // threads
constexpr int CODE = 1 << 30;    // items are fewer than 2^24
constexpr int EACH = 4;          // counts that a thread looks at for free pages
constexpr int RING = 2 * EACH * PLAN;

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

__global__ __launch_bounds__(PLAN) void k_kv_reserve(KvRows B, int lg_page, int32_t *pages, KvRefs R, int32_t *missing, Room *room) {
    __shared__ int part[PLAN / 64], start[PLAN + 1], slot0[PLAN], ring[RING];
    __shared__ int n_fronts;
    const int tid = threadIdx.x;
    if (tid == 0) n_fronts = 0;
    if (missing)
        for (int s = tid; s < B.n_seqs; s += PLAN) missing[s] = 0;
    if (!B.n_rows || !B.cap) return;  // no items; the batch's arrays may be null
    int chunk = -1, items = 0;
    // f(item number, sequence, its page's place in the table, place of its first item) for every item, PLAN at a time; every thread
    // calls it (item -1: none)
    auto each = [&](auto f) {
        int before = 0;
        for (int c = 0; c < B.n_seqs; c += PLAN) {
            if (c != chunk) {
                const int s = c + tid;
                int n = 0;
                __syncthreads();
                if (s < B.n_seqs) {
                    const KvSeq q = kv_seq(B, s);
                    slot0[tid] = q.lo() >> lg_page;
                    n = q.hi(B) > q.lo() ? ((q.hi(B) - 1) >> lg_page) - slot0[tid] + 1 : 0;
                }
                start[tid] = block_scan(n, part, items);
                if (tid == 0) start[PLAN] = items;
                chunk = c;
                __syncthreads();
            }
            for (int i0 = 0; i0 < items; i0 += PLAN) {
                const int i = i0 + tid;
                int s = 0;
#pragma unroll
                for (int o = PLAN / 2; o; o /= 2)  // the last sequence that starts at or before i
                    if (start[s + o] <= i) s += o;
                f(i < items ? before + i : -1, c + s, slot0[s] + i - start[s], slot0[s]);
            }
            before += items;
        }
    };
    auto entry = [&](int s, int slot) { return pages + (size_t)s * B.max_pages + slot; };

    bool shared = false;
    each([&](int item, int s, int slot, int) {
        if (item < 0) return;
        const int p = *entry(s, slot);
        const int want = (unsigned)p >= (unsigned)R.n_pages ? 1 : R.refs[p] > 1 ? 2 : 0;
        room->wants[item] = (uint8_t)want;
        shared |= want == 2;
    });
    if (__syncthreads_or(shared)) {
        each([&](int item, int s, int slot, int) {
            if (item >= 0 && room->wants[item] == 2) atomicSub(R.refs + *entry(s, slot), 1);
        });
        __threadfence();
        __syncthreads();
        each([&](int item, int s, int slot, int) {
            if (item < 0 || room->wants[item] != 2) return;
            int32_t *r = R.refs + *entry(s, slot);
            if (seen(r) <= 0) atomicMin(r, item - CODE);
        });
    }
    __threadfence();
    __syncthreads();
    int head = 0, have = 0, looked = 0;  // the ring's first free page, its free pages, counts looked at
    each([&](int item, int s, int slot, int first) {
        const int want = item < 0 ? 0 : room->wants[item];
        int p = -1;
        bool need = want == 1;
        if (want == 2) {
            p = *entry(s, slot);
            need = seen(R.refs + p) != item - CODE;
            if (!need) __hip_atomic_store(R.refs + p, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        int total;
        const int rank = block_scan(need, part, total);
        while (have < total && looked < R.n_pages) {  // the same in every thread
            int free[EACH], n = 0;
#pragma unroll
            for (int e = 0; e < EACH; e++) {
                const int at = looked + EACH * tid + e;
                free[e] = at < R.n_pages && seen(R.refs + at) == 0;
                n += free[e];
            }
            int more, at = block_scan(n, part, more);
#pragma unroll
            for (int e = 0; e < EACH; e++)
                if (free[e]) ring[(head + have + at++) & (RING - 1)] = looked + EACH * tid + e;
            have += more;
            looked += min(EACH * PLAN, R.n_pages - looked);
            __syncthreads();
        }
        if (need) {
            const int to = rank < have ? ring[(head + rank) & (RING - 1)] : -1;
            *entry(s, slot) = to;
            if (to >= 0) {
                R.refs[to] = 1;
                // what stands in front of the call's rows in the page it leaves
                const KvSeq q = kv_seq(B, s);
                const int in_front = q.lo() & ((1 << lg_page) - 1);
                if (want == 2 && slot == first && in_front)
                    room->fronts[atomicAdd(&n_fronts, 1)] = {p, to, (in_front + KV_BLOCK - 1) / KV_BLOCK, 0};
            } else if (missing) {
                atomicAdd(missing + s, 1);
            }
        }
        const int used = min(have, total);
        head = (head + used) & (RING - 1);
        have -= used;
        __syncthreads();  // the ring's places are read
    });
    __syncthreads();
    if (tid == 0) room->n_fronts = n_fronts;
}

// A block takes a front's head and kind (keys, values), every block of the grid the next ones.
__global__ __launch_bounds__(256) void k_kv_copy_fronts(KvPool P, int d, const Room *room) {
    const int n = room->n_fronts * P.heads * 2;
    for (int u = blockIdx.x; u < n; u += gridDim.x) {
        const int kind = u & 1, h = (u >> 1) % P.heads;
        const Front f = room->fronts[(u >> 1) / P.heads];
        const size_t a = ((size_t)f.src * P.heads + h) << P.lg_b, b = ((size_t)f.dst * P.heads + h) << P.lg_b;
        int8_t *codes = kind ? P.v : P.k;
        const u32x4 *from = reinterpret_cast<const u32x4 *>(codes + a * (KV_BLOCK * d));
        u32x4 *to = reinterpret_cast<u32x4 *>(codes + b * (KV_BLOCK * d));
        for (int i = threadIdx.x; i < f.blocks * d; i += 256) to[i] = from[i];
        float *scale = kind ? P.v_scale : P.k_scale;
        for (int i = threadIdx.x; i < f.blocks; i += 256) scale[b + i] = scale[a + i];
    }
}

// ---- whole pages ------------------------------------------------------------

// Pages src[i] of one pool to dst[i] of another (or the same), i < *count (null: n): a block takes PIECE bytes of a page's
// keys or values, every block of the grid the next ones.
constexpr int PIECE = 16384;
__global__ __launch_bounds__(256) void k_kv_copy(KvPool A, KvPool B, size_t page_bytes, int pieces, const int32_t *src, const int32_t *dst,
                                                 const int32_t *count, int n) {
    const size_t units = (size_t)(count ? *count : n) * 2 * pieces;
    for (size_t u = blockIdx.x; u < units; u += gridDim.x) {
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
            if ((int)threadIdx.x + 256 * j < end) reinterpret_cast<u32x4 *>(to)[threadIdx.x + 256 * j] = v[j];
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
__global__ __launch_bounds__(PLAN) void k_kv_compact(KvRefs R, int32_t *new_ids, int32_t *n_used, Moves *moves) {
    __shared__ int part[PLAN / 64];
    const int tid = threadIdx.x;
    int used = 0;
    for (int p0 = 0; p0 < R.n_pages; p0 += EACH * PLAN) {
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            const int p = p0 + PLAN * e + tid;
            used += p < R.n_pages && R.refs[p] != 0;
        }
    }
    int n;
    block_scan(used, part, n);
    if (tid == 0 && n_used) *n_used = n;
    int holes = 0;
    for (int p0 = 0; p0 < n; p0 += EACH * PLAN) {
        bool hole[EACH];
        int c = 0, total;
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            const int p = p0 + EACH * tid + e;
            hole[e] = p < n && R.refs[p] == 0;
            c += hole[e];
            if (p < n) new_ids[p] = hole[e] ? -1 : p;
        }
        int at = holes + block_scan(c, part, total);
#pragma unroll
        for (int e = 0; e < EACH; e++)
            if (hole[e]) moves->dst[at++] = p0 + EACH * tid + e;
        holes += total;
    }
    __threadfence();
    __syncthreads();
    int moved = 0;
    for (int p0 = n; p0 < R.n_pages; p0 += EACH * PLAN) {
        int ref[EACH], c = 0, total;
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            const int p = p0 + EACH * tid + e;
            ref[e] = p < R.n_pages ? R.refs[p] : 0;
            c += ref[e] != 0;
        }
        int at = moved + block_scan(c, part, total);
#pragma unroll
        for (int e = 0; e < EACH; e++) {
            const int p = p0 + EACH * tid + e;
            int to = -1;
            if (ref[e]) {
                to = seen(moves->dst + at);
                moves->src[at++] = p;
                R.refs[to] = ref[e];
                R.refs[p] = 0;
            }
            if (p < R.n_pages) new_ids[p] = to;
        }
        moved += total;
    }
    if (tid == 0) moves->count = moved;
}

__global__ __launch_bounds__(256) void k_kv_rename(KvTable t, const int32_t *new_ids, int n_pages) {
    const unsigned at = blockIdx.x * 256 + threadIdx.x;
    if (at >= t.entries()) return;
    const int p = t.pages[at];
    if ((unsigned)p < (unsigned)n_pages) t.pages[at] = new_ids[p];
}

dim3 over_entries(const KvTable &t) { return dim3((unsigned)((t.entries() + 255) / 256)); }
constexpr size_t COPY_BLOCKS = 4096;

}  // namespace

size_t kv_pages_bytes() { return std::max(sizeof(Room), sizeof(Moves)); }

static void copy_pages(const KvPool &from, const KvPool &to, int d_head, const int32_t *src, const int32_t *dst, const int32_t *count, int n,
                       hipStream_t s) {
    const size_t bytes = ((size_t)from.heads << from.lg_b) * KV_BLOCK * d_head, pieces = (bytes + PIECE - 1) / PIECE;
    const dim3 g((unsigned)std::max((size_t)1, std::min(COPY_BLOCKS, (size_t)n * 2 * pieces)));
    hipLaunchKernelGGL(k_kv_copy, g, dim3(256), 0, s, from, to, bytes, (int)pieces, src, dst, count, n);
}

hipError_t launch_kv_copy(const KvPool &from, const KvPool &to, int d_head, const int32_t *src, const int32_t *dst, int n, hipStream_t s) {
    copy_pages(from, to, d_head, src, dst, nullptr, n, s);
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
    hipLaunchKernelGGL(k_kv_reserve, dim3(1), dim3(PLAN), 0, s, rows, pool.lg_b + 4, pages, KvRefs{refs, pool.n_pages}, missing, r);
    if (!rows.n_rows || !rows.cap) return hipGetLastError();
    const dim3 g((unsigned)std::min((size_t)2048, (size_t)rows.n_seqs * pool.heads * 2));
    hipLaunchKernelGGL(k_kv_copy_fronts, g, dim3(256), 0, s, pool, d_head, r);
    return hipGetLastError();
}

hipError_t launch_kv_compact(const KvPool &pool, int d_head, const KvTable &t, int32_t *refs, int32_t *new_ids, int32_t *n_used,
                             void *room, hipStream_t s) {
    Moves *m = static_cast<Moves *>(room);
    hipLaunchKernelGGL(k_kv_compact, dim3(1), dim3(PLAN), 0, s, KvRefs{refs, pool.n_pages}, new_ids, n_used, m);
    copy_pages(pool, pool, d_head, m->src, m->dst, &m->count, pool.n_pages / 2, s);
    if (t.entries()) hipLaunchKernelGGL(k_kv_rename, over_entries(t), dim3(256), 0, s, t, new_ids, pool.n_pages);
    return hipGetLastError();
}

}  // namespace rce_qmm
