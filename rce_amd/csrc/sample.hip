// sample.hip -- next tokens from logits: temperature, top-k, top-p, min-p and
// the draw from given uniform numbers (include/rce_qmm.h rce_qmm_sample_dev).
//
// A block per row.  Weights are whole numbers, rint(exp((l - max) / T) 2^S)
// with S = min(50, 62 - ceil(log2 vocab)): a row's sum fits 63 bits, every sum
// is exact and no order of additions matters, so the histograms, made with LDS
// atomics, are deterministic.
//
// The filters keep a prefix of the order (l falling, id rising), told by its
// last element.  A histogram over BINS equal intervals of l says which bin
// holds the end (by counts for top-k, by weights for top-p).  Where the bins up
// to it hold at most NT elements these are collected and sorted, one per thread,
// and everything that follows works on that list.  Else the bin's own elements
// are sorted and cut; a bin of more than NT (many equal logits) goes
// through a radix descent over (order-preserving bits of l, id), 64 bits, 8 a
// pass.
//
// The draw from a row that is no list: run r of the row, q * 256 consecutive
// ids, belongs to wave r % 16; the runs' kept weights are summed and scanned,
// and the wave whose run the draw falls into walks it.
//
// What bounds it: one CU per row, so the instructions of the row's passes over
// LDS (rows above 128 KB: over L2): the first one, the histogram and the collection
// where a list follows, and two more where none does.  A top_k up to NT takes its
// first cut from the threads' own maxima instead of a histogram of all logits.
// 1 x 32000 f32 with top-k 40: 11 us; 500 x 32003 bf16, settings mixed: 65 us (two
// blocks per CU).  Few rows above 128 KB are spread over several CUs, see below.
#include "kv_cache.h"
#include "lds_limit.h"

#include <algorithm>
#include <climits>
#include <type_traits>

namespace rce_qmm {
namespace {

typedef unsigned long long u64;

constexpr int NT = 1024, NW = NT / 64;
constexpr int BINS = 2048, PER = BINS / NT;
constexpr int RUNS = NT;              // runs of a row, at most
constexpr int STEP = 4;               // consecutive ids of a lane
constexpr int ROW_BYTES = 128 << 10;  // a row up to this size is kept in LDS

struct alignas(16) Shared {  // the row follows
    union {                  // in turn
        u64 hist[BINS];
        struct {
            u64 list[NT], weight[NT];
        };
        u64 sums[RUNS];
    };
    double exp2_[128];  // 2^(j / 128)
    u64 wave[NW];
    float red[2 * NW];
    u64 at;      // a place, or an id
    u64 before;  // count or weight in front of a bin
    int bin, n;
};

__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// position in the order: smaller comes first
__device__ __forceinline__ u64 place(float l, int id) { return (u64)(~key_of(l)) << 32 | (uint32_t)id; }
__device__ __forceinline__ float logit_of(u64 place) {
    const uint32_t k = ~(uint32_t)(place >> 32);
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

struct bf16_bits {
    uint16_t u;
};
__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(_Float16 x) { return (float)x; }
__device__ __forceinline__ float widen(bf16_bits x) { return __uint_as_float((uint32_t)x.u << 16); }
__device__ __forceinline__ void narrow(float x, float &t) { t = x; }
__device__ __forceinline__ void narrow(float x, _Float16 &t) { t = (_Float16)x; }
__device__ __forceinline__ void narrow(float x, bf16_bits &t) { t.u = (uint16_t)(__float_as_uint(x) >> 16); }

__device__ __forceinline__ u64 wave_sum64(u64 v) { return lane64(wave_scan64(v), 63); }

// Exclusive prefix sum over the block's threads; total in every thread.
__device__ __forceinline__ u64 block_scan(Shared &sh, u64 v, u64 &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const u64 incl = wave_scan64(v);
    __syncthreads();
    if (lane == 63) sh.wave[wave] = incl;
    __syncthreads();
    u64 run = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < NW; w++) {
        if (w == wave) run = total;
        total += sh.wave[w];
    }
    return run + incl - v;
}

// Sorts one number per thread, n of them (~0 in the threads past n), rising: a
// bitonic network, steps within a wave by lane exchanges.
__device__ __forceinline__ u64 block_sort(Shared &sh, u64 v, int n) {
    const int tid = threadIdx.x;
    for (int size = 2; size < 2 * n; size <<= 1) {
        for (int d = size >> 1; d > 0; d >>= 1) {
            u64 o;
            if (d >= 64) {
                __syncthreads();
                sh.list[tid] = v;
                __syncthreads();
                o = sh.list[tid ^ d];
            } else {
                o = __shfl_xor(v, d);
            }
            const bool up = (tid & size) == 0, low = (tid & d) == 0;
            v = (low == up) == (o < v) ? o : v;
        }
    }
    return v;
}

// 2^S exp((l - max) / T) as a double: t = (l - max) log2e / T = k / 128 + r, k a whole
// number, 2^(k / 128) from the table and the exponent, 2^r by its Taylor series to degree 4
// (|r ln 2| <= 2.71e-3: within 2^-49).
struct Weight {
    float max;
    double c;  // log2e / T
    int S;
    double low;  // -(S + 2): t below it is taken as it, which rounds to weight 0
    __device__ __forceinline__ double value(const Shared &sh, float l) const {
        // the maximum by itself: an infinite one gives NaN, which fmax turns into `low`
        const double t = l == max ? 0.0 : fmax(((double)l - (double)max) * c, low);
        const double k = __builtin_rint(t * 128.0), r = __builtin_fma(k, -1.0 / 128, t);
        const int i = (int)k;
        double p = 0x1.3b2ab6fba4e77p-7;
        p = __builtin_fma(p, r, 0x1.c6b08d704a0bfp-5);
        p = __builtin_fma(p, r, 0x1.ebfbdff82c58ep-3);
        p = __builtin_fma(p, r, 0x1.62e42fefa39efp-1);
        p = __builtin_fma(p, r, 1.0);
        return __builtin_ldexp(sh.exp2_[i & 127] * p, (i >> 7) + S);
    }
    // rounded to a whole number: at most 2^50, so adding 2^52 leaves it in the low bits
    __device__ __forceinline__ static u64 whole(double w) {
        return (u64)(__builtin_bit_cast(long long, w + 0x1p52) - __builtin_bit_cast(long long, 0x1p52));
    }
    __device__ __forceinline__ u64 operator()(const Shared &sh, float l) const { return whole(value(sh, l)); }
};

// Steps of a run: so many that a row has at most RUNS.
__host__ __device__ constexpr int row_q(size_t vocab) { return (int)((vocab + RUNS * 64 * STEP - 1) / (RUNS * 64 * STEP)); }

// The row's logits.  A lane's step is STEP consecutive ids, a run q steps of a wave;
// run run0 + s * NW + wave is the wave's s-th.
template <class T, bool LDS>
struct Row {
    T *copy;  // in LDS: NaN as -inf, -0 as 0, -inf past the end up to a whole number of steps
    int n, q, segs;
    int run0;  // of the block's slice of the row
    // In device memory, as a buffer whose loads return 0 past the row's end (a 16-bit row's end
    // rounded up to a dword).  words: the row starts at a dword.
    __amdgpu_buffer_rsrc_t mem;
    bool words;

    struct alignas(STEP * sizeof(T)) Quad {
        T t[STEP];
    };
    __device__ __forceinline__ void bind(const T *p) {
        words = sizeof(T) == 4 || reinterpret_cast<uintptr_t>(p) % 4 == 0;
        const int bytes = n * (int)sizeof(T);
        mem = __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(p), (short)0, words ? (bytes + 3) & ~3 : bytes, 0x00020000);
    }
    __device__ __forceinline__ Quad load(int id) const {
        const int at = id * (int)sizeof(T);
        if constexpr (sizeof(T) == 4) {
            return __builtin_bit_cast(Quad, __builtin_amdgcn_raw_buffer_load_b128(mem, at, 0, 0));
        } else {
            if (words) return __builtin_bit_cast(Quad, __builtin_amdgcn_raw_buffer_load_b64(mem, at, 0, 0));
            Quad v;
#pragma unroll
            for (int e = 0; e < STEP; e++)
                v.t[e] = __builtin_bit_cast(T, (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(mem, at + 2 * e, 0, 0));
            return v;
        }
    }
    // fmax: NaN as -inf
    __device__ __forceinline__ float clean(int id, T t) const { return id < n ? fmaxf(widen(t) + 0.0f, -INFINITY) : -INFINITY; }
    __device__ __forceinline__ void values(int id, float (&l)[STEP]) const {
        if constexpr (LDS) {
            const Quad v = *reinterpret_cast<const Quad *>(copy + id);
#pragma unroll
            for (int e = 0; e < STEP; e++) l[e] = widen(v.t[e]);
        } else {
            unpack(id, load(id), l);
        }
    }
    __device__ __forceinline__ void unpack(int id, const Quad &v, float (&l)[STEP]) const {
#pragma unroll
        for (int e = 0; e < STEP; e++) l[e] = clean(id + e, v.t[e]);
    }
    __device__ __forceinline__ int first(int run, int j) const { return ((run * q + j) * 64 + (int)(threadIdx.x & 63)) * STEP; }

    // g(run) in front of a run's elements and after the last (the wave's next run), f(id, l) for
    // each STEP of this thread's, l[e] of id + e; -inf past the row's end.  q = 1 in LDS.
    template <class F, class G>
    __device__ __forceinline__ void each(F f, G g) const {
        const int wave = threadIdx.x >> 6;
        float l[STEP];
        if constexpr (LDS) {
            int id = first(run0 + wave, 0);
            for (int s = 0; s < segs; s++, id += NT * STEP) {
                g(run0 + s * NW + wave);
                values(id, l);
                f(id, l);
            }
        } else {
            Quad next = load(first(run0 + wave, 0));
            for (int s = 0; s < segs; s++) {
                const int run = run0 + s * NW + wave;
                g(run);
                for (int j = 0; j < q; j++) {
                    const int id = first(run, j);
                    unpack(id, next, l);
                    next = load(j + 1 < q ? first(run, j + 1) : first(run + NW, 0));
                    f(id, l);
                }
            }
        }
        g(run0 + segs * NW + wave);
    }
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        each(f, [](int) {});
    }
};

// f is between 2^-118 and 2^100, so that the product is not lost: past the range
// it is the last bin, and logits of a range below 2^-88 share the first.  NaN (an infinite maximum's
// own) is bin 0, as v_cvt_i32_f32 has it; it saturates for large values.
struct Bins {
    float max, f;
    __device__ __forceinline__ int of(float l) const {
        const float x = (max - l) * f;
        int b;
        asm("v_cvt_i32_f32 %0, %1" : "=v"(b) : "v"(x));
        return min(b, BINS - 1);
    }
    // not above any logit of the bins 0 .. b: the bin's edge, a 2^-20 of the way to it and a
    // 2^-20 of the maximum lower, far more than the roundings of `of` and of this
    __device__ __forceinline__ float floor(int b) const {
        const float away = (float)(b + 1) / f * (1.0f + 0x1p-20f), slack = fabsf(max) * 0x1p-20f;
        return b >= BINS - 1 || !(fabsf(max) < __builtin_inff()) ? -INFINITY : (max - away) - slack;
    }
};

// The end of what is kept, in the order (l falling, id rising).
struct Keep {
    float l;
    int id;
    // (int, and | and &: no branches)
    __device__ __forceinline__ int has(float x, int i) const { return int(x > l) | (int(x == l) & int(i <= id)); }
};
__device__ __forceinline__ Keep keep_to(u64 place) { return {logit_of(place), (int)(uint32_t)place}; }

// The bin that holds the n-th of the threads' elements, one each where `is`; -1: they are fewer.
__device__ __forceinline__ int nth_bin(Shared &sh, int bin, bool is, int n) {
    const int tid = threadIdx.x;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; i++) sh.hist[i * NT + tid] = 0;
    if (tid == 0) {
        sh.bin = -1;
        sh.n = 0;
    }
    __syncthreads();
    if (is) atomicAdd(&sh.hist[bin], 1ull);
    __syncthreads();
    u64 h[PER], mine = 0, total;
#pragma unroll
    for (int i = 0; i < PER; i++) mine += h[i] = sh.hist[PER * tid + i];
    u64 run = block_scan(sh, mine, total);
#pragma unroll
    for (int i = 0; i < PER; i++) {
        if (run < (u64)n && run + h[i] >= (u64)n) sh.bin = PER * tid + i;
        run += h[i];
    }
    __syncthreads();  // the histogram is read: its room is the list's
    return sh.bin;
}

// Puts the places of the kept elements of bin `bin`, or of all bins up to it, into
// sh.list, in any order; their number (sh.n, 0 before): above NT if they are more.
template <class R>
__device__ __forceinline__ int collect(Shared &sh, const R &row, const Bins &bins, Keep keep, int bin, bool all) {
    const int lane = threadIdx.x & 63;
    const float low = bins.floor(bin);
    bool full = false;
    row.each([&](int id, const float(&l)[STEP]) {
        if (full || !__ballot(fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3])) >= low)) return;
#pragma unroll
        for (int e = 0; e < STEP; e++) {
            const int b = bins.of(l[e]);
            const bool take = int(all ? b <= bin : b == bin) & keep.has(l[e], id + e);
            const u64 m = __ballot(take);
            if (!m) continue;
            int at = 0;  // one addition for the wave
            if (lane == 0) at = atomicAdd(&sh.n, (int)__popcll(m));
            at = __builtin_amdgcn_readfirstlane(at);
            full = at + (int)__popcll(m) > NT;
            at += __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
            if (take && at < NT) sh.list[at] = place(l[e], id + e);
        }
    });
    __syncthreads();
    return sh.n;
}

// What is kept: everything up to `keep`, or of the n >= 0 places in sh.list what cut() was asked for.
// want: the weight that the kept ones have to reach (a list of cut<true>).
struct Kept {
    Keep keep;
    int n;
    double want;
};

// The last kept one of a bin's n elements, v of thread tid by place: where the sum passes `want`.
template <bool WEIGHTS>
__device__ __forceinline__ Keep end_of(Shared &sh, const Weight &W, u64 v, int n, u64 before, double want) {
    const int tid = threadIdx.x;
    const u64 w = tid < n ? (WEIGHTS ? W(sh, logit_of(v)) : 1) : 0;
    u64 sum;
    const u64 ahead = before + block_scan(sh, w, sum);
    if (tid < n && (double)ahead < want && (double)(ahead + w) >= want) sh.at = v;
    __syncthreads();
    return keep_to(sh.at);
}

// Keep only a prefix: the first `count` elements (WEIGHTS false), or the shortest one whose
// weights reach the share `p` of all kept ones'.  limited: the last bin holds only
// weights of 0.  Where the result is a list, it holds more: the cut is still to be made.
// FIRST: everything finite is kept so far.
template <bool WEIGHTS, bool FIRST, class R>
__device__ __forceinline__ void cut(Shared &sh, const R &row, const Bins &bins, const Weight &W, Kept &K, u64 count, double p,
                                    bool limited) {
    const int tid = threadIdx.x;
    const Keep keep = K.keep;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; i++) sh.hist[i * NT + tid] = 0;
    if (tid == 0) {
        sh.bin = -1;
        sh.n = 0;
    }
    __syncthreads();
    row.each([&](int id, const float(&l)[STEP]) {
        if (!FIRST && !__ballot(fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3])) >= keep.l)) return;
#pragma unroll
        for (int e = 0; e < STEP; e++)
            if (FIRST ? l[e] > -INFINITY : keep.has(l[e], id + e)) atomicAdd(&sh.hist[bins.of(l[e])], WEIGHTS ? W(sh, l[e]) : 1ull);
    });
    __syncthreads();
    u64 h[PER], mine = 0, total;
#pragma unroll
    for (int i = 0; i < PER; i++) mine += h[i] = sh.hist[PER * tid + i];
    u64 run = block_scan(sh, mine, total);
    const double want = WEIGHTS ? p * (double)total : (double)count;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        if ((double)run < want && (double)(run + h[i]) >= want) {  // one bin of the row
            sh.bin = PER * tid + i;
            sh.before = run;
            sh.at = run + h[i];
        }
        run += h[i];
    }
    __syncthreads();  // the histogram is read: its room is the list's
    const int bin = sh.bin;
    if (bin < 0 || (limited && bin == BINS - 1)) return;  // fewer elements than wanted, or only weights of 0 beyond
    u64 before = sh.before;

    // the elements of the bins up to this one, of this one alone if they are too many
    bool all = WEIGHTS || sh.at <= (u64)NT;
    int n = collect(sh, row, bins, keep, bin, all);
    if (n > NT && all) {
        all = false;
        __syncthreads();
        if (tid == 0) sh.n = 0;
        __syncthreads();
        n = collect(sh, row, bins, keep, bin, false);
    }
    if (all && n <= NT) {
        K.n = n;
        if (WEIGHTS) K.want = want;
        return;
    }
    if (n <= NT) {
        const u64 v = block_sort(sh, tid < n ? sh.list[tid] : ~0ull, n);
        K.keep = end_of<WEIGHTS>(sh, W, v, n, before, want);
        return;
    }
    // radix descent over the places
    u64 prefix = 0, acc = before;
    for (int s = 56; s >= 0; s -= 8) {
        __syncthreads();
        if (tid < 256) sh.hist[tid] = 0;
        __syncthreads();
        row.each([&](int id, const float(&l)[STEP]) {
#pragma unroll
            for (int e = 0; e < STEP; e++) {
                const u64 v = place(l[e], id + e);
                if (bins.of(l[e]) == bin && keep.has(l[e], id + e) && (s == 56 || v >> (s + 8) == prefix >> (s + 8)))
                    atomicAdd(&sh.hist[(v >> s) & 255u], WEIGHTS ? W(sh, l[e]) : 1ull);
            }
        });
        __syncthreads();
        const u64 c = tid < 256 ? sh.hist[tid] : 0;
        u64 sum;
        const u64 ahead = acc + block_scan(sh, c, sum);
        if ((double)ahead < want && (double)(ahead + c) >= want) {
            sh.at = prefix | (u64)tid << s;
            sh.before = ahead;
        }
        __syncthreads();
        prefix = sh.at;
        acc = sh.before;
    }
    K.keep = keep_to(prefix);
}

// floor(u total), u brought into [0, 1)
__device__ __forceinline__ u64 target(float u, u64 total) {
    u = u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f;
    const u64 t = (u64)((double)u * (double)total);
    return t < total ? t : total - 1;
}

// A row's filters, and what follows from its largest and smallest logit.
struct Filters {
    float temp, min_p, top_p;
    int top_k;
    bool by_count, by_weight, limited;  // limited: the last bin holds only weights of 0
    Weight W;
    Bins bins;
    double least;
    __device__ __forceinline__ void read(const SampleRows &R, int r) {
        temp = R.temperature ? R.temperature[r] : 1.0f;
        min_p = R.min_p ? R.min_p[r] : 0.0f;
        top_p = R.top_p ? R.top_p[r] : 1.0f;
        top_k = R.top_k ? R.top_k[r] : 0;
        by_count = top_k > 0 && (size_t)top_k < R.vocab;
        by_weight = top_p < 1.0f;
    }
    __device__ __forceinline__ bool few() const { return by_count && top_k <= NT; }
    // the most likely token
    __device__ __forceinline__ bool greedy() const { return !(temp > 0.0f) || min_p > 1.0f || top_p <= 0.0f || top_k == 1; }
    __device__ __forceinline__ void range(float hi, float lo, int S) {
        W.max = hi;
        W.c = 1.4426950408889634 / (double)temp;
        W.S = S;
        W.low = -(double)(S + 2);
        // Bins over the logits that have weight, or all of them if those span less.
        const double span = (double)(S + 3) / W.c, wide = (double)hi - (double)lo;
        limited = !(wide < span);
        bins = {hi, (float)fmin(fmax((double)BINS / (limited ? span : wide), 0x1p-118), 0x1p100)};
        least = min_p > 0.0f ? __builtin_ldexp((double)min_p, S) : 0.0;
    }
};

// The largest and the smallest finite logit of this thread's (in all, of the row or
// slice); id: the lowest of the largest (ID).  A row kept in LDS is copied there.
template <bool ID, class T, bool LDS>
__device__ __forceinline__ void extremes(const Row<T, LDS> &row, float &hi, float &lo, int &id_hi) {
    const int tid = threadIdx.x;
    hi = -INFINITY;
    lo = INFINITY;
    id_hi = INT_MAX;
    constexpr int U = ID ? 4 : 8;
    using Quad = typename Row<T, LDS>::Quad;
    const int steps = row.segs * row.q, id0 = row.run0 * row.q * (64 * STEP);
    auto id_of = [&](int step) { return !ID || step < steps ? id0 + (step * NT + tid) * STEP : row.n; };  // past the row's end: nothing
    for (int s = 0; s < steps; s += U) {
        Quad v[U];
#pragma unroll
        for (int k = 0; k < U; k++) v[k] = row.load(id_of(s + k));
#pragma unroll
        for (int k = 0; k < U; k++) {
            const int id = id_of(s + k);
            float l[STEP];
            row.unpack(id, v[k], l);
            Quad c;
#pragma unroll
            for (int e = 0; e < STEP; e++) {
                if constexpr (ID) id_hi = l[e] > hi ? id + e : id_hi;
                hi = fmaxf(hi, l[e]);
                lo = fminf(lo, l[e] > -INFINITY ? l[e] : INFINITY);
                narrow(l[e], c.t[e]);
            }
            if constexpr (LDS)
                if (s + k < steps) *reinterpret_cast<Quad *>(row.copy + id) = c;
        }
    }
}

template <class T, bool LDS>
__device__ __forceinline__ void bind_row(Row<T, LDS> &row, const SampleRows &R, int r, T *copy) {
    row.copy = copy;
    row.n = (int)R.vocab;
    row.q = LDS ? 1 : row_q(R.vocab);
    row.segs = (row.n + row.q * NT * STEP - 1) / (row.q * NT * STEP);
    row.run0 = 0;
    row.bind(static_cast<const T *>(R.logits) + (size_t)r * R.stride);
}

// ---- a row over several blocks --------------------------------------------
//
// Few long rows leave most CUs without work in a block per row, so slices of
// whole runs get a block each in three kernels: the slices' largest and smallest
// logits; their histograms, added up in device memory; the elements of the bin
// where the kept ones end (of all bins up to it, if they are few) and
// the runs' sums of what is kept for certain.  k_sample goes on from there with a
// block per row.  Rows with top-p and a top_k above NT, and lists of
// more than NT elements, are left to its own passes.
//
// 64 x 128000 f32 with top-p: 8 + 20 + 22 + 16 us, the gathering bound by VALU issue (10 M
// instructions, 60 % of its cycles; 16 logits per lane, a third of the instructions in front of
// them) and by its chain of dependent loads: 4 f64 operations fewer per logit, or half the
// blocks, leave its time as it is.  A block per row took 138.  Whole calls, a
// block per row against this (us):
//                      top-p 0.9  none       top-k 40, top-p  top-k 5000, top-p
//   64 x 128000 f32     133   62   61   33    27   35          174  180
//   128                 140   87   64   52    32   43          180  187
//   200                 147  130   71   82    38   53          186  195
//   1 x 30000 (in LDS)   34   25   17   15    12   20           49   61
// The filters' values are not known on the host, so rows that fit LDS and more than 128 of
// them stay with a block per row, also in the calls without a top_k array (which the
// host does see) that the table has faster over several blocks.
constexpr int MAX_SLICES = 64;
struct SplitRow {
    u64 hist[BINS], list[NT], runs[RUNS];
    struct {
        float hi, lo;
        int id;
    } slice[MAX_SLICES];
    int n;
};
constexpr int SPLIT_ROWS = 128, SPLIT_BLOCKS = 512;  // rows of a split call; blocks to make of them (two per CU)
struct Split {
    SplitRow *rows;
    float *tops;       // [rows][slices][NT]: the largest logits of the slices' threads
    int slices, runs;  // runs of a slice: a multiple of NW
    __device__ float &top() const { return tops[((size_t)blockIdx.y * slices + blockIdx.x) * NT + threadIdx.x]; }
};

template <class T>
__device__ __forceinline__ Row<T, false> slice_of(const SampleRows &R, const Split &P) {
    Row<T, false> row;
    bind_row<T, false>(row, R, blockIdx.y, nullptr);
    row.run0 = blockIdx.x * P.runs;
    row.segs = P.runs / NW;
    return row;
}

__device__ __forceinline__ void join_slices(const SplitRow &W, const Split &P, float &hi, float &lo, int &id) {
    const int lane = threadIdx.x & 63;
    const bool is = lane < P.slices;
    const float h = is ? W.slice[lane].hi : -INFINITY;
    hi = wave_max(h);
    lo = -wave_max(is ? -W.slice[lane].lo : -INFINITY);
    const u64 m = __ballot(is && h == hi);  // the first slice of these
    id = m ? W.slice[__builtin_ctzll(m)].id : -1;
}

template <class T>
__global__ __launch_bounds__(NT, 8) void k_sample_extremes(SampleRows R, Split P) {
    __shared__ float red[2 * NW];
    __shared__ int first;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    SplitRow &W = P.rows[blockIdx.y];
    for (int i = blockIdx.x * NT + tid; i < BINS; i += P.slices * NT) W.hist[i] = 0;
    if (blockIdx.x == 0 && tid == 0) W.n = 0;
    float hi, lo;
    int id;
    extremes<true>(slice_of<T>(R, P), hi, lo, id);
    const float own = hi;
    P.top() = own;
    hi = wave_max(hi);
    lo = -wave_max(-lo);
    if (lane == 0) {
        red[wave] = hi;
        red[NW + wave] = lo;
    }
    if (tid == 0) first = INT_MAX;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; w++) {
        hi = fmaxf(hi, red[w]);
        lo = fminf(lo, red[NW + w]);
    }
    if (own == hi && hi > -INFINITY) atomicMin(&first, id);
    __syncthreads();
    if (tid == 0) {
        W.slice[blockIdx.x].hi = hi;
        W.slice[blockIdx.x].lo = lo;
        W.slice[blockIdx.x].id = first;
    }
}

__device__ __forceinline__ bool split_slow(const Filters &f) { return f.by_count && f.by_weight && f.top_k > NT; }

template <class T>
__global__ __launch_bounds__(NT, 8) void k_sample_bins(SampleRows R, Split P, int S) {
    __shared__ Shared sh;
    const int tid = threadIdx.x;
    SplitRow &W = P.rows[blockIdx.y];
    Filters f;
    f.read(R, blockIdx.y);
    float hi, lo;
    int id_hi;
    join_slices(W, P, hi, lo, id_hi);
    if (hi == -INFINITY || f.greedy() || !(f.by_count || f.by_weight) || split_slow(f)) return;
    f.range(hi, lo, S);
    if (tid < 128) sh.exp2_[tid] = exp2((double)tid / 128);
#pragma unroll
    for (int i = 0; i < PER; i++) sh.hist[i * NT + tid] = 0;
    __syncthreads();
    if (f.few()) {
        const float l = P.top();
        if (l > -INFINITY) atomicAdd(&sh.hist[f.bins.of(l)], 1ull);
    } else slice_of<T>(R, P).each([&](int, const float(&l)[STEP]) {
#pragma unroll
        for (int e = 0; e < STEP; e++)
            if (l[e] > -INFINITY) atomicAdd(&sh.hist[f.bins.of(l[e])], f.by_count ? 1ull : f.W(sh, l[e]));
    });
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int b = i * NT + tid;
        if (sh.hist[b]) atomicAdd(&W.hist[b], sh.hist[b]);
    }
}

// How a split row goes on, from its histogram; the same in every block.  It holds
// the weights, or with top-k the counts; for a small top_k those of the threads'
// largest logits alone: at least top_k logits are as large as the top_k-th of these, and
// not many more where the ids' order is no order of l.
struct Plan {
    enum { EVERY, LIST, BIN, SLOW } mode;  // no cut; the list of the bins 0 .. bin, or of `bin` alone; k_sample's own passes
    int bin;
    u64 before;
    double want;
};
__device__ __forceinline__ Plan plan(Shared &sh, const SplitRow &W, const Filters &f) {
    if (!(f.by_count || f.by_weight)) return {Plan::EVERY, BINS, 0, 0.0};
    if (split_slow(f)) return {Plan::SLOW, BINS, 0, 0.0};
    const int tid = threadIdx.x;
    u64 h[PER], mine = 0, total;
#pragma unroll
    for (int i = 0; i < PER; i++) mine += h[i] = W.hist[PER * tid + i];
    if (tid == 0) sh.bin = -1;
    u64 run = block_scan(sh, mine, total);
    const double want = f.by_count ? (double)f.top_k : (double)f.top_p * (double)total;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        if ((double)run < want && (double)(run + h[i]) >= want) {
            sh.bin = PER * tid + i;
            sh.before = run;
            sh.at = run + h[i];
        }
        run += h[i];
    }
    __syncthreads();
    const bool cut = sh.bin >= 0 && !(f.limited && sh.bin == BINS - 1);
    if (f.few()) return {cut ? Plan::LIST : Plan::SLOW, cut ? sh.bin : BINS, 0, 0.0};
    if (!cut) return {Plan::EVERY, BINS, 0, 0.0};
    return {Plan::BIN, sh.bin, sh.before, want};
}

template <class T>
__global__ __launch_bounds__(NT, 8) void k_sample_gather(SampleRows R, Split P, int S) {
    __shared__ Shared sh;
    const int tid = threadIdx.x, lane = tid & 63;
    SplitRow &W = P.rows[blockIdx.y];
    Filters f;
    f.read(R, blockIdx.y);
    float hi, lo;
    int id_hi;
    join_slices(W, P, hi, lo, id_hi);
    if (hi == -INFINITY || f.greedy()) return;
    f.range(hi, lo, S);
    if (tid < 128) sh.exp2_[tid] = exp2((double)tid / 128);
    const Plan p = plan(sh, W, f);
    if (p.mode == Plan::SLOW) return;
    __syncthreads();
    if (tid == 0) sh.n = 0;
    __syncthreads();
    const Row<T, false> row = slice_of<T>(R, P);
    const float low = f.bins.floor(p.bin);
    const bool sums = p.mode != Plan::LIST;
    u64 sum = 0;
    int at = -1;
    row.each(
        [&](int id, const float(&l)[STEP]) {
            if (!__ballot(fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3])) >= low)) return;
#pragma unroll
            for (int e = 0; e < STEP; e++) {
                const int b = l[e] > -INFINITY ? f.bins.of(l[e]) : BINS;
                const bool take = sums ? b == p.bin && b < BINS : b <= p.bin;
                const u64 m = __ballot(take);
                if (m) {
                    int to = 0;
                    if (lane == 0) to = atomicAdd(&sh.n, (int)__popcll(m));
                    to = __builtin_amdgcn_readfirstlane(to);
                    to += __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
                    if (take && to < NT) sh.list[to] = place(l[e], id + e);
                }
                if (sums && b < p.bin) {
                    const double w = f.W.value(sh, l[e]);
                    sum += w >= f.least ? Weight::whole(w) : 0;
                }
            }
        },
        [&](int run) {
            if (sums && at >= 0) {
                sum = wave_sum64(sum);
                if (lane == 0 && at < RUNS) W.runs[at] = sum;
            }
            sum = 0;
            at = run;
        });
    __syncthreads();
    const int n = sh.n;
    if (!n) return;
    if (tid == 0) sh.bin = atomicAdd(&W.n, n);
    __syncthreads();
    const int to = sh.bin + tid;
    if (tid < min(n, NT) && to < NT) W.list[to] = sh.list[tid];
}

// ---- a block per row ------------------------------------------------------

// SPLIT: after the kernels above.
template <class T, bool LDS, bool SPLIT>
__global__ __launch_bounds__(NT, LDS ? 8 : 4) void k_sample(SampleRows R, Split P, int S) {
    extern __shared__ __align__(16) unsigned char lds[];
    Shared &sh = *reinterpret_cast<Shared *>(lds);
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    Row<T, LDS> row;
    bind_row(row, R, r, reinterpret_cast<T *>(lds + sizeof(Shared)));
    Filters f;
    f.read(R, r);
    const float u = R.u[r];
    float hi, lo, hi_t = 0.0f;  // the row's; this thread's
    int id_hi;
    if (tid < 128) sh.exp2_[tid] = exp2((double)tid / 128);
    if constexpr (SPLIT) {
        join_slices(P.rows[r], P, hi, lo, id_hi);
        __syncthreads();
    } else {
        extremes<false>(row, hi, lo, id_hi);
        hi_t = hi;
        hi = wave_max(hi);
        lo = -wave_max(-lo);
        if (lane == 0) {
            sh.red[wave] = hi;
            sh.red[NW + wave] = lo;
        }
        if (tid == 0) sh.at = ~0ull;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NW; w++) {
            hi = fmaxf(hi, sh.red[w]);
            lo = fminf(lo, sh.red[NW + w]);
        }
    }
    auto put = [&](int id, float prob) {
        R.ids[r] = id;
        if (R.probs) R.probs[r] = prob;
    };
    if (hi == -INFINITY) {  // nothing to draw
        if (tid == 0) put(-1, 0.0f);
        return;
    }
    if (f.greedy()) {
        if constexpr (SPLIT) {
            if (tid == 0) put(id_hi, 1.0f);
        } else {
            u64 at = ~0ull;
            row.each([&](int id, const float(&l)[STEP]) {
#pragma unroll
                for (int e = STEP - 1; e >= 0; e--) at = l[e] == hi && (u64)id < at ? (u64)(id + e) : at;
            });
            if (at != ~0ull) atomicMin(&sh.at, at);
            __syncthreads();
            if (tid == 0) put((int)sh.at, 1.0f);
        }
        return;
    }
    f.range(hi, lo, S);
    const Weight &W = f.W;
    const Bins &bins = f.bins;
    const double least = f.least;
    const float top_p = f.top_p;
    const int top_k = f.top_k;
    const bool by_weight = f.by_weight, limited = f.limited;

    Kept K{{-INFINITY, -1}, -1, 0.0};  // everything finite
    int most = NT;         // a list of more than top_k elements so far: top_k
    bool summed = false;   // the runs' sums are known but for the places in sh.list
    bool by_count = f.by_count, left = by_count || by_weight;  // left: filters that are still to be applied
    u64 last = ~0ull;      // thread tid's place of that list
    if constexpr (SPLIT) {
        const SplitRow &X = P.rows[r];
        const Plan p = plan(sh, X, f);
        if (p.mode == Plan::EVERY) {
            left = false;
            summed = true;
        } else if (p.mode != Plan::SLOW && X.n <= NT) {
            __syncthreads();
            const u64 v = tid < X.n ? X.list[tid] : ~0ull;
            left = false;
            if (p.mode == Plan::LIST) {
                sh.list[tid] = v;
                K.n = X.n;
                most = top_k;
                __syncthreads();
            } else {
                last = block_sort(sh, v, X.n);
                K.keep = by_weight ? end_of<true>(sh, W, last, X.n, p.before, p.want)
                                   : end_of<false>(sh, W, last, X.n, p.before, p.want);
                summed = true;
            }
        }
    }
    if (left) {
        if (!SPLIT && by_count && top_k <= NT) {
            // At least top_k logits are as large as the top_k-th largest of the threads'
            // own maxima, and not many more where the ids' order is no order of l.
            const int bin = nth_bin(sh, bins.of(hi_t), hi_t > -INFINITY, top_k);
            if (bin >= 0 && !(limited && bin == BINS - 1)) {
                const int n = collect(sh, row, bins, K.keep, bin, true);
                if (n <= NT) K.n = n;
            }
        }
        if (by_count && K.n < 0) cut<false, true>(sh, row, bins, W, K, (u64)top_k, 0.0, limited);
        if (K.n >= 0) most = top_k;
        if (by_weight && K.n < 0) {
            if (by_count) cut<true, false>(sh, row, bins, W, K, 0, (double)top_p, limited);
            else cut<true, true>(sh, row, bins, W, K, 0, (double)top_p, limited);
        }
    }

    if (K.n >= 0 && K.n <= 64) {  // a list of one wave: ranks and sums by comparing all pairs
        if (wave != 0) return;
        const bool is = lane < K.n;
        const u64 v = is ? sh.list[lane] : ~0ull;
        const double x = is ? W.value(sh, logit_of(v)) : 0.0;
        u64 w = is ? Weight::whole(x) : 0;
        // sums over the elements in front of this lane's, weights through LDS as broadcasts
        auto in_front = [&](auto less, int &count) {
            sh.list[lane] = v;
            sh.weight[lane] = w;
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            u64 sum = 0;
            count = 0;
            for (int j = 0; j < K.n; j += 8) {  // places past the list's end are ~0, their weights 0
                u64 o[8], ow[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    o[e] = sh.list[j + e];
                    ow[e] = sh.weight[j + e];
                }
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const bool l = less(o[e]);
                    count += l;
                    sum += l ? ow[e] : 0;
                }
            }
            return sum;
        };
        int rank;
        u64 ahead = in_front([&](u64 o) { return o < v; }, rank);
        bool in = is && rank < most;
        const u64 all = wave_sum64(in ? w : 0);  // every lane takes part
        if (by_weight) in = in && (double)ahead < (K.want > 0.0 ? K.want : (double)top_p * (double)all);
        in = in && (x >= least);
        w = in ? w : 0;
        const u64 total = wave_sum64(w), want = target(u, total);
        ahead = in_front([&](u64 o) { return (uint32_t)o < (uint32_t)v; }, rank);
        if (want >= ahead && want < ahead + w) put((int)(uint32_t)v, (float)((double)w / (double)total));
        return;
    }
    if (K.n >= 0) {  // a longer one: sorted by place for the filters, by id for the draw
        const u64 v = block_sort(sh, tid < K.n ? sh.list[tid] : ~0ull, K.n);
        const bool is = tid < K.n && tid < most;
        const double x = is ? W.value(sh, logit_of(v)) : 0.0;
        u64 w = is ? Weight::whole(x) : 0, total;
        bool in = is;
        if (by_weight) {
            const u64 ahead = block_scan(sh, w, total);
            in = in && (double)ahead < (K.want > 0.0 ? K.want : (double)top_p * (double)total);
        }
        in = in && (x >= least);
        __syncthreads();
        sh.weight[tid] = w;
        const u64 by_id = block_sort(sh, in ? (v & 0xFFFFFFFFull) << 10 | (u64)tid : ~0ull, K.n);
        __syncthreads();
        w = by_id != ~0ull ? sh.weight[by_id & (NT - 1)] : 0;
        const u64 ahead = block_scan(sh, w, total), want = target(u, total);
        if (want >= ahead && want < ahead + w) put((int)(by_id >> 10), (float)((double)w / (double)total));
        return;
    }

    // the runs' kept weights
    const Keep keep = K.keep;
    auto kept = [&](int id, float l) -> u64 {
        const double w = W.value(sh, l);
        return (keep.has(l, id) & int(w >= least)) ? Weight::whole(w) : 0;
    };
    __syncthreads();
    if (SPLIT && summed) {
        sh.sums[tid] = tid < P.slices * P.runs ? P.rows[r].runs[tid] : 0;
        __syncthreads();
        if (last != ~0ull) {
            const int id = (int)(uint32_t)last;
            const u64 w = kept(id, logit_of(last));
            if (w) atomicAdd(&sh.sums[id / (row.q * 64 * STEP)], w);
        }
    } else {
        sh.sums[tid] = 0;
        __syncthreads();
        u64 sum = 0;
        int at = -1;
        row.each(
            [&](int id, const float(&l)[STEP]) {
                if (!__ballot(fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3])) >= keep.l)) return;
#pragma unroll
                for (int e = 0; e < STEP; e++)
                    if (__ballot(keep.has(l[e], id + e))) sum += kept(id + e, l[e]);
            },
            [&](int run) {
                if (__ballot(sum != 0)) {
                    sum = wave_sum64(sum);
                    if (lane == 0) sh.sums[at] = sum;
                }
                sum = 0;
                at = run;
            });
    }
    __syncthreads();
    static_assert(RUNS == NT, "a thread per run");
    const u64 mine = sh.sums[tid];
    u64 total;
    const u64 ahead = block_scan(sh, mine, total), want = target(u, total);
    if (want >= ahead && want < ahead + mine) {
        sh.bin = tid;
        sh.before = ahead;
    }
    __syncthreads();
    const int run = sh.bin;
    if (wave != run % NW) return;
    u64 acc = sh.before;
    for (int j = 0; j < row.q; j++) {
        const int id = row.first(run, j);
        float l[STEP];
        row.values(id, l);
        u64 w[STEP], c = 0;
#pragma unroll
        for (int e = 0; e < STEP; e++) c += w[e] = kept(id + e, l[e]);
        const u64 incl = wave_scan64(c);
        const u64 hit = __ballot(acc + incl > want);
        if (hit) {
            if (lane == __builtin_ctzll(hit)) {
                u64 run_sum = acc + incl - c;
                int e = 0;
                for (; e < STEP - 1 && run_sum + w[e] <= want; e++) run_sum += w[e];
                put(id + e, (float)((double)w[e] / (double)total));
            }
            return;
        }
        acc += lane64(incl, 63);
    }
}

// LDS of a row kept there: up to a whole number of steps of the block.
template <class T>
size_t row_lds(size_t vocab) {
    return (vocab + NT * STEP - 1) / (NT * STEP) * (NT * STEP) * sizeof(T);
}

}  // namespace

hipError_t sample_prepare_lds() {
    for (const void *fn : {(const void *)k_sample<float, true, false>, (const void *)k_sample<_Float16, true, false>,
                           (const void *)k_sample<bf16_bits, true, false>}) {
        const hipError_t e = ensure_lds_limit(fn, ROW_BYTES + (int)sizeof(Shared));
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

size_t sample_split_bytes() { return SPLIT_ROWS * sizeof(SplitRow) + (size_t)SPLIT_BLOCKS * NT * sizeof(float); }

hipError_t launch_sample(const SampleRows &r, hipStream_t s) {
    if (!r.n_rows) return hipSuccess;
    int lg = 0;
    while ((1ull << lg) < r.vocab) lg++;
    const int S = 62 - lg < 50 ? 62 - lg : 50;
    auto go = [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const size_t lds = row_lds<T>(r.vocab);
        const dim3 rows((unsigned)r.n_rows);
        Split p{static_cast<SplitRow *>(r.split), nullptr, 0, 0};
        if (lds <= ROW_BYTES) {
            hipLaunchKernelGGL((k_sample<T, true, false>), rows, dim3(NT), sizeof(Shared) + lds, s, r, p, S);
        } else if (r.n_rows > SPLIT_ROWS) {
            hipLaunchKernelGGL((k_sample<T, false, false>), rows, dim3(NT), sizeof(Shared), s, r, p, S);
        } else {
            const int runs = (int)((r.vocab + (size_t)row_q(r.vocab) * 64 * STEP - 1) / ((size_t)row_q(r.vocab) * 64 * STEP));
            const int want = std::min(MAX_SLICES, std::max(1, SPLIT_BLOCKS / (int)r.n_rows));
            p.runs = ((runs + want - 1) / want + NW - 1) / NW * NW;
            p.slices = (runs + p.runs - 1) / p.runs;
            p.tops = reinterpret_cast<float *>(p.rows + SPLIT_ROWS);
            const dim3 grid((unsigned)p.slices, (unsigned)r.n_rows);
            hipLaunchKernelGGL((k_sample_extremes<T>), grid, dim3(NT), 0, s, r, p);
            hipLaunchKernelGGL((k_sample_bins<T>), grid, dim3(NT), 0, s, r, p, S);
            hipLaunchKernelGGL((k_sample_gather<T>), grid, dim3(NT), 0, s, r, p, S);
            hipLaunchKernelGGL((k_sample<T, false, true>), rows, dim3(NT), sizeof(Shared), s, r, p, S);
        }
    };
    if (r.dtype == T_F32) go((float *)nullptr);
    else if (r.dtype == T_F16) go((_Float16 *)nullptr);
    else go((bf16_bits *)nullptr);
    return hipGetLastError();
}

}  // namespace rce_qmm
