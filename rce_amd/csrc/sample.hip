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
// where a list follows, and two more where none does.
#include "kv_cache.h"
#include "lds_limit.h"

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

// v of the lane CTRL names (0 where there is none, or for rows outside ROWS).
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ u64 dpp64(u64 v) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xF, false);
    return (u64)hi << 32 | lo;
}
// Inclusive prefix sum over the lanes: within rows of 16 (shifts by 1, 2, 4, 8), then
// lane 15 of rows 0 and 2 into rows 1 and 3, then lane 31 into rows 2 and 3.
__device__ __forceinline__ u64 wave_scan64(u64 v) {
    v += dpp64<0x111>(v);
    v += dpp64<0x112>(v);
    v += dpp64<0x114>(v);
    v += dpp64<0x118>(v);
    v += dpp64<0x142, 0xA>(v);
    v += dpp64<0x143, 0xC>(v);
    return v;
}
__device__ __forceinline__ u64 lane64(u64 v, int l) {
    return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), l) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, l);
}
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

// The row's logits.  A lane's step is STEP consecutive ids, a run q steps of a wave;
// run s * NW + wave is the wave's s-th.
template <class T, bool LDS>
struct Row {
    T *copy;  // in LDS: NaN as -inf, -0 as 0, -inf past the end up to a whole number of steps
    int n, q, segs;
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
            int id = first(wave, 0);
            for (int s = 0; s < segs; s++, id += NT * STEP) {
                g(s * NW + wave);
                values(id, l);
                f(id, l);
            }
        } else {
            Quad next = load(first(wave, 0));
            for (int s = 0; s < segs; s++) {
                const int run = s * NW + wave;
                g(run);
                for (int j = 0; j < q; j++) {
                    const int id = first(run, j);
                    unpack(id, next, l);
                    next = load(j + 1 < q ? first(run, j + 1) : first(run + NW, 0));
                    f(id, l);
                }
            }
        }
        g(segs * NW + wave);
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
        const u64 w = tid < n ? (WEIGHTS ? W(sh, logit_of(v)) : 1) : 0;
        u64 sum;
        const u64 ahead = before + block_scan(sh, w, sum);
        if (tid < n && (double)ahead < want && (double)(ahead + w) >= want) sh.at = v;
        __syncthreads();
        K.keep = keep_to(sh.at);
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

template <class T, bool LDS>
__global__ __launch_bounds__(NT, LDS ? 8 : 4) void k_sample(SampleRows R, int S) {
    extern __shared__ __align__(16) unsigned char lds[];
    Shared &sh = *reinterpret_cast<Shared *>(lds);
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    Row<T, LDS> row;
    row.copy = reinterpret_cast<T *>(lds + sizeof(Shared));
    row.n = (int)R.vocab;
    row.q = LDS ? 1 : (row.n + RUNS * 64 * STEP - 1) / (RUNS * 64 * STEP);
    row.segs = (row.n + row.q * NT * STEP - 1) / (row.q * NT * STEP);
    row.bind(static_cast<const T *>(R.logits) + (size_t)r * R.stride);
    const float temp = R.temperature ? R.temperature[r] : 1.0f;
    const float min_p = R.min_p ? R.min_p[r] : 0.0f;
    const float top_p = R.top_p ? R.top_p[r] : 1.0f;
    const int top_k = R.top_k ? R.top_k[r] : 0;
    const float u = R.u[r];

    // the largest and the smallest finite logit
    float hi = -INFINITY, lo = INFINITY;
    constexpr int U = 8;
    using Quad = typename Row<T, LDS>::Quad;
    const int steps = row.segs * row.q;
    for (int s = 0; s < steps; s += U) {
        Quad v[U];
#pragma unroll
        for (int k = 0; k < U; k++) v[k] = row.load(((s + k) * NT + tid) * STEP);
#pragma unroll
        for (int k = 0; k < U; k++) {
            const int id = ((s + k) * NT + tid) * STEP;
            float l[STEP];
            row.unpack(id, v[k], l);
            Quad c;
#pragma unroll
            for (int e = 0; e < STEP; e++) {
                hi = fmaxf(hi, l[e]);
                lo = fminf(lo, l[e] > -INFINITY ? l[e] : INFINITY);
                narrow(l[e], c.t[e]);
            }
            if constexpr (LDS)
                if (s + k < steps) *reinterpret_cast<Quad *>(row.copy + id) = c;
        }
    }
    if (tid < 128) sh.exp2_[tid] = exp2((double)tid / 128);
    const float hi_t = hi;  // this thread's
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
    auto put = [&](int id, float prob) {
        R.ids[r] = id;
        if (R.probs) R.probs[r] = prob;
    };
    if (hi == -INFINITY) {  // nothing to draw
        if (tid == 0) put(-1, 0.0f);
        return;
    }
    if (!(temp > 0.0f) || min_p > 1.0f || top_p <= 0.0f || top_k == 1) {  // the most likely token
        u64 at = ~0ull;
        row.each([&](int id, const float(&l)[STEP]) {
#pragma unroll
            for (int e = STEP - 1; e >= 0; e--) at = l[e] == hi && (u64)id < at ? (u64)(id + e) : at;
        });
        if (at != ~0ull) atomicMin(&sh.at, at);
        __syncthreads();
        if (tid == 0) put((int)sh.at, 1.0f);
        return;
    }
    Weight W;
    W.max = hi;
    W.c = 1.4426950408889634 / (double)temp;
    W.S = S;
    W.low = -(double)(S + 2);
    // Bins over the logits that have weight, or all of them if those span less.
    const double span = (double)(S + 3) / W.c, range = (double)hi - (double)lo;
    const bool limited = !(range < span);
    const Bins bins{hi, (float)fmin(fmax((double)BINS / (limited ? span : range), 0x1p-118), 0x1p100)};
    const double least = min_p > 0.0f ? __builtin_ldexp((double)min_p, S) : 0.0;

    Kept K{{-INFINITY, -1}, -1, 0.0};  // everything finite
    const bool by_count = top_k > 0 && top_k < row.n, by_weight = top_p < 1.0f;
    if (by_count && top_k <= NT) {
        // At least top_k logits are as large as the top_k-th largest of the threads'
        // own maxima, and not many more where the ids' order is no order of l.
        const int bin = nth_bin(sh, bins.of(hi_t), hi_t > -INFINITY, top_k);
        if (bin >= 0 && !(limited && bin == BINS - 1)) {
            const int n = collect(sh, row, bins, K.keep, bin, true);
            if (n <= NT) K.n = n;
        }
    }
    if (by_count && K.n < 0) cut<false, true>(sh, row, bins, W, K, (u64)top_k, 0.0, limited);
    const int most = K.n >= 0 ? top_k : NT;  // a list of more than top_k elements so far
    if (by_weight && K.n < 0) {
        if (by_count) cut<true, false>(sh, row, bins, W, K, 0, (double)top_p, limited);
        else cut<true, true>(sh, row, bins, W, K, 0, (double)top_p, limited);
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
    for (const void *fn : {(const void *)k_sample<float, true>, (const void *)k_sample<_Float16, true>,
                           (const void *)k_sample<bf16_bits, true>}) {
        const hipError_t e = ensure_lds_limit(fn, ROW_BYTES + (int)sizeof(Shared));
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_sample(const SampleRows &r, hipStream_t s) {
    if (!r.n_rows) return hipSuccess;
    int lg = 0;
    while ((1ull << lg) < r.vocab) lg++;
    const int S = 62 - lg < 50 ? 62 - lg : 50;
    auto go = [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const size_t row = row_lds<T>(r.vocab);
        if (row <= ROW_BYTES)
            hipLaunchKernelGGL((k_sample<T, true>), dim3((unsigned)r.n_rows), dim3(NT), sizeof(Shared) + row, s, r, S);
        else hipLaunchKernelGGL((k_sample<T, false>), dim3((unsigned)r.n_rows), dim3(NT), sizeof(Shared), s, r, S);
    };
    if (r.dtype == T_F32) go((float *)nullptr);
    else if (r.dtype == T_F16) go((_Float16 *)nullptr);
    else go((bf16_bits *)nullptr);
    return hipGetLastError();
}

}  // namespace rce_qmm
