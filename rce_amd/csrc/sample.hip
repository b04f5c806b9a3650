// sample.hip -- next tokens from logits: temperature, top-k, top-p, min-p and
// the draw from given uniform numbers (include/rce_qmm.h rce_qmm_sample_dev).
//
// A block per row.  Weights are whole numbers, rint(exp((l - max) / T) 2^S)
// with S = min(50, 62 - ceil(log2 vocab)): a row's sum fits 63 bits, every sum
// is exact and no order of additions matters, so the histograms, made with LDS
// atomics, are deterministic.
//
// The filters keep a prefix of the order (l falling, id rising): it is told by
// its last element.  To find it, a
// histogram over BINS equal intervals of l says which bin holds the end (by
// counts for top-k, by weights for top-p); that bin's elements are collected,
// sorted, and cut where the count or the sum is reached.  A bin of more than NT
// elements (many equal logits) goes through a radix descent over (order-preserving bits
// of l, id), 64 bits, 8 a pass.
//
// The draw: each wave owns runs of q * 64 consecutive ids (run r of the row
// belongs to wave r % 16); the runs' kept weights are summed and scanned, and the
// wave whose run the draw falls into walks it.
//
// What bounds it: one CU per row, so the row's passes (two to six, from
// registers up to 32768 ids, else from L2) and their double-precision exponentials,
// which only elements that a pass keeps pay for.
#include "kv_cache.h"

#include <type_traits>

namespace rce_qmm {
namespace {

typedef unsigned long long u64;

constexpr int NT = 1024, NW = NT / 64;
constexpr int BINS = 4096;
constexpr int SEGS = 64;    // runs of a wave, at most
constexpr int CACHED = 32;  // ids per thread held in registers

__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// position in the order: smaller comes first
__device__ __forceinline__ u64 place(float l, int id) { return (u64)(~key_of(l)) << 32 | (uint32_t)id; }

struct bf16_bits {
    uint16_t u;
};
__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(_Float16 x) { return (float)x; }
__device__ __forceinline__ float widen(bf16_bits x) { return __uint_as_float((uint32_t)x.u << 16); }

struct Shared {
    u64 hist[BINS];
    u64 sums[SEGS * NW];
    u64 list[NT];
    u64 wave[NW + 1];
    double exp2_[128];  // 2^(j / 128)
    float red[2 * NW];
    u64 at;      // a place, or an id
    u64 before;  // count or weight in front of a bin
    int bin, n;
};

// 2^S exp((l - max) / T) as a double: t = (l - max) log2e / T = k / 128 + r, k a whole
// number, 2^(k / 128) from the table and the exponent, 2^r by its Taylor series to degree 4
// (|r ln 2| <= 2.71e-3: within 2^-49).
struct Weight {
    float max;
    double c;  // log2e / T
    int S;
    double low;  // t below it: weight 0
    __device__ __forceinline__ double value(const Shared &sh, float l) const {
        if (l == max) return __builtin_ldexp(1.0, S);
        const double t = ((double)l - (double)max) * c;
        if (!(t > low)) return 0.0;  // NaN too, of an infinite max and T
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
};

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

// The row's logits.  Run r = seg * NW + wave holds ids r * q * 64 ...; lane
// and step j of a run: id (r * q + j) * 64 + lane.
template <class T, bool REGS>
struct Row {
    const T *p;
    int n, q, segs;
    float x[REGS ? CACHED : 1];

    // id i's logit as loaded, any for ids past the end: the load is not under a
    // condition, so that several are in flight
    __device__ __forceinline__ T raw(int i) const { return p[min(i, n - 1)]; }
    // NaN and ids past the end as -inf, -0 as 0
    __device__ __forceinline__ float value(int i, T t) const {
        const float v = widen(t) + 0.0f;
        return i < n && v == v ? v : -INFINITY;
    }
    __device__ __forceinline__ float load(int i) const { return value(i, raw(i)); }
    __device__ __forceinline__ void fill() {
        if constexpr (REGS) {
            T t[CACHED];
#pragma unroll
            for (int s = 0; s < CACHED; s += 8) {
                if (s >= segs) break;
#pragma unroll
                for (int e = 0; e < 8; e++) t[s + e] = raw((s + e) * NT + (int)threadIdx.x);
            }
#pragma unroll
            for (int s = 0; s < CACHED; s++) x[s] = s < segs ? value(s * NT + (int)threadIdx.x, t[s]) : -INFINITY;
        }
    }
    // f(seg, id, l) for this thread's ids, l = -inf past the row's end.
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        if constexpr (REGS) {
            // opaque, and one after the other: else the passes share 32 keys, ids
            // and places in registers, and spill
            int id = (int)threadIdx.x, m = segs;
            asm volatile("" : "+v"(id), "+s"(m));
#pragma unroll
            for (int s = 0; s < CACHED; s++)
                if (s < m) {
                    float v = x[s];
                    asm volatile("" : "+v"(v), "+v"(id));
                    f(s, id, v);
                    id += NT;
                    __builtin_amdgcn_sched_barrier(0);
                }
        } else {
            const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
            for (int s = 0; s < segs; s++) {
                const int first = (s * NW + wave) * q * 64 + lane;
                for (int j = 0; j < q; j += 4) {  // q is a multiple of 4
                    T t[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) t[e] = raw(first + (j + e) * 64);
#pragma unroll
                    for (int e = 0; e < 4; e++) f(s, first + (j + e) * 64, value(first + (j + e) * 64, t[e]));
                }
            }
        }
    }
};

// f is between 2^-118 and 2^100, so that the product is neither NaN nor lost: past the
// range it is the last bin, and logits of a range below 2^-88 share the first.
struct Bins {
    float max, f;
    __device__ __forceinline__ int of(float l) const {
        return l == max ? 0 : (int)fminf((max - l) * f, (float)(BINS - 1));
    }
};

// Bin b's place in the histogram: a thread's PER bins lie NT apart (no bank conflicts).
constexpr int PER = BINS / NT;
__device__ __forceinline__ int slot_of(int b) { return b % PER * NT + b / PER; }

// The end of what is kept, in the order (l falling, id rising).
struct Keep {
    float l;
    int id;
    __device__ __forceinline__ bool has(float x, int i) const { return x > l || (x == l && i <= id); }
};
__device__ __forceinline__ float logit_of(u64 place) {
    const uint32_t k = ~(uint32_t)(place >> 32);
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ Keep keep_to(u64 place) { return {logit_of(place), (int)(uint32_t)place}; }

// The new end: of what is kept so far only a prefix, the first `want` elements (WEIGHTS false), or the shortest one whose weights reach the
// share `p` of theirs.  limited: the last bin holds only weights of 0.
template <bool WEIGHTS, class R>
__device__ __forceinline__ Keep cut(Shared &sh, const R &row, const Bins &bins, const Weight &W, Keep keep, u64 count,
                                    double p, bool limited) {
    const int tid = threadIdx.x;
    __syncthreads();
    for (int b = tid; b < BINS; b += NT) sh.hist[b] = 0;
    if (tid == 0) sh.bin = -1;
    __syncthreads();
    row.each([&](int, int id, float l) {
        if (keep.has(l, id))
            atomicAdd(&sh.hist[slot_of(bins.of(l))], WEIGHTS ? Weight::whole(W.value(sh, l)) : 1ull);
    });
    __syncthreads();
    u64 h[PER], mine = 0, total;
#pragma unroll
    for (int i = 0; i < PER; i++) mine += h[i] = sh.hist[i * NT + tid];
    u64 run = block_scan(sh, mine, total);
    const double want = WEIGHTS ? p * (double)total : (double)count;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        if ((double)run < want && (double)(run + h[i]) >= want) {  // one bin of the row
            sh.bin = PER * tid + i;
            sh.before = run;
        }
        run += h[i];
    }
    if (tid == 0) sh.n = 0;
    __syncthreads();
    const int bin = sh.bin;
    if (bin < 0 || (limited && bin == BINS - 1)) return keep;  // fewer elements than wanted, or only weights of 0 beyond
    const u64 before = sh.before;
    // the bin's elements
    row.each([&](int, int id, float l) {
        if (bins.of(l) == bin && keep.has(l, id)) {
            const int at = atomicAdd(&sh.n, 1);
            if (at < NT) sh.list[at] = place(l, id);
        }
    });
    __syncthreads();
    const int n = sh.n;
    if (n <= NT) {
        // a bitonic sort, one element per thread; steps within a wave by lane exchanges
        u64 v = tid < n ? sh.list[tid] : ~0ull;
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
        u64 w = 0;
        if (tid < n) w = WEIGHTS ? Weight::whole(W.value(sh, logit_of(v))) : 1;
        u64 all;
        const u64 ahead = before + block_scan(sh, w, all);
        if (tid < n && (double)ahead < want && (double)(ahead + w) >= want) sh.at = v;
        __syncthreads();
        return keep_to(sh.at);
    }
    // radix descent over the places
    u64 prefix = 0, acc = before;
    for (int s = 56; s >= 0; s -= 8) {
        __syncthreads();
        if (tid < 256) sh.hist[tid] = 0;
        __syncthreads();
        row.each([&](int, int id, float l) {
            const u64 v = place(l, id);
            if (bins.of(l) == bin && keep.has(l, id) && (s == 56 || v >> (s + 8) == prefix >> (s + 8)))
                atomicAdd(&sh.hist[(v >> s) & 255u], WEIGHTS ? Weight::whole(W.value(sh, l)) : 1ull);
        });
        __syncthreads();
        const u64 c = tid < 256 ? sh.hist[tid] : 0;
        u64 all;
        const u64 ahead = acc + block_scan(sh, c, all);
        if ((double)ahead < want && (double)(ahead + c) >= want) {
            sh.at = prefix | (u64)tid << s;
            sh.before = ahead;
        }
        __syncthreads();
        prefix = sh.at;
        acc = sh.before;
    }
    return keep_to(prefix);
}

template <class T, bool REGS>
__global__ __launch_bounds__(NT) void k_sample(SampleRows R, int S) {
    __shared__ Shared sh;
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    Row<T, REGS> row;
    row.p = static_cast<const T *>(R.logits) + (size_t)r * R.stride;
    row.n = (int)R.vocab;
    row.q = REGS ? 1 : (row.n + SEGS * NT * 4 - 1) / (SEGS * NT * 4) * 4;
    row.segs = (row.n + row.q * NT - 1) / (row.q * NT);
    row.fill();
    if (tid < 128) sh.exp2_[tid] = exp2((double)tid / 128);
    const float temp = R.temperature ? R.temperature[r] : 1.0f;
    const float min_p = R.min_p ? R.min_p[r] : 0.0f;
    const float top_p = R.top_p ? R.top_p[r] : 1.0f;
    const int top_k = R.top_k ? R.top_k[r] : 0;
    const float u_in = R.u[r];

    // the largest and the smallest finite logit
    float hi = -INFINITY, lo = INFINITY;
    row.each([&](int, int, float l) {
        hi = fmaxf(hi, l);
        lo = fminf(lo, l > -INFINITY ? l : INFINITY);
    });
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
    if (hi == -INFINITY) {  // nothing to draw
        if (tid == 0) {
            R.ids[r] = -1;
            if (R.probs) R.probs[r] = 0.0f;
        }
        return;
    }
    if (!(temp > 0.0f) || min_p > 1.0f || top_p <= 0.0f || top_k == 1) {  // the most likely token
        u64 at = ~0ull;
        row.each([&](int, int id, float l) {
            if (l == hi && at == ~0ull) at = (u64)id;
        });
        if (at != ~0ull) atomicMin(&sh.at, at);
        __syncthreads();
        if (tid == 0) {
            R.ids[r] = (int)sh.at;
            if (R.probs) R.probs[r] = 1.0f;
        }
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

    Keep keep{-INFINITY, -1};  // everything finite
    if (top_k > 0 && top_k < row.n) keep = cut<false>(sh, row, bins, W, keep, (u64)top_k, 0.0, limited);
    if (top_p < 1.0f) keep = cut<true>(sh, row, bins, W, keep, 0, (double)top_p, limited);

    // the runs' kept weights
    const double least = min_p > 0.0f ? __builtin_ldexp((double)min_p, S) : 0.0;
    auto kept = [&](int id, float l) -> u64 {
        if (!keep.has(l, id)) return 0;
        const double w = W.value(sh, l);
        return w >= least ? Weight::whole(w) : 0;
    };
    __syncthreads();
    sh.sums[tid] = 0;
    __syncthreads();
    {
        u64 sum = 0;
        int at = 0;
        row.each([&](int s, int id, float l) {
            if constexpr (REGS) {
                if (__ballot(keep.has(l, id))) {
                    const u64 w = wave_sum64(kept(id, l));
                    if (lane == 0) sh.sums[s * NW + wave] = w;
                }
            } else {
                if (s != at) {
                    if (__ballot(sum != 0)) {
                        sum = wave_sum64(sum);
                        if (lane == 0) sh.sums[at * NW + wave] = sum;
                    }
                    sum = 0;
                    at = s;
                }
                if (__ballot(keep.has(l, id))) sum += kept(id, l);
            }
        });
        if constexpr (!REGS) {
            sum = wave_sum64(sum);
            if (lane == 0) sh.sums[at * NW + wave] = sum;
        }
    }
    __syncthreads();
    static_assert(SEGS * NW == NT, "a thread per run");
    const u64 mine = sh.sums[tid];
    u64 total;
    const u64 ahead = block_scan(sh, mine, total);
    const float u = u_in > 0.0f ? fminf(u_in, 0x1.fffffep-1f) : 0.0f;
    u64 want = (u64)((double)u * (double)total);
    want = want < total ? want : total - 1;
    if (want >= ahead && want < ahead + mine) {
        sh.bin = tid;
        sh.before = ahead;
    }
    __syncthreads();
    const int run = sh.bin;
    if (wave != run % NW) return;
    u64 acc = sh.before;
    for (int j = 0; j < row.q; j++) {
        const int id = (run * row.q + j) * 64 + lane;
        const float l = row.load(id);
        const u64 w = kept(id, l), c = wave_scan64(w);
        const u64 hit = __ballot(acc + c > want);
        if (hit) {
            if (lane == __builtin_ctzll(hit)) {
                R.ids[r] = id;
                if (R.probs) R.probs[r] = (float)((double)w / (double)total);
            }
            return;
        }
        acc += lane64(c, 63);
    }
}

}  // namespace

hipError_t launch_sample(const SampleRows &r, hipStream_t s) {
    if (!r.n_rows) return hipSuccess;
    int lg = 0;
    while ((1ull << lg) < r.vocab) lg++;
    const int S = 62 - lg < 50 ? 62 - lg : 50;
    auto go = [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (r.vocab <= (size_t)CACHED * NT)
            hipLaunchKernelGGL((k_sample<T, true>), dim3((unsigned)r.n_rows), dim3(NT), 0, s, r, S);
        else hipLaunchKernelGGL((k_sample<T, false>), dim3((unsigned)r.n_rows), dim3(NT), 0, s, r, S);
    };
    if (r.dtype == T_F32) go((float *)nullptr);
    else if (r.dtype == T_F16) go((_Float16 *)nullptr);
    else go((bf16_bits *)nullptr);
    return hipGetLastError();
}

}  // namespace rce_qmm
