// sample.hip -- next tokens from logits: temperature, top-k, top-p, min-p and
// the draw from given uniform numbers (include/rce_qmm.h rce_qmm_sample_dev).
//
// A block per row.  Weights are whole numbers, rint(exp((l - max) / T) 2^S)
// with S = 62 - ceil(log2 vocab): a row's sum fits 63 bits, every sum is exact
// and no order of additions matters, so histograms by LDS atomics are
// deterministic.
// The filters keep a prefix of the order (l falling, id rising), which a
// threshold says: keys above `key`, and the first `ties` ids at `key`.  It
// is found by radix descent over the order-preserving bits of l, 8 at a
// time: by counts for top-k, by weights for top-p.
#include "kv_cache.h"

namespace rce_qmm {
namespace {

constexpr int NT = 1024, NW = NT / 64;

typedef unsigned long long u64;

struct Row {
    const void *p;
    uint32_t dtype;
    int n;
};

// l in f32, NaN as -inf, -0 as 0.
__device__ __forceinline__ float logit(const Row &r, int i) {
    float x;
    if (r.dtype == T_F32) x = static_cast<const float *>(r.p)[i];
    else if (r.dtype == T_F16) x = (float)static_cast<const _Float16 *>(r.p)[i];
    else x = __uint_as_float((uint32_t)static_cast<const uint16_t *>(r.p)[i] << 16);
    return x == x ? x + 0.0f : -INFINITY;
}
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

struct Weights {
    float max;
    double inv_t, scale, min_p;  // scale = 2^S
    __device__ __forceinline__ u64 operator()(float l) const {
        if (l == max) return (u64)scale;
        if (l == -INFINITY) return 0;
        const double w = exp(((double)l - (double)max) * inv_t);
        return w > 0.0 ? (u64)rint(w * scale) : 0;  // not above 0: NaN where both max l and T are infinite
    }
};

struct Keep {
    uint32_t key;  // keys above it are kept,
    int ties;      // and the first ids with this key
};

struct Sh {
    u64 hist[256];
    u64 wave[NW];
    int cnt[NW];
    u64 acc;
    uint32_t key;
    int ties, idx;
};

__device__ __forceinline__ u64 wave_sum64(u64 v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
    return v;
}

}  // namespace

__global__ __launch_bounds__(NT) void k_sample(SampleRows R, int shift) {
    __shared__ Sh sh;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const size_t size = R.dtype == T_F32 ? 4 : 2;
    const Row r{static_cast<const char *>(R.logits) + (size_t)row * R.stride * size, R.dtype, (int)R.vocab};
    // the largest key
    uint32_t top = 0;
    for (int i = tid; i < r.n; i += NT) top = max(top, key_of(logit(r, i)));
    if (tid == 0) {
        sh.key = 0;
        sh.idx = r.n;
    }
    __syncthreads();
    atomicMax(&sh.key, top);
    __syncthreads();
    top = sh.key;
    const float max_l = of_key(top);
    if (max_l == -INFINITY) {
        if (tid == 0) {
            R.ids[row] = -1;
            if (R.probs) R.probs[row] = 0.0f;
        }
        return;
    }
    const float t = R.temperature ? R.temperature[row] : 1.0f;
    const float min_p = R.min_p ? R.min_p[row] : 0.0f;
    float top_p = R.top_p ? R.top_p[row] : 1.0f;
    const int top_k = R.top_k ? R.top_k[row] : 0;
    if (!(t > 0.0f) || min_p > 1.0f || top_p <= 0.0f || top_k == 1) {  // the most likely token
        int at = r.n;
        for (int i = tid; i < r.n; i += NT)
            if (key_of(logit(r, i)) == top) {
                at = i;
                break;
            }
        atomicMin(&sh.idx, at);
        __syncthreads();
        if (tid == 0) {
            R.ids[row] = sh.idx;
            if (R.probs) R.probs[row] = 1.0f;
        }
        return;
    }
    Weights W;
    W.max = max_l;
    W.inv_t = 1.0 / (double)t;
    W.scale = (double)(1ull << shift);

    Keep keep{key_of(-INFINITY), 0};
    if (top_k > 0 && top_k < r.n) {
        uint32_t prefix = 0;
        int left = top_k;
        for (int s = 24; s >= 0; s -= 8) {
            if (tid < 256) sh.hist[tid] = 0;
            __syncthreads();
            for (int i = tid; i < r.n; i += NT) {
                const uint32_t k = key_of(logit(r, i));
                if (s == 24 || (k >> (s + 8)) == (prefix >> (s + 8))) atomicAdd(&sh.hist[(k >> s) & 255u], 1ull);
            }
            __syncthreads();
            if (tid == 0) {
                int b = 255, c = left;
                for (; b > 0 && c > (int)sh.hist[b]; b--) c -= (int)sh.hist[b];
                sh.key = prefix | (uint32_t)b << s;
                sh.ties = c;
            }
            __syncthreads();
            prefix = sh.key;
            left = sh.ties;
            __syncthreads();
        }
        keep = {prefix, left};
    }
    // sum of what is kept: above the threshold, and its ties
    if (top_p < 1.0f) {
        u64 s = 0;
        for (int i = tid; i < r.n; i += NT) {
            const float l = logit(r, i);
            if (key_of(l) > keep.key) s += W(l);
        }
        s = wave_sum64(s);
        if (lane == 0) sh.wave[wave] = s;
        __syncthreads();
        u64 total = (u64)keep.ties * W(of_key(keep.key));
        for (int w = 0; w < NW; w++) total += sh.wave[w];
        const double want = (double)top_p * (double)total;
        uint32_t prefix = 0;
        u64 acc = 0;
        for (int s2 = 24; s2 >= 0; s2 -= 8) {
            __syncthreads();
            if (tid < 256) sh.hist[tid] = 0;
            __syncthreads();
            for (int i = tid; i < r.n; i += NT) {
                const float l = logit(r, i);
                const uint32_t k = key_of(l);
                if (k > keep.key && (s2 == 24 || (k >> (s2 + 8)) == (prefix >> (s2 + 8))))
                    atomicAdd(&sh.hist[(k >> s2) & 255u], W(l));
            }
            __syncthreads();
            if (tid == 0) {
                if (keep.ties && (s2 == 24 || (keep.key >> (s2 + 8)) == (prefix >> (s2 + 8))))
                    sh.hist[(keep.key >> s2) & 255u] += (u64)keep.ties * W(of_key(keep.key));
                // from the top: the first bin that reaches `want`, else the lowest with weight
                int b = 0;
                u64 a = acc, before = acc;
                for (int c = 255; c >= 0; c--) {
                    if (!sh.hist[c]) continue;
                    b = c;
                    before = a;
                    a += sh.hist[c];
                    if ((double)a >= want) break;
                }
                sh.acc = before;
                sh.key = prefix | (uint32_t)b << s2;
            }
            __syncthreads();
            prefix = sh.key;
            acc = sh.acc;
        }
        const u64 w = W(of_key(prefix));
        const double m = ceil((want - (double)acc) / (double)w);
        const int most = prefix == keep.key ? keep.ties : r.n;
        keep = {prefix, max(1, (int)fmin(m, (double)most))};
    }
    // draw: a wave per contiguous part of the ids, then 64 at a time in the wave the draw falls into
    const int part = (r.n + NW - 1) / NW, a0 = min(r.n, wave * part), a1 = min(r.n, a0 + part);
    auto passes = [&](float l) { return l == max_l || !(min_p > 0.0f) || exp(((double)l - (double)max_l) * W.inv_t) >= (double)min_p; };
    const u64 wk = passes(of_key(keep.key)) ? W(of_key(keep.key)) : 0;
    u64 sum = 0;
    int ties = 0;
    for (int i = a0 + lane; i < a1; i += 64) {
        const float l = logit(r, i);
        const uint32_t k = key_of(l);
        if (k > keep.key) sum += passes(l) ? W(l) : 0;
        else if (k == keep.key) ties++;
    }
    sum = wave_sum64(sum);
    for (int o = 1; o < 64; o <<= 1) ties += __shfl_xor(ties, o);
    __syncthreads();
    if (lane == 0) {
        sh.wave[wave] = sum;
        sh.cnt[wave] = ties;
    }
    __syncthreads();
    u64 total = 0, before = 0;
    int left = keep.ties, my_left = 0;
    for (int w = 0; w < NW; w++) {
        if (w == wave) {
            before = total;
            my_left = left;
        }
        const int c = min(left, sh.cnt[w]);
        total += sh.wave[w] + (u64)c * wk;
        left -= c;
    }
    const u64 mine = sum + (u64)min(my_left, ties) * wk;
    float u = R.u[row];
    u = u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f;
    u64 want = (u64)((double)u * (double)total);
    if (want >= total) want = total - 1;
    if (!(want >= before && want < before + mine)) return;
    u64 run = before;
    for (int b = a0; b < a1; b += 64) {
        const int i = b + lane;
        const float l = i < a1 ? logit(r, i) : -INFINITY;
        const uint32_t k = i < a1 ? key_of(l) : 0;
        const bool tie = i < a1 && k == keep.key;
        const unsigned long long tm = __ballot(tie);
        const int rank = __popcll(tm & ((1ull << lane) - 1));
        u64 w = k > keep.key ? (passes(l) ? W(l) : 0) : tie && rank < my_left ? wk : 0;
        my_left = max(0, my_left - __popcll(tm));
        u64 c = w;
        for (int o = 1; o < 64; o <<= 1) {
            const u64 y = __shfl_up(c, o);
            if (lane >= o) c += y;
        }
        const unsigned long long hit = __ballot(run + c > want);
        if (hit) {
            const int at = __builtin_ctzll(hit);
            if (lane == at) {
                R.ids[row] = i;
                if (R.probs) R.probs[row] = (float)((double)w / (double)total);
            }
            return;
        }
        run += __shfl(c, 63);
    }
}

hipError_t launch_sample(const SampleRows &r, hipStream_t s) {
    if (!r.n_rows) return hipSuccess;
    int lg = 0;
    while ((1ull << lg) < r.vocab) lg++;
    hipLaunchKernelGGL(k_sample, dim3((unsigned)r.n_rows), dim3(NT), 0, s, r, 62 - lg);
    return hipGetLastError();
}

}  // namespace rce_qmm
