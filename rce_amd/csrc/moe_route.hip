// moe_route.hip -- routing of tokens to experts (include/rce_qmm.h
// rce_qmm_moe_route_dev).
//
// A wave takes a token, or several of few experts; waves share nothing.  A
// round finds the largest key, the lowest expert among equals, and takes it
// away; round r's expert goes to lane r, which weighs it at the end.
//
// Without a bias the order of the scores is that of the logits, whatever the
// scores round to: keys are the logits as 32-bit whole numbers.  A bias is added
// to scores of 64 bits, and groups that count by two experts are compared by
// sums of 64 bits: neighbours in 16-bit logits differ by 2^-8 of a score, but a
// score of 32 bits plus a bias would make equals of what is not.
#include "moe_route.h"

#include <algorithm>
#include <type_traits>
#include <utility>

namespace rce_qmm {
namespace {

// v of the lane that CTRL names.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, true);
}

// f over the lanes of an aligned group of L (8, 16, 32 or 64), the result in all of them.
template <int L, class F>
__device__ __forceinline__ uint32_t over(uint32_t v, F f) {
    v = f(v, dpp<0xB1>(v));   // quad_perm [1,0,3,2]
    v = f(v, dpp<0x4E>(v));   // quad_perm [2,3,0,1]
    v = f(v, dpp<0x141>(v));  // row_half_mirror: the other quad of the 8
    if constexpr (L >= 16) v = f(v, dpp<0x140>(v));  // row_mirror
    if constexpr (L >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = f(r[0], r[1]);
    }
    if constexpr (L >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = f(r[0], r[1]);
    }
    return v;
}
template <int L>
__device__ __forceinline__ uint32_t most(uint32_t v) {
    return over<L>(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}
template <int L>
__device__ __forceinline__ uint32_t least(uint32_t v) {
    return over<L>(v, [](uint32_t a, uint32_t b) { return min(a, b); });
}
template <int L>
__device__ __forceinline__ float sum_over(float x) {
    return __uint_as_float(over<L>(__float_as_uint(x), [](uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
}
template <int CTRL>
__device__ __forceinline__ double dpp64(double x) {
    const uint64_t u = (uint64_t)__double_as_longlong(x);
    return __longlong_as_double((long long)((uint64_t)dpp<CTRL>((uint32_t)(u >> 32)) << 32 | dpp<CTRL>((uint32_t)u)));
}
template <int L>
__device__ __forceinline__ double sum_of(double x) {
    x += dpp64<0xB1>(x);
    x += dpp64<0x4E>(x);
    x += dpp64<0x141>(x);
    if constexpr (L >= 16) x += dpp64<0x140>(x);
    if constexpr (L >= 32) x += __shfl_xor(x, 16);
    if constexpr (L >= 64) x += __shfl_xor(x, 32);
    return x;
}

// Whole numbers in the order of x (not NaN; both zeros are one), all above 0: 0 is no expert.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t ordered(double x) {
    const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
    return u >> 63 ? ~u : u | 0x8000000000000000u;
}
__device__ __forceinline__ float number(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u); }  // of ordered()
constexpr uint32_t NONE32 = 0x007FFFFFu;                 // ordered(-inf)

__device__ __forceinline__ float logit(const void *p, uint32_t t, size_t i) {
    float x;
    if (t == T_F32) x = static_cast<const float *>(p)[i];
    else if (t == T_F16) x = (float)static_cast<const _Float16 *>(p)[i];
    else x = __uint_as_float((uint32_t)static_cast<const uint16_t *>(p)[i] << 16);
    return x != x ? -__builtin_inff() : x;
}

// The score of logit x (top: the row's largest one; total: the sum of exp(x - top)).
__device__ __forceinline__ double score_of(bool sigmoid, float x, float top, double total) {
    if (sigmoid) return 1.0 / (1.0 + exp(-(double)x));
    return (x == top ? 1.0 : exp((double)x - (double)top)) / total;
}

// A token's logits, experts sub + L j (past the last one: -inf).
template <int L, int N>
__device__ __forceinline__ void load(const Routing &A, size_t row, int sub, float (&x)[N]) {
    if (A.dtype == T_F32) {
        const float *p = static_cast<const float *>(A.logits) + row;
#pragma unroll
        for (int j = 0; j < N; j++) x[j] = p[min(sub + L * j, A.n_expert - 1)];
    } else {
        const uint16_t *p = static_cast<const uint16_t *>(A.logits) + row;
        uint16_t u[N];
#pragma unroll
        for (int j = 0; j < N; j++) u[j] = p[min(sub + L * j, A.n_expert - 1)];
        const bool f16 = A.dtype == T_F16;
#pragma unroll
        for (int j = 0; j < N; j++) x[j] = f16 ? (float)__builtin_bit_cast(_Float16, u[j]) : __uint_as_float((uint32_t)u[j] << 16);
    }
#pragma unroll
    for (int j = 0; j < N; j++) x[j] = x[j] == x[j] && sub + L * j < A.n_expert ? x[j] : -__builtin_inff();
}
template <int L, int N>
__device__ __forceinline__ float top_of(const float (&x)[N]) {
    float top = x[0];
#pragma unroll
    for (int j = 1; j < N; j++) top = fmaxf(top, x[j]);
    return number(most<L>(ordered(top)));
}
// The softmax's sum in 64 bits.
template <int L, int N>
__device__ __forceinline__ double total_of(const Routing &A, const float (&x)[N], int sub, float top) {
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < N; j++) sum += sub + L * j >= A.n_expert ? 0.0 : x[j] == top ? 1.0 : exp((double)x[j] - (double)top);
    return sum_of<L>(sum);
}

// Lane `sub` of a token's weighs and writes its choice sub.
template <int L>
__device__ __forceinline__ void finish(const Routing &A, bool is, int64_t at, size_t row, int sub, int id, float top, double total) {
    const float x = logit(A.logits, A.dtype, row + id), b = A.bias ? A.bias[id] : 0.0f;
    double w = 0.0;
    if (sub < A.top_k && x > -__builtin_inff() && b > -__builtin_inff()) w = score_of(A.sigmoid, x, top, total);
    if (A.normalize) {
        const double s = sum_of<L>(w);
        w = s > 0.0 ? w / s : 0.0;
    }
    if (is && sub < A.top_k) {
        const size_t o = (size_t)at * A.top_k + sub;
        A.ids[o] = id;
        A.weights[o] = (float)(w * (double)A.scale);
    }
}

// ---- few experts ------------------------------------------------------------------

// L lanes take a token, N experts each (expert lane + L j), 64 / L tokens to a wave.  K: uint32_t without a bias.
template <class K, int L, int N>
__global__ __launch_bounds__(256) void k_moe_route_few(Routing A) {
    constexpr bool WIDE = std::is_same<K, uint64_t>::value;
    const int lane = threadIdx.x & 63, sub = lane & (L - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t at = ((int64_t)blockIdx.x * 4 + wave) * (64 / L) + lane / L;
    const bool is = at < A.n_tokens;
    const size_t row = (size_t)(is ? at : 0) * A.stride;

    float x[N];
    load<L, N>(A, row, sub, x);
    const float top = top_of<L, N>(x);
    double total = 1.0;
    if (!A.sigmoid && (WIDE || !A.normalize)) total = total_of<L, N>(A, x, sub, top);
    K key[N];
#pragma unroll
    for (int j = 0; j < N; j++) {
        const int e = sub + L * j;
        if constexpr (WIDE) {
            double v = score_of(A.sigmoid, x[j], top, total) + (double)A.bias[min(e, A.n_expert - 1)];
            if (x[j] == -__builtin_inff() || v != v) v = -__builtin_inf();
            key[j] = ordered(v);
        } else {
            key[j] = ordered(x[j]);
        }
        if (e >= A.n_expert) key[j] = 0;
    }
    int id = 0;
    for (int r = 0; r < A.top_k; r++) {
        K best = key[0];
        int e = sub;
#pragma unroll
        for (int j = 1; j < N; j++) {
            e = key[j] > best ? sub + L * j : e;
            best = key[j] > best ? key[j] : best;
        }
        bool mine;
        if constexpr (WIDE) {
            const uint32_t hi = (uint32_t)(best >> 32), top_hi = most<L>(hi);
            const uint32_t lo = hi == top_hi ? (uint32_t)best : 0u, top_lo = most<L>(lo);
            mine = hi == top_hi && lo == top_lo;
        } else {
            mine = best == most<L>(best);
        }
        const int win = (int)least<L>(mine ? (uint32_t)e : ~0u);
        id = sub == r ? win : id;
#pragma unroll
        for (int j = 0; j < N; j++) key[j] = win == sub + L * j ? 0 : key[j];
    }
    finish<L>(A, is, at, row, sub, id, top, total);
}

// ---- a wave per token ------------------------------------------------------------

// Keys of the lanes as the next expert in order: the largest key, the lowest expert among equals: in the masks of
// the lanes that hold it the first bit of the first one that has any.  Takes it away; its key in m.
template <int N>
__device__ __forceinline__ int take(uint32_t (&key)[N], uint32_t &m) {
    uint32_t best = key[0];
#pragma unroll
    for (int j = 1; j < N; j++) best = max(best, key[j]);
    m = __builtin_amdgcn_readfirstlane((int)most<64>(best));
    uint64_t held[N];
    int e = -1;
#pragma unroll
    for (int j = 0; j < N; j++) held[j] = __ballot(key[j] == m);
#pragma unroll
    for (int j = N - 1; j >= 0; j--) e = held[j] ? 64 * j + __builtin_ctzll(held[j]) : e;
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < N; j++) key[j] = lane + 64 * j == e ? 0u : key[j];
    return e;
}
template <int N>
__device__ __forceinline__ int take(uint64_t (&key)[N], uint64_t &m) {
    uint64_t best = key[0];
#pragma unroll
    for (int j = 1; j < N; j++) best = key[j] > best ? key[j] : best;
    const uint32_t hi = most<64>((uint32_t)(best >> 32)), lo = most<64>((uint32_t)(best >> 32) == hi ? (uint32_t)best : 0u);
    m = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)hi) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)lo);
    int e = -1;
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int j = N - 1; j >= 0; j--) {
        const uint64_t held = __ballot(key[j] == m);
        e = held ? 64 * j + __builtin_ctzll(held) : e;
    }
#pragma unroll
    for (int j = 0; j < N; j++) key[j] = lane + 64 * j == e ? 0ull : key[j];
    return e;
}

__device__ __forceinline__ float lane_value(float x, int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), l)); }
__device__ __forceinline__ double lane_value(double x, int l) {
    const uint64_t u = (uint64_t)__double_as_longlong(x);
    return __longlong_as_double((long long)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(u >> 32), l) << 32 |
                                            (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, l)));
}

// A call's groups on a wave's lanes: 1 << lg lanes to a group.
struct Groups {
    int lg = 6, size;
    float per;
    __device__ explicit Groups(const Routing &A) : size(A.n_expert / A.n_group) {
        while ((A.n_group << lg) > 64) lg--;
        per = 1.0f / (float)size;
    }
    // whether expert e's group is in the mask of group g's bits at g << lg
    __device__ bool holds(uint64_t kept, int e) const {
        return kept >> (((int)(((float)e + 0.5f) * per) << lg) & 63) & 1;  // exact for up to 1024 experts
    }
};

// The groups that experts are chosen from, group g's bit at g << lg: a group's lanes find its two largest values (in LDS, v), the
// groups' worth is compared.  slack above 0: `sure` becomes false where two worths are nearer each other than that and what their
// addends' roundings come to, or their addends pass binary32.
template <class V>
__device__ __forceinline__ uint64_t kept_groups(const Routing &A, const V *v, const Groups &G, float slack, bool &sure) {
    const V none = -(V)__builtin_inff();
    const int lg = G.lg, size = G.size, lane = threadIdx.x & 63, P = 1 << lg, g = lane >> lg;
    V a = none, b = none;
    if (g < A.n_group)
        for (int i = lane & (P - 1); i < size; i += P) {
            const V y = v[g * size + i];
            const V low = y > a ? a : y;
            a = y > a ? y : a;
            b = low > b ? low : b;
        }
    for (int o = 1; o < P; o *= 2) {
        const V c = __shfl_xor(a, o), d = __shfl_xor(b, o);
        const V low = c > a ? a : c;
        a = c > a ? c : a;
        b = d > b ? d : b;
        b = low > b ? low : b;
    }
    // of the addends, not of a sum that they cancel in; no expert: below all
    float addends = a > none ? fabsf((float)a) : -1.0f;
    if (A.group_top == 2 && b > none) {
        a += b;
        addends += fabsf((float)b);
    }
    int rank = 0;
    bool near = false;
    for (int i = 0; i < A.n_group; i++) {
        const V o = lane_value(a, i << lg);
        rank += o > a || (o == a && i < g);
        if (slack > 0.0f) {
            const float larger = fmaxf(addends, lane_value(addends, i << lg));
            near |= i != g && larger >= 0.0f && !(fabsf((float)(o - a)) > slack + 0x1p-21f * larger);
        }
    }
    if (slack > 0.0f && __ballot(near && g < A.n_group)) sure = false;
    return __ballot(g < A.n_group && rank < A.topk_group);
}

// Experts lane + 64 j, N a lane.
//
// With a bias, or with groups that count by two experts, scores and sums of 32 bits choose first, and the choice stands where no two
// of what it compared are nearer to each other than their errors reach; else the wave does it again in 64 bits (a call with one such token
// takes 10 us for 5).  A score's error:
//   sigmoid: the exponent's two roundings, 1.5 * 2^-24 |x|, times the slope (|x| s (1 - s) <= 0.23); 2^-23 of the exponential times the slope
//   (<= 1/4); 2^-24 + 2^-23 for the sum and the reciprocal: below 2^-22;
//   softmax, t = top - x: 2.5 * 2^-24 t + 2^-23 of e^-t, in the sum too (its weighted mean of t is at most ln 1024), whose 1024 terms add up in
//   21 roundings (16 a lane, six steps between lanes), reciprocal and product: 45 * 2^-24 of a score, below 2^-18 of the highest.
// A sum with the bias is rounded to 2^-24 of itself.  So is a group's sum of two, whose addends may be far larger than it: two groups' sums
// are off by 2^-23 of what each one's addends come to, less than 2^-21 of the larger.
constexpr float SIGMOID_ERROR = 0x1p-22f, SOFTMAX_ERROR = 0x1p-18f;

__device__ __forceinline__ float rough_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }
__device__ __forceinline__ float rough_sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + rough_exp(-x)); }
// A wave's LDS accesses before and after it, in this order.
__device__ __forceinline__ void together() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The choice of a wave's token by scores and sums of 64 bits: lane r gets choice r.  v: LDS of the wave, 64 N values (GROUPS).
template <int N, bool GROUPS>
__device__ __forceinline__ int choose_exactly(const Routing &A, const float (&x)[N], float top, double *v) {
    const int lane = threadIdx.x & 63;
    double total = 1.0;
    if (!A.sigmoid) total = total_of<64, N>(A, x, lane, top);
    uint64_t key[N];
#pragma unroll
    for (int j = 0; j < N; j++) {
        const int e = lane + 64 * j;
        double y = score_of(A.sigmoid, x[j], top, total);
        if (A.bias) y += (double)A.bias[min(e, A.n_expert - 1)];
        if (x[j] == -__builtin_inff() || y != y) y = -__builtin_inf();
        if constexpr (GROUPS) v[e] = A.bias || A.group_top == 2 ? y : (double)x[j];
        key[j] = e < A.n_expert ? ordered(A.bias ? y : (double)x[j]) : 0ull;
    }
    if constexpr (GROUPS) {
        together();
        bool sure = true;
        const Groups g(A);
        const uint64_t kept = kept_groups<double>(A, v, g, 0.0f, sure);
        together();
#pragma unroll
        for (int j = 0; j < N; j++) key[j] = g.holds(kept, lane + 64 * j) ? key[j] : 0;
    }
    int id = 0;
    for (int r = 0; r < A.top_k; r++) {
        uint64_t m;
        const int e = take<N>(key, m);
        id = lane == r ? e : id;
    }
    return id;
}

template <int N, bool GROUPS>
__global__ __launch_bounds__(256) void k_moe_route(Routing A) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int at = blockIdx.x * 4 + wave;
    if (at >= A.n_tokens) return;
    const size_t row = (size_t)at * A.stride;
    const bool rough = A.bias || (GROUPS && A.group_top == 2);
    __shared__ double values[GROUPS ? 4 : 1][GROUPS ? 64 * N : 1];

    float x[N], v[N], bias[N], error = SIGMOID_ERROR;
    load<64, N>(A, row, lane, x);
#pragma unroll
    for (int j = 0; j < N; j++) bias[j] = A.bias ? A.bias[min(lane + 64 * j, A.n_expert - 1)] : 0.0f;
    float top = 0.0f;
    double total = 1.0;
    if (!A.sigmoid) {
        top = top_of<64, N>(x);
        if (!A.normalize) total = total_of<64, N>(A, x, lane, top);
    }
    if (!rough) {
#pragma unroll
        for (int j = 0; j < N; j++) v[j] = x[j];
    } else {
        if (A.sigmoid) {
#pragma unroll
            for (int j = 0; j < N; j++) v[j] = rough_sigmoid(x[j]);
        } else {
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < N; j++) {
                v[j] = x[j] == top ? 1.0f : rough_exp(x[j] - top);
                sum += lane + 64 * j < A.n_expert ? v[j] : 0.0f;
            }
            sum = __builtin_amdgcn_rcpf(sum_over<64>(sum));
            error = SOFTMAX_ERROR * sum;  // the highest score
#pragma unroll
            for (int j = 0; j < N; j++) v[j] *= sum;
        }
#pragma unroll
        for (int j = 0; j < N; j++) {
            v[j] += bias[j];
            v[j] = x[j] > -__builtin_inff() && v[j] == v[j] ? v[j] : -__builtin_inff();
        }
    }
    uint32_t key[N];
#pragma unroll
    for (int j = 0; j < N; j++) key[j] = lane + 64 * j < A.n_expert ? ordered(A.bias ? v[j] : x[j]) : 0u;
    bool sure = true;
    if constexpr (GROUPS) {
        float *w = reinterpret_cast<float *>(values[wave]);
#pragma unroll
        for (int j = 0; j < N; j++) w[lane + 64 * j] = v[j];
        together();
        const Groups g(A);
        const uint64_t kept = kept_groups<float>(A, w, g, rough ? 4.0f * error + 0x1p-21f : 0.0f, sure);
        together();
#pragma unroll
        for (int j = 0; j < N; j++) key[j] = g.holds(kept, lane + 64 * j) ? key[j] : 0;
    }
    int id = 0;
    uint32_t chosen = 0;  // lane r: the key of choice r
    for (int r = 0; r < A.top_k; r++) {
        uint32_t m;
        const int e = take<N>(key, m);
        id = lane == r ? e : id;
        chosen = lane == r ? m : chosen;
    }
    if (A.bias) {  // neighbours among the chosen, and the last with what comes next
        uint32_t best = key[0];
#pragma unroll
        for (int j = 1; j < N; j++) best = max(best, key[j]);
        best = most<64>(best);
        uint32_t after = (uint32_t)__shfl_down((int)chosen, 1);  // (all lanes take part)
        after = lane + 1 < A.top_k ? after : best;
        const float a = number(chosen), b = number(after);
        if (__ballot(lane < A.top_k && after > NONE32 && !(a - b > 2.0f * error + 0x1p-23f * (fabsf(a) + fabsf(b))))) sure = false;
    }
    if (!__builtin_amdgcn_readfirstlane((int)sure)) id = choose_exactly<N, GROUPS>(A, x, top, values[GROUPS ? wave : 0]);
    finish<64>(A, true, at, row, lane, id, top, total);
}

// ---- four tokens to a wave -----------------------------------------------------------
//
// Many tokens: 16 lanes take one, experts C s .. C s + C - 1 lane s; up to 16 choices.  A key is one word, (level, 1023 - expert),
// so that a round is a maximum over the lanes and the winner's word alone says which it was.  The level: 16 bits of a 16-bit logit
// (no bias: its order exactly); the first 22 bits of a logit of 32; with a bias score + bias in steps of 2^-19 from -4 to 4, off by
// 0.4 steps (sigmoid) or 2.3 (softmax) before it is cut to whole ones: the errors above, 2^-22 each for the sums with the bias and with 4.
// Two levels stand in their order if they are `apart` steps from each other, twice that and one; a token with two
// chosen ones (or the last and the next) nearer than that, or a sum outside -4 .. 4, is done again by the wave in 64 bits.
// Groups are whole lanes, 1, 2, 4 or 8 of them, compared by the sums of their levels (four errors and two cuts).
//
// 12289 x 256 bf16, 4 of 8 groups, 8 experts: 14 us, 330 vector instructions for a token; a wave per token 758 and 22 us.  What bounds it: a
// wave's own chain, 9 rounds of dependent maxima, with three waves per SIMD to share it.
// f(1), f(2), ... as constants.
template <class F, int... I>
__device__ __forceinline__ void each_of(F f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I + 1>{}), ...);
}

template <int C, bool GROUPS>
__global__ __launch_bounds__(256) void k_moe_route_fours(Routing A, int group_lanes, int vec) {
    constexpr int N = C <= 4 ? 1 : C / 4;  // of a wave per token
    const int lane = threadIdx.x & 63, sub = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t first = ((int64_t)blockIdx.x * 4 + wave) * 4, at = first + lane / 16;
    const bool is = at < A.n_tokens;
    const size_t row = (size_t)(is ? at : A.n_tokens - 1) * A.stride;
    const bool rough = A.bias || (GROUPS && A.group_top == 2), f32 = A.dtype == T_F32, f16 = A.dtype == T_F16;
    __shared__ double values[GROUPS ? 4 : 1][GROUPS ? 64 * N : 1];

    // whole lanes of experts, at multiples of their size
    auto pieces = [&](const float *from, float (&y)[C]) {
        float4 p[C / 4];
#pragma unroll
        for (int i = 0; i < C / 4; i++) p[i] = reinterpret_cast<const float4 *>(from)[i];
#pragma unroll
        for (int i = 0; i < C / 4; i++) {
            y[4 * i] = p[i].x;
            y[4 * i + 1] = p[i].y;
            y[4 * i + 2] = p[i].z;
            y[4 * i + 3] = p[i].w;
        }
    };
    const int lane_at = C * min(sub, max(A.n_expert / C, 1) - 1);
    float x[C], bias[C];
    if (A.bias) {
        if (vec & 2) {
            pieces(A.bias + lane_at, bias);
        } else {
#pragma unroll
            for (int j = 0; j < C; j++) bias[j] = A.bias[min(C * sub + j, A.n_expert - 1)];
        }
    }
    if (vec & 1) {
        if (f32) {
            pieces(static_cast<const float *>(A.logits) + row + lane_at, x);
        } else {
            struct alignas(C >= 8 ? 16 : 8) Words {
                uint32_t w[C >= 8 ? 4 : 2];
            };
            constexpr int W = sizeof(Words) / 4;
            const Words *from = reinterpret_cast<const Words *>(static_cast<const uint16_t *>(A.logits) + row + lane_at);
            Words p[C / (2 * W)];
#pragma unroll
            for (int i = 0; i < C / (2 * W); i++) p[i] = from[i];
#pragma unroll
            for (int j = 0; j < C; j++) {
                const uint32_t w = p[j / (2 * W)].w[j / 2 % W];
                x[j] = f16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)(j & 1 ? w >> 16 : w)) : __uint_as_float(j & 1 ? w & 0xFFFF0000u : w << 16);
            }
        }
    } else if (f32) {
#pragma unroll
        for (int j = 0; j < C; j++) x[j] = static_cast<const float *>(A.logits)[row + min(C * sub + j, A.n_expert - 1)];
    } else {
#pragma unroll
        for (int j = 0; j < C; j++) {
            const uint16_t u = static_cast<const uint16_t *>(A.logits)[row + min(C * sub + j, A.n_expert - 1)];
            x[j] = f16 ? (float)__builtin_bit_cast(_Float16, u) : __uint_as_float((uint32_t)u << 16);
        }
    }
    const int mine = min(max(A.n_expert - C * sub, 0), C);  // experts of this lane
#pragma unroll
    for (int j = 0; j < C; j++) x[j] = fmaxf(j < mine ? x[j] : -__builtin_inff(), -__builtin_inff());  // (NaN: -inf)
    float top = 0.0f;
    double total = 1.0;
    if (!A.sigmoid) {
        top = x[0];
#pragma unroll
        for (int j = 1; j < C; j++) top = fmaxf(top, x[j]);
        top = number(most<16>(ordered(top)));
        if (!A.normalize) {
            double sum = 0.0;
#pragma unroll
            for (int j = 0; j < C; j++) sum += j >= mine ? 0.0 : x[j] == top ? 1.0 : exp((double)x[j] - (double)top);
            total = sum_of<16>(sum);
        }
    }

    float v[C];  // what groups go by, and keys with a bias
    bool unsure = false;
    if (!rough) {
#pragma unroll
        for (int j = 0; j < C; j++) v[j] = x[j];
    } else {
        if (A.sigmoid) {
#pragma unroll
            for (int j = 0; j < C; j++) v[j] = rough_sigmoid(x[j]);
        } else {
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < C; j++) {
                v[j] = x[j] == top ? 1.0f : rough_exp(x[j] - top);
                sum += j < mine ? v[j] : 0.0f;
            }
            sum = __builtin_amdgcn_rcpf(sum_over<16>(sum));
#pragma unroll
            for (int j = 0; j < C; j++) v[j] *= sum;
        }
        if (A.bias) {
#pragma unroll
            for (int j = 0; j < C; j++) v[j] += bias[j];
        }
#pragma unroll
        for (int j = 0; j < C; j++) v[j] = x[j] > -__builtin_inff() ? fmaxf(v[j], -__builtin_inff()) : -__builtin_inff();
    }
    uint32_t key[C];
    int apart;
    const uint32_t last = 1023u - C * sub;
    if (A.bias) {
        apart = A.sigmoid ? 2 : 6;
        float far = 0.0f;
#pragma unroll
        for (int j = 0; j < C; j++) {
            const float y = v[j] > -__builtin_inff() ? v[j] : 0.0f;
            far = fmaxf(far, fabsf(y));
            const uint32_t level = (uint32_t)((y + 4.0f) * 0x1p19f);
            key[j] = v[j] > -__builtin_inff() ? level << 10 | (last - j) : last - j;
        }
        unsure = !(far < 3.9f);
    } else if (f32) {
        apart = 1;
#pragma unroll
        for (int j = 0; j < C; j++) key[j] = x[j] > -__builtin_inff() ? (ordered(x[j]) & ~1023u) | (last - j) : last - j;
    } else {  // exact: a logit of 16 bits is the first 19 of its 32 at most
        apart = 0;
#pragma unroll
        for (int j = 0; j < C; j++) key[j] = x[j] > -__builtin_inff() ? (ordered(x[j]) & ~1023u) | (last - j) : last - j;
    }
#pragma unroll
    for (int j = 0; j < C; j++) key[j] = j < mine ? key[j] : 0u;

    if constexpr (GROUPS) {
        // worths in levels, a missing second expert 0's
        uint32_t a = 0, b = 0;
        const bool own = rough && !A.bias;  // keys are the logits', worths the scores'
#pragma unroll
        for (int j = 0; j < C; j++) {
            uint32_t y = key[j] >> 10;
            if (own) y = key[j] >> 10 ? (uint32_t)((v[j] + 4.0f) * 0x1p19f) : 0u;
            b = max(b, min(a, y));
            a = max(a, y);
        }
        auto merge = [&](auto ctrl) {
            constexpr int CTRL = decltype(ctrl)::value;
            const uint32_t c = dpp<CTRL>(a), d = dpp<CTRL>(b);
            b = max(max(b, d), min(a, c));
            a = max(a, c);
        };
        if (group_lanes > 1) merge(std::integral_constant<int, 0xB1>{});
        if (group_lanes > 2) merge(std::integral_constant<int, 0x4E>{});
        if (group_lanes > 4) merge(std::integral_constant<int, 0x141>{});
        const int g = sub / group_lanes;
        if (A.group_top == 2 && a) a += b ? b : 4u << 19;
        // at most 2^23, over the group's number, the lower ones first; lanes without a group last
        const int worth = g < A.n_group ? (int)(a << 5 | (31u - g)) : -1 - g;
        const int near = (rough ? A.sigmoid ? 4 : 12 : apart) << 5;
        int before = 0;
        auto against = [&](auto by) {
            constexpr int K = decltype(by)::value;
            if (K % group_lanes) return;
            const int o = (int)dpp<0x120 + K>((uint32_t)worth);  // row_ror
            before += o > worth;
            unsure |= min(o, worth) >= 32 && abs(o - worth) < near;
        };
        each_of(against, std::make_integer_sequence<int, 15>{});
        if (g >= A.n_group || before >= A.topk_group) {
#pragma unroll
            for (int j = 0; j < C; j++) key[j] = 0;
        }
    }

    uint32_t chosen = 0;  // lane r: the word of choice r
    for (int r = 0; r <= A.top_k; r++) {  // and the next one
        uint32_t m = key[0];
#pragma unroll
        for (int j = 1; j < C; j++) m = max(m, key[j]);
        m = most<16>(m);
        // the levels of this one and the one before it: lane r - 1 holds that
        unsure |= sub == r - 1 && m >> 10 && (int)(chosen >> 10) - (int)(m >> 10) < apart;
        if (r == A.top_k) break;
        chosen = sub == r ? m : chosen;
#pragma unroll
        for (int j = 0; j < C; j++) key[j] = key[j] == m ? 0u : key[j];
    }
    int id = sub < A.top_k ? 1023 - (int)(chosen & 1023u) : 0;
    uint64_t again = __ballot(unsure && is);
    while (again) {
        const int t = __builtin_ctzll(again) / 16;
        again &= ~(0xFFFFull << (16 * t));
        const size_t from = (size_t)(first + t) * A.stride;
        float y[N];
        load<64, N>(A, from, lane, y);
        const int e = choose_exactly<N, GROUPS>(A, y, A.sigmoid ? 0.0f : top_of<64, N>(y), values[GROUPS ? wave : 0]);
        const int to = __shfl(e, sub);
        id = lane / 16 == t ? to : id;
    }
    finish<16>(A, is, at, row, sub, id, top, total);
}

// From so many tokens on four share a wave.  A wave per token : four (us, whole calls, f32 logits):
//   256 experts, 8 groups that count by two, a bias: 2048 tokens 6.8 : 14.9, 4096 12.1 : 11.0, 6000 11.4 : 11.1, 8192 15.4 : 12.2, 16384 23.3 : 15.9;
//   64 experts, 8 groups that count by two, a bias: 2048 5.5 : 6.6, 4096 8.2 : 6.8, 6000 8.3 : 6.9, 16384 16.5 : 7.8;
//   logits alone, 64 experts in 8 groups: 6000 7.0 : 7.4, 8192 8.4 : 9.4, 10000 9.7 : 7.7, 16384 13.5 : 8.6; 32 in 4: 6000 6.1 : 6.5, 10000 8.3 : 7.1;
//   128 experts without groups: 8192 6.8 : 8.9, 10000 7.9 : 7.5, 16384 11.0 : 9.1.
constexpr int FOURS_FROM = 6000, FOURS_FROM_PLAIN = 10000;

}  // namespace

hipError_t launch_moe_route(const Routing &r, hipStream_t s) {
    const bool groups = r.topk_group < r.n_group;
    auto few = [&](auto key, auto lanes, auto each) {
        constexpr int L = decltype(lanes)::value, N = decltype(each)::value;
        const int per = 4 * (64 / L);
        hipLaunchKernelGGL((k_moe_route_few<decltype(key), L, N>), dim3((r.n_tokens + per - 1) / per), dim3(256), 0, s, r);
    };
    auto whole = [&](auto each) {
        constexpr int N = decltype(each)::value;
        const dim3 g((r.n_tokens + 3) / 4), b(256);
        if (groups) hipLaunchKernelGGL((k_moe_route<N, true>), g, b, 0, s, r);
        else hipLaunchKernelGGL((k_moe_route<N, false>), g, b, 0, s, r);
    };
    auto fours = [&](auto each) {
        constexpr int C = decltype(each)::value;
        const int size = r.n_expert / r.n_group, lanes = size / C;
        if (groups && (size % C || (lanes & (lanes - 1)))) return false;
        const size_t bytes = r.dtype == T_F32 ? 4 : 2, piece = std::min((size_t)16, bytes * C);
        auto at = [](const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
        const bool whole = r.n_expert % C == 0;
        const int vec = (whole && at(r.logits, piece) && r.stride * bytes % piece == 0 ? 1 : 0) | (whole && at(r.bias, 16) ? 2 : 0);
        const dim3 g((r.n_tokens + 15) / 16), b(256);
        if (groups) hipLaunchKernelGGL((k_moe_route_fours<C, true>), g, b, 0, s, r, lanes, vec);
        else if constexpr (C > 4) hipLaunchKernelGGL((k_moe_route_fours<C, false>), g, b, 0, s, r, 1, vec);
        return true;
    };
    auto in_fours = [&] {
        if (r.n_tokens < (r.bias || (groups && r.group_top == 2) ? FOURS_FROM : FOURS_FROM_PLAIN) || r.top_k > 16) return false;
        if (r.n_expert <= 64) return groups && fours(std::integral_constant<int, 4>{});
        if (r.n_expert <= 128) return fours(std::integral_constant<int, 8>{});
        return r.n_expert <= 256 && fours(std::integral_constant<int, 16>{});
    };
    auto by_lanes = [&](auto lanes, auto each) {
        if (r.bias) few(uint64_t{}, lanes, each);
        else few(uint32_t{}, lanes, each);
    };
    if (!groups && r.n_expert <= 8) by_lanes(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{});
    else if (!groups && r.n_expert <= 64 && r.top_k <= 16) by_lanes(std::integral_constant<int, 16>{}, std::integral_constant<int, 4>{});
    else if (in_fours()) {}
    else if (r.n_expert <= 64) whole(std::integral_constant<int, 1>{});
    else if (r.n_expert <= 128) whole(std::integral_constant<int, 2>{});
    else if (r.n_expert <= 256) whole(std::integral_constant<int, 4>{});
    else if (r.n_expert <= 512) whole(std::integral_constant<int, 8>{});
    else whole(std::integral_constant<int, 16>{});
    return hipGetLastError();
}

}  // namespace rce_qmm
