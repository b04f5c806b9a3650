// moe_route.hip -- routing of tokens to experts (include/rce_qmm.h
// rce_qmm_moe_route_dev).
//
// L lanes take a token, N experts each (expert lane + L j), 64 / L tokens to a
// wave; waves share nothing.  A round takes the largest key of the lanes' own
// largest ones, the lowest expert among equals, and takes it away; round r's
// expert goes to lane r, which weighs it at the end.
//
// Without a bias the order of the scores is that of the logits, whatever the
// scores round to: keys are the logits as 32-bit whole numbers.  A bias is added
// to scores of 64 bits, and groups that count by two experts are compared by
// sums of 64 bits: neighbours in 16-bit logits differ by 2^-8 of a score, but a
// score of 32 bits plus a bias would make equals of what is not.
#include "moe_route.h"

#include <type_traits>

namespace rce_qmm {
namespace {

// v of the lane that CTRL names.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xF, 0xF, false);
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
__device__ __forceinline__ double sum_of(double x) {
#pragma unroll
    for (int o = 1; o < L; o *= 2) x += __shfl_xor(x, o);
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
constexpr uint32_t NONE32 = 0x007FFFFFu;                 // ordered(-inf)
constexpr uint64_t NONE64 = 0x000FFFFFFFFFFFFFull;

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

template <class K>
struct GroupValue {
    typedef double type;
};
template <>
struct GroupValue<uint32_t> {
    typedef uint32_t type;
};

// K: uint32_t without a bias and with groups by their best expert (or none), else uint64_t.
template <class K, int L, int N, bool GROUPS>
__global__ __launch_bounds__(256) void k_moe_route(Routing A) {
    static_assert(!GROUPS || L == 64, "a token with groups takes a wave");
    constexpr bool WIDE = std::is_same<K, uint64_t>::value;
    typedef typename GroupValue<K>::type V;
    const int lane = threadIdx.x & 63, sub = lane & (L - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t at = ((int64_t)blockIdx.x * 4 + wave) * (64 / L) + lane / L;
    const bool is = at < A.n_tokens;
    const size_t row = (size_t)(is ? at : 0) * A.stride;

    float x[N];
#pragma unroll
    for (int j = 0; j < N; j++) {
        const int e = sub + L * j;
        x[j] = logit(A.logits, A.dtype, row + min(e, A.n_expert - 1));
        if (e >= A.n_expert) x[j] = -__builtin_inff();
    }
    float top = x[0];
#pragma unroll
    for (int j = 1; j < N; j++) top = fmaxf(top, x[j]);
    const uint32_t t32 = most<L>(ordered(top));
    top = __uint_as_float(t32 & 0x80000000u ? t32 & 0x7FFFFFFFu : ~t32);
    // the softmax's sum, where something needs it
    double total = 1.0;
    if (!A.sigmoid && (WIDE || !A.normalize)) {
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < N; j++) sum += sub + L * j >= A.n_expert ? 0.0 : x[j] == top ? 1.0 : exp((double)x[j] - (double)top);
        total = sum_of<L>(sum);
    }

    K key[N];
    V value[N];  // what groups go by
#pragma unroll
    for (int j = 0; j < N; j++) {
        const int e = sub + L * j;
        if constexpr (WIDE) {
            const float b = A.bias ? A.bias[min(e, A.n_expert - 1)] : 0.0f;
            double s = score_of(A.sigmoid, x[j], top, total) + (double)b;
            if (x[j] == -__builtin_inff() || s != s) s = -__builtin_inf();
            value[j] = s;
            key[j] = ordered(A.bias ? s : (double)x[j]);
        } else {
            value[j] = key[j] = ordered(x[j]);
        }
        if (e >= A.n_expert) key[j] = 0;
    }

    if constexpr (GROUPS) {
        __shared__ V values[4][L * N];
        V *v = values[wave];
#pragma unroll
        for (int j = 0; j < N; j++) v[sub + L * j] = value[j];
        __syncthreads();
        // P lanes to a group: its two largest values
        const V none = WIDE ? (V)-__builtin_inf() : (V)NONE32;
        const int size = A.n_expert / A.n_group;
        int lg = 6;  // P = 1 << lg
        while ((A.n_group << lg) > 64) lg--;
        const int P = 1 << lg, g = lane >> lg;
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
        if constexpr (WIDE)
            if (A.group_top == 2 && b > none) a += b;
        int rank = 0;
        for (int i = 0; i < A.n_group; i++) {
            const V o = __shfl(a, i << lg);
            rank += o > a || (o == a && i < g);
        }
        const uint64_t kept = __ballot(g < A.n_group && rank < A.topk_group);
        const float per = 1.0f / (float)size;
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int eg = (int)(((float)(sub + L * j) + 0.5f) * per);  // exact up to 1024 experts
            if (!(kept >> ((eg << lg) & 63) & 1)) key[j] = 0;
        }
    }

    int id = 0;
    bool some = false;
    for (int r = 0; r < A.top_k; r++) {
        K best = key[0];
        int e = sub;
#pragma unroll
        for (int j = 1; j < N; j++) {
            e = key[j] > best ? sub + L * j : e;
            best = key[j] > best ? key[j] : best;
        }
        bool mine;
        bool weighs;
        if constexpr (WIDE) {
            const uint32_t hi = (uint32_t)(best >> 32), top_hi = most<L>(hi);
            const uint32_t lo = hi == top_hi ? (uint32_t)best : 0u, top_lo = most<L>(lo);
            mine = hi == top_hi && lo == top_lo;
            weighs = ((uint64_t)top_hi << 32 | top_lo) > NONE64;
        } else {
            const uint32_t m = most<L>(best);
            mine = best == m;
            weighs = m > NONE32;
        }
        const int win = (int)least<L>(mine ? (uint32_t)e : ~0u);
        if (sub == r) {
            id = win;
            some = weighs;
        }
#pragma unroll
        for (int j = 0; j < N; j++)
            if (win == sub + L * j) key[j] = 0;
    }
    double w = 0.0;
    if (some) w = score_of(A.sigmoid, logit(A.logits, A.dtype, row + id), top, total);
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

}  // namespace

hipError_t launch_moe_route(const Routing &r, hipStream_t s) {
    auto go = [&](auto key, auto lanes, auto each, auto groups) {
        constexpr int L = decltype(lanes)::value, N = decltype(each)::value;
        const int per = 4 * (64 / L);
        hipLaunchKernelGGL((k_moe_route<decltype(key), L, N, decltype(groups)::value>), dim3((r.n_tokens + per - 1) / per), dim3(256), 0, s, r);
    };
    auto whole = [&](auto key, auto groups) {  // a wave per token
        const auto l = std::integral_constant<int, 64>{};
        if (r.n_expert <= 64) go(key, l, std::integral_constant<int, 1>{}, groups);
        else if (r.n_expert <= 128) go(key, l, std::integral_constant<int, 2>{}, groups);
        else if (r.n_expert <= 256) go(key, l, std::integral_constant<int, 4>{}, groups);
        else if (r.n_expert <= 512) go(key, l, std::integral_constant<int, 8>{}, groups);
        else go(key, l, std::integral_constant<int, 16>{}, groups);
    };
    auto pick = [&](auto key) {
        const bool groups = r.topk_group < r.n_group;
        if (groups) whole(key, std::true_type{});
        else if (r.n_expert <= 8) go(key, std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{}, std::false_type{});
        else if (r.n_expert <= 64 && r.top_k <= 16) go(key, std::integral_constant<int, 16>{}, std::integral_constant<int, 4>{}, std::false_type{});
        else whole(key, std::false_type{});
    };
    if (r.bias || (r.topk_group < r.n_group && r.group_top == 2)) pick(uint64_t{});
    else pick(uint32_t{});
    return hipGetLastError();
}

}  // namespace rce_qmm
