// qk_rope.hip -- norms of query and key heads and their rotation in one pass
// (include/rce_qmm.h rce_qmm_qk_norm_rope_dev).
//
// A head of d values x becomes x / sqrt(mean x^2 + eps) * w, in f32, and its
// first 2 * half values turn in pairs (a, b) -> (a c - b s, a s + b c); one
// rounding at the end.  Every value is read and written once: memory bounds it (5 x up to 2500 rows of 40 heads of 128, f16: 152 MB in 30 us,
// as a copy of as much; 37 where the results go through the L2s).  Several chunks of heads to a wave measured the same.
//
// A lane holds two pieces of 8 values (16 or 32 bytes each), d / 16 lanes a
// head.  Where pairs are (i, i + half) the pieces are `half` values apart, so
// that no value of a pair is another lane's.  What does not fit that (heads not
// of 16 values, rotated parts not of 16, addresses not of 16 bytes) goes value by value,
// a wave to a head: 40 heads of 80, f16, 5 x up to 2500 rows with 20 values of each rotated as halves take 112 us, with all 80 (by pieces) 22.
#include "qk_rope.h"

#include <algorithm>

namespace rce_qmm {
namespace {

struct bf16_t {
    uint16_t u;
};
__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(_Float16 x) { return (float)x; }
__device__ __forceinline__ float widen(bf16_t x) { return __uint_as_float((uint32_t)x.u << 16); }
__device__ __forceinline__ void narrow(float &o, float x) { o = x; }
__device__ __forceinline__ void narrow(_Float16 &o, float x) { o = (_Float16)x; }
__device__ __forceinline__ void narrow(bf16_t &o, float x) {
    const uint32_t u = __float_as_uint(x);
    o.u = x != x ? (uint16_t)0x7FC0u : (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}

// The sum over the lanes of an aligned group of `lanes` (a power of two, the same in all lanes), in all of them.
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ float sum_over(float v, int lanes) {
    if (lanes > 1) v += dpp<0xB1>(v);   // quad_perm [1,0,3,2]
    if (lanes > 2) v += dpp<0x4E>(v);   // quad_perm [2,3,0,1]
    if (lanes > 4) v += dpp<0x141>(v);  // row_half_mirror: the other quad of the 8
    if (lanes > 8) v += dpp<0x140>(v);  // row_mirror
    if (lanes > 16) {
        const unsigned u = __float_as_uint(v);
        const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if (lanes > 32) {
        const unsigned u = __float_as_uint(v);
        const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return v;
}

// The position of row r; below 0: none.  The whole wave calls it: 64 sequences' ends a step.
__device__ __forceinline__ int position_of(const QkNormRope &A, int r) {
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = A.rows.n_seqs;  // sequences below lo end at or before r, those from hi on behind it
    while (lo < hi) {
        const int step = (hi - lo + 63) / 64, at = lo + lane * step;
        const int n = __popcll(__ballot(at < hi && A.rows.offsets[min(at, hi - 1) + 1] <= r));
        if (!n) break;
        hi = min(hi, lo + n * step);
        lo += (n - 1) * step + 1;
    }
    if (lo >= A.rows.n_seqs) return -1;
    const KvSeq q = kv_seq(A.rows, lo);
    const int pos = q.len - (q.r1 - r);
    return r >= q.r0 && r < q.r1 && (!A.rope.cs || pos < A.n_pos) ? pos : -1;
}

// A head whose mean square and eps together are below TINY: its squares leave binary32's normal numbers, and the root's reciprocal
// takes a subnormal number for 0.  Its values are times TINY_UP first, eps times that twice, which cancels: values below 2^-45 come
// to less than 2^59, a head's squares to less than 2^118, and the least subnormal value's square to 2^-90.
constexpr float TINY = 0x1p-100f, TINY_UP = 0x1p104f;

template <class T>
struct alignas(16) Piece {
    T t[8];
};

// PAST: results that the caches cannot hold are written past them.
template <bool PAST, class T>
__device__ __forceinline__ void put(T *p, const Piece<T> &o) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    const u32x4 *from = reinterpret_cast<const u32x4 *>(&o);
    u32x4 *to = reinterpret_cast<u32x4 *>(p);
#pragma unroll
    for (int i = 0; i < (int)sizeof(o) / 16; i++) {
        if constexpr (PAST) __builtin_nontemporal_store(from[i], to + i);
        else to[i] = from[i];
    }
}

template <class TI, class TO, bool PAST>
__global__ __launch_bounds__(256) void k_qk_norm_rope(QkNormRope A, int lanes, int chunks) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int unit = blockIdx.x * 4 + wave;
    const int r = unit / chunks;
    if (r >= A.rows.n_rows) return;
    const int sub = lane & (lanes - 1), used = A.d / 16;
    const int head = (unit - r * chunks) * (64 / lanes) + lane / lanes;
    const bool is = head < A.q.n + A.k.n && sub < used;
    const bool key = head >= A.q.n;
    const int h = is ? key ? head - A.q.n : head : 0;
    const int turned = A.interleaved ? 0 : A.rope.half / 8;  // lanes whose pieces are pairs
    const int c0 = !is ? 0 : sub < turned ? sub : turned + sub;
    const int c1 = !is ? 0 : sub < turned ? sub + turned : c0 + used - turned;
    const size_t head_at = (size_t)h * A.d;
    const bool of_k = is ? key : !A.q.n;
    const TI *in = static_cast<const TI *>(of_k ? A.k.in : A.q.in) + (size_t)r * (of_k ? A.k.in_stride : A.q.in_stride) + head_at;
    const Piece<TI> p0 = *reinterpret_cast<const Piece<TI> *>(in + 8 * c0), p1 = *reinterpret_cast<const Piece<TI> *>(in + 8 * c1);
    const float *w = of_k ? A.k.weight : A.q.weight;
    const int pos = position_of(A, r);
    if (pos < 0) return;
    float x[2][8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        x[0][i] = widen(p0.t[i]);
        x[1][i] = widen(p1.t[i]);
    }
    if (A.eps >= 0.0f) {
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
            for (int i = 0; i < 8; i++) s = __builtin_fmaf(x[e][i], x[e][i], s);
        s = sum_over(is ? s : 0.0f, lanes);
        float m = s * (1.0f / (float)A.d) + A.eps;
        if (__ballot(m < TINY)) {
            const float up = m < TINY ? TINY_UP : 1.0f;
            s = 0.0f;
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    x[e][i] *= up;
                    s = __builtin_fmaf(x[e][i], x[e][i], s);
                }
            m = sum_over(is ? s : 0.0f, lanes) * (1.0f / (float)A.d) + A.eps * up * up;
        }
        const float f = __builtin_amdgcn_rsqf(m);
        float y[2][8];
#pragma unroll
        for (int i = 0; i < 8; i++) y[0][i] = y[1][i] = 1.0f;
        if (w) {
            const Piece<float> w0 = *reinterpret_cast<const Piece<float> *>(w + 8 * c0), w1 = *reinterpret_cast<const Piece<float> *>(w + 8 * c1);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                y[0][i] = w0.t[i];
                y[1][i] = w1.t[i];
            }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            x[0][i] *= f * y[0][i];
            x[1][i] *= f * y[1][i];
        }
    }
    if (A.rope.cs) {
        const float *cs = A.rope.cs + (size_t)pos * A.rope.half * 2;
        if (!A.interleaved) {
            if (sub < turned) {
                const Piece<float> t0 = *reinterpret_cast<const Piece<float> *>(cs + 16 * c0), t1 = *reinterpret_cast<const Piece<float> *>(cs + 16 * c0 + 8);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float c = i < 4 ? t0.t[2 * (i & 3)] : t1.t[2 * (i & 3)], s = i < 4 ? t0.t[2 * (i & 3) + 1] : t1.t[2 * (i & 3) + 1];
                    const float a = x[0][i], b = x[1][i];
                    x[0][i] = a * c - b * s;
                    x[1][i] = a * s + b * c;
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int c8 = e ? c1 : c0;
                if (4 * c8 < A.rope.half) {
                    const Piece<float> t = *reinterpret_cast<const Piece<float> *>(cs + 8 * c8);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float a = x[e][2 * i], b = x[e][2 * i + 1];
                        x[e][2 * i] = a * t.t[2 * i] - b * t.t[2 * i + 1];
                        x[e][2 * i + 1] = a * t.t[2 * i + 1] + b * t.t[2 * i];
                    }
                }
            }
        }
    }
    if (!is) return;
    TO *out = static_cast<TO *>(of_k ? A.k.out : A.q.out) + (size_t)r * (of_k ? A.k.out_stride : A.q.out_stride) + head_at;
    Piece<TO> o0, o1;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        narrow(o0.t[i], x[0][i]);
        narrow(o1.t[i], x[1][i]);
    }
    put<PAST>(out + 8 * c0, o0);
    put<PAST>(out + 8 * c1, o1);
}

// Any head: a wave takes one, a lane the pairs lane + 64 j of the rotated part and of what is behind it
// (neighbours there), so that a head written where it was read is safe.
template <class TI, class TO>
__global__ __launch_bounds__(256) void k_qk_norm_rope_any(QkNormRope A) {
    constexpr int J = QK_HEAD / 128;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int heads = A.q.n + A.k.n;
    const int64_t unit = (int64_t)blockIdx.x * 4 + wave;
    const int r = (int)(unit / heads), head = (int)(unit - (int64_t)r * heads);
    if (r >= A.rows.n_rows) return;
    const int pos = position_of(A, r);
    if (pos < 0) return;
    const QkHeads &H = head < A.q.n ? A.q : A.k;
    const size_t head_at = (size_t)(head < A.q.n ? head : head - A.q.n) * A.d;
    const TI *in = static_cast<const TI *>(H.in) + (size_t)r * H.in_stride + head_at;
    TO *out = static_cast<TO *>(H.out) + (size_t)r * H.out_stride + head_at;
    const int half = A.rope.cs ? A.rope.half : 0;
    float a[J], b[J], s = 0.0f;
    auto first = [&](int p) { return p < half && !A.interleaved ? p : 2 * p; };
    auto second = [&](int p) { return p < half && !A.interleaved ? p + half : 2 * p + 1; };
#pragma unroll
    for (int j = 0; j < J; j++) {
        const int p = lane + 64 * j;
        const bool is = p < A.d / 2;
        a[j] = is ? widen(in[first(p)]) : 0.0f;
        b[j] = is ? widen(in[second(p)]) : 0.0f;
        s = __builtin_fmaf(b[j], b[j], __builtin_fmaf(a[j], a[j], s));
    }
    float f = 1.0f;
    if (A.eps >= 0.0f) {
        float m = sum_over(s, 64) * (1.0f / (float)A.d) + A.eps;
        if (m < TINY) {  // the same in all lanes
            s = 0.0f;
#pragma unroll
            for (int j = 0; j < J; j++) {
                a[j] *= TINY_UP;
                b[j] *= TINY_UP;
                s = __builtin_fmaf(b[j], b[j], __builtin_fmaf(a[j], a[j], s));
            }
            m = sum_over(s, 64) * (1.0f / (float)A.d) + A.eps * TINY_UP * TINY_UP;
        }
        f = __builtin_amdgcn_rsqf(m);
    }
#pragma unroll
    for (int j = 0; j < J; j++) {
        const int p = lane + 64 * j;
        if (p >= A.d / 2) break;
        const int i0 = first(p), i1 = second(p);
        if (A.eps >= 0.0f) {
            a[j] *= f * (H.weight ? H.weight[i0] : 1.0f);
            b[j] *= f * (H.weight ? H.weight[i1] : 1.0f);
        }
        if (p < half) {
            const float *cs = A.rope.cs + ((size_t)pos * half + p) * 2;
            const float c = cs[0], t = cs[1], x = a[j], y = b[j];
            a[j] = x * c - y * t;
            b[j] = x * t + y * c;
        }
        TO o;
        narrow(o, a[j]);
        out[i0] = o;
        narrow(o, b[j]);
        out[i1] = o;
    }
}

// Bytes of results that the L2s (32 MB) do not hold for the next call anyway.
constexpr size_t PAST_FROM = (size_t)32 << 20;

bool of_pieces(const QkHeads &h, size_t in_size, size_t out_size) {
    auto ok = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    return !h.n || (ok(h.in) && ok(h.out) && ok(h.weight) && h.in_stride * in_size % 16 == 0 && h.out_stride * out_size % 16 == 0);
}

}  // namespace

hipError_t launch_qk_norm_rope(const QkNormRope &c, hipStream_t s) {
    const size_t in_size = c.in_dtype == T_F32 ? 4 : 2, out_size = c.out_dtype == T_F32 ? 4 : 2;
    const int heads = c.q.n + c.k.n;
    const bool pieces = c.d % 16 == 0 && of_pieces(c.q, in_size, out_size) && of_pieces(c.k, in_size, out_size) &&
                        (!c.rope.cs || (reinterpret_cast<uintptr_t>(c.rope.cs) % 16 == 0 && c.rope.half % (c.interleaved ? 4 : 8) == 0));
    int lanes = 1;
    while (lanes * 16 < c.d) lanes *= 2;
    const int chunks = (heads + 64 / lanes - 1) / (64 / lanes);
    const size_t units = (size_t)c.rows.n_rows * (pieces ? chunks : heads);
    const dim3 g((unsigned)((units + 3) / 4)), b(256);
    const bool past = (size_t)c.rows.n_rows * heads * c.d * out_size >= PAST_FROM;
    auto go = [&](auto ti, auto to) {
        typedef decltype(ti) TI;
        typedef decltype(to) TO;
        if (pieces && past) hipLaunchKernelGGL((k_qk_norm_rope<TI, TO, true>), g, b, 0, s, c, lanes, chunks);
        else if (pieces) hipLaunchKernelGGL((k_qk_norm_rope<TI, TO, false>), g, b, 0, s, c, lanes, chunks);
        else hipLaunchKernelGGL((k_qk_norm_rope_any<TI, TO>), g, b, 0, s, c);
    };
    auto out = [&](auto ti) {
        if (c.out_dtype == T_F32) go(ti, float{});
        else if (c.out_dtype == T_F16) go(ti, _Float16{});
        else go(ti, bf16_t{});
    };
    if (c.in_dtype == T_F32) out(float{});
    else if (c.in_dtype == T_F16) out(_Float16{});
    else out(bf16_t{});
    return hipGetLastError();
}

}  // namespace rce_qmm
