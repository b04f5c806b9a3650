// kv_cache.hip -- the paged 8-bit KV cache: rows of keys and values appended
// (rotated, quantized) and read back (include/rce_qmm.h
// rce_qmm_kv_append_dev, rce_qmm_kv_read_dev).
//
// A block is 16 positions of one kv head, d_head codes each and one scale.
// Both kernels give a wave one block of the keys or of the values: the block's
// largest value is then a reduction inside the wave, and nothing is shared
// between waves.  The scale rule, in f32 with one rounding per operation:
//   d = max|x| / 127 over the call's new rows in the block (below 2^-126: 0),
//   s = d for a block written from its first slot, else max(old s, d),
//   code = rint(x * (1 / s)), earlier slots rint(code * (old s / s)).
// A block whose earlier slots are rescaled carries their rounding twice; the
// scale of a block filled by single tokens grows ln 16 times on average, so
// its error is about 1.4 times that of a block written at once (rms).
#include "kv_cache.h"

#include <type_traits>

namespace rce_qmm {
namespace {

constexpr float TINY = 0x1p-126f;

template <class T>
__device__ __forceinline__ float widen(T x) {
    return (float)x;
}
// bf16 travels as its bits
struct bf16_t {
    uint16_t u;
};
__device__ __forceinline__ float widen(bf16_t x) { return __uint_as_float((uint32_t)x.u << 16); }

// Four consecutive values; VEC: at a multiple of their size.
template <class T, bool VEC>
__device__ __forceinline__ void load4(const T *p, float (&x)[4]) {
    if constexpr (VEC) {
        struct alignas(4 * sizeof(T)) Quad {
            T t[4];
        };
        const Quad q = *reinterpret_cast<const Quad *>(p);
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = widen(q.t[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = widen(p[e]);
    }
}

// The block a wave writes: slots o .. o + n - 1 from the rows row0 ...
struct Task {
    size_t block;  // index in the pool's arrays
    int o, n, row0, pos0;
};

// Item `item` of the call's (sequence, touched block) list, for head h.
__device__ __forceinline__ bool find_block(const KvPool &P, const KvRows &B, int item, int h, Task &t) {
    int seq, idx;
    if (!kv_find(B, item, [&](const KvSeq &q) { return q.hi(B) > q.lo() ? ((q.hi(B) - 1) >> 4) - (q.lo() >> 4) + 1 : 0; },
                 seq, idx))
        return false;
    const KvSeq q = kv_seq(B, seq);
    const int b = (q.lo() >> 4) + idx;
    t.pos0 = max(q.lo(), b << 4);
    const int end = min(q.hi(B), (b + 1) << 4);
    t.o = t.pos0 & 15;
    t.n = end - t.pos0;
    t.row0 = q.r0 + (t.pos0 - q.first());
    const int page = B.pages[(size_t)seq * B.max_pages + (b >> P.lg_b)];
    if ((unsigned)page >= (unsigned)P.n_pages) return false;
    t.block = (((size_t)page * P.heads + h) << P.lg_b) + (b & ((1 << P.lg_b) - 1));
    return true;
}

// The block's new scale from the largest |x| of its new rows, and what its
// codes are formed with (0: codes 0).  NaN passes through.
struct Scale {
    float s, id, ratio;
    bool moved;  // earlier slots need new codes
};
__device__ __forceinline__ Scale new_scale(float amax, bool nan, float old) {
    Scale r;
    float d = nan ? __builtin_nanf("") : amax / 127.0f;
    if (d < TINY) d = 0.0f;
    r.s = old != old || d != d ? __builtin_nanf("") : fmaxf(old, d);
    const bool some = r.s > 0.0f && r.s < __builtin_inff();
    r.id = some ? 1.0f / r.s : 0.0f;
    r.ratio = some ? old / r.s : 0.0f;
    r.moved = !(r.s == old) || !some;
    return r;
}

__device__ __forceinline__ uint32_t code(float x, float f) {
    const float c = __builtin_rintf(x * f);  // NaN only where f is 0: code 0
    return (uint32_t)(int)fminf(fmaxf(c == c ? c : 0.0f, -127.0f), 127.0f) & 255u;
}
__device__ __forceinline__ float decode(uint32_t w, int e) { return (float)(int8_t)(w >> (8 * e)); }

// Keys: a lane holds four consecutive dimensions of a slot, U of them.
template <class T, int D, bool VEC>
__device__ __forceinline__ void append_keys(const KvPool &P, const Task &t, const T *__restrict__ src, size_t stride,
                                            const KvRope &rope) {
    constexpr int QD = D / 4, U = 16 * QD / 64;  // quads of a slot, per lane
    const int lane = threadIdx.x & 63;
    float x[U][4], y[U][4];
    const float old_s = t.o ? P.k_scale[t.block] : 0.0f;
#pragma unroll
    for (int i = 0; i < U; i++) {
        const int u = lane + 64 * i, j = u / QD - t.o;
#pragma unroll
        for (int e = 0; e < 4; e++) x[i][e] = 0.0f;
        if (j >= 0 && j < t.n) load4<T, VEC>(src + (size_t)(t.row0 + j) * stride + u % QD * 4, x[i]);
    }
    if (rope.cs) {
        const int half = rope.half;
#pragma unroll
        for (int i = 0; i < U; i++) {
            const int u = lane + 64 * i, j = u / QD - t.o, d = u % QD * 4;
            if (j < 0 || j >= t.n || d >= 2 * half) continue;
            const T *row = src + (size_t)(t.row0 + j) * stride;
            const float *cs = rope.cs + (size_t)(t.pos0 + j) * half * 2;
            if (VEC && (half & 3) == 0) {  // the quad's partners and its table entries are whole quads too
                const bool lo = d < half;
                const int k = lo ? d : d - half;
                load4<T, VEC>(row + (lo ? d + half : d - half), y[i]);
                float a[4], b[4];
                load4<float, VEC>(cs + 2 * k, a);
                load4<float, VEC>(cs + 2 * k + 4, b);
                const float c[4] = {a[0], a[2], b[0], b[2]}, s[4] = {a[1], a[3], b[1], b[3]};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float xc = x[i][e] * c[e], ys = y[i][e] * s[e];
                    x[i][e] = lo ? xc - ys : ys + xc;
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int dd = d + e;
                    if (dd >= 2 * half) continue;
                    const bool lo = dd < half;
                    const int k = lo ? dd : dd - half;
                    const float p = widen(row[lo ? dd + half : dd - half]);
                    const float xc = x[i][e] * cs[2 * k], ys = p * cs[2 * k + 1];
                    x[i][e] = lo ? xc - ys : ys + xc;
                }
            }
        }
    }
    float amax = 0.0f;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < U; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            amax = fmaxf(amax, fabsf(x[i][e]));
            nan |= x[i][e] != x[i][e];
        }
    const Scale sc = new_scale(wave_max(amax), __ballot(nan) != 0, old_s);
    uint32_t *dst = reinterpret_cast<uint32_t *>(P.k + t.block * (16 * D));
#pragma unroll
    for (int i = 0; i < U; i++) {
        const int u = lane + 64 * i, j = u / QD - t.o;
        if (j >= 0 && j < t.n) {
            uint32_t w = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) w |= code(x[i][e], sc.id) << (8 * e);
            dst[u] = w;
        } else if (j < 0 && sc.moved) {
            const uint32_t q = dst[u];
            uint32_t w = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) w |= code(decode(q, e), sc.ratio) << (8 * e);
            dst[u] = w;
        }
    }
    if (lane == 0) P.k_scale[t.block] = sc.s;
}

// Values: a lane holds the 16 slots of D / 64 dimensions, one 16-byte word of
// codes each.
template <class T, int D>
__device__ __forceinline__ void append_values(const KvPool &P, const Task &t, const T *__restrict__ src, size_t stride) {
    constexpr int U = D / 64;
    const int lane = threadIdx.x & 63;
    const float old_s = t.o ? P.v_scale[t.block] : 0.0f;
    uint4 *dst = reinterpret_cast<uint4 *>(P.v + t.block * (16 * D));
    float x[U][16];
    uint4 had[U];
    const bool whole = t.n == 16;
#pragma unroll
    for (int i = 0; i < U; i++) had[i] = whole ? make_uint4(0, 0, 0, 0) : dst[lane + 64 * i];
#pragma unroll
    for (int j = 0; j < 16; j++)
#pragma unroll
        for (int i = 0; i < U; i++) {
            x[i][j] = 0.0f;
            if (j >= t.o && j < t.o + t.n) x[i][j] = widen(src[(size_t)(t.row0 + j - t.o) * stride + lane + 64 * i]);
        }
    float amax = 0.0f;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < U; i++)
#pragma unroll
        for (int j = 0; j < 16; j++) {
            amax = fmaxf(amax, fabsf(x[i][j]));
            nan |= x[i][j] != x[i][j];
        }
    const Scale sc = new_scale(wave_max(amax), __ballot(nan) != 0, old_s);
#pragma unroll
    for (int i = 0; i < U; i++) {
        const uint32_t w[4] = {had[i].x, had[i].y, had[i].z, had[i].w};
        uint32_t r[4];
#pragma unroll
        for (int q = 0; q < 4; q++) {
            r[q] = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int j = 4 * q + e;
                uint32_t c = (w[q] >> (8 * e)) & 255u;
                if (j < t.o) c = sc.moved ? code(decode(w[q], e), sc.ratio) : c;
                else if (j < t.o + t.n) c = code(x[i][j], sc.id);
                r[q] |= c << (8 * e);
            }
        }
        dst[lane + 64 * i] = make_uint4(r[0], r[1], r[2], r[3]);
    }
    if (lane == 0) P.v_scale[t.block] = sc.s;
}

// Wave w of the grid: (block item, head, keys or values).
template <class T, int D>
__global__ __launch_bounds__(256) void k_kv_append(KvPool P, KvRows B, const T *__restrict__ k, size_t k_stride,
                                                   const T *__restrict__ v, size_t v_stride, int vec, KvRope rope) {
    const unsigned task = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    const int item = task / (2 * P.heads), rest = task - item * (2 * P.heads), h = rest >> 1;
    Task t;
    if (!find_block(P, B, item, h, t)) return;
    if (rest & 1) append_values<T, D>(P, t, v + (size_t)h * D, v_stride);
    else if (vec) append_keys<T, D, true>(P, t, k + (size_t)h * D, k_stride, rope);
    else append_keys<T, D, false>(P, t, k + (size_t)h * D, k_stride, rope);
}

// x, a product rounded to f32, in T: the empty asm keeps the two roundings
// apart (else product and conversion become one v_fma_mix instruction, in
// some places and not in others).
template <class T>
__device__ __forceinline__ T narrow(float x) {
    asm("" : "+v"(x));
    return (T)x;
}
template <>
__device__ __forceinline__ bf16_t narrow<bf16_t>(float x) {
    const uint32_t u = __float_as_uint(x);
    return bf16_t{(uint16_t)(x != x ? 0x7FC0u : (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16)};
}

// One block's slots of the batch's rows: out[row][head][dimension].
template <class T, int D>
__global__ __launch_bounds__(256) void k_kv_read(KvPool P, KvRows B, T *__restrict__ k, T *__restrict__ v) {
    const unsigned task = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    const int item = task / (2 * P.heads), rest = task - item * (2 * P.heads), h = rest >> 1, lane = threadIdx.x & 63;
    T *out = rest & 1 ? v : k;
    Task t;
    if (!out || !find_block(P, B, item, h, t)) return;
    out += ((size_t)t.row0 * P.heads + h) * D;
    const size_t row = (size_t)P.heads * D;
    if (rest & 1) {
        const float s = P.v_scale[t.block];
        const uint4 *src = reinterpret_cast<const uint4 *>(P.v + t.block * (16 * D));
#pragma unroll
        for (int i = 0; i < D / 64; i++) {
            const uint4 q = src[lane + 64 * i];
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int j = 0; j < 16; j++)
                if (j >= t.o && j < t.o + t.n)
                    out[(size_t)(j - t.o) * row + lane + 64 * i] = narrow<T>(decode(w[j >> 2], j & 3) * s);
        }
        return;
    }
    constexpr int QD = D / 4;
    const float s = P.k_scale[t.block];
    const uint32_t *src = reinterpret_cast<const uint32_t *>(P.k + t.block * (16 * D));
#pragma unroll
    for (int i = 0; i < 16 * QD / 64; i++) {
        const int u = lane + 64 * i, j = u / QD - t.o;
        if (j < 0 || j >= t.n) continue;
        const uint32_t w = src[u];
#pragma unroll
        for (int e = 0; e < 4; e++) out[(size_t)j * row + u % QD * 4 + e] = narrow<T>(decode(w, e) * s);
    }
}

// Touched blocks of a call, at most: a sequence of r rows touches up to
// r / 16 + 2 blocks and up to r.
size_t max_blocks(const KvRows &B) {
    const size_t r = (size_t)B.n_rows, n = (size_t)B.n_seqs;
    return r < r / 16 + 2 * n ? r : r / 16 + 2 * n;
}

template <class F>
hipError_t by_head_size(int d, F f) {
    switch (d) {
    case 64: f(std::integral_constant<int, 64>{}); break;
    case 128: f(std::integral_constant<int, 128>{}); break;
    case 192: f(std::integral_constant<int, 192>{}); break;
    case 256: f(std::integral_constant<int, 256>{}); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_append(const KvPool &pool, const KvRows &rows, int d_head, const void *k, size_t k_stride,
                            const void *v, size_t v_stride, uint32_t dtype, const KvRope &rope, hipStream_t s) {
    const size_t tasks = max_blocks(rows) * pool.heads * 2;
    if (!tasks) return hipSuccess;
    const dim3 grid((unsigned)((tasks + 3) / 4));
    return by_head_size(d_head, [&](auto d) {
        constexpr int D = decltype(d)::value;
        auto go = [&](auto *p) {
            using T = std::remove_pointer_t<decltype(p)>;
            const int vec = k_stride % 4 == 0 && reinterpret_cast<uintptr_t>(k) % (4 * sizeof(T)) == 0 &&
                            reinterpret_cast<uintptr_t>(rope.cs) % 16 == 0;
            hipLaunchKernelGGL((k_kv_append<T, D>), grid, dim3(256), 0, s, pool, rows, static_cast<const T *>(k), k_stride,
                               static_cast<const T *>(v), v_stride, vec, rope);
        };
        if (dtype == T_F32) go((float *)nullptr);
        else if (dtype == T_F16) go((_Float16 *)nullptr);
        else go((bf16_t *)nullptr);
    });
}

hipError_t launch_kv_read(const KvPool &pool, const KvRows &rows, int d_head, void *k, void *v, uint32_t dtype,
                          hipStream_t s) {
    const size_t tasks = max_blocks(rows) * pool.heads * 2;
    if (!tasks) return hipSuccess;
    const dim3 grid((unsigned)((tasks + 3) / 4));
    return by_head_size(d_head, [&](auto d) {
        constexpr int D = decltype(d)::value;
        auto go = [&](auto *p) {
            using T = std::remove_pointer_t<decltype(p)>;
            hipLaunchKernelGGL((k_kv_read<T, D>), grid, dim3(256), 0, s, pool, rows, static_cast<T *>(k),
                               static_cast<T *>(v));
        };
        if (dtype == T_F32) go((float *)nullptr);
        else if (dtype == T_F16) go((_Float16 *)nullptr);
        else go((bf16_t *)nullptr);
    });
}

}  // namespace rce_qmm
