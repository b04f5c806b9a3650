// kv_attention.hip -- causal attention of ragged query rows over the paged
// 8-bit KV cache (include/rce_qmm.h rce_qmm_kv_attention_dev).
//
// A unit is 16 query rows of one sequence and kv head: row r of the unit is
// query head r % G of token r / G, G the query heads per kv head (one token of
// up to 16 heads, or several tokens).  Its keys are cut into ranges of `chunk`
// tiles of 64 positions; a block takes one range, its four waves every fourth
// tile, and joins the waves' (m, l, o) in LDS.  A unit of one range is
// finished there; the ranges of a longer one leave (m, l, o) in `parts`, which
// k_kv_join adds up in range order.
//
// Every block plans for itself: it reads the sequences' lengths (device
// memory, no host round trip), forms the total of tiles and from it the chunk
// that spreads them over TARGET blocks, and finds its own range.
//
// A tile of a wave, all on the matrix cores, with no exchange between lanes
// but the maximum over the keys (n = lane % 16 a query row, g = lane / 16 one
// of the tile's four 16-position blocks):
//   S^T = K Q^T   (int8, 16x16x64, exact int32): operand row m of MFMA t is
//                 position 16 (m / 4) + 4 t + m % 4, so that lane (n, g)
//                 gets the scores of positions 16 g + 4 t + i: all 16 of
//                 block g, which share one key scale and one value scale.
//   Q             as LIMBS signed bytes per value of one whole number
//                 rint(q * QMAX / max|q|) (2: 15 bits, 3: 22 bits).
//   O^T += V^T P^T (binary16, 16x16x32): P^T is the lane's own scores in order
//                 (k slot 8 g + j of MFMA u is position 16 g + 8 u + j), V^T the
//                 value codes as stored, 16 positions of a dimension in a
//                 word.  P carries its block's value scale relative to the
//                 tile's largest, times 2^14 (so that small weights stay
//                 normal in binary16); HILO adds a second binary16 term.
#include "kv_cache.h"

#include <climits>
#include <type_traits>

#include "mfma_util.h"

namespace rce_qmm {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int ROWS = 16;    // query rows of a unit
constexpr int WAVES = 4;    // of a block
constexpr int TILE = 64;    // positions of a wave's step
constexpr int TARGET = 512;   // blocks that a call's tiles are spread over (two per CU)
constexpr int MIN_CHUNK = 8;  // tiles of the shortest range

constexpr float LOG2E = 1.4426950408889634f;

struct Args {
    KvPool P;
    KvRows B;
    KvAttention a;
    int G;  // query heads per kv head
};

// The units of a sequence (per kv head) and the tiles of its longest one.
struct Span {
    int units, t0, tiles;
};
__device__ __forceinline__ Span span_of(const Args &A, const KvSeq &q) {
    Span s;
    s.units = (int)(((long long)(q.r1 - q.r0) * A.G + ROWS - 1) / ROWS);
    const int lo = max(0, q.lo() - (A.a.window - 1));
    s.t0 = lo / TILE;
    s.tiles = q.hi(A.B) > q.lo() ? (q.hi(A.B) + TILE - 1) / TILE - s.t0 : 0;
    return s;
}

// Tiles per range, the same in every block of the call.
__device__ __forceinline__ int chunk_of(const Args &A) {
    const int lane = threadIdx.x & 63;
    float total = 0.0f;  // only a size: its rounding moves no result
    for (int s = lane; s < A.B.n_seqs; s += 64) {
        const Span p = span_of(A, kv_seq(A.B, s));
        total += (float)p.units * (float)p.tiles;
    }
    total = wave_sum(total) * (float)A.P.heads;
    return max(MIN_CHUNK, (int)fminf(ceilf(total / (float)TARGET), 1e9f));
}

__device__ __forceinline__ int ranges(int tiles, int chunk) { return tiles ? (tiles + chunk - 1) / chunk : 1; }

// A unit's split ranges are numbered within the call: parts slot (range number * heads + head).
struct Work {
    KvSeq q;
    Span sp;
    int seq, unit, range, n_ranges, slot;  // slot of the unit's range 0, before the head
};

// Range `item` of the list (sequence, unit, range).
__device__ __forceinline__ bool find_work(const Args &A, int item, int chunk, Work &w) {
    const int lane = threadIdx.x & 63;
    int run = 0, srun = 0;
    for (int base = 0; base < A.B.n_seqs; base += 64) {
        const int s = base + lane;
        int c = 0, sc = 0;
        if (s < A.B.n_seqs) {
            const Span p = span_of(A, kv_seq(A.B, s));
            const int n = ranges(p.tiles, chunk);
            c = p.units * n;
            sc = n > 1 ? c : 0;
        }
        const int incl = wave_scan(c), sincl = wave_scan(sc);
        const int total = __builtin_amdgcn_readlane(incl, 63);
        if (item < run + total) {
            const int l = __builtin_ctzll(__ballot(item < run + incl));
            const int at = item - run - __builtin_amdgcn_readlane(incl - c, l);
            w.seq = base + l;
            w.q = kv_seq(A.B, w.seq);
            w.sp = span_of(A, w.q);
            w.n_ranges = ranges(w.sp.tiles, chunk);
            w.unit = at / w.n_ranges;
            w.range = at - w.unit * w.n_ranges;
            w.slot = srun + __builtin_amdgcn_readlane(sincl - sc, l) + w.unit * w.n_ranges;
            return true;
        }
        run += total;
        srun += __builtin_amdgcn_readlane(sincl, 63);
    }
    return false;
}

__device__ __forceinline__ float swap_max(float x) {  // over the lanes with the same lane % 16
    const unsigned u = __builtin_bit_cast(unsigned, x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const float y = fmaxf(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
    const unsigned w = __builtin_bit_cast(unsigned, y);
    const auto q = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return fmaxf(__builtin_bit_cast(float, (unsigned)q[0]), __builtin_bit_cast(float, (unsigned)q[1]));
}
__device__ __forceinline__ float swap_sum(float x) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const float y = __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
    const unsigned w = __builtin_bit_cast(unsigned, y);
    const auto q = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return __builtin_bit_cast(float, (unsigned)q[0]) + __builtin_bit_cast(float, (unsigned)q[1]);
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ float load_any(const void *p, uint32_t t, size_t i) {
    if (t == T_F32) return static_cast<const float *>(p)[i];
    if (t == T_F16) return (float)static_cast<const _Float16 *>(p)[i];
    return __uint_as_float((uint32_t)static_cast<const uint16_t *>(p)[i] << 16);
}
__device__ __forceinline__ void store_any(void *p, uint32_t t, size_t i, float x) {
    if (t == T_F32) static_cast<float *>(p)[i] = x;
    else if (t == T_F16) static_cast<_Float16 *>(p)[i] = (_Float16)x;
    else {
        const uint32_t u = __float_as_uint(x);
        static_cast<uint16_t *>(p)[i] = (uint16_t)(x != x ? 0x7FC0u : (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
    }
}

// Four codes as two binary16 pairs: bytes offset to 0 .. 255 become the low
// byte of 1024 + b, minus 1152.  Exact.
__device__ __forceinline__ void codes4(uint32_t x, half2v &lo, half2v &hi) {
    const uint32_t b = x ^ 0x80808080u;
    const half2v off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    lo = as_h2(__builtin_amdgcn_perm(b, 0x64646464u, 0x00050004u)) + off;
    hi = as_h2(__builtin_amdgcn_perm(b, 0x64646464u, 0x00070006u)) + off;
}

// LDS: the query rows in f32 before the loop, the waves' results after it (at
// most 128 dimensions at a time: 34 KB).
template <int D>
struct Shared {
    static constexpr int PART = D <= 128 ? D : D / 2;
    union {
        alignas(16) float q[ROWS][D + 4];
        alignas(16) float o[WAVES][ROWS][PART + 4];
    };
    float m[WAVES][ROWS], l[WAVES][ROWS];
};

template <int D, bool HILO>
__global__ __launch_bounds__(64 * WAVES) void k_kv_attention(Args A) {
    constexpr int NQ = D / 64, NT = D / 16;
    constexpr int LIMBS = HILO ? 3 : 2;
    constexpr float QMAX = HILO ? 127.0f * 65536.0f : 127.0f * 256.0f;
    __shared__ Shared<D> sh;
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = blockIdx.x % A.P.heads;
    const int chunk = chunk_of(A);
    Work w;
    if (!find_work(A, blockIdx.x / A.P.heads, chunk, w)) return;
    const KvSeq &q = w.q;
    const int G = A.G, first = q.first();
    const int x0 = w.unit * ROWS, n_x = min(ROWS, (q.r1 - q.r0) * G - x0);  // rows of the unit

    // the query rows, rotated, to LDS; rows past the unit's or without a position: zeros
    for (int i = tid; i < ROWS * D; i += 64 * WAVES) {
        const int r = i / D, d = i % D;
        float x = 0.0f;
        const int tok = (x0 + r) / G, pos = first + tok;
        if (r < n_x && pos >= 0 && pos < A.B.cap) {
            const size_t at = (size_t)(q.r0 + tok) * A.a.q_stride + (size_t)(h * G + (x0 + r) % G) * D;
            x = load_any(A.a.q, A.a.q_dtype, at + d);
            const int half = A.a.rope.half;
            if (A.a.rope.cs && d < 2 * half) {
                const bool lo = d < half;
                const int k = lo ? d : d - half;
                const float y = load_any(A.a.q, A.a.q_dtype, at + (lo ? d + half : k));
                const float *cs = A.a.rope.cs + ((size_t)pos * half + k) * 2;
                const float xc = x * cs[0], ys = y * cs[1];
                x = lo ? xc - ys : ys + xc;
            }
        }
        sh.q[r][d] = x;
    }
    __syncthreads();

    // this lane's query row: positions it sees, codes and scale
    int p_hi = -1, p_lo = 0;  // keys p_lo .. p_hi
    if (n < n_x) {
        const int pos = first + (x0 + n) / G;
        if (pos >= 0 && pos < A.B.cap) {
            p_hi = pos;
            p_lo = max(0, pos - (A.a.window - 1));
        }
    }
    i32x4 qf[NQ][LIMBS];
    float qs;
    {
        float amax = 0.0f;
        bool bad = false;
#pragma unroll
        for (int s = 0; s < NQ; s++)
#pragma unroll
            for (int j = 0; j < 16; j++) {
                const float x = fabsf(sh.q[n][64 * s + 16 * g + j]);
                amax = fmaxf(amax, x);
                bad |= !(x < __builtin_inff());
            }
        amax = swap_max(amax);
        bad = swap_max(bad ? 1.0f : 0.0f) != 0.0f;
        // below 2^-100 a row's scores vanish beside any scale in use
        const float id = bad || amax < 0x1p-100f ? 0.0f : QMAX / amax;
        qs = bad ? __builtin_nanf("") : id == 0.0f ? 0.0f : amax / QMAX * A.a.scale * LOG2E;
#pragma unroll
        for (int s = 0; s < NQ; s++)
#pragma unroll
            for (int v = 0; v < 4; v++) {
                uint32_t limb[LIMBS];
#pragma unroll
                for (int b = 0; b < LIMBS; b++) limb[b] = 0;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float x = sh.q[n][64 * s + 16 * g + 4 * v + e];
                    int i = id == 0.0f ? 0 : (int)__builtin_rintf(x * id);
#pragma unroll
                    for (int b = LIMBS - 1; b >= 0; b--) {  // signed bytes, the lowest first
                        const int c = (int)(int8_t)i;
                        limb[b] |= ((uint32_t)c & 255u) << (8 * e);
                        i = (i - c) >> 8;
                    }
                }
#pragma unroll
                for (int b = 0; b < LIMBS; b++) qf[s][b][v] = (int)limb[b];
            }
    }
    __syncthreads();  // sh.q is read; sh.o may be written

    // tiles of this unit and range; keys that every row sees need no mask
    const int u_tok0 = x0 / G, u_tok1 = (x0 + n_x - 1) / G;
    const int u_hi = min(A.B.cap - 1, first + u_tok1), u_first = first + u_tok0;
    const int all_lo = max(0, max(0, u_hi) - (A.a.window - 1)), all_hi = u_first;  // seen by every row (if all have positions)
    int t_lo = max(0, max(u_first, 0) - (A.a.window - 1)) / TILE, t_hi = u_hi < 0 ? 0 : u_hi / TILE + 1;
    t_lo = max(t_lo, w.sp.t0 + w.range * chunk);
    t_hi = min(t_hi, w.sp.t0 + (w.range + 1) * chunk);
    const bool placed = u_first >= 0 && first + u_tok1 < A.B.cap;  // every row has a position
    const int32_t *pages = A.B.pages + (size_t)w.seq * A.B.max_pages;
    const int bmask = (1 << A.P.lg_b) - 1;

    f32x4 acc[NT];
#pragma unroll
    for (int i = 0; i < NT; i++) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    for (int t = t_lo + wave; t < t_hi; t += WAVES) {
        // the K block of this lane's operand rows, the block of its scores
        const int max_block = A.B.cap / KV_BLOCK - 1;
        const int kb = min(4 * t + (n >> 2), max_block), vb = min(4 * t + g, max_block);
        const int kp = pages[kb >> A.P.lg_b], vp = pages[vb >> A.P.lg_b];
        const bool k_ok = (unsigned)kp < (unsigned)A.P.n_pages, v_ok = (unsigned)vp < (unsigned)A.P.n_pages;
        const size_t kblk = (((size_t)(k_ok ? kp : 0) * A.P.heads + h) << A.P.lg_b) + (kb & bmask);
        const size_t vblk = (((size_t)(v_ok ? vp : 0) * A.P.heads + h) << A.P.lg_b) + (vb & bmask);
        const int8_t *kq = A.P.k + kblk * (16 * D) + (n & 3) * D + 16 * g;
        const int8_t *vq = A.P.v + vblk * (16 * D) + n * 16;
        i32x4 ka[4][NQ];
        u32x4 va[NT];
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int s = 0; s < NQ; s++) ka[i][s] = *reinterpret_cast<const i32x4 *>(kq + 4 * i * D + 64 * s);
#pragma unroll
        for (int i = 0; i < NT; i++) va[i] = *reinterpret_cast<const u32x4 *>(vq + 256 * i);
        const float sk = A.P.k_scale[vblk];
        float sv = A.P.v_scale[vblk];

        float x[16];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            i32x4 c[LIMBS];
#pragma unroll
            for (int b = 0; b < LIMBS; b++) {
                c[b] = i32x4{0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < NQ; s++)
                    c[b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(ka[i][s], qf[s][b], c[b], 0, 0, 0);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) {
                // |sum of a limb| <= 256 * 128 * 127: the two lower limbs join in int32
                const float lo = (float)(c[LIMBS - 2][e] * 256 + c[LIMBS - 1][e]);
                if constexpr (HILO) x[4 * i + e] = (float)c[0][e] * 65536.0f + lo;
                else x[4 * i + e] = lo;
            }
        }
        const float f = sk * qs;
        const bool full = placed && TILE * t >= all_lo && TILE * t + TILE - 1 <= all_hi;  // the same in all lanes
        const bool masked = !full || __ballot(!v_ok) != 0;
        if (masked) {
            bool any = false;
#pragma unroll
            for (int j = 0; j < 16; j++) {
                const int p = TILE * t + 16 * g + j;
                const bool see = v_ok && p >= p_lo && p <= p_hi;
                any |= see;
                x[j] = see ? x[j] * f : -INFINITY;
            }
            if (!__ballot(any)) continue;
            // a block that no row sees may hold anything
            const unsigned long long b = __ballot(any);
            if (!((b >> (16 * g)) & 0xFFFFull)) sv = 0.0f;
        } else {
#pragma unroll
            for (int j = 0; j < 16; j++) x[j] = x[j] * f;
        }
        float top = x[0];
#pragma unroll
        for (int j = 1; j < 16; j++) top = fmaxf(top, x[j]);
        const float m_new = fmaxf(m, swap_max(top));
        const float base = m_new == -INFINITY ? 0.0f : m_new;
        const float alpha = exp2_(m - base);
        m = m_new;
        // The tile's largest (finite) scale gets weights up to 2^14; an infinite
        // or NaN one makes NaN of the rows that see its block, no others.
        const float sv_max = swap_max(sv < __builtin_inff() ? sv : 0.0f);
        const float pw = sv_max > 0.0f ? sv / sv_max * 16384.0f : sv < __builtin_inff() ? 0.0f : sv;
        float sum = 0.0f;
        half8 ph[2], pl[2];
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const float e = exp2_(x[j] - base);
            sum += e;
            // where a row does not see a block, its scale (NaN, say) is not the row's
            const float p = masked && x[j] == -INFINITY ? 0.0f : e * pw;
            const _Float16 hi = (_Float16)p;
            ph[j >> 3][j & 7] = hi;
            if constexpr (HILO) pl[j >> 3][j & 7] = (_Float16)(p - (float)hi);
        }
        l = l * alpha + sum;
        const float back = sv_max * 0x1p-14f;
#pragma unroll
        for (int i = 0; i < NT; i++) {
            half2v a[8];
#pragma unroll
            for (int b = 0; b < 4; b++) codes4(va[i][b], a[2 * b], a[2 * b + 1]);
            const half8 v0 = join8(a[0], a[1], a[2], a[3]), v1 = join8(a[4], a[5], a[6], a[7]);
            f32x4 o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, ph[0], o, 0, 0, 0);
            o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, ph[1], o, 0, 0, 0);
            if constexpr (HILO) {
                o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pl[0], o, 0, 0, 0);
                o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pl[1], o, 0, 0, 0);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) acc[i][e] = __builtin_fmaf(acc[i][e], alpha, o[e] * back);
        }
    }
    // join the waves: lane (n, g) holds dimensions 16 i + 4 g + e of row n
    l = swap_sum(l);
    if (g == 0) {
        sh.m[wave][n] = m;
        sh.l[wave][n] = l;
    }
    const bool whole = w.n_ranges == 1;
    float *part = A.a.parts + ((size_t)(w.slot + w.range) * A.P.heads + h) * (ROWS * (D + 2));
    constexpr int PART = Shared<D>::PART;
#pragma unroll
    for (int d0 = 0; d0 < D; d0 += PART) {
        if (d0) __syncthreads();
#pragma unroll
        for (int i = 0; i < PART / 16; i++)
            *reinterpret_cast<f32x4 *>(&sh.o[wave][n][16 * i + 4 * g]) = acc[d0 / 16 + i];
        __syncthreads();
        for (int i = tid; i < ROWS * PART; i += 64 * WAVES) {
            const int r = i / PART, d = i % PART;
            if (r >= n_x) break;
            float top = -INFINITY;
#pragma unroll
            for (int k = 0; k < WAVES; k++) top = fmaxf(top, sh.m[k][r]);
            const float base = top == -INFINITY ? 0.0f : top;
            float o = 0.0f, sum = 0.0f;
#pragma unroll
            for (int k = 0; k < WAVES; k++) {
                const float f = exp2_(sh.m[k][r] - base);
                o = __builtin_fmaf(f, sh.o[k][r][d], o);
                sum = __builtin_fmaf(f, sh.l[k][r], sum);
            }
            if (whole) {
                const size_t at = (size_t)(q.r0 + (x0 + r) / G) * A.a.out_stride + (size_t)(h * G + (x0 + r) % G) * D;
                store_any(A.a.out, A.a.out_dtype, at + d0 + d, sum == 0.0f ? 0.0f : o / sum);
            } else {
                part[r * D + d0 + d] = o;
                if (d0 + d == 0) {
                    part[ROWS * D + r] = top;
                    part[ROWS * D + ROWS + r] = sum;
                }
            }
        }
    }
}

// The split units' ranges, in range order: a wave per (unit, head, row).
template <int D>
__global__ __launch_bounds__(256) void k_kv_join(Args A) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int chunk = chunk_of(A);
    const int task = blockIdx.x * 4 + wave, r = task % ROWS, rest = task / ROWS, h = rest % A.P.heads;
    const int item = rest / A.P.heads;
    int seq, unit;
    if (!kv_find(A.B, item, [&](const KvSeq &q) {
            const Span p = span_of(A, q);
            return ranges(p.tiles, chunk) > 1 ? p.units : 0;
        }, seq, unit))
        return;
    // the ranges before this unit's
    int slot = 0;
    for (int s = lane; s < seq; s += 64) {
        const Span p = span_of(A, kv_seq(A.B, s));
        const int n = ranges(p.tiles, chunk);
        slot += n > 1 ? p.units * n : 0;
    }
    slot = __builtin_amdgcn_readlane(wave_scan(slot), 63);
    const KvSeq q = kv_seq(A.B, seq);
    const int nr = ranges(span_of(A, q).tiles, chunk), x = unit * ROWS + r;
    if (x >= (q.r1 - q.r0) * A.G) return;
    slot += unit * nr;
    const size_t step = (size_t)A.P.heads * (ROWS * (D + 2));
    const float *part = A.a.parts + ((size_t)slot * A.P.heads + h) * (ROWS * (D + 2));
    float top = -INFINITY;
    for (int k = lane; k < nr; k += 64) top = fmaxf(top, part[k * step + ROWS * D + r]);
    top = wave_max(top);
    const float base = top == -INFINITY ? 0.0f : top;
    float o[D / 64], sum = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 64; i++) o[i] = 0.0f;
#pragma unroll 4
    for (int k = 0; k < nr; k++) {
        const float *p = part + k * step;
        const float f = exp2_(p[ROWS * D + r] - base);
        sum = __builtin_fmaf(f, p[ROWS * D + ROWS + r], sum);
#pragma unroll
        for (int i = 0; i < D / 64; i++) o[i] = __builtin_fmaf(f, p[r * D + lane + 64 * i], o[i]);
    }
    const size_t at = (size_t)(q.r0 + x / A.G) * A.a.out_stride + (size_t)(h * A.G + x % A.G) * D;
#pragma unroll
    for (int i = 0; i < D / 64; i++)
        store_any(A.a.out, A.a.out_dtype, at + lane + 64 * i, sum == 0.0f ? 0.0f : o[i] / sum);
}

}  // namespace

// Split units have at least two ranges, all but the last of `chunk` tiles, so
// there are at most twice TARGET of them (heads included), and a rounding
// of the total adds less than one in 2^20.
size_t kv_attention_parts_bytes() { return (size_t)(2 * TARGET + 64) * (ROWS * (256 + 2)) * sizeof(float); }

hipError_t launch_kv_attention(const KvPool &pool, const KvRows &rows, int d_head, const KvAttention &a, hipStream_t s) {
    if (!rows.n_rows) return hipSuccess;
    Args A{pool, rows, a, a.n_q / pool.heads};
    // units of the call at most, and their split ranges
    const size_t x = (size_t)rows.n_rows * A.G, units = x / ROWS + (size_t)rows.n_seqs;
    const size_t u = units < x ? units : x;
    const bool split = rows.cap > MIN_CHUNK * TILE;
    const size_t items = (u + (split ? (2 * TARGET + 64) / pool.heads + 1 : 0)) * pool.heads;
    const dim3 grid((unsigned)items), join((unsigned)((TARGET + 64) * ROWS / 4));
    auto go = [&](auto d) {
        constexpr int D = decltype(d)::value;
        if (a.out_dtype == T_F32) hipLaunchKernelGGL((k_kv_attention<D, true>), grid, dim3(64 * WAVES), 0, s, A);
        else hipLaunchKernelGGL((k_kv_attention<D, false>), grid, dim3(64 * WAVES), 0, s, A);
        if (split) hipLaunchKernelGGL((k_kv_join<D>), join, dim3(256), 0, s, A);
    };
    switch (d_head) {
    case 64: go(std::integral_constant<int, 64>{}); break;
    case 128: go(std::integral_constant<int, 128>{}); break;
    case 192: go(std::integral_constant<int, 192>{}); break;
    case 256: go(std::integral_constant<int, 256>{}); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace rce_qmm
