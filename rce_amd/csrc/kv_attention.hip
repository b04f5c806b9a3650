// kv_attention.hip -- causal attention of ragged query rows over the paged
// 8-bit KV cache (include/rce_qmm.h rce_qmm_kv_attention_dev).
//
// A unit is 16 query rows of one sequence and kv head: row r of the unit is
// query head r % G of token r / G, G the query heads per kv head (one token of
// up to 16 heads, or several tokens).  Its keys are cut into ranges of `chunk`
// tiles of 64 positions; a block takes one range, its four waves every fourth
// tile, and joins the waves' (m, l, o) in LDS.  A unit of one range is
// finished there; the ranges of a longer one leave (m, l, o) in `parts`, which
// k_kv_join adds up in range order.  With first positions that stay visible beside a window (SINKS,
// rce_qmm_kv_attention_sinks_dev) a unit's tiles are four blocks each of what it visits (Span, Visits).
//
// Every block plans for itself: it reads the sequences' lengths (device
// memory, no host round trip), forms the total of tiles and from it the chunk
// that spreads them over TARGET blocks, and finds its own range.  Long enough units
// are cut as one line instead, sequences of many query rows go to k_kv_prompt (both below).
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
//                 largest that its row sees in the tile, times 2^14 (so that small weights stay
//                 normal in binary16), as two binary16 terms: one would round the
//                 weights by up to 2^-11, as much as a binary16 result is rounded
//                 itself, and saves 1 to 3 % (64 x 4096 ragged 81.5 : 79.9 us, 5 rows x 16 x 2000 19.5 : 18.8).
//
// What bounds it: the codes' way from HBM, where there are enough of them.  2 x 131072 ragged, 8
// kv heads of 128, bf16: 340 MB in 70 us (4.9 TB/s, what a copy reaches) and 11 us
// of the join; 64 x 4096 ragged: 348 MB in 82 + 6 us.  Below some 50 MB a block's own
// way from its arguments to its result: 5 rows x 16 x 2000, 41 MB in 19 + 5 us, one
// row x 700 in 11 us (a table of more than SPLIT_FROM tiles: in two ranges and a join, whole calls 10 : 13).
#include "kv_cache.h"

#include <algorithm>
#include <climits>
#include <type_traits>

#include "mfma_util.h"

namespace rce_qmm {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int ROWS = 16;    // query rows of a unit
constexpr int WAVES = 4;    // of a block
constexpr int TILE = 64;    // positions of a wave's step
constexpr int TARGET = 512;   // blocks that a part's tiles are spread over: two per CU
constexpr int MIN_CHUNK = 8;  // tiles of the shortest range
// Tables of up to so many tiles are not split: one sequence of 1000 in one range 16 us, in two 13 and the join 5;
// of 4000 in ranges of 8 tiles 12.5 + 5, in ranges of 24 19 + 5.
constexpr int SPLIT_FROM = 16;
// A single sequence in a table of up to so many tiles has one part whatever its rows turn out to be: 64 rows
// of 64 11 us against 13 with a launch for few rows too, 12 after 5000 21 : 24, 512 after 4096 82 : 87. One row in a
// batch with room for 16: at 4096 positions 18 : 18, at 32768 38 : 32, at 131072 101 : 59.
constexpr int ONE_TABLE = 128;
constexpr int WHOLE = 1 << 24;  // tiles of a range where there is no split
constexpr int P_MIN_CHUNK = 4;  // of units of P_ROWS rows: 3 x 201 f32 in ranges of 4 tiles 21 us, of 8 25, of 2 28
constexpr int LINE_CHUNK = 24;  // tiles per block from which a block may serve several units
constexpr int PAD = 4;          // a unit's prologue and epilogue, in the time of a tile
constexpr int FEW = 32;       // query rows per kv head up to which a sequence is served in units of ROWS
// A call of more than FEW rows per sequence on average has a part in units of P_ROWS.  So has one of LONG rows
// or more besides a token per sequence, which may be one prompt's, where that prompt in units of ROWS could
// come to LONG_TILES tiles for each of TARGET blocks by the table's span.  All in units of ROWS : with the
// part (us, f16, heads of 128), single tokens beside a prompt of that many rows, and those tiles:
//   1020 rows after 1744, 32: 82 : 88;  1196 new, 36: 86 : 78, 5 (heads of 64): 12 : 25;  1996 new, 31: 68 : 94;
//   3992 new, 8: 30 : 53;
//   1899 new, 59: 171 : 176;  1999 new, 62: 139 : 137;  1996 after 1500, 62: 129 : 119;  1792 after 3647, 112: 159 : 137;
//   1996 after 7692, 250: 287 : 194;  3992 after 3000, 500: 350 : 206;  6999 new, 751: 811 : 285.
// LONG: 16 sequences of 5 drafts in long tables are spared the launch (4 us of 27).
constexpr int LONG = 1536, LONG_TILES = 48;

// With sinks no unit visits more tiles than a window's.  Up to SHORT of them a few sequences have one part (a long one is there: units of few rows
// take no longer than its), and units that are TARGET and more are not split: 3 x 500 rows after 9000, a window of 2048: 117 -> 104 us.
// Two parts : one (us, f16, 32 / 8 heads of 128, a window of 1024 where none is named): 3 x 500 rows, 2048 96.4 : 88.4; 16 x 20 rows 39.9 : 33.8;
// 15 single tokens and 1000 rows 58.6 : 51.0, and 4000 121 : 117, and 500 with 3000 89.6 : 86.8; 15 x 4 and 2000 rows, 2048 118.9 : 120.5.
// Of more than SHORT_SEQS sequences one part measured no worse either (31 single tokens and 1000 rows 61.4 : 48, 24 x 300 199 : 190).
constexpr int SHORT = 64, SHORT_SEQS = 16;
// Tiles of the shortest range of few rows there, and beyond.  In ranges of 8 : of 4 (us, whole calls): one row, window 1024, 4 kv heads of 64,
// f32 14.5 : 13.2; window 1500, 8 of 128 17.9 : 15.7; 8 rows, window 1024 20.4 : 19.8; one row, window 8192 21.1 : 22.4.
constexpr int SHORT_CHUNK = 4;

constexpr float LOG2E = 1.4426950408889634f;

struct Args {
    KvPool P;
    KvRows B;
    KvAttention a;
    int G;          // query heads per kv head
    int rows;       // query rows of a unit
    int lo_x, hi_x; // the call's part: sequences of lo_x .. hi_x query rows per kv head
    int target;     // blocks that the part's tiles are spread over
    int min_chunk;  // tiles of the shortest range
    int line;       // 1: the units may be cut as one line
    int vec;        // query rows (1) and rotation table (2) can be read, output rows (4) written 16 bytes at a time
};

// The units of a sequence (per kv head; 0 where it is not of the part) and the tiles of its longest one: t0 .. t0 + tiles - 1.
//
// With sinks a range is cut from what a unit visits, not from the positions: a list of the blocks of 16 positions that the
// sinks reach into (as far as its window does not) and its window's, four of them a tile, number 0 ..; `tiles` is what the
// sequence's longest unit can come to.  Blocks and not tiles of 64 positions stand in a row: 4 sinks and a window of 1024 of 32 tokens
// are 17 tiles, not 18.5 (2 prompts of up to 6000, 338 -> 328 us).
struct Span {
    int units, t0, tiles;
};
template <bool SINKS>
__device__ __forceinline__ Span span_of(const Args &A, const KvSeq &q) {
    Span s;
    const int x = (q.r1 - q.r0) * A.G;
    s.units = x >= A.lo_x && x <= A.hi_x ? (x + A.rows - 1) / A.rows : 0;
    const int lo = max(0, q.lo() - (A.a.window - 1));
    s.t0 = lo / TILE;
    s.tiles = q.hi(A.B) > q.lo() ? (q.hi(A.B) + TILE - 1) / TILE - s.t0 : 0;
    if constexpr (SINKS) {
        if (s.tiles) {
            // a unit's tokens stand in a row, their windows span that many positions together
            const int tokens = min(q.r1 - q.r0, (A.rows - 1) / A.G + 2);
            const int own = (int)(((int64_t)A.a.window + tokens - 2) / KV_BLOCK) + 2, reach = (A.a.sinks + KV_BLOCK - 1) / KV_BLOCK;
            s.tiles = min(s.t0 + s.tiles, (own + reach + 3) / 4);
        }
        s.t0 = 0;
    }
    return s;
}

// The tiles that a unit visits of its range [w_lo, w_hi); its window reaches into the positions p_lo .. p_hi - 1.
template <bool SINKS>
struct Visits {
    int lo, hi, front, back;  // block i of the list is block i below `front`, else i + back
    __device__ Visits(const Args &A, int w_lo, int w_hi, int p_lo, int p_hi) {
        if constexpr (SINKS) {
            const int first = p_lo / KV_BLOCK, end = (p_hi + KV_BLOCK - 1) / KV_BLOCK;
            front = min(min((A.a.sinks + KV_BLOCK - 1) / KV_BLOCK, first), end);
            back = first - front;
            lo = w_lo;
            hi = min(w_hi, (front + max(0, end - first) + 3) / 4);
        } else {
            lo = max(p_lo / TILE, w_lo);
            hi = min((p_hi + TILE - 1) / TILE, w_hi);
        }
    }
    __device__ __forceinline__ int block(int t, int b) const {  // block b of tile t
        if constexpr (!SINKS) return 4 * t + b;
        return 4 * t + b + (4 * t + b < front ? 0 : back);
    }
};
// The cells of a unit in the line (below): its prologue's, then one per tile, one if it has none.
__device__ __forceinline__ int line_cells(const Span &p) { return PAD + max(1, p.tiles); }

// How a part is cut, the same in every block: tiles per range, or in a line cells per block.
struct Cut {
    int chunk;
    bool line;
};
template <bool LINE, bool SINKS>
__device__ __forceinline__ Cut cut_of(const Args &A) {
    const int lane = threadIdx.x & 63;
    float tiles = 0.0f, units = 0.0f;  // only sizes: their rounding moves no result
    for (int s = lane; s < A.B.n_seqs; s += 64) {
        const Span p = span_of<SINKS>(A, kv_seq(A.B, s));
        tiles += (float)p.units * (float)p.tiles;
        if (LINE) units += (float)line_cells(p) * (float)p.units;
    }
    auto chunk = [&](float total) { return (int)fminf(ceilf(wave_sum(total) * (float)A.P.heads / (float)A.target), 1e9f); };
    const int c = chunk(tiles);
    if (LINE && A.line && c >= LINE_CHUNK) {
        const int l = chunk(units);
        if (l < 1 << 20) return {l, true};  // the line's length fits 31 bits
    }
    return {max(A.min_chunk, c), false};
}

__device__ __forceinline__ int ranges(int tiles, int chunk) { return tiles ? (tiles + chunk - 1) / chunk : 1; }
// Tiles of each of a unit's ranges but the last: the ranges are as long as each other.
__device__ __forceinline__ int range_tiles(int tiles, int n) { return (tiles + n - 1) / n; }

// A unit's split ranges are numbered within the call: parts slot (range number * heads + head).
struct Work {
    KvSeq q;
    Span sp;
    int seq, unit;
    int t_lo, t_hi;  // tiles of the range, of the sequence
    int slot;        // of the range, before the head
    bool whole;      // the range is all of the unit's
};

// Range `item` of the list (sequence, unit, range).
template <bool SINKS>
__device__ __forceinline__ bool find_work(const Args &A, int item, int chunk, Work &w) {
    const int lane = threadIdx.x & 63;
    int run = 0, srun = 0;
    for (int base = 0; base < A.B.n_seqs; base += 64) {
        const int s = base + lane;
        int c = 0, sc = 0;
        KvSeq q{0, 0, 0};
        if (s < A.B.n_seqs) {
            q = kv_seq(A.B, s);
            const Span p = span_of<SINKS>(A, q);
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
            w.q = {__builtin_amdgcn_readlane(q.r0, l), __builtin_amdgcn_readlane(q.r1, l), __builtin_amdgcn_readlane(q.len, l)};
            w.sp = span_of<SINKS>(A, w.q);
            const int n = ranges(w.sp.tiles, chunk), step = range_tiles(w.sp.tiles, n);
            const int u = at / n, range = at - u * n;
            w.unit = w.sp.units - 1 - u;  // the units with the most keys first
            w.t_lo = w.sp.t0 + range * step;
            w.t_hi = w.t_lo + step;
            w.slot = srun + __builtin_amdgcn_readlane(sincl - sc, l) + w.unit * n + range;
            w.whole = n == 1;
            return true;
        }
        run += total;
        srun += __builtin_amdgcn_readlane(sincl, 63);
    }
    return false;
}

// ---- the units as one line ------------------------------------------------
//
// Ranges of whole units leave lengths from chunk / 2 to chunk: the CUs that have got
// the short ones wait.  Where a block has LINE_CHUNK tiles or more to do, all units stand in one
// line, PAD cells for the prologue and one per tile each, and block i takes the cells i * chunk ..
// (i + 1) * chunk - 1, of two or more units often.  What it leaves of a unit that it shares goes to
// slot 2 i + 1 if it has the unit's first tile, else 2 i (its first unit).
// 64 sequences of up to 4096: 100 -> 85 us.

// The work at cell `pos` of the line, up to cell `end`; false: none is left.  n: the cells up to the next unit.
template <bool SINKS>
__device__ __forceinline__ bool find_in_line(const Args &A, int item, int pos, int end, Work &w, int &n) {
    const int lane = threadIdx.x & 63;
    int run = 0;
    for (int base = 0; base < A.B.n_seqs; base += 64) {
        const int s = base + lane;
        int c = 0;
        if (s < A.B.n_seqs) {
            const Span p = span_of<SINKS>(A, kv_seq(A.B, s));
            c = p.units * line_cells(p);
        }
        const int incl = wave_scan(c), total = __builtin_amdgcn_readlane(incl, 63);
        if (pos < run + total) {
            const int l = __builtin_ctzll(__ballot(pos < run + incl));
            const int at = pos - run - __builtin_amdgcn_readlane(incl - c, l);
            w.seq = base + l;
            w.q = kv_seq(A.B, w.seq);
            w.sp = span_of<SINKS>(A, w.q);
            const int cells = line_cells(w.sp);
            w.unit = at / cells;
            const int from = at - w.unit * cells, to = min(cells, from + end - pos);
            n = to - from;
            if (to <= PAD) return false;  // the unit's tiles are the next block's
            const int t = max(from, PAD) - PAD;
            w.t_lo = w.sp.t0 + t;
            w.t_hi = w.sp.t0 + min(w.sp.tiles, to - PAD);
            w.slot = 2 * item + (t == 0);
            w.whole = t == 0 && to == cells;
            return true;
        }
        run += total;
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
__device__ __forceinline__ uint32_t bf16_of(float x) {
    const uint32_t u = __float_as_uint(x);
    return x != x ? 0x7FC0u : (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;
}
__device__ __forceinline__ void store_any(void *p, uint32_t t, size_t i, float x) {
    if (t == T_F32) static_cast<float *>(p)[i] = x;
    else if (t == T_F16) static_cast<_Float16 *>(p)[i] = (_Float16)x;
    else static_cast<uint16_t *>(p)[i] = (uint16_t)bf16_of(x);
}

// Four codes as two binary16 pairs: bytes offset to 0 .. 255 become the low
// byte of 1024 + b, minus 1152.  Exact.
__device__ __forceinline__ void codes4(uint32_t x, half2v &lo, half2v &hi) {
    const uint32_t b = x ^ 0x80808080u;
    const half2v off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    lo = as_h2(__builtin_amdgcn_perm(b, 0x64646464u, 0x00050004u)) + off;
    hi = as_h2(__builtin_amdgcn_perm(b, 0x64646464u, 0x00070006u)) + off;
}

// 16 values as LIMBS signed bytes each of rint(x * id), the highest first: one operand register
// group per limb.
template <int LIMBS>
__device__ __forceinline__ void limbs_of(const float (&x)[16], float id, i32x4 (&out)[LIMBS]) {
#pragma unroll
    for (int v = 0; v < 4; v++) {
        uint32_t limb[LIMBS];
#pragma unroll
        for (int b = 0; b < LIMBS; b++) limb[b] = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            int i = id == 0.0f ? 0 : (int)__builtin_rintf(x[4 * v + e] * id);
#pragma unroll
            for (int b = LIMBS - 1; b >= 0; b--) {  // signed bytes, the lowest first
                const int c = (int)(int8_t)i;
                limb[b] |= ((uint32_t)c & 255u) << (8 * e);
                i = (i - c) >> 8;
            }
        }
#pragma unroll
        for (int b = 0; b < LIMBS; b++) out[b][v] = (int)limb[b];
    }
}

// N pieces of 16 values from the value indexes i: at multiples of 16 bytes.
template <int N>
__device__ __forceinline__ void load_pieces(const void *p, uint32_t t, const size_t (&i)[N], float (&x)[N][16]) {
    if (t == T_F32) {
        float4 v[N][4];
#pragma unroll
        for (int s = 0; s < N; s++)
#pragma unroll
            for (int k = 0; k < 4; k++) v[s][k] = reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i[s])[k];
#pragma unroll
        for (int s = 0; s < N; s++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                x[s][4 * k] = v[s][k].x;
                x[s][4 * k + 1] = v[s][k].y;
                x[s][4 * k + 2] = v[s][k].z;
                x[s][4 * k + 3] = v[s][k].w;
            }
        return;
    }
    u32x4 v[N][2];
#pragma unroll
    for (int s = 0; s < N; s++)
#pragma unroll
        for (int k = 0; k < 2; k++) v[s][k] = reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(p) + i[s])[k];
    const bool f16 = t == T_F16;
#pragma unroll
    for (int s = 0; s < N; s++)
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const uint32_t w = v[s][k >> 2][k & 3];
            const half2v e = as_h2(w);
            x[s][2 * k] = f16 ? (float)e.x : __uint_as_float(w << 16);
            x[s][2 * k + 1] = f16 ? (float)e.y : __uint_as_float(w & 0xFFFF0000u);
        }
}

// Row x_row of the sequence and kv head h, rotated to position pos, as codes: the 16 dimensions
// 64 s + 16 g .. of this lane in qf[s], the factor of its base-2 scores in qs.  is: the row has a position.
template <int D, int LIMBS, bool SINKS>
__device__ __forceinline__ void query_codes(const Args &A, const KvSeq &q, int h, int x_row, int pos, bool is, int g,
                                            i32x4 (&qf)[D / 64][LIMBS], float &qs) {
    constexpr int NQ = D / 64;
    constexpr float QMAX = LIMBS == 3 ? 127.0f * 65536.0f : 127.0f * 256.0f;
    float x[NQ][16];
    const int half = A.a.rope.cs ? A.a.rope.half : 0;
    // A row without a position reads row 0 of the call and of the table, and is zeroed after:
    // no load stands under a condition of its lane, all are in flight together.
    const size_t at = is ? (size_t)(q.r0 + x_row / A.G) * A.a.q_stride + (size_t)(h * A.G + x_row % A.G) * D : 0;
    const float *cs = A.a.rope.cs + (size_t)(is ? pos : 0) * half * 2;
    if ((A.vec & 3) == 3 && half % 16 == 0) {  // the pieces' partners are whole pieces too
        size_t own[NQ], other[NQ];
#pragma unroll
        for (int s = 0; s < NQ; s++) {
            const int d = 64 * s + 16 * g;
            own[s] = at + d;
            other[s] = at + (d < half ? d + half : d < 2 * half ? d - half : d);
        }
        load_pieces<NQ>(A.a.q, A.a.q_dtype, own, x);
        // All of a head turned, two operands or more: the lane holds its pieces' partners.  With sinks their pairs turn
        // together, by table values read once (2 x 6000 tokens, window 64 132 -> 119 us); without, that spills registers
        // (3 x 4096 488 -> 497 us).
        const bool partners = NQ % 2 == 0 && 2 * half == D;
        if (SINKS && partners) {
            constexpr int H = NQ / 2;
#pragma unroll
            for (int s = 0; s < H; s++) {
                const float4 *c = reinterpret_cast<const float4 *>(cs + 2 * (64 * s + 16 * g));
                float (&a)[16] = x[s], (&b)[16] = x[(s + H) % NQ];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float4 v = c[j];
                    const float a0 = a[2 * j], a1 = a[2 * j + 1], b0 = b[2 * j], b1 = b[2 * j + 1];
                    a[2 * j] = a0 * v.x - b0 * v.y;
                    a[2 * j + 1] = a1 * v.z - b1 * v.w;
                    b[2 * j] = a0 * v.y + b0 * v.x;
                    b[2 * j + 1] = a1 * v.w + b1 * v.z;
                }
            }
        } else if (half) {
            float y[NQ][16];
            if (!SINKS && partners) {
#pragma unroll
                for (int s = 0; s < NQ; s++)
#pragma unroll
                    for (int j = 0; j < 16; j++) y[s][j] = x[(s + NQ / 2) % NQ][j];
            } else {
                load_pieces<NQ>(A.a.q, A.a.q_dtype, other, y);
            }
#pragma unroll
            for (int s = 0; s < NQ; s++) {
                const int d = 64 * s + 16 * g;
                const bool lo = d < half, turns = d < 2 * half;
                const float4 *c = reinterpret_cast<const float4 *>(cs + 2 * (lo ? d : turns ? d - half : 0));
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float4 v = c[j];
                    const float ac = x[s][2 * j] * v.x, as = y[s][2 * j] * v.y;
                    const float bc = x[s][2 * j + 1] * v.z, bs = y[s][2 * j + 1] * v.w;
                    const float a = lo ? ac - as : as + ac, b = lo ? bc - bs : bs + bc;
                    x[s][2 * j] = turns ? a : x[s][2 * j];
                    x[s][2 * j + 1] = turns ? b : x[s][2 * j + 1];
                }
            }
        }
    } else {
#pragma unroll
        for (int s = 0; s < NQ; s++)
#pragma unroll
            for (int j = 0; j < 16; j++) {
                const int d = 64 * s + 16 * g + j;
                x[s][j] = load_any(A.a.q, A.a.q_dtype, at + d);
                if (d < 2 * half) {
                    const bool lo = d < half;
                    const int k = lo ? d : d - half;
                    const float p = load_any(A.a.q, A.a.q_dtype, at + (lo ? d + half : k));
                    const float xc = x[s][j] * cs[2 * k], ys = p * cs[2 * k + 1];
                    x[s][j] = lo ? xc - ys : ys + xc;
                }
            }
    }
    float amax = 0.0f;
    bool bad = false;
#pragma unroll
    for (int s = 0; s < NQ; s++)
#pragma unroll
        for (int j = 0; j < 16; j++) {
            x[s][j] = is ? x[s][j] : 0.0f;
            amax = fmaxf(amax, fabsf(x[s][j]));
            bad |= !(fabsf(x[s][j]) < __builtin_inff());
        }
    amax = swap_max(amax);
    bad = swap_max(bad ? 1.0f : 0.0f) != 0.0f;
    const float id = bad || amax < 0x1p-100f ? 0.0f : QMAX / amax;
    qs = bad ? __builtin_nanf("") : id == 0.0f ? 0.0f : amax / QMAX * A.a.scale * LOG2E;
#pragma unroll
    for (int s = 0; s < NQ; s++) limbs_of<LIMBS>(x[s], id, qf[s]);
}

// LDS: the waves' results (at most 128 dimensions at a time: 34 KB).
template <int D>
struct Shared {
    static constexpr int PART = D <= 128 ? D : D / 2;
    alignas(16) float o[WAVES][ROWS][PART + 4];
    float m[WAVES][ROWS], l[WAVES][ROWS];
};

template <int D, int LIMBS, bool LINE, bool SINKS>
__global__ __launch_bounds__(64 * WAVES, D * LIMBS <= 256 ? 3 : D <= 192 ? 2 : 1) void k_kv_attention(Args A) {
    constexpr int NQ = D / 64, NT = D / 16;
    __shared__ Shared<D> sh;
    int block = blockIdx.x;
    const Cut cut = cut_of<LINE, SINKS>(A);
    // a line is at most `target` blocks and one more per head; past it the products below would pass 31 bits
    if (LINE && cut.line && block / A.P.heads > A.target) return;
    int line_at = cut.line ? block / A.P.heads * cut.chunk : 0;
    const int line_end = line_at + cut.chunk;
    for (;;) {
        // opaque: what follows from them is not kept in registers from one unit to the next
        int tid = threadIdx.x;
        if constexpr (LINE) asm volatile("" : "+v"(tid), "+s"(block));
        const int lane = tid & 63, n = lane & 15, g = lane >> 4;
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int item = block / A.P.heads, h = block % A.P.heads;
        Work w;
        int n_cells = 0;
        if (LINE && cut.line ? !find_in_line<SINKS>(A, item, line_at, line_end, w, n_cells) : !find_work<SINKS>(A, item, cut.chunk, w)) return;
        const KvSeq &q = w.q;
        const int G = A.G, first = q.first();
        const int x0 = w.unit * ROWS, n_x = min(ROWS, (q.r1 - q.r0) * G - x0);  // rows of the unit

        // this lane's query row: positions it sees, codes and scale
        const int pos = first + (x0 + n) / G;
        const bool is = n < n_x && pos >= 0 && pos < A.B.cap;
        const int p_hi = is ? pos : -1, p_lo = is ? max(0, pos - (A.a.window - 1)) : 0;  // keys p_lo .. p_hi
        i32x4 qf[NQ][LIMBS];
        float qs;
        query_codes<D, LIMBS, SINKS>(A, q, h, x0 + n, pos, is, g, qf, qs);

        // tiles of this unit and range; keys that every row sees need no mask
        const int u_tok0 = x0 / G, u_tok1 = (x0 + n_x - 1) / G;
        const int u_hi = min(A.B.cap - 1, first + u_tok1), u_first = first + u_tok0;
        const int all_lo = max(0, max(0, u_hi) - (A.a.window - 1)), all_hi = u_first;  // seen by every row (if all have positions)
        const Visits<SINKS> visit(A, w.t_lo, w.t_hi, max(0, max(u_first, 0) - (A.a.window - 1)), max(u_hi + 1, 0));
        const bool placed = u_first >= 0 && first + u_tok1 < A.B.cap;  // every row has a position
        const int32_t *pages = A.B.pages + (size_t)w.seq * A.B.max_pages;
        const int bmask = (1 << A.P.lg_b) - 1;

        f32x4 acc[NT];
#pragma unroll
        for (int i = 0; i < NT; i++) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        float m = -INFINITY, l = 0.0f;
        for (int t = visit.lo + wave; t < visit.hi; t += WAVES) {
            // the K block of this lane's operand rows, the block of its scores
            const int max_block = A.B.cap / KV_BLOCK - 1;
            const int kb = min(visit.block(t, n >> 2), max_block), vb = min(visit.block(t, g), max_block);
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
                    if constexpr (LIMBS == 3) x[4 * i + e] = (float)c[0][e] * 65536.0f + lo;
                    else x[4 * i + e] = lo;
                }
            }
            const float f = sk * qs;
            // the tile's first and last position; the same in all lanes
            const int p0 = KV_BLOCK * visit.block(t, 0), p1 = KV_BLOCK * visit.block(t, 3) + KV_BLOCK - 1;
            const bool full = placed && (p0 >= all_lo || (SINKS && p1 < A.a.sinks)) && p1 <= all_hi;
            const bool masked = !full || __ballot(!v_ok) != 0;
            if (masked) {
                bool any = false;
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    const int p = KV_BLOCK * visit.block(t, g) + j;
                    const bool see = v_ok && (p >= p_lo || (SINKS && p < A.a.sinks)) && p <= p_hi;
                    any |= see;
                    x[j] = see ? x[j] * f : -INFINITY;
                }
                if (!__ballot(any)) continue;
                // a block that this lane's row does not see may hold anything, values far larger than
                // all that it does see among it
                if (!any) sv = 0.0f;
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
            // The largest (finite) scale that the row sees in the tile gets weights up to 2^14; an
            // infinite or NaN one makes NaN of the rows that see its block, no others.
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
                pl[j >> 3][j & 7] = (_Float16)(p - (float)hi);
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
                o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pl[0], o, 0, 0, 0);
                o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pl[1], o, 0, 0, 0);
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
        const bool whole = w.whole;
        float *part = A.a.parts + ((size_t)w.slot * A.P.heads + h) * (ROWS * (D + 2));
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
        line_at += n_cells;
        if (!LINE || !cut.line || line_at >= line_end) return;
        __syncthreads();  // sh is read
    }
}

// ---- many query rows ------------------------------------------------------
//
// A block of eight waves takes 128 query rows, a wave 16 of them, with the
// operand layouts of k_kv_attention.  The block shares each tile of 64 positions
// through LDS: the key codes as they are, the values converted to binary16 once, both
// with their 16-byte pieces in another order per row (else reads of one piece of
// 16 rows would fall on the same banks).  The next tile's codes travel to registers meanwhile.
// O stays in the MFMAs' accumulators, in units of `ref`, the largest value
// scale that the row has seen, and of the row's m.  m moves, and O and l are rescaled, only when a
// score passes it by more than LAG (base 2): weights are then at most 2^LAG,
// times UP in binary16 at most 2^15.
// Results in 16 bits take one binary16 term per weight (HILO: two).  Its rounding, 2^-11 at most, adds
// a third to the error of a binary16 result (normwise against 64 bits 2.7e-4, 2.1e-4 for the
// result's own rounding; below 1 % for BF16); a second term costs a third of the time (3 x 4096 f16 565 : 770 us).
// 3 prompts of 4096, 32 query and 8 kv heads of 128, f16: 355 GFLOP in 500 us for the whole call, 0.71
// PFLOP/s, the MFMAs busy 30 % of the time.  What bounds it: the vector unit (16 exponentials, their conversions and
// the scores' of a lane per tile and row) and the reads of LDS, a quarter of them in conflict.
// 3 x 201 rows f32, 16 kv heads of 64, a window of 512: 21 us and 8 of the join; no unit is busy there
// (VALU a third of the time, MFMAs and LDS 3 %): a block's chain of loads and barriers.
// 16 rows and not 32 per wave: MFMAs, exponentials and the vector unit overlap only across
// waves, and 16 rows fit 128 registers (four waves per SIMD; at the price of twice
// the LDS reads per product).
constexpr int P_ROWS = 128, P_WAVES = 8;
constexpr float LAG = 6.0f, UP = 512.0f;  // UP = 2^9
constexpr int UNSEEN = -(1 << 30);  // below all scores of two limbs: at 256 dimensions they reach 256 * 128 * 127 * 256, 0.8 % less

// A lane's accumulators times f: four consecutive values every 16 from value index i; vec:
// at multiples of their size.
template <int NT>
__device__ __forceinline__ void store_row(void *p, uint32_t t, size_t i, bool vec, const f32x4 (&acc)[NT], float f, bool zero) {
    auto at = [&](int k, int e) { return zero ? 0.0f : acc[k][e] * f; };
    if (!vec) {
#pragma unroll
        for (int k = 0; k < NT; k++)
#pragma unroll
            for (int e = 0; e < 4; e++) store_any(p, t, i + 16 * k + e, at(k, e));
    } else if (t == T_F32) {
        float *o = static_cast<float *>(p) + i;
#pragma unroll
        for (int k = 0; k < NT; k++) *reinterpret_cast<float4 *>(o + 16 * k) = make_float4(at(k, 0), at(k, 1), at(k, 2), at(k, 3));
    } else if (t == T_F16) {
        _Float16 *o = static_cast<_Float16 *>(p) + i;
        typedef _Float16 half4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int k = 0; k < NT; k++)
            *reinterpret_cast<half4 *>(o + 16 * k) = half4{(_Float16)at(k, 0), (_Float16)at(k, 1), (_Float16)at(k, 2), (_Float16)at(k, 3)};
    } else {
        uint16_t *o = static_cast<uint16_t *>(p) + i;
#pragma unroll
        for (int k = 0; k < NT; k++)
            *reinterpret_cast<uint2 *>(o + 16 * k) =
                make_uint2(bf16_of(at(k, 0)) | bf16_of(at(k, 1)) << 16, bf16_of(at(k, 2)) | bf16_of(at(k, 3)) << 16);
    }
}

template <int D>
struct PShared {
    alignas(16) int8_t k[TILE * D];      // row: a position, pieces of 16 codes
    alignas(16) _Float16 v[D * TILE];    // row: a dimension, pieces of 8 positions
    float ks[4], vs[4];                  // of the tile's blocks
    int ok[4];                           // 0: no page
};

// Where piece c of a key row of position p lies: the 16 rows of an operand are 16 (m / 4) + m % 4 (+ 4 t).
template <int D>
__device__ __forceinline__ int key_piece(int p, int c) {
    return D % 128 == 0 ? c ^ ((p & 3) | (p >> 2 & 4)) : c ^ ((p >> 1 & 1) | (p >> 3 & 2));
}

template <int D, bool HILO, bool SINKS>
__global__ __launch_bounds__(64 * P_WAVES, D <= 128 ? (HILO ? 3 : 4) : 2) void k_kv_prompt(Args A, const int32_t *__restrict__ page_table) {
    constexpr int NQ = D / 64, NT = D / 16;
    constexpr int LIMBS = HILO ? 3 : 2;
    constexpr bool QUICK = SINKS && !HILO;
    static_assert(!QUICK || (int64_t)D * 128 * 127 * 256 < -(int64_t)UNSEEN, "codes of 128, queries of 127 * 256");
    constexpr float lag = QUICK ? 0.0f : LAG;  // QUICK comes to the maximum only where m was too low
    constexpr int NK = (TILE * D + 16 * 64 * P_WAVES - 1) / (16 * 64 * P_WAVES);  // 16-byte pieces of codes a thread moves
    constexpr int BUFS = D <= 128 ? 2 : 1;  // two where they fit 64 KB
    __shared__ PShared<D> buf[BUFS];
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = blockIdx.x % A.P.heads;
    Work w;
    if (!find_work<SINKS>(A, blockIdx.x / A.P.heads, SINKS && A.min_chunk == WHOLE ? WHOLE : cut_of<false, SINKS>(A).chunk, w)) return;
    const KvSeq &q = w.q;
    const int G = A.G, first = q.first();
    const int x0 = w.unit * P_ROWS, n_x = min(P_ROWS, (q.r1 - q.r0) * G - x0);
    const int xr = wave * 16 + n;  // this lane's row of the unit
    const int tok = (x0 + xr) / G, pos = first + tok;
    const bool is = xr < n_x && pos >= 0 && pos < A.B.cap;

    i32x4 qf[NQ][LIMBS];
    float qs;
    if constexpr (!SINKS) query_codes<D, LIMBS, SINKS>(A, q, h, x0 + xr, pos, is, g, qf, qs);

    const int p_hi = is ? pos : -1, p_lo = is ? max(0, pos - (A.a.window - 1)) : 0;
    // the wave's rows: positions that all of them see, or that any of them sees
    const int w0 = wave * 16, w_n = min(16, n_x - w0);  // rows (none: w_n <= 0)
    const int f0 = first + (x0 + w0) / G, f1 = first + (x0 + w0 + max(w_n, 1) - 1) / G;
    const bool placed = w_n > 0 && f0 >= 0 && f1 < A.B.cap;
    const int w_lo = max(0, max(0, f0) - (A.a.window - 1)), w_hi = w_n > 0 ? min(f1, A.B.cap - 1) : -1;
    const int all_lo = max(0, max(0, f1) - (A.a.window - 1)), all_hi = f0;
    // the block's tiles
    const int u_first = first + x0 / G, u_hi = min(A.B.cap - 1, first + (x0 + n_x - 1) / G);
    const Visits<SINKS> visit(A, w.t_lo, w.t_hi, max(0, max(u_first, 0) - (A.a.window - 1)), max(u_hi + 1, 0));
    const int t_lo = visit.lo, t_hi = visit.hi;
    const int32_t *__restrict__ pages = page_table + (size_t)w.seq * A.B.max_pages;
    const int bmask = (1 << A.P.lg_b) - 1, max_block = A.B.cap / KV_BLOCK - 1;

    // What this thread moves: piece tid + 256 i of the tile's keys (position / (D / 16), 16
    // codes) and of its values (dimension and block: 16 positions).  A wave's pieces i lie in one
    // block: page ids and block addresses are scalar.
    constexpr int BP = D;  // pieces of a block: 16 positions x D codes / 16
    static_assert(BP % 64 == 0, "a wave's pieces lie in one block");
    u32x4 kr[NK], vr[NK];
    float ksr = 0.0f, vsr = 0.0f;
    int pg[NK], pgs = 0, oks = 0;  // the next tile's page ids, loaded a tile ahead
    auto mine = [&](int i) { return 4 * BP % (64 * P_WAVES) == 0 || wave * 64 + 64 * P_WAVES * i < 4 * BP; };  // the same in a wave
    auto block_of = [&](int t, int b) { return min(visit.block(t, b), max_block); };
    auto look = [&](int t) {
#pragma unroll
        for (int i = 0; i < NK; i++)
            if (mine(i)) pg[i] = pages[block_of(t, (wave * 64 + 64 * P_WAVES * i) / BP) >> A.P.lg_b];
        if (tid < 4) pgs = pages[block_of(t, tid) >> A.P.lg_b];
    };
    auto block_at = [&](int page, int blk) -> uint32_t {  // page 0 where there is none
        const uint32_t p = (unsigned)page < (unsigned)A.P.n_pages ? page : 0;
        return ((p * (uint32_t)A.P.heads + (uint32_t)h) << A.P.lg_b) + (uint32_t)(blk & bmask);
    };
    auto fetch = [&](int t) {
#pragma unroll
        for (int i = 0; i < NK; i++) {
            if (!mine(i)) continue;
            const int e = wave * 64 + 64 * P_WAVES * i, b = e / BP;
            const size_t at = (size_t)block_at(pg[i], block_of(t, b)) * (16 * D) + e % BP * 16;
            kr[i] = *reinterpret_cast<const u32x4 *>(A.P.k + at + 16u * lane);
            vr[i] = *reinterpret_cast<const u32x4 *>(A.P.v + at + 16u * lane);
        }
        if (tid < 4) {
            int b = tid;
            asm volatile("" : "+v"(b));  // as below
            const uint32_t blk = block_at(pgs, block_of(t, b));
            ksr = A.P.k_scale[blk];
            vsr = A.P.v_scale[blk];
            oks = (unsigned)pgs < (unsigned)A.P.n_pages;
        }
    };
    auto place = [&](PShared<D> &to) {
#pragma unroll
        for (int i = 0; i < NK; i++) {
            if (!mine(i)) continue;
            const int e = tid + 64 * P_WAVES * i, b = e / BP, r = e % BP;
            {  // keys: position 16 b + r / (D / 16), piece r % (D / 16)
                const int p = 16 * b + r / (D / 16), c = r % (D / 16);
                *reinterpret_cast<u32x4 *>(to.k + p * D + key_piece<D>(p, c) * 16) = kr[i];
            }
            {  // values: dimension r, positions 16 b .. + 15: pieces 2 b, 2 b + 1
                half2v a[8];
#pragma unroll
                for (int k = 0; k < 4; k++) codes4(vr[i][k], a[2 * k], a[2 * k + 1]);
                _Float16 *row = to.v + r * TILE;
                *reinterpret_cast<half8 *>(row + ((2 * b) ^ (r & 7)) * 8) = join8(a[0], a[1], a[2], a[3]);
                *reinterpret_cast<half8 *>(row + ((2 * b + 1) ^ (r & 7)) * 8) = join8(a[4], a[5], a[6], a[7]);
            }
        }
        if (tid < 4) {
            to.ks[tid] = ksr;
            to.vs[tid] = vsr;
            to.ok[tid] = oks;
        }
    };

    f32x4 acc[NT];
#pragma unroll
    for (int i = 0; i < NT; i++) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // (ref from 2^-110 on: UP / ref stays finite, and smaller scales keep 2^-18 of the largest weight)
    float m = -INFINITY, l = 0.0f, ref = 0x1p-110f, inv_ref = UP * 0x1p110f;
    // This lane's operands in LDS: key position 16 (n / 4) + n % 4 + 4 i, piece 4 s + g, and value
    // row n + 16 i, piece 2 g + u.
    const int k_pos = 16 * (n >> 2) + (n & 3);
    const int k_row0 = k_pos * D + key_piece<D>(k_pos, g) * 16, v_row0 = n * TILE + (2 * g ^ (n & 7)) * 8;
    if (t_lo < t_hi) {
        look(t_lo);
        fetch(t_lo);
        look(t_lo + 1);
    }
    // With sinks units are short, and the first tile comes while the query rows do (with the rows' halves read once
    // 2 prompts of up to 6000, window 1024 289 -> 280 us); without, 3 x 201 rows f32 take 31.6 us so, 31.1 the other way.
    if constexpr (SINKS) query_codes<D, LIMBS, SINKS>(A, q, h, x0 + xr, pos, is, g, qf, qs);
    if (t_lo < t_hi) {
        place(buf[0]);
        if (t_lo + 1 < t_hi) fetch(t_lo + 1);
        look(t_lo + 2);
    }
    __syncthreads();
    for (int t = t_lo; t < t_hi; t++) {
        const PShared<D> &sh = buf[(t - t_lo) & (BUFS - 1)];
        const int p0 = KV_BLOCK * visit.block(t, 0), p1 = KV_BLOCK * visit.block(t, 3) + KV_BLOCK - 1;  // its first and last position
        if (p0 <= w_hi && (p1 >= w_lo || (SINKS && p0 < A.a.sinks))) {  // some row of the wave sees it (the same in all lanes)
            const bool full = placed && (p0 >= all_lo || (SINKS && p1 < A.a.sinks)) && p1 <= all_hi;
            const bool masked = !full || !(sh.ok[0] & sh.ok[1] & sh.ok[2] & sh.ok[3]);
            // opaque: what is formed from them would be kept over the loop, in registers that spill
            int k_row = k_row0, v_row = v_row0;
            asm volatile("" : "+v"(k_row), "+v"(v_row));
            int xi[16];  // scores as whole numbers (HILO: without the highest limb, which is xh)
            float xh[HILO ? 16 : 1];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                i32x4 c[LIMBS];
#pragma unroll
                for (int b = 0; b < LIMBS; b++) c[b] = i32x4{0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < NQ; s++) {
                    // key_piece of a row 4 i on is the same, of a piece 4 s on 64 s bytes on (all but bit 2 of
                    // the piece stays)
                    const int8_t *at = sh.k + (D % 128 == 0 ? (k_row ^ (s & 1) * 64) + (s >> 1) * 128 : k_row + 64 * s) + 4 * i * D;
                    const i32x4 a = *reinterpret_cast<const i32x4 *>(at);
#pragma unroll
                    for (int b = 0; b < LIMBS; b++) c[b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, qf[s][b], c[b], 0, 0, 0);
                }
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    xi[4 * i + e] = c[LIMBS - 2][e] * 256 + c[LIMBS - 1][e];
                    if constexpr (HILO) xh[4 * i + e] = (float)c[0][e] * 65536.0f;
                }
            }
            auto score = [&](int e) { return HILO ? xh[HILO ? e : 0] + (float)xi[e] : (float)xi[e]; };
            const float f = sh.ks[g] * qs;
            float sv = sh.vs[g];
            half8 ph[2], pl[2];
            // QUICK: a tile that all its rows see is weighted with the m and ref there are, with no maximum over
            // it.  It stands where no weight is past binary16 (the sum of a lane's 16 bounds each; an m of
            // -infinity and a NaN fail) and the scale is as in the ordinary tile below; else the tile is weighted again,
            // after a new m.  2 prompts of up to 6000, window 1024, 4 sinks, f16 280 -> 262 us; 3 x 500 rows, window 2048 100 -> 93.
            bool done = false;
            if constexpr (QUICK) {
                if (!masked) {
                    const float pw = sv * inv_ref, lw = __builtin_amdgcn_logf(pw), off = lw - m;
                    float sum = 0.0f;
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const float p = exp2_(__builtin_fmaf((float)xi[e], f, off));
                        sum += p;
                        ph[e >> 3][e & 7] = (_Float16)p;
                    }
                    done = !__ballot(!(pw >= 0.125f && pw < 2.0f * UP && sum <= 65504.0f));
                    if (done) l = __builtin_fmaf(sum, exp2_(-lw), l);
                }
            }
            if (!done) {
                float top = -INFINITY;
                uint32_t seen = 0xFFFFu;  // bit e: the row sees the position of score e
                if (HILO || masked) {
                    if (masked) {
                        const int p = KV_BLOCK * visit.block(t, g), lo = max(p_lo - p, 0), hi = min(p_hi - p, 15);
                        seen = sh.ok[g] && lo <= hi ? (0xFFFFu << lo) & (0xFFFFu >> (15 - hi)) : 0u;
                        if constexpr (SINKS) {
                            const int last = min(hi, A.a.sinks - 1 - p);
                            if (sh.ok[g] && last >= 0) seen |= 0xFFFFu >> (15 - last);
                        }
                        if (!seen) sv = 0.0f;  // as in k_kv_attention
                    }
                    asm volatile("" : "+v"(seen));  // else its bits are tested in front of the branch
                    if constexpr (SINKS && !HILO) {
                        // what a row does not see is below all that it sees; a row that sees nothing has no score
                        int x = UNSEEN;
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            const int is = (int)(seen << (31 - e)) >> 31;
                            xi[e] = (xi[e] & is) | (UNSEEN & ~is);
                            x = max(x, xi[e]);
                        }
                        top = seen ? (float)x * f : -INFINITY;
                    } else {
#pragma unroll
                        for (int e = 0; e < 16; e++) top = fmaxf(top, seen >> e & 1 ? score(e) * f : -INFINITY);
                    }
                } else {
                    int x = xi[0];
#pragma unroll
                    for (int e = 1; e < 16; e++) x = max(x, xi[e]);
                    top = (float)x * f;
                }
                top = swap_max(top);
                // `top` above m + LAG, or a larger value scale that the row sees: rescale (lanes alone for the
                // scale: a ballot over both costs registers that spill)
                const bool fin = sv < __builtin_inff();
                const float scale = swap_max(fin ? sv : 0.0f);
                if (__ballot(top > m + lag) || scale > ref) {
                    const float m_new = top > m + lag ? top : m, ref_new = fmaxf(ref, scale);
                    const float alpha = m == -INFINITY ? 0.0f : exp2_(m - m_new);
                    const float back = ref_new > ref ? ref / ref_new * alpha : alpha;
                    l *= alpha;
#pragma unroll
                    for (int i = 0; i < NT; i++)
#pragma unroll
                        for (int e = 0; e < 4; e++) acc[i][e] *= back;
                    m = m_new;
                    ref = ref_new;
                    inv_ref = UP / ref;
                }
                const float base = m == -INFINITY ? 0.0f : m;
                // what the values' scale makes of the weights; an infinite or NaN one makes NaN of the
                // rows that see its block, no others
                const float pw = fin ? sv * inv_ref : sv;
                // The ordinary tile: no mask, value scales above 2^-12 of `ref`.  The scale goes into the
                // exponent, l gets the sum of the weights in f32 over it (the rounded ones would leave out
                // those below 2^-25 / pw: 1 % of the sum of 65536 at 2^-22.6).
                // Two terms (HILO) and all else take the longer way.
                if (!HILO && !QUICK && !masked && !__ballot(!(pw >= 0.125f && pw < 2.0f * UP))) {
                    const float lw = __builtin_amdgcn_logf(pw), off = lw - base;
                    float sum = 0.0f;
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const float p = exp2_(__builtin_fmaf((float)xi[e], f, off));
                        sum += p;
                        ph[e >> 3][e & 7] = (_Float16)p;
                    }
                    l = __builtin_fmaf(sum, exp2_(-lw), l);
                } else if constexpr (SINKS && !HILO) {  // xi is UNSEEN where the row does not see it: the weight is taken out
                    float sum = 0.0f;
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const int is = (int)(seen << (31 - e)) >> 31;
                        const float y = __int_as_float(__float_as_int(exp2_(__builtin_fmaf((float)xi[e], f, -base))) & is);
                        sum += y;
                        ph[e >> 3][e & 7] = (_Float16)__int_as_float(__float_as_int(y * pw) & is);
                    }
                    l += sum;
                } else {
                    float sum = 0.0f;
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const bool see = seen >> e & 1;
                        const float y = see ? exp2_(score(e) * f - base) : 0.0f, p = see ? y * pw : 0.0f;
                        sum += y;
                        const _Float16 hi = (_Float16)p;
                        ph[e >> 3][e & 7] = hi;
                        if constexpr (HILO) pl[e >> 3][e & 7] = (_Float16)(p - (float)hi);
                    }
                    l += sum;
                }
            }
#pragma unroll
            for (int u = 0; u < 2; u++)  // positions 16 g + 8 u ...
#pragma unroll
                for (int i = 0; i < NT; i++) {
                    const half8 a = *reinterpret_cast<const half8 *>(sh.v + (v_row ^ u * 8) + 16 * i * TILE);
                    acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ph[u], acc[i], 0, 0, 0);
                    if constexpr (HILO) acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pl[u], acc[i], 0, 0, 0);
                }
        }
        if constexpr (BUFS == 1) __syncthreads();
        if (t + 1 < t_hi) {  // the next tile to the other buffer, the one after it on its way
            place(buf[(t + 1 - t_lo) & (BUFS - 1)]);
            if (t + 2 < t_hi) fetch(t + 2);
            look(t + 3);
        }
        __syncthreads();
    }
    // lane (n, g) holds dimensions 16 i + 4 g + e of its row
    l = swap_sum(l);
    if (xr >= n_x) return;
    const float unit = ref * (1.0f / UP);
    if (w.whole) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l * unit;
        const size_t at = (size_t)(q.r0 + tok) * A.a.out_stride + (size_t)(h * G + (x0 + xr) % G) * D + 4 * g;
        store_row<NT>(A.a.out, A.a.out_dtype, at, A.vec & 4, acc, inv, l == 0.0f);
    } else {
        float *part = A.a.parts + ((size_t)w.slot * A.P.heads + h) * (P_ROWS * (D + 2));
        store_row<NT>(part, T_F32, (size_t)xr * D + 4 * g, (D + 2) * P_ROWS % 4 == 0, acc, unit, false);
        if (g == 0) {
            part[P_ROWS * D + xr] = m;
            part[P_ROWS * D + P_ROWS + xr] = l;
        }
    }
}

// The split units' ranges, in range order: a wave takes 256 / D consecutive rows of a (unit,
// head), four values per lane, every wave of the grid the next ones; U ranges
// at a time, whose loads depend on nothing.
constexpr int JOIN_BLOCKS = 1024;  // at most: four waves per SIMD
template <int D, bool LINE, bool SINKS>
__global__ __launch_bounds__(256) void k_kv_join(Args A0, Args A1) {
    constexpr int LPR = D / 4, RPW = 64 / LPR;  // lanes of a row, rows of a wave
    constexpr int U = LINE ? 16 : 8;  // a line's units are the long ones
    const Args &A = blockIdx.y ? A1 : A0;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Cut cut = cut_of<LINE, SINKS>(A);
    const int chunk = cut.chunk;
    const bool line = LINE && cut.line;
    const int rows = A.rows;
    for (int task = blockIdx.x * 4 + wave;; task += gridDim.x * 4) {
        const int h = task % A.P.heads;
        int seq, group;
        if (!kv_find(A.B, task / A.P.heads, [&](const KvSeq &q) {
                const Span p = span_of<SINKS>(A, q);
                return p.units && (line || ranges(p.tiles, chunk) > 1) ? ((q.r1 - q.r0) * A.G + RPW - 1) / RPW : 0;
            }, seq, group))
            return;
        // what stands in front of the sequence: cells of the line, or split ranges
        int before = 0;
        for (int s = lane; s < seq; s += 64) {
            const Span p = span_of<SINKS>(A, kv_seq(A.B, s));
            const int n = ranges(p.tiles, chunk);
            before += line ? p.units * line_cells(p) : n > 1 ? p.units * n : 0;
        }
        before = __builtin_amdgcn_readlane(wave_scan(before), 63);
        const KvSeq q = kv_seq(A.B, seq);
        const Span sp = span_of<SINKS>(A, q);
        const int x0 = group * RPW, unit = x0 / rows;
        int slot, nr;  // the first range's; their number
        if (line) {
            const int cells = line_cells(sp), t0 = before + unit * cells;
            const int b0 = (t0 + PAD) / chunk, b1 = (t0 + cells - 1) / chunk;
            if (b0 == b1) continue;
            slot = 2 * b0 + 1;  // the next 2 (b0 + 1), every other slot from there
            nr = b1 - b0 + 1;
        } else {
            nr = ranges(sp.tiles, chunk);
            slot = before + unit * nr;
        }
        const int sub = lane / LPR, x = x0 + sub, r = x % rows, d = lane % LPR * 4;
        if (sub < RPW && x < (q.r1 - q.r0) * A.G) {
            const size_t unit_size = (size_t)rows * (D + 2), step = (size_t)A.P.heads * unit_size * (line ? 2 : 1);
            const float *part0 = A.a.parts + ((size_t)slot * A.P.heads + h) * unit_size;
            const float *part1 = part0 + (size_t)A.P.heads * unit_size;  // of range 1
            float top = -INFINITY, sum = 0.0f;
            f32x4 o[1] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
            for (int k0 = 0; k0 < nr; k0 += U) {
                float m[U], l[U];
                f32x4 v[U];
#pragma unroll
                for (int e = 0; e < U; e++) {
                    const int k = min(k0 + e, nr - 1);
                    const float *p = k ? part1 + (size_t)(k - 1) * step : part0;
                    m[e] = p[rows * D + r];
                    l[e] = p[rows * D + rows + r];
                    v[e] = *reinterpret_cast<const f32x4 *>(p + r * D + d);
                }
                float to = top;
#pragma unroll
                for (int e = 0; e < U; e++) to = fmaxf(to, m[e]);  // the last one again: no change
                const float base = to == -INFINITY ? 0.0f : to, back = exp2_(top - base);
                top = to;
                sum *= back;
#pragma unroll
                for (int i = 0; i < 4; i++) o[0][i] *= back;
#pragma unroll
                for (int e = 0; e < U; e++) {
                    const bool in = k0 + e < nr;  // (a select: past the end may be a NaN times 0)
                    const float f = exp2_(m[e] - base);
                    sum = in ? __builtin_fmaf(f, l[e], sum) : sum;
#pragma unroll
                    for (int i = 0; i < 4; i++) o[0][i] = in ? __builtin_fmaf(f, v[e][i], o[0][i]) : o[0][i];
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) o[0][i] /= sum;
            const size_t at = (size_t)(q.r0 + x / A.G) * A.a.out_stride + (size_t)(h * A.G + x % A.G) * D + d;
            store_row<1>(A.a.out, A.a.out_dtype, at, A.vec & 4, o, 1.0f, sum == 0.0f);
        }
    }
}

}  // namespace

// A part's split units have at least two ranges, all but the last of `chunk` tiles, so that
// there are at most twice `target` of them (heads included); a rounding of the total
// adds less than one in 2^10 (n_seqs is at most 2^20).  In a line the blocks have two slots each, and
// there is at most one block more per head: heads are at most target / 20 there.
constexpr int slots(int target) { return 2 * target + target / 8; }
// Partial results of units of ROWS and of P_ROWS rows.  Room for TARGET blocks of few rows at every
// head size, for 126 (256 dimensions) to 496 of many.
constexpr size_t FEW_PARTS = (size_t)18 << 20, MANY_PARTS = (size_t)34 << 20;
size_t kv_attention_parts_bytes() { return FEW_PARTS + MANY_PARTS; }

hipError_t launch_kv_attention(const KvPool &pool, const KvRows &rows, int d_head, const KvAttention &a, hipStream_t s) {
    if (!rows.n_rows) return hipSuccess;
    const int G = a.n_q / pool.heads;
    const size_t x = (size_t)rows.n_rows * G;
    // positions that the tiles of a sequence span at most; with sinks its longest unit's (span_of; units of P_ROWS hold the most tokens)
    const int64_t tokens = std::min(rows.n_rows, (P_ROWS - 1) / G + 2);
    const int64_t reach = (a.sinks + KV_BLOCK - 1) / KV_BLOCK, own = ((int64_t)a.window + tokens) / KV_BLOCK + 2;
    const int64_t span = a.sinks ? std::min((int64_t)rows.cap, TILE * ((reach + own + 3) / 4)) : (int64_t)rows.cap;
    auto go = [&](auto d, auto with_sinks) {
        constexpr int D = decltype(d)::value;
        constexpr bool SINKS = decltype(with_sinks)::value;
        const bool f32 = a.out_dtype == T_F32;
        int vec = 0;
        if (reinterpret_cast<uintptr_t>(a.q) % 16 == 0 && a.q_stride * (a.q_dtype == T_F32 ? 4 : 2) % 16 == 0) vec |= 1;
        if (reinterpret_cast<uintptr_t>(a.rope.cs) % 16 == 0) vec |= 2;
        if (reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.out_stride * (f32 ? 4 : 2) % 16 == 0) vec |= 4;
        Args join[2];
        int joins = 0;
        bool in_line = false;
        // units of the part at most, and its grid
        auto units = [&](const Args &A, int hi) {
            const size_t n = std::min((size_t)rows.n_seqs, x / std::max(A.lo_x, 1));  // sequences of the part
            const size_t u = std::min(x, x / A.rows + n);
            return hi == INT_MAX ? u : std::min(u, (size_t)rows.n_seqs * ((hi + A.rows - 1) / A.rows));
        };
        auto grid = [&](Args &A, size_t u) {
            const bool split = span > (int64_t)A.min_chunk * TILE;
            if (split) join[joins++] = A;
            return dim3((unsigned)((u + (split ? slots(A.target) / pool.heads + 1 : 0)) * pool.heads));
        };
        auto target = [](size_t room, int unit) { return std::min(TARGET, (int)(room / ((size_t)unit * (D + 2) * sizeof(float)) * 16 / 34)); };
        auto few = [&](int hi) {
            Args A{pool, rows, a, G, ROWS, 0, hi, target(FEW_PARTS, ROWS),
                   span <= SPLIT_FROM * TILE ? WHOLE : SINKS && span <= SHORT * TILE ? SHORT_CHUNK : MIN_CHUNK, 0, vec};
            const size_t u = units(A, hi);
            // can its tiles come to a line at all?
            A.line = span > SPLIT_FROM * TILE && pool.heads * 20 <= A.target &&
                     (double)u * pool.heads * (span / TILE + 2) >= (double)A.target * (LINE_CHUNK - 1);
            in_line = A.line;
            const dim3 g = grid(A, u), b(64 * WAVES);
            if (A.line && f32) hipLaunchKernelGGL((k_kv_attention<D, 3, true, SINKS>), g, b, 0, s, A);
            else if (A.line) hipLaunchKernelGGL((k_kv_attention<D, 2, true, SINKS>), g, b, 0, s, A);
            else if (f32) hipLaunchKernelGGL((k_kv_attention<D, 3, false, SINKS>), g, b, 0, s, A);
            else hipLaunchKernelGGL((k_kv_attention<D, 2, false, SINKS>), g, b, 0, s, A);
        };
        auto many = [&](int lo) {
            Args A{pool, rows, a, G, P_ROWS, lo, INT_MAX, target(MANY_PARTS, P_ROWS), P_MIN_CHUNK, 0, vec};
            // units of much the same length, enough of them: none is split
            if (SINKS && span <= SHORT * TILE && x / P_ROWS * pool.heads >= (size_t)A.target) A.min_chunk = WHOLE;
            A.a.parts += FEW_PARTS / sizeof(float);
            const dim3 g = grid(A, units(A, INT_MAX)), b(64 * P_WAVES);
            if (f32) hipLaunchKernelGGL((k_kv_prompt<D, true, SINKS>), g, b, 0, s, A, rows.pages);
            else hipLaunchKernelGGL((k_kv_prompt<D, false, SINKS>), g, b, 0, s, A, rows.pages);
        };
        const size_t tokens = (size_t)G * rows.n_seqs, more = x > tokens ? x - tokens : 0;
        const bool prompt = more >= (size_t)LONG &&
                            (double)more / ROWS * (span / TILE) * pool.heads >= (double)LONG_TILES * TARGET;
        if (x > (size_t)FEW * rows.n_seqs || prompt) {
            const bool one = (rows.n_seqs == 1 && span <= ONE_TABLE * TILE) || (SINKS && rows.n_seqs <= SHORT_SEQS && span <= SHORT * TILE);
            many(one ? 0 : FEW + 1);
            if (!one) few(FEW);
        } else {
            few(INT_MAX);
        }
        if (!joins) return;
        constexpr int RPB = 4 * (256 / D);  // rows of a block
        const dim3 g((unsigned)std::min((size_t)JOIN_BLOCKS, (x * pool.heads + RPB - 1) / RPB), (unsigned)joins), b(256);
        if (in_line) hipLaunchKernelGGL((k_kv_join<D, true, SINKS>), g, b, 0, s, join[0], join[joins - 1]);
        else hipLaunchKernelGGL((k_kv_join<D, false, SINKS>), g, b, 0, s, join[0], join[joins - 1]);
    };
    auto pick = [&](auto d) {
        if (a.sinks) go(d, std::true_type{});
        else go(d, std::false_type{});
    };
    switch (d_head) {
    case 64: pick(std::integral_constant<int, 64>{}); break;
    case 128: pick(std::integral_constant<int, 128>{}); break;
    case 192: pick(std::integral_constant<int, 192>{}); break;
    case 256: pick(std::integral_constant<int, 256>{}); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace rce_qmm
