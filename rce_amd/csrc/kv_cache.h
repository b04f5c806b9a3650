// kv_cache.h -- the paged 8-bit KV cache (include/rce_qmm.h rce_qmm_kv_*)
// as its kernels see it (kv_cache.hip, kv_attention.hip), and their
// launchers.  Not installed.
#pragma once

#include "qmm_internal.h"

namespace rce_qmm {

constexpr int KV_BLOCK = 16;  // positions that share a scale

// The pool: block b (of B = 1 << lg_b per page) of page p and head h is block
// (p * heads + h) * B + b of each array.
struct KvPool {
    int8_t *k, *v;
    float *k_scale, *v_scale;
    int n_pages, lg_b, heads;
};

// rce_qmm_kv_batch, its counts checked to fit int; cap = positions a
// sequence's table spans.
struct KvRows {
    const int32_t *offsets, *lens, *pages;
    int n_seqs, n_rows, max_pages, cap;
};

struct KvRope {
    const float *cs;  // null: no rotation
    int half;
};

hipError_t launch_kv_append(const KvPool &pool, const KvRows &rows, int d_head, const void *k, size_t k_stride,
                            const void *v, size_t v_stride, uint32_t dtype, const KvRope &rope, hipStream_t s);
hipError_t launch_kv_read(const KvPool &pool, const KvRows &rows, int d_head, void *k, void *v, uint32_t dtype,
                          hipStream_t s);

struct KvAttention {
    const void *q;
    void *out;
    size_t q_stride, out_stride;
    uint32_t q_dtype, out_dtype;
    int n_q;
    int window;   // INT_MAX: none
    float scale;
    KvRope rope;
    float *parts;  // kv_attention_parts_bytes()
};
// Room for the partial results of a call's split key ranges, whatever the call.
size_t kv_attention_parts_bytes();
hipError_t launch_kv_attention(const KvPool &pool, const KvRows &rows, int d_head, const KvAttention &a, hipStream_t s);

struct SampleRows {
    const void *logits;
    uint32_t dtype;
    size_t n_rows, vocab, stride;
    const float *u, *temperature, *top_p, *min_p;
    const int32_t *top_k;
    int32_t *ids;
    float *probs;
    void *split;  // sample_split_bytes(), 16-byte aligned
};
// Room for rows that several blocks share, whatever the call.
size_t sample_split_bytes();
hipError_t launch_sample(const SampleRows &r, hipStream_t s);

#ifdef __HIPCC__
// ---- device helpers -------------------------------------------------------

// One sequence of the batch, offsets brought into range: its rows are
// r0 .. r1 - 1, row r at position len - (r1 - r).
struct KvSeq {
    int r0, r1, len;
    __device__ int first() const { return len - (r1 - r0); }                  // position of the first row
    __device__ int lo() const { return max(0, first()); }                     // positions the rows have in the table:
    __device__ int hi(const KvRows &b) const { return max(lo(), min(len, b.cap)); }  // lo .. hi - 1
};

__device__ __forceinline__ KvSeq kv_seq(const KvRows &b, int s) {
    KvSeq q;
    q.r0 = min(max(b.offsets[s], 0), b.n_rows);
    q.r1 = min(max(b.offsets[s + 1], q.r0), b.n_rows);
    q.len = max(b.lens[s], 0);
    return q;
}

// v of the lane CTRL names (0 where there is none, or for rows outside ROWS).
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ int dpp32(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ unsigned long long dpp64(unsigned long long v) {
    const uint32_t lo = (uint32_t)dpp32<CTRL, ROWS>((int)(uint32_t)v), hi = (uint32_t)dpp32<CTRL, ROWS>((int)(uint32_t)(v >> 32));
    return (unsigned long long)hi << 32 | lo;
}
// Inclusive prefix sum over the wave's lanes: within rows of 16 (shifts by 1, 2, 4, 8), then
// lane 15 of rows 0 and 2 into rows 1 and 3, then lane 31 into rows 2 and 3.
__device__ __forceinline__ int wave_scan(int v) {
    v += dpp32<0x111>(v);
    v += dpp32<0x112>(v);
    v += dpp32<0x114>(v);
    v += dpp32<0x118>(v);
    v += dpp32<0x142, 0xA>(v);
    v += dpp32<0x143, 0xC>(v);
    return v;
}
__device__ __forceinline__ unsigned long long wave_scan64(unsigned long long v) {
    v += dpp64<0x111>(v);
    v += dpp64<0x112>(v);
    v += dpp64<0x114>(v);
    v += dpp64<0x118>(v);
    v += dpp64<0x142, 0xA>(v);
    v += dpp64<0x143, 0xC>(v);
    return v;
}
__device__ __forceinline__ unsigned long long lane64(unsigned long long v, int l) {
    return (unsigned long long)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), l) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, l);
}

// Item `item` of the list that has count(seq) consecutive items for every
// sequence: its sequence and its index there (false: past the list's end).
// The whole wave calls it, 64 sequences a round.
template <class Count>
__device__ __forceinline__ bool kv_find(const KvRows &b, int item, Count count, int &seq, int &idx) {
    const int lane = threadIdx.x & 63;
    int run = 0;
    for (int base = 0; base < b.n_seqs; base += 64) {
        const int s = base + lane;
        const int c = s < b.n_seqs ? count(kv_seq(b, s)) : 0;
        const int incl = wave_scan(c), total = __builtin_amdgcn_readlane(incl, 63);
        if (item < run + total) {
            const int l = __builtin_ctzll(__ballot(item < run + incl));
            seq = base + l;
            idx = item - run - __builtin_amdgcn_readlane(incl - c, l);
            return true;
        }
        run += total;
    }
    return false;
}
#endif

}  // namespace rce_qmm
