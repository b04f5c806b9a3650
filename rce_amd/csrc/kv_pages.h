// kv_pages.h -- the pages of the paged KV cache (include/rce_qmm.h
// rce_qmm_kv_copy_dev, _fork_dev, _release_dev, _reserve_dev, _compact_dev) as
// their kernels see them (kv_pages.hip), and their launchers.  Not installed.
#pragma once

#include "kv_cache.h"

namespace rce_qmm {

// Sequences' tables of pages.
struct KvTable {
    int32_t *pages;
    int n_seqs, max_pages;
    __host__ __device__ size_t entries() const { return (size_t)n_seqs * max_pages; }
};

// Entries name pages 0 .. n_pages - 1 of a pool; refs[p] of them name page p.
struct KvRefs {
    int32_t *refs;
    int n_pages;
};

constexpr size_t KV_COMPACT_PAGES = (size_t)1 << 23;  // of a compacted pool at most
// Room that reserve and compact need at most (a part of the context's buffer).
size_t kv_pages_bytes();

hipError_t launch_kv_copy(const KvPool &from, const KvPool &to, int d_head, const int32_t *src, const int32_t *dst, int n, hipStream_t s);
hipError_t launch_kv_fork(const KvTable &from, const KvTable &to, const int32_t *parents, const KvRefs &refs, hipStream_t s);
hipError_t launch_kv_release(const KvTable &t, int page_tokens, const int32_t *from, const int32_t *to, const KvRefs &refs, hipStream_t s);
hipError_t launch_kv_reserve(const KvPool &pool, const KvRows &rows, int d_head, int32_t *pages, int32_t *refs, int32_t *missing,
                             void *room, hipStream_t s);
hipError_t launch_kv_compact(const KvPool &pool, int d_head, const KvTable &t, int32_t *refs, int32_t *new_ids, int32_t *n_used,
                             void *room, hipStream_t s);

}  // namespace rce_qmm
