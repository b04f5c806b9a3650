// qk_rope.h -- norms of query and key heads with their rotation
// (include/rce_qmm.h rce_qmm_qk_norm_rope_dev): the call as its kernels see
// it, and the launcher.  Not installed.
#pragma once

#include "kv_cache.h"

namespace rce_qmm {

constexpr int QK_HEAD = 1024;  // values of a head at most

struct QkHeads {
    const void *in;
    void *out;
    size_t in_stride, out_stride;  // values from row to row
    const float *weight;           // null: ones
    int n;
};
struct QkNormRope {
    KvRows rows;  // pages and cap are not used
    QkHeads q, k;
    int d;
    uint32_t in_dtype, out_dtype;
    float eps;  // below 0: no norm
    KvRope rope;
    int n_pos;  // of the rotation's table
    bool interleaved;
};
hipError_t launch_qk_norm_rope(const QkNormRope &c, hipStream_t s);

}  // namespace rce_qmm
