// moe_route.h -- routing of tokens to experts (include/rce_qmm.h
// rce_qmm_moe_route_dev): its call as the kernel sees it, and the launcher.
// Not installed.
#pragma once

#include "qmm_internal.h"

namespace rce_qmm {

constexpr int ROUTE_EXPERTS = 1024, ROUTE_GROUPS = 64, ROUTE_TOP_K = 64;  // at most

struct Routing {
    const void *logits;
    uint32_t dtype;
    size_t stride;
    int n_tokens, n_expert;
    int top_k, n_group, topk_group, group_top;
    bool sigmoid, normalize;
    float scale;
    const float *bias;  // null: none
    int32_t *ids;
    float *weights;
};
hipError_t launch_moe_route(const Routing &r, hipStream_t s);

}  // namespace rce_qmm
