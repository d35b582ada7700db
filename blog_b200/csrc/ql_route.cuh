// Choice of experts (ql_route.cu): launch arguments.
#pragma once
#include "ql_common.cuh"

namespace ql {

constexpr int kRouteMaxExperts = 1024, kRouteMaxTop = 32, kRouteMaxGroups = 32;

struct RouteArgs {
    const float *logits;  // [tokens][logits_stride]
    const float *bias;    // [n_experts] or null
    int *top_idx;         // [tokens][k]
    float *top_w;
    int64_t logits_stride;
    int tokens, n_experts, k;
    bool sigmoid, renorm;
    int n_groups, top_groups, group_best;  // n_groups 1: no groups
    float scale;
};

cudaError_t route_launch(const RouteArgs &a, cudaStream_t s);

}  // namespace ql
