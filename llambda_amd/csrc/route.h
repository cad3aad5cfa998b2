// route.h -- routing to experts (route.hip; the MoE layers' gating with a
// router, moe.hip): scores, a selection bias, groups of experts, top-k,
// renormalised weights.
#pragma once

#include <hip/hip_runtime.h>

namespace llhip {

constexpr int kRouteMaxGroups = 64;

// For one token's logits l over `experts` experts, in 64 bits:
//   s = sigmoid(l), or softmax(l) over all experts;  c = s + bias
//   a group (experts / groups neighbours) scores the sum of its `group_rank`
//   highest c; the top_groups highest groups stay (all where groups is 1)
//   the top_k highest c of those are taken, lower index first among equals
//   w = s of the taken, divided by their sum where `norm`, times scale
// (without a bias and with one group the order is the logits', which also
// tells apart scores that round to the same number)
// NaN and l <= -FLT_MAX are never taken and add nothing to a softmax; places
// that stay unfilled hold (-1, 0).
struct RouteSpec {
  const float* bias;  // [experts], or null
  int experts, top_k, groups, top_groups, group_rank;
  int sigmoid, norm;
  float scale;
};

// logits [tokens][experts] -> indices, weights [tokens][top_k].
hipError_t route_launch(const RouteSpec& r, const float* logits, int tokens, int* indices,
                        float* weights, hipStream_t stream);

}  // namespace llhip
