// Gate of a mixture of experts (kernels/route.hip): k of E experts per token, their weights and
// the experts' loads, and the gradient of the weights into the logits.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "kernels/elem.h"

namespace oap {
namespace kern {

constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxK = 32;
constexpr int kRouteMaxGroups = 64;

struct RouteArgs {
  const void* logits;  // [tokens][experts], row stride ld elements
  int64_t ld;
  const float* bias;  // [experts] or null; enters the choice only
  int64_t tokens;
  int experts, k, groups, top_groups;
  bool sigmoid, renormalize;
  float scale;
  float* weights;    // [tokens][k]
  int32_t* indices;  // [tokens][k], -1 where fewer than k experts are left
  int32_t* counts;   // [experts]
  int32_t* partial;  // workspace, route_partial_bytes(tokens, experts)
};

size_t route_partial_bytes(int64_t tokens, int experts);
void route(Elem e, const RouteArgs& a, hipStream_t s);

struct RouteGradArgs {
  const void* logits;
  int64_t ld;
  const float* weights;    // the forward's
  const int32_t* indices;  // the forward's
  const float* grad;       // [tokens][k], of the weights
  int64_t tokens;
  int experts, k;
  bool sigmoid, renormalize;
  float scale;
  void* grad_logits;  // [tokens][experts], contiguous
};

void route_grad(Elem e, const RouteGradArgs& a, hipStream_t s);

}  // namespace kern
}  // namespace oap
