// Host engine of the training ops (dropout, route, softmax cross entropy) for tensors in host
// memory: the same definitions as the kernels, fp32 in and out, sums and choices in fp64.
#pragma once

#include "kernels/dropout.h"
#include "kernels/route.h"
#include "kernels/softmax_ce.h"

namespace oap {

// every pointer of the arguments is host memory; elements are fp32
void dropout_host(const kern::DropoutArgs& a);
void route_host(const kern::RouteArgs& a);
void route_grad_host(const kern::RouteGradArgs& a);
void ce_forward_host(const kern::CeArgs& a, float* loss, float2* stat, float* total, bool mean);
void ce_backward_host(const kern::CeArgs& a, const float2* stat, const float* grad, bool per_row,
                      bool mean, float* dx, float* dw, float* db);

}  // namespace oap
