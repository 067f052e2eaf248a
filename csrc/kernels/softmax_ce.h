// Softmax cross entropy over the rows of a catalogue without keeping the logits
// (kernels/softmax_ce.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "kernels/elem.h"

namespace oap {
namespace kern {

struct CeArgs {
  Elem elem;
  const void* x;  // [n][dim], row stride ldx
  int64_t ldx;
  const void* w;  // [classes][dim], row stride ldw
  int64_t ldw;
  const float* bias;      // [classes] or null; -inf leaves the class out
  const int64_t* target;  // [n]
  int64_t ignore;         // rows with this target have no loss
  int64_t n, classes;
  int dim;
  // forward: gradients will be asked for, whose pass has to see the same logits, to the last bit,
  // as the one that forms the maxima (a row's probabilities are powers of their difference)
  bool train;
};

// loss[i] = log sum_j exp(logit(i, j)) - logit(i, target[i]); stat[i] = the row's (max, sum of
// exp(logit - max)) and, for split operands only, miss[i] = 1 - probability of the target, which
// the gradients read.
// total (one float, or null): the sum of the losses, over the number of rows that have one
// where `mean`.
size_t ce_forward_bytes(const CeArgs& a);
void ce_forward(const CeArgs& a, float* loss, float2* stat, float* miss, float* total, bool mean,
                void* work, hipStream_t s);

// Gradients for the upstream gradient of the losses: one float (per_row false; divided by the
// number of rows that have a loss where `mean`) or one per row.  Any of dx [n][dim],
// dw [classes][dim] (element type) and db [classes] may be null.
size_t ce_backward_bytes(const CeArgs& a, bool want_dx, bool want_dw, bool want_db);
void ce_backward(const CeArgs& a, const float2* stat, const float* miss, const float* grad,
                 bool per_row, bool mean, void* dx, void* dw, float* db, void* work,
                 hipStream_t s);

// How a call is divided: rows of a turn of the forward pass, classes of a piece (of the pass that
// `grad` names), and whether fp32 operands are split in two fp16 numbers
struct CePlan {
  int64_t rows, classes;
  bool split;
};
CePlan ce_plan(const CeArgs& a, bool grad);

}  // namespace kern
}  // namespace oap
