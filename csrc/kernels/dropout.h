// Counter-based dropout of a flat array (kernels/dropout.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "kernels/elem.h"

namespace oap {
namespace kern {

struct DropoutArgs {
  const void* x;
  const void* residual;  // null: none
  void* y;
  int64_t n;
  uint64_t offset;         // global index of element 0
  uint64_t seed;           // the generator's key, unless seed_ptr is given
  const int64_t* seed_ptr;  // device memory, read by the kernel (graph replays see new values)
  uint64_t threshold;      // round(p 2^32)
  float scale;             // 1 / (1 - p); 0 where p = 1
};

// y = keep ? x * scale : 0 (+ residual), rounded once to the element type
void dropout(Elem e, const DropoutArgs& a, hipStream_t s);

}  // namespace kern
}  // namespace oap
