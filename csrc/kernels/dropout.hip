// Dropout whose mask is never stored: element i of the (global) array is kept when word i & 3 of
// Philox4x32-10 at counter i >> 2 is at least round(p 2^32), so the backward pass, another shard
// or the host engine form the same mask from the seed.
#include "kernels/dropout.h"

#include <algorithm>

#include "kernels/philox.h"
#include "runtime/common.h"

namespace oap {
namespace kern {

namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxBlocks = int64_t(1) << 22;  // (a grid has less than 2^32 threads)

template <typename T>
__device__ inline T drop_one(T x, T res, bool has_res, uint32_t w, const DropoutArgs& a) {
  // (selected, not multiplied: an infinity or NaN in a dropped place leaves nothing)
  float y = dropout_keeps(w, a.threshold) ? static_cast<float>(x) * a.scale : 0.f;
  if (has_res) y += static_cast<float>(res);
  return static_cast<T>(y);
}

// One element per thread and turn, for counters or addresses that no wider access takes.
template <typename T>
__global__ __launch_bounds__(kThreads) void oap_dropout_any(DropoutArgs a) {
  const uint64_t key = a.seed_ptr ? uint64_t(*a.seed_ptr) : a.seed;
  const T* res = static_cast<const T*>(a.residual);
  for (int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x; i < a.n;
       i += int64_t(gridDim.x) * kThreads) {
    const uint64_t g = a.offset + uint64_t(i);
    const Philox4 r = philox4x32_10(g >> 2, key);
    const uint32_t w = (g & 2) ? ((g & 1) ? r.w[3] : r.w[2]) : ((g & 1) ? r.w[1] : r.w[0]);
    static_cast<T*>(a.y)[i] = drop_one(static_cast<const T*>(a.x)[i], res ? res[i] : T(0.f),
                                       res != nullptr, w, a);
  }
}

}  // namespace

void dropout(Elem e, const DropoutArgs& a, hipStream_t s) {
  if (a.n <= 0) return;
  const int64_t blocks = std::min<int64_t>(ceil_div(a.n, kThreads), kMaxBlocks);
  elem_dispatch(e, [&](auto t) {
    using T = decltype(t);
    oap_dropout_any<T><<<dim3(unsigned(blocks)), kThreads, 0, s>>>(a);
  });
  OAP_HIP_CHECK(hipGetLastError());
}

}  // namespace kern
}  // namespace oap
