// Dropout whose mask is never stored: element i of the (global) array is kept when word i & 3 of
// Philox4x32-10 at counter i >> 2 is at least round(p 2^32), so the backward pass, another shard
// or the host engine form the same mask from the seed.
//
// Bound by memory: the generator's ten rounds (20 wide multiplications for four elements) run
// under the loads.  1M x 100 fp32: 131 us a pass, 6.1 TB/s; bf16 79 us, 5.0 TB/s.  Where the offset
// is no multiple of four, or an address of 16, every element forms a block of the generator for
// itself, which then bounds it: 330 and 300 us.
#include "kernels/dropout.h"

#include <algorithm>

#include "kernels/philox.h"
#include "runtime/common.h"

namespace oap {
namespace kern {

namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxBlocks = int64_t(1) << 22;  // (a grid has less than 2^32 threads)

__device__ inline uint32_t word_of(const Philox4& r, uint64_t g) {
  return (g & 2) ? ((g & 1) ? r.w[3] : r.w[2]) : ((g & 1) ? r.w[1] : r.w[0]);
}

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
    const uint32_t w = word_of(philox4x32_10(g >> 2, key), g);
    static_cast<T*>(a.y)[i] = drop_one(static_cast<const T*>(a.x)[i], res ? res[i] : T(0.f),
                                       res != nullptr, w, a);
  }
}

// 16 bytes per thread and turn: the words of four neighbouring elements are one block of the
// generator, so an element costs a quarter of it.  Needs offset % 4 == 0 and 16-byte addresses.
template <typename T, bool RES>
__global__ __launch_bounds__(kThreads) void oap_dropout_vec(DropoutArgs a) {
  typedef Vec16<T> V;
  const uint64_t key = a.seed_ptr ? uint64_t(*a.seed_ptr) : a.seed;
  const int64_t nv = a.n / V::n;
  const V* x = static_cast<const V*>(a.x);
  const V* res = static_cast<const V*>(a.residual);
  V* y = static_cast<V*>(a.y);
  int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  for (; i < nv; i += int64_t(gridDim.x) * kThreads) {
    const V v = x[i];
    V r = {};
    if (RES) r = res[i];
    V o;
#pragma unroll
    for (int q = 0; q < V::n / 4; ++q) {
      const uint64_t g = (a.offset >> 2) + uint64_t(i) * (V::n / 4) + q;
      const Philox4 w = philox4x32_10(g, key);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        o.v[4 * q + j] = drop_one(v.v[4 * q + j], r.v[4 * q + j], RES, w.w[j], a);
    }
    y[i] = o;
  }
  // the last, partial vector: one element per thread of the first workgroup
  const int64_t t = nv * V::n + threadIdx.x;
  if (blockIdx.x == 0 && t < a.n) {
    const uint64_t g = a.offset + uint64_t(t);
    const uint32_t w = word_of(philox4x32_10(g >> 2, key), g);
    const T rt = RES ? static_cast<const T*>(a.residual)[t] : T(0.f);
    static_cast<T*>(a.y)[t] =
        drop_one(static_cast<const T*>(a.x)[t], rt, RES, w, a);
  }
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace

void dropout(Elem e, const DropoutArgs& a, hipStream_t s) {
  if (a.n <= 0) return;
  const bool vec = a.offset % 4 == 0 && aligned16(a.x) && aligned16(a.y) && aligned16(a.residual);
  const int64_t items = vec ? a.n / (16 / elem_size(e)) : a.n;
  const int64_t blocks =
      std::max<int64_t>(1, std::min<int64_t>(ceil_div(items, kThreads), kMaxBlocks));
  elem_dispatch(e, [&](auto t) {
    using T = decltype(t);
    if (!vec)
      oap_dropout_any<T><<<dim3(unsigned(blocks)), kThreads, 0, s>>>(a);
    else if (a.residual)
      oap_dropout_vec<T, true><<<dim3(unsigned(blocks)), kThreads, 0, s>>>(a);
    else
      oap_dropout_vec<T, false><<<dim3(unsigned(blocks)), kThreads, 0, s>>>(a);
  });
  OAP_HIP_CHECK(hipGetLastError());
}

}  // namespace kern
}  // namespace oap
