// Element types of the torch-tensor training ops (dropout, route, softmax cross entropy) and
// their conversions: storage in 32 or 16 bits, arithmetic always in fp32 or wider.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace oap {
namespace kern {

enum class Elem : int { F32 = 0, BF16 = 1, F16 = 2 };

inline int elem_size(Elem e) { return e == Elem::F32 ? 4 : 2; }

// Calls f.template operator()<T>() with the C++ type of e.
template <typename F>
void elem_dispatch(Elem e, F&& f) {
  switch (e) {
    case Elem::F32: f(float{}); break;
    case Elem::BF16: f(__bf16{}); break;
    case Elem::F16: f(_Float16{}); break;
  }
}

// 16 bytes of elements, the widest global access of a lane
template <typename T>
struct alignas(16) Vec16 {
  static constexpr int n = 16 / sizeof(T);
  T v[n];
};

}  // namespace kern
}  // namespace oap
