// Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3",
// SC 2011): 128 random bits from a 64-bit counter and a 64-bit key, no state.  Each of ten
// rounds is two 32 x 32 -> 64 bit products, four xors and a key step that is the same for the
// whole wave.
#pragma once

#include <cstdint>

#include "kernels/rng.h"

namespace oap {
namespace kern {

struct Philox4 {
  uint32_t w[4];
};

OAP_HD inline Philox4 philox4x32_10(uint64_t counter, uint64_t key) {
  uint32_t c0 = uint32_t(counter), c1 = uint32_t(counter >> 32), c2 = 0, c3 = 0;
  uint32_t k0 = uint32_t(key), k1 = uint32_t(key >> 32);
#if defined(__clang__)
#pragma unroll
#endif
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = uint64_t(0xD2511F53u) * c0, p1 = uint64_t(0xCD9E8D57u) * c2;
    const uint32_t n0 = uint32_t(p1 >> 32) ^ c1 ^ k0, n2 = uint32_t(p0 >> 32) ^ c3 ^ k1;
    c1 = uint32_t(p1);
    c3 = uint32_t(p0);
    c0 = n0;
    c2 = n2;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

// Whether dropout keeps the element whose 32 random bits are w: the threshold is
// round(p 2^32), so 2^32 (p = 1) keeps nothing.
OAP_HD inline bool dropout_keeps(uint32_t w, uint64_t threshold) {
  return uint64_t(w) >= threshold;
}

}  // namespace kern
}  // namespace oap
