// Gate of a mixture of experts.  Per token: scores s = softmax(z) or sigmoid(z) over its E
// logits; the k experts of the highest choice values c = s + bias (without a bias the order of
// the logits), ties to the lowest index; with groups only the experts of the top groups (a
// group's value is the sum of its two highest c); weights s (over their sum) times a scale.
//
// Layout: L lanes share a token, each with EPL consecutive logits in registers (64 / L tokens a
// wave), so a reduction over a token is log2(L) exchanges for all the wave's tokens at once and
// equal values in a lower lane have the lower index.  One pass over the logits; nothing but the
// k picks is written.
//
// What bounds it is the selection, not the bytes, so it runs on 32-bit keys: the choice value's
// bits in unsigned order, the lowest replaced by the index.  A lane keeps its keys as sorted
// lists of four; a round is the maximum of the list heads, of the lanes (DPP), and a shift of one
// list.  16-bit logits leave room for the whole index in the unused bits, so the keys decide
// exactly.  Otherwise two neighbours in the order may be closer than the key's last bit, or than
// the fp32 error of c: such a token (about one in a thousand of random fp32 logits) is decided
// again from values in 64 bits.  In 32 bits alone two experts' scores would round to the same or
// the other order that often.  262144 x 128 fp32, eight chosen: 55 us forward (the read alone takes
// 26 us).  Equal choice values are always in doubt, one token of a wave after the other: the same
// gate with all logits equal takes 545 us, and 8192 x 256 bf16 with groups 66 us where a bias of
// zeros leaves the ties of 16-bit logits (32 us with a random bias).
#include "kernels/route.h"

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "runtime/common.h"

namespace oap {
namespace kern {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxBlocks = 2048;  // 8 workgroups per CU: loads are counted once per workgroup
constexpr float kLog2e = 1.44269504088896340736f;

template <typename T>
__device__ inline float load_one(const T* p) {
  return static_cast<float>(*p);
}
// A logit as it counts: NaN is an expert that is left out; +inf the largest finite number (its
// score is the limit's, not inf / inf); -0 is 0, equal in the keys too.
__device__ inline float as_logit(float v) {
  v = v == v ? v : -INFINITY;
  return fminf(v, FLT_MAX) + 0.f;
}

// v of lane ^ M in groups of L lanes, or of the lane mirrored in them: either way a reduction of
// a symmetric function after all steps.  VALU only up to 16 lanes.
template <int M>
__device__ inline int lane_xor(int v) {
  if constexpr (M == 1) return __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, true);
  if constexpr (M == 2) return __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, true);
  if constexpr (M == 4) return __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, true);
  if constexpr (M == 8) return __builtin_amdgcn_update_dpp(0, v, 0x140, 0xf, 0xf, true);
  return __shfl_xor(v, M, 64);
}
template <int L, typename F>
__device__ inline int group_reduce(int v, F&& f) {
  v = f(v, lane_xor<1>(v));
  v = f(v, lane_xor<2>(v));
  if constexpr (L >= 8) v = f(v, lane_xor<4>(v));
  if constexpr (L >= 16) v = f(v, lane_xor<8>(v));
  if constexpr (L >= 32) v = f(v, lane_xor<16>(v));
  if constexpr (L >= 64) v = f(v, lane_xor<32>(v));
  return v;
}
template <int L>
__device__ inline float group_max(float v) {
  return __int_as_float(group_reduce<L>(__float_as_int(v), [](int a, int b) {
    return __float_as_int(fmaxf(__int_as_float(a), __int_as_float(b)));
  }));
}
template <int L>
__device__ inline float group_sum(float v) {
  return __int_as_float(group_reduce<L>(__float_as_int(v), [](int a, int b) {
    return __float_as_int(__int_as_float(a) + __int_as_float(b));
  }));
}
template <int L>
__device__ inline unsigned group_umax(unsigned v) {
  return unsigned(group_reduce<L>(int(v), [](int a, int b) {
    return int(unsigned(a) > unsigned(b) ? unsigned(a) : unsigned(b));
  }));
}

// Orders this wave's LDS traffic: its instructions execute in order, so only the compiler has to
// keep them there.
__device__ inline void wave_sync() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_wave_barrier();
}

// Floats in unsigned order and back; 0 is below every number
__device__ inline unsigned ordered(float v) {
  const int b = __float_as_int(v);
  return unsigned(b) ^ (unsigned(b >> 31) | 0x80000000u);
}
__device__ inline float from_ordered(unsigned u) {
  return __int_as_float(int(u ^ (unsigned(~int(u) >> 31) | 0x80000000u)));
}

__device__ inline void order2(unsigned& a, unsigned& b) {
  const unsigned hi = a > b ? a : b, lo = a > b ? b : a;
  a = hi;
  b = lo;
}

// The chosen experts' weights from their logits.  Renormalised weights are ratios of scores, so
// they are formed from exponentials relative to the largest: scores that underflow still have
// them.  zref = the chosen's largest logit (sigmoid: at most 0).
__device__ inline float rel_score(bool sigmoid, float z, float zref) {
  if (!sigmoid) return expf(z - zref);
  return z > 0.f ? 1.f / (1.f + expf(-z)) : expf(z - zref) / (1.f + expf(z));
}

// Decides a token from 64-bit choice values (32-bit logits without a bias), the whole wave for
// one token.  It reads the token's row again and keeps the values in LDS (buf: one double per
// expert, and one per group), so that the many tokens that do not come here pay no registers for
// it.
template <typename T>
__device__ void decide_exactly(const RouteArgs& a, const T* row, int lane, double* buf,
                               int32_t* sel) {
  constexpr int L = 64;
  const double kout = -INFINITY;
  const int E = a.experts;
  const bool grouped = a.top_groups < a.groups, wide = a.bias || grouped;
  auto logit = [&](int e) { return as_logit(load_one(row + e)); };
  if (wide) {
    float zmax = -INFINITY;
    double sum = 0.0;
    if (!a.sigmoid) {
#pragma unroll 1
      for (int e = lane; e < E; e += L) zmax = fmaxf(zmax, logit(e));
      zmax = group_max<L>(zmax);
#pragma unroll 1
      for (int e = lane; e < E; e += L)
        if (logit(e) > -INFINITY) sum += exp(double(logit(e)) - double(zmax));
#pragma unroll
      for (int m = L / 2; m >= 1; m >>= 1) sum += __shfl_xor(sum, m, 64);
    }
#pragma unroll 1
    for (int e = lane; e < E; e += L) {
      const double z = logit(e);
      double c = exp(a.sigmoid ? -z : z - double(zmax));
      c = a.sigmoid ? 1.0 / (1.0 + c) : c / sum;
      if (a.bias) c += double(a.bias[e]);
      buf[e] = z > kout && c == c ? c : kout;
    }
  } else {
#pragma unroll 1
    for (int e = lane; e < E; e += L) buf[e] = logit(e);
  }
  wave_sync();
  if (grouped) {
    const int per = E / a.groups;
    double* gv = buf + E;
#pragma unroll 1
    for (int g = lane; g < a.groups; g += L) {
      double b0 = kout, b1 = kout;
#pragma unroll 1
      for (int e = g * per; e < (g + 1) * per; ++e) {
        b1 = fmax(b1, fmin(b0, buf[e]));
        b0 = fmax(b0, buf[e]);
      }
      gv[g] = b1 > kout ? b0 + b1 : b0;
    }
    wave_sync();
#pragma unroll 1
    for (int g = lane; g < a.groups; g += L) {
      int before = 0;
#pragma unroll 1
      for (int h = 0; h < a.groups; ++h) before += gv[h] > gv[g] || (gv[h] == gv[g] && h < g);
      if (before < a.top_groups) continue;
#pragma unroll 1
      for (int e = g * per; e < (g + 1) * per; ++e) buf[e] = kout;
    }
    wave_sync();
    if (!a.bias) {  // the order of the logits among the open groups
#pragma unroll 1
      for (int e = lane; e < E; e += L)
        if (buf[e] > kout) buf[e] = logit(e);
      wave_sync();
    }
  }
#pragma unroll 1
  for (int r = 0; r < a.k; ++r) {
    double v = kout;
    int i = E;
#pragma unroll 1
    for (int e = lane; e < E; e += L)
      if (buf[e] > v) {
        v = buf[e];
        i = e;
      }
#pragma unroll
    for (int m = L / 2; m >= 1; m >>= 1) {
      const double ov = __shfl_xor(v, m, 64);
      const int oi = __shfl_xor(i, m, 64);
      if (ov > v || (ov == v && oi < i)) {
        v = ov;
        i = oi;
      }
    }
    if (lane == 0) {
      sel[r] = v > kout ? i : -1;
      if (v > kout) buf[i] = kout;
    }
    wave_sync();
  }
}

// WIDE: choice values are computed (a bias, or groups), else they are the logits.
template <typename T, int L, int EPL, bool WIDE>
__global__ __launch_bounds__(kThreads) void oap_route(RouteArgs a, bool vec) {
  constexpr int TPB = kThreads / L, TPW = 64 / L;  // tokens per workgroup and wave, a turn
  constexpr bool kExact = sizeof(T) == 2 && !WIDE;
  constexpr unsigned kIdx = kExact ? 1023u : 15u;  // index bits of a key
  constexpr int NL = EPL / 4;                      // sorted lists of four
  // a wave's doubles of one token and its groups, or floats of all its tokens
  constexpr int kOne = L * EPL + (WIDE ? kRouteMaxGroups : 0), kAll = WIDE ? 32 * EPL : 0;
  constexpr int kBuf = kExact ? 1 : kOne > kAll ? kOne : kAll;
  __shared__ int32_t hist[kRouteMaxExperts];
  __shared__ int32_t sel[TPB * kRouteMaxK];
  __shared__ double buffer[kThreads / 64][kBuf];
  const int tid = threadIdx.x, lane = tid & (L - 1), slot = tid / L;
  const int wlane = tid & 63, wslot = wlane / L;
  double* wbuf = buffer[tid >> 6];
  int32_t* mysel = sel + slot * kRouteMaxK;
  for (int e = tid; e < a.experts; e += kThreads) hist[e] = 0;
  __syncthreads();
  const bool grouped = WIDE && a.top_groups < a.groups;

  for (int64_t t0 = int64_t(blockIdx.x) * TPB; t0 < a.tokens; t0 += int64_t(gridDim.x) * TPB) {
    const int64_t tok = t0 + slot;
    const bool live = tok < a.tokens;
    float z[EPL];
    const T* row = static_cast<const T*>(a.logits) + (live ? tok : 0) * a.ld;
    constexpr int VE = EPL * int(sizeof(T)) < 16 ? EPL : 16 / int(sizeof(T));
    if (vec) {
#pragma unroll
      for (int q = 0; q < EPL / VE; ++q) {
        struct alignas(VE * sizeof(T)) V {
          T v[VE];
        };
        const int e = lane * EPL + q * VE;
        const bool in = live && e < a.experts;
        V v = {};
        if (in) v = *reinterpret_cast<const V*>(row + e);
#pragma unroll
        for (int j = 0; j < VE; ++j) z[q * VE + j] = in ? static_cast<float>(v.v[j]) : -INFINITY;
      }
    } else {
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        const int e = lane * EPL + j;
        z[j] = live && e < a.experts ? load_one(row + e) : -INFINITY;
      }
    }
    float zmax = -INFINITY;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      z[j] = as_logit(z[j]);
      zmax = fmaxf(zmax, z[j]);
    }
    float sum = 0.f;
    if (!a.sigmoid && (WIDE || !a.renormalize)) {
      zmax = group_max<L>(zmax);
      const float ref = zmax > -INFINITY ? zmax : 0.f;
#pragma unroll
      for (int j = 0; j < EPL; ++j) sum += __builtin_amdgcn_exp2f((z[j] - ref) * kLog2e);
      sum = group_sum<L>(sum);
    }
    // Choice values in fp32 are off by err + 2^-24 |v|: a sigmoid by 2^-22 (its argument's rounding
    // and three operations), a softmax by 24 2^-24 of itself (an exponential, a sum over the
    // lanes, a quotient), at most that of the row's largest, 1 / sum; then the bias is added.
    bool doubt = false;
    const float err = a.sigmoid ? 0x1p-22f : 24.f * 0x1p-24f / sum;
    unsigned key[EPL];
    if constexpr (!WIDE) {
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        const unsigned low = kExact ? kIdx - unsigned(lane * EPL + j) : kIdx - unsigned(j);
        key[j] = z[j] > -INFINITY ? (ordered(z[j]) & ~kIdx) | low : 0u;
      }
    } else {
      const float ref = zmax > -INFINITY ? zmax : 0.f;
      float c[EPL];
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        const int e = lane * EPL + j;
        const float s = a.sigmoid
                            ? __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-z[j] * kLog2e))
                            : __builtin_amdgcn_exp2f((z[j] - ref) * kLog2e) *
                                  __builtin_amdgcn_rcpf(sum);
        const float v = a.bias && e < a.experts ? s + a.bias[e] : s;
        c[j] = z[j] > -INFINITY && v == v ? v : -INFINITY;
      }
      if (grouped) {
        const int per = a.experts / a.groups;
        float cmax = 0.f;
#pragma unroll
        for (int j = 0; j < EPL; ++j) cmax = c[j] > -INFINITY ? fmaxf(cmax, fabsf(c[j])) : cmax;
        const float tol = 4.f * err + 0x1p-20f * group_max<L>(cmax);
        float* buf = reinterpret_cast<float*>(wbuf) + wslot * L * EPL;
        wave_sync();
#pragma unroll
        for (int j = 0; j < EPL; ++j) buf[lane * EPL + j] = c[j];
        wave_sync();
        constexpr int NG = (kRouteMaxGroups + L - 1) / L;
        float gv[NG];
#pragma unroll
        for (int q = 0; q < NG; ++q) {
          const int g = lane + q * L;
          float b0 = -INFINITY, b1 = -INFINITY;
          if (g < a.groups)
            for (int e = 0; e < per; ++e) {
              const float v = buf[g * per + e];
              b1 = fmaxf(b1, fminf(b0, v));
              b0 = fmaxf(b0, v);
            }
          gv[q] = b1 > -INFINITY ? b0 + b1 : b0;
        }
        wave_sync();
#pragma unroll
        for (int q = 0; q < NG; ++q)
          if (lane + q * L < a.groups) buf[lane + q * L] = gv[q];
        wave_sync();
        // a group that may or may not be among the top ones leaves the token in doubt
#pragma unroll
        for (int q = 0; q < NG; ++q) {
          const int g = lane + q * L;
          if (g >= a.groups) continue;
          const float mine = gv[q];
          int before = 0, maybe = 0;
          for (int h = 0; h < a.groups; ++h) {
            const float o = buf[h];
            before += o > mine || (o == mine && h < g);
            maybe += h != g && mine > -INFINITY && o > -INFINITY && fabsf(o - mine) <= tol;
          }
          const bool in = before < a.top_groups;
          if (maybe && before - maybe < a.top_groups && before + maybe >= a.top_groups)
            doubt = true;
          gv[q] = in ? 1.f : 0.f;
        }
        wave_sync();
#pragma unroll
        for (int q = 0; q < NG; ++q)
          if (lane + q * L < a.groups) buf[lane + q * L] = gv[q];
        wave_sync();
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
          const int e = lane * EPL + j;
          const int g = e < a.experts ? e / per : 0;
          if (e >= a.experts || buf[g] == 0.f) c[j] = -INFINITY;
        }
      }
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        const float v = a.bias ? c[j] : z[j];
        key[j] = c[j] > -INFINITY ? (ordered(v) & ~kIdx) | (kIdx - unsigned(j)) : 0u;
      }
    }
#pragma unroll
    for (int q = 0; q < NL; ++q) {
      unsigned* l = key + 4 * q;
      order2(l[0], l[1]);
      order2(l[2], l[3]);
      order2(l[0], l[2]);
      order2(l[1], l[3]);
      order2(l[1], l[2]);
    }
    // k rounds, and one more that only looks whether the last pick was certain
    unsigned last = 0;
    const int rounds = kExact ? a.k : a.k + 1;
    for (int r = 0; r < rounds; ++r) {
      unsigned mine = key[0];
#pragma unroll
      for (int q = 1; q < NL; ++q) mine = key[4 * q] > mine ? key[4 * q] : mine;
      const unsigned best = group_umax<L>(mine);
      if constexpr (!kExact) {
        if (r > 0 && best) {
          if (!WIDE || !a.bias) {
            doubt |= (last ^ best) <= kIdx;
          } else {
            const float x = from_ordered(last & ~kIdx), y = from_ordered(best & ~kIdx);
            // (a key leaves out less than 2^-19 of its value)
            doubt |= !(x - y > 2.f * err + 0x1.2p-19f * fmaxf(fabsf(x), fabsf(y)));
          }
        }
        last = best;
      }
      if (r < a.k) {
        // the lowest lane that has it
        const unsigned long long eq = __ballot(mine == best);
        const unsigned long long of = eq >> (wlane & ~(L - 1));
        const bool win = (__ffsll(of) - 1) == lane;
        if (win) {
          const int i = kExact ? int(kIdx - (best & kIdx)) : lane * EPL + int(kIdx - (best & kIdx));
          mysel[r] = best ? i : -1;
        }
#pragma unroll
        for (int q = 0; q < NL; ++q) {
          const bool pop = win && key[4 * q] == best;
#pragma unroll
          for (int j = 0; j < 3; ++j) key[4 * q + j] = pop ? key[4 * q + j + 1] : key[4 * q + j];
          key[4 * q + 3] = pop ? 0u : key[4 * q + 3];
        }
      }
    }
    if constexpr (!kExact) {
      // tokens in doubt, one at a time
      const unsigned long long left = __ballot(doubt && live);
      for (int w = 0; left && w < TPW; ++w) {
        const unsigned long long mask = (L == 64 ? ~0ull : (1ull << L % 64) - 1) << (w * L % 64);
        if (!(left & mask)) continue;
        const int one = (tid >> 6) * TPW + w;
        wave_sync();
        decide_exactly<T>(a, static_cast<const T*>(a.logits) + (t0 + one) * a.ld, wlane, wbuf,
                          sel + one * kRouteMaxK);
        wave_sync();
      }
    }
    wave_sync();
    if (live && a.k <= L) {  // weights: a lane per slot, which reads its logit once
      const int i = lane < a.k ? mysel[lane] : -1;
      const float zr = i >= 0 ? as_logit(load_one(row + i)) : -INFINITY;
      float zref = a.sigmoid ? 0.f : zmax;
      if (a.renormalize) {
        zref = group_max<L>(zr);
        if (a.sigmoid) zref = fminf(zref, 0.f);
      }
      const float score = i >= 0 ? rel_score(a.sigmoid, zr, zref) : 0.f;
      const float norm = a.renormalize ? group_sum<L>(score) : a.sigmoid ? 1.f : sum;
      if (lane < a.k) {
        a.weights[tok * a.k + lane] = i >= 0 ? score / norm * a.scale : 0.f;
        a.indices[tok * a.k + lane] = i;
        if (i >= 0) atomicAdd(&hist[i], 1);
      }
    } else if (live) {
      // lane l of the token takes slots l, l + L, ...
      float zref = -INFINITY, norm = 0.f;
      if (a.renormalize) {
        for (int r = lane; r < a.k; r += L)
          if (mysel[r] >= 0) zref = fmaxf(zref, as_logit(load_one(row + mysel[r])));
        zref = group_max<L>(zref);
        if (a.sigmoid) zref = fminf(zref, 0.f);
        for (int r = lane; r < a.k; r += L)
          if (mysel[r] >= 0)
            norm += rel_score(a.sigmoid, as_logit(load_one(row + mysel[r])), zref);
        norm = group_sum<L>(norm);
      } else {
        zref = a.sigmoid ? 0.f : zmax;
        norm = a.sigmoid ? 1.f : sum;
      }
      for (int r = lane; r < a.k; r += L) {
        const int i = mysel[r];
        float w = 0.f;
        if (i >= 0) {
          w = rel_score(a.sigmoid, as_logit(load_one(row + i)), zref) / norm * a.scale;
          atomicAdd(&hist[i], 1);
        }
        a.weights[tok * a.k + r] = w;
        a.indices[tok * a.k + r] = i;
      }
    }
    wave_sync();
  }
  __syncthreads();
  int32_t* out = gridDim.x == 1 ? a.counts : a.partial + int64_t(blockIdx.x) * a.experts;
  for (int e = tid; e < a.experts; e += kThreads) out[e] = hist[e];
}

// counts[e] = sum over workgroups of their histograms
constexpr int kCountLanes = 64;  // threads per column

__global__ __launch_bounds__(16 * kCountLanes) void oap_route_counts(
    const int32_t* __restrict__ partial, int blocks, int experts, int32_t* __restrict__ counts) {
  __shared__ int32_t acc[16 * kCountLanes];
  const int col = blockIdx.x * 16 + (threadIdx.x & 15), r0 = threadIdx.x >> 4;
  int32_t v = 0;
  if (col < experts) {
#pragma unroll 8
    for (int r = r0; r < blocks; r += kCountLanes) v += partial[int64_t(r) * experts + col];
  }
  acc[threadIdx.x] = v;
  for (int h = kCountLanes / 2; h >= 1; h >>= 1) {
    __syncthreads();
    if (r0 < h) acc[threadIdx.x] += acc[threadIdx.x + 16 * h];
  }
  if (r0 == 0 && col < experts) counts[col] = acc[threadIdx.x];
}

// Gradient of the weights w into the logits (C the chosen, g the gradient of w):
//   renormalised softmax   dz_c = w_c (g_c - sum_C g w / scale)
//   renormalised sigmoid   the same times 1 - s_c
//   sigmoid                dz_c = w_c (1 - s_c) g_c
//   softmax                dz_i = s_i (scale [i in C] g_i - sum_C g w), all experts
// One workgroup forms the rows of a few tokens in LDS (zeros, then the chosen) and writes them
// out in order.  262144 x 128 fp32: 45 us, 3.0 TB/s written, little more than half of a copy's
// rate: the zeros, the chosen (a thread per token) and the write follow each other with a barrier
// between.
// The plain softmax reads its logits three times and writes single elements: 183 us.
constexpr int kGradTile = 8192;  // floats of LDS

template <typename T>
__global__ __launch_bounds__(kThreads) void oap_route_grad(RouteGradArgs a, int tpb) {
  __shared__ __attribute__((aligned(16))) float tile[kGradTile];
  __shared__ float dense[kThreads], zmax[kThreads], rsum[kThreads];
  const int tid = threadIdx.x, E = a.experts, k = a.k;
  const bool all = !a.sigmoid && !a.renormalize;
  const T* z = static_cast<const T*>(a.logits);
  for (int64_t t0 = int64_t(blockIdx.x) * tpb; t0 < a.tokens; t0 += int64_t(gridDim.x) * tpb) {
    const int nt = int(a.tokens - t0 < tpb ? a.tokens - t0 : tpb);
    __syncthreads();
    for (int i = tid; i < (nt * E + 3) / 4; i += kThreads)
      reinterpret_cast<float4*>(tile)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (all) {  // the row's softmax again: 16 lanes per token
      const int lane = tid & 15;
      for (int t = tid >> 4; t < nt; t += kThreads / 16) {
        const T* row = z + (t0 + t) * a.ld;
        float m = -INFINITY;
        for (int e = lane; e < E; e += 16) {
          m = fmaxf(m, as_logit(load_one(row + e)));
        }
        m = group_max<16>(m);
        float s = 0.f;
        for (int e = lane; e < E; e += 16) {
          const float v = as_logit(load_one(row + e));
          s += v > -INFINITY ? expf(v - m) : 0.f;
        }
        s = group_sum<16>(s);
        if (lane == 0) {
          zmax[t] = m;
          rsum[t] = s;
        }
      }
    }
    __syncthreads();
    if (tid < nt) {
      const int64_t b = (t0 + tid) * k;
      float dot = 0.f;
      for (int r = 0; r < k; ++r)
        if (a.indices[b + r] >= 0) dot += a.grad[b + r] * a.weights[b + r];
      dense[tid] = dot;
      const float mean = a.renormalize ? dot / a.scale : 0.f;
      for (int r = 0; r < k; ++r) {
        const int e = a.indices[b + r];
        if (e < 0) continue;
        float d = a.weights[b + r] * (a.grad[b + r] - mean);
        if (a.sigmoid) d *= 1.f / (1.f + expf(load_one(z + (t0 + tid) * a.ld + e)));
        tile[tid * E + e] = d;
      }
    }
    __syncthreads();
    T* out = static_cast<T*>(a.grad_logits) + t0 * E;
    if (all) {
      for (int i = tid; i < nt * E; i += kThreads) {
        const int t = i / E;
        const float v = as_logit(load_one(z + (t0 + t) * a.ld + (i - t * E)));
        float d = tile[i];
        if (v > -INFINITY) d -= expf(v - zmax[t]) / rsum[t] * dense[t];
        out[i] = static_cast<T>(d);
      }
    } else if (E % Vec16<T>::n == 0) {  // the rows are whole 16-byte runs
      for (int i = tid; i < nt * E / Vec16<T>::n; i += kThreads) {
        Vec16<T> o;
#pragma unroll
        for (int q = 0; q < Vec16<T>::n; q += 4) {
          const float4 d = *reinterpret_cast<const float4*>(tile + i * Vec16<T>::n + q);
          o.v[q] = static_cast<T>(d.x);
          o.v[q + 1] = static_cast<T>(d.y);
          o.v[q + 2] = static_cast<T>(d.z);
          o.v[q + 3] = static_cast<T>(d.w);
        }
        reinterpret_cast<Vec16<T>*>(out)[i] = o;
      }
    } else {
      for (int i = tid; i < nt * E; i += kThreads) out[i] = static_cast<T>(tile[i]);
    }
  }
}

int route_lanes(int experts) {
  return experts <= 64 ? 4 : experts <= 128 ? 8 : experts <= 256 ? 16 : experts <= 512 ? 32 : 64;
}

int64_t route_blocks(int64_t tokens, int experts) {
  return std::min<int64_t>(ceil_div(tokens, kThreads / route_lanes(experts)), kMaxBlocks);
}

template <typename T, bool WIDE>
void route_launch(const RouteArgs& a, unsigned blocks, hipStream_t s) {
  const int e = a.experts;
  // 16 bytes of a row at a time (EPL = 4: its four elements)
  const int ve = std::min<int>(e <= 16 ? 4 : 16, 16 / int(sizeof(T)));
  const bool vec = e % ve == 0 && a.ld % ve == 0 &&
                   reinterpret_cast<uintptr_t>(a.logits) % (ve * sizeof(T)) == 0;
  if (e <= 16)
    oap_route<T, 4, 4, WIDE><<<dim3(blocks), kThreads, 0, s>>>(a, vec);
  else if (e <= 64)
    oap_route<T, 4, 16, WIDE><<<dim3(blocks), kThreads, 0, s>>>(a, vec);
  else if (e <= 128)
    oap_route<T, 8, 16, WIDE><<<dim3(blocks), kThreads, 0, s>>>(a, vec);
  else if (e <= 256)
    oap_route<T, 16, 16, WIDE><<<dim3(blocks), kThreads, 0, s>>>(a, vec);
  else if (e <= 512)
    oap_route<T, 32, 16, WIDE><<<dim3(blocks), kThreads, 0, s>>>(a, vec);
  else
    oap_route<T, 64, 16, WIDE><<<dim3(blocks), kThreads, 0, s>>>(a, vec);
}

}  // namespace

size_t route_partial_bytes(int64_t tokens, int experts) {
  const int64_t b = route_blocks(tokens, experts);
  return b <= 1 ? 0 : size_t(b) * size_t(experts) * 4;
}

void route(Elem e, const RouteArgs& a, hipStream_t s) {
  OAP_CHECK(a.experts >= 1 && a.experts <= kRouteMaxExperts && a.k >= 1 && a.k <= kRouteMaxK &&
                a.k <= a.experts && a.groups >= 1 && a.groups <= kRouteMaxGroups &&
                a.experts % a.groups == 0 && a.top_groups >= 1 && a.top_groups <= a.groups &&
                a.tokens >= 0 && a.ld >= a.experts,
            "route: bad shape");
  // (no token: one workgroup still writes the zero counts)
  const unsigned blocks = unsigned(std::max<int64_t>(1, route_blocks(a.tokens, a.experts)));
  const bool wide = a.bias || a.top_groups < a.groups;
  elem_dispatch(e, [&](auto t) {
    using T = decltype(t);
    if (wide)
      route_launch<T, true>(a, blocks, s);
    else
      route_launch<T, false>(a, blocks, s);
  });
  OAP_HIP_CHECK(hipGetLastError());
  if (blocks > 1) {
    oap_route_counts<<<dim3(unsigned(ceil_div(a.experts, 16))), 16 * kCountLanes, 0,
                       s>>>(a.partial, int(blocks), a.experts, a.counts);
    OAP_HIP_CHECK(hipGetLastError());
  }
}

void route_grad(Elem e, const RouteGradArgs& a, hipStream_t s) {
  OAP_CHECK(a.experts >= 1 && a.experts <= kRouteMaxExperts && a.k >= 1 && a.k <= kRouteMaxK,
            "route_grad: bad shape");
  if (a.tokens <= 0) return;
  const int tpb = std::min(kThreads, kGradTile / a.experts);
  const unsigned blocks = unsigned(std::min<int64_t>(ceil_div(a.tokens, tpb), 1 << 20));
  elem_dispatch(e, [&](auto t) {
    using T = decltype(t);
    oap_route_grad<T><<<dim3(blocks), kThreads, 0, s>>>(a, tpb);
  });
  OAP_HIP_CHECK(hipGetLastError());
}

}  // namespace kern
}  // namespace oap
