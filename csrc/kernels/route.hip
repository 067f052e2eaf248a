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
// The values that decide a choice are formed in 64 bits where they are computed (bias, groups):
// in 32 bits two experts' scores round to the same or the other order once in a few thousand
// tokens.  The logits' own order needs no arithmetic.
#include "kernels/route.h"

#include <algorithm>
#include <cmath>

#include "runtime/common.h"

namespace oap {
namespace kern {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxBlocks = 2048;  // 8 workgroups per CU: loads are counted once per workgroup

template <typename T>
__device__ inline float load_one(const T* p) {
  return static_cast<float>(*p);
}

// k, and the order of two candidates: higher value first, then lower index
template <typename K>
struct Best {
  K v;
  int i;
};
template <typename K>
__device__ inline bool beats(const Best<K>& a, const Best<K>& b) {
  return a.v > b.v || (a.v == b.v && a.i < b.i);
}

template <int L, typename V>
__device__ inline V group_max(V v) {
#pragma unroll
  for (int m = L / 2; m >= 1; m >>= 1) {
    const V o = __shfl_xor(v, m, 64);
    v = o > v ? o : v;
  }
  return v;
}
template <int L, typename V>
__device__ inline V group_sum(V v) {
#pragma unroll
  for (int m = L / 2; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
  return v;
}

// The chosen experts' weights from their logits.  Renormalised weights are ratios of scores, so
// they are formed from exponentials relative to the largest: scores that underflow still have
// them.  zref = the chosen's largest logit (sigmoid: at most 0).
__device__ inline float rel_score(bool sigmoid, float z, float zref) {
  if (!sigmoid) return expf(z - zref);
  return z > 0.f ? 1.f / (1.f + expf(-z)) : expf(z - zref) / (1.f + expf(z));
}

template <typename T, typename K, int L, int EPL>
__global__ __launch_bounds__(kThreads) void oap_route(RouteArgs a) {
  constexpr int TPB = kThreads / L;  // tokens per workgroup and turn
  constexpr bool kWide = sizeof(K) == 8;
  __shared__ int32_t hist[kRouteMaxExperts];
  __shared__ float sel_z[TPB * kRouteMaxK];
  __shared__ int32_t sel_i[TPB * kRouteMaxK];
  __shared__ double cbuf[kWide ? kThreads * EPL : 1];
  __shared__ double gval[kWide ? TPB * kRouteMaxGroups : 1];
  __shared__ unsigned long long gmask[TPB];
  const int tid = threadIdx.x, lane = tid & (L - 1), slot = tid / L;
  for (int e = tid; e < a.experts; e += kThreads) hist[e] = 0;
  const float ninf = -INFINITY;
  const bool grouped = a.top_groups < a.groups;

  for (int64_t t0 = int64_t(blockIdx.x) * TPB; t0 < a.tokens; t0 += int64_t(gridDim.x) * TPB) {
    __syncthreads();  // (hist is clear; the last turn's picks are written)
    const int64_t tok = t0 + slot;
    const bool live = tok < a.tokens;
    float z[EPL];
    const T* row = static_cast<const T*>(a.logits) + (live ? tok : 0) * a.ld;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const int e = lane * EPL + j;
      const float v = live && e < a.experts ? load_one(row + e) : ninf;
      z[j] = v == v ? v : ninf;  // a NaN logit is an expert that is left out, as -inf is
    }
    float zmax = z[0];
#pragma unroll
    for (int j = 1; j < EPL; ++j) zmax = fmaxf(zmax, z[j]);
    zmax = group_max<L>(zmax);
    float sum = 0.f;
    if (!a.sigmoid && !a.renormalize) {
#pragma unroll
      for (int j = 0; j < EPL; ++j) sum += z[j] > ninf ? expf(z[j] - zmax) : 0.f;
      sum = group_sum<L>(sum);
    }
    K key[EPL];
    if constexpr (!kWide) {
#pragma unroll
      for (int j = 0; j < EPL; ++j) key[j] = z[j];
    } else {
      const double kout = -INFINITY;
      double s64 = 0.0;
      if (!a.sigmoid) {
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
          key[j] = z[j] > ninf ? exp(double(z[j]) - double(zmax)) : 0.0;
          s64 += key[j];
        }
        s64 = group_sum<L>(s64);
      }
#pragma unroll
      for (int j = 0; j < EPL; ++j) {
        const int e = lane * EPL + j;
        double c = a.sigmoid ? 1.0 / (1.0 + exp(-double(z[j]))) : key[j] / s64;
        if (a.bias && e < a.experts) c += double(a.bias[e]);
        key[j] = z[j] > ninf && c == c ? c : kout;
      }
      if (grouped) {
        const int per = a.experts / a.groups;
        if (lane == 0) gmask[slot] = 0;
#pragma unroll
        for (int j = 0; j < EPL; ++j) cbuf[tid * EPL + j] = key[j];
        __syncthreads();
        const double* c = cbuf + slot * L * EPL;
        for (int g = lane; g < a.groups; g += L) {
          double b0 = kout, b1 = kout;
          for (int e = 0; e < per; ++e) {
            const double v = c[g * per + e];
            b1 = fmax(b1, fmin(b0, v));
            b0 = fmax(b0, v);
          }
          gval[slot * kRouteMaxGroups + g] = b1 > kout ? b0 + b1 : b0;
        }
        __syncthreads();
        const double* gv = gval + slot * kRouteMaxGroups;
        for (int g = lane; g < a.groups; g += L) {
          int before = 0;
          for (int h = 0; h < a.groups; ++h)
            before += gv[h] > gv[g] || (gv[h] == gv[g] && h < g);
          if (before < a.top_groups) atomicOr(&gmask[slot], 1ull << g);
        }
        __syncthreads();
        const unsigned long long open = gmask[slot];
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
          const int g = (lane * EPL + j) / per;
          if (g >= a.groups || !((open >> g) & 1)) key[j] = kout;
        }
      }
      if (!a.bias) {  // the order of the logits among the open groups
#pragma unroll
        for (int j = 0; j < EPL; ++j) key[j] = key[j] > kout ? double(z[j]) : kout;
      }
    }

    // k rounds: every lane's best, the token's best, and its removal
    for (int r = 0; r < a.k; ++r) {
      Best<K> b = {key[0], lane * EPL};
      float bz = z[0];
#pragma unroll
      for (int j = 1; j < EPL; ++j) {
        const bool up = key[j] > b.v;
        b.v = up ? key[j] : b.v;
        b.i = up ? lane * EPL + j : b.i;
        bz = up ? z[j] : bz;
      }
      const int mine = b.i;
#pragma unroll
      for (int m = L / 2; m >= 1; m >>= 1) {
        const Best<K> o = {__shfl_xor(b.v, m, 64), __shfl_xor(b.i, m, 64)};
        if (beats(o, b)) b = o;
      }
      const bool some = b.v > K(ninf);
      if (b.i == mine && live) {
        sel_z[slot * kRouteMaxK + r] = bz;
        sel_i[slot * kRouteMaxK + r] = some ? b.i : -1;
        if (some) atomicAdd(&hist[b.i], 1);
      }
#pragma unroll
      for (int j = 0; j < EPL; ++j)
        if (lane * EPL + j == b.i) key[j] = K(ninf);
    }
    __syncthreads();
    if (live) {
      // weights: lane l of the token takes slots l, l + L, ...
      const float* sz = sel_z + slot * kRouteMaxK;
      const int32_t* si = sel_i + slot * kRouteMaxK;
      float zref = ninf, norm = 1.f;
      if (a.renormalize) {
        for (int r = 0; r < a.k; ++r) zref = si[r] >= 0 ? fmaxf(zref, sz[r]) : zref;
        if (a.sigmoid) zref = fminf(zref, 0.f);
        norm = 0.f;
        for (int r = 0; r < a.k; ++r) norm += si[r] >= 0 ? rel_score(a.sigmoid, sz[r], zref) : 0.f;
      } else {
        zref = a.sigmoid ? 0.f : zmax;
        norm = a.sigmoid ? 1.f : sum;
      }
      for (int r = lane; r < a.k; r += L) {
        const float w = si[r] >= 0 ? rel_score(a.sigmoid, sz[r], zref) / norm * a.scale : 0.f;
        a.weights[tok * a.k + r] = w;
        a.indices[tok * a.k + r] = si[r];
      }
    }
  }
  __syncthreads();
  int32_t* out = gridDim.x == 1 ? a.counts : a.partial + int64_t(blockIdx.x) * a.experts;
  for (int e = tid; e < a.experts; e += kThreads) out[e] = hist[e];
}

// counts[e] = sum over workgroups of their histograms
__global__ __launch_bounds__(kThreads) void oap_route_counts(const int32_t* __restrict__ partial,
                                                             int blocks, int experts,
                                                             int32_t* __restrict__ counts) {
  __shared__ int32_t acc[kThreads];
  const int col = blockIdx.x * 16 + (threadIdx.x & 15), r0 = threadIdx.x >> 4;
  int32_t v = 0;
  if (col < experts)
    for (int r = r0; r < blocks; r += 16) v += partial[int64_t(r) * experts + col];
  acc[threadIdx.x] = v;
  __syncthreads();
  if (r0 == 0 && col < experts) {
    for (int r = 1; r < 16; ++r) v += acc[r * 16 + threadIdx.x];
    counts[col] = v;
  }
}

// Gradient of the weights w into the logits (C the chosen, g the gradient of w):
//   renormalised softmax   dz_c = w_c (g_c - sum_C g w / scale)
//   renormalised sigmoid   the same times 1 - s_c
//   sigmoid                dz_c = w_c (1 - s_c) g_c
//   softmax                dz_i = s_i (scale [i in C] g_i - sum_C g w), all experts
// One workgroup forms the rows of a few tokens in LDS (zeros, then the chosen) and writes them
// out in order: the write of the whole gradient is what bounds it.
constexpr int kGradTile = 8192;  // floats of LDS

template <typename T>
__global__ __launch_bounds__(kThreads) void oap_route_grad(RouteGradArgs a, int tpb) {
  __shared__ float tile[kGradTile];
  __shared__ float dense[kThreads], zmax[kThreads], rsum[kThreads];
  const int tid = threadIdx.x, E = a.experts, k = a.k;
  const bool all = !a.sigmoid && !a.renormalize;
  const T* z = static_cast<const T*>(a.logits);
  for (int64_t t0 = int64_t(blockIdx.x) * tpb; t0 < a.tokens; t0 += int64_t(gridDim.x) * tpb) {
    const int nt = int(a.tokens - t0 < tpb ? a.tokens - t0 : tpb);
    __syncthreads();
    for (int i = tid; i < nt * E; i += kThreads) tile[i] = 0.f;
    if (all) {  // the row's softmax again: 16 lanes per token
      const int lane = tid & 15;
      for (int t = tid >> 4; t < nt; t += kThreads / 16) {
        const T* row = z + (t0 + t) * a.ld;
        float m = -INFINITY;
        for (int e = lane; e < E; e += 16) {
          const float v = load_one(row + e);
          m = v > m ? v : m;
        }
        m = group_max<16>(m);
        float s = 0.f;
        for (int e = lane; e < E; e += 16) {
          const float v = load_one(row + e);
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
    for (int i = tid; i < nt * E; i += kThreads) {
      float d = tile[i];
      if (all) {
        const int t = i / E;
        const float v = load_one(z + (t0 + t) * a.ld + (i - t * E));
        if (v > -INFINITY) d -= expf(v - zmax[t]) / rsum[t] * dense[t];
      }
      out[i] = static_cast<T>(d);
    }
  }
}

int route_lanes(int experts) {
  return experts <= 64 ? 4 : experts <= 128 ? 8 : experts <= 256 ? 16 : experts <= 512 ? 32 : 64;
}

int64_t route_blocks(int64_t tokens, int experts) {
  return std::min<int64_t>(ceil_div(tokens, kThreads / route_lanes(experts)), kMaxBlocks);
}

template <typename T, typename K>
void route_launch(const RouteArgs& a, unsigned blocks, hipStream_t s) {
  const int e = a.experts;
  if (e <= 16)
    oap_route<T, K, 4, 4><<<dim3(blocks), kThreads, 0, s>>>(a);
  else if (e <= 64)
    oap_route<T, K, 4, 16><<<dim3(blocks), kThreads, 0, s>>>(a);
  else if (e <= 128)
    oap_route<T, K, 8, 16><<<dim3(blocks), kThreads, 0, s>>>(a);
  else if (e <= 256)
    oap_route<T, K, 16, 16><<<dim3(blocks), kThreads, 0, s>>>(a);
  else if (e <= 512)
    oap_route<T, K, 32, 16><<<dim3(blocks), kThreads, 0, s>>>(a);
  else
    oap_route<T, K, 64, 16><<<dim3(blocks), kThreads, 0, s>>>(a);
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
      route_launch<T, double>(a, blocks, s);
    else
      route_launch<T, float>(a, blocks, s);
  });
  OAP_HIP_CHECK(hipGetLastError());
  if (blocks > 1) {
    oap_route_counts<<<dim3(unsigned(ceil_div(a.experts, 16))), kThreads, 0, s>>>(
        a.partial, int(blocks), a.experts, a.counts);
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
