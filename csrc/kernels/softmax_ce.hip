// Softmax cross entropy of logits z = x W^T + b over V classes, for N rows of D features:
//   m_n = max_v z_nv,  s_n = sum_v exp(z_nv - m_n),  loss_n = log s_n + (m_n - z_{n, t_n})
//   dz_nv = g_n (exp(z_nv - m_n) / s_n - [v = t_n]),  dx = dz W,  dW = dz^T x,  db_v = sum_n dz_nv
// N V logits are never stored.  The forward pass keeps (max, sum of exp) of each row and class
// tile; the backward pass goes over the classes in pieces, forms a piece's logits again,
// stores its dz in the operand type and multiplies it into dx and dW while it is in cache.
//
// Operands are bf16, fp16, fp32, or (larger fp32 problems) fp32 split in two fp16 numbers.  A
// product then keeps 22 bits of each: x and a piece's classes are copied into split images at
// powers of two, every row of x at its own in the logits (a row is right whatever the others
// hold), a piece's classes at one, and so the rows in dW: a number keeps an absolute 2^-40 of the
// largest there.  dz is stored in fp32 and split as a tile of it is read, at a power of two per row
// for dx (its largest magnitude is known, 1 - p of the target) and per class for dW (from maxima
// that the logits' epilogue keeps): a probability of 2^-60 has its 22 bits where all of its sum are
// as small.  At one scale for all, probabilities below 2^-24 lost bits and those below 2^-39 all.
//
// Roundings: sums, statistics, losses and dx's slabs are fp32, and a result is rounded once.  With
// 16-bit operands dz is rounded to their type (at most 2^-8 of it in bf16, 2^-11 in fp16) before
// it meets W and x, whose own rounding is as large: that is what the matrix units take, and dz in
// two parts would double the work of dX and dW.  db sums dz in fp32 before that rounding.
//
// What bounds it, at 8192 x 131072 x 2048 bf16 (16.7 to 17.1 ms by card for forward and gradients,
// 8 N V D operations): the matrix units under the chip's power limit, 0.98 to 1.10 PF/s in each
// product (a library product of the same shapes 1.23).  At 1024 x 2M x 100 fp32 (11.1 ms): k is
// short, so each tile's epilogue and staging weigh as much as its MFMAs, and dz, written once and
// read twice, is 26 GB.
#include "kernels/softmax_ce.h"

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <mutex>
#include <set>
#include <utility>

#include "kernels/gemm_tile.h"
#include "runtime/common.h"

namespace oap {
namespace kern {

namespace {

// Logits are kept in units of ln 2, z log2(e), so that a power is one v_exp_f32 of a difference.
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.693147180559945309417f;
__device__ inline float pow2(float d) { return __builtin_amdgcn_exp2f(d); }

// Sum of the 32 lanes of each half wave, in all of them: VALU only (an LDS exchange a step would
// cost more than the additions)
template <int CTRL>
__device__ inline float dpp_add(float v) {
  const int o = __builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true);
  return v + __int_as_float(o);
}
__device__ inline float half_wave_sum(float v) {
  v = dpp_add<0xB1>(v);   // quad_perm [1,0,3,2]
  v = dpp_add<0x4E>(v);   // quad_perm [2,3,0,1]
  v = dpp_add<0x141>(v);  // row_half_mirror
  v = dpp_add<0x140>(v);  // row_mirror
  const auto p = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false,
                                                  false);
  return __int_as_float(p[0]) + __int_as_float(p[1]);
}

template <int CTRL>
__device__ inline float dpp_max(float v) {
  return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf,
                                                             true)));
}
__device__ inline float half_wave_max(float v) {
  v = dpp_max<0xB1>(v);
  v = dpp_max<0x4E>(v);
  v = dpp_max<0x141>(v);
  v = dpp_max<0x140>(v);
  const auto p = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false,
                                                  false);
  return fmaxf(__int_as_float(p[0]), __int_as_float(p[1]));
}

// ------------------------------------------------------------------------------ operand images
// dst[row][dp] = src[row][0..dim), zero beyond dim and in rows that are left out (no class as
// target, an upstream gradient of zero, or bias == -inf): an infinity or NaN there must not meet a
// coefficient of zero in the gradients' products, nor a large number set the others' scale.
// Split images of x: dst at a scale per row, and dst2 at the scale of the largest.
template <typename T>
struct PackArgs {
  const T* src;  // null: nothing to do
  int64_t ld, rows;
  int dim, dp;
  const int64_t* target;
  int64_t ignore, classes;
  const float* grad;  // upstream gradient per row, or null
  const float* bias;
  void *dst, *dst2;
  int* rowexp;  // exponents of dst's rows, or null: one scale for all
  int lanes;  // log2 of the lanes of a row
  bool vec;   // rows of src are 16-byte aligned
};

// Eight numbers of a row from column c on, zero beyond its end
template <typename T>
__device__ inline void load8(const PackArgs<T>& a, int64_t row, int c, T (&v)[8]) {
  const T* p = a.src + row * a.ld + c;
  if (a.vec && c + 8 <= a.dim) {
#pragma unroll
    for (int q = 0; q < 8; q += Vec16<T>::n) {
      const Vec16<T> o = *reinterpret_cast<const Vec16<T>*>(p + q);
#pragma unroll
      for (int j = 0; j < Vec16<T>::n; ++j) v[q + j] = o.v[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < a.dim ? p[j] : T(0.f);
  }
}

template <typename T>
__device__ inline bool left_out_row(const PackArgs<T>& a, int64_t row) {
  if (!a.target) return a.bias && a.bias[row] == -INFINITY;
  const int64_t t = a.target[row];
  return t == a.ignore || t < 0 || t >= a.classes || (a.grad && a.grad[row] == 0.f);
}

// Split images: the largest finite magnitude of each operand, by workgroup, and the exponent e
// that takes a largest magnitude into [2^14, 2^15)
constexpr int kMaxBlocks = 512;  // workgroups (and partial maxima) of an operand

__device__ inline int scale_exponent(float top) {
  if (!(top > 0.f && top < INFINITY)) return 0;
  int e;
  frexpf(top, &e);  // top = f 2^e, f in [0.5, 1)
  return min(max(15 - e, -126), 126);
}

template <typename T>
__device__ inline float finite_max(float m, const T (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float x = fabsf(static_cast<float>(v[j]));
    m = x > m && x < INFINITY ? x : m;
  }
  return m;
}

template <typename T>
__device__ inline float largest(const PackArgs<T>& a, int block, int blocks) {
  const int64_t t = int64_t(block) * blockDim.x + threadIdx.x;
  const int lane = int(t & ((1 << a.lanes) - 1));
  float m = 0.f;
  for (int64_t row = t >> a.lanes; row < a.rows; row += int64_t(blocks) * blockDim.x >> a.lanes) {
    if (left_out_row(a, row)) continue;
    for (int c = lane * 8; c < a.dim; c += 8 << a.lanes) {
      T v[8];
      load8(a, row, c, v);
      m = finite_max(m, v);
    }
  }
  return m;
}

// the maximum of 1024 threads' values, in all of them
__device__ inline float block_max(float v, float* red) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v = fmaxf(v, __shfl_xor(v, m, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
  for (int i = 1; i < int(blockDim.x >> 6); ++i) v = fmaxf(v, red[i]);
  return v;
}

// part[0 .. kMaxBlocks): x where one scale for all rows is wanted, part[kMaxBlocks ..): w
template <typename T>
__global__ __launch_bounds__(1024) void oap_ce_largest(PackArgs<T> x, PackArgs<T> w,
                                                       float* __restrict__ part) {
  __shared__ float red[16];
  if (x.src && x.dst2) {
    const float m = block_max(largest(x, blockIdx.x, kMaxBlocks), red);
    if (threadIdx.x == 0) part[blockIdx.x] = m;
  }
  if (w.src) {
    const float m = block_max(largest(w, blockIdx.x, kMaxBlocks), red);
    if (threadIdx.x == 0) part[kMaxBlocks + blockIdx.x] = m;
  }
}

// Eight numbers from column c on, split: runs of 32 numbers, their h, then their l
template <typename T>
__device__ inline void store_split(void* dst, int64_t row, int dp, int c, const T (&v)[8],
                                   float scale, bool out) {
  Vec16<_Float16> h, l;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float x = out ? 0.f : static_cast<float>(v[j]) * scale;
    h.v[j] = static_cast<_Float16>(x);
    l.v[j] = static_cast<_Float16>(x - static_cast<float>(h.v[j]));
  }
  _Float16* d = static_cast<_Float16*>(dst) + 2 * (row * dp + (c & ~31)) + (c & 31);
  *reinterpret_cast<Vec16<_Float16>*>(d) = h;
  *reinterpret_cast<Vec16<_Float16>*>(d + 32) = l;
}

// the share of thread t of `threads`
template <typename T, typename I>
__device__ inline void pack_rows(const PackArgs<T>& a, float scale, int64_t t, int64_t threads) {
  const int lane = int(t & ((1 << a.lanes) - 1));
  for (int64_t row = t >> a.lanes; row < a.rows; row += threads >> a.lanes) {
    const bool out = left_out_row(a, row);
    float first = scale;  // of dst
    if (gt_is_split<I> && a.rowexp) {
      float m = 0.f;
      for (int c = lane * 8; c < a.dim; c += 8 << a.lanes) {
        T v[8];
        load8(a, row, c, v);
        m = finite_max(m, v);
      }
      for (int k = 1 << a.lanes >> 1; k >= 1; k >>= 1) m = fmaxf(m, __shfl_xor(m, k, 64));
      const int e = scale_exponent(m);
      if (lane == 0) a.rowexp[row] = e;
      first = ldexpf(1.f, e);
    }
    for (int c = lane * 8; c < a.dp; c += 8 << a.lanes) {
      T v[8];
      load8(a, row, c, v);
      if constexpr (gt_is_split<I>) {
        store_split(a.dst, row, a.dp, c, v, first, out);
        if (a.dst2) store_split(a.dst2, row, a.dp, c, v, scale, out);
      } else {
#pragma unroll
        for (int q = 0; q < 8; q += Vec16<T>::n) {
          Vec16<T> o;
#pragma unroll
          for (int j = 0; j < Vec16<T>::n; ++j) o.v[j] = out ? T(0.f) : v[q + j];
          if (c + q < a.dp)  // (an fp32 row may end inside the eight)
            *reinterpret_cast<Vec16<T>*>(static_cast<T*>(a.dst) + row * a.dp + c + q) = o;
        }
      }
    }
  }
}

// ------------------------------------------------------------------------------------ logits
struct LogitArgs {
  GtOperand w, x;      // rows: the piece's classes, all rows
  int64_t dp;          // k extent
  const float* bias;   // of the piece, or null
  const int* scale;    // split images: exponent of the piece's classes
  const int* rowexp;   // and of every row
  const int64_t* target;
  int64_t class0;      // first class of the piece
  int64_t n;
  int vtiles, ntiles;
  // statistics
  float2* part;        // [class tile][npad]: max, sum of exp(z - max)
  int64_t npad;
  float* zt;           // [n] target's logit
  // gradient
  const float2* stat;  // [n] the row's (max, sum)
  const float* coef;   // [n] upstream gradient over its largest magnitude, 0: no loss
  float pscale, unscale;  // of the dz image (powers of two)
  void* dz;            // [npad][vp]
  int64_t vp;
  float* dbpart;       // [row tile][vp] sums of dz over the tile's rows, or null
  float* dzmax;        // [row tile][vp] largest |dz| of the tile's rows, or null (split operands)
};

// Tile of a workgroup: workgroups go to the 8 XCDs in turn, so each XCD takes a run of
// consecutive tiles and its L2 sees the same class rows again for every row tile.
__device__ inline int xcd_tile(int b, int total) {
  const int per = total >> 3, rest = total & 7;
  const int x = b & 7, i = b >> 3;
  return x * per + (x < rest ? x : rest) + i;
}

// Tiles in runs of 8 class tiles by all row tiles, the class tile fastest: the 32 workgroups that
// an XCD runs at a time then share 8 + 4 operand panels in its L2.
__device__ inline void tile_at(int t, int mtiles, int ntiles, int& mt, int& nt) {
  const int run = t / (8 * ntiles), first = run * 8;
  const int wide = mtiles - first < 8 ? mtiles - first : 8;
  const int r = t - first * ntiles;
  mt = first + r % wide;
  nt = r / wide;
}

template <typename T>
struct Store {
  typedef T type;
};
template <>
struct Store<GtSplit> {
  typedef float type;
};

// One tile of logits, classes down (in registers) and rows across (lanes): a row's reduction
// over the tile's classes is mostly within the lane.  8192 x 131072 x 2048 bf16: 4.0 ms forward
// (1.10 PF/s), 2.26 ms for each half of the classes with their dz (0.98 PF/s, 1 GiB written).
template <typename T, int BM, int BN, int WAVES_M, bool SINGLE, bool GRAD>
__global__ __launch_bounds__(kGtThreads, gt_occupancy(BM, BN)) void oap_ce_logits(LogitArgs a) {
#pragma clang fp contract(off)
  typedef GtTile<T, BM, kAlongK, BN, kAlongK, WAVES_M, SINGLE> Tile;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ float sbias[BM];
  __shared__ float2 smerge[WAVES_M][BN];
  __shared__ int left_out;
  const int tid = threadIdx.x, lane = tid & 63;
  int vt, nt;
  tile_at(xcd_tile(blockIdx.x, a.vtiles * a.ntiles), a.vtiles, a.ntiles, vt, nt);
  const int v0 = vt * BM, n0 = nt * BN;
  if (tid == 0) left_out = 0;
  __syncthreads();
  for (int i = tid; i < BM; i += kGtThreads) {
    float b = v0 + i >= a.w.rows ? -INFINITY : a.bias ? a.bias[v0 + i] : 0.f;
    // (finite biases stay finite: the type's lowest value is no exclusion)
    if (b > -INFINITY) b = fmaxf(b * kLog2e, -FLT_MAX);
    sbias[i] = b;
    if (b == -INFINITY) left_out = 1;
  }
  __syncthreads();
  const int i0 = Tile::row0(), j0 = Tile::col0();
  int ex[Tile::NI] = {};  // (loaded ahead of the products, which hide the wait)
  if constexpr (gt_is_split<T>) {
#pragma unroll
    for (int ni = 0; ni < Tile::NI; ++ni) {
      const int64_t n = n0 + j0 + 32 * ni;
      ex[ni] = a.rowexp[n < a.n ? n : a.n - 1];
    }
  }
  gt_f32x16 acc[Tile::MI][Tile::NI];
  Tile::clear(acc);
  Tile::run(a.w, a.x, v0, n0, 0, a.dp, lds, acc);
  // what takes a row's sums of products to logits in units of ln 2 (finite: a sum of 0 stays 0)
  float per[Tile::NI];
#pragma unroll
  for (int ni = 0; ni < Tile::NI; ++ni) {
    per[ni] = kLog2e;
    if constexpr (gt_is_split<T>)
      per[ni] = fminf(ldexpf(kLog2e, -(*a.scale + ex[ni])), FLT_MAX);
  }
  const bool masked = left_out != 0, plain = !masked && !a.bias;
  if (!plain) {
#pragma unroll
    for (int mi = 0; mi < Tile::MI; ++mi)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float b = sbias[i0 + Tile::row_of(mi, e)];
#pragma unroll
        for (int ni = 0; ni < Tile::NI; ++ni)
          acc[mi][ni][e] = __builtin_fmaf(acc[mi][ni][e], per[ni], b);
      }
  }
  if (masked) {  // a class that is left out has no logit, whatever its weights hold
#pragma unroll
    for (int mi = 0; mi < Tile::MI; ++mi)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const bool out = sbias[i0 + Tile::row_of(mi, e)] == -INFINITY;
#pragma unroll
        for (int ni = 0; ni < Tile::NI; ++ni) acc[mi][ni][e] = out ? -INFINITY : acc[mi][ni][e];
      }
  }
  // acc: the logits in units of ln 2, or (plain) the sums, which a factor takes there.  The product
  // is rounded before a maximum is taken off: in one multiply-add, logits of 1e4 to 1e9 would lie
  // 2^-11 to 2^6 off their own maximum, larger ones beyond the range of a power.
#pragma unroll
  for (int ni = 0; ni < Tile::NI; ++ni) {
    const int j = j0 + 32 * ni;
    const int64_t n = n0 + j;
    const float unit = plain ? per[ni] : 1.f;
    const int64_t tg = n < a.n ? a.target[n] - a.class0 - v0 - i0 : -1;
    // the target's offset where it may be one of this lane's classes, else -1 (i0 holds the half
    // wave's four, so the last of a lane's offsets is also the last within the tile)
    const int tgt = tg >= 0 && tg <= Tile::row_of(Tile::MI - 1, 15) ? int(tg) : -1;
    if constexpr (!GRAD) {
      float m = -INFINITY;
#pragma unroll
      for (int mi = 0; mi < Tile::MI; ++mi)
#pragma unroll
        for (int e = 0; e < 16; ++e) m = fmaxf(m, acc[mi][ni][e]);
      m *= unit;
      float sum = 0.f;
      const float ref = m > -INFINITY ? m : 0.f;
#pragma unroll
      for (int mi = 0; mi < Tile::MI; ++mi)
#pragma unroll
        for (int e = 0; e < 16; ++e) sum += pow2(acc[mi][ni][e] * unit - ref);
      if (__ballot(tgt >= 0)) {
        float zt = 0.f;
        bool mine = false;
#pragma unroll
        for (int mi = 0; mi < Tile::MI; ++mi)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const bool hit = tgt == Tile::row_of(mi, e);
            zt = hit ? acc[mi][ni][e] : zt;
            mine |= hit;
          }
        if (mine) a.zt[n] = zt * unit;
      }
      const float mo = __shfl_xor(m, 32, 64), so = __shfl_xor(sum, 32, 64);
      const float mm = fmaxf(m, mo), mr = mm > -INFINITY ? mm : 0.f;
      // (a part that is -inf throughout has the sum 0; NaN stays in the sums)
      const float st = sum * pow2(m - mr) + so * pow2(mo - mr);
      if (lane < 32) smerge[Tile::wave_m()][j] = make_float2(mm, st);
    } else {
      const float2 st = n < a.n ? a.stat[n] : make_float2(0.f, 0.f);
      const float c = n < a.n ? a.coef[n] * a.pscale : 0.f;  // (the image's scale in it)
      const float cs = c == 0.f || st.y == 0.f ? 0.f : c / st.y;
      // (a row without a loss has no gradient, whatever its logits are)
      const float ref = c == 0.f ? INFINITY : st.x > -INFINITY ? st.x : 0.f;
#pragma unroll
      for (int mi = 0; mi < Tile::MI; ++mi)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          acc[mi][ni][e] = pow2(acc[mi][ni][e] * unit - ref) * cs;
      if (__ballot(tgt >= 0)) {
        const int hit = tgt >= 0 && sbias[i0 + tgt] == -INFINITY ? -1 : tgt;
#pragma unroll
        for (int mi = 0; mi < Tile::MI; ++mi)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            acc[mi][ni][e] -= hit == Tile::row_of(mi, e) ? c : 0.f;
      }
    }
  }
  if constexpr (!GRAD) {
    __syncthreads();
    for (int j = tid; j < BN; j += kGtThreads) {
      float m = -INFINITY;
#pragma unroll
      for (int k = 0; k < WAVES_M; ++k) m = fmaxf(m, smerge[k][j].x);
      const float ref = m > -INFINITY ? m : 0.f;
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < WAVES_M; ++k) s += smerge[k][j].y * pow2(smerge[k][j].x - ref);
      a.part[int64_t(vt) * a.npad + n0 + j] = make_float2(m, s);
    }
  } else {
    if (a.dbpart) {
      float* sdb = reinterpret_cast<float*>(lds);  // [wave column][BM]
#pragma unroll
      for (int mi = 0; mi < Tile::MI; ++mi)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float v = 0.f;
#pragma unroll
          for (int ni = 0; ni < Tile::NI; ++ni) v += acc[mi][ni][e];
          v = half_wave_sum(v);
          if ((lane & 31) == 0) sdb[Tile::wave_n() * BM + i0 + Tile::row_of(mi, e)] = v;
        }
      __syncthreads();
      for (int i = tid; i < BM; i += kGtThreads) {
        float v = 0.f;
        for (int k = 0; k < Tile::WAVES_N; ++k) v += sdb[k * BM + i];
        a.dbpart[int64_t(nt) * a.vp + v0 + i] = v * a.unscale;
      }
    }
    if constexpr (gt_is_split<T>) {
      if (a.dzmax) {
        float* smx = reinterpret_cast<float*>(lds);  // [wave column][BM]
        if (a.dbpart) __syncthreads();
#pragma unroll
        for (int mi = 0; mi < Tile::MI; ++mi)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float v = 0.f;
#pragma unroll
            for (int ni = 0; ni < Tile::NI; ++ni) v = fmaxf(v, fabsf(acc[mi][ni][e]));
            v = half_wave_max(v);
            if ((lane & 31) == 0) smx[Tile::wave_n() * BM + i0 + Tile::row_of(mi, e)] = v;
          }
        __syncthreads();
        for (int i = tid; i < BM; i += kGtThreads) {
          float v = 0.f;
          for (int k = 0; k < Tile::WAVES_N; ++k) v = fmaxf(v, smx[k * BM + i]);
          a.dzmax[int64_t(nt) * a.vp + v0 + i] = v;
        }
      }
    }
    // dz through LDS, [row][BM classes], the 16-byte chunk c of row j at slot c ^ (j & SW), then
    // out in whole rows; in parts of 32 rows of every wave where the tile is larger than LDS
    constexpr int CPR = BM * int(sizeof(T)) / 16, ROW = BM * int(sizeof(T));
    constexpr int SW = CPR < 16 ? CPR - 1 : 15;
    constexpr bool kWhole = BN * ROW <= Tile::kLds;
    constexpr int PARTS = kWhole ? 1 : Tile::NI, NP = Tile::NI / PARTS;  // blocks of a part
    constexpr int PW = Tile::WN / PARTS, PR = BN / PARTS;                // rows of it
    static_assert(PR * ROW <= Tile::kLds, "a part of the dz tile fits the staging buffer");
    typedef typename Store<T>::type H;  // what is stored: T, or fp32 for split operands
    struct alignas(4 * sizeof(H)) Four {
      H v[4];
    };
    auto at = [&](int j, int byte) {
      return reinterpret_cast<Four*>(lds + j * ROW + (((byte >> 4) ^ (j & SW)) << 4) + (byte & 15));
    };
    // (a thread's chunk k of rows j1, j1 + RS, ... of a part)
    constexpr int RS = kGtThreads / CPR;
    const int k = tid % CPR, j1 = tid / CPR;
    const int64_t pitch = a.vp * int64_t(sizeof(T));
    char* out = static_cast<char*>(a.dz) + int64_t(n0) * pitch + v0 * int64_t(sizeof(T)) + k * 16;
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
      __syncthreads();
#pragma unroll
      for (int np = 0; np < NP; ++np)
#pragma unroll
        for (int mi = 0; mi < Tile::MI; ++mi)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int ni = part * NP + np;
            const int j = Tile::wave_n() * PW + 32 * np + (lane & 31);
            const int i = i0 + Tile::row_of(mi, 4 * g);
            Four f;
#pragma unroll
            for (int e = 0; e < 4; ++e) f.v[e] = static_cast<H>(acc[mi][ni][4 * g + e]);
            *at(j, i * int(sizeof(T))) = f;
          }
      __syncthreads();
#pragma unroll
      for (int it = 0; it < PR / RS; ++it) {
        const int j = j1 + it * RS;
        const int row = j / PW * Tile::WN + part * PW + j % PW;  // of the tile
        *reinterpret_cast<float4*>(out + row * pitch) =
            *reinterpret_cast<const float4*>(lds + j * ROW + ((k ^ (j & SW)) << 4));
      }
    }
  }
}

// A few rows (up to eight): the class rows are read once from memory and that is what bounds it,
// so they go straight into registers.  G lanes share a class, ITERS 16-byte chunks each; the rows
// of x stay in registers.  The sums over the lanes are formed so that a lane ends with the logit of
// one row (as many rows at once as there are), and keeps that row's (max, sum) over the group's
// classes; the workgroup joins them.
// 2M x 100 fp32: one row 130 us (6.1 TB/s), four 140, eight 166 (tiles: 237 and 260); 8-byte loads
// 202, single elements (101 features) 206 us.  One row in bf16, 8-byte loads: 118 us, 3.4 TB/s:
// half the bytes in as many loads, with twice the conversions in each.
struct FewArgs {
  const void *w, *x;
  int64_t ldw, ldx, classes;
  int n, dim;
  int width;  // bytes of a load that the class rows' alignment allows: 16, 8, or 0 for an element
  const float* bias;
  const int64_t* target;
  float2* part;  // [workgroup][n]
  float* zt;
};

constexpr int kFewBlocks = 1024;  // 4 per CU: their loads in flight are enough
constexpr int kFewRows = 8;
// chunks of a lane: the rows of x take 64 registers, or 128 (eight rows)
constexpr int few_iters(int rows, int element) { return rows > 1 && element == 2 ? 2 : 4; }

// One step of a sum over lanes, B the bit in which the lane's partner differs.  The partners of 8
// and 4 differ in the lower bits too, so the steps go from the highest bit down.
template <int B>
__device__ inline float lane_partner(float v) {
  constexpr int CTRL = B == 8 ? 0x140 : B == 4 ? 0x141 : B == 2 ? 0x4E : 0xB1;
  return __int_as_float(
      __builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
// sum of a in the lanes without bit B, of b in those with it
template <int B>
__device__ inline float lane_halves(float a, float b, int lane) {
  const unsigned ua = unsigned(__float_as_int(a)), ub = unsigned(__float_as_int(b));
  if constexpr (B == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(ua, ub, false, false);
    return __int_as_float(int(r[0])) + __int_as_float(int(r[1]));
  } else if constexpr (B == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(ua, ub, false, false);
    return __int_as_float(int(r[0])) + __int_as_float(int(r[1]));
  } else {
    const bool second = lane & B;
    return (second ? b : a) + lane_partner<B>(second ? a : b);
  }
}
// z[0 .. N) summed over groups of 2 B lanes; the group's lanes end with N / (2 B)-ths of the rows
template <int B, int N>
__device__ inline float lane_sums(float (&z)[N], int lane) {
  if constexpr (B == 0) {
    return z[0];
  } else if constexpr (N == 1) {
    float w[1] = {lane_halves<B>(z[0], z[0], lane)};
    return lane_sums<B / 2>(w, lane);
  } else {
    float w[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) w[i] = lane_halves<B>(z[i], z[i + N / 2], lane);
    return lane_sums<B / 2>(w, lane);
  }
}

// WIDE: the class rows are whole 16-byte chunks
template <typename T, int N, int G, bool WIDE>
__global__ __launch_bounds__(256) void oap_ce_few(FewArgs a) {
  constexpr int CH = gt_chunk<T>(), GROUPS = 256 / G, ITERS = few_iters(N, sizeof(T));
  constexpr int PER = G / N;  // lanes of a group that end with the same row
  static_assert(PER >= 1, "a lane for every row");
  struct alignas(8) Half {
    T v[CH / 2];
  };
  __shared__ float2 red[N][GROUPS];
  const int q = threadIdx.x & (G - 1), g = threadIdx.x / G, mine = q / PER;
  float x[N][ITERS][CH];
#pragma unroll
  for (int r = 0; r < N; ++r)
#pragma unroll
    for (int i = 0; i < ITERS; ++i)
#pragma unroll
      for (int j = 0; j < CH; ++j) {
        const int k = (q + i * G) * CH + j;
        x[r][i][j] = r < a.n && k < a.dim
                         ? static_cast<float>(static_cast<const T*>(a.x)[r * a.ldx + k])
                         : 0.f;
      }
  const int64_t tgt = mine < a.n && q % PER == 0 ? a.target[mine] : -1;
  float m = -INFINITY, s = 0.f;
  const T* w = static_cast<const T*>(a.w);
  for (int64_t c = int64_t(blockIdx.x) * GROUPS + g; c < a.classes;
       c += int64_t(gridDim.x) * GROUPS) {
    Vec16<T> v[ITERS];
#pragma unroll
    for (int i = 0; i < ITERS; ++i) {
      v[i] = {};
      const int k = (q + i * G) * CH;
      const T* p = w + c * a.ldw + k;
      if (WIDE) {
        if (k < a.dim) v[i] = *reinterpret_cast<const Vec16<T>*>(p);
      } else if (a.width == 8) {
#pragma unroll
        for (int h = 0; h < CH; h += CH / 2)
          if (k + h < a.dim) {
            const Half o = *reinterpret_cast<const Half*>(p + h);
#pragma unroll
            for (int j = 0; j < CH / 2; ++j) v[i].v[h + j] = o.v[j];
          }
      } else {
#pragma unroll
        for (int j = 0; j < CH; ++j)
          if (k + j < a.dim) v[i].v[j] = p[j];
      }
    }
    float b = a.bias ? a.bias[c] : 0.f;
    const bool out = b == -INFINITY;
    if (!out) b = fmaxf(b * kLog2e, -FLT_MAX);
    float sums[N];
#pragma unroll
    for (int r = 0; r < N; ++r) {
      sums[r] = 0.f;
#pragma unroll
      for (int i = 0; i < ITERS; ++i)
#pragma unroll
        for (int j = 0; j < CH; ++j)
          sums[r] = __builtin_fmaf(x[r][i][j], static_cast<float>(v[i].v[j]), sums[r]);
    }
    float z = lane_sums<G / 2>(sums, q);
    z = out ? -INFINITY : __builtin_fmaf(z, kLog2e, b);
    if (c == tgt) a.zt[mine] = z;
    // (NaN stays in the sum)
    const float mm = fmaxf(m, z), ref = mm > -INFINITY ? mm : 0.f;
    s = s * pow2(m - ref) + pow2(z - ref);
    m = mm;
  }
  if (q % PER == 0) red[mine][g] = make_float2(m, s);
  __syncthreads();
  if (threadIdx.x < unsigned(a.n)) {
    const int r = threadIdx.x;
    float mm = -INFINITY, ss = 0.f;
    for (int k = 0; k < GROUPS; ++k) {
      const float2 p = red[r][k];
      const float t = fmaxf(mm, p.x), ref = t > -INFINITY ? t : 0.f;
      ss = ss * pow2(mm - ref) + p.y * pow2(p.x - ref);
      mm = t;
    }
    a.part[int64_t(blockIdx.x) * a.n + r] = make_float2(mm, ss);
  }
}

// Rows: (max, sum) of every class tile into the row's and the loss, log(sum) + (max - z_t): the
// difference is formed first, so logits of any size keep the loss's own precision.  A workgroup
// takes `cols` rows (a power of two) and shares the class tiles of each among its other threads.
// A single workgroup goes over all rows and forms the total as well.
struct RowArgs {
  const float2* part;
  int tiles;
  int64_t npad, n;
  int cols;
  const int64_t* target;
  int64_t ignore, classes;
  const float* zt;
  float* loss;
  float2* stat;
  float* miss;   // 1 - probability of the target, or null
  float* total;  // null: none, or in a launch of its own
  int mean;
};

// (sum, count) of the workgroup's threads in a fixed order, in fp64; into *total
__device__ inline void total_of(double s, unsigned long long k, int mean, float* total) {
  __shared__ double red[1024];
  __shared__ unsigned long long cnt[1024];
  red[threadIdx.x] = s;
  cnt[threadIdx.x] = k;
  for (int h = 512; h >= 1; h >>= 1) {
    __syncthreads();
    if (threadIdx.x < unsigned(h)) {
      red[threadIdx.x] += red[threadIdx.x + h];
      cnt[threadIdx.x] += cnt[threadIdx.x + h];
    }
  }
  if (threadIdx.x == 0) *total = float(mean ? red[0] / double(cnt[0] ? cnt[0] : 1) : red[0]);
}

__global__ __launch_bounds__(1024) void oap_ce_rows(RowArgs a) {
  __shared__ float2 red[1024];
  const int cols = a.cols, c = threadIdx.x & (cols - 1), r0 = threadIdx.x / cols;
  const int nr = 1024 / cols;
  double sum = 0.0;
  unsigned long long count = 0;
  for (int64_t first = int64_t(blockIdx.x) * cols; first < a.n;
       first += int64_t(gridDim.x) * cols) {
    const int64_t row = first + c;
    float m = -INFINITY, s = 0.f;
    if (row < a.n) {
      for (int t = r0; t < a.tiles; t += nr) {
        const float2 p = a.part[int64_t(t) * a.npad + row];
        const float mm = fmaxf(m, p.x), ref = mm > -INFINITY ? mm : 0.f;
        s = s * pow2(m - ref) + p.y * pow2(p.x - ref);
        m = mm;
      }
    }
    __syncthreads();
    red[threadIdx.x] = make_float2(m, s);
    for (int h = nr / 2; h >= 1; h >>= 1) {
      __syncthreads();
      if (r0 < h) {
        const float2 p = red[threadIdx.x + h * cols];
        const float mm = fmaxf(m, p.x), ref = mm > -INFINITY ? mm : 0.f;
        s = s * pow2(m - ref) + p.y * pow2(p.x - ref);
        m = mm;
        red[threadIdx.x] = make_float2(m, s);
      }
    }
    if (r0 == 0 && row < a.n) {
      a.stat[row] = make_float2(m, s);
      const int64_t t = a.target[row];
      float l;
      if (t == a.ignore)
        l = 0.f;
      else if (t < 0 || t >= a.classes)
        l = NAN;
      else if (a.zt[row] == -INFINITY)
        l = INFINITY;
      else {
        l = log2f(s) + (m - a.zt[row]);
        l = l < 0.f ? 0.f : l * kLn2;  // (below 0 by roundings only)
      }
      a.loss[row] = l;
      if (a.miss) a.miss[row] = -expm1f(-l);
      if (t != a.ignore) {
        sum += double(l);
        ++count;
      }
    }
  }
  if (gridDim.x == 1 && a.total) total_of(sum, count, a.mean, a.total);
}

// Sum (or mean over the rows that have a loss)
__global__ __launch_bounds__(1024) void oap_ce_total(RowArgs a) {
  double s = 0.0;
  unsigned long long k = 0;
  for (int64_t i = threadIdx.x; i < a.n; i += 1024)
    if (a.target[i] != a.ignore) {
      s += double(a.loss[i]);
      ++k;
    }
  total_of(s, k, a.mean, a.total);
}

// Upstream gradient of every row as g_n = gscale * coef_n with |coef_n| <= 1: products of the
// coefficient with a probability then fit 16 bits.  Rows without a loss (or with a target that
// is no class) get the coefficient 0.  gscale is the largest magnitude that is a number, and a
// row's gradient that is none is its coefficient: it reaches that row's dx, and no other's.
struct CoefArgs {
  const float* grad;  // null: nothing to do
  int per_row, mean;
  const int64_t* target;
  int64_t ignore, classes, n;
  float* coef;
  float* gscale;
  // split operands, for dx: the power of two of each row's dz, or null
  float* rowscale;
  const float* miss;
};

// |dz| of a row is at most |c| (1 - p of the target): the target's own, and the sum of all others'.
// It goes to [2^12, 2^13), which leaves room for the roundings of the loss, from which 1 - p comes
// (2^-23 and what its sums lose beside a one), and of the logits, which differ between the passes
// by what the scales of their pieces round (2^-40 of the largest weight).
__device__ inline float row_scale(float c, float miss) {
  float top = miss + 0x1p-20f;
  top = fabsf(c) * (top < 1.f ? top : 1.f);
  return ldexpf(1.f, scale_exponent(top) - 2);
}

__device__ inline void coefficients(const CoefArgs& a) {
  __shared__ float red[1024];
  __shared__ unsigned long long cnt[1024];
  float m = 0.f;
  unsigned long long k = 0;
  for (int64_t i = threadIdx.x; i < a.n; i += 1024) {
    const int64_t t = a.target[i];
    k += t != a.ignore;
    if (t >= 0 && t < a.classes && t != a.ignore) {
      const float g = a.per_row ? fabsf(a.grad[i]) : 1.f;
      m = g > m && g < INFINITY ? g : m;
    }
  }
  red[threadIdx.x] = m;
  cnt[threadIdx.x] = k;
  for (int h = 512; h >= 1; h >>= 1) {
    __syncthreads();
    if (threadIdx.x < unsigned(h)) {
      red[threadIdx.x] = fmaxf(red[threadIdx.x], red[threadIdx.x + h]);
      cnt[threadIdx.x] += cnt[threadIdx.x + h];
    }
  }
  __syncthreads();
  const float top = red[0];
  if (threadIdx.x == 0)  // (0 if no row has a loss)
    *a.gscale = a.per_row || top == 0.f
                    ? top
                    : a.mean ? a.grad[0] / float(cnt[0] ? cnt[0] : 1) : a.grad[0];
  for (int64_t i = threadIdx.x; i < a.n; i += 1024) {
    const int64_t t = a.target[i];
    const bool has = t >= 0 && t < a.classes && t != a.ignore;
    float c = has ? 1.f : 0.f;
    if (has && a.per_row) {
      const float g = a.grad[i];
      c = !(fabsf(g) < INFINITY) ? g : top == 0.f ? 0.f : g / top;
    }
    a.coef[i] = c;
    if (a.rowscale) a.rowscale[i] = row_scale(c, a.miss[i]);
  }
}

// What a launch of logits reads: the rows' coefficients (workgroup 0), the image of x and that
// of the piece's classes (shares of the other workgroups), in one launch.  Split images: part
// holds the partial maxima, and the exponents go to scale[0] (x, dst2) and scale[1] (classes).
template <typename T, typename I>
__global__ __launch_bounds__(1024) void oap_ce_prepare(CoefArgs coef, PackArgs<T> x,
                                                       PackArgs<T> w, const float* part,
                                                       int* scale) {
  if (coef.grad && blockIdx.x == 0) {
    coefficients(coef);
    return;
  }
  const int skip = coef.grad ? 1 : 0;
  const int64_t first = int64_t(blockIdx.x - skip) * 1024 + threadIdx.x;
  const int64_t stride = int64_t(gridDim.x - skip) * 1024;
  float sx = 1.f, sw = 1.f;
  if constexpr (gt_is_split<I>) {
    __shared__ float red[16];
    const int t = threadIdx.x;
    if (x.src && x.dst2) {
      const int e = scale_exponent(block_max(t < kMaxBlocks ? part[t] : 0.f, red));
      if (first == 0) scale[0] = e;
      sx = ldexpf(1.f, e);
    }
    const int e = scale_exponent(block_max(t < kMaxBlocks ? part[kMaxBlocks + t] : 0.f, red));
    if (first == 0) scale[1] = e;
    sw = ldexpf(1.f, e);
  }
  if (x.src) pack_rows<T, I>(x, sx, first, stride);
  if (w.src) pack_rows<T, I>(w, sw, first, stride);
}

// ------------------------------------------------------------------------------------- products
struct ProdArgs {
  GtOperand a, b;
  int64_t k;           // extent
  int64_t m, n;        // valid rows / columns of the result
  int mtiles, ntiles, splits;
  void* out;           // dW: [m][n] elements; dx: fp32 slabs [split][m][n]
  int add;             // dx: add to the slab
  const float* gscale; // dW
  const int* scale;    // split operands: the exponent of b, or null
  float unscale;
  const float* bias;   // dW: rows of classes that are left out are zero
};

// the exponent of a power of two
__device__ inline int exponent_of(float p) { return (__float_as_int(p) >> 23) - 127; }

// dx: a slab per split of k (classes of the piece); the same workgroup adds the next piece's
// part to the same elements, so the order of the sums is fixed.  65536 classes of 8192 x 2048
// bf16: 2.12 ms (1.04 PF/s); dW of them 2.13 ms (1.03 PF/s).
template <typename T, int BM, int BN, int WAVES_M>
__device__ void dx_tile(const ProdArgs& a, int block, char* lds) {
  typedef GtTile<T, BM, kAlongK, BN, kAcrossK, WAVES_M, false, gt_is_split<T>> Tile;
  const int t = xcd_tile(block, a.mtiles * a.ntiles * a.splits);
  const int sp = t / (a.mtiles * a.ntiles), u = t - sp * a.mtiles * a.ntiles;
  int mt, nt;
  tile_at(u, a.mtiles, a.ntiles, mt, nt);
  const int64_t blocks = (a.k + Tile::BK - 1) / Tile::BK;
  const int64_t k0 = blocks * sp / a.splits * Tile::BK;
  const int64_t k1 = sp + 1 == a.splits ? a.k : blocks * (sp + 1) / a.splits * Tile::BK;
  gt_f32x16 acc[Tile::MI][Tile::NI];
  Tile::clear(acc);
  Tile::run(a.a, a.b, mt * BM, nt * BN, k0, k1, lds, acc);
  const int64_t i0 = int64_t(mt) * BM + Tile::row0(), j0 = nt * BN + Tile::col0();
  float* out = static_cast<float*>(a.out) + (int64_t(sp) * a.m + i0) * a.n + j0;
#pragma unroll
  for (int mi = 0; mi < Tile::MI; ++mi)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      // (four rows at a time, from an address that is not kept for the others)
      float* q = out + Tile::row_of(mi, 4 * g) * a.n;
      asm volatile("" : "+v"(q)::"memory");
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t i = i0 + Tile::row_of(mi, 4 * g + e);
        if (i >= a.m) continue;
        int ex = 0;
        if constexpr (gt_is_split<T>) ex = *a.scale + exponent_of(a.a.scale[i]);
#pragma unroll
        for (int ni = 0; ni < Tile::NI; ++ni)
          if (j0 + 32 * ni < a.n) {
            float* o = q + e * a.n + 32 * ni;
            float v = acc[mi][ni][4 * g + e];
            if constexpr (gt_is_split<T>) v = ldexpf(v, -ex);
            *o = a.add ? *o + v : v;
          }
      }
    }
}

template <typename S, typename T, int BM, int BN, int WAVES_M>
__device__ void dw_tile(const ProdArgs& a, int block, char* lds) {
  typedef GtTile<T, BM, kAcrossK, BN, kAcrossK, WAVES_M, false, gt_is_split<T>> Tile;
  int mt, nt;
  tile_at(xcd_tile(block, a.mtiles * a.ntiles), a.mtiles, a.ntiles, mt, nt);
  gt_f32x16 acc[Tile::MI][Tile::NI];
  Tile::clear(acc);
  Tile::run(a.a, a.b, mt * BM, nt * BN, 0, a.k, lds, acc);
  const float g = *a.gscale;
  S* out = static_cast<S*>(a.out);
  const int64_t i0 = int64_t(mt) * BM + Tile::row0(), j0 = nt * BN + Tile::col0();
#pragma unroll
  for (int mi = 0; mi < Tile::MI; ++mi)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int64_t i = i0 + Tile::row_of(mi, e);
      if (i >= a.m) continue;
      const bool out_of = a.bias && a.bias[i] == -INFINITY;
      int ex = 0;
      if constexpr (gt_is_split<T>) ex = *a.scale + exponent_of(a.a.scale[i]);
#pragma unroll
      for (int ni = 0; ni < Tile::NI; ++ni) {
        const int64_t j = j0 + 32 * ni;
        float v = acc[mi][ni][e];
        if constexpr (gt_is_split<T>)
          v = ldexpf(v, -ex);
        else
          v *= a.unscale;
        if (j < a.n) out[i * a.n + j] = static_cast<S>(out_of ? 0.f : v * g);
      }
    }
}

// Both products of a piece in one launch, dx's workgroups (each with more of k) first: the last of
// one fill up with the first of the other (bf16 with gradients, 3000 x 20000 x 784 618 against 628
// us, 300 x 50001 x 1000 235 against 259 us).  The largest tiles have no registers for both and
// take a launch each.
enum GradPart { kBoth, kDx, kDw };
template <typename S, typename T, int B, GradPart PART>
__global__ __launch_bounds__(kGtThreads, gt_occupancy(B, B)) void oap_ce_grads(ProdArgs x,
                                                                            ProdArgs w, int nx) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  if (PART == kDx || (PART == kBoth && int(blockIdx.x) < nx))
    dx_tile<T, B, B, 2>(x, blockIdx.x, lds);
  else
    dw_tile<S, T, B, B, 2>(w, blockIdx.x - nx, lds);
}

// What is left of a piece: db of its classes (the first workgroups), and after the last piece the
// slabs of dx into the result.
template <typename T>
struct FinishArgs {
  const float* gscale;
  const float* coef;
  const float* bias;    // of the piece, or null
  const float* dbpart;  // [row tile][vp], or null
  int rtiles;
  int64_t vp, classes;
  float* db;
  const float* slab;  // [split][count], or null
  int splits;
  int64_t count;
  int dim;
  float unscale;
  T* dx;
};

template <typename T>
__global__ __launch_bounds__(256) void oap_ce_finish(FinishArgs<T> a) {
  const int dbblocks = a.dbpart ? int((a.classes + 255) / 256) : 0;
  const float g = *a.gscale;
  if (int(blockIdx.x) < dbblocks) {
    const int64_t v = int64_t(blockIdx.x) * 256 + threadIdx.x;
    if (v >= a.classes) return;
    float s = 0.f;
    for (int t = 0; t < a.rtiles; ++t) s += a.dbpart[int64_t(t) * a.vp + v];
    // (a class that is left out has no gradient, whatever the rows' upstream gradients are)
    a.db[v] = a.bias && a.bias[v] == -INFINITY ? 0.f : s * g;
    return;
  }
  const float scale = g * a.unscale;
  for (int64_t i = int64_t(blockIdx.x - dbblocks) * 256 + threadIdx.x; i < a.count;
       i += int64_t(gridDim.x - dbblocks) * 256) {
    float v = 0.f;
    for (int s = 0; s < a.splits; ++s) v += a.slab[int64_t(s) * a.count + i];
    v *= scale;
    // an upstream gradient that is no number leaves the rows without a loss at 0
    if (!(fabsf(scale) < INFINITY) && a.coef[i / a.dim] == 0.f) v = 0.f;
    a.dx[i] = static_cast<T>(v);
  }
}

// Split operands: the power of two that takes a class's largest |dz| of the piece to [2^14, 2^15)
// (classes beyond the piece's end, which fill its last tiles: 1)
__global__ __launch_bounds__(256) void oap_ce_class_scales(const float* __restrict__ dzmax,
                                                           int rtiles, int64_t vp, int64_t classes,
                                                           float* __restrict__ scale) {
  const int64_t v = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (v >= vp) return;
  float m = 0.f;
  if (v < classes)
    for (int t = 0; t < rtiles; ++t) m = fmaxf(m, dzmax[int64_t(t) * vp + v]);
  scale[v] = ldexpf(1.f, scale_exponent(m));
}

template <typename S>
__global__ __launch_bounds__(256) void oap_ce_fill0(S* __restrict__ p, int64_t count) {
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < count;
       i += int64_t(gridDim.x) * 256)
    p[i] = S(0.f);
}

// ------------------------------------------------------------------------------------- planning
struct Plan {
  bool split;               // fp32 operands as two fp16 numbers
  int64_t dp;               // features of an image's row, to a whole chunk
  bool x_direct, w_direct;  // the operand is read where it lies
  int64_t rows;             // rows per turn of the forward pass
  int bm, bn;               // class and row tile of the logits
  int64_t npad;
  int64_t piece;            // classes per piece, a multiple of 256
  bool single;              // logits of 128 x 128 with one staging buffer
  int xtile, wtile;         // square tiles of dx and dW
  int splits;
};

bool direct(const CeArgs& a, const void* p, int64_t ld) {
  const int ch = 16 / elem_size(a.elem);
  return a.dim % ch == 0 && ld % ch == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0 &&
         ld < (int64_t(1) << 20);
}

// Of one dz image or one class image.  Smaller pieces stay in the last-level cache, but their
// products fill the chip less evenly and dx's slabs are added to more often: 2^28, 2^29, 2^30, 2^31
// take 18.2, 17.2, 17.0, 17.1 ms at 8192 x 131072 x 2048 bf16 and 12.2, 11.8, 11.0, 11.1 ms at
// 1024 x 2M x 100 fp32.
constexpr int64_t kPieceBytes = int64_t(1) << 30;

// fp32 problems of more than 128 rows and at least this many products take the split operands:
// their images cost two launches and two passes over the weights (1024 x 20000 x 128: 182 against
// 250 us with gradients, 2048 x 20000 x 1000 1.18 against 2.44 ms; 300 x 5000 x 512 146 against
// 134 us, 200 x 20000 x 300 without gradients 49 against 50 us; 192 x 1M x 100 1.89 against 2.15
// ms, but 128 x 1M x 100, one row tile, 1.61 against 1.38 ms, without gradients 422 against 292).
constexpr double kSplitWork = 1.5e9;

// Tiles of 128 x 128, two or more of which share a CU, or of 256 x 256: one's epilogue overlaps
// another's MFMAs, but a byte from LDS feeds half as many.  fp32 MFMAs are slow enough for LDS at
// any size (1024 x 2M x 100 in fp32 MFMAs: 19.9 against 24.4 ms); in 16 bits the small ones are
// faster while the epilogue weighs (forward and gradients, bf16: 3000 x 20000 x 784 0.66 against
// 0.68 ms, 4096 x 65536 x 512 1.44 against 1.52 ms; 8192 x 131072 x 2048 18.9 against 16.6 ms).
// Where tiles of 128 leave CUs empty, tiles of 64 finish sooner.
int tile_of(const CeArgs& a, int64_t rows, int64_t cols) {
  if (ceil_div(rows, 128) * ceil_div(cols, 128) < 192) return 64;
  return a.elem == Elem::F32 || a.dim <= 1024 ? 128 : 256;
}

bool split_fp32(const CeArgs& a) {
  return a.elem == Elem::F32 && a.n > 128 &&
         double(a.n) * double(a.classes) * a.dim >= kSplitWork;
}

Plan make_plan(const CeArgs& a, bool grad) {
  Plan p;
  const int es = elem_size(a.elem);
  p.split = split_fp32(a);
  p.dp = int64_t(round_up(size_t(a.dim), size_t(p.split ? 32 : 16 / es)));
  // (the gradients read images in which the rows that are left out are zero)
  p.x_direct = !p.split && !grad && direct(a, a.x, a.ldx);
  p.w_direct = !p.split && direct(a, a.w, a.ldw) && !(grad && a.bias);
  p.bm = tile_of(a, a.classes, a.n);
  p.bn = a.n <= 64 ? 64 : p.bm;
  // 256 classes a tile where the chip's 512 places for them fill twice: a byte of the operands
  // feeds a third more products (bf16: 3000 x 20000 x 784 with gradients 632 against 661 us, 700 x
  // 50001 x 1000 without 103 against 109 us; fewer tiles leave places empty: 300 x 50001 x 1000
  // 67 against 60 us).
  if (es == 2 && p.bm == 128 && p.bn == 128 &&
      ceil_div(a.classes, 256) * ceil_div(a.n, 128) >= 1024)
    p.bm = 256;
  // One buffer lets a third workgroup share the CU.  16 bits gain at every k that takes this tile
  // (4096 x 200000 x 128 1.82 against 1.99 ms, 4096 x 65536 x 512 1.38 against 1.42 ms), split
  // operands while k is short (1024 x 2M x 100 11.0 against 11.9 ms; nothing is gained at 2048 x
  // 20000 x 1000).  fp32 keeps two: that loop skips the empty steps of a short k.
  p.single = es == 2 || (p.split && p.dp <= 512);
  // few rows of many classes (16 x 2M x 100 fp32 in tiles of 32 rows 260 us, of 64 390 us; one
  // buffer for those of 64, 377 against 394 us, two for those of 32, 188 against 201 us for 8 x
  // 400000 x 1000 bf16)
  if (p.bn == 64 && p.bm > 64) {
    p.bm = 256;
    if (a.n <= 32) p.bn = 32;
  }
  // the forward pass keeps 8 bytes of each row and class tile: as many rows at a time as take
  // 1 GiB, at least 4096
  p.rows = a.n;
  if (!grad) {
    const int64_t fit = (int64_t(1) << 30) / 8 / ceil_div(a.classes, p.bm) / p.bn * p.bn;
    p.rows = std::min<int64_t>(a.n, std::max<int64_t>(fit, 4096));
  }
  p.npad = int64_t(round_up(size_t(p.rows), size_t(p.bn)));
  const int64_t vpad = int64_t(round_up(size_t(a.classes), 256));
  int64_t per = p.dp;  // elements per class of the largest image
  if (grad) per = std::max(per, p.npad);
  p.piece = kPieceBytes / (per * es) / 256 * 256;
  if (!grad && p.w_direct) p.piece = vpad;
  p.piece = std::max<int64_t>(256, std::min({p.piece, vpad, int64_t(1) << 20}));
  p.wtile = tile_of(a, std::min(p.piece, a.classes), a.dim);
  // dx: two workgroups per CU between the tiles and the splits of k, of at least 256 classes (128
  // where even so there are few)
  p.xtile = a.elem == Elem::F32 || a.dim <= 1024 ? 128 : 256;
  int64_t tiles = ceil_div(a.n, p.xtile) * ceil_div(a.dim, p.xtile), by_k = p.piece / 256;
  if (a.n <= 64 || tiles * by_k < 192) {
    p.xtile = 64;
    tiles = ceil_div(a.n, 64) * ceil_div(a.dim, 64);
    by_k = p.piece / 128;
  }
  p.splits = int(std::max<int64_t>(1, std::min<int64_t>(by_k, 512 / tiles)));
  return p;
}

int few_width(const CeArgs& a) {
  const int64_t es = elem_size(a.elem);
  const uintptr_t of = uintptr_t(a.dim * es) | uintptr_t(a.ldw * es) |
                       reinterpret_cast<uintptr_t>(a.w);
  return of % 16 == 0 ? 16 : of % 8 == 0 ? 8 : 0;
}

// Whether oap_ce_few takes the call: the rows and features that its lane groups cover.  In 16 bits
// the conversions weigh, and tiles are faster (4 x 400000 x 1000 bf16 179 against 281 us) unless
// they need an image of classes that are not aligned (4 x 2M x 100 bf16 369 against 124 us).  A
// training call takes tiles, as its gradients do: the sums of the two run in another order, and
// with logits of 1e7 their last bits are whole powers of e.
bool few_rows(const CeArgs& a) {
  const int es = elem_size(a.elem);
  if (a.train || a.n > kFewRows || a.dim > 64 * few_iters(int(a.n), es) * 16 / es) return false;
  return es == 4 || a.n == 1 || (a.n <= 4 && few_width(a) < 16);
}

struct Carver {
  char* base;
  size_t used = 0;
  template <typename T>
  T* take(size_t count) {
    T* p = reinterpret_cast<T*>(base + used);
    used += round_up(count * sizeof(T), 256);
    return p;
  }
};

// More than 64 KiB of LDS is asked for once per kernel and device.
template <typename F>
void set_lds(F kernel, int bytes) {
  static std::mutex mu;
  static std::set<std::pair<const void*, int>> done;
  int device = 0;
  OAP_HIP_CHECK(hipGetDevice(&device));
  std::lock_guard<std::mutex> lock(mu);
  if (!done.emplace(reinterpret_cast<const void*>(kernel), device).second) return;
  OAP_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                    hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
}

unsigned stride_grid(int64_t threads) {
  return unsigned(std::max<int64_t>(1, std::min<int64_t>(ceil_div(threads, 256), 8192)));
}

// S: type of x, w and their gradients; T: of the products' operands
template <typename S, typename T>
struct Ce {
  struct Work {
    T *ximg, *ximg2, *wimg, *dz;
    float2* part;
    float *zt, *coef, *gscale, *slab, *dbpart, *largest, *dzmax, *classscale, *rowscale;
    int *scale, *rowexp;
  };

  static PackArgs<S> pack(const void* src, int64_t ld, int64_t rows, const CeArgs& a, int64_t dp,
                          const int64_t* target, const float* bias, T* dst) {
    PackArgs<S> r = {};
    r.src = static_cast<const S*>(src);
    r.ld = ld;
    r.rows = rows;
    r.dim = a.dim;
    r.dp = int(dp);
    r.target = target;
    r.ignore = a.ignore;
    r.classes = a.classes;
    r.bias = bias;
    r.dst = dst;
    while (r.lanes < 6 && (8 << r.lanes) < dp) ++r.lanes;
    r.vec = ld % gt_chunk<S>() == 0 && reinterpret_cast<uintptr_t>(src) % 16 == 0;
    return r;
  }
  static void prepare(const CoefArgs& coef, const PackArgs<S>& x, const PackArgs<S>& w,
                      const Work& k, hipStream_t s) {
    if (!coef.grad && !x.src && !w.src) return;
    if constexpr (gt_is_split<T>) {
      oap_ce_largest<S><<<kMaxBlocks, 1024, 0, s>>>(x, w, k.largest);
      OAP_HIP_CHECK(hipGetLastError());
    }
    const int64_t items = std::max(x.src ? x.rows << x.lanes : 0, w.src ? w.rows << w.lanes : 0);
    const int64_t blocks = std::min<int64_t>(ceil_div(items, 1024), 2048);
    oap_ce_prepare<S, T><<<dim3(unsigned(std::max<int64_t>(1, blocks) + (coef.grad ? 1 : 0))),
                           1024, 0, s>>>(coef, x, w, k.largest, k.scale);
    OAP_HIP_CHECK(hipGetLastError());
  }

  template <int BM, int BN, int WAVES_M, bool SINGLE, bool GRAD>
  static void logits_tile(const LogitArgs& l, hipStream_t s) {
    auto k = oap_ce_logits<T, BM, BN, WAVES_M, SINGLE, GRAD>;
    constexpr int lds = GtTile<T, BM, kAlongK, BN, kAlongK, WAVES_M, SINGLE>::kLds;
    set_lds(k, lds);
    k<<<dim3(unsigned(l.vtiles * l.ntiles)), kGtThreads, lds, s>>>(l);
    OAP_HIP_CHECK(hipGetLastError());
  }

  template <bool GRAD>
  static void logits(const Plan& p, const LogitArgs& l, hipStream_t s) {
    if (p.bm == 64)
      logits_tile<64, 64, 2, false, GRAD>(l, s);
    else if (p.bn == 32)
      logits_tile<256, 32, 4, false, GRAD>(l, s);
    else if (p.bn == 64)
      logits_tile<256, 64, 4, true, GRAD>(l, s);
    else if (p.bn == 128 && p.bm == 256) {
      if constexpr (sizeof(T) == 2) logits_tile<256, 128, 2, true, GRAD>(l, s);
    } else if (p.bn == 128 && p.single)
      logits_tile<128, 128, 2, sizeof(T) == 2 || gt_is_split<T>, GRAD>(l, s);
    else if (p.bn == 128)
      logits_tile<128, 128, 2, sizeof(T) == 2, GRAD>(l, s);
    else if constexpr (sizeof(T) == 2)
      logits_tile<256, 256, 2, false, GRAD>(l, s);
  }

  static size_t carve_forward(const CeArgs& a, const Plan& p, void* base, Work& w) {
    Carver c{static_cast<char*>(base)};
    w = {};
    if (few_rows(a)) {
      w.part = c.take<float2>(size_t(kFewBlocks) * a.n);
      w.zt = c.take<float>(a.n);
      return c.used;
    }
    w.ximg = p.x_direct ? nullptr : c.take<T>(size_t(p.rows) * p.dp);
    w.wimg = p.w_direct ? nullptr : c.take<T>(size_t(std::min(p.piece, a.classes)) * p.dp);
    w.part = c.take<float2>(size_t(ceil_div(a.classes, p.bm)) * p.npad);
    w.zt = c.take<float>(p.rows);
    w.largest = c.take<float>(2 * kMaxBlocks);
    w.scale = c.take<int>(2);
    w.rowexp = p.split ? c.take<int>(p.rows) : nullptr;
    return c.used;
  }

  static size_t carve_backward(const CeArgs& a, const Plan& p, void* base, bool dx, bool dw,
                               bool db, Work& w) {
    Carver c{static_cast<char*>(base)};
    w = {};
    w.ximg = p.x_direct ? nullptr : c.take<T>(size_t(a.n) * p.dp);
    w.wimg = p.w_direct ? nullptr : c.take<T>(size_t(std::min(p.piece, a.classes)) * p.dp);
    w.largest = c.take<float>(2 * kMaxBlocks);
    w.scale = c.take<int>(2);
    w.rowexp = p.split ? c.take<int>(p.rows) : nullptr;
    w.ximg2 = p.split && dw ? c.take<T>(size_t(a.n) * p.dp) : nullptr;
    w.coef = c.take<float>(a.n);
    w.gscale = c.take<float>(1);
    w.dz = c.take<T>(size_t(p.npad) * p.piece);
    w.slab = dx ? c.take<float>(size_t(p.splits) * a.n * a.dim) : nullptr;
    w.dbpart = db ? c.take<float>(size_t(p.npad / p.bn) * p.piece) : nullptr;
    if (p.split && dw) {
      w.dzmax = c.take<float>(size_t(p.npad / p.bn) * p.piece);
      w.classscale = c.take<float>(p.piece);
    }
    w.rowscale = p.split && dx ? c.take<float>(a.n) : nullptr;
    return c.used;
  }

  static void forward(const CeArgs& all, float* loss, float2* stat, float* miss, float* total,
                      bool mean, void* work, hipStream_t s) {
    const Plan p = make_plan(all, false);
    Work w;
    carve_forward(all, p, work, w);
    if (few_rows(all)) {
      const int blocks = few(all, w, s);
      rows(all, w, blocks, all.n, loss, stat, nullptr, total, mean, s);
      return;
    }
    for (int64_t r0 = 0; r0 < all.n; r0 += p.rows) {
      CeArgs a = all;
      a.n = std::min(p.rows, all.n - r0);
      a.x = static_cast<const S*>(all.x) + r0 * all.ldx;
      a.target = all.target + r0;
      forward_rows(a, p, w, s);
      rows(a, w, int(ceil_div(a.classes, p.bm)), p.npad, loss + r0, stat + r0,
           p.split ? miss + r0 : nullptr, p.rows == all.n ? total : nullptr, mean, s);
    }
    if (total && p.rows < all.n) sum_losses(all, loss, total, mean, s);
  }

  // (max, sum) of all class tiles for the rows of a
  static void forward_rows(const CeArgs& a, const Plan& p, const Work& w, hipStream_t s) {
    const S* wt = static_cast<const S*>(a.w);
    LogitArgs l = {};
    PackArgs<S> px = {}, pw = {};
    l.x = {a.x, a.ldx, a.n, p.dp};
    if (!p.x_direct) {
      px = pack(a.x, a.ldx, a.n, a, p.dp, a.target, nullptr, w.ximg);
      px.rowexp = w.rowexp;
      l.x = {w.ximg, p.dp, a.n, p.dp};
    }
    l.dp = p.dp;
    l.scale = w.scale + 1;
    l.rowexp = w.rowexp;
    l.target = a.target;
    l.n = a.n;
    l.ntiles = int(ceil_div(a.n, p.bn));
    l.npad = p.npad;
    l.zt = w.zt;
    for (int64_t c0 = 0; c0 < a.classes; c0 += p.piece) {
      const int64_t nc = std::min(p.piece, a.classes - c0);
      const float* bias = a.bias ? a.bias + c0 : nullptr;
      l.w = {wt + c0 * a.ldw, a.ldw, nc, p.dp};
      if (!p.w_direct) {
        pw = pack(wt + c0 * a.ldw, a.ldw, nc, a, p.dp, nullptr, bias, w.wimg);
        l.w = {w.wimg, p.dp, nc, p.dp};
      }
      prepare({}, px, pw, w, s);
      px.src = nullptr;
      l.bias = bias;
      l.class0 = c0;
      l.vtiles = int(ceil_div(nc, p.bm));
      l.part = w.part + c0 / p.bm * p.npad;
      logits<false>(p, l, s);
    }
  }

  // One workgroup for little work (the total needs no launch of its own then), else at least one
  // per CU.
  static void rows(const CeArgs& a, const Work& w, int tiles, int64_t npad, float* loss,
                   float2* stat, float* miss, float* total, bool mean, hipStream_t s) {
    RowArgs r = {w.part, tiles, npad, a.n,  1,     a.target, a.ignore, a.classes,
                 w.zt,   loss,  stat, miss, total, mean};
    const bool one = a.n * tiles <= 16384;
    while (r.cols < 64 && r.cols * (one ? 1 : 256) < a.n) r.cols *= 2;
    if (a.n >= 8) r.cols = std::max(r.cols, 8);
    oap_ce_rows<<<dim3(one ? 1 : unsigned(ceil_div(a.n, r.cols))), 1024, 0, s>>>(r);
    OAP_HIP_CHECK(hipGetLastError());
    if (total && !one && ceil_div(a.n, r.cols) > 1) sum_losses(a, loss, total, mean, s);
  }
  static void sum_losses(const CeArgs& a, const float* loss, float* total, bool mean,
                         hipStream_t s) {
    RowArgs r = {};
    r.n = a.n;
    r.target = a.target;
    r.ignore = a.ignore;
    r.loss = const_cast<float*>(loss);
    r.total = total;
    r.mean = mean;
    oap_ce_total<<<1, 1024, 0, s>>>(r);
    OAP_HIP_CHECK(hipGetLastError());
  }

  template <int N, int G>
  static int few_launch(const FewArgs& f, hipStream_t s) {
    const int blocks =
        int(std::max<int64_t>(1, std::min<int64_t>(kFewBlocks, ceil_div(f.classes, 256 / G))));
    if (f.width == 16)
      oap_ce_few<S, N, G, true><<<dim3(unsigned(blocks)), 256, 0, s>>>(f);
    else
      oap_ce_few<S, N, G, false><<<dim3(unsigned(blocks)), 256, 0, s>>>(f);
    OAP_HIP_CHECK(hipGetLastError());
    return blocks;
  }
  template <int N>
  static int few_lanes(const FewArgs& f, hipStream_t s) {
    const int per = few_iters(N, sizeof(S)) * gt_chunk<S>();  // features of a lane
    if (f.dim <= 8 * per) return few_launch<N, 8>(f, s);
    if (f.dim <= 16 * per) return few_launch<N, 16>(f, s);
    if (f.dim <= 32 * per) return few_launch<N, 32>(f, s);
    return few_launch<N, 64>(f, s);
  }
  static int few(const CeArgs& a, const Work& w, hipStream_t s) {
    FewArgs f = {};
    f.w = a.w;
    f.x = a.x;
    f.ldw = a.ldw;
    f.ldx = a.ldx;
    f.classes = a.classes;
    f.n = int(a.n);
    f.dim = a.dim;
    f.width = few_width(a);
    f.bias = a.bias;
    f.target = a.target;
    f.part = w.part;
    f.zt = w.zt;
    if (a.n == 1) return few_lanes<1>(f, s);
    if constexpr (sizeof(S) == 4)
      if (a.n > 4) return few_lanes<8>(f, s);
    return few_lanes<4>(f, s);
  }

  // dx's tiles and dW's; none where out is null
  template <int B, GradPart PART>
  static void grads_tile(const ProdArgs& x, const ProdArgs& w, hipStream_t s) {
    constexpr bool raw = gt_is_split<T>;
    constexpr int lds = std::max(GtTile<T, B, kAlongK, B, kAcrossK, 2, false, raw>::kLds,
                                 GtTile<T, B, kAcrossK, B, kAcrossK, 2, false, raw>::kLds);
    const int nx = x.out && PART != kDw ? x.mtiles * x.ntiles * x.splits : 0;
    const int nw = w.out && PART != kDx ? w.mtiles * w.ntiles : 0;
    if (nx + nw == 0) return;
    auto k = oap_ce_grads<S, T, B, PART>;
    set_lds(k, lds);
    k<<<dim3(unsigned(nx + nw)), kGtThreads, lds, s>>>(x, w, nx);
    OAP_HIP_CHECK(hipGetLastError());
  }
  static void grads(int tile, const ProdArgs& x, const ProdArgs& w, hipStream_t s) {
    if (tile == 64) {
      grads_tile<64, kBoth>(x, w, s);
    } else if (tile == 128) {
      grads_tile<128, kBoth>(x, w, s);
    } else if constexpr (sizeof(T) == 2) {
      grads_tile<256, kDx>(x, w, s);
      grads_tile<256, kDw>(x, w, s);
    }
  }

  static void products(const CeArgs& a, const Plan& p, const Work& w, const LogitArgs& l,
                       int64_t nc, int64_t c0, float unscale, void* dx, void* dw,
                       hipStream_t s) {
    ProdArgs gx = {}, gw = {};
    gx.n = gw.n = a.dim;
    gx.gscale = gw.gscale = w.gscale;
    gx.unscale = gw.unscale = unscale;
    gx.a = {w.dz, p.piece, a.n, p.piece, w.rowscale};
    gw.a = {w.dz, p.piece, p.npad, p.piece, w.classscale};
    if (dx) {
      gx.b = l.w;
      gx.scale = w.scale + 1;
      gx.k = nc;
      gx.m = a.n;
      gx.mtiles = int(ceil_div(a.n, p.xtile));
      gx.ntiles = int(ceil_div(a.dim, p.xtile));
      gx.splits = p.splits;
      gx.out = w.slab;
      gx.add = c0 > 0;
    }
    if (dw) {
      gw.b = l.x;
      if (p.split) gw.b.p = w.ximg2;
      gw.scale = w.scale;
      gw.k = a.n;
      gw.m = nc;
      gw.mtiles = int(ceil_div(nc, p.wtile));
      gw.ntiles = int(ceil_div(a.dim, p.wtile));
      gw.splits = 1;
      gw.out = static_cast<S*>(dw) + c0 * a.dim;
      gw.bias = a.bias ? a.bias + c0 : nullptr;
    }
    if (p.xtile == p.wtile) {
      grads(p.xtile, gx, gw, s);
    } else {
      grads(p.xtile, gx, {}, s);
      grads(p.wtile, {}, gw, s);
    }
  }

  static void backward(const CeArgs& a, const float2* stat, const float* miss, const float* grad,
                       bool per_row, bool mean, void* dx, void* dw, float* db, void* work,
                       hipStream_t s) {
    const Plan p = make_plan(a, true);
    Work w;
    carve_backward(a, p, work, dx, dw, db, w);
    const S* wt = static_cast<const S*>(a.w);
    // fp16 images hold dz times 2^14: |dz| <= 1 stays finite and 2^-28 is still a normal number
    const float pscale = a.elem == Elem::F16 ? 0x1p14f : 1.f;
    const CoefArgs coef = {grad,   per_row,  mean,       a.target, a.ignore, a.classes, a.n,
                           w.coef, w.gscale, w.rowscale, miss};
    LogitArgs l = {};
    PackArgs<S> px = pack(a.x, a.ldx, a.n, a, p.dp, a.target, nullptr, w.ximg), pw = {};
    px.grad = per_row ? grad : nullptr;
    px.rowexp = w.rowexp;
    px.dst2 = w.ximg2;
    l.x = {w.ximg, p.dp, a.n, p.dp};
    l.dp = p.dp;
    l.scale = w.scale + 1;
    l.rowexp = w.rowexp;
    l.target = a.target;
    l.n = a.n;
    l.ntiles = int(p.npad / p.bn);
    l.npad = p.npad;
    l.stat = stat;
    l.coef = w.coef;
    l.pscale = pscale;
    l.unscale = 1.f / pscale;
    l.dz = w.dz;
    l.vp = p.piece;
    l.dbpart = w.dbpart;
    l.dzmax = w.dzmax;
    for (int64_t c0 = 0; c0 < a.classes; c0 += p.piece) {
      const int64_t nc = std::min(p.piece, a.classes - c0);
      const bool last = c0 + nc == a.classes;
      const float* bias = a.bias ? a.bias + c0 : nullptr;
      l.w = {wt + c0 * a.ldw, a.ldw, nc, p.dp};
      if (!p.w_direct) {
        pw = pack(wt + c0 * a.ldw, a.ldw, nc, a, p.dp, nullptr, bias, w.wimg);
        l.w = {w.wimg, p.dp, nc, p.dp};
      }
      prepare(c0 ? CoefArgs{} : coef, px, pw, w, s);
      px.src = nullptr;
      l.bias = bias;
      l.class0 = c0;
      l.vtiles = int(ceil_div(nc, p.bm));
      logits<true>(p, l, s);
      if (w.dzmax) {
        oap_ce_class_scales<<<dim3(unsigned(p.piece / 256)), 256, 0, s>>>(
            w.dzmax, l.ntiles, p.piece, nc, w.classscale);
        OAP_HIP_CHECK(hipGetLastError());
      }
      products(a, p, w, l, nc, c0, 1.f / pscale, dx, dw, s);
      FinishArgs<S> f = {};
      f.gscale = w.gscale;
      f.coef = w.coef;
      f.bias = bias;
      int64_t blocks = 0;
      if (db) {
        f.dbpart = w.dbpart;
        f.rtiles = l.ntiles;
        f.vp = p.piece;
        f.classes = nc;
        f.db = db + c0;
        blocks = ceil_div(nc, 256);
      }
      if (dx && last) {
        f.slab = w.slab;
        f.splits = p.splits;
        f.count = a.n * a.dim;
        f.dim = a.dim;
        f.unscale = 1.f / pscale;
        f.dx = static_cast<S*>(dx);
        blocks += stride_grid(f.count);
      }
      if (blocks > 0) {
        oap_ce_finish<S><<<dim3(unsigned(blocks)), 256, 0, s>>>(f);
        OAP_HIP_CHECK(hipGetLastError());
      }
    }
  }

  static void zeros(const CeArgs& a, void* dx, void* dw, float* db, hipStream_t s) {
    const int64_t nx = a.n * a.dim, nw = a.classes * a.dim;
    if (dx && nx) oap_ce_fill0<S><<<stride_grid(nx), 256, 0, s>>>(static_cast<S*>(dx), nx);
    if (dw && nw) oap_ce_fill0<S><<<stride_grid(nw), 256, 0, s>>>(static_cast<S*>(dw), nw);
    if (db && a.classes)
      oap_ce_fill0<float><<<stride_grid(a.classes), 256, 0, s>>>(db, a.classes);
    OAP_HIP_CHECK(hipGetLastError());
  }
};

void check(const CeArgs& a) {
  OAP_CHECK(a.n >= 0 && a.n < (int64_t(1) << 31) - 256 && a.classes >= 1 &&
                a.classes < (int64_t(1) << 31) - 256 && a.dim >= 1 && a.dim <= (1 << 20) &&
                a.ldx >= a.dim && a.ldw >= a.dim,
            "softmax_cross_entropy: bad shape");
  OAP_CHECK(ceil_div(a.n, 64) * ceil_div(a.classes, 64) < (int64_t(1) << 31),
            "softmax_cross_entropy: " << a.n << " x " << a.classes << " tiles are too many");
}

// f(Ce<..>{}) for the element type and the plan's operands
template <typename F>
void ce_dispatch(const CeArgs& a, F&& f) {
  switch (a.elem) {
    case Elem::BF16: f(Ce<__bf16, __bf16>{}); break;
    case Elem::F16: f(Ce<_Float16, _Float16>{}); break;
    case Elem::F32:
      if (split_fp32(a))
        f(Ce<float, GtSplit>{});
      else
        f(Ce<float, float>{});
      break;
  }
}

}  // namespace

CePlan ce_plan(const CeArgs& a, bool grad) {
  check(a);
  const Plan p = make_plan(a, grad);
  return {p.rows, p.piece, p.split};
}

size_t ce_forward_bytes(const CeArgs& a) {
  check(a);
  if (a.n == 0) return 0;
  size_t r = 0;
  ce_dispatch(a, [&](auto t) {
    typename decltype(t)::Work w;
    r = decltype(t)::carve_forward(a, make_plan(a, false), nullptr, w);
  });
  return r;
}

void ce_forward(const CeArgs& a, float* loss, float2* stat, float* miss, float* total, bool mean,
                void* work, hipStream_t s) {
  check(a);
  if (a.n == 0) {  // no row: the sum and the mean are 0
    if (total) oap_ce_fill0<float><<<1, 256, 0, s>>>(total, 1);
    OAP_HIP_CHECK(hipGetLastError());
    return;
  }
  ce_dispatch(a, [&](auto t) {
    decltype(t)::forward(a, loss, stat, miss, total, mean, work, s);
  });
}

size_t ce_backward_bytes(const CeArgs& a, bool want_dx, bool want_dw, bool want_db) {
  check(a);
  if (a.n == 0) return 0;
  size_t r = 0;
  ce_dispatch(a, [&](auto t) {
    typename decltype(t)::Work w;
    r = decltype(t)::carve_backward(a, make_plan(a, true), nullptr, want_dx, want_dw, want_db,
                                        w);
  });
  return r;
}

void ce_backward(const CeArgs& a, const float2* stat, const float* miss, const float* grad,
                 bool per_row, bool mean, void* dx, void* dw, float* db, void* work,
                 hipStream_t s) {
  check(a);
  ce_dispatch(a, [&](auto t) {
    if (a.n == 0)
      decltype(t)::zeros(a, dx, dw, db, s);
    else
      decltype(t)::backward(a, stat, miss, grad, per_row, mean, dx, dw, db, work, s);
  });
}

}  // namespace kern
}  // namespace oap
