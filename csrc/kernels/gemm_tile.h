// Tile core of the products of the softmax cross entropy: C[m, n] = sum_k A(m, k) B(n, k) in
// bf16 or fp16 on v_mfma_f32_32x32x16 with fp32 sums.  Each operand lies in memory either with k
// along its rows (kAlongK: element (r, k) at r * ld + k) or with k across them (kAcrossK: at
// k * ld + r), so no operand is ever transposed in memory.
//
// A workgroup of 8 waves owns a BM x BN tile.  k advances in blocks of 64, staged by
// global_load_lds (16 bytes a lane) into one of two LDS buffers while the other feeds the MFMAs:
// one barrier a block.
//  * kAlongK: 128 bytes of each row; the 16-byte chunk c of row r lies at slot c ^ (r & 7), so
//    the eight rows that a fragment read (ds_read_b128) touches at once use different banks.
//  * kAcrossK: 64 rows of k with R elements each, read by ds_read_b64_tr_b16: the 16 lanes of
//    a group pass the addresses of 4 x 16 elements (4 of k, 16 of r) and get them transposed,
//    lane i the four k of r = i.  Two reads make a fragment.  The 64-byte granule of a row is
//    xor-ed with bits of k, so the four k rows of a read use different banks.
// global_load_lds writes its 64 lanes' data in lane order, so both permutations are applied to
// the global addresses.
//
// fp32 operands come as three bf16 planes per row (x = h + m + l, 8 bits each: all 24 bits of
// the significand); the six plane products above 2^-24 are summed as if k were six times as
// long, smallest first.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace oap {
namespace kern {

typedef __bf16 gt_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 gt_f16x8 __attribute__((ext_vector_type(8)));
typedef short gt_s16x4 __attribute__((ext_vector_type(4)));
typedef short gt_s16x8 __attribute__((ext_vector_type(8)));
typedef float gt_f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void* gt_lds_ptr;
typedef __attribute__((address_space(3))) gt_s16x4* gt_lds_s16x4;
typedef const __attribute__((address_space(1))) void* gt_glb_ptr;

template <typename T>
struct GtVec;
template <>
struct GtVec<__bf16> {
  typedef gt_bf16x8 type;
};
template <>
struct GtVec<_Float16> {
  typedef gt_f16x8 type;
};

__device__ inline gt_f32x16 gt_mfma(gt_bf16x8 a, gt_bf16x8 b, gt_f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ inline gt_f32x16 gt_mfma(gt_f16x8 a, gt_f16x8 b, gt_f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

constexpr int kGtK = 64;         // elements of k per block
constexpr int kGtThreads = 512;  // 8 waves

// `rows` x `cols` elements in memory, row stride `ld`; plane q of a row starts at q * plane.
// Reads beyond the last row or the last whole 16 bytes of a row are moved back onto them, so
// what lies there is the caller's to leave out.  cols is a multiple of 8, p 16-byte aligned.
struct GtOperand {
  const void* p;
  int64_t ld;
  int64_t rows, cols;
  int64_t plane;
};

enum GtOrder { kAlongK, kAcrossK };

// One operand of R rows in a tile; W waves' worth of pieces.
template <typename T, int R, GtOrder ORDER>
struct GtSide {
  static constexpr int kBytes = R * kGtK * 2;  // of a staged block
  static constexpr int kPieces = kBytes / 1024;
  static constexpr int kChunks = R / 8;  // 16-byte chunks of a k row (kAcrossK)
  typedef typename GtVec<T>::type V8;

  // xor on the chunk index of k row r
  __device__ static int swizzle(int r) {
    return R >= 256 ? (r & 7) << 2 : R == 128 ? (r & 3) << 2 : ((r >> 1) & 1) << 2;
  }

  // Global address of this lane's 16 bytes of piece `piece` for k block 0 of the range
  struct Source {
    const char* p;
    int64_t row, limit;  // kAcrossK: k row and the last valid one
    int64_t step;        // bytes per k block
    int64_t ld;          // bytes
    __device__ const char* at(int64_t kb, int64_t plane_bytes) const {
      if (ORDER == kAlongK) return p + kb * step + plane_bytes;
      const int64_t r = row + kb * kGtK;
      return p + (r < limit ? r : limit) * ld + plane_bytes;
    }
  };
  __device__ static Source source(const GtOperand& o, int piece, int lane, int64_t r0,
                                  int64_t k0) {
    Source s;
    s.ld = o.ld * 2;
    s.limit = o.rows - 1;
    if (ORDER == kAlongK) {
      const int64_t r = r0 + piece * 8 + (lane >> 3);
      const int chunk = (lane & 7) ^ (lane >> 3);
      s.p = static_cast<const char*>(o.p) + (r < o.rows ? r : o.rows - 1) * s.ld + k0 * 2 +
            chunk * 16;
      s.step = kGtK * 2;
      s.row = 0;
    } else {
      const int kr = piece * (64 / kChunks) + lane / kChunks;
      const int chunk = (lane % kChunks) ^ swizzle(kr);
      const int64_t c = r0 + chunk * 8;
      s.p = static_cast<const char*>(o.p) + (c < o.cols ? c : o.cols - 8) * 2;
      s.step = 0;
      s.row = k0 + kr;
    }
    return s;
  }

  // Per-lane LDS offsets of the fragments of rows base + 32 i
  template <int N>
  struct Reader {
    int off[ORDER == kAlongK ? 1 : N][2];
    int r7;
    __device__ void init(int lane, int base) {
      if (ORDER == kAlongK) {
        off[0][0] = (base + (lane & 31)) * 128;
        r7 = lane & 7;
      } else {
        const int g = lane >> 4, s = lane & 15;
#pragma unroll
        for (int i = 0; i < (ORDER == kAlongK ? 1 : N); ++i)
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const int k = 8 * (g >> 1) + (s >> 2) + 4 * q;
            const int chunk = (base + 32 * i + 16 * (g & 1)) / 8 + ((s & 3) >> 1);
            off[i][q] = k * R * 2 + (chunk ^ swizzle(k)) * 16 + (s & 1) * 8;
          }
      }
    }
    __device__ V8 read(const char* block, int i, int ks, int lane) const {
      if constexpr (ORDER == kAlongK) {
        const int slot = ((2 * ks + (lane >> 5)) ^ r7) * 16;
        return *reinterpret_cast<const V8*>(block + off[0][0] + i * 32 * 128 + slot);
      } else {
        const char* p = block + ks * 16 * R * 2;
        const gt_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((gt_lds_s16x4)(p + off[i][0]));
        const gt_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((gt_lds_s16x4)(p + off[i][1]));
        const gt_s16x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        return __builtin_bit_cast(V8, v);
      }
    }
  };
};

// Element (row i, column j) of acc[mi][ni][e] in lane l of wave (wm, wn):
//   i = wm * WM + 32 mi + 8 (e >> 2) + 4 (l >> 5) + (e & 3),   j = wn * WN + 32 ni + (l & 31)
template <typename T, int BM_, GtOrder OA, int BN_, GtOrder OB, int WAVES_M, int PLANES>
struct GtTile {
  static constexpr int BM = BM_, BN = BN_;
  static constexpr int WAVES_N = 8 / WAVES_M;
  static constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N;
  static constexpr int MI = WM / 32, NI = WN / 32;
  typedef GtSide<T, BM, OA> SideA;
  typedef GtSide<T, BN, OB> SideB;
  static constexpr int kBuf = SideA::kBytes + SideB::kBytes;
  static constexpr int kLds = 2 * kBuf;
  static constexpr int kPairs = PLANES == 3 ? 6 : 1;
  static constexpr int kLoadsA = SideA::kPieces / 8, kLoadsB = SideB::kPieces / 8;
  typedef typename GtVec<T>::type V8;
  static_assert(MI >= 1 && NI >= 1 && kLoadsB >= 1 && (PLANES == 1 || PLANES == 3), "tile");

  // acc += A[m0.., k0..k1) B[n0.., k0..k1)^T; k0, k1 multiples of 64.  Every thread of the
  // workgroup calls it; all LDS reads are done when it returns.
  __device__ static void run(const GtOperand& A, const GtOperand& B, int64_t m0, int64_t n0,
                             int64_t k0, int64_t k1, char* lds, gt_f32x16 (&acc)[MI][NI]) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    typename SideA::Source sa[kLoadsA];
    typename SideB::Source sb[kLoadsB];
#pragma unroll
    for (int i = 0; i < kLoadsA; ++i) sa[i] = SideA::source(A, wave * kLoadsA + i, lane, m0, k0);
#pragma unroll
    for (int i = 0; i < kLoadsB; ++i) sb[i] = SideB::source(B, wave * kLoadsB + i, lane, n0, k0);
    typename SideA::template Reader<MI> ra;
    typename SideB::template Reader<NI> rb;
    ra.init(lane, (wave / WAVES_N) * WM);
    rb.init(lane, (wave % WAVES_N) * WN);
    const int nk = int((k1 - k0) / kGtK), total = nk * kPairs;
    auto stage = [&](int it, int buf) {
      int kb = it, pa = 0, pb = 0;
      if (kPairs > 1) {
        const int pair = it / nk;
        kb = it - pair * nk;
        // (l,h) (h,l) (m,m) (m,h) (h,m) (h,h)
        pa = pair == 0 ? 2 : (pair == 2 || pair == 3) ? 1 : 0;
        pb = pair == 1 ? 2 : (pair == 2 || pair == 4) ? 1 : 0;
      }
      char* da = lds + buf * kBuf + wave * kLoadsA * 1024;
      char* db = lds + buf * kBuf + SideA::kBytes + wave * kLoadsB * 1024;
#pragma unroll
      for (int i = 0; i < kLoadsA; ++i)
        __builtin_amdgcn_global_load_lds((gt_glb_ptr)(sa[i].at(kb, pa * A.plane * 2)),
                                         (gt_lds_ptr)(da + i * 1024), 16, 0, 0);
#pragma unroll
      for (int i = 0; i < kLoadsB; ++i)
        __builtin_amdgcn_global_load_lds((gt_glb_ptr)(sb[i].at(kb, pb * B.plane * 2)),
                                         (gt_lds_ptr)(db + i * 1024), 16, 0, 0);
    };
    if (total > 0) stage(0, 0);
    for (int it = 0; it < total; ++it) {
      const int buf = it & 1;
      // this wave's pieces of the block landed, then everyone's; and every wave has read the
      // other buffer (its reads fed MFMAs that were issued before the barrier)
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      const char* la = lds + buf * kBuf;
      const char* lb = la + SideA::kBytes;
      constexpr int KS = kGtK / 16;
      if constexpr (OA == kAcrossK || OB == kAcrossK) {
        // all of the block's fragments are read before the next block's loads are issued: the
        // compiler waits for every load in flight before a transposed read
        V8 a[KS][MI], b[KS][NI];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
          for (int i = 0; i < MI; ++i) a[ks][i] = ra.read(la, i, ks, lane);
#pragma unroll
          for (int j = 0; j < NI; ++j) b[ks][j] = rb.read(lb, j, ks, lane);
        }
        if (it + 1 < total) stage(it + 1, buf ^ 1);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[i][j] = gt_mfma(a[ks][i], b[ks][j], acc[i][j]);
      } else {
        if (it + 1 < total) stage(it + 1, buf ^ 1);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          V8 a[MI], b[NI];
#pragma unroll
          for (int i = 0; i < MI; ++i) a[i] = ra.read(la, i, ks, lane);
#pragma unroll
          for (int j = 0; j < NI; ++j) b[j] = rb.read(lb, j, ks, lane);
#pragma unroll
          for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[i][j] = gt_mfma(a[i], b[j], acc[i][j]);
        }
      }
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }

  __device__ static int wave_m() { return (threadIdx.x >> 6) / WAVES_N; }
  __device__ static int wave_n() { return (threadIdx.x >> 6) % WAVES_N; }
  // first row / column of this wave's part of the tile, and of the lane in a 32 x 32 block
  __device__ static int row0() { return wave_m() * WM + 4 * ((threadIdx.x & 63) >> 5); }
  __device__ static int col0() { return wave_n() * WN + (threadIdx.x & 31); }
  __device__ static constexpr int row_of(int mi, int e) { return 32 * mi + 8 * (e >> 2) + (e & 3); }
  __device__ static void clear(gt_f32x16 (&acc)[MI][NI]) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  }
};

}  // namespace kern
}  // namespace oap
