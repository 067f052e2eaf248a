// Tile core of the products of the softmax cross entropy: C[m, n] = sum_k A(m, k) B(n, k) on the
// matrix units, in bf16 or fp16 (v_mfma_f32_32x32x16), in fp32 (v_mfma_f32_32x32x2) or in fp32 as
// two fp16 numbers (GtSplit), with fp32 sums.  Each operand lies in memory either with k along its
// rows (kAlongK: element (r, k) at r * ld + k) or with k across them (kAcrossK: at k * ld + r), so
// no operand is ever transposed in memory.
//
// A workgroup of 4 waves, one per SIMD, owns a BM x BN tile; a wave's part of up to 128 x 128
// keeps 256 accumulators, so a byte read from LDS feeds the most MFMAs.  k advances in blocks of
// 128 bytes of a row (64 or 32 elements) in two LDS buffers: the next block is loaded into
// registers while this one is multiplied, and written to the other buffer before the last of
// its four steps; one barrier a block, and behind it the last step's MFMAs cover the first reads
// of the next block.
//  * kAlongK: 128 bytes of each row; the 16-byte chunk c of row r lies at slot c ^ ((r >> 1) & 7),
//    so the 16 rows that a fragment read (ds_read_b128) touches at once use all 64 banks.
//  * kAcrossK, 16 bits: 64 rows of k, read by ds_read_b64_tr_b16: the 16 lanes of a group pass
//    the addresses of 4 x 16 elements (4 of k, 16 of r) and get them transposed, lane i the four
//    k of r = i.  Two reads make a fragment.  The 64-byte granule of a row is xor-ed with bits
//    of k, so the four k rows of a read use different banks.
//  * kAcrossK, fp32: 32 rows of k, read by ds_read_b32 (32 lanes along a row).
//
// GtSplit: a matrix scaled by a power of two so that its largest magnitude lies in [2^14, 2^15),
// each number the sum of two fp16, h + l.  A product is l h + h l + h h: it leaves out l l and
// the rounding of l, each below 2^-22 of the product, and numbers below 2^-15 of the matrix's
// largest keep an absolute error of 2^-40 of that.  Three 16-bit MFMAs take a fifth of the time
// of the fp32 ones.  A row lies as runs of 32 numbers, their 32 h and then their 32 l, so 128
// bytes of a row hold 32 k in either order of k.
//
// The A operand may lie in fp32 instead (RAW) and is split on its way to LDS, at a power of two of
// its own for each row of the result: a row then keeps 22 bits of its numbers, or 2^-40 of its
// largest, whatever the others hold, and the scale needs to be known only when the tile is read.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace oap {
namespace kern {

typedef __bf16 gt_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 gt_f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 gt_f16x4 __attribute__((ext_vector_type(4)));
typedef short gt_s16x4 __attribute__((ext_vector_type(4)));
typedef short gt_s16x8 __attribute__((ext_vector_type(8)));
typedef float gt_f32x4 __attribute__((ext_vector_type(4)));
typedef float gt_f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned gt_u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) gt_s16x4* gt_lds_s16x4;

// A fragment: the 16 bytes of a lane that one step of k multiplies
template <typename T>
struct GtFrag;
template <>
struct GtFrag<__bf16> {
  typedef gt_bf16x8 type;
};
template <>
struct GtFrag<_Float16> {
  typedef gt_f16x8 type;
};
template <>
struct GtFrag<float> {
  typedef gt_f32x4 type;
};
struct GtSplit {
  _Float16 h, l;
};
struct gt_split8 {
  gt_f16x8 h, l;
};
template <>
struct GtFrag<GtSplit> {
  typedef gt_split8 type;
};

__device__ inline gt_f32x16 gt_mfma(gt_bf16x8 a, gt_bf16x8 b, gt_f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ inline gt_f32x16 gt_mfma(gt_f16x8 a, gt_f16x8 b, gt_f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ inline gt_f32x16 gt_mfma(gt_f32x4 a, gt_f32x4 b, gt_f32x16 c) {
#pragma unroll
  for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

__device__ inline gt_f32x16 gt_mfma(const gt_split8& a, const gt_split8& b, gt_f32x16 c) {
  c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.l, b.h, c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a.h, b.l, c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a.h, b.h, c, 0, 0, 0);
}
template <typename T>
constexpr bool gt_is_split = false;
template <>
constexpr bool gt_is_split<GtSplit> = true;
// steps of k per block, and MFMAs of a step's 32 x 32 product
template <typename T>
constexpr int gt_steps = gt_is_split<T> ? 2 : 4;
template <typename T>
constexpr int gt_mfmas = gt_is_split<T> ? 3 : sizeof(T) == 4 ? 4 : 1;

constexpr int kGtThreads = 256;  // 4 waves
// waves per SIMD that a tile's registers allow
constexpr int gt_occupancy(int bm, int bn) { return bm * bn <= 256 * 128 ? 2 : 1; }

// elements of k per block, and per 16-byte chunk
template <typename T>
constexpr int gt_block() {
  return 128 / int(sizeof(T));
}
template <typename T>
constexpr int gt_chunk() {
  return 16 / int(sizeof(T));
}

// `rows` x `cols` elements in memory, row stride `ld`; cols and ld are multiples of a chunk
// (GtSplit: of 32) and p is 16-byte aligned.  256 rows span less than 2^31 bytes.  k beyond the
// extent of the operand reads as 0; rows beyond `rows` (kAlongK) or columns beyond `cols`
// (kAcrossK) read as some others, and the results they belong to are the caller's to leave out.
struct GtOperand {
  const void* p;
  int64_t ld;
  int64_t rows, cols;
  const float* scale;  // RAW: the power of two of each row (kAlongK) or column (kAcrossK)
};

enum GtOrder { kAlongK, kAcrossK };

// One operand of R rows of a tile
template <typename T, int R, GtOrder ORDER, bool RAW = false>
struct GtSide {
  static constexpr int BK = gt_block<T>(), CH = gt_chunk<T>();
  static constexpr int kBytes = R * 128;                // of a staged block
  static constexpr int kLoads = kBytes / 16 / kGtThreads;  // 16-byte loads of a thread
  static constexpr int kChunks = R / CH;                // chunks of a k row (kAcrossK)
  static constexpr int kRowBytes = R * int(sizeof(T));  // of a k row (kAcrossK)
  static constexpr int kStep = ORDER == kAlongK ? kGtThreads / 8 : kGtThreads / kChunks;
  static constexpr bool kSplit = gt_is_split<T>;
  static constexpr bool kTransposed = ORDER == kAcrossK && (sizeof(T) == 2 || kSplit);
  // LDS reads of a fragment
  static constexpr int kReads = (ORDER == kAlongK ? 1 : kTransposed ? 2 : 4) * (kSplit ? 2 : 1);
  static constexpr int kWrites = (RAW ? 2 : 1) * kLoads;  // LDS writes of a thread
  typedef typename GtFrag<T>::type Frag;
  static_assert(kLoads >= 1, "a thread stages at least 16 bytes of each operand");
  static_assert(!RAW || kSplit, "only split operands are made from fp32");

  // xor on the chunk index of k row r
  __device__ static int swizzle(int r) {
    if (!kTransposed) return 0;
    return kRowBytes >= 512 ? (r & 7) << 2 : kRowBytes == 256 ? (r & 3) << 2 : ((r >> 1) & 1) << 2;
  }

  // The thread's loads: rows r, r + kStep, ... of a block (rows of the tile, or rows of k)
  struct Loader {
    const char* base;  // uniform: the tile's first element at the range's first k
    uint32_t off[kLoads];
    uint32_t ldb;      // bytes of a row in memory
    int left;          // k from the block's first to the end of the operand or the range
    int sub;           // the thread's place in k within a block: its chunk's first k, or row
    uint32_t lds;      // byte in the staged block
    // RAW: of the thread's rows (kAlongK) or its four columns
    float mul[RAW ? (ORDER == kAlongK ? kLoads : 4) : 1];

    __device__ void init(const GtOperand& o, int64_t r0, int64_t k0, int64_t k1) {
      const int t = threadIdx.x;
      ldb = uint32_t(o.ld * sizeof(T));
      if (ORDER == kAlongK) {
        const int r = t >> 3, chunk = t & 7;
        base = static_cast<const char*>(o.p) + r0 * o.ld * sizeof(T) + k0 * sizeof(T);
        const int64_t last = o.rows - 1 - r0;  // >= 0: a tile starts within the operand
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          const int q = r + i * kStep;
          off[i] = uint32_t(q < last ? q : last) * ldb + chunk * 16;
          if constexpr (RAW) mul[i] = o.scale[r0 + (q < last ? q : last)];
        }
        left = int((k1 < o.cols ? k1 : o.cols) - k0);
        sub = kSplit && !RAW ? 0 : chunk * CH;
        // (RAW: four numbers, whose h are half a chunk, and their l four chunks on)
        lds = RAW ? r * 128 + (((chunk >> 1) ^ ((r >> 1) & 7)) << 4) + (chunk & 1) * 8
                  : r * 128 + ((chunk ^ ((r >> 1) & 7)) << 4);
      } else {
        const int k = t / kChunks, chunk = t % kChunks;
        base = static_cast<const char*>(o.p) + k0 * o.ld * sizeof(T) + r0 * sizeof(T);
        const int64_t last = o.cols - CH - r0;  // >= 0
        const int64_t c = int64_t(chunk) * CH;
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
          off[i] = uint32_t(k + i * kStep) * ldb + uint32_t((c < last ? c : last) * sizeof(T));
        left = int((k1 < o.rows ? k1 : o.rows) - k0);
        sub = k;
        const int at = RAW ? (chunk & ~7) + ((chunk & 7) >> 1) : chunk;
        lds = k * kRowBytes + ((at ^ swizzle(k)) << 4) + (RAW ? (chunk & 1) * 8 : 0);
        if constexpr (RAW) {
#pragma unroll
          for (int j = 0; j < 4; ++j) mul[j] = o.scale[r0 + (c < last ? c : last) + j];
        }
      }
    }
    // loads the block and steps to the next.  Buffer loads: an offset beyond the resource reads
    // as 0, so what lies beyond the extent of k needs no branch (a branch would make the compiler
    // wait for the loads where its paths join).
    __device__ void load(gt_u32x4 (&v)[kLoads]) {
      const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), short(0),
                                                          0x7fffffff, 0x00020000);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int k = sub + (ORDER == kAlongK ? 0 : i * kStep);
        const uint32_t o = k < left ? off[i] : 0x80000000u;
        v[i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, o, 0, 0);
      }
      base += ORDER == kAlongK ? 128u : BK * ldb;
      left -= BK;
    }
    __device__ void store(char* block, const gt_u32x4 (&v)[kLoads]) const {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        constexpr int kRow = ORDER == kAlongK ? 128 : kRowBytes;
        if constexpr (RAW) {
          const gt_f32x4 f = __builtin_bit_cast(gt_f32x4, v[i]);
          gt_f16x4 h, l;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float x = f[j] * mul[ORDER == kAlongK ? i : j];
            h[j] = static_cast<_Float16>(x);
            l[j] = static_cast<_Float16>(x - static_cast<float>(h[j]));
          }
          *reinterpret_cast<gt_f16x4*>(block + lds + i * kStep * kRow) = h;
          *reinterpret_cast<gt_f16x4*>(block + (lds ^ 64) + i * kStep * kRow) = l;
        } else {
          *reinterpret_cast<gt_u32x4*>(block + lds + i * kStep * kRow) = v[i];
        }
      }
    }
  };

  // Fragments of the rows base + 32 i
  template <int N>
  struct Reader {
    static constexpr int kOffs = kTransposed ? N : 1, kPlanes = kSplit ? 2 : 1;
    int off[kOffs][kPlanes][2];
    int x7;
    __device__ void init(int lane, int base) {
      if (ORDER == kAlongK) {
        off[0][0][0] = (base + (lane & 31)) * 128;
        x7 = (lane >> 1) & 7;
      } else if (!kTransposed) {
        off[0][0][0] = 4 * (lane >> 5) * kRowBytes + (base + (lane & 31)) * 4;
      } else {
        const int g = lane >> 4, s = lane & 15;
#pragma unroll
        for (int i = 0; i < kOffs; ++i)
#pragma unroll
          for (int p = 0; p < kPlanes; ++p)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const int k = 8 * (g >> 1) + (s >> 2) + 4 * q;
              const int first = (base + 32 * i) / 8 * kPlanes + 4 * p;  // chunk of the run
              const int chunk = first + 2 * (g & 1) + ((s & 3) >> 1);
              off[i][p][q] = k * kRowBytes + ((chunk ^ swizzle(k)) << 4) + (s & 1) * 8;
            }
      }
    }
    template <typename V>
    __device__ static V transposed(const char* lo, const char* hi) {
      const gt_s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((gt_lds_s16x4)lo);
      const gt_s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((gt_lds_s16x4)hi);
      const gt_s16x8 v = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
      return __builtin_bit_cast(V, v);
    }
    __device__ Frag read(const char* block, int i, int ks, int lane) const {
      if constexpr (ORDER == kAlongK) {
        const char* p = block + off[0][0][0] + i * 32 * 128;
        const int c = 2 * ks + (lane >> 5);
        if constexpr (kSplit) {
          Frag f;
          f.h = *reinterpret_cast<const gt_f16x8*>(p + ((c ^ x7) << 4));
          f.l = *reinterpret_cast<const gt_f16x8*>(p + (((c + 4) ^ x7) << 4));
          return f;
        } else {
          return *reinterpret_cast<const Frag*>(p + ((c ^ x7) << 4));
        }
      } else if constexpr (!kTransposed) {
        const char* p = block + off[0][0][0] + ks * 8 * kRowBytes + i * 32 * 4;
        Frag f;
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = *reinterpret_cast<const float*>(p + j * kRowBytes);
        return f;
      } else {
        const char* p = block + ks * 16 * kRowBytes;
        if constexpr (kSplit) {
          Frag f;
          f.h = transposed<gt_f16x8>(p + off[i][0][0], p + off[i][0][1]);
          f.l = transposed<gt_f16x8>(p + off[i][1][0], p + off[i][1][1]);
          return f;
        } else {
          return transposed<Frag>(p + off[i][0][0], p + off[i][0][1]);
        }
      }
    }
  };
};

// Element (row i, column j) of acc[mi][ni][e] in lane l of wave (wm, wn):
//   i = wm * WM + 32 mi + 8 (e >> 2) + 4 (l >> 5) + (e & 3),   j = wn * WN + 32 ni + (l & 31)
//
// SINGLE: one LDS buffer and two barriers a block.  Half the LDS lets a third workgroup share the
// CU, which hides more than the second buffer does while k is short.
template <typename T, int BM_, GtOrder OA, int BN_, GtOrder OB, int WAVES_M_, bool SINGLE = false,
          bool RAW_A = false>
struct GtTile {
  static constexpr int BM = BM_, BN = BN_;
  static constexpr int WAVES_M = WAVES_M_, WAVES_N = 4 / WAVES_M;
  static constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N;
  static constexpr int MI = WM / 32, NI = WN / 32;
  typedef GtSide<T, BM, OA, RAW_A> SideA;
  typedef GtSide<T, BN, OB> SideB;
  static constexpr int BK = SideA::BK;
  static constexpr int kBuf = SideA::kBytes + SideB::kBytes;
  static constexpr int kLds = (SINGLE ? 1 : 2) * kBuf;
  // the last block apart, with only its occupied steps (the largest tiles' registers do not have
  // room for a second copy of the loop's body, and their k is long)
  static constexpr bool kTail = gt_occupancy(BM, BN) > 1 && !gt_is_split<T>;
  typedef typename GtFrag<T>::type Frag;
  static_assert(MI >= 1 && NI >= 1, "tile");

  // Order of one step: the next step's fragment reads, and the step's share of global loads or
  // LDS writes, are spread over its MFMAs, so the reads are in flight from the step's beginning;
  // left to itself the compiler reads a fragment just before its use and waits for it.
  template <bool LOADS, bool STORES>
  __device__ static void interleave() {
    constexpr int kMfmas = MI * NI * gt_mfmas<T>;
    constexpr int kReads = SideA::kReads * MI + SideB::kReads * NI;
    constexpr int kMoves = SideA::kLoads + SideB::kLoads;
    constexpr int kWrites = SideA::kWrites + SideB::kWrites;
    constexpr int G = kMfmas < 8 ? kMfmas : 8;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      // the reads in the first half of the step, LDS writes in the second
      constexpr int kR = STORES ? (2 * kReads + G - 1) / G : (kReads + G - 1) / G;
      if (!STORES || g < G / 2) __builtin_amdgcn_sched_group_barrier(0x100, kR, 0);
      if (LOADS) __builtin_amdgcn_sched_group_barrier(0x020, (kMoves + G - 1) / G, 0);
      if (STORES && g >= G / 2)
        __builtin_amdgcn_sched_group_barrier(0x200, (2 * kWrites + G - 1) / G, 0);
      __builtin_amdgcn_sched_group_barrier(0x008, kMfmas / G, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  }

  // acc += A[m0.., k0..k1) B[n0.., k0..k1)^T; k0 a multiple of a block.  Every thread of the
  // workgroup calls it; all LDS reads are done when it returns.
  __device__ static void run(const GtOperand& A, const GtOperand& B, int64_t m0, int64_t n0,
                             int64_t k0, int64_t k1, char* lds, gt_f32x16 (&acc)[MI][NI]) {
    if (k1 <= k0) return;
    const int lane = threadIdx.x & 63;
    typename SideA::Loader ga;
    typename SideB::Loader gb;
    ga.init(A, m0, k0, k1);
    gb.init(B, n0, k0, k1);
    typename SideA::template Reader<MI> ra;
    typename SideB::template Reader<NI> rb;
    ra.init(lane, wave_m() * WM);
    rb.init(lane, wave_n() * WN);
    const int nk = int((k1 - k0 + BK - 1) / BK);
    gt_u32x4 va[SideA::kLoads], vb[SideB::kLoads];
    Frag a[2][MI], b[2][NI];
    auto fetch = [&](const char* block, int ks, int f) {
#pragma unroll
      for (int i = 0; i < MI; ++i) a[f][i] = ra.read(block, i, ks, lane);
#pragma unroll
      for (int j = 0; j < NI; ++j) b[f][j] = rb.read(block + SideA::kBytes, j, ks, lane);
    };
    auto multiply = [&](int f) {
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = gt_mfma(a[f][i], b[f][j], acc[i][j]);
    };
    if constexpr (SINGLE) {
      ga.load(va);
      gb.load(vb);
      for (int it = 0; it < nk; ++it) {
        ga.store(lds, va);
        gb.store(lds + SideA::kBytes, vb);
        __syncthreads();
        ga.load(va);
        gb.load(vb);
        fetch(lds, 0, 0);
#pragma unroll
        for (int ks = 0; ks < gt_steps<T>; ++ks) {
          if (ks + 1 < gt_steps<T>) fetch(lds, ks + 1, (ks + 1) & 1);
          multiply(ks & 1);
          interleave<false, false>();
        }
        __syncthreads();
      }
      return;
    }
    ga.load(va);
    gb.load(vb);
    ga.store(lds, va);
    gb.store(lds + SideA::kBytes, vb);
    if constexpr (gt_is_split<T>) {
      ga.load(va);
      gb.load(vb);
    }
    __syncthreads();
    fetch(lds, 0, 0);
    if constexpr (gt_is_split<T>) {
      // two short steps a block: the loads are issued behind the barrier, a block ahead
      for (int it = 0; it < nk; ++it) {
        const char* cur = lds + (it & 1) * kBuf;
        char* nxt = lds + ((it + 1) & 1) * kBuf;
        fetch(cur, 1, 1);
        multiply(0);
        ga.store(nxt, va);
        gb.store(nxt + SideA::kBytes, vb);
        interleave<false, true>();
        __syncthreads();
        fetch(nxt, 0, 0);
        ga.load(va);
        gb.load(vb);
        multiply(1);
        interleave<true, false>();
      }
      __syncthreads();
      return;
    }
    // (the loads beyond the range give zeros that are staged unread: no branch)
    for (int it = 0; it < (kTail ? nk - 1 : nk); ++it) {
      const char* cur = lds + (it & 1) * kBuf;
      char* nxt = lds + ((it + 1) & 1) * kBuf;
      ga.load(va);
      gb.load(vb);
      fetch(cur, 1, 1);
      multiply(0);
      interleave<true, false>();
      fetch(cur, 2, 0);
      multiply(1);
      interleave<false, false>();
      fetch(cur, 3, 1);
      multiply(0);
      ga.store(nxt, va);
      gb.store(nxt + SideA::kBytes, vb);
      interleave<false, true>();
      // every wave has read this block and written its part of the next
      __syncthreads();
      fetch(nxt, 0, 0);
      multiply(1);
      interleave<false, false>();
    }
    if constexpr (!kTail) {
      __syncthreads();
      return;
    }
    // the last block: only the steps that hold any k
    const char* cur = lds + ((nk - 1) & 1) * kBuf;
    const int steps = int((k1 - k0 - int64_t(nk - 1) * BK + BK / 4 - 1) / (BK / 4));
    fetch(cur, 1, 1);
    multiply(0);
    interleave<false, false>();
    if (steps > 1) {
      fetch(cur, 2, 0);
      multiply(1);
      interleave<false, false>();
    }
    if (steps > 2) {
      fetch(cur, 3, 1);
      multiply(0);
      interleave<false, false>();
    }
    if (steps > 3) multiply(1);
    __syncthreads();
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
