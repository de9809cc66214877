// Tiled matrix products on gfx950's matrix cores, for the kernels of
// luma_xent.hip: acc[m][n] += sum_k A(m, k) B(n, k) over one workgroup's tile,
// with either operand stored k-contiguous or m- (n-) contiguous.
//
// A workgroup's K loop runs in stages of 64 bytes of k per row (32 elements of
// 16 bits, 16 of float32).  Stages go from memory into LDS without passing
// registers (16 bytes a lane), kStages of them in a ring, two in flight while
// one is multiplied; each wavefront reads the fragments of the stage behind
// into a second set of registers while the matrix unit works on the first.
// Fragments are 16 bytes a lane: lane l of a 16x16 tile holds row l % 16 and
// the 16 bytes of k at 16 * (l / 16), which is what v_mfma_f32_16x16x32 takes;
// four v_mfma_f32_16x16x4_f32 take its four floats (any order of k serves, as
// long as both operands have it).  An m-contiguous operand of 16 bits is read
// with ds_read_b64_tr_b16, which turns a 4 x 16 block on the way.
//
// The rows of a stage lie in LDS without padding (what the direct loads need),
// their 16-byte chunks permuted so that the lanes of one read meet different
// banks: k-contiguous rows of 64 bytes by chunk ^ (row / 2 % 4), m-contiguous
// ones by whole 16-element blocks, block ^ (a function of k).
//
// Loads go through buffer descriptors that end where the operand ends: rows
// past the end read as zeros, and so does k past the end of a k-contiguous row
// (its lanes are given an offset past the end).
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/luma.h"

namespace luma {
namespace gemm {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) char lds_char;

constexpr int kRow = 64;       // bytes of k per stage and row
constexpr int kStages = 4;

// Which direction of an operand is contiguous.
constexpr int kAlongK = 0, kAlongM = 1;

template <int DT>
constexpr int kSize = DT == LUMA_GRAD_F32 ? 4 : 2;      // bytes of an element
template <int DT>
constexpr int kStep = kRow / kSize<DT>;                  // elements of k per stage

// One operand: `rows` rows of `row_bytes` used bytes, `ld` bytes apart; the
// rows are m (kAlongK) or k (kAlongM).  p and ld are multiples of 16 bytes,
// and so is row_bytes of a kAlongK operand.
struct Operand {
  const char *p;
  int64_t ld, rows, row_bytes;
};

template <int DT>
__device__ __forceinline__ v4f mma(const v4u &a, const v4u &b, v4f c) {
  if constexpr (DT == LUMA_GRAD_BF16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a),
                                                   __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  } else if constexpr (DT == LUMA_GRAD_F16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a),
                                                  __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0,
                                               0, 0);
    return c;
  }
}

// The block of a kAlongM row in whose place a block's elements lie: block ^ this.
template <int DT>
__device__ __forceinline__ int turn(int k) {
  if (DT == LUMA_GRAD_F32) return (k >> 2) & 3;    // lanes of one read: k = j, 4 + j, 8 + j, 12 + j
  return (k & 3) | ((k >> 1) & 4);                 // k = 8 g .. 8 g + 3
}

// One operand's stages: ROWS of m (or n) by 64 bytes of k.
template <int DT, int ALONG, int ROWS, int THREADS>
struct Tile {
  static constexpr int kBytes = ROWS * kRow;
  static constexpr int kWaves = THREADS / 64;
  // 1 KB loads of a wavefront; with more wavefronts than loads some load the same bytes twice
  static constexpr int kTotal = kBytes / 1024;
  static constexpr int kLoads = (kTotal + kWaves - 1) / kWaves;
  static_assert(kBytes % 1024 == 0 && (kTotal % kWaves == 0 || kTotal < kWaves), "tile size");
  static constexpr int kLine = ROWS * kSize<DT>;                // bytes of a kAlongM row
  static constexpr int kBlock = 16 * kSize<DT>;                 // bytes of 16 elements
  static constexpr int kTurn = kLine / kBlock - 1;              // mask of block numbers

  const char *base;      // of the next stage to be loaded
  int64_t left;          // bytes from base to the operand's end
  int64_t step;          // bytes from stage to stage
  int k_left;            // kAlongK: bytes of k from base to the row's end
  uint32_t voff[kLoads];
  uint32_t chunk[kLoads];

  __device__ __forceinline__ void init(const Operand &o, int64_t m0, int64_t k0) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t end = (o.rows - 1) * o.ld + o.row_bytes;
    const int64_t at = ALONG == kAlongK ? m0 * o.ld + k0 * kSize<DT> : k0 * o.ld + m0 * kSize<DT>;
    base = o.p + at;
    left = end - at;
    step = ALONG == kAlongK ? kRow : kStep<DT> * o.ld;
    const int64_t kl = o.row_bytes - k0 * kSize<DT>;
    k_left = ALONG == kAlongK ? (int)(kl < 0x40000000 ? kl : 0x40000000) : 0;
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
      const int at_lds = ((wave * kLoads + q) % kTotal) * 1024 + lane * 16;
      if (ALONG == kAlongK) {
        const int row = at_lds / kRow, pos = (at_lds % kRow) / 16;
        chunk[q] = (pos ^ ((row >> 1) & 3)) * 16;
        voff[q] = (uint32_t)(row * o.ld) + chunk[q];
      } else {
        const int k = at_lds / kLine, in = at_lds % kLine;
        const int block = (in / kBlock) ^ (turn<DT>(k) & kTurn);
        chunk[q] = 0;
        voff[q] = (uint32_t)(k * o.ld) + block * kBlock + in % kBlock;
      }
    }
  }

  // Sends the next stage on its way into s.
  __device__ __forceinline__ void load(char *s) {
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int records = left <= 0 ? 0 : left < 0x7FFFFFFF ? (int)left : 0x7FFFFFFF;
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, records, 0x00020000);
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
      uint32_t v = voff[q];
      if (ALONG == kAlongK && k_left < kRow && (int)chunk[q] >= k_left) v = 0xFFFFFFF0u;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rsrc, (__attribute__((address_space(3))) void *)(s + ((wave * kLoads + q) % kTotal) * 1024),
          16, v, 0, 0, 0);
    }
    base += step;
    left -= step;
    if (ALONG == kAlongK) k_left -= kRow;
  }

  // Where this lane's part of the fragments of COUNT blocks from block `first`
  // (a multiple of COUNT) lies.
  static __device__ __forceinline__ int where(int first) {
    const int lane = threadIdx.x & 63;
    if (ALONG == kAlongK) {
      const int row = first * 16 + (lane & 15);
      return row * kRow + (((lane >> 4) ^ ((row >> 1) & 3)) * 16);
    }
    if (DT == LUMA_GRAD_F32)
      return (lane >> 4) * 4 * kLine + ((first ^ ((lane >> 4) & kTurn)) * kBlock) + (lane & 15) * 4;
    const int k = 8 * (lane >> 4) + ((lane & 15) >> 2);
    return k * kLine + ((first ^ (turn<DT>(k) & kTurn)) * kBlock) + (lane & 3) * 8;
  }

  // Fragment of block first + i.
  static __device__ __forceinline__ v4u read(const char *s, int where, int i) {
    if constexpr (ALONG == kAlongK) {
      return *(const v4u *)(s + where + i * 16 * kRow);
    } else if constexpr (DT == LUMA_GRAD_F32) {
      const char *p = s + (where ^ (i * kBlock));
      v4u f;
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = *(const uint32_t *)(p + j * kLine);
      return f;
    } else {
      const char *p = s + (where ^ (i * kBlock));
      typedef __attribute__((address_space(3))) v4s lds_v4s;
      const v2u lo = __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)p));
      const v2u hi = __builtin_bit_cast(
          v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)(p + 4 * kLine)));
      return v4u{lo[0], lo[1], hi[0], hi[1]};
    }
  }
};

// A tile's shape: WM x WN wavefronts of TM x TN 16x16 blocks.
template <int TM_, int TN_, int WM_, int WN_>
struct Shape {
  static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_;
  static constexpr int BM = 16 * TM * WM, BN = 16 * TN * WN;
  static constexpr int kThreads = 64 * WM * WN;
};

// Outstanding direct loads at most N, this wavefront's LDS reads done, then all
// wavefronts here.
template <int N>
__device__ __forceinline__ void wait_and_meet() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// acc[i][j] (+)= the product over k0 <= k < k1 of this wavefront's blocks.
// k1 - k0 is rounded up to whole rounds of the ring: past k1 operands must
// read as zeros (past the operands' end), unless k1 - k0 is a multiple of
// kStages * kStep.
template <int DT, int AA, int AB, typename S>
__device__ __forceinline__ void product(const Operand &a, const Operand &b, int64_t m0, int64_t n0,
                                        int64_t k0, int64_t k1, v4f (&acc)[S::TM][S::TN]) {
  typedef Tile<DT, AA, S::BM, S::kThreads> A;
  typedef Tile<DT, AB, S::BN, S::kThreads> B;
  constexpr int kLoads = A::kLoads + B::kLoads;
  // (a variable for each stage: the compiler then knows that a stage's reads
  // do not wait for another's loads)
  __shared__ __align__(1024) char a0[A::kBytes], a1[A::kBytes], a2[A::kBytes], a3[A::kBytes];
  __shared__ __align__(1024) char b0[B::kBytes], b1[B::kBytes], b2[B::kBytes], b3[B::kBytes];
  A ta;
  B tb;
  ta.init(a, m0, k0);
  tb.init(b, n0, k0);
  const int wave = threadIdx.x >> 6;
  const int wa = A::where((wave / S::WN) * S::TM), wb = B::where((wave % S::WN) * S::TN);
  v4u fa[2][S::TM], fb[2][S::TN];

  auto fill = [&](char *sa, char *sb) {
    ta.load(sa);
    tb.load(sb);
  };
  auto fetch = [&](const char *sa, const char *sb, v4u (&xa)[S::TM], v4u (&xb)[S::TN]) {
#pragma unroll
    for (int j = 0; j < S::TN; ++j) xb[j] = B::read(sb, wb, j);
#pragma unroll
    for (int i = 0; i < S::TM; ++i) xa[i] = A::read(sa, wa, i);
  };
  auto multiply = [&](const v4u (&xa)[S::TM], const v4u (&xb)[S::TN]) {
#pragma unroll
    for (int i = 0; i < S::TM; ++i)
#pragma unroll
      for (int j = 0; j < S::TN; ++j) acc[i][j] = mma<DT>(xa[i], xb[j], acc[i][j]);
  };

  fill(a0, b0);
  fill(a1, b1);
  fill(a2, b2);
  wait_and_meet<2 * kLoads>();
  fetch(a0, b0, fa[0], fb[0]);
  const int rounds = (int)((k1 - k0 + kStages * kStep<DT> - 1) / (kStages * kStep<DT>));
  for (int r = 0; r < rounds; ++r) {
    wait_and_meet<kLoads>();
    fill(a3, b3);
    fetch(a1, b1, fa[1], fb[1]);
    multiply(fa[0], fb[0]);
    wait_and_meet<kLoads>();
    fill(a0, b0);
    fetch(a2, b2, fa[0], fb[0]);
    multiply(fa[1], fb[1]);
    wait_and_meet<kLoads>();
    fill(a1, b1);
    fetch(a3, b3, fa[1], fb[1]);
    multiply(fa[0], fb[0]);
    wait_and_meet<kLoads>();
    fill(a2, b2);
    fetch(a0, b0, fa[0], fb[0]);
    multiply(fa[1], fb[1]);
  }
  // (nothing of the ring is in flight when the workgroup goes on or ends)
  wait_and_meet<0>();
}

// The tile of this workgroup: consecutive workgroups go to the eight XCDs in
// turn, so each XCD is given one run of tiles, and runs of kGroup tiles along m
// with every n, so that the tiles at work on an XCD at a time share panels in
// its L2.
constexpr int kXcds = 8, kGroup = 8;

__device__ __forceinline__ void tile_of(int tiles_m, int tiles_n, int splits, int &m, int &n,
                                        int &split) {
  const int total = tiles_m * tiles_n * splits;
  const int xcd = blockIdx.x % kXcds, i = blockIdx.x / kXcds;
  const int each = total / kXcds, more = total % kXcds;
  int t = xcd * each + min(xcd, more) + i;
  split = t / (tiles_m * tiles_n);
  t -= split * tiles_m * tiles_n;
  const int group = t / (kGroup * tiles_n), first = group * kGroup;
  const int size = min(kGroup, tiles_m - first);
  t -= group * kGroup * tiles_n;
  m = first + t % size;
  n = t / size;
}

}  // namespace gemm
}  // namespace luma
