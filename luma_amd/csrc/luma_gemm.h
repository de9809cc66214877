// Tiled matrix products on gfx950's matrix cores, for the kernels of
// luma_xent.hip: acc[m][n] += sum_k A(m, k) B(n, k) over one workgroup's tile,
// with either operand stored k-contiguous or m- (n-) contiguous.
//
// A workgroup's K loop runs in stages of 64 bytes of k per row (32 elements of
// 16 bits, 16 of float32), two to a pair.  Pairs go from memory into LDS without
// passing registers (16 bytes a lane), one under way while the other is
// multiplied, with one barrier a pair; each wavefront reads the fragments of the
// next stage into a second set of registers while the matrix unit works on the
// first.
// Fragments are 16 bytes a lane: lane l of a 16x16 tile holds row l % 16 and
// the 16 bytes of k at 16 * (l / 16), which is what v_mfma_f32_16x16x32 takes;
// four v_mfma_f32_16x16x4_f32 take its four floats (any order of k serves, as
// long as both operands have it).  An m-contiguous operand of 16 bits is read
// with ds_read_b64_tr_b16, which turns a 4 x 16 block on the way.
//
// The rows lie in LDS without padding (what the direct loads need), their
// 16-byte chunks permuted so that the lanes of one read meet different banks:
// k-contiguous rows by chunk ^ (row % 8), m-contiguous ones by whole 16-element
// blocks, block ^ (a function of k).
//
// Measured on the logits of 8,192 x 4,096 by 128,256 x 4,096 bfloat16 (8.6
// TFLOP; a library product of that size, its result written, 5.96 ms): 6.4 to
// 6.6 ms, 1.3 PFLOP/s, the matrix unit busy 69% of the time at the 1.65 GHz
// that the power limit leaves.  Before: a barrier for each stage and the
// compiler's order 7.2 ms (it sank the LDS reads below the matrix instructions,
// to the barrier); stages of 64-byte lines 6.7.  Not kept: 32 x 32 x 16
// instructions 7.2; wavefronts of 128 x 96 8.9; of 128 x 128 (accumulators moved
// and spilled) 25; workgroups that run on from tile to tile 7.1 (no gain at
// h = 768 either).
//
// Loads go through buffer descriptors that end where the operand ends: rows
// past the end read as zeros, and so does k past the end of a k-contiguous row
// (its lanes are given an offset past the end).
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/luma.h"

namespace luma {
namespace gemm {

typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) char lds_char;

constexpr int kRow = 64;       // bytes of k per stage and row
constexpr int kStages = 4;     // in LDS: two pairs

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

// A tile's shape: WM x WN wavefronts of TM x TN blocks of 16 x 16.
template <int TM_, int TN_, int WM_, int WN_>
struct Shape {
  static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_;
  static constexpr int BM = 16 * TM * WM, BN = 16 * TN * WN;
  static constexpr int kThreads = 64 * WM * WN;
};

// A wavefront's accumulators: TM x TN blocks of 16 x 16 (instructions of 32 x 32
// took 7% longer here).  A block is a quad per lane: four consecutive rows of
// one column.
template <int DT, typename S>
struct Acc {
  v4f t[S::TM][S::TN];

  __device__ __forceinline__ Acc() { clear(); }
  // Whether any of this lane's sums is a NaN.
  __device__ __forceinline__ bool nan() const {
    bool any = false;
#pragma unroll
    for (int i = 0; i < S::TM; ++i)
#pragma unroll
      for (int j = 0; j < S::TN; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) any |= t[i][j][r] != t[i][j][r];
    return any;
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < S::TM; ++i)
#pragma unroll
      for (int j = 0; j < S::TN; ++j) t[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
  }
  __device__ __forceinline__ void mma_bf16(int i, int j, const v4u &a, const v4u &b) {
    t[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
        __builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), t[i][j], 0, 0, 0);
  }
  __device__ __forceinline__ void mma(int i, int j, const v4u &a, const v4u &b) {
    if constexpr (DT == LUMA_GRAD_BF16) {
      mma_bf16(i, j, a, b);
    } else if constexpr (DT == LUMA_GRAD_F16) {
      t[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
          __builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), t[i][j], 0, 0, 0);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        t[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[k]),
                                                       __uint_as_float(b[k]), t[i][j], 0, 0, 0);
    }
  }
};

// The row of a pair of blocks of 16 that row `r` of block `i` of them takes, so
// that a lane's two quads are eight consecutive rows (kPaired), or 16 i + r.
constexpr int kPlain = 0, kPaired = 1;
template <int ORDER>
__device__ __forceinline__ constexpr int row_of(int i, int r) {
  return ORDER == kPaired ? 8 * (r >> 2) + 4 * i + (r & 3) : 16 * i + r;
}

// The block of a kAlongM row in whose place a block's elements lie: block ^ this.
// (The lanes of one read have k = j, 4 + j, 8 + j, 12 + j; of 16 bits 8 g .. 8 g + 3,
// one block of each or, kPaired, half of two.)
template <int DT, int ORDER>
__device__ __forceinline__ int turn(int k) {
  if (DT == LUMA_GRAD_F32) return (k >> 2) & 3;
  return ((k & 3) | ((k >> 1) & 4)) << (ORDER == kPaired ? 1 : 0);
}

// One operand's pairs of stages: ROWS of m (or n) by 128 bytes of k.  In LDS, a
// kAlongK pair is ROWS lines of 128 bytes (a whole cache line of the operand: its
// two stages are its halves), a kAlongM pair a line of ROWS elements for each k.
template <int DT, int ALONG, int ORDER, int ROWS, int THREADS>
struct Tile {
  static constexpr int kBytes = 2 * ROWS * kRow;                // of a pair
  static constexpr int kWaves = THREADS / 64;
  // 1 KB loads of a wavefront; with more wavefronts than loads some load the same bytes twice
  static constexpr int kTotal = kBytes / 1024;
  static constexpr int kLoads = (kTotal + kWaves - 1) / kWaves;
  static_assert(kBytes % 1024 == 0 && (kTotal % kWaves == 0 || kTotal < kWaves), "tile size");
  static constexpr int kLine = ROWS * kSize<DT>;                // bytes of a kAlongM line
  static constexpr int kBlock = 16 * kSize<DT>;                 // bytes of 16 elements
  static constexpr int kTurn = kLine / kBlock - 1;              // mask of block numbers

  const char *base;      // of the next pair of stages to be loaded
  int64_t left;          // bytes from base to the operand's end
  int64_t step;          // bytes from pair to pair
  int past;              // kAlongK: < 0 where this lane's chunk is past the row's end
  int at_lds[kLoads];
  uint32_t voff[kLoads];

  __device__ __forceinline__ void init(const Operand &o, int64_t m0, int64_t k0) {
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int lane = threadIdx.x & 63;
    const int64_t end = (o.rows - 1) * o.ld + o.row_bytes;
    const int64_t at = ALONG == kAlongK ? m0 * o.ld + k0 * kSize<DT> : k0 * o.ld + m0 * kSize<DT>;
    base = o.p + at;
    left = end - at;
    step = 2 * (ALONG == kAlongK ? kRow : kStep<DT> * o.ld);
#pragma unroll
    for (int q = 0; q < kLoads; ++q) {
      at_lds[q] = ((wave * kLoads + q) % kTotal) * 1024;
      const int at = at_lds[q] + lane * 16;
      if (ALONG == kAlongK) {
        // (line r % 8 is the same for all of a lane's loads, and so is the chunk)
        const int line = at / (2 * kRow), chunk = (at % (2 * kRow) / 16 ^ (line & 7)) * 16;
        const int row = line / 32 * 32 + row_of<ORDER>(line / 16 % 2, line % 16);
        voff[q] = (uint32_t)(row * o.ld) + chunk;
        const int64_t kl = o.row_bytes - k0 * kSize<DT>;
        past = (int)(kl < 0x40000000 ? kl : 0x40000000) - 1 - chunk;
      } else {
        const int k = at / kLine, in = at % kLine;
        const int block = (in / kBlock) ^ (turn<DT, ORDER>(k) & kTurn);
        voff[q] = (uint32_t)(k * o.ld) + block * kBlock + in % kBlock;
      }
    }
  }

  // Sends the next pair of stages on its way into s.  ONCE: nothing else reads
  // these bytes (non-temporal).
  template <bool ONCE>
  __device__ __forceinline__ void load(char *s) {
    typedef __attribute__((address_space(3))) void lds_void;
    const int high = (int)(left >> 31);
    const int records = high == 0 ? (int)left : high < 0 ? 0 : 0x7FFFFFFF;
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, records, 0x00020000);
    // (an offset past any end where k is)
    const uint32_t none = ALONG == kAlongK ? past & 0x80000000u : 0u;
#pragma unroll
    for (int q = 0; q < kLoads; ++q)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void *)(s + at_lds[q]), 16,
                                               voff[q] | none, 0, 0, ONCE ? 2 : 0);
    base += step;
    left -= step;
    if (ALONG == kAlongK) past -= 2 * kRow;
  }

  // Where this lane's part of the fragments of a run of blocks lies, the run
  // starting at block `first` and its length a power of two that divides it.
  static __device__ __forceinline__ int where(int first) {
    const int lane = threadIdx.x & 63;
    if (ALONG == kAlongK) {
      const int line = first * 16 + (lane & 15);
      return line * 2 * kRow + (((lane >> 4) ^ (line & 7)) * 16);
    }
    if (DT == LUMA_GRAD_F32)
      return (lane >> 4) * 4 * kLine + ((first ^ ((lane >> 4) & kTurn)) * kBlock) + (lane & 15) * 4;
    const int k = 8 * (lane >> 4) + ((lane & 15) >> 2), q = lane & 3;
    const int block = ORDER == kPaired ? first + (q >> 1) : first;
    return k * kLine + ((block ^ (turn<DT, ORDER>(k) & kTurn)) * kBlock) +
           (ORDER == kPaired ? (q & 1) * 16 : q * 8);
  }

  // Fragment of block first + i in the pair's stage h.
  static __device__ __forceinline__ v4u read(const char *s, int h, int where, int i) {
    if constexpr (ALONG == kAlongK) {
      return *(const v4u *)(s + (where ^ (h * kRow)) + i * 16 * 2 * kRow);
    } else if constexpr (DT == LUMA_GRAD_F32) {
      const char *p = s + h * kStep<DT> * kLine + (where ^ (i * kBlock));
      v4u f;
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = *(const uint32_t *)(p + j * kLine);
      return f;
    } else {
      const char *p = s + h * kStep<DT> * kLine +
                      (ORDER == kPaired ? (where ^ (i / 2 * 2 * kBlock)) + i % 2 * 8
                                        : where ^ (i * kBlock));
      typedef __attribute__((address_space(3))) v4s lds_v4s;
      const v2u lo = __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)p));
      const v2u hi = __builtin_bit_cast(
          v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)(p + 4 * kLine)));
      return v4u{lo[0], lo[1], hi[0], hi[1]};
    }
  }
};

// Outstanding direct loads at most N, this wavefront's LDS reads done, then all
// wavefronts here.
template <int N>
__device__ __forceinline__ void wait_and_meet() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// The order of one half of a pair of stages: a fragment's read after every few
// matrix instructions, and LOADS loads into LDS after the first ones.
template <int MMAS, int READS, int LOADS>
__device__ __forceinline__ void spread() {
#pragma unroll
  for (int q = 0; q < LOADS; ++q) {
    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x20, 1, 0);
  }
  constexpr int kEach = (MMAS - LOADS) / READS > 0 ? (MMAS - LOADS) / READS : 1;
#pragma unroll
  for (int q = 0; q < READS; ++q) {
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x8, kEach, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x8, MMAS, 0);
  __builtin_amdgcn_sched_barrier(0);
}

// Float32 as a sum of three bfloat16, x = hi + mid + lo with nothing left over
// (each takes the next 8 of its 24 bits; a lo below 2^-126 may be lost).
struct Split {
  v4u hi, mid, lo;
  // of the eight values of two fragments
  __device__ __forceinline__ Split(const v4u &a, const v4u &b) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const v4u &x = e < 2 ? a : b;
      v2f f = {__uint_as_float(x[2 * (e & 1)]), __uint_as_float(x[2 * (e & 1) + 1])};
      hi[e] = take(f);
      mid[e] = take(f);
      lo[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f, v2bf));
    }
  }
  static __device__ __forceinline__ uint32_t take(v2f &f) {
    const uint32_t b = __builtin_bit_cast(uint32_t, __builtin_convertvector(f, v2bf));
    f[0] -= __uint_as_float(b << 16);
    f[1] -= __uint_as_float(b & 0xFFFF0000u);
    return b;
  }
};

// acc (+)= the product over k0 <= k < k1 of this wavefront's blocks.
// k1 - k0 is rounded up to whole rounds of the ring: past k1 operands must
// read as zeros (past the operands' end), unless k1 - k0 is a multiple of
// kStages * kStep.
template <int DT, int AA, int AB, int ORDER, typename S, bool ONCE>
__device__ __forceinline__ void product(const Operand &a, const Operand &b, int64_t m0, int64_t n0,
                                        int64_t k0, int64_t k1, Acc<DT, S> &acc) {
#ifdef __HIP_DEVICE_COMPILE__   // (the host's compiler has no use for it)
  typedef Tile<DT, AA, ORDER, S::BM, S::kThreads> A;
  typedef Tile<DT, AB, kPlain, S::BN, S::kThreads> B;
  constexpr int kLoads = A::kLoads + B::kLoads;
  constexpr int kMmas = S::TM * S::TN * (DT == LUMA_GRAD_F32 ? 4 : 1), kReads = S::TM + S::TN;
  // (a variable for each pair: the compiler then knows that a pair's reads do not
  // wait for another's loads)
  __shared__ __align__(1024) char a0[A::kBytes], a1[A::kBytes];
  __shared__ __align__(1024) char b0[B::kBytes], b1[B::kBytes];
  A ta;
  B tb;
  const int wave = threadIdx.x >> 6;
  const int wa = A::where((wave / S::WN) * S::TM);
  const int wb = B::where((wave % S::WN) * S::TN);
  auto fill = [&](char *sa, char *sb) {
    ta.template load<ONCE>(sa);
    tb.template load<false>(sb);
  };
  const int rounds = (int)((k1 - k0 + kStages * kStep<DT> - 1) / (kStages * kStep<DT>));

  if constexpr (DT == LUMA_GRAD_F32 && S::TM * S::TN >= 16) {
    // Six products of bfloat16 parts for one of float32 (all but mid lo, lo mid
    // and lo lo, together about 2^-24 of the product): the matrix unit takes
    // bfloat16 16 times as fast as float32.  A pair of stages (32 of k) makes
    // one bfloat16 fragment.  (Smaller tiles take the float32 instruction: their
    // time is latency, which taking the parts adds to.)
    auto parts = [&](const char *xa, const char *xb) {
      v4u hi[S::TN], mid[S::TN], lo[S::TN];
#pragma unroll
      for (int j = 0; j < S::TN; ++j) {
        const Split y(B::read(xb, 0, wb, j), B::read(xb, 1, wb, j));
        hi[j] = y.hi, mid[j] = y.mid, lo[j] = y.lo;
      }
      // (while block i is multiplied, the parts of the next are taken and the one
      // behind is read; the fences keep the compiler from doing all at once,
      // for which there are no registers)
      Split x(A::read(xa, 0, wa, 0), A::read(xa, 1, wa, 0));
      v4u f0 = A::read(xa, 0, wa, 1), f1 = A::read(xa, 1, wa, 1);
#pragma unroll
      for (int i = 0; i < S::TM; ++i) {
        __builtin_amdgcn_sched_barrier(0);
        const Split now = x;
        if (i + 1 < S::TM) x = Split(f0, f1);
        if (i + 2 < S::TM) f0 = A::read(xa, 0, wa, i + 2), f1 = A::read(xa, 1, wa, i + 2);
        // (the small ones first)
#pragma unroll
        for (int j = 0; j < S::TN; ++j) acc.mma_bf16(i, j, now.lo, hi[j]);
#pragma unroll
        for (int j = 0; j < S::TN; ++j) acc.mma_bf16(i, j, now.hi, lo[j]);
#pragma unroll
        for (int j = 0; j < S::TN; ++j) acc.mma_bf16(i, j, now.mid, mid[j]);
#pragma unroll
        for (int j = 0; j < S::TN; ++j) acc.mma_bf16(i, j, now.mid, hi[j]);
#pragma unroll
        for (int j = 0; j < S::TN; ++j) acc.mma_bf16(i, j, now.hi, mid[j]);
#pragma unroll
        for (int j = 0; j < S::TN; ++j) acc.mma_bf16(i, j, now.hi, hi[j]);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    auto run = [&](auto pair) {
      ta.init(a, m0, k0);
      tb.init(b, n0, k0);
      fill(a0, b0);
      for (int r = 0; r < rounds; ++r) {
        wait_and_meet<0>();
        fill(a1, b1);
        pair(a0, b0);
        wait_and_meet<0>();
        fill(a0, b0);
        pair(a1, b1);
      }
      wait_and_meet<0>();
    };
    run(parts);
    // Of an infinity (or a value that rounds to one) the parts leave NaN: a sum
    // that is NaN is formed again by the float32 instruction, a row of blocks
    // at a time.
    if (__syncthreads_or(acc.nan())) {
#pragma unroll
      for (int i = 0; i < S::TM; ++i) {
        Acc<DT, Shape<1, S::TN, S::WM, S::WN>> again;
        run([&](const char *xa, const char *xb) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < S::TN; ++j)
              again.mma(0, j, A::read(xa, h, wa, i), B::read(xb, h, wb, j));
        });
#pragma unroll
        for (int j = 0; j < S::TN; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (acc.t[i][j][r] != acc.t[i][j][r]) acc.t[i][j][r] = again.t[0][j][r];
      }
    }
  } else {
    ta.init(a, m0, k0);
    tb.init(b, n0, k0);
    v4u fa[2][S::TM], fb[2][S::TN];

    auto fetch = [&](const char *sa, const char *sb, int h) {
#pragma unroll
      for (int j = 0; j < S::TN; ++j) fb[h][j] = B::read(sb, h, wb, j);
#pragma unroll
      for (int i = 0; i < S::TM; ++i) fa[h][i] = A::read(sa, h, wa, i);
    };
    auto multiply = [&](int h) {
#pragma unroll
      for (int i = 0; i < S::TM; ++i)
#pragma unroll
        for (int j = 0; j < S::TN; ++j) acc.mma(i, j, fa[h][i], fb[h][j]);
    };

    // One pair of stages, x; the loads under way fill the next one, y.
    auto pair = [&](char *xa, char *xb, char *ya, char *yb) {
      fetch(xa, xb, 1);
      multiply(0);
      spread<kMmas, kReads, 0>();
      wait_and_meet<0>();
      fill(xa, xb);
      fetch(ya, yb, 0);
      multiply(1);
      spread<kMmas, kReads, kLoads>();
    };

    fill(a0, b0);
    fill(a1, b1);
    wait_and_meet<kLoads>();
    fetch(a0, b0, 0);
    for (int r = 0; r < rounds; ++r) {
      pair(a0, b0, a1, b1);
      pair(a1, b1, a0, b0);
    }
  }
  // (nothing of the ring is in flight when the workgroup goes on or ends)
  wait_and_meet<0>();
#endif
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
