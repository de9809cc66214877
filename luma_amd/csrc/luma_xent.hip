// Cross entropy over a vocabulary without the logits (include/luma.h,
// luma_xent_forward / luma_xent_backward).
//
// Forward:   logits tile by tile (W X^T, vocabulary along the accumulators'
//            rows, so that a lane holds many words of one token), and from each
//            tile, in registers, every token's largest logit, its sum of
//            exp(l - largest), and the target's logit; then a join over the
//            vocabulary's tiles.
// Backward:  for each piece of the vocabulary: the logits again, from them
//            D = r_i (exp(l - top_i) / sum_i - [target]) in the operands' type; then
//            d_weight's rows of the piece = D^T X and d_hidden += D W.
//            r_i is the token's gradient times a power of two that brings the
//            largest to about 2^kTop (float16's range is short); the products
//            are scaled back in float32, which is exact.  One gradient for all
//            tokens (a mean, a sum) stays out of D altogether.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include "../../include/luma.h"
#include "luma_error.h"
#include "luma_gemm.h"

namespace luma {
namespace {

using namespace gemm;

constexpr float kLog2e = 1.44269504088896340736f;

template <int DT>
struct Elem;
template <>
struct Elem<LUMA_GRAD_F32> {
  typedef float type;
  static __device__ __forceinline__ float round(float f) { return f; }
};
template <>
struct Elem<LUMA_GRAD_BF16> {
  typedef __bf16 type;
  static __device__ __forceinline__ __bf16 round(float f) { return (__bf16)f; }
};
template <>
struct Elem<LUMA_GRAD_F16> {
  typedef _Float16 type;
  static __device__ __forceinline__ _Float16 round(float f) { return (_Float16)f; }
};

template <int DT>
using Four = typename Elem<DT>::type __attribute__((ext_vector_type(4), aligned(2)));

// (D is the workspace's: its rows are whole tiles of words, 512 bytes aligned)
template <int DT>
using Eight = typename Elem<DT>::type __attribute__((ext_vector_type(8), aligned(16)));

// Stores four consecutive elements of a row, those before `end`.
template <int DT>
__device__ __forceinline__ void store4(typename Elem<DT>::type *p, int64_t at, int64_t end, v4f f) {
  if (at + 4 <= end) {
    Four<DT> o;
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = Elem<DT>::round(f[r]);
    if constexpr (DT == LUMA_GRAD_F32) {
      typedef float v4fu __attribute__((ext_vector_type(4), aligned(4)));
      *(v4fu *)(p + at) = v4fu{o[0], o[1], o[2], o[3]};
    } else {
      *(Four<DT> *)(p + at) = o;
    }
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (at + r < end) p[at + r] = Elem<DT>::round(f[r]);
  }
}

struct Grid {
  int tiles_m, tiles_n, splits;
};

// Few tokens: one tile holds them all, and the weight is read once.
template <typename S>
constexpr bool kFew = S::BM > S::BN;

// This lane's first row and column of its wavefront's accumulators; its quad i
// of column j is rows m + row(i) .. + 3 and column n + 16 j.
template <typename S, int ORDER>
struct Place {
  int64_t m, n;
  __device__ __forceinline__ Place(int tm, int tn) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    m = (int64_t)tm * S::BM + (wave / S::WN) * S::TM * 16 + row_of<ORDER>(0, lane >> 4 << 2);
    n = (int64_t)tn * S::BN + (wave % S::WN) * S::TN * 16 + (lane & 15);
  }
  static __device__ __forceinline__ constexpr int row(int i) {
    return i / 2 * 32 + row_of<ORDER>(i & 1, 0);
  }
};

// -- forward --------------------------------------------------------------------

// (largest, sum) of two sets of words together.
__device__ __forceinline__ float2 join(float2 a, float2 b) {
  const float top = fmaxf(a.x, b.x);
  if (top == -__builtin_inff()) return make_float2(top, a.y + b.y);
  return make_float2(top, a.y * __builtin_amdgcn_exp2f((a.x - top) * kLog2e) +
                              b.y * __builtin_amdgcn_exp2f((b.x - top) * kLog2e));
}

// Bound by the matrix cores (2 n h v operations; few tokens: by reading the
// weight once).  The vocabulary lies along the accumulators' rows, so that a
// lane holds 32 words of a token and the largest and the sum are formed in
// registers, with two steps across lanes and one across wavefronts.  8,192
// tokens: h = 4096, v = 128256 6.5 ms (1.3 PFLOP/s); h = 768, v = 50257 0.63 to
// 0.72 ms (a library product of that size, its result written, 0.58: a third of
// a tile's time is its first loads and its exponentials).  One token of the
// former: 175 us (6.0 TB/s).
//
// Every token's (largest logit, sum of exp(l - largest)) over each tile's words:
// part[tile of words from v0][token]; picked[token] = the target's logit.
template <int DT, typename S>
__global__ __launch_bounds__(S::kThreads) void logits_kernel(Operand w, Operand x, int64_t v0,
                                                             int64_t v, int64_t n, int64_t h,
                                                             const int64_t *target, Grid g,
                                                             float2 *part, float *picked) {
  int tm, tn, split;
  tile_of(g.tiles_m, g.tiles_n, 1, tm, tn, split);
  Acc<DT, S> acc;
  product<DT, kAlongK, kAlongK, kPlain, S, kFew<S>>(w, x, v0 + (int64_t)tm * S::BM,
                                                    (int64_t)tn * S::BN, 0, h, acc);
  typedef Place<S, kPlain> P;
  P at(tm, tn);
  at.m += v0;
  const bool whole = v0 + (int64_t)(tm + 1) * S::BM <= v;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / S::WN, wn = wave % S::WN;
  __shared__ float2 records[S::WM][S::BN];
#pragma unroll
  for (int j = 0; j < S::TN; ++j) {
    const int64_t token = at.n + 16 * j;
    const int64_t t = token < n ? target[token] : -1;
    // the target's word from this lane's first; < 0 for none here
    const int64_t far = t < v ? t - at.m : -1;
    const int d = far >= 0 && far < 16 * S::TM ? (int)far : -1;
    if (__ballot(d >= 0)) {
      float mine = 0.0f;
      bool found = false;
#pragma unroll
      for (int q = 0; q < S::TM; ++q)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (d == P::row(q) + r) {
            mine = acc.t[q][j][r];
            found = true;
          }
      if (found) picked[token] = mine;
    }
    float top = -__builtin_inff();
#pragma unroll
    for (int q = 0; q < S::TM; ++q)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (whole || at.m + P::row(q) + r < v) top = fmaxf(top, acc.t[q][j][r]);
#pragma unroll
    for (int o = 16; o < 64; o *= 2) top = fmaxf(top, __shfl_xor(top, o));
    // (all -inf: their exponentials are 0 and not NaN)
    const float base = top == -__builtin_inff() ? 0.0f : top;
    float sum = 0.0f;
#pragma unroll
    for (int q = 0; q < S::TM; ++q)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float e = __builtin_amdgcn_exp2f((acc.t[q][j][r] - base) * kLog2e);
        if (whole || at.m + P::row(q) + r < v) sum += e;
      }
#pragma unroll
    for (int o = 16; o < 64; o *= 2) sum += __shfl_xor(sum, o);
    if (lane < 16)
      records[wm][wn * S::TN * 16 + 16 * j + lane] = make_float2(top, sum);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < S::BN; i += S::kThreads) {
    const int64_t token = (int64_t)tn * S::BN + i;
    float2 a = records[0][i];
#pragma unroll
    for (int k = 1; k < S::WM; ++k) a = join(a, records[k][i]);
    if (token < n) part[(int64_t)tm * n + token] = a;
  }
}

constexpr int kJoinThreads = 1024;

// Bound by latency for few tokens (one token, 1,002 records: 4.5 us, with 32
// threads to a token 10.5 us), by memory for many.
//
// Each token's largest logit, sum and loss from its `parts` records, TOKENS to a workgroup (the
// records of one shared out to 1024 / TOKENS threads); with a reduction, each
// workgroup's sums (in float64) of the losses and of the targets that count.
template <int TOKENS>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(const float2 *part, int parts,
                                                            const float *picked,
                                                            const int64_t *target, int64_t n,
                                                            int64_t v, int64_t ignore,
                                                            float *stats, float *loss,
                                                            double2 *sums) {
  constexpr int kSlices = kJoinThreads / TOKENS;
  __shared__ float2 lds[kSlices][TOKENS + 1];
  const int tok = threadIdx.x % TOKENS, slice = threadIdx.x / TOKENS;
  const int64_t token = (int64_t)blockIdx.x * TOKENS + tok;
  float2 a = make_float2(-__builtin_inff(), 0.0f);
  if (token < n) {
    // (kAhead records in flight: a token has hundreds, and the loads' latency
    // is what they take)
    constexpr int kAhead = 8;
    int p = slice;
    for (; p + (kAhead - 1) * kSlices < parts; p += kAhead * kSlices) {
      float2 b[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) b[k] = part[(int64_t)(p + k * kSlices) * n + token];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) a = join(a, b[k]);
    }
    for (; p < parts; p += kSlices) a = join(a, part[(int64_t)p * n + token]);
  }
  lds[slice][tok] = a;
  __syncthreads();
  for (int s = kSlices / 2; s > 0; s /= 2) {
    if (slice < s && slice + s < parts) lds[slice][tok] = a = join(a, lds[slice + s][tok]);
    __syncthreads();
  }
  if (threadIdx.x >= 64) return;      // (the rest is the first wavefront's)
  double value = 0.0, count = 0.0;
  if (slice == 0 && token < n) {
    const int64_t t = target[token];
    float l = 0.0f;
    if (t != ignore) {
      // (not lse - l: a small loss is the difference of nearly equal numbers)
      l = t >= 0 && t < v ? (a.x - picked[token]) + logf(a.y) : __builtin_nanf("");
      count = 1.0;
    }
    stats[token] = a.x;
    stats[n + token] = a.y;
    if (!sums) loss[token] = l;
    value = (double)l;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    value += __shfl_xor(value, o);
    count += __shfl_xor(count, o);
  }
  if (sums && threadIdx.x == 0) sums[blockIdx.x] = make_double2(value, count);
}

// The loss from the workgroups' sums.
__global__ __launch_bounds__(256) void reduce_kernel(const double2 *sums, int64_t count,
                                                     int reduction, float *stats_n, float *loss) {
  __shared__ double2 lds[4];
  double a = 0.0, b = 0.0;
  for (int64_t i = threadIdx.x; i < count; i += 256) {
    a += sums[i].x;
    b += sums[i].y;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    a += __shfl_xor(a, o);
    b += __shfl_xor(b, o);
  }
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = make_double2(a, b);
  __syncthreads();
  if (threadIdx.x != 0) return;
  a = lds[0].x + lds[1].x + lds[2].x + lds[3].x;
  b = lds[0].y + lds[1].y + lds[2].y + lds[3].y;
  *stats_n = (float)b;
  *loss = (float)(reduction == LUMA_XENT_MEAN ? a / b : a);
}

// -- backward -------------------------------------------------------------------

// The header of the tokens' factors: what the products are scaled back by.
struct Rows {
  float back;
  float pad[63];
};

// Each token's factor r_i: the gradient of its loss times a power of two that
// brings the largest to 2^(TOP - 1) .. 2^TOP; 0 for an ignored target, NaN for
// one outside the vocabulary.  With one gradient g for all tokens r_i is the
// power of two 2^(TOP - 1) alone and the products are scaled back by g over it: D is then
// p - [target] itself, whose target's entry is nearly -1 and rounds to little; of
// g (p - [target]) every token's would be off by the same up to 2^-9.
struct Factors {
  const float *grad;
  const int64_t *target;
  const float *stats;
  int64_t n, v, ignore;
  int reduction;
  Rows *head;       // rows_kernel's (LUMA_XENT_NONE)
  float *rows;

  // One gradient for all tokens.
  __device__ __forceinline__ float one() const {
    return reduction == LUMA_XENT_MEAN ? grad[0] / stats[2 * n] : grad[0];
  }
  __device__ __forceinline__ float factor(int64_t t, float g) const {
    return t == ignore ? 0.0f : t >= 0 && t < v ? g : __builtin_nanf("");
  }
  template <int TOP>
  __device__ __forceinline__ float row(int64_t i, int64_t t) const {
    if (reduction == LUMA_XENT_NONE) return rows[i];
    const float g = one();
    // (an infinity's or a NaN's tokens get it, the ignored ones 0)
    return factor(t, __builtin_isfinite(g) ? __builtin_ldexpf(0.5f, TOP) : g);
  }
  template <int TOP>
  __device__ __forceinline__ float back() const {
    if (reduction == LUMA_XENT_NONE) return head->back;
    const float g = one();
    return __builtin_isfinite(g) ? g * __builtin_ldexpf(2.0f, -TOP) : 1.0f;
  }
};

template <int DT>
constexpr int kTop = DT == LUMA_GRAD_F16 ? 15 : 0;

template <int TOP>
__global__ __launch_bounds__(1024) void rows_kernel(Factors f) {
  __shared__ float lds[16];
  float top = 0.0f;      // the largest finite |g|
  for (int64_t i = threadIdx.x; i < f.n; i += 1024) {
    const float a = __builtin_fabsf(f.factor(f.target[i], f.grad[i]));
    if (a < __builtin_inff()) top = fmaxf(top, a);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 16; ++w) top = fmaxf(top, lds[w]);
  int e = 0;
  if (top > 0.0f) {
    __builtin_frexpf(top, &e);           // top = f 2^e, f in [0.5, 1)
    e = TOP - e;
    e = e > 100 ? 100 : e < -100 ? -100 : e;
  }
  const float up = __builtin_ldexpf(1.0f, e);
  for (int64_t i = threadIdx.x; i < f.n; i += 1024)
    f.rows[i] = f.factor(f.target[i], f.grad[i] * up);
  if (threadIdx.x == 0) f.head->back = __builtin_ldexpf(1.0f, -e);
}

// As logits_kernel, and D written: 8,192 tokens, h = 4096, v = 128256 6.7 ms, h =
// 768, v = 50257 0.72 to 0.80 ms (8-byte stores 0.84).  Eight words of a token are
// a lane's (kPaired).  TWO: what the rounding leaves too, n rows further down.
//
// D's rounding to 16 bits, against float32 products of a float32 D (errors of
// the gradients against 64 bits, relative, of which the gradients' own rounding
// is 1.66e-3 in bfloat16 and 2.07e-4 in float16): 8,192 tokens, h = 768, v =
// 50257 bfloat16 1.84e-3 to 1.95e-3, with one gradient for all; 1,021 tokens, h =
// 1000, v = 32003 float16 2.8e-4, with one for each.  Linear layer and cross
// entropy of whole 16-bit logits: 2.6e-3 to 2.8e-3 and 4.5e-4.  A second part for
// all tokens would be six products in place of four.
//
// D of words [v0, v0 + tiles_m BM), 0 past the vocabulary: d[token][word - v0].
template <int DT, typename S, bool TWO>
__global__ __launch_bounds__(S::kThreads) void slope_kernel(Operand w, Operand x, int64_t v0,
                                                            int64_t v, int64_t n, int64_t h,
                                                            Factors factors, Grid g,
                                                            typename Elem<DT>::type *d,
                                                            int64_t ld) {
  int tm, tn, split;
  tile_of(g.tiles_m, g.tiles_n, 1, tm, tn, split);
  Acc<DT, S> acc;
  product<DT, kAlongK, kAlongK, kPaired, S, kFew<S>>(w, x, v0 + (int64_t)tm * S::BM,
                                                     (int64_t)tn * S::BN, 0, h, acc);
  typedef Place<S, kPaired> P;
  const P at(tm, tn);
#pragma unroll
  for (int j = 0; j < S::TN; ++j) {
    const int64_t token = at.n + 16 * j;
    if (token >= n) continue;
    const int64_t word = factors.target[token];
    const float top = factors.stats[token], part = 1.0f / factors.stats[n + token];
    const float row = factors.row<kTop<DT>>(token, word);
    const int64_t t = word - v0 - at.m;
    typename Elem<DT>::type *out = d + token * ld + at.m;
#pragma unroll
    for (int q = 0; q < S::TM; q += 2) {
      Eight<DT> f, rest;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float p = __builtin_amdgcn_exp2f((acc.t[q + e / 4][j][e % 4] - top) * kLog2e) * part;
        if (t == P::row(q) + e) p -= 1.0f;
        // (an ignored token's logits may be anything)
        const float g = row == 0.0f || v0 + at.m + P::row(q) + e >= v ? 0.0f : p * row;
        f[e] = Elem<DT>::round(g);
        if (TWO) rest[e] = Elem<DT>::round(g - (float)f[e]);
      }
      *(Eight<DT> *)(out + P::row(q)) = f;
      if (TWO) *(Eight<DT> *)(out + n * ld + P::row(q)) = rest;
    }
  }
}

// -- logits of few tokens, or of few words ----------------------------------------
//
// A tile's workgroup walks along k a pair of stages at a time, each a memory's
// latency long: with one tile to a CU or less that is the time.  Here a tile is
// kFewRows words by 16 TN tokens, k is shared out to the workgroup's wavefronts,
// which read their fragments straight from memory, a row's 512 (TN 4: 256) bytes
// at a time, wait for nobody and join their sums in LDS.  For few tokens the
// weight is read once, in longer runs than a tile's 128 bytes a row.

constexpr int kFewRows = 32, kFewWaves = 8, kFewThreads = 64 * kFewWaves;

template <int DT, int TN>
struct FewSums {
  static constexpr int kTokens = 16 * TN;
  static constexpr int kAhead = TN == 1 ? 8 : 4;      // 64-byte chunks of k per step
  static constexpr int kPer = kFewRows * kTokens / kFewThreads;    // sums per thread
  static_assert(kPer == TN, "a thread's sums are consecutive words of one token");
  // (padded: the four rows that a wavefront writes at a time lie in other banks)
  typedef float Lds[kFewWaves][kFewRows][kTokens + 4];

  // This thread's token and first word of a tile.
  static __device__ __forceinline__ int token() { return threadIdx.x % kTokens; }
  static __device__ __forceinline__ int word() { return threadIdx.x / kTokens * kPer; }

  template <bool WHOLE>
  static __device__ __forceinline__ void step(const char *const (&a)[2], const char *const (&b)[TN],
                                              int chunk, int bytes,
                                              Acc<DT, Shape<2, TN, 1, 1>> &acc) {
    const int part = (threadIdx.x & 63) >> 4;
    v4u fa[kAhead][2], fb[kAhead][TN];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int at = (chunk + u) * kRow;
      const bool in = WHOLE || at + part * 16 < bytes;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        // (one tile holds all tokens: nothing else reads these words)
        fa[u][i] = !in ? v4u{0, 0, 0, 0}
                   : TN == 1 ? __builtin_nontemporal_load((const v4u *)(a[i] + at))
                             : *(const v4u *)(a[i] + at);
#pragma unroll
      for (int j = 0; j < TN; ++j)
        fb[u][j] = in ? *(const v4u *)(b[j] + at) : v4u{0, 0, 0, 0};
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc.mma(i, j, fa[u][i], fb[u][j]);
  }

  // This thread's logits: words m0 + word() .. of token n0 + token().  Words and
  // tokens past the operands' ends take the last one's.
  static __device__ __forceinline__ void run(const Operand &w, const Operand &x, int64_t m0,
                                             int64_t n0, Lds &lds, float (&out)[kPer]) {
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int lane = threadIdx.x & 63, r = lane & 15;
    const char *a[2], *b[TN];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      a[i] = w.p + min(m0 + 16 * i + r, w.rows - 1) * w.ld + (lane >> 4) * 16;
#pragma unroll
    for (int j = 0; j < TN; ++j)
      b[j] = x.p + min(n0 + 16 * j + r, x.rows - 1) * x.ld + (lane >> 4) * 16;
    Acc<DT, Shape<2, TN, 1, 1>> acc;
    const int bytes = (int)w.row_bytes, chunks = (bytes + kRow - 1) / kRow;
    for (int c = wave * kAhead; c < chunks; c += kFewWaves * kAhead) {
      if ((c + kAhead) * kRow <= bytes)
        step<true>(a, b, c, bytes, acc);
      else
        step<false>(a, b, c, bytes, acc);
    }
    __syncthreads();               // (the tile before has been read)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          lds[wave][16 * i + (lane >> 4) * 4 + e][16 * j + r] = acc.t[i][j][e];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      out[e] = 0.0f;
#pragma unroll
      for (int k = 0; k < kFewWaves; ++k) out[e] += lds[k][word() + e][token()];
    }
  }
};

// logits_kernel's records, one for each of gridDim.x runs of tiles of words.
template <int DT, int TN>
__global__ __launch_bounds__(kFewThreads) void few_logits_kernel(Operand w, Operand x, int64_t v,
                                                                 int64_t n, const int64_t *target,
                                                                 float2 *part, float *picked) {
  typedef FewSums<DT, TN> F;
  __shared__ typename F::Lds lds;
  __shared__ float2 records[kFewThreads / F::kTokens][F::kTokens];
  const int64_t n0 = (int64_t)blockIdx.y * F::kTokens, token = n0 + F::token();
  const int64_t t = token < n ? target[token] : -1;
  float2 a = make_float2(-__builtin_inff(), 0.0f);
  for (int64_t m0 = (int64_t)blockIdx.x * kFewRows; m0 < v; m0 += (int64_t)gridDim.x * kFewRows) {
    float l[F::kPer];
    F::run(w, x, m0, n0, lds, l);
#pragma unroll
    for (int e = 0; e < F::kPer; ++e) {
      const int64_t word = m0 + F::word() + e;
      if (word >= v) continue;
      if (word == t) picked[token] = l[e];
      // (exp(l - l): 0 for -inf, NaN for inf and NaN)
      a = join(a, make_float2(l[e], l[e] == -__builtin_inff() ? 0.0f : 1.0f + (l[e] - l[e])));
    }
  }
  records[threadIdx.x / F::kTokens][F::token()] = a;
  __syncthreads();
  if (threadIdx.x >= F::kTokens || token >= n) return;
  for (int k = 1; k < kFewThreads / F::kTokens; ++k) a = join(a, records[k][F::token()]);
  part[(int64_t)blockIdx.x * n + token] = a;
}

// slope_kernel's D.
template <int DT, int TN, bool TWO>
__global__ __launch_bounds__(kFewThreads) void few_slope_kernel(Operand w, Operand x, int64_t v0,
                                                                int64_t v, int64_t padded,
                                                                int64_t n, Factors factors,
                                                                typename Elem<DT>::type *d,
                                                                int64_t ld) {
  typedef FewSums<DT, TN> F;
  __shared__ typename F::Lds lds;
  const int64_t n0 = (int64_t)blockIdx.y * F::kTokens, token = n0 + F::token();
  const int64_t t = token < n ? factors.target[token] : 0;
  const float top = token < n ? factors.stats[token] : 0.0f;
  const float part = token < n ? 1.0f / factors.stats[n + token] : 0.0f;
  const float row = token < n ? factors.row<kTop<DT>>(token, t) : 0.0f;
  for (int64_t m0 = (int64_t)blockIdx.x * kFewRows; m0 < padded;
       m0 += (int64_t)gridDim.x * kFewRows) {
    float l[F::kPer] = {};
    if (v0 + m0 < v) F::run(w, x, v0 + m0, n0, lds, l);     // (else padding)
    if (token >= n) continue;
#pragma unroll
    for (int e = 0; e < F::kPer; ++e) {
      const int64_t at = m0 + F::word() + e, word = v0 + at;
      float p = __builtin_amdgcn_exp2f((l[e] - top) * kLog2e) * part;
      if (word == t) p -= 1.0f;
      const float f = row == 0.0f || word >= v ? 0.0f : p * row;
      const typename Elem<DT>::type hi = Elem<DT>::round(f);
      d[token * ld + at] = hi;
      if (TWO) d[(n + token) * ld + at] = Elem<DT>::round(f - (float)hi);
    }
  }
}

// D W and D^T X.  Bound by the matrix cores; both operands of the second and one
// of the first lie with k along their lines, which the LDS reads turn, so that
// nothing is transposed in memory.  8,192 tokens, h = 4096, v = 128256: 6.1 and
// 6.3 ms (1.4 PFLOP/s); h = 768, v = 50257: 0.57 and 0.52 ms.  A few tokens'
// d_weight is bound by writing it (one token: 1.05 GB in 325 us, 128 x 128 tiles
// 400 us, non-temporal stores no faster).
//
// A product into float32 (out[split][n][m], added to what is there with `add`)
// or, with out16, scaled back into the operands' type.
template <int DT, int AB, typename S>
__global__ __launch_bounds__(S::kThreads) void product_kernel(Operand a, Operand b, int64_t m,
                                                              int64_t n, int64_t k,
                                                              int64_t k_split, Grid g, int add,
                                                              float *out, Factors factors,
                                                              typename Elem<DT>::type *out16) {
  int tm, tn, split;
  tile_of(g.tiles_m, g.tiles_n, g.splits, tm, tn, split);
  const int64_t k0 = split * k_split, k1 = min(k, k0 + k_split);
  // (a lane's eight consecutive columns are one store; of float32 four are)
  constexpr int kOrder = DT == LUMA_GRAD_F32 ? kPlain : kPaired;
  Acc<DT, S> acc;
  product<DT, kAlongM, AB, kOrder, S, kFew<S> && AB == kAlongK>(
      a, b, (int64_t)tm * S::BM, (int64_t)tn * S::BN, k0, k1, acc);
  typedef Place<S, kOrder> P;
  const P at(tm, tn);
  const bool aligned = m % 8 == 0 && (uintptr_t)out16 % 16 == 0;
  const float f = out16 ? factors.back<kTop<DT>>() : 1.0f;
#pragma unroll
  for (int j = 0; j < S::TN; ++j) {
    const int64_t row = at.n + 16 * j;
    if (row >= n) continue;
#pragma unroll
    for (int q = 0; q < S::TM; q += 2) {
      const int64_t col = at.m + P::row(q), next = at.m + P::row(q + 1);
      if (out16) {
        const v4f c = acc.t[q][j] * f, d = acc.t[q + 1][j] * f;
        if (kOrder == kPaired && aligned && col + 8 <= m) {
          Eight<DT> o;
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = Elem<DT>::round(e < 4 ? c[e & 3] : d[e & 3]);
          *(Eight<DT> *)(out16 + row * m + col) = o;
        } else {
          store4<DT>(out16 + row * m, col, m, c);
          store4<DT>(out16 + row * m, next, m, d);
        }
      } else {
        float *o = out + (int64_t)split * n * m + row * m;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int64_t at = k ? next : col;
          v4f c = acc.t[q + k][j];
          if (add)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (at + r < m) c[r] += o[at + r];
          store4<LUMA_GRAD_F32>(o, at, m, c);
        }
      }
    }
  }
}

// Bound by memory.  The sum of `splits` float32 products, scaled back, in the operands' type.
template <int DT>
__global__ __launch_bounds__(256) void sum_kernel(const float *part, int splits, int64_t count,
                                                  Factors factors,
                                                  typename Elem<DT>::type *out) {
  const float f = factors.back<kTop<DT>>();
  for (int64_t i = (blockIdx.x * 256ll + threadIdx.x) * 4; i < count; i += gridDim.x * 1024ll) {
    v4f s = {0.f, 0.f, 0.f, 0.f};
    if (i + 4 <= count) {
      typedef float v4fu __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll 4
      for (int k = 0; k < splits; ++k) s += *(const v4fu *)(part + k * count + i);
    } else {
      for (int k = 0; k < splits; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (i + r < count) s[r] += part[k * count + i + r];
    }
    store4<DT>(out, i, count, s * f);
  }
}

// A copy of a strided matrix with rows of `ld` elements, zeros past its columns.
template <typename T>
__global__ __launch_bounds__(256) void pack_kernel(const T *in, int64_t rows, int64_t cols,
                                                   int64_t ld_in, T *out, int64_t ld) {
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < rows * ld; i += gridDim.x * 256ll) {
    const int64_t r = i / ld, c = i % ld;
    out[i] = c < cols ? in[r * ld_in + c] : (T)0;
  }
}

// -- host -----------------------------------------------------------------------

typedef Shape<8, 4, 2, 4> Big;       // 256 x 256
typedef Shape<4, 4, 2, 2> Mid;       // 128 x 128
typedef Shape<2, 2, 2, 2> Small;     // 64 x 64
typedef Shape<2, 4, 4, 1> Thin64;    // 128 x 64: few tokens
typedef Shape<2, 1, 4, 1> Thin16;    // 128 x 16
enum ShapeId { kBig, kMid, kSmall, kThin64, kThin16 };
constexpr int64_t kTwoParts = 64;    // tokens: up to here D is kept in two parts (kFew's shapes)
constexpr int kBM[] = {256, 128, 64, 128, 128}, kBN[] = {256, 128, 64, 64, 16};
constexpr int64_t kChip = 256;                 // CUs

int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
int64_t tiles(int64_t x, int64_t size) { return (x + size - 1) / size; }

// The tile for a product of m x n whose k can be split in up to `splits`: the
// largest whose workgroups fill the chip.
int shape_for(int64_t m, int64_t n, int64_t splits) {
  if (n <= 16) return kThin16;
  if (n <= 64) return kThin64;
  if (tiles(m, 256) * tiles(n, 256) * splits >= 192) return kBig;
  if (tiles(m, 128) * tiles(n, 128) * splits >= 128) return kMid;
  return kSmall;
}

// Into how many parts k is split, and each part's length (a multiple of
// `round`).  A part is a workgroup per tile: they should come in whole rounds of
// the chip, but each part's float32 sums are written and read again.  The cost
// of s parts, in bytes of that traffic's time: a round takes `deep` bytes' time
// for an element of k (a 256 x 256 tile at about 5 TFLOP/s per CU of 16-bit
// products takes 26 ns, in which the chip moves 100 KB), and the sums 8 s m n.
int64_t split_k(int shape, int64_t m, int64_t n, int64_t k, int64_t round, int64_t &each) {
  const int64_t t = tiles(m, kBM[shape]) * tiles(n, kBN[shape]);
  const int64_t at_once = shape == kBig ? kChip : shape == kMid ? 2 * kChip : 4 * kChip;
  const double deep = 100e3 * kBM[shape] * kBN[shape] / (256.0 * 256.0) * at_once / kChip;
  const int64_t most = tiles(k, 4 * round) < 64 ? tiles(k, 4 * round) : 64;
  int64_t best = 1;
  double least = 0.0;
  for (int64_t s = 1; s <= most; ++s) {
    const int64_t part = up(tiles(k, s), round);
    const double cost = (double)tiles(t * s, at_once) * part * deep +
                        (s > 1 ? 8.0 * s * m * n + 16e6 : 0.0);
    if (s == 1 || cost < least) best = s, least = cost;
  }
  each = up(tiles(k, best), round);
  return tiles(k, each);
}

// Of `words` words, those whose 256 x 256 tiles with `others` along the other
// side make whole rounds of the chip (0: fewer than one round).
int64_t whole_rounds(int64_t others, int64_t words) {
  const int64_t rows = tiles(others, 256), rounds = tiles(words, 256) * rows / kChip;
  const int64_t main = kChip * rounds / rows * 256;
  return main < words ? main : words;
}

// Of `words` words of logits, those that take 256 x 256 tiles; the others take
// 128 x 128, where that is shorter than a last round that few tiles fill (two of
// them are on a CU at a time and take about 0.55 of a round; their launch
// starts after the rounds').
int64_t big_words(int64_t n, int64_t words) {
  if (shape_for(words, n, 1) != kBig) return 0;
  const int64_t main = whole_rounds(n, words);
  if (main == 0 || main == words) return words;
  const int64_t rest = tiles(words - main, 128) * tiles(n, 128);
  return 0.55 * tiles(rest, 2 * kChip) + 0.1 < 1.0 ? main : words;
}

// Words per piece of the vocabulary: pieces of about equal length, each at most
// kPieceBytes of D (pieces of 256 MB, which the last-level cache holds: d_hidden
// of 8,192 x 768 tokens takes 0.90 ms in four, 0.60 in one).
constexpr int64_t kPieceBytes = 1 << 30;
constexpr int64_t kPieceTiles = 1 << 15;   // a tile's offsets into 64 rows of D stay below 2^31
int64_t piece_for(int64_t n, int64_t v, int64_t size) {
  const int64_t all = tiles(v, 256);
  int64_t most = kPieceBytes / (n * size * 256);
  if (most < 1) most = 1;
  if (most > kPieceTiles) most = kPieceTiles;
  return tiles(all, tiles(all, most)) * 256;
}

struct Plan {
  int64_t size;                 // bytes of an element
  bool pack_x, pack_w;
  int64_t ld_x, ld_w;           // elements, of what the products read
  int64_t at_x, at_w;           // of the packed copies
  bool few;                     // logits by few_logits_kernel, few_slope_kernel
  int64_t big;                  // else: words of logits (of a piece) in 256 x 256 tiles
  int rest;                     // tile shape of the others
  // forward
  int64_t parts, at_part, at_picked, at_sums, blocks;
  // backward
  int64_t rows_d;               // rows of D: n, or 2 n where it is kept in two parts
  int64_t piece, ld_d;          // words per piece; elements per row of D
  int hidden;                   // tile shape
  int64_t hidden_splits, hidden_k;
  int64_t at_head, at_rows, at_d, at_hidden, at_weight;
  int64_t bytes;
};

// Tokens per workgroup of the join: one, while they are too few to fill the chip.
int64_t join_tokens(int64_t n) { return n <= kChip ? 1 : 32; }

// Whether the logits of n tokens and `words` words go without tiles: where less
// than a quarter of the chip would have one, and k is long (us for the loss,
// tiles / without; tokens x h x words): float32 10 x 4096 x 100 92 / 31, 300 x
// 4096 x 28 76 / 64, bfloat16 1 x 4096 x 28 42 / 23; but 50 x 768 x 5000 24 / 25,
// 128 x 2048 x 3000 23 / 27, 1 x 4096 x 128256 171 / 334.
bool few_for(int64_t words, int64_t n, int64_t k_bytes) {
  const int shape = shape_for(words, n, 1);
  return tiles(words, kBM[shape]) * tiles(n, kBN[shape]) < kChip / 4 && k_bytes >= 32 * kRow;
}
int few_tn(int64_t words, int64_t n) {
  return tiles(words, kFewRows) * tiles(n, 16) < kChip ? 1 : 4;
}
// Runs of tiles of words: about four workgroups to a CU in all.
int64_t few_runs(int64_t words, int64_t n, int tn) {
  const int64_t groups = tiles(n, 16 * tn), most = groups < 1024 ? 1024 / groups : 1;
  const int64_t all = tiles(words, kFewRows);
  return all < most ? all : most;
}

int weight_shape(const LumaXentArgs *a, int64_t words) {
  return shape_for(a->h, words < 65 ? 65 : words, tiles(a->n, 1024));
}

bool plan(const LumaXentArgs *a, bool backward, Plan &p) {
  p = Plan{};
  p.size = a->dtype == LUMA_GRAD_F32 ? 4 : 2;
  const int64_t group = 16 / p.size, round = (kStages * kRow) / p.size;
  auto direct = [&](const void *q, int64_t ld, int64_t rows) {
    return (uintptr_t)q % 16 == 0 && a->h % group == 0 && (ld % group == 0 || rows == 1);
  };
  p.pack_x = !direct(a->hidden, a->ld_hidden, a->n);
  p.pack_w = !direct(a->weight, a->ld_weight, a->v);
  p.ld_x = p.pack_x ? up(a->h, group) : a->ld_hidden;
  p.ld_w = p.pack_w ? up(a->h, group) : a->ld_weight;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += up(bytes, 256);
    return here;
  };
  auto logits_plan = [&](int64_t words) {
    p.few = few_for(words, a->n, a->h * p.size);
    p.big = big_words(a->n, words);
    p.rest = p.big ? kMid : shape_for(words, a->n, 1);
  };
  // D is rounded to the operands' type, as a 16-bit matrix operand has to be; what
  // that costs is about as much again as half of the gradients' own rounding.  Of
  // few tokens nearly the whole gradient is the target's entry, off by up to half
  // a step.  Their products wait for the weight (or write its gradient), so a
  // second part costs nothing: it is n more rows of D, and X is there twice.
  const bool two = backward && a->n <= kTwoParts && p.size == 2;
  p.rows_d = two ? 2 * a->n : a->n;
  if (two) {
    p.pack_x = true;
    p.ld_x = up(a->h, group);
  }
  if (p.pack_x) p.at_x = take(p.rows_d * p.ld_x * p.size);
  if (p.pack_w) p.at_w = take(a->v * p.ld_w * p.size);
  if (!backward) {
    logits_plan(a->v);
    p.parts = p.few ? few_runs(a->v, a->n, few_tn(a->v, a->n))
                    : tiles(p.big, 256) + tiles(a->v - p.big, kBM[p.rest]);
    p.blocks = tiles(a->n, join_tokens(a->n));
    p.at_part = take(p.parts * a->n * sizeof(float2));
    p.at_picked = take(a->n * sizeof(float));
    p.at_sums = take(p.blocks * sizeof(double2));
  } else {
    p.piece = piece_for(p.rows_d, a->v, p.size);
    // (the same tiles as the forward's: the largest logit is then the same
    // number, and its probability 1 / sum exactly)
    logits_plan(p.piece < a->v ? p.piece : a->v);
    p.ld_d = p.piece;
    p.at_head = take(sizeof(Rows));
    p.at_rows = take(a->n * sizeof(float));
    p.at_d = take(p.rows_d * p.ld_d * p.size);
    int64_t each, sums = 0;
    if (a->d_hidden) {
      p.hidden = shape_for(a->h, p.rows_d, tiles(p.ld_d, 1024));
      p.hidden_splits = split_k(p.hidden, a->h, p.rows_d, p.ld_d, round, p.hidden_k);
      if (p.hidden_splits > 1 || p.piece < a->v || p.rows_d > a->n)
        p.at_hidden = take(p.hidden_splits * p.rows_d * a->h * sizeof(float));
    }
    if (a->d_weight) {
      const int64_t last = a->v - (a->v - 1) / p.piece * p.piece;
      const int64_t first = p.piece < a->v ? p.piece : a->v;
      for (const int64_t words : {whole_rounds(a->h, first), first - whole_rounds(a->h, first),
                                  whole_rounds(a->h, last), last - whole_rounds(a->h, last)}) {
        if (words == 0) continue;
        const int shape = weight_shape(a, words);
        const int64_t splits = split_k(shape, a->h, words, p.rows_d, round, each);
        if (splits > 1 && splits * words > sums) sums = splits * words;
      }
      if (sums) p.at_weight = take(sums * a->h * sizeof(float));
    }
  }
  p.bytes = at;
  return true;
}

bool check_args(const LumaXentArgs *a, bool backward) {
  if (!a) return fail("luma_xent: null arguments"), false;
  if (a->n < 1 || a->h < 1 || a->v < 1) return fail("luma_xent: empty operands"), false;
  if (a->n > INT32_MAX / 2 || a->h > 1 << 20 || a->v > INT32_MAX / 2)
    return fail("luma_xent: operands too large"), false;
  if (a->dtype < LUMA_GRAD_F32 || a->dtype > LUMA_GRAD_F16)
    return fail("luma_xent: unknown type"), false;
  if (a->reduction < LUMA_XENT_NONE || a->reduction > LUMA_XENT_MEAN)
    return fail("luma_xent: unknown reduction"), false;
  if (!a->hidden || !a->weight || !a->target || !a->stats || (!backward && !a->loss) ||
      (backward && !a->grad_loss))
    return fail("luma_xent: null operand"), false;
  if ((a->ld_hidden < a->h && a->n > 1) || (a->ld_weight < a->h && a->v > 1))
    return fail("luma_xent: rows overlap"), false;
  if (a->ld_hidden > 1 << 21 || a->ld_weight > 1 << 21)
    return fail("luma_xent: rows too far apart"), false;
  // (a launch's workgroups are counted in 32 bits, and so are its threads: 512 to
  // a 256 x 256 tile)
  if (tiles(a->n, 256) * tiles(a->v, 256) > UINT32_MAX / 512 ||
      tiles(a->n, 16) * tiles(a->v, 64) > INT32_MAX ||
      tiles(a->h, 64) * tiles(a->v, 64) > INT32_MAX / 64 ||
      tiles(a->h, 64) * tiles(a->n, 16) > INT32_MAX / 64)
    return fail("luma_xent: operands too large"), false;
  return true;
}

template <typename F>
void with_shape(int shape, F f) {
  switch (shape) {
    case kBig: return f(Big{});
    case kMid: return f(Mid{});
    case kSmall: return f(Small{});
    case kThin64: return f(Thin64{});
    default: return f(Thin16{});
  }
}

template <typename F>
void with_few(int64_t words, int64_t n, F f) {
  if (few_tn(words, n) == 1)
    f(std::integral_constant<int, 1>{});
  else
    f(std::integral_constant<int, 4>{});
}

Grid grid_of(int shape, int64_t m, int64_t n, int64_t splits) {
  return Grid{(int)tiles(m, kBM[shape]), (int)tiles(n, kBN[shape]), (int)splits};
}

template <int DT>
void pack(const void *in, int64_t rows, int64_t cols, int64_t ld_in, char *out, int64_t ld,
          hipStream_t s) {
  typedef typename Elem<DT>::type T;
  const int64_t blocks = tiles(rows * ld, 256 * 8);
  pack_kernel<T><<<(int)(blocks < 8192 ? blocks : 8192), 256, 0, s>>>((const T *)in, rows, cols,
                                                                      ld_in, (T *)out, ld);
}

// The operands as the products read them.
template <int DT>
void operands(const LumaXentArgs *a, const Plan &p, Operand &x, Operand &w, hipStream_t s) {
  char *ws = (char *)a->workspace;
  for (int64_t r = 0; p.pack_x && r < p.rows_d; r += a->n)
    pack<DT>(a->hidden, a->n, a->h, a->ld_hidden, ws + p.at_x + r * p.ld_x * p.size, p.ld_x, s);
  if (p.pack_w) pack<DT>(a->weight, a->v, a->h, a->ld_weight, ws + p.at_w, p.ld_w, s);
  const int64_t bytes = up(a->h, 16 / p.size) * p.size;
  x = Operand{p.pack_x ? ws + p.at_x : (const char *)a->hidden, p.ld_x * p.size, a->n, bytes};
  w = Operand{p.pack_w ? ws + p.at_w : (const char *)a->weight, p.ld_w * p.size, a->v, bytes};
}

template <int DT>
void forward(const LumaXentArgs *a, const Plan &p, hipStream_t s) {
  Operand x, w;
  operands<DT>(a, p, x, w, s);
  char *ws = (char *)a->workspace;
  float2 *part = (float2 *)(ws + p.at_part);
  float *picked = (float *)(ws + p.at_picked);
  double2 *sums = a->reduction == LUMA_XENT_NONE ? nullptr : (double2 *)(ws + p.at_sums);
  auto logits = [&](int shape_id, int64_t v0, int64_t words, float2 *out) {
    if (words == 0) return;
    with_shape(shape_id, [&](auto shape) {
      typedef decltype(shape) S;
      const Grid g = grid_of(shape_id, words, a->n, 1);
      logits_kernel<DT, S><<<g.tiles_m * g.tiles_n, S::kThreads, 0, s>>>(
          w, x, v0, a->v, a->n, a->h, a->target, g, out, picked);
    });
  };
  if (p.few) {
    with_few(a->v, a->n, [&](auto tn) {
      constexpr int TN = decltype(tn)::value;
      const dim3 grid((int)p.parts, (int)tiles(a->n, 16 * TN));
      few_logits_kernel<DT, TN><<<grid, kFewThreads, 0, s>>>(w, x, a->v, a->n, a->target, part,
                                                            picked);
    });
  } else {
    logits(kBig, 0, p.big, part);
    logits(p.rest, p.big, a->v - p.big, part + tiles(p.big, 256) * a->n);
  }
  const auto join = join_tokens(a->n) == 1 ? join_kernel<1> : join_kernel<32>;
  join<<<(int)p.blocks, kJoinThreads, 0, s>>>(part, (int)p.parts, picked, a->target, a->n, a->v,
                                              a->ignore_index, a->stats, a->loss, sums);
  if (sums)
    reduce_kernel<<<1, 256, 0, s>>>(sums, p.blocks, a->reduction, a->stats + 2 * a->n, a->loss);
}

template <int DT>
void sum_splits(const float *part, int64_t splits, int64_t count, const Factors &factors,
                void *out, hipStream_t s) {
  const int64_t blocks = tiles(count, 1024);
  sum_kernel<DT><<<(int)(blocks < 4096 ? blocks : 4096), 256, 0, s>>>(
      part, (int)splits, count, factors, (typename Elem<DT>::type *)out);
}

template <int DT>
void backward(const LumaXentArgs *a, const Plan &p, hipStream_t s) {
  typedef typename Elem<DT>::type T;
  Operand x, w;
  operands<DT>(a, p, x, w, s);
  char *ws = (char *)a->workspace;
  Rows *head = (Rows *)(ws + p.at_head);
  float *rows = (float *)(ws + p.at_rows);
  T *d = (T *)(ws + p.at_d);
  float *hidden = (float *)(ws + p.at_hidden), *weight = (float *)(ws + p.at_weight);
  const Factors factors = {a->grad_loss, a->target,    a->stats, a->n, a->v,
                           a->ignore_index, a->reduction, head,     rows};
  if (a->reduction == LUMA_XENT_NONE) rows_kernel<kTop<DT>><<<1, 1024, 0, s>>>(factors);
  const bool whole = p.piece >= a->v;        // one piece
  const bool direct = p.hidden_splits == 1 && whole && p.rows_d == a->n;
  const Operand twice = {x.p, x.ld, p.rows_d, x.row_bytes};
  for (int64_t v0 = 0; v0 < a->v; v0 += p.piece) {
    const int64_t words = a->v - v0 < p.piece ? a->v - v0 : p.piece;
    // (the products take k up to the padding: D is 0 there)
    const int64_t padded = up(words, 256);
    auto slope = [&](int shape_id, int64_t w0, int64_t count) {
      if (count <= 0) return;
      with_shape(shape_id, [&](auto shape) {
        typedef decltype(shape) S;
        const Grid g = grid_of(shape_id, count, a->n, 1);
        auto go = [&](auto two) {
          slope_kernel<DT, S, decltype(two)::value>
              <<<g.tiles_m * g.tiles_n, S::kThreads, 0, s>>>(w, x, v0 + w0, a->v, a->n, a->h,
                                                             factors, g, d + w0, p.ld_d);
        };
        if constexpr (kFew<S> && DT != LUMA_GRAD_F32) {
          if (p.rows_d > a->n) return go(std::true_type{});
        }
        go(std::false_type{});
      });
    };
    if (p.few) {
      with_few(a->v, a->n, [&](auto tn) {
        constexpr int TN = decltype(tn)::value;
        const dim3 grid((int)few_runs(padded, a->n, TN), (int)tiles(a->n, 16 * TN));
        auto go = [&](auto two) {
          few_slope_kernel<DT, TN, decltype(two)::value><<<grid, kFewThreads, 0, s>>>(
              w, x, v0, a->v, padded, a->n, factors, d, p.ld_d);
        };
        if constexpr (DT != LUMA_GRAD_F32) {
          if (p.rows_d > a->n) return go(std::true_type{});
        }
        go(std::false_type{});
      });
    } else {
      // (whole tiles: all of the padding, or whole_rounds')
      const int64_t big = p.big < words ? p.big : padded;
      slope(kBig, 0, big);
      slope(p.rest, big, padded - big);
    }
    const Operand wp = {w.p + v0 * w.ld, w.ld, words, w.row_bytes};
    if (a->d_hidden) {
      const Operand dk = {(const char *)d, p.ld_d * p.size, p.rows_d, padded * p.size};
      with_shape(p.hidden, [&](auto shape) {
        typedef decltype(shape) S;
        const Grid g = grid_of(p.hidden, a->h, p.rows_d, p.hidden_splits);
        product_kernel<DT, kAlongK, S><<<g.tiles_m * g.tiles_n * g.splits, S::kThreads, 0, s>>>(
            wp, dk, a->h, p.rows_d, padded, p.hidden_k, g, v0 > 0, hidden, factors,
            direct ? (T *)a->d_hidden : nullptr);
      });
    }
    if (a->d_weight) {
      // (the tiles that make whole rounds of the chip, then the rest)
      const int64_t main = whole_rounds(a->h, words);
      const int64_t cut[] = {0, main, words};
      for (int c = 0; c < 2; ++c) {
        const int64_t w0 = cut[c], count = cut[c + 1] - w0;
        if (count == 0) continue;
        const Operand dm = {(const char *)(d + w0), p.ld_d * p.size, p.rows_d,
                            (padded - w0) * p.size};
        T *out = (T *)a->d_weight + (v0 + w0) * a->h;
        const int shape_id = weight_shape(a, count);
        int64_t each;
        const int64_t splits =
            split_k(shape_id, a->h, count, p.rows_d, kStages * kRow / p.size, each);
        with_shape(shape_id, [&](auto shape) {
          typedef decltype(shape) S;
          if constexpr (S::BN >= 64) {
            const Grid g = grid_of(shape_id, a->h, count, splits);
            product_kernel<DT, kAlongM, S>
                <<<g.tiles_m * g.tiles_n * g.splits, S::kThreads, 0, s>>>(
                    twice, dm, a->h, count, p.rows_d, each, g, 0, weight, factors,
                    splits == 1 ? out : nullptr);
          }
        });
        if (splits > 1) sum_splits<DT>(weight, splits, count * a->h, factors, out, s);
      }
    }
  }
  if (a->d_hidden && !direct)
    sum_splits<DT>(hidden, p.hidden_splits * (p.rows_d / a->n), a->n * a->h, factors,
                   a->d_hidden, s);
}

template <typename F>
void with_type(int dtype, F f) {
  switch (dtype) {
    case LUMA_GRAD_F32: return f(std::integral_constant<int, LUMA_GRAD_F32>{});
    case LUMA_GRAD_BF16: return f(std::integral_constant<int, LUMA_GRAD_BF16>{});
    default: return f(std::integral_constant<int, LUMA_GRAD_F16>{});
  }
}

}  // namespace
}  // namespace luma

using namespace luma;

extern "C" {

int64_t luma_xent_workspace_bytes(const LumaXentArgs *a, int32_t backward) {
  Plan p;
  if (!check_args(a, backward != 0) || !plan(a, backward != 0, p)) return -1;
  return p.bytes;
}

int luma_xent_forward(const LumaXentArgs *a, void *stream) {
  Plan p;
  if (!check_args(a, false) || !plan(a, false, p)) return -1;
  if (!a->workspace || (uintptr_t)a->workspace % 256 || a->workspace_bytes < p.bytes)
    return fail("luma_xent_forward: workspace too small or not aligned");
  with_type(a->dtype, [&](auto dt) { forward<decltype(dt)::value>(a, p, (hipStream_t)stream); });
  return check_launch("luma_xent_forward");
}

int luma_xent_backward(const LumaXentArgs *a, void *stream) {
  Plan p;
  if (!check_args(a, true) || !plan(a, true, p)) return -1;
  if (!a->workspace || (uintptr_t)a->workspace % 256 || a->workspace_bytes < p.bytes)
    return fail("luma_xent_backward: workspace too small or not aligned");
  if (!a->d_hidden && !a->d_weight) return 0;
  with_type(a->dtype, [&](auto dt) { backward<decltype(dt)::value>(a, p, (hipStream_t)stream); });
  return check_launch("luma_xent_backward");
}

}  // extern "C"
