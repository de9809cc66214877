// Rows of elements in eights, and dropout's draws: what the kernels of the
// residual stream (luma_residual.hip) and of the tokens' losses (luma_policy.hip)
// share.
#pragma once
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <type_traits>

#include "../../include/luma.h"
#include "luma_philox.h"

namespace luma {
namespace rows {

template <int DT>
struct Elem;
template <>
struct Elem<LUMA_GRAD_F32> {
  typedef float type;
};
template <>
struct Elem<LUMA_GRAD_BF16> {
  typedef __bf16 type;
};
template <>
struct Elem<LUMA_GRAD_F16> {
  typedef _Float16 type;
};

// (element alignment only: a row may begin anywhere)
template <typename T, int N>
using Vec = T __attribute__((ext_vector_type(N), aligned(sizeof(T)), may_alias));

// N elements of a row of h from column c on; 0 past the row's end.
template <int N, typename T>
__device__ __forceinline__ Vec<T, N> load(const T *row, int64_t c, int64_t h) {
  if (c + N <= h) return *(const Vec<T, N> *)(row + c);
  Vec<T, N> v;
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = c + j < h ? row[c + j] : (T)0.0f;
  return v;
}

// Rounds f to nearest and stores those of the elements that lie in the row.
template <int N, typename T>
__device__ __forceinline__ void store(T *row, int64_t c, int64_t h, const float *f) {
  if (c + N <= h) {
    Vec<T, N> v;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = (T)f[j];
    *(Vec<T, N> *)(row + c) = v;
    return;
  }
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (c + j < h) row[c + j] = (T)f[j];
}

template <int N, typename T>
__device__ __forceinline__ void widen(const Vec<T, N> &v, float *f) {
#pragma unroll
  for (int j = 0; j < N; ++j) f[j] = (float)v[j];
}

// Dropout's draws.  Element e (its index in the operand, rows one after the
// other) has 32 bits u(e): the high ones are half e % 8 of the block with
// counter (e / 8, 0, call), the low ones that half of (e / 8, 1, call), the key
// is the seed.  It is dropped where u < p 2^32 (rounded), so p is met to 2^-33.
// The high half decides but for one element in 65,536, and the second block is
// drawn for those alone: eight elements for the ten rounds of one block.
struct Draw {
  uint32_t k0, k1, call;
  uint32_t high, low;   // the limit p 2^32 in halves (high: up to 65,536)
  float scale;          // 1 / (1 - p)
};

__device__ __forceinline__ Draw draw_of(const LumaDropout &d) {
  Draw o;
  const uint64_t seed = d.seed_at ? *(const uint64_t *)d.seed_at : d.seed;
  o.k0 = (uint32_t)seed;
  o.k1 = (uint32_t)(seed >> 32);
  o.call = d.call;
  const double limit = __builtin_floor(d.p * 4294967296.0 + 0.5);
  const uint64_t t = (uint64_t)limit;
  o.high = (uint32_t)(t >> 16);
  o.low = (uint32_t)t & 0xFFFFu;
  o.scale = d.p < 1.0 ? (float)(1.0 / (1.0 - d.p)) : 0.0f;
  return o;
}

// Bit j: whether element 8 block + j is kept.
__device__ __forceinline__ uint32_t kept_of_block(uint64_t block, const Draw &d) {
  const U4 top = philox4x32_10_v((uint32_t)block, (uint32_t)(block >> 32), 0u, d.call, d.k0, d.k1,
                                 kPhiloxM0, kPhiloxM1);
  uint32_t kept = 0u, even = 0u;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t u = u4_half(top, j);
    kept |= u >= d.high ? 1u << j : 0u;
    even |= u == d.high ? 1u << j : 0u;
  }
  if (even && d.low) {
    const U4 below = philox4x32_10_v((uint32_t)block, (uint32_t)(block >> 32), 1u, d.call, d.k0,
                                     d.k1, kPhiloxM0, kPhiloxM1);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if ((even >> j & 1u) && u4_half(below, j) < d.low) kept &= ~(1u << j);
  }
  return kept;
}

// Bit j: whether element e + j is kept, j < 8.
__device__ __forceinline__ uint32_t kept_from(uint64_t e, const Draw &d) {
  const uint32_t at = (uint32_t)e & 7u;
  uint32_t kept = kept_of_block(e >> 3, d);
  if (at) kept = (kept | kept_of_block((e >> 3) + 1, d) << 8) >> at;
  return kept;
}

// f(type) of an element type's code.
template <typename F>
void with_type(int dtype, F f) {
  switch (dtype) {
    case LUMA_GRAD_F32: return f(float{});
    case LUMA_GRAD_BF16: return f(__bf16{});
    default: return f(_Float16{});
  }
}

// f(stream's type, branch's type): the same, or a float32 stream.
template <typename F>
void with_types(int stream, int branch, F f) {
  with_type(branch, [&](auto b) {
    typedef decltype(b) B;
    if (stream == branch) return f(B{}, B{});
    f(float{}, B{});
  });
}

inline bool known_type(int dtype) { return dtype >= LUMA_GRAD_F32 && dtype <= LUMA_GRAD_F16; }

// Sum of v over the L lanes (a power of two, at most 64) that hold one row.
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int m = 1; m < L; m <<= 1) v += __shfl_xor(v, m);
  return v;
}

}  // namespace rows
}  // namespace luma
