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

// N elements with the alignment of one: a row may begin anywhere.  (Typedefs of
// their own: in an alias template the attribute is lost, and the compiler then
// takes 16-byte alignment for given.)
template <typename T, int N>
struct VecOf;
template <>
struct VecOf<float, 4> {
  typedef float type __attribute__((ext_vector_type(4), aligned(4), may_alias));
};
template <>
struct VecOf<__bf16, 4> {
  typedef __bf16 type __attribute__((ext_vector_type(4), aligned(2), may_alias));
};
template <>
struct VecOf<__bf16, 8> {
  typedef __bf16 type __attribute__((ext_vector_type(8), aligned(2), may_alias));
};
template <>
struct VecOf<_Float16, 4> {
  typedef _Float16 type __attribute__((ext_vector_type(4), aligned(2), may_alias));
};
template <>
struct VecOf<_Float16, 8> {
  typedef _Float16 type __attribute__((ext_vector_type(8), aligned(2), may_alias));
};
template <>
struct VecOf<uint8_t, 4> {
  typedef uint8_t type __attribute__((ext_vector_type(4), aligned(1), may_alias));
};
template <>
struct VecOf<float, 1> {
  typedef float type __attribute__((ext_vector_type(1), aligned(4), may_alias));
};
template <>
struct VecOf<__bf16, 1> {
  typedef __bf16 type __attribute__((ext_vector_type(1), aligned(2), may_alias));
};
template <>
struct VecOf<_Float16, 1> {
  typedef _Float16 type __attribute__((ext_vector_type(1), aligned(2), may_alias));
};
template <>
struct VecOf<uint8_t, 1> {
  typedef uint8_t type __attribute__((ext_vector_type(1), aligned(1), may_alias));
};
template <typename T, int N>
using Vec = typename VecOf<T, N>::type;

// N elements of a row of h >= N from column c on, as one load.  WHOLE: h is a
// multiple of N; 0 outside.  Else without a condition (where the branches of a few
// met, the compiler waited for each load: 524 x 5,616 of cut rows 15.3 us, so 11.9;
// of whole ones the condition is as good and takes fewer registers): of a run that
// the row's end cuts, and of one outside, the row's N last elements, of which
// settle() makes, when they are used, what lies in the row, moved down, and 0s.
template <int N, bool WHOLE = false, bool NT = false, typename T>
__device__ __forceinline__ Vec<T, N> load_raw(const T *row, int64_t c, int64_t h) {
  static_assert(alignof(Vec<T, N>) == sizeof(T), "an element's alignment");
  if constexpr (WHOLE) {
    if (c >= h) {
      Vec<T, N> v;
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = (T)0.0f;
      return v;
    }
  } else {
    c = c < h - N ? c : h - N;
  }
  if constexpr (NT) return __builtin_nontemporal_load((const Vec<T, N> *)(row + c));
  return *(const Vec<T, N> *)(row + c);
}

template <int N, bool WHOLE = false, typename V>
__device__ __forceinline__ V settle(V v, int64_t c, int64_t h) {
  if constexpr (WHOLE) return v;
  if (c < h && c + N > h) {
    for (int64_t cut = c + N - h; cut > 0; --cut) {
#pragma unroll
      for (int j = 0; j + 1 < N; ++j) v[j] = v[j + 1];
      v[N - 1] = (decltype(v[0] + v[0]))0.0f;
    }
  }
  constexpr int kWords = sizeof(V) / 4;
  if constexpr (kWords > 0) {
    typedef uint32_t Words __attribute__((ext_vector_type(kWords)));
    return __builtin_bit_cast(V, __builtin_bit_cast(Words, v) & (c < h ? ~0u : 0u));
  }
  if (c >= h) v = (V)(decltype(v[0] + v[0]))0.0f;
  return v;
}

template <int N, bool WHOLE = false, bool NT = false, typename T>
__device__ __forceinline__ Vec<T, N> load(const T *row, int64_t c, int64_t h) {
  const Vec<T, N> v = load_raw<N, WHOLE, NT>(row, c, h);
  return settle<N, WHOLE>(v, c, h);
}

template <typename T, int N>
__device__ __forceinline__ Vec<T, N> rounded(const float *f) {      // to nearest
  Vec<T, N> v;
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = (T)f[j];
  return v;
}

// Stores those of the elements that lie in the row.
template <int N, bool WHOLE = false, bool NT = false, typename T>
__device__ __forceinline__ void store(T *row, int64_t c, int64_t h, Vec<T, N> v) {
  if (c >= h) return;
  if (WHOLE || c + N <= h) {
    if constexpr (NT)
      __builtin_nontemporal_store(v, (Vec<T, N> *)(row + c));
    else
      *(Vec<T, N> *)(row + c) = v;
  } else {
    for (int64_t at = c; at < h; ++at) {
      row[at] = v[0];
#pragma unroll
      for (int j = 0; j + 1 < N; ++j) v[j] = v[j + 1];
    }
  }
}

template <int N, bool WHOLE = false, bool NT = false, typename T>
__device__ __forceinline__ void store(T *row, int64_t c, int64_t h, const float *f) {
  store<N, WHOLE, NT>(row, c, h, rounded<T, N>(f));
}

// f - about for those of the N elements from column c on that lie in the row, 0
// for the others.
template <int N, bool WHOLE = false>
__device__ __forceinline__ void differences(float *f, float about, int64_t c, int64_t h) {
  if constexpr (WHOLE) about = c < h ? about : 0.0f;      // (f is 0 outside)
#pragma unroll
  for (int j = 0; j < N; ++j) f[j] -= about;
  if (!WHOLE && c + N > h) {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (c + j >= h) f[j] = 0.0f;
  }
}

template <int N, typename V>
__device__ __forceinline__ void widen(V v, float *f) {
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

// Bit j: whether element 8 block + j is kept.  The verdicts are the signs of
// differences of 17-bit numbers, gathered bit by bit (a select through a condition
// takes several times a whole-number operation's time).
__device__ __forceinline__ uint32_t kept_of_block(uint64_t block, const Draw &d) {
  const U4 top = philox4x32_10_v((uint32_t)block, (uint32_t)(block >> 32), 0u, d.call, d.k0, d.k1,
                                 kPhiloxM0, kPhiloxM1);
  uint32_t kept = 0u, most = 0u;
#pragma unroll
  for (int j = 7; j >= 0; --j) {
    const uint32_t off = d.high - 1u - u4_half(top, j);     // negative: kept
    kept = __builtin_amdgcn_alignbit(kept, off, 31);        // kept << 1 | off >> 31
    most = most > off ? most : off;                         // -1: some half is the limit's
  }
  if (most == 0xFFFFFFFFu && d.low) {
    const U4 below = philox4x32_10_v((uint32_t)block, (uint32_t)(block >> 32), 1u, d.call, d.k0,
                                     d.k1, kPhiloxM0, kPhiloxM1);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (u4_half(top, j) == d.high && u4_half(below, j) < d.low) kept &= ~(1u << j);
  }
  return kept;
}

// N elements, kept (bit j of `kept`) and scaled, or 0.
template <int N>
__device__ __forceinline__ void keep(float *f, uint32_t kept, float scale) {
#pragma unroll
  for (int j = 0; j < N; ++j)
    f[j] = __uint_as_float(__float_as_uint(f[j] * scale) &
                           (uint32_t)__builtin_amdgcn_sbfe((int)kept, j, 1));
}

// Dropout of K runs of N elements a lane, run k from element e + k step on, those
// for which inside(k).  aligned: e is a multiple of N, step of 8, and so a pair of
// lanes with runs of four has one block: it draws two runs' blocks at a time.
template <int K, int N, typename F>
__device__ __forceinline__ void drop(float (&f)[K][N], uint64_t e, uint64_t step, bool aligned,
                                     const Draw &d, F inside) {
  if (aligned && N == 4) {
    const bool odd = threadIdx.x & 1;
#pragma unroll
    for (int k = 0; k < K; k += 2) {
      const uint64_t at = e + k * step;
      const uint32_t own = kept_of_block((k + 1 < K && odd ? at + step : at) >> 3, d);
      const uint32_t other = __builtin_amdgcn_update_dpp(0, own, 0xB1, 0xF, 0xF, true);
      const uint32_t here = k + 1 < K && odd ? other : own;
      keep<N>(f[k], odd ? here >> 4 : here, d.scale);
      if (k + 1 < K) {
        const uint32_t next = odd ? own >> 4 : other;
        keep<N>(f[k + 1 < K ? k + 1 : k], next, d.scale);
      }
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (!inside(k)) continue;
    const uint64_t from = e + k * step;
    const uint32_t at = (uint32_t)from & 7u;
    uint32_t kept = kept_of_block(from >> 3, d) >> at;
    if (!aligned && at + N > 8) kept |= kept_of_block((from >> 3) + 1, d) << (8 - at);
    keep<N>(f[k], kept, d.scale);
  }
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

inline bool known_type(int dtype) { return dtype >= LUMA_GRAD_F32 && dtype <= LUMA_GRAD_F16; }

// v of the lane that a DPP control word names (row-local exchanges in the vector
// unit; a shuffle through LDS takes some 100 cycles, and a sum six of them).
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __uint_as_float(
      __builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, 0xF, 0xF, true));
}

// Sum of v over the L lanes (a power of two, at most 64) that hold one row, in
// each of them: pairs and quads, halves of a row of 16 mirrored, the row
// mirrored, then rows and halves of the wavefront exchanged.
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
  if constexpr (L >= 2) v += dpp<0xB1>(v);
  if constexpr (L >= 4) v += dpp<0x4E>(v);
  if constexpr (L >= 8) v += dpp<0x141>(v);
  if constexpr (L >= 16) v += dpp<0x140>(v);
  if constexpr (L >= 32) {
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  }
  if constexpr (L >= 64) {
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  }
  return v;
}

// The same for the 64 lanes' float64 numbers (16 or fewer: the lanes of a row).
template <int CTRL>
__device__ __forceinline__ double dpp(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t low = __builtin_amdgcn_update_dpp(0, (uint32_t)u, CTRL, 0xF, 0xF, true);
  const uint32_t high = __builtin_amdgcn_update_dpp(0, (uint32_t)(u >> 32), CTRL, 0xF, 0xF, true);
  return __builtin_bit_cast(double, (uint64_t)high << 32 | low);
}

template <int L>
__device__ __forceinline__ double lanes_sum(double v) {
  v += dpp<0xB1>(v);
  v += dpp<0x4E>(v);
  if constexpr (L >= 8) v += dpp<0x141>(v);
  if constexpr (L >= 16) v += dpp<0x140>(v);
  auto both = [&](auto low, auto high) {
    v = __builtin_bit_cast(double, (uint64_t)high[0] << 32 | low[0]) +
        __builtin_bit_cast(double, (uint64_t)high[1] << 32 | low[1]);
  };
  if constexpr (L >= 32) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t l = (uint32_t)u, h = (uint32_t)(u >> 32);
    both(__builtin_amdgcn_permlane16_swap(l, l, false, false),
         __builtin_amdgcn_permlane16_swap(h, h, false, false));
  }
  if constexpr (L >= 64) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t l = (uint32_t)u, h = (uint32_t)(u >> 32);
    both(__builtin_amdgcn_permlane32_swap(l, l, false, false),
         __builtin_amdgcn_permlane32_swap(h, h, false, false));
  }
  return v;
}

}  // namespace rows
}  // namespace luma
