// The global norm of many gradients and clipping by it (include/luma.h,
// luma_grad_norm / luma_grad_clip / luma_grad_scale).
//
//   ||g||_p = (sum |g|^p)^(1/p), p = 1, 2, inf, over all rows together;
//   clip:  g <- round(g * c),  c = min(1, max_norm / (||g||_p + 1e-6)).
//
// Bound by HBM: the norm reads every gradient once, clipping reads it again
// and writes it.  The rows are cut into tiles of LUMA_GRAD_TILE elements, and
// each wavefront takes one run of consecutive tiles: it finds its first row by
// a 64-way search (a 20,000-row table takes three loads) and walks on from
// there, so a row of one element costs one iteration and not a workgroup, and
// a long row is read in 16-byte loads, kInFlight of them in flight per lane.
// The norm's loads are non-temporal (2.8e9 bfloat16 take 815 us, 6.9 TB/s; cached
// 914; a kernel that reads and does nothing else reaches 7.0 and 6.2 TB/s; the
// scaling, which finds part of the rows in the last-level cache, is a tenth
// slower so).  Loading rows and tiles a step ahead gained nothing.
// Partial sums go to one double per workgroup; the kernel behind (the join, or
// every workgroup of the scaling) sums those in a fixed order: no atomics, so
// no order that changes from run to run, and no counter to reset.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <string.h>

#include "../../include/luma.h"
#include "luma_error.h"

namespace luma {
namespace {

constexpr int kWaves = 8;                 // wavefronts per workgroup
constexpr int kThreads = 64 * kWaves;
// Two workgroups to a CU (1,024 in two rounds: 141 us for the norm of 20,000
// tensors of 118M float32 together, 512: 112).
constexpr int kBlocks = 512;
constexpr int kInFlight = 8;
constexpr float kTiny = 1e-6f;            // torch's guard against a norm of zero

// (element alignment only: a gradient may be a view anywhere in a bucket)
typedef uint32_t vu4u __attribute__((ext_vector_type(4), aligned(2), may_alias));
typedef uint32_t vu4a __attribute__((ext_vector_type(4), aligned(4), may_alias));

struct Rows {
  LumaGrad row[LUMA_GRADS_INLINE];
};

__device__ __forceinline__ float bf16_float(uint32_t b) { return __uint_as_float(b << 16); }

__device__ __forceinline__ uint32_t float_bf16(float f) {   // to nearest even
  const uint32_t u = __float_as_uint(f);
  return f != f ? 0x7FC0u : (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;
}

// g * c rounded to float32, as torch forms it before it rounds to the
// gradient's type (left alone, the compiler makes one instruction of the
// product and the half conversion, which rounds once).
__device__ __forceinline__ float times(float g, float c) {
  float x = g * c;
  asm("" : "+v"(x));
  return x;
}

// The elements of one 16-byte group by gradient type.
template <int DT>
struct Type;
template <>
struct Type<LUMA_GRAD_F32> {
  typedef float elem;
  typedef vu4a vec;
  static constexpr int kVec = 4;
  static __device__ __forceinline__ float get(const vec &v, int j) { return __uint_as_float(v[j]); }
  static __device__ __forceinline__ void put(vec &v, int j, float f) { v[j] = __float_as_uint(f); }
  static __device__ __forceinline__ float one(elem e) { return e; }
  static __device__ __forceinline__ elem round(float f) { return f; }
};
template <>
struct Type<LUMA_GRAD_BF16> {
  typedef uint16_t elem;
  typedef vu4u vec;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float get(const vec &v, int j) {
    return __uint_as_float(j & 1 ? v[j >> 1] & 0xFFFF0000u : v[j >> 1] << 16);
  }
  static __device__ __forceinline__ void put(vec &v, int j, float f) {
    const uint32_t b = float_bf16(f);
    v[j >> 1] = j & 1 ? v[j >> 1] | (b << 16) : b;
  }
  static __device__ __forceinline__ float one(elem e) { return bf16_float(e); }
  static __device__ __forceinline__ elem round(float f) { return (elem)float_bf16(f); }
};
template <>
struct Type<LUMA_GRAD_F16> {
  typedef uint16_t elem;
  typedef vu4u vec;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float one(elem e) {
    return __half2float(__ushort_as_half(e));
  }
  static __device__ __forceinline__ elem round(float f) {
    return __half_as_ushort(__float2half_rn(f));
  }
  static __device__ __forceinline__ float get(const vec &v, int j) {
    return one((elem)(j & 1 ? v[j >> 1] >> 16 : v[j >> 1] & 0xFFFFu));
  }
  static __device__ __forceinline__ void put(vec &v, int j, float f) {
    const uint32_t b = round(f);
    v[j >> 1] = j & 1 ? v[j >> 1] | (b << 16) : b;
  }
};

// One element into the running sum.  Float64: the square of a float32 is
// exact, and neither overflows nor vanishes; at bfloat16's 3.3e12 elements/s
// the conversions and sums take about a quarter of the vector unit's time.
// The largest |g| is kept by its bits (NaN above infinity).
template <int NORM>
struct Sum {
  double s = 0.0;
  __device__ __forceinline__ void take(float g) {
    const double d = (double)g;
    s = NORM == LUMA_NORM_L2 ? __builtin_fma(d, d, s) : s + __builtin_fabs(d);
  }
  __device__ __forceinline__ double value() const { return s; }
};
template <>
struct Sum<LUMA_NORM_INF> {
  uint32_t s = 0u;
  __device__ __forceinline__ void take(float g) {
    s = max(s, __float_as_uint(g) & 0x7FFFFFFFu);
  }
  __device__ __forceinline__ double value() const { return (double)__uint_as_float(s); }
};

template <int NORM>
__device__ __forceinline__ double join(double a, double b) {
  if (NORM != LUMA_NORM_INF) return a + b;
  return (a >= b || a != a) ? a : b;      // (a NaN stays)
}

// Sum over the workgroup, in thread 0 .. and, through LDS, in every thread.
template <int NORM>
__device__ __forceinline__ double block_sum(double v, double *lds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = join<NORM>(v, __shfl_xor(v, o));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = lds[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) v = join<NORM>(v, lds[w]);
  return v;
}

// The row that holds tile t: the last one with first_tile <= t.  rows[0] has
// first_tile <= t.
__device__ __forceinline__ int find_row(const LumaGrad *rows, int n, int t) {
  const int lane = threadIdx.x & 63;
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) >> 6;
    const int64_t i = (int64_t)lo + (int64_t)lane * step;
    const bool le = i < hi && rows[i].first_tile <= t;
    const int k = __popcll(__ballot(le));
    lo += (k - 1) * step;
    hi = min(hi, lo + step);
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// Runs f(row, first element, end element) over this wavefront's share of the
// tiles [base, base + tiles), upwards or (DOWN) from its end.
template <bool DOWN, typename F>
__device__ __forceinline__ void walk(const LumaGrad *rows, int n, int base, int tiles, F f) {
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int64_t w = (int64_t)blockIdx.x * kWaves + wave, W = (int64_t)gridDim.x * kWaves;
  int t = base + (int)(tiles * w / W);
  int end = base + (int)(tiles * (w + 1) / W);
  if (t >= end) return;
  for (int r = find_row(rows, n, DOWN ? end - 1 : t); t < end; r += DOWN ? -1 : 1) {
    const LumaGrad g = rows[r];
    const int64_t a = (int64_t)max(t - g.first_tile, 0) * LUMA_GRAD_TILE;
    const int64_t b = min(g.numel, (int64_t)(end - g.first_tile) * LUMA_GRAD_TILE);
    f(g, a, b);
    if (DOWN)
      end = g.first_tile;
    else
      t = g.first_tile + (int)((g.numel + LUMA_GRAD_TILE - 1) / LUMA_GRAD_TILE);
  }
}

template <int DT, int NORM>
__device__ __forceinline__ void sum_span(const void *data, int64_t a, int64_t b, Sum<NORM> &sum) {
  typedef Type<DT> T;
  typedef typename T::vec vec;
  constexpr int kStep = 64 * T::kVec;
  const typename T::elem *p = (const typename T::elem *)data;
  const int lane = threadIdx.x & 63;
  int64_t i = a + lane * T::kVec;
  for (; i + (int64_t)(kInFlight - 1) * kStep + T::kVec <= b; i += kInFlight * kStep) {
    vec v[kInFlight];
#pragma unroll
    for (int k = 0; k < kInFlight; ++k) v[k] = __builtin_nontemporal_load((const vec *)(p + i + k * kStep));
#pragma unroll
    for (int k = 0; k < kInFlight; ++k)
#pragma unroll
      for (int j = 0; j < T::kVec; ++j) sum.take(T::get(v[k], j));
  }
  for (; i + T::kVec <= b; i += kStep) {
    const vec v = __builtin_nontemporal_load((const vec *)(p + i));
#pragma unroll
    for (int j = 0; j < T::kVec; ++j) sum.take(T::get(v, j));
  }
  const int64_t last = a + ((b - a) & ~(int64_t)(T::kVec - 1)) + lane;   // the row's partial group
  if (last < b) sum.take(T::one(p[last]));
}

template <int NORM>
__device__ __forceinline__ void norm_body(const LumaGrad *rows, int n, int base, int tiles,
                                          double *partials) {
  __shared__ double lds[kWaves];
  Sum<NORM> sum;
  walk<false>(rows, n, base, tiles, [&](const LumaGrad &g, int64_t a, int64_t b) {
    if (g.dtype == LUMA_GRAD_F32)
      sum_span<LUMA_GRAD_F32>(g.data, a, b, sum);
    else if (g.dtype == LUMA_GRAD_BF16)
      sum_span<LUMA_GRAD_BF16>(g.data, a, b, sum);
    else
      sum_span<LUMA_GRAD_F16>(g.data, a, b, sum);
  });
  const double v = block_sum<NORM>(sum.value(), lds);
  if (threadIdx.x == 0) partials[blockIdx.x] = v;
}

template <int NORM>
__global__ __launch_bounds__(kThreads) void norm_inline(const Rows rows, int n, int base,
                                                        int tiles, double *partials) {
  norm_body<NORM>(rows.row, n, base, tiles, partials);
}

template <int NORM>
__global__ __launch_bounds__(kThreads) void norm_table(const LumaGrad *rows, int n, int tiles,
                                                       double *partials) {
  norm_body<NORM>(rows, n, 0, tiles, partials);
}

// The norm before its root from the workgroups' partial sums, in every thread.
template <int NORM>
__device__ __forceinline__ double total_power(const double *partials, int count) {
  __shared__ double lds[kWaves];
  double v = 0.0;
  for (int i = threadIdx.x; i < count; i += kThreads) v = join<NORM>(v, partials[i]);
  return block_sum<NORM>(v, lds);
}

template <int NORM>
__device__ __forceinline__ float root(double power) {
  return (float)(NORM == LUMA_NORM_L2 ? __builtin_sqrt(power) : power);
}

// min(1, max_norm / (norm + 1e-6)) in float32; a NaN stays.  (torch multiplies by
// the reciprocal, which may be one unit in the last place away.)
__device__ __forceinline__ float clip_factor(float norm, float max_norm) {
  const float c = max_norm / (norm + kTiny);
  return c > 1.0f ? 1.0f : c;
}

template <int NORM>
__global__ __launch_bounds__(kThreads) void join_kernel(const double *partials, int count,
                                                        float max_norm, float *total,
                                                        double *power, const float *grad_scale,
                                                        float *step_scale) {
  const double p = total_power<NORM>(partials, count);
  if (threadIdx.x != 0) return;
  const float scale = grad_scale ? *grad_scale : 1.0f;
  float norm = root<NORM>(p);
  if (grad_scale) norm = (float)((double)norm / (double)scale);
  if (total) *total = norm;
  if (power) *power = p;
  if (step_scale) *step_scale = scale / clip_factor(norm, max_norm);
}

// From the end down: what the norm read last is read first, while the last-level
// cache (256 MB) still holds it (118M float32 in 20,000 rows: 173 us upwards, 165
// down, 5.7 TB/s).
template <int DT>
__device__ __forceinline__ void scale_span(void *data, int64_t a, int64_t b, float c) {
  typedef Type<DT> T;
  typedef typename T::vec vec;
  constexpr int kStep = 64 * T::kVec;
  typename T::elem *p = (typename T::elem *)data;
  const int lane = threadIdx.x & 63;
  const int64_t last = a + ((b - a) & ~(int64_t)(T::kVec - 1)) + lane;   // the row's partial group
  if (last < b) p[last] = T::round(times(T::one(p[last]), c));
  auto scaled = [&](const vec &v) {
    vec o;
#pragma unroll
    for (int j = 0; j < T::kVec; ++j) T::put(o, j, times(T::get(v, j), c));
    return o;
  };
  // whole steps of the wavefront and one that some lanes have
  int64_t i = a + ((b - a) / kStep * kStep) + lane * T::kVec;
  if (i + T::kVec <= b) *(vec *)(p + i) = scaled(*(const vec *)(p + i));
  i -= kStep;
  for (; i - (int64_t)(kInFlight - 1) * kStep >= a; i -= kInFlight * kStep) {
    vec v[kInFlight];
#pragma unroll
    for (int k = 0; k < kInFlight; ++k) v[k] = *(const vec *)(p + i - k * kStep);
#pragma unroll
    for (int k = 0; k < kInFlight; ++k) *(vec *)(p + i - k * kStep) = scaled(v[k]);
  }
  for (; i >= a; i -= kStep) *(vec *)(p + i) = scaled(*(const vec *)(p + i));
}

// NORM < 0: the norm is *total's; else from the partial sums (workgroup 0
// writes it to *total and *power).
template <int NORM>
__device__ __forceinline__ void scale_body(const LumaGrad *rows, int n, int base, int tiles,
                                           const double *partials, int count, float max_norm,
                                           float *total, double *power) {
  float norm;
  if constexpr (NORM < 0) {
    norm = *total;
  } else {
    const double p = total_power<NORM>(partials, count);
    norm = root<NORM>(p);
    if (base == 0 && blockIdx.x == 0 && threadIdx.x == 0) {
      *total = norm;
      if (power) *power = p;
    }
  }
  const float c = clip_factor(norm, max_norm);
  if (c == 1.0f) return;
  walk<true>(rows, n, base, tiles, [&](const LumaGrad &g, int64_t a, int64_t b) {
    if (g.dtype == LUMA_GRAD_F32)
      scale_span<LUMA_GRAD_F32>(g.data, a, b, c);
    else if (g.dtype == LUMA_GRAD_BF16)
      scale_span<LUMA_GRAD_BF16>(g.data, a, b, c);
    else
      scale_span<LUMA_GRAD_F16>(g.data, a, b, c);
  });
}

template <int NORM>
__global__ __launch_bounds__(kThreads) void scale_inline(const Rows rows, int n, int base,
                                                         int tiles, const double *partials,
                                                         int count, float max_norm, float *total,
                                                         double *power) {
  scale_body<NORM>(rows.row, n, base, tiles, partials, count, max_norm, total, power);
}

template <int NORM>
__global__ __launch_bounds__(kThreads) void scale_table(const LumaGrad *rows, int n, int tiles,
                                                        const double *partials, int count,
                                                        float max_norm, float *total,
                                                        double *power) {
  scale_body<NORM>(rows, n, 0, tiles, partials, count, max_norm, total, power);
}

// -- host ---------------------------------------------------------------------

int64_t tiles_of(int64_t numel) { return (numel - 1) / LUMA_GRAD_TILE + 1; }

// Checks the rows and gives their tiles; < 0 (and the error set) if they are
// not what the kernels assume.
int64_t check_args(const LumaNormArgs *a) {
  if (!a || !a->grads) return fail("luma_grad_norm: null arguments"), -1;
  if (a->n <= 0) return fail("luma_grad_norm: no rows"), -1;
  if (!a->total && !a->power) return fail("luma_grad_norm: no output"), -1;
  if (a->norm < LUMA_NORM_L2 || a->norm > LUMA_NORM_INF)
    return fail("luma_grad_norm: unknown norm"), -1;
  if (!a->table && a->n > LUMA_GRADS_NO_TABLE)
    return fail("luma_grad_norm: too many rows without a device table"), -1;
  int64_t tiles = 0;
  for (int32_t i = 0; i < a->n; ++i) {
    const LumaGrad &g = a->grads[i];
    if (!g.data || g.numel <= 0) return fail("luma_grad_norm: an empty row"), -1;
    if (g.dtype < LUMA_GRAD_F32 || g.dtype > LUMA_GRAD_F16)
      return fail("luma_grad_norm: unknown gradient type"), -1;
    if (g.first_tile != tiles) return fail("luma_grad_norm: first_tile does not add up"), -1;
    tiles += tiles_of(g.numel);
    if (tiles > INT32_MAX) return fail("luma_grad_norm: too many elements"), -1;
  }
  return tiles;
}

// The launches of one pass: all rows from the device table, or
// LUMA_GRADS_INLINE at a time; each of at most `most` workgroups.
template <typename FT, typename FI>
void launches(const LumaNormArgs *a, int64_t tiles, FT with_table, FI with_rows) {
  auto blocks = [](int64_t t, int most) {
    const int64_t b = (t + kWaves - 1) / kWaves;
    return (int)(b < most ? b : most);
  };
  if (a->table) {
    with_table(blocks(tiles, kBlocks));
    return;
  }
  const int calls = (a->n + LUMA_GRADS_INLINE - 1) / LUMA_GRADS_INLINE;
  const int most = LUMA_NORM_PARTIALS / calls < kBlocks ? LUMA_NORM_PARTIALS / calls : kBlocks;
  Rows rows;
  for (int c = 0; c < calls; ++c) {
    const int first = c * LUMA_GRADS_INLINE;
    const int n = a->n - first < LUMA_GRADS_INLINE ? a->n - first : LUMA_GRADS_INLINE;
    memcpy(rows.row, a->grads + first, n * sizeof(LumaGrad));
    const int base = a->grads[first].first_tile;
    const int64_t end = first + n < a->n ? a->grads[first + n].first_tile : tiles;
    with_rows(rows, n, base, (int)(end - base), blocks(end - base, most));
  }
}
static_assert(LUMA_GRADS_NO_TABLE / LUMA_GRADS_INLINE <= LUMA_NORM_PARTIALS,
              "a partial sum per launch");
static_assert(sizeof(Rows) <= 4096 - 128, "the launch's arguments");

template <int NORM>
int partial_sums(const LumaNormArgs *a, int64_t tiles, hipStream_t s) {
  int count = 0;
  launches(
      a, tiles,
      [&](int blocks) {
        norm_table<NORM><<<blocks, kThreads, 0, s>>>(a->table, a->n, (int)tiles, a->partials);
        count = blocks;
      },
      [&](const Rows &rows, int n, int base, int t, int blocks) {
        norm_inline<NORM><<<blocks, kThreads, 0, s>>>(rows, n, base, t, a->partials + count);
        count += blocks;
      });
  return count;
}

template <int NORM>
void scale(const LumaNormArgs *a, int64_t tiles, int count, hipStream_t s) {
  launches(
      a, tiles,
      [&](int blocks) {
        scale_table<NORM><<<blocks, kThreads, 0, s>>>(a->table, a->n, (int)tiles, a->partials,
                                                      count, (float)a->max_norm, a->total,
                                                      a->power);
      },
      [&](const Rows &rows, int n, int base, int t, int blocks) {
        scale_inline<NORM><<<blocks, kThreads, 0, s>>>(rows, n, base, t, a->partials, count,
                                                       (float)a->max_norm, a->total, a->power);
      });
}

template <int NORM>
void norm(const LumaNormArgs *a, int64_t tiles, hipStream_t s) {
  const int count = partial_sums<NORM>(a, tiles, s);
  join_kernel<NORM><<<1, kThreads, 0, s>>>(a->partials, count, (float)a->max_norm, a->total,
                                           a->power, a->grad_scale, a->step_scale);
}

template <int NORM>
void clip(const LumaNormArgs *a, int64_t tiles, hipStream_t s) {
  scale<NORM>(a, tiles, partial_sums<NORM>(a, tiles, s), s);
}

}  // namespace
}  // namespace luma

using namespace luma;

extern "C" {

int luma_grad_norm(const LumaNormArgs *a, void *stream) {
  const int64_t tiles = check_args(a);
  if (tiles < 0) return -1;
  if (!a->partials) return fail("luma_grad_norm: null workspace");
  if (a->step_scale && !(a->max_norm >= 0.0)) return fail("luma_grad_norm: max_norm < 0");
  hipStream_t s = (hipStream_t)stream;
  switch (a->norm) {
    case LUMA_NORM_L2: norm<LUMA_NORM_L2>(a, tiles, s); break;
    case LUMA_NORM_L1: norm<LUMA_NORM_L1>(a, tiles, s); break;
    default: norm<LUMA_NORM_INF>(a, tiles, s);
  }
  return check_launch("luma_grad_norm");
}

int luma_grad_clip(const LumaNormArgs *a, void *stream) {
  const int64_t tiles = check_args(a);
  if (tiles < 0) return -1;
  if (!a->partials || !a->total) return fail("luma_grad_clip: null workspace or total");
  if (!(a->max_norm >= 0.0)) return fail("luma_grad_clip: max_norm < 0");
  hipStream_t s = (hipStream_t)stream;
  switch (a->norm) {
    case LUMA_NORM_L2: clip<LUMA_NORM_L2>(a, tiles, s); break;
    case LUMA_NORM_L1: clip<LUMA_NORM_L1>(a, tiles, s); break;
    default: clip<LUMA_NORM_INF>(a, tiles, s);
  }
  return check_launch("luma_grad_clip");
}

int luma_grad_scale(const LumaNormArgs *a, void *stream) {
  const int64_t tiles = check_args(a);
  if (tiles < 0) return -1;
  if (!a->total) return fail("luma_grad_scale: null total");
  if (!(a->max_norm >= 0.0)) return fail("luma_grad_scale: max_norm < 0");
  scale<-1>(a, tiles, 0, (hipStream_t)stream);
  return check_launch("luma_grad_scale");
}

}  // extern "C"
