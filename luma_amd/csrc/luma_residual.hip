// The residual stream's operators (include/luma.h): layer normalisation, alone
// or of the sum that a block's border forms, and dropout.
//
//   total = round(residual + dropout(x));  s = total (or x)
//   m = mean(s),  r = 1 / sqrt(mean((s - m)^2) + eps),  z = (s - m) r
//   y = z weight + bias
//   d_s = r (g - mean(g) - z mean(g z)) + d_total,  g = d_y weight
//   d_weight = sum_rows d_y z,  d_bias = sum_rows d_y
//
// All of them are bound by HBM (a few operations an element, and 30 integer ones
// for a draw): every operand is read once and every result written once.  A
// row lies in the registers of a team of L lanes, K eights of elements a lane,
// between its loads and its stores; rows that no team holds (h > kWidest) are
// read again, from the caches.
#include "luma_error.h"
#include "luma_rows.h"

// Unit 0: the entry points, dropout and the forward; unit 1: the backward (side
// by side: a minute each).
#ifndef LUMA_UNIT
#define LUMA_UNIT 0
#endif

namespace luma {
namespace residual {

using namespace rows;

constexpr int64_t kWidest = 16384;     // elements of a row that a team holds
constexpr int64_t kLargest = (int64_t)1 << 24;
constexpr int kLongThreads = 1024;     // of a workgroup that holds no row
constexpr int kJoinCols = 32, kJoinRows = 32;
constexpr int64_t kMostThreads = (int64_t)1 << 31;   // of one launch

// Which team holds a row of h: the narrowest that does with one eight a lane.
template <int L_, int K_>
struct Team {
  static constexpr int L = L_, K = K_;
  static constexpr int kThreads = L < 256 ? 256 : L;
  static constexpr int kTeams = kThreads / L;
};

inline int lanes_of(int64_t h) {
  int lanes = 8;
  while (lanes < 1024 && lanes * 8 < h) lanes *= 2;
  return lanes;
}

template <typename F>
void with_team(int64_t h, F f) {
  switch (lanes_of(h)) {
    case 8: return f(Team<8, 1>{});
    case 16: return f(Team<16, 1>{});
    case 32: return f(Team<32, 1>{});
    case 64: return f(Team<64, 1>{});
    case 128: return f(Team<128, 1>{});
    case 256: return f(Team<256, 1>{});
    case 512: return f(Team<512, 1>{});
    default: return h <= 8192 ? f(Team<1024, 1>{}) : f(Team<1024, 2>{});
  }
}

// Workgroups that the backward keeps on the chip, each with its own sums of the
// weight's and bias's gradients.
inline int64_t grad_blocks(int64_t n, int64_t h) {
  if (h > kWidest) {      // (norm_long_sums_kernel's shares of the rows)
    const int64_t most = 1024 / ((h + 2047) / 2048);
    return most < 1 ? 1 : n < most ? n : most;
  }
  const int64_t lanes = lanes_of(h), threads = lanes < 256 ? 256 : lanes;
  const int64_t most = 256 * (1024 / threads), need = (n + threads / lanes - 1) / (threads / lanes);
  return need < most ? need : most;
}

// launch(first, blocks) for runs of the workgroups that one launch can hold.
template <typename F>
void in_runs(int64_t blocks, int threads, F launch) {
  const int64_t most = kMostThreads / threads;
  for (int64_t first = 0; first < blocks; first += most)
    launch(first, (uint32_t)(blocks - first < most ? blocks - first : most));
}

// Sum of v over a team's lanes, in all of them; `at`: a float for each of the
// workgroup's wavefronts, used for this sum alone until the next barrier but one.
template <int L>
__device__ __forceinline__ float team_sum(float v, float *at) {
  v = lanes_sum<(L < 64 ? L : 64)>(v);
  if constexpr (L > 64) {
    const int wave = threadIdx.x / 64;
    if (threadIdx.x % 64 == 0) at[wave] = v;
    __syncthreads();
    const int first = wave / (L / 64) * (L / 64);
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < L / 64; ++i) v += at[first + i];
  }
  return v;
}

// Eight of the weight or bias, of float32 or the branch's type.
template <typename B>
__device__ __forceinline__ void load_param(const void *p, bool wide, int64_t c, int64_t h,
                                           float fill, float *f) {
  if (!p) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = fill;
  } else if (wide) {
    widen<8, float>(load<8>((const float *)p, c, h), f);
  } else {
    widen<8, B>(load<8>((const B *)p, c, h), f);
  }
}

// f, kept and scaled or dropped.
__device__ __forceinline__ void drop8(float *f, uint64_t e, const Draw &d) {
  const uint32_t kept = kept_from(e, d);
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = kept >> j & 1u ? f[j] * d.scale : 0.0f;
}

void backward(const LumaLayerNormArgs *a, hipStream_t s);

#if LUMA_UNIT == 0

// -- dropout ----------------------------------------------------------------------

constexpr int kDropThreads = 256;

// U eights a thread, a workgroup's next to each other.
template <typename I, typename O, int U>
__global__ __launch_bounds__(kDropThreads) void dropout_kernel(LumaDropoutArgs a) {
  const I *x = (const I *)a.x;
  const O *residual = (const O *)a.residual;
  O *y = (O *)a.y;
  const bool draws = a.drop.p > 0.0;
  const Draw d = draw_of(a.drop);
  const int64_t first = ((int64_t)blockIdx.x * U * kDropThreads + threadIdx.x) * 8;
  Vec<I, 8> in[U];
  Vec<O, 8> add[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t e = first + u * (kDropThreads * 8);
    in[u] = load<8>(x, e, a.numel);
    if (residual) add[u] = load<8>(residual, e, a.numel);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t e = first + u * (kDropThreads * 8);
    if (e >= a.numel) break;
    float f[8], r[8];
    widen<8, I>(in[u], f);
    if (draws) drop8(f, (uint64_t)e, d);
    if (residual) {
      widen<8, O>(add[u], r);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = r[j] + f[j];
    }
    store<8>(y, e, a.numel, f);
  }
}

template <typename I, typename O>
void dropout(const LumaDropoutArgs *a, hipStream_t s) {
  const int64_t eights = (a->numel + 7) / 8;
  if (eights >= 256 * 1024) {
    const int64_t each = 4 * kDropThreads;
    dropout_kernel<I, O, 4><<<(uint32_t)((eights + each - 1) / each), kDropThreads, 0, s>>>(*a);
  } else {
    dropout_kernel<I, O, 1>
        <<<(uint32_t)((eights + kDropThreads - 1) / kDropThreads), kDropThreads, 0, s>>>(*a);
  }
}

// -- the forward ------------------------------------------------------------------

// The row's elements before its norm: x, or the sum (also stored).
template <typename S, typename B, bool RES>
__device__ __forceinline__ void row_elements(const LumaLayerNormArgs &a, const Draw &d, int64_t row,
                                             int64_t c, float *f) {
  if constexpr (!RES) {
    widen<8, S>(load<8>((const S *)a.x + row * a.ld_x, c, a.h), f);
  } else {
    float r[8];
    widen<8, S>(load<8>((const S *)a.residual + row * a.ld_residual, c, a.h), r);
    widen<8, B>(load<8>((const B *)a.x + row * a.ld_x, c, a.h), f);
    if (a.drop.p > 0.0 && c < a.h) drop8(f, (uint64_t)(row * a.h + c), d);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (float)(S)(r[j] + f[j]);
    store<8>((S *)a.total + row * a.h, c, a.h, f);
  }
}

// The mean of h elements about `about` with the squares about it: m and r.  The
// mean of the differences is not quite 0 where the elements stand far from 0;
// it is put into both.
__device__ __forceinline__ void moments(float about, float first, float second, float h, float eps,
                                        float &off, float &m, float &r) {
  off = first / h;
  float v = second / h - off * off;
  v = v < 0.0f ? 0.0f : v;
  m = about + off;
  r = 1.0f / sqrtf(v + eps);
}

template <typename S, typename B, bool RES, typename T>
__global__ __launch_bounds__(T::kThreads) void norm_kernel(LumaLayerNormArgs a,
                                                             int64_t block) {
  constexpr int L = T::L, K = T::K;
  __shared__ float at[3][T::kThreads / 64];
  const int lane = threadIdx.x % L;
  const int64_t row = (block + blockIdx.x) * T::kTeams + threadIdx.x / L;
  const bool live = row < a.n;
  Draw d;
  if constexpr (RES) d = draw_of(a.drop);
  float f[K][8], sum = 0.0f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t c = (int64_t)(k * L + lane) * 8;
    if (live) {
      row_elements<S, B, RES>(a, d, row, c, f[k]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[k][j] = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += f[k][j];      // (0 past the row)
  }
  float w[K][8], b[K][8];
  const bool wide = a.param == LUMA_GRAD_F32;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t c = (int64_t)(k * L + lane) * 8;
    load_param<B>(a.weight, wide, c, a.h, 1.0f, w[k]);
    load_param<B>(a.bias, wide, c, a.h, 0.0f, b[k]);
  }
  const float h = (float)a.h;
  const float about = team_sum<L>(sum, at[0]) / h;
  float first = 0.0f, second = 0.0f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t c = (int64_t)(k * L + lane) * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      f[k][j] = c + j < a.h ? f[k][j] - about : 0.0f;
      first += f[k][j];
      second = __builtin_fmaf(f[k][j], f[k][j], second);
    }
  }
  first = team_sum<L>(first, at[1]);
  second = team_sum<L>(second, at[2]);
  float off, m, r;
  moments(about, first, second, h, (float)a.eps, off, m, r);
  if (!live) return;
  if (a.stats && lane == 0) {
    a.stats[row] = m;
    a.stats[a.n + row] = r;
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int64_t c = (int64_t)(k * L + lane) * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      f[k][j] = __builtin_fmaf((f[k][j] - off) * r, w[k][j], b[k][j]);
    store<8>((B *)a.y + row * a.h, c, a.h, f[k]);
  }
}

// A row that no team holds, one workgroup each: three passes over it.
template <typename S, typename B, bool RES>
__global__ __launch_bounds__(kLongThreads) void norm_long_kernel(LumaLayerNormArgs a, int64_t block) {
  constexpr int L = kLongThreads, kStep = L * 8;
  __shared__ float at[3][L / 64];
  const int64_t row = block + blockIdx.x;
  Draw d;
  if constexpr (RES) d = draw_of(a.drop);
  const S *s = RES ? (const S *)a.total + row * a.h : (const S *)a.x + row * a.ld_x;
  float f[8], sum = 0.0f;
  for (int64_t c = threadIdx.x * 8; c < a.h; c += kStep) {
    row_elements<S, B, RES>(a, d, row, c, f);
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += f[j];
  }
  const float h = (float)a.h;
  const float about = team_sum<L>(sum, at[0]) / h;
  float first = 0.0f, second = 0.0f;
  // (a thread reads the elements of the sum that it wrote itself)
  for (int64_t c = threadIdx.x * 8; c < a.h; c += kStep) {
    widen<8, S>(load<8>(s, c, a.h), f);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float g = c + j < a.h ? f[j] - about : 0.0f;
      first += g;
      second = __builtin_fmaf(g, g, second);
    }
  }
  first = team_sum<L>(first, at[1]);
  second = team_sum<L>(second, at[2]);
  float off, m, r;
  moments(about, first, second, h, (float)a.eps, off, m, r);
  if (a.stats && threadIdx.x == 0) {
    a.stats[row] = m;
    a.stats[a.n + row] = r;
  }
  const bool wide = a.param == LUMA_GRAD_F32;
  for (int64_t c = threadIdx.x * 8; c < a.h; c += kStep) {
    float w[8], b[8];
    load_param<B>(a.weight, wide, c, a.h, 1.0f, w);
    load_param<B>(a.bias, wide, c, a.h, 0.0f, b);
    widen<8, S>(load<8>(s, c, a.h), f);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      f[j] = __builtin_fmaf((f[j] - about - off) * r, w[j], b[j]);
    store<8>((B *)a.y + row * a.h, c, a.h, f);
  }
}

template <typename S, typename B, bool RES>
void forward(const LumaLayerNormArgs *a, hipStream_t s) {
  if (a->h > kWidest) {
    in_runs(a->n, kLongThreads, [&](int64_t first, uint32_t blocks) {
      norm_long_kernel<S, B, RES><<<blocks, kLongThreads, 0, s>>>(*a, first);
    });
    return;
  }
  with_team(a->h, [&](auto team) {
    typedef decltype(team) T;
    in_runs((a->n + T::kTeams - 1) / T::kTeams, T::kThreads, [&](int64_t first, uint32_t blocks) {
      norm_kernel<S, B, RES, T><<<blocks, T::kThreads, 0, s>>>(*a, first);
    });
  });
}

// -- checks -----------------------------------------------------------------------

bool check_drop(const LumaDropout &d) {
  if (!(d.p >= 0.0 && d.p <= 1.0)) return fail("luma: the share dropped is not in [0, 1]"), false;
  if (d.reserved) return fail("luma: reserved fields must be 0"), false;
  return true;
}

bool check_types(int32_t stream, int32_t branch) {
  if (!known_type(stream) || !known_type(branch)) return fail("luma: unknown type"), false;
  if (stream != branch && stream != LUMA_GRAD_F32)
    return fail("luma: the stream's type is neither float32 nor the branch's"), false;
  return true;
}

bool check_args(const LumaLayerNormArgs *a, bool backward) {
  if (!a) return fail("luma_layer_norm: null arguments"), false;
  if (a->n < 1 || a->h < 1) return fail("luma_layer_norm: empty operands"), false;
  if (a->n > INT32_MAX || a->h > kLargest)
    return fail("luma_layer_norm: operands too large"), false;
  if (!check_types(a->stream, a->branch) || !check_drop(a->drop)) return false;
  if (a->param != LUMA_GRAD_F32 && a->param != a->branch)
    return fail("luma_layer_norm: the weight's type is neither float32 nor the branch's"), false;
  if (!(a->eps >= 0.0)) return fail("luma_layer_norm: eps is negative"), false;
  if (a->reserved) return fail("luma_layer_norm: reserved fields must be 0"), false;
  const bool adds = a->residual != nullptr || (backward && a->total != nullptr);
  if (a->drop.p > 0.0 && !adds)
    return fail("luma_layer_norm: dropout is of a branch, beside a residual"), false;
  if (!backward) {
    if (!a->x || !a->y || (adds && !a->total))
      return fail("luma_layer_norm: null operand"), false;
    // (rows may lie on each other: an expanded operand is only read)
    if (a->n > 1 && (a->ld_x < 0 || (adds && a->ld_residual < 0)))
      return fail("luma_layer_norm: rows lie backwards"), false;
  } else {
    if (!(adds ? a->total : a->x) || !a->d_y || !a->stats)
      return fail("luma_layer_norm: null operand"), false;
    if (!adds && (a->d_total || a->d_residual))
      return fail("luma_layer_norm: gradients of a sum without one"), false;
  }
  return true;
}

#endif  // LUMA_UNIT == 0

#if LUMA_UNIT == 1

// -- the backward -----------------------------------------------------------------

// One row's share of the gradients in a lane's eight columns: from s and d_y,
// z and g, and into the sums over the rows.
struct Eight {
  float z[8], g[8];
};

template <typename S, typename B>
__device__ __forceinline__ void eight(const Vec<S, 8> &s, const Vec<B, 8> &dy, const float *w,
                                      float m, float r, Eight &o, float *dw, float *db, float &s1,
                                      float &s2) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float d = (float)dy[j];
    o.z[j] = ((float)s[j] - m) * r;
    o.g[j] = d * w[j];
    s1 += o.g[j];
    s2 = __builtin_fmaf(o.g[j], o.z[j], s2);
    dw[j] = __builtin_fmaf(d, o.z[j], dw[j]);
    db[j] += d;
  }
}

// d_s of eight columns, and what is stored of it.
template <typename S, typename B>
__device__ __forceinline__ void finish(const LumaLayerNormArgs &a, const Draw &d, int64_t row,
                                       int64_t c, const Eight &e, const Vec<S, 8> &dt, float r,
                                       float mean_g, float mean_gz) {
  float f[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    f[j] = r * (e.g[j] - mean_g - e.z[j] * mean_gz);
    if (a.d_total) f[j] += (float)dt[j];
  }
  if (!a.total) {
    store<8>((S *)a.d_x + row * a.h, c, a.h, f);
    return;
  }
  if (a.d_residual) store<8>((S *)a.d_residual + row * a.h, c, a.h, f);
  if (a.d_x) {
    if (a.drop.p > 0.0 && c < a.h) drop8(f, (uint64_t)(row * a.h + c), d);
    store<8>((B *)a.d_x + row * a.h, c, a.h, f);
  }
}

// A team's sums over its rows go into LDS, those of the workgroup's teams
// together to the workspace: [block][d_weight, d_bias][h].
template <typename T>
__device__ __forceinline__ void put_sums(const float (&v)[T::K][8], float *lds, float *out,
                                         int64_t h) {
  constexpr int L = T::L, K = T::K, kRow = L * K * 8;
  if constexpr (T::kTeams == 1) {
#pragma unroll
    for (int k = 0; k < K; ++k)
      store<8>(out, (int64_t)(k * L + threadIdx.x) * 8, h, v[k]);
  } else {
    const int lane = threadIdx.x % L, team = threadIdx.x / L;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j) lds[team * kRow + (k * L + lane) * 8 + j] = v[k][j];
    __syncthreads();
    for (int64_t c = threadIdx.x; c < h; c += T::kThreads) {
      float sum = 0.0f;
#pragma unroll 8
      for (int t = 0; t < T::kTeams; ++t) sum += lds[t * kRow + c];
      out[c] = sum;
    }
  }
}

template <typename S, typename B, typename T>
__global__ __launch_bounds__(T::kThreads) void norm_grad_kernel(LumaLayerNormArgs a) {
  constexpr int L = T::L, K = T::K;
  __shared__ float at[2][2][T::kThreads / 64];
  __shared__ float lds[T::kTeams == 1 ? 1 : T::kThreads * K * 8];
  const int lane = threadIdx.x % L, team = threadIdx.x / L;
  const S *s = a.total ? (const S *)a.total : (const S *)a.x;
  const int64_t ld = a.total ? a.h : a.ld_x;
  const B *dy = (const B *)a.d_y;
  const bool stores = a.d_x || a.d_residual;
  Draw d;
  if (a.drop.p > 0.0) d = draw_of(a.drop);
  const bool wide = a.param == LUMA_GRAD_F32;
  float w[K][8], dw[K][8], db[K][8];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    load_param<B>(a.weight, wide, (int64_t)(k * L + lane) * 8, a.h, 1.0f, w[k]);
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[k][j] = db[k][j] = 0.0f;
  }
  const float h = (float)a.h;
  int turn = 0;
  for (int64_t base = (int64_t)blockIdx.x * T::kTeams; base < a.n;
       base += (int64_t)gridDim.x * T::kTeams) {
    const int64_t row = base + team;
    const bool live = row < a.n;
    Vec<S, 8> vs[K], vt[K];
    Vec<B, 8> vd[K];
    float m = 0.0f, r = 0.0f;
    if (live) {
      m = a.stats[row];
      r = a.stats[a.n + row];
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t c = (int64_t)(k * L + lane) * 8;
      const int64_t end = live ? a.h : 0;      // (a row past the last: zeros)
      vs[k] = load<8>(s + row * ld, c, end);
      vd[k] = load<8>(dy + row * a.h, c, end);
      if (a.d_total) vt[k] = load<8>((const S *)a.d_total + row * a.h, c, end);
    }
    Eight e[K];
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
      eight<S, B>(vs[k], vd[k], w[k], m, r, e[k], dw[k], db[k], s1, s2);
    if (stores) {
      s1 = lanes_sum<(L < 64 ? L : 64)>(s1);
      s2 = lanes_sum<(L < 64 ? L : 64)>(s2);
      if constexpr (L > 64) {
        // (one barrier a row: the next row's sums go to the other half)
        const int wave = threadIdx.x / 64;
        if (threadIdx.x % 64 == 0) {
          at[turn][0][wave] = s1;
          at[turn][1][wave] = s2;
        }
        __syncthreads();
        const int first = wave / (L / 64) * (L / 64);
        s1 = s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < L / 64; ++i) {
          s1 += at[turn][0][first + i];
          s2 += at[turn][1][first + i];
        }
        turn ^= 1;
      }
      if (live) {
#pragma unroll
        for (int k = 0; k < K; ++k)
          finish<S, B>(a, d, row, (int64_t)(k * L + lane) * 8, e[k], vt[k], r, s1 / h, s2 / h);
      }
    }
  }
  float *out = (float *)a.workspace + (int64_t)blockIdx.x * 2 * a.h;
  if (a.d_weight) put_sums<T>(dw, lds, out, a.h);
  if (a.d_bias) put_sums<T>(db, lds, out + a.h, a.h);
}

// A row that no team holds: d_s in two passes over it.
template <typename S, typename B>
__global__ __launch_bounds__(kLongThreads) void norm_long_grad_kernel(LumaLayerNormArgs a,
                                                                  int64_t block) {
  constexpr int L = kLongThreads, kStep = L * 8;
  __shared__ float at[2][L / 64];
  const int64_t row = block + blockIdx.x;
  const S *s = a.total ? (const S *)a.total + row * a.h : (const S *)a.x + row * a.ld_x;
  const B *dy = (const B *)a.d_y + row * a.h;
  const bool wide = a.param == LUMA_GRAD_F32;
  Draw d;
  if (a.drop.p > 0.0) d = draw_of(a.drop);
  const float m = a.stats[row], r = a.stats[a.n + row], h = (float)a.h;
  float s1 = 0.0f, s2 = 0.0f, dw[8] = {}, db[8] = {};
  auto at_column = [&](int64_t c, Eight &e) {
    float w[8];
    load_param<B>(a.weight, wide, c, a.h, 1.0f, w);
    eight<S, B>(load<8>(s, c, a.h), load<8>(dy, c, a.h), w, m, r, e, dw, db, s1, s2);
  };
  Eight e;
  for (int64_t c = threadIdx.x * 8; c < a.h; c += kStep) at_column(c, e);
  s1 = team_sum<L>(s1, at[0]);
  s2 = team_sum<L>(s2, at[1]);
  const float mean_g = s1 / h, mean_gz = s2 / h;
  for (int64_t c = threadIdx.x * 8; c < a.h; c += kStep) {
    at_column(c, e);
    Vec<S, 8> dt;
    if (a.d_total) dt = load<8>((const S *)a.d_total + row * a.h, c, a.h);
    finish<S, B>(a, d, row, c, e, dt, r, mean_g, mean_gz);
  }
}

// Its share of d_weight and d_bias: 2,048 columns a workgroup, the rows shared
// out over gridDim.y.
template <typename S, typename B>
__global__ __launch_bounds__(256) void norm_long_sums_kernel(LumaLayerNormArgs a) {
  const int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (c >= a.h) return;
  const int64_t ld = a.total ? a.h : a.ld_x;
  const S *s = a.total ? (const S *)a.total : (const S *)a.x;
  const float one[8] = {1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f, 1.0f};
  float s1 = 0.0f, s2 = 0.0f, dw[8] = {}, db[8] = {};
  Eight e;
  for (int64_t row = blockIdx.y; row < a.n; row += gridDim.y)
    eight<S, B>(load<8>(s + row * ld, c, a.h), load<8>((const B *)a.d_y + row * a.h, c, a.h), one,
                a.stats[row], a.stats[a.n + row], e, dw, db, s1, s2);
  float *out = (float *)a.workspace + (int64_t)blockIdx.y * 2 * a.h;
  store<8>(out, c, a.h, dw);
  store<8>(out + a.h, c, a.h, db);
}

// d_weight and d_bias from the workgroups' sums: 32 columns a workgroup, whose 32
// rows of threads take every 32nd sum each, in a fixed order.
template <typename P>
__global__ __launch_bounds__(kJoinCols *kJoinRows) void join_kernel(const float *part,
                                                                    int64_t blocks, int64_t h,
                                                                    P *d_weight, P *d_bias) {
  __shared__ float lds[kJoinRows][kJoinCols + 1];
  const int col = threadIdx.x % kJoinCols, from = threadIdx.x / kJoinCols;
  const int64_t c = (int64_t)blockIdx.x * kJoinCols + col;
  P *out = blockIdx.y ? d_bias : d_weight;
  if (!out) return;
  float sum = 0.0f;
  if (c < h) {
    const float *p = part + (int64_t)blockIdx.y * h + c;
#pragma unroll 8
    for (int64_t b = from; b < blocks; b += kJoinRows) sum += p[b * 2 * h];
  }
  lds[from][col] = sum;
  __syncthreads();
  if (from == 0 && c < h) {
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kJoinRows; ++i) sum += lds[i][col];
    out[c] = (P)sum;
  }
}

void backward(const LumaLayerNormArgs *a, hipStream_t stream) {
  const int64_t blocks = grad_blocks(a->n, a->h);
  const bool sums = a->d_weight || a->d_bias, stores = a->d_x || a->d_residual;
  if (!sums && !stores) return;
  with_types(a->stream, a->branch, [&](auto s, auto b) {
    typedef decltype(s) S;
    typedef decltype(b) B;
    if (a->h > kWidest) {
      if (stores)
        in_runs(a->n, kLongThreads, [&](int64_t first, uint32_t count) {
          norm_long_grad_kernel<S, B><<<count, kLongThreads, 0, stream>>>(*a, first);
        });
      if (sums)
        norm_long_sums_kernel<S, B><<<dim3((uint32_t)((a->h + 2047) / 2048), (uint32_t)blocks), 256,
                                      0, stream>>>(*a);
      return;
    }
    with_team(a->h, [&](auto team) {
      typedef decltype(team) T;
      norm_grad_kernel<S, B, T><<<(uint32_t)blocks, T::kThreads, 0, stream>>>(*a);
    });
  });
  if (!sums) return;
  with_type(a->param, [&](auto p) {
    typedef decltype(p) P;
    const dim3 grid((uint32_t)((a->h + kJoinCols - 1) / kJoinCols), 2);
    join_kernel<P><<<grid, kJoinCols * kJoinRows, 0, stream>>>(
        (const float *)a->workspace, blocks, a->h, (P *)a->d_weight, (P *)a->d_bias);
  });
}

#endif  // LUMA_UNIT == 1

}  // namespace residual
}  // namespace luma

#if LUMA_UNIT == 0

using namespace luma;
using namespace luma::residual;

extern "C" {

int luma_dropout(const LumaDropoutArgs *a, void *stream) {
  if (!a) return fail("luma_dropout: null arguments");
  if (a->numel < 1) return fail("luma_dropout: empty operands");
  if (a->numel > (int64_t)1 << 36) return fail("luma_dropout: operands too large");
  if (!check_drop(a->drop)) return -1;
  if (!known_type(a->in) || !known_type(a->out) ||
      (a->in != a->out && a->in != LUMA_GRAD_F32 && a->out != LUMA_GRAD_F32))
    return fail("luma_dropout: unknown types");
  if (!a->x || !a->y) return fail("luma_dropout: null operand");
  with_type(a->in, [&](auto i) {
    with_type(a->out, [&](auto o) {
      typedef decltype(i) I;
      typedef decltype(o) O;
      if constexpr (std::is_same<I, O>::value || std::is_same<I, float>::value ||
                    std::is_same<O, float>::value)
        dropout<I, O>(a, (hipStream_t)stream);
    });
  });
  return check_launch("luma_dropout");
}

int64_t luma_layer_norm_workspace_bytes(const LumaLayerNormArgs *a) {
  if (!a) return fail("luma_layer_norm: null arguments"), -1;
  if (a->n < 1 || a->h < 1) return fail("luma_layer_norm: empty operands"), -1;
  if (a->n > INT32_MAX || a->h > kLargest)
    return fail("luma_layer_norm: operands too large"), -1;
  return grad_blocks(a->n, a->h) * 2 * a->h * (int64_t)sizeof(float);
}

int luma_layer_norm_forward(const LumaLayerNormArgs *a, void *stream) {
  if (!check_args(a, false)) return -1;
  with_types(a->stream, a->branch, [&](auto s, auto b) {
    typedef decltype(s) S;
    typedef decltype(b) B;
    if (a->residual)
      forward<S, B, true>(a, (hipStream_t)stream);
    else
      forward<S, B, false>(a, (hipStream_t)stream);
  });
  return check_launch("luma_layer_norm_forward");
}

int luma_layer_norm_backward(const LumaLayerNormArgs *a, void *stream) {
  if (!check_args(a, true)) return -1;
  if ((a->d_weight || a->d_bias) &&
      (!a->workspace || (uintptr_t)a->workspace % 16 ||
       a->workspace_bytes < luma_layer_norm_workspace_bytes(a)))
    return fail("luma_layer_norm_backward: workspace too small or not aligned");
  backward(a, (hipStream_t)stream);
  return check_launch("luma_layer_norm_backward");
}

}  // extern "C"

#endif  // LUMA_UNIT == 0
