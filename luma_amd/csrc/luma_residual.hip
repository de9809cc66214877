// The residual stream's operators (include/luma.h): layer normalisation, alone
// or of the sum that a block's border forms, and dropout.
//
//   total = round(residual + dropout(x));  s = total (or x)
//   m = mean(s),  r = 1 / sqrt(mean((s - m)^2) + eps),  z = (s - m) r
//   y = z weight + bias
//   d_s = r (g - mean(g) - z mean(g z)) + d_total,  g = d_y weight
//   d_weight = sum_rows d_y z,  d_bias = sum_rows d_y
//
// All of them are bound by HBM (a few operations an element, and for a draw ten
// rounds of the generator for eight): every operand is read once and every result written once.  A
// row lies in the registers of a team of L lanes, K runs of 16 bytes a lane, between
// its loads and its stores, the next row's loads under way; rows that no team holds
// (h > kWidest) are read again, from the caches.  Measured: 16,384 x 4,096 bfloat16
// (residual + x, no draws) 93 to 94 us forward, 5.8 TB/s, and 90 to 93 backward, 5.9 (kernels
// that only move as much, two tensors in and two out or three and one, 91 and 86);
// 8,192 x 4,096 of a float32 stream and a bfloat16 branch 68 us forward, 6.0; dropout
// of 100M bfloat16 64 to 68 us, 6.3 to 5.9.  Small ones are launches: 2,048 x 128
// float32 3.5 us, backward 3.9 and 3.0 (the join).  Not kept: sums by shuffles through
// LDS (8,192 x 768, float32 and bfloat16, with draws: backward 33 us, by moves in the
// vector unit 28); a wavefront a row of 4,096 (forward 191 us).
#include "luma_error.h"
#include "luma_rows.h"

// Units, compiled side by side (a minute each): 0 holds the entry points and
// dropout, 1 to 3 the forward of a branch of float32, bfloat16 and float16, 4 to 6
// the backward.
#ifndef LUMA_UNIT
#define LUMA_UNIT 0
#endif
#define LUMA_FORWARD (LUMA_UNIT >= 1 && LUMA_UNIT <= 3)
#define LUMA_BACKWARD (LUMA_UNIT >= 4)

namespace luma {
namespace residual {

using namespace rows;

// Elements of a row that a team holds.  2,048 x 16,384 float32 onto a residual 95 us
// forward and 119 backward, by the kernels of longer rows 124 and 198.  A lane then has
// 32 float32 of everything and spills: up to 96 bytes forward and 236 backward, of cut
// rows 876 and 984 (16,381 columns 237 and 326 us, by the kernels of longer rows 129
// and 203).
constexpr int64_t kWidest = 16384;
constexpr int64_t kLargest = (int64_t)1 << 24;
// Of a workgroup that holds no row.  64 x 65,536 float32 onto a residual 30 us forward
// and 48 backward, with 512 threads 42 and 55; 1,024 x 32,768 134 and 206, 137 and 207.
constexpr int kLongThreads = 1024;
// Of a workgroup that joins sums.  2,048 x 128 float32, the backward with its join 5.6 us,
// with 64 x 16 threads 5.5, with 16 x 64 6.4; 16,384 x 4,096 175, 175 and 177.
constexpr int kJoinCols = 32, kJoinRows = 32;
constexpr int64_t kMostThreads = (int64_t)1 << 31;   // of one launch

// Elements that a lane has next to each other: 16 bytes of the stream's type, so
// that each load or store of a wavefront is one run of memory.  (Eight float32 a
// lane, in two loads of every other 16 bytes: 8,192 x 4,096 of a float32 stream
// and a bfloat16 branch 77 us with non-temporal accesses, 74 without.)
template <typename S>
constexpr int kVec = 16 / sizeof(S);

// A team of L lanes holds a row, K runs of V elements a lane (WHOLE: rows of whole
// runs).
template <int L_, int K_, int V_, bool WHOLE_>
struct Team {
  static constexpr int L = L_, K = K_, V = V_;
  static constexpr bool WHOLE = WHOLE_;
  static constexpr int kRow = L * K * V;
  static constexpr int kThreads = L < 256 ? 256 : L;
  static constexpr int kTeams = kThreads / L;

  // The column of this thread's run k.
  static __device__ __forceinline__ int64_t column(int k) {
    return (k * L + (int)(threadIdx.x % L)) * V;
  }
};

// f(team) of the narrowest team that holds a row of h.  Lanes without elements cost
// their instructions (8,192 x 768 in teams for 2,048 took 1.4 times as long), a
// wavefront needs no barrier for its sums (8,192 x 768 bfloat16 backward 15.7 us
// in teams of 64 lanes, 21.7 in 128), and a lane of a wide row has eight elements at
// least, for what a row costs besides (and, of float32, two runs: drop()), and as few
// as that, for the backward's five numbers an element (16,384 x 4,096 bfloat16: 512
// lanes 90 and 86 us, 256 lanes 95 and 88).
template <int V, bool WHOLE, typename F>
void with_team(int64_t h, F f) {
  const int64_t runs = (h + V - 1) / V;
  if (runs <= 8) return f(Team<8, 1, V, WHOLE>{});
  if (runs <= 16) return f(Team<16, 1, V, WHOLE>{});
  if (runs <= 32) return f(Team<32, 1, V, WHOLE>{});
  if (runs <= 64) return f(Team<64, 1, V, WHOLE>{});
  if (runs <= 128) return f(Team<64, 2, V, WHOLE>{});
  if (runs <= 192) return f(Team<64, 3, V, WHOLE>{});
  if constexpr (V == 4) {
    if (runs <= 256) return f(Team<128, 2, V, WHOLE>{});
    if (runs <= 384) return f(Team<128, 3, V, WHOLE>{});
    if (runs <= 512) return f(Team<256, 2, V, WHOLE>{});
  } else {
    if (runs <= 256) return f(Team<256, 1, V, WHOLE>{});
    if (runs <= 512) return f(Team<512, 1, V, WHOLE>{});
  }
  if (runs <= 768) return f(Team<256, 3, V, WHOLE>{});
  if (runs <= 1024) return f(Team<512, 2, V, WHOLE>{});
  if (runs <= 1536) return f(Team<512, 3, V, WHOLE>{});
  if (V == 8 || runs <= 2048) return f(Team<512, 4, V, WHOLE>{});
  if constexpr (V == 4) f(Team<512, 8, V, WHOLE>{});
}

template <int V, typename F>
void with_team(int64_t h, F f) {
  if (h < V)      // (no run of V: an element a lane)
    f(Team<8, 1, 1, true>{});
  else if (h % V == 0)
    with_team<V, true>(h, f);
  else
    with_team<V, false>(h, f);
}

// Whether a call's operands (so many of the stream's type and of the branch's) are
// more than the last-level cache holds: they then go past it (16,384 x 4,096
// bfloat16, 537 MB: backward 91 us, cached 101; of 75 MB the forward takes 14.5 us so
// and 13.4 cached).  Rows of whole runs in teams of a wavefront and more have kernels for
// that.  The others would gain less or are fewer, and have none (bfloat16 onto a residual,
// forward and backward: 16,384 x 4,093 132 and 137 us, past the cache 126 and 134; 51,105
// x 1,078 100 and 95, so 102 and 93; 1,048,576 x 64 100 and 98, so 95 and 86).
inline bool apart(const LumaLayerNormArgs *a, int streams, int branches) {
  const int64_t size = streams * (a->stream == LUMA_GRAD_F32 ? 4 : 2) +
                       branches * (a->branch == LUMA_GRAD_F32 ? 4 : 2);
  return a->n * a->h * size > (int64_t)256 << 20;
}

// Workgroups of T that a call of n rows is given: `threads` threads of each of the
// 256 CUs, or fewer.
template <typename T>
int64_t blocks_of(int64_t n, int threads) {
  const int64_t most = 256 * (threads < T::kThreads ? 1 : threads / T::kThreads);
  const int64_t need = (n + T::kTeams - 1) / T::kTeams;
  return need < most ? need : most;
}

// (The backward: more workgroups are more sums to join; 16,384 x 4,096 bfloat16 in
// teams of 256 lanes 91 us and 2.7 for the join, with twice as many 95 and 3.4.)
constexpr int kForwardThreads = 1024, kGradThreads = 512;

// Workgroups of the backward, each with its own sums of the weight's and bias's
// gradients.
inline int64_t grad_blocks(int64_t n, int64_t h, int stream) {
  if (h > kWidest) {      // (norm_long_sums_kernel's shares of the rows)
    const int64_t most = 1024 / ((h + 2047) / 2048);
    return most < 1 ? 1 : n < most ? n : most;
  }
  int64_t blocks = 0;
  auto count = [&](auto team) { blocks = blocks_of<decltype(team)>(n, kGradThreads); };
  if (stream == LUMA_GRAD_F32)
    with_team<4>(h, count);
  else
    with_team<8>(h, count);
  return blocks;
}

// launch(first, blocks) for runs of the workgroups that one launch can hold.
template <typename F>
void in_runs(int64_t blocks, int threads, F launch) {
  const int64_t most = kMostThreads / threads;
  for (int64_t first = 0; first < blocks; first += most)
    launch(first, (uint32_t)(blocks - first < most ? blocks - first : most));
}

// Sum of v over a team's lanes, in all of them; `at`: a float for each of the
// workgroup's wavefronts, that no wavefront writes again before the next barrier.
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

// Two at once.
template <int L>
__device__ __forceinline__ void team_sum2(float &u, float &v, float *at_u, float *at_v) {
  u = lanes_sum<(L < 64 ? L : 64)>(u);
  v = lanes_sum<(L < 64 ? L : 64)>(v);
  if constexpr (L > 64) {
    const int wave = threadIdx.x / 64;
    if (threadIdx.x % 64 == 0) {
      at_u[wave] = u;
      at_v[wave] = v;
    }
    __syncthreads();
    const int first = wave / (L / 64) * (L / 64);
    u = v = 0.0f;
#pragma unroll
    for (int i = 0; i < L / 64; ++i) {
      u += at_u[first + i];
      v += at_v[first + i];
    }
  }
}

// The elements of the weight (1 without one) and the bias (0) at the columns of K
// runs, of P; all loads go out before the first is looked at.
template <int K, int V, bool WHOLE, typename P, typename F>
__device__ __forceinline__ void params_of(const P *weight, const P *bias, int64_t h, F column,
                                          float (&w)[K][V], float (&b)[K][V]) {
  constexpr int N = V * sizeof(P) > 16 ? 4 : V, R = V / N;
  // (without one the other is read in its place: no condition, see load_raw)
  const P *pw = weight ? weight : bias, *pb = bias ? bias : weight;
  Vec<P, N> raw_w[K][R], raw_b[K][R];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < R; ++i) {
      raw_w[k][i] = load_raw<N, WHOLE>(pw, column(k) + i * N, h);
      raw_b[k][i] = load_raw<N, WHOLE>(pb, column(k) + i * N, h);
    }
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < R; ++i) {
      widen<N>(settle<N, WHOLE>(raw_w[k][i], column(k) + i * N, h), w[k] + i * N);
      widen<N>(settle<N, WHOLE>(raw_b[k][i], column(k) + i * N, h), b[k] + i * N);
    }
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (!weight) w[k][j] = 1.0f;
      if (!bias) b[k][j] = 0.0f;
    }
}

// Of float32 or of the branch's type B.
template <int K, int V, bool WHOLE, typename B, typename F>
__device__ __forceinline__ void load_params(const void *weight, const void *bias, bool wide,
                                            int64_t h, F column, float (&w)[K][V],
                                            float (&b)[K][V]) {
  if (!weight && !bias) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        w[k][j] = 1.0f;
        b[k][j] = 0.0f;
      }
  } else if (std::is_same<B, float>::value || wide) {
    params_of<K, V, WHOLE>((const float *)weight, (const float *)bias, h, column, w, b);
  } else {
    params_of<K, V, WHOLE>((const B *)weight, (const B *)bias, h, column, w, b);
  }
}

// The forward and the backward of a branch of type B (units 1 to 6).
template <typename B>
void forward_of(const LumaLayerNormArgs *a, hipStream_t s);
template <typename B>
void backward_of(const LumaLayerNormArgs *a, hipStream_t s);

#if LUMA_UNIT == 0

// -- dropout ----------------------------------------------------------------------

constexpr int kDropThreads = 256, kDropRuns = 2;
constexpr int64_t kL2Bytes = (int64_t)32 << 20;      // of all XCDs

// Two runs a thread, a workgroup's next to each other: a pair of lanes has one
// draw for each of float32's runs, and two are under way at a time (100M bfloat16,
// 403 MB: one run 88 us, two 64, four 65, eight 70; 4.1M onto a residual 6.0, 6.0,
// 6.8, 10).  A run is 16 bytes of the wider type (its lanes' 8 bytes of the other are
// one run of memory, too).  What the L2 caches do not hold goes past them (100M
// bfloat16 64 us, cached 74; 8 MB the same).
template <typename I, typename O, int V, bool NT>
__global__ __launch_bounds__(kDropThreads) void dropout_kernel(LumaDropoutArgs a) {
  constexpr int U = kDropRuns;
  const I *x = (const I *)a.x;
  const O *residual = (const O *)a.residual;
  O *y = (O *)a.y;
  const bool draws = a.drop.p > 0.0;
  const Draw d = draw_of(a.drop);
  const int64_t first = ((int64_t)blockIdx.x * U * kDropThreads + threadIdx.x) * V;
  Vec<I, V> in[U];
  Vec<O, V> add[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t e = first + u * (kDropThreads * V);
    in[u] = load<V, false, NT>(x, e, a.numel);
    if (residual) add[u] = load<V, false, NT>(residual, e, a.numel);
  }
  float f[U][V];
#pragma unroll
  for (int u = 0; u < U; ++u) widen<V>(in[u], f[u]);
  constexpr int kStep = kDropThreads * V;
  if (draws) drop(f, first, kStep, true, d, [&](int u) { return first + u * kStep < a.numel; });
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t e = first + u * kStep;
    if (e >= a.numel) break;
    if (residual) {
#pragma unroll
      for (int j = 0; j < V; ++j) f[u][j] = (float)add[u][j] + f[u][j];
    }
    store<V, false, NT>(y, e, a.numel, f[u]);
  }
}

template <typename I, typename O>
void dropout(const LumaDropoutArgs *a, hipStream_t s) {
  constexpr int V = kVec<I> < kVec<O> ? kVec<I> : kVec<O>;
  const int64_t bytes = a->numel * (int64_t)(sizeof(I) + sizeof(O) * (a->residual ? 2 : 1));
  const int64_t each = (int64_t)kDropThreads * kDropRuns * V;
  // (fewer elements than a run has: one workgroup, an element a lane)
  const auto kernel = a->numel < V       ? dropout_kernel<I, O, 1, false>
                      : bytes > kL2Bytes ? dropout_kernel<I, O, V, true>
                                         : dropout_kernel<I, O, V, false>;
  kernel<<<(uint32_t)((a->numel + each - 1) / each), kDropThreads, 0, s>>>(*a);
}

#endif  // LUMA_UNIT == 0

#if LUMA_FORWARD

// -- the forward ------------------------------------------------------------------

// How the elements before a norm come about.
// x, residual + x, residual + dropout(x) (of rows with a cut run: either sum)
constexpr int kAlone = 0, kAdds = 1, kDrops = 2;

// A run of a row's columns as they are read: x, and the residual.
template <typename S, typename B, int HOW, int V, bool WHOLE, bool NT>
struct Columns {
  typedef typename std::conditional<HOW == kAlone, S, B>::type X;
  Vec<X, V> x;
  typename std::conditional<HOW == kAlone, char, Vec<S, V>>::type residual;

  __device__ __forceinline__ void load(const LumaLayerNormArgs &a, int64_t row, int64_t c) {
    x = load_raw<V, WHOLE, NT>((const X *)a.x + row * a.ld_x, c, a.h);
    if constexpr (HOW != kAlone)
      residual = load_raw<V, WHOLE, NT>((const S *)a.residual + row * a.ld_residual, c, a.h);
  }

  __device__ __forceinline__ void branch(const LumaLayerNormArgs &a, int64_t c, float *f) const {
    widen<V>(settle<V, WHOLE>(x, c, a.h), f);
  }

  // f, x or what dropout has left of it, becomes the sum, which is stored.
  __device__ __forceinline__ void sum(const LumaLayerNormArgs &a, int64_t row, int64_t c,
                                      float *f) const {
    if constexpr (HOW != kAlone) {
      const Vec<S, V> r = settle<V, WHOLE>(residual, c, a.h);
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = (float)(S)((float)r[j] + f[j]);
      store<V, WHOLE, NT>((S *)a.total + row * a.h, c, a.h, f);
    }
  }
};

// 1 / sqrt(v): the instruction, within a unit in the last place, which takes
// numbers below 2^-126 for 0.
__device__ __forceinline__ float rsqrt_of(float v) {
  if (v < 1e-30f) return __builtin_amdgcn_rsqf(v * 1.8446744e19f) * 4.2949673e9f;
  return __builtin_amdgcn_rsqf(v);
}

// The mean and the deviation from the sums of the differences from `about` and of
// their squares: m = about + off and r.  The mean of the differences is not quite
// 0 where the elements stand far from 0; it is put into both.
__device__ __forceinline__ void moments(float about, float first, float second, float one_h,
                                        float eps, float &off, float &m, float &r) {
  off = first * one_h;
  float v = second * one_h - off * off;
  v = v < 0.0f ? 0.0f : v;
  m = about + off;
  r = rsqrt_of(v + eps);
}

// A team goes from row to row, the next one's loads under way while it forms the
// sums of one.
template <typename S, typename B, int HOW, bool NT, typename T>
__global__ __launch_bounds__(T::kThreads) void norm_kernel(LumaLayerNormArgs a) {
  constexpr int L = T::L, K = T::K, V = T::V;
  __shared__ float at[2][3][T::kThreads / 64];
  const int64_t step = (int64_t)gridDim.x * T::kTeams;
  int64_t row = (int64_t)blockIdx.x * T::kTeams + threadIdx.x / L;
  Draw d;
  if constexpr (HOW == kDrops) d = draw_of(a.drop);
  Columns<S, B, HOW, V, T::WHOLE, NT> next[K];
  auto load = [&](int64_t of) {
    // (of cut rows without a condition, see load_raw: past the last row that again)
    if (T::WHOLE && of >= a.n) return;
    of = of < a.n ? of : a.n - 1;
#pragma unroll
    for (int k = 0; k < K; ++k) next[k].load(a, of, T::column(k));
  };
  load(row);
  float w[K][V], b[K][V];
  load_params<K, V, T::WHOLE, B>(a.weight, a.bias, a.param == LUMA_GRAD_F32, a.h,
                                 [](int k) { return T::column(k); }, w, b);
  const float one_h = 1.0f / (float)a.h;
  // A row's results are stored while the next one is formed: whoever waits for that
  // one's elements waits for all accesses before, and would wait for these stores
  // (16,384 x 4,096 bfloat16 93 us, otherwise 97).  A wavefront alone has others
  // beside it that need not wait (8,192 x 768 float32: 14.1 us, so 15.2).
  constexpr bool kLate = L > 64;
  Vec<B, V> y[K];
  float m = 0.0f, r = 0.0f;
  auto put = [&](int64_t of) {
#pragma unroll
    for (int k = 0; k < K; ++k)
      store<V, T::WHOLE, NT>((B *)a.y + of * a.h, T::column(k), a.h, y[k]);
    if (a.stats && threadIdx.x % L == 0) {
      a.stats[of] = m;
      a.stats[a.n + of] = r;
    }
  };
  // (the workgroup's teams make as many turns as its first, which has the most rows)
  int turn = 0;
  for (int64_t base = (int64_t)blockIdx.x * T::kTeams; base < a.n;
       base += step, row += step, turn ^= 1) {
    const bool live = row < a.n;
    float f[K][V], sum = 0.0f;
    if (live) {
#pragma unroll
      for (int k = 0; k < K; ++k) next[k].branch(a, T::column(k), f[k]);
      if constexpr (HOW == kDrops) {
        // (WHOLE teams: of a sum without draws there are others)
        if (T::WHOLE || a.drop.p > 0.0)
          drop(f, (uint64_t)(row * a.h + T::column(0)), L * V, a.h % 8 == 0, d,
               [&](int k) { return T::column(k) < a.h; });
      }
#pragma unroll
      for (int k = 0; k < K; ++k) {
        next[k].sum(a, row, T::column(k), f[k]);
#pragma unroll
        for (int j = 0; j < V; ++j) sum += f[k][j];      // (0 past the row)
      }
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) f[k][j] = 0.0f;
    }
    if (kLate && row >= step) put(row - step);
    load(row + step);
    const float about = team_sum<L>(sum, at[turn][0]) * one_h;
    float first = 0.0f, second = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      differences<V, T::WHOLE>(f[k], about, T::column(k), a.h);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        first += f[k][j];
        second = __builtin_fmaf(f[k][j], f[k][j], second);
      }
    }
    team_sum2<L>(first, second, at[turn][1], at[turn][2]);
    float off;
    moments(about, first, second, one_h, (float)a.eps, off, m, r);
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int j = 0; j < V; ++j)
        f[k][j] = __builtin_fmaf((f[k][j] - off) * r, w[k][j], b[k][j]);
      y[k] = rounded<B, V>(f[k]);
    }
    if (!kLate && live) put(row);
  }
  // (row is the one after the last turn's, whether that was there or not)
  if (kLate && row - step < a.n) put(row - step);
}

// A row that no team holds, one workgroup each: three passes over it.
template <typename S, typename B, int HOW>
__global__ __launch_bounds__(kLongThreads) void norm_long_kernel(LumaLayerNormArgs a, int64_t block) {
  constexpr int L = kLongThreads, V = kVec<S>, kStep = L * V;
  __shared__ float at[3][L / 64];
  const int64_t row = block + blockIdx.x;
  Draw d;
  if constexpr (HOW == kDrops) d = draw_of(a.drop);
  const S *s = HOW == kAlone ? (const S *)a.x + row * a.ld_x : (const S *)a.total + row * a.h;
  float g[1][V], (&f)[V] = g[0], sum = 0.0f;
  for (int64_t c = threadIdx.x * V; c < a.h; c += kStep) {
    Columns<S, B, HOW, V, false, false> in;
    in.load(a, row, c);
    in.branch(a, c, f);
    if constexpr (HOW == kDrops)
      drop(g, (uint64_t)(row * a.h + c), 0, a.h % 8 == 0, d, [](int) { return true; });
    in.sum(a, row, c, f);
#pragma unroll
    for (int j = 0; j < V; ++j) sum += f[j];
  }
  const float one_h = 1.0f / (float)a.h;
  const float about = team_sum<L>(sum, at[0]) * one_h;
  float first = 0.0f, second = 0.0f;
  // (a thread reads the elements of the sum that it wrote itself)
  for (int64_t c = threadIdx.x * V; c < a.h; c += kStep) {
    widen<V>(load<V>(s, c, a.h), f);
    differences<V>(f, about, c, a.h);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      first += f[j];
      second = __builtin_fmaf(f[j], f[j], second);
    }
  }
  team_sum2<L>(first, second, at[1], at[2]);
  float off, m, r;
  moments(about, first, second, one_h, (float)a.eps, off, m, r);
  if (a.stats && threadIdx.x == 0) {
    a.stats[row] = m;
    a.stats[a.n + row] = r;
  }
  for (int64_t c = threadIdx.x * V; c < a.h; c += kStep) {
    float w[1][V], b[1][V];
    load_params<1, V, false, B>(a.weight, a.bias, a.param == LUMA_GRAD_F32, a.h,
                                [&](int) { return c; }, w, b);
    widen<V>(load<V>(s, c, a.h), f);
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = __builtin_fmaf((f[j] - about - off) * r, w[0][j], b[0][j]);
    store<V>((B *)a.y + row * a.h, c, a.h, f);
  }
}

template <typename S, typename B, int HOW>
void forward(const LumaLayerNormArgs *a, hipStream_t s) {
  if (a->h > kWidest) {
    in_runs(a->n, kLongThreads, [&](int64_t first, uint32_t blocks) {
      norm_long_kernel<S, B, HOW><<<blocks, kLongThreads, 0, s>>>(*a, first);
    });
    return;
  }
  with_team<kVec<S>>(a->h, [&](auto team) {
    typedef decltype(team) T;
    if constexpr (T::WHOLE || HOW != kAdds) {
      auto kernel = norm_kernel<S, B, HOW, false, T>;
      if constexpr (T::WHOLE && T::L >= 64)
        if (apart(a, HOW == kAlone ? 1 : 2, HOW == kAlone ? 1 : 2))
          kernel = norm_kernel<S, B, HOW, true, T>;
      kernel<<<(uint32_t)blocks_of<T>(a->n, kForwardThreads), T::kThreads, 0, s>>>(*a);
    }
  });
}

template <typename S, typename B>
void forward(const LumaLayerNormArgs *a, hipStream_t s) {
  if (!a->residual)
    forward<S, B, kAlone>(a, s);
  else if (a->drop.p == 0.0 && (a->h % kVec<S> == 0 || a->h > kWidest))
    forward<S, B, kAdds>(a, s);
  else
    forward<S, B, kDrops>(a, s);
}

template <typename B>
void forward_of(const LumaLayerNormArgs *a, hipStream_t s) {
  if (std::is_same<B, float>::value || a->stream != LUMA_GRAD_F32)
    forward<B, B>(a, s);
  else
    forward<float, B>(a, s);
}

template void forward_of<Elem<LUMA_UNIT - 1>::type>(const LumaLayerNormArgs *, hipStream_t);

#endif  // LUMA_FORWARD

#if LUMA_UNIT == 0

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
    if (!adds && a->n > 1 && a->ld_x < 0)
      return fail("luma_layer_norm: rows lie backwards"), false;
    if (!adds && (a->d_total || a->d_residual))
      return fail("luma_layer_norm: gradients of a sum without one"), false;
  }
  return true;
}

#endif  // LUMA_UNIT == 0

#if LUMA_BACKWARD

// -- the backward -----------------------------------------------------------------

// A run of a row's columns as the backward reads them.
template <typename S, typename B, int V, bool WHOLE>
struct GradColumns {
  Vec<S, V> s, d_total;
  Vec<B, V> d_y;

  template <bool NT>
  __device__ __forceinline__ void load(const LumaLayerNormArgs &a, int64_t row, int64_t c) {
    const S *from = (const S *)(a.total ? a.total : a.x) + row * (a.total ? a.h : a.ld_x);
    s = load_raw<V, WHOLE, NT>(from, c, a.h);
    d_y = load_raw<V, WHOLE, NT>((const B *)a.d_y + row * a.h, c, a.h);
    if (a.d_total) d_total = load_raw<V, WHOLE, NT>((const S *)a.d_total + row * a.h, c, a.h);
  }

  __device__ __forceinline__ void settle(const LumaLayerNormArgs &a, int64_t c) {
    s = rows::settle<V, WHOLE>(s, c, a.h);
    d_y = rows::settle<V, WHOLE>(d_y, c, a.h);
    if (a.d_total) d_total = rows::settle<V, WHOLE>(d_total, c, a.h);
  }

  // Into the row's sums of g and g z, and the columns' of d_y z and d_y.
  __device__ __forceinline__ void sums(const float *w, float m, float r, float *dw, float *db,
                                       float &s1, float &s2) const {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float d = (float)d_y[j], z = ((float)s[j] - m) * r, g = d * w[j];
      s1 += g;
      s2 = __builtin_fmaf(g, z, s2);
      dw[j] = __builtin_fmaf(d, z, dw[j]);
      db[j] += d;
    }
  }

  // z and g are formed again of what was read: kept from the sums on they would
  // take two registers an element.
  __device__ __forceinline__ void forget() {
    typedef uint32_t Words __attribute__((ext_vector_type(4)));
    if constexpr (sizeof(Words) == sizeof(s)) {
      Words b = __builtin_bit_cast(Words, s);
      asm("" : "+v"(b));
      s = __builtin_bit_cast(decltype(s), b);
    }
  }

  // d_s.
  __device__ __forceinline__ void stream(const LumaLayerNormArgs &a, const float *w, float m,
                                         float r, float mean_g, float mean_gz, float *f) const {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float z = ((float)s[j] - m) * r, g = (float)d_y[j] * w[j];
      f[j] = r * (g - mean_g - z * mean_gz);
    }
    if (a.d_total) {
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] += (float)d_total[j];
    }
  }
};

// f(first, how many) for pairs of K runs.
template <int K, int K0 = 0, typename F>
__device__ __forceinline__ void in_pairs(F f) {
  if constexpr (K0 < K) {
    f(std::integral_constant<int, K0>{}, std::integral_constant<int, (K0 + 1 < K ? 2 : 1)>{});
    in_pairs<K, K0 + 2>(f);
  }
}

// Stores K runs of d_s, and what dropout leaves of it.
template <typename S, typename B, bool DROPS, bool WHOLE, bool NT, int K, int V, typename F>
__device__ __forceinline__ void store_grads(const LumaLayerNormArgs &a, const Draw &d, int64_t row,
                                            float (&f)[K][V], int64_t step, F column) {
  if (S *to = (S *)(a.total ? a.d_residual : a.d_x)) {
#pragma unroll
    for (int k = 0; k < K; ++k) store<V, WHOLE, NT>(to + row * a.h, column(k), a.h, f[k]);
  }
  if (!a.total || !a.d_x) return;
  if constexpr (DROPS) {
    // (WHOLE teams: where nothing is drawn there are others)
    if (WHOLE || a.drop.p > 0.0)
      drop(f, (uint64_t)(row * a.h + column(0)), step, a.h % 8 == 0, d,
           [&](int k) { return column(k) < a.h; });
  }
#pragma unroll
  for (int k = 0; k < K; ++k)
    store<V, WHOLE, NT>((B *)a.d_x + row * a.h, column(k), a.h, f[k]);
}

// A team's sums over its rows go into LDS, those of the workgroup's teams
// together to the workspace: [block][d_weight, d_bias][h].
template <typename T>
__device__ __forceinline__ void put_sums(const float (&v)[T::K][T::V], float *lds, float *out,
                                         int64_t h) {
  if constexpr (T::kTeams == 1) {
    constexpr int N = T::V < 4 ? T::V : 4;
#pragma unroll
    for (int k = 0; k < T::K; ++k)
#pragma unroll
      for (int i = 0; i < T::V; i += N) store<N, T::WHOLE>(out, T::column(k) + i, h, v[k] + i);
  } else {
    const int team = threadIdx.x / T::L;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < T::K; ++k)
#pragma unroll
      for (int j = 0; j < T::V; ++j) lds[team * T::kRow + T::column(k) + j] = v[k][j];
    __syncthreads();
    for (int64_t c = threadIdx.x; c < h; c += T::kThreads) {
      float sum = 0.0f;
#pragma unroll 8
      for (int t = 0; t < T::kTeams; ++t) sum += lds[t * T::kRow + c];
      out[c] = sum;
    }
  }
}

// A team goes from row to row; the next one's loads are under way while it forms
// the sums of one (with 32 elements a lane there are no registers for
// it).
template <typename S, typename B, bool DROPS, bool NT, typename T>
__global__ __launch_bounds__(T::kThreads) void norm_grad_kernel(LumaLayerNormArgs a) {
  constexpr int L = T::L, K = T::K, V = T::V;
  constexpr bool kAhead = K * V <= 24;
  __shared__ float at[2][2][T::kThreads / 64];
  __shared__ float lds[T::kTeams == 1 ? 1 : T::kTeams * T::kRow];
  const int64_t step = (int64_t)gridDim.x * T::kTeams;
  int64_t row = (int64_t)blockIdx.x * T::kTeams + threadIdx.x / L;
  const bool stores = a.d_x || a.d_residual;
  Draw d;
  if constexpr (DROPS) d = draw_of(a.drop);
  GradColumns<S, B, V, T::WHOLE> now[K], next[kAhead ? K : 1];
  float m = 0.0f, r = 0.0f, next_m = 0.0f, next_r = 0.0f;
  auto load = [&](auto &to, int64_t of, float &to_m, float &to_r) {
    // (of cut rows without a condition, see load_raw: past the last row that again)
    if (T::WHOLE && of >= a.n) return;
    of = of < a.n ? of : a.n - 1;
    to_m = a.stats[of];
    to_r = a.stats[a.n + of];
#pragma unroll
    for (int k = 0; k < K; ++k) to[k].template load<NT>(a, of, T::column(k));
  };
  if constexpr (kAhead) load(next, row, next_m, next_r);
  float w[K][V], dw[K][V], db[K][V];
  load_params<K, V, T::WHOLE, B>(a.weight, nullptr, a.param == LUMA_GRAD_F32, a.h,
                                 [](int k) { return T::column(k); }, w, dw);
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) dw[k][j] = db[k][j] = 0.0f;
  const float one_h = 1.0f / (float)a.h;
  int turn = 0;
  for (int64_t base = (int64_t)blockIdx.x * T::kTeams; base < a.n;
       base += step, row += step, turn ^= 1) {
    const bool live = row < a.n;
    if constexpr (kAhead) {
#pragma unroll
      for (int k = 0; k < K; ++k) now[k] = next[k];
      m = next_m;
      r = next_r;
      load(next, row + step, next_m, next_r);
    } else {
      load(now, row, m, r);
    }
    float s1 = 0.0f, s2 = 0.0f;
    if (live) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        now[k].settle(a, T::column(k));
        now[k].sums(w[k], m, r, dw[k], db[k], s1, s2);
      }
    }
    if (!stores) continue;
    // (one barrier a row: the next row's sums go to the other half)
    team_sum2<L>(s1, s2, at[turn][0], at[turn][1]);
    if (!live) continue;
    // (two runs at a time: drop()'s draws are for as many, and f takes few registers)
    in_pairs<K>([&](auto first, auto count) {
      constexpr int K0 = decltype(first)::value, N = decltype(count)::value;
      float f[N][V];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        now[K0 + k].forget();
        now[K0 + k].stream(a, w[K0 + k], m, r, s1 * one_h, s2 * one_h, f[k]);
      }
      store_grads<S, B, DROPS, T::WHOLE, NT>(a, d, row, f, L * V,
                                             [](int k) { return T::column(K0 + k); });
    });
  }
  float *out = (float *)a.workspace + (int64_t)blockIdx.x * 2 * a.h;
  if (a.d_weight) put_sums<T>(dw, lds, out, a.h);
  if (a.d_bias) put_sums<T>(db, lds, out + a.h, a.h);
}

// A row that no team holds: d_s in two passes over it.
template <typename S, typename B>
__global__ __launch_bounds__(kLongThreads) void norm_long_grad_kernel(LumaLayerNormArgs a,
                                                                  int64_t block) {
  constexpr int L = kLongThreads, V = kVec<S>, kStep = L * V;
  __shared__ float at[2][L / 64];
  const int64_t row = block + blockIdx.x;
  const Draw d = draw_of(a.drop);
  const float m = a.stats[row], r = a.stats[a.n + row], one_h = 1.0f / (float)a.h;
  float s1 = 0.0f, s2 = 0.0f, w[1][V], none[1][V], dw[V] = {}, db[V] = {};
  GradColumns<S, B, V, false> in;
  auto weights = [&](int64_t c) {
    load_params<1, V, false, B>(a.weight, nullptr, a.param == LUMA_GRAD_F32, a.h,
                                [&](int) { return c; }, w, none);
  };
  for (int64_t c = threadIdx.x * V; c < a.h; c += kStep) {
    weights(c);
    in.template load<false>(a, row, c);
    in.settle(a, c);
    in.sums(w[0], m, r, dw, db, s1, s2);
  }
  team_sum2<L>(s1, s2, at[0], at[1]);
  for (int64_t c = threadIdx.x * V; c < a.h; c += kStep) {
    weights(c);
    in.template load<false>(a, row, c);
    in.settle(a, c);
    float f[1][V];
    in.stream(a, w[0], m, r, s1 * one_h, s2 * one_h, f[0]);
    store_grads<S, B, true, false, false>(a, d, row, f, 0, [&](int) { return c; });
  }
}

// Its share of d_weight and d_bias: 256 lanes' columns a workgroup, the rows shared
// out over gridDim.y.
template <typename S, typename B>
__global__ __launch_bounds__(256) void norm_long_sums_kernel(LumaLayerNormArgs a) {
  constexpr int V = kVec<S>;
  const int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
  if (c >= a.h) return;
  float s1 = 0.0f, s2 = 0.0f, one[V], dw[V] = {}, db[V] = {};
#pragma unroll
  for (int j = 0; j < V; ++j) one[j] = 1.0f;
  a.d_total = nullptr;
  GradColumns<S, B, V, false> in;
  for (int64_t row = blockIdx.y; row < a.n; row += gridDim.y) {
    in.template load<false>(a, row, c);
    in.settle(a, c);
    in.sums(one, a.stats[row], a.stats[a.n + row], dw, db, s1, s2);
  }
  float *out = (float *)a.workspace + (int64_t)blockIdx.y * 2 * a.h;
#pragma unroll
  for (int i = 0; i < V; i += 4) {
    store<4>(out, c + i, a.h, dw + i);
    store<4>(out + a.h, c + i, a.h, db + i);
  }
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

template <typename S, typename B>
void backward(const LumaLayerNormArgs *a, hipStream_t stream) {
  const int64_t blocks = grad_blocks(a->n, a->h, a->stream);
  const bool sums = a->d_weight || a->d_bias, stores = a->d_x || a->d_residual;
  if (!sums && !stores) return;
  if (a->h > kWidest) {
    if (stores)
      in_runs(a->n, kLongThreads, [&](int64_t first, uint32_t count) {
        norm_long_grad_kernel<S, B><<<count, kLongThreads, 0, stream>>>(*a, first);
      });
    const int64_t each = 256 * kVec<S>;
    if (sums)
      norm_long_sums_kernel<S, B><<<dim3((uint32_t)((a->h + each - 1) / each), (uint32_t)blocks), 256,
                                    0, stream>>>(*a);
  } else {
    // (what is read and stored of the stream's type and of the branch's)
    const int streams = 1 + (a->d_total != nullptr) + ((a->total ? a->d_residual : a->d_x) != nullptr);
    const bool nt = apart(a, streams, 1 + (a->total && a->d_x));
    const bool drops = a->drop.p > 0.0 && a->d_x;
    with_team<kVec<S>>(a->h, [&](auto team) {
      typedef decltype(team) T;
      auto kernel = norm_grad_kernel<S, B, true, false, T>;
      if constexpr (T::WHOLE) {
        if (!drops) kernel = norm_grad_kernel<S, B, false, false, T>;
        if constexpr (T::L >= 64)
          if (nt)
            kernel = drops ? norm_grad_kernel<S, B, true, true, T>
                           : norm_grad_kernel<S, B, false, true, T>;
      }
      kernel<<<(uint32_t)blocks, T::kThreads, 0, stream>>>(*a);
    });
  }
  if (!sums) return;
  with_type(a->param, [&](auto p) {
    typedef decltype(p) P;
    const dim3 grid((uint32_t)((a->h + kJoinCols - 1) / kJoinCols), 2);
    join_kernel<P><<<grid, kJoinCols * kJoinRows, 0, stream>>>(
        (const float *)a->workspace, blocks, a->h, (P *)a->d_weight, (P *)a->d_bias);
  });
}

template <typename B>
void backward_of(const LumaLayerNormArgs *a, hipStream_t s) {
  if (std::is_same<B, float>::value || a->stream != LUMA_GRAD_F32)
    backward<B, B>(a, s);
  else
    backward<float, B>(a, s);
}

template void backward_of<Elem<LUMA_UNIT - 4>::type>(const LumaLayerNormArgs *, hipStream_t);

#endif  // LUMA_BACKWARD

}  // namespace residual
}  // namespace luma

#if LUMA_UNIT == 0

using namespace luma;
using namespace luma::residual;

extern "C" {

int luma_dropout(const LumaDropoutArgs *a, void *stream) {
  if (!a) return fail("luma_dropout: null arguments");
  if (a->numel < 1) return fail("luma_dropout: empty operands");
  // (2,048 elements a workgroup at least: 2^31 threads)
  if (a->numel > (int64_t)1 << 34) return fail("luma_dropout: operands too large");
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
  if (!known_type(a->stream)) return fail("luma_layer_norm: unknown type"), -1;
  return grad_blocks(a->n, a->h, a->stream) * 2 * a->h * (int64_t)sizeof(float);
}

int luma_layer_norm_forward(const LumaLayerNormArgs *a, void *stream) {
  if (!check_args(a, false)) return -1;
  with_type(a->branch, [&](auto b) { forward_of<decltype(b)>(a, (hipStream_t)stream); });
  return check_launch("luma_layer_norm_forward");
}

int luma_layer_norm_backward(const LumaLayerNormArgs *a, void *stream) {
  if (!check_args(a, true)) return -1;
  if ((a->d_weight || a->d_bias) &&
      (!a->workspace || (uintptr_t)a->workspace % 16 ||
       a->workspace_bytes < luma_layer_norm_workspace_bytes(a)))
    return fail("luma_layer_norm_backward: workspace too small or not aligned");
  with_type(a->branch, [&](auto b) { backward_of<decltype(b)>(a, (hipStream_t)stream); });
  return check_launch("luma_layer_norm_backward");
}

}  // extern "C"

#endif  // LUMA_UNIT == 0
