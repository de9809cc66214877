// The clipped policy loss of sampled tokens with a KL term (include/luma.h,
// luma_policy_forward / luma_policy_backward).
//
//   r = exp(l - l_old),  value = -min(r A, clip(r) A) + kl (exp(q) - 1 - q),  q = l_ref - l
//   d value / d l = -r A (or 0 where the clipped product is the smaller) + kl (1 - exp(q))
//
// A few numbers are read for each token and one is written: bound by HBM for
// large batches and by launches for small ones.  A workgroup takes a piece of
// one long row, or whole short rows, a wavefront each, and leaves one record of
// its sums; a join makes the loss of them in a fixed order (no atomics).  Up to
// kAlone short rows are one workgroup's, which joins them itself: one launch.
// The backward forms the token's terms again, which is cheaper than keeping
// them: the operands of small batches are still in the caches.  Measured: 512 x
// 8,192 float32 15.7 us (54 MB, 3.4 TB/s), 4.5 for the join, 16.3 backward (71 MB, 4.4
// TB/s); 16 x 65 5.4 and 4.5 us; 61 x 4,097 without sums 4.9.  (With the sums by
// shuffles through LDS, and always formed, 16 x 65 took 7.8 us forward.)
// The limits below carry a forward's (with its join) and a backward's times, calls in a
// row, float32, with a reference and a mask.
#include "luma_error.h"
#include "luma_rows.h"

namespace luma {
namespace policy {

using namespace rows;

constexpr int kThreads = 256, kWaves = kThreads / 64;
// Tokens of a lane at a time, 16 bytes of float32 (rows of fewer: 1).  32 x 1,024 20.4
// and 7.0 us, one at a time 24.0 and 7.4; 512 x 8,192 18.5 and 15.5, so 18.5 and 13.6;
// rows that fill no wavefront lose by four: 20,000 x 60 18.3 and 14.9, so 10.7 and 8.3.
constexpr int kTokens = 4;
// Tokens of a row that a wavefront takes whole; longer ones are cut in pieces.  2,000 x
// 600 9.6 and 7.0 us, with a limit of 512 10.3 and 6.4; 2,000 x 1,500 14.4 and 11.1, with
// one of 2,048 14.5 and 12.7.  Few rows would rather be cut: 64 x 600 8.5 and 6.0, by
// pieces 5.7 and 3.2.
constexpr int64_t kShort = 1024;
constexpr int64_t kMostLong = (int64_t)1 << 22;   // longer rows (a workgroup each)
// Short rows that one workgroup takes, and joins: one launch for two, on the host too.
// 16 x 65 5.3 us forward, in two launches 6.3; 4 x 1,024 7.1 and 9.2.  More tokens are
// sooner done by more workgroups: 32 x 10 7.5 and 6.3, 16 x 1,024 11.3 and 9.4, 32 x 1,024
// 20.4 and 9.7, and 64 x 10 would take 12.9 in one, 6.5 in two.
constexpr int64_t kAlone = 32;
// Of the workgroup that joins or takes all.  16 x 65 5.3 us forward, with 512 6.4, with
// 256 9.8; the join of 2,000 x 1,500's records (all 14.4, 14.6, 15.7).
constexpr int kJoinThreads = 1024;
// Workgroups, about.  2,000 x 1,500 14.4 and 11.1 us, with twice as many 17.2 and 12.6;
// 20,000 x 60 18.3 and 14.9, with half 18.1 and 15.4; 512 x 8,192 18.5 and 15.5, with half
// 16.7 and 13.8, with twice 22.6 and 15.0.
constexpr int64_t kBlocks = 2048;

// A workgroup's sums.
struct Part {
  double value;        // of the values; of whole rows' means for the mean of sequences
  double kl, moved;    // of exp(q) - 1 - q, of r - 1 - log r
  double count, clipped, sequences;      // (whole numbers)
};

// A wavefront's: the first three differ from lane to lane, the counts do not.
struct Sums {
  double value = 0.0, kl = 0.0, moved = 0.0;
  int64_t count = 0, clipped = 0, sequences = 0;
};

// How a call is shared out.
struct Plan {
  bool shorts;         // whole rows, a wavefront each; else pieces of rows
  int64_t piece;       // tokens of a piece
  int64_t pieces;      // of a row
  int64_t each;        // rows of a wavefront, one after the other
  int64_t blocks;
};

inline Plan plan(const LumaPolicyArgs *a) {
  Plan p;
  p.shorts = a->length <= kShort;
  if (p.shorts) {
    p.piece = a->length;
    p.pieces = 1;
    p.each = (a->rows + kBlocks * kWaves - 1) / (kBlocks * kWaves);
    const int64_t rows = p.each * kWaves;
    p.blocks = (a->rows + rows - 1) / rows;
  } else {
    // (pieces of at least 1,024 tokens, longer where that makes too many)
    const int64_t steps = (a->length + kShort - 1) / kShort, total = steps * a->rows;
    const int64_t run = (total + kBlocks - 1) / kBlocks;
    p.piece = (run < steps ? run : steps) * kShort;
    p.pieces = (a->length + p.piece - 1) / p.piece;
    p.each = 1;
    p.blocks = p.pieces * a->rows;
  }
  return p;
}

// exp(x) and exp(x) - 1 - x, the latter by its series where it is a difference
// of near numbers (the terms left out are below 2^-24 of it).
__device__ __forceinline__ void exp_excess(float x, float &e, float &excess) {
  e = expf(x);
  float s = 1.0f / 40320.0f;
  s = __builtin_fmaf(s, x, 1.0f / 5040.0f);
  s = __builtin_fmaf(s, x, 1.0f / 720.0f);
  s = __builtin_fmaf(s, x, 1.0f / 120.0f);
  s = __builtin_fmaf(s, x, 1.0f / 24.0f);
  s = __builtin_fmaf(s, x, 1.0f / 6.0f);
  s = __builtin_fmaf(s, x, 0.5f);
  // (of an infinite x, too, exp(x) is the larger: what is taken from it stays finite)
  const float less = __builtin_fminf(x, 3e38f);
  excess = __builtin_fabsf(x) < 0.5f ? s * x * x : e - 1.0f - less;
}

struct Limits {
  double up, low;               // of l - l_old
  float high_ratio, low_ratio;  // 1 + clip_high, 1 - clip_low
  float kl;
};

struct Token {
  float value, grad, kl, moved;
  bool clipped;
};

__device__ __forceinline__ Token token(float l, float old, float ref, bool has_ref, float adv,
                                       const Limits &lim) {
  Token t;
  // (float64 holds the difference of float32 numbers of like sizes exactly)
  const double d = (double)l - (double)old;
  float r;
  exp_excess((float)d, r, t.moved);
  const bool up = d > lim.up, low = d < lim.low;
  t.clipped = adv > 0.0f ? up : low && adv < 0.0f;
  const float held = up ? lim.high_ratio : lim.low_ratio;
  // (an advantage of 0 makes nothing of a ratio that passes float32, not 0 inf)
  const float product = adv == 0.0f && r > 1.0f ? 0.0f : r * adv;
  t.value = t.clipped ? -held * adv : -product;
  t.grad = t.clipped ? 0.0f : -product;
  t.kl = 0.0f;
  if (has_ref) {
    const float q = ref - l;
    float e;
    exp_excess(q, e, t.kl);
    // (exp(q) - 1 with the excess's digits)
    const float minus = __builtin_fabsf(q) < 0.5f ? t.kl + q : e - 1.0f;
    // (a weight of 0 leaves the term out: an infinite one times 0 is no number)
    if (lim.kl != 0.0f) {
      t.value = __builtin_fmaf(lim.kl, t.kl, t.value);
      t.grad = __builtin_fmaf(-lim.kl, minus, t.grad);
    }
  }
  return t;
}

// A row's operands at a lane's tokens.
template <typename T>
struct Row {
  const T *logp, *old, *ref;
  const float *advantage;
  const uint8_t *mask;
  float one;           // the row's advantage
  bool each;

  __device__ __forceinline__ Row(const LumaPolicyArgs &a, int64_t row) {
    logp = (const T *)a.logp + row * a.ld_logp;
    old = (const T *)a.old_logp + row * a.ld_old;
    ref = a.ref_logp ? (const T *)a.ref_logp + row * a.ld_ref : nullptr;
    mask = a.mask ? a.mask + row * a.ld_mask : nullptr;
    advantage = a.advantage + row * a.ld_advantage;
    each = a.advantage_each != 0;
    one = each ? 0.0f : *advantage;
  }
};

template <typename T, int N>
struct Tokens {
  Vec<T, N> l, old, ref;
  Vec<float, N> adv;
  Vec<uint8_t, N> mask;
  uint32_t keep;       // bit j: token j counts

  // The loads of tokens t .. t + N - 1 of a row of `length`,
  __device__ __forceinline__ void load(const Row<T> &r, int64_t t, int64_t length) {
    l = load_raw<N>(r.logp, t, length);
    old = load_raw<N>(r.old, t, length);
    if (r.ref) ref = load_raw<N>(r.ref, t, length);
    if (r.each) adv = load_raw<N>(r.advantage, t, length);
    if (r.mask) mask = load_raw<N>(r.mask, t, length);
  }

  // and what is before `end`.
  __device__ __forceinline__ void settle(const Row<T> &r, int64_t t, int64_t length, int64_t end) {
    l = rows::settle<N>(l, t, length);
    old = rows::settle<N>(old, t, length);
    if (r.ref) ref = rows::settle<N>(ref, t, length);
    if (r.each) adv = rows::settle<N>(adv, t, length);
    const int64_t left = end - t;
    keep = left >= N ? (1u << N) - 1u : left > 0 ? (1u << left) - 1u : 0u;
    if (r.mask) {
      mask = rows::settle<N>(mask, t, length);
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (!mask[j]) keep &= ~(1u << j);
    }
  }

  __device__ __forceinline__ Token at(const Row<T> &r, int j, const Limits &lim) const {
    return token((float)l[j], (float)old[j], r.ref ? (float)ref[j] : 0.0f, r.ref != nullptr,
                 r.each ? adv[j] : r.one, lim);
  }
};

// Tokens base + N lane of a row, base from `first` in steps of `step` (those of a
// wavefront) to before `end`, into s.  FIGURES: with what only a log wants.
template <typename T, int N, bool FIGURES>
__device__ __forceinline__ void row_sums(const LumaPolicyArgs &a, const Limits &lim, int64_t row,
                                         int64_t first, int64_t step, int64_t end, Sums &s) {
  const Row<T> r(a, row);
  const int64_t lane = threadIdx.x % 64 * N;
  float *out = a.reduction == LUMA_XENT_NONE ? a.loss + row * a.length : nullptr;
  Tokens<T, N> next;
  if (first < end) next.load(r, first + lane, a.length);
  for (int64_t base = first; base < end; base += step) {
    Tokens<T, N> in = next;
    if (base + step < end) next.load(r, base + step + lane, a.length);
    in.settle(r, base + lane, a.length, end);
    float v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const Token k = in.at(r, j, lim);
      const bool keep = in.keep >> j & 1u;
      v[j] = keep ? k.value : 0.0f;
      s.value += (double)v[j];
      s.count += __builtin_popcountll(__ballot(keep));
      if constexpr (FIGURES) {
        s.kl += (double)(keep ? k.kl : 0.0f);
        s.moved += (double)(keep ? k.moved : 0.0f);
        s.clipped += __builtin_popcountll(__ballot(keep && k.clipped));
      }
    }
    if (out) store<N>(out, base + lane, end, v);
  }
}

// The sums of W wavefronts, in the lanes of the first (W a power of two from 4 to 16).
template <int W, bool FIGURES>
__device__ __forceinline__ Part block_sum(Sums s, Part *lds) {
  s.value = lanes_sum<64>(s.value);
  if constexpr (FIGURES) {
    s.kl = lanes_sum<64>(s.kl);
    s.moved = lanes_sum<64>(s.moved);
  }
  if (threadIdx.x % 64 == 0)
    lds[threadIdx.x / 64] = Part{s.value,         s.kl,
                                 s.moved,         (double)s.count,
                                 (double)s.clipped, (double)s.sequences};
  __syncthreads();
  Part p = lds[threadIdx.x % W];
  p.value = lanes_sum<W>(p.value);
  p.count = lanes_sum<W>(p.count);
  p.sequences = lanes_sum<W>(p.sequences);
  if constexpr (FIGURES) {
    p.kl = lanes_sum<W>(p.kl);
    p.moved = lanes_sum<W>(p.moved);
    p.clipped = lanes_sum<W>(p.clipped);
  }
  return p;
}

// The loss and what goes with it, by one thread.
template <bool FIGURES>
__device__ __forceinline__ void finish(const LumaPolicyArgs &a, const Part &p) {
  const double n = p.count, s = p.sequences;
  if (a.reduction == LUMA_XENT_SUM) *a.loss = (float)p.value;
  if (a.reduction == LUMA_XENT_MEAN) *a.loss = (float)(p.value / n);
  if (a.reduction == LUMA_POLICY_SEQUENCE) *a.loss = (float)(p.value / s);
  if (a.share)
    a.share[a.rows] = a.reduction == LUMA_XENT_MEAN          ? (float)(1.0 / n)
                      : a.reduction == LUMA_POLICY_SEQUENCE ? (float)(1.0 / s)
                                                             : 1.0f;
  if constexpr (FIGURES) {
    a.stats[0] = (float)(p.clipped / n);
    a.stats[1] = (float)(p.kl / n);
    a.stats[2] = (float)(p.moved / n);
    a.stats[3] = (float)p.count;
  }
}

// A wavefront's whole rows; a sequence's mean is taken here.
template <typename T, int N, bool FIGURES>
__device__ __forceinline__ void whole_rows(const LumaPolicyArgs &a, const Limits &lim,
                                           int64_t first, int64_t end, Sums &s) {
  const bool lead = threadIdx.x % 64 == 0;
  for (int64_t row = first; row < end; ++row) {
    if (a.reduction != LUMA_POLICY_SEQUENCE) {
      row_sums<T, N, FIGURES>(a, lim, row, 0, 64 * N, a.length, s);
      continue;
    }
    const double value = s.value;
    const int64_t count = s.count;
    s.value = 0.0;
    row_sums<T, N, FIGURES>(a, lim, row, 0, 64 * N, a.length, s);
    const double own = (double)(s.count - count);
    s.value = value + (own ? s.value / own : 0.0);
    s.sequences += own != 0.0;
    if (lead && a.share) a.share[row] = own ? (float)(1.0 / own) : 0.0f;
  }
}

template <typename T, int N, bool FIGURES>
__global__ __launch_bounds__(kThreads) void sums_kernel(LumaPolicyArgs a, Limits lim, Plan plan) {
  __shared__ Part lds[kWaves];
  Sums s;
  if (plan.shorts) {
    const int64_t first = ((int64_t)blockIdx.x * kWaves + threadIdx.x / 64) * plan.each;
    const int64_t end = first + plan.each < a.rows ? first + plan.each : a.rows;
    whole_rows<T, N, FIGURES>(a, lim, first, end, s);
  } else {
    const int64_t row = blockIdx.x / plan.pieces, first = blockIdx.x % plan.pieces * plan.piece;
    const int64_t end = first + plan.piece < a.length ? first + plan.piece : a.length;
    row_sums<T, N, FIGURES>(a, lim, row, first + threadIdx.x / 64 * (64 * N), kThreads * N, end, s);
  }
  // (each token's loss alone: nothing is summed)
  if (!FIGURES && a.reduction == LUMA_XENT_NONE) return;
  const Part p = block_sum<kWaves, FIGURES>(s, lds);
  if (threadIdx.x == 0) ((Part *)a.workspace)[blockIdx.x] = p;
}

template <bool FIGURES>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(LumaPolicyArgs a, Plan plan) {
  __shared__ Part lds[kJoinThreads / 64];
  const Part *part = (const Part *)a.workspace;
  Part p = {};
  auto take = [&](const Part &o) {
    p.kl += o.kl;
    p.moved += o.moved;
    p.count += o.count;
    p.clipped += o.clipped;
    p.sequences += o.sequences;
  };
  if (!plan.shorts && a.reduction == LUMA_POLICY_SEQUENCE) {
    // (a thread a row: few long rows keep most threads idle, and the forward of 1 x
    // 1,000,000 takes 148 us, for the mean over the tokens 7.7; 8 x 131,072 30 and 7.7)
    for (int64_t row = threadIdx.x; row < a.rows; row += kJoinThreads) {
      double value = 0.0, count = 0.0;
      for (int64_t i = 0; i < plan.pieces; ++i) {
        const Part o = part[row * plan.pieces + i];
        take(o);
        value += o.value;
        count += o.count;
      }
      p.value += count ? value / count : 0.0;
      p.sequences += count != 0.0;
      if (a.share) a.share[row] = count ? (float)(1.0 / count) : 0.0f;
    }
  } else {
    for (int64_t i = threadIdx.x; i < plan.blocks; i += kJoinThreads) {
      const Part o = part[i];
      take(o);
      p.value += o.value;
    }
  }
  // (here the counts differ from lane to lane, too)
  double *const sums[] = {&p.value, &p.count, &p.sequences, &p.kl, &p.moved, &p.clipped};
#pragma unroll
  for (int i = 0; i < (FIGURES ? 6 : 3); ++i) *sums[i] = lanes_sum<64>(*sums[i]);
  if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = p;
  __syncthreads();
  if (threadIdx.x >= 64) return;
  p = lds[threadIdx.x % (kJoinThreads / 64)];
#pragma unroll
  for (int i = 0; i < (FIGURES ? 6 : 3); ++i) *sums[i] = lanes_sum<kJoinThreads / 64>(*sums[i]);
  if (threadIdx.x == 0) finish<FIGURES>(a, p);
}

// A few short rows in one launch.
template <typename T, int N, bool FIGURES>
__global__ __launch_bounds__(kJoinThreads) void alone_kernel(LumaPolicyArgs a, Limits lim) {
  constexpr int W = kJoinThreads / 64;
  __shared__ Part lds[W];
  Sums s;
  for (int64_t row = threadIdx.x / 64; row < a.rows; row += W)
    whole_rows<T, N, FIGURES>(a, lim, row, row + 1, s);
  if (!FIGURES && a.reduction == LUMA_XENT_NONE) return;
  const Part p = block_sum<W, FIGURES>(s, lds);
  if (threadIdx.x == 0) finish<FIGURES>(a, p);
}

template <typename T, int N>
__device__ __forceinline__ void row_grads(const LumaPolicyArgs &a, const Limits &lim, int64_t row,
                                          int64_t first, int64_t step, int64_t end) {
  const Row<T> r(a, row);
  const bool none = a.reduction == LUMA_XENT_NONE;
  const float *each = none ? a.grad_loss + row * a.length : nullptr;
  float g = 1.0f;
  if (!none) g = *a.grad_loss * a.share[a.rows];
  if (a.reduction == LUMA_POLICY_SEQUENCE) g *= a.share[row];
  Tokens<T, N> next;
  if (first < end) next.load(r, first, a.length);
  for (int64_t t = first; t < end; t += step) {
    Tokens<T, N> in = next;
    if (t + step < end) next.load(r, t + step, a.length);
    float o[N], f[N];
    if (none) {
      widen<N>(load<N>(each, t, a.length), f);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = g;
    }
    in.settle(r, t, a.length, end);
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = in.keep >> j & 1u ? in.at(r, j, lim).grad * f[j] : 0.0f;
    store<N>((T *)a.d_logp + row * a.length, t, end, o);
  }
}

template <typename T, int N>
__global__ __launch_bounds__(kThreads) void grad_kernel(LumaPolicyArgs a, Limits lim, Plan plan) {
  if (plan.shorts) {
    const int64_t first = ((int64_t)blockIdx.x * kWaves + threadIdx.x / 64) * plan.each;
    const int64_t end = first + plan.each < a.rows ? first + plan.each : a.rows;
    for (int64_t row = first; row < end; ++row)
      row_grads<T, N>(a, lim, row, threadIdx.x % 64 * N, 64 * N, a.length);
  } else {
    const int64_t row = blockIdx.x / plan.pieces, first = blockIdx.x % plan.pieces * plan.piece;
    const int64_t end = first + plan.piece < a.length ? first + plan.piece : a.length;
    row_grads<T, N>(a, lim, row, first + threadIdx.x * N, kThreads * N, end);
  }
}

// f(type, how many tokens a lane takes at a time).
template <typename F>
void with_tokens(const LumaPolicyArgs *a, F f) {
  with_type(a->dtype, [&](auto t) {
    if (a->length < kTokens)
      f(t, std::integral_constant<int, 1>{});
    else
      f(t, std::integral_constant<int, kTokens>{});
  });
}

Limits limits_of(const LumaPolicyArgs *a) {
  Limits l;
  l.up = log1p(a->clip_high);
  l.low = a->clip_low >= 1.0 ? -INFINITY : log1p(-a->clip_low);
  l.high_ratio = (float)(1.0 + a->clip_high);
  l.low_ratio = (float)(1.0 - a->clip_low);
  l.kl = (float)a->kl_weight;
  return l;
}

bool alone(const LumaPolicyArgs *a) { return a->length <= kShort && a->rows <= kAlone; }

// Whether workgroups' records are left to be joined.
bool joins(const LumaPolicyArgs *a) {
  return !alone(a) && (a->stats || a->reduction != LUMA_XENT_NONE);
}

bool check_args(const LumaPolicyArgs *a, bool backward) {
  if (!a) return fail("luma_policy: null arguments"), false;
  if (a->rows < 1 || a->length < 1) return fail("luma_policy: empty operands"), false;
  if (a->rows > INT32_MAX || a->length > INT32_MAX || a->rows > ((int64_t)1 << 40) / a->length)
    return fail("luma_policy: operands too large"), false;
  // (a workgroup each, if they are long)
  if (a->length > kShort && a->rows > kMostLong)
    return fail("luma_policy: operands too large"), false;
  if (!known_type(a->dtype)) return fail("luma_policy: unknown type"), false;
  if (a->reduction < LUMA_XENT_NONE || a->reduction > LUMA_POLICY_SEQUENCE)
    return fail("luma_policy: unknown reduction"), false;
  if (!(a->clip_low >= 0.0 && a->clip_low <= 1.0))
    return fail("luma_policy: clip_low is not in [0, 1]"), false;
  if (!(a->clip_high >= 0.0)) return fail("luma_policy: clip_high is negative"), false;
  if (a->kl_weight != a->kl_weight) return fail("luma_policy: kl_weight is NaN"), false;
  if (a->reserved) return fail("luma_policy: reserved fields must be 0"), false;
  if (!a->logp || !a->old_logp || !a->advantage) return fail("luma_policy: null operand"), false;
  if (backward ? !a->grad_loss || !a->d_logp || (a->reduction != LUMA_XENT_NONE && !a->share)
               : !a->loss)
    return fail("luma_policy: null operand"), false;
  if (a->rows > 1 && (a->ld_logp < 0 || a->ld_old < 0 || (a->ref_logp && a->ld_ref < 0) ||
                      a->ld_advantage < 0 || (a->mask && a->ld_mask < 0)))
    return fail("luma_policy: rows lie backwards"), false;
  return true;
}

}  // namespace policy
}  // namespace luma

using namespace luma;
using namespace luma::policy;

extern "C" {

int64_t luma_policy_workspace_bytes(const LumaPolicyArgs *a) {
  if (!check_args(a, false)) return -1;
  return joins(a) ? plan(a).blocks * (int64_t)sizeof(Part) : 0;
}

int luma_policy_forward(const LumaPolicyArgs *a, void *stream) {
  if (!check_args(a, false)) return -1;
  const hipStream_t s = (hipStream_t)stream;
  const Limits lim = limits_of(a);
  const Plan p = plan(a);
  if (joins(a) && (!a->workspace || (uintptr_t)a->workspace % 16 ||
                   a->workspace_bytes < p.blocks * (int64_t)sizeof(Part)))
    return fail("luma_policy_forward: workspace too small or not aligned");
  with_tokens(a, [&](auto t, auto tokens) {
    typedef decltype(t) T;
    constexpr int N = decltype(tokens)::value;
    if (alone(a)) {
      const auto kernel = a->stats ? alone_kernel<T, N, true> : alone_kernel<T, N, false>;
      kernel<<<1, kJoinThreads, 0, s>>>(*a, lim);
    } else {
      const auto kernel = a->stats ? sums_kernel<T, N, true> : sums_kernel<T, N, false>;
      kernel<<<(uint32_t)p.blocks, kThreads, 0, s>>>(*a, lim, p);
    }
  });
  if (joins(a)) {
    const auto kernel = a->stats ? join_kernel<true> : join_kernel<false>;
    kernel<<<1, kJoinThreads, 0, s>>>(*a, p);
  }
  return check_launch("luma_policy_forward");
}

int luma_policy_backward(const LumaPolicyArgs *a, void *stream) {
  if (!check_args(a, true)) return -1;
  const Plan p = plan(a);
  with_tokens(a, [&](auto t, auto tokens) {
    grad_kernel<decltype(t), decltype(tokens)::value>
        <<<(uint32_t)p.blocks, kThreads, 0, (hipStream_t)stream>>>(*a, limits_of(a), p);
  });
  return check_launch("luma_policy_backward");
}

}  // extern "C"
