/*
 * luma.h -- C ABI of the MI355X (gfx950) LUMA optimizer-step library
 * (libluma_hip.so).  Plain C types only; every pointer documented as
 * "device" is HIP device memory owned by the caller.  The library never
 * allocates, never synchronises the stream it is given, and never throws:
 * each entry point returns 0 on success or a nonzero status whose text is
 * available from luma_last_error().
 *
 * Every per-step quantity lives in device memory: each tensor's step count,
 * scales and grids sit in its slot, and the step-dependent scalars are
 * derived on the device from the param group's hyper-parameters.  A launch
 * sequence captured into a HIP graph therefore advances correctly on every
 * replay (the reference keeps its step counter on the device for the same
 * reason, optimizer.py:382-387).
 *
 * What each entry point replaces in the reference (IgorYashch/LUMA 0.1.0):
 *
 *   luma_step          -- the per-parameter loop body of LUMA.step for all
 *                         parameters at once: luma_init_step (t = 1,
 *                         src/luma_optimizer/functional.py:183-228) and
 *                         luma_update_step (t >= 2, functional.py:231-298),
 *                         i.e. the Triton pipelines luma_triton_init_step /
 *                         luma_triton_step (triton_kernel.py:409-492); with
 *                         LumaScaling, also GradScaler's unscale_ and
 *                         skip-on-overflow around it (the reference runs
 *                         them outside the optimizer).
 *   luma_step_profiled -- luma_step with event records between its launches.
 *   luma_step_noalloc  -- luma_step with its workspace inside the library
 *                         (no counterpart in the reference; for callers that
 *                         cannot allocate).
 *   luma_step_tensor   -- one tensor, no device tables: the per-tensor
 *                         functional ops luma_triton_step /
 *                         luma_triton_init_step (triton_kernel.py:409-492).
 *   luma_set_scales    -- the scale half of load_state_dict /
 *                         _init_triton_buffers (optimizer.py:146-183,341-387).
 *   luma_get_scales    -- the S_m / S_v / step read-back of state_dict
 *                         (optimizer.py:119-144).
 *   luma_decode        -- the decode of export_adamw_state
 *                         (optimizer.py:231-235, functional.py:113-126).
 *   luma_quantize      -- the quantisation of import_adamw_state
 *                         (optimizer.py:304-321, functional.py:133-176).
 *   luma_hyper_rows    -- the step-dependent scalars of functional.py:209-213,
 *                         262-264, 278 as the device derives them (for
 *                         checking against the host's double arithmetic).
 *   luma_grad_norm, luma_grad_clip, luma_grad_scale
 *                      -- torch.nn.utils.get_total_norm, clip_grad_norm_ and
 *                         clip_grads_with_norm_ as the reference's benchmark
 *                         uses them around its step (no kernel of its own).
 *   luma_xent_forward, luma_xent_backward
 *                      -- torch.nn.functional.cross_entropy of a linear
 *                         layer's outputs, as the reference's benchmark
 *                         trains on (no kernel of its own).
 *   luma_layer_norm_forward, luma_layer_norm_backward, luma_dropout
 *                      -- torch's layer norm, dropout and residual sum of the
 *                         models that the reference's benchmark trains (no
 *                         kernel of its own).
 *   luma_policy_forward, luma_policy_backward
 *                      -- nothing: the loss of a model that is tuned on its
 *                         own answers, on luma_xent_forward's losses.
 *   luma_philox4x32    -- host-side Philox4x32-10 block function used by the
 *                         stochastic rounding (Salmon et al., SC'11); the
 *                         reference's Triton path draws from tl.rand
 *                         (triton_kernel.py:103,124).
 */
#ifndef LUMA_H
#define LUMA_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define LUMA_ABI_VERSION 12

/*
 * Elements per chunk-table entry (one workgroup's share of a tensor): the
 * default and the largest.  luma_step accepts any power of two from
 * LUMA_CHUNK_ELEMS_MIN to LUMA_CHUNK_ELEMS per launch (LumaStepArgs.chunk_elems);
 * smaller chunks give small tensor sets more workgroups.
 */
#define LUMA_CHUNK_ELEMS 131072
#define LUMA_CHUNK_ELEMS_MIN 2048
#define LUMA_STEP_TENSOR_CHUNK_MIN 16384   /* shortest chunk luma_step_tensor uses */

/*
 * Tensors of at most this many elements are best stepped one wavefront each
 * with an exact pass 1 (LumaStepArgs.small_chunks): a workgroup of their own
 * would spend most of its time in set-up, and the fast pass 1's wavefront
 * route (medium_chunks) runs a partial group for them.
 */
#define LUMA_SMALL_TENSOR 256

/*
 * Tensors above LUMA_SMALL_TENSOR and of at most this many elements are best
 * stepped one wavefront each (LumaStepArgs.medium_chunks): a whole
 * workgroup would leave most of its wavefronts idle on them.  (In a set that
 * leaves the chip idle that costs nothing: LUMA_FLAG_SPLIT.)
 */
#define LUMA_MEDIUM_TENSOR 8192

/*
 * Bytes of one slot: a tensor's persistent device state (step count, S_m,
 * S_v, grids).  A fresh slot must be zero-filled (step count 0: the next
 * step is the reference's init step).  16-byte aligned.
 */
#define LUMA_SLOT_BYTES 512

/*
 * Code summaries.  A tensor may carry a summary array that its steps keep:
 * one uint32 per thread of each chunk's workgroup, LUMA_SUMMARY_WORDS words
 * per chunk, chunk c of the tensor at words [c * LUMA_SUMMARY_WORDS,
 * (c + 1) * LUMA_SUMMARY_WORDS).  Each step's pass 2 writes, for every
 * thread, a bound on the codes it stored in its share of the chunk: the
 * largest |Q_m| and the smallest Q_w, widened by the step's certified
 * decision margin.  The next step's pass 1 bounds each thread's |m'| and v'
 * from that word and the gradients alone, and reads a wave's codes only when
 * some thread could hold the tensor's maximum.  Results do not depend on the
 * summaries; they only save reads.  They are used only when the slot records
 * that the previous step wrote them with the same chunk length (luma_set_scales
 * and luma_quantize clear that record), and only for chunks whose words fit
 * in summary_words.  A caller that rewrites a tensor's codes by other means
 * between steps must also rewrite its slot with luma_set_scales, or pass a
 * NULL summary.  luma_summary_words gives the words a tensor needs.
 */
#define LUMA_SUMMARY_WORDS 256

/* Gradient element types. */
#define LUMA_GRAD_F32 0
#define LUMA_GRAD_BF16 1
#define LUMA_GRAD_F16 2

/*
 * Where the stochastic-rounding uniforms come from.  Under
 * LUMA_NOISE_INJECTED a tensor whose u_m or u_w is NULL draws from Philox as
 * under LUMA_NOISE_PHILOX, so a caller may inject uniforms for some tensors
 * of a step only.
 */
#define LUMA_NOISE_PHILOX 0   /* counter-based Philox4x32-10, keyed per (seed, step, param) */
#define LUMA_NOISE_INJECTED 1 /* caller-supplied u_m / u_w float32 arrays in [0, 1) */

/* luma_step flags. */
#define LUMA_FLAG_EXACT_ONLY 1 /* take the exact per-element path everywhere */
/*
 * Let the step give a small set more workgroups than it has chunk records:
 * the medium records take a workgroup each where luma_split_plan says so, and
 * the workgroup records (those medium ones among them) are split into
 * 2^(its value) parts of down to LUMA_CHUNK_ELEMS_MIN elements, which then are
 * the chunks (of the code summaries too).  The results do not depend on it.
 * `partials` then needs luma_workspace_bytes(n_chunks + LUMA_SPLIT_CHUNKS)
 * (luma_step_tensor: plus LUMA_SPLIT_CHUNKS likewise; luma_step_noalloc's own
 * workspace has the room, and beyond LUMA_NOALLOC_MAX_CHUNKS -
 * LUMA_SPLIT_CHUNKS chunks it ignores the flag).  Without the flag every
 * record is one chunk.
 */
#define LUMA_FLAG_SPLIT 2
#define LUMA_SPLIT_CHUNKS 1024
/*
 * For LUMA_FLAG_SPLIT, in luma_step's flags: the elements of the longest medium
 * tensor, which luma_split_plan's rule takes (absent: LUMA_MEDIUM_TENSOR).
 */
#define LUMA_FLAG_LONGEST_SHIFT 8
#define LUMA_FLAG_LONGEST(elems) ((int32_t)(elems) << LUMA_FLAG_LONGEST_SHIFT)

/* One parameter tensor taking part in a step. */
typedef struct LumaTensor {
  float *param;         /* device f32 [numel], updated in place            */
  const void *grad;     /* device f32 / bf16 / f16 [numel]                  */
  int16_t *q_m;         /* device [numel] signed log-grid momentum codes    */
  int16_t *q_w;         /* device [numel] uint16 preconditioner codes       */
  const float *u_m;     /* device [numel] injected uniforms, or NULL        */
  const float *u_w;     /* device [numel] injected uniforms, or NULL        */
  void *slot;           /* device, LUMA_SLOT_BYTES: this tensor's state     */
  uint32_t *summary;    /* device code summaries kept across steps, or NULL */
  int64_t summary_words;/* words at summary (see luma_summary_words)       */
  int64_t numel;        /* elements                                          */
  int64_t param_id;     /* position of the parameter in param_groups order  */
  int64_t elem_offset;  /* index of element 0 in the whole parameter when this
                           tensor is one shard of it, else 0: the Philox
                           counters follow the whole parameter's element
                           index, so shards draw independent uniforms       */
  int32_t grad_dtype;   /* LUMA_GRAD_*                                       */
  int32_t group;        /* index into the LumaGroup table                    */
  int32_t first_chunk;  /* index of this tensor's first LumaChunk            */
  int32_t reserved;     /* 0                                                 */
} LumaTensor;

/* Chunk c of a tensor covers elements [c*C, min(numel, (c+1)*C)), C the launch's chunk length. */
typedef struct LumaChunk {
  int32_t tensor; /* index into the LumaTensor table */
  int32_t index;  /* chunk number within that tensor */
} LumaChunk;

/*
 * A param group's hyper-parameters as the Python doubles the reference holds
 * (optimizer.py:80-92).  Per step the device derives, exactly as the
 * reference's double arithmetic and each rounded once to float32:
 * beta1, 1 - beta1, beta2, 1 - beta2, 1 - weight_decay*lr,
 * -(lr / (1 - beta1^t)), 1 - beta2^t and eps, where beta^t is the correctly
 * rounded power (Python's ** agrees with it after the float32 rounding).
 */
typedef struct LumaGroup {
  double lr, beta1, beta2, eps, weight_decay;
  double reserved; /* 0 */
} LumaGroup;

/*
 * Mixed-precision scaling (torch.amp.GradScaler's contract for optimizers
 * that unscale inside their step, `_step_supports_amp_scaling`):
 *   grad_scale -- device float32 scalar, or NULL.  The gradients hold
 *                 scale * g; each element is unscaled exactly as
 *                 GradScaler.unscale_ would store it:
 *                 dtype(f32(grad) * f32(1 / (double)scale)), rounded to
 *                 nearest even in the gradient's own dtype.
 *   found_inf  -- device float32 scalar, or NULL.  Nonzero: the whole step
 *                 does nothing (parameters, codes, scales and step counts
 *                 unchanged), with no host synchronisation.
 */
typedef struct LumaScaling {
  const float *grad_scale;
  const float *found_inf;
} LumaScaling;

typedef struct LumaStepArgs {
  const LumaTensor *tensors; /* device */
  int32_t n_tensors;
  int32_t n_chunks;
  const LumaChunk *chunks;   /* device */
  const LumaGroup *groups;   /* device */
  float *partials;           /* device workspace, luma_workspace_bytes(n_chunks), 16-byte aligned */
  uint64_t base_seed;        /* LUMA._base_seed as its two's-complement bits */
  int32_t noise_mode;        /* LUMA_NOISE_* */
  int32_t flags;             /* LUMA_FLAG_* */
  int32_t chunk_elems;       /* chunk length C of the chunk table: a power of two in
                                [LUMA_CHUNK_ELEMS_MIN, LUMA_CHUNK_ELEMS]; 0 = LUMA_CHUNK_ELEMS */
  int32_t small_chunks;      /* the last small_chunks records of the chunk table, one
                                chunk per tensor, are stepped one wavefront each (four
                                per workgroup): pass 1 by the exact path, pass 2 by the
                                fast kernel's wavefront route; meant for tensors of at
                                most LUMA_SMALL_TENSOR elements (any tensor is stepped
                                correctly).  0: every chunk takes a workgroup */
  int32_t medium_chunks;     /* the medium_chunks records just before the small ones
                                are stepped one wavefront each, four per workgroup, in
                                the same launches and by the same fast kernels as the
                                others (8 elements per lane and iteration); meant for
                                tensors of at most LUMA_MEDIUM_TENSOR elements, one
                                chunk each (any chunk is stepped correctly).  Such
                                tensors keep no code summaries.  LUMA_FLAG_SPLIT may
                                give them a workgroup each instead.  0: none */
  int32_t reserved;          /* 0 */
  LumaScaling scaling;       /* both NULL: unscaled gradients, always step */
} LumaStepArgs;

/* One slot write (array in device memory). */
typedef struct LumaScaleInit {
  void *slot;    /* device slot */
  int64_t step;  /* the tensor's step count t */
  double s_m;    /* S_m as stored by the reference (>= 1e-9) */
  double s_v;    /* S_v (>= 0) */
  double eps;    /* the group's eps */
} LumaScaleInit;

int luma_abi_version(void);
const char *luma_last_error(void);

/*
 * Struct sizes as compiled, for binding checks: LumaTensor, LumaChunk,
 * LumaGroup, LumaScaleInit, LumaStepArgs, slot bytes, LUMA_CHUNK_ELEMS, 0.
 */
void luma_layout(int32_t out[8]);

/* Bytes of workspace luma_step / luma_step_tensor / luma_quantize need for n_chunks chunks. */
size_t luma_workspace_bytes(int32_t n_chunks);

/*
 * How LUMA_FLAG_SPLIT shares out a launch of `records` workgroup records of
 * chunk_elems elements (luma_step: n_chunks - medium_chunks - small_chunks),
 * `medium` and `small` records (medium_chunks, small_chunks), the longest
 * medium tensor of `medium_longest` elements (0: LUMA_MEDIUM_TENSOR): returns
 * log2 of the parts of a workgroup record; *wide (may be NULL) is 1 where the
 * medium records take a workgroup each, which then are split too.
 */
int32_t luma_split_plan(int32_t records, int32_t medium, int32_t small, int32_t medium_longest,
                        int32_t chunk_elems, int32_t *wide);

/* luma_split_plan of `records` workgroup records alone. */
int32_t luma_split_shift(int32_t records, int32_t chunk_elems);

/* Summary words a tensor of numel elements needs for chunks of chunk_elems elements. */
int64_t luma_summary_words(int64_t numel, int32_t chunk_elems);

/*
 * One optimizer step for every tensor in the table: pass 1 (decode + EMA +
 * per-chunk maxima), per-tensor finalize (new S_m/S_v and grid in float64,
 * step count + 1, step scalars), pass 2 (re-decode + EMA + AdamW update +
 * LogSR re-quantisation).  A tensor whose slot holds step count 0 takes the
 * init step.  Three kernel launches on `stream` (a hipStream_t): the small
 * tensors (small_chunks > 0) are stepped by workgroups of the pass-1 and
 * pass-2 launches past their own (with LUMA_FLAG_EXACT_ONLY by a kernel of
 * their own in each pass); no host synchronisation.  No device table is written, so the sequence may
 * be captured into a HIP graph and replayed.
 */
int luma_step(const LumaStepArgs *args, void *stream);

/*
 * luma_step that also records caller-created hipEvent_t events[0..3] on the
 * stream: before pass 1, after pass 1, after finalize, after pass 2 (NULL
 * entries are skipped).  Used to time each kernel on its own stream.
 */
int luma_step_profiled(const LumaStepArgs *args, void *stream, void *const events[4]);

/*
 * Largest n_chunks luma_step_noalloc takes: its workspace is a fixed device
 * array of 16 bytes per chunk (4 MiB per GPU).
 */
#define LUMA_NOALLOC_MAX_CHUNKS 262144

/*
 * luma_step that allocates nothing and takes no workspace: args->partials is
 * ignored, and pass 1's per-chunk maxima go to a fixed array inside the
 * library (one per GPU, kept until the process ends), so no memory is
 * allocated on any call, the first included.  No counterpart in the
 * reference: it is for callers that cannot allocate (code under HIP graph
 * capture, tight serving loops, harnesses that forbid hipMalloc).  Limits:
 * n_chunks <= LUMA_NOALLOC_MAX_CHUNKS (else an error, nothing launched); the
 * stream's device must be the current device; calls that overlap on one GPU
 * (other streams, other threads) share that GPU's array and race.
 */
int luma_step_noalloc(const LumaStepArgs *args, void *stream);

/*
 * luma_step for one tensor with no device tables: *tensor, *group and
 * *scaling (may be NULL) are host structs read during the call
 * (tensor->first_chunk is ignored).  The chunk length is LUMA_CHUNK_ELEMS,
 * halved down to LUMA_STEP_TENSOR_CHUNK_MIN while the tensor has fewer than
 * 4096 chunks; `partials` needs
 * luma_workspace_bytes(ceil(numel / LUMA_STEP_TENSOR_CHUNK_MIN)).
 */
int luma_step_tensor(const LumaTensor *tensor, const LumaGroup *group, float *partials,
                     uint64_t base_seed, int32_t noise_mode, int32_t flags,
                     const LumaScaling *scaling, void *stream);

/* Write step count, S_m and S_v of n slots (items: device array) and derive their grids. */
int luma_set_scales(const LumaScaleInit *items, int32_t n, void *stream);

/*
 * Read n slots (slots: device array of slot pointers): S_m, S_v into
 * scales[2*i], scales[2*i+1] and the step count into steps[i] (device).
 */
int luma_get_scales(void *const *slots, int32_t n, double *scales, int64_t *steps, void *stream);

/*
 * Decode one tensor's codes into float32 m (exp_avg) and v (exp_avg_sq) on
 * the grid of the slot's current step, with the group's eps.
 */
int luma_decode(const int16_t *q_m, const int16_t *q_w, int64_t numel, const void *slot,
                double eps, float *m_out, float *v_out, void *stream);

/*
 * Quantise given float32 m, v (clamped at 0) into codes with fresh scales
 * S_m = max(max|m|, 1e-9), S_v = max(max v, 0), stored into the slot with
 * step count `step`.  Uniforms: Philox keyed by seed (noise_mode 0) or
 * u_m/u_w (noise_mode 1).  `partials` needs
 * luma_workspace_bytes(ceil(numel / LUMA_CHUNK_ELEMS)).
 */
int luma_quantize(const float *m, const float *v, int64_t numel, int16_t *q_m, int16_t *q_w,
                  void *slot, int64_t step, double eps, uint64_t seed, int32_t noise_mode,
                  const float *u_m, const float *u_w, float *partials, void *stream);

/*
 * The step scalars the device derives for steps t0 .. t0+n-1 of *group (a
 * host struct): 8 floats per step into out (device): beta1, 1-beta1, beta2,
 * 1-beta2, decay, -eta, bc2, eps.
 */
int luma_hyper_rows(const LumaGroup *group, int64_t t0, int32_t n, float *out, void *stream);

/*
 * The global norm of many gradients, and clipping by it.
 *
 * ||g||_p over all elements of all rows together; the reference's benchmark
 * clips with torch.nn.utils.clip_grad_norm_ between backward() and step()
 * (benchmarks/bench_nanogpt.py).  Sums are formed in float64 (a float32
 * gradient's square is exact there and cannot overflow or vanish) in an order
 * that the rows' sizes and the way they are passed (LumaNormArgs.table or not)
 * determine: the same call gives the same bits every time, and the same rows
 * passed the other way the same sum but for float64's rounding.  A NaN anywhere
 * makes the norm NaN.
 */
#define LUMA_NORM_L2 0
#define LUMA_NORM_L1 1
#define LUMA_NORM_INF 2

/* Elements per tile: the unit in which the rows are shared out to wavefronts. */
#define LUMA_GRAD_TILE 2048
/* Rows that one launch carries among its arguments (no device table). */
#define LUMA_GRADS_INLINE 160
/* Rows that may go without a device table. */
#define LUMA_GRADS_NO_TABLE (LUMA_GRADS_INLINE * 256)
/* Doubles of workspace (LumaNormArgs.partials). */
#define LUMA_NORM_PARTIALS 1024

/* One gradient; dense, elements in any order, aligned to its element type. */
typedef struct LumaGrad {
  void *data;          /* device f32 / bf16 / f16 [numel]                       */
  int64_t numel;       /* >= 1                                                   */
  int32_t dtype;       /* LUMA_GRAD_*                                            */
  int32_t first_tile;  /* sum of ceil(numel / LUMA_GRAD_TILE) of the rows before */
} LumaGrad;

typedef struct LumaNormArgs {
  const LumaGrad *grads; /* HOST: the rows, read during the call                 */
  const LumaGrad *table; /* device copy of them; NULL (n <= LUMA_GRADS_NO_TABLE):
                            the rows travel as launch arguments, a launch per
                            LUMA_GRADS_INLINE of them (may then be captured into
                            a HIP graph)                                         */
  int32_t n;             /* rows                                                 */
  int32_t norm;          /* LUMA_NORM_*                                          */
  double max_norm;       /* clipping: the largest norm, >= 0                     */
  double *partials;      /* device workspace, LUMA_NORM_PARTIALS doubles         */
  float *total;          /* device scalar: the norm (luma_grad_scale reads it)   */
  double *power;         /* device scalar or NULL: the norm before its root (the
                            sum of |g|^p; the largest |g|), to be joined with
                            other GPUs'                                          */
  const float *grad_scale; /* device scalar or NULL: the gradients hold scale * g,
                            and *total and *step_scale are for g
                            (luma_grad_norm only)                                */
  float *step_scale;     /* device scalar or NULL: what LumaScaling.grad_scale has
                            to be for a step that clips by max_norm as it reads
                            the gradients: grad_scale (or 1) over the clip factor
                            (luma_grad_norm only)                                */
} LumaNormArgs;

/* *total (and *power) of the rows; the gradients are only read. */
int luma_grad_norm(const LumaNormArgs *args, void *stream);

/*
 * luma_grad_norm, then every gradient times min(1, max_norm / (*total + 1e-6))
 * in place, rounded to nearest in its own type (nothing is written where the
 * factor is 1).  No two rows may share memory.
 */
int luma_grad_clip(const LumaNormArgs *args, void *stream);

/* The second half of luma_grad_clip, with the norm that *total holds. */
int luma_grad_scale(const LumaNormArgs *args, void *stream);

/*
 * The cross entropy of a vocabulary's logits, without the logits.
 *
 * For token i with hidden state x_i, target t_i and the weight's rows w_j:
 *   l_ij = x_i . w_j,  lse_i = log sum_j exp(l_ij),  loss_i = lse_i - l_i,t_i
 * and for the gradient g_i of loss_i
 *   D_ij = g_i (exp(l_ij - lse_i) - [j = t_i]),  d_hidden = D W,  d_weight = D^T X.
 * The logits are formed tile by tile on the matrix cores and never written; the
 * backward forms them again and keeps D for one piece of the vocabulary at a
 * time, in the operands' type.  The reference's benchmark takes torch's cross
 * entropy of whole logits (benchmarks/bench_nanogpt.py).
 *
 * A target equal to ignore_index has loss 0 and gradient 0, and does not count
 * in the mean; any other target outside [0, v) has loss (and gradients) NaN.
 */
#define LUMA_XENT_NONE 0   /* loss[n]                                              */
#define LUMA_XENT_SUM 1    /* loss[1]                                              */
#define LUMA_XENT_MEAN 2   /* loss[1], over the targets that are not ignored       */

typedef struct LumaXentArgs {
  const void *hidden;    /* device [n][h], rows ld_hidden elements apart         */
  const void *weight;    /* device [v][h], rows ld_weight elements apart         */
  const int64_t *target; /* device [n]                                           */
  int64_t n, h, v;       /* each >= 1                                            */
  int64_t ld_hidden, ld_weight;
  int64_t ignore_index;
  int32_t dtype;         /* LUMA_GRAD_*: both operands and both gradients        */
  int32_t reduction;     /* LUMA_XENT_*                                          */
  float *loss;           /* forward: device [n] or [1]                           */
  float *stats;          /* device [2 n + 1]: each token's largest logit, then each
                            one's sum of exp(l - largest), then the number of
                            targets that count (a sum or a mean); the forward
                            writes it, the backward reads it                     */
  const float *grad_loss;/* backward: device [n] or [1]                          */
  void *d_hidden;        /* backward: device [n][h] dense, or NULL               */
  void *d_weight;        /* backward: device [v][h] dense, or NULL               */
  void *workspace;       /* device, 256-byte aligned                             */
  int64_t workspace_bytes;
} LumaXentArgs;

/* Bytes of workspace that the call needs (from the sizes, the type and the
 * operands' addresses and strides); < 0: the arguments are refused. */
int64_t luma_xent_workspace_bytes(const LumaXentArgs *args, int32_t backward);
int luma_xent_forward(const LumaXentArgs *args, void *stream);
int luma_xent_backward(const LumaXentArgs *args, void *stream);

/*
 * Dropout whose mask is drawn from a counter-based generator and never stored.
 *
 * Element e of an operand (its index, rows one after the other) has 32 bits
 * u(e): the high 16 are half e % 8 (of the words x, y, z, w from the low end) of
 * the Philox4x32-10 block with counter (lo32(e / 8), hi32(e / 8), 0, call) and
 * the seed as key, the low 16 that half of the block with counter word 1 in
 * place of 0.  It is dropped (0, whatever it holds) where u(e) <
 * floor(p 2^32 + 1/2) and scaled by 1 / (1 - p) where not.  The backward draws
 * the same bits again.
 */
typedef struct LumaDropout {
  const int64_t *seed_at; /* device: the seed, read by the kernels; or NULL        */
  uint64_t seed;          /* the seed where seed_at is NULL                        */
  double p;               /* in [0, 1]; 0: nothing is drawn                        */
  uint32_t call;          /* tells the calls that share a seed from each other     */
  uint32_t reserved;      /* 0                                                     */
} LumaDropout;

/* y = residual + dropout(x), or dropout(x) without a residual; dense. */
typedef struct LumaDropoutArgs {
  const void *x;          /* device [numel], type `in`                             */
  const void *residual;   /* device [numel], type `out`, or NULL                   */
  void *y;                /* device [numel], type `out`                            */
  int64_t numel;          /* 1 to 2^34                                             */
  int32_t in, out;        /* LUMA_GRAD_*: the same, or one of them float32         */
  LumaDropout drop;
} LumaDropoutArgs;

/* (the backward is the same call on y's gradient, without a residual) */
int luma_dropout(const LumaDropoutArgs *args, void *stream);

/*
 * Layer normalisation over rows of h elements, alone or of the sum that a
 * block's border forms:
 *   s = x, or s = total = round(residual + dropout(x)) where residual is given;
 *   m = mean(s), r = 1 / sqrt(mean((s - m)^2) + eps), z = (s - m) r,
 *   y = z weight + bias
 * and for y's and total's gradients d_y, d_total, with g = d_y weight:
 *   d_s = r (g - mean(g) - z mean(g z)) + d_total,
 *   d_x = d_s, or d_residual = d_s and d_x = dropout's gradient of d_s,
 *   d_weight = sum over the rows of d_y z, d_bias = that of d_y.
 * Everything is formed in float32 and rounded once.  The sum's rounding to the
 * stream's type comes before its norm, so that y is the norm of the sum that a
 * program goes on with, and the backward, which reads that, has the same z.
 */
typedef struct LumaLayerNormArgs {
  const void *x;          /* device [n][h], rows ld_x elements apart; of the stream's
                             type, with a residual of the branch's                 */
  const void *residual;   /* device [n][h], rows ld_residual apart, or NULL        */
  const void *weight;     /* device [h] or NULL (1)                                */
  const void *bias;       /* device [h] or NULL (0)                                */
  int64_t n, h;           /* each >= 1; n below 2^31, h at most 2^24               */
  int64_t ld_x, ld_residual;
  int32_t stream;         /* LUMA_GRAD_*: of the residual and total                */
  int32_t branch;         /* LUMA_GRAD_*: of y; the stream's, or the stream is float32 */
  int32_t param;          /* LUMA_GRAD_*: of weight and bias: float32 or the branch's */
  int32_t reserved;       /* 0                                                     */
  double eps;
  LumaDropout drop;       /* of x, with a residual                                 */
  void *y;                /* forward: device [n][h] dense                          */
  void *total;            /* device [n][h] dense, with a residual: the forward writes
                             it, the backward reads it (and not x or residual)     */
  float *stats;           /* device [2 n]: each row's m, then each one's r; the
                             forward writes it (or NULL), the backward reads it    */
  const void *d_y;        /* backward: device [n][h] dense, the branch's type      */
  const void *d_total;    /* backward: device [n][h] dense, the stream's, or NULL  */
  void *d_x;              /* backward: device [n][h] dense, x's type, or NULL      */
  void *d_residual;       /* backward: device [n][h] dense, the stream's, or NULL  */
  void *d_weight;         /* backward: device [h], or NULL                         */
  void *d_bias;           /* backward: device [h], or NULL                         */
  void *workspace;        /* backward: device, 16-byte aligned                     */
  int64_t workspace_bytes;
} LumaLayerNormArgs;

/* Bytes of workspace that the backward needs (from n, h and stream); < 0: refused. */
int64_t luma_layer_norm_workspace_bytes(const LumaLayerNormArgs *args);
int luma_layer_norm_forward(const LumaLayerNormArgs *args, void *stream);
int luma_layer_norm_backward(const LumaLayerNormArgs *args, void *stream);

/*
 * The clipped policy loss of sampled tokens, with a KL term.
 *
 * For a token's log-probability l under the policy that learns, l_old under the
 * one that drew it, l_ref under a reference, and its advantage A:
 *   r = exp(l - l_old),  value = -min(r A, clip(r, 1 - clip_low, 1 + clip_high) A)
 *   q = l_ref - l,       value += kl_weight (exp(q) - 1 - q)
 * and d value / d l = -r A where r A is the smaller (or both are the same),
 * else 0, plus kl_weight (1 - exp(q)); a kl_weight of 0 leaves the term out,
 * whatever it is, and an A of 0 the ratio, if it is a number.  Which side of a
 * limit r lies on is decided on l - l_old in float64; values are float32, sums
 * float64.  A token whose mask is 0 has value and gradient 0, and counts
 * nowhere; nothing is formed of what its operands hold.
 */
#define LUMA_POLICY_SEQUENCE 3 /* the mean over the sequences that have tokens of each
                                  one's mean; LUMA_XENT_NONE, _SUM and _MEAN (over
                                  the tokens) are the others                       */
/* Floats at `stats`. */
#define LUMA_POLICY_STATS 4

typedef struct LumaPolicyArgs {
  const void *logp;       /* device [rows][length], rows ld_logp elements apart    */
  const void *old_logp;
  const void *ref_logp;   /* or NULL: no KL term                                   */
  const float *advantage; /* device [rows], or [rows][length] (advantage_each)     */
  const uint8_t *mask;    /* device [rows][length], 0 or 1, or NULL: every token   */
  int64_t rows, length;   /* each >= 1 and below 2^31, 2^40 tokens at most; rows of
                             more than 1,024: up to 2^22 of them                   */
  int64_t ld_logp, ld_old, ld_ref, ld_advantage, ld_mask;
  int32_t advantage_each; /* 1: an advantage for each token                        */
  int32_t dtype;          /* LUMA_GRAD_*: the log-probabilities and d_logp         */
  int32_t reduction;
  int32_t reserved;       /* 0                                                     */
  double clip_low, clip_high, kl_weight;
  float *loss;            /* forward: device [rows][length] dense, or [1]          */
  float *stats;           /* forward: device [LUMA_POLICY_STATS]: the share of the
                             tokens whose ratio was clipped, the means of exp(q) - 1
                             - q and of r - 1 - log r, the number of tokens; or NULL */
  float *share;           /* device [rows + 1]: each row's and the whole's factor of a
                             mean; the forward writes it (or NULL: there will be no
                             backward), the backward reads it                      */
  const float *grad_loss; /* backward: device [rows][length] dense, or [1]         */
  void *d_logp;           /* backward: device [rows][length] dense                 */
  void *workspace;        /* forward: device, 16-byte aligned                      */
  int64_t workspace_bytes;
} LumaPolicyArgs;

/* Bytes of workspace that the forward needs (from the sizes); < 0: refused. */
int64_t luma_policy_workspace_bytes(const LumaPolicyArgs *args);
int luma_policy_forward(const LumaPolicyArgs *args, void *stream);
int luma_policy_backward(const LumaPolicyArgs *args, void *stream);

/* Host: one Philox4x32-10 block. */
void luma_philox4x32(const uint32_t ctr[4], const uint32_t key[2], uint32_t out[4]);

#ifdef __cplusplus
}
#endif

#endif /* LUMA_H */
