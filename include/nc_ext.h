/*
 * nc_ext.h — side API of the B200 newch engine.
 *
 * These entry points have no counterpart in newch's engine/include/nc.h, whose ABI stays frozen.
 * They sit where newch plans its optional engine/src/ext/ module (newch CLAUDE.md:83-85): device
 * facts, data-parallel set-up (NCCL over NVLink/NVSwitch) and counters for benchmarks. A newch
 * user needs none of them: data parallelism can also be switched on purely through the
 * environment (NC_RANK, NC_WORLD_SIZE, NC_NCCL_ID_FILE), read by nc_init.
 */
#ifndef NC_EXT_H
#define NC_EXT_H

#include "nc.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Number of visible CUDA devices (0 when there is none or the driver is missing). */
NC_API int nc_ext_device_count(void);
/* Name of the context's device, e.g. "NVIDIA B200". */
NC_API const char *nc_ext_device_name(const nc_ctx *ctx);
/* Waits for all work enqueued by the context; returns its status code (kernel-found errors become
 * NC_ERR_ARG, CUDA failures NC_ERR_STATE). */
NC_API int nc_ext_synchronize(nc_ctx *ctx);
/* Kernels this context has enqueued since nc_init. */
NC_API int64_t nc_ext_launch_count(const nc_ctx *ctx);
/* "ffma", "tf32" or "3xtf32": how fp32 GEMMs run (NC_GEMM env; force_reference forces "ffma"). */
NC_API const char *nc_ext_gemm_mode(const nc_ctx *ctx);

/* Writes an NCCL unique id (bytes) into buf; returns its length or -1. Rank 0 calls it and sends
 * the bytes to the other ranks by any host channel. */
NC_API int nc_ext_nccl_unique_id(void *buf, int cap);
/* Joins the context to a data-parallel group of `world` ranks. After this, nc_optim_step averages
 * the gradients of all ranks (one all-reduce of the flat gradient buffer) before updating.
 * Returns NC_OK or an error status. */
NC_API int nc_ext_dp_init(nc_ctx *ctx, int rank, int world, const void *id, int id_len);
NC_API int nc_ext_dp_world(const nc_ctx *ctx);
/* Dropout streams of a data-parallel group that reproduce newch's gradient accumulation over the
 * ranks' batches (rank r's step draws what newch draws for the r-th micro-batch of an accumulated
 * step): every step of every rank takes at most `draws_per_step` random numbers, rank r starts r
 * strides into each step's span of world * draws_per_step draws, and nc_step_end moves it to its
 * place in the next span. Call after nc_ext_dp_init, at the point training starts. 0 turns the
 * interleaving off. Returns NC_OK or NC_ERR_ARG. */
NC_API int nc_ext_dp_rng_stride(nc_ctx *ctx, int64_t draws_per_step);
/* Random numbers taken from the context's stream since it was seeded. */
NC_API int64_t nc_ext_rng_position(const nc_ctx *ctx);

/* The cudaStream_t every kernel of this context runs on. */
NC_API void *nc_ext_stream(nc_ctx *ctx);
/* Per-kernel timing with CUDA events on the context's stream (costs a little per launch). */
NC_API int nc_ext_timing(nc_ctx *ctx, int on);
/* Sum of device milliseconds and the number of timed launches of kernels whose name starts with
 * `prefix` ("" = all) since timing was switched on. */
NC_API int nc_ext_kernel_time(nc_ctx *ctx, const char *prefix, double *ms, int64_t *count);
/* Timed kernel class i (0-based): its name, total device milliseconds, launches and the algorithmic
 * work of those launches (FLOPs, and bytes that must move: each logical input read once, each
 * output written once). Returns 0 when i is past the last class. */
NC_API int nc_ext_kernel_entry(nc_ctx *ctx, int i, const char **name, double *ms, int64_t *count, double *flops,
                               double *bytes);
/* Clears the accumulated timings (timing stays on). */
NC_API void nc_ext_timing_reset(nc_ctx *ctx);

/* Failure-reporting probe: launches one kernel whose tensor-core pipeline wait (an mbarrier that
 * never completes) gives up after its 2 s bound, as every tcgen05 kernel's waits do, then
 * synchronizes. Returns the context status: NC_ERR_STATE with "pipeline wait timed out" in
 * nc_error. The device stays usable: nc_clear_error and continue. */
NC_API int nc_ext_pipeline_wait_probe(nc_ctx *ctx);

/* Cross-entropy forward on caller-owned device buffers that allocates nothing. It has no
 * counterpart in newch; the arithmetic is the engine's nc_cross_entropy (newch
 * engine/src/ops/ops_nn.c:107-149): prob[rows, classes] = softmax(logits) and
 * *loss = -mean(log prob[r, labels[r]]), with the mean summed in double in a fixed order.
 *
 * For callers that must not have device memory allocated on their behalf while they run (a runtime
 * that owns and accounts for the whole device pool, a latency-critical loop, a process at its
 * memory limit): the only scratch is a static device array of NC_EXT_CE_NOALLOC_MAX_ROWS floats.
 * All pointers are device pointers; `stream` is a cudaStream_t (NULL = the legacy default stream).
 * The call is asynchronous. Returns NC_OK, NC_ERR_ARG (rows < 0, rows > NC_EXT_CE_NOALLOC_MAX_ROWS,
 * classes <= 0, or a NULL pointer; nothing is launched) or NC_ERR_STATE (CUDA set-up or launch
 * failure).
 * - The first call on a device (made with that device current) looks up the static array's address
 *   in the current CUDA context; a later call under another context (after cudaDeviceReset, say)
 *   looks it up again. Make such a first call before any stream capture begins.
 * - Launch failures are taken from the launches themselves: an error the caller left pending in the
 *   runtime's last-error slot is neither reported nor cleared.
 * - *status must start at zero; a label outside [0, classes) sets it to 2 (that row's label is
 *   read as class 0). The static array needs no initialisation.
 * - Calls on one device share the static array: calls that can run at the same time (on streams
 *   with no ordering between them) race on it. Calls ordered on one stream are safe. */
#define NC_EXT_CE_NOALLOC_MAX_ROWS 262144
NC_API int nc_ext_cross_entropy_fwd_noalloc(const float *logits, const int32_t *labels, int64_t rows,
                                            int64_t classes, float *prob, float *loss, int *status, void *stream);

/* ---- tensors on the device -----------------------------------------------------------------------
 * Address of t's element 0 in device memory (a view's own first element; strides as created), with host
 * writes pushed and pending values computed. The data is that of the context's stream: a reader or writer on
 * another stream orders itself after nc_ext_stream (an event, or nc_ext_synchronize) and before the next op.
 * write != 0 says that the caller will write through the address: host mirrors are dropped and pending values
 * that read t are computed first (ask again before each round of writes). The address holds until t is released
 * or, for a temporary, until nc_step_end. NULL when t is NULL or holds no data, or the context has an error. */
NC_API void *nc_ext_device_data(nc_tensor *t, int write);
/* nc_backward from any f32 tensor y with dy as the gradient of it (same shape, any strides, same context)
 * instead of a scalar loss with gradient 1. dy is read, never written or kept; it may be a gradient that a pass
 * left (a retained one's of an intermediate tensor keeps its values until nc_step_end; a leaf's is read as it was
 * and then added to, as in every pass). Returns the context status. */
NC_API int nc_ext_backward_from(nc_tensor *y, nc_tensor *dy);

/* ---- query/key norms with rotary positions -------------------------------------------------------
 * x [batch, tokens, heads, dim] f32 (any strides; a slice of a fused projection is read in place) holds
 * query heads, then key heads. Each head's vector is divided by its root mean square (x * (mean x^2 +
 * eps)^-1/2), multiplied by q_weight (the first q_heads heads) or k_weight (the others), both [dim] f32 or
 * NULL for none, and rotated by its position: pair i, of dim / 2, is elements (i, dim/2 + i), or (2i, 2i + 1)
 * with NC_EXT_ROPE_INTERLEAVED. One pass over x; the result is contiguous and has x's shape.
 *
 * positions: i32 [tokens, n_axes] or [batch, tokens, n_axes] (time, height, width, ...; any i32 value), or
 * NULL with one axis: the token's index. The first sections[0] pairs follow axis 0, the next sections[1] axis
 * 1, and so on; pairs behind the last section are not rotated. Pair i turns by base^(-i / (dim/2)) radians per
 * step of its axis; with NC_EXT_ROPE_AXIS_FREQ by base^(-j / sections[a]), j counting from the start of its
 * section, so that every axis has the whole range of frequencies. Angles are formed in 64 bits.
 * NC_EXT_ROPE_NO_NORM leaves the division out (weights still apply).
 *
 * dim is even, 2 to 256; 1 to 3 axes; the sections sum to at most dim / 2. Gradients reach x, q_weight and
 * k_weight, in an order of summation that is the same every time. */
enum { NC_EXT_ROPE_INTERLEAVED = 1, NC_EXT_ROPE_AXIS_FREQ = 2, NC_EXT_ROPE_NO_NORM = 4 };
typedef struct {
    int q_heads;
    int n_axes;
    int sections[3];
    float base;
    float eps;
    int flags;
} nc_ext_rope_opts;
NC_API nc_tensor *nc_ext_qk_norm_rope(nc_tensor *x, nc_tensor *q_weight, nc_tensor *k_weight, nc_tensor *positions,
                                      const nc_ext_rope_opts *opts);

/* ---- losses on logits for tuning a language model ---------------------------------------------------
 * Both take f32 logits [rows, vocab] or [batch, tokens, vocab] (any strides with adjacent vocabulary entries:
 * a slice of tokens is read in place), i32 labels and mask of the leading shape (mask NULL: every row counts,
 * else rows whose entry is not 0; other integer types are converted), and return a scalar with gradients to
 * the logits. Rows that the mask leaves out are not read: their logits, labels and other entries may hold
 * anything, and their gradient is 0. A counted label outside [0, vocab) is an error (found on the device at
 * the latest: NC_ERR_ARG at the next synchronisation). Logits of -infinity have probability 0. Log
 * probabilities are subtracted and summed, and the KL term formed, in 64 bits, ratios and what is clipped of them
 * in 32; sums run in the same order every time.
 *
 * Everything but the logits is a constant: while gradients are enabled, an input of the others that requires
 * grad is refused. */

/* The clipped policy loss with a KL term: with lp the log probability of a row's action, ratio = exp(lp -
 * old_logp) and away = ref_logp - lp,
 *   loss = mean over counted rows of  -min(ratio A, clip(ratio, 1 - clip_low, 1 + clip_high) A)
 *                                     + kl_coef (exp(away) - away - 1)
 * (0 when no row counts). old_logp, ref_logp and advantages are f32 of the leading shape; ref_logp may be NULL
 * when kl_coef is 0. *logp (when logp is not NULL) becomes lp of every row as f32, 0 for rows left out,
 * without gradient. clip_low lies in [0, 1], clip_high is at least 0, kl_coef finite. */
typedef struct {
    float clip_low;
    float clip_high;
    float kl_coef;
} nc_ext_policy_opts;
NC_API nc_tensor *nc_ext_policy_loss(nc_tensor *logits, nc_tensor *actions, nc_tensor *old_logp, nc_tensor *ref_logp,
                                     nc_tensor *advantages, nc_tensor *mask, const nc_ext_policy_opts *opts,
                                     nc_tensor **logp);

/* The preference loss of pairs of answers: logits [2 pairs, tokens, vocab], the preferred answers first, in
 * the order of the others. With s the sum of an answer's counted log probabilities and h = beta ((s - ref) of
 * the preferred - (s - ref) of the other),
 *   loss = mean over pairs of  -(1 - label_smoothing) log sigmoid(h) - label_smoothing log sigmoid(-h)
 * ref_logp: f32 [2 pairs], the reference model's sums, or NULL for 0. *seq_logp (when seq_logp is not NULL)
 * becomes s as f32 [2 pairs], without gradient. beta is positive, label_smoothing lies in [0, 0.5]. */
NC_API nc_tensor *nc_ext_preference_loss(nc_tensor *logits, nc_tensor *labels, nc_tensor *ref_logp, nc_tensor *mask,
                                         float beta, float label_smoothing, nc_tensor **seq_logp);

/* ---- AdamW with 8-bit moments ------------------------------------------------------------------------
 * nc_adamw with 16 bytes of memory traffic and 2.03 bytes of state per element instead of 28 and 8: both
 * moments are kept as one byte an element and an fp32 maximum s per block of 256 elements of a parameter,
 *   m = sign(c) s (c / 127)^2, c in [-127, 127];   v = s (c / 255)^4, c in [0, 255], 0 for v = 0 only,
 * each rounded to the nearest code (in sqrt|m| and v^(1/4)) after the step. The step uses the moments before
 * that rounding, in fp32. Blocks whose largest value is below 2^-94 count as zero; a v beyond fp32, from
 * a finite gradient, is held as the largest float (the step itself divides by infinity: it moves nothing); a gradient
 * that is not finite makes the moments of its block not finite. The handle works with every nc_optim_* call, gradient
 * accumulation and data parallelism included; nc_optim_state shows the moments as floats, and floats written
 * through it are encoded again before the next step (v by its absolute value). Defaults as nc_adamw. A parameter is given once. */
NC_API nc_optim *nc_ext_adamw8(nc_ctx *ctx, nc_tensor **params, int n, nc_optim_opts opts);
/* The moments of an optimizer that keeps two (Adam, AdamW, AdamW in 8 bits, RMSprop with momentum: its momentum
 * and square average) copied to or from a contiguous f32 tensor [2, elements] on the device: row 0 m, row 1 v, the parameters one
 * after the other. 8-bit moments are decoded and encoded; encoding what was decoded restores them bit for
 * bit. Together with nc_optim_get_step / set_step a checkpoint without a host copy. get_state
 * shows what was written through nc_optim_state's pointers, and they stay good for more until the next step;
 * put_state replaces everything and ends them (take them again). Return the context status. */
NC_API int nc_ext_optim_get_state(nc_optim *o, nc_tensor *values);
NC_API int nc_ext_optim_put_state(nc_optim *o, nc_tensor *values);

#ifdef __cplusplus
}
#endif

#endif /* NC_EXT_H */
