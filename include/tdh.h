/*
 * tdh.h — C ABI of libtdh.so: tiny-dnn's training hot path on one AMD Instinct
 * MI355X (gfx950), hand-written HIP.
 *
 * The entry points are what tiny-dnn's operator layer binds for this path: each
 * one replaces the body of an OpKernel::compute (or of the free function the
 * reference calls in its place) and is cited next to its declaration (paths
 * relative to the tiny-dnn tree).
 *
 * Conventions
 *  - Every tensor argument is a DEVICE pointer obtained from tdh_malloc, dense
 *    fp32 (the operators of language models: the element type they are called with), [batch][flat] with tiny-dnn's per-sample CHW layout
 *    index = (H*c + y)*W + x  (tiny_dnn/util/util.h:168-173). Conv weights are
 *    OIHW, fully-connected weights [in][out] row-major.
 *  - Convolution inputs/gradients are UNPADDED; padding::same is applied
 *    implicitly by the kernels (the reference copies into padded buffers,
 *    tiny_dnn/core/params/conv_params.h:106-166).
 *  - Weight/bias gradients are produced already reduced over the batch (the sum
 *    over samples that edge::merge_grads computes, tiny_dnn/node.h:89-103) in a
 *    fixed order: the same inputs always give the same bits.
 *  - All work is queued on one library-owned stream; calls return without
 *    waiting for the GPU except tdh_sync, tdh_memcpy_d2h and tdh_event_elapsed_ms.
 *  - Every function returns TDH_OK (0) or a negative tdh_status; the message for
 *    the last failure on the calling thread is tdh_last_error(). The C++ host
 *    layer turns failures into tiny_dnn::nn_error, the reference's convention
 *    (tiny_dnn/util/nn_error.h:19-26).
 *  - Single caller thread (the reference's training thread); not re-entrant.
 */
#ifndef TDH_H
#define TDH_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum tdh_status {
  TDH_OK                = 0,
  TDH_ERR_INVALID       = -1, /* bad argument / unsupported shape */
  TDH_ERR_HIP           = -2, /* a HIP runtime call failed */
  TDH_ERR_NOT_INIT      = -3, /* tdh_init has not been called */
  TDH_ERR_UNSUPPORTED   = -4, /* valid in the reference but not built here */
  TDH_ERR_OOM           = -5
} tdh_status;

/* activation_layer subclasses (tiny_dnn/activations/) */
enum { TDH_ACT_TANH = 0, TDH_ACT_RELU = 1, TDH_ACT_SOFTMAX = 2, TDH_ACT_SIGMOID = 3,
       TDH_ACT_LEAKY_RELU = 4, TDH_ACT_ELU = 5, TDH_ACT_SELU = 6, TDH_ACT_SOFTPLUS = 7,
       TDH_ACT_SOFTSIGN = 8, TDH_ACT_ASINH = 9, TDH_ACT_TANH_P1M2 = 10, TDH_ACT_NONE = -1 };
/* loss functions (tiny_dnn/lossfunctions/loss_function.h) */
enum { TDH_LOSS_MSE = 0, TDH_LOSS_CE_MULTICLASS = 1, TDH_LOSS_CE = 2 };
/* optimizers (tiny_dnn/optimizers/optimizer.h) */
enum { TDH_OPT_SGD = 0, TDH_OPT_MOMENTUM = 1, TDH_OPT_ADAM = 2, TDH_OPT_ADAGRAD = 3,
       TDH_OPT_RMSPROP = 4, TDH_OPT_ADAMAX = 5, TDH_OPT_NESTEROV = 6 };
/* layer kinds of a sequential network */
enum { TDH_L_CONV = 0, TDH_L_FC = 1, TDH_L_MAXPOOL = 2, TDH_L_AVEPOOL = 3, TDH_L_ACT = 4,
       TDH_L_BATCHNORM = 5, TDH_L_DROPOUT = 6 };

/* element types of the operators that take a dtype (the others are fp32) */
enum { TDH_F32 = 0, TDH_BF16 = 1, TDH_F16 = 2 };
/* activations of a gated feed-forward block's gate: silu, gelu (erf), gelu (tanh form), sigmoid, relu, identity */
enum { TDH_GATE_SILU = 0, TDH_GATE_GELU = 1, TDH_GATE_GELU_TANH = 2, TDH_GATE_SIGMOID = 3, TDH_GATE_RELU = 4,
       TDH_GATE_NONE = 5 };
/* what a pair's margin m costs in tdh_preference_loss */
enum { TDH_PREF_SIGMOID = 0, TDH_PREF_SQUARED = 1, TDH_PREF_HINGE = 2 };

/* core::conv_params (tiny_dnn/core/params/conv_params.h:63-90) */
typedef struct tdh_conv_desc {
  int32_t in_w, in_h, in_c;
  int32_t k_w, k_h, out_c;
  int32_t w_stride, h_stride;
  int32_t w_dilation, h_dilation; /* forward only, as in the reference; backward needs 1 */
  int32_t pad_same;               /* 0 = padding::valid, 1 = padding::same */
  int32_t has_bias;
  const uint8_t *tbl;             /* HOST pointer: NULL or connection_table [in_c][out_c] */
} tdh_conv_desc;

/* core::maxpool_params (tiny_dnn/core/params/maxpool_params.h:17-34) and the
 * constructor arguments of average_pooling_layer */
typedef struct tdh_pool_desc {
  int32_t in_w, in_h, in_c;
  int32_t pool_w, pool_h;
  int32_t stride_w, stride_h;
  int32_t pad_same;
  int32_t ceil_mode;
} tdh_pool_desc;

/* Hyper-parameters plus the scalar state tiny-dnn keeps inside the optimizer
 * object: adam/adamax advance b1_t (and b2_t) once per update() call, i.e. once
 * per weight TENSOR (tiny_dnn/optimizers/optimizer.h:112-127,153-165). */
typedef struct tdh_opt {
  int32_t kind;
  float alpha, lambda, mu, b1, b2, eps;
  float b1_t, b2_t;
} tdh_opt;

typedef struct tdh_layer {
  int32_t kind;
  int32_t act; /* TDH_L_ACT: activation kind */
  tdh_conv_desc conv;
  tdh_pool_desc pool;
  int32_t fc_in, fc_out, fc_bias;
  float act_p[2]; /* TDH_L_ACT: constructor parameters of the kinds that have them (see tdh_act_fwd_p) */
  /* TDH_L_BATCHNORM: batch_normalization_layer(in_spatial_size, in_channels, epsilon, momentum)
   * (tiny_dnn/layers/batch_normalization_layer.h:54-72); tensors are [batch][channels][spatial] */
  int32_t bn_channels, bn_spatial;
  float bn_eps, bn_momentum;
  /* TDH_L_DROPOUT: dropout_layer(in_dim, dropout_rate) (tiny_dnn/layers/dropout_layer.h:32-39);
   * in_dim is the size of the layer in front */
  float dropout_rate;
} tdh_layer;

/* ------------------------------------------------------------ library state */
int tdh_init(int device);
int tdh_shutdown(void);
const char *tdh_last_error(void);
const char *tdh_version(void);
/* name, compute units and memory of the device selected by tdh_init */
int tdh_device_info(char *name, size_t name_len, int32_t *compute_units, size_t *global_mem_bytes);

/* ----------------------------------------------------------- device memory */
int tdh_malloc(void **dptr, size_t bytes);
int tdh_free(void *dptr);
int tdh_memcpy_h2d(void *dst, const void *src, size_t bytes);
int tdh_memcpy_d2h(void *dst, const void *src, size_t bytes); /* waits for queued work */
int tdh_memcpy_d2d(void *dst, const void *src, size_t bytes);
int tdh_fill_zero(void *dptr, size_t bytes);                  /* fill kernel, graph-safe */
int tdh_sync(void);

/* timing on the library stream */
int tdh_event_create(void **event);
int tdh_event_destroy(void *event);
int tdh_event_record(void *event);
int tdh_event_elapsed_ms(void *start, void *stop, float *ms); /* waits for `stop` */

/* Per-kernel timing of everything launched between begin and end: each launch carries
 * a pair of events that the runtime stamps with the begin and the end of that kernel's
 * execution, and is booked under a kernel tag with its algorithmic work (unit 0 = FLOP,
 * 1 = bytes); a tag's time is the sum over its kernels. A captured train step runs
 * eagerly while profiling is on, so whole-step throughput is measured with profiling
 * off. tdh_profile_end waits for the GPU; entries are then read back by index, ordered
 * by total time (largest first). */
int tdh_profile_begin(void);
int tdh_profile_end(int32_t *n_entries);
int tdh_profile_entry(int32_t index, char *tag, size_t tag_len, int64_t *launches,
                      double *total_ms, double *work_per_launch, int32_t *work_unit);
/* The tag of the index-th kernel launch of the profiled region, in dispatch order ("-" for a
 * launch outside any tag); TDH_ERR_INVALID (no error text) past the last one. It lets a trace
 * of the same run, which knows kernels only by symbol, be read tag by tag. */
int tdh_profile_launch(int32_t index, char *tag, size_t tag_len);
/* A mark in the kernel stream that a trace can find: three launches of the fill kernel on
 * `dptr` (which they clear), booked under the tag "profile_mark", never under the tag of a
 * workload's own fills. */
int tdh_profile_mark(void *dptr, size_t bytes);

/* shape helpers: conv_out_length / pool_out_length (tiny_dnn/util/util.h:329-363) */
int tdh_conv_out_w(const tdh_conv_desc *d);
int tdh_conv_out_h(const tdh_conv_desc *d);
int tdh_pool_out_w(const tdh_pool_desc *d);
int tdh_pool_out_h(const tdh_pool_desc *d);

/* ------------------------------------------------------------- convolution */
/* Conv2dOp::compute (tiny_dnn/core/kernels/conv2d_op.h:23-51,
 * conv2d_op_internal.h:13-74): y = conv(x, w) + b */
int tdh_conv2d_fwd(const tdh_conv_desc *d, int batch, const float *x, const float *w,
                   const float *b, float *y);
/* Conv2dGradOp::compute (tiny_dnn/core/kernels/conv2d_grad_op.h:22-50,
 * conv2d_op_internal.h:78-181). dx is overwritten; dw/db are overwritten
 * (accumulate = 0) or added to (accumulate = 1, the reference's += into gradients
 * that update_weight later clears). Any of dx, dw, db may be NULL to skip it. */
int tdh_conv2d_bwd(const tdh_conv_desc *d, int batch, const float *x, const float *w,
                   const float *dy, float *dx, float *dw, float *db, int accumulate);

/* tdh_conv2d_bwd for callers that cannot allocate (tight serving loops, harnesses that forbid
 * hipMalloc). It has no counterpart in the reference. It is refused (TDH_ERR_INVALID) while a
 * network step of this library is being captured or holds the scratch buffer, and
 * (TDH_ERR_UNSUPPORTED) for a descriptor with a connection table. Same
 * arguments, kernels and results as tdh_conv2d_bwd (a shape whose three-part kernels would not fit
 * runs the fp32 ones instead), but the kernels' scratch (split partial
 * sums, packed filters) lies in a static 64 MiB device array that the library holds on every
 * device it is initialised on, and the call allocates and frees nothing. A shape whose scratch
 * need exceeds the array is refused with TDH_ERR_INVALID (the message states both sizes); use
 * tdh_conv2d_bwd for it. All calls on one GPU share that GPU's array: calls are ordered by the
 * library stream, two processes' or threads' calls that overlap on one GPU would race. */
int tdh_conv2d_bwd_static(const tdh_conv_desc *d, int batch, const float *x, const float *w,
                          const float *dy, float *dx, float *dw, float *db, int accumulate);

/* --------------------------------------------------------- fully connected */
/* FullyConnectedOp::compute (tiny_dnn/core/kernels/fully_connected_op.h:25-63,
 * fully_connected_op_internal.h:15-36) */
int tdh_fc_fwd(int in, int out, int has_bias, int batch, const float *x, const float *w,
               const float *b, float *y);
/* FullyConnectedGradOp::compute (tiny_dnn/core/kernels/fully_connected_grad_op.h:22-52,
 * fully_connected_op_internal.h:38-71) */
int tdh_fc_bwd(int in, int out, int has_bias, int batch, const float *x, const float *w,
               const float *dy, float *dx, float *dw, float *db, int accumulate);

/* ----------------------------------------------------------------- pooling */
/* MaxPoolOp::compute (tiny_dnn/core/kernels/maxpool_op.h:23-61,
 * maxpool_op_internal.h:16-40). argmax[batch][out] = flat per-sample CHW index of
 * the first maximum in (dy,dx) scan order (the reference's out2inmax, held as
 * int32 here). */
int tdh_maxpool_fwd(const tdh_pool_desc *d, int batch, const float *x, float *y,
                    int32_t *argmax);
/* MaxPoolGradOp::compute (tiny_dnn/core/kernels/maxpool_grad_op.h:22-46,
 * maxpool_op_internal.h:42-57) */
int tdh_maxpool_bwd(const tdh_pool_desc *d, int batch, const float *dy, const int32_t *argmax,
                    float *dx);
/* AvePoolOp: tiny_average_pooling_kernel (tiny_dnn/layers/average_pooling_layer.h:25-55);
 * w and b hold one trainable scale / bias per channel */
int tdh_avepool_fwd(const tdh_pool_desc *d, int batch, const float *x, const float *w,
                    const float *b, float *y);
/* AvePoolGradOp: tiny_average_pooling_back_kernel
 * (tiny_dnn/layers/average_pooling_layer.h:58-106) */
int tdh_avepool_bwd(const tdh_pool_desc *d, int batch, const float *x, const float *w,
                    const float *dy, float *dx, float *dw, float *db, int accumulate);

/* ------------------------------------------------- activations and losses */
/* activation_layer::forward_propagation / back_propagation
 * (tiny_dnn/activations/activation_layer.h:74-91; tanh_layer.h:24-38,
 * relu_layer.h:25-39, softmax_layer.h:24-55, sigmoid_layer.h:24-38).
 * len = per-sample vector length; the backward uses the layer OUTPUT y. */
int tdh_act_fwd(int kind, int batch, int len, const float *x, float *y);
int tdh_act_bwd(int kind, int batch, int len, const float *y, const float *dy, float *dx);
/* The same for every activation layer, with the layer's constructor parameters p[2]:
 * leaky_relu {epsilon} (leaky_relu_layer.h:74-88), elu {alpha} (elu_layer.h:37-52),
 * selu {lambda, alpha} (selu_layer.h:82-99), softplus {beta, threshold}
 * (softplus_layer.h:84-102), softsign (softsign_layer.h:24-40), asinh (asinh_layer.h:24-38),
 * tanh_p1m2 (tanh_p1m2_layer.h:24-40); p is ignored by the other kinds and NULL selects the
 * constructor defaults. The backward takes the layer input x as well, as the reference's
 * backward_activation does: selu and softsign read it (x may be NULL for the others).
 * tdh_act_fwd / tdh_act_bwd are these calls with p = NULL and x = NULL. */
void tdh_act_default_params(int kind, float *p);
int tdh_act_fwd_p(int kind, const float *p, int batch, int len, const float *x, float *y);
int tdh_act_bwd_p(int kind, const float *p, int batch, int len, const float *x, const float *y,
                  const float *dy, float *dx);
/* batch_normalization_layer (tiny_dnn/layers/batch_normalization_layer.h:127-169): tensors are
 * [batch][channels][spatial]. train != 0: mean and variance receive this batch's moments
 * (util/math_functions.h:25-96: variance over max(1, batch*spatial - 1)); train == 0: they are
 * read (the moving averages). stddev[c] = sqrt(variance[c] + eps) is written either way and is
 * what the backward pass divides by. y = (x - mean) / stddev. */
int tdh_batchnorm_fwd(int channels, int spatial, int batch, float eps, int train, const float *x,
                      float *mean, float *variance, float *stddev, float *y);
/* batch_normalization_layer::back_propagation (batch_normalization_layer.h:87-125):
 * dx = (dy - mean(dy) - mean(dy*y) * y) / stddev, means per channel over batch and space */
int tdh_batchnorm_bwd(int channels, int spatial, int batch, const float *y, const float *dy,
                      const float *stddev, float *dx);
/* batch_normalization_layer::post_update (batch_normalization_layer.h:171-177):
 * mean = momentum*mean + (1-momentum)*mean_cur, the same for the variance */
int tdh_batchnorm_update_moving(int channels, float momentum, const float *mean_cur,
                                const float *var_cur, float *mean, float *variance);
/* dropout_layer (tiny_dnn/layers/dropout_layer.h:84-117): mask is [batch][len] bytes of 0/1, drawn
 * by the caller as the reference draws it (bernoulli(rate) per element, sample after sample);
 * train != 0: y = mask * scale * x with scale = 1/(1-rate), else y = x (mask may be NULL).
 * Backward (dropout_layer.h:62-82): dx = mask * dy, without the scale. */
int tdh_dropout_fwd(int batch, int len, int train, float scale, const uint8_t *mask, const float *x,
                    float *y);
int tdh_dropout_bwd(int batch, int len, const uint8_t *mask, const float *dy, float *dx);
/* gradient<E> for a mini-batch (tiny_dnn/lossfunctions/loss_function.h:191-218) */
int tdh_loss_grad(int kind, int batch, int len, const float *y, const float *t, float *dy);
/* softmax_layer backward applied to cross_entropy_multiclass::df in one kernel:
 * dz = y * sum(t) - t  (= y - t for one-hot targets) */
int tdh_softmax_xent_grad(int batch, int len, const float *y, const float *t, float *dz);

/* -------------------------------------------- operators of language models
 * They have no counterpart in the reference. `dtype` (TDH_F32, TDH_BF16, TDH_F16) is the element type of the
 * tensors declared void *; those declared float * are fp32 in every type. Sums are held in 32 bits or more, and
 * results are rounded once, to nearest. Tensors are aligned to their elements. No output may overlap
 * an input or another output, except where it is said that it may be an input. The same inputs give the same bits. */

/* Gated feed-forward block: z = x W + b, h = act(z_gate) * z_up. x [batch][in], w [in][2*hidden] with the gate's
 * columns first, b [2*hidden] (has_bias), h [batch][hidden]. z [batch][2*hidden], fp32, is what the backward pass
 * reads; NULL where there is none (inference). in up to 2^21, hidden up to 2^20, batch up to 2^24 (TDH_F32: 2^20), and
 * no tensor of 2^31 elements. */
int tdh_gated_ff_fwd(int dtype, int act, int in, int hidden, int has_bias, int batch, const void *x, const void *w,
                     const void *b, void *h, float *z);
/* dz = (dh * z_up * act'(z_gate), dh * act(z_gate)), dx = dz W^T, dw = x^T dz, db = the sum of dz over the batch. dx is overwritten;
 * dw and db (as in tdh_fc_bwd) overwritten, or added to with accumulate != 0. Any of dx, dw, db may be NULL.
 * In the 16-bit types dz is rounded to that type once, as the operand of the two products (not for up to four samples); in
 * TDH_F16 times a power of two that brings its largest finite value into [2^14, 2^15), so dz need not be in the type's range.
 * The derivative of relu at zero is 0. */
int tdh_gated_ff_bwd(int dtype, int act, int in, int hidden, int has_bias, int batch, const void *x, const void *w,
                     const float *z, const void *dh, void *dx, void *dw, void *db, int accumulate);

/* Dropout with the mask drawn on the device and stored nowhere: y = [residual +] (kept ? x / (1 - rate) : 0).
 * Element i is dropped where word i % 4 of Philox4x32-10 with counter (i / 4, offset) and key seed (low words
 * first) lies below floor(rate * 2^32): the same (seed, offset) gives the same mask, another offset another one.
 * A training step counts offset up, with a number of its own for every dropout layer in it. n elements in any layout;
 * residual may be NULL; y may be x or residual; 0 <= rate < 1. Unlike tdh_dropout_fwd, whose mask and missing
 * scale on the way back are the reference's, rate is the share that is dropped and the backward pass scales. */
int tdh_dropout_seeded_fwd(int dtype, size_t n, float rate, uint64_t seed, uint64_t offset, const void *x,
                           const void *residual, void *y);
/* dx = kept ? dy / (1 - rate) : 0 (the residual's gradient is dy itself); dx may be dy */
int tdh_dropout_seeded_bwd(int dtype, size_t n, float rate, uint64_t seed, uint64_t offset, const void *dy, void *dx);

/* Log-probabilities of given tokens: logp[r] = logits[r][target[r]] - m - log(s), m the row's maximum and
 * s = sum_j exp(logits[r][j] - m). Row r starts ld elements behind row r-1 (ld >= vocab). A row with a negative
 * target does not count (prompt, padding): its logits are not read, logp and stats are 0. A target of vocab or more
 * gives NaN. stats [rows][2] receives (m, s), from which the gradient is computed; NULL where there is none. vocab up to
 * 2^30, and fewer than 2^24 rows, of more than 65504 bytes fewer than 2^22; the same of the losses below. */
int tdh_token_logprob_fwd(int dtype, int rows, int vocab, const void *logits, size_t ld, const int32_t *target,
                          float *logp, float *stats);
/* dlogits[r][j] = dlogp[r] * ((j == target[r]) - exp(logits[r][j] - m) / s), zero in rows that do not count.
 * Rows of dlogits are ld_d elements apart; it may be logits itself (with ld_d == ld). */
int tdh_token_logprob_bwd(int dtype, int rows, int vocab, const void *logits, size_t ld, const int32_t *target,
                          const float *stats, const float *dlogp, void *dlogits, size_t ld_d);

/* Clipped policy loss with a KL term. Of row r, with the token target[r] (negative: the row does not count),
 *   ratio = exp(logp - old_logp), gap = ref_logp - logp,
 *   row_loss = weight * (-min(ratio * advantage, clamp(ratio, 1 - clip_low, 1 + clip_high) * advantage)
 *                        + kl_coef * (exp(gap) - gap - 1)),
 * loss[0] = the sum of row_loss, and dlogits its gradient. weight NULL: 1 for every row (1 / rows makes a mean). It is a
 * factor and no mask: 0 times an infinite loss is NaN, and rows whose values mean nothing have a negative target.
 * ref_logp NULL or kl_coef 0: no KL term. Any of logp, row_loss, loss and dlogits may be NULL; dlogits as in
 * tdh_token_logprob_bwd. Where the two sides of the minimum are equal the gradient is the first one's. */
typedef struct tdh_policy_desc {
  float clip_low, clip_high, kl_coef;
} tdh_policy_desc;
int tdh_policy_loss(const tdh_policy_desc *p, int dtype, int rows, int vocab, const void *logits, size_t ld,
                    const int32_t *target, const float *old_logp, const float *ref_logp, const float *advantage,
                    const float *weight, float *logp, float *row_loss, float *loss, void *dlogits, size_t ld_d);

/* Preference loss on paired log ratios. Sequence s is rows seq_start[s] .. seq_start[s+1]-1 (2*pairs + 1 ascending
 * values within 0 .. rows; a sequence may be empty); 2p is pair p's chosen answer, 2p+1 the rejected one. With
 * seq_logp[s] the sum of logp over the sequence's rows that count and ref_logp[s] the same of the reference
 * model (NULL: 0),
 *   margin = beta * ((seq_logp - ref_logp)[2p] - (seq_logp - ref_logp)[2p+1]), and its loss
 *   TDH_PREF_SIGMOID  (1 - smoothing) * log(1 + exp(-margin)) + smoothing * log(1 + exp(margin)), without the side whose
 *                     factor is 0
 *   TDH_PREF_SQUARED  ((margin - 1/2) / beta)^2
 *   TDH_PREF_HINGE    max(0, 1 - margin)   (derivative 0 at 1)
 * loss[0] = the mean over the pairs, dlogits its gradient. Any of logp [rows], seq_logp [2*pairs], margin [pairs],
 * loss and dlogits may be NULL; dlogits as above. Rows of logp and dlogits outside the sequences keep what they hold. */
typedef struct tdh_preference_desc {
  int32_t kind;
  float beta, smoothing;
} tdh_preference_desc;
int tdh_preference_loss(const tdh_preference_desc *p, int dtype, int pairs, int rows, int vocab, const void *logits, size_t ld,
                        const int32_t *target, const int32_t *seq_start, const float *ref_logp, float *logp,
                        float *seq_logp, float *margin, float *loss, void *dlogits, size_t ld_d);

/* Layer normalisation of rows: y = (x - mean) * rstd * gamma + beta with the row's mean and rstd = 1 / sqrt(variance + eps), the variance
 * over len. Rows of x are ld elements apart, of y ld_y (both >= len). gamma [len] and beta [len], or NULL for 1 and 0. stats [rows][2]
 * receives (mean, rstd), which the backward pass reads; NULL where there is none. y may be x (with ld_y == ld). eps is positive and
 * normal, len up to 2^24, fewer than 2^24 rows; sums are fp32, so the squares of a row's deviations have to add up to less than 2^127. */
int tdh_layernorm_fwd(int dtype, int rows, int len, float eps, const void *x, size_t ld, const void *gamma, const void *beta,
                      void *y, size_t ld_y, float *stats);
/* With xhat = (x - mean) * rstd and g = dy * gamma: dx = rstd * (g - mean(g) - xhat * mean(g * xhat)), means over the row; dgamma = the sum
 * over the rows of dy * xhat, dbeta = that of dy. dx is overwritten, and may be dy (with ld_dx == ld_dy); dgamma and dbeta are
 * overwritten, or added to with accumulate != 0. Any of dx, dgamma and dbeta may be NULL. Sums are fp32 here too: those of |g|, |g (x - mean)| and |dy xhat|
 * have to stay in its range. */
int tdh_layernorm_bwd(int dtype, int rows, int len, const void *x, size_t ld, const void *gamma, const float *stats,
                      const void *dy, size_t ld_dy, void *dx, size_t ld_dx, void *dgamma, void *dbeta, int accumulate);

/* A token of every row of logits, drawn with the row's number u in [0, 1). Of the tokens whose logit is not -inf, likeliest first and equal ones
 * by their index, these are left:
 *   the first top_k (0: all), of those
 *   the shortest beginning whose share of their probability softmax(logits / temperature) is top_p or more (1: all), of those
 *   the ones with at least min_p times the probability of the likeliest (0: all),
 * always the first one. token[r] is the first one left, by index, at which the sum of the probabilities of those left exceeds u times the sum
 * over all of them. temperature 0 takes the likeliest. logp[r] is the token's log-probability under softmax(logits), which
 * tdh_policy_loss takes as old_logp; logq[r] the one that it was drawn with; kept[r] how many were left; any of the three may be NULL. A u below 0
 * or NaN counts as 0, of 1 or more as the last number below 1, 1 - 2^-24. A row with NaN or +inf, or nothing but -inf, gives token -1, kept 0 and NaN.
 * Probabilities are computed to 2e-12 of themselves and summed as whole multiples of 2^-41 of the likeliest's or finer (vocab up to 2^17; of 2^(b - 58) up to
 * 2^b), so a call with the same inputs gives the same tokens.
 * settings (device, [rows]): each row's own descriptor in the place of p, or NULL. Values out of range there: top_k below 1
 * and top_p of 1 or more, and NaN, leave all; top_p of 0 or less the likeliest; min_p of 0 or less, and NaN, all, above 1 what has the likeliest's
 * logit; a temperature that is 0 or less or NaN takes the likeliest, an infinite one leaves all equal. vocab up to 2^30, fewer than 2^22 rows,
 * ld elements apart. */
typedef struct tdh_sample_desc {
  float temperature;
  int32_t top_k;
  float top_p, min_p;
} tdh_sample_desc;
int tdh_sample_tokens(const tdh_sample_desc *p, const tdh_sample_desc *settings, int dtype, int rows, int vocab, const void *logits, size_t ld,
                      const float *u, int32_t *token, float *logp, float *logq, int32_t *kept);

/* Products with weights in 8 bits. A row of weights holds one output's, wq [out][tdh_q8_row(in)], where bytes behind `in` are 0; output n stands for
 * wq[n] * wscale[n]. tdh_fc_q8_pack makes them of w [in][out]: wscale[n] = max |w[.][n]| / 127, wq = w / wscale rounded to nearest. */
size_t tdh_q8_row(int in); /* `in` rounded up to 16 */
int tdh_fc_q8_pack(int dtype, int in, int out, const void *w, int8_t *wq, float *wscale);
/* y = x W + b with every sample of x in 8 bits too: scale = max |x| / 127 of the sample (fp32), q = x / scale (fp32) rounded to nearest, ties to
 * even; y[m][n] = (sum_k q[m][k] wq[n][k]) * scale[m] * wscale[n] + b[n], the sum in 32-bit integers, which is exact. A sample with NaN or an
 * infinity gives NaN. in up to 2^17, out up to 2^20, batch up to 2^24, no tensor of 2^31 elements. wq lies on a 16-byte boundary. */
int tdh_fc_q8_fwd(int dtype, int in, int out, int has_bias, int batch, const void *x, const int8_t *wq, const float *wscale,
                  const void *b, void *y);

/* n elements from one element type to another, rounded to nearest: fp32 weights to the 16-bit ones that a block
 * computes with, and its 16-bit gradients to the fp32 ones that tdh_opt_update takes */
int tdh_cast(int dst_dtype, int src_dtype, size_t n, const void *src, void *dst);

/* -------------------------------------------------------------- optimizers */
/* layer::update_weight for one tensor (tiny_dnn/layers/layer.h:663-682) followed by
 * optimizer::update (tiny_dnn/optimizers/optimizer.h): g = merged_grad * grad_scale,
 * then the update of `kind`. tiny-dnn's own grad_scale is 1 (its rcp_batch_size is
 * taken from the weight edge, whose data tensor has one entry). s0/s1 are the
 * optimizer's per-weight state vectors (may be NULL where unused). *o is updated on
 * the host exactly as the reference updates b1_t/b2_t. */
int tdh_opt_update(tdh_opt *o, size_t n, const float *merged_grad, float grad_scale, float *w,
                   float *s0, float *s1);
void tdh_opt_default(tdh_opt *o, int kind);

/* The update of a matrix by its orthogonalised momentum (K. Jordan et al., "Muon: an optimizer for hidden layers in neural networks", 2024). It has no
 * counterpart in the reference. Of a matrix U, steps times from X = U / (|U| + eps), |U| the root of the sum of squares:
 *   A = X X^T, X <- a X + (b A + c A A) X       (A = X^T X on the right-hand side where there are more rows than columns)
 * which takes every singular value s to s (a + b s^2 + c s^4) and leaves the singular vectors: the result O is near the orthogonal factor of U.
 * products: TDH_F32 or TDH_F16, what the products' operands are held in. TDH_F32: in two fp16 parts, 22 bits, as precise as products in fp32. TDH_F16:
 * rounded to fp16 around known magnitudes. O is off by 3e-4 to 1.3e-3 of its size after five steps with a, b, c as they are by default; where a few singular
 * values are a thousand times the others, by 4e-3 to 8e-3 (of TDH_F32 by 4e-5), and three times that with every step more, since what is off beside the large
 * ones grows as the small ones do. X itself is held in 22 bits of either kind, and sums in fp32. Small matrices (up to 96 x 128, 64 x 256,
 * 32 x 512 and less, or turned round) go as TDH_F32 does.
 * Coefficients that take a singular value of at most 1 beyond 4 in any step are refused. Up to 16384 on the shorter side, 2^20 on the longer and
 * 2^30 elements in all. */
typedef struct tdh_muon {
  float alpha, mu, lambda; /* learning rate, momentum, decay */
  float scale;             /* of the update, beside alpha: sqrt(max(1, out / in)) and the like */
  int32_t nesterov;
  int32_t steps;           /* 0 to 32 */
  float a, b, c, eps;
  int32_t products;
} tdh_muon;
void tdh_muon_default(tdh_muon *o);
/* y = O of x [rows][cols]; may be x. alpha, mu, lambda, scale and nesterov are not read. */
int tdh_orthogonalize(const tdh_muon *o, int dtype, int rows, int cols, const void *x, void *y);
/* With g = merged_grad * grad_scale (merged_grad in dtype, weights and momentum in fp32, all [rows][cols]):
 *   momentum = mu * momentum + g, U = nesterov ? g + mu * momentum : momentum, w = w - alpha * (scale * O + lambda * w) */
int tdh_muon_update(const tdh_muon *o, int dtype, int rows, int cols, const void *merged_grad, float grad_scale, float *w, float *momentum);

/* ------------------------------------------------------ sequential network */
/* network<sequential>::fit / train_onebatch (tiny_dnn/network.h:840-926) with
 * every tensor resident on the device. */
typedef struct tdh_net tdh_net;

enum {
  TDH_NET_FUSE_ACT_GRAD = 1, /* fold activation gradients into the next layer's dX epilogue */
  TDH_NET_GRAPH         = 2, /* replay the step as a captured HIP graph */
  /* A net whose activations of one sample fit in a workgroup's local memory (LeNet-5) trains in
   * two to five launches: one workgroup per sample runs forward, the loss gradient and the input
   * gradients of the layers (the first block and the way back to it, a channel a workgroup, in launches of
   * their own for small batches); one launch computes the weight and bias gradients over groups of samples, whose
   * sizes follow from the layers and the batch. Where one group of all samples is the faster way, as in most nets
   * up to 16 or 32 samples, that launch updates as well; else every group leaves a slice, which the optimizer
   * launch adds up. Inside a group the order of a sum is fixed but is not the samples'; the slices are added in
   * the groups' order, also by a step without an update, which adds them to the gradient tensors
   * (edge::merge_grads, tiny_dnn/node.h:89-103). Every layer output, input gradient and max-pool record is still
   * written to memory. Nets that do not qualify (size, more than 2^26 parameters x max_batch, batch
   * normalization, dropout, a softmax that is not the closing layer of a cross_entropy_multiclass net) ignore
   * the flag. */
  TDH_NET_SAMPLE_STEP   = 4,
  /* Training never reads the gradient with respect to the net's input, which the reference
   * computes like every other (layer::backward of the first layer fills the gradient of its
   * data edge, tiny_dnn/layers/layer.h:557-575). With this flag a net whose first layer is a
   * convolution or a fully-connected layer leaves that product out: tdh_net_layer_dx(net, 0)
   * returns NULL after a step, everything else is what it is without the flag. Other first
   * layers ignore the flag. */
  TDH_NET_NO_INPUT_GRAD = 8
};

int tdh_net_create(const tdh_layer *layers, int n_layers, int max_batch, int flags,
                   tdh_net **net);
int tdh_net_destroy(tdh_net *net);
size_t tdh_net_in_size(const tdh_net *net);
size_t tdh_net_out_size(const tdh_net *net);
size_t tdh_net_layer_out_size(const tdh_net *net, int layer);
/* which: 0 = weight, 1 = bias; of a batch-norm layer (which has neither) 2 = moving mean,
 * 3 = moving variance (batch_normalization_layer.h:171-202, one value per channel, not touched
 * by the optimizer); sizes in floats */
size_t tdh_net_param_size(const tdh_net *net, int layer, int which);
int tdh_net_set_param(tdh_net *net, int layer, int which, const float *host_src);
int tdh_net_get_param(tdh_net *net, int layer, int which, float *host_dst);
/* optimizer::reset() as network::fit calls it before training (tiny_dnn/network.h:856,
 * tiny_dnn/optimizers/optimizer.h:36-38): clears the per-weight state vectors */
int tdh_net_reset_optimizer(tdh_net *net);
/* network::set_netphase (tiny_dnn/network.h:438-442): train != 0 is net_phase::train, the
 * state of a new net. In the train phase a batch-norm layer normalises by the moments of the
 * batch and every update moves its running averages (post_update), a dropout layer applies
 * its mask; in the test phase batch-norm uses the running averages and dropout is the identity. */
int tdh_net_set_phase(tdh_net *net, int train);
/* The mask that the following passes of dropout layer `layer` apply: host bytes [batch][len] of
 * 0/1, drawn by the caller as the reference draws them (bernoulli(dropout_rate) per element,
 * sample after sample, tiny_dnn/layers/dropout_layer.h:99-102), once per train step. The copy
 * is queued on the library stream, behind the kernels of the step before. */
int tdh_net_set_dropout_mask(tdh_net *net, int layer, int batch, const uint8_t *host_mask);
/* From now on dropout layer `layer` draws its masks itself, on the device (until tdh_net_set_dropout_mask hands it one
 * again): pass number p behind this call, counting train steps and forward passes in the train phase, does what
 * tdh_dropout_seeded_fwd and tdh_dropout_seeded_bwd do with (seed, offset + p), so the layer drops a share dropout_rate and scales
 * both ways. Nothing is uploaded between the steps, a captured step draws another mask at every replay, and
 * tdh_net_train_steps takes such a net. Layers of one net get seeds of their own, or offsets far apart. It has no
 * counterpart in the reference. */
int tdh_net_set_dropout_generator(tdh_net *net, int layer, uint64_t seed, uint64_t offset);
/* nodes::update_weights (tiny_dnn/nodes.h:103-107): layer::update_weight of every layer, front
 * to back, weight before bias, on the gradients accumulated since the last update, which are
 * then cleared (tiny_dnn/layers/layer.h:663-682). What tdh_net_train_step does with
 * do_update != 0, as a call of its own (network::update_weights, tiny_dnn/network.h:209-213). */
int tdh_net_update_weights(tdh_net *net, tdh_opt *opt);
/* nodes::clear_grads (tiny_dnn/nodes.h:118-122): zeroes every weight and bias gradient */
int tdh_net_clear_grads(tdh_net *net);
/* device views valid until the net is destroyed. The weights may be written through them between any
 * two calls: once a convolution's weights have been asked for here, a net packs the filters
 * that a pass or step reads anew in every call (one launch of a few microseconds at most), where it
 * otherwise keeps packed copies beside the weights. To look at weights, or to set them now and then,
 * tdh_net_get_param and tdh_net_set_param cost the following calls nothing. */
float *tdh_net_param(tdh_net *net, int layer, int which);
/* the layer's output as the last pass left it, or NULL where that pass never wrote it to
 * memory: in a train step with TDH_NET_FUSE_ACT_GRAD a convolution kernel that also writes the
 * pointwise activation or computes the 2x2 max-pool behind the convolution keeps the
 * convolution's own output in registers (nothing in the backward pass reads it: the gradients
 * of tanh, relu and sigmoid are functions of their outputs), with a pool directly behind the
 * convolution only in layers of few input channels or few tiles and in rows of fewer than 24 pixels;
 * tdh_net_forward always writes it */
const float *tdh_net_layer_out(const tdh_net *net, int layer);
/* the gradient with respect to the layer's input as the last step left it, or NULL where
 * that step never wrote it to memory: with TDH_NET_FUSE_ACT_GRAD the gradient of a folded
 * activation's output only exists in registers, and the backward kernels of a first
 * convolution (few input channels, stride 1) in front of a 2x2 / stride-2 max-pool read the
 * pooled gradient and the argmax records instead of the pool's input gradient */
const float *tdh_net_layer_dx(const tdh_net *net, int layer);
const float *tdh_net_layer_grad(const tdh_net *net, int layer, int which);
const int32_t *tdh_net_layer_argmax(const tdh_net *net, int layer);
/* x: [batch][in_size], t: [batch][out_size], device pointers */
int tdh_net_forward(tdh_net *net, int batch, const float *x);
/* fprop, loss gradient, bprop and (do_update != 0) update_weights + clear_grads */
int tdh_net_train_step(tdh_net *net, tdh_opt *opt, int loss_kind, int batch, const float *x,
                       const float *t, int do_update);
/* n_steps (1 to 8) consecutive train steps with update, step s on the mini-batch x[s], t[s]
 * (arrays of device pointers, which may repeat): what the loop over mini-batches of
 * network::fit does (tiny_dnn/network.h:866-879, one train_once per mini-batch) when the
 * batches are on the device already. The results are those of n_steps calls of
 * tdh_net_train_step; with TDH_NET_GRAPH the steps are captured into one graph, so a replay
 * starts once for all of them (a few microseconds each time, which is a tenth of a LeNet-5
 * step). A net with a dropout layer in the train phase is refused, unless that layer draws
 * its masks itself (tdh_net_set_dropout_generator): handed-over masks change between the steps. */
int tdh_net_train_steps(tdh_net *net, tdh_opt *opt, int loss_kind, int batch, int n_steps,
                        const float *const *x, const float *const *t);

/* ------------------------------------------------ batches from host memory */
/* network::fit hands each mini-batch over as host vectors (tiny_dnn/network.h:866-879;
 * layer::set_in_data copies them into the first layer, tiny_dnn/layers/layer.h:230-251).
 * A feeder takes them ahead of time: tdh_feeder_stage hands a batch in pageable host memory to
 * a worker thread of the feeder, which copies it into a pinned slot and queues its upload on a
 * copy stream at once; tdh_feeder_acquire makes the library stream wait for the upload of the
 * oldest staged batch and returns the device pointers to hand to tdh_net_train_step /
 * tdh_net_forward. Up to two batches may be staged and not yet acquired (stage, stage, then
 * acquire, stage, step, acquire, stage, step ...: the upload of a batch then overlaps the step
 * before it; staging one batch ahead works as well), a third is refused with TDH_ERR_INVALID.
 * x: [batch][x_len], t: [batch][t_len] floats; x_host / t_host must stay valid and unchanged
 * until the tdh_feeder_acquire that returns that batch. Queue every piece of work that reads a
 * batch before acquiring the next one: its device slot is reused by the second stage call
 * after that. */
typedef struct tdh_feeder tdh_feeder;
int tdh_feeder_create(size_t x_len, size_t t_len, int max_batch, tdh_feeder **feeder);
int tdh_feeder_destroy(tdh_feeder *feeder);
int tdh_feeder_stage(tdh_feeder *feeder, int batch, const float *x_host, const float *t_host);
int tdh_feeder_acquire(tdh_feeder *feeder, const float **x_dev, const float **t_dev, int *batch);

#ifdef __cplusplus
}
#endif
#endif /* TDH_H */
