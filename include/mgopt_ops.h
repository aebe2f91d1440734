/*
 * mgopt_ops.h -- C ABI of the operators of a training step around its matrix
 * products and attention (libmgopt.so): token embedding, query/key norms with
 * the rotary rotation, the MLP's activation with an 8-bit checkpoint, and the
 * clipped policy loss.  Their gradients are the ones the optimizer step
 * (mgopt.h) reads.
 *
 * Conventions are those of mgopt.h: *_dev arguments are device pointers to
 * memory of the caller's, calls are asynchronous on `stream` and wait for
 * nothing, the return value is 0 or a hipError_t / MGOPT_E_* code that
 * mgopt_last_error() explains.  Calls launch on the current device, which must
 * be the stream's.  They allocate nothing, so they can be captured in a graph.
 * Element types are MGOPT_F32, MGOPT_F16 and MGOPT_BF16; strides count
 * elements; the last dimension is always contiguous.  Arithmetic, sums and
 * statistics are held in 32 bits or more and rounded once to the output's type.
 * Same inputs give the same bits: no result depends on the order of atomics.
 */
#ifndef MGOPT_OPS_H
#define MGOPT_OPS_H

#include <stdint.h>

#include "mgopt.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- token embedding -------------------------------------------------------- */

/* out[t] = scale * weight[ids[t]] for n ids of id_bytes (4 or 8) bytes; weight
 * is [rows][width], out [n][width], both contiguous.  An id outside
 * [0, rows) gives a row of NaN. */
MGOPT_API int mgopt_embedding(const void* ids_dev, int32_t id_bytes, int64_t n, const void* weight_dev,
                              int32_t weight_dtype, int64_t rows, int64_t width, float scale, void* out_dev,
                              int32_t out_dtype, void* stream);

MGOPT_API int64_t mgopt_embedding_grad_workspace(int64_t n, int64_t rows, int64_t width);

/* grad[v] = scale * sum of grad_out[t] over the t with ids[t] = v, and, with
 * accumulate, added to what grad[v] holds: then only rows that the ids name are
 * read and written, otherwise every row is written.  grad_out is [n][width],
 * grad [rows][width], both contiguous.  Ids outside [0, rows) and equal to
 * padding_idx (-1: none) add nothing.  workspace_dev:
 * mgopt_embedding_grad_workspace bytes, 16-byte aligned.  Fewer than 2^30 ids
 * and 2^31 rows (MGOPT_E_LIMIT). */
MGOPT_API int mgopt_embedding_grad(const void* ids_dev, int32_t id_bytes, int64_t n, const void* grad_out_dev,
                                   int32_t grad_out_dtype, void* grad_dev, int32_t grad_dtype, int64_t rows,
                                   int64_t width, float scale, int64_t padding_idx, int32_t accumulate,
                                   void* workspace_dev, void* stream);

/* ---- the MLP's activation ------------------------------------------------ */

#define MGOPT_ACT_SILU 0       /* x / (1 + exp(-x)) */
#define MGOPT_ACT_GELU_TANH 1  /* x (1 + tanh(sqrt(2/pi) (x + 0.044715 x^3))) / 2 */
#define MGOPT_ACT_GROUP 128    /* elements of a row that share a scale in a checkpoint */

/* y = act(gate) * up, or act(gate) where up_dev is NULL, for `rows` rows of
 * `width` elements; y is contiguous.  With codes_dev and scales_dev, also the
 * 8-bit checkpoint of gate and up that mgopt_gated_act_backward reads: with
 * G = ceil(width / 128) groups a row, codes_dev (8-byte aligned) holds
 * [inputs][rows][G * 128] int8 and scales_dev [inputs][rows][G] floats, inputs
 * being gate and, where there is one, up.  A group whose largest magnitude is
 * m holds scale = m * (1/127) and the integers nearest to x * (127 / m), ties
 * to even; m below 2^-119 counts as 0, and a group with an inf or a NaN has
 * the scale NaN. */
MGOPT_API int mgopt_gated_act(const void* gate_dev, int64_t gate_stride, const void* up_dev, int64_t up_stride,
                              int32_t dtype, int64_t rows, int64_t width, int32_t act, void* y_dev, int8_t* codes_dev,
                              float* scales_dev, void* stream);

/* From the gradient of y and the checkpoint (g, u): d_gate = dy * u * act'(g),
 * d_up = dy * act(g) (d_up_dev is NULL exactly where gated is 0, and u is 1
 * then), and, where y_dev is not NULL, y = act(g) * u again, contiguous. */
MGOPT_API int mgopt_gated_act_backward(const void* grad_out_dev, int64_t grad_out_stride, const int8_t* codes_dev,
                                       const float* scales_dev, int32_t gated, int32_t dtype, int64_t rows,
                                       int64_t width, int32_t act, void* d_gate_dev, int64_t d_gate_stride,
                                       void* d_up_dev, int64_t d_up_stride, void* y_dev, void* stream);

/* ---- query/key norms and the rotation -------------------------------------- */

#define MGOPT_MAX_HEAD_DIM 512

/* The heads of one side.  Every *_stride is {batch, token, head}, in elements;
 * a head's `dim` elements are contiguous.
 *   x_dev         the projection's output; out_dev the result (forward only).
 *   grad_dev      the gradient of out, d_x_dev that of x, d_weight_dev that of
 *                 weight_dev, of its type (backward only). */
typedef struct mgopt_heads {
    const void* x_dev;
    const void* weight_dev;
    void* out_dev;
    const void* grad_dev;
    void* d_x_dev;
    void* d_weight_dev;
    int64_t x_stride[3];
    int64_t out_stride[3];
    int64_t grad_stride[3];
    int64_t d_x_stride[3];
    int32_t heads;
    int32_t reserved;
} mgopt_heads;

/* cos_dev and sin_dev hold table_rows rows of rotary / 2 floats, one per
 * position.  positions_dev: of position_bytes (4 or 8) bytes, position_stride
 * apart from one sequence to the next (0: all alike), or NULL for 0, 1, ...  A
 * position outside the table makes its token's rotated elements NaN.  Pairs are
 * (i, i + rotary / 2), or (2i, 2i + 1) with interleaved; elements from `rotary`
 * on are not rotated.  At most 2^28 tokens. */
typedef struct mgopt_qk_args {
    mgopt_heads q;
    mgopt_heads k;
    const float* cos_dev;
    const float* sin_dev;
    const void* positions_dev;
    void* workspace_dev; /* backward: mgopt_qk_norm_rope_workspace(dim) bytes */
    int64_t table_rows;
    int64_t position_stride;
    int64_t batch;
    int64_t length;
    int32_t dim;
    int32_t rotary;
    int32_t dtype;
    int32_t weight_dtype;
    int32_t position_bytes;
    int32_t interleaved;
    float eps;
    int32_t reserved;
} mgopt_qk_args;

/* out = rotate(x / sqrt(mean(x^2) + eps) * weight) for every head. */
MGOPT_API int mgopt_qk_norm_rope(const mgopt_qk_args* args, void* stream);

MGOPT_API int64_t mgopt_qk_norm_rope_workspace(int32_t dim);

/* d_x and d_weight from x and the gradient of out. */
MGOPT_API int mgopt_qk_norm_rope_backward(const mgopt_qk_args* args, void* stream);

/* ---- the clipped policy loss ---------------------------------------------- */

#define MGOPT_MASK_NONE 0   /* every row counts once */
#define MGOPT_MASK_BYTES 1  /* one byte a row: 0 leaves it out */
#define MGOPT_MASK_F32 2    /* a weight a row */

/* Row n holds the logits of one token.
 *   logits_dev     [rows] of `vocab` elements, logits_stride elements apart.
 *   targets_dev    the token that was taken, of target_bytes (4 or 8) bytes.
 *   old_logp_dev, advantages_dev, ref_logp_dev (NULL: no KL term): [rows].
 *   mask_dev       by mask_kind.  A row of weight 0 is not read: its target,
 *                  logits and other values may be anything.
 *   clip_low,
 *   clip_high      the ratio is clipped to [1 - clip_low, 1 + clip_high].
 *   grad_scale_dev a factor of the gradient (a loss scaler's scale, or the
 *                  gradient of the loss), or NULL.
 *   log_probs_dev  [rows]: each row's log-probability of its target, 0 for a
 *                  row of weight 0.
 *   d_logits_dev   the gradient, of the logits' type, or NULL; it may be
 *                  logits_dev itself with the same stride.
 *   workspace_dev  mgopt_policy_workspace(rows) bytes, 16-byte aligned.
 * A target outside [0, vocab) in a row that counts makes the loss and that
 * row's gradient NaN. */
typedef struct mgopt_policy_args {
    const void* logits_dev;
    const void* targets_dev;
    const float* old_logp_dev;
    const float* advantages_dev;
    const float* ref_logp_dev;
    const void* mask_dev;
    const float* grad_scale_dev;
    float* log_probs_dev;
    void* d_logits_dev;
    void* workspace_dev;
    int64_t rows;
    int64_t vocab;
    int64_t logits_stride;
    int64_t d_logits_stride;
    double clip_low;
    double clip_high;
    double kl_coef;
    double temperature; /* from 2^-120 to 2^120 */
    int32_t dtype;
    int32_t target_bytes;
    int32_t mask_kind;
    int32_t reserved;
} mgopt_policy_args;

MGOPT_API int64_t mgopt_policy_workspace(int64_t rows);

/* Writes log_probs_dev.  Reads logits, targets and mask.  The workspace may be
 * NULL: fewer than 128 long rows are then not cut in slices, and their sums, of
 * another order, may differ in the last bits. */
MGOPT_API int mgopt_token_log_probs(const mgopt_policy_args* args, void* stream);

/* With logp = log_softmax(logits / temperature)[target], ratio =
 * exp(logp - old_logp) and r = ref_logp - logp:
 *   policy = -min(ratio * A, clip(ratio) * A)    kl = exp(r) - r - 1
 * loss_dev[0] = mean(policy) + kl_coef * mean(kl), parts_dev[0..2] =
 * mean(policy), mean(kl) and the share of rows whose gradient the clip holds at
 * 0, all weighted by the mask (0 where the weights' sum is 0).  With d_logits_dev,
 * also the gradient of grad_scale * loss, reading the logits once; without it,
 * the workspace keeps what mgopt_policy_loss_backward needs. */
MGOPT_API int mgopt_policy_loss(const mgopt_policy_args* args, float* loss_dev, float* parts_dev, void* stream);

/* The gradient of grad_scale * loss, after mgopt_policy_loss without
 * d_logits_dev on the same arguments, log_probs_dev and workspace_dev: the same
 * bits as mgopt_policy_loss gives with d_logits_dev. */
MGOPT_API int mgopt_policy_loss_backward(const mgopt_policy_args* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* MGOPT_OPS_H */
