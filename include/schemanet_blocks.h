/*
 * schemanet_blocks.h -- C ABI of libschemanet_hip.so, second part: the operators of deep residual graph networks and of large
 * sets of answers.  The conventions are those of schemanet_hip.h (plain device pointers, sizes, a hipStream_t as void*;
 * nothing allocates, synchronises or throws; 0 = enqueued, < 0 = rejected with a message in sn_last_error()).
 *
 * Types of the tensors are given by SN_F32 / SN_BF16 / SN_F16; all arithmetic is fp32, each result is rounded once.
 * Strides count elements, rows are contiguous, no alignment beyond the element's own is needed.
 */
#ifndef SCHEMANET_BLOCKS_H
#define SCHEMANET_BLOCKS_H

#include "schemanet_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define SN_F32 0
#define SN_BF16 1
#define SN_F16 2

/* Version of this header's declarations, bumped on any change of a signature or of a by-pointer struct. */
int sn_blocks_abi_version(void);

/* ------------------------------------------------------------------------------------------
 * 8-bit checkpoints of activations
 * A row of n features is kept in blocks of 32: code byte q in -127 .. 127 and one exponent byte e a block, the value is
 * q * 2^(e - 133).  2^(e - 133) is the smallest power of two s with max|x| < 127.5 s, q = round-half-even(x / s): every kept
 * value is exact in bfloat16.  e is at least 8 (magnitudes under 2^-126 are kept as zero); e = 255 marks a block that held an
 * infinity or a NaN: all its values come back as NaN.
 * codes [rows, npad] int8, exps [rows, npad / 32] uint8, npad = n rounded up to 32 (the codes beyond n are zero).
 * ------------------------------------------------------------------------------------------ */
int sn_checkpoint8(const void *x, int dtype, int64_t rows, int n, int64_t row_stride, void *codes, void *exps, void *stream);
/* out [rows, n] contiguous; SN_F16: kept values beyond 65504 come back as 65504 (8 bits round 65024 .. 65504 up to 65536) */
int sn_checkpoint8_restore(const void *codes, const void *exps, int64_t rows, int n, void *out, int dtype, void *stream);

/* dw [out_features, in_features] = sum_r dy[r, :]^T kept[r, :], db [out_features] = sum_r dy[r, :] (NULL: not wanted), kept =
 * the checkpoint of an activation [rows, in_features].  The products run on the bf16 matrix cores with fp32 sums: kept is exact
 * in bf16, dy is taken as one (bf16), two (fp16) or three (fp32) bf16 pieces that add up to it.  out_dtype: type of dw and db.
 * workspace: sn_checkpoint8_weight_grad_workspace bytes (0 for bad arguments). */
size_t sn_checkpoint8_weight_grad_workspace(int64_t rows, int out_features, int in_features, int dy_dtype);
int sn_checkpoint8_weight_grad(const void *dy, int dy_dtype, int64_t dy_row_stride, const void *codes, const void *exps, int64_t rows,
                               int out_features, int in_features, void *dw, void *db, int out_dtype, void *workspace,
                               size_t workspace_bytes, void *stream);

/* ------------------------------------------------------------------------------------------
 * the end of a residual block and the norm before the next one
 *     p = N_post(branch) (or branch);  y = x + scale * sigmoid(gate) * p;  h = N_pre(y)
 * N = LayerNorm over the features (rms = 0) or division by the root mean square (rms = 1), times a weight, plus a bias (NULL: none).
 * ------------------------------------------------------------------------------------------ */
#define SN_BLOCK_NORMS_MAX_WIDTH 4096
typedef struct sn_block_norms_args {
    uint32_t struct_size;                 /* sizeof(sn_block_norms_args) */
    int32_t dtype;                        /* x, branch, gate, y, h and the gradients of x, branch, gate, y, h */
    int32_t param_dtype;                  /* scale, the norms' weights and biases and their gradients */
    int32_t rms;
    int64_t rows;
    int32_t width;                        /* 1 .. SN_BLOCK_NORMS_MAX_WIDTH */
    int32_t rows_per_graph;               /* with n_valid: row r belongs to graph r / rows_per_graph */
    const int32_t *n_valid;               /* rows of a graph from n_valid[g] on are not read; they get zeros (NULL: every row counts) */
    float eps;
    int32_t has_post, has_pre;
    const void *x, *branch, *gate;        /* [rows, width]; gate may be NULL */
    int64_t x_stride, branch_stride, gate_stride;
    const void *scale;                    /* [width] or NULL */
    const void *post_weight, *post_bias, *pre_weight, *pre_bias;   /* [width]; weights needed with has_*, biases may be NULL */
    void *y, *h;                          /* forward results [rows, width] contiguous; h with has_pre */
    float *stats;                         /* [rows, 4]: mean and 1 / deviation of both norms; forward writes (NULL: not wanted), backward reads */
    void *x_codes, *x_exps, *branch_codes, *branch_exps, *gate_codes, *gate_exps;
                                          /* 8-bit checkpoints of the three inputs: forward writes them (x_codes NULL: not wanted); backward
                                           * reads them in place of x, branch and gate when x_codes is not NULL */
    const void *dy, *dh;                  /* backward inputs [rows, width]; either may be NULL (= zeros) */
    int64_t dy_stride, dh_stride;
    void *dx, *dbranch, *dgate;           /* [rows, width] contiguous; NULL: not wanted */
    void *dscale, *dpost_weight, *dpost_bias, *dpre_weight, *dpre_bias;      /* [width]; NULL: not wanted */
    void *workspace;                      /* backward: sn_block_norms_workspace(rows, width) bytes */
    size_t workspace_bytes;
} sn_block_norms_args;

int sn_block_norms_forward(const sn_block_norms_args *args, void *stream);
size_t sn_block_norms_workspace(int64_t rows, int width);
int sn_block_norms_backward(const sn_block_norms_args *args, void *stream);

/* ------------------------------------------------------------------------------------------
 * log probabilities of given tokens, with entropy and top alternatives
 * logits [rows, n]; target [rows] int64.  p = softmax(logits).
 *   log_probs[r] = log p[target], 0 where target == ignore_index, NaN where the target is outside 0 .. n - 1;
 *   entropy[r] = -sum p log p;   top_ids / top_log_probs [rows, k]: the k largest, the lowest index first among equals
 *   stats [rows, 3]: max, sum of exp(x - max), entropy - what the backward pass reads (NULL: not wanted).
 *   workspace: sn_label_log_probs_workspace bytes (0: none needed, NULL will do).
 * A row whose every logit is -inf has no distribution: log_probs -inf, entropy 0, gradient 0.  A NaN or +inf logit makes the
 * row's outputs NaN (the ids are then those of the largest finite or +inf logits, -1 where there are
 * fewer than k).
 * ------------------------------------------------------------------------------------------ */
#define SN_SCORES_MAX_TOP 64
size_t sn_label_log_probs_workspace(int64_t rows, int64_t n, int k);
int sn_label_log_probs(const void *logits, int dtype, int64_t rows, int64_t n, int64_t row_stride, const int64_t *target, int64_t ignore_index,
                       int k, float *log_probs, float *entropy, float *stats, float *top_log_probs, int64_t *top_ids, void *workspace,
                       size_t workspace_bytes, void *stream);
/* grad [rows, n] contiguous, in the logits' type: g_log_probs[r] (delta(target) - p) - g_entropy[r] p (log p + entropy);
 * either upstream gradient may be NULL.  A row whose upstream gradients are zeros (g_log_probs of an ignored target counts as zero) is
 * not read and gets zeros, unless its target lies outside. */
int sn_label_log_probs_backward(const void *logits, int dtype, int64_t rows, int64_t n, int64_t row_stride, const int64_t *target,
                                int64_t ignore_index, const float *stats, const float *g_log_probs, const float *g_entropy, void *grad,
                                void *stream);

#ifdef __cplusplus
}
#endif
#endif /* SCHEMANET_BLOCKS_H */
