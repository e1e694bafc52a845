/*
 * tinydeform_dense.h -- C ABI of the dense operators beside deformable attention (libtinydeform.so): attention among
 * tokens, forward and backward, and layer norm with a residual, forward and backward.
 *
 * The conventions of tinydeform.h hold: plain device pointers, int64 sizes, a hipStream_t passed as void*; the library
 * never allocates, frees or synchronises, callers own every buffer (workspaces included), each call may be captured in
 * a HIP graph; TD_OK or a negative TD_E* code is returned, with td_last_error() describing the failure. dtype is TD_F32,
 * TD_F16, TD_BF16 or TD_F64; outputs do not overlap inputs; sums, softmax statistics and norms are float32 (float64 for
 * TD_F64).
 * No counterpart in the reference, whose operator is deformable attention alone.
 */
#ifndef TINYDEFORM_DENSE_H
#define TINYDEFORM_DENSE_H

#include <stdint.h>

#include "tinydeform.h"

#ifdef __cplusplus
extern "C" {
#endif

#define TD_ATTN_MAX_HEAD_DIM 256
#define TD_NORM_MAX_CHANNELS 16384

#define TD_MASK_NONE 0
#define TD_MASK_BYTES 1 /* non-zero: the query may not attend to the key */
#define TD_MASK_FLOAT 2 /* in dtype, added to the scaled scores; -inf: the query may not attend to the key */

/*
 * Attention among tokens: with G = H / Hk heads sharing each key head,
 *   t[b,h,i,j]  = scale * query[b,i,h] . key[b,j,h / G] (+ mask[b,h,i,j])
 *   out[b,i,h]  = sum_j softmax_j(t[b,h,i,:])[j] value[b,j,h / G]
 * over the keys j that padding, mask and causal leave. A row that they leave nothing gives 0 (and gradients of 0). A key
 * that key_padding excludes is not read into any result, whatever it holds; the keys and values of the others are
 * expected to be finite. causal: query i sees the keys j <= i + K - Q (the last query sees every key).
 */
typedef struct td_attn_args {
    int32_t dtype;
    int32_t mask_type; /* TD_MASK_* */
    int32_t causal;
    int32_t reserved; /* 0 */
    /* Hk divides H; D <= TD_ATTN_MAX_HEAD_DIM; Q, K, B * Q * H, B * K * Hk <= INT32_MAX - 1023 */
    int64_t B, Q, K, H, Hk, D;
    double scale;              /* finite, > 0 */
    const void* query;         /* [B, Q, H, D], element strides below (batch, token, head; not negative), the last one 1 */
    const void* key;           /* [B, K, Hk, D] */
    const void* value;         /* [B, K, Hk, D] */
    int64_t query_stride[3], key_stride[3], value_stride[3];
    const void* mask;          /* [B, H, Q, K]: element strides (batch, head, query), 0 where shared, the last one 1 */
    int64_t mask_stride[3];
    const uint8_t* key_padding; /* [B, K] contiguous, non-zero: no query attends to the key; or NULL */
    void* out;                  /* [B, Q, H * D] contiguous */
    void* stats;                /* [B, H, Q, 2] float32 (float64): the backward's softmax statistics; or NULL */
    void* out_low;              /* TD_F16, TD_BF16: like out, what rounding took from it, in dtype: the backward's
                                   grad_out . out then has twice the bits. Or NULL */
} td_attn_args;

/* Bytes of workspace td_attn_forward needs (0 for many problems; a mask takes an eighth of a byte an entry), or a negative
 * TD_E* code. No memory is read. */
int64_t td_attn_forward_workspace(const td_attn_args* args);
int td_attn_forward(const td_attn_args* args, void* workspace, int64_t workspace_bytes, void* stream);

/*
 * Gradients of td_attn_forward, the probabilities computed again from the scores and `stats`. args: as in the forward
 * call, with the out, stats and out_low (or NULL) that it wrote. grad_out [B, Q, H * D], grad_query [B, Q, H, D],
 * grad_key and grad_value [B, K, Hk, D] are contiguous, in dtype; grad_query, or grad_key and grad_value together, may be
 * NULL (not computed).
 * No atomics: the results are the same on every run.
 */
int64_t td_attn_backward_workspace(const td_attn_args* args);
int td_attn_backward(const td_attn_args* args, const void* grad_out, void* grad_query, void* grad_key,
                     void* grad_value, void* workspace, int64_t workspace_bytes, void* stream);

/*
 * Layer norm over the last dimension of x (+ residual), rows [rows, C] contiguous:
 *   h = x + residual;  out = (h - mean(h)) * rstd(h) * weight + bias,  rstd = 1 / sqrt(var(h) + eps)
 * residual, weight and bias may be NULL. h is not rounded to dtype. stats [rows, 2] float32 (float64), or NULL, receives
 * mean and rstd for the backward. C <= TD_NORM_MAX_CHANNELS.
 */
int td_layer_norm_forward(int dtype, const void* x, const void* residual, const void* weight, const void* bias,
                          void* out, void* stats, int64_t rows, int64_t C, double eps, void* stream);

/*
 * Its gradients: grad_x [rows, C] (also the residual's), grad_weight and grad_bias [C] (NULL: not computed). The column
 * sums over the rows are taken in float32 (float64) in a fixed order, by way of the workspace.
 */
int64_t td_layer_norm_backward_workspace(int dtype, int64_t rows, int64_t C);
int td_layer_norm_backward(int dtype, const void* x, const void* residual, const void* weight, const void* stats,
                           const void* grad_out, void* grad_x, void* grad_weight, void* grad_bias, int64_t rows,
                           int64_t C, void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* TINYDEFORM_DENSE_H */
