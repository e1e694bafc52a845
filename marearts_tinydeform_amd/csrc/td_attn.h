// Attention among tokens: what the forward and backward kernels share (td_attn.hip, td_attn_forward.hip,
// td_attn_backward.hip).
#pragma once

#include "../../include/tinydeform_dense.h"
#include "td_internal.h"

namespace td {

// Heads that share a key head are rows of one problem: row r of (batch b, key head hk) is query r / G of head
// hk * G + r % G, so that a tile of rows reads each key once and the key gradients of shared heads are one sum.
struct AttnParams {
    const void *q, *k, *v, *mask;
    const uint8_t* pad;
    void *out;
    void *stats;  // [B, H, Q, 2]: the maximum of each row's scores and log2 of the sum of 2^(score - maximum), in base 2
    int64_t qs[3], ks[3], vs[3], ms[3];  // batch, token (query), head strides in elements
    int B, Q, K, H, Hk, D, G;
    int rows;       // Q * G
    FastDiv gdiv;   // r / G
    int mask_type;  // TD_MASK_*
    int causal;
    int64_t diag;   // K - Q: with causal, query i sees the keys j <= i + diag
    double scale;
    float c;        // scale * log2(e): scores in base 2
    void* out_low;  // 16-bit types: out's rounding errors, or null
    // a mask as bits (attn_mask_kernel): row b * bs[0] + h * bs[1] + i * bs[2] has words of 32 keys, set for pairs left
    // out; kinds[(that row's 32-row tile)][word]: MaskKind of the 32 x 32 pairs
    uint32_t* bits;
    uint8_t* kinds;
    int64_t bs[3], kinds_bs[2];  // rows; tiles (kinds_bs: batch, head), 0 where shared
    int words;                   // of a row
    // backward
    const void* go;
    void *dq, *dk, *dv;
    void* delta;    // float64: [B, H, Q], grad_out . out
    // workspace of the forward's key split, of the backward
    void* ws;
};

enum MaskKind { kMaskNone = 0, kMaskBits = 1, kMaskValues = 2, kMaskAll = 3 };

AttnParams attn_params(const td_attn_args& a);
// The mask as bits, at `at` (16-byte aligned); returns the bytes they take, a multiple of 16. With at null only that.
int64_t plan_mask(AttnParams& p, void* at);
int launch_mask(int dtype, const AttnParams& p, hipStream_t stream);

// On the matrix units, for float32, float16 and bfloat16 (td_attn_forward.hip)
int64_t attn_forward_workspace(int dtype, const AttnParams& p);
int launch_attn_forward(int dtype, const AttnParams& p, hipStream_t stream);
template <typename T>
int launch_attn_forward_t(int dtype, const AttnParams& p, hipStream_t stream);
// ... and the gradients (td_attn_backward.hip)
int64_t attn_backward_workspace(int dtype, const AttnParams& p);
int launch_attn_backward(int dtype, const AttnParams& p, hipStream_t stream);
template <typename T>
int launch_attn_backward_t(int dtype, const AttnParams& p, hipStream_t stream);
// Head widths the matrix-unit kernels are built for (80 in 96, 2 x 8 x 4096, bfloat16: forward 168 us in 128, 138 in 96, dQ 219
// and 170, dK and dV 343 and 240)
inline int padded_width(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : D <= 128 ? 128 : 256; }

// float64 (td_attn.hip). Every launcher returns 0 or a negative TD_E* code after recording a message.
int launch_attn_forward_f64(const AttnParams& p, hipStream_t stream);
int launch_attn_backward_f64(const AttnParams& p, hipStream_t stream);

}  // namespace td
