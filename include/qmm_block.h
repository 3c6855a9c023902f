/*
 * qmm_block.h -- C ABI of the operators around the quantized linear of a DiT
 * block on B200 (sm_100a): MXFP4 quantisation and product, q/k norm with
 * multi-axis rotary positions, and the norms before and after a block fused
 * with its gate and residual.
 *
 * Same library and conventions as qmm.h: plain device pointers, int64_t
 * counts, an opaque stream, nothing allocated, asynchronous launches, a
 * qmm_status returned and the message of the last failure in
 * qmm_last_error().  Forward only: the library serves inference.
 */
#ifndef QMM_BLOCK_H
#define QMM_BLOCK_H

#include "qmm.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element type of an operand.  The first two are qmm_dtype's values. */
typedef enum qmm_elem {
    QMM_ELEM_BF16 = 0,
    QMM_ELEM_F32 = 1,
    QMM_ELEM_F16 = 2
} qmm_elem;

/* ------------------------------------------------------------------ MXFP4 */

/*
 * An MXFP4 matrix [rows, k]: E2M1 codes (sign, 2 exponent bits, 1 mantissa
 * bit: 0, .5, 1, 1.5, 2, 3, 4, 6) and one E8M0 scale 2^(e - 127) for each 32
 * consecutive columns (e = 255: NaN).
 *   codes  : uint8 [rows, 16 * ceil(k / 32)], row-major; column 2 j in the low
 *            four bits of byte j, column 2 j + 1 in the high four; columns
 *            past k are code 0.  16-byte aligned.
 *   scales : qmm_mx4_scale_bytes(rows, k) bytes, 16-byte aligned, in the order
 *            in which the tensor cores take them: tiles of 128 rows x 4
 *            blocks (512 bytes), tile (R, B) at (R * T + B) * 512 with T =
 *            2 * ceil(k / 256); row r and block b of the tile at byte
 *            16 * (r % 32) + 4 * (r / 32) + b.  Blocks past ceil(k / 32) are 0;
 *            rows past `rows` may hold anything.
 */
typedef struct qmm_mx4 {
    const uint8_t *codes;
    const uint8_t *scales;
    int64_t rows;
    int64_t k;
} qmm_mx4;

/* Bytes of an MXFP4 matrix's codes and scales (0 for rows or k <= 0).  Host-only. */
QMM_API uint64_t qmm_mx4_code_bytes(int64_t rows, int64_t k);
QMM_API uint64_t qmm_mx4_scale_bytes(int64_t rows, int64_t k);

/*
 * x [rows, k] (row r at x + r * row_stride elements; elem: qmm_elem) to MXFP4.
 * Per block of 32 columns (the last one may be short): e = floor(log2(max|x|))
 * - 2 + 127, at least 0, and 0 for a block of zeros; codes are x / 2^(e - 127)
 * rounded to the nearest (ties to the even code), 6 where that is past 6.  A
 * block with an infinity or NaN gets scale 255 and codes 0: it stands for NaN.
 */
QMM_API qmm_status qmm_mx4_quantize(const void *x, int32_t elem, int64_t rows, int64_t k, int64_t row_stride,
                                    uint8_t *codes, uint8_t *scales, void *stream);

/* dst [rows, k] (row-major, contiguous; bf16, f32 or f16) = the values of `w`.
 * bf16 and f32 hold every value below 2^128 exactly (scales 253 and 254 reach
 * past it: infinity); f16 rounds (past 65504: infinity). */
QMM_API qmm_status qmm_mx4_dequantize(const qmm_mx4 *w, void *dst, int32_t elem, void *stream);

/* Scales between row-major order (uint8 [rows, ceil(k / 32)], as checkpoints
 * store them) and the order of qmm_mx4. */
QMM_API qmm_status qmm_mx4_tile_scales(const uint8_t *row_major, int64_t rows, int64_t k, uint8_t *scales,
                                       void *stream);
QMM_API qmm_status qmm_mx4_row_scales(const uint8_t *scales, int64_t rows, int64_t k, uint8_t *row_major,
                                      void *stream);

/*
 * y [m, n] (bf16, row-major) = residual + gate * act(x . W^T + bias), or
 * residual * (gate * act(...)) with QMM_EPILOGUE_RESIDUAL_MUL, one rounding to
 * bf16; W [n, k] MXFP4.  x is either MXFP4 (x_codes and x_scales; x NULL) or a
 * matrix of bf16, f32 or f16 (x, x_elem, x_row_stride), which is first
 * quantised by the rule of qmm_mx4_quantize, within the product where m is
 * small, else into `workspace` (16-byte aligned,
 * qmm_mx4_linear_workspace_bytes(m, n, k) bytes: 0 in the former case, never
 * more than qmm_mx4_workspace_bytes(m, k)).  Products of codes
 * and scales are exact, sums are f32.  bias, gate bf16 [n] or NULL; residual
 * bf16 [m, n] or NULL, it may alias y.  y must not overlap x, W or workspace.
 * Calls that share a workspace must be ordered on one stream.  Every operand,
 * W among them, is read only after the kernels ahead on the stream have
 * completed, whatever qmm_set_weights_immutable says: W may come straight out
 * of qmm_mx4_quantize.
 */
typedef struct qmm_mx4_linear_args {
    qmm_mx4 w;
    int64_t m;
    const void *x;
    int64_t x_row_stride;
    const uint8_t *x_codes;
    const uint8_t *x_scales;
    const uint16_t *bias;
    const uint16_t *gate;
    const uint16_t *residual;
    uint16_t *y;
    void *workspace;
    uint64_t workspace_bytes;
    int32_t x_elem;
    int32_t activation;
} qmm_mx4_linear_args;

QMM_API uint64_t qmm_mx4_workspace_bytes(int64_t m, int64_t k);
QMM_API uint64_t qmm_mx4_linear_workspace_bytes(int64_t m, int64_t n, int64_t k);
QMM_API qmm_status qmm_mx4_linear(const qmm_mx4_linear_args *a, void *stream);

/* ----------------------------------------------------------------- rotary */

/*
 * RMSNorm per head of q and k and rotary positions with several axes:
 *   v   = x * rsqrt(mean(x^2) + eps) * weight          (weight NULL: v = x)
 *   phi = 2 pi * positions[token, axis_p] * turns_p    for pair p of a head
 *   (a, b) of pair p -> (a cos phi - b sin phi, a sin phi + b cos phi)
 * with (a, b) columns (2 p, 2 p + 1) of the head (adjacent) or (p, pairs + p)
 * (halves); columns from 2 * pairs on are only normalised.  f32 arithmetic,
 * one rounding.  Whole turns are dropped before the sine and cosine: the angle
 * is right to about 2^-23 turns at positions up to 2^24, whole or not, and to
 * 2^-52 of the position in turns beyond (whole positions up to 2^48; turns up
 * to 1 / (2 pi); 2^-21 turns at 2^31).
 *
 * q [batch, tokens, q_heads, dim] and k [batch, tokens, k_heads, dim] lie at
 * the given element strides (batch, token, head; columns are contiguous), as
 * do the outputs; an output may be its input (same address and strides) but
 * must not overlap it otherwise.  k NULL: q alone.  `turns` f32 [pairs, 2]:
 * each frequency (turns a position) as a leading and a trailing term; axis
 * uint8 [pairs], each below `axes`; positions [batch or 1, tokens, axes]
 * int32, int64 or f32 (pos_kind 0, 1, 2), contiguous but for pos_batch_stride
 * (0: shared).  dim up to 256; q_weight and k_weight [dim] in q's type.
 */
typedef struct qmm_rotary_args {
    const void *q;
    const void *k;
    void *q_out;
    void *k_out;
    const void *q_weight;
    const void *k_weight;
    const void *positions;
    const float *turns;
    const uint8_t *axis;
    int64_t batch;
    int64_t tokens;
    int64_t q_stride[3];
    int64_t k_stride[3];
    int64_t q_out_stride[3];
    int64_t k_out_stride[3];
    int64_t pos_batch_stride;
    int32_t q_heads;
    int32_t k_heads;
    int32_t dim;
    int32_t pairs;
    int32_t axes;
    int32_t adjacent;
    int32_t pos_kind;
    int32_t elem;
    float eps;
} qmm_rotary_args;

QMM_API qmm_status qmm_qk_norm_rotary(const qmm_rotary_args *a, void *stream);

/* ------------------------------------------------------------------ norms */

typedef enum qmm_norm {
    QMM_NORM_NONE = 0,
    QMM_NORM_RMS = 1,   /* t * rsqrt(mean(t^2) + eps) */
    QMM_NORM_LAYER = 2  /* (t - mean) * rsqrt(var + eps) */
} qmm_norm;

/*
 * The seam between two sublayers, one pass per row:
 *   h  = norm_post(branch) * post_weight
 *   x' = residual_scale * x + gate * h                   -> x_out
 *   n  = norm_pre(x') * pre_weight * (1 + scale) + shift -> n_out, or MXFP4
 * in f32 (statistics included; n is formed from the unrounded x'), one
 * rounding per output.  x, x_out and n_out hold x_elem, branch holds
 * branch_elem; each has its own row stride in elements.  branch NULL:
 * x' = residual_scale * x.  x_out NULL: x' is not stored.  Vectors hold
 * vec_elem: post_weight, pre_weight [hidden]; gate, shift, scale [groups,
 * hidden] (row r uses group r / (rows / groups); vec_stride elements between
 * groups); each may be NULL.  n leaves as n_out, as MXFP4 (n_codes and
 * n_scales, the layout of qmm_mx4 [rows, hidden]), or not at all (all NULL).
 * x_out may be x or branch (same address and stride), n_out may be branch or x
 * likewise; otherwise outputs must not overlap inputs.  hidden up to 32768.
 */
typedef struct qmm_gated_norm_args {
    const void *x;
    const void *branch;
    void *x_out;
    void *n_out;
    uint8_t *n_codes;
    uint8_t *n_scales;
    const void *post_weight;
    const void *pre_weight;
    const void *gate;
    const void *shift;
    const void *scale;
    int64_t rows;
    int64_t hidden;
    int64_t x_stride;
    int64_t branch_stride;
    int64_t x_out_stride;
    int64_t n_out_stride;
    int64_t gate_stride;
    int64_t shift_stride;
    int64_t scale_stride;
    int64_t groups;
    int32_t x_elem;
    int32_t branch_elem;
    int32_t vec_elem;
    int32_t post;
    int32_t pre;
    float residual_scale;
    float eps;
} qmm_gated_norm_args;

QMM_API qmm_status qmm_gated_residual_norm(const qmm_gated_norm_args *a, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* QMM_BLOCK_H */
