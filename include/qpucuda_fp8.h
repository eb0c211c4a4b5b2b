/*
 * Block-scaled FP8 (e4m3) linear: row quantizer, weight quantizer and matrix
 * product, device pointers, asynchronous on the context stream. No counterpart
 * in the reference, whose quantized linear is int8 with one scale per row; this
 * is the same linear for weights published as e4m3 with one fp32 scale per
 * 128 x 128 block.
 *
 *   scale of a group   s = max(RN(max|x| / 448), 2^-60)
 *   value              q = e4m3(RN(x / s)), round to nearest even, at most 448
 *   product            y[m, n] = sum_k (qx[m, k] sx[m, k / 128]) (qw[n, k] sw[n / 128, k / 128]) + bias[n]
 *
 * A group of rows with a NaN or an infinity dequantizes to NaN, and so do the
 * outputs of that row; no other row is affected. Every call allocates nothing
 * and may be captured into a CUDA graph.
 * The product's waits inside a kernel are bounded. One that runs out leaves
 * outputs unwritten or incomplete and ends without a CUDA error; the next
 * qpucuda_context_synchronize returns QPUCUDA_TIMEOUT.
 */
#ifndef QPUCUDA_FP8_H
#define QPUCUDA_FP8_H

#include "qpucuda_runtime.h"

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif
#if defined(__GNUC__)
#pragma GCC visibility push(default)
#endif

/* Columns (and weight rows) that share one scale. */
#define QPUCUDA_FP8_GROUP 128u

/* Element types of activations and outputs. */
typedef enum qpucuda_dtype {
    QPUCUDA_DTYPE_F32 = 0,
    QPUCUDA_DTYPE_BF16 = 1,
    QPUCUDA_DTYPE_F16 = 2
} qpucuda_dtype;

typedef struct qpucuda_fp8_quantize_desc {
    const void *x;           /* [source rows][cols], or [..][2 * cols] = gate | up when gated */
    int x_type;              /* qpucuda_dtype */
    size_t x_stride;         /* elements */
    uint32_t rows;           /* quantized rows */
    uint32_t cols;
    int gated;               /* nonzero: quantize silu(gate) * up, computed in fp32 */
    /* Row r is made from source row row_source[r] / row_divisor; a negative entry gives a zero
     * row, as does one past source_rows. NULL: row r from source row r. */
    const int32_t *row_source;
    uint32_t row_divisor;
    uint32_t source_rows;
    uint8_t *q;              /* [rows] rows of q_stride bytes, 16-byte aligned */
    /* A multiple of 16, at least cols. The bytes past cols that a 16-byte vector of x reaches (up to 7,
     * up to 3 of fp32) are written as the quantized zeros they stand for: zero, or NaN (0x7F) in a group
     * whose scale is NaN. The others are left as they are. */
    size_t q_stride;
    float *scales;           /* group g of row r at r * scale_row_stride + g * scale_group_stride */
    size_t scale_row_stride;
    size_t scale_group_stride;
} qpucuda_fp8_quantize_desc;

/* Rows to e4m3 with one scale per 128 columns (the last group may be shorter). */
qpucuda_status qpucuda_fp8_quantize_rows(qpucuda_context *context, const qpucuda_fp8_quantize_desc *desc);

/* Matrices [batch][rows][cols] (row stride x_stride, matrices rows * x_stride apart) to e4m3
 * values [batch][rows] of q_stride bytes and scales [batch][ceil(rows/128)][ceil(cols/128)]. */
qpucuda_status qpucuda_fp8_quantize_blocks(
    qpucuda_context *context,
    const void *x, int x_type, size_t x_stride,
    uint32_t batch, uint32_t rows, uint32_t cols,
    uint8_t *q, size_t q_stride,
    float *scales);

typedef struct qpucuda_fp8_gemm_desc {
    const uint8_t *a;        /* e4m3 [rows] of a_stride bytes; bytes past k do not count */
    size_t a_stride;         /* a multiple of 16, base 16-byte aligned (as w) */
    const float *a_scales;   /* strided as in qpucuda_fp8_quantize_desc */
    size_t a_scale_row_stride;
    size_t a_scale_group_stride;
    const uint8_t *w;        /* e4m3 [max(experts, 1)][n] of w_stride bytes */
    size_t w_stride;
    const float *w_scales;   /* [max(experts, 1)][ceil(n/128)][ceil(k/128)] */
    const float *bias;       /* [n] or NULL; NULL with experts */
    uint32_t rows, n, k;
    /* 0: one matrix. Otherwise rows [offsets[e], offsets[e + 1]) meet matrix e (offsets: device
     * int32 [experts + 1], ascending from 0 to at most rows; clamped to that), and rows from
     * offsets[experts] on become zero. At most QPUCUDA_MAX_EXPERTS. */
    uint32_t experts;
    const int32_t *offsets;
    void *out;               /* [rows][n]; shares no bytes with what the call reads */
    int out_type;            /* qpucuda_dtype */
    size_t out_stride;       /* elements */
    /* Nonzero: w, w_scales and offsets were complete before the kernel queued just before this one
     * started, so they may be read while that kernel is still running. */
    int weights_settled;
} qpucuda_fp8_gemm_desc;

#define QPUCUDA_MAX_EXPERTS 1024u

qpucuda_status qpucuda_fp8_gemm(qpucuda_context *context, const qpucuda_fp8_gemm_desc *desc);

/* The product of rows that are quantized in the same call: gemm->a, a_stride, a_scales, rows and k
 * must be quantize's, whose q and scales serve as scratch and hold nothing certain afterwards (a few
 * rows of a small matrix never leave the kernel). With weights_settled the weight must also not be
 * written by the work queued just before this call; offsets may be. */
qpucuda_status qpucuda_fp8_linear(qpucuda_context *context, const qpucuda_fp8_quantize_desc *quantize,
                                  const qpucuda_fp8_gemm_desc *gemm);

#if defined(__GNUC__)
#pragma GCC visibility pop
#endif
#ifdef __cplusplus
}
#endif

#endif
