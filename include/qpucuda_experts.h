/*
 * Tokens sorted by expert and back: the routing around a layer of experts
 * (qpucuda_fp8_gemm with experts), with its gradients. Device pointers,
 * asynchronous on the context stream, no allocation, deterministic (no
 * floating-point atomics). No counterpart in the reference.
 *
 * Every token t makes `choices` choices; choice (t, j) has the flat index
 * t * choices + j. Rows are ordered by expert, then by flat index; an expert id
 * outside [0, experts) drops the choice.
 * Outputs share no bytes with what a call reads.
 *
 *   offsets[e], offsets[e + 1]   the rows of expert e
 *   source[row]                  the flat index at that row, -1 from offsets[experts] on
 *   position[t, j]               the row of that choice, -1 when dropped
 */
#ifndef QPUCUDA_EXPERTS_H
#define QPUCUDA_EXPERTS_H

#include "qpucuda_fp8.h"

#ifdef __cplusplus
extern "C" {
#endif
#if defined(__GNUC__)
#pragma GCC visibility push(default)
#endif

/* Scratch bytes of qpucuda_expert_sort (0 is possible). */
size_t qpucuda_expert_sort_workspace(uint32_t tokens, uint32_t choices, uint32_t experts);

/* ids: [tokens][choices] int32, or int64 when ids_64 is nonzero. experts <= QPUCUDA_MAX_EXPERTS,
 * tokens * choices < 2^31. workspace: 4-byte aligned, used by this call alone until it has run. */
qpucuda_status qpucuda_expert_sort(
    qpucuda_context *context,
    const void *ids, int ids_64,
    uint32_t tokens, uint32_t choices, uint32_t experts,
    int32_t *offsets, int32_t *source, int32_t *position,
    void *workspace, size_t workspace_bytes);

/* rows[position[t, j]] = x[t]; rows from offsets[experts] on (read from `offsets`) become zero.
 * x [tokens][width], rows [tokens * choices][width], both of `type` (qpucuda_dtype). */
qpucuda_status qpucuda_expert_gather(
    qpucuda_context *context,
    const void *x, int type, size_t x_stride,
    uint32_t tokens, uint32_t choices, uint32_t width,
    const int32_t *position, const int32_t *offsets, uint32_t experts,
    void *rows, size_t rows_stride);

/* out[t] = sum_j weight[t, j] * rows[position[t, j]] in fp32, in the order of j, rounded once.
 * weights NULL: all one, which is the gradient of qpucuda_expert_gather. */
qpucuda_status qpucuda_expert_combine(
    qpucuda_context *context,
    const void *rows, int type, size_t rows_stride,
    uint32_t tokens, uint32_t choices, uint32_t width,
    const int32_t *position, const float *weights,
    void *out, size_t out_stride);

/* The gradients of qpucuda_expert_combine: grad_rows[position[t, j]] = weight[t, j] * grad[t],
 * zero from offsets[experts] on; grad_weights[t, j] = <rows[position[t, j]], grad[t]> in fp32,
 * zero when dropped. */
qpucuda_status qpucuda_expert_combine_backward(
    qpucuda_context *context,
    const void *rows, int type, size_t rows_stride,
    const void *grad, size_t grad_stride,
    uint32_t tokens, uint32_t choices, uint32_t width,
    const int32_t *position, const int32_t *offsets, uint32_t experts,
    const float *weights,
    void *grad_rows, size_t grad_rows_stride,
    float *grad_weights);

#if defined(__GNUC__)
#pragma GCC visibility pop
#endif
#ifdef __cplusplus
}
#endif

#endif
