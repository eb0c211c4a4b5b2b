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

typedef struct qpucuda_expert_sort_desc {
    const void *ids;         /* [tokens][choices] int32, or int64 when ids_64 is nonzero */
    int ids_64;
    uint32_t tokens, choices, experts; /* experts <= QPUCUDA_MAX_EXPERTS, tokens * choices < 2^31 */
    int32_t *offsets, *source, *position;
    void *workspace;         /* 4-byte aligned, used by this call alone until it has run */
    size_t workspace_bytes;
} qpucuda_expert_sort_desc;

qpucuda_status qpucuda_expert_sort(qpucuda_context *context, const qpucuda_expert_sort_desc *desc);

/* One move of rows between the tokens' order, [tokens][width], and the experts', [tokens *
 * choices][width]; strides in elements. */
typedef struct qpucuda_expert_rows_desc {
    int type;                /* qpucuda_dtype of source, grad and out */
    uint32_t tokens, choices, width, experts;
    const int32_t *position, *offsets; /* of the sort; combine reads no offsets */
    const float *weights;    /* [tokens][choices]; gather has none */
    const void *source;
    size_t source_stride;
    const void *grad;        /* combine_backward: the gradient of the tokens, and where the weights' goes */
    size_t grad_stride;
    float *grad_weights;
    void *out;
    size_t out_stride;
} qpucuda_expert_rows_desc;

/* Tokens to the experts' order: out[position[t, j]] = source[t]; rows from offsets[experts] on become
 * zero. */
qpucuda_status qpucuda_expert_gather(qpucuda_context *context, const qpucuda_expert_rows_desc *desc);

/* And back: out[t] = sum_j weight[t, j] * source[position[t, j]] in fp32, in the order of j, rounded
 * once. weights NULL: all one, which is the gradient of qpucuda_expert_gather. */
qpucuda_status qpucuda_expert_combine(qpucuda_context *context, const qpucuda_expert_rows_desc *desc);

/* The gradients of qpucuda_expert_combine, whose source is given again: out[position[t, j]] =
 * weight[t, j] * grad[t], zero from offsets[experts] on; grad_weights[t, j] = <source[position[t, j]],
 * grad[t]> in fp32, zero when dropped. */
qpucuda_status qpucuda_expert_combine_backward(qpucuda_context *context, const qpucuda_expert_rows_desc *desc);

#if defined(__GNUC__)
#pragma GCC visibility pop
#endif
#ifdef __cplusplus
}
#endif

#endif
