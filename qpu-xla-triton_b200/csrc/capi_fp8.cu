// C entry points of the block-scaled FP8 linear (include/qpucuda_fp8.h) and of the expert routing
// (include/qpucuda_experts.h): argument checks, the context's submission rules, then the launches
// on the context stream. Nothing here allocates.
#include <climits>

#include "qpucuda_fp8_internal.h"
#include "qpucuda_internal.h"

using namespace qpucuda;

namespace {

bool aligned(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
bool known_type(int type) { return type == QPUCUDA_DTYPE_F32 || type == QPUCUDA_DTYPE_BF16 || type == QPUCUDA_DTYPE_F16; }
size_t type_bytes(int type) { return type == QPUCUDA_DTYPE_F32 ? 4 : 2; }

qpucuda_status launched(qpucuda_context *context, cudaError_t error, const char *what) {
    if (error == cudaErrorInvalidValue) return cuda_fail(context, error, what, QPUCUDA_INVALID_ARGUMENT);
    if (error != cudaSuccess) return cuda_fail(context, error, what, QPUCUDA_SUBMISSION_FAILED);
    return QPUCUDA_OK;
}

template <typename Launch>
qpucuda_status submit(qpucuda_context *context, const char *what, Launch &&launch) {
    std::lock_guard<std::mutex> lock(context->mutex);
    const qpucuda_status status = begin_submit(context);
    if (status != QPUCUDA_OK) return status;
    DeviceGuard guard(context->device);
    return launched(context, launch(), what);
}

// tokens * choices rows, indexed by int32.
bool routing_fits(uint32_t tokens, uint32_t choices, uint32_t experts) {
    return choices != 0 && experts != 0 && experts <= QPUCUDA_MAX_EXPERTS &&
           static_cast<uint64_t>(tokens) * choices <= static_cast<uint64_t>(INT32_MAX);
}

bool present(const void *p) { return p != nullptr && aligned(p, 4); }

// What every move of rows reads and writes.
bool rows_fit(const qpucuda_expert_rows_desc &desc) {
    return known_type(desc.type) && desc.width != 0 && present(desc.position) && desc.source != nullptr && desc.out != nullptr &&
           desc.source_stride >= desc.width && desc.out_stride >= desc.width && aligned(desc.source, type_bytes(desc.type)) &&
           aligned(desc.out, type_bytes(desc.type));
}

// Argument checks: QPUCUDA_OK, or the refusal with its message. `rows` is not zero.
qpucuda_status check_quantize(qpucuda_context *context, const qpucuda_fp8_quantize_desc *desc) {
    const uint64_t width = static_cast<uint64_t>(desc->cols) * (desc->gated != 0 ? 2u : 1u);
    if (!known_type(desc->x_type) || desc->cols == 0 || desc->cols > INT32_MAX || desc->x == nullptr || desc->q == nullptr ||
        desc->scales == nullptr || desc->x_stride < width || desc->q_stride < desc->cols || desc->q_stride % 16 != 0 ||
        !aligned(desc->q, 16) || !aligned(desc->x, type_bytes(desc->x_type)) || !aligned(desc->scales, 4)) {
        return fail(context, QPUCUDA_INVALID_ARGUMENT,
                    "fp8_quantize_rows: needs fp32, bf16 or fp16 rows, and 16-byte aligned values with row strides "
                    "that are multiples of 16 and hold the columns");
    }
    if (desc->row_source != nullptr && (desc->row_divisor == 0 || !aligned(desc->row_source, 4))) {
        return fail(context, QPUCUDA_INVALID_ARGUMENT, "fp8_quantize_rows: row_divisor must be positive");
    }
    return QPUCUDA_OK;
}

qpucuda_status check_gemm(qpucuda_context *context, const qpucuda_fp8_gemm_desc *desc) {
    const uint64_t matrices = desc->experts != 0 ? desc->experts : 1u;
    if (!known_type(desc->out_type) || desc->n == 0 || desc->k == 0 || desc->k > INT32_MAX || desc->rows > INT32_MAX ||
        desc->n > INT32_MAX / 4 ||
        desc->a == nullptr || desc->a_scales == nullptr || desc->w == nullptr || desc->w_scales == nullptr ||
        desc->out == nullptr || desc->a_stride < desc->k || desc->w_stride < desc->k || desc->a_stride % 16 != 0 ||
        desc->w_stride % 16 != 0 || !aligned(desc->a, 16) || !aligned(desc->w, 16) || desc->out_stride < desc->n ||
        !aligned(desc->out, type_bytes(desc->out_type)) || !aligned(desc->a_scales, 4) || !aligned(desc->w_scales, 4) ||
        !aligned(desc->bias, 4) || !aligned(desc->offsets, 4)) {
        return fail(context, QPUCUDA_INVALID_ARGUMENT,
                    "fp8_gemm: operands need 16-byte aligned rows and in-range strides, the output fp32, bf16 or fp16");
    }
    if (desc->experts > QPUCUDA_MAX_EXPERTS || (desc->experts != 0 && (desc->offsets == nullptr || desc->bias != nullptr)) ||
        matrices * desc->n > static_cast<uint64_t>(INT32_MAX)) {
        return fail(context, QPUCUDA_INVALID_ARGUMENT,
                    "fp8_gemm: experts need offsets and no bias, at most %u of them and 2^31 weight rows in all",
                    QPUCUDA_MAX_EXPERTS);
    }
    if (!(context->cc_major == 10 && context->cc_minor == 0)) {
        return fail(context, QPUCUDA_CAPABILITY_MISSING, "fp8_gemm: the tcgen05 FP8 product needs an sm_100 device");
    }
    return QPUCUDA_OK;
}

}  // namespace

extern "C" {

qpucuda_status qpucuda_fp8_quantize_rows(qpucuda_context *context, const qpucuda_fp8_quantize_desc *desc) {
    if (context == nullptr || desc == nullptr) return QPUCUDA_INVALID_ARGUMENT;
    if (desc->rows == 0) return QPUCUDA_OK;
    const qpucuda_status checked = check_quantize(context, desc);
    if (checked != QPUCUDA_OK) return checked;
    return submit(context, "fp8_quantize_rows",
                  [&] { return launch_fp8_quantize_rows(*desc, context->sm_count, context->stream); });
}

qpucuda_status qpucuda_fp8_quantize_blocks(qpucuda_context *context, const void *x, int x_type, size_t x_stride,
                                           uint32_t batch, uint32_t rows, uint32_t cols, uint8_t *q, size_t q_stride,
                                           float *scales) {
    if (context == nullptr) return QPUCUDA_INVALID_ARGUMENT;
    if (batch == 0 || rows == 0) return QPUCUDA_OK;
    if (!known_type(x_type) || cols == 0 || cols > INT32_MAX || x == nullptr || q == nullptr || scales == nullptr ||
        x_stride < cols || q_stride < cols || !aligned(x, type_bytes(x_type)) || !aligned(scales, 4) || batch > 65535u ||
        rows > 65535u * QPUCUDA_FP8_GROUP) {
        return fail(context, QPUCUDA_INVALID_ARGUMENT, "fp8_quantize_blocks: invalid pointers, types or extents");
    }
    return submit(context, "fp8_quantize_blocks", [&] {
        return launch_fp8_quantize_blocks(x, x_type, x_stride, batch, rows, cols, q, q_stride, scales, context->stream);
    });
}

qpucuda_status qpucuda_fp8_gemm(qpucuda_context *context, const qpucuda_fp8_gemm_desc *desc) {
    if (context == nullptr || desc == nullptr) return QPUCUDA_INVALID_ARGUMENT;
    if (desc->rows == 0) return QPUCUDA_OK;
    const qpucuda_status checked = check_gemm(context, desc);
    if (checked != QPUCUDA_OK) return checked;
    return submit(context, "fp8_gemm",
                  [&] { return launch_fp8_gemm(*desc, context->d_error, context->sm_count, context->stream); });
}

qpucuda_status qpucuda_fp8_linear(qpucuda_context *context, const qpucuda_fp8_quantize_desc *quantize,
                                  const qpucuda_fp8_gemm_desc *gemm) {
    if (context == nullptr || quantize == nullptr || gemm == nullptr) return QPUCUDA_INVALID_ARGUMENT;
    if (quantize->rows == 0 && gemm->rows == 0) return QPUCUDA_OK;
    if (quantize->rows != gemm->rows || quantize->cols != gemm->k || quantize->q != gemm->a ||
        quantize->q_stride != gemm->a_stride || quantize->scales != gemm->a_scales ||
        quantize->scale_row_stride != gemm->a_scale_row_stride || quantize->scale_group_stride != gemm->a_scale_group_stride) {
        return fail(context, QPUCUDA_INVALID_ARGUMENT, "fp8_linear: the product must read the rows that are quantized");
    }
    qpucuda_status checked = check_quantize(context, quantize);
    if (checked == QPUCUDA_OK) checked = check_gemm(context, gemm);
    if (checked != QPUCUDA_OK) return checked;
    return submit(context, "fp8_linear",
                  [&] { return launch_fp8_linear(*quantize, *gemm, context->d_error, context->sm_count, context->stream); });
}

size_t qpucuda_expert_sort_workspace(uint32_t tokens, uint32_t choices, uint32_t experts) {
    return routing_fits(tokens, choices, experts) ? expert_sort_workspace(tokens, choices, experts) : 0;
}

qpucuda_status qpucuda_expert_sort(qpucuda_context *context, const qpucuda_expert_sort_desc *desc) {
    if (context == nullptr || desc == nullptr) return QPUCUDA_INVALID_ARGUMENT;
    const qpucuda_expert_sort_desc &d = *desc;
    if (!routing_fits(d.tokens, d.choices, d.experts) || d.offsets == nullptr || !aligned(d.offsets, 4) ||
        (d.tokens != 0 && (d.ids == nullptr || d.source == nullptr || d.position == nullptr ||
                           !aligned(d.ids, d.ids_64 != 0 ? 8 : 4) || !aligned(d.source, 4) || !aligned(d.position, 4)))) {
        return fail(context, QPUCUDA_INVALID_ARGUMENT,
                    "expert_sort: needs 1 to %u experts, at least one choice and fewer than 2^31 of them", QPUCUDA_MAX_EXPERTS);
    }
    const size_t needed = expert_sort_workspace(d.tokens, d.choices, d.experts);
    if (needed != 0 && (d.workspace == nullptr || d.workspace_bytes < needed || !aligned(d.workspace, 4))) {
        return fail(context, QPUCUDA_INVALID_ARGUMENT, "expert_sort: the workspace is smaller than %zu bytes", needed);
    }
    return submit(context, "expert_sort", [&] { return launch_expert_sort(d, context->stream); });
}

qpucuda_status qpucuda_expert_gather(qpucuda_context *context, const qpucuda_expert_rows_desc *desc) {
    if (context == nullptr || desc == nullptr) return QPUCUDA_INVALID_ARGUMENT;
    if (desc->tokens == 0) return QPUCUDA_OK;
    if (!routing_fits(desc->tokens, desc->choices, desc->experts) || !rows_fit(*desc) || !present(desc->offsets)) {
        return fail(context, QPUCUDA_INVALID_ARGUMENT, "expert_gather: invalid pointers, types or extents");
    }
    return submit(context, "expert_gather", [&] { return launch_expert_gather(*desc, context->sm_count, context->stream); });
}

qpucuda_status qpucuda_expert_combine(qpucuda_context *context, const qpucuda_expert_rows_desc *desc) {
    if (context == nullptr || desc == nullptr) return QPUCUDA_INVALID_ARGUMENT;
    if (desc->tokens == 0) return QPUCUDA_OK;
    if (!routing_fits(desc->tokens, desc->choices, 1) || !rows_fit(*desc) || !aligned(desc->weights, 4)) {
        return fail(context, QPUCUDA_INVALID_ARGUMENT, "expert_combine: invalid pointers, types or extents");
    }
    return submit(context, "expert_combine", [&] { return launch_expert_combine(*desc, context->sm_count, context->stream); });
}

qpucuda_status qpucuda_expert_combine_backward(qpucuda_context *context, const qpucuda_expert_rows_desc *desc) {
    if (context == nullptr || desc == nullptr) return QPUCUDA_INVALID_ARGUMENT;
    if (desc->tokens == 0) return QPUCUDA_OK;
    if (!routing_fits(desc->tokens, desc->choices, desc->experts) || !rows_fit(*desc) || !present(desc->offsets) ||
        !present(desc->weights) || !present(desc->grad_weights) || desc->grad == nullptr || desc->grad_stride < desc->width ||
        !aligned(desc->grad, type_bytes(desc->type))) {
        return fail(context, QPUCUDA_INVALID_ARGUMENT, "expert_combine_backward: invalid pointers, types or extents");
    }
    return submit(context, "expert_combine_backward",
                  [&] { return launch_expert_combine_backward(*desc, context->sm_count, context->stream); });
}

}  // extern "C"
