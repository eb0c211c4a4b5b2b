// Launchers of the block-scaled FP8 linear and of the expert routing (arguments already checked).
#pragma once

#include <cuda_runtime.h>

#include "qpucuda_experts.h"
#include "qpucuda_fp8.h"

namespace qpucuda {

cudaError_t launch_fp8_quantize_rows(const qpucuda_fp8_quantize_desc &desc, int sm_count, cudaStream_t stream);
cudaError_t launch_fp8_quantize_blocks(const void *x, int x_type, size_t x_stride, uint32_t batch, uint32_t rows,
                                       uint32_t cols, uint8_t *q, size_t q_stride, float *scales, cudaStream_t stream);
// Whether the rows (and, gated, their second halves) can be read in 16-byte vectors.
bool fp8_vector_rows(const qpucuda_fp8_quantize_desc &desc);
// error_word: the context's, for the kernel's bounded waits. cudaErrorInvalidValue when an operand
// cannot be described to the copy engine.
cudaError_t launch_fp8_gemm(const qpucuda_fp8_gemm_desc &desc, unsigned int *error_word, int sm_count,
                            cudaStream_t stream);
// The rows quantized, then their product; a few rows of a small matrix in one launch, which leaves
// quantize.q and .scales as they were.
cudaError_t launch_fp8_linear(const qpucuda_fp8_quantize_desc &quantize, const qpucuda_fp8_gemm_desc &gemm, unsigned int *error_word,
                              int sm_count, cudaStream_t stream);

size_t expert_sort_workspace(uint32_t tokens, uint32_t choices, uint32_t experts);
cudaError_t launch_expert_sort(const qpucuda_expert_sort_desc &desc, cudaStream_t stream);
cudaError_t launch_expert_gather(const qpucuda_expert_rows_desc &desc, int sm_count, cudaStream_t stream);
cudaError_t launch_expert_combine(const qpucuda_expert_rows_desc &desc, int sm_count, cudaStream_t stream);
cudaError_t launch_expert_combine_backward(const qpucuda_expert_rows_desc &desc, int sm_count, cudaStream_t stream);

}  // namespace qpucuda
