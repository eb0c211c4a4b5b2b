// Quantizers of the block-scaled FP8 linear: activations to e4m3 with one scale per row and 128
// columns, weights to e4m3 with one scale per 128 x 128 block.
//
//   s = max(RN(max|x| / 448), 2^-60),   q = e4m3(RN(x / s)), round to nearest even
//
// 448 is the largest e4m3 value. The floor keeps s (and the product of a row's and a weight's
// scale, at least 2^-120) a normal number; a group below 448 * 2^-60 only loses relative precision.
// The maximum propagates NaN: a group with a NaN or an infinity has such a scale and dequantizes to
// NaN throughout.
#include "fp8_quantize.cuh"
#include "qpucuda_fp8_internal.h"
#include "qpucuda_internal.h"

namespace qpucuda {
namespace {

struct RowsParams {
    const void *x;
    size_t x_stride;
    uint32_t rows, cols, groups;
    const int32_t *row_source;
    uint32_t row_divisor, source_rows;
    uint8_t *q;
    size_t q_stride;
    float *scales;
    size_t scale_row_stride, scale_group_stride;
};

// One group is 128 columns of a row: kVector elements on each of 32 (fp32) or 16 (16-bit) lanes, so
// every lane moves 16 bytes and the maximum is a shuffle reduction inside those lanes. A warp takes
// STEPS steps of one or two neighbouring groups of one row, at fixed distances from one address, and
// loads them all before it uses the first (39 against 27 us). Each input is read once, each output
// written once. 32768 x 8192 bf16: 145 us (5.6 TB/s), 4096 x 8192 fp32: 29 us (5.8 TB/s), bf16 20 us
// (5.1), gated bf16: 39 us (4.3). At 4096 x 8192 bf16 neither the issue slots (57 %, about 14 instructions a
// value) nor the warps (54 %) are full: a warp's loads, maximum and stores follow one another.
constexpr int kRowsThreads = 128;

template <typename T, bool GATED, bool VECTOR, int STEPS>
__global__ void __launch_bounds__(kRowsThreads) quantize_rows_fp8_kernel(const RowsParams params, uint32_t chunks) {
    constexpr int kLanes = 128 / kVector<T>;
    constexpr int kPerStep = 32 / kLanes;
    // The source may be the previous kernel's output. Once it is complete, the product that follows
    // may start and stream its weights while the rows are quantized.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t lane = threadIdx.x & 31u;
    const uint32_t inner = lane * kVector<T>;  // column inside a step
    const uint64_t total = static_cast<uint64_t>(params.rows) * chunks;
    const uint64_t warps = static_cast<uint64_t>(gridDim.x) * (kRowsThreads / 32);
    for (uint64_t item = static_cast<uint64_t>(blockIdx.x) * (kRowsThreads / 32) + threadIdx.x / 32; item < total; item += warps) {
        uint32_t row, chunk;
        if (total <= 0xFFFFFFFFull) {
            row = static_cast<uint32_t>(item) / chunks;
            chunk = static_cast<uint32_t>(item) - row * chunks;
        } else {
            row = static_cast<uint32_t>(item / chunks);
            chunk = static_cast<uint32_t>(item - static_cast<uint64_t>(row) * chunks);
        }
        uint32_t source = row;
        if (params.row_source != nullptr) {
            const int32_t entry = params.row_source[row];
            source = entry < 0 ? 0xFFFFFFFFu : static_cast<uint32_t>(entry) / params.row_divisor;
        }
        const bool present = source < params.source_rows;
        const uint32_t column0 = chunk * (STEPS * kPerStep * 128u) + inner;
        const T *x = static_cast<const T *>(params.x) + (present ? static_cast<size_t>(source) * params.x_stride : 0) + column0;
        constexpr uint32_t kStep = kPerStep * 128;
        const uint32_t remaining = present && column0 < params.cols ? params.cols - column0 : 0u;
        Vector<T> raw[STEPS], raw_up[GATED ? STEPS : 1];
        load_steps<T, VECTOR>(x, remaining, kStep, raw);
        if constexpr (GATED) load_steps<T, VECTOR>(x + params.cols, remaining, kStep, raw_up);
        uint8_t *q = params.q + static_cast<size_t>(row) * params.q_stride + column0;
        const uint32_t group0 = column0 / 128u;
        float *scales = params.scales + static_cast<size_t>(row) * params.scale_row_stride + static_cast<size_t>(group0) * params.scale_group_stride;
#pragma unroll
        for (int u = 0; u < STEPS; ++u) {
            float v[kVector<T>], amax = 0.0f;
#pragma unroll
            for (int i = 0; i < kVector<T>; ++i) v[i] = to_float(raw[u].items[i]);
            if constexpr (GATED) {
                float up[kVector<T>];
#pragma unroll
                for (int i = 0; i < kVector<T>; ++i) up[i] = to_float(raw_up[u].items[i]);
                silu_times(v, up);
            }
#pragma unroll
            for (int i = 0; i < kVector<T>; ++i) amax = max_nan(amax, fabsf(v[i]));
            const float scale = group_scale(group_max<kLanes>(amax));
            uint32_t packed[kVector<T> / 4];
            quantize_values(v, scale, packed);
            if (column0 + u * (kPerStep * 128u) < params.cols) {
                // q rows are padded to 16 bytes, so a vector that starts below cols fits
                if constexpr (kVector<T> == 8) {
                    *reinterpret_cast<uint2 *>(q + u * kPerStep * 128) = make_uint2(packed[0], packed[kVector<T> / 4 - 1]);
                } else {
                    *reinterpret_cast<uint32_t *>(q + u * kPerStep * 128) = packed[0];
                }
                if (lane % kLanes == 0) scales[static_cast<size_t>(u * kPerStep) * params.scale_group_stride] = scale;
            }
        }
    }
}

// One CTA per 128 x 128 block, held in registers between its maximum and its values: a warp's lanes
// take four neighbouring columns each, its rows are 16 apart. WHOLE: rows of x and q allow vectors of
// four; the ragged blocks of such a matrix go element by element all the same. Runs once per weight,
// when it is prepared: 28672 x 8192 fp32 195 us (6.0 TB/s; 488 us with a second read in place of the
// registers), bf16 343 (2.1 TB/s: a lane loads 8 bytes a row where fp32 loads 16).
constexpr int kBlockThreads = 512;

template <typename T>
struct alignas(4 * sizeof(T)) Four {
    T items[4];
};

template <typename T, bool WHOLE>
__global__ void __launch_bounds__(kBlockThreads, 2) quantize_blocks_fp8_kernel(const T *__restrict__ x, size_t x_stride,
                                                                            uint32_t rows, uint32_t cols, uint8_t *q,
                                                                            size_t q_stride, float *scales) {
    constexpr int kWarps = kBlockThreads / 32;
    constexpr int kRows = 128 / kWarps;
    __shared__ float warp_max[kWarps];
    const uint32_t warp = threadIdx.x / 32u, lane = threadIdx.x & 31u;
    const uint32_t row0 = blockIdx.y * 128u + warp, col0 = blockIdx.x * 128u + lane * 4u;
    const size_t batch = blockIdx.z;
    const T *matrix = x + batch * rows * x_stride;
    uint8_t *values = q + batch * rows * q_stride;
    const bool vector = WHOLE && col0 + 4 <= cols;
    Four<T> x4[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const uint32_t row = row0 + i * kWarps;
        const T *at = matrix + static_cast<size_t>(row) * x_stride + col0;
        if (vector && row < rows) {
            x4[i] = *reinterpret_cast<const Four<T> *>(at);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) x4[i].items[j] = row < rows && col0 + j < cols ? at[j] : from_float<T>(0.0f);
        }
    }
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) amax = max_nan(amax, fabsf(to_float(x4[i].items[j])));
    amax = group_max<32>(amax);
    if (lane == 0) warp_max[warp] = amax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) amax = max_nan(amax, warp_max[w]);
    const float scale = group_scale(amax);
    if (threadIdx.x == 0) scales[(batch * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x] = scale;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
        const uint32_t row = row0 + i * kWarps;
        uint32_t packed[1];
        const float v[4] = {to_float(x4[i].items[0]), to_float(x4[i].items[1]), to_float(x4[i].items[2]), to_float(x4[i].items[3])};
        quantize_values(v, scale, packed);
        uint8_t *at = values + static_cast<size_t>(row) * q_stride + col0;
        if (vector && row < rows) {
            *reinterpret_cast<uint32_t *>(at) = packed[0];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (row < rows && col0 + j < cols) at[j] = static_cast<uint8_t>(packed[0] >> (8 * j));
        }
    }
}

template <typename T>
cudaError_t launch_blocks(const void *x, size_t x_stride, uint32_t batch, uint32_t rows, uint32_t cols, uint8_t *q, size_t q_stride,
                          float *scales, cudaStream_t stream) {
    const dim3 grid((cols + 127u) / 128u, (rows + 127u) / 128u, batch);
    const bool whole = reinterpret_cast<uintptr_t>(x) % (4 * sizeof(T)) == 0 && x_stride % 4 == 0 &&
                       reinterpret_cast<uintptr_t>(q) % 4 == 0 && q_stride % 4 == 0;
    auto kernel = whole ? quantize_blocks_fp8_kernel<T, true> : quantize_blocks_fp8_kernel<T, false>;
    kernel<<<grid, kBlockThreads, 0, stream>>>(static_cast<const T *>(x), x_stride, rows, cols, q, q_stride, scales);
    return cudaGetLastError();
}

template <typename T, bool GATED, bool VECTOR, int STEPS>
cudaError_t launch_rows(const RowsParams &params, int sm_count, cudaStream_t stream) {
    constexpr uint32_t kGroups = static_cast<uint32_t>(32 / (128 / kVector<T>)) * STEPS;
    const uint32_t chunks = (params.groups + kGroups - 1) / kGroups;
    const uint64_t warps = static_cast<uint64_t>(params.rows) * chunks;
    uint64_t blocks = (warps + kRowsThreads / 32 - 1) / (kRowsThreads / 32);
    const uint64_t most = static_cast<uint64_t>(sm_count) * 64u;
    if (blocks > most) blocks = most;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(blocks));
    config.blockDim = dim3(kRowsThreads);
    config.stream = stream;
    config.attrs = &attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, quantize_rows_fp8_kernel<T, GATED, VECTOR, STEPS>, params, chunks);
}

// Four steps a warp where that still gives every SM 16 warps, one otherwise (us, one and four steps: gated
// fp16 333 x 5632 3.6 and 4.4, 1024 x 5632 8.5 and 8.2; fp32 333 x 5632 4.1 and 3.8).
template <typename T, bool GATED>
cudaError_t launch_rows_steps(const RowsParams &params, bool vector, int sm_count, cudaStream_t stream) {
    constexpr uint64_t kGroups = 4u * (32u / (128u / kVector<T>));  // of a warp with four steps
    const bool many = params.groups >= 4 && static_cast<uint64_t>(params.rows) * params.groups >= static_cast<uint64_t>(sm_count) * 16u * kGroups;
    if (vector) {
        return many ? launch_rows<T, GATED, true, 4>(params, sm_count, stream) : launch_rows<T, GATED, true, 1>(params, sm_count, stream);
    }
    return many ? launch_rows<T, GATED, false, 4>(params, sm_count, stream) : launch_rows<T, GATED, false, 1>(params, sm_count, stream);
}

template <typename T>
cudaError_t launch_rows_type(const qpucuda_fp8_quantize_desc &desc, int sm_count, cudaStream_t stream) {
    RowsParams params{};
    params.x = desc.x;
    params.x_stride = desc.x_stride;
    params.rows = desc.rows;
    params.cols = desc.cols;
    params.groups = (desc.cols + 127u) / 128u;
    params.row_source = desc.row_source;
    params.row_divisor = desc.row_divisor;
    params.source_rows = desc.row_source != nullptr ? desc.source_rows : desc.rows;
    params.q = desc.q;
    params.q_stride = desc.q_stride;
    params.scales = desc.scales;
    params.scale_row_stride = desc.scale_row_stride;
    params.scale_group_stride = desc.scale_group_stride;
    const bool vector = fp8_vector_rows(desc);
    return desc.gated != 0 ? launch_rows_steps<T, true>(params, vector, sm_count, stream)
                           : launch_rows_steps<T, false>(params, vector, sm_count, stream);
}

}  // namespace

bool fp8_vector_rows(const qpucuda_fp8_quantize_desc &desc) {
    const size_t items = desc.x_type == QPUCUDA_DTYPE_F32 ? 4 : 8;  // of 16 bytes
    return (reinterpret_cast<uintptr_t>(desc.x) & 15u) == 0 && desc.x_stride % items == 0 && (desc.gated == 0 || desc.cols % items == 0);
}

cudaError_t launch_fp8_quantize_rows(const qpucuda_fp8_quantize_desc &desc, int sm_count, cudaStream_t stream) {
    switch (desc.x_type) {
        case QPUCUDA_DTYPE_F32: return launch_rows_type<float>(desc, sm_count, stream);
        case QPUCUDA_DTYPE_BF16: return launch_rows_type<__nv_bfloat16>(desc, sm_count, stream);
        case QPUCUDA_DTYPE_F16: return launch_rows_type<__half>(desc, sm_count, stream);
    }
    return cudaErrorInvalidValue;
}

cudaError_t launch_fp8_quantize_blocks(const void *x, int x_type, size_t x_stride, uint32_t batch, uint32_t rows,
                                       uint32_t cols, uint8_t *q, size_t q_stride, float *scales,
                                       cudaStream_t stream) {
    switch (x_type) {
        case QPUCUDA_DTYPE_F32: return launch_blocks<float>(x, x_stride, batch, rows, cols, q, q_stride, scales, stream);
        case QPUCUDA_DTYPE_BF16: return launch_blocks<__nv_bfloat16>(x, x_stride, batch, rows, cols, q, q_stride, scales, stream);
        case QPUCUDA_DTYPE_F16: return launch_blocks<__half>(x, x_stride, batch, rows, cols, q, q_stride, scales, stream);
    }
    return cudaErrorInvalidValue;
}

}  // namespace qpucuda
