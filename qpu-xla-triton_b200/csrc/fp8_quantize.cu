// Quantizers of the block-scaled FP8 linear: activations to e4m3 with one scale per row and 128
// columns, weights to e4m3 with one scale per 128 x 128 block.
//
//   s = max(RN(max|x| / 448), 2^-60),   q = e4m3(RN(x / s)), round to nearest even
//
// 448 is the largest e4m3 value. The floor keeps s (and the product of a row's and a weight's
// scale, at least 2^-120) a normal number; a group below 448 * 2^-60 only loses relative precision.
// The maximum propagates NaN: a group with a NaN or an infinity has such a scale and dequantizes to
// NaN throughout.
#include <cuda_fp8.h>

#include "element.cuh"
#include "qpucuda_fp8_internal.h"
#include "qpucuda_internal.h"

namespace qpucuda {
namespace {

constexpr float kE4m3Max = 448.0f;
constexpr float kScaleFloor = 8.673617379884035e-19f;  // 2^-60

__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// max(RN(amax / 448), 2^-60), the quotient by Markstein's correction of a product with the rounded
// reciprocal: q0 = RN(a y) with y = RN(1 / 448) is within one step of a / 448, the remainder a - 448 q0
// is exact in an fma, and RN(q0 + remainder * y) is then the rounded quotient (amax above 2^-100;
// anything smaller ends at the floor). An infinite amax gives NaN, which serves as well.
__device__ __forceinline__ float group_scale(float amax) {
    constexpr float kReciprocal = 1.0f / 448.0f;
    const float q0 = __fmul_rn(amax, kReciprocal);
    const float remainder = __fmaf_rn(-q0, kE4m3Max, amax);
    return max_nan(__fmaf_rn(remainder, kReciprocal, q0), kScaleFloor);
}

__device__ __forceinline__ float reciprocal(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    return static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3)) |
           (static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3)) << 16);
}

// e4m3(RN(x / s)) of N values without a division each. The products with two reciprocals, 2^-20
// below and above an approximate one (which is within 2^-23; each product rounds by 2^-24), lie on
// either side of x / s, so of RN(x / s) too. Rounding to e4m3 is monotonic: where both give the same
// value, so does RN(x / s), in the subnormal range and at zero as well. Otherwise (a border within
// 2^-20, 1.5e-5 of the values) the quotients of all N are formed.
template <int N>
__device__ __forceinline__ void quantize_values(const float (&v)[N], float scale, uint32_t (&packed)[N / 4]) {
    const float inverse = reciprocal(scale);
    const float below = inverse * (1.0f - 9.5367431640625e-07f), above = inverse * (1.0f + 9.5367431640625e-07f);
    bool differ = false;
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        packed[i / 4] = e4m3x4(v[i] * below, v[i + 1] * below, v[i + 2] * below, v[i + 3] * below);
        differ |= packed[i / 4] != e4m3x4(v[i] * above, v[i + 1] * above, v[i + 2] * above, v[i + 3] * above);
    }
    if (differ) {
#pragma unroll
        for (int i = 0; i < N; i += 4)
            packed[i / 4] = e4m3x4(__fdiv_rn(v[i], scale), __fdiv_rn(v[i + 1], scale), __fdiv_rn(v[i + 2], scale), __fdiv_rn(v[i + 3], scale));
    }
}

// silu(g) * u in fp32. exp(-g) overflows to infinity below g = -88.7, where the quotient is then -0
// as it should be to fp32's range.
__device__ __forceinline__ float silu_times(float g, float u) { return __fdividef(g, 1.0f + __expf(-g)) * u; }

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

// Elements [column, column + kVector) of a row as fp32, zero past cols.
template <typename T, bool VECTOR>
__device__ __forceinline__ void load_row(const T *row, uint32_t column, uint32_t cols, float (&v)[kVector<T>]) {
    if (VECTOR && column + kVector<T> <= cols) {
        Vector<T> raw;
        raw.bits = load_stream16(row + column);
#pragma unroll
        for (int i = 0; i < kVector<T>; ++i) v[i] = to_float(raw.items[i]);
    } else {
#pragma unroll
        for (int i = 0; i < kVector<T>; ++i) v[i] = column + i < cols ? to_float(row[column + i]) : 0.0f;
    }
}

// One group is 128 columns of a row: kVector elements on each of 32 (fp32) or 16 (16-bit) lanes, so
// every lane moves 16 bytes and the maximum is a shuffle reduction inside those lanes. A warp takes
// kUnroll steps of one or two neighbouring groups and loads them all before it uses the first.
// Reads each input once and writes each output once: bound by HBM.
constexpr int kRowsThreads = 256;
constexpr int kUnroll = 4;

template <typename T, bool GATED, bool VECTOR>
__global__ void __launch_bounds__(kRowsThreads) quantize_rows_fp8_kernel(const RowsParams params) {
    constexpr int kLanes = 128 / kVector<T>;
    constexpr int kPerStep = 32 / kLanes;
    constexpr int kPerWarp = kPerStep * kUnroll;
    // The source may be the previous kernel's output. Once it is complete, the product that follows
    // may start and stream its weights while the rows are quantized.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t lane = threadIdx.x & 31u;
    const uint64_t total = static_cast<uint64_t>(params.rows) * params.groups;
    const uint64_t warps = static_cast<uint64_t>(gridDim.x) * (kRowsThreads / 32);
    for (uint64_t item0 = (static_cast<uint64_t>(blockIdx.x) * (kRowsThreads / 32) + threadIdx.x / 32) * kPerWarp;
         item0 < total; item0 += warps * kPerWarp) {
        const uint64_t first = item0 + lane / kLanes;
        uint32_t row, group;
        if (total <= 0xFFFFFFFFull) {
            row = static_cast<uint32_t>(first) / params.groups;
            group = static_cast<uint32_t>(first) - row * params.groups;
        } else {
            row = static_cast<uint32_t>(first / params.groups);
            group = static_cast<uint32_t>(first - static_cast<uint64_t>(row) * params.groups);
        }
        float v[kUnroll][kVector<T>];
        uint32_t rows[kUnroll], groups[kUnroll];
        const uint32_t inner = (lane % kLanes) * kVector<T>;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            rows[u] = row;
            groups[u] = group;
            const uint32_t column = group * 128u + inner;
            int64_t source = row < params.rows ? static_cast<int64_t>(row) : -1;
            if (source >= 0 && params.row_source != nullptr) {
                const int32_t entry = params.row_source[row];
                source = entry < 0 ? -1 : static_cast<int64_t>(static_cast<uint32_t>(entry) / params.row_divisor);
                if (source >= static_cast<int64_t>(params.source_rows)) source = -1;
            }
#pragma unroll
            for (int i = 0; i < kVector<T>; ++i) v[u][i] = 0.0f;
            if (source >= 0 && column < params.cols) {
                const T *x = static_cast<const T *>(params.x) + static_cast<size_t>(source) * params.x_stride;
                load_row<T, VECTOR>(x, column, params.cols, v[u]);
                if (GATED) {
                    float up[kVector<T>];
                    load_row<T, VECTOR>(x + params.cols, column, params.cols, up);
#pragma unroll
                    for (int i = 0; i < kVector<T>; ++i) v[u][i] = silu_times(v[u][i], up[i]);
                }
            }
            group += kPerStep;
            while (group >= params.groups) {
                group -= params.groups;
                ++row;
            }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            float amax = 0.0f;
#pragma unroll
            for (int i = 0; i < kVector<T>; ++i) amax = max_nan(amax, fabsf(v[u][i]));
#pragma unroll
            for (int offset = kLanes / 2; offset > 0; offset >>= 1)
                amax = max_nan(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, offset));
            const float scale = group_scale(amax);
            uint32_t packed[kVector<T> / 4];
            quantize_values(v[u], scale, packed);
            const uint32_t column = groups[u] * 128u + inner;
            if (rows[u] < params.rows) {
                // q rows are padded to 16 bytes, so a vector that starts below cols fits
                if (column < params.cols) {
                    uint8_t *q = params.q + static_cast<size_t>(rows[u]) * params.q_stride + column;
                    if constexpr (kVector<T> == 8) {
                        *reinterpret_cast<uint2 *>(q) = make_uint2(packed[0], packed[kVector<T> / 4 - 1]);
                    } else {
                        *reinterpret_cast<uint32_t *>(q) = packed[0];
                    }
                }
                if (inner == 0)
                    params.scales[static_cast<size_t>(rows[u]) * params.scale_row_stride +
                                  static_cast<size_t>(groups[u]) * params.scale_group_stride] = scale;
            }
        }
    }
}

// One CTA per 128 x 128 block: its maximum, then its values (the second read hits the caches).
// Runs once per weight, when it is prepared.
template <typename T>
__global__ void __launch_bounds__(256) quantize_blocks_fp8_kernel(const T *__restrict__ x, size_t x_stride,
                                                                  uint32_t rows, uint32_t cols, uint8_t *q,
                                                                  size_t q_stride, float *scales) {
    __shared__ float warp_max[8];
    const uint32_t row0 = blockIdx.y * 128u, col0 = blockIdx.x * 128u;
    const size_t batch = blockIdx.z;
    const T *matrix = x + batch * rows * x_stride;
    uint8_t *values = q + batch * rows * q_stride;
    const uint32_t column = col0 + (threadIdx.x & 127u);
    const uint32_t end = min(rows, row0 + 128u);
    float amax = 0.0f;
    if (column < cols)
        for (uint32_t r = row0 + threadIdx.x / 128u; r < end; r += 2)
            amax = max_nan(amax, fabsf(to_float(matrix[static_cast<size_t>(r) * x_stride + column])));
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, offset));
    if ((threadIdx.x & 31u) == 0) warp_max[threadIdx.x / 32u] = amax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) amax = max_nan(amax, warp_max[w]);
    const float scale = group_scale(amax);
    if (threadIdx.x == 0) scales[(batch * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x] = scale;
    if (column < cols)
        for (uint32_t r = row0 + threadIdx.x / 128u; r < end; r += 2) {
            const float v = __fdiv_rn(to_float(matrix[static_cast<size_t>(r) * x_stride + column]), scale);
            values[static_cast<size_t>(r) * q_stride + column] = __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
        }
}

template <typename T, bool GATED>
cudaError_t launch_rows(const RowsParams &params, bool vector, int sm_count, cudaStream_t stream) {
    constexpr uint64_t kPerBlock = static_cast<uint64_t>(32 / (128 / kVector<T>)) * kUnroll * (kRowsThreads / 32);
    const uint64_t total = static_cast<uint64_t>(params.rows) * params.groups;
    uint64_t blocks = (total + kPerBlock - 1) / kPerBlock;
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
    return vector ? cudaLaunchKernelEx(&config, quantize_rows_fp8_kernel<T, GATED, true>, params)
                  : cudaLaunchKernelEx(&config, quantize_rows_fp8_kernel<T, GATED, false>, params);
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
    params.source_rows = desc.source_rows;
    params.q = desc.q;
    params.q_stride = desc.q_stride;
    params.scales = desc.scales;
    params.scale_row_stride = desc.scale_row_stride;
    params.scale_group_stride = desc.scale_group_stride;
    // 16-byte loads need aligned rows and, gated, an aligned second half.
    const bool vector = (reinterpret_cast<uintptr_t>(desc.x) & 15u) == 0 && desc.x_stride % kVector<T> == 0 &&
                        (desc.gated == 0 || desc.cols % kVector<T> == 0);
    return desc.gated != 0 ? launch_rows<T, true>(params, vector, sm_count, stream)
                           : launch_rows<T, false>(params, vector, sm_count, stream);
}

}  // namespace

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
    const dim3 grid((cols + 127u) / 128u, (rows + 127u) / 128u, batch);
    switch (x_type) {
        case QPUCUDA_DTYPE_F32:
            quantize_blocks_fp8_kernel<<<grid, 256, 0, stream>>>(static_cast<const float *>(x), x_stride, rows, cols, q,
                                                                 q_stride, scales);
            break;
        case QPUCUDA_DTYPE_BF16:
            quantize_blocks_fp8_kernel<<<grid, 256, 0, stream>>>(static_cast<const __nv_bfloat16 *>(x), x_stride, rows,
                                                                 cols, q, q_stride, scales);
            break;
        case QPUCUDA_DTYPE_F16:
            quantize_blocks_fp8_kernel<<<grid, 256, 0, stream>>>(static_cast<const __half *>(x), x_stride, rows, cols, q,
                                                                 q_stride, scales);
            break;
        default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

}  // namespace qpucuda
