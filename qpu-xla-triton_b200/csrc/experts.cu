// Tokens sorted by expert and back (include/qpucuda_experts.h).
//
// The sort is a stable counting sort in integers. A choice's row is
//   offsets[e] + (choices of e in earlier chunks) + (in earlier warps of its chunk) + (earlier in its warp),
// every term an exact count, so the order never depends on timing. Moving the rows is bound by HBM:
// each kernel reads a token's vector once, in registers, for all of its choices, and writes each
// row once.
#include "element.cuh"
#include "qpucuda_fp8_internal.h"
#include "qpucuda_internal.h"

namespace qpucuda {
namespace {

// ---- sort -----------------------------------------------------------------------------------

constexpr int kSortThreads = 512;
constexpr int kSortWarps = kSortThreads / 32;
// A chunk is one CTA's share. Up to kSortChunk choices take one CTA and one launch; above, at most
// kSortMaxChunks CTAs, so that each can add up the counts of all chunks by itself.
constexpr uint32_t kSortChunk = 4096;
constexpr uint32_t kSortMaxChunks = 64;
constexpr uint32_t kMaxExperts = QPUCUDA_MAX_EXPERTS;

uint32_t sort_chunk(uint32_t total) {
    const uint32_t least = (total + kSortMaxChunks - 1) / kSortMaxChunks;
    const uint32_t chunk = least > kSortChunk ? least : kSortChunk;
    return (chunk + kSortThreads - 1) / kSortThreads * kSortThreads;
}

template <typename Id>
__device__ __forceinline__ uint32_t expert_of(const Id *ids, uint32_t index, uint32_t end, uint32_t experts) {
    if (index >= end) return kMaxExperts;
    const Id id = ids[index];
    return id >= 0 && id < static_cast<Id>(experts) ? static_cast<uint32_t>(id) : kMaxExperts;
}

// counts[chunk][expert] of one chunk per CTA.
template <typename Id>
__global__ void __launch_bounds__(kSortThreads) expert_count_kernel(const Id *__restrict__ ids, uint32_t total,
                                                                    uint32_t chunk, uint32_t experts, int32_t *counts) {
    __shared__ int32_t histogram[kMaxExperts];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    for (uint32_t e = threadIdx.x; e < experts; e += kSortThreads) histogram[e] = 0;
    __syncthreads();
    const uint32_t begin = blockIdx.x * chunk;
    const uint32_t end = min(total, begin + chunk);
    for (uint32_t i = begin + threadIdx.x; i < end; i += kSortThreads) {
        const uint32_t e = expert_of(ids, i, end, experts);
        if (e < experts) atomicAdd(&histogram[e], 1);
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < experts; e += kSortThreads)
        counts[static_cast<size_t>(blockIdx.x) * experts + e] = histogram[e];
}

// Rows of one chunk per CTA. counts: [gridDim.x][experts], or null for a single chunk.
template <typename Id>
__global__ void __launch_bounds__(kSortThreads) expert_scatter_kernel(const Id *__restrict__ ids, uint32_t total,
                                                                      uint32_t chunk, uint32_t experts,
                                                                      const int32_t *counts, int32_t *offsets,
                                                                      int32_t *source, int32_t *position) {
    extern __shared__ int32_t next[];  // [kSortWarps][experts]: counts, then the next row of (warp, expert)
    __shared__ int32_t warp_sums[kSortWarps];
    __shared__ int32_t kept;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t warp = threadIdx.x / 32u, lane = threadIdx.x & 31u;
    for (uint32_t i = threadIdx.x; i < kSortWarps * experts; i += kSortThreads) next[i] = 0;
    __syncthreads();
    const uint32_t begin = blockIdx.x * chunk;
    const uint32_t end = min(total, begin + chunk);
    const uint32_t share = chunk / kSortWarps;  // a multiple of 32
    const uint32_t warp_begin = begin + warp * share;
    const uint32_t warp_end = min(end, warp_begin + share);
    int32_t *own = next + warp * experts;
    for (uint32_t i = warp_begin + lane; i < warp_end; i += 32) {
        const uint32_t e = expert_of(ids, i, warp_end, experts);
        if (e < experts) atomicAdd(&own[e], 1);
    }
    __syncthreads();
    // Thread t takes experts 2t and 2t + 1: their counts over this chunk's warps become offsets
    // inside the chunk, their totals over all chunks are scanned into the experts' first rows.
    int32_t in_all[2], before[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const uint32_t e = 2u * threadIdx.x + s;
        in_all[s] = before[s] = 0;
        if (e < experts) {
            int32_t in_chunk = 0;
            for (int w = 0; w < kSortWarps; ++w) {
                const int32_t count = next[w * experts + e];
                next[w * experts + e] = in_chunk;
                in_chunk += count;
            }
            in_all[s] = in_chunk;
            if (counts != nullptr) {
                int32_t sum = 0;
                for (uint32_t c = 0; c < gridDim.x; ++c) {
                    if (c == blockIdx.x) before[s] = sum;
                    sum += counts[static_cast<size_t>(c) * experts + e];
                }
                in_all[s] = sum;
            }
        }
    }
    const int32_t pair = in_all[0] + in_all[1];
    int32_t inclusive = pair;
#pragma unroll
    for (int offset = 1; offset < 32; offset <<= 1) {
        const int32_t other = __shfl_up_sync(0xFFFFFFFFu, inclusive, offset);
        if (lane >= static_cast<uint32_t>(offset)) inclusive += other;
    }
    if (lane == 31) warp_sums[warp] = inclusive;
    __syncthreads();
    int32_t first = inclusive - pair;
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w)
        if (static_cast<uint32_t>(w) < warp) first += warp_sums[w];
    if (threadIdx.x == kSortThreads - 1) kept = first + pair;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const uint32_t e = 2u * threadIdx.x + s;
        if (e < experts) {
            for (int w = 0; w < kSortWarps; ++w) next[w * experts + e] += first + before[s];
            if (blockIdx.x == 0) offsets[e] = first;
        }
        first += in_all[s];
    }
    __syncthreads();
    if (blockIdx.x == 0 && threadIdx.x == 0) offsets[experts] = kept;
    for (uint32_t i0 = warp_begin; i0 < warp_end; i0 += 32) {
        const uint32_t i = i0 + lane;
        const uint32_t e = expert_of(ids, i, warp_end, experts);
        const uint32_t same = __match_any_sync(0xFFFFFFFFu, e);
        const uint32_t earlier = __popc(same & ((1u << lane) - 1u));
        int32_t row = -1;
        if (e < experts) row = own[e] + static_cast<int32_t>(earlier);
        __syncwarp();
        if (e < experts && earlier == 0) own[e] += __popc(same);
        __syncwarp();
        if (i < warp_end) {
            position[i] = row;
            if (row >= 0) source[row] = static_cast<int32_t>(i);
        }
    }
    const uint32_t stride = gridDim.x * kSortThreads;
    for (uint32_t row = static_cast<uint32_t>(kept) + blockIdx.x * kSortThreads + threadIdx.x; row < total; row += stride)
        source[row] = -1;
}

// ---- rows -------------------------------------------------------------------------------------

constexpr int kRowThreads = 256;

// VEC elements of T move as one: 16 bytes, or a single element where a base or a stride is not a
// multiple of 16 bytes.
template <typename T, int VEC>
struct Pack {
    T items[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack(const T *p) {
    Pack<T, VEC> result;
    if constexpr (VEC == 1) {
        result.items[0] = *p;
    } else {
        *reinterpret_cast<uint4 *>(&result) = load_stream16(p);
    }
    return result;
}

template <typename T, int VEC>
__device__ __forceinline__ void store_pack(T *p, const Pack<T, VEC> &value) {
    if constexpr (VEC == 1) {
        *p = value.items[0];
    } else {
        *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(&value);
    }
}

// (row, pack) of a flat index; the division is 32 bits wide where the whole range is.
__device__ __forceinline__ void split_index(uint64_t index, uint64_t total, uint32_t packs, uint32_t &row, uint32_t &pack) {
    if (total <= 0xFFFFFFFFull) {
        row = static_cast<uint32_t>(index) / packs;
        pack = static_cast<uint32_t>(index) - row * packs;
    } else {
        row = static_cast<uint32_t>(index / packs);
        pack = static_cast<uint32_t>(index - static_cast<uint64_t>(row) * packs);
    }
}

// The rows no expert owns, [offsets[experts], count), become zero.
template <typename T, int VEC>
__device__ __forceinline__ void zero_tail(T *rows, size_t stride, uint32_t count, uint32_t packs, const int32_t *end) {
    const int32_t raw = *end;
    const uint32_t first = raw < 0 ? 0u : min(static_cast<uint32_t>(raw), count);
    const uint64_t total = static_cast<uint64_t>(count - first) * packs;
    const uint64_t step = static_cast<uint64_t>(gridDim.x) * blockDim.x;
    Pack<T, VEC> zero;
#pragma unroll
    for (int i = 0; i < VEC; ++i) zero.items[i] = from_float<T>(0.0f);
    for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += step) {
        uint32_t row, pack;
        split_index(i, total, packs, row, pack);
        store_pack<T, VEC>(rows + static_cast<size_t>(first + row) * stride + static_cast<size_t>(pack) * VEC, zero);
    }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kRowThreads) expert_gather_kernel(const T *__restrict__ x, size_t x_stride,
                                                                    uint32_t tokens, uint32_t choices, uint32_t packs,
                                                                    const int32_t *position, const int32_t *end,
                                                                    T *rows, size_t rows_stride) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t count = tokens * choices;
    const uint64_t total = static_cast<uint64_t>(tokens) * packs;
    const uint64_t step = static_cast<uint64_t>(gridDim.x) * kRowThreads;
    for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * kRowThreads + threadIdx.x; i < total; i += step) {
        uint32_t token, pack;
        split_index(i, total, packs, token, pack);
        const size_t column = static_cast<size_t>(pack) * VEC;
        const Pack<T, VEC> value = load_pack<T, VEC>(x + static_cast<size_t>(token) * x_stride + column);
        const int32_t *at = position + static_cast<size_t>(token) * choices;
        for (uint32_t j = 0; j < choices; ++j) {
            const uint32_t row = static_cast<uint32_t>(at[j]);  // -1 is out of range as well
            if (row < count) store_pack<T, VEC>(rows + static_cast<size_t>(row) * rows_stride + column, value);
        }
    }
    zero_tail<T, VEC>(rows, rows_stride, count, packs, end);
}

// out[t] = sum_j w[t, j] rows[position[t, j]]: fp32 in the order of j, rounded once. The rows of up
// to kAhead choices are loaded before the first is added.
constexpr int kAhead = 4;

template <typename T, int VEC, bool WEIGHTED>
__global__ void __launch_bounds__(kRowThreads) expert_combine_kernel(const T *__restrict__ rows, size_t rows_stride,
                                                                     uint32_t tokens, uint32_t choices, uint32_t packs,
                                                                     const int32_t *position, const float *weights,
                                                                     T *out, size_t out_stride) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t count = tokens * choices;
    const uint64_t total = static_cast<uint64_t>(tokens) * packs;
    const uint64_t step = static_cast<uint64_t>(gridDim.x) * kRowThreads;
    for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * kRowThreads + threadIdx.x; i < total; i += step) {
        uint32_t token, pack;
        split_index(i, total, packs, token, pack);
        const size_t column = static_cast<size_t>(pack) * VEC;
        const size_t at = static_cast<size_t>(token) * choices;
        float sum[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) sum[v] = 0.0f;
        for (uint32_t j0 = 0; j0 < choices; j0 += kAhead) {
            Pack<T, VEC> value[kAhead];
            bool present[kAhead];
            float weight[kAhead];
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                const uint32_t row = j0 + a < choices ? static_cast<uint32_t>(position[at + j0 + a]) : count;
                present[a] = row < count;
                weight[a] = 1.0f;
                if (present[a]) {
                    value[a] = load_pack<T, VEC>(rows + static_cast<size_t>(row) * rows_stride + column);
                    if (WEIGHTED) weight[a] = weights[at + j0 + a];
                }
            }
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                if (!present[a]) continue;
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    const float x = to_float(value[a].items[v]);
                    sum[v] = WEIGHTED ? fmaf(weight[a], x, sum[v]) : sum[v] + x;
                }
            }
        }
        Pack<T, VEC> result;
#pragma unroll
        for (int v = 0; v < VEC; ++v) result.items[v] = from_float<T>(sum[v]);
        store_pack<T, VEC>(out + static_cast<size_t>(token) * out_stride + column, result);
    }
}

// One CTA per token: grad[t] is read once per kAhead choices, each choice's row once; its dot
// product with grad[t] is summed per thread, then over the CTA in a fixed order.
template <typename T, int VEC>
__global__ void __launch_bounds__(kRowThreads)
    expert_combine_backward_kernel(const T *__restrict__ rows, size_t rows_stride, const T *__restrict__ grad,
                                   size_t grad_stride, uint32_t tokens, uint32_t choices, uint32_t packs,
                                   const int32_t *position, const int32_t *end, const float *weights, T *grad_rows,
                                   size_t grad_rows_stride, float *grad_weights) {
    __shared__ float partial[kRowThreads / 32][kAhead];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t count = tokens * choices;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x / 32u, warps = blockDim.x / 32u;
    for (uint32_t token = blockIdx.x; token < tokens; token += gridDim.x) {
        const T *g = grad + static_cast<size_t>(token) * grad_stride;
        const size_t at = static_cast<size_t>(token) * choices;
        for (uint32_t j0 = 0; j0 < choices; j0 += kAhead) {
            uint32_t row[kAhead];
            float weight[kAhead], dot[kAhead];
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                row[a] = j0 + a < choices ? static_cast<uint32_t>(position[at + j0 + a]) : count;
                weight[a] = row[a] < count ? weights[at + j0 + a] : 0.0f;
                dot[a] = 0.0f;
            }
            for (uint32_t pack = threadIdx.x; pack < packs; pack += blockDim.x) {
                const size_t column = static_cast<size_t>(pack) * VEC;
                const Pack<T, VEC> upstream = load_pack<T, VEC>(g + column);
                Pack<T, VEC> value[kAhead];
#pragma unroll
                for (int a = 0; a < kAhead; ++a)
                    if (row[a] < count) value[a] = load_pack<T, VEC>(rows + static_cast<size_t>(row[a]) * rows_stride + column);
#pragma unroll
                for (int a = 0; a < kAhead; ++a) {
                    if (row[a] >= count) continue;
                    Pack<T, VEC> scaled;
#pragma unroll
                    for (int v = 0; v < VEC; ++v) {
                        const float u = to_float(upstream.items[v]);
                        dot[a] = fmaf(to_float(value[a].items[v]), u, dot[a]);
                        scaled.items[v] = from_float<T>(weight[a] * u);
                    }
                    store_pack<T, VEC>(grad_rows + static_cast<size_t>(row[a]) * grad_rows_stride + column, scaled);
                }
            }
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
#pragma unroll
                for (int offset = 16; offset > 0; offset >>= 1) dot[a] += __shfl_xor_sync(0xFFFFFFFFu, dot[a], offset);
                if (lane == 0) partial[warp][a] = dot[a];
            }
            __syncthreads();
            if (threadIdx.x < kAhead && j0 + threadIdx.x < choices) {
                float sum = 0.0f;
                for (uint32_t w = 0; w < warps; ++w) sum += partial[w][threadIdx.x];
                grad_weights[at + j0 + threadIdx.x] = sum;  // nothing was added for a dropped choice
            }
            __syncthreads();
        }
    }
    zero_tail<T, VEC>(grad_rows, grad_rows_stride, count, packs, end);
}

// ---- launches -----------------------------------------------------------------------------------

template <typename... Parameters, typename... Arguments>
cudaError_t launch(void (*kernel)(Parameters...), uint32_t blocks, uint32_t threads, size_t shared, cudaStream_t stream,
                   Arguments... arguments) {
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(blocks);
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = shared;
    config.stream = stream;
    config.attrs = &attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, static_cast<Parameters>(arguments)...);
}

bool vector_rows(const void *base, size_t stride, size_t item) {
    return (reinterpret_cast<uintptr_t>(base) & 15u) == 0 && stride * item % 16u == 0;
}

uint32_t row_blocks(uint64_t items, int sm_count) {
    const uint64_t blocks = (items + kRowThreads - 1) / kRowThreads;
    const uint64_t most = static_cast<uint64_t>(sm_count) * 32u;
    return static_cast<uint32_t>(blocks < most ? (blocks == 0 ? 1 : blocks) : most);
}

template <typename Id>
cudaError_t sort_typed(const Id *ids, uint32_t total, uint32_t experts, int32_t *offsets, int32_t *source,
                       int32_t *position, int32_t *counts, cudaStream_t stream) {
    static PerDeviceOnce configured;
    const cudaError_t error = configured.run([] {
        return cudaFuncSetAttribute(expert_scatter_kernel<Id>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    static_cast<int>(kSortWarps * kMaxExperts * sizeof(int32_t)));
    });
    if (error != cudaSuccess) return error;
    const uint32_t chunk = sort_chunk(total);
    const uint32_t chunks = total == 0 ? 1u : (total + chunk - 1) / chunk;
    if (chunks > 1) {
        const cudaError_t counted =
            launch(expert_count_kernel<Id>, chunks, kSortThreads, 0, stream, ids, total, chunk, experts, counts);
        if (counted != cudaSuccess) return counted;
    }
    return launch(expert_scatter_kernel<Id>, chunks, kSortThreads, kSortWarps * experts * sizeof(int32_t), stream, ids,
                  total, chunk, experts, chunks > 1 ? counts : nullptr, offsets, source, position);
}

template <typename T, int VEC>
cudaError_t gather_typed(const void *x, size_t x_stride, uint32_t tokens, uint32_t choices, uint32_t width,
                         const int32_t *position, const int32_t *end, void *rows, size_t rows_stride, int sm_count,
                         cudaStream_t stream) {
    const uint32_t packs = width / VEC;
    return launch(expert_gather_kernel<T, VEC>, row_blocks(static_cast<uint64_t>(tokens) * packs, sm_count), kRowThreads,
                  0, stream, static_cast<const T *>(x), x_stride, tokens, choices, packs, position, end,
                  static_cast<T *>(rows), rows_stride);
}

template <typename T, int VEC>
cudaError_t combine_typed(const void *rows, size_t rows_stride, uint32_t tokens, uint32_t choices, uint32_t width,
                          const int32_t *position, const float *weights, void *out, size_t out_stride, int sm_count,
                          cudaStream_t stream) {
    const uint32_t packs = width / VEC;
    const uint32_t blocks = row_blocks(static_cast<uint64_t>(tokens) * packs, sm_count);
    auto kernel = weights != nullptr ? expert_combine_kernel<T, VEC, true> : expert_combine_kernel<T, VEC, false>;
    return launch(kernel, blocks, kRowThreads, 0, stream, static_cast<const T *>(rows), rows_stride, tokens, choices,
                  packs, position, weights, static_cast<T *>(out), out_stride);
}

template <typename T, int VEC>
cudaError_t combine_backward_typed(const void *rows, size_t rows_stride, const void *grad, size_t grad_stride,
                                   uint32_t tokens, uint32_t choices, uint32_t width, const int32_t *position,
                                   const int32_t *end, const float *weights, void *grad_rows, size_t grad_rows_stride,
                                   float *grad_weights, int sm_count, cudaStream_t stream) {
    const uint32_t packs = width / VEC;
    uint32_t threads = 32;
    while (threads < kRowThreads && threads < packs) threads *= 2;
    const uint32_t most = static_cast<uint32_t>(sm_count) * 64u;
    return launch(expert_combine_backward_kernel<T, VEC>, tokens < most ? tokens : most, threads, 0, stream,
                  static_cast<const T *>(rows), rows_stride, static_cast<const T *>(grad), grad_stride, tokens, choices,
                  packs, position, end, weights, static_cast<T *>(grad_rows), grad_rows_stride, grad_weights);
}

// Calls f<T, VEC>(...) for the element type, 16-byte vectors where every row allows them.
#define QPUCUDA_ROWS_DISPATCH(f, type, vector, ...)                                          \
    switch (type) {                                                                          \
        case QPUCUDA_DTYPE_F32: return vector ? f<float, 4>(__VA_ARGS__) : f<float, 1>(__VA_ARGS__);             \
        case QPUCUDA_DTYPE_BF16:                                                             \
            return vector ? f<__nv_bfloat16, 8>(__VA_ARGS__) : f<__nv_bfloat16, 1>(__VA_ARGS__);                 \
        case QPUCUDA_DTYPE_F16: return vector ? f<__half, 8>(__VA_ARGS__) : f<__half, 1>(__VA_ARGS__);           \
    }                                                                                        \
    return cudaErrorInvalidValue

size_t item_bytes(int type) { return type == QPUCUDA_DTYPE_F32 ? 4 : 2; }

}  // namespace

size_t expert_sort_workspace(uint32_t tokens, uint32_t choices, uint32_t experts) {
    const uint64_t total = static_cast<uint64_t>(tokens) * choices;
    if (total == 0 || total > 0x7FFFFFFFull) return 0;
    const uint32_t chunk = sort_chunk(static_cast<uint32_t>(total));
    const uint32_t chunks = static_cast<uint32_t>((total + chunk - 1) / chunk);
    return chunks > 1 ? static_cast<size_t>(chunks) * experts * sizeof(int32_t) : 0;
}

cudaError_t launch_expert_sort(const void *ids, bool ids_64, uint32_t tokens, uint32_t choices, uint32_t experts,
                               int32_t *offsets, int32_t *source, int32_t *position, void *workspace, int sm_count,
                               cudaStream_t stream) {
    (void)sm_count;
    const uint32_t total = tokens * choices;
    int32_t *counts = static_cast<int32_t *>(workspace);
    return ids_64 ? sort_typed(static_cast<const long long *>(ids), total, experts, offsets, source, position, counts, stream)
                  : sort_typed(static_cast<const int32_t *>(ids), total, experts, offsets, source, position, counts, stream);
}

cudaError_t launch_expert_gather(const void *x, int type, size_t x_stride, uint32_t tokens, uint32_t choices,
                                 uint32_t width, const int32_t *position, const int32_t *offsets, uint32_t experts,
                                 void *rows, size_t rows_stride, int sm_count, cudaStream_t stream) {
    const size_t item = item_bytes(type);
    const bool vector = width * item % 16u == 0 && vector_rows(x, x_stride, item) && vector_rows(rows, rows_stride, item);
    QPUCUDA_ROWS_DISPATCH(gather_typed, type, vector, x, x_stride, tokens, choices, width, position, offsets + experts,
                          rows, rows_stride, sm_count, stream);
}

cudaError_t launch_expert_combine(const void *rows, int type, size_t rows_stride, uint32_t tokens, uint32_t choices,
                                  uint32_t width, const int32_t *position, const float *weights, void *out,
                                  size_t out_stride, int sm_count, cudaStream_t stream) {
    const size_t item = item_bytes(type);
    const bool vector = width * item % 16u == 0 && vector_rows(rows, rows_stride, item) && vector_rows(out, out_stride, item);
    QPUCUDA_ROWS_DISPATCH(combine_typed, type, vector, rows, rows_stride, tokens, choices, width, position, weights, out,
                          out_stride, sm_count, stream);
}

cudaError_t launch_expert_combine_backward(const void *rows, int type, size_t rows_stride, const void *grad,
                                           size_t grad_stride, uint32_t tokens, uint32_t choices, uint32_t width,
                                           const int32_t *position, const int32_t *offsets, uint32_t experts,
                                           const float *weights, void *grad_rows, size_t grad_rows_stride,
                                           float *grad_weights, int sm_count, cudaStream_t stream) {
    const size_t item = item_bytes(type);
    const bool vector = width * item % 16u == 0 && vector_rows(rows, rows_stride, item) &&
                        vector_rows(grad, grad_stride, item) && vector_rows(grad_rows, grad_rows_stride, item);
    QPUCUDA_ROWS_DISPATCH(combine_backward_typed, type, vector, rows, rows_stride, grad, grad_stride, tokens, choices,
                          width, position, offsets + experts, weights, grad_rows, grad_rows_stride, grad_weights,
                          sm_count, stream);
}

}  // namespace qpucuda
