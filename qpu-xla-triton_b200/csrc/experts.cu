// Tokens sorted by expert and back (include/qpucuda_experts.h).
//
// The sort is a stable counting sort in integers. A choice's row is
//   offsets[e] + (choices of e in earlier chunks) + (in earlier warps of its chunk) + (earlier in its warp),
// every term an exact count, so the order never depends on timing. Up to 32768 choices (a prompt of
// 4096 tokens with 8 choices) it is one launch of one cluster, whose CTAs read each other's counts in
// distributed shared memory; above, a kernel counts the chunks first. Its time is latency: 16384
// choices of 32 experts about 6 us, 160000 of 128 about 12.
//
// Moving the rows is bound by HBM: each kernel reads a token's vector once, in registers, for all of
// its choices, and writes each row once. 20000 tokens x 8 choices of 2048 bf16: copies 124 us (5.9
// TB/s of the 738 MB), sums 116 us (6.4 TB/s), gradients of the sums 227 us (6.1 TB/s); 6.56 TB/s is the
// measured copy.
#include "element.cuh"
#include "qpucuda_fp8_internal.h"
#include "qpucuda_internal.h"
#include "sm100_fp8.cuh"

namespace qpucuda {
namespace {

// ---- sort -----------------------------------------------------------------------------------

constexpr int kSortThreads = 512;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortAhead = 8;
// A chunk is one CTA's share. Up to kSortCluster CTAs of one cluster share kSortCluster * kSortChunk
// choices, whose ranks stay in registers; above, the CTAs of a grid each add up the counts of all
// chunks, at most kSortMaxChunks of them, and rank their choices a second time.
constexpr uint32_t kSortChunk = 4096;
constexpr uint32_t kSortCluster = 8;
constexpr uint32_t kSortMaxChunks = 64;
constexpr uint32_t kMaxExperts = QPUCUDA_MAX_EXPERTS;
static_assert(kSortChunk == kSortThreads * kSortAhead, "a cluster's choices stay in registers");

bool sort_in_cluster(uint32_t total) { return total <= kSortCluster * kSortChunk; }

uint32_t sort_chunk(uint32_t total) {
    const uint32_t parts = sort_in_cluster(total) ? kSortCluster : kSortMaxChunks;
    const uint32_t chunk = (total + parts - 1) / parts;
    return (chunk == 0 ? 1 : (chunk + kSortThreads - 1) / kSortThreads) * kSortThreads;
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

// Whole warp: the order of each lane's choice among the warp's choices of its expert so far, counted
// on in `own`.
__device__ __forceinline__ int32_t rank_in_warp(int32_t *own, uint32_t e, uint32_t experts, uint32_t lane) {
    const uint32_t same = __match_any_sync(0xFFFFFFFFu, e);
    const uint32_t earlier = __popc(same & ((1u << lane) - 1u));
    int32_t rank = 0;
    if (e < experts) rank = own[e] + static_cast<int32_t>(earlier);
    __syncwarp();
    if (e < experts && earlier == 0) own[e] += __popc(same);
    __syncwarp();
    return rank;
}

// Rows of one chunk per CTA. CLUSTER: the grid is one cluster, whose CTAs publish their chunk's
// counts in shared memory behind `next`. Otherwise counts: [gridDim.x][experts].
template <typename Id, bool CLUSTER>
__global__ void __launch_bounds__(kSortThreads) expert_scatter_kernel(const Id *__restrict__ ids, uint32_t total,
                                                                      uint32_t chunk, uint32_t experts,
                                                                      const int32_t *counts, int32_t *offsets,
                                                                      int32_t *source, int32_t *position) {
    extern __shared__ int32_t next[];  // [kSortWarps + 1][experts]: counts, then the first row of (warp, expert)
    __shared__ int32_t warp_sums[kSortWarps];
    __shared__ int32_t kept;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t warp = threadIdx.x / 32u, lane = threadIdx.x & 31u;
    const uint32_t begin = blockIdx.x * chunk;
    const uint32_t end = min(total, begin + chunk);
    const uint32_t share = chunk / kSortWarps;  // a multiple of 32
    const uint32_t warp_begin = begin + warp * share;
    const uint32_t warp_end = min(end, warp_begin + share);
    int32_t *own = next + warp * experts;
    uint32_t e[kSortAhead];
    int32_t rank[kSortAhead];
    // kSortAhead steps of 32 ids are loaded before the first is used.
    auto load = [&](uint32_t i0) {
#pragma unroll
        for (int a = 0; a < kSortAhead; ++a) e[a] = expert_of(ids, i0 + 32 * a + lane, warp_end, experts);
    };
    if (CLUSTER) load(warp_begin);
    for (uint32_t i = threadIdx.x; i < kSortWarps * experts; i += kSortThreads) next[i] = 0;
    __syncthreads();
    if (CLUSTER) {
#pragma unroll
        for (int a = 0; a < kSortAhead; ++a)
            if (32u * a < share) rank[a] = rank_in_warp(own, e[a], experts, lane);
    } else {
        for (uint32_t i0 = warp_begin; i0 < warp_end; i0 += 32 * kSortAhead) {
            load(i0);
#pragma unroll
            for (int a = 0; a < kSortAhead; ++a)
                if (e[a] < experts) atomicAdd(&own[e[a]], 1);
        }
    }
    __syncthreads();
    // Thread t takes experts 2t and 2t + 1: their counts over this chunk's warps become offsets
    // inside the chunk, their totals over all chunks are scanned into the experts' first rows.
    int32_t in_all[2], before[2];
    int32_t *published = next + kSortWarps * experts;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const uint32_t x = 2u * threadIdx.x + s;
        in_all[s] = before[s] = 0;
        if (x < experts) {
            int32_t count[kSortWarps], in_chunk = 0;
#pragma unroll
            for (int w = 0; w < kSortWarps; ++w) count[w] = next[w * experts + x];
#pragma unroll
            for (int w = 0; w < kSortWarps; ++w) {
                next[w * experts + x] = in_chunk;
                in_chunk += count[w];
            }
            in_all[s] = in_chunk;
            if (CLUSTER) published[x] = in_chunk;
        }
    }
    if (gridDim.x > 1) {
        if (CLUSTER) sm100::cluster_sync();
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const uint32_t x = 2u * threadIdx.x + s;
            if (x < experts) {
                int32_t sum = 0;
                for (uint32_t c0 = 0; c0 < gridDim.x; c0 += kSortCluster) {
                    int32_t count[kSortCluster];
#pragma unroll
                    for (uint32_t c = 0; c < kSortCluster; ++c) {
                        count[c] = 0;
                        if (c0 + c < gridDim.x)
                            count[c] = CLUSTER ? sm100::load_cluster_s32(sm100::map_to_rank(sm100::smem_u32(published + x), c0 + c))
                                               : counts[static_cast<size_t>(c0 + c) * experts + x];
                    }
#pragma unroll
                    for (uint32_t c = 0; c < kSortCluster; ++c) {
                        if (c0 + c == blockIdx.x) before[s] = sum;
                        sum += count[c];
                    }
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
        const uint32_t x = 2u * threadIdx.x + s;
        if (x < experts) {
#pragma unroll
            for (int w = 0; w < kSortWarps; ++w) next[w * experts + x] += first + before[s];
            if (blockIdx.x == 0) offsets[x] = first;
        }
        first += in_all[s];
    }
    __syncthreads();
    if (blockIdx.x == 0 && threadIdx.x == 0) offsets[experts] = kept;
    auto place = [&](uint32_t i, int32_t row) {
        if (i < warp_end) {
            position[i] = row;
            if (row >= 0) source[row] = static_cast<int32_t>(i);
        }
    };
    if (CLUSTER) {
#pragma unroll
        for (int a = 0; a < kSortAhead; ++a)
            if (32u * a < share) place(warp_begin + 32 * a + lane, e[a] < experts ? own[e[a]] + rank[a] : -1);
    } else {
        for (uint32_t i0 = warp_begin; i0 < warp_end; i0 += 32 * kSortAhead) {
            load(i0);
#pragma unroll
            for (int a = 0; a < kSortAhead; ++a) {
                const int32_t row = rank_in_warp(own, e[a], experts, lane);
                place(i0 + 32 * a + lane, e[a] < experts ? row : -1);
            }
        }
    }
    const uint32_t stride = gridDim.x * kSortThreads;
    for (uint32_t row = static_cast<uint32_t>(kept) + blockIdx.x * kSortThreads + threadIdx.x; row < total; row += stride)
        source[row] = -1;
    if (CLUSTER && gridDim.x > 1) sm100::cluster_sync();  // no CTA ends while another reads its counts
}

// ---- rows -------------------------------------------------------------------------------------

constexpr int kRowThreads = 256;

// The elements of a row that one thread moves: kVector<T> of them, 16 bytes. Where every base and row
// stride is a multiple of 16 bytes (ALIGNED) they are contiguous and move as one; otherwise they are
// 32 apart, so that a warp's loads and stores of single elements stay contiguous.
template <typename T, bool ALIGNED>
struct Columns {
    uint32_t first, width;

    // packs of a row; a warp never crosses the row's end when elements are 32 apart
    static uint32_t packs(uint32_t width) {
        constexpr uint32_t kItems = kVector<T>;
        return ALIGNED ? width / kItems : (width + 32 * kItems - 1) / (32 * kItems) * 32;
    }
    __device__ __forceinline__ Columns(uint32_t pack, uint32_t width_)
        : first(ALIGNED ? pack * kVector<T> : pack / 32 * (32 * kVector<T>) + pack % 32), width(width_) {}

    __device__ __forceinline__ void load(const T *row, Vector<T> &v) const {
        if constexpr (ALIGNED) {
            v.bits = load_stream16(row + first);
        } else {
#pragma unroll
            for (int i = 0; i < kVector<T>; ++i) {
                v.items[i] = from_float<T>(0.0f);
                if (first + 32 * i < width) v.items[i] = __ldg(row + first + 32 * i);
            }
        }
    }
    __device__ __forceinline__ void store(T *row, const Vector<T> &v) const {
        if constexpr (ALIGNED) {
            *reinterpret_cast<uint4 *>(row + first) = v.bits;
        } else {
#pragma unroll
            for (int i = 0; i < kVector<T>; ++i)
                if (first + 32 * i < width) row[first + 32 * i] = v.items[i];
        }
    }
};

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
template <typename T, bool ALIGNED>
__device__ __forceinline__ void zero_tail(T *rows, size_t stride, uint32_t count, uint32_t width, uint32_t packs, const int32_t *end) {
    const int32_t raw = *end;
    const uint32_t first = raw < 0 ? 0u : min(static_cast<uint32_t>(raw), count);
    const uint64_t total = static_cast<uint64_t>(count - first) * packs;
    const uint64_t step = static_cast<uint64_t>(gridDim.x) * blockDim.x;
    Vector<T> zero;
    zero.bits = make_uint4(0, 0, 0, 0);
    for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += step) {
        uint32_t row, pack;
        split_index(i, total, packs, row, pack);
        Columns<T, ALIGNED>(pack, width).store(rows + static_cast<size_t>(first + row) * stride, zero);
    }
}

// A token's choices are taken kAhead at a time: their rows are known, and where they are read also
// loaded, before the first is used.
constexpr int kAhead = 4;

// The row of choice j0 + a, or `count` (no row) when it is dropped or there is none.
__device__ __forceinline__ void choice_rows(const int32_t *position, uint32_t j0, uint32_t choices, uint32_t count, uint32_t (&row)[kAhead]) {
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
        const uint32_t at = j0 + a < choices ? static_cast<uint32_t>(__ldg(position + j0 + a)) : count;  // -1 is out of range as well
        row[a] = min(at, count);
    }
}

template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kRowThreads) expert_gather_kernel(const T *__restrict__ x, size_t x_stride,
                                                                    uint32_t tokens, uint32_t choices, uint32_t width,
                                                                    uint32_t packs, const int32_t *__restrict__ position,
                                                                    const int32_t *end, T *rows, size_t rows_stride) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t count = tokens * choices;
    const uint64_t total = static_cast<uint64_t>(tokens) * packs;
    const uint64_t step = static_cast<uint64_t>(gridDim.x) * kRowThreads;
    for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * kRowThreads + threadIdx.x; i < total; i += step) {
        uint32_t token, pack;
        split_index(i, total, packs, token, pack);
        const Columns<T, ALIGNED> columns(pack, width);
        Vector<T> value;
        columns.load(x + static_cast<size_t>(token) * x_stride, value);
        const int32_t *at = position + static_cast<size_t>(token) * choices;
        for (uint32_t j0 = 0; j0 < choices; j0 += kAhead) {
            uint32_t row[kAhead];
            choice_rows(at, j0, choices, count, row);
#pragma unroll
            for (int a = 0; a < kAhead; ++a)
                if (row[a] < count) columns.store(rows + static_cast<size_t>(row[a]) * rows_stride, value);
        }
    }
    zero_tail<T, ALIGNED>(rows, rows_stride, count, width, packs, end);
}

// out[t] = sum_j w[t, j] rows[position[t, j]]: fp32 in the order of j, rounded once.
template <typename T, bool ALIGNED, bool WEIGHTED>
__global__ void __launch_bounds__(kRowThreads) expert_combine_kernel(const T *__restrict__ rows, size_t rows_stride,
                                                                     uint32_t tokens, uint32_t choices, uint32_t width,
                                                                     uint32_t packs, const int32_t *__restrict__ position,
                                                                     const float *__restrict__ weights, T *out,
                                                                     size_t out_stride) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t count = tokens * choices;
    const uint64_t total = static_cast<uint64_t>(tokens) * packs;
    const uint64_t step = static_cast<uint64_t>(gridDim.x) * kRowThreads;
    for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * kRowThreads + threadIdx.x; i < total; i += step) {
        uint32_t token, pack;
        split_index(i, total, packs, token, pack);
        const Columns<T, ALIGNED> columns(pack, width);
        const size_t at = static_cast<size_t>(token) * choices;
        float sum[kVector<T>];
#pragma unroll
        for (int v = 0; v < kVector<T>; ++v) sum[v] = 0.0f;
        for (uint32_t j0 = 0; j0 < choices; j0 += kAhead) {
            uint32_t row[kAhead];
            choice_rows(position + at, j0, choices, count, row);
            Vector<T> value[kAhead];
            float weight[kAhead];
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                weight[a] = 1.0f;
                if (row[a] < count) {
                    columns.load(rows + static_cast<size_t>(row[a]) * rows_stride, value[a]);
                    if (WEIGHTED) weight[a] = __ldg(weights + at + j0 + a);
                }
            }
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                if (row[a] >= count) continue;
#pragma unroll
                for (int v = 0; v < kVector<T>; ++v) {
                    const float x = to_float(value[a].items[v]);
                    sum[v] = WEIGHTED ? fmaf(weight[a], x, sum[v]) : sum[v] + x;
                }
            }
        }
        Vector<T> result;
#pragma unroll
        for (int v = 0; v < kVector<T>; ++v) result.items[v] = from_float<T>(sum[v]);
        columns.store(out + static_cast<size_t>(token) * out_stride, result);
    }
}

// One CTA per token: grad[t] is read once per kAhead choices, each choice's row once; its dot
// product with grad[t] is summed per thread, then over the CTA in a fixed order.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kRowThreads)
    expert_combine_backward_kernel(const T *__restrict__ rows, size_t rows_stride, const T *__restrict__ grad,
                                   size_t grad_stride, uint32_t tokens, uint32_t choices, uint32_t width, uint32_t packs,
                                   const int32_t *__restrict__ position, const int32_t *end,
                                   const float *__restrict__ weights, T *grad_rows, size_t grad_rows_stride,
                                   float *grad_weights) {
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
            choice_rows(position + at, j0, choices, count, row);
            float weight[kAhead], dot[kAhead];
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                weight[a] = row[a] < count ? __ldg(weights + at + j0 + a) : 0.0f;
                dot[a] = 0.0f;
            }
            for (uint32_t pack = threadIdx.x; pack < packs; pack += blockDim.x) {
                const Columns<T, ALIGNED> columns(pack, width);
                Vector<T> upstream, value[kAhead];
                columns.load(g, upstream);
#pragma unroll
                for (int a = 0; a < kAhead; ++a)
                    if (row[a] < count) columns.load(rows + static_cast<size_t>(row[a]) * rows_stride, value[a]);
#pragma unroll
                for (int a = 0; a < kAhead; ++a) {
                    if (row[a] >= count) continue;
                    Vector<T> scaled;
#pragma unroll
                    for (int v = 0; v < kVector<T>; ++v) {
                        const float u = to_float(upstream.items[v]);
                        dot[a] = fmaf(to_float(value[a].items[v]), u, dot[a]);
                        scaled.items[v] = from_float<T>(weight[a] * u);
                    }
                    columns.store(grad_rows + static_cast<size_t>(row[a]) * grad_rows_stride, scaled);
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
    zero_tail<T, ALIGNED>(grad_rows, grad_rows_stride, count, width, packs, end);
}

// ---- launches -----------------------------------------------------------------------------------

template <typename... Parameters, typename... Arguments>
cudaError_t launch(void (*kernel)(Parameters...), uint32_t blocks, uint32_t threads, size_t shared, uint32_t cluster,
                   cudaStream_t stream, Arguments... arguments) {
    cudaLaunchAttribute attributes[2] = {};
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = cluster;
    attributes[1].val.clusterDim.y = 1;
    attributes[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(blocks);
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = shared;
    config.stream = stream;
    config.attrs = attributes;
    config.numAttrs = cluster > 1 ? 2 : 1;
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
    constexpr size_t kTable = (kSortWarps + 1) * sizeof(int32_t);  // per expert
    static PerDeviceOnce configured;
    const cudaError_t error = configured.run([] {
        const int bytes = static_cast<int>(kTable * kMaxExperts);
        const cudaError_t first = cudaFuncSetAttribute(expert_scatter_kernel<Id, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        return first != cudaSuccess
                   ? first
                   : cudaFuncSetAttribute(expert_scatter_kernel<Id, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    });
    if (error != cudaSuccess) return error;
    const uint32_t chunk = sort_chunk(total);
    const uint32_t chunks = total == 0 ? 1u : (total + chunk - 1) / chunk;
    if (sort_in_cluster(total)) {
        return launch(expert_scatter_kernel<Id, true>, chunks, kSortThreads, kTable * experts, chunks, stream, ids, total, chunk,
                      experts, nullptr, offsets, source, position);
    }
    const cudaError_t counted = launch(expert_count_kernel<Id>, chunks, kSortThreads, 0, 1, stream, ids, total, chunk, experts, counts);
    if (counted != cudaSuccess) return counted;
    return launch(expert_scatter_kernel<Id, false>, chunks, kSortThreads, kTable * experts, 1, stream, ids, total, chunk, experts,
                  counts, offsets, source, position);
}

template <typename T, bool ALIGNED>
cudaError_t gather_typed(const qpucuda_expert_rows_desc &d, int sm_count, cudaStream_t stream) {
    const uint32_t packs = Columns<T, ALIGNED>::packs(d.width);
    return launch(expert_gather_kernel<T, ALIGNED>, row_blocks(static_cast<uint64_t>(d.tokens) * packs, sm_count), kRowThreads,
                  0, 1, stream, static_cast<const T *>(d.source), d.source_stride, d.tokens, d.choices, d.width, packs,
                  d.position, d.offsets + d.experts, static_cast<T *>(d.out), d.out_stride);
}

template <typename T, bool ALIGNED>
cudaError_t combine_typed(const qpucuda_expert_rows_desc &d, int sm_count, cudaStream_t stream) {
    const uint32_t packs = Columns<T, ALIGNED>::packs(d.width);
    const uint32_t blocks = row_blocks(static_cast<uint64_t>(d.tokens) * packs, sm_count);
    auto kernel = d.weights != nullptr ? expert_combine_kernel<T, ALIGNED, true> : expert_combine_kernel<T, ALIGNED, false>;
    return launch(kernel, blocks, kRowThreads, 0, 1, stream, static_cast<const T *>(d.source), d.source_stride, d.tokens,
                  d.choices, d.width, packs, d.position, d.weights, static_cast<T *>(d.out), d.out_stride);
}

template <typename T, bool ALIGNED>
cudaError_t combine_backward_typed(const qpucuda_expert_rows_desc &d, int sm_count, cudaStream_t stream) {
    const uint32_t packs = Columns<T, ALIGNED>::packs(d.width);
    uint32_t threads = 32;
    while (threads < kRowThreads && threads < packs) threads *= 2;
    const uint32_t most = static_cast<uint32_t>(sm_count) * 64u;
    return launch(expert_combine_backward_kernel<T, ALIGNED>, d.tokens < most ? d.tokens : most, threads, 0, 1, stream,
                  static_cast<const T *>(d.source), d.source_stride, static_cast<const T *>(d.grad), d.grad_stride, d.tokens,
                  d.choices, d.width, packs, d.position, d.offsets + d.experts, d.weights, static_cast<T *>(d.out), d.out_stride,
                  d.grad_weights);
}

// Calls f<T, ALIGNED>(...) for the element type.
#define QPUCUDA_ROWS_DISPATCH(f, type, aligned, ...)                                                              \
    switch (type) {                                                                                               \
        case QPUCUDA_DTYPE_F32: return aligned ? f<float, true>(__VA_ARGS__) : f<float, false>(__VA_ARGS__);      \
        case QPUCUDA_DTYPE_BF16:                                                                                  \
            return aligned ? f<__nv_bfloat16, true>(__VA_ARGS__) : f<__nv_bfloat16, false>(__VA_ARGS__);          \
        case QPUCUDA_DTYPE_F16: return aligned ? f<__half, true>(__VA_ARGS__) : f<__half, false>(__VA_ARGS__);    \
    }                                                                                                             \
    return cudaErrorInvalidValue

size_t item_bytes(int type) { return type == QPUCUDA_DTYPE_F32 ? 4 : 2; }

bool vector_moves(const qpucuda_expert_rows_desc &desc) {
    const size_t item = item_bytes(desc.type);
    return desc.width * item % 16u == 0 && vector_rows(desc.source, desc.source_stride, item) &&
           vector_rows(desc.out, desc.out_stride, item);
}

}  // namespace

size_t expert_sort_workspace(uint32_t tokens, uint32_t choices, uint32_t experts) {
    const uint64_t total = static_cast<uint64_t>(tokens) * choices;
    if (total == 0 || total > 0x7FFFFFFFull) return 0;
    if (sort_in_cluster(static_cast<uint32_t>(total))) return 0;
    const uint32_t chunk = sort_chunk(static_cast<uint32_t>(total));
    return static_cast<size_t>((total + chunk - 1) / chunk) * experts * sizeof(int32_t);
}

cudaError_t launch_expert_sort(const qpucuda_expert_sort_desc &d, cudaStream_t stream) {
    const uint32_t total = d.tokens * d.choices;
    int32_t *counts = static_cast<int32_t *>(d.workspace);
    return d.ids_64 != 0
               ? sort_typed(static_cast<const long long *>(d.ids), total, d.experts, d.offsets, d.source, d.position, counts, stream)
               : sort_typed(static_cast<const int32_t *>(d.ids), total, d.experts, d.offsets, d.source, d.position, counts, stream);
}

cudaError_t launch_expert_gather(const qpucuda_expert_rows_desc &given, int sm_count, cudaStream_t stream) {
    // A copy, whatever the elements: pairs of 16-bit ones move as one of 32 bits where they may (4096 x 4 of
    // 2046 bf16, in a captured graph 11 us, 15 one by one).
    qpucuda_expert_rows_desc desc = given;
    if (desc.type != QPUCUDA_DTYPE_F32) {
        const uint64_t either = reinterpret_cast<uintptr_t>(desc.source) / 2 | reinterpret_cast<uintptr_t>(desc.out) / 2 | desc.width |
                                desc.source_stride | desc.out_stride;
        if (either % 2 != 0) return gather_typed<__nv_bfloat16, false>(desc, sm_count, stream);
        desc.type = QPUCUDA_DTYPE_F32;
        desc.width /= 2;
        desc.source_stride /= 2;
        desc.out_stride /= 2;
    }
    return vector_moves(desc) ? gather_typed<float, true>(desc, sm_count, stream) : gather_typed<float, false>(desc, sm_count, stream);
}

cudaError_t launch_expert_combine(const qpucuda_expert_rows_desc &desc, int sm_count, cudaStream_t stream) {
    QPUCUDA_ROWS_DISPATCH(combine_typed, desc.type, vector_moves(desc), desc, sm_count, stream);
}

cudaError_t launch_expert_combine_backward(const qpucuda_expert_rows_desc &desc, int sm_count, cudaStream_t stream) {
    const bool aligned = vector_moves(desc) && vector_rows(desc.grad, desc.grad_stride, item_bytes(desc.type));
    QPUCUDA_ROWS_DISPATCH(combine_backward_typed, desc.type, aligned, desc, sm_count, stream);
}

}  // namespace qpucuda
