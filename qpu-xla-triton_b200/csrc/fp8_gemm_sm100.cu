// Block-scaled FP8 product for sm_100a: y[m, n] = sum_b sx[m, b] sw[n / 128, b] p[m, n, b] (+ bias[n]),
// p[m, n, b] the e4m3 dot product over the 128 columns of block b, accumulated in fp32 by
// tcgen05.mma (kind::f8f6f4). The scales are arbitrary fp32, so p leaves tensor memory after every
// block and is added to fp32 registers as fma(p, sx * sw, acc): two roundings of a factor and one of
// the sum per block.
//
// With experts, the rows [offsets[e], offsets[e + 1]) meet matrix e. Tiles are cut inside an
// expert's rows; the rows of the next expert that a tile's copy also brings in are computed and
// not stored, the rows no expert owns are zeroed.
//
// Two kernels. A few rows per matrix are bound by the weight's bytes (narrow); many by the tensor
// cores and, at one multiply-add per product of 128 columns beside them, by the board's power (wide).
#include <algorithm>
#include <atomic>
#include <cstring>
#include <type_traits>

#include "fp8_quantize.cuh"
#include "qpucuda_fp8_internal.h"
#include "qpucuda_internal.h"
#include "sm100_fp8.cuh"

namespace qpucuda {
namespace {

using namespace sm100;

constexpr int kBlockN = 128;  // output columns (weight rows) per tile = one row of weight scales
constexpr int kBlockK = 128;  // columns per stage = one scale group = one swizzle row
constexpr int kMmaK = 32;     // columns per tcgen05.mma kind::f8f6f4
constexpr uint32_t kMaxSplit = 8;

struct GemmParams {
    uint32_t rows, n, k;
    uint32_t k_blocks, n_blocks;
    uint32_t experts;  // 0: one matrix
    const int32_t *offsets;
    const float *a_scales;
    size_t a_scale_row_stride, a_scale_group_stride;
    const float *w_scales;
    const float *bias;
    void *out;
    size_t out_stride;
    uint32_t weights_settled;
    uint32_t tma_store;  // the output's rows can be written by the copy engine
    unsigned int *error_word;
};

// Rows that the product quantizes itself.
struct FusedRows {
    const void *x;
    size_t stride;
    int type;
    uint32_t gated;
    uint32_t vector;  // rows and, gated, their second halves allow 16-byte loads
};

// The rows of one tile: [row0, row_end) of matrix `expert`, at most the tile's height of them.
struct Tile {
    uint32_t expert, row0, row_end;
    bool valid;
};

// Whole warp. Tile number `slot` among the tiles of `height` rows cut inside every expert's rows.
// Offsets that do not ascend within [0, rows] are clamped, so every tile stays inside the rows.
__device__ __forceinline__ Tile find_tile(const GemmParams &params, uint32_t height, uint32_t slot, uint32_t lane) {
    Tile tile{0, 0, 0, false};
    if (params.experts == 0) {
        tile.row0 = slot * height;
        tile.row_end = min(params.rows, tile.row0 + height);
        tile.valid = tile.row0 < params.rows;
        return tile;
    }
    const int32_t rows = static_cast<int32_t>(params.rows);
    for (uint32_t e0 = 0; e0 < params.experts; e0 += 32) {
        const uint32_t e = e0 + lane;
        int32_t begin = 0, end = 0;
        if (e < params.experts) {
            begin = min(max(params.offsets[e], 0), rows);
            end = min(max(params.offsets[e + 1], begin), rows);
        }
        const uint32_t tiles = (static_cast<uint32_t>(end - begin) + height - 1) / height;
        uint32_t through = tiles;
#pragma unroll
        for (int offset = 1; offset < 32; offset <<= 1) {
            const uint32_t other = __shfl_up_sync(0xFFFFFFFFu, through, offset);
            if (lane >= static_cast<uint32_t>(offset)) through += other;
        }
        const uint32_t holders = __ballot_sync(0xFFFFFFFFu, slot < through);
        if (holders != 0) {
            const int holder = __ffs(static_cast<int>(holders)) - 1;
            const uint32_t inside = slot - (__shfl_sync(0xFFFFFFFFu, through, holder) - __shfl_sync(0xFFFFFFFFu, tiles, holder));
            tile.expert = e0 + holder;
            tile.row0 = static_cast<uint32_t>(__shfl_sync(0xFFFFFFFFu, begin, holder)) + inside * height;
            tile.row_end = min(static_cast<uint32_t>(__shfl_sync(0xFFFFFFFFu, end, holder)), tile.row0 + height);
            tile.valid = true;
            return tile;
        }
        slot -= __shfl_sync(0xFFFFFFFFu, through, 31);
    }
    return tile;
}

// First row that no expert owns.
__device__ __forceinline__ uint32_t owned_rows(const GemmParams &params) {
    if (params.experts == 0) return params.rows;
    return static_cast<uint32_t>(min(max(params.offsets[params.experts], 0), static_cast<int32_t>(params.rows)));
}

// ---- the narrow kernel ------------------------------------------------------------------------

// Few rows: the weight is the M = 128 operand and NT rows are the N operand, so they cost a tile of NT =
// 16 or 32 and not 128. Tensor memory lane = output column, tensor memory column = row. Two CTAs an SM
// keep 2 x 5 stages of 16 KB of weights under way. 4 x 28672 x 8192: 42 us back to back, 235 MB read
// once (5.6 TB/s, 0.85 of the measured copy). NT = 64 and 128 were slower than the wide kernel or than
// NT = 32 twice (64 x 11008 x 4096: 23 us at 64, 19 at 32).
//
// A few rows of a small matrix are quantized by the product itself: every CTA those of its K blocks,
// at most kFusedBlocks, into shared memory, while its first weights arrive. One launch instead of two
// (1 x 2048 x 2048 bf16: 14.4 -> 12.4 us a call, 5.3 -> 4.4 in a captured graph), as long as its four
// warps are done in three steps each (4 x 2048 x 5632, three steps: 7.5 -> 6.9 us in a graph; 16 x 2048
// x 2048, four: 6.0 -> 6.4).
constexpr uint32_t kFusedBlocks = 8;
constexpr uint32_t kFusedSteps = 3;

template <int NT, bool FUSED>
struct Narrow {
    static constexpr int kWarps = 4;  // epilogue: one per lane quarter
    static constexpr int kThreads = 64 + 32 * kWarps;
    static constexpr int kCtasPerSm = 2;
    static constexpr int kWBytes = kBlockN * kBlockK;
    static constexpr int kXBytes = NT * kBlockK;
    static constexpr int kStageBytes = kWBytes + (FUSED ? 0 : kXBytes);
    static constexpr int kFusedBytes = FUSED ? static_cast<int>(kFusedBlocks) * (kXBytes + NT * 4) : 0;  // values, then scales
    static constexpr int kStages = 5;
    static constexpr int kBuffers = 4;  // tensor memory accumulators
    static constexpr int kTmemColumns = kBuffers * NT;      // a power of two
    static constexpr int kScaleFloats = 2 * NT;             // per warp: this block's and the next's
    // Other CTAs' sums arrive in memory of their own, as long as they want, where there is room for it.
    static constexpr bool kOwnSums = NT == 16;
    static constexpr int kSumBytes = kOwnSums ? NT * kBlockN * 4 : 0;
    static constexpr size_t kSharedBytes =
        static_cast<size_t>(kStages) * kStageBytes + kFusedBytes + kSumBytes + kWarps * kScaleFloats * sizeof(float) + 1024 + 256;
    static_assert(kTmemColumns * kCtasPerSm <= 512, "tensor memory");
    static_assert(kSharedBytes * kCtasPerSm + 2048 <= 227 * 1024, "shared memory");
    static_assert(static_cast<size_t>(NT) * kBlockN * 4 <= static_cast<size_t>(kStages) * kStageBytes, "split sums");
};

// Groups of this CTA's rows and K blocks, `items` of them, quantized by four warps: group i is row
// i / blocks, block i % blocks. Values go to `values` in the MMA's layout ([block][row] of 128 bytes,
// 128-byte swizzle), scales to scales[block * NT + row].
template <typename T, bool GATED, int NT>
__device__ __forceinline__ void fuse_rows(const FusedRows &rows, const GemmParams &params, uint32_t row0, uint32_t items,
                                          uint32_t kb_begin, uint32_t blocks, uint8_t *values, float *scales, uint32_t worker,
                                          uint32_t lane) {
    constexpr int kLanes = 128 / kVector<T>;
    constexpr uint32_t kPerStep = 32 / kLanes;
    const uint32_t inner = lane % kLanes * kVector<T>;
    for (uint32_t first = worker * kPerStep; first < items; first += 4 * kPerStep) {
        const uint32_t item = first + lane / kLanes;
        const bool present = item < items;
        const uint32_t row = present ? item / blocks : 0u, block = present ? item % blocks : 0u;
        const uint32_t column = (kb_begin + block) * kBlockK + inner;
        const T *x = static_cast<const T *>(rows.x) + static_cast<size_t>(row0 + row) * rows.stride + column;
        const uint32_t remaining = present && column < params.k ? params.k - column : 0u;
        Vector<T> raw[1], raw_up[1];
        if (rows.vector != 0) {
            load_steps<T, true>(x, remaining, 128u, raw);
            if (GATED) load_steps<T, true>(x + params.k, remaining, 128u, raw_up);
        } else {
            load_steps<T, false>(x, remaining, 128u, raw);
            if (GATED) load_steps<T, false>(x + params.k, remaining, 128u, raw_up);
        }
        float v[kVector<T>], amax = 0.0f;
#pragma unroll
        for (int i = 0; i < kVector<T>; ++i) v[i] = to_float(raw[0].items[i]);
        if constexpr (GATED) {
            float up[kVector<T>];
#pragma unroll
            for (int i = 0; i < kVector<T>; ++i) up[i] = to_float(raw_up[0].items[i]);
            silu_times(v, up);
        }
#pragma unroll
        for (int i = 0; i < kVector<T>; ++i) amax = max_nan(amax, fabsf(v[i]));
        const float scale = group_scale(group_max<kLanes>(amax));
        uint32_t packed[kVector<T> / 4];
        quantize_values(v, scale, packed);
        if (present) {
            uint8_t *q = values + (block * NT + row) * 128u + (((inner >> 4) ^ (row & 7u)) << 4) + (inner & 15u);
            if constexpr (kVector<T> == 8) {
                *reinterpret_cast<uint2 *>(q) = make_uint2(packed[0], packed[kVector<T> / 4 - 1]);
            } else {
                *reinterpret_cast<uint32_t *>(q) = packed[0];
            }
            if (lane % kLanes == 0) scales[block * NT + row] = scale;
        }
    }
}

template <int STAGES, int BUFFERS>
struct Control {
    uint64_t full[STAGES];
    uint64_t empty[STAGES];
    uint64_t tmem_full[BUFFERS];
    uint64_t tmem_empty[BUFFERS];
    uint64_t drain;
    uint64_t rows_ready;  // the product's own quantized rows are in place
    uint32_t tmem_base;
    volatile int abort_flag;
    uint32_t copies;      // stages that warp 0's first thread has set under way
    uint32_t multiplied;  // warp 1's has issued an MMA
};

// Parity of the phase that the last of `issued` copies into `stage` completes, the stages taken in turn.
__host__ __device__ constexpr uint32_t last_phase(uint32_t issued, uint32_t stage, uint32_t stages) {
    return ((issued - stage + stages - 1) / stages - 1) & 1u;
}
static_assert(last_phase(1, 0, 5) == 0 && last_phase(5, 4, 5) == 0 && last_phase(6, 0, 5) == 1 && last_phase(6, 1, 5) == 0 &&
                  last_phase(10, 4, 5) == 1 && last_phase(11, 0, 5) == 0 && last_phase(11, 1, 5) == 1,
              "stages 0 to issued - 1, each pass of the ring the other parity");

// A wait of this CTA ran out, in whichever warp: no role takes another step, but the copies and the MMAs that
// were issued must end before the CTA gives up its memory, also where the warp that issued them had nothing
// left to wait for. Each by the thread that issued them; the waits are bounded.
template <int STAGES>
__device__ __forceinline__ void drain_copies(uint64_t *full, uint32_t issued) {
    for (uint32_t s = 0; s < STAGES && s < issued; ++s) wait_drain(smem_u32(&full[s]), last_phase(issued, s, STAGES));
}
template <bool PAIR>
__device__ __forceinline__ void drain_mmas(uint64_t *drain) {
    if constexpr (PAIR) {
        mma_commit_pair_local(smem_u32(drain));
    } else {
        mma_commit(smem_u32(drain));
    }
    wait_drain(smem_u32(drain), 0);
}

// Grid: x = column block * split + rank in the cluster, y = tile of rows. The CTAs of a cluster
// share a tile and split its K blocks; their sums meet in distributed shared memory in rank order,
// so the result does not depend on timing.
//   warp 0   copies: a weight and a row box per stage
//   warp 1   tensor memory and MMA: 4 MMAs per stage into the next of kBuffers accumulators
//   others   each block's accumulator into registers, scaled; then the sums over the cluster, the store
template <int NT, bool FUSED, typename Out>
__global__ void __launch_bounds__(Narrow<NT, FUSED>::kThreads, Narrow<NT, FUSED>::kCtasPerSm)
    fp8_gemm_narrow_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a,
                           const GemmParams params, const FusedRows fused) {
    using Shape = Narrow<NT, FUSED>;
    using Ctl = Control<Shape::kStages, Shape::kBuffers>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *stage_w = smem;
    uint8_t *stage_x = smem + Shape::kStages * Shape::kWBytes;  // FUSED: one tile per K block of this CTA
    float *fused_scales = reinterpret_cast<float *>(stage_x + kFusedBlocks * Shape::kXBytes);
    float *sums = reinterpret_cast<float *>(Shape::kOwnSums ? smem + Shape::kStages * Shape::kStageBytes + Shape::kFusedBytes : smem);
    float *scale_rows = reinterpret_cast<float *>(smem + Shape::kStages * Shape::kStageBytes + Shape::kFusedBytes + Shape::kSumBytes);
    Ctl *control = reinterpret_cast<Ctl *>(scale_rows + Shape::kWarps * Shape::kScaleFloats);
    static_assert(sizeof(Ctl) <= 256, "control block");

    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t split = cluster_size();  // a power of two
    const uint32_t split_shift = __ffs(static_cast<int>(split)) - 1;
    const uint32_t rank = cluster_rank();
    const uint32_t n_block = blockIdx.x / split;
    const uint32_t n0 = n_block * kBlockN;

    if (threadIdx.x == 0) {
        for (int s = 0; s < Shape::kStages; ++s) {
            mbar_init(smem_u32(&control->full[s]), 1);
            mbar_init(smem_u32(&control->empty[s]), 1);
        }
        for (int b = 0; b < Shape::kBuffers; ++b) {
            mbar_init(smem_u32(&control->tmem_full[b]), 1);
            mbar_init(smem_u32(&control->tmem_empty[b]), Shape::kWarps);
        }
        mbar_init(smem_u32(&control->drain), 1);
        mbar_init(smem_u32(&control->rows_ready), 1);
        control->abort_flag = 0;
        control->copies = control->multiplied = 0;
        mbar_init_fence();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&control->tmem_base)),
                     "r"(Shape::kTmemColumns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (Shape::kOwnSums && split > 1) cluster_arrive();  // this CTA's memory may be written from now on
    const uint32_t tmem_base = control->tmem_base;
    const bool early = params.weights_settled != 0;
    // Weights and offsets that the previous kernel does not write are read before it has finished;
    // the rows, and every store, wait for it.
    if (!early) asm volatile("griddepcontrol.wait;" ::: "memory");
    const Tile tile = find_tile(params, NT, blockIdx.y, lane);
    const uint32_t kb_begin = static_cast<uint32_t>(static_cast<uint64_t>(params.k_blocks) * rank / split);
    const uint32_t kb_end = static_cast<uint32_t>(static_cast<uint64_t>(params.k_blocks) * (rank + 1) / split);
    const int row0 = static_cast<int>(tile.row0);

    if (!tile.valid) {
        if (early) asm volatile("griddepcontrol.wait;" ::: "memory");
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    } else if (warp == 0) {
        if (lane == 0) {
            prefetch_tensor_map(&map_w);
            if (!FUSED) prefetch_tensor_map(&map_a);
            const int w_row = static_cast<int>(tile.expert * params.n + n0);
            auto load_w = [&](uint32_t kb, uint32_t stage) {
                const uint32_t full = smem_u32(&control->full[stage]);
                mbar_expect_tx(full, Shape::kStageBytes);
                tma_load_2d(smem_u32(stage_w + stage * Shape::kWBytes), &map_w, full, static_cast<int>(kb * kBlockK), w_row);
            };
            auto load_x = [&](uint32_t kb, uint32_t stage) {
                if (FUSED) return;
                tma_load_2d(smem_u32(stage_x + stage * Shape::kXBytes), &map_a, smem_u32(&control->full[stage]),
                            static_cast<int>(kb * kBlockK), row0);
            };
            const uint32_t count = kb_end - kb_begin;
            const uint32_t ahead = min(count, static_cast<uint32_t>(Shape::kStages));
            for (uint32_t s = 0; s < ahead; ++s) load_w(kb_begin + s, s);
            if (early) asm volatile("griddepcontrol.wait;" ::: "memory");
            asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
            for (uint32_t s = 0; s < ahead; ++s) load_x(kb_begin + s, s);
            uint32_t stage = 0, phase = 1, copies = ahead;
            if (ahead == Shape::kStages) {
                for (uint32_t i = ahead; i < count; ++i) {
                    if (!wait_bounded(smem_u32(&control->empty[stage]), phase ^ 1u, &control->abort_flag, params.error_word)) break;
                    load_w(kb_begin + i, stage);
                    load_x(kb_begin + i, stage);
                    ++copies;
                    if (++stage == Shape::kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            control->copies = copies;
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0) {
            if (early) asm volatile("griddepcontrol.wait;" ::: "memory");
            asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
            constexpr uint32_t instr = fp8_instr_desc(kBlockN, NT);
            uint32_t stage = 0, phase = 0, buffer = 0, buffer_phase = 1;
            bool ok = true, any = false;
            if (FUSED) ok = wait_bounded(smem_u32(&control->rows_ready), 0, &control->abort_flag, params.error_word);
            for (uint32_t kb = kb_begin; ok && kb < kb_end; ++kb) {
                ok = wait_bounded(smem_u32(&control->tmem_empty[buffer]), buffer_phase, &control->abort_flag, params.error_word) &&
                     wait_bounded(smem_u32(&control->full[stage]), phase, &control->abort_flag, params.error_word);
                if (!ok) break;
                tc_fence_after();
                const uint64_t w = smem_desc_sw128(smem_u32(stage_w + stage * Shape::kWBytes));
                const uint64_t x = smem_desc_sw128(smem_u32(stage_x + (FUSED ? kb - kb_begin : stage) * Shape::kXBytes));
#pragma unroll
                for (int kk = 0; kk < kBlockK / kMmaK; ++kk)
                    mma_fp8(tmem_base + buffer * NT, w + static_cast<uint64_t>(kk * (kMmaK >> 4)),
                            x + static_cast<uint64_t>(kk * (kMmaK >> 4)), instr, kk != 0 ? 1u : 0u);
                mma_commit(smem_u32(&control->empty[stage]));
                mma_commit(smem_u32(&control->tmem_full[buffer]));
                any = true;
                if (++stage == Shape::kStages) {
                    stage = 0;
                    phase ^= 1u;
                }
                if (++buffer == Shape::kBuffers) {
                    buffer = 0;
                    buffer_phase ^= 1u;
                }
            }
            control->multiplied = any ? 1u : 0u;
        }
        __syncwarp();
    } else {
        if (early) asm volatile("griddepcontrol.wait;" ::: "memory");
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
        constexpr int kColumns = NT;  // sums of a thread
        const uint32_t worker = warp - 2u;
        const uint32_t quarter = warp & 3u;  // tensor memory lanes this warp may read
        float *scales = scale_rows + worker * Shape::kScaleFloats;
        const float *w_scales = params.w_scales + (static_cast<size_t>(tile.expert) * params.n_blocks + n_block) * params.k_blocks;
        if constexpr (FUSED) {
            const uint32_t blocks = kb_end - kb_begin;
            const uint32_t items = (tile.row_end - tile.row0) * blocks;
            auto quantize = [&](auto element, auto gated) {
                fuse_rows<decltype(element), decltype(gated)::value, NT>(fused, params, tile.row0, items, kb_begin, blocks, stage_x,
                                                                         fused_scales, worker, lane);
            };
            auto choose = [&](auto element) {
                if (fused.gated != 0) {
                    quantize(element, std::true_type{});
                } else {
                    quantize(element, std::false_type{});
                }
            };
            if (fused.type == QPUCUDA_DTYPE_F32) {
                choose(float{});
            } else if (fused.type == QPUCUDA_DTYPE_BF16) {
                choose(__nv_bfloat16{});
            } else {
                choose(__half{});
            }
            fence_proxy_async_shared();  // the MMA reads what was just written
            asm volatile("bar.sync 1, 128;" ::: "memory");
            if (worker == 0 && lane == 0) mbar_arrive(smem_u32(&control->rows_ready));
        }
        const float *a_scales = FUSED ? fused_scales : params.a_scales + static_cast<size_t>(tile.row0) * params.a_scale_row_stride;
        // Lane j stages row j's scale; rows past the tile hold zeros or another expert's values and
        // are not stored. Fetched two blocks ahead.
        const bool staging = lane < kColumns && tile.row0 + lane < (FUSED ? tile.row_end : params.rows);
        const size_t scale_row = FUSED ? 1 : params.a_scale_row_stride, scale_block = FUSED ? NT : params.a_scale_group_stride;
        const uint32_t scale_first = FUSED ? kb_begin : 0u;
        auto fetch = [&](uint32_t kb, float &row_scale, float &w_scale) {
            const bool inside = kb < kb_end;
            w_scale = inside ? __ldg(w_scales + kb) : 0.0f;
            row_scale = inside && staging
                            ? a_scales[static_cast<size_t>(lane) * scale_row + static_cast<size_t>(kb - scale_first) * scale_block]
                            : 0.0f;
        };
        float row_now, row_next, w_now, w_next;
        fetch(kb_begin, row_now, w_now);
        fetch(kb_begin + 1, row_next, w_next);
        uint64_t acc[kColumns / 2];
#pragma unroll
        for (int i = 0; i < kColumns / 2; ++i) acc[i] = 0;
        const uint32_t taddr = tmem_base + ((quarter * 32u) << 16);
        uint32_t buffer = 0, buffer_phase = 0;
        bool ok = true;
        for (uint32_t kb = kb_begin; kb < kb_end; ++kb) {
            float *products = scales + (kb & 1u) * kColumns;
            if (lane < kColumns) products[lane] = row_now * w_now;
            row_now = row_next;
            w_now = w_next;
            fetch(kb + 2, row_next, w_next);
            if (lane == 0) ok = wait_bounded(smem_u32(&control->tmem_full[buffer]), buffer_phase, &control->abort_flag, params.error_word);
            ok = __shfl_sync(0xFFFFFFFFu, ok ? 1 : 0, 0) != 0;  // also orders the products' stores before their loads
            __syncwarp();
            if (!ok) break;
            tc_fence_after();
            uint32_t r[kColumns];
            if constexpr (kColumns == 16) {
                tmem_load_x16(taddr + buffer * NT, r);
            } else {
                tmem_load_x32(taddr + buffer * NT, r);
            }
            tmem_wait_load(r);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&control->tmem_empty[buffer]));
#pragma unroll
            for (int i = 0; i < kColumns; i += 4) {
                const ulonglong2 s = *reinterpret_cast<const ulonglong2 *>(products + i);
                acc[i / 2] = fma2(pack2(r[i], r[i + 1]), s.x, acc[i / 2]);
                acc[i / 2 + 1] = fma2(pack2(r[i + 2], r[i + 3]), s.y, acc[i / 2 + 1]);
            }
            if (++buffer == Shape::kBuffers) {
                buffer = 0;
                buffer_phase ^= 1u;
            }
        }
        const uint32_t column = quarter * 32u + lane;  // output column inside the block
        if (split > 1) {
            // The tile's rows in turn over the ranks: each row's sums go to its rank, as [rank][row /
            // split][column]; into its stages only once the MMAs of the whole cluster have completed.
            __syncwarp();
            if (!Shape::kOwnSums) cluster_arrive();
            cluster_wait();
            const uint32_t rows = tile.row_end - tile.row0;
            const uint32_t mine = smem_u32(sums) + ((rank * NT >> split_shift) * kBlockN + column) * 4u;
#pragma unroll
            for (uint32_t i = 0; i < kColumns; ++i) {
                const float v = (i & 1u) ? high(acc[i / 2]) : low(acc[i / 2]);
                if (i < rows) store_cluster(map_to_rank(mine + (i >> split_shift) * (kBlockN * 4u), i & (split - 1u)), v);
            }
            __syncwarp();
        } else if (ok && n0 + column < params.n) {
            const float bias = params.bias != nullptr ? __ldg(params.bias + n0 + column) : 0.0f;
            Out *out = static_cast<Out *>(params.out) + static_cast<size_t>(tile.row0) * params.out_stride + n0 + column;
            const uint32_t rows = tile.row_end - tile.row0;
#pragma unroll
            for (uint32_t i = 0; i < kColumns; ++i) {
                const float v = (i & 1u) ? high(acc[i / 2]) : low(acc[i / 2]);
                if (i < rows) out[i * params.out_stride] = from_float<Out>(v + bias);
            }
        }
    }
    if (split > 1) {
        __syncwarp();
        if (warp < 2 || !tile.valid) {
            if (!Shape::kOwnSums) cluster_arrive();
            cluster_wait();
        }
        cluster_sync();  // every rank's sums are in place; no CTA touches another's memory from here on
        if (tile.valid && warp >= 2) {
            const uint32_t rows = tile.row_end - tile.row0;
            const uint32_t column = threadIdx.x - 64u;  // 128 across
            const bool inside = n0 + column < params.n;
            const float bias = params.bias != nullptr && inside ? __ldg(params.bias + n0 + column) : 0.0f;
            for (uint32_t row = rank; row < rows; row += split) {
                float sum = 0.0f;
#pragma unroll
                for (uint32_t r = 0; r < kMaxSplit; ++r)
                    if (r < split) sum += sums[((r * NT >> split_shift) + (row >> split_shift)) * kBlockN + column];
                if (inside)
                    static_cast<Out *>(params.out)[static_cast<size_t>(tile.row0 + row) * params.out_stride + n0 + column] =
                        from_float<Out>(sum + bias);
            }
        }
    }
    if (params.experts != 0 && rank == 0 && warp >= 2) {
        const uint32_t column = n0 + threadIdx.x - 64u;
        if (column < params.n)
            for (uint32_t row = owned_rows(params) + blockIdx.y; row < params.rows; row += gridDim.y)
                static_cast<Out *>(params.out)[static_cast<size_t>(row) * params.out_stride + column] = from_float<Out>(0.0f);
    }
    tc_fence_before();
    __syncthreads();
    if (control->abort_flag != 0) {
        if (threadIdx.x == 0) drain_copies<Shape::kStages>(control->full, control->copies);
        if (threadIdx.x == 32 && control->multiplied != 0) drain_mmas<false>(&control->drain);
        __syncthreads();
    }
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(Shape::kTmemColumns)
                     : "memory");
    }
}

// A narrow product's tiles: their height, their number at most (whatever the offsets) and the CTAs
// that share the K blocks of one.
struct NarrowLaunch {
    int height;
    uint32_t tiles, split;
};

template <int NT, bool FUSED, typename Out>
cudaError_t launch_narrow(const CUtensorMap &map_w, const CUtensorMap &map_a, const GemmParams &params, const NarrowLaunch &launch,
                          const FusedRows &fused, cudaStream_t stream) {
    using Shape = Narrow<NT, FUSED>;
    static PerDeviceOnce configured;
    const cudaError_t error = configured.run([] {
        return cudaFuncSetAttribute(fp8_gemm_narrow_kernel<NT, FUSED, Out>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    static_cast<int>(Shape::kSharedBytes));
    });
    if (error != cudaSuccess) return error;
    cudaLaunchAttribute attributes[2] = {};
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = launch.split;
    attributes[1].val.clusterDim.y = 1;
    attributes[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(params.n_blocks * launch.split, launch.tiles, 1);
    config.blockDim = dim3(Shape::kThreads);
    config.dynamicSmemBytes = Shape::kSharedBytes;
    config.stream = stream;
    config.attrs = attributes;
    config.numAttrs = 2;
    return cudaLaunchKernelEx(&config, fp8_gemm_narrow_kernel<NT, FUSED, Out>, map_w, map_a, params, fused);
}

template <typename Out>
cudaError_t launch_narrow_rows(const CUtensorMap &map_w, const CUtensorMap &map_a, const GemmParams &params,
                               const NarrowLaunch &launch, const FusedRows *fused, cudaStream_t stream) {
    if (fused != nullptr) return launch_narrow<16, true, Out>(map_w, map_a, params, launch, *fused, stream);
    const FusedRows none{};
    return launch.height == 16 ? launch_narrow<16, false, Out>(map_w, map_a, params, launch, none, stream)
                               : launch_narrow<32, false, Out>(map_w, map_a, params, launch, none, stream);
}

// ---- the wide kernel --------------------------------------------------------------------------

// Many rows: 128 rows are the M operand, 256 output columns the N operand, so tensor memory lane =
// row and the factor sx * sw is one number per thread and block (a row's scale; the two halves of
// the columns are two rows of weight scales, one for each group of four epilogue warps).
//
// Per block of 128 columns a CTA's MMAs take 512 cycles in a pair (768 alone: both operands then come
// from one SM's shared memory), its eight epilogue warps read 128 KB of tensor memory and form 32768
// multiply-adds in registers meanwhile. 4096 x 28672 x 8192 bf16 in pairs: 900 us in a short run, 2.1
// PFLOP/s (1.28 of the measured bf16 burst); 1040 us, 1.11, once the 1000 W limit holds the clock at 1.6 GHz.
// By parts, in runs of one length: 920 us whole, without the sums 845, without reading the accumulators
// either 745, the MMAs alone 650. Where power does not decide (4096 x 5632 x 8192, 170 us: tensor pipe 57 %
// active, issue slots 38 %) the pipe waits for the accumulators' way through registers.
constexpr int kWideM = 128;
constexpr int kWideN = 256;
constexpr uint64_t kGroupBytes = 40ull << 20;  // rows of a group of tiles: part of the 126 MB L2
constexpr uint64_t kGroupRows = 16;
constexpr int kWideWarps = 8;  // epilogue: lane quarters x column halves
constexpr int kWideThreads = 128 + 32 * kWideWarps;
// Registers a thread: an epilogue thread holds 128 sums and 32 loaded values, the other four warps
// hold next to nothing. Launched with 168 each (three warps per scheduler), handed over to
// 40 + 2 x 232 = 3 x 168.
constexpr int kWideFewRegisters = 40;
constexpr int kWideManyRegisters = 232;
static_assert(128 * kWideFewRegisters + 256 * kWideManyRegisters <= 384 * 168, "register hand-over");
// A stage per CTA. Alone: 128 rows and 256 weight rows. In a pair (cluster of two, tcgen05
// cta_group::2, a tile of 256 x 256): 128 rows and this CTA's half of the weight rows, which both
// CTAs' MMAs read; a third less shared-memory traffic per product.
template <bool PAIR>
struct Wide {
    static constexpr int kRows = PAIR ? 2 * kWideM : kWideM;  // of a tile
    static constexpr int kStages = PAIR ? 4 : 3;
    static constexpr int kABytes = kWideM * kBlockK;
    static constexpr int kWBytes = (PAIR ? kWideN / 2 : kWideN) * kBlockK;
    static constexpr int kStageBytes = kABytes + kWBytes;
};
constexpr int kWideBoxBytes = 4096;    // 32 rows x 128 bytes of the output
constexpr int kWideStoreBytes = 2 * kWideBoxBytes;  // per epilogue warp, on their way out
// The experts' tables: their first tiles and first rows, with one entry past the end each.
constexpr size_t kWideTableBytes = 2 * (QPUCUDA_MAX_EXPERTS + 1) * sizeof(uint32_t);
template <bool PAIR>
constexpr size_t wide_shared_bytes() {
    return Wide<PAIR>::kStages * Wide<PAIR>::kStageBytes + kWideWarps * kWideStoreBytes + kWideTableBytes + 256 + 1024;
}
static_assert(wide_shared_bytes<false>() <= 227 * 1024 && wide_shared_bytes<true>() <= 227 * 1024, "shared memory");

struct WideLaunch {
    bool pair;
    uint32_t split;
    uint64_t tiles;  // at most, whatever the offsets
    uint32_t n_tiles, group_rows;
};

struct WideTile {
    uint32_t expert, row0, row_end, n0;
};

// Tile order inside a matrix: groups of group_rows row blocks, the row block fastest inside a group,
// so the rows of a group stay in L2 while its columns stream past and each weight tile is read from
// DRAM once per group.
__device__ __forceinline__ void order_tile(uint32_t tile, uint32_t m_blocks, uint32_t n_tiles, uint32_t group_rows,
                                           uint32_t &m_block, uint32_t &n_tile) {
    const uint32_t group_tiles = group_rows * n_tiles;
    const uint32_t group = tile / group_tiles;
    const uint32_t first = group * group_rows;
    const uint32_t height = min(group_rows, m_blocks - first);
    const uint32_t local = tile - group * group_tiles;
    m_block = first + local % height;
    n_tile = local / height;
}

// first_tile[e]: tiles of the experts before e. The last e with first_tile[e] <= tile holds it, in its
// rows from first_row[e] on.
template <uint32_t HEIGHT>
__device__ __forceinline__ WideTile locate(const GemmParams &params, const uint32_t *first_tile, const uint32_t *first_row,
                                           uint32_t n_tiles, uint32_t group_rows, uint32_t tile) {
    WideTile result;
    uint32_t begin = 0, end = params.rows, local = tile;
    result.expert = 0;
    if (params.experts != 0) {
        uint32_t low_e = 0, high_e = params.experts;  // first_tile[low_e] <= tile < first_tile[high_e]
        while (high_e - low_e > 1) {
            const uint32_t middle = (low_e + high_e) / 2;
            if (first_tile[middle] <= tile) {
                low_e = middle;
            } else {
                high_e = middle;
            }
        }
        result.expert = low_e;
        local = tile - first_tile[low_e];
        begin = first_row[low_e];
        end = max(first_row[low_e + 1], begin);
    }
    uint32_t m_block, n_tile;
    order_tile(local, (end - begin + HEIGHT - 1) / HEIGHT, n_tiles, group_rows, m_block, n_tile);
    result.row0 = begin + m_block * HEIGHT;
    result.row_end = min(end, result.row0 + HEIGHT);
    result.n0 = n_tile * kWideN;
    return result;
}

// 64 bytes of each of a warp's 32 rows, transposed through shared memory so that four lanes write
// one row's 64 bytes. Slot c of row r lies at slot c ^ ((r >> 1) & 3): no bank conflicts either way.
template <typename Out>
__device__ __forceinline__ void store_chunk(uint4 *buffer, const float (&v)[64 / sizeof(Out)], Out *out, size_t out_stride,
                                            uint32_t rows, uint32_t columns, bool vector, uint32_t lane) {
    constexpr int kColumns = 64 / sizeof(Out);
    constexpr int kPerSlot = kColumns / 4;
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        Vector<Out> slot;
#pragma unroll
        for (int i = 0; i < kPerSlot; ++i) slot.items[i] = from_float<Out>(v[c * kPerSlot + i]);
        buffer[lane * 4 + (c ^ ((lane >> 1) & 3))] = slot.bits;
    }
    __syncwarp();
    if (vector && columns >= kColumns) {
        const uint32_t c = lane & 3u;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const uint32_t r = i * 8u + lane / 4u;
            const uint4 value = buffer[r * 4 + (c ^ ((r >> 1) & 3))];
            if (r < rows) *reinterpret_cast<uint4 *>(out + r * out_stride + c * kPerSlot) = value;
        }
    } else if (lane < kColumns) {
        const Out *items = reinterpret_cast<const Out *>(buffer);
        for (uint32_t r = 0; r < min(rows, 32u); ++r)
            if (lane < columns)
                out[r * out_stride + lane] = items[(r * 4 + ((lane / kPerSlot) ^ ((r >> 1) & 3))) * kPerSlot + lane % kPerSlot];
    }
}

template <int N>
__device__ __forceinline__ void add_bias(const GemmParams &params, uint32_t n, float (&v)[N]) {
    if (params.bias == nullptr) return;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += n + i < params.n ? __ldg(params.bias + n + i) : 0.0f;
}

// One box of a warp's 32 rows (a row to a lane, 128 bytes each) on its way out. Staged in shared
// memory in the 128-byte swizzle (16-byte slot c of row r at c ^ (r & 7): no bank conflicts) and copied
// out from there: by the copy engine while the warp goes on, where the output's rows are aligned and
// all 32 are the tile's (`map` then), else by the warp, eight lanes to a row. A warp's boxes take its two
// buffers in turn, over all of its tiles (a ragged last tile can have an odd number of boxes), and each
// box is one group of copies, so a buffer is free once no more than the newest group is still being read.
template <typename Out>
__device__ __forceinline__ void store_box(uint8_t *buffer, const float (&v)[128 / sizeof(Out)], const CUtensorMap *map, Out *out,
                                          size_t out_stride, int row, uint32_t column, uint32_t rows, uint32_t columns, bool vector,
                                          uint32_t lane) {
    constexpr uint32_t kColumns = 128 / sizeof(Out);
    constexpr uint32_t kPerSlot = kColumns / 8;
    uint4 *slots = reinterpret_cast<uint4 *>(buffer);
    if (lane == 0) bulk_wait_read_all_but_one();  // the copy that last read this buffer is two copies back
    __syncwarp();
#pragma unroll
    for (uint32_t c = 0; c < 8; ++c) {
        Vector<Out> slot;
#pragma unroll
        for (uint32_t i = 0; i < kPerSlot; ++i) slot.items[i] = from_float<Out>(v[c * kPerSlot + i]);
        slots[lane * 8u + (c ^ (lane & 7u))] = slot.bits;
    }
    if (map != nullptr) {
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) {
            tma_store_2d(map, smem_u32(buffer), static_cast<int>(column * sizeof(Out)), row);
            bulk_commit();
        }
        return;
    }
    __syncwarp();
    if (vector && columns >= kColumns) {
        const uint32_t c = lane & 7u;
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            const uint32_t r = i * 4u + lane / 8u;
            const uint4 value = slots[r * 8u + (c ^ (r & 7u))];
            if (r < rows) *reinterpret_cast<uint4 *>(out + r * out_stride + c * kPerSlot) = value;
        }
    } else {
        const Out *items = reinterpret_cast<const Out *>(buffer);
        for (uint32_t r = 0; r < min(rows, 32u); ++r)
#pragma unroll
            for (uint32_t j = lane; j < kColumns; j += 32)
                if (j < columns) out[r * out_stride + j] = items[(r * 8u + ((j / kPerSlot) ^ (r & 7u))) * kPerSlot + j % kPerSlot];
    }
    if (lane == 0) bulk_commit();  // an empty group keeps the count of two buffers
    __syncwarp();
}

// Persistent: one CTA (or pair) per SM (or two) walks tiles 0, 1, ... in steps of the CTAs or pairs.
//   warp 0   copies: a row box and the weight boxes per stage (a pair's bytes all complete on rank 0's barriers)
//   warp 1   tensor memory and MMA (rank 0 alone in a pair): 4 MMAs per stage into one of two accumulators
//   warp 2   the experts' table of tiles, warp 3 nothing
//   4 to 11  each block's accumulator into registers, scaled; at the tile's end the store
// SPLIT: few tiles. The CTAs of a cluster share one tile's K blocks and add their sums, in slice
// order, through distributed shared memory; each CTA has one tile. The sums are pushed to the CTA that
// adds them: 96 KB leave each of four CTAs in 2.9 us, 16 bytes a cycle, and take 5.6 to be read from
// the other side.
template <typename Out, bool PAIR, bool SPLIT>
__global__ void __launch_bounds__(kWideThreads, 1)
    fp8_gemm_wide_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a,
                         const __grid_constant__ CUtensorMap map_out,
                         const GemmParams params, uint32_t n_tiles, uint32_t group_rows, uint32_t most_tiles) {
    using Shape = Wide<PAIR>;
    constexpr int kStages = Shape::kStages;
    using Ctl = Control<kStages, 2>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *stage_w = smem;
    uint8_t *stage_a = smem + kStages * Shape::kWBytes;
    uint8_t *store = smem + kStages * Shape::kStageBytes;
    uint32_t *first_tile = reinterpret_cast<uint32_t *>(store + kWideWarps * kWideStoreBytes);
    Ctl *control = reinterpret_cast<Ctl *>(store + kWideWarps * kWideStoreBytes + kWideTableBytes);
    uint32_t *first_row = first_tile + QPUCUDA_MAX_EXPERTS + 1;
    static_assert(sizeof(Ctl) <= 256 && kWideTableBytes % 8 == 0, "control block");

    const uint32_t warp = threadIdx.x >> 5;
    const uint32_t lane = threadIdx.x & 31;
    static_assert(!(PAIR && SPLIT), "a cluster is a pair or shares K");
    const uint32_t rank = PAIR ? cluster_rank() : 0u;
    const uint32_t slices = SPLIT ? cluster_size() : 1u;
    const uint32_t slice = SPLIT ? cluster_rank() : 0u;
    const uint32_t tile_first = PAIR ? blockIdx.x / 2 : blockIdx.x / slices;
    const uint32_t tile_step = PAIR ? gridDim.x / 2 : (SPLIT ? 0x80000000u : gridDim.x);
    const uint32_t kb_begin = SPLIT ? static_cast<uint32_t>(static_cast<uint64_t>(params.k_blocks) * slice / slices) : 0u;
    const uint32_t kb_end = SPLIT ? static_cast<uint32_t>(static_cast<uint64_t>(params.k_blocks) * (slice + 1) / slices) : params.k_blocks;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(smem_u32(&control->full[s]), 1);
            mbar_init(smem_u32(&control->empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(smem_u32(&control->tmem_full[b]), 1);
            mbar_init(smem_u32(&control->tmem_empty[b]), (PAIR ? 2 : 1) * kWideWarps);
        }
        mbar_init(smem_u32(&control->drain), 1);
        control->abort_flag = 0;
        control->copies = control->multiplied = 0;
        mbar_init_fence();
    }
    if (warp == 1) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&control->tmem_base)),
                         "r"(2 * kWideN)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&control->tmem_base)),
                         "r"(2 * kWideN)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    // The rows' copies, the offsets and every store come after the previous kernel. Weights are not
    // read early here: the tiles are long.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (warp == 2 && params.experts != 0) {
        uint32_t before = 0;
        const int32_t rows = static_cast<int32_t>(params.rows);
        for (uint32_t e0 = 0; e0 < params.experts; e0 += 32) {
            const uint32_t e = e0 + lane;
            uint32_t tiles = 0;
            if (e < params.experts) {
                const int32_t begin = min(max(params.offsets[e], 0), rows);
                const int32_t end = min(max(params.offsets[e + 1], begin), rows);
                tiles = (static_cast<uint32_t>(end - begin) + Shape::kRows - 1) / Shape::kRows * n_tiles;
            }
            uint32_t through = tiles;
#pragma unroll
            for (int offset = 1; offset < 32; offset <<= 1) {
                const uint32_t other = __shfl_up_sync(0xFFFFFFFFu, through, offset);
                if (lane >= static_cast<uint32_t>(offset)) through += other;
            }
            if (e < params.experts) {
                first_tile[e] = before + through - tiles;
                first_row[e] = static_cast<uint32_t>(min(max(params.offsets[e], 0), rows));
            }
            before += __shfl_sync(0xFFFFFFFFu, through, 31);
        }
        if (lane == 0) {
            first_tile[params.experts] = before;
            first_row[params.experts] = static_cast<uint32_t>(min(max(params.offsets[params.experts], 0), rows));
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (PAIR) cluster_sync();  // both CTAs' barriers exist before any arrival or copy of the other
    tc_fence_after();
    const uint32_t tmem_base = control->tmem_base;
    // no more than ascending offsets can make
    const uint32_t total = params.experts != 0 ? min(first_tile[params.experts], most_tiles) : most_tiles;

    if (warp == 0) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWideFewRegisters));
        if (lane == 0) {
            prefetch_tensor_map(&map_w);
            prefetch_tensor_map(&map_a);
            uint32_t stage = 0, phase = 0, copies = 0;
            bool ok = true;
            for (uint32_t t = tile_first; ok && t < total; t += tile_step) {
                const WideTile tile = locate<Shape::kRows>(params, first_tile, first_row, n_tiles, group_rows, t);
                const int w_row = static_cast<int>(tile.expert * params.n + tile.n0 + rank * kBlockN);
                const int a_row = static_cast<int>(tile.row0 + rank * kWideM);
                for (uint32_t kb = kb_begin; kb < kb_end; ++kb) {
                    ok = wait_bounded(smem_u32(&control->empty[stage]), phase ^ 1u, &control->abort_flag, params.error_word);
                    if (!ok) break;
                    const uint32_t full = smem_u32(&control->full[stage]);
                    const int x = static_cast<int>(kb * kBlockK);
                    if constexpr (PAIR) {
                        if (rank == 0) mbar_expect_tx(full, 2 * Shape::kStageBytes);
                        const uint32_t leader_full = map_to_rank(full, 0);
                        tma_load_2d_pair(smem_u32(stage_a + stage * Shape::kABytes), &map_a, leader_full, x, a_row);
                        tma_load_2d_pair(smem_u32(stage_w + stage * Shape::kWBytes), &map_w, leader_full, x, w_row);
                    } else {
                        mbar_expect_tx(full, Shape::kStageBytes);
                        tma_load_2d(smem_u32(stage_a + stage * Shape::kABytes), &map_a, full, x, a_row);
                        tma_load_2d(smem_u32(stage_w + stage * Shape::kWBytes), &map_w, full, x, w_row);
                        tma_load_2d(smem_u32(stage_w + stage * Shape::kWBytes + Shape::kWBytes / 2), &map_w, full, x, w_row + kBlockN);
                    }
                    ++copies;
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            control->copies = copies;
        }
        __syncwarp();
        if constexpr (SPLIT) {
            cluster_sync();
            cluster_sync();
        }
    } else if (warp == 1) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWideFewRegisters));
        if (lane == 0 && rank == 0) {
            constexpr uint32_t instr = fp8_instr_desc(Shape::kRows, kWideN);
            uint32_t stage = 0, phase = 0, buffer = 0, buffer_phase = 1;
            bool ok = true, any = false;
            for (uint32_t t = tile_first; ok && t < total; t += tile_step) {
                for (uint32_t kb = kb_begin; kb < kb_end; ++kb) {
                    ok = wait_bounded(smem_u32(&control->tmem_empty[buffer]), buffer_phase, &control->abort_flag, params.error_word) &&
                         wait_bounded(smem_u32(&control->full[stage]), phase, &control->abort_flag, params.error_word);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t a = smem_desc_sw128(smem_u32(stage_a + stage * Shape::kABytes));
                    const uint64_t w = smem_desc_sw128(smem_u32(stage_w + stage * Shape::kWBytes));
#pragma unroll
                    for (int kk = 0; kk < kBlockK / kMmaK; ++kk) {
                        const uint64_t step = static_cast<uint64_t>(kk * (kMmaK >> 4));
                        if constexpr (PAIR) {
                            mma_fp8_pair(tmem_base + buffer * kWideN, a + step, w + step, instr, kk != 0 ? 1u : 0u);
                        } else {
                            mma_fp8(tmem_base + buffer * kWideN, a + step, w + step, instr, kk != 0 ? 1u : 0u);
                        }
                    }
                    if constexpr (PAIR) {  // frees the stage and fills the accumulator in both CTAs
                        mma_commit_pair(smem_u32(&control->tmem_full[buffer]));
                        mma_commit_pair(smem_u32(&control->empty[stage]));
                    } else {
                        mma_commit(smem_u32(&control->empty[stage]));
                        mma_commit(smem_u32(&control->tmem_full[buffer]));
                    }
                    any = true;
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                    if (++buffer == 2) {
                        buffer = 0;
                        buffer_phase ^= 1u;
                    }
                }
            }
            control->multiplied = any ? 1u : 0u;
        }
        __syncwarp();
        if constexpr (SPLIT) {
            cluster_sync();
            cluster_sync();
        }
    } else if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kWideFewRegisters));
        if constexpr (SPLIT) {
            cluster_sync();
            cluster_sync();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kWideManyRegisters));
        const uint32_t worker = warp - 4u;
        const uint32_t quarter = warp & 3u;
        const uint32_t half = worker / 4u;
        uint8_t *buffer_out = store + worker * kWideStoreBytes;
        uint32_t box = 0;  // the buffer of this warp's next box, in turn across its tiles
        const uint32_t taddr = tmem_base + ((quarter * 32u) << 16) + half * (kWideN / 2);
        const bool vector = (reinterpret_cast<uintptr_t>(params.out) & 15u) == 0 && params.out_stride * sizeof(Out) % 16 == 0;
        const uint32_t tmem_full0 = smem_u32(&control->tmem_full[0]);
        // released on the barrier of the CTA that issues the MMAs
        const uint32_t tmem_empty0 = PAIR ? map_to_rank(smem_u32(&control->tmem_empty[0]), 0) : smem_u32(&control->tmem_empty[0]);
        uint32_t buffer = 0, buffer_phase = 0;
        const uint32_t part_shift = slices == 2 ? 4u : 3u;  // SPLIT: log2 of the float4 columns of a CTA's part of a half
        bool summed = false;
        for (uint32_t t = tile_first; t < total; t += tile_step) {
            const WideTile tile = locate<Shape::kRows>(params, first_tile, first_row, n_tiles, group_rows, t);
            const uint32_t n0 = tile.n0 + half * (kWideN / 2);
            const uint32_t row0 = tile.row0 + rank * kWideM + quarter * 32u;
            const bool row_inside = row0 + lane < tile.row_end;
            const bool block_inside = n0 < params.n;
            const float *w_scales = params.w_scales + (static_cast<size_t>(tile.expert) * params.n_blocks + n0 / kBlockN) * params.k_blocks;
            const float *a_scales = params.a_scales + static_cast<size_t>(row0 + lane) * params.a_scale_row_stride;
            // A block's factor is fetched two blocks ahead; the fetches of the last two repeat the last block.
            const float *a_at = (row_inside ? a_scales : params.a_scales) + static_cast<size_t>(kb_begin) * params.a_scale_group_stride;
            const float *w_at = (block_inside ? w_scales : params.w_scales) + kb_begin;
            uint32_t fetched = kb_begin;
            auto fetch = [&](float &a, float &w) {
                a = *a_at;
                w = __ldg(w_at);
                if (++fetched < kb_end) {
                    a_at += params.a_scale_group_stride;
                    ++w_at;
                }
            };
            float a_now, w_now, a_next, w_next;
            fetch(a_now, w_now);
            fetch(a_next, w_next);
            uint64_t acc[64];
#pragma unroll
            for (int i = 0; i < 64; ++i) acc[i] = 0;
            // 32 columns at a time through two sets of registers, the next load under way while the
            // previous one is added; the accumulator is given back before its second half is added.
            // No load crosses the loop's end: a set carried around costs 32 moves (1060 against 910 us
            // at 4096 x 28672 x 8192).
            uint32_t even[32], odd[32];
            auto add = [&](int c, const uint32_t (&r)[32], uint64_t factors) {
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[c * 16 + i] = fma2(pack2(r[2 * i], r[2 * i + 1]), factors, acc[c * 16 + i]);
            };
            auto arrived = [&]() {
                const bool full = wait_bounded(tmem_full0 + buffer * 8u, buffer_phase, &control->abort_flag, params.error_word);
                const bool all = __all_sync(0xFFFFFFFFu, full) != 0;
                tc_fence_after();
                return all;
            };
            bool ok = arrived();
            for (uint32_t kb = kb_begin; ok && kb < kb_end; ++kb) {
                const float factor = a_now * w_now;
                const uint64_t factors = pack2(factor, factor);
                a_now = a_next;
                w_now = w_next;
                fetch(a_next, w_next);
                const uint32_t block = taddr + buffer * kWideN;
                tmem_load_x32(block, even);
                tmem_wait_load(even);
                tmem_load_x32(block + 32, odd);
                add(0, even, factors);
                tmem_wait_load(odd);
                tmem_load_x32(block + 64, even);
                add(1, odd, factors);
                tmem_wait_load(even);
                tmem_load_x32(block + 96, odd);
                tmem_wait_load(odd);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if constexpr (PAIR) {
                        arrive_cluster(tmem_empty0 + buffer * 8u);
                    } else {
                        mbar_arrive(tmem_empty0 + buffer * 8u);
                    }
                }
                if (++buffer == 2) {
                    buffer = 0;
                    buffer_phase ^= 1u;
                }
                if (kb + 1 < kb_end) ok = arrived();
                add(2, even, factors);
                add(3, odd, factors);
            }
            if (!ok) break;
            if constexpr (SPLIT) {
                // The only tile of this CTA. Each of the cluster's CTAs adds up its share of the columns, a
                // part of both halves: the sums go to the stages of the CTA they belong to, free once the
                // cluster's MMAs have completed, as [slice][half][column / 4][row] float4.
                __syncwarp();
                cluster_sync();
                if (row0 < tile.row_end) {
                    const uint32_t mine = smem_u32(smem) + ((((slice * 2u + half) << part_shift) * kWideM) + quarter * 32u + lane) * 16u;
#pragma unroll
                    for (uint32_t i = 0; i < 32; ++i) {
                        const uint32_t owner = i >> part_shift, place = i - (owner << part_shift);
                        store_cluster4(map_to_rank(mine + place * (kWideM * 16u), owner),
                                       make_float4(low(acc[2 * i]), high(acc[2 * i]), low(acc[2 * i + 1]), high(acc[2 * i + 1])));
                    }
                }
                __syncwarp();
                cluster_sync();
                summed = true;
                continue;
            }
            if (row0 >= tile.row_end || !block_inside) continue;
            constexpr int kChunk = 128 / static_cast<int>(sizeof(Out));
            const uint32_t rows = tile.row_end - row0;
            // Rows past an expert's would be overwritten by a copy of the whole box; rows past the output
            // are cut off by it. So are columns, but only to 16 bytes: the last, partly filled box goes
            // the other way.
            const bool whole = params.tma_store != 0 && (params.experts == 0 || rows >= 32);
#pragma unroll
            for (int c = 0; c < kWideN / 2; c += kChunk) {
                const uint32_t n = n0 + c;
                if (n >= params.n) break;
                float v[kChunk];
#pragma unroll
                for (int i = 0; i < kChunk; i += 2) {
                    v[i] = low(acc[(c + i) / 2]);
                    v[i + 1] = high(acc[(c + i) / 2]);
                }
                add_bias(params, n, v);
                store_box<Out>(buffer_out + box, v, whole && n + kChunk <= params.n ? &map_out : nullptr,
                               static_cast<Out *>(params.out) + static_cast<size_t>(row0) * params.out_stride + n, params.out_stride,
                               static_cast<int>(row0), n, rows, params.n - n, vector, lane);
                box ^= kWideBoxBytes;
            }
        }
        if constexpr (SPLIT) {
            if (!summed) {  // no tile, or given up
                __syncwarp();
                cluster_sync();
                cluster_sync();
            } else {
                const WideTile tile = locate<Shape::kRows>(params, first_tile, first_row, n_tiles, group_rows, tile_first);
                constexpr uint32_t kChunk = 64 / sizeof(Out);
                const uint32_t row0 = tile.row0 + quarter * 32u;
                const uint32_t columns = 4u << part_shift;
                const uint32_t n0 = tile.n0 + half * (kWideN / 2) + slice * columns;
                if (row0 < tile.row_end) {
                    for (uint32_t c = 0; c < columns && n0 + c < params.n; c += kChunk) {
                        const float4 *part = reinterpret_cast<const float4 *>(smem) +
                                             ((half << part_shift) + c / 4u) * kWideM + quarter * 32u + lane;
                        float v[kChunk] = {};
                        for (uint32_t r = 0; r < slices; ++r, part += (2u << part_shift) * kWideM) {
#pragma unroll
                            for (uint32_t i = 0; i < kChunk / 4; ++i) {
                                const float4 term = part[i * kWideM];
                                v[4 * i] += term.x;
                                v[4 * i + 1] += term.y;
                                v[4 * i + 2] += term.z;
                                v[4 * i + 3] += term.w;
                            }
                        }
                        const uint32_t n = n0 + c;
                        add_bias(params, n, v);
                        store_chunk<Out>(reinterpret_cast<uint4 *>(buffer_out), v, static_cast<Out *>(params.out) + static_cast<size_t>(row0) * params.out_stride + n,
                                         params.out_stride, tile.row_end - row0, params.n - n, vector, lane);
                    }
                }
            }
        }
        if (params.experts != 0) {
            // rows no expert owns
            const uint32_t step = gridDim.x * kWideWarps;
            for (uint32_t row = owned_rows(params) + blockIdx.x * kWideWarps + worker; row < params.rows; row += step)
                for (uint32_t n = lane; n < params.n; n += 32)
                    static_cast<Out *>(params.out)[static_cast<size_t>(row) * params.out_stride + n] = from_float<Out>(0.0f);
        }
        if (lane == 0) bulk_wait_all();  // every copy out is complete before the CTA ends
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (control->abort_flag != 0) {
        if (threadIdx.x == 0) {
            // Only rank 0's barriers see a pair's copies; the other CTA gives its own a bounded 200 us.
            if (!PAIR || cluster_rank() == 0) {
                drain_copies<kStages>(control->full, control->copies);
            } else {
                const uint64_t start = globaltimer();
                while (globaltimer() - start < 200000ull) {
                }
            }
        }
        if (threadIdx.x == 32 && control->multiplied != 0) drain_mmas<PAIR>(&control->drain);
        __syncthreads();
    }
    // Neither CTA of a pair leaves while the other may still signal its barriers, read its shared
    // memory or write its tensor memory.
    if constexpr (PAIR) cluster_sync();
    if (warp == 1) {
        tc_fence_after();
        if constexpr (PAIR) {
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(2 * kWideN) : "memory");
        } else {
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(2 * kWideN) : "memory");
        }
    }
}

template <typename Out, bool PAIR, bool SPLIT>
cudaError_t configure_wide() {
    return cudaFuncSetAttribute(fp8_gemm_wide_kernel<Out, PAIR, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                static_cast<int>(wide_shared_bytes<PAIR>()));
}

// Pairs that can be resident at once, cached per device (0: not known yet).
int resident_pairs(int sm_count) {
    static std::atomic<int> cached[64] = {};
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return sm_count / 2;
    const int known = cached[device].load(std::memory_order_relaxed);
    if (known > 0) return known;
    cudaLaunchAttribute attribute = {};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = 2;
    attribute.val.clusterDim.y = 1;
    attribute.val.clusterDim.z = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(sm_count & ~1));
    config.blockDim = dim3(kWideThreads);
    config.dynamicSmemBytes = wide_shared_bytes<true>();
    config.attrs = &attribute;
    config.numAttrs = 1;
    int pairs = 0;
    if (cudaOccupancyMaxActiveClusters(&pairs, fp8_gemm_wide_kernel<float, true, false>, &config) != cudaSuccess || pairs <= 0) {
        (void)cudaGetLastError();
        return sm_count / 2;
    }
    cached[device].store(pairs, std::memory_order_relaxed);
    return pairs;
}

// split: CTAs of a cluster that share a tile's K blocks (1, 2 or 4; then tiles * split CTAs, one tile each).
template <typename Out, bool PAIR, bool SPLIT>
cudaError_t launch_wide(const CUtensorMap &map_w, const CUtensorMap &map_a, GemmParams params, const WideLaunch &launch,
                        int sm_count, cudaStream_t stream) {
    static PerDeviceOnce configured;
    const cudaError_t error = configured.run([] {
        const cudaError_t first = configure_wide<Out, PAIR, SPLIT>();
        return first != cudaSuccess || !PAIR ? first : configure_wide<float, true, false>();  // resident_pairs asks about this one
    });
    if (error != cudaSuccess) return error;
    const uint64_t resident = PAIR ? static_cast<uint64_t>(resident_pairs(sm_count)) : (SPLIT ? launch.tiles : static_cast<uint64_t>(sm_count));
    const uint64_t walkers = launch.tiles < resident ? launch.tiles : resident;
    const uint32_t cluster = PAIR ? 2u : launch.split;
    cudaLaunchAttribute attributes[2] = {};
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = cluster;
    attributes[1].val.clusterDim.y = 1;
    attributes[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(walkers * cluster));
    config.blockDim = dim3(kWideThreads);
    config.dynamicSmemBytes = wide_shared_bytes<PAIR>();
    config.stream = stream;
    config.attrs = attributes;
    config.numAttrs = cluster > 1 ? 2 : 1;
    CUtensorMap map_out;
    std::memset(&map_out, 0, sizeof(map_out));
    params.tma_store = encode_tensor_map_2d_u8(&map_out, params.out, static_cast<uint64_t>(params.n) * sizeof(Out), params.rows,
                                               params.out_stride * sizeof(Out), 128u, 32u)
                           ? 1u
                           : 0u;
    return cudaLaunchKernelEx(&config, fp8_gemm_wide_kernel<Out, PAIR, SPLIT>, map_w, map_a, map_out, params, launch.n_tiles,
                              launch.group_rows, static_cast<uint32_t>(launch.tiles));
}

template <typename Out>
cudaError_t launch_wide_type(const CUtensorMap &map_w, const CUtensorMap &map_a, const GemmParams &params, const WideLaunch &launch,
                             int sm_count, cudaStream_t stream) {
    if (launch.pair) return launch_wide<Out, true, false>(map_w, map_a, params, launch, sm_count, stream);
    if (launch.split > 1) return launch_wide<Out, false, true>(map_w, map_a, params, launch, sm_count, stream);
    return launch_wide<Out, false, false>(map_w, map_a, params, launch, sm_count, stream);
}

// Rows per matrix from which pairs' tiles of 256 rows are worth their padding with uneven experts: 512
// rows each (4096 tokens, 4 of 32, 5632 x 2048) took 303 us in pairs and 292 alone, 1024 rows 525 and 534.
constexpr uint64_t kPairShare = 1024;

GemmParams gemm_params(const qpucuda_fp8_gemm_desc &desc, unsigned int *error_word) {
    GemmParams params{};
    params.rows = desc.rows;
    params.n = desc.n;
    params.k = desc.k;
    params.k_blocks = (desc.k + kBlockK - 1) / kBlockK;
    params.n_blocks = (desc.n + kBlockN - 1) / kBlockN;
    params.experts = desc.experts;
    params.offsets = desc.offsets;
    params.a_scales = desc.a_scales;
    params.a_scale_row_stride = desc.a_scale_row_stride;
    params.a_scale_group_stride = desc.a_scale_group_stride;
    params.w_scales = desc.w_scales;
    params.bias = desc.bias;
    params.out = desc.out;
    params.out_stride = desc.out_stride;
    params.weights_settled = desc.weights_settled != 0 ? 1u : 0u;
    params.error_word = error_word;
    return params;
}

// Tiles of `height` rows, at most, whatever the offsets: one partly filled tile per matrix.
uint64_t most_tiles(const qpucuda_fp8_gemm_desc &desc, uint64_t filled, uint64_t height) {
    return (desc.rows + filled * (height - 1)) / height;
}

NarrowLaunch plan_narrow(const qpucuda_fp8_gemm_desc &desc, const GemmParams &params, uint64_t share, uint64_t filled, uint64_t sms) {
    NarrowLaunch launch{};
    // 16 rows, or 32 where a matrix has more (uneven experts: more than 4 on average)
    launch.height = share <= (desc.experts != 0 ? 4u : 16u) ? 16 : 32;
    const uint64_t tiles = most_tiles(desc, filled, static_cast<uint64_t>(launch.height));
    launch.tiles = static_cast<uint32_t>(tiles);
    // K is split over a cluster while the tiles leave SMs idle, two CTAs each.
    launch.split = 1;
    while (launch.split < kMaxSplit && tiles * params.n_blocks * launch.split * 2 <= sms * 2 && launch.split * 2 <= params.k_blocks)
        launch.split *= 2;
    return launch;
}

WideLaunch plan_wide(const qpucuda_fp8_gemm_desc &desc, const GemmParams &params, uint64_t share, uint64_t filled, uint64_t sms) {
    WideLaunch launch{};
    launch.n_tiles = (desc.n + kWideN - 1) / kWideN;
    // Pairs where tiles of 256 rows hold hardly more padding than tiles of 128.
    const uint64_t single_tiles = most_tiles(desc, filled, kWideM), pair_tiles = most_tiles(desc, filled, 2 * kWideM);
    launch.pair = sms >= 2 && (desc.experts != 0 ? share >= kPairShare : pair_tiles * 2 * 12 <= single_tiles * 13);
    launch.split = 1;
    if ((launch.pair ? pair_tiles : single_tiles) * launch.n_tiles * 2 <= sms) {
        launch.pair = false;
        while (launch.split < 4 && single_tiles * launch.n_tiles * launch.split * 2 <= sms && params.k_blocks >= 16) launch.split *= 2;
    }
    launch.tiles = (launch.pair ? pair_tiles : single_tiles) * launch.n_tiles;
    const uint64_t group = kGroupBytes / (static_cast<uint64_t>(launch.pair ? 2 * kWideM : kWideM) * desc.k);
    const uint64_t row_blocks = launch.tiles / launch.n_tiles;
    launch.group_rows = static_cast<uint32_t>(std::min(std::max(group, kGroupRows), row_blocks));
    return launch;
}

// Which kernel? Up to 64 rows per expert, wide tiles once they fill the SMs: the wide kernel's deeper
// copies then stream the weights at least as fast (32 experts of 5632 x 2048 with 8 rows each: 70 us
// wide, 73 narrow; with 32 rows 77 against 104). One matrix takes the narrow kernel up to 32 rows, its
// tile. Beyond, the estimate of both in tenths of a microsecond: the blocks of K that a CTA walks
// through, 0.3 us each with two narrow CTAs an SM and 0.4 us each with a wide one, over the rounds of
// CTAs, what a further round of narrow CTAs costs (the wide ones stay), and what a split adds. Measured us, narrow and wide: one matrix of 2048 x 2048, 65 rows 7.5 and
// 9.4, 512 rows 11.2 and 12.5; 2048 x 5632, 128 rows 11.3 and 13.9, 192 rows 16.4 and 14.3; 1024 x 8192,
// 128 rows 9.9 and 16.2, 384 rows 20.7 and 16.7; 4096 x 4096, 64 rows 10.0 and 10.7, 65 rows 13.7 and
// 11.7; 11008 x 4096, 33 rows 17.7 and 14.6.
bool use_wide(const NarrowLaunch &narrow, const WideLaunch &wide, const GemmParams &params, uint64_t share, uint64_t filled, uint64_t sms) {
    if (filled > 1 && share <= 64) return share > 4 && filled * wide.n_tiles * 4 >= sms * 3;
    if (share <= 32) return false;
    const uint64_t tiles = static_cast<uint64_t>(narrow.tiles) * params.n_blocks;
    const uint64_t narrow_rounds = (tiles * narrow.split + 2 * sms - 1) / (2 * sms);
    const uint64_t narrow_time =
        (narrow.split > 1 ? 22 + 20 / narrow.split : 0) + 30 * (narrow_rounds - 1) + 3 * narrow_rounds * params.k_blocks / narrow.split;
    const uint64_t wide_rounds = (wide.tiles * (wide.pair ? 2 : wide.split) + sms - 1) / sms;
    const uint64_t wide_time = (wide.split > 1 ? 20 + 5 * wide.split : 15) + 4 * wide_rounds * params.k_blocks / wide.split;
    return wide_time < narrow_time;
}

cudaError_t launch_gemm(const qpucuda_fp8_gemm_desc &desc, const qpucuda_fp8_quantize_desc *quantize, unsigned int *error_word,
                        int sm_count, cudaStream_t stream) {
    const GemmParams params = gemm_params(desc, error_word);
    const uint64_t matrices = desc.experts != 0 ? desc.experts : 1u;
    const uint64_t filled = matrices < desc.rows ? matrices : desc.rows;  // matrices that can have rows
    const uint64_t share = (desc.rows + matrices - 1) / matrices;
    const uint64_t sms = static_cast<uint64_t>(sm_count);
    CUtensorMap map_w, map_a;
    const WideLaunch wide = plan_wide(desc, params, share, filled, sms);
    const NarrowLaunch narrow = plan_narrow(desc, params, share, filled, sms);
    if (use_wide(narrow, wide, params, share, filled, sms)) {
        if (quantize != nullptr) {
            const cudaError_t error = launch_fp8_quantize_rows(*quantize, sm_count, stream);
            if (error != cudaSuccess) return error;
        }
        if (wide.tiles > 0x3FFFFFFFull) return cudaErrorInvalidValue;
        if (!encode_tensor_map_2d_u8(&map_w, desc.w, desc.k, matrices * desc.n, desc.w_stride, kBlockK, kBlockN) ||
            !encode_tensor_map_2d_u8(&map_a, desc.a, desc.k, desc.rows, desc.a_stride, kBlockK, kWideM)) {
            return cudaErrorInvalidValue;
        }
        switch (desc.out_type) {
            case QPUCUDA_DTYPE_F32: return launch_wide_type<float>(map_w, map_a, params, wide, sm_count, stream);
            case QPUCUDA_DTYPE_BF16: return launch_wide_type<__nv_bfloat16>(map_w, map_a, params, wide, sm_count, stream);
            case QPUCUDA_DTYPE_F16: return launch_wide_type<__half>(map_w, map_a, params, wide, sm_count, stream);
        }
        return cudaErrorInvalidValue;
    }
    FusedRows fused{};
    bool fuse = false;
    if (quantize != nullptr) {
        const uint64_t blocks = (params.k_blocks + narrow.split - 1) / narrow.split;
        fuse = desc.experts == 0 && quantize->row_source == nullptr && narrow.tiles == 1 && narrow.height == 16 &&
               blocks <= kFusedBlocks &&
               blocks * desc.rows <= kFusedSteps * 4u * (quantize->x_type == QPUCUDA_DTYPE_F32 ? 1u : 2u);  // groups of a step
        if (fuse) {
            fused.x = quantize->x;
            fused.stride = quantize->x_stride;
            fused.type = quantize->x_type;
            fused.gated = quantize->gated != 0 ? 1u : 0u;
            fused.vector = fp8_vector_rows(*quantize) ? 1u : 0u;
        } else {
            const cudaError_t error = launch_fp8_quantize_rows(*quantize, sm_count, stream);
            if (error != cudaSuccess) return error;
        }
    }
    if (!encode_tensor_map_2d_u8(&map_w, desc.w, desc.k, matrices * desc.n, desc.w_stride, kBlockK, kBlockN)) return cudaErrorInvalidValue;
    if (fuse) {
        map_a = map_w;  // not used
    } else if (!encode_tensor_map_2d_u8(&map_a, desc.a, desc.k, desc.rows, desc.a_stride, kBlockK, static_cast<uint32_t>(narrow.height))) {
        return cudaErrorInvalidValue;
    }
    const FusedRows *rows = fuse ? &fused : nullptr;
    switch (desc.out_type) {
        case QPUCUDA_DTYPE_F32: return launch_narrow_rows<float>(map_w, map_a, params, narrow, rows, stream);
        case QPUCUDA_DTYPE_BF16: return launch_narrow_rows<__nv_bfloat16>(map_w, map_a, params, narrow, rows, stream);
        case QPUCUDA_DTYPE_F16: return launch_narrow_rows<__half>(map_w, map_a, params, narrow, rows, stream);
    }
    return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_fp8_gemm(const qpucuda_fp8_gemm_desc &desc, unsigned int *error_word, int sm_count, cudaStream_t stream) {
    return launch_gemm(desc, nullptr, error_word, sm_count, stream);
}

cudaError_t launch_fp8_linear(const qpucuda_fp8_quantize_desc &quantize, const qpucuda_fp8_gemm_desc &gemm, unsigned int *error_word,
                              int sm_count, cudaStream_t stream) {
    return launch_gemm(gemm, &quantize, error_word, sm_count, stream);
}

}  // namespace qpucuda
