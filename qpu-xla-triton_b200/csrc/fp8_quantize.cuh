// e4m3 groups of 128 columns: the arithmetic shared by the quantizer kernels and by the product that
// quantizes its own rows, so that both give the same bytes and scales.
#pragma once

#include <cuda_fp8.h>

#include "element.cuh"
#include "sm100_fp8.cuh"

namespace qpucuda {

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

// e4m3(RN(x / s)) of N values, two to an instruction. A hardware division per value, or a branch to
// one near the borders of e4m3 (bf16 values over a bf16 maximum lie on borders in 1 of 500 cases, so
// half of the warps took it), costs more than the copy itself. Markstein's correction instead, twice:
// with y = RN(1 / s), q1 = RN(q0 + (x - q0 s) y) is within one step of x / s, its remainder is exact in
// an fma, and RN(q1 + (x - q1 s) y) is the rounded quotient (Markstein 1990). That needs remainders
// above the smallest normal number: true for every quotient above 2^-10, the smallest border of e4m3,
// as s is at least 2^-60; smaller quotients end as zero whatever their last bits.
//
// The steps run on n = -q: the last of them adds remainder * -y to n, which for x = -0 is -0 + (+0), the
// negative of the wanted -0; on q itself the sum of -0 and +0 would lose the sign. The four signs of a word
// are turned at the end, but for a group of NaNs, whose bytes stay 0x7F.
template <int N>
__device__ __forceinline__ void quantize_values(const float (&v)[N], float scale, uint32_t (&packed)[N / 4]) {
    using sm100::fma2;
    using sm100::pack2;
    const float inverse = __frcp_rn(scale);
    const uint64_t minus_y = pack2(-inverse, -inverse), s = pack2(scale, scale), zero = pack2(-0.0f, -0.0f);
    const uint32_t signs = scale == scale ? 0x80808080u : 0u;
    uint16_t pairs[N / 2];
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const uint64_t x = pack2(v[i], v[i + 1]);
        uint64_t n = fma2(x, minus_y, zero);
        n = fma2(fma2(n, s, x), minus_y, n);
        n = fma2(fma2(n, s, x), minus_y, n);
        pairs[i / 2] = __nv_cvt_float2_to_fp8x2(make_float2(sm100::low(n), sm100::high(n)), __NV_SATFINITE, __NV_E4M3);
    }
#pragma unroll
    for (int i = 0; i < N / 4; ++i) packed[i] = (pairs[2 * i] | (static_cast<uint32_t>(pairs[2 * i + 1]) << 16)) ^ signs;
}

__device__ __forceinline__ float reciprocal(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// v = silu(v) * up = v / (1 + exp(-v)) * up in fp32, every step to the last bit: a value that the
// quantizer then rounds to three bits should not land on the other side of a border for an
// approximation's sake. The quotient is Markstein's: q0 = g y with y within 2^-23 of 1 / d, corrected
// by its exact remainder, is within 2^-45 of g / d before it is rounded; as above its negative is
// formed, and multiplied by -up. Below -87 the denominator's
// reciprocal is no normal number, and the hardware's division (-0 once exp overflows) takes over.
// 4096 x 8192 bf16: 39 us, with a division per value 46, with the fast exp and quotient 31.
template <int N>
__device__ __forceinline__ void silu_times(float (&v)[N], const float (&up)[N]) {
    using sm100::fma2;
    using sm100::pack2;
    float least = 0.0f, d[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        d[i] = __fadd_rn(1.0f, expf(-v[i]));
        least = fminf(least, v[i]);
    }
    if (least < -87.0f) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __fmul_rn(__fdiv_rn(v[i], d[i]), up[i]);
        return;
    }
    const uint64_t zero = pack2(-0.0f, -0.0f);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const uint64_t g = pack2(v[i], v[i + 1]), minus_y = pack2(reciprocal(-d[i]), reciprocal(-d[i + 1]));
        uint64_t n = fma2(g, minus_y, zero);
        n = fma2(fma2(n, pack2(d[i], d[i + 1]), g), minus_y, n);
        v[i] = __fmul_rn(sm100::low(n), -up[i]);
        v[i + 1] = __fmul_rn(sm100::high(n), -up[i + 1]);
    }
}

// 16 bytes at x in the widest words that its alignment allows: in Words, or, two bytes off a word, in three
// words between two halves.
template <typename Word, typename T>
__device__ __forceinline__ uint4 load_words(const T *x) {
    constexpr int kWords = 16 / sizeof(Word);
    alignas(16) Word words[kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i) words[i] = reinterpret_cast<const Word *>(x)[i];
    return *reinterpret_cast<const uint4 *>(words);
}
template <typename T>
__device__ __forceinline__ uint4 load_halves(const T *x) {
    const uint16_t *halves = reinterpret_cast<const uint16_t *>(x);
    const uint32_t *words = reinterpret_cast<const uint32_t *>(halves + 1);
    const uint32_t first = halves[0], a = words[0], b = words[1], c = words[2], last = halves[7];
    return make_uint4(first | (a << 16), __funnelshift_r(a, b, 16), __funnelshift_r(b, c, 16), (c >> 16) | (last << 16));
}

// kVector elements at x, zero from `remaining` of them on. Full vectors first and the ragged end of a
// row in a pass of its own, so that nothing stands between the loads of several steps. Unaligned rows:
// the alignment is the same for all lanes of a row, which are 16 bytes apart (4096 x 8191 bf16 22 us, 33
// element by element).
template <typename T, bool VECTOR, int STEPS>
__device__ __forceinline__ void load_steps(const T *x, uint32_t remaining, uint32_t step, Vector<T> (&raw)[STEPS]) {
    constexpr uint32_t kItems = kVector<T>;
    auto each = [&](auto load) {
#pragma unroll
        for (int u = 0; u < STEPS; ++u) {
            raw[u].bits = make_uint4(0, 0, 0, 0);
            if (remaining >= u * step + kItems) raw[u].bits = load(x + u * step);
        }
    };
    const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(x));
    if (VECTOR) {
        each([](const T *at) { return load_stream16(at); });
    } else if ((off & 7u) == 0) {
        each([](const T *at) { return load_words<uint2>(at); });
    } else if (sizeof(T) == 4 || (off & 3u) == 0) {
        each([](const T *at) { return load_words<uint32_t>(at); });
    } else {
        each([](const T *at) { return load_halves(at); });
    }
    if (remaining % step != 0 && remaining % step < kItems) {
#pragma unroll
        for (int u = 0; u < STEPS; ++u) {
            const uint32_t left = remaining > u * step ? remaining - u * step : 0u;
            if (left < kItems) {
#pragma unroll
                for (uint32_t i = 0; i < kItems; ++i)
                    if (i < left) raw[u].items[i] = x[u * step + i];
            }
        }
    }
}

// The group's maximum, with each of its lanes holding some of its values' maximum.
template <int LANES>
__device__ __forceinline__ float group_max(float amax) {
#pragma unroll
    for (int offset = LANES / 2; offset > 0; offset >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, offset));
    return amax;
}

}  // namespace qpucuda
