// Products of 16-bit operands (bf16, float16): argument block, element types, the epilogue's activations.
#pragma once
#include <type_traits>

#include "mi8_gemm.h"

namespace mi8 {
namespace half {

constexpr int kStepK = 64;  // elements of K per LDS stage: 128 bytes of every row

// C[M, N] = act(A . B^T + bias) + residual.  Either operand lies with its K contiguous ([rows][K], "by rows") or with its rows contiguous
// ([K][rows], "by K"); pitches are in elements and multiples of 8, addresses of 16 bytes.
//   sizes, rows in groups (A by rows): rows of A and C are in E groups, group e is multiplied with B + e * b_group_stride;
//          rows behind the last group give zeros
//   sizes, K in groups (both by K): C[e] = A[K of e]^T . B[K of e], matrices of M x N one after the other
struct HalfArgs {
    const uint8_t* A;
    const uint8_t* B;
    uint16_t* C;
    int64_t lda, ldb, ldc;
    int M, N, K;
    const int64_t* sizes;
    int E;
    int64_t b_group_stride;  // elements
    const void* bias;        // [N]; null: none
    int bias_f32;
    const uint16_t* residual;
    int64_t ldr;
    int act;  // mi8_activation
    uint16_t* z;  // null, or where A . B^T + bias goes
    int64_t ldz;
    int tiles_m, tiles_n;
    // K in slices (no groups): slice s sums slice_k (a multiple of the step) of K into partial [s][M][ld_partial], which launch_join adds up
    int slices, slice_k;
    float* partial;  // null: one slice, straight to C
    int64_t ld_partial;  // a multiple of 4
    int wide;  // C, z and residual take 16 bytes at multiples of 8 columns
};

struct Bf16 {
    static constexpr int kCode = MI8_BF16;
    static __device__ __forceinline__ float lo(uint32_t v) { return bits_to_f32(v << 16); }
    static __device__ __forceinline__ float hi(uint32_t v) { return bits_to_f32(v & 0xFFFF0000u); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16(a, b); }
};
struct F16 {
    static constexpr int kCode = MI8_F16;
    typedef _Float16 pair_t __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ float lo(uint32_t v) { return (float)__builtin_bit_cast(pair_t, v)[0]; }
    static __device__ __forceinline__ float hi(uint32_t v) { return (float)__builtin_bit_cast(pair_t, v)[1]; }
    static __device__ __forceinline__ uint32_t pack(float a, float b) { return __builtin_bit_cast(uint32_t, (pair_t){(_Float16)a, (_Float16)b}); }
};

typedef float v4f __attribute__((ext_vector_type(4)));

// D += first . second^T of 16 rows x 32 K each: lane l has row l % 16, eight K from a place that follows from l / 16
template <typename T>
__device__ __forceinline__ v4f mma(const gemm::v4i& first, const gemm::v4i& second, const v4f& c)
{
#ifdef __HIP_DEVICE_COMPILE__
    if constexpr (T::kCode == MI8_BF16) {
        typedef __bf16 v8 __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, first), __builtin_bit_cast(v8, second), c, 0, 0, 0);
    } else {
        typedef _Float16 v8 __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, first), __builtin_bit_cast(v8, second), c, 0, 0, 0);
    }
#else
    return c;
#endif
}

// The same with the accumulator tied to the result, in accumulator registers: left to the register allocator, a share of 64 accumulators is copied in and
// out of ordinary registers around every step.  (The compiler does not know when the result is there: whoever reads it next waits.)
template <typename T>
__device__ __forceinline__ void mma_tied(const gemm::v4i& first, const gemm::v4i& second, v4f& c, bool fresh)
{
    if constexpr (T::kCode == MI8_BF16) {
        if (fresh)
            asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, 0" : "=a"(c) : "v"(first), "v"(second));
        else
            asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(first), "v"(second));
    } else {
        if (fresh)
            asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, 0" : "=a"(c) : "v"(first), "v"(second));
        else
            asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(first), "v"(second));
    }
}

// ---- activations.  All in float32 on the hardware's exponential and reciprocal (within about 1 and 2 units in the last place).

__device__ __forceinline__ float exp_neg(float x) { return __builtin_amdgcn_exp2f(x * -1.4426950408889634f); }  // e^-x

// 1 / (1 + e^-x): e^-x overflows to infinity for large negative x, whose reciprocal is 0
__device__ __forceinline__ float logistic(float x) { return __builtin_amdgcn_rcpf(1.0f + exp_neg(x)); }

// A float32 whose products with itself stay finite; a NaN passes through
__device__ __forceinline__ float tamed(float x) { return clamp_keep_nan(x, 1e4f); }

// The normal distribution's upper tail q = erfc(|x| / sqrt 2) / 2 and e = exp(-x^2 / 2).  q / e is smooth in t = 1 / (1 + 0.265 |x|) and goes to 0
// with it: t times a polynomial of degree 6, fitted for least relative error over |x| = 0 .. 14, beyond which e is 0 in float32 (with the
// rounding of its evaluation within 1e-6, where bf16 and float16 values have half steps of 2e-3 and 5e-4).
struct NormalTail {
    float q, e;
};
__device__ __forceinline__ NormalTail normal_tail(float x)
{
    const float e = __builtin_amdgcn_exp2f(x * x * -0.72134752f);
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.265f, __builtin_fabsf(x), 1.0f));
    float p = -0.06778666078457006f;
    p = __builtin_fmaf(p, t, 0.19527177f);
    p = __builtin_fmaf(p, t, -0.06636097974606796f);
    p = __builtin_fmaf(p, t, 0.14249185322351035f);
    p = __builtin_fmaf(p, t, 0.0829472170053685f);
    p = __builtin_fmaf(p, t, 0.10783664227949369f);
    p = __builtin_fmaf(p, t, 0.10559984701564744f);
    return NormalTail{p * t * e, e};
}

constexpr float kTanhC = 1.5957691216057308f;  // 2 sqrt(2 / pi): (1 + tanh(u)) / 2 = logistic(2 u)
constexpr float kTanhCube = 0.044715f;

__device__ __forceinline__ float activate(int act, float x)
{
    switch (act) {  // (uniform)
        case MI8_ACT_RELU: return x <= 0.0f ? 0.0f : x;
        case MI8_ACT_SILU: return x * logistic(x);
        case MI8_ACT_GELU: {
            const NormalTail n = normal_tail(x);
            return x * (x > 0.0f ? 1.0f - n.q : n.q);
        }
        case MI8_ACT_GELU_TANH: {
            const float c = tamed(x);
            return x * logistic(kTanhC * c * __builtin_fmaf(kTanhCube * c, c, 1.0f));
        }
        default: return x;
    }
}

// (ReLU has none here: times_slope() chooses)
__device__ __forceinline__ float activation_slope(int act, float x)
{
    const float c = tamed(x);
    if (act == MI8_ACT_SILU) {
        const float s = logistic(c);
        return s * __builtin_fmaf(c, 1.0f - s, 1.0f);
    }
    if (act == MI8_ACT_GELU) {
        const NormalTail n = normal_tail(c);
        return __builtin_fmaf(c * 0.3989422804f, n.e, c > 0.0f ? 1.0f - n.q : n.q);
    }
    if (act == MI8_ACT_GELU_TANH) {
        const float cube = kTanhCube * c * c, s = logistic(kTanhC * c * (1.0f + cube));
        return s * __builtin_fmaf(c * (1.0f - s) * kTanhC, __builtin_fmaf(3.0f, cube, 1.0f), 1.0f);
    }
    return 1.0f;
}

// One choice of the function for many elements: a choice for each costs more than the function does (float16, 16384 x 1024 -> 2816, 256 x 256 tiles:
// no activation 98 us; SiLU 143 with a choice for each element, 106 with one for 32; the exact GELU 166 and 120).
template <typename F>
__device__ __forceinline__ void for_act(int act, F&& f)
{
    switch (act) {  // (uniform)
        case MI8_ACT_RELU: f(std::integral_constant<int, MI8_ACT_RELU>{}); break;
        case MI8_ACT_SILU: f(std::integral_constant<int, MI8_ACT_SILU>{}); break;
        case MI8_ACT_GELU: f(std::integral_constant<int, MI8_ACT_GELU>{}); break;
        case MI8_ACT_GELU_TANH: f(std::integral_constant<int, MI8_ACT_GELU_TANH>{}); break;
        default: break;
    }
}
template <int ROWS>
__device__ __forceinline__ void activate(int act, float (&x)[ROWS][8])
{
    for_act(act, [&](auto tag) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < ROWS; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) x[k][e] = activate(decltype(tag)::value, x[k][e]);
    });
}
__device__ __forceinline__ void times_slope(int act, const float (&x)[8], float (&g)[8])
{
    for_act(act, [&](auto tag) __attribute__((always_inline)) {
        constexpr int kAct = decltype(tag)::value;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (kAct == MI8_ACT_RELU)
                g[e] = x[e] <= 0.0f ? 0.0f : g[e];  // (a product would make NaN of an infinite gradient where the unit is off)
            else
                g[e] *= activation_slope(kAct, x[e]);
        }
    });
}

// mi8_half_gemm.hip; variant: a mi8_half_variant
int launch_tiles(const HalfArgs& p, int hp_dtype, bool a_by_k, bool b_by_k, int variant, hipStream_t st);
// mi8_half_rows.hip: both operands by rows, up to kMostRows rows of A
constexpr int kMostRows = 16;
int launch_rows(const HalfArgs& p, int hp_dtype, hipStream_t st);
// mi8_half_pointwise.hip: C from the partial sums of p.slices slices of K
int launch_join(const HalfArgs& p, int hp_dtype, hipStream_t st);

}  // namespace half
}  // namespace mi8
