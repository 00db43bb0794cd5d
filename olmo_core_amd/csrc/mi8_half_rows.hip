// Products of up to 16 rows, both operands by rows: y = x W^T for a generation loop's handful of tokens.
//
// The time is reading W once.  Tiles would give it to as many compute units as W has blocks of 64 rows, each walking all of K with the latency of
// its steps (4096 -> 4096: 18 us where the read takes 7, 11008 -> 4096 41 where it takes 18).  Here a workgroup has 16 rows of W and its eight waves an
// eighth of K each: they stream disjoint pieces of W straight into MFMA operands, the loads of eight steps in flight, and their sums meet in LDS (4096 -> 4096
// 8.6 us, 11008 -> 4096 18.1; 16 rows of x, which every workgroup reads out of the L2, 11.3 and 23.9).  A W of many rows fills the chip with
// tiles, which then read it at 4.8 TB/s (4096 -> 11008 18.7 us, here 22.2).
//
// Rows of x past the last one are zeros that are not loaded, rows of W past the edge repeat the last one and are not stored, K past the end is zeros.
#include "mi8_elements.h"

namespace mi8 {
using namespace gemm;
namespace half {
namespace {

constexpr int kWaves = 8;
constexpr int kBatch = 4;  // steps of 64 K loaded at a time, two such batches in registers

template <typename T>
__global__ __launch_bounds__(kWaves * 64) void half_rows_kernel(const HalfArgs p)
{
    __shared__ v4f sums[kWaves][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, kb = lane >> 4;
    const int n0 = (int)blockIdx.x * 16;
    const int steps = (p.K + kStepK - 1) / kStepK, per = (steps + kWaves - 1) / kWaves;
    const int from = wave * per, to = from + per < steps ? from + per : steps;
    const bool here = r16 < p.M;
    const uint8_t* const wp = p.B + ((int64_t)(n0 + r16 < p.N ? n0 + r16 : p.N - 1) * p.ldb + kb * 16) * 2;
    const uint8_t* const xp = p.A + ((int64_t)(here ? r16 : 0) * p.lda + kb * 16) * 2;

    v4f acc = {0, 0, 0, 0};
    v4i fx[2][kBatch][2], fw[2][kBatch][2];
    auto load = [&](auto set_tag, int s0) __attribute__((always_inline)) {
        constexpr int S = decltype(set_tag)::value;
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int64_t at = (int64_t)(s0 + u) * (kStepK * 2) + q * 16;
                const bool in = s0 + u < to && (s0 + u) * kStepK + kb * 16 + q * 8 < p.K;
                fw[S][u][q] = in ? *reinterpret_cast<const v4i*>(wp + at) : (v4i){0, 0, 0, 0};
                fx[S][u][q] = in && here ? *reinterpret_cast<const v4i*>(xp + at) : (v4i){0, 0, 0, 0};
            }
    };
    auto multiply = [&](auto set_tag) __attribute__((always_inline)) {
        constexpr int S = decltype(set_tag)::value;
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
#pragma unroll
            for (int q = 0; q < 2; ++q) acc = mma<T>(fw[S][u][q], fx[S][u][q], acc);
    };
    const std::integral_constant<int, 0> set0;
    const std::integral_constant<int, 1> set1;
    load(set0, from);
    for (int s = from; s < to; s += 2 * kBatch) {
        load(set1, s + kBatch);
        multiply(set0);
        if (s + kBatch >= to) break;  // (uniform)
        load(set0, s + 2 * kBatch);
        multiply(set1);
    }
    sums[wave][lane] = acc;
    __syncthreads();
    if (wave != 0 || !here) return;
    // element j of lane l is C[l % 16][4 (l / 16) + j]
    v4f v = sums[0][lane];
#pragma unroll
    for (int k = 1; k < kWaves; ++k) v += sums[k][lane];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int c = n0 + 4 * kb + j;
        if (c >= p.N) continue;
        float f = v[j];
        if (p.bias) f += p.bias_f32 ? reinterpret_cast<const float*>(p.bias)[c] : T::lo(reinterpret_cast<const uint16_t*>(p.bias)[c]);
        if (p.z) p.z[r16 * p.ldz + c] = (uint16_t)T::pack(f, 0.0f);
        f = activate(p.act, f);
        if (p.residual) f += T::lo(p.residual[r16 * p.ldr + c]);
        p.C[r16 * p.ldc + c] = (uint16_t)T::pack(f, 0.0f);
    }
}

}  // namespace

int launch_rows(const HalfArgs& p, int hp_dtype, hipStream_t st)
{
    hipLaunchKernelGGL(hp_dtype == MI8_BF16 ? half_rows_kernel<Bf16> : half_rows_kernel<F16>, dim3((unsigned)ceil_div(p.N, 16)), dim3(kWaves * 64), 0, st, p);
    return launch_status("mi8_gemm_half");
}

}  // namespace half
}  // namespace mi8
