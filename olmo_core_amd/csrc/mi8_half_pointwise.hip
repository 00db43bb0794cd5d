// What surrounds the products of 16-bit operands: copies of operands that 16-byte loads cannot take, and the gradient of their epilogue.
//
// Both are bound by memory; a lane takes eight consecutive columns.
#include "mi8_elements.h"

namespace mi8 {
namespace half {
namespace {

constexpr int kThreads = 256;
constexpr int kCols = 512;  // columns of a workgroup: eight a lane

__global__ __launch_bounds__(kThreads) void pad_kernel(const uint16_t* __restrict__ x, int64_t ld_x, int64_t rows, int cols, uint16_t* __restrict__ out, int64_t ld_out)
{
    const int64_t chunks = ld_out / 8, total = rows * chunks;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
        const int64_t r = i / chunks;
        const int c = (int)(i - r * chunks) * 8;
        Eight<Bf16> v;  // (bits)
        v.load(x + r * ld_x, c, cols);
        *reinterpret_cast<u32x4_t*>(out + r * ld_out + c) = v.v;
    }
}

struct EpilogueGrad {
    const uint16_t* grad;
    const uint16_t* z;
    uint16_t* dz;
    float* partial;  // [row chunks][N]
    int64_t ld_grad, ld_z, ld_dz, M;
    int N, act;
    int64_t chunk_rows;
};

// Workgroup (column block, row chunk): its four waves take every fourth row, two at a time, and their sums meet in LDS.
template <typename T>
__global__ __launch_bounds__(kThreads) void epilogue_grad_kernel(const EpilogueGrad p)
{
    __shared__ float sums[4][kCols];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c = (int)blockIdx.x * kCols + lane * 8;
    const int64_t first = (int64_t)blockIdx.y * p.chunk_rows, end = first + p.chunk_rows < p.M ? first + p.chunk_rows : p.M;
    constexpr int kRows = 2;
    float sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int64_t r0 = first + wave; r0 < end; r0 += 4 * kRows) {
        Eight<T> g8[kRows], z8[kRows];
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            const int64_t r = r0 + 4 * k;
            const int n = r < end ? p.N : 0;
            g8[k].load(p.grad + r * p.ld_grad, c, n);
            if (p.z) z8[k].load(p.z + r * p.ld_z, c, n);
        }
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            const int64_t r = r0 + 4 * k;
            float g[8];
            g8[k].get(g);
            if (p.z) {
                float z[8];
                z8[k].get(z);
                times_slope(p.act, z, g);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] += g[e];
            if (p.dz && r < end && c < p.ld_dz) *reinterpret_cast<u32x4_t*>(p.dz + r * p.ld_dz + c) = Eight<T>::pack(g);  // (zeros behind N)
        }
    }
    if (!p.partial) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[wave][lane * 8 + e] = sum[e];
    __syncthreads();
    for (int k = threadIdx.x; k < kCols; k += kThreads) {
        const int col = (int)blockIdx.x * kCols + k;
        if (col < p.N) p.partial[(int64_t)blockIdx.y * p.N + col] = (sums[0][k] + sums[1][k]) + (sums[2][k] + sums[3][k]);
    }
}

// out[c] = sum over the row chunks: 16 columns a workgroup, its 16 groups of lanes on every 16th chunk
__global__ __launch_bounds__(kThreads) void sum_chunks_kernel(const float* __restrict__ partial, int chunks, int N, void* out, int out_dtype)
{
    __shared__ float sums[16][16];
    const int c = (int)blockIdx.x * 16 + threadIdx.x % 16, k0 = threadIdx.x / 16;
    float s = 0.0f;
    if (c < N)
#pragma unroll 4
        for (int k = k0; k < chunks; k += 16) s += partial[(int64_t)k * N + c];
    sums[k0][threadIdx.x % 16] = s;
    __syncthreads();
    if (k0 != 0 || c >= N) return;
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < 16; ++k) s += sums[k][threadIdx.x];
    if (out_dtype == MI8_F32)
        static_cast<float*>(out)[c] = s;
    else
        static_cast<uint16_t*>(out)[c] = (uint16_t)(out_dtype == MI8_BF16 ? Bf16::pack(s, 0.0f) : F16::pack(s, 0.0f));
}

// C = act(the slices' sums + bias) + residual, eight columns of a row a lane
template <typename T>
__global__ __launch_bounds__(kThreads) void join_kernel(const HalfArgs p)
{
    const int chunks = (p.N + 7) / 8;
    const int64_t total = (int64_t)p.M * chunks;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
        const int64_t r = i / chunks;
        const int c = (int)(i - r * chunks) * 8;
        float row[1][8] = {};
        float(&f)[8] = row[0];
#pragma unroll 4
        for (int s = 0; s < p.slices; ++s) {
            const float* from = p.partial + ((int64_t)s * p.M + r) * p.ld_partial + c;
            const v4f a = *reinterpret_cast<const v4f*>(from), b = c + 4 < p.ld_partial ? *reinterpret_cast<const v4f*>(from + 4) : (v4f){0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                f[e] += a[e];
                f[4 + e] += b[e];
            }
        }
        float x[8];
        if (p.bias && p.bias_f32) {
            Eight<F32> b;
            b.load(p.bias, c, p.N);
            b.get(x);
        } else if (p.bias) {
            Eight<T> b;
            b.load(p.bias, c, p.N);
            b.get(x);
        }
        if (p.bias)
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] += x[e];
        if (p.z) Eight<T>::store(p.z + r * p.ldz, c, p.N, f);
        activate(p.act, row);
        if (p.residual) {
            Eight<T> b;
            b.load(p.residual + r * p.ldr, c, p.N);
            b.get(x);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] += x[e];
        }
        Eight<T>::store(p.C + r * p.ldc, c, p.N, f);
    }
}

// Row chunks of a column sum: as many as give about eight workgroups a compute unit, of at least 16 rows.
int64_t row_chunks(int64_t M, int64_t N)
{
    const int64_t wanted = ceil_div(2048, ceil_div(N, kCols)), most = ceil_div(M, 16);
    const int64_t n = wanted < most ? wanted : most;
    return n < 1 ? 1 : n;
}

}  // namespace

int launch_join(const HalfArgs& p, int hp_dtype, hipStream_t st)
{
    const int64_t blocks = ceil_div((int64_t)p.M * ((p.N + 7) / 8), kThreads);
    hipLaunchKernelGGL(hp_dtype == MI8_BF16 ? join_kernel<Bf16> : join_kernel<F16>, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(kThreads), 0, st, p);
    return launch_status("mi8_gemm_half");
}

}  // namespace half
}  // namespace mi8

using namespace mi8;

extern "C" int mi8_half_pad(const void* x, int64_t ld_x, int64_t rows, int64_t cols, void* out, int64_t ld_out, void* stream)
{
    MI8_REQUIRE(rows >= 0 && cols >= 0 && cols < (1 << 30), MI8_ERR_ARG, "mi8_half_pad: bad size");
    MI8_REQUIRE(ld_out >= cols && ld_out % 8 == 0 && aligned16(out), MI8_ERR_UNSUPPORTED, "mi8_half_pad: the copy needs 16-byte rows");
    if (rows == 0 || ld_out == 0) return MI8_OK;
    MI8_REQUIRE(x != nullptr && out != nullptr, MI8_ERR_ARG, "mi8_half_pad: null pointer");
    const int64_t blocks = ceil_div(rows * (ld_out / 8), half::kThreads);
    hipLaunchKernelGGL(half::pad_kernel, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(half::kThreads), 0, static_cast<hipStream_t>(stream),
                       static_cast<const uint16_t*>(x), ld_x, rows, (int)cols, static_cast<uint16_t*>(out), ld_out);
    return launch_status("mi8_half_pad");
}

extern "C" int64_t mi8_half_epilogue_grad_workspace_words(int64_t M, int64_t N) { return M <= 0 || N <= 0 ? 0 : half::row_chunks(M, N) * N; }

extern "C" int mi8_half_epilogue_grad(int hp_dtype, const void* grad, int64_t ld_grad, const void* z, int64_t ld_z, int activation, int64_t M, int64_t N, void* dz,
                                      int64_t ld_dz, void* bias_grad, int bias_dtype, float* workspace, void* stream)
{
    const char* what = "mi8_half_epilogue_grad";
    MI8_REQUIRE(hp_dtype == MI8_BF16 || hp_dtype == MI8_F16, MI8_ERR_ARG, "%s: element type %d is neither bf16 nor float16", what, hp_dtype);
    MI8_REQUIRE(M >= 0 && N >= 0 && N < (1 << 30) && ld_grad >= 0, MI8_ERR_ARG, "%s: bad size", what);
    MI8_REQUIRE(activation >= MI8_ACT_NONE && activation <= MI8_ACT_GELU_TANH, MI8_ERR_ARG, "%s: unknown activation %d", what, activation);
    MI8_REQUIRE(z == nullptr || ld_z >= N, MI8_ERR_ARG, "%s: z's pitch is smaller than its rows", what);
    MI8_REQUIRE(dz == nullptr || (ld_dz >= N && ld_dz < N + 512 && ld_dz % 8 == 0 && aligned16(dz)), MI8_ERR_UNSUPPORTED, "%s: dz needs 16-byte rows", what);
    MI8_REQUIRE(bias_grad == nullptr || bias_dtype == hp_dtype || bias_dtype == MI8_F32, MI8_ERR_ARG, "%s: the bias is float32 or of the operands' type", what);
    MI8_REQUIRE(bias_grad == nullptr || workspace != nullptr || M == 0 || N == 0, MI8_ERR_ARG, "%s: no workspace", what);
    if (N == 0 || (!dz && !bias_grad)) return MI8_OK;
    MI8_REQUIRE(grad != nullptr || M == 0, MI8_ERR_ARG, "%s: null pointer", what);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const int64_t chunks = M == 0 ? 0 : half::row_chunks(M, N);
    if (M > 0) {
        half::EpilogueGrad p{};
        p.grad = static_cast<const uint16_t*>(grad);
        p.z = static_cast<const uint16_t*>(z);
        p.dz = static_cast<uint16_t*>(dz);
        p.partial = bias_grad ? workspace : nullptr;
        p.ld_grad = ld_grad;
        p.ld_z = ld_z;
        p.ld_dz = ld_dz;
        p.M = M;
        p.N = (int)N;
        p.act = activation;
        p.chunk_rows = ceil_div(M, chunks);
        const dim3 grid((unsigned)ceil_div(dz && ld_dz > N ? ld_dz : N, half::kCols), (unsigned)chunks);
        auto kern = hp_dtype == MI8_BF16 ? half::epilogue_grad_kernel<half::Bf16> : half::epilogue_grad_kernel<half::F16>;
        hipLaunchKernelGGL(kern, grid, dim3(half::kThreads), 0, st, p);
        if (int rc = launch_status(what)) return rc;
    }
    if (!bias_grad) return MI8_OK;
    hipLaunchKernelGGL(half::sum_chunks_kernel, dim3((unsigned)ceil_div(N, 16)), dim3(half::kThreads), 0, st, workspace, (int)chunks, (int)N, bias_grad, bias_dtype);
    return launch_status(what);
}
