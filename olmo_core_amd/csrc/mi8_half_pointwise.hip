// What surrounds the products of 16-bit operands: copies of operands that 16-byte loads cannot take, and the gradient of their epilogue.
//
// Both are bound by memory.  Rows whose pitch and address are whole 16-byte chunks are read eight columns a lane; others an element a lane, consecutive
// lanes on consecutive columns.
#include "mi8_half.h"

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
        const uint16_t* src = x + r * ld_x + c;
        uint32_t v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = c + e < cols ? src[e] : 0;
        *reinterpret_cast<uint4*>(out + r * ld_out + c) = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
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

// Workgroup (column block, row chunk): its four waves take every fourth row, and their sums meet in LDS.
template <typename T, bool WIDE>
__global__ __launch_bounds__(kThreads) void epilogue_grad_kernel(const EpilogueGrad p)
{
    __shared__ float sums[4][kCols];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c0 = (int)blockIdx.x * kCols;
    const int64_t first = (int64_t)blockIdx.y * p.chunk_rows, end = first + p.chunk_rows < p.M ? first + p.chunk_rows : p.M;
    // column e of this lane
    auto column = [&](int e) __attribute__((always_inline)) { return c0 + (WIDE ? lane * 8 + e : e * 64 + lane); };
    float sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int64_t r = first + wave; r < end; r += 4) {
        float g[8], z[8];
        if constexpr (WIDE) {
            const int c = c0 + lane * 8;
            uint4 a = make_uint4(0, 0, 0, 0), b = a;
            if (c < p.N) {
                a = load_stream16(p.grad + r * p.ld_grad + c);
                if (p.z) b = load_stream16(p.z + r * p.ld_z + c);
            }
            const uint32_t ga[4] = {a.x, a.y, a.z, a.w}, za[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                g[2 * e] = T::lo(ga[e]);
                g[2 * e + 1] = T::hi(ga[e]);
                z[2 * e] = T::lo(za[e]);
                z[2 * e + 1] = T::hi(za[e]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool in = column(e) < p.N;
                g[e] = in ? T::lo(p.grad[r * p.ld_grad + column(e)]) : 0.0f;
                z[e] = in && p.z ? T::lo(p.z[r * p.ld_z + column(e)]) : 0.0f;
            }
        }
        if (p.z)
#pragma unroll
            for (int e = 0; e < 8; ++e) g[e] *= activation_slope(p.act, z[e]);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += g[e];
        if (!p.dz) continue;
        if constexpr (WIDE) {
            const int c = c0 + lane * 8;
            if (c < p.ld_dz)
                *reinterpret_cast<uint4*>(p.dz + r * p.ld_dz + c) = make_uint4(T::pack(g[0], g[1]), T::pack(g[2], g[3]), T::pack(g[4], g[5]), T::pack(g[6], g[7]));
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (column(e) < p.ld_dz) p.dz[r * p.ld_dz + column(e)] = (uint16_t)T::pack(g[e], 0.0f);  // (zeros behind N)
        }
    }
    if (!p.partial) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[wave][column(e) - c0] = sum[e];
    __syncthreads();
    for (int c = threadIdx.x; c < kCols; c += kThreads)
        if (c0 + c < p.N) p.partial[(int64_t)blockIdx.y * p.N + c0 + c] = (sums[0][c] + sums[1][c]) + (sums[2][c] + sums[3][c]);
}

// out[c] = sum over the row chunks: 64 columns a workgroup, its waves on every fourth chunk
__global__ __launch_bounds__(kThreads) void sum_chunks_kernel(const float* __restrict__ partial, int chunks, int N, void* out, int out_dtype)
{
    __shared__ float sums[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = (int)blockIdx.x * 64 + lane;
    float s = 0.0f;
    if (c < N)
        for (int k = wave; k < chunks; k += 4) s += partial[(int64_t)k * N + c];
    sums[wave][lane] = s;
    __syncthreads();
    if (wave != 0 || c >= N) return;
    s = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
    if (out_dtype == MI8_F32)
        static_cast<float*>(out)[c] = s;
    else
        static_cast<uint16_t*>(out)[c] = (uint16_t)(out_dtype == MI8_BF16 ? Bf16::pack(s, 0.0f) : F16::pack(s, 0.0f));
}

// Row chunks of a column sum: as many as give about four workgroups a compute unit, of at least 32 rows.
int64_t row_chunks(int64_t M, int64_t N)
{
    const int64_t wanted = ceil_div(1024, ceil_div(N, kCols)), most = ceil_div(M, 32);
    const int64_t n = wanted < most ? wanted : most;
    return n < 1 ? 1 : n;
}

}  // namespace
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
        const bool wide = N % 8 == 0 && ld_grad % 8 == 0 && aligned16(grad) && (!z || (ld_z % 8 == 0 && aligned16(z)));
        const dim3 grid((unsigned)ceil_div(dz && ld_dz > N ? ld_dz : N, half::kCols), (unsigned)chunks);
        auto kern = hp_dtype == MI8_BF16 ? (wide ? half::epilogue_grad_kernel<half::Bf16, true> : half::epilogue_grad_kernel<half::Bf16, false>)
                                         : (wide ? half::epilogue_grad_kernel<half::F16, true> : half::epilogue_grad_kernel<half::F16, false>);
        hipLaunchKernelGGL(kern, grid, dim3(half::kThreads), 0, st, p);
        if (int rc = launch_status(what)) return rc;
    }
    if (!bias_grad) return MI8_OK;
    hipLaunchKernelGGL(half::sum_chunks_kernel, dim3((unsigned)ceil_div(N, 64)), dim3(half::kThreads), 0, st, workspace, (int)chunks, (int)N, bias_grad, bias_dtype);
    return launch_status(what);
}
