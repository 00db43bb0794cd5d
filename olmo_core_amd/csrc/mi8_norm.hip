// A block's output on its way into the residual stream, and the norm in front of the next block, in one pass over the data:
//
//     v = norm(branch) post        norm(a) = a rsqrt(mean(a^2) + eps)
//     h = residual_scale residual + scale gate drop(v)
//     n = norm(h) pre
//
// and the gradients of all its inputs, every part optional.  With a = the row, hat = norm(a), y = hat w: the gradient of a norm is
//     da = rsqrt(..) (dy w - hat mean(dy w hat)),   dw = sum over rows of dy hat.
//
// Bound by memory: forward one read of branch and residual, one write of h and n; backward one read of branch, h and the two gradients, one
// write of the inputs' gradients.  A row lives in the registers of the lanes that own it (16 lanes to 1024, up to four chunks of eight elements each); the
// statistics are float32 sums over those lanes, and h is rounded to its type only when it is stored: the second norm sees it unrounded.
// The backward takes hat = h rsqrt(..) from the stored h and the forward's rsqrt.  The dropped elements are made again from the counter (mi8_philox.h).
//
// Sums over rows (post, pre, gate): every workgroup keeps them for the rows it walks in registers, column by column, writes them out once, and a second
// launch adds the workgroups' in order: no atomics, the same bits on every run.
#include "mi8_elements.h"
#include "mi8_philox.h"

namespace mi8 {
namespace {

struct NormArgs {
    const uint8_t* branch;
    const uint8_t* residual;
    uint8_t* stream;
    uint8_t* normed;
    int64_t ld_branch, ld_residual;  // bytes
    const void *post, *pre, *gate;
    int post_f32, pre_f32, gate_f32;
    int post_norm, pre_norm;
    int64_t rows;
    int D;
    float scale, residual_scale, eps;
    Dropout drop;
    float *branch_rstd, *stream_rstd;  // [rows]; forward: may be null
    // gradients
    const uint8_t *stream_grad, *normed_grad;
    int64_t ld_stream_grad, ld_normed_grad;
    uint8_t *branch_grad, *residual_grad;
    float* partial;  // [workgroups][3][D]: post, pre, gate; null: none wanted
    int want_post, want_pre, want_gate;
};

// Eight weights (float32, or T) of columns c .. c + 7
template <typename T, bool WIDE>
__device__ __forceinline__ void load_weight(const void* w, int f32, int c, int n, float (&f)[8])
{
    if (f32) {
        Eight<F32> r;
        r.template load<WIDE>(w, c, n);
        r.get(f);
    } else {
        Eight<T> r;
        r.template load<WIDE>(w, c, n);
        r.get(f);
    }
}

// Sum over the LANES lanes that own a row.  More than a wave: through LDS, in turns of two places (a barrier of the other place lies between two uses).
template <int LANES>
struct RowSum {
    int turn = 0;
    __device__ __forceinline__ float operator()(float v)
    {
#pragma unroll
        for (int off = (LANES < 64 ? LANES : 64) / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
        if constexpr (LANES > 64) {
            constexpr int W = LANES / 64;
            __shared__ float sums[2][W];
            const int wave = threadIdx.x >> 6;
            if ((threadIdx.x & 63) == 0) sums[turn][wave] = v;
            __syncthreads();
            v = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w) v += sums[turn][w];
            turn ^= 1;
        }
        return v;
    }
};

template <int LANES>
constexpr int kBlock = LANES <= 64 ? 256 : LANES;  // threads of a workgroup

template <typename TB, typename TS, int LANES, int CHUNKS, bool WIDE>
__global__ __launch_bounds__(kBlock<LANES>) void norm_forward_kernel(const NormArgs p)
{
    constexpr int kRows = kBlock<LANES> / LANES;
    const int t = threadIdx.x % LANES, D = p.D;
    const uint64_t key = p.drop.seed_on_device ? (uint64_t)p.drop.seed_on_device[0] : p.drop.seed;
    const float inv_d = 1.0f / (float)D;
    RowSum<LANES> row_sum;
    for (int64_t row0 = (int64_t)blockIdx.x * kRows; row0 < p.rows; row0 += (int64_t)gridDim.x * kRows) {
        const int64_t r = row0 + threadIdx.x / LANES;
        const bool live = r < p.rows;
        const int n = live ? D : 0;  // (lanes of a row past the last one load zeros and store nothing)
        Eight<TB> raw_u[CHUNKS];
        Eight<TS> raw_r[CHUNKS];
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j) raw_u[j].template load<WIDE>(p.branch + r * p.ld_branch, (j * LANES + t) * 8, n);
        if (p.residual)
#pragma unroll
            for (int j = 0; j < CHUNKS; ++j) raw_r[j].template load<WIDE>(p.residual + r * p.ld_residual, (j * LANES + t) * 8, n);
        float h[CHUNKS][8];
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j) raw_u[j].get(h[j]);
        if (p.post_norm) {
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < CHUNKS; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) s = __builtin_fmaf(h[j][e], h[j][e], s);
            const float rstd = rsqrtf(row_sum(s) * inv_d + p.eps);
            if (p.branch_rstd && live && t == 0) p.branch_rstd[r] = rstd;
#pragma unroll
            for (int j = 0; j < CHUNKS; ++j) {
#pragma unroll
                for (int e = 0; e < 8; ++e) h[j][e] *= rstd;
                if (p.post) {
                    float w[8];
                    load_weight<TB, WIDE>(p.post, p.post_f32, (j * LANES + t) * 8, D, w);
#pragma unroll
                    for (int e = 0; e < 8; ++e) h[j][e] *= w[e];
                }
            }
        }
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j) {
            const int c = (j * LANES + t) * 8;
            if (p.drop.threshold) {
                const uint32_t m = kept8(r * D + c, p.drop.offset, key, p.drop.threshold);
#pragma unroll
                for (int e = 0; e < 8; ++e) h[j][e] = m >> e & 1 ? h[j][e] * p.drop.factor : 0.0f;
            }
            if (p.gate) {
                float w[8];
                load_weight<TB, WIDE>(p.gate, p.gate_f32, c, D, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) h[j][e] *= w[e];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) h[j][e] *= p.scale;
            if (p.residual) {
                float x[8];
                raw_r[j].get(x);
#pragma unroll
                for (int e = 0; e < 8; ++e) h[j][e] = __builtin_fmaf(p.residual_scale, x[e], h[j][e]);
            }
            if (p.stream) Eight<TS>::template store<WIDE>(p.stream + r * D * Eight<TS>::kBytes, c, n, h[j]);
#pragma unroll
            for (int e = 0; e < 8; ++e) s = __builtin_fmaf(h[j][e], h[j][e], s);
        }
        if (!p.pre_norm) continue;
        const float rstd = rsqrtf(row_sum(s) * inv_d + p.eps);
        if (p.stream_rstd && live && t == 0) p.stream_rstd[r] = rstd;
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j) {
            const int c = (j * LANES + t) * 8;
#pragma unroll
            for (int e = 0; e < 8; ++e) h[j][e] *= rstd;
            if (p.pre) {
                float w[8];
                load_weight<TB, WIDE>(p.pre, p.pre_f32, c, D, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) h[j][e] *= w[e];
            }
            Eight<TB>::template store<WIDE>(p.normed + r * D * Eight<TB>::kBytes, c, n, h[j]);
        }
    }
}

template <typename TB, typename TS, int LANES, int CHUNKS, bool WIDE>
__global__ __launch_bounds__(kBlock<LANES>) void norm_backward_kernel(const NormArgs p)
{
    constexpr int kRows = kBlock<LANES> / LANES;
    const int t = threadIdx.x % LANES, D = p.D;
    const uint64_t key = p.drop.seed_on_device ? (uint64_t)p.drop.seed_on_device[0] : p.drop.seed;
    const float inv_d = 1.0f / (float)D;
    const bool need_u = p.post_norm || p.want_gate;
    RowSum<LANES> row_sum;
    float post_sum[CHUNKS][8] = {}, pre_sum[CHUNKS][8] = {}, gate_sum[CHUNKS][8] = {};
    for (int64_t row0 = (int64_t)blockIdx.x * kRows; row0 < p.rows; row0 += (int64_t)gridDim.x * kRows) {
        const int64_t r = row0 + threadIdx.x / LANES;
        const bool live = r < p.rows;
        const int n = live ? D : 0;
        Eight<TS> raw_dh[CHUNKS], raw_h[CHUNKS];
        Eight<TB> raw_dn[CHUNKS], raw_u[CHUNKS];
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j) {
            const int c = (j * LANES + t) * 8;
            if (p.stream_grad) raw_dh[j].template load<WIDE>(p.stream_grad + r * p.ld_stream_grad, c, n);
            if (p.normed_grad) {
                raw_dn[j].template load<WIDE>(p.normed_grad + r * p.ld_normed_grad, c, n);
                raw_h[j].template load<WIDE>(p.stream + r * D * Eight<TS>::kBytes, c, n);
            }
            if (need_u) raw_u[j].template load<WIDE>(p.branch + r * p.ld_branch, c, n);
        }
        float g[CHUNKS][8];  // the gradient on its way up
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j) {
            if (p.stream_grad)
                raw_dh[j].get(g[j]);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) g[j][e] = 0.0f;
        }
        if (p.normed_grad) {
            const float rstd = live ? p.stream_rstd[r] : 0.0f;
            float dn[CHUNKS][8], s = 0.0f;
#pragma unroll
            for (int j = 0; j < CHUNKS; ++j) {
                float hat[8];
                raw_h[j].get(hat);
                raw_dn[j].get(dn[j]);
                float w[8];
                if (p.pre) load_weight<TB, WIDE>(p.pre, p.pre_f32, (j * LANES + t) * 8, D, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    hat[e] *= rstd;
                    pre_sum[j][e] = __builtin_fmaf(dn[j][e], hat[e], pre_sum[j][e]);
                    if (p.pre) dn[j][e] *= w[e];
                    s = __builtin_fmaf(dn[j][e], hat[e], s);
                }
            }
            const float mean = row_sum(s) * inv_d;
#pragma unroll
            for (int j = 0; j < CHUNKS; ++j) {
                float hat[8];
                raw_h[j].get(hat);
#pragma unroll
                for (int e = 0; e < 8; ++e) g[j][e] += rstd * (dn[j][e] - hat[e] * rstd * mean);
            }
        }
        if (p.residual_grad)
#pragma unroll
            for (int j = 0; j < CHUNKS; ++j) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = p.residual_scale * g[j][e];
                Eight<TS>::template store<WIDE>(p.residual_grad + r * D * Eight<TS>::kBytes, (j * LANES + t) * 8, n, x);
            }
        if (!p.branch_grad && !p.want_post && !p.want_gate) continue;  // (uniform)
        const float rstd = p.post_norm && live ? p.branch_rstd[r] : 0.0f;
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j) {
            const int c = (j * LANES + t) * 8;
            float hat[8], w[8], gate[8];
            const uint32_t m = p.drop.threshold ? kept8(r * D + c, p.drop.offset, key, p.drop.threshold) : 0xFFu;
            if (need_u) raw_u[j].get(hat);
            if (p.post) load_weight<TB, WIDE>(p.post, p.post_f32, c, D, w);
            if (p.gate) load_weight<TB, WIDE>(p.gate, p.gate_f32, c, D, gate);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (p.post_norm) hat[e] *= rstd;
                g[j][e] = m >> e & 1 ? g[j][e] * (p.scale * p.drop.factor) : 0.0f;
                if (p.want_gate) gate_sum[j][e] = __builtin_fmaf(g[j][e], !(m >> e & 1) ? 0.0f : p.post ? hat[e] * w[e] : hat[e], gate_sum[j][e]);
                if (p.gate) g[j][e] *= gate[e];
                if (p.post_norm) {
                    post_sum[j][e] = __builtin_fmaf(g[j][e], hat[e], post_sum[j][e]);
                    if (p.post) g[j][e] *= w[e];
                    s = __builtin_fmaf(g[j][e], hat[e], s);
                }
            }
        }
        if (p.post_norm) {
            const float mean = row_sum(s) * inv_d;
#pragma unroll
            for (int j = 0; j < CHUNKS; ++j) {
                float hat[8];
                raw_u[j].get(hat);
#pragma unroll
                for (int e = 0; e < 8; ++e) g[j][e] = rstd * (g[j][e] - hat[e] * rstd * mean);
            }
        }
        if (p.branch_grad)
#pragma unroll
            for (int j = 0; j < CHUNKS; ++j) Eight<TB>::template store<WIDE>(p.branch_grad + r * D * Eight<TB>::kBytes, (j * LANES + t) * 8, n, g[j]);
    }
    if (!p.partial) return;
    float* out = p.partial + (int64_t)blockIdx.x * 3 * D;
    auto write = [&](const float (&sum)[CHUNKS][8], float* to) __attribute__((always_inline)) {
        if constexpr (kRows == 1) {
#pragma unroll
            for (int j = 0; j < CHUNKS; ++j) Eight<F32>::template store<WIDE>(to, (j * LANES + t) * 8, D, sum[j]);
        } else {  // the workgroup's rows meet in LDS
            constexpr int W = LANES * 8 * CHUNKS;
            __shared__ float meet[kRows][W];
            __syncthreads();
#pragma unroll
            for (int j = 0; j < CHUNKS; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) meet[threadIdx.x / LANES][(j * LANES + t) * 8 + e] = sum[j][e];
            __syncthreads();
            for (int c = threadIdx.x; c < D; c += kBlock<LANES>) {
                float v = 0.0f;
#pragma unroll
                for (int k = 0; k < kRows; ++k) v += meet[k][c];
                to[c] = v;
            }
        }
    };
    if (p.want_post) write(post_sum, out);
    if (p.want_pre) write(pre_sum, out + D);
    if (p.want_gate) write(gate_sum, out + 2 * D);
}

// out[q][c] = sum of the workgroups' partial sums: 64 columns of one of the three a workgroup, its waves on every fourth
struct SumArgs {
    const float* partial;
    int groups, D;
    void* out[3];
    int dtype[3];
};
__global__ __launch_bounds__(256) void norm_sums_kernel(const SumArgs p)
{
    __shared__ float sums[4][64];
    const int q = (int)blockIdx.y;
    if (!p.out[q]) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = (int)blockIdx.x * 64 + lane;
    float s = 0.0f;
    if (c < p.D)
        for (int g = wave; g < p.groups; g += 4) s += p.partial[((int64_t)g * 3 + q) * p.D + c];
    sums[wave][lane] = s;
    __syncthreads();
    if (wave != 0 || c >= p.D) return;
    s = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
    if (p.dtype[q] == MI8_F32)
        static_cast<float*>(p.out[q])[c] = s;
    else
        static_cast<uint16_t*>(p.out[q])[c] = (uint16_t)(p.dtype[q] == MI8_BF16 ? half::Bf16::pack(s, 0.0f) : half::F16::pack(s, 0.0f));
}

constexpr int kMostFeatures = 1024 * 2 * 8;

// Lanes of a row by its length.  Forward: a wave a row as long as it holds it, then as few waves as do (a sum over the row is a barrier).  Backward: one
// chunk a lane, whose column sums and gradients are a hundred registers; with two or four chunks a lane there is one wave on a SIMD.
int backward_lanes(int64_t D) { return D <= 128 ? 16 : D <= 512 ? 64 : D <= 1024 ? 128 : D <= 2048 ? 256 : D <= 4096 ? 512 : 1024; }

// Workgroups of the backward: what lives on the chip at once, since each writes 3 D sums.
int64_t backward_groups(int64_t rows, int64_t D)
{
    const int lanes = backward_lanes(D);
    const int64_t most = (int64_t)num_compute_units() * (lanes <= 256 ? 4 : 1024 / lanes), wanted = ceil_div(rows, lanes <= 64 ? 256 / lanes : 1);
    return wanted < most ? wanted : most;
}

template <typename TB, typename TS, int LANES, int CHUNKS>
int forward(const NormArgs& p, bool wide, hipStream_t st)
{
    const int64_t wanted = ceil_div(p.rows, kBlock<LANES> / LANES), most = (int64_t)num_compute_units() * (2048 / kBlock<LANES>);
    auto kern = wide ? norm_forward_kernel<TB, TS, LANES, CHUNKS, true> : norm_forward_kernel<TB, TS, LANES, CHUNKS, false>;
    hipLaunchKernelGGL(kern, dim3((unsigned)(wanted < most ? wanted : most)), dim3(kBlock<LANES>), 0, st, p);
    return launch_status("mi8_residual_norm_forward");
}

template <typename TB, typename TS, int LANES, int CHUNKS>
int backward(const NormArgs& p, bool wide, hipStream_t st)
{
    auto kern = wide ? norm_backward_kernel<TB, TS, LANES, CHUNKS, true> : norm_backward_kernel<TB, TS, LANES, CHUNKS, false>;
    hipLaunchKernelGGL(kern, dim3((unsigned)backward_groups(p.rows, p.D)), dim3(kBlock<LANES>), 0, st, p);
    return launch_status("mi8_residual_norm_backward");
}

template <typename TB, typename TS>
int run(const NormArgs& p, bool wide, bool back, hipStream_t st)
{
    const int D = p.D;
    if (back) {
        switch (backward_lanes(D)) {
            case 16: return backward<TB, TS, 16, 1>(p, wide, st);
            case 64: return backward<TB, TS, 64, 1>(p, wide, st);
            case 128: return backward<TB, TS, 128, 1>(p, wide, st);
            case 256: return backward<TB, TS, 256, 1>(p, wide, st);
            case 512: return backward<TB, TS, 512, 1>(p, wide, st);
            default: return D <= 8192 ? backward<TB, TS, 1024, 1>(p, wide, st) : backward<TB, TS, 1024, 2>(p, wide, st);
        }
    }
    if (D <= 128) return forward<TB, TS, 16, 1>(p, wide, st);
    if (D <= 512) return forward<TB, TS, 64, 1>(p, wide, st);
    if (D <= 1024) return forward<TB, TS, 64, 2>(p, wide, st);
    if (D <= 2048) return forward<TB, TS, 64, 4>(p, wide, st);
    if (D <= 4096) return forward<TB, TS, 256, 2>(p, wide, st);
    if (D <= 8192) return forward<TB, TS, 256, 4>(p, wide, st);
    return forward<TB, TS, 1024, 2>(p, wide, st);
}

int run_types(const NormArgs& p, int branch_dtype, int stream_dtype, bool wide, bool backward, hipStream_t st)
{
    if (branch_dtype == MI8_BF16)
        return stream_dtype == MI8_F32 ? run<half::Bf16, F32>(p, wide, backward, st) : run<half::Bf16, half::Bf16>(p, wide, backward, st);
    if (branch_dtype == MI8_F16)
        return stream_dtype == MI8_F32 ? run<half::F16, F32>(p, wide, backward, st) : run<half::F16, half::F16>(p, wide, backward, st);
    return run<F32, F32>(p, wide, backward, st);
}

// The argument block, or an error
int arguments(const mi8_residual_norm* a, NormArgs& p, bool& wide, const char* what)
{
    MI8_REQUIRE(a != nullptr, MI8_ERR_ARG, "%s: null argument", what);
    MI8_REQUIRE(float_type(a->branch_dtype) && (a->stream_dtype == a->branch_dtype || a->stream_dtype == MI8_F32), MI8_ERR_ARG,
                "%s: the stream is of the branch's type or float32", what);
    MI8_REQUIRE(a->rows >= 0 && a->features >= 0 && a->features <= kMostFeatures, MI8_ERR_UNSUPPORTED, "%s: up to %d features", what, kMostFeatures);
    MI8_REQUIRE(a->threshold <= 65536, MI8_ERR_ARG, "%s: threshold past 65536", what);
    const struct { const void* p; int dtype; } weights[3] = {{a->post, a->post_dtype}, {a->pre, a->pre_dtype}, {a->gate, a->gate_dtype}};
    for (const auto& w : weights)
        MI8_REQUIRE(w.p == nullptr || w.dtype == a->branch_dtype || w.dtype == MI8_F32, MI8_ERR_ARG, "%s: weights are float32 or of the branch's type", what);
    MI8_REQUIRE((a->post == nullptr || a->post_norm) && (a->pre == nullptr || a->pre_norm), MI8_ERR_ARG, "%s: a weight without its norm", what);
    const int sb = bytes_of(a->branch_dtype), ss = bytes_of(a->stream_dtype);
    p = NormArgs{};
    p.branch = static_cast<const uint8_t*>(a->branch);
    p.residual = static_cast<const uint8_t*>(a->residual);
    p.stream = static_cast<uint8_t*>(a->stream);
    p.normed = static_cast<uint8_t*>(a->normed);
    p.ld_branch = a->ld_branch * sb;
    p.ld_residual = a->ld_residual * ss;
    p.post = a->post;
    p.pre = a->pre;
    p.gate = a->gate;
    p.post_f32 = a->post_dtype == MI8_F32;
    p.pre_f32 = a->pre_dtype == MI8_F32;
    p.gate_f32 = a->gate_dtype == MI8_F32;
    p.post_norm = a->post_norm != 0;
    p.pre_norm = a->pre_norm != 0;
    p.rows = a->rows;
    p.D = (int)a->features;
    p.scale = a->scale;
    p.residual_scale = a->residual_scale;
    p.eps = a->eps;
    p.drop = Dropout{a->seed, a->offset, a->seed_on_device, a->threshold, a->factor};
    p.branch_rstd = a->branch_rstd;
    p.stream_rstd = a->stream_rstd;
    p.stream_grad = static_cast<const uint8_t*>(a->stream_grad);
    p.normed_grad = static_cast<const uint8_t*>(a->normed_grad);
    p.ld_stream_grad = a->ld_stream_grad * ss;
    p.ld_normed_grad = a->ld_normed_grad * sb;
    p.branch_grad = static_cast<uint8_t*>(a->branch_grad);
    p.residual_grad = static_cast<uint8_t*>(a->residual_grad);
    p.want_post = a->post_grad != nullptr;
    p.want_pre = a->pre_grad != nullptr;
    p.want_gate = a->gate_grad != nullptr;
    // whole 16-byte chunks everywhere: eight elements of any of them, at multiples of eight elements
    wide = p.D % 8 == 0 && a->ld_branch % 8 == 0 && a->ld_residual % 8 == 0 && a->ld_stream_grad % 8 == 0 && a->ld_normed_grad % 8 == 0;
    const void* all[] = {a->branch, a->residual, a->stream, a->normed, a->post, a->pre, a->gate, a->stream_grad, a->normed_grad, a->branch_grad, a->residual_grad};
    for (const void* q : all) wide = wide && aligned16(q);
    return MI8_OK;
}

}  // namespace
}  // namespace mi8

using namespace mi8;

extern "C" int mi8_residual_norm_forward(const mi8_residual_norm* args, void* stream)
{
    const char* what = "mi8_residual_norm_forward";
    NormArgs p;
    bool wide;
    if (int rc = arguments(args, p, wide, what)) return rc;
    if (p.rows == 0 || p.D == 0) return MI8_OK;
    MI8_REQUIRE(p.branch && (p.stream || p.normed), MI8_ERR_ARG, "%s: null pointer", what);
    MI8_REQUIRE(!p.pre_norm || p.normed, MI8_ERR_ARG, "%s: nowhere to put the norm of the stream", what);
    return run_types(p, args->branch_dtype, args->stream_dtype, wide, false, static_cast<hipStream_t>(stream));
}

extern "C" int64_t mi8_residual_norm_workspace_words(int64_t rows, int64_t features)
{
    return rows <= 0 || features <= 0 ? 0 : backward_groups(rows, features) * 3 * features;
}

extern "C" int mi8_residual_norm_backward(const mi8_residual_norm* args, float* workspace, void* stream)
{
    const char* what = "mi8_residual_norm_backward";
    NormArgs p;
    bool wide;
    if (int rc = arguments(args, p, wide, what)) return rc;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const bool sums = p.want_post || p.want_pre || p.want_gate;
    if (p.D == 0) return MI8_OK;
    MI8_REQUIRE(!p.want_post || p.post_norm, MI8_ERR_ARG, "%s: gradient of a weight without its norm", what);
    MI8_REQUIRE(!p.want_pre || p.pre_norm, MI8_ERR_ARG, "%s: gradient of a weight without its norm", what);
    if (p.rows > 0) {
        MI8_REQUIRE(p.stream_grad || p.normed_grad, MI8_ERR_ARG, "%s: no gradient", what);
        MI8_REQUIRE(!p.normed_grad || (p.pre_norm && p.stream && p.stream_rstd), MI8_ERR_ARG, "%s: the stream and its statistics are needed", what);
        MI8_REQUIRE(!p.post_norm || p.branch_rstd, MI8_ERR_ARG, "%s: the branch's statistics are needed", what);
        MI8_REQUIRE(!(p.post_norm || p.want_gate) || p.branch, MI8_ERR_ARG, "%s: the branch is needed", what);
        MI8_REQUIRE(!sums || workspace, MI8_ERR_ARG, "%s: no workspace", what);
        p.partial = sums ? workspace : nullptr;
        if (int rc = run_types(p, args->branch_dtype, args->stream_dtype, wide, true, st)) return rc;
    }
    if (!sums) return MI8_OK;
    SumArgs s{};
    s.partial = workspace;
    s.groups = p.rows > 0 ? (int)backward_groups(p.rows, p.D) : 0;
    s.D = p.D;
    void* outs[3] = {args->post_grad, args->pre_grad, args->gate_grad};
    // (a weight's gradient has its type; one that has no weight does not occur)
    const int dtypes[3] = {args->post_dtype, args->pre_dtype, args->gate_dtype};
    for (int q = 0; q < 3; ++q) {
        s.out[q] = outs[q];
        s.dtype[q] = dtypes[q];
    }
    hipLaunchKernelGGL(norm_sums_kernel, dim3((unsigned)ceil_div(p.D, 64), 3), dim3(256), 0, st, s);
    return launch_status(what);
}
