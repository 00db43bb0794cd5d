// A block's output on its way into the residual stream, and the norm in front of the next block, in one pass over the data:
//
//     v = norm(branch) post        norm(a) = a rsqrt(mean(a^2) + eps)
//     h = residual_scale residual + scale gate drop(v)
//     n = norm(h) pre
//
// and the gradients of all its inputs, every part optional.  With a = the row, hat = norm(a), y = hat w: the gradient of a norm is
//     da = rsqrt(..) (dy w - hat mean(dy w hat)),   dw = sum over rows of dy hat.
//
// Bound by memory: forward one read of branch and residual, one write of h and n; backward one read of branch and residual, or h, and of the two gradients, one
// write of the inputs' gradients.  A row lives in the registers of the lanes that own it (16 lanes to 1024, one or two chunks of eight elements each); the
// statistics are float32 sums over those lanes, and h is rounded to its type only when it is stored: the second norm sees it unrounded.  The next row's
// loads are issued as soon as this one's are in float32, in front of the sums over the row.
// The backward makes h again, unrounded, where it is given the branch: the gradient of a weight keeps the accuracy of its terms (from an h that was stored in
// bf16: 2.3e-3 of the definition in 64 bits instead of the rounding's 1.7e-3, and 1.6e-3 instead of 1e-7 in float32).  Beside a norm or a gate on the branch that is the
// residual in place of h, the same bytes; a plain join moves six tensors for five (bf16, 16384 x 4096: 161 us
// for 155, 8192 x 8192 167 for 149).  Without the branch it takes h as it is stored,
// which is for a float32 stream or a norm alone.  The dropped elements are made again from the counter (mi8_philox.h).
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
    int remake;  // the stream is made again from branch and residual
    const uint8_t *stream_grad, *normed_grad;
    int64_t ld_stream_grad, ld_normed_grad;
    uint8_t *branch_grad, *residual_grad;
    float* partial;  // [workgroups][3][D]: post, pre, gate; null: none wanted
    int want_post, want_pre, want_gate;
};

// Eight weights (float32, or T) of columns c .. c + 7; w null: ones
template <typename T, bool WHOLE, bool LONG>
__device__ __forceinline__ void load_weight(const void* w, int f32, int c, int n, float (&f)[8])
{
    if (w == nullptr) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = 1.0f;
    } else if (f32) {
        Eight<F32> r;
        r.template load<WHOLE, LONG>(w, c, n);
        r.get(f);
    } else {
        Eight<T> r;
        r.template load<WHOLE, LONG>(w, c, n);
        r.get(f);
    }
}

// A weight's elements of this lane, ones where there is none: held in registers for all rows, or, where a lane has too many, read again for each (from
// the caches).  Multiplying with ones costs less than a choice: values that pass a branch are copied.
template <typename T, int LANES, int CHUNKS, bool HELD, bool WHOLE>
struct Weight {
    float v[HELD ? CHUNKS : 1][8];
    const void* w;
    int f32, D;
    __device__ __forceinline__ Weight(const void* w_, int f32_, int D_) : w(w_), f32(f32_), D(D_)
    {
        if constexpr (HELD)
#pragma unroll
            for (int j = 0; j < CHUNKS; ++j) load_weight<T, WHOLE, (LANES > 16)>(w, f32, (j * LANES + threadIdx.x % LANES) * 8, D, v[j]);
    }
    __device__ __forceinline__ void times(float (&x)[8], int j) const
    {
        float now[8];
        if constexpr (!HELD) load_weight<T, WHOLE, (LANES > 16)>(w, f32, (j * LANES + threadIdx.x % LANES) * 8, D, now);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= HELD ? v[j][e] : now[e];
    }
};

template <int CTRL, int ROWS>
__device__ __forceinline__ float plus_dpp(float v)
{
    return v + __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, ROWS, 0xF, true));
}

// Sum over the LANES lanes that own a row (16, or all of a wave or of the workgroup), by moves inside the vector unit.  More than a wave: through
// LDS, in turns of two places (a barrier of the other place lies between two uses).
template <int LANES>
struct RowSum {
    int turn = 0;
    __device__ __forceinline__ float operator()(float v)
    {
        v = plus_dpp<0xB1, 0xF>(v);   // quad_perm [1,0,3,2]
        v = plus_dpp<0x4E, 0xF>(v);   // quad_perm [2,3,0,1]
        v = plus_dpp<0x141, 0xF>(v);  // row_half_mirror
        v = plus_dpp<0x140, 0xF>(v);  // row_mirror: every lane has its 16 lanes' sum
        if constexpr (LANES == 16) return v;
        v = plus_dpp<0x142, 0xA>(v);  // row_bcast 15, 31: lane 63 has the wave's
        v = plus_dpp<0x143, 0xC>(v);
        v = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), 63));
        if constexpr (LANES > 64) {
            constexpr int W = LANES / 64;
            __shared__ float sums[2][W];
            if ((threadIdx.x & 63) == 0) sums[turn][threadIdx.x >> 6] = v;
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

// Are the next row's loads issued before this one is done?
template <int LANES, int CHUNKS>
constexpr bool kAhead = LANES * CHUNKS <= 1024;

// Between a lane's chunks where registers are short: what one loads is not fetched while another is worked on
template <int LANES, int CHUNKS>
__device__ __forceinline__ void apart()
{
    if constexpr (!kAhead<LANES, CHUNKS>) __builtin_amdgcn_sched_barrier(0);
}

// Sums of a lane's columns over the rows that it walks: in registers, or in LDS, each lane its own places of 16 bytes, neighbours next to each other
template <int LANES, int CHUNKS, bool IN_LDS, int WHICH>
struct ColumnSum {
    float v[IN_LDS ? 1 : CHUNKS][8];
    float4* at;
    __device__ __forceinline__ ColumnSum() : v{}
    {
        if constexpr (IN_LDS) {
            __shared__ float4 sums[CHUNKS * 2 * LANES];
            at = sums + threadIdx.x;
#pragma unroll
            for (int k = 0; k < CHUNKS * 2; ++k) at[k * LANES] = float4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    __device__ __forceinline__ void add(const float (&a)[8], const float (&b)[8], int j, bool wanted)
    {
        if constexpr (IN_LDS) {
            if (!wanted) return;  // (uniform)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float4& s = at[(j * 2 + h) * LANES];
                float4 x = s;
                x.x = __builtin_fmaf(a[4 * h], b[4 * h], x.x);
                x.y = __builtin_fmaf(a[4 * h + 1], b[4 * h + 1], x.y);
                x.z = __builtin_fmaf(a[4 * h + 2], b[4 * h + 2], x.z);
                x.w = __builtin_fmaf(a[4 * h + 3], b[4 * h + 3], x.w);
                s = x;
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[j][e] = __builtin_fmaf(a[e], b[e], v[j][e]);
        }
    }
    __device__ __forceinline__ void get(float (&x)[8], int j) const
    {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (IN_LDS)
                x[e] = reinterpret_cast<const float*>(at + (j * 2 + e / 4) * LANES)[e % 4];
            else
                x[e] = v[j][e];
        }
    }
};

// The state of a row's dropout: a bit an element, all set where there is none
__device__ __forceinline__ uint32_t kept_of(const Dropout& d, int64_t first, uint64_t key)
{
    uint32_t m = 0xFFu;
    if (d.threshold) m = kept8(first, d.offset, key, d.threshold);
    return m;
}

template <typename TB, typename TS, int LANES, int CHUNKS, bool WHOLE>
__global__ __launch_bounds__(kBlock<LANES>, LANES == 1024 ? 4 : 3) void norm_forward_kernel(const NormArgs p)
{
    constexpr int kRows = kBlock<LANES> / LANES;
    constexpr bool kLong = LANES > 16;  // (rows of more than 128)
    const int t = threadIdx.x % LANES, D = p.D;
    const uint64_t key = p.drop.seed_on_device ? (uint64_t)p.drop.seed_on_device[0] : p.drop.seed;
    const float inv_d = 1.0f / (float)D, factor = p.scale * (p.drop.threshold ? p.drop.factor : 1.0f);
    RowSum<LANES> row_sum;
    typedef Weight<TB, LANES, CHUNKS, LANES != 1024, WHOLE> W;
    const W post(p.post, p.post_f32, D), pre(p.pre, p.pre_f32, D), gate(p.gate, p.gate_f32, D);
    const int64_t stride = (int64_t)gridDim.x * kRows;
    int64_t row0 = (int64_t)blockIdx.x * kRows;
    Eight<TB> raw_u[CHUNKS];
    Eight<TS> raw_r[CHUNKS] = {};
    auto load = [&](int64_t from) __attribute__((always_inline)) {  // (rows past the last one: zeros)
        const int64_t r = from + threadIdx.x / LANES;
        const int n = r < p.rows ? D : 0;
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j) raw_u[j].template load<WHOLE, kLong>(p.branch + r * p.ld_branch, (j * LANES + t) * 8, n);
        if (p.residual)
#pragma unroll
            for (int j = 0; j < CHUNKS; ++j) raw_r[j].template load<WHOLE, kLong>(p.residual + r * p.ld_residual, (j * LANES + t) * 8, n);
    };
    if (kAhead<LANES, CHUNKS>) load(row0);
    for (; row0 < p.rows; row0 += stride) {
        const int64_t r = row0 + threadIdx.x / LANES;
        const bool live = r < p.rows;
        const int n = live ? D : 0;
        if constexpr (!kAhead<LANES, CHUNKS>) {
#pragma unroll
            for (int j = 0; j < CHUNKS; ++j) raw_r[j] = {};  // (nothing that is not loaded lives on from row to row)
            load(row0);
        }
        float h[CHUNKS][8], res[CHUNKS][8];
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j) {
            apart<LANES, CHUNKS>();
            raw_u[j].get(h[j]);
            raw_r[j].get(res[j]);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (kAhead<LANES, CHUNKS>) load(row0 + stride);
        __builtin_amdgcn_sched_barrier(0);
        float rstd = 1.0f;
        if (p.post_norm) {
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < CHUNKS; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) s = __builtin_fmaf(h[j][e], h[j][e], s);
            rstd = rsqrtf(row_sum(s) * inv_d + p.eps);
            if (p.branch_rstd && live && t == 0) p.branch_rstd[r] = rstd;
        }
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j) {
            apart<LANES, CHUNKS>();
            const int c = (j * LANES + t) * 8;
            const uint32_t m = kept_of(p.drop, r * D + c, key);
#pragma unroll
            for (int e = 0; e < 8; ++e) h[j][e] *= rstd;
            post.times(h[j], j);
            gate.times(h[j], j);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                h[j][e] = __builtin_fmaf(p.residual_scale, res[j][e], m >> e & 1 ? h[j][e] * factor : 0.0f);
                s = __builtin_fmaf(h[j][e], h[j][e], s);
            }
            if (p.stream) Eight<TS>::template store<WHOLE, kLong>(p.stream + r * D * Eight<TS>::kBytes, c, n, h[j]);
        }
        if (!p.pre_norm) continue;
        rstd = rsqrtf(row_sum(s) * inv_d + p.eps);
        if (p.stream_rstd && live && t == 0) p.stream_rstd[r] = rstd;
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j) {
            apart<LANES, CHUNKS>();
#pragma unroll
            for (int e = 0; e < 8; ++e) h[j][e] *= rstd;
            pre.times(h[j], j);
            Eight<TB>::template store<WHOLE, kLong>(p.normed + r * D * Eight<TB>::kBytes, (j * LANES + t) * 8, n, h[j]);
        }
    }
}

template <typename TB, typename TS, int LANES, int CHUNKS, bool WHOLE>
__global__ __launch_bounds__(kBlock<LANES>, LANES == 1024 ? 4 : 2) void norm_backward_kernel(const NormArgs p)
{
    constexpr int kRows = kBlock<LANES> / LANES;
    constexpr bool kLong = LANES > 16;  // (rows of more than 128)
    const int t = threadIdx.x % LANES, D = p.D;
    const uint64_t key = p.drop.seed_on_device ? (uint64_t)p.drop.seed_on_device[0] : p.drop.seed;
    const float inv_d = 1.0f / (float)D, factor = p.scale * (p.drop.threshold ? p.drop.factor : 1.0f);
    const uint8_t* const other = p.remake ? p.residual : p.normed_grad ? p.stream : nullptr;  // of the stream's type
    const int64_t ld_other = p.remake ? p.ld_residual : (int64_t)D * Eight<TS>::kBytes;
    // the stream as the forward made it, or as it is stored: other times this, plus the branch where it is read
    const float other_factor = p.remake ? p.residual_scale : 1.0f;
    RowSum<LANES> row_sum;
    typedef Weight<TB, LANES, CHUNKS, LANES != 1024, WHOLE> W;
    const W post(p.post, p.post_f32, D), pre(p.pre, p.pre_f32, D), gate(p.gate, p.gate_f32, D);
    ColumnSum<LANES, CHUNKS, LANES == 1024, 0> post_sum;
    ColumnSum<LANES, CHUNKS, false, 1> pre_sum;
    ColumnSum<LANES, CHUNKS, LANES == 1024, 2> gate_sum;
    const int64_t stride = (int64_t)gridDim.x * kRows;
    int64_t row0 = (int64_t)blockIdx.x * kRows;
    Eight<TB> raw_u[CHUNKS] = {}, raw_dn[CHUNKS] = {};
    Eight<TS> raw_other[CHUNKS] = {}, raw_dh[CHUNKS] = {};
    auto load = [&](int64_t from) __attribute__((always_inline)) {  // (rows past the last one: zeros)
        const int64_t r = from + threadIdx.x / LANES;
        const int n = r < p.rows ? D : 0;
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j) {
            apart<LANES, CHUNKS>();
            const int c = (j * LANES + t) * 8;
            if (p.branch) raw_u[j].template load<WHOLE, kLong>(p.branch + r * p.ld_branch, c, n);
            if (other) raw_other[j].template load<WHOLE, kLong>(other + r * ld_other, c, n);
            if (p.normed_grad) raw_dn[j].template load<WHOLE, kLong>(p.normed_grad + r * p.ld_normed_grad, c, n);
            if (p.stream_grad) raw_dh[j].template load<WHOLE, kLong>(p.stream_grad + r * p.ld_stream_grad, c, n);
        }
    };
    if (kAhead<LANES, CHUNKS>) load(row0);
    for (; row0 < p.rows; row0 += stride) {
        const int64_t r = row0 + threadIdx.x / LANES;
        const bool live = r < p.rows;
        const int n = live ? D : 0;
        if constexpr (!kAhead<LANES, CHUNKS>) {
#pragma unroll
            for (int j = 0; j < CHUNKS; ++j) {  // (nothing that is not loaded lives on from row to row)
                raw_u[j] = raw_dn[j] = {};
                raw_other[j] = raw_dh[j] = {};
            }
            load(row0);
        }
        float branch_rstd = 1.0f, stream_rstd = 0.0f;
        if (p.post_norm && live) branch_rstd = p.branch_rstd[r];
        if (p.normed_grad && live) stream_rstd = p.stream_rstd[r];
        float u[CHUNKS][8], hat[CHUNKS][8], dn[CHUNKS][8], g[CHUNKS][8];  // u: the branch, normed if it is; g: the gradient on its way up
        uint32_t kept[CHUNKS];
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j) {
            apart<LANES, CHUNKS>();
            raw_u[j].get(u[j]);
            raw_other[j].get(hat[j]);
            raw_dn[j].get(dn[j]);
            raw_dh[j].get(g[j]);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (kAhead<LANES, CHUNKS>) load(row0 + stride);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j) {
            apart<LANES, CHUNKS>();
            kept[j] = kept_of(p.drop, r * D + (j * LANES + t) * 8, key);
#pragma unroll
            for (int e = 0; e < 8; ++e) u[j][e] *= branch_rstd;
        }
        if (p.normed_grad) {
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < CHUNKS; ++j) {
            apart<LANES, CHUNKS>();
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = u[j][e];
                post.times(v, j);
                gate.times(v, j);
#pragma unroll
                for (int e = 0; e < 8; ++e) hat[j][e] = __builtin_fmaf(other_factor, hat[j][e], kept[j] >> e & 1 ? v[e] * factor : 0.0f) * stream_rstd;
                pre_sum.add(dn[j], hat[j], j, true);
                pre.times(dn[j], j);
#pragma unroll
                for (int e = 0; e < 8; ++e) s = __builtin_fmaf(dn[j][e], hat[j][e], s);
            }
            const float mean = row_sum(s) * inv_d;
#pragma unroll
            for (int j = 0; j < CHUNKS; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) g[j][e] = __builtin_fmaf(stream_rstd, dn[j][e] - hat[j][e] * mean, g[j][e]);
        }
        if (p.residual_grad)
#pragma unroll
            for (int j = 0; j < CHUNKS; ++j) {
            apart<LANES, CHUNKS>();
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = p.residual_scale * g[j][e];
                Eight<TS>::template store<WHOLE, kLong>(p.residual_grad + r * D * Eight<TS>::kBytes, (j * LANES + t) * 8, n, x);
            }
        if (!p.branch_grad && !p.want_post && !p.want_gate) continue;  // (uniform)
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < CHUNKS; ++j) {
            apart<LANES, CHUNKS>();
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                g[j][e] = kept[j] >> e & 1 ? g[j][e] * factor : 0.0f;
                v[e] = kept[j] >> e & 1 ? u[j][e] : 0.0f;  // (what was dropped reaches no gradient, whatever it was)
            }
            post.times(v, j);
            gate_sum.add(g[j], v, j, p.want_gate);
            gate.times(g[j], j);
            post_sum.add(g[j], u[j], j, p.want_post);
            post.times(g[j], j);
#pragma unroll
            for (int e = 0; e < 8; ++e) s = __builtin_fmaf(g[j][e], u[j][e], s);
        }
        if (p.post_norm) {
            const float mean = row_sum(s) * inv_d;
#pragma unroll
            for (int j = 0; j < CHUNKS; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) g[j][e] = branch_rstd * (g[j][e] - u[j][e] * mean);
        }
        if (p.branch_grad)
#pragma unroll
            for (int j = 0; j < CHUNKS; ++j) Eight<TB>::template store<WHOLE, kLong>(p.branch_grad + r * D * Eight<TB>::kBytes, (j * LANES + t) * 8, n, g[j]);
    }
    if (!p.partial) return;
    float* out = p.partial + (int64_t)blockIdx.x * 3 * D;
    auto write = [&](const auto& sum, float* to) __attribute__((always_inline)) {
        if constexpr (kRows == 1) {
#pragma unroll
            for (int j = 0; j < CHUNKS; ++j) {
                float x[8];
                sum.get(x, j);
                Eight<F32>::template store<WHOLE, kLong>(to, (j * LANES + t) * 8, D, x);
            }
        } else {  // the workgroup's rows meet in LDS
            constexpr int kWidth = LANES * 8 * CHUNKS;
            __shared__ float meet[kRows][kWidth];
            __syncthreads();
#pragma unroll
            for (int j = 0; j < CHUNKS; ++j)
#pragma unroll
                for (int e = 0; e < 8; ++e) meet[threadIdx.x / LANES][(j * LANES + t) * 8 + e] = sum.v[j][e];
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

// out[q][c] = sum of the workgroups' partial sums: 16 columns of one of the three a workgroup, its 16 groups of lanes on every 16th
struct SumArgs {
    const float* partial;
    int groups, D;
    void* out[3];
    int dtype[3];
};
__global__ __launch_bounds__(256) void norm_sums_kernel(const SumArgs p)
{
    __shared__ float sums[16][16];
    const int q = (int)blockIdx.y;
    if (!p.out[q]) return;
    const int c = (int)blockIdx.x * 16 + threadIdx.x % 16, g0 = threadIdx.x / 16;
    float s = 0.0f;
    if (c < p.D)
#pragma unroll 8
        for (int g = g0; g < p.groups; g += 16) s += p.partial[((int64_t)g * 3 + q) * p.D + c];
    sums[g0][threadIdx.x % 16] = s;
    __syncthreads();
    if (g0 != 0 || c >= p.D) return;
    s = 0.0f;
#pragma unroll
    for (int g = 0; g < 16; ++g) s += sums[g][threadIdx.x];
    if (p.dtype[q] == MI8_F32)
        static_cast<float*>(p.out[q])[c] = s;
    else
        static_cast<uint16_t*>(p.out[q])[c] = (uint16_t)(p.dtype[q] == MI8_BF16 ? half::Bf16::pack(s, 0.0f) : half::F16::pack(s, 0.0f));
}

constexpr int kMostFeatures = 1024 * 2 * 8;

// Lanes of a row by its length.  Forward: two chunks a lane, a wave a row as long as it holds it (a sum over more is a barrier).  Backward: one chunk a
// lane, whose column sums, weights and gradients are over a hundred registers (16384 x 4096 bf16 with every part: 172 us with two waves on a SIMD and
// those registers, 272 with four waves and scratch memory).  Rows past 4096 take 1024 lanes, 128 registers each: the sums of post and gate live in LDS,
// the weights are read again from the caches, and past 8192 no loads run ahead.  What still goes to scratch memory past 8192 is 208 to 264 bytes a
// lane of 16-bit rows, 140 to 204 of float32 ones; between 4096 and 8192 it is nothing but for 16-bit rows of whole chunks with a float32 stream and odd float32
// rows (12 to 36).  Backward of 2^26 bf16 elements, a float32 stream: 4096 columns 225 us, 8192 264 (5.4, 4.6 TB/s), 11008 389, 16384 363; 11003 631.
int backward_lanes(int64_t D) { return D <= 128 ? 16 : D <= 512 ? 64 : D <= 1024 ? 128 : D <= 2048 ? 256 : D <= 4096 ? 512 : 1024; }

// Workgroups of the backward: what lives on the chip at once, since each writes 3 D sums, and of four turns at least.
int64_t backward_groups(int64_t rows, int64_t D)
{
    const int lanes = backward_lanes(D);
    const int64_t most = (int64_t)num_compute_units() * (lanes <= 256 ? 4 : 1024 / lanes), wanted = ceil_div(rows, 4 * (lanes <= 64 ? 256 / lanes : 1));
    return wanted < most ? wanted : most;
}

template <typename TB, typename TS, int LANES, int CHUNKS>
int forward(const NormArgs& p, hipStream_t st)
{
    const int64_t wanted = ceil_div(p.rows, kBlock<LANES> / LANES), most = (int64_t)num_compute_units() * (2048 / kBlock<LANES>);
    auto kern = p.D % 8 == 0 ? norm_forward_kernel<TB, TS, LANES, CHUNKS, true> : norm_forward_kernel<TB, TS, LANES, CHUNKS, false>;
    hipLaunchKernelGGL(kern, dim3((unsigned)(wanted < most ? wanted : most)), dim3(kBlock<LANES>), 0, st, p);
    return launch_status("mi8_residual_norm_forward");
}

template <typename TB, typename TS, int LANES, int CHUNKS>
int backward(const NormArgs& p, hipStream_t st)
{
    auto kern = p.D % 8 == 0 ? norm_backward_kernel<TB, TS, LANES, CHUNKS, true> : norm_backward_kernel<TB, TS, LANES, CHUNKS, false>;
    hipLaunchKernelGGL(kern, dim3((unsigned)backward_groups(p.rows, p.D)), dim3(kBlock<LANES>), 0, st, p);
    return launch_status("mi8_residual_norm_backward");
}

template <typename TB, typename TS>
int run(const NormArgs& p, bool back, hipStream_t st)
{
    const int D = p.D;
    if (back) {
        switch (backward_lanes(D)) {
            case 16: return backward<TB, TS, 16, 1>(p, st);
            case 64: return backward<TB, TS, 64, 1>(p, st);
            case 128: return backward<TB, TS, 128, 1>(p, st);
            case 256: return backward<TB, TS, 256, 1>(p, st);
            case 512: return backward<TB, TS, 512, 1>(p, st);
            default: return D <= 8192 ? backward<TB, TS, 1024, 1>(p, st) : backward<TB, TS, 1024, 2>(p, st);
        }
    }
    if (D <= 128) return forward<TB, TS, 16, 1>(p, st);
    if (D <= 512) return forward<TB, TS, 64, 1>(p, st);
    if (D <= 1024) return forward<TB, TS, 64, 2>(p, st);
    if (D <= 2048) return forward<TB, TS, 128, 2>(p, st);
    if (D <= 4096) return forward<TB, TS, 256, 2>(p, st);
    if (D <= 8192) return forward<TB, TS, 512, 2>(p, st);
    return forward<TB, TS, 1024, 2>(p, st);
}

int run_types(const NormArgs& p, int branch_dtype, int stream_dtype, bool backward, hipStream_t st)
{
    if (branch_dtype == MI8_BF16)
        return stream_dtype == MI8_F32 ? run<half::Bf16, F32>(p, backward, st) : run<half::Bf16, half::Bf16>(p, backward, st);
    if (branch_dtype == MI8_F16)
        return stream_dtype == MI8_F32 ? run<half::F16, F32>(p, backward, st) : run<half::F16, half::F16>(p, backward, st);
    return run<F32, F32>(p, backward, st);
}

// The argument block, or an error
int arguments(const mi8_residual_norm* a, NormArgs& p, const char* what)
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
    return MI8_OK;
}

}  // namespace
}  // namespace mi8

using namespace mi8;

extern "C" int mi8_residual_norm_forward(const mi8_residual_norm* args, void* stream)
{
    const char* what = "mi8_residual_norm_forward";
    NormArgs p;
    if (int rc = arguments(args, p, what)) return rc;
    if (p.rows == 0 || p.D == 0) return MI8_OK;
    MI8_REQUIRE(p.branch && (p.stream || p.normed), MI8_ERR_ARG, "%s: null pointer", what);
    MI8_REQUIRE(!p.pre_norm || p.normed, MI8_ERR_ARG, "%s: nowhere to put the norm of the stream", what);
    return run_types(p, args->branch_dtype, args->stream_dtype, false, static_cast<hipStream_t>(stream));
}

extern "C" int64_t mi8_residual_norm_workspace_words(int64_t rows, int64_t features)
{
    return rows <= 0 || features <= 0 ? 0 : backward_groups(rows, features) * 3 * features;
}

extern "C" int mi8_residual_norm_backward(const mi8_residual_norm* args, float* workspace, void* stream)
{
    const char* what = "mi8_residual_norm_backward";
    NormArgs p;
    if (int rc = arguments(args, p, what)) return rc;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const bool sums = p.want_post || p.want_pre || p.want_gate;
    if (p.D == 0) return MI8_OK;
    MI8_REQUIRE(!p.want_post || p.post_norm, MI8_ERR_ARG, "%s: gradient of a weight without its norm", what);
    MI8_REQUIRE(!p.want_pre || p.pre_norm, MI8_ERR_ARG, "%s: gradient of a weight without its norm", what);
    if (p.rows > 0) {
        MI8_REQUIRE(p.stream_grad || p.normed_grad, MI8_ERR_ARG, "%s: no gradient", what);
        MI8_REQUIRE(!p.normed_grad || (p.pre_norm && (p.stream || p.branch) && p.stream_rstd), MI8_ERR_ARG, "%s: the stream and its statistics are needed", what);
        p.remake = p.normed_grad && p.branch;
        MI8_REQUIRE(!p.post_norm || p.branch_rstd, MI8_ERR_ARG, "%s: the branch's statistics are needed", what);
        MI8_REQUIRE(!(p.post_norm || p.want_gate) || p.branch, MI8_ERR_ARG, "%s: the branch is needed", what);
        MI8_REQUIRE(!sums || workspace, MI8_ERR_ARG, "%s: no workspace", what);
        p.partial = sums ? workspace : nullptr;
        if (int rc = run_types(p, args->branch_dtype, args->stream_dtype, true, st)) return rc;
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
    hipLaunchKernelGGL(norm_sums_kernel, dim3((unsigned)ceil_div(p.D, 16), 3), dim3(256), 0, st, s);
    return launch_status(what);
}
