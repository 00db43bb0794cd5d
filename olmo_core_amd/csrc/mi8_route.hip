// Routing of tokens to experts: from router logits [tokens, experts] to the top_k experts of every token, their weights and the
// number of slots of every expert; and the gradient of the logits.
//
//   s_e = softmax(l)_e or sigmoid(l_e)      the scores
//   c_e = s_e + bias_e                      what the choice is made by (the bias balances the load and is no part of a weight)
//   groups of consecutive experts: the `kept` ones with the largest sum of their two largest c; the others are not chosen from
//   i_1 .. i_k: the largest c first, the lowest index of equal ones;  w_j = scale * s_{i_j} (normalize: / sum of the chosen s)
//
// What bounds it: reading the logits once (4 MB at 16384 x 64 in two bytes, 17 MB at 16384 x 256 in four) and, at these
// sizes, the arithmetic of the choice.  Sixteen lanes share a token, so that every reduction is four moves inside the vector unit (DPP)
// and a wave has four tokens; a lane holds V consecutive experts.
//
// The choice is the one of exact arithmetic.  Without a bias it goes by the logits themselves, which order the scores.  With a bias, or by sums
// of groups, the scores' float32 errors could swap neighbours: where two values that decide are closer than those errors (one wave in
// some hundred), the wave repeats its choice in 64 bits.
#include "mi8_block.h"

namespace mi8 {
namespace {

struct RouteArgs {
    const void* logits;
    const float* bias;  // null, or [experts]
    int64_t tokens;
    int experts, top_k, groups, kept, softmax, normalize;
    float scale;
    float* weights;       // [tokens, top_k]
    int64_t* indices;     // [tokens, top_k]
    int64_t* counts;      // [experts] (a launch of one workgroup)
    int32_t* partial;     // [workgroups, experts] (others)
};

constexpr int kMostExperts = 512, kMostTopK = 64, kMostGroups = 32;
constexpr int kOneBlock = 128;  // tokens that one workgroup takes by itself

template <int HP>
struct Logit;
template <>
struct Logit<MI8_BF16> {
    typedef uint16_t type;
    __device__ static float value(uint16_t v) { return bits_to_f32((uint32_t)v << 16); }
    __device__ static uint16_t round(float f)
    {
        return (uint16_t)(pack_bf16(f, f) & 0xFFFFu);
    }
};
template <>
struct Logit<MI8_F16> {
    typedef _Float16 type;
    __device__ static float value(_Float16 v) { return (float)v; }
    __device__ static _Float16 round(float f) { return (_Float16)f; }
};
template <>
struct Logit<MI8_F32> {
    typedef float type;
    __device__ static float value(float v) { return v; }
    __device__ static float round(float f) { return f; }
};

// ---- reductions over the 16 lanes of a token -----------------------------------------------------------------------

template <int CTRL>
__device__ __forceinline__ float dpp(float v) { return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true)); }
template <int CTRL>
__device__ __forceinline__ int dpp(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, true); }
template <int CTRL>
__device__ __forceinline__ double dpp(double v)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)dpp<CTRL>((int)(uint32_t)u), hi = (uint32_t)dpp<CTRL>((int)(uint32_t)(u >> 32));
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
constexpr int kSwap1 = 0xB1, kSwap2 = 0x4E, kMirror8 = 0x141, kMirror16 = 0x140;  // quad_perm [1,0,3,2], [2,3,0,1], row_half_mirror, row_mirror

template <typename T, typename Op>
__device__ __forceinline__ T over16(T v, Op op)
{
    v = op(v, dpp<kSwap1>(v));
    v = op(v, dpp<kSwap2>(v));
    v = op(v, dpp<kMirror8>(v));
    return op(v, dpp<kMirror16>(v));
}
template <typename T>
__device__ __forceinline__ T larger(T a, T b) { return a > b ? a : b; }
template <typename T>
__device__ __forceinline__ T max16(T v) { return over16(v, [](T a, T b) { return larger(a, b); }); }
template <typename T>
__device__ __forceinline__ T sum16(T v) { return over16(v, [](T a, T b) { return a + b; }); }
__device__ __forceinline__ int min16(int v) { return over16(v, [](int a, int b) { return a < b ? a : b; }); }

template <typename T>
__device__ __forceinline__ T sigmoid(T l);
template <>
__device__ __forceinline__ float sigmoid(float l) { return 1.0f / (1.0f + expf(-l)); }
template <>
__device__ __forceinline__ double sigmoid(double l) { return 1.0 / (1.0 + exp(-l)); }

// what one lane of a wave wrote to LDS is there for the others (their LDS operations run in order)
__device__ __forceinline__ void wave_lds() { asm volatile("" ::: "memory"); __builtin_amdgcn_wave_barrier(); }

// The two largest of a set
template <typename T>
struct Two {
    T m1, m2;
    __device__ __forceinline__ void take(T v)
    {
        m2 = larger(m2, v < m1 ? v : m1);
        m1 = larger(m1, v);
    }
    template <int CTRL>
    __device__ __forceinline__ void merge()
    {
        const T o1 = dpp<CTRL>(m1), o2 = dpp<CTRL>(m2);
        m2 = larger(larger(m2, o2), o1 < m1 ? o1 : m1);
        m1 = larger(m1, o1);
    }
};

// A token's choice from c[V] (-infinity where the lane has no expert) into choice[top_k] (LDS of the token; group_scores likewise).  Returns
// whether values that decide are not further apart than `border` (0: not asked).
template <typename T, int V>
__device__ __forceinline__ bool choose(const RouteArgs& a, const T (&c)[V], const int l16, const T border, int* choice, T* group_scores)
{
    constexpr T kLeast = -__builtin_huge_val();
    const int first = l16 * V;
    bool near = false;
    // An expert that is out - not there, of no kept group, or chosen - has its bit set.  Of experts whose c is -infinity the lowest index that is
    // left has its turn (top_k is at most the size of the kept groups).
    uint32_t out = 0;
#pragma unroll
    for (int p = 0; p < V; ++p)
        if (first + p >= a.experts) out |= 1u << p;
    if (a.groups > 1) {
        const int size = a.experts / a.groups, lanes = size / V;
        const bool whole = size % V == 0;  // a lane's experts are of one group
        if (whole && (lanes == 1 || lanes == 2 || lanes == 4 || lanes == 8)) {
            Two<T> two{kLeast, kLeast};
#pragma unroll
            for (int p = 0; p < V; ++p) two.take(c[p]);
            if (lanes > 1) two.template merge<kSwap1>();
            if (lanes > 2) two.template merge<kSwap2>();
            if (lanes > 4) two.template merge<kMirror8>();
            if (first < a.experts && l16 % lanes == 0) group_scores[l16 / lanes] = size > 1 ? two.m1 + two.m2 : two.m1;
        } else {
            for (int g = 0; g < a.groups; ++g) {
                Two<T> two{kLeast, kLeast};
#pragma unroll
                for (int p = 0; p < V; ++p) two.take(first + p >= g * size && first + p < (g + 1) * size ? c[p] : kLeast);
                two.template merge<kSwap1>();
                two.template merge<kSwap2>();
                two.template merge<kMirror8>();
                two.template merge<kMirror16>();
                if (l16 == 0) group_scores[g] = size > 1 ? two.m1 + two.m2 : two.m1;
            }
        }
        wave_lds();
        // a group is kept if fewer than `kept` groups are before it
        auto kept = [&](int g) __attribute__((always_inline)) {
            const T mine = group_scores[g];
            int before = 0;
            for (int o = 0; o < a.groups; ++o) {
                const T other = group_scores[o];
                before += (other > mine || (other == mine && o < g)) ? 1 : 0;
                if (o != g && !(other > mine + 2 * border || other < mine - 2 * border)) near = true;
            }
            return before < a.kept;
        };
        if (first < a.experts) {
            int g = first / size, next = (g + 1) * size;
            bool keep = kept(g);
            if (whole) {
                if (!keep) out = ~0u;
            } else {
#pragma unroll
                for (int p = 0; p < V; ++p) {
                    if (first + p == next && first + p < a.experts) {
                        keep = kept(++g);
                        next += size;
                    }
                    if (!keep) out |= 1u << p;
                }
            }
        }
        near = near && border > 0;
    }
    T previous = 0;
    for (int j = 0; j <= a.top_k; ++j) {
        T best = kLeast;
        int at = 1 << 20;
#pragma unroll
        for (int p = V - 1; p >= 0; --p)
            if (!(out >> p & 1) && c[p] >= best) {
                best = c[p];
                at = first + p;
            }
        const T top = max16(best);
        if (j > 0 && border > 0 && !(previous - top > border)) near = true;  // (also between the last that is chosen and the next)
        previous = top;
        if (j == a.top_k) break;
        const int winner = min16(best == top ? at : 1 << 20);
        if (winner / V == l16) out |= 1u << (winner % V);
        if (l16 == 0) choice[j] = winner;
    }
    wave_lds();
    return near;
}

template <int HP, int V, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void route_kernel(RouteArgs a)
{
    __shared__ int hist[kMostExperts];
    __shared__ int choices[WAVES * 4][kMostTopK];
    __shared__ float scores[WAVES * 4][kMostGroups];
    __shared__ double scores64[WAVES * 4][kMostGroups];
    typedef typename Logit<HP>::type logit_t;
    const int tid = threadIdx.x, l16 = tid & 15;
    const int slot = tid >> 4;
    for (int e = tid; e < a.experts; e += WAVES * 64) hist[e] = 0;
    __syncthreads();
    const int first = l16 * V;
    const logit_t* logits = reinterpret_cast<const logit_t*>(a.logits);
    for (int64_t t0 = (int64_t)blockIdx.x * WAVES * 4; t0 < a.tokens; t0 += (int64_t)gridDim.x * WAVES * 4) {
        const int64_t token = t0 + slot;
        const bool valid = token < a.tokens;
        const logit_t* row = logits + (valid ? token : a.tokens - 1) * a.experts;
        float l[V];
#pragma unroll
        for (int p = 0; p < V; ++p) l[p] = first + p < a.experts ? Logit<HP>::value(row[first + p]) : -__builtin_huge_valf();
        float top = l[0];
#pragma unroll
        for (int p = 1; p < V; ++p) top = larger(top, l[p]);
        top = max16(top);
        const bool by_score = a.bias != nullptr || a.groups > 1;
        float total = 1.0f;
        if (a.softmax) {  // (the sum is needed for the weights in any case)
            total = 0.0f;
#pragma unroll
            for (int p = 0; p < V; ++p) total += l[p] > -__builtin_huge_valf() || l[p] != l[p] ? expf(l[p] - top) : 0.0f;
            total = sum16(total);
        }
        {
            float c[V];
            float border = 0.0f;
            if (by_score) {
                float most = 1.0f;
#pragma unroll
                for (int p = 0; p < V; ++p) {
                    float s = a.softmax ? (total > 0.0f ? expf(l[p] - top) / total : 0.0f) : sigmoid(l[p]);
                    if (a.bias && first + p < a.experts) {
                        const float b = a.bias[first + p];
                        s += b;
                        most = larger(most, fabsf(b) < 3e38f ? fabsf(b) : 1.0f);
                    }
                    c[p] = first + p < a.experts && s == s ? s : -__builtin_huge_valf();
                }
                // a score is off by less than 2^-21 (a few roundings of values up to 1), a sum with the bias by 2^-24 of it more
                border = max16(most) * 0x1p-20f;
            } else {
#pragma unroll
                for (int p = 0; p < V; ++p) c[p] = l[p] == l[p] ? l[p] : -__builtin_huge_valf();
            }
            const bool near = choose<float, V>(a, c, l16, border, choices[slot], scores[slot]);
            if (by_score && __builtin_amdgcn_ballot_w64(near)) {  // (uniform)
                double d[V], sum = 1.0;
                if (a.softmax) {
                    sum = 0.0;
#pragma unroll
                    for (int p = 0; p < V; ++p) sum += l[p] > -__builtin_huge_valf() || l[p] != l[p] ? exp((double)l[p] - (double)top) : 0.0;
                    sum = sum16(sum);
                }
#pragma unroll
                for (int p = 0; p < V; ++p) {
                    double s = a.softmax ? (sum > 0.0 ? exp((double)l[p] - (double)top) / sum : 0.0) : sigmoid((double)l[p]);
                    if (a.bias && first + p < a.experts) s += (double)a.bias[first + p];
                    d[p] = first + p < a.experts && s == s ? s : -__builtin_huge_val();
                }
                choose<double, V>(a, d, l16, 0.0, choices[slot], scores64[slot]);
            }
        }
        // the weights: lane j of a token has the j-th expert
        float chosen_sum = 0.0f;
        for (int j0 = 0; j0 < a.top_k; j0 += 16) {
            const int j = j0 + l16;
            float s = 0.0f;
            if (j < a.top_k) {
                const float v = Logit<HP>::value(row[choices[slot][j]]);
                s = a.softmax ? (total > 0.0f || total != total ? expf(v - top) / total : 0.0f) : sigmoid(v);
            }
            chosen_sum += sum16(s);
        }
        const float by = a.normalize ? (chosen_sum != 0.0f ? a.scale / chosen_sum : 0.0f) : a.scale;
        for (int j = l16; j < a.top_k; j += 16) {
            const int e = choices[slot][j];
            const float v = Logit<HP>::value(row[e]);
            const float s = a.softmax ? (total > 0.0f || total != total ? expf(v - top) / total : 0.0f) : sigmoid(v);
            if (valid) {
                a.weights[token * a.top_k + j] = s * by;
                a.indices[token * a.top_k + j] = e;
                atomicAdd(&hist[e], 1);
            }
        }
    }
    __syncthreads();
    for (int e = tid; e < a.experts; e += WAVES * 64) {
        if (a.counts)
            a.counts[e] = hist[e];
        else
            a.partial[(int64_t)blockIdx.x * a.experts + e] = hist[e];
    }
}

// counts[e] = sum over workgroups of partial[.][e]: 16 experts a workgroup, 16 threads each
__global__ __launch_bounds__(256) void route_counts_kernel(const int32_t* partial, int rows, int experts, int64_t* counts)
{
    __shared__ int sums[16][16];
    const int e = (int)blockIdx.x * 16 + (threadIdx.x & 15), part = threadIdx.x >> 4;
    int n = 0;
    if (e < experts)
        for (int r = part; r < rows; r += 16) n += partial[(int64_t)r * experts + e];
    sums[part][threadIdx.x & 15] = n;
    __syncthreads();
    if (part == 0 && e < experts) {
        int64_t all = 0;
#pragma unroll
        for (int p = 0; p < 16; ++p) all += sums[p][threadIdx.x];
        counts[e] = all;
    }
}

// ---- gradient of the logits ----------------------------------------------------------------------------------------------
//   normalize:  ds_j = scale (g_j - sum_m g_m w_m / scale) / D,  D the sum of the chosen s;  otherwise ds_j = scale g_j
//   sigmoid:    dl_e = ds_e s_e (1 - s_e);   softmax: dl_e = s_e (ds_e - sum_m ds_m s_m)
// ds is zero but for the chosen experts, and the softmax's sum is zero with normalize (the weights do not depend on the sum of all
// exponentials): only softmax without normalize has a gradient for all experts.  Bound by writing it.
struct RouteGradArgs {
    const void* logits;
    const float* weights;
    const int64_t* indices;
    const float* grad;
    int64_t tokens;
    int experts, top_k, softmax, normalize;
    float scale;
    void* out;
};

template <int HP, int V>
__global__ __launch_bounds__(256) void route_grad_kernel(RouteGradArgs a)
{
    typedef typename Logit<HP>::type logit_t;
    __shared__ float ds[16][kMostExperts];
    const int l16 = threadIdx.x & 15, slot = threadIdx.x >> 4;
    const int64_t token = (int64_t)blockIdx.x * 16 + slot;
    if (token >= a.tokens) return;  // (lanes of whole tokens; no barrier of the workgroup below)
    const logit_t* row = reinterpret_cast<const logit_t*>(a.logits) + token * a.experts;
    logit_t* out = reinterpret_cast<logit_t*>(a.out) + token * a.experts;
    for (int e = l16; e < a.experts; e += 16) ds[slot][e] = 0.0f;
    float dot = 0.0f;  // sum of g_m w_m / scale, the gradient's part that all chosen share
    for (int j = l16; j < a.top_k; j += 16) dot += a.grad[token * a.top_k + j] * a.weights[token * a.top_k + j];
    dot = sum16(dot);
    const bool all = a.softmax && !a.normalize;
    const float mean = a.normalize && a.scale != 0.0f ? dot / a.scale : 0.0f;
    wave_lds();
    for (int j = l16; j < a.top_k; j += 16) {
        const int64_t e = a.indices[token * a.top_k + j];
        if (e < 0 || e >= a.experts) continue;
        const float g = a.grad[token * a.top_k + j];
        if (all) {
            ds[slot][e] = a.scale * g;
        } else {
            // w_j (g_j - mean), with the sigmoid's (1 - s_j)
            const float v = a.weights[token * a.top_k + j] * (g - mean);
            ds[slot][e] = a.softmax ? v : v * sigmoid(-Logit<HP>::value(row[e]));
        }
    }
    wave_lds();
    if (!all) {
        for (int e = l16; e < a.experts; e += 16) out[e] = Logit<HP>::round(ds[slot][e]);
        return;
    }
    const int first = l16 * V;
    float l[V], top = -__builtin_huge_valf();
#pragma unroll
    for (int p = 0; p < V; ++p) {
        l[p] = first + p < a.experts ? Logit<HP>::value(row[first + p]) : -__builtin_huge_valf();
        top = larger(top, l[p]);
    }
    top = max16(top);
    float total = 0.0f;
#pragma unroll
    for (int p = 0; p < V; ++p) {
        l[p] = l[p] > -__builtin_huge_valf() || l[p] != l[p] ? expf(l[p] - top) : 0.0f;
        total += l[p];
    }
    total = sum16(total);
    // (dot is sum of g w = sum of ds s: w = scale s)
#pragma unroll
    for (int p = 0; p < V; ++p)
        if (first + p < a.experts) out[first + p] = Logit<HP>::round(total > 0.0f || total != total ? l[p] / total * (ds[slot][first + p] - dot) : 0.0f);
}

int route_blocks(int64_t tokens)
{
    const int64_t blocks = ceil_div(tokens, 16);
    return tokens <= kOneBlock ? 1 : blocks < 512 ? (int)blocks : 512;
}

template <int HP, int V>
int launch_route(const RouteArgs& a, hipStream_t st)
{
    constexpr int kWaves = V > 8 ? 8 : 16;  // (what 128 or 256 registers a lane allow)
    if (a.tokens <= kOneBlock)
        hipLaunchKernelGGL((route_kernel<HP, V, kWaves>), dim3(1), dim3(kWaves * 64), 0, st, a);
    else
        hipLaunchKernelGGL((route_kernel<HP, V, 4>), dim3(route_blocks(a.tokens)), dim3(256), 0, st, a);
    return launch_status("mi8_moe_route");
}

template <int HP>
int launch_route_experts(const RouteArgs& a, hipStream_t st)
{
    if (a.experts <= 16) return launch_route<HP, 1>(a, st);
    if (a.experts <= 64) return launch_route<HP, 4>(a, st);
    if (a.experts <= 128) return launch_route<HP, 8>(a, st);
    if (a.experts <= 256) return launch_route<HP, 16>(a, st);
    return launch_route<HP, 32>(a, st);
}

template <int HP>
int launch_route_grad(const RouteGradArgs& a, hipStream_t st)
{
    const dim3 grid((unsigned)ceil_div(a.tokens, 16));
    if (a.experts <= 64)
        hipLaunchKernelGGL((route_grad_kernel<HP, 4>), grid, dim3(256), 0, st, a);
    else if (a.experts <= 256)
        hipLaunchKernelGGL((route_grad_kernel<HP, 16>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((route_grad_kernel<HP, 32>), grid, dim3(256), 0, st, a);
    return launch_status("mi8_moe_route_grad");
}

int check_route(int64_t tokens, int32_t experts, int32_t top_k, int hp_dtype, const char* what)
{
    MI8_REQUIRE(hp_dtype == MI8_BF16 || hp_dtype == MI8_F32 || hp_dtype == MI8_F16, MI8_ERR_ARG, "%s: logits must be bf16, float16 or float32", what);
    MI8_REQUIRE(tokens > 0 && experts > 0 && top_k > 0, MI8_ERR_ARG, "%s: no tokens, no experts or no choice", what);
    MI8_REQUIRE(experts <= kMostExperts && top_k <= kMostTopK && top_k <= experts && tokens < ((int64_t)1 << 32), MI8_ERR_UNSUPPORTED,
                "%s: at most %d experts, of which at most %d are chosen", what, kMostExperts, kMostTopK);
    return MI8_OK;
}

}  // namespace
}  // namespace mi8

using namespace mi8;

extern "C" int64_t mi8_moe_route_workspace_words(int64_t tokens, int32_t experts)
{
    return tokens > kOneBlock && experts > 0 ? (int64_t)route_blocks(tokens) * experts : 0;
}

extern "C" int mi8_moe_route(const void* logits, int hp_dtype, int64_t tokens, int32_t experts, int32_t top_k, int32_t softmax, const float* bias,
                             int32_t groups, int32_t groups_kept, int32_t normalize, float scale, int32_t* workspace, float* weights,
                             int64_t* indices, int64_t* counts, void* stream)
{
    if (int rc = check_route(tokens, experts, top_k, hp_dtype, "mi8_moe_route")) return rc;
    MI8_REQUIRE(logits && weights && indices && counts, MI8_ERR_ARG, "mi8_moe_route: null pointer");
    MI8_REQUIRE(groups > 0 && groups <= kMostGroups && experts % groups == 0 && groups_kept > 0 && groups_kept <= groups, MI8_ERR_UNSUPPORTED,
                "mi8_moe_route: %d experts in %d groups of which %d are kept (at most %d groups of equal size)", experts, groups, groups_kept, kMostGroups);
    MI8_REQUIRE(top_k <= experts / groups * groups_kept, MI8_ERR_UNSUPPORTED, "mi8_moe_route: %d experts of %d groups of %d are too few to choose %d",
                experts / groups * groups_kept, groups_kept, experts / groups, top_k);
    MI8_REQUIRE(tokens <= kOneBlock || workspace, MI8_ERR_ARG, "mi8_moe_route: needs mi8_moe_route_workspace_words() words");
    // (all groups kept: nothing is left out)
    RouteArgs a{logits, bias, tokens, experts, top_k, groups_kept == groups ? 1 : groups, groups_kept, softmax, normalize, scale, weights, indices,
                tokens <= kOneBlock ? counts : nullptr, workspace};
    hipStream_t st = (hipStream_t)stream;
    const int rc = hp_dtype == MI8_BF16  ? launch_route_experts<MI8_BF16>(a, st)
                   : hp_dtype == MI8_F16 ? launch_route_experts<MI8_F16>(a, st)
                                         : launch_route_experts<MI8_F32>(a, st);
    if (rc || tokens <= kOneBlock) return rc;
    hipLaunchKernelGGL(route_counts_kernel, dim3((experts + 15) / 16), dim3(256), 0, st, workspace, route_blocks(tokens), experts, counts);
    return launch_status("mi8_moe_route(counts)");
}

extern "C" int mi8_moe_route_grad(const void* logits, int hp_dtype, int64_t tokens, int32_t experts, int32_t top_k, int32_t softmax, int32_t normalize,
                                  float scale, const float* weights, const int64_t* indices, const float* grad, void* grad_logits, void* stream)
{
    if (int rc = check_route(tokens, experts, top_k, hp_dtype, "mi8_moe_route_grad")) return rc;
    MI8_REQUIRE(logits && weights && indices && grad && grad_logits, MI8_ERR_ARG, "mi8_moe_route_grad: null pointer");
    RouteGradArgs a{logits, weights, indices, grad, tokens, experts, top_k, softmax, normalize, scale, grad_logits};
    hipStream_t st = (hipStream_t)stream;
    if (hp_dtype == MI8_BF16) return launch_route_grad<MI8_BF16>(a, st);
    if (hp_dtype == MI8_F16) return launch_route_grad<MI8_F16>(a, st);
    return launch_route_grad<MI8_F32>(a, st);
}
