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
// Without a bias or groups the choice goes by the logits themselves, which order the scores; else it is the one of 64-bit scores.  With a bias, or by sums
// of groups, the scores' float32 errors could swap neighbours: where two values that decide are closer than those errors (kBorder), or equal, the wave
// repeats its choice in 64 bits: with scores of normal logits 0.1 to 2 % of the waves where there is a bias, up to 9 % of float32 and 8 to 21 % of
// bf16 logits in groups without one (equal logits are equal scores there).
#include "mi8_block.h"

namespace mi8 {
namespace {

struct RouteArgs {
    const void* logits;
    const float* bias;  // null, or [experts]
    int64_t tokens;
    int experts, top_k, groups, kept, softmax, normalize;
    int wide;       // rows start at multiples of 16 bytes
    int wide_bias;  // there is a bias, and it may be read in pieces of 16 bytes
    float scale;
    float* weights;       // [tokens, top_k]
    int64_t* indices;     // [tokens, top_k]
    int64_t* counts;      // [experts] (a launch of one workgroup)
    int32_t* partial;     // [workgroups, experts] (others)
};

constexpr int kMostExperts = 512, kMostTopK = 64, kMostGroups = 32;
constexpr int kMostBlocks = 1024;
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
template <int CTRL>
__device__ __forceinline__ int64_t dpp(int64_t v) { return __builtin_bit_cast(int64_t, dpp<CTRL>(__builtin_bit_cast(double, v))); }
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
// Integers in the order of the values (no NaN; the two zeros are one): a maximum of them is one instruction
__device__ __forceinline__ int key_of(float v)
{
    const int u = __builtin_bit_cast(int, v + 0.0f);
    return u ^ (u >> 31 & 0x7FFFFFFF);
}
__device__ __forceinline__ float value_of(int k) { return __builtin_bit_cast(float, k ^ (k >> 31 & 0x7FFFFFFF)); }
__device__ __forceinline__ int64_t key_of(double v)
{
    const int64_t u = __builtin_bit_cast(int64_t, v + 0.0);
    return u ^ (u >> 63 & 0x7FFFFFFFFFFFFFFF);
}
__device__ __forceinline__ double value_of(int64_t k) { return __builtin_bit_cast(double, k ^ (k >> 63 & 0x7FFFFFFFFFFFFFFF)); }
template <typename T>
__device__ __forceinline__ T max16(T v) { return over16(v, [](T a, T b) { return larger(a, b); }); }
template <typename T>
__device__ __forceinline__ T sum16(T v) { return over16(v, [](T a, T b) { return a + b; }); }
__device__ __forceinline__ int min16(int v) { return over16(v, [](int a, int b) { return a < b ? a : b; }); }

// e^x for x up to 88, off by two units in the last place of a normal number (0 or so below 2^-126): 2^(x log2 e) by the instruction, the product's rounding (and the constant's) put right to first
// order.  Below -150 it is 0 as at -150; a NaN stays one.
__device__ __forceinline__ float exp32(float x)
{
    constexpr float kLog2e = 0x1.715476p+0f, kLog2eRest = 0x1.4ae0bep-26f, kLn2 = 0x1.62e430p-1f;
    x = x < -150.0f ? -150.0f : x;
    const float t = x * kLog2e;
    const float rest = __builtin_fmaf(x, kLog2eRest, __builtin_fmaf(x, kLog2e, -t));
    const float e = __builtin_amdgcn_exp2f(t);
    return __builtin_fmaf(e, rest * kLn2, e);
}
// 1 / x for finite x of ordinary size: the instruction and one step of Newton's
__device__ __forceinline__ float inverse32(float x)
{
    const float r = __builtin_amdgcn_rcpf(x);
    return __builtin_fmaf(__builtin_fmaf(-x, r, 1.0f), r, r);
}
template <typename T>
__device__ __forceinline__ T sigmoid(T l);
template <>
__device__ __forceinline__ float sigmoid(float l) { return inverse32(1.0f + exp32(-l > 88.0f ? 88.0f : -l)); }
template <>
__device__ __forceinline__ double sigmoid(double l) { return 1.0 / (1.0 + exp(-l)); }

// term(P) + .. + term(P + N - 1): the sums of four in pairs, so that no term meets more than 6 additions of the 31 it would with N = 32
template <int P, int N, typename Term>
__device__ __forceinline__ float lane_sum(const Term& term)
{
    if constexpr (N > 4) {
        const float head = lane_sum<P, N / 2>(term);
        return head + lane_sum<P + N / 2, N / 2>(term);
    } else {
        float s = term(P);
#pragma unroll
        for (int p = 1; p < N; ++p) s += term(P + p);
        return s;
    }
}

// How close values that decide may be, as a share of the largest bias (1 if that is less), before float32 could have them in the wrong order.  In
// u = 2^-24, a score s is off by at most
//   softmax  26 s: exp32 4, the rounding of l - top (d for e^-d: less than 1 of the largest score), inverse32 2, the product 1; the sum of all: its
//            terms' exp32 4, their roundings of l - top (weighted by the terms, less than 4 with 512 of them), 10 additions (6 in the lane, 4 across)
//   sigmoid   7 s: exp32 4, the addition of 1, inverse32 2
// Two experts: softmax scores add up to 1, so 26 together, sigmoids 14, and each sum with the bias b is rounded, 2 (1 + b): 30 max(1, b).  Groups are
// compared by sums of two, with twice the border: the scores' errors 26 (four of a softmax add up to 1) or 28, four sums with the bias and two of two
// 8 (1 + b), the comparison's own sum 4 max(1, b): 48 max(1, b).
constexpr float kBorder = 0x1p-19f;  // 32 u

constexpr float kLittle = 0x1p-100f;          // (float32 loses scores below 2^-126)
constexpr float kLeastExponent = -709.7827f;  // e^this is 2^-1024: where all chosen scores are less they count as zero, as in 64 bits

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

// A token's choice from c[V] into choice[top_k] (LDS of the token; group_scores likewise).  An expert that is out - not there, of no kept group, or
// chosen - has the least key; one whose c is -infinity comes before it, the lowest index first (top_k is at most the size of the kept groups).  Returns
// whether values that decide are not further apart than `border` (0: not asked).
template <typename T, int V>
__device__ __forceinline__ bool choose(const RouteArgs& a, const T (&c)[V], const int l16, const T border, int* choice, T* group_scores)
{
    constexpr T kLeast = -__builtin_huge_val();
    typedef decltype(key_of(kLeast)) key_t;
    constexpr key_t kOut = (key_t)1 << (8 * sizeof(key_t) - 1);
    const int first = l16 * V;
    bool near = false;
    key_t key[V];
#pragma unroll
    for (int p = 0; p < V; ++p) key[p] = first + p < a.experts ? key_of(c[p]) : kOut;
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
#pragma unroll
            for (int p = 0; p < V; ++p) {
                if (!whole && first + p == next && first + p < a.experts) {
                    keep = kept(++g);
                    next += size;
                }
                key[p] = keep ? key[p] : kOut;
            }
        }
        near = near && border > 0;
    }
    T previous = 0;
    for (int j = 0; j <= a.top_k; ++j) {
        key_t top = key[0];
#pragma unroll
        for (int p = 1; p < V; ++p) top = larger(top, key[p]);
        top = max16(top);
        if (border > 0) {
            const T value = value_of(top);
            if (j > 0 && !(previous - value > border)) near = true;  // (also between the last that is chosen and the next)
            previous = value;
        }
        if (j == a.top_k) break;
        int at = 1 << 20;
#pragma unroll
        for (int p = V - 1; p >= 0; --p) at = key[p] == top ? p : at;
        const int winner = min16(at + first);
#pragma unroll
        for (int p = 0; p < V; ++p) key[p] = winner == first + p ? kOut : key[p];
        if (l16 == 0) choice[j] = winner;
    }
    wave_lds();
    return near;
}

// The same from the logits in 64 bits
template <int HP, int V>
__device__ __forceinline__ void choose_in_64_bits(const RouteArgs& a, const typename Logit<HP>::type* row, const int l16, int* choice,
                                                            double* group_scores)
{
    const int first = l16 * V;
    double d[V], top = -__builtin_huge_val(), sum = 0.0;
#pragma unroll
    for (int p = 0; p < V; ++p) {
        d[p] = first + p < a.experts ? (double)Logit<HP>::value(row[first + p]) : -__builtin_huge_val();
        top = larger(top, d[p]);
    }
    if (a.softmax) {
        top = max16(top);
#pragma unroll
        for (int p = 0; p < V; ++p) {
            d[p] = d[p] > -__builtin_huge_val() || d[p] != d[p] ? exp(d[p] - top) : 0.0;
            sum += d[p];
        }
        sum = sum16(sum);
    }
#pragma unroll
    for (int p = 0; p < V; ++p) {
        double s = a.softmax ? (sum > 0.0 ? d[p] / sum : 0.0) : sigmoid(d[p]);
        if (a.bias && first + p < a.experts) s += (double)a.bias[first + p];
        d[p] = first + p < a.experts && s == s ? s : -__builtin_huge_val();
    }
    choose<double, V>(a, d, l16, 0.0, choice, group_scores);
}

template <int HP, int V, int WAVES>
__global__ __launch_bounds__(WAVES * 64, WAVES == 4 ? (V > 16 ? 2 : V > 8 ? 3 : 4) : 1) void route_kernel(RouteArgs a)
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
        constexpr int kPer16 = 16 / (int)sizeof(logit_t);
        if (V % kPer16 == 0 && a.wide) {  // (uniform)
#pragma unroll
            for (int c = 0; c < V / kPer16; ++c) {
                struct alignas(16) { logit_t v[kPer16]; } piece;
                if (first + c * kPer16 < a.experts) piece = *reinterpret_cast<const decltype(piece)*>(row + first + c * kPer16);
#pragma unroll
                for (int p = 0; p < kPer16; ++p) l[c * kPer16 + p] = first + c * kPer16 < a.experts ? Logit<HP>::value(piece.v[p]) : -__builtin_huge_valf();
            }
        } else {
#pragma unroll
            for (int p = 0; p < V; ++p) l[p] = first + p < a.experts ? Logit<HP>::value(row[first + p]) : -__builtin_huge_valf();
        }
        float top = l[0];
#pragma unroll
        for (int p = 1; p < V; ++p) top = larger(top, l[p]);
        top = max16(top);
        const bool by_score = a.bias != nullptr || a.groups > 1;
        float total = 1.0f;
        if (a.softmax) {  // (the sum is needed for the weights in any case)
            total = sum16(lane_sum<0, V>([&](int p) __attribute__((always_inline)) { return l[p] > -__builtin_huge_valf() || l[p] != l[p] ? exp32(l[p] - top) : 0.0f; }));
        }
        const float inv_total = inverse32(total);
        {
            float c[V];
            float border = 0.0f;
            if (by_score) {
                float most = 1.0f, bias[V];
#pragma unroll
                for (int p = 0; p < V; ++p) bias[p] = 0.0f;
                if (V % 4 == 0 && a.wide_bias) {  // (uniform)
#pragma unroll
                    for (int p = 0; p < V; p += 4)
                        if (first + p < a.experts) {
                            const float4 b = *reinterpret_cast<const float4*>(a.bias + first + p);
                            bias[p] = b.x, bias[p + 1] = b.y, bias[p + 2] = b.z, bias[p + 3] = b.w;
                        }
                } else if (a.bias) {
#pragma unroll
                    for (int p = 0; p < V; ++p)
                        if (first + p < a.experts) bias[p] = a.bias[first + p];
                }
#pragma unroll
                for (int p = 0; p < V; ++p) {
                    float s = a.softmax ? (total > 0.0f ? exp32(l[p] - top) * inv_total : 0.0f) : sigmoid(l[p]);
                    s += bias[p];
                    most = larger(most, fabsf(bias[p]) < 3e38f ? fabsf(bias[p]) : 1.0f);
                    c[p] = first + p < a.experts && s == s ? s : -__builtin_huge_valf();
                }
                border = max16(most) * kBorder;
            } else {
#pragma unroll
                for (int p = 0; p < V; ++p) c[p] = l[p] == l[p] ? l[p] : -__builtin_huge_valf();
            }
            const bool near = choose<float, V>(a, c, l16, border, choices[slot], scores[slot]);
            if (by_score && __builtin_amdgcn_ballot_w64(near))  // (uniform)
                choose_in_64_bits<HP, V>(a, row, l16, choices[slot], scores64[slot]);
        }
        // the weights: lane j of a token has the j-th expert (and 16 further on)
        float low = 0.0f;
        bool little = false, shifted = false;  // a chosen score is little; (a token's) scores are divided by e^low
        auto score = [&](int j, int& e) __attribute__((always_inline)) {
            e = choices[slot][j];
            const float v = Logit<HP>::value(row[e]);
            if (shifted) return a.softmax ? exp32(v - low) : exp32(v - low) * sigmoid(-v);
            const float s = a.softmax ? (total > 0.0f || total != total ? exp32(v - top) * inv_total : 0.0f) : sigmoid(v);
            little = little || s < kLittle;
            return s;
        };
        int e = 0;
        float s = l16 < a.top_k ? score(l16, e) : 0.0f;
        float by = a.scale;
        if (a.normalize) {
            float sum;
            auto add = [&]() __attribute__((always_inline)) {
                sum = sum16(s);
                for (int j = 16; j < a.top_k; j += 16) {
                    int unused;
                    sum += sum16(j + l16 < a.top_k ? score(j + l16, unused) : 0.0f);
                }
            };
            add();
            // Scores near or below the least normal number: relative to the largest chosen one they are not.  s / e^low is e^(l - low) / (1 + e^l) for
            // low, the largest chosen logit, up to 0 (beyond, a little score has no normal weight), and the sum of all exponentials is a common factor.
            if (__builtin_amdgcn_ballot_w64(little)) {  // (uniform)
                float most = -__builtin_huge_valf();
                for (int j = l16; j < a.top_k; j += 16) most = larger(most, Logit<HP>::value(row[choices[slot][j]]));
                most = max16(most);
                if (max16((int)little) && (a.softmax ? most - top : most) >= kLeastExponent && (a.softmax || most <= 0.0f)) {
                    shifted = true;
                    low = most;
                }
                if (l16 < a.top_k) s = score(l16, e);
                add();
            }
            by = sum != 0.0f ? a.scale / sum : 0.0f;
        }
        auto store = [&](int j, int expert, float value) __attribute__((always_inline)) {
            a.weights[token * a.top_k + j] = value * by;
            a.indices[token * a.top_k + j] = expert;
            atomicAdd(&hist[expert], 1);
        };
        if (valid && l16 < a.top_k) store(l16, e, s);
        for (int j = l16 + 16; valid && j < a.top_k; j += 16) {
            const float more = score(j, e);
            store(j, e, more);
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

// counts[e] = sum over workgroups of partial[.][e]: 16 experts a workgroup, 64 threads each, all of whose reads are in flight together
__global__ __launch_bounds__(1024) void route_counts_kernel(const int32_t* partial, int rows, int experts, int64_t* counts)
{
    __shared__ int sums[64][17];
    const int e = (int)blockIdx.x * 16 + (threadIdx.x & 15), part = threadIdx.x >> 4;
    int n[kMostBlocks / 64];
#pragma unroll
    for (int i = 0; i < kMostBlocks / 64; ++i) {
        const int r = part + 64 * i;
        n[i] = e < experts && r < rows ? partial[(int64_t)r * experts + e] : 0;
    }
#pragma unroll
    for (int i = 1; i < kMostBlocks / 64; ++i) n[0] += n[i];
    sums[part][threadIdx.x & 15] = n[0];
    __syncthreads();
    if (part < 16 && (int)blockIdx.x * 16 + part < experts) {  // sixteen lanes an expert
        int all = 0;
#pragma unroll
        for (int p = 0; p < 4; ++p) all += sums[(threadIdx.x & 15) + 16 * p][part];
        all = over16(all, [](int a, int b) { return a + b; });
        if ((threadIdx.x & 15) == 0) counts[blockIdx.x * 16 + part] = all;
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
        l[p] = l[p] > -__builtin_huge_valf() || l[p] != l[p] ? exp32(l[p] - top) : 0.0f;
        total += l[p];
    }
    total = sum16(total);
    const float inv_total = inverse32(total);
    // (dot is sum of g w = sum of ds s: w = scale s)
#pragma unroll
    for (int p = 0; p < V; ++p)
        if (first + p < a.experts) out[first + p] = Logit<HP>::round(total > 0.0f || total != total ? l[p] * inv_total * (ds[slot][first + p] - dot) : 0.0f);
}

int route_blocks(int64_t tokens)
{
    const int64_t blocks = ceil_div(tokens, 16);
    return tokens <= kOneBlock ? 1 : blocks < kMostBlocks ? (int)blocks : kMostBlocks;
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
    MI8_REQUIRE(experts <= kMostExperts && top_k <= kMostTopK && top_k <= experts && tokens < ((int64_t)1 << 31), MI8_ERR_UNSUPPORTED,
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
    RouteArgs a{logits, bias, tokens, experts, top_k, groups_kept == groups ? 1 : groups, groups_kept, softmax, normalize,
                aligned16(logits) && experts * (hp_dtype == MI8_F32 ? 4 : 2) % 16 == 0, bias && aligned16(bias) && experts % 4 == 0, scale, weights, indices,
                tokens <= kOneBlock ? counts : nullptr, workspace};
    hipStream_t st = (hipStream_t)stream;
    const int rc = hp_dtype == MI8_BF16  ? launch_route_experts<MI8_BF16>(a, st)
                   : hp_dtype == MI8_F16 ? launch_route_experts<MI8_F16>(a, st)
                                         : launch_route_experts<MI8_F32>(a, st);
    if (rc || tokens <= kOneBlock) return rc;
    hipLaunchKernelGGL(route_counts_kernel, dim3((experts + 15) / 16), dim3(1024), 0, st, workspace, route_blocks(tokens), experts, counts);
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
