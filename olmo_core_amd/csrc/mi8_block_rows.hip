// A few rows times a weight with block scales, the rows quantised on the way: y = q(x) . B^T for the tokens of a generation step.
//
// Bound by reading the weight once.  A workgroup of four or eight waves takes 32 rows of it, each wave its share of K.  The bytes go
// straight to LDS, whole 128-byte lines, into a ring that is the wave's own: four blocks (16 KB a wave) in flight and not a barrier.
// (Read from memory in the layout of the MFMA's fragments, 16 bytes of another row every lane, one row times
// 11008 x 4096 took 15.5 us where this takes 12.2; a cast and a product of 64 x 64 tiles 4.0 + 10.7.)  The
// activations come from the L2 in their own type: a lane has 32 of the 128 values of a block and row, four lanes share its largest magnitude, and
// the values become float8 in registers, as the casts of mi8_block_cast.hip make them - no launch and no memory for that.  It costs
// every workgroup the conversion of all rows, hence 16 of them (of 32, in two MFMA tiles, the conversion took longer than a launch of its own), and
// hence 32 rows of weight, not 16.  The waves' sums meet in LDS, in the order of K.
#include "mi8_block_gemm.h"
#include "mi8_gemm.h"
#include "mi8_groups.h"

namespace mi8 {
using namespace gemm;
using namespace block;
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));

struct BlockRowsArgs {
    const void* x;      // [M, K]
    int64_t ldx;
    const uint8_t* B;   // rows of ldb bytes
    const uint8_t* eb;  // scales of B
    int64_t ldb;
    void* C;            // [M, N]
    int M, N, K, nk;
    const int64_t* sizes;  // (groups of rows)
    int E;
    int64_t b_group_stride, eb_group_stride;
};

constexpr int kRowsN = 32;

// 32 values of a row as they are in memory, and as float8: four lanes (16 and 32 apart) have the block
template <int HP>
struct Raw;
template <>
struct Raw<MI8_BF16> {
    v4i v[4];
    __device__ __forceinline__ uint32_t absmax() const
    {
        typedef uint16_t pair_t __attribute__((ext_vector_type(2)));
        uint32_t m = 0;
#pragma unroll
        for (int c = 0; c < 16; ++c)
            m = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(pair_t, m), __builtin_bit_cast(pair_t, (uint32_t)v[c / 4][c % 4] & 0x7FFF7FFFu)));
        return umax32(m << 16, m & 0xFFFF0000u);
    }
    __device__ __forceinline__ float at(int i) const
    {
        const uint32_t w = (uint32_t)v[i / 8][i / 2 % 4];
        return bits_to_f32(i & 1 ? w & 0xFFFF0000u : w << 16);
    }
};
template <>
struct Raw<MI8_F32> {
    v4i v[8];
    __device__ __forceinline__ uint32_t absmax() const
    {
        uint32_t m = 0;
#pragma unroll
        for (int c = 0; c < 32; ++c) m = umax32(m, (uint32_t)v[c / 4][c % 4] & 0x7FFFFFFFu);
        return m;
    }
    __device__ __forceinline__ float at(int i) const { return bits_to_f32((uint32_t)v[i / 4][i % 4]); }
};

template <int HP>
__device__ __forceinline__ v8i quantise32(const Raw<HP>& x, uint32_t& exponent)
{
    uint32_t m = x.absmax();
    auto pair = __builtin_amdgcn_permlane16_swap(m, m, false, false);  // (rows of 16 lanes 0 and 1, 2 and 3)
    m = umax32(pair[0], pair[1]);
    pair = __builtin_amdgcn_permlane32_swap(m, m, false, false);
    m = umax32(pair[0], pair[1]);
    float s;
    uint8_t byte;
    scale_of(m, s, byte);
    exponent = byte;
    v8i q;
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = (int)cvt4<MI8_E4M3, false>(x.at(4 * i) * s, x.at(4 * i + 1) * s, x.at(4 * i + 2) * s, x.at(4 * i + 3) * s);
    return q;
}

typedef __attribute__((address_space(1))) const void* rows_global_t;
typedef __attribute__((address_space(3))) void* rows_lds_t;
typedef const __attribute__((address_space(3))) v4i* rows_frag_t;

constexpr int kSlot = kRowsN * BK, kSlots = 4;  // a block of K of the workgroup's rows of B; how many of them a wave has in flight
constexpr int rows_vmcnt(int n) { return (n & 15) | ((n >> 4) << 14) | 0x0F70; }  // s_waitcnt: at most n memory operations in flight
constexpr int rows_lds_bytes(int waves) { return waves * (kSlots * kSlot + 16 * (kRowsN + 1) * 4); }

// HP: type of x and of the output.
template <int HP, bool GROUPED, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 2) void block_rows_kernel(BlockRowsArgs a)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    float (*sums)[16][kRowsN + 1] = reinterpret_cast<float (*)[16][kRowsN + 1]>(lds + WAVES * kSlots * kSlot);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, kb = lane >> 4;
    const int n0 = (int)blockIdx.x * kRowsN;
    typedef typename std::conditional<HP == MI8_BF16, uint16_t, float>::type out_t;

    int64_t row0 = 0;
    int rows = a.M;
    const uint8_t* B = a.B;
    const uint8_t* eb = a.eb;
    if constexpr (GROUPED) {
        const GroupSpan s = locate_group<128, false>(a.sizes, a.E, a.M, (int)blockIdx.y < a.E ? (int64_t)blockIdx.y : a.E - 1);
        if ((int)blockIdx.y == a.E) {  // the rows behind the last group
            for (int64_t i = threadIdx.x; i < (a.M - s.rows_before - s.m) * kRowsN; i += WAVES * 64)
                if (n0 + i % kRowsN < a.N) reinterpret_cast<out_t*>(a.C)[(s.rows_before + s.m + i / kRowsN) * a.N + n0 + i % kRowsN] = 0;
            return;
        }
        row0 = s.rows_before;
        rows = (int)s.m;
        B += s.e * a.b_group_stride;
        eb += s.e * a.eb_group_stride;
    }
    constexpr int kChunks = HP == MI8_BF16 ? 4 : 8;  // loads of 16 bytes for 32 values
    constexpr int kIssued = kChunks + 1 + 4;         // memory operations of a block: rows of x, scales, rows of B
    const int per_wave = (a.nk + WAVES - 1) / WAVES;
    const int first = wave * per_wave, last = first + per_wave < a.nk ? first + per_wave : a.nk;
    // B: a load of the wave fills eight rows of a slot, 128 bytes each (16-byte pieces swizzled as the fragment reads want them); rows past the
    // last one re-read it (their sums are not stored).  A wave reads only what it has loaded itself: no barriers.
    uint8_t* ring = lds + wave * kSlots * kSlot;
    const int lr = lane >> 3;
    uint32_t b_at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = 8 * i + lr, n = n0 + r < a.N ? r : a.N - 1 - n0;
        b_at[i] = (uint32_t)(n * (int)a.ldb) + (uint32_t)(((lane & 7) ^ swz16(r)) << 4);
    }
    const uint8_t* b_tile = B + (int64_t)n0 * a.ldb;
    auto fetch_b = [&](int k, int slot) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            __builtin_amdgcn_global_load_lds((rows_global_t)(b_tile + (int64_t)k * BK + b_at[i]), (rows_lds_t)(ring + slot * kSlot + 8 * i * BK), 16, 0, 0);
    };
    uint32_t f_at[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) f_at[q] = (uint32_t)(uintptr_t)(rows_lds_t)ring + (uint32_t)(r16 * BK) + ((uint32_t)((2 * kb + q) ^ swz16(r16)) << 4);
    const int64_t eb_step = padded(a.N);
    const uint8_t* e_row = eb + n0 / 128 * 128 + 8 * r16 + n0 % 128 / 16;  // two tiles' bytes, next to each other

    for (int m0 = 0; m0 < rows; m0 += 16) {  // (one pass unless a group has more rows)
        v4f acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
        const int m = m0 + r16;
        const bool valid = m < rows;
        // (a lane whose row or column is not there points past the end and gets zeros)
        const __amdgpu_buffer_rsrc_t x_rows = __builtin_amdgcn_make_buffer_rsrc(
            (void*)(reinterpret_cast<const uint8_t*>(a.x) + (row0 + m0) * a.ldx * HpVec<HP>::kBytes), 0, (int)(uint32_t)((rows - m0 < 16 ? rows - m0 : 16) * a.ldx * HpVec<HP>::kBytes),
            0x00020000);
        const int x_at = (r16 * (int)a.ldx + 32 * kb) * HpVec<HP>::kBytes, columns = a.K - 32 * kb;
        auto fetch = [&](Raw<HP>& to, int k) __attribute__((always_inline)) {
            const int at = valid ? x_at : 0x7FFFFF00;
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {  // (K % 16 == 0: a load is inside a row or outside)
                const int there = k * 128 + c * (32 / kChunks) < columns ? at + 16 * c : 0x7FFFFF00;
                to.v[c] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(x_rows, there, k * 128 * HpVec<HP>::kBytes, 0));
            }
        };
        Raw<HP> x[kSlots];
        uint32_t e[kSlots];
        auto issue = [&](int k, int u) __attribute__((always_inline)) {
            fetch(x[u], k);
            e[u] = *reinterpret_cast<const uint16_t*>(e_row + k * eb_step);
            fetch_b(k, u);
        };
#pragma unroll
        for (int u = 0; u < kSlots; ++u) {
            if (first + u < last) issue(first + u, u);
            asm volatile("" ::: "memory");  // (the waits below count operations: those of a block stay behind the ones of the block before)
            __builtin_amdgcn_sched_barrier(0);
        }
        for (int k0 = first; k0 < last; k0 += kSlots) {
#pragma unroll
            for (int u = 0; u < kSlots; ++u) {
                const int k = k0 + u;
                if (k >= last) break;  // (uniform)
                // what was issued for this block has landed; that of up to three later ones may be in flight (operations complete in order)
                if (k + 3 < last)
                    __builtin_amdgcn_s_waitcnt(rows_vmcnt(3 * kIssued));
                else if (k + 2 < last)
                    __builtin_amdgcn_s_waitcnt(rows_vmcnt(2 * kIssued));
                else if (k + 1 < last)
                    __builtin_amdgcn_s_waitcnt(rows_vmcnt(kIssued));
                else
                    __builtin_amdgcn_s_waitcnt(rows_vmcnt(0));
                asm volatile("" ::: "memory");
                v4i b[2][2];
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int h = 0; h < 2; ++h) b[t][h] = *reinterpret_cast<rows_frag_t>((uintptr_t)(f_at[h] + u * kSlot + t * 16 * BK));
                uint32_t ea;
                const v8i q = quantise32<HP>(x[u], ea);
                acc[0] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(__builtin_shufflevector(b[0][0], b[0][1], 0, 1, 2, 3, 4, 5, 6, 7), q, acc[0], 0, 0, 0,
                                                                          (int)e[u], 0, (int)ea);
                acc[1] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(__builtin_shufflevector(b[1][0], b[1][1], 0, 1, 2, 3, 4, 5, 6, 7), q, acc[1], 0, 0, 1,
                                                                          (int)e[u], 0, (int)ea);
                __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the slot has been read
                asm volatile("" ::: "memory");
                if (k + kSlots < last) issue(k + kSlots, u);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        // acc[t][j] of lane l: row l % 16, column 16 t + 4 (l / 16) + j
        if (m0 > 0) __syncthreads();  // (the sums before have been read)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) sums[wave][r16][16 * t + 4 * kb + j] = acc[t][j];
        __syncthreads();
#pragma unroll
        for (int part = 0; part < 8 / WAVES; ++part) {
            const int at = part * WAVES * 64 + threadIdx.x, r = at / kRowsN, c = at % kRowsN;
            float s = sums[0][r][c];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) s += sums[w][r][c];
            if (m0 + r < rows && n0 + c < a.N) {
                if constexpr (HP == MI8_BF16)
                    reinterpret_cast<uint16_t*>(a.C)[(row0 + m0 + r) * a.N + n0 + c] = f32_to_bf16_bits(s);
                else
                    reinterpret_cast<float*>(a.C)[(row0 + m0 + r) * a.N + n0 + c] = s;
            }
        }
    }
}

template <int HP, bool GROUPED, int WAVES>
int launch_rows(const BlockRowsArgs& a, hipStream_t st)
{
    auto kern = block_rows_kernel<HP, GROUPED, WAVES>;
    static std::atomic<uint64_t> configured{0};
    if (int rc = reserve_dynamic_lds(reinterpret_cast<const void*>(kern), rows_lds_bytes(WAVES), configured, "mi8_block_rows")) return rc;
    hipLaunchKernelGGL(kern, dim3((unsigned)ceil_div(a.N, kRowsN), GROUPED ? a.E + 1 : 1), dim3(WAVES * 64), rows_lds_bytes(WAVES), st, a);
    return launch_status("mi8_block_rows");
}

// Eight waves, of which a compute unit holds one workgroup, where there is one for each; beyond, four, of which it holds two.
template <int HP>
int launch_rows(const BlockRowsArgs& a, hipStream_t st)
{
    if (ceil_div(a.N, kRowsN) * (a.sizes ? a.E : 1) <= 256) return a.sizes ? launch_rows<HP, true, 8>(a, st) : launch_rows<HP, false, 8>(a, st);
    return a.sizes ? launch_rows<HP, true, 4>(a, st) : launch_rows<HP, false, 4>(a, st);
}

}  // namespace
}  // namespace mi8

using namespace mi8;

extern "C" int64_t mi8_block_rows_max(int32_t num_groups) { return num_groups > 0 ? 512 : 16; }

extern "C" int mi8_block_rows(const void* x, int hp_dtype, int64_t M, const void* b, int64_t ldb, int64_t b_group_stride, const void* b_scales,
                              const int64_t* group_sizes, int32_t num_groups, int64_t N, int64_t K, void* out, void* stream)
{
    MI8_REQUIRE(x && b && b_scales && out, MI8_ERR_ARG, "mi8_block_rows: null pointer");
    MI8_REQUIRE(hp_dtype == MI8_BF16 || hp_dtype == MI8_F32, MI8_ERR_ARG, "mi8_block_rows: x must be bf16 or float32");
    MI8_REQUIRE(M > 0 && N > 0 && K > 0 && num_groups >= 0 && (num_groups == 0) == (group_sizes == nullptr), MI8_ERR_ARG, "mi8_block_rows: empty problem");
    MI8_REQUIRE(M <= mi8_block_rows_max(num_groups) && num_groups < 65535, MI8_ERR_UNSUPPORTED, "mi8_block_rows: %lld rows, at most %lld", (long long)M,
                (long long)mi8_block_rows_max(num_groups));
    MI8_REQUIRE(K % 16 == 0 && K < (1 << 24) && N < (1 << 30) && ldb % 16 == 0 && ldb >= block::padded(K) && ldb < (1 << 26) && b_group_stride % 16 == 0, MI8_ERR_UNSUPPORTED,
                "mi8_block_rows: K (below 2^24) and the pitches must be multiples of 16, ldb at least round_up(K, 128) and below 2^26");
    MI8_REQUIRE(aligned16(x) && aligned16(b) && aligned16(b_scales) && (reinterpret_cast<uintptr_t>(out) & 3) == 0, MI8_ERR_UNSUPPORTED,
                "mi8_block_rows: x, weight and scales must be 16-byte aligned");
    BlockRowsArgs a{x, K, (const uint8_t*)b, (const uint8_t*)b_scales, ldb, out, (int)M, (int)N, (int)K, (int)ceil_div(K, 128), group_sizes, num_groups,
                    b_group_stride, mi8_block_scale_bytes(N, K)};
    hipStream_t st = (hipStream_t)stream;
    return hp_dtype == MI8_BF16 ? launch_rows<MI8_BF16>(a, st) : launch_rows<MI8_F32>(a, st);
}
