// Products of float8 operands with block scales (mi8_block.h):  C[M, N] = sum over blocks of K of 2^(ea + eb) A_block . B_block^T,
// dense, for ragged groups of rows (the experts of a routed layer) and over ragged groups of tokens (their weight gradients).
//
// One block is one step of v_mfma_scale_f32_16x16x128_f8f6f4, whose scale operands are the exponent bytes of the 16 rows of
// either matrix: the scales are applied in the matrix pipe and every partial sum meets the float32 accumulator with its own.
// A step needs BM + BN bytes of them beside (BM + BN) * 128 of operands; they travel with the operands (one more load per
// wave into a 256-byte slot of the stage) and are read from LDS as one register for the tiles of a wave's side.
#include "mi8_block_gemm.h"
#include "mi8_gemm_ring.h"
#include "mi8_groups.h"

namespace mi8 {
using namespace gemm;
using namespace block;
namespace {

typedef __attribute__((address_space(1))) const void* block_global_t;
typedef const __attribute__((address_space(3))) uint32_t* block_word_t;

// One tile's product: rows [0, rows) of `a` by rows [0, cols) of `b` over nk blocks of 128.
struct BlockTile {
    const uint8_t* a;
    const uint8_t* b;
    int64_t lda, ldb;
    const uint8_t* ea;  // scales of the 128-row group that holds the tile's first row, first block of K
    const uint8_t* eb;
    int64_t ea_step, eb_step;  // bytes from a block of K to the next
    int a_half, b_half;        // (tiles of 64 rows or columns) which half of their 128
    int rows, cols, nk;
    void* c;
    int64_t ldc;
    int c_f32;
};

constexpr int kBlockThreads = 256;
template <int BM, int BN, int ST>
constexpr int kBlockLdsBytes = ST * ((BM + BN) * BK + 256);

// Tiles of BM x BN (64 x 64, 128 x 64, 64 x 128: two workgroups on a compute unit; one of 128 x 128 with 96 KB of LDS to itself took 1.4 times as long
// as two of 128 x 64), four waves of (BM / 2) x (BN / 2), a ring of ST stages that the operands reach from
// L2 without passing through registers.  Fragments (and the two registers of exponents) of a step are read from LDS during the
// step before, in two sets.
template <int BM, int BN, int ST>
__device__ __forceinline__ void block_tile(const BlockTile& t, uint8_t* lds)
{
    constexpr int WTM = BM / 2, WTN = BN / 2, TM = WTM / 16, TN = WTN / 16;
    constexpr int STAGE = (BM + BN) * BK + 256;
    constexpr int LA = BM / 32, LB = BN / 32, LD = LA + LB + 1;
    static_assert((BM == 64 || BM == 128) && (BN == 64 || BN == 128) && ST >= 3 && LD * (ST - 1) < 64, "tile shape");
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    const int r16 = lane & 15, kb = lane >> 4;

    // ---- loads: load i of a wave fills rows 8 (4 i + wave) .. + 7; rows past the edge re-read the last one
    const __amdgpu_buffer_rsrc_t da = __builtin_amdgcn_make_buffer_rsrc((void*)t.a, 0, (int)(uint32_t)((int64_t)(t.rows - 1) * t.lda + t.nk * BK), 0x00020000);
    const __amdgpu_buffer_rsrc_t db = __builtin_amdgcn_make_buffer_rsrc((void*)t.b, 0, (int)(uint32_t)((int64_t)(t.cols - 1) * t.ldb + t.nk * BK), 0x00020000);
    const int lr = lane >> 3, chunk16 = ((lane & 7) ^ swz16(lr)) * 16;
    int off[LA + LB];
#pragma unroll
    for (int i = 0; i < LA + LB; ++i) {
        const bool is_a = i < LA;
        int r = 8 * (4 * (is_a ? i : i - LA) + wave) + lr;
        const int last = (is_a ? t.rows : t.cols) - 1;
        r = r < last ? r : last;
        off[i] = (int)((uint32_t)r * (uint32_t)(is_a ? t.lda : t.ldb)) + chunk16;
    }
    // words of exponents: BM / 4 of A, BN / 4 of B.  128 rows are 32 consecutive words; a half of 64 rows has every other one,
    // the four bytes of its four MFMA tiles.
    const uint8_t* e_src;
    int64_t e_step;
    {
        int w = lane < (BM + BN) / 4 ? lane : (BM + BN) / 4 - 1;
        const bool is_a = w < BM / 4;
        w = is_a ? w : w - BM / 4;
        const bool small = is_a ? BM == 64 : BN == 64;
        e_src = (is_a ? t.ea : t.eb) + 4 * (small ? 2 * w + (is_a ? t.a_half : t.b_half) : w);
        e_step = is_a ? t.ea_step : t.eb_step;
    }
    const int nk = t.nk;
    auto issue_one = [&](int i, int k, int slot) __attribute__((always_inline)) {
        uint8_t* st = lds + slot * STAGE;
        if (i == LA + LB) {  // (steps are issued in order: the source moves on)
            __builtin_amdgcn_global_load_lds((block_global_t)e_src, (ring_lds_t)(st + (BM + BN) * BK), 4, 0, 0);
            e_src += e_step;
            return;
        }
        const bool is_a = i < LA;
        ring_load(is_a ? da : db, st + ((is_a ? 0 : BM) + 8 * (4 * (is_a ? i : i - LA) + wave)) * BK, off[i], k * BK);
    };
    auto issue = [&](int k, int slot) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < LD; ++i) issue_one(i, k, slot);
    };

    // ---- fragment reads: half q of a lane's 32 K bytes; MFMA tile t adds 2048 t
    uint32_t fa_at[2], fb_at[2], ea_at, eb_at;
    {
        const uint32_t lds0 = (uint32_t)(uintptr_t)(ring_lds_t)lds;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const uint32_t chunk = (uint32_t)((2 * kb + q) ^ swz16(r16)) << 4;
            fa_at[q] = lds0 + (uint32_t)((wm * WTM + r16) * BK) + chunk;
            fb_at[q] = lds0 + (uint32_t)((BM + wn * WTN + r16) * BK) + chunk;
        }
        // a wave of 64 rows: the word of its four tiles; of 32 rows: two of a word's four bytes
        ea_at = lds0 + (BM + BN) * BK + 4 * (BM == 128 ? 2 * r16 + wm : r16);
        eb_at = lds0 + (BM + BN) * BK + BM + 4 * (BN == 128 ? 2 * r16 + wn : r16);
    }
    const int a_shift = BM == 128 ? 0 : 16 * wm, b_shift = BN == 128 ? 0 : 16 * wn;

    ring_v4f acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = (ring_v4f){0, 0, 0, 0};

    struct Set { v4i a[TM][2], b[TN][2]; uint32_t ea, eb; };
    Set set[2];
    constexpr int kMma = TM * TN, kReads = 2 * (TM + TN) + 2;
    auto read_one = [&](Set& s, int x, uint32_t at) __attribute__((always_inline)) {
        if (x == 0) {
            s.ea = *reinterpret_cast<block_word_t>((uintptr_t)(ea_at + at));
        } else if (x == 1) {
            s.eb = *reinterpret_cast<block_word_t>((uintptr_t)(eb_at + at));
        } else {
            const int y = (x - 2) >> 1, q = x & 1;
            if (y < TM)
                s.a[y][q] = *reinterpret_cast<ring_frag_t>((uintptr_t)(fa_at[q] + at + y * 16 * BK));
            else
                s.b[y - TM][q] = *reinterpret_cast<ring_frag_t>((uintptr_t)(fb_at[q] + at + (y - TM) * 16 * BK));
        }
    };
    // D' = B . A^T: the first operand is the B fragment, its exponents come first
#define MI8_BLOCK_MMA(I, J)                                                                                                        \
    case 4 * (I) + (J):                                                                                                            \
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(                                                             \
            __builtin_shufflevector(s.b[j][0], s.b[j][1], 0, 1, 2, 3, 4, 5, 6, 7),                                                \
            __builtin_shufflevector(s.a[i][0], s.a[i][1], 0, 1, 2, 3, 4, 5, 6, 7), acc[i][j], 0, 0, J, (int)eb, I, (int)ea);      \
        break;
    auto mma_one = [&](const Set& s, int x, uint32_t ea, uint32_t eb) __attribute__((always_inline)) {
        const int i = x / TN, j = x % TN;
        switch (4 * i + j) {
            MI8_BLOCK_MMA(0, 0) MI8_BLOCK_MMA(0, 1) MI8_BLOCK_MMA(0, 2) MI8_BLOCK_MMA(0, 3)
            MI8_BLOCK_MMA(1, 0) MI8_BLOCK_MMA(1, 1) MI8_BLOCK_MMA(1, 2) MI8_BLOCK_MMA(1, 3)
            MI8_BLOCK_MMA(2, 0) MI8_BLOCK_MMA(2, 1) MI8_BLOCK_MMA(2, 2) MI8_BLOCK_MMA(2, 3)
            MI8_BLOCK_MMA(3, 0) MI8_BLOCK_MMA(3, 1) MI8_BLOCK_MMA(3, 2) MI8_BLOCK_MMA(3, 3)
        }
    };
#undef MI8_BLOCK_MMA

    int slot = 0;
    auto k_step = [&](int k, auto set_tag, auto steady_tag) __attribute__((always_inline)) {
        constexpr int S = decltype(set_tag)::value;
        constexpr bool kSteady = decltype(steady_tag)::value;
        // this wave's loads of step k + 1 have landed (those of up to ST - 2 later steps may be in flight) and its fragments of
        // step k arrived; after the barrier every wave's, so that slot k may be filled again
        ring_wait_steps<LD, ST - 2>(kSteady ? ST - 2 : nk - 2 - k);
        asm volatile("s_barrier" ::: "memory");
        const uint32_t ea = set[S].ea >> a_shift, eb = set[S].eb >> b_shift;
        auto body = [&](auto with_reads, auto with_loads) __attribute__((always_inline)) {
            uint32_t at = (uint32_t)((slot == ST - 1 ? 0 : slot + 1) * STAGE);
            asm volatile("" : "+v"(at));
#pragma unroll
            for (int x = 0; x < kMma; ++x) {
                mma_one(set[S], x, ea, eb);
                if constexpr (decltype(with_reads)::value) {
#pragma unroll
                    for (int y = x * kReads / kMma; y < (x + 1) * kReads / kMma; ++y) read_one(set[S ^ 1], y, at);
                }
                if constexpr (decltype(with_loads)::value) {
#pragma unroll
                    for (int y = x * LD / kMma; y < (x + 1) * LD / kMma; ++y) issue_one(y, k + ST, slot);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        if constexpr (kSteady) {
            body(std::true_type{}, std::true_type{});
        } else {
            if (k + ST < nk) issue(k + ST, slot);
            asm volatile("" ::: "memory");
            if (k + 1 < nk)
                body(std::true_type{}, std::false_type{});
            else
                body(std::false_type{}, std::false_type{});
        }
        slot = slot == ST - 1 ? 0 : slot + 1;
    };
    if (nk > 0) {
#pragma unroll
        for (int s = 0; s < ST; ++s) {
            if (s < nk) issue(s, s);
            asm volatile("" ::: "memory");  // (the waits count operations: those of a step stay behind the ones of the step before)
            __builtin_amdgcn_sched_barrier(0);
        }
        ring_wait_steps<LD, ST - 1>(nk - 1);
        asm volatile("s_barrier" ::: "memory");
#pragma unroll
        for (int x = 0; x < kReads; ++x) read_one(set[0], x, 0);
    }
    const std::integral_constant<int, 0> set0;
    const std::integral_constant<int, 1> set1;
    int k = 0;
    for (; k + 1 + ST < nk; k += 2) {  // both steps have loads to issue
        k_step(k, set0, std::true_type{});
        k_step(k + 1, set1, std::true_type{});
    }
    for (; k + 1 < nk; k += 2) {
        k_step(k, set0, std::false_type{});
        k_step(k + 1, set1, std::false_type{});
    }
    if (k < nk) k_step(k, set0, std::false_type{});

    // ---- epilogue: acc[i][j][e] of lane l is C[row = 16 i + l % 16][col = 16 j + 4 (l / 16) + e] of the wave tile
    const int row0 = wm * WTM + r16, col0 = wn * WTN + 4 * kb;
    if (t.c_f32) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
                if (row0 + 16 * i < t.rows && col0 + 16 * j < t.cols)
                    *reinterpret_cast<ring_v4f*>(reinterpret_cast<float*>(t.c) + (int64_t)(row0 + 16 * i) * t.ldc + col0 + 16 * j) = acc[i][j];
        return;
    }
    // bf16 rows leave through LDS (the ring is free now): whole row segments of the wave tile, 16 bytes per lane
    constexpr int PITCH = WTN * 2 + 16;  // (the pad spreads the rows of a store over the banks)
    static_assert(4 * WTM * PITCH <= ST * STAGE, "output staging");
    __syncthreads();
    uint8_t* stg = lds + wave * (WTM * PITCH);
    constexpr int LPR = WTN / 8, RPI = 64 / LPR;  // lanes per row, rows per store
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
            *reinterpret_cast<uint2*>(stg + (16 * i + r16) * PITCH + (16 * j + 4 * kb) * 2) =
                make_uint2(pack_bf16x2(acc[i][j][0], acc[i][j][1]), pack_bf16x2(acc[i][j][2], acc[i][j][3]));
#pragma unroll
    for (int it = 0; it < WTM / RPI; ++it) {
        const int rw = it * RPI + lane / LPR, c8 = (lane % LPR) * 8;
        const v4i v = *reinterpret_cast<const v4i*>(stg + rw * PITCH + c8 * 2);
        const int row = wm * WTM + rw, col = wn * WTN + c8;
        if (row < t.rows && col < t.cols) *reinterpret_cast<v4i*>(reinterpret_cast<uint16_t*>(t.c) + (int64_t)row * t.ldc + col) = v;
    }
}

// ---- the problems ------------------------------------------------------------------------------------------------

__device__ __forceinline__ int at_most(int64_t v, int most) { return v < most ? (int)v : most; }

// tile `block` of a dense product whose tiles are dealt to the XCDs an eighth each, contiguous
template <int BM, int BN, int ST>
__device__ __forceinline__ void dense_tile(const BlockArgs& p, const int block, uint8_t* lds)
{
    GemmArgs order;
    order.tiles_m = p.tiles_m;
    order.tiles_n = p.tiles_n;
    const int total = p.tiles_m * p.tiles_n, per_xcd = (total + 7) / 8, index = block % 8 * per_xcd + block / 8;
    if (block / 8 >= per_xcd || index >= total) return;
    int tm, tn;
    tile_coords(order, index, tm, tn);
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
    BlockTile t;
    t.a = p.A + m0 * p.lda;
    t.b = p.B + n0 * p.ldb;
    t.lda = p.lda;
    t.ldb = p.ldb;
    t.ea = p.ea + m0 / 128 * 128;
    t.eb = p.eb + n0 / 128 * 128;
    t.ea_step = padded(p.M);
    t.eb_step = padded(p.N);
    t.a_half = (int)(m0 / 64) & 1;
    t.b_half = (int)(n0 / 64) & 1;
    t.rows = at_most(p.M - m0, BM);
    t.cols = at_most(p.N - n0, BN);
    t.nk = p.nk;
    t.c = reinterpret_cast<uint8_t*>(p.C) + (m0 * p.ldc + n0) * (p.c_f32 ? 4 : 2);
    t.ldc = p.ldc;
    t.c_f32 = p.c_f32;
    block_tile<BM, BN, ST>(t, lds);
}

template <int BM, int BN, int ST>
__global__ __launch_bounds__(kBlockThreads, 2) void block_gemm_kernel(BlockArgs p)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    dense_tile<BM, BN, ST>(p, (int)blockIdx.x, lds);
}

// Several products in one grid, each dealt to the XCDs by itself: of two that fill half of the chip each, one need not wait for the other.  The two
// of a linear's backward, us one by one / together: 100 tokens x 1024 x 1024 7.6 / 5.3, 512 x 1024 x 2816 13.8 / 11.0, 2048 x 2048 x 2048
// 27.1 / 24.2, 300 x 4096 x 4096 26.6 / 26.7.
struct BlockBatch {
    BlockArgs item[MI8_BLOCK_GEMM_BATCH];
    int first[MI8_BLOCK_GEMM_BATCH];  // first workgroup, a multiple of 8
    int count;
};

template <int BM, int BN, int ST>
__global__ __launch_bounds__(kBlockThreads, 2) void block_gemm_batch_kernel(BlockBatch p)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    int i = 0;
#pragma unroll
    for (int j = 1; j < MI8_BLOCK_GEMM_BATCH; ++j)
        if (j < p.count && (int)blockIdx.x >= p.first[j]) i = j;
    dense_tile<BM, BN, ST>(p.item[i], (int)blockIdx.x - p.first[i], lds);
}

// Rows [row, row + BM) of the output, where there are any, become zero in columns [col, col + BN).
template <int BM, int BN>
__device__ __forceinline__ void zero_rows(const BlockArgs& p, int64_t row, int64_t col)
{
    const int bytes = p.c_f32 ? 4 : 2, chunks = BN * bytes / 16;  // (N % 8 == 0: rows are whole chunks)
    for (int i = (int)threadIdx.x; i < BM * chunks; i += kBlockThreads) {
        const int64_t r = row + i / chunks, at = (col * bytes) + i % chunks * 16;
        if (r < p.M && at < (int64_t)p.N * bytes) *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(p.C) + r * p.ldc * bytes + at) = make_uint4(0, 0, 0, 0);
    }
}

// out[rows of e] = A[rows of e] . B_e^T, zero behind the last group
template <int BM, int BN, int ST>
__global__ __launch_bounds__(kBlockThreads, 2) void block_grouped_kernel(BlockArgs p)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int tn = (int)blockIdx.x % p.tiles_n, part = (int)blockIdx.x / p.tiles_n;
    const int unit = part * BM / 128;  // of 128 rows, as the scales are laid out
    const GroupSpan s = locate_group<128, true>(p.sizes, p.E, p.M, unit);
    if (s.e >= p.E) {  // behind the last group: the grid has a part of its own for all of its rows
        const int64_t first = s.rows_before + (unit - s.units_before) * 128 + part * BM % 128;
        zero_rows<BM, BN>(p, first, (int64_t)tn * BN);
        return;
    }
    const int64_t inside = (int64_t)(unit - s.units_before) * 128 + part * BM % 128;  // first row, counted from the group's
    if (inside >= s.m) return;
    const int64_t m0 = s.rows_before + inside, n0 = (int64_t)tn * BN;
    BlockTile t;
    t.a = p.A + m0 * p.lda;
    t.b = p.B + s.e * p.b_group_stride + n0 * p.ldb;
    t.lda = p.lda;
    t.ldb = p.ldb;
    t.ea = p.ea + (int64_t)unit * 128;
    t.eb = p.eb + s.e * p.eb_group_stride + n0 / 128 * 128;
    t.ea_step = p.axis;
    t.eb_step = padded(p.N);
    t.a_half = part * BM / 64 & 1;
    t.b_half = (int)(n0 / 64) & 1;
    t.rows = at_most(s.m - inside, BM);
    t.cols = at_most(p.N - n0, BN);
    t.nk = p.nk;
    t.c = reinterpret_cast<uint8_t*>(p.C) + (m0 * p.ldc + n0) * (p.c_f32 ? 4 : 2);
    t.ldc = p.ldc;
    t.c_f32 = p.c_f32;
    block_tile<BM, BN, ST>(t, lds);
}

// out[e] [M, N] = A[:, blocks of e] . B[:, blocks of e]^T; a group without tokens gives zeros
template <int BM, int BN, int ST>
__global__ __launch_bounds__(kBlockThreads, 2) void block_grouped_wgrad_kernel(BlockArgs p)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int per_group = p.tiles_m * p.tiles_n;
    const int e = (int)blockIdx.x / per_group, rest = (int)blockIdx.x % per_group;
    const int64_t m0 = (int64_t)(rest / p.tiles_n) * BM, n0 = (int64_t)(rest % p.tiles_n) * BN;
    const GroupSpan s = locate_group<128, false>(p.sizes, p.E, p.tokens, e);
    const int64_t first = s.units_before;  // block of K
    BlockTile t;
    t.a = p.A + m0 * p.lda + first * 128;
    t.b = p.B + n0 * p.ldb + first * 128;
    t.lda = p.lda;
    t.ldb = p.ldb;
    t.ea_step = padded(p.M);
    t.eb_step = padded(p.N);
    t.ea = p.ea + first * t.ea_step + m0 / 128 * 128;
    t.eb = p.eb + first * t.eb_step + n0 / 128 * 128;
    t.a_half = (int)(m0 / 64) & 1;
    t.b_half = (int)(n0 / 64) & 1;
    t.rows = at_most(p.M - m0, BM);
    t.cols = at_most(p.N - n0, BN);
    t.nk = (int)((s.m + 127) / 128);
    t.c = reinterpret_cast<uint8_t*>(p.C) + ((e * (int64_t)p.M + m0) * p.ldc + n0) * (p.c_f32 ? 4 : 2);
    t.ldc = p.ldc;
    t.c_f32 = p.c_f32;
    block_tile<BM, BN, ST>(t, lds);
}

template <int BM, int BN, int ST>
int launch_dense(BlockArgs& p, hipStream_t st)
{
    auto kern = block_gemm_kernel<BM, BN, ST>;
    static std::atomic<uint64_t> configured{0};
    if (int rc = reserve_dynamic_lds(reinterpret_cast<const void*>(kern), kBlockLdsBytes<BM, BN, ST>, configured, "mi8_gemm_fp8_block")) return rc;
    p.tiles_m = (int)ceil_div(p.M, BM);
    p.tiles_n = (int)ceil_div(p.N, BN);
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
    MI8_REQUIRE(tiles < ((int64_t)1 << 30), MI8_ERR_UNSUPPORTED, "mi8_gemm_fp8_block: grid too large");
    hipLaunchKernelGGL(kern, dim3((unsigned)round_up(tiles, 8)), dim3(kBlockThreads), (kBlockLdsBytes<BM, BN, ST>), st, p);
    return launch_status("mi8_gemm_fp8_block");
}

template <int BM, int BN, int ST>
int launch_batch(BlockBatch& p, hipStream_t st)
{
    auto kern = block_gemm_batch_kernel<BM, BN, ST>;
    static std::atomic<uint64_t> configured{0};
    if (int rc = reserve_dynamic_lds(reinterpret_cast<const void*>(kern), kBlockLdsBytes<BM, BN, ST>, configured, "mi8_gemm_fp8_block_batch")) return rc;
    int64_t blocks = 0;
    for (int i = 0; i < p.count; ++i) {
        BlockArgs& t = p.item[i];
        t.tiles_m = (int)ceil_div(t.M, BM);
        t.tiles_n = (int)ceil_div(t.N, BN);
        p.first[i] = (int)blocks;
        blocks += round_up((int64_t)t.tiles_m * t.tiles_n, 8);
        MI8_REQUIRE(blocks < ((int64_t)1 << 30), MI8_ERR_UNSUPPORTED, "mi8_gemm_fp8_block_batch: grid too large");
    }
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(kBlockThreads), (kBlockLdsBytes<BM, BN, ST>), st, p);
    return launch_status("mi8_gemm_fp8_block_batch");
}

template <int BM, int BN, int ST>
int launch_grouped(BlockArgs& p, hipStream_t st)
{
    auto kern = block_grouped_kernel<BM, BN, ST>;
    static std::atomic<uint64_t> configured{0};
    if (int rc = reserve_dynamic_lds(reinterpret_cast<const void*>(kern), kBlockLdsBytes<BM, BN, ST>, configured, "mi8_grouped_gemm_fp8_block")) return rc;
    p.tiles_n = (int)ceil_div(p.N, BN);
    // (128-row units of the groups, at most axis / 128 together with those of the rows behind them but for a part of one)
    const int64_t blocks = (p.axis / 128 + 1) * (128 / BM) * p.tiles_n;
    MI8_REQUIRE(blocks < ((int64_t)1 << 31), MI8_ERR_UNSUPPORTED, "mi8_grouped_gemm_fp8_block: grid too large");
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(kBlockThreads), (kBlockLdsBytes<BM, BN, ST>), st, p);
    return launch_status("mi8_grouped_gemm_fp8_block");
}

template <int BM, int BN, int ST>
int launch_wgrad(BlockArgs& p, hipStream_t st)
{
    auto kern = block_grouped_wgrad_kernel<BM, BN, ST>;
    static std::atomic<uint64_t> configured{0};
    if (int rc = reserve_dynamic_lds(reinterpret_cast<const void*>(kern), kBlockLdsBytes<BM, BN, ST>, configured, "mi8_grouped_wgrad_fp8_block")) return rc;
    p.tiles_m = (int)ceil_div(p.M, BM);
    p.tiles_n = (int)ceil_div(p.N, BN);
    const int64_t blocks = (int64_t)p.E * p.tiles_m * p.tiles_n;
    MI8_REQUIRE(blocks < ((int64_t)1 << 31), MI8_ERR_UNSUPPORTED, "mi8_grouped_wgrad_fp8_block: grid too large");
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(kBlockThreads), (kBlockLdsBytes<BM, BN, ST>), st, p);
    return launch_status("mi8_grouped_wgrad_fp8_block");
}

// (row offsets inside a tile of 256 rows are 32 bits)
bool persistent_fits(const BlockArgs& p) { return !p.c_f32 && p.lda < (1 << 23) && p.ldb < (1 << 23) && p.ldc < (1 << 22); }

// ---- which kernel a product runs on -----------------------------------------------------------------------------------
// By estimated time, with the constants of the kernels without block scales (mi8_gemm.hip), which these meet within 10 %.  us, tiles of 64 x 64 /
// 128 x 64 / 64 x 128 / 256 x 256: 64 x 4096 x 4096 9.2 / 11.1 / 11.0 / 38.6, 1537 x 2048 x 2048 16.2 / 12.6 / 12.1 / 22.7,
// 777 x 11008 x 4096 64 / 50 / 51 / 43, 777 x 4096 x 11008 69 / 54 / 54 / 92, 2048 x 8192 x 2048 65 / 45 / 45 / 32,
// 4096 x 4096 x 4096 109 / 85 / 81 / 52, 6000 x 768 x 2048 21 / 18 / 18 / 23, 16384 x 1024 x 1024 35 / 25 / 25 / 20.

enum BlockKernel { kBlock64, kBlock128x64, kBlock64x128, kBlock256, kNumBlockKernels };

struct TileCost {
    int bm, bn;
    double step0, step1, step2, tile;  // us a step with one tile on a compute unit: few of them busy .. all; with two; us a tile besides
    double many, many_tile;            // where units get three tiles and more
};
constexpr TileCost kTileCosts[] = {{64, 64, 0.113, 0.181, 0.335, 1.33, 0.39, 1.2}, {128, 64, 0.169, 0.294, 0.524, 1.67, 0.64, 1.2}, {64, 128, 0.171, 0.295, 0.533, 1.72, 0.64, 1.2}};

// `tiles` tiles of `steps` blocks each
double ring_time(const TileCost& r, double tiles, double steps)
{
    const double per_cu = __builtin_ceil(tiles / 256), busy = tiles / 256 < 1 ? tiles / 256 : 1;
    if (per_cu > 2) return 2.6 + 0.5 * per_cu * (steps * r.many + r.many_tile);
    return 2.6 + (per_cu > 1 ? steps * r.step2 : steps * (r.step0 + (r.step1 - r.step0) * busy)) + r.tile;
}

double persistent_time(double tiles, double steps)
{
    const double rounds = __builtin_floor(tiles / 256), left = tiles - 256 * rounds, crowd = (2 * left - 256) / 256;
    return 3.0 + rounds * (1.35 * steps + 5) + (left > 0 ? steps * (1 + 0.35 * (crowd > 0 ? crowd : 0)) + 5 : 0);
}

// tiles(bm, bn): how many there are
template <typename Tiles>
BlockKernel choose_kernel(Tiles tiles, double steps, bool persistent)
{
    int best = kBlock64;
    double time = ring_time(kTileCosts[0], tiles(64, 64), steps);
    for (int k = kBlock128x64; k <= kBlock64x128; ++k) {
        const double t = ring_time(kTileCosts[k], tiles(kTileCosts[k].bm, kTileCosts[k].bn), steps);
        if (t < time) {
            best = k;
            time = t;
        }
    }
    if (persistent && persistent_time(tiles(256, 256), steps) < time) best = kBlock256;
    return (BlockKernel)best;
}

// (the sizes are on the device: with popularity as skewed as routers make it about half of the groups add a tile that is partly empty)
BlockKernel choose_grouped(int64_t T, int64_t N, int64_t steps, int32_t num_groups, bool persistent)
{
    const double partial = 0.5 * (double)(num_groups < T ? num_groups : T);
    return choose_kernel([&](int bm, int bn) { return ((double)T / bm + partial) * (double)ceil_div(N, bn); }, (double)steps, persistent);
}

BlockKernel choose_wgrad(int64_t T, int64_t N, int64_t Kl, int32_t num_groups, bool persistent)
{
    return choose_kernel([&](int bm, int bn) { return (double)num_groups * (double)(ceil_div(N, bm) * ceil_div(Kl, bn)); }, (double)T / 128 / num_groups + 0.5,
                         persistent);
}

int check_operands(const BlockArgs& p, int64_t K, int64_t M, int64_t N, int out_dtype, const char* what)
{
    MI8_REQUIRE(p.A && p.B && p.ea && p.eb && p.C, MI8_ERR_ARG, "%s: null pointer", what);
    MI8_REQUIRE(out_dtype == MI8_BF16 || out_dtype == MI8_F32, MI8_ERR_ARG, "%s: output must be bf16 or float32", what);
    MI8_REQUIRE(M > 0 && N > 0 && K > 0, MI8_ERR_ARG, "%s: empty problem", what);
    MI8_REQUIRE(M < (1 << 30) && N < (1 << 30) && K < (1 << 30), MI8_ERR_UNSUPPORTED, "%s: problem too large", what);
    MI8_REQUIRE(p.lda % 16 == 0 && p.ldb % 16 == 0 && p.lda >= block::padded(K) && p.ldb >= block::padded(K) && p.lda < (1 << 24) && p.ldb < (1 << 24),
                MI8_ERR_UNSUPPORTED, "%s: operand rows must be round_up(K, 128) bytes or more, a multiple of 16, below 2^24", what);
    MI8_REQUIRE(N % 8 == 0 && p.ldc % 8 == 0 && p.ldc >= N, MI8_ERR_UNSUPPORTED, "%s: N and the output's row pitch must be multiples of 8", what);
    MI8_REQUIRE(aligned16(p.A) && aligned16(p.B) && aligned16(p.ea) && aligned16(p.eb) && aligned16(p.C), MI8_ERR_UNSUPPORTED,
                "%s: operands, scales and output must be 16-byte aligned", what);
    return MI8_OK;
}

}  // namespace
}  // namespace mi8

using namespace mi8;

extern "C" int mi8_gemm_fp8_block(const void* a, int64_t lda, const void* a_scales, const void* b, int64_t ldb, const void* b_scales, int64_t M,
                                  int64_t N, int64_t K, void* out, int out_dtype, int64_t ldc, int variant, void* stream)
{
    BlockArgs p{(const uint8_t*)a, (const uint8_t*)b, (const uint8_t*)a_scales, (const uint8_t*)b_scales, out, lda, ldb, ldc, (int)M, (int)N,
                (int)ceil_div(K, 128), out_dtype == MI8_F32, 0, 0, nullptr, 0, 0, 0, 0, 0};
    if (int rc = check_operands(p, K, M, N, out_dtype, "mi8_gemm_fp8_block")) return rc;
    hipStream_t st = (hipStream_t)stream;
    MI8_REQUIRE(variant >= -1 && variant < kNumBlockKernels && (variant != kBlock256 || persistent_fits(p)), MI8_ERR_UNSUPPORTED,
                "mi8_gemm_fp8_block: no variant %d, or not for this problem", variant);
    const auto tiles = [&](int bm, int bn) { return (double)(ceil_div(M, bm) * ceil_div(N, bn)); };
    const int k = variant >= 0 ? variant : choose_kernel(tiles, p.nk, persistent_fits(p));
    return k == kBlock256 ? launch_persistent(p, st) : k == kBlock128x64 ? launch_dense<128, 64, 3>(p, st)
           : k == kBlock64x128 ? launch_dense<64, 128, 3>(p, st) : launch_dense<64, 64, 4>(p, st);
}

extern "C" int mi8_gemm_fp8_block_batch(const mi8_block_product* items, int32_t count, void* stream)
{
    MI8_REQUIRE(items && count > 0 && count <= MI8_BLOCK_GEMM_BATCH, MI8_ERR_ARG, "mi8_gemm_fp8_block_batch: 1 to %d products", MI8_BLOCK_GEMM_BATCH);
    BlockBatch p{};
    p.count = count;
    bool together = true;
    double steps = 0, weight = 0;
    for (int i = 0; i < count; ++i) {
        const mi8_block_product& t = items[i];
        p.item[i] = BlockArgs{(const uint8_t*)t.a, (const uint8_t*)t.b, (const uint8_t*)t.a_scales, (const uint8_t*)t.b_scales, t.out, t.lda, t.ldb, t.ldc, (int)t.M,
                              (int)t.N, (int)ceil_div(t.K, 128), t.out_dtype == MI8_F32, 0, 0, nullptr, 0, 0, 0, 0, 0};
        if (int rc = check_operands(p.item[i], t.K, t.M, t.N, t.out_dtype, "mi8_gemm_fp8_block_batch")) return rc;
        const auto tiles = [&](int bm, int bn) { return (double)(ceil_div(t.M, bm) * ceil_div(t.N, bn)); };
        together = together && choose_kernel(tiles, p.item[i].nk, persistent_fits(p.item[i])) != kBlock256;
        steps += tiles(64, 64) * p.item[i].nk;
        weight += tiles(64, 64);
    }
    if (!together || count == 1) {  // (one of them is large: each on its own kernel)
        for (int i = 0; i < count; ++i) {
            const mi8_block_product& t = items[i];
            if (int rc = mi8_gemm_fp8_block(t.a, t.lda, t.a_scales, t.b, t.ldb, t.b_scales, t.M, t.N, t.K, t.out, t.out_dtype, t.ldc, -1, stream)) return rc;
        }
        return MI8_OK;
    }
    const auto all_tiles = [&](int bm, int bn) {
        double n = 0;
        for (int i = 0; i < count; ++i) n += (double)(ceil_div(items[i].M, bm) * ceil_div(items[i].N, bn));
        return n;
    };
    hipStream_t st = (hipStream_t)stream;
    const BlockKernel k = choose_kernel(all_tiles, steps / weight, false);
    return k == kBlock128x64 ? launch_batch<128, 64, 3>(p, st) : k == kBlock64x128 ? launch_batch<64, 128, 3>(p, st) : launch_batch<64, 64, 4>(p, st);
}

extern "C" int mi8_grouped_gemm_fp8_block(const void* a, int64_t lda, const void* a_scales, const void* b, int64_t ldb, int64_t b_group_stride,
                                          const void* b_scales, const int64_t* group_sizes, int32_t num_groups, int64_t T, int64_t N, int64_t K,
                                          void* out, int out_dtype, int64_t ldc, void* stream)
{
    MI8_REQUIRE(group_sizes && num_groups > 0, MI8_ERR_ARG, "mi8_grouped_gemm_fp8_block: no groups");
    BlockArgs p{(const uint8_t*)a, (const uint8_t*)b, (const uint8_t*)a_scales, (const uint8_t*)b_scales, out, lda, ldb, ldc, (int)T, (int)N,
                (int)ceil_div(K, 128), out_dtype == MI8_F32, 0, 0, group_sizes, num_groups, b_group_stride, mi8_block_scale_bytes(N, K),
                T > 0 ? mi8_grouped_padded_rows(T, num_groups) : 0, T};
    if (int rc = check_operands(p, K, T, N, out_dtype, "mi8_grouped_gemm_fp8_block")) return rc;
    MI8_REQUIRE(b_group_stride % 16 == 0, MI8_ERR_UNSUPPORTED, "mi8_grouped_gemm_fp8_block: the group stride must be a multiple of 16");
    hipStream_t st = (hipStream_t)stream;
    const BlockKernel k = choose_grouped(T, N, p.nk, num_groups, persistent_fits(p));
    return k == kBlock256 ? launch_persistent_grouped(p, st) : k == kBlock128x64 ? launch_grouped<128, 64, 3>(p, st)
           : k == kBlock64x128 ? launch_grouped<64, 128, 3>(p, st) : launch_grouped<64, 64, 4>(p, st);
}

extern "C" int mi8_grouped_wgrad_fp8_block(const void* a_t, const void* a_scales, const void* b_t, const void* b_scales, int64_t ld_t,
                                           const int64_t* group_sizes, int32_t num_groups, int64_t T, int64_t N, int64_t Kl, void* out,
                                           int out_dtype, void* stream)
{
    MI8_REQUIRE(group_sizes && num_groups > 0, MI8_ERR_ARG, "mi8_grouped_wgrad_fp8_block: no groups");
    MI8_REQUIRE(T > 0, MI8_ERR_ARG, "mi8_grouped_wgrad_fp8_block: empty problem");
    const int64_t axis = mi8_grouped_padded_rows(T, num_groups);
    BlockArgs p{(const uint8_t*)a_t, (const uint8_t*)b_t, (const uint8_t*)a_scales, (const uint8_t*)b_scales, out, ld_t, ld_t, Kl, (int)N, (int)Kl, 0,
                out_dtype == MI8_F32, 0, 0, group_sizes, num_groups, 0, 0, axis, T};
    if (int rc = check_operands(p, axis, N, Kl, out_dtype, "mi8_grouped_wgrad_fp8_block")) return rc;
    hipStream_t st = (hipStream_t)stream;
    const BlockKernel k = choose_wgrad(T, N, Kl, num_groups, persistent_fits(p));
    return k == kBlock256 ? launch_persistent_wgrad(p, st) : k == kBlock128x64 ? launch_wgrad<128, 64, 3>(p, st)
           : k == kBlock64x128 ? launch_wgrad<64, 128, 3>(p, st) : launch_wgrad<64, 64, 4>(p, st);
}

extern "C" int32_t mi8_grouped_gemm_fp8_block_variant(int64_t T, int64_t N, int64_t K, int32_t num_groups, int out_dtype)
{
    if (T <= 0 || N <= 0 || K <= 0 || num_groups <= 0) return -1;
    BlockArgs p{};
    p.lda = p.ldb = block::padded(K);
    p.ldc = N;
    p.c_f32 = out_dtype == MI8_F32;
    return choose_grouped(T, N, ceil_div(K, 128), num_groups, persistent_fits(p));
}

extern "C" int32_t mi8_grouped_wgrad_fp8_block_variant(int64_t T, int64_t N, int64_t Kl, int32_t num_groups, int out_dtype)
{
    if (T <= 0 || N <= 0 || Kl <= 0 || num_groups <= 0) return -1;
    BlockArgs p{};
    p.lda = p.ldb = mi8_grouped_padded_rows(T, num_groups);
    p.ldc = Kl;
    p.c_f32 = out_dtype == MI8_F32;
    return choose_wgrad(T, N, Kl, num_groups, persistent_fits(p));
}
