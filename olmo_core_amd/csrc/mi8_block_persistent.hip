// Persistent product of operands with block scales: 256 x 256 tiles of one workgroup, four waves of 128 x 128 on 16x16x128 MFMAs,
// operands from global memory straight to LDS two steps ahead, one 128-byte step per block of scales.
//
// The loop is that of the persistent kernel without block scales (mi8_gemm_m16.hip), which feeds the matrix pipe at the rate the
// chip's power allows: per step 64 MFMAs a wave in two phases of 32, A fragments of tiles 4-7 read during the first, all of the next
// step's B fragments and A tiles 0-3 during the second, eight direct loads a phase.  What the scales add to a step: one more direct
// load of a wave (256 bytes: every other wave those of A's or of B's 256 rows), two 8-byte reads of LDS, and four registers in two
// sets (a step's and the next one's).  The bytes lie so that a lane's eight are those of its row in the wave's eight tiles.
//
// Tiles start at multiples of 128 rows, where the scales do; rows past the edge re-read the last one and are not stored.
#include <type_traits>

#include "mi8_block_gemm.h"
#include "mi8_gemm_tiles.h"

namespace mi8 {
using namespace gemm;
namespace block {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(1))) const void* gptr_t;
typedef __attribute__((address_space(3))) void* lptr_t;
typedef const __attribute__((address_space(3))) v4i* lfrag_t;
typedef const __attribute__((address_space(3))) v2i* lscale_t;

constexpr int kStage = (BM + BN) * BK;  // 64 KB
constexpr int kStaging = 4 * 4096;      // output staging of the waves
constexpr int kScaleSlot = BM + BN;     // a step's scales
constexpr int kLdsBytes = 2 * kStage + kStaging + 2 * kScaleSlot;
constexpr int kThreads = 256;
constexpr int WT = 128, NT = WT / 16;   // wave tile, MFMA tiles along its edge
constexpr int kLoads = 8;               // direct loads per operand, step and wave (8 rows each)

// write-through, streaming: a tile's 128 KB are read by a later kernel, and left in the L2 would displace the operands
constexpr int kOutStoreAux = 1 | 2 | 16;  // sc0, nt, sc1

constexpr int vmcnt(int n) { return (n & 15) | ((n >> 4) << 14) | 0x0F70; }

struct Tile {
    const uint8_t* a;
    const uint8_t* b;
    const uint8_t* ea;
    const uint8_t* eb;
    int nk;
    int rows, cols;  // of the 256 x 256 that exist
    int a_rows;      // rows of A that may be read
    uint16_t* c;     // null: no tile
};

// The kernel's argument (a problem, which starts with its BlockArgs) as it is in memory.  What describes the next tile is read again for every
// tile: held in scalar registers it is spilled into lanes of vector registers, and read back from them in every step of the K loop, where the one
// wave of a SIMD has 32 cycles between two MFMAs (64 equal groups, 131072 x 1024 x 2048: 30 such reads a step, 259 us; 22 and 250 this way).
typedef const __attribute__((address_space(4))) BlockArgs* args_t;
__device__ __forceinline__ args_t args_in_memory()
{
    args_t p = (args_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return p;
}

// ---- problems: how a tile index maps to operands ---------------------------------------------------------------------

struct Dense {
    BlockArgs p;
    static constexpr bool kXcdRanges = true;
    typedef NoCache Cache;
    __device__ __forceinline__ Cache prepare() const { return Cache{}; }
    __device__ __forceinline__ int total_tiles(const Cache&) const { return p.tiles_m * p.tiles_n; }
    __device__ __forceinline__ int64_t ea_step() const { return padded(p.M); }
    __device__ __forceinline__ int64_t eb_step() const { return padded(p.N); }
    __device__ __forceinline__ Tile tile(int t, const Cache&) const
    {
        const args_t p = args_in_memory();
        GemmArgs order;
        order.tiles_m = p->tiles_m;
        order.tiles_n = p->tiles_n;
        int tm, tn;
        tile_coords(order, t, tm, tn);
        const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
        Tile d;
        d.a = p->A + m0 * p->lda;
        d.b = p->B + n0 * p->ldb;
        d.ea = p->ea + m0;
        d.eb = p->eb + n0;
        d.nk = p->nk;
        d.rows = p->M - m0 < BM ? (int)(p->M - m0) : BM;
        d.cols = p->N - n0 < BN ? (int)(p->N - n0) : BN;
        d.a_rows = d.rows;
        d.c = reinterpret_cast<uint16_t*>(p->C) + m0 * p->ldc + n0;
        return d;
    }
};

// Rows of A in groups: a tile covers up to 256 rows of one group.  Tiles behind the groups' clear the rows behind the last one.
struct Grouped {
    BlockArgs p;
    static constexpr bool kXcdRanges = true;
    struct Cache {
        GroupCache rows256, rows128;
        int units, used;  // 256-row tiles of the groups, rows of the groups
    };
    __device__ __forceinline__ Cache prepare() const
    {
        Cache c{build_group_cache<256>(p.sizes, p.E, p.M), build_group_cache<128>(p.sizes, p.E, p.M), 0, 0};
        const GroupSpan end = locate_group_cached<256, true>(c.rows256, p.sizes, p.E, p.M, (int64_t)1 << 60);
        c.units = (int)end.units_before;
        if (c.rows256.valid) {
            const int last = p.E - 1;
            c.used = __builtin_amdgcn_readlane(c.rows256.start, last) + __builtin_amdgcn_readlane(c.rows256.m, last);
        } else {
            c.used = (int)end.rows_before;
        }
        return c;
    }
    __device__ __forceinline__ int total_tiles(const Cache& c) const { return (c.units + (p.M - c.used + 255) / 256) * p.tiles_n; }
    __device__ __forceinline__ int64_t ea_step() const { return p.axis; }
    __device__ __forceinline__ int64_t eb_step() const { return padded(p.N); }
    __device__ __forceinline__ Tile tile(int t, const Cache& c) const
    {
        const args_t p = args_in_memory();
        const int mt = t / p->tiles_n;
        const int64_t n0 = (int64_t)(t % p->tiles_n) * BN;
        Tile d;
        d.cols = p->N - n0 < BN ? (int)(p->N - n0) : BN;
        if (mt >= c.units) {
            const int64_t m0 = c.used + (int64_t)(mt - c.units) * BM;
            d.a = d.b = d.ea = d.eb = nullptr;
            d.nk = 0;
            d.a_rows = 0;
            d.rows = p->M - m0 < BM ? (int)(p->M - m0) : BM;
            d.c = reinterpret_cast<uint16_t*>(p->C) + m0 * p->ldc + n0;
            return d;
        }
        const GroupSpan s = locate_group_cached<256, true>(c.rows256, p->sizes, p->E, p->M, mt);
        const int64_t unit128 = locate_group_cached<128, false>(c.rows128, p->sizes, p->E, p->M, s.e).units_before;
        const int64_t inside = (mt - s.units_before) * BM, m0 = s.rows_before + inside;
        d.a = p->A + m0 * p->lda;
        d.b = p->B + s.e * p->b_group_stride + n0 * p->ldb;
        d.ea = p->ea + unit128 * 128 + inside;
        d.eb = p->eb + s.e * p->eb_group_stride + n0;
        d.nk = p->nk;
        d.rows = s.m - inside < BM ? (int)(s.m - inside) : BM;
        d.a_rows = p->M - m0 < BM ? (int)(p->M - m0) : BM;
        d.c = reinterpret_cast<uint16_t*>(p->C) + m0 * p->ldc + n0;
        return d;
    }
};

// Blocks of K in groups: out[e] = A[:, blocks of e] . B[:, blocks of e]^T.  Tile order and balance as for the weight gradients without block
// scales (mi8_gemm_tiles.h): the tiles of a group, which share its operands, go to one XCD, the groups to the XCDs by size.
struct GroupedK {
    BlockArgs p;
    static constexpr bool kXcdRanges = false;
    typedef WgradCache Cache;
    __device__ __forceinline__ Cache prepare() const
    {
        GroupedWgradProblem order{};
        order.sizes = p.sizes;
        order.E = p.E;
        order.T = p.tokens;
        return order.prepare();
    }
    __host__ __device__ __forceinline__ int grid_tiles() const { return GroupedWgradProblem::grid_tiles(p.E, p.tiles_m * p.tiles_n); }
    __device__ __forceinline__ int total_tiles(const Cache&) const { return grid_tiles(); }
    __device__ __forceinline__ int64_t ea_step() const { return padded(p.M); }
    __device__ __forceinline__ int64_t eb_step() const { return padded(p.N); }
    __device__ __forceinline__ Tile tile(int t, const Cache& c) const
    {
        const args_t p = args_in_memory();
        const int per_group = p->tiles_m * p->tiles_n;
        const int xcd = t & 7, slot = t >> 3;
        const int k = slot / per_group, rest = slot % per_group;
        const int rank = (k & 1) ? 8 * k + 7 - xcd : 8 * k + xcd;
        Tile d{};
        if (rank >= p->E) return d;
        const int e = c.g.valid ? __builtin_amdgcn_readlane(c.group_at_rank, rank) : rank;
        const GroupSpan s = locate_group_cached<128, false>(c.g, p->sizes, p->E, p->tokens, e);
        const int64_t m0 = (int64_t)(rest / p->tiles_n) * BM, n0 = (int64_t)(rest % p->tiles_n) * BN, first = s.units_before;
        d.a = p->A + m0 * p->lda + first * 128;
        d.b = p->B + n0 * p->ldb + first * 128;
        d.ea = p->ea + first * padded(p->M) + m0;
        d.eb = p->eb + first * padded(p->N) + n0;
        d.nk = (int)((s.m + 127) / 128);
        d.a_rows = d.rows = p->M - m0 < BM ? (int)(p->M - m0) : BM;
        d.cols = p->N - n0 < BN ? (int)(p->N - n0) : BN;
        d.c = reinterpret_cast<uint16_t*>(p->C) + (e * (int64_t)p->M + m0) * p->ldc + n0;
        return d;
    }
};

// ---- the kernel ------------------------------------------------------------------------------------------------------

template <typename Problem>
__global__ __launch_bounds__(kThreads, 1) void block_persistent_kernel(Problem pb)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    const int r16 = lane & 15, kb = lane >> 4;
    const BlockArgs& p = pb.p;

    // ---- this workgroup's tiles: a contiguous range of the order for each XCD, or strided over the grid
    const typename Problem::Cache cache = pb.prepare();
    const int total = pb.total_tiles(cache), block = (int)blockIdx.x, blocks = (int)gridDim.x;
    int first_tile = block, tile_stride = blocks, last_tile = total;
    if constexpr (Problem::kXcdRanges) {
        const int per_xcd = (total + 7) / 8, xcd = block & 7;
        first_tile = xcd * per_xcd + (block >> 3);
        tile_stride = (blocks + 7 - xcd) >> 3;
        last_tile = xcd * per_xcd + per_xcd < total ? xcd * per_xcd + per_xcd : total;
    }
    const int my_tiles = first_tile < last_tile ? (last_tile - first_tile + tile_stride - 1) / tile_stride : 0;
    if (my_tiles == 0) return;
    auto my_tile = [&](int i) __attribute__((always_inline)) { return pb.tile(first_tile + i * tile_stride, cache); };

    // ---- fragment and scale reads of the stage being read (half q of the lane's 32 bytes of K); tile t adds 2048 t
    uint32_t ra[2], rb[2], rea, reb;
    {
        const uint32_t lds0 = (uint32_t)(uintptr_t)(lptr_t)lds;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const uint32_t chunk = (uint32_t)((2 * kb + q) ^ swz16(r16));
            ra[q] = lds0 + (uint32_t)((wm * WT + r16) * BK) + (chunk << 4);
            rb[q] = lds0 + (uint32_t)(BM * BK + (wn * WT + r16) * BK) + (chunk << 4);
        }
        rea = lds0 + 2 * kStage + kStaging + wm * 128 + 8 * r16;
        reb = lds0 + 2 * kStage + kStaging + BM + wn * 128 + 8 * r16;
    }
    auto flip_read_stage = [&](int to_stage) __attribute__((always_inline)) {
        const uint32_t delta = to_stage ? (uint32_t)kStage : (uint32_t)(-kStage);
        const uint32_t escale = to_stage ? (uint32_t)kScaleSlot : (uint32_t)(-kScaleSlot);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            ra[q] += delta;
            rb[q] += delta;
        }
        rea += escale;
        reb += escale;
    };
    auto read_a = [&](v4i (&f)[2], int tile, int q) __attribute__((always_inline)) {
        f[q] = *reinterpret_cast<lfrag_t>((uintptr_t)(ra[q] + tile * 16 * BK));
    };
    auto read_b = [&](v4i (&f)[2], int tile, int q) __attribute__((always_inline)) {
        f[q] = *reinterpret_cast<lfrag_t>((uintptr_t)(rb[q] + tile * 16 * BK));
    };

    // ---- load cursor: the step that is fetched next, two ahead of the one computed; past the last tile it repeats valid data
    int ld_tile = -1, ld_kt = 0, ld_nk = 0;
    const uint8_t *ld_a = nullptr, *ld_b = nullptr, *ld_ea = nullptr, *ld_eb = nullptr;
    uint32_t last_a = 0, last_b = 0;  // byte offset of the last row that exists
    int words_a = 0, words_b = 0;     // scales of the rows that exist, in words, less one
    auto next_load_tile = [&]() __attribute__((always_inline)) {
        while (ld_tile + 1 < my_tiles) {
            ++ld_tile;
            const Tile d = my_tile(ld_tile);
            if (d.nk > 0 && d.c != nullptr) {
                ld_a = d.a;
                ld_b = d.b;
                ld_ea = d.ea;
                ld_eb = d.eb;
                ld_nk = d.nk;
                ld_kt = 0;
                last_a = (uint32_t)(d.a_rows - 1) * (uint32_t)p.lda;
                last_b = (uint32_t)(d.cols - 1) * (uint32_t)p.ldb;
                words_a = d.rows > 128 ? 63 : 31;
                words_b = d.cols > 128 ? 63 : 31;
                return;
            }
        }
        if (ld_a) {  // no further tile with work: back to the start of the current one
            ld_a -= (int64_t)ld_kt * BK;
            ld_b -= (int64_t)ld_kt * BK;
            ld_ea -= ld_kt * pb.ea_step();
            ld_eb -= ld_kt * pb.eb_step();
            ld_kt = 0;
        }
    };
    auto advance_load_cursor = [&]() __attribute__((always_inline)) {
        ++ld_kt;
        ld_a += BK;
        ld_b += BK;
        ld_ea += pb.ea_step();
        ld_eb += pb.eb_step();
        if (ld_kt >= ld_nk) next_load_tile();
    };
    next_load_tile();

    // wave w fills rows [64 w + 8 x, +8) of an operand, x = 0..7; lane -> row 64 w + 8 x + lane / 8, position lane % 8, which holds
    // global chunk (lane % 8) ^ swz16(row)
    const int lr = lane >> 3;
    const uint32_t row_a = (uint32_t)(lr * (int)p.lda), row_b = (uint32_t)(lr * (int)p.ldb);
    const uint32_t chunk_of[2] = {(uint32_t)((lane & 7) ^ swz16(lr)) << 4, (uint32_t)((lane & 7) ^ swz16(8 + lr)) << 4};
    auto dma_one = [&](int stage, bool is_a, int x) __attribute__((always_inline)) {
        const int row = wave * 64 + 8 * x;
        uint32_t rows = (uint32_t)row * (uint32_t)(is_a ? p.lda : p.ldb);
        asm volatile("" : "+s"(rows));  // opaque: the sum stays one add at the load instead of sixteen resident registers
        uint32_t o = (is_a ? row_a : row_b) + rows;
        const uint32_t last = is_a ? last_a : last_b;
        o = (o < last ? o : last) + chunk_of[x & 1];
        __builtin_amdgcn_global_load_lds((gptr_t)((is_a ? ld_a : ld_b) + o), (lptr_t)(lds + stage * kStage + (is_a ? 0 : BM * BK) + row * BK), 16, 0, 0);
    };
    auto dma_scales = [&](int stage) __attribute__((always_inline)) {  // even waves: A's, odd waves: B's
        const int words = wn ? words_b : words_a;
        const int w = lane < words ? lane : words;
        __builtin_amdgcn_global_load_lds((gptr_t)((wn ? ld_eb : ld_ea) + 4 * w),
                                         (lptr_t)(lds + 2 * kStage + kStaging + stage * kScaleSlot + wn * BM), 4, 0, 0);
    };

    v4f acc[NT][NT];
    v4i fa_lo[4][2], fa_hi[4][2], fb[2][NT][2];
    v2i ea[2], eb[2];  // (sets) exponent bytes of tiles 0-3 and 4-7
    // D' = B . A^T: the first operand is the B fragment, its exponents come first.  Instructions of their own with the accumulator tied to the result
    // (left to the register allocator some do not accumulate in place and the moves spill); op_sel / op_sel_hi: bits 0 / 1 of the byte of either
    // scale register.  fresh: the first touch in a tile takes 0 as its addend.
    auto mma = [&](const v4i (&a)[2], const v4i (&b)[2], v4f& c, bool fresh, int ia, int jb, const v2i& sa, const v2i& sb) __attribute__((always_inline)) {
        const v8i fa8 = __builtin_shufflevector(a[0], a[1], 0, 1, 2, 3, 4, 5, 6, 7);
        const v8i fb8 = __builtin_shufflevector(b[0], b[1], 0, 1, 2, 3, 4, 5, 6, 7);
        const int sca = ia < 4 ? sa[0] : sa[1], scb = jb < 4 ? sb[0] : sb[1];
#define MI8_MS_ASM(JB, IA)                                                                                                  \
    case JB * 4 + IA:                                                                                                      \
        if (fresh)                                                                                                         \
            asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, 0, %3, %4 op_sel:[" #JB "&1," #IA "&1,0] "        \
                         "op_sel_hi:[" #JB ">>1," #IA ">>1,0] cbsz:0 blgp:0"                                               \
                         : "=a"(c)                                                                                         \
                         : "v"(fb8), "v"(fa8), "v"(scb), "v"(sca));                                                       \
        else                                                                                                               \
            asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[" #JB "&1," #IA "&1,0] "       \
                         "op_sel_hi:[" #JB ">>1," #IA ">>1,0] cbsz:0 blgp:0"                                               \
                         : "+a"(c)                                                                                         \
                         : "v"(fb8), "v"(fa8), "v"(scb), "v"(sca));                                                       \
        break;
        switch ((jb & 3) * 4 + (ia & 3)) {
            MI8_MS_ASM(0, 0) MI8_MS_ASM(0, 1) MI8_MS_ASM(0, 2) MI8_MS_ASM(0, 3)
            MI8_MS_ASM(1, 0) MI8_MS_ASM(1, 1) MI8_MS_ASM(1, 2) MI8_MS_ASM(1, 3)
            MI8_MS_ASM(2, 0) MI8_MS_ASM(2, 1) MI8_MS_ASM(2, 2) MI8_MS_ASM(2, 3)
            MI8_MS_ASM(3, 0) MI8_MS_ASM(3, 1) MI8_MS_ASM(3, 2) MI8_MS_ASM(3, 3)
        }
#undef MI8_MS_ASM
    };
    // what a step's first phase starts from: A tiles 0-3, all B tiles and the scales of the stage the read addresses point at, into set 0
    auto read_step_head = [&]() __attribute__((always_inline)) {
        ea[0] = *reinterpret_cast<lscale_t>((uintptr_t)rea);
        eb[0] = *reinterpret_cast<lscale_t>((uintptr_t)reb);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            read_a(fa_lo[t], t, 0);
            read_a(fa_lo[t], t, 1);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            read_b(fb[0][t], t, 0);
            read_b(fb[0][t], t, 1);
        }
    };

    if (ld_a != nullptr) {  // (uniform) prologue: the stages of steps 0 and 1
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int x = 0; x < kLoads; ++x) dma_one(s, true, x);
#pragma unroll
            for (int x = 0; x < kLoads; ++x) dma_one(s, false, x);
            dma_scales(s);
            advance_load_cursor();
        }
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __syncthreads();
    read_step_head();

    int step = 0;
    for (int cp_tile = 0; cp_tile < my_tiles; ++cp_tile) {
        const Tile td = my_tile(cp_tile);
        if (td.c == nullptr) continue;  // (uniform)
        // The wait between the phases: all loads but the eight of the first phase have landed, so the other stage is complete.  A tile's first
        // step follows the previous tile's epilogue, whose 32 stores are younger than those loads and may stay outstanding as well.
        // Either barrier is passed with the wave's reads of LDS in registers (lgkmcnt 0): the loads behind it fill what they read.
        auto k_step = [&](bool fresh, auto set_tag) __attribute__((always_inline)) {
            constexpr int S = decltype(set_tag)::value;
            const int cur = step & 1;
            __builtin_amdgcn_s_waitcnt(0xc07f);      // lgkmcnt(0)
            asm volatile("s_barrier" ::: "memory");  // every wave has what it reads of this stage's B rows, A tiles 0-3 and scales
#pragma unroll
            for (int x = 0; x < 32; ++x) {
                const int j = x >> 2, i = x & 3;
                mma(fa_lo[i], fb[S][j], acc[i][j], fresh, i, j, ea[S], eb[S]);
                if (x < 8) read_a(fa_hi[x >> 1], 4 + (x >> 1), x & 1);
                if (x >= 8 && x % 3 == 2) dma_one(cur, false, (x - 8) / 3);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (fresh)
                __builtin_amdgcn_s_waitcnt(vmcnt(8 + 32) & 0xF0FF);
            else
                __builtin_amdgcn_s_waitcnt(vmcnt(8) & 0xF0FF);
            asm volatile("s_barrier" ::: "memory");
            flip_read_stage(cur ^ 1);
#pragma unroll
            for (int x = 0; x < 32; ++x) {
                const int j = x >> 2, i = x & 3;
                mma(fa_hi[i], fb[S][j], acc[4 + i][j], fresh, 4 + i, j, ea[S], eb[S]);
                if (x < 16) read_b(fb[S ^ 1][x >> 1], x >> 1, x & 1);
                if (x >= 16 && x < 24) read_a(fa_lo[(x - 16) >> 1], (x - 16) >> 1, x & 1);
                if (x == 24) ea[S ^ 1] = *reinterpret_cast<lscale_t>((uintptr_t)rea);
                if (x == 25) eb[S ^ 1] = *reinterpret_cast<lscale_t>((uintptr_t)reb);
                if (i == 1) dma_one(cur, true, x >> 2);
                if (x == 30) dma_scales(cur);
                __builtin_amdgcn_sched_barrier(0);
            }
            advance_load_cursor();
            ++step;
        };
        if (td.nk > 0) {
            const std::integral_constant<int, 0> set0;
            const std::integral_constant<int, 1> set1;
            k_step(true, set0);
            int kt = 1;
            for (; kt + 1 < td.nk; kt += 2) {
                k_step(false, set1);
                k_step(false, set0);
            }
            if (kt < td.nk) k_step(false, set1);
        } else {  // an empty group, or rows behind the last one: zeros
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = (v4f){0, 0, 0, 0};
        }

        // ---- epilogue: acc[i][j][e] of lane l is C[row = 16 i + l % 16][col = 16 j + 4 (l / 16) + e] of the wave tile.  The output leaves through the
        // wave's staging area, 32 rows x 64 columns at a time, a pass's rows going to memory after the conversion of the next one.
        asm volatile("s_nop 15\n\ts_nop 15");  // (the last MFMA has retired)
        uint8_t* stg = lds + 2 * kStage + wave * 4096;
        const uint32_t stg_lds = (uint32_t)(uintptr_t)(lptr_t)stg;
        const int ldc_bytes = (int)p.ldc * 2;
        const __amdgpu_buffer_rsrc_t c_rows = __builtin_amdgcn_make_buffer_rsrc(td.c, 0, td.rows * ldc_bytes, 0x00020000);
        v4i staged[4];
        auto store_staged = [&](int jq, int ih) __attribute__((always_inline)) {
            // (a lane's store past the rows or columns that exist gets an offset past the end and is dropped)
            const int col = wn * WT + jq * 64 + (lane & 7) * 8;
            const int at = (wm * WT + ih * 32 + (lane >> 3)) * ldc_bytes + col * 2;
#pragma unroll
            for (int it = 0; it < 4; ++it)
                __builtin_amdgcn_raw_buffer_store_b128(staged[it], c_rows, col < td.cols ? at + it * 8 * ldc_bytes : 0x7FFFFFF0, 0, kOutStoreAux);
        };
#pragma unroll
        for (int jq = 0; jq < 2; ++jq)
#pragma unroll
            for (int ih = 0; ih < 4; ++ih) {
                uint2 o[2][4];
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int jj = 0; jj < 4; ++jj) {
                        float v[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e)  // (instructions of their own: the scheduler would move all 256 copies to the top and spill)
                            asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v[e]) : "a"(acc[2 * ih + t][4 * jq + jj][e]));
                        o[t][jj].x = pack_bf16x2(v[0], v[1]);
                        o[t][jj].y = pack_bf16x2(v[2], v[3]);
                    }
                asm volatile("" ::: "memory");
                if (jq + ih > 0) {
                    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the previous pass's rows are in registers
                    store_staged(ih == 0 ? jq - 1 : jq, ih == 0 ? 3 : ih - 1);
                }
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int jj = 0; jj < 4; ++jj) {
                        const int row = 16 * t + r16, cw = 16 * jj + 4 * kb;
                        const int chunk = (cw >> 3) ^ ((row >> 1) & 7);
                        const uint32_t saddr = stg_lds + (uint32_t)(row * 128 + chunk * 16 + (cw & 4) * 2);
                        // (asm: before an LDS store it knows of, the compiler waits for every direct-to-LDS load in flight)
                        asm volatile("ds_write_b64 %0, %1" ::"v"(saddr), "v"(o[t][jj]) : "memory");
                    }
                __builtin_amdgcn_s_waitcnt(0xc07f);
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int it = 0; it < 4; ++it) {
                    const int rw = it * 8 + (lane >> 3);
                    staged[it] = *reinterpret_cast<const v4i*>(stg + rw * 128 + (((lane & 7) ^ ((rw >> 1) & 7)) << 4));
                }
                asm volatile("" ::: "memory");
            }
        __builtin_amdgcn_s_waitcnt(0xc07f);
        store_staged(1, 3);
        // (read again: these registers are free during the epilogue, which would spill otherwise)
        __builtin_amdgcn_sched_barrier(0);
        read_step_head();
    }
    // loads issued for steps past the end have landed before the LDS is released
    __builtin_amdgcn_s_waitcnt(0x0070);
    __syncthreads();
}

template <typename Problem>
int launch(const Problem& pb, int64_t tiles, hipStream_t st, const char* what)
{
    auto kern = block_persistent_kernel<Problem>;
    static std::atomic<uint64_t> configured{0};
    if (int rc = reserve_dynamic_lds(reinterpret_cast<const void*>(kern), kLdsBytes, configured, what)) return rc;
    // one workgroup per compute unit, or as many as there are tiles, a multiple of 8 (every XCD takes an eighth of them, rounded up)
    const int64_t wanted = round_up(tiles, 8), cus = num_compute_units();
    hipLaunchKernelGGL(kern, dim3((unsigned)(wanted < cus ? wanted : cus)), dim3(kThreads), kLdsBytes, st, pb);
    return launch_status(what);
}

}  // namespace

int launch_persistent(BlockArgs& p, hipStream_t st)
{
    p.tiles_m = (int)ceil_div(p.M, BM);
    p.tiles_n = (int)ceil_div(p.N, BN);
    return launch(Dense{p}, (int64_t)p.tiles_m * p.tiles_n, st, "mi8_gemm_fp8_block");
}

int launch_persistent_grouped(BlockArgs& p, hipStream_t st)
{
    p.tiles_n = (int)ceil_div(p.N, BN);
    return launch(Grouped{p}, (ceil_div(p.M, BM) + p.E) * p.tiles_n, st, "mi8_grouped_gemm_fp8_block");
}

int launch_persistent_wgrad(BlockArgs& p, hipStream_t st)
{
    p.tiles_m = (int)ceil_div(p.M, BM);
    p.tiles_n = (int)ceil_div(p.N, BN);
    const GroupedK pb{p};
    return launch(pb, pb.grid_tiles(), st, "mi8_grouped_wgrad_fp8_block");
}

}  // namespace block
}  // namespace mi8
