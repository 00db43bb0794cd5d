// Products of bf16 and float16 matrices on tiles: y = x W^T and its two gradients, dense and for rows sorted by expert, with bias,
// activation and residual in the epilogue.
//
// Operands.  A tile's step is 64 elements of K.  Either operand may lie with its K contiguous (a weight or an activation in the forward) or with its
// rows contiguous (both operands of a weight gradient, the weight in the gradient of the input); both go from global memory straight to LDS, a 16-byte
// chunk a lane, and both take the same 128 bytes of LDS per row and step.
//   [row][64 K]: chunk c (8 K) of row r lies at c ^ swz16(r); a fragment is one 16-byte read.
//   [K][rows]: a K line holds the rows' elements side by side, in units of 16 rows; unit u of line k lies at u ^ f(k).  A fragment is two reads of 4 K
//   that gfx950's LDS transposes on the way (16 lanes read 4 lines x 32 bytes and get 4 K of one row each).  f spreads the eight lines that half
//   a wave reads at once over the banks.
// Which eight K a lane gets is the same for both, so any mix of them multiplies.  No operand is transposed in memory.
//
// Steps.  Two phases, each half of a wave's A tiles against all of its B tiles.  During the first the other A tiles of the stage are read, during the
// second the next stage's, each pair of B tiles into the registers of the pair that has just been multiplied.  A stage's rows are filled again for the
// step ST later as soon as every wave has read them: B's during the first phase, A's during the second, so that the loads have one to one and a half
// steps to arrive and go out evenly (all sixteen of a step within a quarter of a phase held up the MFMAs behind them: 16384 x 11008 -> 4096
// 1430 us).
//
// Edges cost nothing: an operand's buffer descriptor ends where its rows (or its K lines) end, lanes past it get zeros, and stores past C are
// dropped.  Only a last step that is not 64 K long masks the chunks past K of [row][K] operands.
//
// Workgroups walk tiles: an XCD takes a contiguous range of the order (neighbouring tiles share operand panels in its L2); the loads of the next tile's
// first steps are in flight during the epilogue.  Epilogue: where nothing is added, rounded and exchanged between lanes so that
// four of them store 64 bytes of a row; else 32 rows (in 128 x 128 tiles 16) x 64 columns a wave at a time through LDS in float32, so that bias, activation
// and residual act on the unrounded sum.  (Everything through LDS: 10 to 11 us a tile of 256 x 256 instead of 6, one wave on a SIMD waiting for each step: 64 experts
// of 1024 x 2048, 131072 rows, gradient of the input 585 us, now 536.)
//
// Bound by the matrix pipe and the clock that its power allows (counters: forward busy 76 % of the cycles at 1.76 GHz, gradient of the input 70 % at 1.80, of the
// weight 68 % at 1.83, no bank conflict in any): bf16, 16384 x 11008 -> 4096, forward 1000 to 1090 us, gradient of the input 1030 to 1110, of the weight 1070 to
// 1140 (1.3 to 1.48 PFLOP/s); 64 experts of 1024 x 2048, 131072 rows, 495, 536, 490 us.
#include <utility>

#include "mi8_gemm_tiles.h"
#include "mi8_elements.h"

namespace mi8 {
using namespace gemm;
namespace half {
namespace {

typedef __attribute__((address_space(3))) void* lptr_t;
typedef const __attribute__((address_space(3))) v4i* lfrag_t;
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s* ltr_t;

constexpr int kThreads = 256;
constexpr int kRowBytes = kStepK * 2;     // of an operand row per stage
// row tiles of a wave that the epilogue takes at a time, and what its staging of them takes (two 128 x 128 workgroups have 160 KB together)
template <int BM>
constexpr int kRowTiles = BM == 128 ? 1 : 2;
template <int BM, int BN>
constexpr int kStagingWave = 16 * kRowTiles<BM> * (BN < 128 ? BN / 2 : 64) * 4;
constexpr int kOutStoreAux = 1 | 2 | 16;   // sc0, nt, sc1: written through, a later kernel reads it

constexpr int vmcnt(int n) { return (n & 15) | ((n >> 4) << 14) | 0x0F70; }

// Four K of one row from four lines.  (The parameter's restrict tells the compiler that this read is of LDS that it knows: without, it waits for
// every direct load in flight before it.)
__device__ __forceinline__ v4s read_transposed(ltr_t __restrict p)
{
#ifdef __HIP_DEVICE_COMPILE__
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(p);
#else
    return v4s{};
#endif
}

// Lanes 16 kb .. 16 kb + 15 have columns 4 kb .. 4 kb + 3 of x and of y: afterwards two lanes' x, or y, one behind the other
__device__ __forceinline__ void exchange(uint32_t x, uint32_t y, uint32_t& first, uint32_t& second)
{
#ifdef __HIP_DEVICE_COMPILE__
    const auto halves = __builtin_amdgcn_permlane32_swap(x, y, false, false);  // x of lanes 0 - 31, y of lanes 0 - 31; x of lanes 32 - 63, y of those
    const auto rows = __builtin_amdgcn_permlane16_swap(halves[0], halves[1], false, false);
    first = rows[0];
    second = rows[1];
#endif
}

// f of the comment above, of a line of R rows.  256 bytes or more: the low two bits of k and bit 4 (lanes 0 - 31 read lines k .. k + 3 of two
// 16-line blocks); 128 bytes: two lines fill the banks, so bit 1 and bit 4.
template <int R>
__device__ __forceinline__ int line_swizzle(int k)
{
    return R >= 128 ? (k & 3) | ((k >> 4) & 1) << 2 : ((k >> 1) & 1) | ((k >> 4) & 1) << 1;
}

// One operand of R rows a tile: where its loads come from and its fragments lie.
template <bool BY_K, int R>
struct Operand {
    static constexpr int kLoads = R * kRowBytes / 1024 / 4;  // direct loads of a wave and step, 1 KB each
    static constexpr int kLanesPerLine = R / 8;              // (BY_K)
    static constexpr int kLinesPerLoad = BY_K ? 64 / kLanesPerLine : 8;

    // ---- loads.  base, bytes: the buffer descriptor of the step that is fetched next; past the last tile it is empty
    int ld;                // bytes between rows / lines
    uint32_t off[kLoads];  // this lane's, of each load: resident, a load is two instructions then
    int lane_chunk;        // (by rows) chunk of the step that this lane loads
    const uint8_t* base = nullptr;
    int bytes = 0, k_left = 0;  // k_left: of the contraction
    int last_line;              // (by K) bytes of the last line that are read

    // (made again for every tile: held through the epilogue they would spill)
    __device__ __forceinline__ void set_offsets(int64_t ld_elements, int lane, int wave)
    {
        ld = (int)ld_elements * 2;
        asm volatile("" : "+v"(lane));  // opaque: not the same as the last tile's
#pragma unroll
        for (int x = 0; x < kLoads; ++x) {
            const int first = first_of(wave, x);
            if constexpr (BY_K) {
                const int line = first + lane / kLanesPerLine, at = lane % kLanesPerLine;
                off[x] = (uint32_t)line * (uint32_t)ld + (uint32_t)((((at >> 1) ^ line_swizzle<R>(line)) << 5) + ((at & 1) << 4));
            } else {
                lane_chunk = (lane & 7) ^ swz16(lane >> 3);
                off[x] = (uint32_t)(first + (lane >> 3)) * (uint32_t)ld + (uint32_t)lane_chunk * 16;
            }
        }
    }
    // p: the operand's first row and K of the tile; rows: of the tile that exist; k: length of the contraction (0: no further tile)
    __device__ __forceinline__ void start(const uint8_t* p, int rows, int k)
    {
        // (all uniform, which the compiler loses track of where they come from a list of group sizes)
        const uint64_t at64 = reinterpret_cast<uint64_t>(p);
        base = reinterpret_cast<const uint8_t*>((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(at64 >> 32)) << 32 |
                                                (uint32_t)__builtin_amdgcn_readfirstlane((int)at64));
        rows = __builtin_amdgcn_readfirstlane(rows);
        k = __builtin_amdgcn_readfirstlane(k);
        k_left = k;
        if constexpr (BY_K) {
            last_line = (rows + 7) / 8 * 16;
            bytes = ((k < kStepK ? k : kStepK) - 1) * ld + last_line;
        } else {
            bytes = (rows - 1) * ld + (k + 7) / 8 * 16;
        }
        if (k == 0) bytes = 0;
    }
    __device__ __forceinline__ void advance()
    {
        base += BY_K ? kStepK * ld : kRowBytes;
        k_left -= kStepK;
        if constexpr (BY_K) {
            if (k_left < kStepK) bytes = (k_left - 1) * ld + last_line;  // (uniform; the last step of a tile, and what start() replaces)
        } else {
            bytes -= kRowBytes;
        }
    }
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t descriptor() const { return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, bytes, 0x00020000); }
    // What is added to a lane's offsets where its chunk of the step at hand is past K (by rows): more than a descriptor has
    __device__ __forceinline__ uint32_t past_end() const { return BY_K || lane_chunk * 8 < k_left ? 0u : 0x80000000u; }
    // the first row (by rows) or line (by K) that load x of wave w fills
    __device__ static __forceinline__ int first_of(int wave, int x) { return BY_K ? wave * 16 + x * kLinesPerLoad : (wave * kLoads + x) * 8; }
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t d, uint32_t past, uint8_t* stage, int wave, int x) const
    {
#ifdef __HIP_DEVICE_COMPILE__
        __builtin_amdgcn_raw_ptr_buffer_load_lds(d, (lptr_t)(stage + first_of(wave, x) * (BY_K ? R * 2 : kRowBytes)), 16, (int)(off[x] + past), 0, 0, 0);
#endif
    }

    // ---- fragments of rows first + 16 t
    uint32_t at[2];
    __device__ __forceinline__ void init_reads(uint32_t lds0, int first, int lane)
    {
        const int r16 = lane & 15, kb = lane >> 4;
        if constexpr (BY_K) {
            const int k = 16 * kb + (r16 >> 2);
            at[0] = lds0 + (uint32_t)(k * R * 2 + (((first >> 4) ^ line_swizzle<R>(k)) << 5) + (r16 & 3) * 8);
        } else {
#pragma unroll
            for (int q = 0; q < 2; ++q) at[q] = lds0 + (uint32_t)((first + r16) * kRowBytes + (((2 * kb + q) ^ swz16(r16)) << 4));
        }
    }
    // addresses in a stage; opaque, so that what is added for tiles goes into the instructions
    struct At {
        uint32_t v[2];
    };
    __device__ __forceinline__ At in_stage(uint32_t stage_off) const
    {
        At r{{at[0] + stage_off, BY_K ? 0 : at[1] + stage_off}};
        asm volatile("" : "+v"(r.v[0]));
        if constexpr (!BY_K) asm volatile("" : "+v"(r.v[1]));
        return r;
    }
    __device__ static __forceinline__ v4i read(int t, int q, const At& from)
    {
        if constexpr (BY_K) {
            uint32_t a = from.v[0] ^ (uint32_t)(t << 5);
            const v4s x = read_transposed((ltr_t)(uintptr_t)(a + q * 8 * R * 2)), y = read_transposed((ltr_t)(uintptr_t)(a + (q * 8 + 4) * R * 2));
            return __builtin_bit_cast(v4i, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            return *reinterpret_cast<lfrag_t>((uintptr_t)(from.v[q] + t * 16 * kRowBytes));
        }
    }
};

// What a workgroup needs to know about a tile.  rows == 0: none.
struct Tile {
    const uint8_t *a, *b;
    int k;           // length of the contraction (0: zeros)
    int a_rows;      // rows of A in the tile (those past rows are not stored)
    int rows, cols;  // of C that exist in the tile
    int64_t row0;    // of C
    int col0;
};

// The kernel's argument as it is in memory.  What describes a tile and its epilogue is read again for every tile: held in scalar registers it
// is spilled into lanes of vector registers, and read back from them between the MFMAs of every step.
typedef const __attribute__((address_space(4))) HalfArgs* args_t;
__device__ __forceinline__ args_t args_in_memory()
{
    args_t p = (args_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return p;
}

template <bool GROUP_K, int BM, int BN>
struct Problem {
    struct Cache {
        GroupCache g;
        int units, used, group_at_rank;
        int spread;  // (K in groups) the groups' tiles are spread over the XCDs
    };
    __device__ static __forceinline__ Cache prepare(const HalfArgs& p)
    {
        Cache c{};
        if (!p.sizes) return c;
        if constexpr (GROUP_K) {
            GroupedWgradProblem order{};
            order.sizes = p.sizes;
            order.E = p.E;
            order.T = p.K;
            const WgradCache w = order.prepare();
            c.g = w.g;
            c.group_at_rank = w.group_at_rank;
            c.spread = c.g.valid && (int64_t)__builtin_amdgcn_readlane(c.g.m, __builtin_amdgcn_readlane(c.group_at_rank, 0)) * 7 > p.K;
        } else {
            c.g = build_group_cache<BM>(p.sizes, p.E, p.M);
            const GroupSpan end = locate_group_cached<BM, true>(c.g, p.sizes, p.E, p.M, (int64_t)1 << 60);
            c.units = (int)end.units_before;
            if (c.g.valid)
                c.used = __builtin_amdgcn_readlane(c.g.start, p.E - 1) + __builtin_amdgcn_readlane(c.g.m, p.E - 1);
            else
                c.used = (int)end.rows_before;
        }
        return c;
    }
    __device__ static __forceinline__ int total(const HalfArgs& p, const Cache& c)
    {
        if (!p.sizes) return p.tiles_m * p.tiles_n * p.slices;
        if constexpr (GROUP_K) return 8 * (c.spread ? p.E * ((p.tiles_m * p.tiles_n + 7) >> 3) : ((p.E + 7) >> 3) * p.tiles_m * p.tiles_n);
        return (c.units + (p.M - c.used + BM - 1) / BM) * p.tiles_n;
    }
    __device__ static __forceinline__ int rest(int of, int from, int most) { return of - from < most ? of - from : most; }
    template <bool A_BY_K, bool B_BY_K>
    __device__ static __forceinline__ Tile tile(const Cache& c, int t)
    {
        const args_t q = args_in_memory();
        Tile d{};
        if (!q->sizes || GROUP_K) {
            int tm, tn, e = 0;
            int64_t k0 = 0;
            d.k = q->K;
            if (!q->sizes) {
                const int tiles = q->tiles_m * q->tiles_n;
                e = t / tiles;  // (the slice: its partial sums lie where a group's matrix would)
                t -= e * tiles;
                k0 = (int64_t)e * q->slice_k;
                d.k = rest(q->K, (int)k0, q->slice_k);
                GemmArgs order;
                order.tiles_m = q->tiles_m;
                order.tiles_n = q->tiles_n;
                tile_coords(order, t, tm, tn);
            } else {
                // The groups by size.  One after the other to the XCDs, whose tiles of it share its operands in the L2, or, where the longest is more than an
                // XCD's part of all of them, an eighth of a group's tiles to each XCD.  us of 64 groups, the longest an eighth, 1024 x 2048: 520 / 591; 8 groups,
                // the longest a half, 1792 x 1024: 332 / 160.
                const int per_group = q->tiles_m * q->tiles_n, slot = t >> 3, xcd = t & 7;
                int rank, in;
                if (c.spread) {
                    const int per_xcd = (per_group + 7) >> 3;
                    rank = slot / per_xcd;
                    in = ((xcd + rank) & 7) * per_xcd + slot % per_xcd;
                } else {
                    const int k = slot / per_group;
                    rank = (k & 1) ? 8 * k + 7 - xcd : 8 * k + xcd;
                    in = slot % per_group;
                }
                if (rank >= q->E || in >= per_group) return d;
                e = c.g.valid ? __builtin_amdgcn_readlane(c.group_at_rank, rank) : rank;
                const GroupSpan s = locate_group_cached<128, false>(c.g, q->sizes, q->E, q->K, e);
                k0 = s.rows_before;
                d.k = (int)s.m;
                tm = in / q->tiles_n;
                tn = in % q->tiles_n;
            }
            const int m0 = tm * BM, n0 = tn * BN;
            d.rows = d.a_rows = rest(q->M, m0, BM);
            d.cols = rest(q->N, n0, BN);
            d.a = q->A + (A_BY_K ? k0 * q->lda + m0 : m0 * q->lda + k0) * 2;
            d.b = q->B + (B_BY_K ? k0 * q->ldb + n0 : n0 * q->ldb + k0) * 2;
            d.row0 = (int64_t)e * q->M + m0;
            d.col0 = n0;
            return d;
        }
        const int mt = t / q->tiles_n;
        d.col0 = t % q->tiles_n * BN;
        d.cols = rest(q->N, d.col0, BN);
        if (mt >= c.units) {
            d.row0 = c.used + (int64_t)(mt - c.units) * BM;
            d.rows = rest(q->M, (int)d.row0, BM);
            return d;
        }
        const GroupSpan s = locate_group_cached<BM, true>(c.g, q->sizes, q->E, q->M, mt);
        const int inside = (int)(mt - s.units_before) * BM;
        d.row0 = s.rows_before + inside;
        d.rows = d.a_rows = rest((int)s.m, inside, BM);
        d.k = q->K;
        d.a = q->A + d.row0 * q->lda * 2;
        d.b = q->B + (s.e * q->b_group_stride + (B_BY_K ? (int64_t)d.col0 : d.col0 * q->ldb)) * 2;
        return d;
    }
};

// f(constant 0) .. f(constant N - 1), written out
template <typename F, int... X>
__device__ __forceinline__ void written_out(std::integer_sequence<int, X...>, F&& f)
{
    (f(std::integral_constant<int, X>{}), ...);
}

// f(constant pass) for the uniform pass < N
template <int N, int AT = 0, typename F>
__device__ __forceinline__ void for_pass(int pass, F&& f)
{
    if constexpr (AT < N) {
        if (pass == AT)
            f(std::integral_constant<int, AT>{});
        else
            for_pass<N, AT + 1>(pass, f);
    }
}

template <typename T, bool A_BY_K, bool B_BY_K, bool GROUP_K, int BM, int BN, int ST>
__global__ __launch_bounds__(kThreads, BM > 128 ? 1 : 2) void half_tiles_kernel(const HalfArgs p)
{
    constexpr int WTM = BM / 2, WTN = BN / 2, TM = WTM / 16, TN = WTN / 16;
    constexpr int STAGE = (BM + BN) * kRowBytes;
    typedef Problem<GROUP_K, BM, BN> P;
    typedef Operand<A_BY_K, BM> OpA;
    typedef Operand<B_BY_K, BN> OpB;
    constexpr int LD = OpA::kLoads + OpB::kLoads;
    static_assert(ST >= 2 && LD * ST < 64, "the loads in flight are counted in six bits");
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    const int r16 = lane & 15, kb = lane >> 4;

    const typename P::Cache cache = P::prepare(p);
    const int total = P::total(p, cache), block = (int)blockIdx.x, blocks = (int)gridDim.x;
    int first_tile = block, tile_stride = blocks, last_tile = total;
    if (!GROUP_K || !p.sizes) {
        const int per_xcd = (total + 7) / 8, xcd = block & 7;
        first_tile = xcd * per_xcd + (block >> 3);
        tile_stride = (blocks + 7 - xcd) >> 3;
        last_tile = xcd * per_xcd + per_xcd < total ? xcd * per_xcd + per_xcd : total;
    }
    const int my_tiles = first_tile < last_tile ? (last_tile - first_tile + tile_stride - 1) / tile_stride : 0;
    if (my_tiles == 0) return;
    auto my_tile = [&](int i) __attribute__((always_inline)) { return P::template tile<A_BY_K, B_BY_K>(cache, first_tile + i * tile_stride); };

    OpA oa;
    OpB ob;
    oa.set_offsets(p.lda, lane, wave);
    ob.set_offsets(p.ldb, lane, wave);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lptr_t)lds;
    oa.init_reads(lds0, wm * WTM, lane);
    ob.init_reads(lds0 + BM * kRowBytes, wn * WTN, lane);

    // ---- load cursor: the step that is fetched next; past the last tile its descriptors are empty
    int ld_tile = -1;
    auto next_load_tile = [&]() __attribute__((always_inline)) {
        while (ld_tile + 1 < my_tiles) {
            ++ld_tile;
            const Tile d = my_tile(ld_tile);
            if (d.rows > 0 && d.k > 0) {
                oa.start(d.a, d.a_rows, d.k);
                ob.start(d.b, d.cols, d.k);
                return;
            }
        }
        oa.start(nullptr, 1, 0);
        ob.start(nullptr, 1, 0);
    };
    auto advance = [&]() __attribute__((always_inline)) {
        oa.advance();
        ob.advance();
        if (oa.k_left <= 0) next_load_tile();  // (uniform)
    };
    next_load_tile();
    v4f acc[TM][TN];
    // A tiles 0 .. TM / 2 - 1 and the rest; B tiles; [half of the step's K]
    constexpr int TH = TM / 2;
    v4i fa_lo[TH][2], fa_hi[TH][2], fb[TN][2];
    const v4f zero = {0, 0, 0, 0};

    auto read_head = [&](uint32_t stage_off) __attribute__((always_inline)) {
        const typename OpA::At at_a = oa.in_stage(stage_off);
        const typename OpB::At at_b = ob.in_stage(stage_off);
#pragma unroll
        for (int x = 0; x < 2 * TH; ++x) fa_lo[x >> 1][x & 1] = oa.read(x >> 1, x & 1, at_a);
#pragma unroll
        for (int x = 0; x < 2 * TN; ++x) fb[x >> 1][x & 1] = ob.read(x >> 1, x & 1, at_b);
    };

    // ---- prologue: the first ST steps are on their way, what the first one starts from in registers
    {
#pragma unroll
        for (int s = 0; s < ST; ++s) {
            const uint32_t past_a = oa.past_end(), past_b = ob.past_end();
            const __amdgpu_buffer_rsrc_t da = oa.descriptor(), db = ob.descriptor();
#pragma unroll
            for (int x = 0; x < OpB::kLoads; ++x) ob.load(db, past_b, lds + s * STAGE + BM * kRowBytes, wave, x);
#pragma unroll
            for (int x = 0; x < OpA::kLoads; ++x) oa.load(da, past_a, lds + s * STAGE, wave, x);
            advance();
        }
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
        asm volatile("s_barrier" ::: "memory");
        read_head(0);
    }

    constexpr int CW = WTN < 64 ? WTN : 64;                            // columns that the epilogue stages at a time
    constexpr int JT = CW / 16, CHUNKS = CW / 4, LPR = CW / 8, RPI = 64 / LPR;  // ... lanes per row, rows per access
    constexpr int RT = kRowTiles<BM>, kRows = 16 * RT / RPI;           // ... row tiles at a time, accesses for them
    constexpr int kPasses = TM / RT * (WTN / CW);
    constexpr int kStores = kPasses * kRows;                           // of a wave and tile, where rows are whole 16-byte chunks
    static_assert(LD * (ST - 1) + kStores < 64, "operations in flight are counted in six bits");
    // stores of whole 16-byte chunks of a row, one a lane and access: 1, two with z, 3 where nothing is added to the product; 0: there are odd ones
    const int stores = !p.wide ? 0 : p.z ? 2 : p.bias || p.residual || p.act != MI8_ACT_NONE ? 1 : 3;
    int slot = 0;
    for (int i = 0; i < my_tiles; ++i) {
        const Tile td = my_tile(i);
        if (td.rows == 0) continue;  // (uniform)
        auto k_step = [&](auto fresh_tag) __attribute__((always_inline)) {
            constexpr bool kFresh = decltype(fresh_tag)::value;
            // A phase: the A tiles of one half, all B tiles, both halves of K.  B tiles go in pairs, so that two MFMAs into one accumulator lie TM apart.
            constexpr int kPhase = 2 * TH * TN, kPair = 2 * TM;
            const int next = slot + 1 == ST ? 0 : slot + 1;
            uint8_t* const stage = lds + slot * STAGE;
            const uint32_t here = (uint32_t)(slot * STAGE), there = (uint32_t)(next * STAGE);
            auto mma_one = [&](auto x_tag, auto& fa, auto hi_tag) __attribute__((always_inline)) {
                constexpr int x = decltype(x_tag)::value, r = x % kPair, q = r / TM, tj = 2 * (x / kPair) + r % TM / TH, ti = r % TH;
                v4f& c = acc[decltype(hi_tag)::value * TH + ti][tj];
                if constexpr (BM > 128)
                    mma_tied<T>(fb[tj][q], fa[ti][q], c, kFresh && q == 0);
                else
                    c = mma<T>(fb[tj][q], fa[ti][q], kFresh && q == 0 ? zero : c);
            };
            // ---- phase A.  The stage's B rows are free once every wave has what it read of them in the last phase (its last reads are given a quarter
            // of this one to arrive); they are filled for the step ST later, and this stage's other A tiles are read.
            {
                const uint32_t past_b = ob.past_end();
                const __amdgpu_buffer_rsrc_t db = ob.descriptor();
                const typename OpA::At at_a = oa.in_stage(here);
                constexpr int kBar = kPhase / 4, kLeft = kPhase - kBar;
                written_out(std::make_integer_sequence<int, kPhase>{}, [&](auto x_tag) __attribute__((always_inline)) {
                    constexpr int x = decltype(x_tag)::value;
                    mma_one(x_tag, fa_lo, std::integral_constant<int, 0>{});
                    if constexpr (x >= kBar) {
                        constexpr int l = x - kBar;
#pragma unroll
                        for (int y = l * OpB::kLoads / kLeft; y < (l + 1) * OpB::kLoads / kLeft; ++y) ob.load(db, past_b, stage + BM * kRowBytes, wave, y);
                    }
#pragma unroll
                    for (int y = 0; y < 2 * TH; ++y)
                        if (y * kPhase / (4 * TH) + kBar == x) fa_hi[y >> 1][y & 1] = oa.read(TH + (y >> 1), y & 1, at_a);
                    if constexpr (x == kBar - 1) {
                        __builtin_amdgcn_sched_barrier(0);
                        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
                        asm volatile("s_barrier" ::: "memory");
                    }
                    __builtin_amdgcn_sched_barrier(0);
                });
            }
            // ---- phase B.  The next stage has landed (all but the loads of later steps and phase A's) and this one has been read, in every wave: its A rows
            // are filled, and the next step's first A tiles and, pair by pair as they are used up, its B tiles are read.
            {
                const uint32_t past_a = oa.past_end();
                const __amdgpu_buffer_rsrc_t da = oa.descriptor();
                const typename OpA::At at_a = oa.in_stage(there);
                const typename OpB::At at_b = ob.in_stage(there);
                // (a tile's first step follows an epilogue, whose stores are younger than the loads waited for, or the prologue, which has waited for all)
                constexpr int kYounger = LD * (ST - 2) + OpB::kLoads;
                if (kFresh && stores == 2)  // (as far as can be counted)
                    __builtin_amdgcn_s_waitcnt(vmcnt(kYounger + 2 * kStores < 63 ? kYounger + 2 * kStores : 63) & 0xF0FF);  // and lgkmcnt(0)
                else if (kFresh && stores)
                    __builtin_amdgcn_s_waitcnt(vmcnt(kYounger + kStores) & 0xF0FF);
                else
                    __builtin_amdgcn_s_waitcnt(vmcnt(kYounger) & 0xF0FF);
                asm volatile("s_barrier" ::: "memory");
                __builtin_amdgcn_sched_barrier(0);
                written_out(std::make_integer_sequence<int, kPhase>{}, [&](auto x_tag) __attribute__((always_inline)) {
                    constexpr int x = decltype(x_tag)::value, pair = x / kPair, r = x % kPair, kLoading = kPhase * 3 / 4;
                    mma_one(x_tag, fa_hi, std::integral_constant<int, 1>{});
                    if constexpr (pair == 0) {
#pragma unroll
                        for (int y = 0; y < 2 * TH; ++y)
                            if (y * kPair / (2 * TH) == x) fa_lo[y >> 1][y & 1] = oa.read(y >> 1, y & 1, at_a);
                    } else if constexpr (r < 4) {
                        fb[2 * (pair - 1) + (r >> 1)][r & 1] = ob.read(2 * (pair - 1) + (r >> 1), r & 1, at_b);
                    }
                    if constexpr (x < kLoading) {
#pragma unroll
                        for (int y = x * OpA::kLoads / kLoading; y < (x + 1) * OpA::kLoads / kLoading; ++y) oa.load(da, past_a, stage, wave, y);
                    }
                    if constexpr (x == kLoading) oa.advance();
                    if constexpr (x == (kLoading + 1 < kPhase ? kLoading + 1 : kLoading)) ob.advance();
                    __builtin_amdgcn_sched_barrier(0);
                });
#pragma unroll
                for (int y = 0; y < 4; ++y) fb[TN - 2 + (y >> 1)][y & 1] = ob.read(TN - 2 + (y >> 1), y & 1, at_b);
                if (oa.k_left <= 0) next_load_tile();  // (uniform)
            }
            slot = next;
        };
        if (td.k > 0) {
            oa.set_offsets(p.lda, lane, wave);
            ob.set_offsets(p.ldb, lane, wave);
            k_step(std::true_type{});
            for (int k = kStepK; k < td.k; k += kStepK) k_step(std::false_type{});
        } else {  // an empty group, or rows behind the last one
#pragma unroll
            for (int a = 0; a < TM; ++a)
#pragma unroll
                for (int b = 0; b < TN; ++b) acc[a][b] = zero;
        }

        // ---- epilogue: acc[a][b][e] of lane l is C[16 a + l % 16][16 b + 4 (l / 16) + e] of the wave tile
        asm volatile("s_nop 15\n\ts_nop 15");  // (the last MFMA has retired: the stores to LDS below are the compiler's blind spot)
        const args_t q = args_in_memory();
        if constexpr (BM <= 128) {
            if (q->partial) {  // (uniform) a slice's sums
#pragma unroll
                for (int a = 0; a < TM; ++a)
#pragma unroll
                    for (int b = 0; b < TN; ++b) {
                        const int row = wm * WTM + 16 * a + r16, col = wn * WTN + 16 * b + 4 * kb;
                        if (row < td.rows && col < td.cols) *reinterpret_cast<v4f*>(q->partial + (td.row0 + row) * q->ld_partial + td.col0 + col) = acc[a][b];
                    }
                read_head((uint32_t)(slot * STAGE));
                continue;
            }
        }
        const int64_t ldc = q->ldc;
        const __amdgpu_buffer_rsrc_t c_rows = __builtin_amdgcn_make_buffer_rsrc((void*)(q->C + td.row0 * ldc + td.col0), 0, (int)((int64_t)td.rows * ldc * 2), 0x00020000);
        if (stores == 3) {
            // Nothing to add: straight from the accumulators.  Of two tiles side by side a lane has four columns each; two exchanges between the rows of
            // 16 lanes give it eight columns of one, and four lanes 64 bytes of a row.
#pragma unroll
            for (int a = 0; a < TM; ++a) {
                const int row = wm * WTM + 16 * a + r16;
#pragma unroll
                for (int b = 0; b < TN; b += 2) {
                    uint32_t first[2], second[2];
                    v4f x = acc[a][b], y = acc[a][b + 1];
                    if constexpr (BM > 128) {  // (read here and not before: copies of all of them would spill)
                        asm volatile("" : "+a"(x));
                        asm volatile("" : "+a"(y));
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) exchange(T::pack(x[2 * h], x[2 * h + 1]), T::pack(y[2 * h], y[2 * h + 1]), first[h], second[h]);
                    const int col = wn * WTN + 16 * b + 8 * kb;
                    __builtin_amdgcn_raw_buffer_store_b128((u32x4_t){first[0], first[1], second[0], second[1]}, c_rows, col < td.cols ? (int)((row * ldc + col) * 2) : 0x7FFFFFF0, 0,
                                                           kOutStoreAux);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            read_head((uint32_t)(slot * STAGE));
            continue;
        }
        uint8_t* const stg = lds + ST * STAGE + wave * kStagingWave<BM, BN>;
        const uint32_t stg_at = (uint32_t)(uintptr_t)(lptr_t)stg + (uint32_t)(r16 * CW * 4);
        const int row0 = wm * WTM, col0 = wn * WTN;
        // Pass (jq, a): RT x 16 rows x CW columns.  A loop, not copies of it: only what writes the accumulators to LDS is chosen by the pass.  The next
        // pass's are written as soon as this one's are in registers.
        auto stage_pass = [&](int pass) __attribute__((always_inline)) {
            for_pass<kPasses>(pass, [&](auto pass_tag) __attribute__((always_inline)) {
                constexpr int a0 = decltype(pass_tag)::value % (TM / RT) * RT, j0 = decltype(pass_tag)::value / (TM / RT) * JT;
#pragma unroll
                for (int a = 0; a < RT; ++a)
#pragma unroll
                    for (int b = 0; b < JT; ++b) {
                        const uint32_t at = stg_at + (uint32_t)(a * 16 * CW * 4) + (uint32_t)(((4 * b + kb) ^ (r16 & (CHUNKS - 1))) << 4);
                        // (asm: before an LDS store it knows of, the compiler waits for every direct load in flight)
                        const v4f v = acc[a0 + a][j0 + b];
                        if constexpr (BM > 128)  // (LDS stores take accumulator registers; copies of them would be moved out of this loop and spill)
                            asm volatile("ds_write_b128 %0, %1" ::"v"(at), "a"(v) : "memory");
                        else
                            asm volatile("ds_write_b128 %0, %1" ::"v"(at), "v"(v) : "memory");
                    }
            });
        };
        stage_pass(0);
        const uint16_t* const residual = q->residual;
        const int act = q->act;
        float bias[8];
        Eight<T> next_residual[kRows];  // of the pass at hand, loaded during the one before
        auto load_residual = [&](int pass) __attribute__((always_inline)) {
            const int col = col0 + pass / (TM / RT) * CW + (lane % LPR) * 8;
#pragma unroll
            for (int it = 0; it < kRows; ++it) {
                const int row = row0 + pass % (TM / RT) * (16 * RT) + it * RPI + lane / LPR;
                next_residual[it].load(residual + (td.row0 + row) * q->ldr + td.col0, col, row < td.rows ? td.cols : 0);
            }
        };
        if (residual) load_residual(0);
#pragma unroll 1
        for (int pass = 0; pass < kPasses; ++pass) {
            const int pass_row = row0 + pass % (TM / RT) * (16 * RT), col = col0 + pass / (TM / RT) * CW + (lane % LPR) * 8;
            if (pass % (TM / RT) == 0) {
#pragma unroll
                for (int e = 0; e < 8; ++e) bias[e] = 0.0f;
                if (q->bias && q->bias_f32) {
                    Eight<F32> b;
                    b.load(reinterpret_cast<const float*>(q->bias) + td.col0, col, td.cols);
                    b.get(bias);
                } else if (q->bias) {
                    Eight<T> b;
                    b.load(reinterpret_cast<const uint16_t*>(q->bias) + td.col0, col, td.cols);
                    b.get(bias);
                }
            }
            __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
            __builtin_amdgcn_wave_barrier();
            v4f v[kRows][2];
            Eight<T> r[kRows];
#pragma unroll
            for (int it = 0; it < kRows; ++it) {
                const int rw = it * RPI + lane / LPR, chunk = (lane % LPR) * 2;
#pragma unroll
                for (int h = 0; h < 2; ++h) v[it][h] = *reinterpret_cast<const v4f*>(stg + rw * CW * 4 + (((chunk + h) ^ (rw & (CHUNKS - 1))) << 4));
                r[it] = next_residual[it];
            }
            __builtin_amdgcn_s_waitcnt(0xc07f);
            __builtin_amdgcn_wave_barrier();
            if (pass + 1 < kPasses) {
                stage_pass(pass + 1);
                if (residual) load_residual(pass + 1);
            }
            float f[kRows][8];
            int rows[kRows], n[kRows];
#pragma unroll
            for (int it = 0; it < kRows; ++it) {
                rows[it] = pass_row + it * RPI + lane / LPR;
                n[it] = rows[it] < td.rows ? td.cols : 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) f[it][e] = v[it][e >> 2][e & 3] + bias[e];
            }
            if (stores == 2) {  // (the vmcnt of the next step counts on one store for each, whatever its lanes)
                const int64_t ldz = q->ldz;
                const __amdgpu_buffer_rsrc_t z_rows = __builtin_amdgcn_make_buffer_rsrc((void*)(q->z + td.row0 * ldz + td.col0), 0, (int)((int64_t)td.rows * ldz * 2), 0x00020000);
#pragma unroll
                for (int it = 0; it < kRows; ++it)
                    __builtin_amdgcn_raw_buffer_store_b128(Eight<T>::pack(f[it]), z_rows, col < td.cols ? (int)((rows[it] * ldz + col) * 2) : 0x7FFFFFF0, 0, kOutStoreAux);
            } else if (!stores && q->z) {
#pragma unroll
                for (int it = 0; it < kRows; ++it) Eight<T>::store(q->z + (td.row0 + rows[it]) * q->ldz + td.col0, col, n[it], f[it]);
            }
            if (act != MI8_ACT_NONE) activate(act, f);
            if (residual) {
#pragma unroll
                for (int it = 0; it < kRows; ++it) {
                    float x[8];
                    r[it].get(x);
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[it][e] += x[e];
                }
            }
            if (stores) {  // (uniform)
#pragma unroll
                for (int it = 0; it < kRows; ++it)
                    __builtin_amdgcn_raw_buffer_store_b128(Eight<T>::pack(f[it]), c_rows, col < td.cols ? (int)((rows[it] * ldc + col) * 2) : 0x7FFFFFF0, 0, kOutStoreAux);
            } else {
#pragma unroll
                for (int it = 0; it < kRows; ++it) Eight<T>::store(q->C + (td.row0 + rows[it]) * ldc + td.col0, col, n[it], f[it]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        // (read again: these registers are free during the epilogue, which would spill otherwise)
        read_head((uint32_t)(slot * STAGE));
    }
    // loads issued for steps past the end have landed before the LDS is released
    __builtin_amdgcn_s_waitcnt(0x0070);
    __syncthreads();
}

template <typename T, bool A_BY_K, bool B_BY_K, bool GROUP_K, int BM, int BN, int ST>
int launch(HalfArgs p, hipStream_t st)
{
    auto kern = half_tiles_kernel<T, A_BY_K, B_BY_K, GROUP_K, BM, BN, ST>;
    constexpr int kLds = ST * (BM + BN) * kRowBytes + 4 * kStagingWave<BM, BN>;
    static std::atomic<uint64_t> configured{0};
    if (int rc = reserve_dynamic_lds(reinterpret_cast<const void*>(kern), kLds, configured, "mi8_gemm_half")) return rc;
    p.tiles_m = (int)ceil_div(p.M, BM);
    p.tiles_n = (int)ceil_div(p.N, BN);
    int64_t tiles = (int64_t)p.tiles_m * p.tiles_n * p.slices;
    if (p.sizes) tiles = GROUP_K ? (int64_t)8 * p.E * ceil_div(tiles, 8) : (ceil_div(p.M, BM) + p.E) * p.tiles_n;
    // as many workgroups as live on the chip at once, or as there are tiles, a multiple of 8 (an XCD takes an eighth of them)
    const int64_t wanted = round_up(tiles, 8), most = (int64_t)num_compute_units() * (BM > 128 ? 1 : 2);
    hipLaunchKernelGGL(kern, dim3((unsigned)(wanted < most ? wanted : most)), dim3(kThreads), kLds, st, p);
    return launch_status("mi8_gemm_half");
}

template <typename T, int BM, int BN, int ST>
int launch_layout(const HalfArgs& p, bool a_by_k, bool b_by_k, hipStream_t st)
{
    if (a_by_k) return launch<T, true, true, true, BM, BN, ST>(p, st);
    if (b_by_k) return launch<T, false, true, false, BM, BN, ST>(p, st);
    return launch<T, false, false, false, BM, BN, ST>(p, st);
}

template <typename T>
int launch_variant(const HalfArgs& p, bool a_by_k, bool b_by_k, int variant, hipStream_t st)
{
    switch (variant) {
        case MI8_HALF_256: return launch_layout<T, 256, 256, 2>(p, a_by_k, b_by_k, st);
        case MI8_HALF_192:  // (lines of 192 rows do not divide into loads: A by rows)
            return b_by_k ? launch<T, false, true, false, 192, 256, 2>(p, st) : launch<T, false, false, false, 192, 256, 2>(p, st);
        case MI8_HALF_128: return launch_layout<T, 128, 128, 2>(p, a_by_k, b_by_k, st);
        default: return launch_layout<T, 64, 64, 4>(p, a_by_k, b_by_k, st);
    }
}

}  // namespace

int launch_tiles(const HalfArgs& p, int hp_dtype, bool a_by_k, bool b_by_k, int variant, hipStream_t st)
{
    return hp_dtype == MI8_BF16 ? launch_variant<Bf16>(p, a_by_k, b_by_k, variant, st) : launch_variant<F16>(p, a_by_k, b_by_k, variant, st);
}

}  // namespace half
}  // namespace mi8

// ---- C ABI ---------------------------------------------------------------------------------------------------------------

using namespace mi8;

namespace {

// What a product's launch takes, as a model of rounds of tiles fitted to measurements: a round's time is its steps times what a step takes, and a constant
// (prologue, epilogue, launch).  A step takes longer the more of the chip works (the clock falls): us with one workgroup, and with the chip full, below; between
// them about as the square of the part that works, and as long as with a full chip where compute units have two workgroups.  Measured, for 256 x 256 and K =
// 4096: 64 tiles 78 us, 192 tiles 88, a round of four full ones 97.  192 x 256 is for the sizes that leave much of a last round of 256 x 256 idle: bf16
// 777 x 4096 -> 11008 79 us (256: 91, 128: 87), 6000 x 11008 -> 4096 382 (439, 447).  One constant stands for both epilogues, straight from the accumulators and
// through LDS, which differ by 4 us in a full tile of 256 x 256.  Of 152 dense products of 48 to 16384 rows in all three layouts, no choice was over 8 % off the best tile.
struct TileCost {
    int variant;
    int64_t rows, cols, per_cu;
    double one, full, fixed;
    int64_t tiles(int64_t M, int64_t N) const { return ceil_div(M, rows) * ceil_div(N, cols); }
};
constexpr TileCost kTiles[] = {
    {MI8_HALF_256, 256, 256, 1, 1.05, 1.42, 10.0}, {MI8_HALF_128, 128, 128, 2, 0.41, 0.79, 6.0}, {MI8_HALF_64, 64, 64, 2, 0.21, 0.345, 5.0}, {MI8_HALF_192, 192, 256, 1, 0.84, 1.07, 8.0},
};
constexpr int kSquare = 3;  // the first ones: for every layout, and for groups

double rounds_us(const TileCost& t, int64_t tiles, int64_t steps, int64_t cus)
{
    const int64_t slots = cus * t.per_cu, full = tiles / slots, rest = tiles % slots;
    double us = full * (steps * t.full + t.fixed);
    const double part = (double)rest / slots;
    if (rest) us += steps * (rest <= cus ? t.one + (t.full - t.one) * part * part : t.full) + t.fixed;
    return us;
}

struct Choice {
    int variant;
    int64_t slices, slice_k;
};

// few_rows: the layouts that launch_rows takes; slices: whether K may be cut.  A product of few tiles and a long K is cut where the partial sums' way through
// memory costs less than the idle compute units (48 x 11008 -> 4096: one slice 41 us, eight 17).
Choice choose(int64_t M, int64_t N, int64_t K, bool few_rows, bool a_by_k, bool may_slice)
{
    const int64_t cus = num_compute_units(), steps = ceil_div(K, half::kStepK);
    Choice best{MI8_HALF_64, 1, round_up(K, half::kStepK)};
    double least = 1e30;
    for (const TileCost& t : kTiles) {
        if (a_by_k && t.variant == MI8_HALF_192) continue;
        const int64_t tiles = t.tiles(M, N);
        for (int64_t s = 1; s <= 16; s *= 2) {
            const int64_t each = ceil_div(steps, s);
            if (s > 1 && (!may_slice || t.rows > 128 || each < 8 || (s - 1) * each >= steps)) break;
            const double us = rounds_us(t, tiles * s, each, cus) + (s > 1 ? 4.0 + 8.0 * s * M * N / 4e6 : 0.0);
            if (us < least) {
                least = us;
                best = Choice{t.variant, s, each * half::kStepK};
            }
        }
    }
    // (W at 4.2 TB/s and x out of the L2)
    if (few_rows && M <= half::kMostRows && 3.5 + 2.0 * N * K / 4.2e6 * (1.0 + 0.02 * M) < least) return Choice{MI8_HALF_ROWS, 1, 0};
    return best;
}

// Rows in groups whose sizes the host does not know: half a tile of every group is taken to be empty.  Of 40 products of 96 to 131072 rows in 8 to 64 groups of
// skewed sizes, six were 8 to 15 % off the best tile (us: 64 groups of 2048 -> 1024, 32000 rows 165, in 256 x 256 144; 8 of 512 -> 256, 8000 rows 8.4, in 64 x 64 7.3).
int choose_grouped(int64_t T, int64_t N, int64_t K, int64_t groups)
{
    const int64_t cus = num_compute_units(), used = groups < T ? groups : T;
    int best = MI8_HALF_64;
    double least = 1e30;
    for (int i = 0; i < kSquare; ++i) {
        const TileCost& t = kTiles[i];
        const double us = rounds_us(t, (ceil_div(T, t.rows) + used / 2) * ceil_div(N, t.cols), ceil_div(K, half::kStepK), cus);
        if (us < least) {
            least = us;
            best = t.variant;
        }
    }
    return best;
}

// K in groups: the chip's share of all steps, but no less than the longest group's, which is taken to have eight times its share of K, up to a half: routing
// is that uneven (64 experts' tokens by Zipf's law: 8).  us of 32 groups of 65536 rows, 512 x 1024: 256 x 256 275, 128 x 128 142, 64 x 64 207.
// Of 20 such products none was over 3 % off the best tile.  A tile walks all of its group's K, so a long group bounds the launch: those 142 us stand against 48 of
// operations, 58 us of 8 groups of 32768 rows, 256 x 512, against 10 of bytes.
int choose_wgrad(int64_t T, int64_t M, int64_t N, int64_t groups)
{
    const int64_t cus = num_compute_units(), longest = 8 * T / groups < T / 2 ? 8 * T / groups : T / 2;
    int best = MI8_HALF_64;
    double least = 1e30;
    for (int i = 0; i < kSquare; ++i) {
        const TileCost& t = kTiles[i];
        const double each = (double)t.tiles(M, N), steps = (double)T / half::kStepK + 0.5 * groups;
        double us = each * (steps * t.full + groups * t.fixed * 0.8) / (cus * t.per_cu);
        const double floor = ceil_div(longest, half::kStepK) * t.one + t.fixed;
        us = us < floor ? floor : us;
        if (us < least) {
            least = us;
            best = t.variant;
        }
    }
    return best;
}

// what every operand, pitch and size has to meet
int check(const char* what, int hp_dtype, const void* a, int64_t lda, const void* b, int64_t ldb, int64_t M, int64_t N, int64_t K, const void* out, int64_t ldc)
{
    MI8_REQUIRE(hp_dtype == MI8_BF16 || hp_dtype == MI8_F16, MI8_ERR_ARG, "%s: element type %d is neither bf16 nor float16", what, hp_dtype);
    MI8_REQUIRE(M >= 0 && N >= 0 && K >= 0, MI8_ERR_ARG, "%s: negative size", what);
    MI8_REQUIRE(M < (1 << 30) && N < (1 << 30) && K < (1 << 30), MI8_ERR_UNSUPPORTED, "%s: sizes up to 2^30", what);
    MI8_REQUIRE(M == 0 || N == 0 || (out && (K == 0 || (a && b))), MI8_ERR_ARG, "%s: null pointer", what);
    MI8_REQUIRE(aligned16(a) && aligned16(b), MI8_ERR_UNSUPPORTED, "%s: operands need 16-byte alignment", what);
    MI8_REQUIRE(lda % 8 == 0 && ldb % 8 == 0, MI8_ERR_UNSUPPORTED, "%s: operand pitches must be multiples of 8", what);
    MI8_REQUIRE(lda < (1 << 22) && ldb < (1 << 22) && ldc < (1 << 22), MI8_ERR_UNSUPPORTED, "%s: pitches up to 2^22 (32-bit offsets inside a tile)", what);
    MI8_REQUIRE(ldc >= N, MI8_ERR_ARG, "%s: the output's pitch is smaller than its rows", what);
    return MI8_OK;
}

bool takes16(const void* p, int64_t ld) { return p == nullptr || (aligned16(p) && ld % 8 == 0); }

}  // namespace

extern "C" int mi8_gemm_half(int hp_dtype, const void* a, int64_t lda, int a_by_k, const void* b, int64_t ldb, int b_by_k, int64_t M, int64_t N, int64_t K,
                             const mi8_half_epilogue* epilogue, void* out, int64_t ldc, int variant, void* workspace,
                             void* stream)
{
    const char* what = "mi8_gemm_half";
    if (int rc = check(what, hp_dtype, a, lda, b, ldb, M, N, K, out, ldc)) return rc;
    MI8_REQUIRE(!a_by_k || b_by_k, MI8_ERR_UNSUPPORTED, "%s: A by K goes with B by K", what);
    MI8_REQUIRE(lda >= round_up(a_by_k ? M : K, 8) && ldb >= round_up(b_by_k ? N : K, 8), MI8_ERR_ARG, "%s: a pitch is smaller than its rows", what);
    MI8_REQUIRE(variant >= MI8_HALF_ANY && variant <= MI8_HALF_192, MI8_ERR_ARG, "%s: unknown variant %d", what, variant);
    half::HalfArgs p{};
    p.A = static_cast<const uint8_t*>(a);
    p.B = static_cast<const uint8_t*>(b);
    p.C = static_cast<uint16_t*>(out);
    p.lda = lda;
    p.ldb = ldb;
    p.ldc = ldc;
    p.M = (int)M;
    p.N = (int)N;
    p.K = (int)K;
    p.wide = N % 8 == 0 && takes16(out, ldc);
    if (epilogue) {
        MI8_REQUIRE(epilogue->activation >= MI8_ACT_NONE && epilogue->activation <= MI8_ACT_GELU_TANH, MI8_ERR_ARG, "%s: unknown activation %d", what,
                    epilogue->activation);
        MI8_REQUIRE(epilogue->bias == nullptr || epilogue->bias_dtype == hp_dtype || epilogue->bias_dtype == MI8_F32, MI8_ERR_ARG,
                    "%s: the bias is float32 or of the operands' type", what);
        MI8_REQUIRE((epilogue->residual == nullptr || epilogue->ld_residual >= N) && (epilogue->z == nullptr || epilogue->ld_z >= N), MI8_ERR_ARG,
                    "%s: a pitch of the epilogue is smaller than its rows", what);
        p.bias = epilogue->bias;
        p.bias_f32 = epilogue->bias_dtype == MI8_F32;
        p.residual = static_cast<const uint16_t*>(epilogue->residual);
        p.ldr = epilogue->ld_residual;
        p.act = epilogue->activation;
        p.z = static_cast<uint16_t*>(epilogue->z);
        p.ldz = epilogue->ld_z;
        p.wide = p.wide && takes16(p.residual, p.ldr) && takes16(p.z, p.ldz) && p.ldz < (1 << 22);
    }
    if (M == 0 || N == 0) return MI8_OK;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const bool by_rows = !a_by_k && !b_by_k;
    Choice c{variant, 1, round_up(K, half::kStepK)};
    if (variant == MI8_HALF_ANY) c = choose(M, N, K, by_rows, a_by_k, workspace != nullptr);
    MI8_REQUIRE(c.variant != MI8_HALF_ROWS || (by_rows && M <= half::kMostRows), MI8_ERR_UNSUPPORTED, "%s: more than a few rows", what);
    MI8_REQUIRE(c.variant != MI8_HALF_192 || !a_by_k, MI8_ERR_UNSUPPORTED, "%s: tiles of 192 rows of A by K", what);
    if (c.variant == MI8_HALF_ROWS) return half::launch_rows(p, hp_dtype, st);
    p.slices = (int)c.slices;
    p.slice_k = (int)c.slice_k;
    if (c.slices == 1) return half::launch_tiles(p, hp_dtype, a_by_k, b_by_k, c.variant, st);
    half::HalfArgs slices = p;
    slices.partial = p.partial = static_cast<float*>(workspace);
    slices.ld_partial = p.ld_partial = round_up(N, 4);
    slices.wide = 0;
    if (int rc = half::launch_tiles(slices, hp_dtype, a_by_k, b_by_k, c.variant, st)) return rc;
    return half::launch_join(p, hp_dtype, st);
}

extern "C" int64_t mi8_gemm_half_workspace_bytes(int64_t M, int64_t N, int64_t K, int a_by_k, int b_by_k)
{
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    const Choice c = choose(M, N, K, !a_by_k && !b_by_k, a_by_k, true);
    return c.slices > 1 ? c.slices * M * round_up(N, 4) * 4 : 0;
}

extern "C" int mi8_gemm_half_variant(int64_t M, int64_t N, int64_t K, int a_by_k, int b_by_k, int32_t* slices)
{
    if (M <= 0 || N <= 0) return -1;
    const Choice c = choose(M, N, K, !a_by_k && !b_by_k, a_by_k, true);
    if (slices) *slices = (int32_t)c.slices;
    return c.variant;
}

extern "C" int mi8_grouped_gemm_half_variant(int64_t T, int64_t N, int64_t K, int32_t num_groups)
{
    return T <= 0 || N <= 0 || num_groups <= 0 ? -1 : choose_grouped(T, N, K, num_groups);
}

extern "C" int mi8_grouped_wgrad_half_variant(int64_t T, int64_t M, int64_t N, int32_t num_groups)
{
    return M <= 0 || N <= 0 || num_groups <= 0 ? -1 : choose_wgrad(T, M, N, num_groups);
}

extern "C" int mi8_grouped_gemm_half(int hp_dtype, const void* a, int64_t lda, const void* b, int64_t ldb, int b_by_k, int64_t b_group_stride,
                                     const int64_t* group_sizes, int32_t num_groups, int64_t T, int64_t N, int64_t K, void* out, int64_t ldc,
                                     int variant, void* stream)
{
    const char* what = "mi8_grouped_gemm_half";
    if (int rc = check(what, hp_dtype, a, lda, b, ldb, T, N, K, out, ldc)) return rc;
    MI8_REQUIRE(lda >= round_up(K, 8) && ldb >= round_up(b_by_k ? N : K, 8), MI8_ERR_ARG, "%s: a pitch is smaller than its rows", what);
    MI8_REQUIRE(group_sizes != nullptr && num_groups > 0, MI8_ERR_ARG, "%s: needs the sizes of at least one group", what);
    MI8_REQUIRE(b_group_stride >= 0 && b_group_stride % 8 == 0, MI8_ERR_UNSUPPORTED, "%s: the groups' matrices must start at multiples of 8 elements", what);
    MI8_REQUIRE(variant >= MI8_HALF_ANY && variant <= MI8_HALF_64, MI8_ERR_ARG, "%s: unknown variant %d", what, variant);
    MI8_REQUIRE((ceil_div(T, 64) + num_groups) * ceil_div(N, 64) < (int64_t)1 << 31, MI8_ERR_UNSUPPORTED, "%s: too many tiles", what);
    if (T == 0 || N == 0) return MI8_OK;
    half::HalfArgs p{};
    p.A = static_cast<const uint8_t*>(a);
    p.B = static_cast<const uint8_t*>(b);
    p.C = static_cast<uint16_t*>(out);
    p.lda = lda;
    p.ldb = ldb;
    p.ldc = ldc;
    p.M = (int)T;
    p.N = (int)N;
    p.K = (int)K;
    p.slices = 1;
    p.sizes = group_sizes;
    p.E = num_groups;
    p.b_group_stride = b_group_stride;
    p.wide = N % 8 == 0 && takes16(out, ldc);
    if (variant == MI8_HALF_ANY) variant = choose_grouped(T, N, K, num_groups);
    return half::launch_tiles(p, hp_dtype, false, b_by_k, variant, static_cast<hipStream_t>(stream));
}

extern "C" int mi8_grouped_wgrad_half(int hp_dtype, const void* a, int64_t lda, const void* b, int64_t ldb, const int64_t* group_sizes, int32_t num_groups,
                                      int64_t T, int64_t M, int64_t N, void* out, int variant, void* stream)
{
    const char* what = "mi8_grouped_wgrad_half";
    if (int rc = check(what, hp_dtype, a, lda, b, ldb, M, N, T, out, N)) return rc;
    MI8_REQUIRE(lda >= round_up(M, 8) && ldb >= round_up(N, 8), MI8_ERR_ARG, "%s: a pitch is smaller than its rows", what);
    MI8_REQUIRE(group_sizes != nullptr && num_groups > 0, MI8_ERR_ARG, "%s: needs the sizes of at least one group", what);
    MI8_REQUIRE(variant >= MI8_HALF_ANY && variant <= MI8_HALF_64, MI8_ERR_ARG, "%s: unknown variant %d", what, variant);
    MI8_REQUIRE((num_groups + 7) * ceil_div(M, 64) * ceil_div(N, 64) < (int64_t)1 << 31, MI8_ERR_UNSUPPORTED, "%s: too many tiles", what);
    if (M == 0 || N == 0) return MI8_OK;
    half::HalfArgs p{};
    p.A = static_cast<const uint8_t*>(a);
    p.B = static_cast<const uint8_t*>(b);
    p.C = static_cast<uint16_t*>(out);
    p.lda = lda;
    p.ldb = ldb;
    p.ldc = N;
    p.M = (int)M;
    p.N = (int)N;
    p.K = (int)T;
    p.slices = 1;
    p.sizes = group_sizes;
    p.E = num_groups;
    p.wide = N % 8 == 0 && takes16(out, N);
    if (variant == MI8_HALF_ANY) variant = choose_wgrad(T, M, N, num_groups);
    return half::launch_tiles(p, hp_dtype, true, true, variant, static_cast<hipStream_t>(stream));
}
