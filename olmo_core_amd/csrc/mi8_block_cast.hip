// Casts to float8 with block scales (mi8_block.h): one scale per 128 elements of a row (activations, gradients) for a copy that
// is contracted along its rows, one per 128 elements of a column for a transposed copy that is contracted along the tokens, or
// one per 128 x 128 for both copies (weights).
//
// All maxima of a 128 x 128 tile are inside it, so a workgroup reads its tile once, keeps it in registers (64 values a thread,
// eight rows by eight columns) and writes both copies: the casts are bound by 4 bytes of memory traffic an element (2 in, 1 + 1
// out), where scales over whole rows and columns take a pass for the maxima first.
#include "mi8_block.h"
#include "mi8_groups.h"

namespace mi8 {
namespace {

using namespace block;

struct BlockCastArgs {
    const void* x;       // [batch * rows, cols], contiguous
    int64_t rows, cols;  // of one matrix
    uint8_t* out;        // null, or [batch * rows, ld_out]
    int64_t ld_out;
    uint8_t* e_out;      // [batch][cols blocks][padded rows]
    uint8_t* out_t;      // null, or [batch][cols, ld_t]
    int64_t ld_t;
    uint8_t* e_out_t;    // [batch][row blocks][padded cols]
    int tiles_c;
    // (grouped) rows are groups of consecutive rows; the transposed copy and all scales live on an axis on which every group
    // starts at a multiple of 128
    const int64_t* sizes;
    int groups;
    int64_t axis;  // length of that axis
};

typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pk_umax(uint32_t a, uint32_t b)
{
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, a), __builtin_bit_cast(u16x2_t, b)));
}

// A thread's eight rows by eight columns as they are in memory, and maxima of their magnitudes: words of one float32 pattern, or of two
// bf16 patterns (columns 2 c and 2 c + 1), which take the same comparisons.
template <int HP>
struct Patch;
template <>
struct Patch<MI8_BF16> {
    static constexpr int kWords = 4;  // of eight columns
    uint32_t w[8][4];
    __device__ __forceinline__ void load(int i, const uint8_t* p, bool ok)
    {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (ok) v = load_stream16(p);
        w[i][0] = v.x, w[i][1] = v.y, w[i][2] = v.z, w[i][3] = v.w;
    }
    __device__ __forceinline__ uint32_t magnitude(int i, int c) const { return w[i][c] & 0x7FFF7FFFu; }
    __device__ static __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return pk_umax(a, b); }
    __device__ static __forceinline__ uint32_t widest(uint32_t m) { return umax32(m << 16, m & 0xFFFF0000u); }  // as float32 bits
    __device__ static __forceinline__ uint32_t column(const uint32_t* m, int j) { return j & 1 ? m[j / 2] & 0xFFFF0000u : m[j / 2] << 16; }
    __device__ __forceinline__ float at(int i, int j) const { return bits_to_f32(j & 1 ? w[i][j / 2] & 0xFFFF0000u : w[i][j / 2] << 16); }
};
template <>
struct Patch<MI8_F32> {
    static constexpr int kWords = 8;
    uint32_t w[8][8];
    __device__ __forceinline__ void load(int i, const uint8_t* p, bool ok)
    {
        uint4 u = make_uint4(0, 0, 0, 0), v = u;
        if (ok) {
            u = load_stream16(p);
            v = load_stream16(p + 16);
        }
        w[i][0] = u.x, w[i][1] = u.y, w[i][2] = u.z, w[i][3] = u.w;
        w[i][4] = v.x, w[i][5] = v.y, w[i][6] = v.z, w[i][7] = v.w;
    }
    __device__ __forceinline__ uint32_t magnitude(int i, int c) const { return w[i][c] & 0x7FFFFFFFu; }
    __device__ static __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return umax32(a, b); }
    __device__ static __forceinline__ uint32_t widest(uint32_t m) { return m; }
    __device__ static __forceinline__ uint32_t column(const uint32_t* m, int j) { return m[j]; }
    __device__ __forceinline__ float at(int i, int j) const { return bits_to_f32(w[i][j]); }
};

template <int HP, int CTRL>
__device__ __forceinline__ uint32_t larger_dpp(uint32_t v) { return Patch<HP>::larger(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true)); }
template <int HP>
__device__ __forceinline__ uint32_t max_over16(uint32_t v)  // of 16 lanes, in all of them
{
    v = larger_dpp<HP, 0xB1>(v);   // quad_perm [1,0,3,2]
    v = larger_dpp<HP, 0x4E>(v);   // quad_perm [2,3,0,1]
    v = larger_dpp<HP, 0x141>(v);  // row_half_mirror
    return larger_dpp<HP, 0x140>(v);  // row_mirror
}
template <int HP>
__device__ __forceinline__ uint32_t max_over_rows(uint32_t v)  // of the lanes 16 and 32 apart
{
    auto pair = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = Patch<HP>::larger(pair[0], pair[1]);
    pair = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return Patch<HP>::larger(pair[0], pair[1]);
}

template <int HP>
struct CastLds {
    __attribute__((aligned(16))) uint8_t flip[128 * 128];
    uint32_t maxima[4][16 * Patch<HP>::kWords];
    __attribute__((aligned(16))) uint8_t bytes[2][128];
};

// One tile: the block-th of a matrix.  SQUARE: one scale per tile.  GROUPED: see BlockCastArgs.
template <int HP, bool SQUARE, bool GROUPED>
__device__ __forceinline__ void cast_tile(const BlockCastArgs& a, const int64_t block, const int64_t matrix, CastLds<HP>& lds)
{
    typedef Patch<HP> P;
    uint8_t* const flip = lds.flip;
    auto& maxima = lds.maxima;
    auto& bytes = lds.bytes;
    const int tid = threadIdx.x;
    const int cg = tid & 15, rg = tid >> 4;  // columns 8 cg .., rows 8 rg ..
    const int wave = tid >> 6;
    const int tc = (int)(block % a.tiles_c);
    const int64_t tr = block / a.tiles_c;  // tile of rows (of the padded axis)

    int64_t row0, row_first, rows_here, e_pitch, e_tile;
    if constexpr (GROUPED) {
        const gemm::GroupSpan s = gemm::locate_group<128, true>(a.sizes, a.groups, a.rows, tr);
        if (s.e >= a.groups) return;
        const int64_t inside = (tr - s.units_before) * 128;
        row0 = row_first = s.rows_before + inside;
        rows_here = s.m - inside;
        e_pitch = a.axis;
        e_tile = tr;
    } else {
        row0 = tr * 128;
        row_first = matrix * a.rows + row0;
        rows_here = a.rows - row0;
        e_pitch = padded(a.rows);
        e_tile = tr;
    }
    if (rows_here > 128) rows_here = 128;
    const int64_t col = (int64_t)tc * 128 + 8 * cg;
    const bool col_ok = col < a.cols;

    P x;
    const uint8_t* src = reinterpret_cast<const uint8_t*>(a.x) + ((row_first + 8 * rg) * a.cols + col) * HpVec<HP>::kBytes;
#pragma unroll
    for (int i = 0; i < 8; ++i) x.load(i, src + i * a.cols * HpVec<HP>::kBytes, col_ok && 8 * rg + i < rows_here);

    uint32_t row_max[8], col_max[P::kWords];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        row_max[i] = x.magnitude(i, 0);
#pragma unroll
        for (int c = 1; c < P::kWords; ++c) row_max[i] = P::larger(row_max[i], x.magnitude(i, c));
    }
    if constexpr (SQUARE) {
        uint32_t m = row_max[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) m = P::larger(m, row_max[i]);
        m = max_over_rows<HP>(max_over16<HP>(m));
        if ((tid & 63) == 0) maxima[wave][0] = m;
        __syncthreads();
        m = P::widest(P::larger(P::larger(maxima[0][0], maxima[1][0]), P::larger(maxima[2][0], maxima[3][0])));
#pragma unroll
        for (int i = 0; i < 8; ++i) row_max[i] = m;
    } else {
        if (a.out_t) {  // (uniform)
#pragma unroll
            for (int c = 0; c < P::kWords; ++c) {
                uint32_t m = x.magnitude(0, c);
#pragma unroll
                for (int i = 1; i < 8; ++i) m = P::larger(m, x.magnitude(i, c));
                col_max[c] = max_over_rows<HP>(m);
            }
            if ((tid & 63) < 16) {
#pragma unroll
                for (int c = 0; c < P::kWords; ++c) maxima[wave][P::kWords * cg + c] = col_max[c];
            }
            __syncthreads();
#pragma unroll
            for (int c = 0; c < P::kWords; ++c) {
                const int at = P::kWords * cg + c;
                col_max[c] = P::larger(P::larger(maxima[0][at], maxima[1][at]), P::larger(maxima[2][at], maxima[3][at]));
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) row_max[i] = P::widest(max_over16<HP>(row_max[i]));
    }

    if (a.out) {  // (uniform)
        uint8_t* dst = a.out + (row_first + 8 * rg) * a.ld_out + col;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float s;
            uint8_t byte;
            scale_of(row_max[i], s, byte);
            const uint32_t lo = cvt4<MI8_E4M3, false>(x.at(i, 0) * s, x.at(i, 1) * s, x.at(i, 2) * s, x.at(i, 3) * s);
            const uint32_t hi = cvt4<MI8_E4M3, false>(x.at(i, 4) * s, x.at(i, 5) * s, x.at(i, 6) * s, x.at(i, 7) * s);
            if (8 * rg + i < rows_here) *reinterpret_cast<uint2*>(dst + i * a.ld_out) = make_uint2(lo, hi);
            if (cg == 0) bytes[0][scale_at(8 * rg + i)] = byte;
        }
    }
    if (a.out_t) {
        float s[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            uint8_t byte;
            scale_of(SQUARE ? row_max[0] : P::column(col_max, j), s[j], byte);
            if (rg == 0) bytes[1][scale_at(8 * cg + j)] = byte;
        }
        // column c of the tile becomes 128 bytes of LDS, their 8-byte pieces XORed with c / 8 (the 16 lanes of a piece are 1024 bytes apart)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t lo = cvt4<MI8_E4M3, false>(x.at(0, j) * s[j], x.at(1, j) * s[j], x.at(2, j) * s[j], x.at(3, j) * s[j]);
            const uint32_t hi = cvt4<MI8_E4M3, false>(x.at(4, j) * s[j], x.at(5, j) * s[j], x.at(6, j) * s[j], x.at(7, j) * s[j]);
            *reinterpret_cast<uint2*>(flip + (8 * cg + j) * 128 + ((rg ^ cg) << 3)) = make_uint2(lo, hi);
        }
    }
    __syncthreads();
    if (a.out_t) {
        const int p = tid & 7;
        uint8_t* dst = a.out_t + (matrix * a.cols + (int64_t)tc * 128) * a.ld_t + tr * 128 + 16 * p;
#pragma unroll
        for (int it = 0; it < 4; ++it) {
            const int c = it * 32 + (tid >> 3), turn = c >> 3;
            uint4 v = *reinterpret_cast<const uint4*>(flip + c * 128 + (((2 * p) ^ (turn & ~1)) << 3));
            if (turn & 1) v = make_uint4(v.z, v.w, v.x, v.y);
            if ((int64_t)tc * 128 + c < a.cols) *reinterpret_cast<uint4*>(dst + (int64_t)c * a.ld_t) = v;
        }
    }
    if (tid < 32 && a.out) {
        const int64_t blocks = a.tiles_c;
        uint8_t* e = a.e_out + (matrix * blocks + tc) * e_pitch + e_tile * 128;
        reinterpret_cast<uint32_t*>(e)[tid] = reinterpret_cast<const uint32_t*>(bytes[0])[tid];
    } else if (tid >= 32 && tid < 64 && a.out_t) {
        const int64_t blocks = GROUPED ? a.axis / 128 : e_pitch / 128;
        uint8_t* e = a.e_out_t + (matrix * blocks + tr) * padded(a.cols) + (int64_t)tc * 128;
        reinterpret_cast<uint32_t*>(e)[tid - 32] = reinterpret_cast<const uint32_t*>(bytes[1])[tid - 32];
    }
}

template <int HP, bool SQUARE, bool GROUPED>
__global__ __launch_bounds__(256) void block_cast_kernel(BlockCastArgs a)
{
    __shared__ CastLds<HP> lds;
    cast_tile<HP, SQUARE, GROUPED>(a, blockIdx.x, blockIdx.y, lds);
}

// Several casts in one launch: those of a layer of ordinary size take as long to start as to run.  Rows of 1999 x 1024 and a weight of
// 2816 x 1024, bf16, both copies: 11.2 us one by one, 7.7 together.
struct BlockCastBatch {
    BlockCastArgs item[MI8_BLOCK_CAST_BATCH];
    int square[MI8_BLOCK_CAST_BATCH];
    uint32_t tiles[MI8_BLOCK_CAST_BATCH];      // of a matrix
    uint32_t first[MI8_BLOCK_CAST_BATCH];      // first workgroup of an item
    int count;
};

template <int HP>
__global__ __launch_bounds__(256) void block_cast_batch_kernel(BlockCastBatch p)
{
    __shared__ CastLds<HP> lds;
    int i = 0;
#pragma unroll
    for (int j = 1; j < MI8_BLOCK_CAST_BATCH; ++j)
        if (j < p.count && blockIdx.x >= p.first[j]) i = j;
    const uint32_t b = blockIdx.x - p.first[i];
    const BlockCastArgs& a = p.item[i];
    if (a.sizes)
        cast_tile<HP, false, true>(a, b, 0, lds);
    else if (p.square[i])
        cast_tile<HP, true, false>(a, b % p.tiles[i], b / p.tiles[i], lds);
    else
        cast_tile<HP, false, false>(a, b % p.tiles[i], b / p.tiles[i], lds);
}

template <bool SQUARE, bool GROUPED>
int launch_cast(const BlockCastArgs& a, int hp_dtype, int64_t tiles_r, int64_t batch, hipStream_t st, const char* what)
{
    MI8_REQUIRE(tiles_r * a.tiles_c < ((int64_t)1 << 31) && batch < 65536, MI8_ERR_UNSUPPORTED, "%s: grid too large", what);
    const dim3 grid((unsigned)(tiles_r * a.tiles_c), (unsigned)batch);
    if (hp_dtype == MI8_BF16)
        hipLaunchKernelGGL((block_cast_kernel<MI8_BF16, SQUARE, GROUPED>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((block_cast_kernel<MI8_F32, SQUARE, GROUPED>), grid, dim3(256), 0, st, a);
    return launch_status(what);
}

// what both entry points ask of their outputs
int check_outputs(const BlockCastArgs& a, int hp_dtype, int64_t token_axis, const char* what)
{
    MI8_REQUIRE(a.x && (a.out || a.out_t), MI8_ERR_ARG, "%s: null pointer", what);
    MI8_REQUIRE(hp_dtype == MI8_BF16 || hp_dtype == MI8_F32, MI8_ERR_ARG, "%s: input must be bf16 or float32", what);
    MI8_REQUIRE(a.rows > 0 && a.cols > 0, MI8_ERR_ARG, "%s: empty tensor", what);
    MI8_REQUIRE(a.cols % 16 == 0 && aligned16(a.x), MI8_ERR_UNSUPPORTED, "%s: needs cols %% 16 == 0 and 16-byte alignment", what);
    MI8_REQUIRE(a.rows < ((int64_t)1 << 31) - 128 && a.cols < ((int64_t)1 << 31) - 128, MI8_ERR_UNSUPPORTED, "%s: tensor too large", what);
    MI8_REQUIRE(!a.out || (a.e_out && aligned16(a.out) && aligned16(a.e_out) && a.ld_out % 16 == 0 && a.ld_out >= padded(a.cols)), MI8_ERR_UNSUPPORTED,
                "%s: rows of the copy need their scales, 16-byte alignment and round_up(cols, 128) bytes", what);
    MI8_REQUIRE(!a.out_t || (a.e_out_t && aligned16(a.out_t) && aligned16(a.e_out_t) && a.ld_t % 16 == 0 && a.ld_t >= token_axis), MI8_ERR_UNSUPPORTED,
                "%s: rows of the transposed copy need their scales, 16-byte alignment and %lld bytes", what, (long long)token_axis);
    return MI8_OK;
}

BlockCastArgs cast_args(const mi8_block_cast_item& t)
{
    return BlockCastArgs{t.x, t.rows, t.cols, (uint8_t*)t.out, t.ld_out, (uint8_t*)t.scales, (uint8_t*)t.out_t, t.ld_t, (uint8_t*)t.scales_t,
                         (int)ceil_div(t.cols, 128), t.group_sizes, t.num_groups, t.group_sizes && t.rows > 0 ? mi8_grouped_padded_rows(t.rows, t.num_groups) : 0};
}

}  // namespace
}  // namespace mi8

using namespace mi8;

extern "C" int64_t mi8_block_scale_bytes(int64_t rows, int64_t K)
{
    return rows > 0 && K > 0 ? block::padded(rows) * ceil_div(K, 128) : 0;
}

extern "C" int mi8_cast_block(const void* x, int hp_dtype, int64_t rows, int64_t cols, int32_t matrices, int32_t square, void* out,
                              int64_t ld_out, void* scales, void* out_t, int64_t ld_t, void* scales_t, void* stream)
{
    MI8_REQUIRE(matrices > 0, MI8_ERR_ARG, "mi8_cast_block: no matrices");
    BlockCastArgs a{x, rows, cols, (uint8_t*)out, ld_out, (uint8_t*)scales, (uint8_t*)out_t, ld_t, (uint8_t*)scales_t, (int)ceil_div(cols, 128),
                    nullptr, 0, 0};
    if (int rc = check_outputs(a, hp_dtype, block::padded(rows), "mi8_cast_block")) return rc;
    const int64_t tiles_r = ceil_div(rows, 128);
    return square ? launch_cast<true, false>(a, hp_dtype, tiles_r, matrices, (hipStream_t)stream, "mi8_cast_block")
                  : launch_cast<false, false>(a, hp_dtype, tiles_r, matrices, (hipStream_t)stream, "mi8_cast_block");
}

extern "C" int mi8_grouped_cast_block(const void* x, int hp_dtype, int64_t T, int64_t cols, const int64_t* group_sizes, int32_t num_groups,
                                      void* out, int64_t ld_out, void* scales, void* out_t, int64_t ld_t, void* scales_t, void* stream)
{
    MI8_REQUIRE(group_sizes && num_groups > 0, MI8_ERR_ARG, "mi8_grouped_cast_block: no groups");
    const int64_t axis = T > 0 ? mi8_grouped_padded_rows(T, num_groups) : 0;
    BlockCastArgs a{x, T, cols, (uint8_t*)out, ld_out, (uint8_t*)scales, (uint8_t*)out_t, ld_t, (uint8_t*)scales_t, (int)ceil_div(cols, 128),
                    group_sizes, num_groups, axis};
    if (int rc = check_outputs(a, hp_dtype, axis, "mi8_grouped_cast_block")) return rc;
    return launch_cast<false, true>(a, hp_dtype, axis / 128, 1, (hipStream_t)stream, "mi8_grouped_cast_block");
}

extern "C" int mi8_cast_block_batch(const mi8_block_cast_item* items, int32_t count, void* stream)
{
    MI8_REQUIRE(items && count > 0 && count <= MI8_BLOCK_CAST_BATCH, MI8_ERR_ARG, "mi8_cast_block_batch: 1 to %d items", MI8_BLOCK_CAST_BATCH);
    BlockCastBatch p{};
    p.count = count;
    int64_t blocks = 0;
    for (int i = 0; i < count; ++i) {
        const mi8_block_cast_item& t = items[i];
        MI8_REQUIRE(t.matrices > 0 && t.num_groups >= 0 && (t.num_groups > 0) == (t.group_sizes != nullptr) && !(t.group_sizes && (t.square || t.matrices != 1)),
                    MI8_ERR_ARG, "mi8_cast_block_batch: groups of rows are one matrix without square blocks");
        MI8_REQUIRE(t.hp_dtype == items[0].hp_dtype, MI8_ERR_UNSUPPORTED, "mi8_cast_block_batch: items of one type");
        p.item[i] = cast_args(t);
        const int64_t axis = t.group_sizes ? p.item[i].axis : block::padded(t.rows);
        if (int rc = check_outputs(p.item[i], t.hp_dtype, axis, "mi8_cast_block_batch")) return rc;
        p.square[i] = t.square;
        const int64_t tiles = axis / 128 * p.item[i].tiles_c;
        MI8_REQUIRE(tiles < ((int64_t)1 << 31) && blocks + tiles * t.matrices < ((int64_t)1 << 31), MI8_ERR_UNSUPPORTED, "mi8_cast_block_batch: grid too large");
        p.tiles[i] = (uint32_t)tiles;
        p.first[i] = (uint32_t)blocks;
        blocks += tiles * t.matrices;
    }
    hipStream_t st = (hipStream_t)stream;
    if (items[0].hp_dtype == MI8_BF16)
        hipLaunchKernelGGL((block_cast_batch_kernel<MI8_BF16>), dim3((unsigned)blocks), dim3(256), 0, st, p);
    else
        hipLaunchKernelGGL((block_cast_batch_kernel<MI8_F32>), dim3((unsigned)blocks), dim3(256), 0, st, p);
    return launch_status("mi8_cast_block_batch");
}
