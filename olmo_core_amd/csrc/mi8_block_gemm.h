// Products with block scales: the argument block that the kernels of mi8_block_gemm.hip and mi8_block_persistent.hip share.
#pragma once
#include "mi8_block.h"

namespace mi8 {
namespace block {

struct BlockArgs {
    const uint8_t* A;
    const uint8_t* B;
    const uint8_t* ea;
    const uint8_t* eb;
    void* C;
    int64_t lda, ldb, ldc;
    int M, N, nk;  // (groups of rows: M is the number of rows of all of them)
    int c_f32;
    int tiles_m, tiles_n;
    // groups: rows of A, or blocks of K, in consecutive groups whose sizes are on the device; their scales (and blocks of K) lie on
    // an axis of `axis` rows on which every group starts at a multiple of 128
    const int64_t* sizes;
    int E;
    int64_t b_group_stride, eb_group_stride, axis;
    int64_t tokens;  // (groups of blocks of K) rows of all groups
};

// Persistent kernel with 256 x 256 tiles (mi8_block_persistent.hip): bf16 output, operand pitches below 2^23, output pitch below 2^22
int launch_persistent(BlockArgs& p, hipStream_t st);
int launch_persistent_grouped(BlockArgs& p, hipStream_t st);
int launch_persistent_wgrad(BlockArgs& p, hipStream_t st);

}  // namespace block
}  // namespace mi8
