// Microscaled 4-bit floating point: the element and scale types shared by the quantiser (fp4.cu) and the
// block-scaled tensor-core product (fp4_umma.cu).
//
//   element  E2M1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign; two a byte, the even element in the low nibble
//   mxfp4    32 elements of a row share 2^(byte - 127) (E8M0; 255 is NaN)
//   nvfp4    16 elements share an E4M3 scale (0x7f is NaN), the row an fp32 factor
//
// Scales lie in tiles of 512 bytes, 128 rows x 4 blocks: byte (row % 32) * 16 + row % 128 / 32 * 4 + block % 4 of tile
// [row / 128][block / 4].  That is the order in which a tile goes to tensor memory as one 32 x 128-bit copy, so a weight
// keeps no second copy of its scales.  Rows and blocks that pad a tile hold zero bytes.
#pragma once

#include "common.cuh"

namespace rwkv7 {
namespace fp4 {
constexpr int MX = 0, NV = 1;  // RWKV7_FP4_MX, RWKV7_FP4_NV
constexpr int SCALE_TILE_ROWS = 128, SCALE_TILE_BLOCKS = 4, SCALE_TILE_BYTES = 512;

__host__ __device__ constexpr int block_of(int format) { return format == MX ? 32 : 16; }
// tiles along K
__host__ __device__ constexpr int k_tiles(int K, int format) { return (K / block_of(format) + SCALE_TILE_BLOCKS - 1) / SCALE_TILE_BLOCKS; }
__host__ __device__ constexpr int64_t scale_bytes(int64_t rows, int K, int format) {
    return (rows + SCALE_TILE_ROWS - 1) / SCALE_TILE_ROWS * k_tiles(K, format) * SCALE_TILE_BYTES;
}
// byte offset of the four scales of blocks 4t .. 4t + 3 of `row`
__host__ __device__ constexpr int64_t scale_word(int64_t row, int t, int ktiles) {
    return (row / 128 * ktiles + t) * SCALE_TILE_BYTES + row % 32 * 16 + row % 128 / 32 * 4;
}
}  // namespace fp4

// rows to codes, scale tiles and (nvfp4) row scales; sizes and pointers already checked
int launch_fp4_quant(const void* x, int64_t ldx, uint8_t* packed, uint8_t* scales, float* row_scale, int rows, int K, int format,
                     int dtype, cudaStream_t st);
}  // namespace rwkv7
