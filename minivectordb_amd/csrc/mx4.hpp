// mx4.hpp -- microscaled 4-bit rows: the format, and the launches that mx4.hip offers to the C ABI (engine.hip).
//
// A row of `dim` components is cut into blocks of 32.  A block is a scale 2^(s - 127), one byte s (255 = not a number), and 32
// codes of 4 bits {sign, two bits of exponent, one of mantissa}: +-{0, 0.5, 1, 1.5, 2, 3, 4, 6}.  With m the largest magnitude
// of the block s - 127 = floor(log2 m) - 2, not below -127, and a code is x / 2^(s - 127) rounded to the nearest magnitude
// (ties to the even code), at most 6: m / 2^(s - 127) lies in [4, 8), so only what is above 6 loses more than a rounding.
// A block that holds a NaN or an infinity has s = 255 and zero codes: every product with it is NaN.
//
// Packed row, mx4_row_bytes(dim) bytes, 16-byte aligned:
//   nb x 16 bytes of codes (component 2 i of a block in the low half of its byte i), nb = 2 * ceil(dim / 64) blocks,
//   nb scale bytes, zeros up to a multiple of 16.
// Components past `dim` have code 0, blocks past it also scale byte 0: they add nothing to a product.  The number of blocks is
// even because one matrix instruction takes 64 components (two blocks); codes and scales of a row are kept together so
// that a row is one run of memory, 272 bytes at dim 512 (4.25 bits a component).
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace mvdb {

constexpr int kMx4MaxDim = 4096;      // quantise, expand, product
constexpr int kMx4ScanMaxDim = 1024;  // scan (as the traversal)
constexpr int kMx4ScanMaxK = 128;

__host__ __device__ constexpr int mx4_blocks(int dim) { return 2 * ((dim + 63) / 64); }
__host__ __device__ constexpr int mx4_row_bytes(int dim) { return 16 * mx4_blocks(dim) + (mx4_blocks(dim) + 15) / 16 * 16; }

// dtype of the rows that are quantised: 0 f32, 1 bf16, 2 f16; ld = components from one row to the next
hipError_t mx4_launch_quantize(const void *x, int dtype, int64_t rows, int dim, int64_t ld, uint8_t *packed, hipStream_t s);
hipError_t mx4_launch_expand(const uint8_t *packed, int64_t rows, int dim, float *values, hipStream_t s);
// out[q][r], ldo floats from one query to the next
hipError_t mx4_launch_product(const uint8_t *q, int nq, const uint8_t *rows, int n, int dim, float *out, int64_t ldo, hipStream_t s);
size_t mx4_scan_workspace(int nq, int n, int dim, int k);
// ws: mx4_scan_workspace bytes, 16-byte aligned, used by this call until it has run on the stream
hipError_t mx4_launch_scan(const uint8_t *q, int nq, const uint8_t *rows, int n, int dim, int k, const uint32_t *allow, int32_t *out_ids,
                           float *out_val, int32_t *out_count, void *ws, hipStream_t s);

}  // namespace mvdb
