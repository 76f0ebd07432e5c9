// mx4_rows.hip.hpp -- rows -> packed 4-bit rows and back (format: mx4.hpp).
#pragma once

#include <hip/hip_runtime.h>

#include "mx4.hpp"

namespace mvdb {

// Eight components at any byte alignment: the hardware takes unaligned global accesses, so rows of any stride go the same way.
struct __attribute__((packed, aligned(2))) Mx4Half8 {
	uint16_t v[8];
};
struct __attribute__((packed, aligned(4))) Mx4Float8 {
	float v[8];
};
struct __attribute__((packed, aligned(4))) Mx4Float4 {
	float v[4];
};

// the eight components [col, col + 8) of a row as f32; those at or past dim are 0
template <int DTYPE>
__device__ __forceinline__ void mx4_load8(const void *x, int64_t at, int col, int dim, float (&f)[8])
{
	if constexpr (DTYPE == 0) {
		const float *p = static_cast<const float *>(x) + at;
		if (col + 8 <= dim) {
			const Mx4Float8 t = *reinterpret_cast<const Mx4Float8 *>(p);
#pragma unroll
			for (int i = 0; i < 8; i++) f[i] = t.v[i];
		} else {
#pragma unroll
			for (int i = 0; i < 8; i++) f[i] = col + i < dim ? p[i] : 0.f;
		}
	} else {
		const uint16_t *p = static_cast<const uint16_t *>(x) + at;
		uint16_t h[8];
		if (col + 8 <= dim) {
			const Mx4Half8 t = *reinterpret_cast<const Mx4Half8 *>(p);
#pragma unroll
			for (int i = 0; i < 8; i++) h[i] = t.v[i];
		} else {
#pragma unroll
			for (int i = 0; i < 8; i++) h[i] = col + i < dim ? p[i] : (uint16_t)0;
		}
#pragma unroll
		for (int i = 0; i < 8; i++) {
			if constexpr (DTYPE == 1)
				f[i] = __uint_as_float((unsigned)h[i] << 16);
			else
				f[i] = (float)__builtin_bit_cast(_Float16, h[i]);
		}
	}
}

// One thread per 8 components (4 bytes of codes), four threads a block, eight a pair of blocks; `per_row` = 4 nb threads a row, so a
// pair never crosses a row.  The largest magnitude is taken over the bit patterns: for |x| they are ordered as the values
// are, and a NaN or an infinity is at least 0x7f800000.  Bound by memory: 1 M x 384 f32 in 340 us, 5.1 TB/s read and written.
template <int DTYPE>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const void *x, int64_t rows, int dim, int64_t ld, int nb, int row_bytes, uint8_t *packed)
{
	const int per_row = 4 * nb;
	const int64_t first = (int64_t)blockIdx.x * 256;
	const int64_t row0 = first / per_row;
	const int u = (int)(first - row0 * per_row) + (int)threadIdx.x;  // < per_row + 256
	const int dr = u / per_row, part = u - dr * per_row;
	const int64_t row = row0 + dr;
	if (row >= rows) return;  // (whole rows: the eight lanes of a pair leave together)
	const int col = part * 8;
	float f[8];
	mx4_load8<DTYPE>(x, row * ld + col, col, dim, f);
	unsigned top = 0;
#pragma unroll
	for (int i = 0; i < 8; i++) {
		const unsigned b = __float_as_uint(f[i]) & 0x7fffffffu;
		top = b > top ? b : top;
	}
#pragma unroll
	for (int d = 1; d <= 2; d <<= 1) {
		const unsigned o = (unsigned)__shfl_xor((int)top, d, 64);
		top = o > top ? o : top;
	}
	const int e = (int)(top >> 23);
	const bool bad = e == 255;
	const int s = bad ? 255 : (e > 2 ? e - 2 : 0);
	// 2^(s - 127) as a float: s = 0 is the subnormal 2^-127
	const float scale = __uint_as_float(s > 0 ? (unsigned)s << 23 : 0x00400000u);
	unsigned codes = 0;
	// v_cvt_scalef32_pk_fp4_f32 rounds x / scale to nearest, ties to even, and saturates at 6
	codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[0], f[1], scale, 0);
	codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[2], f[3], scale, 1);
	codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[4], f[5], scale, 2);
	codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, f[6], f[7], scale, 3);
	uint8_t *out = packed + row * row_bytes;
	*reinterpret_cast<unsigned *>(out + part * 4) = bad ? 0u : codes;
	const int other = __shfl_xor(s, 4, 64);  // the scale of the pair's other block
	uint8_t *tail = out + 16 * nb;
	if ((part & 7) == 0) *reinterpret_cast<uint16_t *>(tail + (part >> 2)) = (uint16_t)(s | (other << 8));
	const int pad = row_bytes - 17 * nb;  // even, at most 14
	if (2 * part < pad) *reinterpret_cast<uint16_t *>(tail + nb + 2 * part) = 0;
}

// One thread per 4 components, kMx4ExpandRun times 256 threads apart: a store writes 16 neighbouring bytes a lane, 1 KB a wave (8 components a
// thread, two stores of 16 bytes 32 apart: 568 us instead of 300 for 1 M x 384).  Bound by the writing of the values, 5.8 TB/s.
constexpr int kMx4ExpandRun = 4;

__global__ __launch_bounds__(256) void mx4_expand_kernel(const uint8_t *packed, int64_t rows, int dim, int nb, int row_bytes, float *values)
{
	const int per_row = (dim + 3) / 4;
	const int64_t first = (int64_t)blockIdx.x * (256 * kMx4ExpandRun);
	const int64_t row0 = first / per_row;
	const int u0 = (int)(first - row0 * per_row) + (int)threadIdx.x;
	unsigned codes[kMx4ExpandRun];
	int s[kMx4ExpandRun];
	int64_t at[kMx4ExpandRun];
	int left[kMx4ExpandRun];
#pragma unroll
	for (int j = 0; j < kMx4ExpandRun; j++) {
		const int u = u0 + 256 * j, dr = u / per_row, part = u - dr * per_row;
		const int64_t row = row0 + dr;
		left[j] = row < rows ? dim - part * 4 : 0;
		const uint8_t *in = packed + (row < rows ? row : 0) * row_bytes;
		codes[j] = *reinterpret_cast<const uint16_t *>(in + part * 2);
		s[j] = in[16 * nb + (part >> 3)];
		at[j] = row * dim + part * 4;
	}
#pragma unroll
	for (int j = 0; j < kMx4ExpandRun; j++) {
		if (left[j] <= 0) continue;
		const float scale = s[j] == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float(s[j] > 0 ? (unsigned)s[j] << 23 : 0x00400000u);
		Mx4Float4 t;
#pragma unroll
		for (int i = 0; i < 4; i++) {
			const unsigned c = (codes[j] >> (4 * i)) & 15u, ex = (c >> 1) & 3u, m = c & 1u;
			// 2^(ex - 1) (1 + m / 2), or m / 2 where ex = 0
			const float mag = ex ? __uint_as_float(((ex + 126u) << 23) | (m << 22)) : 0.5f * (float)m;
			t.v[i] = ((c & 8u) ? -mag : mag) * scale;
		}
		if (left[j] >= 4) {
			*reinterpret_cast<Mx4Float4 *>(values + at[j]) = t;
		} else {
#pragma unroll
			for (int i = 0; i < 3; i++)
				if (i < left[j]) values[at[j] + i] = t.v[i];
		}
	}
}

// workgroups of 256 threads for rows x per_row threads; what a grid can hold is checked by the caller
inline int64_t mx4_row_groups(int64_t rows, int dim) { return (rows * 4 * mx4_blocks(dim) + 255) / 256; }

hipError_t mx4_launch_quantize(const void *x, int dtype, int64_t rows, int dim, int64_t ld, uint8_t *packed, hipStream_t s)
{
	const int nb = mx4_blocks(dim), rb = mx4_row_bytes(dim);
	const int64_t step = (int64_t)1 << 22;  // rows a launch: at most 2^31 threads at the widest row
	for (int64_t r = 0; r < rows; r += step) {
		const int64_t m = rows - r < step ? rows - r : step;
		const dim3 grid((unsigned)mx4_row_groups(m, dim));
		uint8_t *o = packed + r * rb;
		if (dtype == 0)
			hipLaunchKernelGGL((mx4_quantize_kernel<0>), grid, dim3(256), 0, s, static_cast<const float *>(x) + r * ld, m, dim, ld, nb, rb, o);
		else if (dtype == 1)
			hipLaunchKernelGGL((mx4_quantize_kernel<1>), grid, dim3(256), 0, s, static_cast<const uint16_t *>(x) + r * ld, m, dim, ld, nb, rb, o);
		else
			hipLaunchKernelGGL((mx4_quantize_kernel<2>), grid, dim3(256), 0, s, static_cast<const uint16_t *>(x) + r * ld, m, dim, ld, nb, rb, o);
	}
	return hipGetLastError();
}

hipError_t mx4_launch_expand(const uint8_t *packed, int64_t rows, int dim, float *values, hipStream_t s)
{
	const int nb = mx4_blocks(dim), rb = mx4_row_bytes(dim);
	const int64_t step = (int64_t)1 << 22;
	for (int64_t r = 0; r < rows; r += step) {
		const int64_t m = rows - r < step ? rows - r : step;
		const int64_t groups = (m * ((dim + 3) / 4) + 256 * kMx4ExpandRun - 1) / (256 * kMx4ExpandRun);
		hipLaunchKernelGGL(mx4_expand_kernel, dim3((unsigned)groups), dim3(256), 0, s, packed + r * rb, m, dim, nb, rb,
		                   values + r * dim);
	}
	return hipGetLastError();
}

}  // namespace mvdb
