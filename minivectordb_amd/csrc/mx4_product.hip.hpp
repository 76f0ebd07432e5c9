// mx4_product.hip.hpp -- every dot product of packed queries and packed rows (format: mx4.hpp).
#pragma once

#include <hip/hip_runtime.h>

#include "mx4.hpp"

namespace mvdb {

using mx4_v4i = __attribute__((ext_vector_type(4))) int;
using mx4_v8i = __attribute__((ext_vector_type(8))) int;
using mx4_v16f = __attribute__((ext_vector_type(16))) float;

// D += A B over 64 components: v_mfma_scale_f32_32x32x64_f8f6f4, both operands 4-bit.  Lane l holds row (A) or column (B)
// l & 31, block l >> 5 of the two: 16 bytes of codes, and that block's scale in byte OA (OB) of its scale register.  D: column
// l & 31, row 8 (i / 4) + 4 (l >> 5) + i % 4 in register i.  The products are multiples of 1/4 of the scales' product, so as long as the
// scales of a row lie within a few powers of two the f32 sums are exact.
template <int OA, int OB>
__device__ __forceinline__ mx4_v16f mx4_mfma(const mx4_v4i &a, int sa, const mx4_v4i &b, int sb, const mx4_v16f &c)
{
	const mx4_v8i a8 = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, b8 = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
	return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a8, b8, c, 4, 4, OA, sa, OB, sb);
}

// A wave computes 64 queries x 64 rows, a workgroup (2 x 2 waves) 128 x 128; fragments come straight from memory.  Column c of the
// result is row c, or (step > 1) row 64 * step * (c / 64) + c % 64: the 64-row tiles that are multiples of step.  Columns past the
// last row hold products that nobody reads.
__global__ __launch_bounds__(256) void mx4_product_kernel(const uint8_t *q, int nq, const uint8_t *rows, int n, int ksteps, int row_bytes, float *out,
                                                          int64_t ldo, int qtiles, int cols, int64_t step)
{
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
	const int half = lane >> 5, r32 = lane & 31;
	const int qt = blockIdx.x % qtiles, rt = blockIdx.x / qtiles;
	const int q0 = qt * 128 + (wave >> 1) * 64, r0 = rt * 128 + (wave & 1) * 64;
	if (q0 >= nq || r0 >= cols) return;
	const uint8_t *qp[2], *rp[2];
#pragma unroll
	for (int t = 0; t < 2; t++) {
		const int qi = q0 + t * 32 + r32, col = r0 + t * 32 + r32;
		const int64_t ri = col + (int64_t)(col & ~63) * (step - 1);
		qp[t] = q + (int64_t)(qi < nq ? qi : nq - 1) * row_bytes;
		rp[t] = rows + (ri < n ? ri : n - 1) * row_bytes;
	}
	mx4_v16f acc[2][2];
#pragma unroll
	for (int t = 0; t < 2; t++)
#pragma unroll
		for (int u = 0; u < 2; u++)
#pragma unroll
			for (int i = 0; i < 16; i++) acc[t][u][i] = 0.f;
	const int scales = 32 * ksteps;  // offset of the scale bytes
	for (int s = 0; s < ksteps; s++) {
		mx4_v4i a[2], b[2];
		int sa[2], sb[2];
#pragma unroll
		for (int t = 0; t < 2; t++) {
			a[t] = *reinterpret_cast<const mx4_v4i *>(qp[t] + (2 * s + half) * 16);
			b[t] = *reinterpret_cast<const mx4_v4i *>(rp[t] + (2 * s + half) * 16);
			sa[t] = qp[t][scales + 2 * s + half];
			sb[t] = rp[t][scales + 2 * s + half];
		}
#pragma unroll
		for (int t = 0; t < 2; t++)
#pragma unroll
			for (int u = 0; u < 2; u++) acc[t][u] = mx4_mfma<0, 0>(a[t], sa[t], b[u], sb[u], acc[t][u]);
	}
#pragma unroll
	for (int t = 0; t < 2; t++)
#pragma unroll
		for (int u = 0; u < 2; u++) {
			const int col = r0 + u * 32 + r32;
#pragma unroll
			for (int i = 0; i < 16; i++) {
				const int qi = q0 + t * 32 + 8 * (i >> 2) + 4 * half + (i & 3);
				if (qi < nq && col < cols) out[qi * ldo + col] = acc[t][u][i];
			}
		}
}

// `cols` columns
inline hipError_t mx4_launch_product_tiles(const uint8_t *q, int nq, const uint8_t *rows, int n, int cols, int64_t step, int ksteps, int row_bytes, float *out,
                                           int64_t ldo, hipStream_t s)
{
	const int64_t rtiles = ((int64_t)cols + 127) / 128;
	const int64_t qstep = 1 << 16;  // queries a launch (what one grid can hold)
	for (int64_t q0 = 0; q0 < nq; q0 += qstep) {
		const int m = (int)(nq - q0 < qstep ? nq - q0 : qstep), qtiles = (m + 127) / 128;
		const int64_t rstep = ((int64_t)1 << 22) / qtiles;
		for (int64_t r0 = 0; r0 < rtiles; r0 += rstep) {
			const int64_t c = rtiles - r0 < rstep ? rtiles - r0 : rstep;
			const int64_t col = r0 * 128, row = col * step;
			if (row >= n) break;
			hipLaunchKernelGGL(mx4_product_kernel, dim3((unsigned)(c * qtiles)), dim3(256), 0, s, q + q0 * row_bytes, m, rows + row * row_bytes,
			                   (int)(n - row), ksteps, row_bytes, out + q0 * ldo + col, ldo, qtiles, (int)(cols - col), step);
		}
	}
	return hipGetLastError();
}

hipError_t mx4_launch_product(const uint8_t *q, int nq, const uint8_t *rows, int n, int dim, float *out, int64_t ldo, hipStream_t s)
{
	return mx4_launch_product_tiles(q, nq, rows, n, n, 1, mx4_blocks(dim) / 2, mx4_row_bytes(dim), out, ldo, s);
}

}  // namespace mvdb
