// mx4_product.hip.hpp -- every dot product of packed queries and packed rows (format: mx4.hpp).
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

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

// The fragments of 32 packed rows of KS steps of 64 components, and their scale bytes: pieces 2 s + half of step s
template <int KS>
struct Mx4Frag {
	mx4_v4i d[KS];
	int sc[(KS + 1) / 2];  // byte 0: the scale of an even step, byte 2: of the odd one after it
};

template <int KS>
__device__ __forceinline__ void mx4_load_frag(Mx4Frag<KS> &f, const uint8_t *row, int half)
{
#pragma unroll
	for (int s = 0; s < KS; s++)
		f.d[s] = *reinterpret_cast<const mx4_v4i *>(row + (2 * s + half) * 16);
	const int *sp = reinterpret_cast<const int *>(row + 32 * KS);
#pragma unroll
	for (int s = 0; s < (KS + 1) / 2; s++)
		f.sc[s] = sp[s];
}
template <int KS>
__device__ __forceinline__ void mx4_shift_scales(Mx4Frag<KS> &f, int half)
{
#pragma unroll
	for (int s = 0; s < (KS + 1) / 2; s++) f.sc[s] = (int)((unsigned)f.sc[s] >> (8 * half));
}

// go(KS) for a row of `ks` steps, 1 .. 16
template <int KS = 1, typename F>
inline void mx4_for_steps(int ks, F go)
{
	if (ks == KS)
		go(std::integral_constant<int, KS>{});
	else if constexpr (KS < 16)
		mx4_for_steps<KS + 1>(ks, go);
}

struct Mx4Product {
	const uint8_t *q, *rows;
	int nq, n;
	float *out;
	int64_t ldo;
	int groups, run;  // groups of 32 * mx4_product_frags queries; steps of 128 rows a workgroup
	int block;  // chunks of an XCD that are gone through for one group of queries after the other
};

// fragments of 32 queries a wave holds: as many as leave room in its registers for the rows
__host__ __device__ constexpr int mx4_product_frags(int ks) { return ks <= 8 ? 2 : 1; }

// Bound by the writing of the result (4 bytes for every 2 * dim operations): 1000 x 262 144 x 384 in 189-207 us (5.3-5.8 TB/s; a copy reaches 5.2
// read and written, a fill 6.8), 4096 x 65 536 x 512 in 214 us.  A wave holds 64 queries (32 where rows are long) in registers and takes 32 rows at
// a time, the next ones on their way meanwhile; the four waves of a workgroup take neighbouring rows, so that together they write 512 bytes of each
// of 64 result rows.  Queries are the rows of D, so a store writes 128 bytes of two result rows.  The workgroups of one XCD go through a block of
// rows that stays in its L2, one group of queries after the other: what is written at a time lies side by side in a result row rather than at
// one place of many rows, which a power of two as the row length would put into the same memory channels.
template <int KS, bool STREAM>
__global__ __launch_bounds__(256, 2) void mx4_product_kernel(Mx4Product a)
{
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, r32 = lane & 31;
	const int j8 = blockIdx.x >> 3, j = j8 % (a.groups * a.block);
	const int group = j / a.block;
	const int64_t chunk = ((int64_t)(j8 / (a.groups * a.block)) * a.block + j % a.block) * 8 + (blockIdx.x & 7);
	constexpr int row_bytes = mx4_row_bytes(64 * KS);
	int64_t col0 = chunk * a.run * 128 + wave * 32;
	if (col0 >= a.n) return;
	constexpr int C = mx4_product_frags(KS);
	const int q0 = group * 32 * C;
	Mx4Frag<KS> qf[C];
#pragma unroll
	for (int c = 0; c < C; c++) {
		const int q = q0 + c * 32 + r32;
		mx4_load_frag<KS>(qf[c], a.q + (int64_t)(q < a.nq ? q : a.nq - 1) * row_bytes, half);
	}
	const int64_t end = (chunk + 1) * a.run * 128 < a.n ? (chunk + 1) * a.run * 128 : a.n;
	auto load = [&](int64_t col, Mx4Frag<KS> &f) {
		const int64_t at = col + r32;
		mx4_load_frag<KS>(f, a.rows + (at < a.n ? at : a.n - 1) * row_bytes, half);
	};
	auto use = [&](int64_t col, Mx4Frag<KS> &f) {
		mx4_shift_scales(f, half);
		mx4_v16f acc[C];
		const mx4_v16f zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
		for (int s = 0; s < KS; s++) {
#pragma unroll
			for (int c = 0; c < C; c++) {
				const mx4_v16f &in = s == 0 ? zero : acc[c];
				acc[c] = (s & 1) ? mx4_mfma<2, 2>(qf[c].d[s], qf[c].sc[s / 2], f.d[s], f.sc[s / 2], in)
				                 : mx4_mfma<0, 0>(qf[c].d[s], qf[c].sc[s / 2], f.d[s], f.sc[s / 2], in);
			}
		}
#pragma unroll
		for (int c = 0; c < C; c++) asm volatile("" : "+v"(acc[c]));  // keeps the products out of the branches below: see mx4_tile (mx4_scan.hip.hpp)
		const bool full = q0 + 32 * C <= a.nq && col + 32 <= a.n;
		float *o = a.out + (q0 + 4 * half) * a.ldo + col + r32;
		if (full) {
#pragma unroll
			for (int c = 0; c < C; c++)
#pragma unroll
				for (int i = 0; i < 16; i++) {
					float *p = o + (c * 32 + 8 * (i >> 2) + (i & 3)) * a.ldo;
					if constexpr (STREAM)
						__builtin_nontemporal_store(acc[c][i], p);
					else
						*p = acc[c][i];
				}
		} else if (col + r32 < a.n) {
#pragma unroll
			for (int c = 0; c < C; c++)
#pragma unroll
				for (int i = 0; i < 16; i++) {
					const int q = c * 32 + 8 * (i >> 2) + (i & 3);
					if (q0 + 4 * half + q < a.nq) o[q * a.ldo] = acc[c][i];
				}
		}
	};
	// the first rows are asked for before the queries are waited for
	auto ready = [&]() {
		__builtin_amdgcn_sched_barrier(0);
#pragma unroll
		for (int c = 0; c < C; c++) mx4_shift_scales(qf[c], half);
	};
	if constexpr (KS <= 8) {
		Mx4Frag<KS> f0, f1;
		load(col0, f0);
		ready();
		while (true) {
			if (col0 + 128 < end) load(col0 + 128, f1);
			__builtin_amdgcn_sched_barrier(0);
			use(col0, f0);
			col0 += 128;
			if (col0 >= end) break;
			if (col0 + 128 < end) load(col0 + 128, f0);
			__builtin_amdgcn_sched_barrier(0);
			use(col0, f1);
			col0 += 128;
			if (col0 >= end) break;
		}
	} else {
		Mx4Frag<KS> f;
		load(col0, f);
		ready();
		while (true) {
			use(col0, f);
			col0 += 128;
			if (col0 >= end) break;
			load(col0, f);
		}
	}
}

// Rows of more than 16 steps (dim > 1024): a wave computes 64 queries x 64 rows, a workgroup (2 x 2 waves) 128 x 128, both operands step by step.  Bound by
// its loads, which nothing hides: 37 x 50 021 x 2048 in 30 us (rows and result at the copy rate: 12), 256 x 65 536 x 2048 in 141 us (27).
__global__ __launch_bounds__(256) void mx4_product_long_kernel(const uint8_t *q, int nq, const uint8_t *rows, int n, int ksteps, int row_bytes, float *out,
                                                               int64_t ldo, int qtiles)
{
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
	const int half = lane >> 5, r32 = lane & 31;
	const int qt = blockIdx.x % qtiles, rt = blockIdx.x / qtiles;
	const int q0 = qt * 128 + (wave >> 1) * 64, r0 = rt * 128 + (wave & 1) * 64;
	if (q0 >= nq || r0 >= n) return;
	const uint8_t *qp[2], *rp[2];
#pragma unroll
	for (int t = 0; t < 2; t++) {
		const int qi = q0 + t * 32 + r32, ri = r0 + t * 32 + r32;
		qp[t] = q + (int64_t)(qi < nq ? qi : nq - 1) * row_bytes;
		rp[t] = rows + (int64_t)(ri < n ? ri : n - 1) * row_bytes;
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
				if (qi < nq && col < n) out[qi * ldo + col] = acc[t][u][i];
			}
		}
}

constexpr int kMx4ProductQ = 4096;       // queries a launch
constexpr int kMx4ProductGroups = 4096;  // workgroups a launch, about
constexpr int64_t kMx4BlockBytes = 4 << 20;  // rows of a block: an XCD's L2
constexpr int64_t kMx4StreamBytes = 256 << 20;  // results that are larger than the caches go past them

hipError_t mx4_launch_product(const uint8_t *q, int nq, const uint8_t *rows, int n, int dim, float *out, int64_t ldo, hipStream_t s)
{
	constexpr int row_steps = 16;  // rows that mx4_product_kernel holds in registers
	const int ksteps = mx4_blocks(dim) / 2, row_bytes = mx4_row_bytes(dim);
	const int64_t rtiles = ((int64_t)n + 127) / 128;
	if (ksteps <= row_steps) {
		Mx4Product a{};
		a.rows = rows;
		a.n = n;
		a.ldo = ldo;
		const bool stream = (int64_t)nq * n * 4 > kMx4StreamBytes;
		for (int64_t q0 = 0; q0 < nq; q0 += kMx4ProductQ) {
			a.nq = (int)(nq - q0 < kMx4ProductQ ? nq - q0 : kMx4ProductQ);
			a.q = q + q0 * row_bytes;
			a.out = out + q0 * ldo;
			const int frags = mx4_product_frags(ksteps);
			a.groups = (a.nq + 32 * frags - 1) / (32 * frags);
			// about kMx4ProductGroups workgroups, each with a run of steps that pays for its queries (37 x 50 021 x 1000: two steps 9.0 us, one
			// 10.9 us; 1 to 256 queries, 5000 to 100 000 rows, dims 100 to 1000: two are up to 18 % faster where that makes more than 600
			// workgroups, and nothing differs below); but all of a small result's at once
			const int64_t run = rtiles * a.groups / kMx4ProductGroups, least = rtiles * a.groups >= 512 ? 2 : 1;
			a.run = (int)(run < least ? least : run > 16 ? 16 : run);
			const int64_t chunks = (rtiles + a.run - 1) / a.run;
			const int64_t per_xcd = (chunks + 7) / 8, fit = kMx4BlockBytes / ((int64_t)a.run * 128 * row_bytes);
			// Blocks of an L2 or of one chunk, measured over 256 to 4096 queries, 40 000 to 524 288 rows, dims 100, 384, 1000 (times by blocks of one chunk
			// / of an L2).  Many queries over result rows of moderate length write side by side only in blocks of an L2 (x 65 536 x 384: 1000 queries
			// 71 / 56 us, 4096 243 / 216; 1000 to 4096 queries, 65 536 to 131 072 rows: 1.00 to 1.21).  Up to 512 queries, and over longer result rows, the
			// workgroups in flight spread over enough columns by themselves and share each row at once (512 x 65 536 x 384 28 / 30 us, 512 x 262 144 x
			// 384 102 / 115, 2048 x 262 144 x 384 398 / 451; 160 000 and 200 000 rows: 0.92 to 1.11).  Rows above dim 512, whose groups are half as large,
			// gain nothing from them (x 1000: 0.89 to 1.01 with more than 1000 queries).
			const bool blocks_of_l2 = ksteps <= 8 && a.groups > 8 && n < 150000 && fit >= 1;
			a.block = (int)(blocks_of_l2 ? (fit < per_xcd ? fit : per_xcd) : 1);
			const int64_t blocks = (per_xcd + a.block - 1) / a.block * a.block * 8 * a.groups;
			mx4_for_steps(ksteps, [&](auto steps) {
				constexpr int KS = decltype(steps)::value;
				if (stream)
					hipLaunchKernelGGL((mx4_product_kernel<KS, true>), dim3((unsigned)blocks), dim3(256), 0, s, a);
				else
					hipLaunchKernelGGL((mx4_product_kernel<KS, false>), dim3((unsigned)blocks), dim3(256), 0, s, a);
			});
		}
		return hipGetLastError();
	}
	for (int64_t q0 = 0; q0 < nq; q0 += kMx4ProductQ) {
		const int m = (int)(nq - q0 < kMx4ProductQ ? nq - q0 : kMx4ProductQ), qtiles = (m + 127) / 128;
		const int64_t rstep = ((int64_t)1 << 22) / qtiles;  // what one grid can hold
		for (int64_t r0 = 0; r0 < rtiles; r0 += rstep) {
			const int64_t c = rtiles - r0 < rstep ? rtiles - r0 : rstep;
			hipLaunchKernelGGL(mx4_product_long_kernel, dim3((unsigned)(c * qtiles)), dim3(256), 0, s, q + q0 * row_bytes, m, rows + r0 * 128 * row_bytes,
			                   (int)(n - r0 * 128), ksteps, row_bytes, out + q0 * ldo + r0 * 128, ldo, qtiles);
		}
	}
	return hipGetLastError();
}

}  // namespace mvdb
