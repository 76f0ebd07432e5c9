// mx4_scan.hip.hpp -- the k largest dot products of each packed query with the packed rows (format: mx4.hpp).
//
// Order: value descending, then id ascending.  A candidate is one 64-bit key, larger = earlier in that order: the value's bits made
// monotone in the upper half, ~id in the lower.  0 is no key (it would be a NaN with the sign bit).  Rows whose `allow` bit is not set
// and rows whose product is NaN are no candidates.
#pragma once

#include <hip/hip_runtime.h>

#include "mx4.hpp"
#include "mx4_product.hip.hpp"

namespace mvdb {

using mx4_key = unsigned long long;

__device__ __forceinline__ mx4_key mx4_make_key(float v, unsigned id)
{
	if (v != v) return 0;
	const unsigned b = __float_as_uint(v + 0.f);  // -0 is 0
	return ((mx4_key)(b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u)) << 32) | (unsigned)~id;
}
__device__ __forceinline__ float mx4_key_value(mx4_key key)
{
	const unsigned u = (unsigned)(key >> 32);
	return __uint_as_float(u ^ ((u >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ int mx4_key_id(mx4_key key) { return (int)~(unsigned)key; }

// One workgroup per query over its row of scores: candidates above the k-th best so far are gathered in LDS, and sorted and cut to
// the best k whenever the next 256 might not fit.
constexpr int kMx4Gather = 1024;

__device__ inline void mx4_sort_desc(mx4_key *keys, int size)  // bitonic, size a power of two
{
	for (int w = 2; w <= size; w <<= 1)
		for (int d = w >> 1; d >= 1; d >>= 1) {
			for (int i = threadIdx.x; i < size / 2; i += blockDim.x) {
				const int a = 2 * i - (i & (d - 1)), b = a + d;
				const mx4_key x = keys[a], y = keys[b];
				if ((x < y) == ((a & w) == 0)) {
					keys[a] = y;
					keys[b] = x;
				}
			}
			__syncthreads();
		}
}

__global__ __launch_bounds__(256) void mx4_select_kernel(const float *scores, int n, int k, const uint32_t *allow, int32_t *out_ids, float *out_val,
                                                         int32_t *out_count)
{
	__shared__ mx4_key keys[kMx4Gather];
	__shared__ int count;
	const int tid = threadIdx.x;
	const float *sc = scores + (int64_t)blockIdx.x * n;
	if (tid == 0) count = 0;
	mx4_key bound = 0;
	__syncthreads();
	auto cut = [&](int have) {  // the best k, sorted
		for (int i = have + tid; i < kMx4Gather; i += 256) keys[i] = 0;
		__syncthreads();
		mx4_sort_desc(keys, kMx4Gather);
		if (tid == 0) count = have < k ? have : k;
		if (have >= k) bound = keys[k - 1];
		__syncthreads();
	};
	for (int64_t base = 0; base < n; base += 256) {
		const int64_t id = base + tid;
		if (id < n && (!allow || ((allow[id >> 5] >> (id & 31)) & 1u))) {
			const mx4_key key = mx4_make_key(sc[id], (unsigned)id);
			if (key > bound) keys[atomicAdd(&count, 1)] = key;
		}
		__syncthreads();
		const int have = count;
		__syncthreads();
		if (have > kMx4Gather - 256) cut(have);
	}
	cut(count);
	const int have = count;
	for (int i = tid; i < k; i += 256) {
		const mx4_key key = i < have ? keys[i] : 0;
		out_ids[(int64_t)blockIdx.x * k + i] = i < have ? mx4_key_id(key) : -1;
		out_val[(int64_t)blockIdx.x * k + i] = i < have ? mx4_key_value(key) : 0.f;
	}
	if (tid == 0) out_count[blockIdx.x] = have;
}

// queries whose scores are held at a time: at most 1 GiB of them, but one query's always
inline int mx4_scan_slab(int nq, int n)
{
	const int64_t fit = ((int64_t)1 << 28) / (n > 0 ? n : 1);
	return (int)(fit < 1 ? 1 : fit < nq ? fit : nq);
}

size_t mx4_scan_workspace(int nq, int n, int k)
{
	(void)k;
	return nq > 0 && n > 0 ? (size_t)mx4_scan_slab(nq, n) * n * 4 : 16;
}

hipError_t mx4_launch_scan(const uint8_t *q, int nq, const uint8_t *rows, int n, int dim, int k, const uint32_t *allow, int32_t *out_ids,
                           float *out_val, int32_t *out_count, void *ws, hipStream_t s)
{
	float *scores = static_cast<float *>(ws);
	const int slab = mx4_scan_slab(nq, n), rb = mx4_row_bytes(dim);
	for (int q0 = 0; q0 < nq; q0 += slab) {
		const int m = nq - q0 < slab ? nq - q0 : slab;
		const hipError_t e = mx4_launch_product(q + (int64_t)q0 * rb, m, rows, n, dim, scores, n, s);
		if (e != hipSuccess) return e;
		hipLaunchKernelGGL(mx4_select_kernel, dim3(m), dim3(256), 0, s, scores, n, k, allow, out_ids + (int64_t)q0 * k, out_val + (int64_t)q0 * k,
		                   out_count + q0);
	}
	return hipGetLastError();
}

}  // namespace mvdb
