// mx4_scan.hip.hpp -- the k largest dot products of each packed query with the packed rows (format: mx4.hpp).
//
// Order: value descending, then id ascending.  A candidate is one 64-bit key, larger = earlier in that order: the value's bits made
// monotone in the upper half, ~id in the lower.  0 is no key (it would be a NaN with the sign bit).  Rows whose `allow` bit is not set
// and rows whose product is NaN are no candidates; a row is taken out by giving its blocks the scale 255, which makes every product NaN,
// and a NaN is never >= a bound.
//
// Two ways, by the number of queries:
//
// CHUNKS (few queries): a workgroup computes the products of its own run of rows, keeps them in LDS and picks the best k of each
// query there; a second launch picks the best k of those.  Every row is read once, and two launches are all there is.
//
// LEVELS (many queries): the rows are taken in levels of 64-row tiles, each about `ratio` times the one before it: level 0 is every
// ratio^L-th tile, level l the tiles that are multiples of ratio^(L - l) and not of ratio^(L - l + 1).  After a level the k-th best key so
// far is a bound: k rows are at least that good, so only keys above it matter, and as the rows seen so far are spread evenly over the
// store about k (ratio - 1) keys of the next level are (whatever order the rows are in, unless they repeat with the tiles' period).
// Level 0 has no bound: its products go to memory.  From then on a product that passes the bound is pushed into a queue of its wave in LDS, and
// from there into the query's buffer of kMx4Cap keys; mx4_pick_kernel cuts the buffer to its best k after every level.  A buffer that
// overflows marks its query, and mx4_rescue_kernel does those over, one workgroup each.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

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

// ---------------------------------------------------------------------------------------------- selection
// LDS of mx4_block_kth
struct Mx4PickLds {
	int hist[256];
	mx4_key lo[16], hi[16];  // per wave
	int pick, above, total;
};

// The k-th largest of the keys key_at(0 .. m) (0 = none) of a workgroup of T threads: the key that exactly min(k, keys) are >= to; 1 where
// there are at most k.  Radix selection, eight bits at a time from the highest bit in which the keys differ: scores lie within a few powers of
// two, so their leading bits would all fall into one bin.  It ends as soon as a bin is wanted whole.
template <int T, typename F>
__device__ mx4_key mx4_block_kth(F key_at, int m, int k, Mx4PickLds &l)
{
	const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
	mx4_key lo = ~0ull, hi = 0;
	int have = 0;
	for (int i = tid; i < m; i += T) {
		const mx4_key key = key_at(i);
		if (key) {
			lo = key < lo ? key : lo;
			hi = key > hi ? key : hi;
			have++;
		}
	}
	if (tid == 0) l.total = 0;
#pragma unroll
	for (int d = 32; d >= 1; d >>= 1) {
		const mx4_key ol = ((mx4_key)(unsigned)__shfl_xor((int)(lo >> 32), d, 64) << 32) | (unsigned)__shfl_xor((int)(unsigned)lo, d, 64);
		const mx4_key oh = ((mx4_key)(unsigned)__shfl_xor((int)(hi >> 32), d, 64) << 32) | (unsigned)__shfl_xor((int)(unsigned)hi, d, 64);
		lo = ol < lo ? ol : lo;
		hi = oh > hi ? oh : hi;
		have += __shfl_xor(have, d, 64);
	}
	__syncthreads();
	if (lane == 0) {
		l.lo[wave] = lo;
		l.hi[wave] = hi;
		atomicAdd(&l.total, have);
	}
	__syncthreads();
#pragma unroll
	for (int w = 0; w < T / 64; w++) {
		lo = l.lo[w] < lo ? l.lo[w] : lo;
		hi = l.hi[w] > hi ? l.hi[w] : hi;
	}
	if (l.total <= k) return 1;
	// (more than k keys, so two at least, all different: hi != lo)
	int top = 64 - __builtin_clzll(hi ^ lo);  // bits [0, top) differ
	mx4_key fixed = top < 64 ? hi >> top << top : 0;
	int need = k;
	while (true) {
		const int shift = top > 8 ? top - 8 : 0;
		const unsigned bins = 1u << (top - shift);
		for (int i = tid; i < 256; i += T) l.hist[i] = 0;
		__syncthreads();
		for (int i = tid; i < m; i += T) {
			const mx4_key key = key_at(i);
			if (key && (top == 64 || (key >> top) == (fixed >> top))) atomicAdd(&l.hist[(unsigned)(key >> shift) & (bins - 1)], 1);
		}
		__syncthreads();
		if (wave == 0) {  // the bin that holds the need-th from above
			int c[4], s = 0;
#pragma unroll
			for (int j = 3; j >= 0; j--) {
				s += l.hist[lane * 4 + j];
				c[j] = s;  // keys in the bins of this lane from j up
			}
			int above = s;  // inclusive suffix sum over the lanes
#pragma unroll
			for (int d = 1; d < 64; d <<= 1) {
				const int o = __shfl_down(above, d, 64);
				above += lane + d < 64 ? o : 0;
			}
			above -= s;  // keys in the lanes above
#pragma unroll
			for (int j = 0; j < 4; j++) {
				const int higher = above + (j < 3 ? c[j + 1 < 4 ? j + 1 : 3] : 0);
				if (higher < need && above + c[j] >= need) {
					l.pick = lane * 4 + j;
					l.above = higher;
				}
			}
		}
		__syncthreads();
		const int bin = l.pick, in_bin = l.hist[bin];
		need -= l.above;
		fixed |= (mx4_key)bin << shift;
		top = shift;
		__syncthreads();
		if (in_bin == need || shift == 0) return fixed;
	}
}

// What a selection does with the best k: the caller's arrays, or (a level that is not the last) back into the buffer, with the k-th as
// the bound of the next level.  The keys >= the k-th are gathered in LDS and put in order by their rank (they are all different).
struct Mx4Out {
	int32_t *ids, *count;
	float *val;
	mx4_key *keys, *bound;  // keys != nullptr: not the last level
	int32_t *fill;
};

template <int T, typename F>
__device__ void mx4_block_topk(F key_at, int m, int k, int64_t q, int64_t stride, const Mx4Out &o, Mx4PickLds &l, mx4_key *best)
{
	const int tid = threadIdx.x;
	const mx4_key kth = mx4_block_kth<T>(key_at, m, k, l);
	if (tid == 0) l.pick = 0;
	__syncthreads();
	for (int i = tid; i < m; i += T) {
		const mx4_key key = key_at(i);
		if (key >= kth) best[atomicAdd(&l.pick, 1)] = key;  // (kth >= 1)
	}
	__syncthreads();
	const int have = l.pick;  // <= k <= kMx4ScanMaxK
	for (int i = tid; i < k; i += T) {
		mx4_key key = 0;
		int at = i;
		if (i < have) {
			key = best[i];
			at = 0;
			for (int j = 0; j < have; j++) at += best[j] > key ? 1 : 0;
		}
		if (o.keys) {
			if (i < have) o.keys[q * stride + at] = key;
			if (i < have && at == k - 1) o.bound[q] = key;
		} else {
			o.ids[q * k + at] = i < have ? mx4_key_id(key) : -1;
			o.val[q * k + at] = i < have ? mx4_key_value(key) : 0.f;
		}
	}
	if (tid == 0) {
		if (o.keys) {
			o.fill[q] = have;
			if (have < k) o.bound[q] = 0;
		} else {
			o.count[q] = have;
		}
	}
}

// Rows of level 0 and of a level's tile i.  step = ratio^(L - l); tiles of level l >= 1: step * (i + i / (ratio - 1) + 1).
__host__ __device__ inline int64_t mx4_level_tile(int64_t i, int64_t step, int ratio) { return ratio ? step * (i + i / (ratio - 1) + 1) : step * i; }

// one workgroup per query: the best k of level 0's products (m of them, product j belongs to row (j / 64) * 64 * step + j % 64)
__global__ __launch_bounds__(256) void mx4_pick_first_kernel(const float *scores, int m, int64_t step, int n, int k, const uint32_t *allow, Mx4Out o,
                                                             int64_t stride, int32_t *over)
{
	__shared__ Mx4PickLds l;
	__shared__ mx4_key best[kMx4ScanMaxK];
	const int64_t q = blockIdx.x;
	const float *sc = scores + q * m;
	auto key_at = [&](int j) -> mx4_key {
		const int64_t id = (int64_t)(j >> 6) * 64 * step + (j & 63);
		if (id >= n || (allow && !((allow[id >> 5] >> (id & 31)) & 1u))) return 0;
		return mx4_make_key(sc[j], (unsigned)id);
	};
	if (over && threadIdx.x == 0) over[q] = 0;
	mx4_block_topk<256>(key_at, m, k, q, stride, o, l, best);
}

// one workgroup per query: the best k of its buffer
template <int T>
__global__ __launch_bounds__(T) void mx4_pick_kernel(const mx4_key *keys, const int32_t *fill, int cap, int k, Mx4Out o, int32_t *over)
{
	__shared__ Mx4PickLds l;
	__shared__ mx4_key best[kMx4ScanMaxK];
	const int64_t q = blockIdx.x;
	const mx4_key *mine = keys + q * cap;
	int m = fill ? fill[q] : cap;
	if (m > cap) {  // keys were lost
		m = cap;
		if (threadIdx.x == 0) over[q] = 1;
	}
	if (o.keys) __syncthreads();  // fill[q] has been read by everybody before it is written
	auto key_at = [&](int j) -> mx4_key { return mine[j]; };
	mx4_block_topk<T>(key_at, m, k, q, cap, o, l, best);
}

// ---------------------------------------------------------------------------------------------- queries in registers
// The fragments of 32 queries (columns of D) for KS steps of 64 components, and their scale bytes: pieces 2 s + half of step s.  KS is
// at least the row's number of steps; what is past it stays 0.
template <int KS>
struct Mx4Frag {
	mx4_v4i d[KS];
	int sc[(KS + 1) / 2];  // byte 0: the scale of an even step, byte 2: of the odd one after it
};

// exact: KS is the row's number of steps
template <int KS, bool EXACT>
__device__ __forceinline__ void mx4_load_frag(Mx4Frag<KS> &f, const uint8_t *row, int half, int ksteps)
{
#pragma unroll
	for (int s = 0; s < KS; s++)
		if (EXACT || s < ksteps) f.d[s] = *reinterpret_cast<const mx4_v4i *>(row + (2 * s + half) * 16);
	const int *sp = reinterpret_cast<const int *>(row + 32 * (EXACT ? KS : ksteps));
#pragma unroll
	for (int s = 0; s < (KS + 1) / 2; s++)
		if (EXACT || 2 * s < ksteps) f.sc[s] = sp[s];
}
template <int KS>
__device__ __forceinline__ void mx4_shift_scales(Mx4Frag<KS> &f, int half)
{
#pragma unroll
	for (int s = 0; s < (KS + 1) / 2; s++) f.sc[s] = (int)((unsigned)f.sc[s] >> (8 * half));
}

// acc[c] = the products of the 32 rows in `a` (rows of D) with the 32 queries in b[c]
template <int KS, bool EXACT, int C>
__device__ __forceinline__ void mx4_tile(const Mx4Frag<KS> &a, const Mx4Frag<KS> (&b)[C], int ksteps, mx4_v16f (&acc)[C])
{
	const mx4_v16f zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
	for (int s = 0; s < KS; s++)
		if (EXACT || s < ksteps) {
#pragma unroll
			for (int c = 0; c < C; c++) {
				const mx4_v16f &in = s == 0 ? zero : acc[c];
				acc[c] = (s & 1) ? mx4_mfma<2, 2>(a.d[s], a.sc[s / 2], b[c].d[s], b[c].sc[s / 2], in)
				                 : mx4_mfma<0, 0>(a.d[s], a.sc[s / 2], b[c].d[s], b[c].sc[s / 2], in);
			}
		}
	// A matrix instruction reads its operands from all lanes, whatever the execution mask.  The compiler may move it into a branch that only
	// some lanes take when nothing but that branch uses the result, and the shifts of the scales with it, which do obey the mask: this use
	// keeps both here.
#pragma unroll
	for (int c = 0; c < C; c++) asm volatile("" : "+v"(acc[c]));
}

// ---------------------------------------------------------------------------------------------- chunks
constexpr int kMx4ChunkQ = 8;        // queries a launch, at most
constexpr int kMx4ChunkRows = 2048;  // rows a workgroup, at most

// A workgroup = 4 waves; a wave takes 32 rows at a time.  Queries are the columns of D, so with nq <= 8 of 32 columns used three
// quarters of the matrix work is for nothing: it is a few us at a million rows, against the reading of them.
template <int KS, bool EXACT>
__global__ __launch_bounds__(256) void mx4_chunk_kernel(const uint8_t *q, int nq, const uint8_t *rows, int n, int ksteps, int row_bytes, int k, int chunk,
                                                        const uint32_t *allow, mx4_key *out, int64_t stride)
{
	extern __shared__ float sc[];  // [nq][chunk]
	__shared__ Mx4PickLds l;
	const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, r32 = lane & 31;
	Mx4Frag<KS> b[1];
	mx4_load_frag<KS, EXACT>(b[0], q + (int64_t)(r32 < nq ? r32 : nq - 1) * row_bytes, half, ksteps);
	mx4_shift_scales(b[0], half);
	const int64_t first = (int64_t)blockIdx.x * chunk;
	const int m = (int)(n - first < chunk ? n - first : chunk);
	const uint8_t *base = rows + first * row_bytes;
	for (int t = wave * 32; t < m; t += 128) {
		const int r = t + r32 < m ? t + r32 : m - 1;
		Mx4Frag<KS> a;
		mx4_load_frag<KS, EXACT>(a, base + (int64_t)r * row_bytes, half, ksteps);
		mx4_shift_scales(a, half);
		mx4_v16f acc[1];
		mx4_tile<KS, EXACT, 1>(a, b, ksteps, acc);
		if (r32 < nq) {
#pragma unroll
			for (int i = 0; i < 16; i++) {
				const int at = t + 8 * (i >> 2) + 4 * half + (i & 3);
				if (at < m) sc[r32 * chunk + at] = acc[0][i];
			}
		}
	}
	__syncthreads();
	for (int qi = 0; qi < nq; qi++) {
		auto key_at = [&](int j) -> mx4_key {
			const int64_t id = first + j;
			if (allow && !((allow[id >> 5] >> (id & 31)) & 1u)) return 0;
			return mx4_make_key(sc[qi * chunk + j], (unsigned)id);
		};
		const mx4_key kth = mx4_block_kth<256>(key_at, m, k, l);
		mx4_key *o = out + qi * stride + (int64_t)blockIdx.x * k;
		if (tid == 0) l.pick = 0;
		__syncthreads();
		for (int j = tid; j < m; j += 256) {
			const mx4_key key = key_at(j);
			if (key >= kth) o[atomicAdd(&l.pick, 1)] = key;
		}
		__syncthreads();
		const int have = l.pick;
		for (int j = have + tid; j < k; j += 256) o[j] = 0;
		__syncthreads();
	}
}

// ---------------------------------------------------------------------------------------------- levels
constexpr int kMx4Cap = 2048;      // keys of a query's buffer
constexpr int kMx4FirstTiles = 16;  // 64-row tiles of level 0, at most
constexpr int kMx4Queue = 192;     // keys of a wave's queue

struct Mx4Level {
	const uint8_t *q, *rows;
	const uint32_t *allow;
	int nq, n, ksteps, row_bytes;
	int64_t step;    // see mx4_level_tile
	int ratio, tiles;
	mx4_key *keys;   // [nq][kMx4Cap]
	int32_t *fill;   // [nq] keys in the buffer (may run past kMx4Cap)
	const mx4_key *bound;  // [nq], 0 = none
};

// A wave's queue of candidates
struct Mx4Queue {
	mx4_key key[kMx4Queue];
	int q[kMx4Queue];
};

// Empty the queue: one atomic per key, 64 in flight.
__device__ __forceinline__ void mx4_flush(const Mx4Level &a, Mx4Queue &w, int &n, int lane)
{
	asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
	for (int i = lane; i < n; i += 64) {
		const mx4_key key = w.key[i];
		const int q = w.q[i];
		const int slot = atomicAdd(&a.fill[q], 1);
		if (slot < kMx4Cap) a.keys[(int64_t)q * kMx4Cap + slot] = key;
	}
	asm volatile("" ::: "memory");
	n = 0;
}

// Candidates of one 32 x 32 tile: rows row0 .. + 31, query `q` in this lane's column
__device__ __forceinline__ void mx4_push(const Mx4Level &a, const mx4_v16f &acc, float bound, mx4_key bkey, int q, int64_t row0, int half, int lane, Mx4Queue &w,
                                         int &n)
{
#pragma unroll
	for (int i = 0; i < 16; i++) {
		if (__ballot(acc[i] >= bound)) {
			const mx4_key key = mx4_make_key(acc[i], (unsigned)(row0 + 8 * (i >> 2) + 4 * half + (i & 3)));
			const bool p = acc[i] >= bound && key > bkey;
			const unsigned long long who = __ballot(p);
			if (n + 64 > kMx4Queue) mx4_flush(a, w, n, lane);
			if (p) {
				const int at = n + (int)__builtin_amdgcn_mbcnt_hi((unsigned)(who >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)who, 0));
				w.key[at] = key;
				w.q[at] = q;
			}
			n += __popcll(who);
		}
	}
}

// Independent waves: each holds 64 queries and takes every (waves)-th half tile of the level straight from memory.
template <int KS, bool EXACT>
__global__ __launch_bounds__(256, 2) void mx4_stream_kernel(Mx4Level a, int qgroups)
{
	__shared__ Mx4Queue queue[4];
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, r32 = lane & 31;
	const int gw = blockIdx.x * 4 + wave, group = gw % qgroups;
	const int64_t first = gw / qgroups, waves = (int64_t)gridDim.x * 4 / qgroups;  // (the grid is a multiple of qgroups waves)
	if (first >= waves) return;
	Mx4Queue &w = queue[wave];
	int qn = 0;
	Mx4Frag<KS> b[2];
	float bound[2];
	mx4_key bkey[2];
	int qi[2];
#pragma unroll
	for (int c = 0; c < 2; c++) {
		qi[c] = group * 64 + c * 32 + r32;
		const int qs = qi[c] < a.nq ? qi[c] : a.nq - 1;
		mx4_load_frag<KS, EXACT>(b[c], a.q + (int64_t)qs * a.row_bytes, half, a.ksteps);
		mx4_shift_scales(b[c], half);
		bkey[c] = a.bound[qs];
		// no query in this column: nothing is >= NaN
		bound[c] = qi[c] >= a.nq ? __uint_as_float(0x7fc00000u) : bkey[c] ? mx4_key_value(bkey[c]) : -__builtin_inff();
	}
	for (int64_t i = first; i < 2 * (int64_t)a.tiles; i += waves) {
		const int64_t row0 = mx4_level_tile(i >> 1, a.step, a.ratio) * 64 + (i & 1) * 32;
		if (row0 >= a.n) continue;
		unsigned keep = row0 + 32 <= a.n ? 0xffffffffu : (1u << (a.n - row0)) - 1u;
		if (a.allow) keep &= a.allow[row0 >> 5];
		if (keep == 0) continue;
		const int64_t r = row0 + r32 < a.n ? row0 + r32 : a.n - 1;
		Mx4Frag<KS> f;
		mx4_load_frag<KS, EXACT>(f, a.rows + r * a.row_bytes, half, a.ksteps);
		const bool out = !((keep >> r32) & 1u);
#pragma unroll
		for (int s = 0; s < (KS + 1) / 2; s++) f.sc[s] = out ? -1 : f.sc[s];
		mx4_shift_scales(f, half);
		mx4_v16f acc[2];
		mx4_tile<KS, EXACT, 2>(f, b, a.ksteps, acc);
#pragma unroll
		for (int c = 0; c < 2; c++) {
			float m = acc[c][0];
#pragma unroll
			for (int j = 1; j < 16; j++) m = __builtin_fmaxf(m, acc[c][j]);
			if (__ballot(m >= bound[c])) mx4_push(a, acc[c], bound[c], bkey[c], qi[c], row0, half, lane, w, qn);
		}
	}
	mx4_flush(a, w, qn, lane);
}

// The queries whose buffer overflowed, from the beginning: a workgroup for each, 128 rows at a time, candidates gathered in LDS and cut
// to the best k when the next 128 might not fit.
template <int KS, bool EXACT>
__global__ __launch_bounds__(256) void mx4_rescue_kernel(Mx4Level a, int k, const int32_t *over, Mx4Out o)
{
	__shared__ Mx4PickLds l;
	__shared__ mx4_key keys[kMx4Cap], best[kMx4ScanMaxK];
	__shared__ int count;
	const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, r32 = lane & 31;
	for (int q = blockIdx.x; q < a.nq; q += gridDim.x) {
		if (!over[q]) continue;
		Mx4Frag<KS> b[1];
		mx4_load_frag<KS, EXACT>(b[0], a.q + (int64_t)q * a.row_bytes, half, a.ksteps);
		mx4_shift_scales(b[0], half);
		mx4_key kth = 1;  // keys below it are not wanted
		if (tid == 0) count = 0;
		__syncthreads();
		for (int64_t base = 0; base < a.n; base += 128) {
			const int64_t row0 = base + wave * 32;
			if (row0 < a.n) {
				const int64_t r = row0 + r32 < a.n ? row0 + r32 : a.n - 1;
				Mx4Frag<KS> f;
				mx4_load_frag<KS, EXACT>(f, a.rows + r * a.row_bytes, half, a.ksteps);
				mx4_shift_scales(f, half);
				mx4_v16f acc[1];
				mx4_tile<KS, EXACT, 1>(f, b, a.ksteps, acc);
				if (r32 == 0) {  // every column holds the same query
#pragma unroll
					for (int i = 0; i < 16; i++) {
						const int64_t id = row0 + 8 * (i >> 2) + 4 * half + (i & 3);
						if (id < a.n && (!a.allow || ((a.allow[id >> 5] >> (id & 31)) & 1u))) {
							const mx4_key key = mx4_make_key(acc[0][i], (unsigned)id);
							if (key >= kth) keys[atomicAdd(&count, 1)] = key;
						}
					}
				}
			}
			__syncthreads();
			const int have = count;
			if (have > kMx4Cap - 128) {
				auto key_at = [&](int j) -> mx4_key { return keys[j]; };
				kth = mx4_block_kth<256>(key_at, have, k, l);
				if (tid == 0) l.pick = 0;
				__syncthreads();
				for (int j = tid; j < have; j += 256)
					if (keys[j] >= kth) best[atomicAdd(&l.pick, 1)] = keys[j];
				__syncthreads();
				const int m = l.pick;
				for (int j = tid; j < m; j += 256) keys[j] = best[j];
				if (tid == 0) count = m;
			}
			__syncthreads();
		}
		auto key_at = [&](int j) -> mx4_key { return keys[j]; };
		const int have = count;
		__syncthreads();
		mx4_block_topk<256>(key_at, have, k, q, 0, o, l, best);
		__syncthreads();
	}
}

// ---------------------------------------------------------------------------------------------- the plan
constexpr int kMx4SlabQ = 8192;  // queries whose buffers are held at a time

struct Mx4Plan {
	bool chunks;
	int chunk, parts;  // chunks: rows of one, how many
	int levels, ratio, first_rows;  // levels after level 0; rows of level 0 (a multiple of 64)
	int64_t step0;
	int slab;
	size_t ws;
};

inline Mx4Plan mx4_plan(int nq, int n, int k)
{
	Mx4Plan p{};
	auto up = [](size_t b) { return (b + 255) & ~(size_t)255; };
	p.chunks = nq <= kMx4ChunkQ;
	if (p.chunks) {
		int64_t c = ((int64_t)n + 511) / 512;  // about two workgroups a compute unit
		c = (c + 127) / 128 * 128;
		p.chunk = (int)(c < 512 ? 512 : c > kMx4ChunkRows ? kMx4ChunkRows : c);
		p.parts = (int)(((int64_t)n + p.chunk - 1) / p.chunk);
		p.ws = up((size_t)nq * p.parts * k * 8 + 8);
		return p;
	}
	const int64_t tiles = ((int64_t)n + 63) / 64;
	// k (ratio - 1) keys are expected of a level: at most a quarter of the buffer
	const int most = kMx4Cap / 4 / k < 4 ? 4 : kMx4Cap / 4 / k > 10 ? 10 : kMx4Cap / 4 / k;
	p.levels = 0;
	p.ratio = 0;
	p.step0 = 1;
	if (tiles > kMx4FirstTiles) {
		for (p.levels = 1;; p.levels++) {
			for (p.ratio = 2; p.ratio <= most; p.ratio++) {
				p.step0 = 1;
				for (int l = 0; l < p.levels; l++) p.step0 *= p.ratio;
				if (p.step0 * kMx4FirstTiles >= tiles) break;
			}
			if (p.ratio <= most) break;
		}
	}
	p.first_rows = (int)((tiles + p.step0 - 1) / p.step0) * 64;
	p.slab = nq < kMx4SlabQ ? nq : kMx4SlabQ;
	p.ws = up((size_t)p.slab * kMx4Cap * 8) + up((size_t)p.slab * 8) + 2 * up((size_t)p.slab * 4) + up((size_t)p.slab * p.first_rows * 4 + 4);
	return p;
}

size_t mx4_scan_workspace(int nq, int n, int k) { return mx4_plan(nq, n, k).ws; }

template <int KS, bool EXACT>
hipError_t mx4_scan_chunks(const Mx4Plan &p, const uint8_t *q, int nq, const uint8_t *rows, int n, int ksteps, int row_bytes, int k, const uint32_t *allow,
                           const Mx4Out &o, void *ws, hipStream_t s)
{
	mx4_key *keys = static_cast<mx4_key *>(ws);
	const int64_t stride = (int64_t)p.parts * k;
	const size_t lds = (size_t)nq * p.chunk * 4;
	static bool set[16] = {};
	int dev = 0;
	if (hipGetDevice(&dev) != hipSuccess) return hipErrorInvalidDevice;
	if (dev < 0 || dev >= 16 || !set[dev]) {
		const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(&mx4_chunk_kernel<KS, EXACT>), hipFuncAttributeMaxDynamicSharedMemorySize,
		                                         kMx4ChunkQ * kMx4ChunkRows * 4);
		if (e != hipSuccess) return e;
		if (dev >= 0 && dev < 16) set[dev] = true;
	}
	if (p.parts > 0)
		hipLaunchKernelGGL((mx4_chunk_kernel<KS, EXACT>), dim3(p.parts), dim3(256), lds, s, q, nq, rows, n, ksteps, row_bytes, k, p.chunk, allow, keys, stride);
	hipLaunchKernelGGL((mx4_pick_kernel<1024>), dim3(nq), dim3(1024), 0, s, keys, static_cast<const int32_t *>(nullptr), (int)stride, k, o,
	                   static_cast<int32_t *>(nullptr));
	return hipGetLastError();
}

template <int KS, bool EXACT>
hipError_t mx4_scan_levels(const Mx4Plan &p, const uint8_t *q, int nq, const uint8_t *rows, int n, int ksteps, int row_bytes, int k, const uint32_t *allow,
                           const Mx4Out &last, void *ws, hipStream_t s)
{
	auto up = [](size_t b) { return (b + 255) & ~(size_t)255; };
	uint8_t *w = static_cast<uint8_t *>(ws);
	Mx4Level a{};
	a.q = q;
	a.rows = rows;
	a.allow = allow;
	a.nq = nq;
	a.n = n;
	a.ksteps = ksteps;
	a.row_bytes = row_bytes;
	a.keys = reinterpret_cast<mx4_key *>(w);
	w += up((size_t)p.slab * kMx4Cap * 8);
	mx4_key *bound = reinterpret_cast<mx4_key *>(w);
	w += up((size_t)p.slab * 8);
	a.bound = bound;
	a.fill = reinterpret_cast<int32_t *>(w);
	w += up((size_t)p.slab * 4);
	int32_t *over = reinterpret_cast<int32_t *>(w);
	w += up((size_t)p.slab * 4);
	float *scores = reinterpret_cast<float *>(w);
	const Mx4Out mid = {nullptr, nullptr, nullptr, a.keys, bound, a.fill};
	const int m = p.first_rows;
	hipError_t e = mx4_launch_product_tiles(q, nq, rows, n, m, p.step0, ksteps, row_bytes, scores, m, s);
	if (e != hipSuccess) return e;
	hipLaunchKernelGGL(mx4_pick_first_kernel, dim3(nq), dim3(256), 0, s, scores, m, p.step0, n, k, allow, p.levels ? mid : last, (int64_t)kMx4Cap, over);
	const int64_t tiles = ((int64_t)n + 63) / 64;
	a.ratio = p.ratio;
	a.step = p.step0;
	const int qgroups = (nq + 63) / 64;
	for (int l = 1; l <= p.levels; l++) {
		const int64_t before = (tiles + a.step - 1) / a.step;
		a.step /= p.ratio;
		a.tiles = (int)((tiles + a.step - 1) / a.step - before);
		if (a.tiles > 0) {
			int64_t waves = 2 * (int64_t)a.tiles * qgroups;
			if (waves > 2048) waves = 2048;
			int64_t per = (waves + qgroups - 1) / qgroups;  // waves a query group
			const int64_t blocks = (per * qgroups + 3) / 4;
			hipLaunchKernelGGL((mx4_stream_kernel<KS, EXACT>), dim3((unsigned)blocks), dim3(256), 0, s, a, qgroups);
		}
		hipLaunchKernelGGL((mx4_pick_kernel<256>), dim3(nq), dim3(256), 0, s, a.keys, a.fill, kMx4Cap, k, l < p.levels ? mid : last, over);
	}
	if (p.levels)
		hipLaunchKernelGGL((mx4_rescue_kernel<KS, EXACT>), dim3(nq < 512 ? nq : 512), dim3(256), 0, s, a, k, over, last);
	return hipGetLastError();
}

hipError_t mx4_launch_scan(const uint8_t *q, int nq, const uint8_t *rows, int n, int dim, int k, const uint32_t *allow, int32_t *out_ids,
                           float *out_val, int32_t *out_count, void *ws, hipStream_t s)
{
	const Mx4Plan p = mx4_plan(nq, n, k);
	const int rb = mx4_row_bytes(dim), ks = mx4_blocks(dim) / 2;
	const int slab = p.chunks ? nq : p.slab;
	for (int64_t q0 = 0; q0 < nq; q0 += slab) {
		const int m = (int)(nq - q0 < slab ? nq - q0 : slab);
		Mx4Out o{};
		o.ids = out_ids + q0 * k;
		o.val = out_val + q0 * k;
		o.count = out_count + q0;
		hipError_t e = hipErrorInvalidValue;
		auto go = [&](auto steps, auto exact) {
			constexpr int KS = decltype(steps)::value;
			constexpr bool EXACT = decltype(exact)::value;
			e = p.chunks ? mx4_scan_chunks<KS, EXACT>(p, q + q0 * rb, m, rows, n, ks, rb, k, allow, o, ws, s)
			             : mx4_scan_levels<KS, EXACT>(p, q + q0 * rb, m, rows, n, ks, rb, k, allow, o, ws, s);
		};
		using std::integral_constant;
		switch (ks) {
		case 1: go(integral_constant<int, 1>{}, std::true_type{}); break;
		case 2: go(integral_constant<int, 2>{}, std::true_type{}); break;
		case 3: go(integral_constant<int, 3>{}, std::true_type{}); break;
		case 4: go(integral_constant<int, 4>{}, std::true_type{}); break;
		case 5: go(integral_constant<int, 5>{}, std::true_type{}); break;
		case 6: go(integral_constant<int, 6>{}, std::true_type{}); break;
		case 7: go(integral_constant<int, 7>{}, std::true_type{}); break;
		case 8: go(integral_constant<int, 8>{}, std::true_type{}); break;
		case 9: case 10: case 11: go(integral_constant<int, 12>{}, std::false_type{}); break;
		case 12: go(integral_constant<int, 12>{}, std::true_type{}); break;
		case 13: case 14: case 15: go(integral_constant<int, 16>{}, std::false_type{}); break;
		case 16: go(integral_constant<int, 16>{}, std::true_type{}); break;
		default: break;
		}
		if (e != hipSuccess) return e;
	}
	return hipSuccess;
}

}  // namespace mvdb
