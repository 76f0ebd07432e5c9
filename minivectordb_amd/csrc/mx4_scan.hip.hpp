// mx4_scan.hip.hpp -- the k largest dot products of each packed query with the packed rows (format: mx4.hpp).
//
// Order: value descending, then id ascending.  A candidate is one 64-bit key, larger = earlier in that order: the value's bits made
// monotone in the upper half, ~id in the lower.  0 is no key (it would be a NaN with the sign bit).  Rows whose `allow` bit is not set
// and rows whose product is NaN are no candidates; a row is taken out by giving its blocks the scale 255, which makes every product NaN,
// and a NaN is never >= a bound.
//
// Two ways, by the number of queries (1 M rows x 384, k 10: 8 queries 56 us in chunks, 9 queries 72 us in levels, 64 queries 79 us):
//
// CHUNKS (up to 8 queries): a workgroup computes the products of its own run of rows, keeps them in LDS and picks the best k of each
// query there; a second launch picks the best k of those.  Every row is read once, and two launches are all there is.
//
// LEVELS (more): the 64-row tiles are taken in levels, each about `ratio` times the one before it.  All tiles stand in one order, tile
// p of it being tile (p M) mod T of the T there are, M near T / golden ratio and without a common divisor, and a level is a run of that order.
// The tiles seen up to any level are spread evenly over the store (mx4_spread), and a layout that repeats every so many tiles (pages dealt out
// in turn to tenants, one of which the filter keeps) is met at about its share in every level, where tiles at equal distances see all of it or nothing:
// 1 M x 384, every 8th tile allowed, 300 queries take 146 us, at equal distances 8.4 ms.  (Counted over 300 stores of up to 40 000 tiles and periods of up to
// 128: 1 to 2 % of the pairs are still too much for a level's lists, 15 to 21 % at equal distances.)  The price is 1 % at 4096 queries x 1 M x
// 512 and 3 % at 40 M rows, 8 GB that are no longer read from end to end.  After a level the k-th best key so far is a bound: k rows are at least that good,
// so only keys above it matter, and about k (ratio - 1) keys of the next level are, unless the next level is better than what was seen.
// Level 0 has no bound: it is one chunk.  From then on a lane whose product passes the bound appends it to a list of its own,
// which needs no atomics: a lane only ever sees one query a fragment, and what it takes at a stretch of the order lies far apart, so lists stay short.
// mx4_pick_kernel gathers a query's lists after every level and keeps the best k.  A list that overflows marks its query, and
// mx4_rescue_kernel does those over, one workgroup each.
#pragma once

#include <hip/hip_runtime.h>

#include <atomic>
#include <cmath>
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
constexpr int kMx4Best = 256;  // candidates that are put in order by counting, at most

struct __attribute__((aligned(16))) Mx4PickLds {
	mx4_key best[kMx4Best + 8];
	int hist[256];
	unsigned lo[16], hi[16];  // per wave
	int pick, above, in_bin, total, count;
};

// Barrier of the T threads that share a selection.  The LDS operations of one wave execute in order, so a wave alone needs none.
template <int T>
__device__ __forceinline__ void mx4_sync()
{
	if constexpr (T > 64)
		__syncthreads();
	else
		asm volatile("" ::: "memory");
}

// over the 64 lanes of a wave, by row shifts and broadcasts (no LDS): the largest value, and the inclusive prefix sum
template <int CTRL>
__device__ __forceinline__ unsigned mx4_dpp_max(unsigned x)
{
	const unsigned y = (unsigned)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xf, 0xf, false);
	return y > x ? y : x;
}
__device__ __forceinline__ unsigned mx4_wave_max(unsigned x)
{
	x = mx4_dpp_max<0x111>(x);
	x = mx4_dpp_max<0x112>(x);
	x = mx4_dpp_max<0x114>(x);
	x = mx4_dpp_max<0x118>(x);
	x = mx4_dpp_max<0x142>(x);
	x = mx4_dpp_max<0x143>(x);
	return (unsigned)__builtin_amdgcn_readlane((int)x, 63);
}
__device__ __forceinline__ int mx4_wave_scan(int x)
{
	x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);
	x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
	x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
	x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
	x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);
	x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
	return x;
}

// The bin, from above, of the need-th key in l.hist (wave 0): l.pick, the keys above it and in it, and all there are
__device__ __forceinline__ void mx4_find_bin(Mx4PickLds &l, int need, int lane)
{
	int c[4], sum = 0;  // lane l has the bins 255 - 4 l down to 252 - 4 l
#pragma unroll
	for (int j = 0; j < 4; j++) {
		c[j] = l.hist[255 - 4 * lane - j];
		sum += c[j];
	}
	const int upto = mx4_wave_scan(sum);
	int higher = upto - sum;
	if (lane == 63) l.total = upto;
#pragma unroll
	for (int j = 0; j < 4; j++) {
		if (higher < need && higher + c[j] >= need) {
			l.pick = 255 - 4 * lane - j;
			l.above = higher;
			l.in_bin = c[j];
		}
		higher += c[j];
	}
}

// The best of the keys that T threads (a workgroup, or a wave of one) hold, N a thread (0 = none): l.best[0 .. returned count), in no order, has the best
// min(k, keys) of them, and at most kMx4Best.  A histogram over 256 equal steps from the smallest value to the largest gives the step of the
// k-th key, and everything from that step up is the answer: the best of a few thousand products lie far apart, so that is a few keys more than k
// (and few atomics meet in a bin).  Where it is too many, or the values are not finite, the keys are looked at bit by bit instead, eight at a time
// from the highest in which the values differ, until few enough share the k-th key's.
// l.best is written before the last barrier in here; the caller's next one has to come before l is used again.
template <int T, int N>
__device__ int mx4_block_best(const mx4_key (&key)[N], int k, Mx4PickLds &l)
{
	const int tid = threadIdx.x & (T - 1), lane = tid & 63, wave = tid >> 6;
	unsigned hi = 0, nlo = 0;  // of the values: the largest, and the largest complement
#pragma unroll
	for (int j = 0; j < N; j++) {
		const unsigned v = (unsigned)(key[j] >> 32);
		hi = key[j] && v > hi ? v : hi;
		nlo = key[j] && ~v > nlo ? ~v : nlo;
	}
	hi = mx4_wave_max(hi);
	nlo = mx4_wave_max(nlo);
	if (lane == 0) {
		l.hi[wave] = hi;
		l.lo[wave] = nlo;
	}
	for (int i = tid; i < 256; i += T) l.hist[i] = 0;
	if (tid == 0) l.count = 0;
	mx4_sync<T>();
#pragma unroll
	for (int w = 0; w < T / 64; w++) {
		hi = l.hi[w] > hi ? l.hi[w] : hi;
		nlo = l.lo[w] > nlo ? l.lo[w] : nlo;
	}
	const float most = mx4_key_value((mx4_key)hi << 32), least = mx4_key_value((mx4_key)~nlo << 32), span = most - least;
	bool done = false;
	if (hi != 0 && span > 1e-30f && span < 3e38f) {
		const float scale = 255.f / span;  // (subtraction, product and conversion keep the order of the values)
		int bin[N];
#pragma unroll
		for (int j = 0; j < N; j++) {
			const float x = key[j] ? (mx4_key_value(key[j]) - least) * scale : -1.f;
			bin[j] = x < 255.f ? (int)x : 255;
			if (bin[j] >= 0) atomicAdd(&l.hist[bin[j]], 1);
		}
		mx4_sync<T>();
		if (wave == 0) mx4_find_bin(l, k, lane);
		mx4_sync<T>();
		const int from = l.total < k ? 0 : l.pick;
		if (l.total < k || l.above + l.in_bin <= kMx4Best) {
#pragma unroll
			for (int j = 0; j < N; j++)
				if (bin[j] >= from) l.best[atomicAdd(&l.count, 1)] = key[j];
			done = true;
		} else {
			mx4_sync<T>();
			for (int i = tid; i < 256; i += T) l.hist[i] = 0;
			mx4_sync<T>();
		}
	}
	if (!done) {
		const unsigned differ = hi ^ ~nlo;
		int top = hi == 0 || differ == 0 ? 32 : 64 - __builtin_clz(differ);  // bits [0, top) differ
		mx4_key from = hi == 0 || top == 64 ? 0 : (mx4_key)hi << 32 >> top << top;  // the bits above them
		int need = k, above = 0;
		while (true) {
			const int shift = top > 8 ? top - 8 : 0;
			const unsigned bins = 1u << (top - shift);
#pragma unroll
			for (int j = 0; j < N; j++)
				if (key[j] && (top == 64 || (key[j] >> top) == (from >> top))) atomicAdd(&l.hist[(unsigned)(key[j] >> shift) & (bins - 1)], 1);
			mx4_sync<T>();
			if (wave == 0) mx4_find_bin(l, need, lane);
			mx4_sync<T>();
			if (l.total < need) {  // fewer than k keys: all of them
				from = 1;
				break;
			}
			const int in_bin = l.in_bin;
			above += l.above;
			need -= l.above;
			from |= (mx4_key)l.pick << shift;
			top = shift;
			if (above + in_bin <= kMx4Best || shift == 0) break;
			mx4_sync<T>();
			for (int i = tid; i < 256; i += T) l.hist[i] = 0;
			mx4_sync<T>();
		}
#pragma unroll
		for (int j = 0; j < N; j++)
			if (key[j] && key[j] >= from) l.best[atomicAdd(&l.count, 1)] = key[j];
	}
	mx4_sync<T>();
	return l.count;
}

// What a selection does with the best k: the caller's arrays, or (a level that is not the last) kept for the next, with the k-th as its bound.
struct Mx4Out {
	int32_t *ids, *count;
	float *val;
	mx4_key *keys, *bound;  // keys != nullptr: not the last level; [.][kMx4ScanMaxK]
	int32_t *fill;
};

// how many of the `have` keys in l.best (followed by zeros up to a multiple of 8) are larger
__device__ __forceinline__ int mx4_rank(const Mx4PickLds &l, int have, mx4_key key)
{
	int at = 0;
	for (int j = 0; j < have; j += 8) {
		ulonglong2 b[4];
#pragma unroll
		for (int i = 0; i < 4; i++) b[i] = *reinterpret_cast<const ulonglong2 *>(&l.best[j + 2 * i]);
#pragma unroll
		for (int i = 0; i < 4; i++) at += (b[i].x > key ? 1 : 0) + (b[i].y > key ? 1 : 0);
	}
	return at;
}
template <int T>
__device__ __forceinline__ void mx4_pad_best(Mx4PickLds &l, int have)
{
	const int tid = threadIdx.x & (T - 1);
	if (tid < 8) l.best[have + tid] = 0;
	mx4_sync<T>();
}

// The best k of the `have` keys in l.best to query q's place, in order: a key's place is the number of larger ones (no two are the same).
template <int T>
__device__ void mx4_block_put(int have, int k, int64_t q, const Mx4Out &o, Mx4PickLds &l)
{
	const int tid = threadIdx.x & (T - 1), out = have < k ? have : k;
	mx4_pad_best<T>(l, have);
	for (int i = tid; i < (have > k ? have : k); i += T) {
		mx4_key key = 0;
		int at = i;
		if (i < have) {
			key = l.best[i];
			at = mx4_rank(l, have, key);
			if (at >= k) continue;
		}
		if (o.keys) {
			if (i < have) o.keys[q * kMx4ScanMaxK + at] = key;
			if (i < have && at == k - 1) o.bound[q] = key;
		} else {
			o.ids[q * k + at] = i < have ? mx4_key_id(key) : -1;
			o.val[q * k + at] = i < have ? mx4_key_value(key) : 0.f;
		}
	}
	if (tid == 0) {
		if (o.keys) {
			o.fill[q] = out;
			if (out < k) o.bound[q] = 0;
		} else {
			o.count[q] = out;
		}
	}
}
// The best k of them, or fewer and zeros, in any order, to k places
template <int T>
__device__ void mx4_block_leave(int have, int k, mx4_key *dst, Mx4PickLds &l)
{
	const int tid = threadIdx.x & (T - 1);
	mx4_pad_best<T>(l, have);
	for (int i = tid; i < (have > k ? have : k); i += T) {
		const mx4_key key = i < have ? l.best[i] : 0;
		const int at = have > k ? mx4_rank(l, have, key) : i;
		if (at < k) dst[at] = key;
	}
}

// one workgroup per query: the best k of the `m` keys that the chunks left (0 = none), 7 x 1024 at a time beside the best so far.  Bound by its steps,
// each of which waits for the one before: 4.6 us for 4890 keys
__global__ __launch_bounds__(1024) void mx4_pick_chunks_kernel(const mx4_key *keys, int m, int k, Mx4Out o)
{
	__shared__ Mx4PickLds l;
	const int64_t q = blockIdx.x;
	const int tid = threadIdx.x;
	const mx4_key *mine = keys + q * m;
	int have = 0;
	for (int64_t base = 0; base < m; base += 7 * 1024) {
		mx4_key key[8];
#pragma unroll
		for (int j = 0; j < 7; j++) key[j] = base + j * 1024 + tid < m ? mine[base + j * 1024 + tid] : 0;
		key[7] = tid < have ? l.best[tid] : 0;
		__syncthreads();
		have = mx4_block_best<1024, 8>(key, k, l);
		__syncthreads();
	}
	mx4_block_put<1024>(have, k, q, o, l);
}

// What a list holds: keys, or (many queries) records of four neighbouring rows of which at least one may be a candidate: the first one's id, and the
// products (NaN: a row that does not count).
struct __attribute__((packed, aligned(4))) Mx4Record {
	float v[4];
	unsigned id;
};
__device__ __forceinline__ void mx4_keys_of(const mx4_key &r, mx4_key (&key)[1]) { key[0] = r; }
__device__ __forceinline__ void mx4_keys_of(const Mx4Record &r, mx4_key (&key)[4])
{
#pragma unroll
	for (int t = 0; t < 4; t++) key[t] = mx4_make_key(r.v[t], r.id + t);
}

// Keys of all lists of a query.  The plan sees to it that a random order of the rows stays far below them; what asks for more is a run of neighbouring
// rows that are all candidates and that the levels before have missed, at most about 64 x 2.7 ratio of them.
constexpr int kMx4Gather = 2048, kMx4GatherFewQueries = 4096;
constexpr int kMx4GatherWave = 768;  // the most that a wave deals with

// T threads per query (a workgroup, or a wave of one): the best k of what it had and of its lists, CAP keys in all.  Bound by its steps, each of
// which waits for the one before: 14 us for 333 queries with 512 lists and 1000 keys each, 9 us for 1000 with 256 and 90, 13 us for 4096 with 32 and 90
// (a wave each).
template <int T, int CAP, typename R, int LISTS, int P>
__global__ __launch_bounds__(256) void mx4_pick_kernel(const R *lists, const int32_t *counts, int parts, int list, const mx4_key *before,
                                                       const int32_t *nbefore, const mx4_key *bound, int nq, int k, Mx4Out o, int32_t *over)
{
	__shared__ Mx4PickLds ls[256 / T];
	__shared__ __attribute__((aligned(16))) mx4_key keyss[256 / T][CAP];
	__shared__ int totals[256 / T], losts[256 / T];
	const int tid = threadIdx.x & (T - 1), me = threadIdx.x / T;
	const int64_t q = (int64_t)blockIdx.x * (256 / T) + me;
	if (q >= nq) return;  // (T = 256: never; T = 64: whole waves, which share nothing)
	Mx4PickLds &l = ls[me];
	mx4_key *keys = keyss[me];
	int &total = totals[me], &lost = losts[me];
	mx4_key old[(kMx4ScanMaxK + T - 1) / T];  // loads that wait for nothing
#pragma unroll
	for (int j = 0; j < (kMx4ScanMaxK + T - 1) / T; j++) old[j] = j * T + tid < kMx4ScanMaxK ? before[q * kMx4ScanMaxK + j * T + tid] : 0;
	const int had = nbefore[q];
	const mx4_key beat = bound[q];  // (this kernel writes it, after the last of its threads has read it)
	if (tid == 0) {
		total = had;
		lost = 0;
	}
	mx4_sync<T>();
#pragma unroll
	for (int j = 0; j < (kMx4ScanMaxK + T - 1) / T; j++)
		if (j * T + tid < had) keys[j * T + tid] = old[j];
	// LISTS lists a thread at a time, and P records of each: loads that wait for nothing, as many as most lists hold
	constexpr int N = sizeof(R) == sizeof(mx4_key) ? 1 : 4;
	auto gather = [&](const R (&r)[P], int count) {
		mx4_key key[P][N];
		int n = 0;
#pragma unroll
		for (int j = 0; j < P; j++) {
			mx4_keys_of(r[j], key[j]);
#pragma unroll
			for (int t = 0; t < N; t++) {
				key[j][t] = j < count && (N == 1 || key[j][t] > beat) ? key[j][t] : 0;  // (a key that stands alone has been compared)
				n += key[j][t] ? 1 : 0;
			}
		}
		int at = atomicAdd(&total, n);
#pragma unroll
		for (int j = 0; j < P; j++)
#pragma unroll
			for (int t = 0; t < N; t++)
				if (key[j][t]) {
					if (at < CAP) keys[at] = key[j][t];
					at++;
				}
	};
	for (int i = tid; i < parts; i += LISTS * T) {
		const R *src[LISTS];
		R r[LISTS][P];
		int c[LISTS];
#pragma unroll
		for (int u = 0; u < LISTS; u++) {
			const int at = i + u * T < parts ? i + u * T : parts - 1;
			src[u] = lists + (q * parts + at) * list;
			c[u] = counts[q * parts + at];
#pragma unroll
			for (int j = 0; j < P; j++) r[u][j] = src[u][j];  // (a list has 32 places at least)
		}
#pragma unroll
		for (int u = 0; u < LISTS; u++) {
			if (i + u * T >= parts || c[u] == 0) continue;
			if (c[u] == list - 1) lost = 1;
			gather(r[u], c[u]);
			for (int at = P; at < c[u]; at += P) {
#pragma unroll
				for (int j = 0; j < P; j++) r[u][j] = src[u][at + j < c[u] ? at + j : at];
				gather(r[u], c[u] - at);
			}
		}
	}
	mx4_sync<T>();
	const int m = total < CAP ? total : CAP;
	if (tid == 0 && (lost || total > CAP)) over[q] = 1;
	mx4_key key[CAP / T];
#pragma unroll
	for (int j = 0; j < CAP / T; j++) key[j] = j * T + tid < m ? keys[j * T + tid] : 0;
	const int have = mx4_block_best<T>(key, k, l);
	mx4_block_put<T>(have, k, q, o, l);
}

// ---------------------------------------------------------------------------------------------- products of 32 rows
// acc[c] = the products of the 32 rows in `a` (rows of D) with the 32 queries in b[c]
template <int KS, int C>
__device__ __forceinline__ void mx4_tile(const Mx4Frag<KS> &a, const Mx4Frag<KS> (&b)[C], mx4_v16f (&acc)[C])
{
	const mx4_v16f zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
	for (int s = 0; s < KS; s++) {
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

// ---------------------------------------------------------------------------------------------- the order of the tiles
// Tile at place p of the order, (p M) mod T, from spread = ceil(2^64 M / T): p spread = 2^64 p M / T + e p with 0 <= e < 1, so its lower 64 bits are
// 2^64 ((p M) mod T) / T + e p, and times T / 2^64 that is (p M) mod T + e p T / 2^64: less than 1 more, as p and T are at most 2^25.
__device__ __forceinline__ unsigned mx4_tile_at(uint64_t spread, unsigned tiles, unsigned p)
{
	return (unsigned)__umul64hi(p * spread, (uint64_t)tiles);
}
// The tiles up to any place leave no gap of more than 2.7 times the mean one as long as the continued fraction of M / T has no large term.  The fraction
// of the golden ratio has none, but that of a whole M beside T / golden ratio is like it only in its first half: the first M from there on whose terms are
// at most 5 (6 are tried on average, 64 at most: then the best of them, of 7 in the worst of 300 T up to 40 000).  T >= 2.
inline uint64_t mx4_spread(uint32_t tiles)
{
	const uint32_t from = (uint32_t)(0.6180339887498949 * tiles);
	uint32_t best = 1, best_term = ~0u;
	for (uint32_t i = 0; i < 64 && best_term > 5; i++) {
		const uint32_t m = (i & 1) ? from - (i + 1) / 2 : from + i / 2;
		if (m == 0 || m >= tiles) continue;  // (what wraps below 0 is large)
		uint32_t a = tiles, b = m, term = 0;
		while (b) {
			const uint32_t t = a / b, c = a - t * b;
			term = t > term ? t : term;
			a = b;
			b = c;
		}
		if (a != 1 || term >= best_term) continue;
		best = m;
		best_term = term;
	}
	return (uint64_t)((((unsigned __int128)best << 64) + tiles - 1) / tiles);
}

// ---------------------------------------------------------------------------------------------- chunks
constexpr int kMx4ChunkQ = 8;        // queries of a workgroup
constexpr int kMx4ChunkRows = 2048;  // rows a workgroup, at most
constexpr int kMx4ChunkThreads = 512;
constexpr int64_t kMx4ChunkKeys = 1 << 17;  // keys that the chunks leave for a query, at most: one workgroup goes through them
static_assert(kMx4ChunkThreads / 64 >= kMx4ChunkQ, "a wave for each query");

// A wave takes 32 rows at a time, the next ones on their way meanwhile.  Queries are the columns of D, so with nq <= 8 of 32 columns used three
// quarters of the matrix work is for nothing: it is a few us at a million rows, against the reading of them:
// 33.6 us for 1 M x 384 and one query, 6.2 TB/s.  As level 0 of many queries every workgroup reads the same 2048 rows, 16 bytes of a row a lane, which
// fits an address path that takes a lane a cycle (counted, not measured): 21 us for 1000 queries, 45 us for 4096 (x 512).
template <int KS>
__global__ __launch_bounds__(kMx4ChunkThreads) void mx4_chunk_kernel(const uint8_t *q, int nq, const uint8_t *rows, int n, int k, int chunk,
                                                                     const uint32_t *allow, mx4_key *out, int64_t stride, uint64_t spread,
                                                                     unsigned tiles, Mx4Out o, int32_t *over, int qper)
{
	extern __shared__ __attribute__((aligned(16))) float sc[];  // [nq][chunk]
	__shared__ Mx4PickLds l[kMx4ChunkQ];
	constexpr int row_bytes = mx4_row_bytes(64 * KS);
	const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5, r32 = lane & 31;
	const int64_t first = (int64_t)blockIdx.x * chunk;
	const int64_t end = spread ? chunk : n - first;  // (tiles apart: the host gives as many as there are, one may end early)
	const int m = (int)(end < chunk ? end : chunk);
	const int qbase = blockIdx.y * qper;
	q += (int64_t)qbase * row_bytes;
	nq = nq - qbase < qper ? nq - qbase : qper;
	// row of place t, a multiple of 64 that all lanes agree on: rows in a run, or (spread, one workgroup for them all) the first tiles of the order
	auto row_of = [&](int t) -> int64_t { return spread ? (int64_t)mx4_tile_at(spread, tiles, (unsigned)t >> 6) * 64 : first + t; };
	Mx4Frag<KS> b[1], f0, f1;
	auto load = [&](int t, Mx4Frag<KS> &f) {
		const int64_t r = row_of(t & ~63) + (t & 32) + r32;
		mx4_load_frag<KS>(f, rows + (r < n ? r : n - 1) * row_bytes, half);
	};
	auto use = [&](int t, Mx4Frag<KS> &f) {
		mx4_shift_scales(f, half);
		mx4_v16f acc[1];
		mx4_tile<KS, 1>(f, b, acc);
		if (r32 < nq) {
#pragma unroll
			for (int g = 0; g < 4; g++) {
				const int at = t + 8 * g + 4 * half;
				float *o = sc + r32 * chunk + at;  // (chunk is a multiple of 4)
				if (at + 4 <= m) {
					*reinterpret_cast<float4 *>(o) = make_float4(acc[0][4 * g], acc[0][4 * g + 1], acc[0][4 * g + 2], acc[0][4 * g + 3]);
				} else {
#pragma unroll
					for (int j = 0; j < 3; j++)
						if (at + j < m) o[j] = acc[0][4 * g + j];
				}
			}
		}
	};
	constexpr int STEP = kMx4ChunkThreads / 2;  // 32 rows a wave
	int t = wave * 32;
	mx4_load_frag<KS>(b[0], q + (int64_t)(r32 < nq ? r32 : nq - 1) * row_bytes, half);
	if (t < m) load(t, f0);
	__builtin_amdgcn_sched_barrier(0);
	mx4_shift_scales(b[0], half);
	while (t < m) {
		if (t + STEP < m) load(t + STEP, f1);
		__builtin_amdgcn_sched_barrier(0);
		use(t, f0);
		t += STEP;
		if (t >= m) break;
		if (t + STEP < m) load(t + STEP, f0);
		__builtin_amdgcn_sched_barrier(0);
		use(t, f1);
		t += STEP;
	}
	__syncthreads();
	// One query at a time by the workgroup, or a query a wave: the first takes the less time for one or two, the second for more.
	auto pick = [&](auto threads, Mx4PickLds &l, int qi) {
		constexpr int T = decltype(threads)::value, N = kMx4ChunkRows / T;
		mx4_key key[N];
#pragma unroll
		for (int j = 0; j < N; j++) {
			const int at = j * T + (tid & (T - 1));
			key[j] = 0;
			if (j * T >= m) continue;
			const int64_t id = row_of(j * T + (T > 64 ? wave * 64 : 0)) + lane;
			const bool in = at < m && id < n && (!allow || ((allow[id >> 5] >> (id & 31)) & 1u));
			key[j] = in ? mx4_make_key(sc[qi * chunk + at], (unsigned)id) : 0;
		}
		const int have = mx4_block_best<T>(key, k, l);
		if (out) {  // one chunk of several
			mx4_block_leave<T>(have, k, out + (qbase + qi) * stride + (int64_t)blockIdx.x * k, l);
		} else {
			mx4_block_put<T>(have, k, qbase + qi, o, l);
			if (over && (tid & (T - 1)) == 0) over[qbase + qi] = 0;
		}
		mx4_sync<T>();
	};
	if (nq <= 2) {
		for (int qi = 0; qi < nq; qi++) pick(std::integral_constant<int, kMx4ChunkThreads>{}, l[0], qi);
	} else if (wave < nq) {
		pick(std::integral_constant<int, 64>{}, l[wave], wave);
	}
}

// ---------------------------------------------------------------------------------------------- levels
constexpr int kMx4FirstTiles = 32;  // 64-row tiles of level 0, at most
static_assert(kMx4FirstTiles * 64 <= kMx4ChunkRows, "level 0 is one chunk");

struct Mx4Level {
	const uint8_t *q, *rows;
	const uint32_t *allow;
	int nq, n;
	uint64_t spread;  // see mx4_tile_at
	unsigned all;     // tiles of the store
	unsigned first;   // place of the level's first tile in the order
	int each, more;   // tiles in a row that a wave pair (stream) or workgroup (stage) takes, the first `more` of them one more: tiles of
	                  // neighbouring rows, which may all hold candidates, are far apart in the order, so they go to different lists
	const mx4_key *bound;  // [nq], 0 = none
	void *lists;       // [nq][parts][list] keys or records
	int32_t *counts;   // [nq][parts] how many a list holds; list - 1: some may be lost
	int parts, list;
};

// tile i of a level, first row
__device__ __forceinline__ int64_t mx4_tile_row(const Mx4Level &a, unsigned i) { return (int64_t)mx4_tile_at(a.spread, a.all, a.first + i) * 64; }

// a word of the filter at a place that all lanes agree on, through the scalar cache (a vector load would wait for the LDS-DMA loads before it)
__device__ __forceinline__ uint32_t mx4_allow_word(const uint32_t *allow, int64_t at)
{
	using const_ptr_t = const __attribute__((address_space(4))) uint32_t *;
	return ((const_ptr_t)(allow))[at];
}

// Queries of a wave: C fragments of 32, and for each this lane's query, its bound and its list
template <int KS, int C>
struct Mx4Queries {
	Mx4Frag<KS> b[C];
	float bound[C];
	mx4_key bkey[C];
	unsigned at[C], last[C];  // byte offsets of the list's next place and of its last (at most 262 144 lists of a few KB: mx4_plan)
};

template <typename R, int KS, int C>
__device__ __forceinline__ void mx4_load_queries(Mx4Queries<KS, C> &w, const Mx4Level &a, int q0, int part, int half, int r32)
{
#pragma unroll
	for (int c = 0; c < C; c++) {
		const int q = q0 + c * 32 + r32, qs = q < a.nq ? q : a.nq - 1;
		mx4_load_frag<KS>(w.b[c], a.q + (int64_t)qs * mx4_row_bytes(64 * KS), half);
		mx4_shift_scales(w.b[c], half);
		w.bkey[c] = a.bound[qs];
		// no query in this column: nothing is >= NaN
		w.bound[c] = q >= a.nq ? __uint_as_float(0x7fc00000u) : w.bkey[c] ? mx4_key_value(w.bkey[c]) : -__builtin_inff();
		w.at[c] = ((unsigned)qs * a.parts + part) * a.list * (unsigned)sizeof(R);
		w.last[c] = w.at[c] + (a.list - 1) * (unsigned)sizeof(R);
	}
}
template <typename R, int KS, int C>
__device__ __forceinline__ void mx4_store_counts(const Mx4Queries<KS, C> &w, const Mx4Level &a, int q0, int part, int r32)
{
#pragma unroll
	for (int c = 0; c < C; c++)
		if (q0 + c * 32 + r32 < a.nq) a.counts[(int64_t)(q0 + c * 32 + r32) * a.parts + part] = a.list - 1 - (int)((w.last[c] - w.at[c]) / sizeof(R));
}

// the largest of four neighbouring products, and `top` and four more: one after the other, which is two instructions (v_max3_f32), where a tree of
// them is four to six (two, and the operands of the pairs made canonical)
__device__ __forceinline__ float mx4_most(float top, const mx4_v16f &acc, int g)
{
	return __builtin_fmaxf(__builtin_fmaxf(__builtin_fmaxf(__builtin_fmaxf(top, acc[4 * g]), acc[4 * g + 1]), acc[4 * g + 2]), acc[4 * g + 3]);
}
__device__ __forceinline__ float mx4_most(const mx4_v16f &acc, int g)
{
	return __builtin_fmaxf(__builtin_fmaxf(__builtin_fmaxf(acc[4 * g], acc[4 * g + 1]), acc[4 * g + 2]), acc[4 * g + 3]);
}

// Test of a lane's 16 products with each of its queries: the largest, and whether any may be a candidate.
template <int KS, int C>
__device__ __forceinline__ bool mx4_test(const Mx4Queries<KS, C> &w, const mx4_v16f (&acc)[C], float (&top)[C])
{
	bool any = false;
#pragma unroll
	for (int c = 0; c < C; c++) {
		top[c] = mx4_most(acc[c], 0);
#pragma unroll
		for (int g = 1; g < 4; g++) top[c] = mx4_most(top[c], acc[c], g);
		any |= top[c] >= w.bound[c];
	}
	return any;
}

// One more in this lane's list.  The last place of a list is written over and over, and its number says that some may be lost.
template <typename R, int KS, int C>
__device__ __forceinline__ void mx4_append_one(Mx4Queries<KS, C> &w, const Mx4Level &a, int c, const R &r)
{
	*reinterpret_cast<R *>(static_cast<char *>(a.lists) + w.at[c]) = r;
	const unsigned next = w.at[c] + (unsigned)sizeof(R);
	w.at[c] = next < w.last[c] ? next : w.last[c];
}

// Append what passed; rows row0 .. + 31.  As keys, one by one; or four products at a time, in one record, where which of them pass is found by
// mx4_pick_kernel.  Records take fewer instructions here, where they keep the matrix instructions waiting, and more there (1 M rows x 384, k 100:
// 1000 queries 316 us with keys, 288 with records); with few queries a wave has few candidates and mx4_pick_kernel many lists (64 queries: 104 and 127).
template <typename R, int KS, int C>
__device__ __forceinline__ void mx4_append(Mx4Queries<KS, C> &w, const Mx4Level &a, const mx4_v16f (&acc)[C], const float (&top)[C], int64_t row0, int half)
{
	unsigned id0 = (unsigned)row0 + 4 * half;
	asm volatile("" : "+v"(id0));  // the ids are formed here, where they are rarely wanted, not in the caller's loop
#pragma unroll
	for (int c = 0; c < C; c++) {
		if (!__ballot(top[c] >= w.bound[c])) continue;
#pragma unroll
		for (int g = 0; g < 4; g++) {
			const float m = mx4_most(acc[c], g);
			if (__ballot(m >= w.bound[c])) {
				if constexpr (sizeof(R) == sizeof(Mx4Record)) {
					// (an equal product behind the bound's id is no candidate: rows that are all alike fill no lists)
					const unsigned id = id0 + 8 * g;
					if ((m > w.bound[c]) | ((m >= w.bound[c]) & (~id > (unsigned)w.bkey[c])))
						mx4_append_one(w, a, c, Mx4Record{{acc[c][4 * g], acc[c][4 * g + 1], acc[c][4 * g + 2], acc[c][4 * g + 3]}, id});
				} else {
#pragma unroll
					for (int j = 0; j < 4; j++) {
						const float v = acc[c][4 * g + j];
						if (__ballot(v >= w.bound[c])) {
							const unsigned b = __float_as_uint(v + 0.f);  // mx4_make_key of a number
							const mx4_key key = ((mx4_key)(b ^ ((unsigned)((int)b >> 31) | 0x80000000u)) << 32) | ~(id0 + 8 * g + j);
							if (v >= w.bound[c] && key > w.bkey[c]) mx4_append_one(w, a, c, key);
						}
					}
				}
			}
		}
	}
}

// fragments of 32 queries a wave of the stream kernel holds
__host__ __device__ constexpr int mx4_stream_frags(int ks) { return ks <= 8 ? 2 : 1; }

// Independent waves: each holds 64 queries (32 where rows are long) and takes its half of a run of the level's tiles straight from memory, the next
// one's rows under way while it multiplies.  Bound by the reading of the rows up to 64 queries (9 queries: the last level of 1 M x 384 in 30 us), above
// by their reading once for every 64: 256 queries 76 us, where tiles shared in LDS take as long and cost more at their start.
template <int KS>
__global__ __launch_bounds__(256, 2) void mx4_stream_kernel(Mx4Level a, int qgroups)
{
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, r32 = lane & 31;
	const int gw = blockIdx.x * 4 + wave, group = gw % qgroups, first = gw / qgroups;
	if (first >= a.parts / 2) return;
	constexpr int row_bytes = mx4_row_bytes(64 * KS);
	constexpr int C = mx4_stream_frags(KS);
	Mx4Queries<KS, C> w;
	mx4_load_queries<mx4_key>(w, a, group * 32 * C, 2 * first + half, half, r32);
	const int pair = first >> 1, from = pair * a.each + (pair < a.more ? pair : a.more), total = a.each + (pair < a.more ? 1 : 0);
	// this wave's half of the pair's tile i: its first row and which of its rows count, and (unless none does) the rows
	auto load = [&](int i, Mx4Frag<KS> &f, int64_t &row0, unsigned &keep) {
		row0 = mx4_tile_row(a, from + i) + (first & 1) * 32;
		keep = 0;
		if (row0 >= a.n) return;
		keep = row0 + 32 <= a.n ? 0xffffffffu : (1u << (a.n - row0)) - 1u;
		if (a.allow) keep &= mx4_allow_word(a.allow, row0 >> 5);
		if (keep == 0) return;
		const int64_t r = row0 + r32 < a.n ? row0 + r32 : a.n - 1;
		mx4_load_frag<KS>(f, a.rows + r * row_bytes, half);
	};
	auto use = [&](Mx4Frag<KS> &f, int64_t row0, unsigned keep) {
		if (keep == 0) return;
		const bool out = !((keep >> r32) & 1u);
#pragma unroll
		for (int s = 0; s < (KS + 1) / 2; s++) f.sc[s] = out ? -1 : f.sc[s];
		mx4_shift_scales(f, half);
		mx4_v16f acc[C];
		mx4_tile<KS, C>(f, w.b, acc);
		float top[C];
		if (__builtin_expect(__ballot(mx4_test(w, acc, top)) != 0, 0)) mx4_append<mx4_key>(w, a, acc, top, row0, half);
	};
	if constexpr (KS <= 12) {
		Mx4Frag<KS> f0, f1;
		int64_t row0, row1;
		unsigned keep0 = 0, keep1 = 0;
		int i = 0;
		if (i < total) load(i, f0, row0, keep0);
		while (i < total) {
			keep1 = 0;
			if (i + 1 < total) load(i + 1, f1, row1, keep1);
			__builtin_amdgcn_sched_barrier(0);
			use(f0, row0, keep0);
			if (++i >= total) break;
			keep0 = 0;
			if (i + 1 < total) load(i + 1, f0, row0, keep0);
			__builtin_amdgcn_sched_barrier(0);
			use(f1, row1, keep1);
			i++;
		}
	} else {
		for (int i = 0; i < total; i++) {
			Mx4Frag<KS> f;
			int64_t row0;
			unsigned keep;
			load(i, f, row0, keep);
			use(f, row0, keep);
		}
	}
	mx4_store_counts<mx4_key>(w, a, group * 32 * C, 2 * first + half, r32);
}

// Tiles of 64 rows, staged in LDS for up to 8 waves of 64 queries each.  Groups of tiles come by LDS-DMA into two places in turn: while one group is
// worked on the tiles of the next are asked for, one after the other.  One barrier a group: a wave that appends keeps the others waiting there, the
// less the further the barriers are apart (4096 queries, 900 000 x 512, 168 candidates a query: barriers 1 tile apart 960 us, 2 tiles 880 us).
// An image row is the packed row, plus one slot of 16 bytes where that makes the stride an odd number of slots: then the 16 lanes that an LDS read
// serves at a time hit 16 different slots.  Two waves a SIMD.  4096 queries, 900 000 x 512: 728-746 us, 5.1 PFLOP/s (this card sustains 6.6 on random
// operands); 1000 queries, x 384: 167 us, 4.2 PFLOP/s.
static __device__ __align__(16) int g_mx4_nan[4] = {-1, -1, -1, -1};  // scales 255: the blocks of a row that is left out

__host__ __device__ constexpr int mx4_image_slots(int row_bytes) { return (row_bytes / 16) | 1; }

// tiles of a group (a power of two): as many as LDS has room for twice
__host__ __device__ constexpr int mx4_stage_group(int ks) { return ks <= 8 ? 4 : 2; }
__host__ __device__ constexpr size_t mx4_stage_lds(int ks) { return (size_t)2 * mx4_stage_group(ks) * mx4_image_slots(mx4_row_bytes(64 * ks)) * 1024; }

template <int KS>
__global__ __launch_bounds__(512, 2) void mx4_stage_kernel(Mx4Level a, int qtiles)
{
	extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, r32 = lane & 31;
	const int nwaves = blockDim.x >> 6;
	// blocks with equal blockIdx % 8 share an XCD and its L2: they take the same tiles for their different queries
	const int j8 = blockIdx.x >> 3, qtile = j8 % qtiles;
	const int split = (blockIdx.x & 7) + 8 * (j8 / qtiles);
	constexpr int row_bytes = mx4_row_bytes(64 * KS);
	const int slots = row_bytes / 16, islots = slots | 1;
	const int tile_bytes = islots * 64 * 16;
	constexpr int G = mx4_stage_group(KS);
	const int q0 = (qtile * nwaves + wave) * 64;
	Mx4Queries<KS, 2> w;
	mx4_load_queries<Mx4Record>(w, a, q0, 2 * split + half, half, r32);
	const int from = split * a.each + (split < a.more ? split : a.more), ntiles = a.each + (split < a.more ? 1 : 0);

	using lds_ptr_t = __attribute__((address_space(3))) void *;
	using glb_ptr_t = __attribute__((address_space(1))) const void *;
	// this wave's share of tile t: instructions wave, wave + nwaves, ... of islots, 64 slots of 16 bytes each
	auto fetch = [&](int t) {
		const int64_t row0 = mx4_tile_row(a, from + t);
		const uint8_t *base = a.rows + row0 * row_bytes;
		unsigned char *dst = lds + (t & (2 * G - 1)) * tile_bytes;
		if (islots == slots && !a.allow && row0 + 64 <= a.n) {  // the image is the tile as it lies in memory
			for (int i = wave; i < islots; i += nwaves)
				__builtin_amdgcn_global_load_lds((glb_ptr_t)(base + i * 1024 + (unsigned)lane * 16), (lds_ptr_t)(dst + i * 1024), 16, 0, 0);
			return;
		}
		uint64_t keep = row0 + 64 <= a.n ? ~0ull : (1ull << (a.n - row0)) - 1;
		if (a.allow) {
			const uint64_t lo = mx4_allow_word(a.allow, row0 >> 5), hi = row0 + 32 < a.n ? mx4_allow_word(a.allow, (row0 >> 5) + 1) : 0u;
			keep &= lo | (hi << 32);
		}
		for (int i = wave; i < islots; i += nwaves) {
			const int slot = i * 64 + lane;
			const int r = slot / islots, pos = slot - r * islots;
			const void *src = base + (r * slots + (pos < slots ? pos : 0)) * 16;
			// a row that is left out has scales 255; past the last row nothing is read
			const bool off = !((keep >> r) & 1) && (pos >= 2 * KS || row0 + r >= a.n);
			src = off ? static_cast<const void *>(g_mx4_nan) : src;
			__builtin_amdgcn_global_load_lds((glb_ptr_t)src, (lds_ptr_t)(dst + i * 1024), 16, 0, 0);
		}
	};
	auto image = [&](int t, int h) -> const unsigned char * { return lds + (t & (2 * G - 1)) * tile_bytes + (h * 32 + r32) * islots * 16; };
	for (int t = 0; t < G && t < ntiles; t++) fetch(t);
	constexpr bool AHEAD = KS <= 8;  // room in the registers for the fragments of the next 32 rows
	Mx4Frag<KS> f0, f1;
	constexpr bool PIPED = KS <= 12;
	// Two sets of accumulators (where there is room): the products of one 32 rows are tested while those of the next are computed.
	mx4_v16f accA[2], accB[2];
#pragma unroll
	for (int c = 0; c < 2; c++)
#pragma unroll
		for (int i = 0; i < 16; i++) accB[c][i] = __uint_as_float(0x7fc00000u);
	int64_t rowB = 0;
	auto step = [&](Mx4Frag<KS> &f, mx4_v16f (&now)[2], mx4_v16f (&then)[2], int64_t row) {
		mx4_shift_scales(f, half);
		if constexpr (!PIPED) {
			mx4_tile<KS, 2>(f, w.b, now);
			float top[2];
			if (__builtin_expect(__ballot(mx4_test(w, now, top)) != 0, 0)) mx4_append<Mx4Record>(w, a, now, top, row, half);
			return;
		}
		const mx4_v16f zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
		float top[2];
#pragma unroll
		for (int s = 0; s < KS; s++) {
#pragma unroll
			for (int c = 0; c < 2; c++) {
				const mx4_v16f &in = s == 0 ? zero : now[c];
				now[c] = (s & 1) ? mx4_mfma<2, 2>(f.d[s], f.sc[s / 2], w.b[c].d[s], w.b[c].sc[s / 2], in)
				                 : mx4_mfma<0, 0>(f.d[s], f.sc[s / 2], w.b[c].d[s], w.b[c].sc[s / 2], in);
			}
			__builtin_amdgcn_sched_barrier(0);
#pragma unroll
			for (int p = s * 8 / KS; p < (s + 1) * 8 / KS; p++) {  // a share of the test behind every two matrix instructions
				const int c = p >> 2, g = p & 3;
				top[c] = g == 0 ? mx4_most(then[c], 0) : mx4_most(top[c], then[c], g);
			}
			__builtin_amdgcn_sched_barrier(0);
		}
#pragma unroll
		for (int c = 0; c < 2; c++) asm volatile("" : "+v"(now[c]));  // see mx4_tile
		bool any = false;
#pragma unroll
		for (int c = 0; c < 2; c++) any |= top[c] >= w.bound[c];
		if (__builtin_expect(__ballot(any) != 0, 0)) mx4_append<Mx4Record>(w, a, then, top, row, half);
	};
	for (int t = 0; t < ntiles; t += G) {
		asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's share of the group is there ...
		__builtin_amdgcn_s_barrier();                     // ... and everybody's, and the group before it is done with
		asm volatile("" ::: "memory");
		if (AHEAD) mx4_load_frag<KS>(f0, image(t, 0), half);
		for (int u = t; u < t + G && u < ntiles; u++) {
			if (u + G < ntiles) fetch(u + G);
			const int64_t row0 = mx4_tile_row(a, from + u);
			if (!AHEAD) mx4_load_frag<KS>(f0, image(u, 0), half);
			if (AHEAD) {
				mx4_load_frag<KS>(f1, image(u, 1), half);
				__builtin_amdgcn_sched_barrier(0);
			}
			step(f0, accA, accB, PIPED ? rowB : row0);
			if (!AHEAD) mx4_load_frag<KS>(f1, image(u, 1), half);
			if (AHEAD) {
				mx4_load_frag<KS>(f0, image(u + 1, 0), half);  // (behind the group's last tile: never used)
				__builtin_amdgcn_sched_barrier(0);
			}
			step(f1, PIPED ? accB : accA, accA, PIPED ? row0 : row0 + 32);
			rowB = row0 + 32;
		}
		asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this wave's reads of the tiles are done before it passes the next barrier
	}
	if (PIPED) {
		float top[2];
		if (__ballot(mx4_test(w, accB, top))) mx4_append<Mx4Record>(w, a, accB, top, rowB, half);
	}
	mx4_store_counts<Mx4Record>(w, a, q0, 2 * split + half, r32);
}

// (by value: `first ? x[1] : x[0]` is a place in memory)
__device__ __forceinline__ float mx4_select(bool first, float a, float b) { return first ? a : b; }

// The queries that lost keys, from the beginning: a workgroup for each, 128 rows at a time, candidates gathered in LDS and cut
// to the best k when the next 128 might not fit; from then on what is below all that were kept is none.  Bound by its steps, 0.6
// to 0.7 us for 128 rows (300 queries, 96 000 x 64, all of them done over: 0.46 ms; without that bound, and one lane going through the products,
// 2.98 ms).  Beside queries that fit it is a cliff: one of 300 at 1 M x 384 makes 146 us 5.5 ms, all of them 6.0 ms.  With a filter groups of 128 rows none
// of which may be returned are passed over (one page of 1024 rows in 8 allowed: 8.5 ms for all 300 without that, 1.5 ms with), and without one there is no
// test for it (a test at run time instead of two kernels: 6.5 ms for the 6.0).
template <int KS, bool FILTER>
__global__ __launch_bounds__(256) void mx4_rescue_kernel(Mx4Level a, int k, const int32_t *over, Mx4Out o)
{
	__shared__ Mx4PickLds l;
	__shared__ mx4_key keys[kMx4Gather];
	__shared__ mx4_key least;  // of those that were kept, if that is k
	__shared__ int count;
	const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, r32 = lane & 31;
	for (int q = blockIdx.x; q < a.nq; q += gridDim.x) {
		if (!over[q]) continue;
		Mx4Frag<KS> b[1];
		mx4_load_frag<KS>(b[0], a.q + (int64_t)q * mx4_row_bytes(64 * KS), half);
		mx4_shift_scales(b[0], half);
		int have = 0;
		if (tid == 0) {
			count = 0;
			least = 0;
		}
		__syncthreads();
		auto load = [&](int64_t row0, Mx4Frag<KS> &f) {
			const int64_t r = row0 + r32 < a.n ? row0 + r32 : a.n - 1;
			mx4_load_frag<KS>(f, a.rows + r * mx4_row_bytes(64 * KS), half);
		};
		// With a filter, groups of 128 rows none of which may be returned are passed over: bit i of `some` says that group i of the 64 from row
		// `from` on has one and has not been dealt with.
		int64_t from = FILTER ? -64 * 128 : -128;
		uint64_t some = 0;
		auto step = [&]() -> int64_t {  // the next 128 rows, or past the last
			if constexpr (!FILTER) return from += 128;
			while (some == 0) {
				from += 64 * 128;
				if (from >= a.n) return a.n;
				const int64_t at = from + lane * 128;
				bool any = false;
#pragma unroll
				for (int i = 0; i < 4; i++)
					if (at + 32 * i < a.n) any |= a.allow[(at >> 5) + i] != 0;
				some = __ballot(any);
			}
			const int bit = __builtin_ctzll(some);
			some &= some - 1;
			return from + bit * 128;
		};
		Mx4Frag<KS> f, next;
		int64_t base = step();
		load(base + wave * 32, next);
		while (base < a.n) {
			const int64_t row0 = base + wave * 32;
			f = next;
			base = step();
			load(base + wave * 32, next);
			if (row0 < a.n) {
				mx4_shift_scales(f, half);
				mx4_v16f acc[1];
				mx4_tile<KS, 1>(f, b, acc);
				// every column holds the same query: column i < 16 deals with the i-th of its products
				float v = acc[0][0];
#pragma unroll
				for (int i = 1; i < 16; i++) v = mx4_select(r32 == i, acc[0][i], v);
				const int64_t id = row0 + 8 * (r32 >> 2) + 4 * half + (r32 & 3);
				if (r32 < 16 && id < a.n && (!FILTER || ((a.allow[id >> 5] >> (id & 31)) & 1u))) {
					const mx4_key key = mx4_make_key(v, (unsigned)id);
					if (key > least) keys[atomicAdd(&count, 1)] = key;
				}
			}
			__syncthreads();
			if (count > kMx4Gather - 128 || base >= a.n) {  // cut to the best
				mx4_key key[kMx4Gather / 256];
#pragma unroll
				for (int j = 0; j < kMx4Gather / 256; j++) key[j] = j * 256 + tid < count ? keys[j * 256 + tid] : 0;
				__syncthreads();
				if (tid == 0) least = ~(mx4_key)0;
				have = mx4_block_best<256>(key, k, l);
				for (int j = tid; j < have; j += 256) {
					keys[j] = l.best[j];
					if (have >= k) atomicMin(&least, l.best[j]);
				}
				if (tid == 0) {
					count = have;
					if (have < k) least = 0;
				}
			}
			__syncthreads();
		}
		mx4_block_put<256>(have, k, q, o, l);
		__syncthreads();
	}
}

// ---------------------------------------------------------------------------------------------- the plan
constexpr int kMx4SlabQ = 8192;       // queries that are dealt with at a time
constexpr int kMx4StreamGroups = 4;   // up to so many groups of 64 queries: mx4_stream_kernel, more: mx4_stage_kernel
constexpr int kMx4StreamWaves = 2048;
constexpr int kMx4MostRatio = 10, kMx4MostRatioFew = 52;  // many queries: 4 to 14 are within 3 %; few: a candidate costs little against a launch

struct Mx4Plan {
	bool chunks, few;  // few: keys that a query gathers in a level
	int chunk, parts, list;  // chunks: rows of one, how many; levels: lists of a query, places of a list
	int levels, ratio, first_rows;  // levels after level 0; rows of level 0 (a multiple of 64)
	int64_t step0;  // ratio^levels: one in so many tiles is in level 0
	int slab, qgroups, qtiles, splits, record;  // record: bytes of what a list holds
	size_t ws;
};

inline size_t mx4_up(size_t b) { return (b + 255) & ~(size_t)255; }

inline Mx4Plan mx4_plan(int nq, int n, int dim, int k)
{
	Mx4Plan p{};
	// about two workgroups a compute unit
	const int64_t c = (((int64_t)n + 511) / 512 + 127) / 128 * 128;
	p.chunk = (int)(c < 512 ? 512 : c > kMx4ChunkRows ? kMx4ChunkRows : c);
	p.parts = (int)(((int64_t)n + p.chunk - 1) / p.chunk);
	p.chunks = nq <= kMx4ChunkQ && (int64_t)p.parts * k <= kMx4ChunkKeys;
	if (p.chunks) {
		p.ws = mx4_up((size_t)nq * p.parts * k * 8 + 8);
		return p;
	}
	p.slab = nq < kMx4SlabQ ? nq : kMx4SlabQ;
	p.qgroups = (p.slab + 63) / 64;
	const int64_t tiles = ((int64_t)n + 63) / 64;
	// The rows of a level that beat the bound are about ratio x Gamma(k) in number, if the levels are alike: more than ratio (k + 6 sqrt(k) + 12)
	// about once in 10^9 queries, and that many a query can gather
	const bool many = p.qgroups > kMx4StreamGroups;
	int most = many ? kMx4MostRatio : kMx4MostRatioFew;
	auto gathered = [&](int ratio) { return ratio * (k + 6 * std::sqrt((double)k) + 12); };
	while (most > 4 && gathered(most) > kMx4Gather) most--;
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
	p.few = nq >= 2048 && gathered(p.ratio) <= kMx4GatherWave - 256;  // (by waves instead of workgroups, 30 000 and 300 000 rows, a whole scan:
	// 1000 queries 11 to 15 % slower, 1400 5 to 8, 1800 1 to 4 faster, 4096 7 to 12)
	p.first_rows = (int)((tiles + p.step0 - 1) / p.step0) * 64;
	if (many) {
		p.qtiles = (p.qgroups + 7) / 8;
		// 8 x qtiles workgroups at a time: one a compute unit, as long as there is a tile for each
		const int64_t most_splits = 8 * (32 / p.qtiles < 1 ? 1 : 32 / p.qtiles), some = (tiles + 7) / 8 * 8;
		p.splits = (int)(some < 8 ? 8 : some < most_splits ? some : most_splits);
	} else {
		const int wide = 32 * mx4_stream_frags(mx4_blocks(dim) / 2);
		p.qgroups = (p.slab + wide - 1) / wide;
		const int64_t most_waves = kMx4StreamWaves / p.qgroups;
		p.splits = (int)(2 * tiles < most_waves ? (tiles ? 2 * tiles : 2) : most_waves & ~1);  // (waves, in pairs)
	}
	p.parts = 2 * p.splits;
	// a list's share of a level's candidates, with the same margin, and room for neighbouring rows that are all candidates, three tiles of them in
	// records and two in keys; whole cache lines, so that the first few lie in one
	const double share = (double)k * (p.ratio > 1 ? p.ratio - 1 : 0) / p.parts;
	const int least = (int)(share + 6 * std::sqrt(share)) + (many ? 25 : 60), line = many ? 32 : 16;
	p.list = (least + line - 1) / line * line;
	p.record = many ? sizeof(Mx4Record) : sizeof(mx4_key);
	p.ws = mx4_up((size_t)p.slab * kMx4ScanMaxK * 8) + mx4_up((size_t)p.slab * 8) + 2 * mx4_up((size_t)p.slab * 4);
	if (p.levels) p.ws += mx4_up((size_t)p.slab * p.parts * 4) + mx4_up((size_t)p.slab * p.parts * p.list * p.record);
	return p;
}

size_t mx4_scan_workspace(int nq, int n, int dim, int k) { return mx4_plan(nq, n, dim, k).ws; }

// once per kernel and device: how much LDS a launch may ask for
template <int KS, int WHICH>
struct Mx4Mark {
	static inline std::atomic<bool> set[16] = {};
};
inline hipError_t mx4_allow_lds(const void *fn, int bytes, std::atomic<bool> (&set)[16])
{
	int dev = 0;
	if (hipGetDevice(&dev) != hipSuccess) return hipErrorInvalidDevice;
	const bool known = dev >= 0 && dev < 16;
	if (known && set[dev].load(std::memory_order_relaxed)) return hipSuccess;
	const hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
	if (e == hipSuccess && known) set[dev].store(true, std::memory_order_relaxed);
	return e;
}

template <int KS>
hipError_t mx4_scan_chunks(const Mx4Plan &p, const uint8_t *q, int nq, const uint8_t *rows, int n, int k, const uint32_t *allow,
                           const Mx4Out &o, void *ws, hipStream_t s)
{
	mx4_key *keys = static_cast<mx4_key *>(ws);
	const int64_t stride = (int64_t)p.parts * k;
	const size_t lds = (size_t)nq * p.chunk * 4;
	const hipError_t e = mx4_allow_lds(reinterpret_cast<const void *>(&mx4_chunk_kernel<KS>), kMx4ChunkQ * kMx4ChunkRows * 4, Mx4Mark<KS, 0>::set);
	if (e != hipSuccess) return e;
	if (p.parts > 0)
		hipLaunchKernelGGL((mx4_chunk_kernel<KS>), dim3(p.parts, 1), dim3(kMx4ChunkThreads), lds, s, q, nq, rows, n, k, p.chunk, allow, keys, stride, (uint64_t)0,
		                   0u, Mx4Out{}, static_cast<int32_t *>(nullptr), kMx4ChunkQ);
	hipLaunchKernelGGL(mx4_pick_chunks_kernel, dim3(nq), dim3(1024), 0, s, keys, (int)stride, k, o);
	return hipGetLastError();
}

template <int KS>
hipError_t mx4_scan_levels(const Mx4Plan &p, const uint8_t *q, int nq, const uint8_t *rows, int n, int k, const uint32_t *allow,
                           const Mx4Out &last, void *ws, hipStream_t s)
{
	uint8_t *w = static_cast<uint8_t *>(ws);
	auto take = [&](size_t bytes) -> void * {
		void *at = w;
		w += mx4_up(bytes);
		return at;
	};
	mx4_key *best = static_cast<mx4_key *>(take((size_t)p.slab * kMx4ScanMaxK * 8));
	mx4_key *bound = static_cast<mx4_key *>(take((size_t)p.slab * 8));
	int32_t *nbest = static_cast<int32_t *>(take((size_t)p.slab * 4));
	int32_t *over = static_cast<int32_t *>(take((size_t)p.slab * 4));
	Mx4Level a{};
	a.q = q;
	a.rows = rows;
	a.allow = allow;
	a.nq = nq;
	a.n = n;
	a.bound = bound;
	a.parts = p.parts;
	if (p.levels) {
		a.all = (unsigned)(((int64_t)n + 63) / 64);
		a.spread = mx4_spread(a.all);
		a.counts = static_cast<int32_t *>(take((size_t)p.slab * p.parts * 4));
		a.list = p.list;
		a.lists = take((size_t)p.slab * p.parts * p.list * p.record);
	}
	const Mx4Out mid = {nullptr, nullptr, nullptr, best, bound, nbest};
	const bool stage = p.qtiles > 0;
	const int nwaves = stage ? (p.qgroups + p.qtiles - 1) / p.qtiles : 0;
	constexpr size_t lds = mx4_stage_lds(KS);
	static_assert(lds <= 160 * 1024, "LDS of a compute unit");
	hipError_t e = hipSuccess;
	if (p.levels && stage)
		e = mx4_allow_lds(reinterpret_cast<const void *>(&mx4_stage_kernel<KS>), (int)lds,
		                  Mx4Mark<KS, 1>::set);
	if (e == hipSuccess)
		e = mx4_allow_lds(reinterpret_cast<const void *>(&mx4_chunk_kernel<KS>), kMx4ChunkQ * kMx4ChunkRows * 4, Mx4Mark<KS, 0>::set);
	if (e != hipSuccess) return e;
	const int qper = nq >= 256 * kMx4ChunkQ ? kMx4ChunkQ : (nq + 255) / 256;  // a workgroup for every compute unit if there are queries enough
	hipLaunchKernelGGL((mx4_chunk_kernel<KS>), dim3(1, (nq + qper - 1) / qper), dim3(kMx4ChunkThreads),
	                   (size_t)qper * (p.first_rows ? p.first_rows : 64) * 4, s, q, nq, rows, n, k, p.first_rows, allow,
	                   static_cast<mx4_key *>(nullptr), (int64_t)0, a.spread, a.all, p.levels ? mid : last, over, qper);
	int64_t step = p.step0;
	for (int l = 1; l <= p.levels; l++) {
		a.first = (unsigned)((a.all + step - 1) / step);
		step /= p.ratio;
		const int tiles = (int)((a.all + step - 1) / step - a.first), takers = stage ? p.splits : p.splits / 2;
		a.each = tiles / takers;
		a.more = tiles % takers;
		if (stage)
			hipLaunchKernelGGL((mx4_stage_kernel<KS>), dim3(p.qtiles * p.splits), dim3(64 * nwaves), lds, s, a, p.qtiles);
		else
			hipLaunchKernelGGL((mx4_stream_kernel<KS>), dim3((unsigned)((p.splits * p.qgroups + 3) / 4)), dim3(256), 0, s, a, p.qgroups);
		const Mx4Out &out = l < p.levels ? mid : last;
		auto pick = [&](auto kernel, auto record, int groups) {
			hipLaunchKernelGGL(kernel, dim3(groups), dim3(256), 0, s, static_cast<const decltype(record) *>(a.lists), a.counts, a.parts, a.list, best, nbest, bound,
			                   nq, k, out, over);
		};
		if (p.few)
			pick(mx4_pick_kernel<64, kMx4GatherWave, Mx4Record, 1, 4>, Mx4Record{}, (nq + 3) / 4);
		else if (stage)
			pick(mx4_pick_kernel<256, kMx4Gather, Mx4Record, 1, 4>, Mx4Record{}, nq);
		else
			pick(mx4_pick_kernel<256, kMx4GatherFewQueries, mx4_key, 4, 2>, mx4_key{}, nq);
	}
	if (p.levels && allow)
		hipLaunchKernelGGL((mx4_rescue_kernel<KS, true>), dim3(nq < 512 ? nq : 512), dim3(256), 0, s, a, k, over, last);
	else if (p.levels)
		hipLaunchKernelGGL((mx4_rescue_kernel<KS, false>), dim3(nq < 512 ? nq : 512), dim3(256), 0, s, a, k, over, last);
	return hipGetLastError();
}

hipError_t mx4_launch_scan(const uint8_t *q, int nq, const uint8_t *rows, int n, int dim, int k, const uint32_t *allow, int32_t *out_ids,
                           float *out_val, int32_t *out_count, void *ws, hipStream_t s)
{
	const Mx4Plan p = mx4_plan(nq, n, dim, k);
	const int rb = mx4_row_bytes(dim), ks = mx4_blocks(dim) / 2;
	const int slab = p.chunks ? nq : p.slab;
	for (int64_t q0 = 0; q0 < nq; q0 += slab) {
		const int m = (int)(nq - q0 < slab ? nq - q0 : slab);
		Mx4Out o{};
		o.ids = out_ids + q0 * k;
		o.val = out_val + q0 * k;
		o.count = out_count + q0;
		hipError_t e = hipErrorInvalidValue;
		auto go = [&](auto steps) {
			constexpr int KS = decltype(steps)::value;
			e = p.chunks ? mx4_scan_chunks<KS>(p, q + q0 * rb, m, rows, n, k, allow, o, ws, s)
			             : mx4_scan_levels<KS>(p, q + q0 * rb, m, rows, n, k, allow, o, ws, s);
		};
		mx4_for_steps(ks, go);
		if (e != hipSuccess) return e;
	}
	return hipSuccess;
}

}  // namespace mvdb
