// seqbeam.cu -- the n best continuations of groups of beams (calm_b200_seq_beam_select in include/calm_b200_seq.h).
//
// Two launches.  k_beam_slice reads every logit once: a CTA takes a slice of one row and leaves the slice's maximum, its sum of exponentials against that maximum
// and its n best tokens.  k_beam_merge, one CTA a group and launched while the slices still run, forms each row's log-sum from its slices and picks the group's n best
// from their lists.
//   log sum_u exp x_u = m + log sum_s exp(m_s - m) S_s,   S_s = sum_(u in s) exp(x_u - m_s),   m = max m_s
// Inside a row the order of scores is the order of logits, so a slice compares logits, as they are, and tokens (64-bit keys: ordered bits of the logit, then the lower
// token), and so does the merge; beams are compared in 64 bits by scores + (x - log-sum).
// Four beams of 32000 fp32 logits take 9.0 us (0.08 of bytes), 256 rows of 128256 32.2 us (4.1 TB/s; 20.1 of bytes), 400 rows of 128256 bf16 51.5 us.  Bound: few rows, the
// latency of two launches and of a slice's end (the looks at its chunks, about 4 us); many, the latency of a warp's chunk - copy, maximum, sum - with 13.7 warps an SM in the mean (whole rows a CTA: two on 108 SMs, one on 40), and a
// 16-bit row the instructions of a logit.  Twice the bytes in flight a warp leaves two CTAs an SM: 160 rows 32.2 for 24.2 us.
#include "seqops.cuh"
#include "tc05.cuh"

#include <stddef.h>

#include <algorithm>

namespace seqops {
namespace {

constexpr int BM_THREADS = 256, BM_WARPS = BM_THREADS / 32, BM_PER = 16; // logits that a thread takes at a time: a chunk
constexpr int BM_TILE = BM_THREADS * BM_PER, BM_SLICE = 64, BM_TILES = 160; // a CTA's at a time; tiles that a slice should have at most, and has at most
constexpr int BM_RING = 4096;                                            // bytes that a warp has in flight
constexpr int BM_MAX = 64;                                               // n
constexpr int BM_LIST = 1024;                                            // chunks that may hold one of a slice's n highest
constexpr int BM_KEYS = (1 + BM_PER) * BM_MAX;                           // single candidates
constexpr int BM_LISTS = 256;                                            // slices of a group's rows
constexpr int BM_MOST = 1 << 27;                                         // candidates of a group: so many fit BM_LISTS / beams slices of BM_TILES - 1 tiles, whatever the beams
constexpr int BM_CAND = 4096;                                            // candidates of a group that the merge compares with one another

struct BeamArgs {
	const void* logits;
	long long group_stride, row_stride;
	const float* scores;
	int beams, vocab, n, slices;
	int *tokens, *parents;
	float* best;
	u64* keys;      // [rows][slices][n], highest first, 0: none
	float2* sums;   // [rows][slices]: maximum, sum of exponentials
};

__device__ __forceinline__ uint32_t order_bits(float v) { // unsigned order = order of values; +0 and -0 are one
	const uint32_t u = __float_as_uint(v + 0.f);
	return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t o) { return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ u64 beam_key(float v, uint32_t index) { return v > -INFINITY ? (u64)order_bits(v) << 32 | (uint32_t)~index : 0; }

// How many of list[0 .. c) (c rounded up to an even number, filled with zeros) are above `key`.
__device__ __forceinline__ int rank_in(const u64* list, int c, u64 key) {
	int r = 0;
	const ulonglong2* p = reinterpret_cast<const ulonglong2*>(list);
#pragma unroll 8
	for (int i = 0; i < (c + 1) / 2; ++i) {
		const ulonglong2 w = p[i];
		r += (w.x > key) + (w.y > key);
	}
	return r;
}
// A CTA's shared memory: rings of bulk copies while it reads its slice, then what it finds the slice's n highest with; behind it the highest logit of every chunk, [tiles][threads].
struct BeamEnd {
	alignas(16) float top[BM_LIST]; // (read four at a time, keys two at a time)
	uint32_t chunk[BM_LIST];
	alignas(16) u64 key[BM_KEYS + 2];
	alignas(16) u64 best[BM_THREADS];
	u64 sorted[BM_MAX];
};
struct BeamSlice {
	union {
		alignas(128) unsigned char ring[BM_WARPS][BM_RING];
		BeamEnd end;
	};
	uint64_t full[BM_WARPS][4];
	uint32_t least[BM_WARPS], low; // order bits
	float red[BM_WARPS];
	int count;
	u64 bound;
};
static_assert(offsetof(BeamEnd, key) % 16 == 0 && offsetof(BeamEnd, best) % 16 == 0 && sizeof(BeamSlice) % 16 == 0, "read 16 bytes at a time");

// The n highest of key[0 .. c), in order, take the front; returns how many there are.  Keys differ, so their ranks do.
__device__ __noinline__ int keep_best(BeamSlice& b, int c, int n) { // (functions of their own: the loop over the logits keeps its registers)
	const int tid = threadIdx.x;
	if (tid == 0 && (c & 1)) b.end.key[c] = 0;
	__syncthreads();
	for (int i = tid; i < c; i += BM_THREADS) {
		const u64 k = b.end.key[i];
		const int r = rank_in(b.end.key, c, k);
		if (r < n) b.end.sorted[r] = k;
	}
	__syncthreads();
	const int have = min(c, n);
	if (tid < have) b.end.key[tid] = b.end.sorted[tid];
	__syncthreads();
	return have;
}
// The slice's n highest where too many values are as high as the n-th (rows of few different values): all of it once more, tile by tile.  The n-th highest of the threads' highest
// values is no higher than the tile's n-th, and only n threads hold anything from it on: at most n * BM_PER values, whatever the tile looks like.
template <typename T>
__device__ __noinline__ int slow_tiles(BeamSlice& b, const uint4* base, unsigned begin, unsigned end, unsigned shift, unsigned total, int n) {
	constexpr int VE = 16 / sizeof(T), NV = BM_PER / VE;
	const int tid = threadIdx.x;
	int k = 0;
	for (unsigned v0 = begin; v0 < end; v0 += NV * BM_THREADS) {
		u64 key[BM_PER], mine = 0;
#pragma unroll
		for (int j = 0; j < NV; ++j) {
			const unsigned o = v0 + j * BM_THREADS + tid;
			uint4 w = make_uint4(0, 0, 0, 0);
			if (o < end) w = ldg_stream(base + o);
			float v[VE];
			unpack16<T>(w, v);
#pragma unroll
			for (int e = 0; e < VE; ++e) {
				const unsigned at = o * VE + e;
				key[j * VE + e] = o < end && at >= shift && at < total ? beam_key(v[e], at - shift) : 0;
				mine = max(mine, key[j * VE + e]);
			}
		}
		b.end.best[tid] = mine;
		if (tid == 0) b.bound = 1, b.count = k; // fewer than n threads with values: everything
		const int valid = __syncthreads_count(mine != 0);
		if (valid >= n && mine && rank_in(b.end.best, BM_THREADS, mine) == n - 1) b.bound = mine;
		__syncthreads();
		if (mine >= b.bound) {
#pragma unroll
			for (int i = 0; i < BM_PER; ++i)
				if (key[i] >= b.bound) b.end.key[atomicAdd(&b.count, 1)] = key[i];
		}
		__syncthreads();
		k = keep_best(b, b.count, n);
	}
	return k;
}
// The slice's n highest from the highest logits of its chunks: the n-th highest of those is no higher than the slice's n-th, so the n highest lie in the chunks from it on.  m: the
// thread's highest logit.  Returns how many there are, in order at the front of key.
template <typename T>
__device__ __noinline__ int slice_best(BeamSlice& b, const float* tops, int tiles, float m, const uint4* base, unsigned begin, unsigned end, unsigned shift, unsigned total, int n) {
	constexpr int VE = 16 / sizeof(T), NV = BM_PER / VE;
	constexpr unsigned WSTEP = NV * 32, STEP = WSTEP * BM_WARPS;
	const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
	// a value that n chunks reach: the least, over the warps with logits, of the k-th highest of a warp's threads, k warps >= n
	const int warps = min(BM_WARPS, (int)((end - begin + WSTEP - 1) / WSTEP));
	uint32_t u = m > -INFINITY ? order_bits(m) : 0, x = 0;
	for (int k = (n + warps - 1) / warps; k > 0; --k) {
		x = __reduce_max_sync(0xffffffffu, u);
		if (__ffs(__ballot_sync(0xffffffffu, u == x)) - 1 == lane) u = 0;
	}
	if (lane == 0) b.least[warp] = x;
	if (tid == 0) b.count = 0, b.low = 0xffffffffu;
	__syncthreads();
	uint32_t from = b.least[0];
#pragma unroll
	for (int i = 1; i < BM_WARPS; ++i)
		if (i < warps) from = min(from, b.least[i]);
	const float least = from ? order_value(from) : -INFINITY;
	if (m >= least && m > -INFINITY)
		for (int i = 0; i < tiles; ++i) {
			const float v = tops[i * BM_THREADS + tid];
			if (v >= least && v > -INFINITY) {
				const int at = atomicAdd(&b.count, 1);
				if (at < BM_LIST) b.end.top[at] = v, b.end.chunk[at] = i * BM_THREADS + tid;
			}
		}
	__syncthreads();
	const int c = b.count;
	__syncthreads();
	if (c > BM_LIST) return slow_tiles<T>(b, base, begin, end, shift, total, n);
	// chunks with fewer than n higher ones
	if (tid < (-c & 3)) b.end.top[c + tid] = -INFINITY;
	if (tid == 0) b.count = 0;
	__syncthreads();
	for (int i = tid; i < c; i += BM_THREADS) {
		const float mine = b.end.top[i];
		int higher = 0;
#pragma unroll 4
		for (int k = 0; k < (c + 3) / 4; ++k) {
			const float4 t = reinterpret_cast<const float4*>(b.end.top)[k];
			higher += (t.x > mine) + (t.y > mine) + (t.z > mine) + (t.w > mine);
		}
		if (higher < n) {
			const int at = atomicAdd(&b.count, 1);
			if (at < BM_THREADS) reinterpret_cast<uint32_t*>(b.end.best)[at] = b.end.chunk[i];
			atomicMin(&b.low, order_bits(mine));
		}
	}
	__syncthreads();
	const int left = b.count;
	const float low = left >= n ? order_value(b.low) : -INFINITY;
	__syncthreads();
	if (left > BM_THREADS) return slow_tiles<T>(b, base, begin, end, shift, total, n);
	// their logits, from memory once more
	if (tid == 0) b.count = 0;
	__syncthreads();
	for (int i = tid; i < left * NV; i += BM_THREADS) {
		const unsigned chunk = reinterpret_cast<const uint32_t*>(b.end.best)[i / NV], owner = chunk % BM_THREADS;
		const unsigned o = begin + chunk / BM_THREADS * STEP + owner / 32 * WSTEP + i % NV * 32 + owner % 32;
		if (o >= end) continue;
		float v[VE];
		unpack16<T>(ldg_stream(base + o), v);
#pragma unroll
		for (int e = 0; e < VE; ++e) {
			const unsigned at = o * VE + e;
			if (v[e] >= low && v[e] > -INFINITY && at >= shift && at < total) {
				const int to = atomicAdd(&b.count, 1);
				if (to < BM_KEYS) b.end.key[to] = beam_key(v[e], at - shift);
			}
		}
	}
	__syncthreads();
	const int keys = b.count;
	__syncthreads();
	return keys > BM_KEYS ? slow_tiles<T>(b, base, begin, end, shift, total, n) : keep_best(b, keys, n);
}

// After a wait that gave up: waits, bounded again, for the copies in flight - of this tile and of those requested ahead - before their memory becomes something else.
template <int STAGES>
__device__ __noinline__ void beam_drain(uint64_t* full, int stage, uint32_t parity, unsigned at, unsigned end, unsigned step) {
	for (int k = 0; k < STAGES && at < end; ++k, at += step) {
		mbar_wait_warp(full + stage, parity);
		if (++stage == STAGES) stage = 0, parity ^= 1;
	}
}

// Per logit: a maximum, a difference, a product, an exponential, an addition (with a fused multiply-add against the maximum times log2(e) a row of the type's lowest values, whose
// product is infinite, would have no sum); per chunk one value kept.  No barrier between warps until the slice has been read.
constexpr float BM_L2E = 1.4426950408889634f;
template <typename T>
__global__ void __launch_bounds__(BM_THREADS, 4) k_beam_slice(const BeamArgs a) {
	constexpr int VE = 16 / sizeof(T), NV = BM_PER / VE, STAGES = BM_RING / (NV * 512);
	constexpr unsigned WSTEP = NV * 32, STEP = WSTEP * BM_WARPS; // vectors of a warp's part of a tile, of a tile
	extern __shared__ __align__(128) unsigned char slice_sm[];
	BeamSlice& b = *reinterpret_cast<BeamSlice*>(slice_sm);
	float* const tops = reinterpret_cast<float*>(slice_sm + sizeof(BeamSlice));
	pdl_launch_next();
	const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, slice = blockIdx.x, row = blockIdx.y, n = a.n;
	u64* const out = a.keys + ((size_t)row * a.slices + slice) * n;
	if (!(fabsf(a.scores[row]) < INFINITY)) { // this beam is not there
		for (int i = tid; i < n; i += BM_THREADS) out[i] = 0;
		if (tid == 0) a.sums[(size_t)row * a.slices + slice] = make_float2(-INFINITY, 0.f);
		return;
	}
	// the row from the 16-byte boundary at or before its first element: elements [shift, total) of `base` are its own
	const T* p = (const T*)a.logits + (long long)(row / a.beams) * a.group_stride + (long long)(row % a.beams) * a.row_stride;
	const unsigned shift = (unsigned)(((uintptr_t)p & 15) / sizeof(T));
	const uint4* const base = reinterpret_cast<const uint4*>(p - shift);
	const unsigned total = a.vocab + shift, vectors = (total + VE - 1) / VE, each = (vectors + a.slices - 1) / a.slices;
	const unsigned begin = min(vectors, slice * each), end = min(vectors, begin + each); // in vectors
	// each warp has a ring of its own
	uint64_t* const full = b.full[warp];
	unsigned asked = begin + warp * WSTEP; // the warp's part of the next tile to request
	const uint64_t policy = l2_policy_evict_first();
	auto request = [&](int stage) { // one lane
		if (asked < end) {
			const uint32_t bytes = min(end - asked, WSTEP) * 16;
			mbar_expect_tx(full + stage, bytes);
			tma_load_1d_hint(b.ring[warp] + stage * (NV * 512), base + asked, bytes, full + stage, policy);
		}
	};
	if (lane == 0) {
#pragma unroll
		for (int i = 0; i < STAGES; ++i) mbar_init(full + i, 1);
		mbar_init_fence();
	}
#pragma unroll
	for (int i = 0; i < STAGES; ++i) {
		if (lane == 0) request(i);
		asked += STEP;
	}
	__syncwarp();
	float m = -INFINITY, s = 0.f; // the thread's maximum and sum
	int stage = 0, tiles = 0;
	uint32_t parity = 0;
	bool lost = false; // a copy never came
	for (unsigned v0 = begin; v0 < end; v0 += STEP, ++tiles) {
		float v[BM_PER];
		{
			uint4 w[NV];
			if (v0 + warp * WSTEP < end && !lost) {
				if (!mbar_wait_warp(full + stage, parity)) lost = true, beam_drain<STAGES>(full, stage, parity, v0 + warp * WSTEP, end, STEP);
				const uint4* const src = reinterpret_cast<const uint4*>(b.ring[warp] + stage * (NV * 512)) + lane;
#pragma unroll
				for (int j = 0; j < NV; ++j) w[j] = src[j * 32];
			}
#pragma unroll
			for (int j = 0; j < NV; ++j) unpack16<T>(w[j], *reinterpret_cast<float(*)[VE]>(v + j * VE));
		}
		if (v0 * VE < shift || v0 + STEP > end || (v0 + STEP) * VE > total) { // the row's first and last tile: places outside it
#pragma unroll
			for (int i = 0; i < BM_PER; ++i) {
				const unsigned o = v0 + warp * WSTEP + (i / VE) * 32 + lane, e = o * VE + i % VE;
				if (o >= end || e < shift || e >= total) v[i] = -INFINITY;
			}
		}
		__syncwarp(); // all lanes have read
		if (lane == 0 && !lost) request(stage);
		asked += STEP;
		if (++stage == STAGES) stage = 0, parity ^= 1;
		float top = -INFINITY; // (a NaN is passed over)
#pragma unroll
		for (int i = 0; i < BM_PER; i += 2) top = fmaxf(fmaxf(top, v[i]), v[i + 1]);
		tops[tiles * BM_THREADS + tid] = top;
		if (top > m) s = m > -INFINITY && top < INFINITY ? s * ex2((m - top) * BM_L2E) : 0.f, m = top;
		u64 part[2] = {0, 0};
		const u64 down = pair_of(-m, -m), l2e = pair_of(BM_L2E, BM_L2E);
#pragma unroll
		for (int i = 0; i < BM_PER / 2; ++i) {
			const float2 y = halves(mul2(add2(pair_of(v[2 * i], v[2 * i + 1]), down), l2e));
			part[i & 1] = add2(part[i & 1], pair_of(ex2(y.x), ex2(y.y)));
		}
		const float2 both = halves(add2(part[0], part[1]));
		float sum = both.x + both.y;
		if (!(sum < INFINITY)) { // a NaN among the logits, nothing but -inf so far, or +inf: rare
			sum = 0.f;
			if (m > -INFINITY)
#pragma unroll
				for (int i = 0; i < BM_PER; ++i) sum += m == INFINITY ? (v[i] == INFINITY ? 1.f : 0.f) : v[i] > -INFINITY ? ex2((v[i] - m) * BM_L2E) : 0.f;
		}
		s += sum;
	}
	const float wm = warp_max(m);
	if (lane == 0) b.red[warp] = wm;
	const bool broken = __syncthreads_or(lost);
	float bm = b.red[0];
#pragma unroll
	for (int i = 1; i < BM_WARPS; ++i) bm = fmaxf(bm, b.red[i]);
	const float ws = warp_sum(m == bm ? s : m > -INFINITY && bm < INFINITY ? s * ex2((m - bm) * BM_L2E) : 0.f);
	__syncthreads();
	if (lane == 0) b.red[warp] = ws;
	const int k = begin < end ? slice_best<T>(b, tops, tiles, m, base, begin, end, shift, total, n) : 0;
	for (int i = tid; i < n; i += BM_THREADS) out[i] = i < k ? b.end.key[i] : 0;
	__syncthreads();
	if (tid == 0) {
		float sum = b.red[0];
#pragma unroll
		for (int i = 1; i < BM_WARPS; ++i) sum += b.red[i];
		a.sums[(size_t)row * a.slices + slice] = make_float2(bm, broken ? NAN : bm > -INFINITY ? sum : 0.f); // (without a sum the row has no candidates)
	}
}

// A candidate's score and, as one number that is higher for what comes first among equal scores, its beam, its logit and its token: of one beam the higher logit comes first
// also where 64 bits do not tell the scores apart (a logit of 1e-20 and one of 2e-20 beside a maximum of 5).
struct BeamCand {
	double d[BM_CAND];
	u64 i[BM_CAND];
};
__device__ __forceinline__ bool above(double d, u64 i, double e, u64 j) { return d > e || (d == e && i > j); }

__global__ void __launch_bounds__(BM_THREADS) k_beam_merge(const BeamArgs a) {
	extern __shared__ __align__(16) unsigned char merge_sm[];
	BeamCand& cand = *reinterpret_cast<BeamCand*>(merge_sm);
	__shared__ double log_sum[BM_MAX], head_d[BM_THREADS];
	__shared__ float row_max[BM_MAX];
	__shared__ u64 head_i[BM_THREADS];
	__shared__ int count;
	__shared__ double bound_d[BM_THREADS / 64];
	__shared__ u64 bound_i[BM_THREADS / 64];
	const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = blockIdx.x, n = a.n, K = a.beams, S = a.slices, lists = K * S;
	if (tid == 0) count = 0;
	pdl_wait_prev();
	for (int b = warp; b < K; b += BM_THREADS / 32) { // a row's log-sum from its slices
		const float2* p = a.sums + (size_t)(g * K + b) * S;
		float m = -INFINITY;
		for (int i = lane; i < S; i += 32) m = fmaxf(m, p[i].x);
		m = warp_max(m);
		double sum = 0.;
		for (int i = lane; i < S; i += 32) {
			const float2 q = p[i];
			if (q.x > -INFINITY) sum += q.x == m ? (double)q.y : exp((double)q.x - (double)m) * q.y;
		}
#pragma unroll
		for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
		if (lane == 0) row_max[b] = m, log_sum[b] = log(sum);
	}
	__syncthreads();
	const u64* const keys = a.keys + (size_t)g * lists * n;
	const int bits = 32 - __clz(a.vocab - 1); // of a token; beams and tokens have 28 together at most
	auto value = [&](int list, u64 k, double& d) { // a candidate of a list; false: it is none
		const int b = list / S;
		const float x = order_value((uint32_t)(k >> 32)), m = row_max[b];
		d = (double)a.scores[g * K + b] + ((x == m ? 0. : (double)x - (double)m) - log_sum[b]);
		return k != 0 && d > -INFINITY;
	};
	auto place = [&](int list, u64 k) { return (u64)(K - 1 - list / S) << (32 + bits) | k >> 32 << bits | (uint32_t)(a.vocab - 1 - (int)~(uint32_t)k); };
	// Lists are in order.  Of the values at one depth of all lists the r-th highest, r (depth + 1) >= n, has n values at or above it; at the least such depth at most r lists reach
	// it there, so what is at or above it is at most r n values and the others' first `depth`: n lists' worth.  Where lists are few, other threads look at twice that depth, four
	// times, ...: the highest of the bounds leaves far fewer (64 lists of 64 values: the lowest list's head bounds nothing).
	int width = 64;
	while (width < lists) width *= 2;
	const int set = tid / width, list = tid % width, depth = ((n + lists - 1) / lists << set) - 1, r = (n + depth) / (depth + 1);
	double d = 0.;
	const u64 head = list < lists && depth < n ? keys[list * n + depth] : 0;
	const bool have = value(min(list, lists - 1), head, d);
	u64 i = have ? place(list, head) : 0;
	head_d[tid] = have ? d : -INFINITY, head_i[tid] = i;
	if (list == 0) bound_d[set] = -INFINITY, bound_i[set] = 0; // fewer than r lists reach the depth: everything
	__syncthreads();
	if (have) {
		int rank = 0;
#pragma unroll 8
		for (int k = 0; k < lists; ++k) rank += above(head_d[set * width + k], head_i[set * width + k], d, i);
		if (rank == r - 1) bound_d[set] = d, bound_i[set] = i;
	}
	__syncthreads();
	double low_d = bound_d[0];
	u64 low_i = bound_i[0];
	for (int k = 1; k < BM_THREADS / width; ++k)
		if (above(bound_d[k], bound_i[k], low_d, low_i)) low_d = bound_d[k], low_i = bound_i[k];
	for (int e0 = tid; e0 < lists * n; e0 += 4 * BM_THREADS) {
		u64 k[4];
#pragma unroll
		for (int u = 0; u < 4; ++u) k[u] = e0 + u * BM_THREADS < lists * n ? keys[e0 + u * BM_THREADS] : 0;
#pragma unroll
		for (int u = 0; u < 4; ++u) {
			if (e0 - tid + u * BM_THREADS >= lists * n) break;
			const int from = min((e0 + u * BM_THREADS) / n, lists - 1);
			if (value(from, k[u], d) && d >= low_d && (d > low_d || place(from, k[u]) >= low_i)) {
				const int at = atomicAdd(&count, 1);
				if (at < BM_CAND) cand.d[at] = d, cand.i[at] = place(from, k[u]);
			}
		}
	}
	__syncthreads();
	const int c = min(count, BM_CAND), base = g * n;
	for (int e = tid; e < c; e += BM_THREADS) {
		d = cand.d[e], i = cand.i[e];
		int rank = 0;
#pragma unroll 8
		for (int k = 0; k < c; ++k) {
			const double o = cand.d[k];
			rank += o > d;
			if (o == d && k != e) rank += cand.i[k] > i; // (seldom)
		}
		if (rank < n) a.tokens[base + rank] = a.vocab - 1 - (int)(i & ((1ull << bits) - 1)), a.parents[base + rank] = K - 1 - (int)(i >> (32 + bits)), a.best[base + rank] = (float)d;
	}
	for (int e = c + tid; e < n; e += BM_THREADS) a.tokens[base + e] = a.parents[base + e] = -1, a.best[base + e] = -INFINITY;
}

// Slices of a row: a tile each where rows are few, three CTAs an SM in all where they are many (148 / 296 / 444 / 592 CTAs in all: 160 rows of 128256 fp32 30.5 / 30.9 / 24.2 /
// 34.7 us, 100 rows 26.4 / 20.3 / 18.1 / 24.1, 64 rows 18.2 / 15.9 / 16.5 / 18.2: a slice's end costs about the same whatever its length), two an SM for the longest rows.
int beam_slices(int groups, int beams, int vocab) {
	const int want = std::max(std::min(cdiv(vocab, BM_TILE), 148 * 3 / std::max(1, groups * beams)), cdiv(vocab, BM_TILE * BM_SLICE));
	return std::max(cdiv(vocab, BM_TILE * (BM_TILES - 1)), std::min(want, BM_LISTS / beams)); // (a row that starts behind a 16-byte boundary may reach into one tile more)
}
size_t beam_shared(const BeamArgs& a, int size) { // tiles of a slice, as the kernel cuts them at the worst alignment
	const int ve = 16 / size, each = cdiv(cdiv(a.vocab + ve - 1, ve), a.slices);
	return sizeof(BeamSlice) + (size_t)cdiv(each, BM_TILE / ve) * BM_THREADS * sizeof(float);
}
size_t beam_keys(int groups, int beams, int vocab, int n) { return ((size_t)groups * beams * beam_slices(groups, beams, vocab) * n * sizeof(u64) + 15) & ~(size_t)15; }

template <typename T>
cudaError_t beam_launch(const BeamArgs& a, dim3 grid, cudaStream_t st) {
	static std::atomic<uint64_t> done{0};
	const cudaError_t e = allow(k_beam_slice<T>, sizeof(BeamSlice) + BM_TILES * BM_THREADS * sizeof(float), done);
	return e == cudaSuccess ? launch(st, false, 1, k_beam_slice<T>, grid, dim3(BM_THREADS), beam_shared(a, sizeof(T)), a) : e;
}

int beam_check(int groups, int beams, int vocab, int n) {
	if (groups < 0 || beams < 1 || beams > 64) return refuse("beam: %d groups of %d beams (at most 64 beams)", groups, beams);
	if (vocab < 1 || (long long)beams * vocab > BM_MOST) return refuse("beam: %d beams over %d tokens: at most 2^27 candidates a group", beams, vocab);
	if (n < 1 || n > BM_MAX) return refuse("beam: n = %d is not in 1 .. %d", n, BM_MAX);
	if ((long long)groups * beams > 65535) return refuse("beam: %d rows in all, at most 65535", groups * beams);
	return 0;
}
} // namespace
} // namespace seqops

extern "C" size_t calm_b200_seq_beam_workspace(int groups, int beams, int vocab, int n) {
	using namespace seqops;
	if (beam_check(groups, beams, vocab, n)) return 0;
	return beam_keys(groups, beams, vocab, n) + (size_t)groups * beams * beam_slices(groups, beams, vocab) * sizeof(float2);
}

extern "C" int calm_b200_seq_beam_select(const struct SeqBeam* q, void* stream) {
	using namespace seqops;
	if (!q) return refuse("beam: no arguments");
	if (const int rc = beam_check(q->groups, q->beams, q->vocab, q->n)) return rc;
	if (!type_ok(q->type)) return refuse("beam: unknown type %d", q->type);
	if (q->groups == 0) return 0;
	if (!q->logits || !q->scores || !q->tokens || !q->parents || !q->best || !q->workspace) return refuse("beam: a pointer is missing");
	if ((uintptr_t)q->logits % type_size(q->type)) return refuse("beam: the logits are not aligned to their type");
	if (((uintptr_t)q->scores | (uintptr_t)q->tokens | (uintptr_t)q->parents | (uintptr_t)q->best) % 4) return refuse("beam: scores or results are not aligned to 4 bytes");
	if ((uintptr_t)q->workspace % 16) return refuse("beam: the workspace is not aligned to 16 bytes");
	if (q->workspace_bytes < calm_b200_seq_beam_workspace(q->groups, q->beams, q->vocab, q->n)) return refuse("beam: the workspace has %zu bytes, %zu are needed", q->workspace_bytes, calm_b200_seq_beam_workspace(q->groups, q->beams, q->vocab, q->n));
	BeamArgs a;
	a.logits = q->logits, a.group_stride = q->group_stride, a.row_stride = q->row_stride, a.scores = q->scores;
	a.beams = q->beams, a.vocab = q->vocab, a.n = q->n, a.slices = beam_slices(q->groups, q->beams, q->vocab);
	a.tokens = q->tokens, a.parents = q->parents, a.best = q->best;
	a.keys = (u64*)q->workspace, a.sums = (float2*)((char*)q->workspace + beam_keys(q->groups, q->beams, q->vocab, q->n));
	const cudaStream_t st = (cudaStream_t)stream;
	const dim3 grid(a.slices, q->groups * q->beams);
	cudaError_t e = q->type == SEQ_F32 ? beam_launch<float>(a, grid, st) : q->type == SEQ_BF16 ? beam_launch<__nv_bfloat16>(a, grid, st) : beam_launch<__half>(a, grid, st);
	if (e != cudaSuccess) return failed("beam", e);
	static std::atomic<uint64_t> done{0};
	e = allow(k_beam_merge, sizeof(BeamCand), done);
	if (e == cudaSuccess) e = launch(st, true, 1, k_beam_merge, dim3(q->groups), dim3(BM_THREADS), sizeof(BeamCand), a);
	return e == cudaSuccess ? 0 : failed("beam", e);
}
