// seqbeam.cu -- the n best continuations of groups of beams (calm_b200_seq_beam_select in include/calm_b200_seq.h).
//
// Two launches.  k_beam_slice reads every logit once: a CTA takes a slice of one row and leaves the slice's maximum, its sum of exponentials against that maximum
// and its n best tokens.  k_beam_merge, one CTA a group and launched while the slices still run, forms each row's log-sum from its slices and picks the group's n best
// from their lists.
//   log sum_u exp x_u = m + log sum_s exp(m_s - m) S_s,   S_s = sum_(u in s) exp(x_u - m_s),   m = max m_s
// Inside a row the order of scores is the order of logits, so a slice compares logits, as they are, and tokens (64-bit keys: ordered bits of the logit, then the lower
// token); beams are compared in 64 bits by scores + (x - log-sum).  Bound: the logits' way through memory; a single request's few rows, the latency of two
// launches.
#include "seqops.cuh"

#include <algorithm>

namespace seqops {
namespace {

constexpr int BM_THREADS = 256, BM_PER = 16, BM_TILE = BM_THREADS * BM_PER; // elements a thread and a CTA take at a time
constexpr int BM_MAX = 64;                                                  // n
constexpr int BM_ROOM = 4;                                                  // keys wait for their order until there are more than BM_ROOM n
constexpr int BM_KEYS = (BM_ROOM + BM_PER) * BM_MAX;                        // those and the ones of a tile that may join them
constexpr int BM_LISTS = 256;                                               // slices of a group's rows
constexpr int BM_CAND = 4096;                                               // candidates of a group that the merge compares with one another
typedef unsigned long long u64;

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
// The n highest of keys[0 .. c), in order, take the front; returns how many there are.  Keys differ, so their ranks do.
__device__ int keep_best(u64* keys, int c, int n, u64* sorted) {
	const int tid = threadIdx.x;
	if (tid == 0 && (c & 1)) keys[c] = 0;
	__syncthreads();
	for (int i = tid; i < c; i += BM_THREADS) {
		const u64 k = keys[i];
		const int r = rank_in(keys, c, k);
		if (r < n) sorted[r] = k;
	}
	__syncthreads();
	const int have = min(c, n);
	if (tid < have) keys[tid] = sorted[tid];
	__syncthreads();
	return have;
}

template <typename T>
__global__ void __launch_bounds__(BM_THREADS) k_beam_slice(const BeamArgs a) {
	constexpr int VE = 16 / sizeof(T), NV = BM_PER / VE;
	constexpr float L2E = 1.4426950408889634f;
	__shared__ __align__(16) u64 keys[BM_KEYS + 1], best[BM_THREADS], sorted[BM_MAX];
	__shared__ int count;
	__shared__ u64 bound;
	__shared__ float red_m[BM_THREADS / 32], red_s[BM_THREADS / 32];
	pdl_launch_next();
	const int tid = threadIdx.x, slice = blockIdx.x, row = blockIdx.y, n = a.n;
	u64* const out = a.keys + ((size_t)row * a.slices + slice) * n;
	if (!(a.scores[row] > -INFINITY)) { // this beam is not there
		for (int i = tid; i < n; i += BM_THREADS) out[i] = 0;
		if (tid == 0) a.sums[(size_t)row * a.slices + slice] = make_float2(-INFINITY, 0.f);
		return;
	}
	// the row from the 16-byte boundary at or before its first element: elements [shift, total) of `base` are its own
	const T* p = (const T*)a.logits + (long long)(row / a.beams) * a.group_stride + (long long)(row % a.beams) * a.row_stride;
	const int shift = (int)(((uintptr_t)p & 15) / sizeof(T));
	const T* base = p - shift;
	const long long total = (long long)a.vocab + shift;
	const long long vectors = (total + VE - 1) / VE, each = (vectors + a.slices - 1) / a.slices;
	const long long begin = min(vectors, slice * each) * VE, end = min(total, (slice + 1) * each * VE);
	float m = -INFINITY, s = 0.f, tau = -INFINITY; // the thread's maximum and sum; a later token counts only above tau
	int c = 0;                                     // keys kept
	bool first = true;
	for (long long t0 = begin; t0 < end; t0 += BM_TILE) {
		float v[BM_PER];
		uint4 w[NV];
#pragma unroll
		for (int j = 0; j < NV; ++j) {
			const long long o = t0 + (long long)(j * BM_THREADS + tid) * VE;
			if (o < end) w[j] = ldg_stream(reinterpret_cast<const uint4*>(base + o));
		}
#pragma unroll
		for (int j = 0; j < NV; ++j) {
			const long long o = t0 + (long long)(j * BM_THREADS + tid) * VE;
			float u[VE];
			unpack16<T>(w[j], u);
			const bool inside = o >= shift && o + VE <= end;
#pragma unroll
			for (int e = 0; e < VE; ++e) v[j * VE + e] = inside || (o + e >= shift && o + e < end) ? fmaxf(u[e], -INFINITY) : -INFINITY; // (fmaxf: a NaN becomes -inf)
		}
		float top = v[0];
#pragma unroll
		for (int i = 1; i < BM_PER; ++i) top = fmaxf(top, v[i]);
		if (top > m) {
			if (m > -INFINITY) s *= top == INFINITY ? 0.f : exp2f((m - top) * L2E);
			m = top;
		}
		if (m < INFINITY) {
			if (m > -INFINITY) {
				float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
				for (int i = 0; i < BM_PER; ++i) part[i & 3] += exp2f((v[i] - m) * L2E);
				s += (part[0] + part[1]) + (part[2] + part[3]);
			}
		} else {
#pragma unroll
			for (int i = 0; i < BM_PER; ++i) s += v[i] == INFINITY ? 1.f : 0.f;
		}
		auto index = [&](int i) { return (uint32_t)(t0 + (long long)((i / VE) * BM_THREADS + tid) * VE + i % VE - shift); };
		if (!__syncthreads_or(top > tau)) continue;
		bool pick = first;
		if (!first) { // few values pass tau: they join the kept ones, unless there is no room for all
			if (tid == 0) count = c;
			__syncthreads();
			if (top > tau) {
#pragma unroll
				for (int i = 0; i < BM_PER; ++i)
					if (v[i] > tau) {
						const int at = atomicAdd(&count, 1);
						if (at < BM_KEYS) keys[at] = beam_key(v[i], index(i));
					}
			}
			__syncthreads();
			pick = count > BM_KEYS; // what was written behind the kept keys is forgotten
			if (!pick) c = count;
			__syncthreads();
		}
		if (pick) {
			// The n-th highest of the threads' highest values is no higher than the tile's n-th, and only n threads hold anything from it on: at most
			// n * BM_PER values, whatever the tile looks like.
			u64 mine = 0;
#pragma unroll
			for (int i = 0; i < BM_PER; ++i) mine = max(mine, beam_key(v[i], index(i)));
			best[tid] = mine;
			if (tid == 0) bound = 1, count = c; // fewer than n threads with values: everything
			const int valid = __syncthreads_count(mine != 0);
			if (valid >= n && mine && rank_in(best, BM_THREADS, mine) == n - 1) bound = mine;
			__syncthreads();
			if (mine >= bound) {
#pragma unroll
				for (int i = 0; i < BM_PER; ++i) {
					const u64 k = beam_key(v[i], index(i));
					if (k >= bound) keys[atomicAdd(&count, 1)] = k;
				}
			}
			__syncthreads();
			c = count;
			first = false;
		}
		if (pick || c > BM_ROOM * n) {
			c = keep_best(keys, c, n, sorted);
			tau = c == n ? order_value((uint32_t)(keys[n - 1] >> 32)) : -INFINITY;
		}
	}
	c = keep_best(keys, c, n, sorted);
	for (int i = tid; i < n; i += BM_THREADS) out[i] = i < c ? keys[i] : 0;
	const float wm = warp_max(m);
	if ((tid & 31) == 0) red_m[tid >> 5] = wm;
	__syncthreads();
	float bm = red_m[0];
#pragma unroll
	for (int i = 1; i < BM_THREADS / 32; ++i) bm = fmaxf(bm, red_m[i]);
	const float ws = warp_sum(m == bm ? s : m > -INFINITY ? s * exp2f((m - bm) * L2E) : 0.f);
	if ((tid & 31) == 0) red_s[tid >> 5] = ws;
	__syncthreads();
	if (tid == 0) {
		float sum = red_s[0];
#pragma unroll
		for (int i = 1; i < BM_THREADS / 32; ++i) sum += red_s[i];
		a.sums[(size_t)row * a.slices + slice] = make_float2(bm, bm > -INFINITY ? sum : 0.f);
	}
}

struct BeamCand {
	double d[BM_CAND];
	uint32_t i[BM_CAND];
};
__device__ __forceinline__ bool above(double d, uint32_t i, double e, uint32_t j) { return d > e || (d == e && i < j); }

__global__ void __launch_bounds__(BM_THREADS) k_beam_merge(const BeamArgs a) {
	extern __shared__ __align__(16) unsigned char merge_sm[];
	BeamCand& cand = *reinterpret_cast<BeamCand*>(merge_sm);
	__shared__ double log_sum[BM_MAX], head_d[BM_THREADS];
	__shared__ float row_max[BM_MAX];
	__shared__ uint32_t head_i[BM_THREADS];
	__shared__ int count;
	__shared__ double bound_d;
	__shared__ uint32_t bound_i;
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
	auto value = [&](int list, int at, double& d, uint32_t& i) { // candidate `at` of a list; false: there is none
		const u64 k = keys[(size_t)list * n + at];
		const int b = list / S;
		const float x = order_value((uint32_t)(k >> 32)), m = row_max[b];
		d = (double)a.scores[g * K + b] + ((x == m ? 0. : (double)x - (double)m) - log_sum[b]);
		i = (uint32_t)b * (uint32_t)a.vocab + ~(uint32_t)k;
		return k != 0 && d > -INFINITY;
	};
	// Lists are in order.  Of the values at one depth of all lists the r-th highest, r (depth + 1) >= n, has n values at or above it; at most r lists reach it
	// there, so what is at or above it is at most r n values and the others' first `depth`: n lists' worth.
	const int depth = max(0, (n + lists - 1) / lists - 1), r = (n + depth) / (depth + 1);
	double d = 0.;
	uint32_t i = 0;
	const bool have = tid < lists && value(tid, depth, d, i);
	head_d[tid] = have ? d : -INFINITY, head_i[tid] = have ? i : 0xffffffffu;
	if (tid == 0) bound_d = -INFINITY, bound_i = 0xffffffffu; // fewer than r lists reach the depth: everything
	const int valid = __syncthreads_count(have);
	if (have && valid >= r) {
		int rank = 0;
#pragma unroll 8
		for (int k = 0; k < lists; ++k) rank += above(head_d[k], head_i[k], d, i);
		if (rank == r - 1) bound_d = d, bound_i = i;
	}
	__syncthreads();
	for (int e = tid; e < lists * n; e += BM_THREADS)
		if (value(e / n, e % n, d, i) && !above(bound_d, bound_i, d, i)) {
			const int at = atomicAdd(&count, 1);
			if (at < BM_CAND) cand.d[at] = d, cand.i[at] = i;
		}
	__syncthreads();
	const int c = min(count, BM_CAND), base = g * n;
	for (int e = tid; e < c; e += BM_THREADS) {
		d = cand.d[e], i = cand.i[e];
		int rank = 0;
#pragma unroll 8
		for (int k = 0; k < c; ++k) rank += above(cand.d[k], cand.i[k], d, i);
		if (rank < n) a.tokens[base + rank] = (int)(i % (uint32_t)a.vocab), a.parents[base + rank] = (int)(i / (uint32_t)a.vocab), a.best[base + rank] = (float)d;
	}
	for (int e = c + tid; e < n; e += BM_THREADS) a.tokens[base + e] = a.parents[base + e] = -1, a.best[base + e] = -INFINITY;
}

// Slices of a row: a tile each where rows are few, as many as keep all CTAs of one wave resident where they are many.
int beam_slices(int groups, int beams, int vocab) {
	const int rows = groups * beams, tiles = cdiv(vocab, BM_TILE);
	return std::max(1, std::min({tiles, cdiv(148 * 6, rows), BM_LISTS / beams}));
}
size_t beam_keys(int groups, int beams, int vocab, int n) { return ((size_t)groups * beams * beam_slices(groups, beams, vocab) * n * sizeof(u64) + 15) & ~(size_t)15; }

int beam_check(int groups, int beams, int vocab, int n) {
	if (groups < 0 || beams < 1 || beams > 64) return refuse("beam: %d groups of %d beams (at most 64 beams)", groups, beams);
	if (vocab < 1 || (long long)beams * vocab >= (1LL << 31)) return refuse("beam: %d beams over %d tokens: at most 2^31 candidates", beams, vocab);
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
	if ((uintptr_t)q->workspace % 16) return refuse("beam: the workspace is not aligned to 16 bytes");
	if (q->workspace_bytes < calm_b200_seq_beam_workspace(q->groups, q->beams, q->vocab, q->n)) return refuse("beam: the workspace has %zu bytes, %zu are needed", q->workspace_bytes, calm_b200_seq_beam_workspace(q->groups, q->beams, q->vocab, q->n));
	BeamArgs a;
	a.logits = q->logits, a.group_stride = q->group_stride, a.row_stride = q->row_stride, a.scores = q->scores;
	a.beams = q->beams, a.vocab = q->vocab, a.n = q->n, a.slices = beam_slices(q->groups, q->beams, q->vocab);
	a.tokens = q->tokens, a.parents = q->parents, a.best = q->best;
	a.keys = (u64*)q->workspace, a.sums = (float2*)((char*)q->workspace + beam_keys(q->groups, q->beams, q->vocab, q->n));
	const cudaStream_t st = (cudaStream_t)stream;
	const dim3 grid(a.slices, q->groups * q->beams);
	auto kernel = q->type == SEQ_F32 ? k_beam_slice<float> : q->type == SEQ_BF16 ? k_beam_slice<__nv_bfloat16> : k_beam_slice<__half>;
	cudaError_t e = launch(st, false, 1, kernel, grid, dim3(BM_THREADS), 0, a);
	if (e != cudaSuccess) return failed("beam", e);
	if ((e = cudaFuncSetAttribute(k_beam_merge, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(BeamCand))) != cudaSuccess) return failed("beam", e);
	e = launch(st, true, 1, k_beam_merge, dim3(q->groups), dim3(BM_THREADS), sizeof(BeamCand), a);
	return e == cudaSuccess ? 0 : failed("beam", e);
}
