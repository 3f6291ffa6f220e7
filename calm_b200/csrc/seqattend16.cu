// seqattend16.cu -- attention over a paged cache in 16 bits, where groups of sequences share a prefix (calm_b200_seq_attend16 in include/calm_b200_seq.h).

#include "seqcache16.cuh"

namespace seqops {
namespace {

typedef __nv_bfloat16 bf16;

// what the kernels know of the cache, the batch and its groups
struct C16 {
	const uint16_t *k, *v;
	const int* table;
	int pages, heads, page, dim, slots, table_pages;
	int page_shift; // log2 of page, -1: no power of two
	const int *start, *count, *slot, *pos0;
	int n;
	int groups;
	const int *first, *members, *positions, *group;
	__device__ __forceinline__ int reach(int slot) const { return (unsigned)slot < (unsigned)slots && pages > 0 ? (int)min((long long)table_pages * page, INT_MAX - 256LL) : 0; } // positions that the table has
	__device__ __forceinline__ int page_index(int pos) const { return page_shift >= 0 ? pos >> page_shift : pos / page; }
	__device__ __forceinline__ int page_row(int pos) const { return page_shift >= 0 ? pos & (page - 1) : pos % page; }
};
struct Attend {
	const uint16_t* q;
	long long q_row, q_head;
	uint16_t* out;
	long long o_row, o_head;
	int rows, heads, group; // group: query heads a key head
	float scale, softcap;
	int window;
	const float* sinks;
	int families;     // 1: groups with their prefixes and own keys, and the sequences of no group; 0: every sequence behind what it shares
	int shares, each; // shares of a tile's keys, chunks of each
	int cluster;      // 1: the shares of a tile are a cluster
	int before;       // places of `stats` and `sums` that the prefixes' shares have
	int places;       // all of them
	float2* stats;    // [rows][heads][places]: reference, denominator
	float* sums;      // [rows][heads][places][dim]
};
constexpr float A16_LOG2E = 1.4426950408889634f;
// Softmax weights are rounded to the cache's type on their way into the products (a relative 2^-9 or 2^-12 each, as the values themselves were), sums of them are not.  A row's reference
// moves when a chunk's largest exponent passes it by A16_MOST, to A16_SET below that: fp16 weights stay under 2^15 and the largest is 2^10 or more, so that what it rounds as a subnormal is 2^-35 of the largest.
constexpr float A16_MOST = 15.f, A16_SET = 10.f;

// ---------------------------------------------------------------- few rows
// A CTA takes 8 NQ rows (pairs of token and query head) that read one key head: of one sequence, or of the sequences of a group one after another.  It walks a list of keys: those of the group's
// prefix, which all rows see, then those of each sequence of its rows, which only that sequence's rows see, in chunks of 32.  So a prefix is read once for 8 NQ rows, and a call of few rows needs one launch.
// Each warp walks chunks of its own with references and sums of its own (no barrier between warps until the end), fed by a ring of asynchronous copies, into m16n8k16 products whose 16 rows are keys (scores: keys x queries) or
// channels (values: channels x queries), so that eight rows of queries fill one.
constexpr int AR_WARPS = 4, AR_KEYS = 32;
constexpr int AR_SHARES = 64;                // of a tile's keys at most
constexpr int AR_TILE = 16, AR_CLUSTER = 16; // rows of a CTA at most; shares that a thread-block cluster folds at most

template <int D>
struct ArStage { // a warp's chunk: the next one's keys come while its values are used, the next one's values while their keys are
	uint16_t k[AR_KEYS * D], v[AR_KEYS * D];
};
template <int D>
__host__ __device__ constexpr size_t ar_ring() { // (the sums of the warps take its place)
	const size_t a = (size_t)AR_WARPS * sizeof(ArStage<D>), b = ((size_t)AR_WARPS * 8 * (D + 4) + (size_t)AR_TILE * (D + 2)) * sizeof(float);
	return a > b ? a : b;
}
template <int D, int NQ>
constexpr size_t ar_smem() { return (size_t)8 * NQ * D * 2 + ar_ring<D>(); }

template <typename T>
__device__ __forceinline__ void mma_16(float (&c)[4], const uint32_t (&a)[4], uint2 b) {
	if constexpr (std::is_same<T, bf16>::value)
		asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
		             : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
		             : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
	else
		asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
		             : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
		             : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
	if constexpr (std::is_same<T, bf16>::value) {
		const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
		return *reinterpret_cast<const uint32_t*>(&h);
	} else {
		const __half2 h = __floats2half2_rn(x, y);
		return *reinterpret_cast<const uint32_t*>(&h);
	}
}
template <typename T>
__device__ __forceinline__ uint16_t round16(float x) {
	const T h = from_f32<T>(x);
	return *reinterpret_cast<const uint16_t*>(&h);
}
// whether one of the two halves is infinite or no number
template <typename T>
__device__ __forceinline__ bool odd2(uint32_t x) {
	constexpr uint32_t E = std::is_same<T, bf16>::value ? 0x7f80 : 0x7c00;
	return (x & E) == E || (x >> 16 & E) == E;
}
// The halves that are finite, the others as zero; `inf`: +-1 for each infinity, `nan`: 1 for each that is no number (zero else)
template <typename T>
__device__ __forceinline__ uint32_t split2(uint32_t x, uint32_t& inf, uint32_t& nan) {
	constexpr uint32_t E = std::is_same<T, bf16>::value ? 0x7f80 : 0x7c00, M = 0x7fff ^ E, ONE = std::is_same<T, bf16>::value ? 0x3f80 : 0x3c00;
	uint32_t y = 0;
	inf = nan = 0;
#pragma unroll
	for (int s = 0; s < 32; s += 16) {
		const uint32_t h = x >> s & 0xffff;
		if ((h & E) != E) y |= h << s;
		else if (h & M) nan |= ONE << s;
		else inf |= (ONE | (h & 0x8000)) << s;
	}
	return y;
}

// a sequence of the batch whose description makes sense
__device__ __forceinline__ bool there(const C16& c, int rows, int b) {
	const int n = c.count[b], p0 = c.pos0[b], start = c.start[b];
	return n >= 1 && p0 >= 0 && p0 <= INT_MAX - n && start >= 0 && n <= rows - start;
}
// The rows of work unit z: tokens t0 .. t0 + tokens - 1 of the sequences first .. last; `prefix` positions are the group's.  false: nothing to do
struct Unit {
	int first, last, t0, tokens, prefix;
};
__device__ __forceinline__ bool unit_of(const C16& c, const Attend& a, int z, Unit& u) {
	if (a.families && z < c.groups) {
		const int f = c.first[z], m = c.members[z];
		if (f < 0 || m < 1 || f > c.n - m) return false;
		const long long t0 = c.start[f], t1 = (long long)c.start[f + m - 1] + c.count[f + m - 1];
		if (t0 < 0 || t1 <= t0 || t1 > a.rows) return false;
		u.first = f, u.last = f + m - 1, u.t0 = (int)t0, u.tokens = (int)(t1 - t0), u.prefix = max(c.positions[z], 0);
		return true;
	}
	const int b = a.families ? z - c.groups : z, g = c.groups ? c.group[b] : -1;
	const bool grouped = (unsigned)g < (unsigned)c.groups;
	if ((a.families && grouped) || !there(c, a.rows, b)) return false;
	u.first = u.last = b, u.t0 = c.start[b], u.tokens = c.count[b], u.prefix = grouped ? max(c.positions[g], 0) : 0;
	return true;
}
__device__ __forceinline__ int low_of(const Attend& a, int pos) { return a.window > 0 ? max(0, pos - a.window + 1) : 0; }

template <typename T, int D, int NQ>
__global__ void __launch_bounds__(32 * AR_WARPS, D <= 128 ? 3 : 1) k_c16_rows(const C16 c, const Attend a) {
	constexpr bool KEEP = D * NQ <= 128; // the queries' fragments stay in registers
	constexpr int KS = D / 16, MT = D / 16, PIECES = D / 8, TILE = 8 * NQ, LD = D + 4;
	extern __shared__ __align__(128) unsigned char ar_sm[];
	uint2* const qf = reinterpret_cast<uint2*>(ar_sm); // B fragments [KS][NQ][32]
	ArStage<D>* const ring = reinterpret_cast<ArStage<D>*>(ar_sm + (size_t)TILE * D * 2);
	__shared__ float fold_m[AR_WARPS][TILE], fold_l[AR_WARPS][TILE];
	__shared__ int row_seq[TILE], row_pos[TILE], row_seg[TILE];
	__shared__ int seg_slot[TILE + 1], seg_lo[TILE + 1], seg_hi[TILE + 1], seg_base[TILE + 1]; // the prefix and the sequences of the tile's rows: keys lo .. hi - 1 of a slot, first chunk
	__shared__ int list[4];                                                                     // segments, chunks, the rows' least and largest position
	const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
	const int kvh = blockIdx.y / a.shares, share = blockIdx.y - kvh * a.shares;
	Unit u;
	if (a.before) pdl_launch_next();
	if (!unit_of(c, a, blockIdx.z, u) || (long long)blockIdx.x * TILE >= (long long)u.tokens * a.group) {
		if (a.before) pdl_wait_prev();
		return;
	}
	const int row0 = blockIdx.x * TILE, rows = (int)min((long long)TILE, (long long)u.tokens * a.group - row0);
	const int H = c.heads, dim = c.dim;

	// which sequence and position each row has
	if (tid < TILE) row_seq[tid] = row_pos[tid] = -1;
	__syncthreads();
	for (int b = u.first + tid; b <= u.last; b += 32 * AR_WARPS)
		if (there(c, a.rows, b)) {
			const long long r0 = (long long)(c.start[b] - u.t0) * a.group - row0, r1 = r0 + (long long)c.count[b] * a.group;
			for (long long r = max(r0, 0LL); r < min(r1, (long long)rows); ++r) row_seq[r] = b, row_pos[r] = c.pos0[b] + (int)((r - r0) / a.group);
		}
	__syncthreads();
	if (warp == 0) {
		const int seq = lane < TILE ? row_seq[lane] : -1, pos = lane < TILE ? row_pos[lane] : -1;
		const int left = __shfl_up_sync(0xffffffffu, seq, 1), right = __shfl_down_sync(0xffffffffu, seq, 1);
		const bool head = seq >= 0 && (lane == 0 || left != seq), tail = seq >= 0 && (lane == 31 || right != seq);
		const uint32_t heads = __ballot_sync(0xffffffffu, head);
		const int seg = __popc(heads & (0xffffffffu >> (31 - lane))); // (1: the first; 0: the prefix)
		const int least = __reduce_min_sync(0xffffffffu, seq >= 0 ? pos : INT_MAX), most = __reduce_max_sync(0xffffffffu, pos);
		if (lane < TILE) row_seg[lane] = seq >= 0 ? seg : -1;
		if (head) {
			const int slot = c.slot[seq];
			seg_slot[seg] = slot, seg_lo[seg] = max(u.prefix, low_of(a, pos));
		}
		if (tail) seg_hi[seg] = min(pos + 1, c.reach(c.slot[seq]));
		if (lane == 0) {
			const int slot = c.slot[u.first];
			const bool with = a.families && least != INT_MAX;
			seg_slot[0] = slot, seg_lo[0] = with ? low_of(a, least) : 0, seg_hi[0] = with ? min(min(u.prefix, most + 1), c.reach(slot)) : 0;
		}
		__syncwarp();
		const int segs = __popc(heads) + 1;
		int chunks = lane < segs ? (max(seg_hi[lane] - seg_lo[lane], 0) + AR_KEYS - 1) / AR_KEYS : 0, sum = chunks;
#pragma unroll
		for (int o = 1; o < 32; o *= 2) {
			const int x = __shfl_up_sync(0xffffffffu, sum, o);
			if (lane >= o) sum += x;
		}
		if (lane < segs) seg_base[lane] = sum - chunks;
		if (lane == segs - 1) list[0] = segs, list[1] = sum, list[2] = least, list[3] = most;
	}
	__syncthreads();
	const int segs = list[0], total = list[1], least = list[2], most = list[3];
	const int my_base = lane < segs ? seg_base[lane] : INT_MAX; // (at most 17 segments)
	const int begin = (int)min((long long)total, (long long)share * a.each), end = share == a.shares - 1 ? total : min(total, begin + a.each); // (more keys than were planned for: the last share's)
	const bool whole = a.shares == 1 || (a.cluster && total <= a.each); // no other share has keys
	if (whole && share > 0) return;                                     // (nor does any of the cluster wait)

	// the chunk to request: its segment, first position and end; the page of this lane's key, as the table has it: a load that nothing waits for where it is asked for
	ArStage<D>& s = ring[warp];
	int next = begin + warp, next_seg = 0, next_pos = 0, next_hi = 0, next_page = 0, next_row = 0;
	uint32_t next_seen = 0;
	bool page_ok = false;
	auto look = [&]() {
		const bool some = next < end;
		next_seg = some ? __popc(__ballot_sync(0xffffffffu, my_base <= next)) - 1 : 0;
		// (segments without keys start where the next one does: the last of those that start here has the chunk)
		next_hi = seg_hi[next_seg], next_pos = seg_lo[next_seg] + (next - seg_base[next_seg]) * AR_KEYS;
		const int pos = next_pos + lane, at = c.page_index(max(pos, 0));
		page_ok = some && pos < next_hi && at < c.table_pages;
		next_page = page_ok ? __ldg(c.table + (size_t)seg_slot[next_seg] * c.table_pages + at) : -1;
	};
	look();
	const int piece = lane % PIECES, prow = lane / PIECES; // which piece of which row of a group of 32 pieces this lane copies
	auto copy = [&](uint16_t* to, const uint16_t* from) { // the next chunk's keys or values
		const uint32_t dst = smem_u32(to);
		if (next_seen == 0xffffffffu && dim == D) {
#pragma unroll
			for (int i = 0; i < PIECES; ++i) { // 32 rows of PIECES pieces, 32 pieces at a time
				const int r = i * (32 / PIECES) + prow;
				const long long o = (long long)__shfl_sync(0xffffffffu, next_row, r) * D;
				cp16(dst + (r * PIECES + (piece ^ (r & 7))) * 16, from + o + piece * 8);
			}
		} else {
#pragma unroll
			for (int i = 0; i < PIECES; ++i) { // keys that are not there are zeros
				const int r = i * (32 / PIECES) + prow;
				const long long o = (long long)__shfl_sync(0xffffffffu, next_row, r) * dim;
				const bool some = (next_seen >> r & 1) && piece * 8 < dim;
				cp16(dst + (r * PIECES + (piece ^ (r & 7))) * 16, some ? from + o + piece * 8 : from, some);
			}
		}
	};
	auto request_keys = [&]() {
		if (next < end) {
			const bool some = page_ok && (unsigned)next_page < (unsigned)c.pages;
			next_seen = __ballot_sync(0xffffffffu, some);
			next_row = some ? (next_page * H + kvh) * c.page + c.page_row(next_pos + lane) : 0; // (rows of a pool: under 2^31)
			copy(s.k, c.k);
		}
		asm volatile("cp.async.commit_group;" ::: "memory");
	};
	int cur_seg = 0, cur_pos = 0;
	uint32_t cur_seen = 0;
	auto request_values = [&]() { // of the chunk whose keys were requested last
		cur_seg = next_seg, cur_pos = next_pos, cur_seen = next_seen;
		if (next < end) {
			copy(s.v, c.v);
			next += AR_WARPS;
			look();
		}
		asm volatile("cp.async.commit_group;" ::: "memory");
	};
	request_keys(), request_values();

	// queries as B fragments
	for (int i = tid; i < KS * NQ * 32; i += 32 * AR_WARPS) {
		const int k = i / (NQ * 32), r = (i / 32 % NQ) * 8 + (i >> 2 & 7), d = k * 16 + (i & 3) * 2, rr = row0 + min(r, rows - 1);
		const uint16_t* q = a.q + (long long)(u.t0 + rr / a.group) * a.q_row + (long long)(kvh * a.group + rr % a.group) * a.q_head + d;
		const bool some = r < rows && d < dim; // (16 channels are there or not)
		uint2 x = make_uint2(0, 0);
		if (some) x.x = q[0] | (uint32_t)q[1] << 16, x.y = q[8] | (uint32_t)q[9] << 16;
		qf[i] = x;
	}
	__syncthreads();
	uint2 qr[KEEP ? KS * NQ : 1];
	if (KEEP) {
#pragma unroll
		for (int i = 0; i < KS * NQ; ++i) qr[i] = qf[i * 32 + lane];
	}
	auto qfrag = [&](int i) { return KEEP ? qr[i] : qf[i * 32 + lane]; };
	const float qscale = a.softcap > 0.f ? a.scale : a.scale * A16_LOG2E;

	float acc[MT][NQ][4], m[NQ][2], l[NQ][2]; // queries 2t and 2t + 1 of each eight; m: the reference
	int rpos[NQ][2], rseg[NQ][2];
#pragma unroll
	for (int q = 0; q < NQ; ++q) {
#pragma unroll
		for (int i = 0; i < MT; ++i) acc[i][q][0] = acc[i][q][1] = acc[i][q][2] = acc[i][q][3] = 0.f;
#pragma unroll
		for (int e = 0; e < 2; ++e) m[q][e] = -INFINITY, l[q][e] = 0.f, rpos[q][e] = row_pos[8 * q + 2 * t + e], rseg[q][e] = row_seg[8 * q + 2 * t + e];
	}
	const int wide = low_of(a, most); // from here on, and up to `least`, every row sees every key of a segment that is its own
	const uint32_t lrow = lane & 7;

	for (int chunk = begin + warp; chunk < end; chunk += AR_WARPS) {
		const int seg = cur_seg, pos = cur_pos;
		const uint32_t seen = cur_seen;
		asm volatile("cp.async.wait_group 1;" ::: "memory"); // the keys; the values are the group behind them
		__syncwarp();
		// scores: rows g and g + 8 of product i are keys 16 i + g, + 8
		float z[2][NQ][4];
#pragma unroll
		for (int i = 0; i < 2; ++i)
#pragma unroll
			for (int q = 0; q < NQ; ++q) z[i][q][0] = z[i][q][1] = z[i][q][2] = z[i][q][3] = 0.f;
#pragma unroll
		for (int k = 0; k < KS; ++k) {
			if (16 * k >= dim) break;
			uint2 b[NQ];
#pragma unroll
			for (int q = 0; q < NQ; ++q) b[q] = qfrag(k * NQ + q);
#pragma unroll
			for (int i = 0; i < 2; ++i) {
				uint32_t A[4];
				ldsm_x4(s.k + ((16 * i + (lane & 8) + lrow) * PIECES + ((2 * k + (lane >> 4)) ^ lrow)) * 8, A);
#pragma unroll
				for (int q = 0; q < NQ; ++q) mma_16<T>(z[i][q], A, b[q]);
			}
		}
		__syncwarp(); // every lane has its keys
		request_keys();
		if (a.softcap > 0.f) {
			const float cap = a.softcap * A16_LOG2E, by = qscale / a.softcap;
#pragma unroll
			for (int i = 0; i < 2; ++i)
#pragma unroll
				for (int q = 0; q < NQ; ++q)
#pragma unroll
					for (int e = 0; e < 4; ++e) z[i][q][e] = cap * tanhf(z[i][q][e] * by);
		} else {
#pragma unroll
			for (int i = 0; i < 2; ++i)
#pragma unroll
				for (int q = 0; q < NQ; ++q)
#pragma unroll
					for (int e = 0; e < 4; ++e) z[i][q][e] *= qscale;
		}
		const bool all = seen == 0xffffffffu && (seg == 0 || segs == 2) && pos >= wide && pos + AR_KEYS - 1 <= least;
		if (!all) { // some row does not see some key; this thread's keys are 8 j + g
#pragma unroll
			for (int j = 0; j < 4; ++j) {
				const int kp = pos + 8 * j + g;
				const bool some = seen >> (8 * j + g) & 1;
#pragma unroll
				for (int q = 0; q < NQ; ++q)
#pragma unroll
					for (int e = 0; e < 2; ++e)
						if (!(some && kp <= rpos[q][e] && kp >= low_of(a, rpos[q][e]) && (seg == 0 || seg == rseg[q][e]))) z[j >> 1][q][(j & 1) * 2 + e] = -INFINITY;
			}
		}
		bool move = false;
#pragma unroll
		for (int q = 0; q < NQ; ++q)
#pragma unroll
			for (int e = 0; e < 2; ++e) move |= fmaxf(fmaxf(z[0][q][e], z[0][q][2 + e]), fmaxf(z[1][q][e], z[1][q][2 + e])) > m[q][e] + A16_MOST;
		if (__any_sync(0xffffffffu, move)) { // references move
#pragma unroll
			for (int q = 0; q < NQ; ++q) {
				float f[2];
#pragma unroll
				for (int e = 0; e < 2; ++e) {
					float top = fmaxf(fmaxf(z[0][q][e], z[0][q][2 + e]), fmaxf(z[1][q][e], z[1][q][2 + e]));
#pragma unroll
					for (int o = 4; o < 32; o *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
					const float mn = top > m[q][e] + A16_MOST ? top - A16_SET : m[q][e];
					f[e] = m[q][e] == -INFINITY ? 0.f : ex2(m[q][e] - mn);
					m[q][e] = mn, l[q][e] *= f[e];
				}
#pragma unroll
				for (int i = 0; i < MT; ++i) acc[i][q][0] *= f[0], acc[i][q][1] *= f[1], acc[i][q][2] *= f[0], acc[i][q][3] *= f[1];
			}
		}
		// weights, from keys x queries to the B fragments of queries x keys
		uint2 p[2][NQ];
#pragma unroll
		for (int q = 0; q < NQ; ++q) {
			const float base[2] = {m[q][0] == -INFINITY ? 0.f : m[q][0], m[q][1] == -INFINITY ? 0.f : m[q][1]};
#pragma unroll
			for (int i = 0; i < 2; ++i) {
#pragma unroll
				for (int e = 0; e < 4; ++e) {
					z[i][q][e] = ex2(z[i][q][e] - base[e & 1]);
					l[q][e & 1] += z[i][q][e];
				}
				p[i][q] = make_uint2(transposed(pack2<T>(z[i][q][0], z[i][q][1])), transposed(pack2<T>(z[i][q][2], z[i][q][3])));
			}
		}
		asm volatile("cp.async.wait_group 1;" ::: "memory"); // the values; the next keys are the group behind them
		__syncwarp();
		// values: rows g and g + 8 of product i are channels 16 i + g, + 8
#pragma unroll
		for (int kk = 0; kk < 2; ++kk)
#pragma unroll
			for (int i = 0; i < MT; ++i) {
				if (16 * i >= dim) break;
				uint32_t A[4];
				ldsm_x4_t(s.v + ((16 * kk + (lane >> 4) * 8 + lrow) * PIECES + ((2 * i + (lane >> 3 & 1)) ^ lrow)) * 8, A);
				if (!all && __any_sync(0xffffffffu, odd2<T>(A[0]) || odd2<T>(A[1]) || odd2<T>(A[2]) || odd2<T>(A[3]))) { // a value that is not finite reaches the rows that see its key and no others
					uint32_t inf[4], nan[4];
#pragma unroll
					for (int x = 0; x < 4; ++x) A[x] = split2<T>(A[x], inf[x], nan[x]);
#pragma unroll
					for (int q = 0; q < NQ; ++q) {
						float s_inf[4] = {0.f, 0.f, 0.f, 0.f}, s_nan[4] = {0.f, 0.f, 0.f, 0.f};
						mma_16<T>(s_inf, inf, p[kk][q]), mma_16<T>(s_nan, nan, p[kk][q]);
#pragma unroll
						for (int x = 0; x < 4; ++x) {
							if (s_nan[x] != 0.f) acc[i][q][x] = NAN;
							else if (s_inf[x] != 0.f) acc[i][q][x] += s_inf[x] * INFINITY;
						}
					}
				}
#pragma unroll
				for (int q = 0; q < NQ; ++q) mma_16<T>(acc[i][q], A, p[kk][q]);
			}
		__syncwarp(); // every lane has its values
		request_values();
	}
	asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
	for (int q = 0; q < NQ; ++q)
#pragma unroll
		for (int e = 0; e < 2; ++e) {
#pragma unroll
			for (int o = 4; o < 32; o *= 2) l[q][e] += __shfl_xor_sync(0xffffffffu, l[q][e], o);
			if (g == 0) fold_m[warp][8 * q + 2 * t + e] = m[q][e], fold_l[warp][8 * q + 2 * t + e] = l[q][e];
		}
	if (a.before) pdl_wait_prev(); // the prefixes' shares

	// the warps' sums as one, eight rows at a time
	float* const sums = reinterpret_cast<float*>(ring); // [warps][8][LD]
	float* const own = sums + AR_WARPS * 8 * LD;        // [TILE][D + 2]: what this share of a cluster found
	const int prefix_places = whole && c.groups && (unsigned)c.group[u.first] < (unsigned)c.groups ? a.before : 0;
#pragma unroll
	for (int q = 0; q < NQ; ++q) {
		if (8 * q >= rows) break;
		__syncthreads();
#pragma unroll
		for (int e = 0; e < 2; ++e) {
			float* const to = sums + (warp * 8 + 2 * t + e) * LD + g;
#pragma unroll
			for (int i = 0; i < MT; ++i) to[16 * i] = acc[i][q][e], to[16 * i + 8] = acc[i][q][2 + e];
		}
		__syncthreads();
		for (int rr = warp; rr < min(8, rows - 8 * q); rr += AR_WARPS) {
			const int r = 8 * q + rr;
			if (row_seq[r] < 0) continue;
			float mx = fold_m[0][r], den = 0.f, wt[AR_WARPS];
#pragma unroll
			for (int w = 1; w < AR_WARPS; ++w) mx = fmaxf(mx, fold_m[w][r]);
#pragma unroll
			for (int w = 0; w < AR_WARPS; ++w) wt[w] = fold_m[w][r] == -INFINITY ? 0.f : ex2(fold_m[w][r] - mx), den = fmaf(wt[w], fold_l[w][r], den);
			const int token = u.t0 + (row0 + r) / a.group, head = kvh * a.group + (row0 + r) % a.group;
			const size_t place = ((size_t)token * a.heads + head) * a.places;
			if (whole) {
				// with the prefix's shares, and a sink: one more term of the denominator
				const float sk = a.sinks ? a.sinks[head] * A16_LOG2E : -INFINITY;
				float top = fmaxf(mx, sk), pm = -INFINITY, pl = 0.f;
				if (lane < prefix_places) {
					const float2 st = a.stats[place + lane];
					pm = st.x, pl = st.y;
				}
				top = fmaxf(top, warp_max(pm));
				const float pw = pm == -INFINITY ? 0.f : ex2(pm - top), down = mx == -INFINITY ? 0.f : ex2(mx - top);
				den = den * down + warp_sum(pw * pl);
				if (a.sinks) den += at_sink(sk, top);
				const float norm = den > 0.f ? 1.f / den : den == 0.f ? 0.f : den; // (0: nothing was seen; a NaN stays one)
				for (int d0 = 0; d0 < dim; d0 += 32) {
					const int d = d0 + lane;
					float v = 0.f;
					if (d < dim) {
#pragma unroll
						for (int w = 0; w < AR_WARPS; ++w) v = fmaf(wt[w], sums[(w * 8 + rr) * LD + d], v);
						v *= down;
					}
					for (int k = 0; k < prefix_places; ++k) {
						const float f = __shfl_sync(0xffffffffu, pw, k);
						if (f != 0.f && d < dim) v = fmaf(f, a.sums[(place + k) * dim + d], v);
					}
					if (d < dim) a.out[token * a.o_row + head * a.o_head + d] = round16<T>(v * norm);
				}
			} else {
				float2* const st = a.cluster ? reinterpret_cast<float2*>(own + r * (D + 2) + D) : a.stats + place + a.before + share;
				float* const to = a.cluster ? own + r * (D + 2) : a.sums + (place + a.before + share) * dim;
				if (lane == 0) *st = make_float2(mx, den);
				if (mx != -INFINITY || a.cluster)
					for (int d = lane; d < dim; d += 32) {
						float v = 0.f;
#pragma unroll
						for (int w = 0; w < AR_WARPS; ++w) v = fmaf(wt[w], sums[(w * 8 + rr) * LD + d], v);
						to[d] = v;
					}
			}
		}
	}
	if (whole || !a.cluster) return;
	// A cluster's shares: each CTA finishes its part of the outputs from all of them.
	__shared__ float wz[AR_CLUSTER][TILE], inv[TILE];
	const int shares = min(a.shares, (total + a.each - 1) / a.each);
	cluster_sync();
	if (tid < rows) {
		const int head = kvh * a.group + (row0 + tid) % a.group;
		const float sk = a.sinks ? a.sinks[head] * A16_LOG2E : -INFINITY;
		float ms[AR_CLUSTER], ls[AR_CLUSTER], mx = sk, den = 0.f;
#pragma unroll
		for (int k = 0; k < AR_CLUSTER; ++k) {
			ms[k] = -INFINITY, ls[k] = 0.f;
			if (k < shares) ms[k] = cluster_load_f32(cluster_addr(own + tid * (D + 2) + D, k)), ls[k] = cluster_load_f32(cluster_addr(own + tid * (D + 2) + D + 1, k));
		}
#pragma unroll
		for (int k = 0; k < AR_CLUSTER; ++k) mx = fmaxf(mx, ms[k]);
#pragma unroll
		for (int k = 0; k < AR_CLUSTER; ++k)
			if (k < shares) {
				const float f = ms[k] == -INFINITY ? 0.f : ex2(ms[k] - mx);
				wz[k][tid] = f, den = fmaf(f, ls[k], den);
			}
		if (a.sinks) den += at_sink(sk, mx);
		inv[tid] = den > 0.f ? 1.f / den : den; // (0: nothing was seen)
	}
	__syncthreads();
	const int all = rows * dim, from = (int)((long long)all * share / a.shares), to = (int)((long long)all * (share + 1) / a.shares);
	for (int e = from + tid; e < to; e += 32 * AR_WARPS) {
		const int r = e / dim, d = e - r * dim;
		float v = 0.f;
#pragma unroll 8
		for (int k = 0; k < shares; ++k) v = fmaf(cluster_load_f32(cluster_addr(own + r * (D + 2) + d, k)), wz[k][r], v);
		if (row_seq[r] >= 0) a.out[(u.t0 + (row0 + r) / a.group) * a.o_row + (kvh * a.group + (row0 + r) % a.group) * a.o_head + d] = round16<T>(v * inv[r]);
	}
	cluster_sync(); // no CTA leaves while another reads what it found
}

// Folds the shares of one (token, head), in the order of their places: a warp for each.
template <typename T>
__global__ void __launch_bounds__(128) k_c16_fold(const C16 c, const Attend a) {
	pdl_wait_prev();
	const int b = blockIdx.z, kvh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
	if (!there(c, a.rows, b)) return;
	const int n = c.count[b], start = c.start[b];
	const int from = a.before && !(c.groups && (unsigned)c.group[b] < (unsigned)c.groups) ? a.before : 0; // (a sequence of no group has no shares of a prefix)
	for (long long row = (long long)blockIdx.x * 4 + warp; row < (long long)n * a.group; row += gridDim.x * 4) {
		const int token = start + (int)(row / a.group), head = kvh * a.group + (int)(row % a.group);
		const size_t place = ((size_t)token * a.heads + head) * a.places;
		const float sk = a.sinks ? a.sinks[head] * A16_LOG2E : -INFINITY;
		float mx = sk, den = 0.f;
		for (int s = from + lane; s < a.places; s += 32) mx = fmaxf(mx, a.stats[place + s].x);
		mx = warp_max(mx);
		float v[8];
#pragma unroll
		for (int k = 0; k < 8; ++k) v[k] = 0.f;
		for (int s0 = from; s0 < a.places; s0 += 32) {
			const float2 st = s0 + lane < a.places ? a.stats[place + s0 + lane] : make_float2(-INFINITY, 0.f);
			const float w = st.x == -INFINITY ? 0.f : ex2(st.x - mx);
			den = fmaf(w, st.y, den);
			for (int s = s0; s < min(a.places, s0 + 32); ++s) {
				const float f = __shfl_sync(0xffffffffu, w, s - s0);
				if (f == 0.f) continue; // (nothing may have been written there)
				const float* const p = a.sums + (place + s) * c.dim;
#pragma unroll
				for (int k = 0; k < 8; ++k)
					if (32 * k + lane < c.dim) v[k] = fmaf(f, p[32 * k + lane], v[k]);
			}
		}
		den = warp_sum(den);
		if (a.sinks) den += at_sink(sk, mx);
		const float norm = den > 0.f ? 1.f / den : den == 0.f ? 0.f : den; // (0: nothing was seen; a NaN stays one)
#pragma unroll
		for (int k = 0; k < 8; ++k)
			if (32 * k + lane < c.dim) a.out[token * a.o_row + head * a.o_head + 32 * k + lane] = round16<T>(v[k] * norm);
	}
}

// ---------------------------------------------------------------- the host's side
// How the work is cut: rows of a CTA, shares of a tile's keys and the chunks of each, whether a cluster folds the shares.
struct A16Plan {
	int tile, shares, each, cluster;
	int units; // of the grid
	long long most_rows; // of a unit
};
constexpr int AR_ROOM = 148 * 3; // CTAs that run at a time

A16Plan a16_plan(const SeqCache16& c, const SeqPortions& p, const SeqShared* s, const SeqAttend16& a) {
	A16Plan r = {};
	const int group = a.heads / c.heads, groups = s ? s->n : 0;
	const long long tokens = std::max<long long>(p.longest, groups ? s->tokens : 0), rows = tokens * group;
	r.units = p.n + groups, r.most_rows = rows;
	const int units = groups ? std::max(groups, 1) : p.n; // (about: which sequences are in no group is the device's to know)
	auto ctas = [&](int tile) { return (long long)units * cdiv(rows, tile) * c.heads; };
	r.tile = rows > 8 ? 16 : 8;
	const int own = groups ? std::max(s->most_own, 1) : std::max(a.most_keys, 1);
	long long keys = (groups ? s->longest : 0) + (long long)own * (groups ? std::min<long long>(cdiv(r.tile, group), std::max(s->tokens, 1)) : 1);
	if (a.window > 0) keys = std::min(keys, (long long)a.window + r.tile / group + own);
	const int chunks = std::max(1, (int)std::min<long long>(cdiv(keys, AR_KEYS), INT_MAX / 2));
	const long long n = std::max(1LL, ctas(r.tile)), room = AR_ROOM;
	long long shares = n >= room ? 1 : n > room / 2 ? cdiv(6 * room, n) : room / n;
	shares = std::max(1LL, std::min({shares, (long long)cdiv(chunks, n > room / 2 ? 2 * AR_WARPS : AR_WARPS), (long long)AR_SHARES}));
	r.cluster = shares > 1 && n <= room / 2;
	if (r.cluster) shares = shares >= 16 ? 16 : shares >= 8 ? 8 : shares >= 4 ? 4 : 2;
	r.each = cdiv(chunks, shares), r.shares = r.cluster ? (int)shares : cdiv(chunks, r.each);
	return r;
}
int a16_places(const A16Plan& p) { return p.shares > 1 && !p.cluster ? p.shares : 0; }
size_t a16_bytes(const SeqCache16& c, const SeqAttend16& a, const A16Plan& p) { return (size_t)a.q.rows * a.heads * a16_places(p) * (c.dim * sizeof(float) + sizeof(float2)); }

int check_attend16(const SeqCache16* c, const SeqPortions* p, const SeqShared* s, const SeqAttend16* a) {
	if (const int rc = check_cache16("attend16", c, p)) return rc;
	if (!a) return refuse("attend16: no arguments");
	if (const int rc = check_rows("attend16", "q", a->q)) return rc;
	if (const int rc = check_rows("attend16", "out", a->out)) return rc;
	if (a->q.type != c->type || a->out.type != c->type) return refuse("attend16: q has type %d, out %d, the cache %d: one type for all", a->q.type, a->out.type, c->type);
	if (a->out.rows < a->q.rows) return refuse("attend16: out has %d rows, q %d", a->out.rows, a->q.rows);
	if (a->heads < 1 || a->heads % c->heads) return refuse("attend16: %d query heads over %d key heads", a->heads, c->heads);
	if (a->heads > 65535) return refuse("attend16: at most 65535 query heads");
	const long long group = a->heads / c->heads;
	if (s) {
		if (s->n < 0 || s->n > p->n || s->longest < 0 || s->tokens < 0 || s->most_own < 0) return refuse("attend16: %d groups of %d sequences, longest %d, tokens %d", s->n, p->n, s->longest, s->tokens);
		if (s->n && (!s->first || !s->count || !s->positions || !s->group)) return refuse("attend16: the groups' description is missing");
		if (((uintptr_t)s->first | (uintptr_t)s->count | (uintptr_t)s->positions | (uintptr_t)s->group) % 4) return refuse("attend16: the groups' description is not aligned to 4 bytes");
		if (p->n + s->n > 65535) return refuse("attend16: %d sequences and %d groups: at most 65535", p->n, s->n);
	}
	if (std::max(p->longest, s && s->n ? s->tokens : 0) * group > INT_MAX - 256) return refuse("attend16: %d tokens of %d query heads a key head: at most 2^31 pairs a sequence or group", std::max(p->longest, s ? s->tokens : 0), (int)group);
	if ((uintptr_t)a->sinks % 4) return refuse("attend16: sinks are not aligned to 4 bytes");
	if (!(a->scale == a->scale) || a->window < 0 || !(a->softcap >= 0.f)) return refuse("attend16: scale, window or softcap out of range");
	return 0;
}

template <typename T, int D, int NQ>
cudaError_t rows_launch(const C16& c, const Attend& a, dim3 grid, bool after, cudaStream_t st) {
	constexpr size_t smem = ar_smem<D, NQ>();
	static std::atomic<uint64_t> done{0};
	cudaError_t e = allow(k_c16_rows<T, D, NQ>, smem, done, true);
	if (e == cudaSuccess) e = launch(st, after, a.cluster ? a.shares : 1, k_c16_rows<T, D, NQ>, grid, dim3(32 * AR_WARPS), smem, c, a);
	return e;
}
template <typename T, int D>
cudaError_t rows_tile(int tile, const C16& c, const Attend& a, dim3 grid, bool after, cudaStream_t st) {
	return tile == 8 ? rows_launch<T, D, 1>(c, a, grid, after, st) : rows_launch<T, D, 2>(c, a, grid, after, st);
}
template <typename T>
cudaError_t rows_wide(int tile, const C16& c, const Attend& a, dim3 grid, bool after, cudaStream_t st) {
	return c.dim <= 64 ? rows_tile<T, 64>(tile, c, a, grid, after, st) : c.dim <= 128 ? rows_tile<T, 128>(tile, c, a, grid, after, st) : rows_tile<T, 256>(tile, c, a, grid, after, st);
}
} // namespace
} // namespace seqops

extern "C" size_t calm_b200_seq_attend16_workspace(const struct SeqCache16* cache, const struct SeqPortions* batch, const struct SeqShared* shared, const struct SeqAttend16* args) {
	using namespace seqops;
	if (check_attend16(cache, batch, shared, args)) return 0;
	return a16_bytes(*cache, *args, a16_plan(*cache, *batch, shared, *args));
}

extern "C" int calm_b200_seq_attend16(const struct SeqCache16* cache, const struct SeqPortions* batch, const struct SeqShared* shared, const struct SeqAttend16* q, void* stream) {
	using namespace seqops;
	if (const int rc = check_attend16(cache, batch, shared, q)) return rc;
	if (batch->n == 0 || batch->longest == 0) return 0;
	const A16Plan plan = a16_plan(*cache, *batch, shared, *q);
	const size_t need = a16_bytes(*cache, *q, plan);
	if (need && (!q->workspace || (uintptr_t)q->workspace % 16 || q->workspace_bytes < need)) return refuse("attend16: the workspace has %zu bytes (16-byte aligned), %zu are needed", q->workspace ? q->workspace_bytes : (size_t)0, need);
	C16 c = {};
	c.k = (const uint16_t*)cache->k, c.v = (const uint16_t*)cache->v, c.table = cache->table, c.pages = cache->pages, c.heads = cache->heads, c.page = cache->page, c.dim = cache->dim;
	c.slots = cache->slots, c.table_pages = cache->table_pages, c.page_shift = log2_of(cache->page), c.start = batch->start, c.count = batch->count, c.slot = batch->slot, c.pos0 = batch->pos0, c.n = batch->n;
	if (shared && shared->n) c.groups = shared->n, c.first = shared->first, c.members = shared->count, c.positions = shared->positions, c.group = shared->group;
	Attend a = {};
	a.q = (const uint16_t*)q->q.p, a.q_row = q->q.row_stride, a.q_head = q->q.head_stride, a.out = (uint16_t*)q->out.p, a.o_row = q->out.row_stride, a.o_head = q->out.head_stride;
	a.rows = q->q.rows, a.heads = q->heads, a.group = q->heads / cache->heads, a.scale = q->scale, a.softcap = q->softcap, a.window = q->window, a.sinks = q->sinks;
	a.families = 1, a.shares = plan.shares, a.each = plan.each, a.cluster = plan.cluster, a.before = 0, a.places = a16_places(plan);
	a.sums = (float*)q->workspace, a.stats = (float2*)(a.sums + (size_t)a.rows * a.heads * a.places * c.dim);
	const dim3 grid(cdiv(plan.most_rows, plan.tile), cache->heads * plan.shares, plan.units);
	if (grid.y > 65535) return refuse("attend16: too many key heads");
	const cudaStream_t st = (cudaStream_t)stream;
	const bool half = cache->type == SEQ_F16;
	cudaError_t e = half ? rows_wide<__half>(plan.tile, c, a, grid, false, st) : rows_wide<bf16>(plan.tile, c, a, grid, false, st);
	if (e == cudaSuccess && a.places) {
		const dim3 fold(std::min(cdiv((long long)batch->longest * a.group, 4), 65535), cache->heads, batch->n);
		e = launch(st, true, 1, half ? k_c16_fold<__half> : k_c16_fold<bf16>, fold, dim3(128), 0, c, a);
	}
	return e == cudaSuccess ? 0 : failed("attend16", e);
}
