// seqattend16.cu -- attention over a paged cache in 16 bits, where groups of sequences share a prefix (calm_b200_seq_attend16 in include/calm_b200_seq.h).

#include "seqcache16.cuh"
#include "tc05.cuh"

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
	int groups, alone; // groups; sequences of none
	const int *first, *members, *positions, *group, *lonely;
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
	int out_vec;            // four channels of a result at a time
	float scale, softcap;
	int window;
	const float* sinks;
	int families;     // 1: groups with their prefixes and own keys, and the sequences of no group; 0: every sequence behind what it shares;
	                  // -t: k_c16_rows has the sequences of at most t tokens with their prefixes, k_c16_tiles the others, both at once
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
// Bound: memory where keys are many - 32 sequences of up to 6000 keys, 8 key heads of 128 channels (500 MB) 86 us, 5.8 TB/s with the fold - and the way of a chunk (copy, products, softmax, products) where they are few: 4 sequences
// behind 4000 shared ones 13.2 us, 64 CTAs. Masked or capped scores cost instructions: 18 sequences of 5 tokens, window 2048, cap and sinks 37 us at 0.4 of the issue slots.
constexpr int AR_KEYS = 32; // (of a warp's chunk)
constexpr int AR_SHARES = 64;                // of a tile's keys at most
constexpr int AR_TILE = 16, AR_CLUSTER = 8; // rows of a CTA at most; shares that a thread-block cluster folds

template <int D>
struct ArStage { // a warp's chunk: the next one's keys come while its values are used, the next one's values while their keys are
	uint16_t k[AR_KEYS * D], v[AR_KEYS * D];
};
template <int D, int W>
__host__ __device__ constexpr size_t ar_ring() { // (the sums of the warps take its place)
	const size_t a = (size_t)W * sizeof(ArStage<D>), b = ((size_t)W * AR_TILE * (D + 4) + (size_t)AR_TILE * (D + 2)) * sizeof(float);
	return a > b ? a : b;
}
template <int D, int NQ, int W>
constexpr size_t ar_smem() { return (size_t)8 * NQ * D * 2 + ar_ring<D, W>(); }

template <typename T>
__device__ __forceinline__ void mma_16(float (&c)[4], const uint32_t (&a)[4], uint2 b) {
	if constexpr (std::is_same<T, bf16>::value)
		asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
		             : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
		             : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
	else
		asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
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
// four neighbouring channels of a result
template <typename T>
__device__ __forceinline__ void put4(uint16_t* to, bool vec, const float4& v) {
	const uint2 w = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w));
	if (vec) *reinterpret_cast<uint2*>(to) = w;
	else to[0] = (uint16_t)w.x, to[1] = (uint16_t)(w.x >> 16), to[2] = (uint16_t)w.y, to[3] = (uint16_t)(w.y >> 16);
}
__device__ __forceinline__ void add4(float4& v, float f, const float4& x) { v.x = fmaf(f, x.x, v.x), v.y = fmaf(f, x.y, v.y), v.z = fmaf(f, x.z, v.z), v.w = fmaf(f, x.w, v.w); }
__device__ __forceinline__ float4 times4(const float4& v, float f) { return make_float4(v.x * f, v.y * f, v.z * f, v.w * f); }
// `sum` becomes no number where one of the two halves is infinite or no number
template <typename T>
__device__ __forceinline__ void odd2(uint32_t x, uint32_t& sum) {
	if constexpr (std::is_same<T, bf16>::value) {
		const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&x), __nv_bfloat162(__float2bfloat16_rn(0.f), __float2bfloat16_rn(0.f)), *reinterpret_cast<const __nv_bfloat162*>(&sum));
		sum = *reinterpret_cast<const uint32_t*>(&r);
	} else {
		const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&x), __half2(__float2half_rn(0.f), __float2half_rn(0.f)), *reinterpret_cast<const __half2*>(&sum));
		sum = *reinterpret_cast<const uint32_t*>(&r);
	}
}
// The halves that are finite, the others as zero; `up`: 1 for each +infinity, `down`: 1 for each -infinity, both for each that is no number (zero else)
template <typename T>
__device__ __forceinline__ uint32_t split2(uint32_t x, uint32_t& up, uint32_t& down) {
	constexpr uint32_t E = std::is_same<T, bf16>::value ? 0x7f80 : 0x7c00, M = 0x7fff ^ E, ONE = std::is_same<T, bf16>::value ? 0x3f80 : 0x3c00;
	uint32_t y = 0;
	up = down = 0;
#pragma unroll
	for (int s = 0; s < 32; s += 16) {
		const uint32_t h = x >> s & 0xffff;
		if ((h & E) != E) y |= h << s;
		else {
			if (h & M || !(h & 0x8000)) up |= ONE << s;
			if (h & M || h & 0x8000) down |= ONE << s;
		}
	}
	return y;
}

// a sequence of the batch whose description makes sense
__device__ __forceinline__ bool there(const C16& c, int rows, int b) {
	const int n = c.count[b], p0 = c.pos0[b], start = c.start[b];
	return n >= 1 && p0 >= 0 && p0 <= INT_MAX - n && start >= 0 && n <= rows - start;
}
// The rows of a work unit: tokens t0 .. t0 + tokens - 1 of the sequences first .. last; `prefix` positions are the group's, found through sequence `lead`.  false: nothing to do
struct Unit {
	int first, last, lead, t0, tokens, prefix;
};
__device__ __forceinline__ bool group_unit(const C16& c, const Attend& a, int g, Unit& u) {
	const int f = c.first[g], m = c.members[g];
	if (f < 0 || m < 1 || f > c.n - m) return false;
	const long long t0 = c.start[f], t1 = (long long)c.start[f + m - 1] + c.count[f + m - 1];
	if (t0 < 0 || t1 <= t0 || t1 > a.rows) return false;
	u.first = u.lead = f, u.last = f + m - 1, u.t0 = (int)t0, u.tokens = (int)(t1 - t0), u.prefix = max(c.positions[g], 0);
	return true;
}
// a sequence; one that names a group is among that group's and has its rows among the group's
__device__ __forceinline__ bool own_unit(const C16& c, const Attend& a, int b, Unit& u) {
	const int g = c.groups ? c.group[b] : -1;
	if (!there(c, a.rows, b)) return false;
	u.prefix = 0, u.lead = -1;
	if ((unsigned)g < (unsigned)c.groups) {
		if (!group_unit(c, a, g, u) || b < u.first || b > u.last || c.start[b] < u.t0 || c.start[b] + c.count[b] > u.t0 + u.tokens) return false;
	}
	u.first = u.last = b, u.t0 = c.start[b], u.tokens = c.count[b];
	return true;
}
// v += what the shares at up to 32 places hold of four channels; lane k has the weight of place k.  All of them are asked for before one is used; where nothing weighs, nothing may have been written.
__device__ __forceinline__ void add_places(float4& v, const float* p, size_t stride, int places, float weight) {
#pragma unroll 1
	for (int k0 = 0; k0 < places; k0 += 8) {
		float4 x[8];
#pragma unroll
		for (int k = 0; k < 8; ++k)
			if (k0 + k < places) x[k] = *reinterpret_cast<const float4*>(p + (k0 + k) * stride);
#pragma unroll
		for (int k = 0; k < 8; ++k) {
			const float f = __shfl_sync(0xffffffffu, weight, k0 + k);
			if (k0 + k < places && f != 0.f) add4(v, f, x[k]);
		}
	}
}
// Soft caps: cap tanh(s / cap), off by 12 2^-24 of the score at most, whatever the cap.  For |u| = |s / cap| <= 1 it is s times the fifth convergent of tanh(u) / u = 1 / (1 + u^2 / (3 + u^2 / (5 + ...))), Lambert's
// continued fraction, (945 + 105 u^2 + u^4) / (945 + 420 u^2 + 15 u^4): off by 2^-24, with the roundings of two quotients' parts, a reciprocal and three products.  Else cap (1 - t) / (1 + t) with t = e^(-2 |u|), where 1 - t
// is 0.86 or more.  (That form alone is off by 2^-21 of the cap: at a cap of 10^6 no score is left.)
struct Cap {
	float by, most; // u of a product of query and key; the cap for exponents of 2
};
__device__ __forceinline__ Cap cap_of(const Attend& a) { // (u is 0 where scores are, and an infinity where they are)
	return {a.scale == 0.f ? 0.f : copysignf(fmaxf(fabsf(a.scale / a.softcap), 1.4e-45f), a.scale), fminf(a.softcap * A16_LOG2E, 3.40282347e38f)};
}
__device__ __forceinline__ float over(float x, float y) { // x / y for 1 <= y <= 2
	float r;
	asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y));
	return x * r;
}
// N products of query and key as capped exponents of 2; a warp reckons both forms where one of its scores is past the cap (a prompt of 8192 tokens, 32 heads over 8 of 128 channels: 1181 us, 1461 where all warps do, 597
// without a cap; a division in each form 1320 and 3407).
template <int N>
__device__ __forceinline__ void cap_scores(float (&z)[N], const Cap& cap, float qscale) {
	float top = 0.f;
#pragma unroll
	for (int i = 0; i < N; ++i) top = fmaxf(top, fabsf(z[i]));
	auto form = [&](float x, bool far) {
		const float u = x * cap.by, w = u * u;
		float num = x * qscale * fmaf(w, fmaf(w, 1.f / 945.f, 1.f / 9.f), 1.f), den = fmaf(w, fmaf(w, 1.f / 63.f, 4.f / 9.f), 1.f);
		if (far) {
			const float t = ex2(-2.f * A16_LOG2E * fabsf(u));
			num = fabsf(u) > 1.f ? copysignf(fmaf(-cap.most, t, cap.most), u) : num, den = fabsf(u) > 1.f ? 1.f + t : den;
		}
		return over(num, den);
	};
	if (__any_sync(0xffffffffu, top * fabsf(cap.by) > 1.f)) {
#pragma unroll
		for (int i = 0; i < N; ++i) z[i] = form(z[i], true);
	} else {
#pragma unroll
		for (int i = 0; i < N; ++i) z[i] = form(z[i], false);
	}
}
// chunks of the keys lo .. hi - 1, the first of which begins at a multiple of a chunk
__device__ __forceinline__ int chunks_of(int lo, int hi) { return hi > lo ? (hi - lo / AR_KEYS * AR_KEYS + AR_KEYS - 1) / AR_KEYS : 0; }
__device__ __forceinline__ int low_of(const Attend& a, int pos) { return a.window > 0 ? max(0, pos - a.window + 1) : 0; }

// CAP: with a soft cap.  (One kernel for both: 13.6 us for 13.2 without a cap, four beams behind 4000 positions, 18.3 for 17.8, 8 groups of 8 behind 3000.)
template <typename T, int D, int NQ, int W, bool CAP>
__global__ void __launch_bounds__(32 * W, W > 4 || D > 128 ? 1 : 3) k_c16_rows(const C16 c, const Attend a) {
	constexpr bool KEEP = D * NQ <= 128; // the queries' fragments stay in registers
	constexpr int KS = D / 16, MT = D / 16, PIECES = D / 8, TILE = 8 * NQ, LD = D + 4;
	extern __shared__ __align__(128) unsigned char ar_sm[];
	uint2* const qf = reinterpret_cast<uint2*>(ar_sm); // B fragments [KS][NQ][32]
	ArStage<D>* const ring = reinterpret_cast<ArStage<D>*>(ar_sm + (size_t)TILE * D * 2);
	__shared__ float fold_m[W][TILE], fold_l[W][TILE];
	__shared__ int row_seq[TILE], row_pos[TILE], row_seg[TILE], row_slot[TILE];
	__shared__ int seg_slot[TILE + 1], seg_lo[TILE + 1], seg_hi[TILE + 1], seg_base[TILE + 1]; // the prefix and the sequences of the tile's rows: keys lo .. hi - 1 of a slot, first chunk
	__shared__ long long row_place[TILE];                                                       // where a row's results go
	__shared__ int list[4];                                                                     // segments, chunks, the rows' least and largest position
	const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
	const int kvh = blockIdx.y / a.shares, share = blockIdx.y - kvh * a.shares;
	Unit u;
	if (a.before) pdl_launch_next();
	const int z = blockIdx.z;
	const bool grouped = a.families == 1 && c.groups;
	const int b = grouped ? (z < c.groups ? 0 : c.lonely[z - c.groups]) : z;
	bool some_rows = grouped && z < c.groups ? group_unit(c, a, z, u) : (unsigned)b < (unsigned)c.n && own_unit(c, a, b, u);
	if (some_rows && ((grouped && z >= c.groups && u.lead >= 0) || (u.first == u.last && !there(c, a.rows, u.first)))) some_rows = false; // (a sequence that its group has; a group of one that makes no sense)
	if (D <= 128 && some_rows && a.families < 0 && u.tokens > -a.families) some_rows = false;
	// The kernel before this one has ended when this one has: all blocks wait for what they read of it, or where they read nothing one does.
	auto wait = [&]() {
		if (a.before || (D <= 128 && a.families < 0 && !(blockIdx.x | blockIdx.y | blockIdx.z))) pdl_wait_prev();
	};
	if (!some_rows || (long long)blockIdx.x * TILE >= (long long)u.tokens * a.group) {
		wait();
		return;
	}
	const int row0 = blockIdx.x * TILE, rows = (int)min((long long)TILE, (long long)u.tokens * a.group - row0);
	const int H = c.heads, dim = c.dim;

	// the queries are asked for first
	constexpr int QF = KS * NQ * 32 / (32 * W) > 0 ? KS * NQ * 32 / (32 * W) : 1; // fragments of a thread
	uint2 qx[QF];
	{
		static_assert(W % NQ == 0, "all fragments of a thread are of one row");
		const int r = warp % NQ * 8 + g, rr = row0 + min(r, rows - 1), token = rr / a.group;
		const uint16_t* const q = a.q + (long long)(u.t0 + token) * a.q_row + (long long)(kvh * a.group + rr - token * a.group) * a.q_head + 2 * t;
#pragma unroll
		for (int f = 0; f < QF; ++f) {
			const int d = (warp + f * W) / NQ * 16;
			qx[f] = make_uint2(0, 0);
			if (r < rows && d < dim) qx[f].x = q[d] | (uint32_t)q[d + 1] << 16, qx[f].y = q[d + 8] | (uint32_t)q[d + 9] << 16; // (16 channels are there or not)
		}
	}
	// The first chunks of a prefix are asked for before the rest is known.  (Their keys are known without the rows where there is no window.)
	ArStage<D>& s = ring[warp];
	const int lead_slot = a.families && u.lead >= 0 ? c.slot[u.lead] : -1;
	const int prefix = a.window == 0 ? min(a.families ? u.prefix : 0, c.reach(lead_slot)) : 0;
	int next = (int)min((long long)INT_MAX / 2, (long long)share * a.each) + warp, next_seg = 0, next_pos = 0, next_lo = 0, next_hi = 0, next_page = 0, next_row = 0; // the chunk to request
	uint32_t next_seen = 0;
	bool page_ok = false;
	const bool early = next < chunks_of(0, prefix) && (share == a.shares - 1 || warp < a.each);
	auto ask = [&](bool some, int slot) { // for the page of this lane's key, as the table has it: a load that nothing waits for where it is asked for
		const int pos = next_pos + lane, at = c.page_index(max(pos, 0));
		page_ok = some && pos >= next_lo && pos < next_hi && at < c.table_pages;
		next_page = page_ok ? __ldg(c.table + (size_t)slot * c.table_pages + at) : -1;
	};
	if (early) next_hi = prefix, next_pos = next * AR_KEYS, ask(true, lead_slot);
	constexpr int EACH = 32 / PIECES;                      // rows that a warp copies at a time
	const int piece = lane % PIECES, prow = lane / PIECES; // which piece of which of them this lane copies
	const bool eights = c.page % 8 == 0 && dim == D;       // eight keys from a multiple of eight on lie side by side
	auto copy = [&](uint16_t* to, const uint16_t* from) { // the next chunk's keys or values
		const uint32_t dst = smem_u32(to);
		if (next_seen == 0xffffffffu && eights) {
#pragma unroll
			for (int g = 0; g < AR_KEYS / 8; ++g) {
				const uint16_t* const src = from + (long long)__shfl_sync(0xffffffffu, next_row, g * 8) * D + prow * D + piece * 8;
#pragma unroll
				for (int i = 0; i < 8; i += EACH) cp16(dst + (g * 8 + i) * PIECES * 16 + prow * PIECES * 16 + (((piece ^ prow) ^ i) << 4), src + i * D);
			}
		} else {
#pragma unroll 4
			for (int i = 0; i < PIECES; ++i) { // keys that are not there are zeros
				const int r = i * EACH + prow;
				const long long o = (long long)__shfl_sync(0xffffffffu, next_row, r) * dim;
				const bool some = (next_seen >> r & 1) && piece * 8 < dim;
				cp16(dst + (r * PIECES + (piece ^ (r & 7))) * 16, some ? from + o + piece * 8 : from, some);
			}
		}
	};
	auto copy_keys = [&]() {
		const bool some = page_ok && (unsigned)next_page < (unsigned)c.pages;
		next_seen = __ballot_sync(0xffffffffu, some);
		next_row = some ? (next_page * H + kvh) * c.page + c.page_row(next_pos + lane) : 0; // (rows of a pool: under 2^31)
		copy(s.k, c.k);
	};
	if (early) {
		copy_keys();
		asm volatile("cp.async.commit_group;" ::: "memory");
		copy(s.v, c.v);
		asm volatile("cp.async.commit_group;" ::: "memory");
	}
	// which sequence and position each row has; the segments of the tile's list of keys: 0 the prefix, then every sequence of its rows
	const bool alone = u.first == u.last;
	if (alone) { // one sequence: nothing to look for
		const int p0 = c.pos0[u.first] + (u.t0 - c.start[u.first]), low = p0 + row0 / a.group, high = p0 + (row0 + rows - 1) / a.group; // (a group of one has its sequence's rows)
		if (tid < TILE) row_seq[tid] = tid < rows ? u.first : -1, row_pos[tid] = tid < rows ? p0 + (row0 + tid) / a.group : -1, row_seg[tid] = tid < rows ? 1 : -1;
		if (tid == 0) {
			const int slot = c.slot[u.first], reach = c.reach(slot);
			const bool with = a.families && u.prefix > 0;
			const int lo0 = with ? low_of(a, low) : 0, hi0 = with ? (a.window ? min(min(u.prefix, high + 1), c.reach(lead_slot)) : prefix) : 0, lo1 = max(u.prefix, low_of(a, low)), hi1 = min(high + 1, reach);
			const int n0 = chunks_of(lo0, hi0), n1 = chunks_of(lo1, hi1);
			seg_slot[0] = lead_slot, seg_slot[1] = slot, seg_lo[0] = lo0, seg_hi[0] = hi0, seg_lo[1] = lo1, seg_hi[1] = hi1, seg_base[0] = 0, seg_base[1] = n0;
			list[0] = 2, list[1] = n0 + n1, list[2] = low, list[3] = high;
		}
	} else {
		if (tid < TILE) row_seq[tid] = row_pos[tid] = -1;
		__syncthreads();
		for (int b = u.first + tid; b <= u.last; b += 32 * W) {
			const int slot = c.slot[b], pos0 = c.pos0[b], start = c.start[b], count = c.count[b];
			if (!there(c, a.rows, b)) continue;
			const long long r0 = (long long)(start - u.t0) * a.group - row0, r1 = r0 + (long long)count * a.group;
			for (long long r = max(r0, 0LL); r < min(r1, (long long)rows); ++r) row_seq[r] = b, row_pos[r] = pos0 + (int)((unsigned)(r - r0) / (unsigned)a.group), row_slot[r] = slot;
		}
		__syncthreads();
		if (warp == 0) {
			const int seq = lane < TILE ? row_seq[lane] : -1, pos = lane < TILE ? row_pos[lane] : -1, slot = seq >= 0 ? row_slot[lane] : -1;
			const int left = __shfl_up_sync(0xffffffffu, seq, 1), right = __shfl_down_sync(0xffffffffu, seq, 1);
			const bool head = seq >= 0 && (lane == 0 || left != seq), tail = seq >= 0 && (lane == 31 || right != seq);
			const uint32_t heads = __ballot_sync(0xffffffffu, head);
			const int seg = __popc(heads & (0xffffffffu >> (31 - lane))); // (1: the first; 0: the prefix)
			const int least = __reduce_min_sync(0xffffffffu, seq >= 0 ? pos : INT_MAX), most = __reduce_max_sync(0xffffffffu, pos);
			if (lane < TILE) row_seg[lane] = seq >= 0 ? seg : -1;
			if (head) seg_slot[seg] = slot, seg_lo[seg] = max(u.prefix, low_of(a, pos));
			if (tail) seg_hi[seg] = min(pos + 1, c.reach(slot));
			if (lane == 0) {
				const bool with = u.prefix > 0 && least != INT_MAX;
				seg_slot[0] = lead_slot, seg_lo[0] = with ? low_of(a, least) : 0, seg_hi[0] = with ? (a.window ? min(min(u.prefix, most + 1), c.reach(lead_slot)) : prefix) : 0;
			}
			__syncwarp();
			const int segs = __popc(heads) + 1;
			int chunks = lane < segs ? chunks_of(seg_lo[lane], seg_hi[lane]) : 0, sum = chunks;
#pragma unroll
			for (int o = 1; o < 32; o *= 2) {
				const int x = __shfl_up_sync(0xffffffffu, sum, o);
				if (lane >= o) sum += x;
			}
			if (lane < segs) seg_base[lane] = sum - chunks;
			if (lane == segs - 1) list[0] = segs, list[1] = sum, list[2] = least, list[3] = most;
		}
	}
#pragma unroll
	for (int f = 0; f < QF; ++f)
		if (tid + f * 32 * W < KS * NQ * 32) qf[tid + f * 32 * W] = qx[f]; // B fragments
	__syncthreads();
	const int segs = list[0], total = list[1], least = list[2], most = list[3];
	const int begin = (int)min((long long)total, (long long)share * a.each), end = share == a.shares - 1 ? total : min(total, begin + a.each); // (more keys than were planned for: the last share's)
	const bool whole = a.shares == 1 || (a.cluster && total <= a.each); // no other share has keys

	if (whole && share > 0) {
		asm volatile("cp.async.wait_all;" ::: "memory");
		return; // (nor does any of the cluster wait)
	}
	const int my_base = lane < segs ? seg_base[lane] : INT_MAX; // (at most 17 segments)
	auto look = [&]() { // the chunk to request next: its segment, first position and end
		const bool some = next < end;
		// (segments without keys start where the next one does: the last of those that start here has the chunk)
		next_seg = some ? __popc(__ballot_sync(0xffffffffu, my_base <= next)) - 1 : 0;
		next_lo = seg_lo[next_seg], next_hi = seg_hi[next_seg], next_pos = (next_lo / AR_KEYS + next - seg_base[next_seg]) * AR_KEYS;
		ask(some, seg_slot[next_seg]);
	};
	int cur_seg = 0, cur_pos = next_pos;
	uint32_t cur_seen = next_seen;
	auto request_values = [&]() { // of the chunk whose keys were requested last
		cur_seg = next_seg, cur_pos = next_pos, cur_seen = next_seen;
		if (next < end) {
			copy(s.v, c.v);
			next += W;
			look();
		}
		asm volatile("cp.async.commit_group;" ::: "memory");
	};
	auto request_keys = [&]() {
		if (next < end) copy_keys();
		asm volatile("cp.async.commit_group;" ::: "memory");
	};
	if (early) next += W, look(); // (both are on their way)
	else look(), request_keys(), request_values();

	uint2 qr[KEEP ? KS * NQ : 1];
	if (KEEP) {
#pragma unroll
		for (int i = 0; i < KS * NQ; ++i) qr[i] = qf[i * 32 + lane];
	}
	auto qfrag = [&](int i) { return KEEP ? qr[i] : qf[i * 32 + lane]; };
	const float qscale = a.scale * A16_LOG2E;

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

	for (int chunk = begin + warp; chunk < end; chunk += W) {
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
		// (fragments of two steps are asked for while the last two's are used)
		constexpr int AHEAD = 2;
		uint32_t A[2][AHEAD][2][4];
		uint2 B[2][AHEAD][NQ];
		auto fetch = [&](int k0, uint32_t (&to)[AHEAD][2][4], uint2 (&b)[AHEAD][NQ]) {
#pragma unroll
			for (int k = 0; k < AHEAD; ++k) {
#pragma unroll
				for (int q = 0; q < NQ; ++q) b[k][q] = qfrag((k0 + k) * NQ + q);
#pragma unroll
				for (int i = 0; i < 2; ++i) ldsm_x4(s.k + ((16 * i + (lane & 8) + lrow) * PIECES + ((2 * (k0 + k) + (lane >> 4)) ^ lrow)) * 8, to[k][i]);
			}
		};
		fetch(0, A[0], B[0]);
#pragma unroll
		for (int k0 = 0; k0 < KS; k0 += AHEAD) {
			if (k0 + AHEAD < KS) fetch(k0 + AHEAD, A[(k0 / AHEAD + 1) & 1], B[(k0 / AHEAD + 1) & 1]);
#pragma unroll
			for (int k = 0; k < AHEAD; ++k)
				if (16 * (k0 + k) < dim) // (channels that are not there: nothing was copied)
#pragma unroll
					for (int i = 0; i < 2; ++i)
#pragma unroll
						for (int q = 0; q < NQ; ++q) mma_16<T>(z[i][q], A[(k0 / AHEAD) & 1][k][i], B[(k0 / AHEAD) & 1][k][q]);
		}
		__syncwarp(); // every lane has its keys
		request_keys();
		if constexpr (CAP) {
			cap_scores(reinterpret_cast<float(&)[8 * NQ]>(z), cap_of(a), qscale);
		} else {
#pragma unroll
			for (int i = 0; i < 2; ++i)
#pragma unroll
				for (int q = 0; q < NQ; ++q)
#pragma unroll
					for (int e = 0; e < 4; ++e) z[i][q][e] *= qscale;
		}
		const bool all = seen == 0xffffffffu && (seg == 0 || segs == 2) && pos >= wide && pos + AR_KEYS - 1 <= least;
		auto sees_key = [&](int j, int q, int e) { // this thread's keys are 8 j + g
			const int kp = pos + 8 * j + g;
			return (seen >> (8 * j + g) & 1) && kp <= rpos[q][e] && kp >= low_of(a, rpos[q][e]) && (seg == 0 || seg == rseg[q][e]);
		};
		if (!all) { // some row does not see some key
#pragma unroll
			for (int j = 0; j < 4; ++j)
#pragma unroll
				for (int q = 0; q < NQ; ++q)
#pragma unroll
					for (int e = 0; e < 2; ++e)
						if (!sees_key(j, q, e)) z[j >> 1][q][(j & 1) * 2 + e] = -INFINITY;
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
		bool odd = false; // where rows see different keys: a value that is not finite reaches the rows that see its key and no others
		if (!all) {
			uint32_t sum = 0;
#pragma unroll 4
			for (int i = 0; i < PIECES; ++i)
				if (piece * 8 < dim) {
					const int r = i * EACH + prow;
					const uint4 w = *reinterpret_cast<const uint4*>(s.v + (r * PIECES + (piece ^ (r & 7))) * 8);
					odd2<T>(w.x, sum), odd2<T>(w.y, sum), odd2<T>(w.z, sum), odd2<T>(w.w, sum);
				}
			odd = __any_sync(0xffffffffu, sum & 0x7fff7fff);
		}
		auto values = [&](int x, uint32_t (&to)[4]) { // step x: keys 16 (x / MT), channels 16 (x % MT)
			ldsm_x4_t(s.v + ((16 * (x / MT) + (lane >> 4) * 8 + lrow) * PIECES + ((2 * (x % MT) + (lane >> 3 & 1)) ^ lrow)) * 8, to);
		};
		if (!odd) {
			constexpr int DEPTH = 4;
			uint32_t V[2][DEPTH][4];
#pragma unroll
			for (int x = 0; x < DEPTH; ++x) values(x, V[0][x]);
#pragma unroll
			for (int x0 = 0; x0 < 2 * MT; x0 += DEPTH) {
				if (x0 + DEPTH < 2 * MT)
#pragma unroll
					for (int x = 0; x < DEPTH; ++x) values(x0 + DEPTH + x, V[(x0 / DEPTH + 1) & 1][x]);
#pragma unroll
				for (int x = 0; x < DEPTH; ++x)
					if (16 * ((x0 + x) % MT) < dim)
#pragma unroll
						for (int q = 0; q < NQ; ++q) mma_16<T>(acc[(x0 + x) % MT][q], V[(x0 / DEPTH) & 1][x], p[(x0 + x) / MT][q]);
			}
		} else {
#pragma unroll
			for (int i = 0; i < 2; ++i) {
				uint2 sees[NQ]; // 1 for each key that a row sees, even if its weight rounds to nothing
#pragma unroll
				for (int q = 0; q < NQ; ++q) {
					auto two = [&](int j) { return transposed(pack2<T>(sees_key(j, q, 0) ? 1.f : 0.f, sees_key(j, q, 1) ? 1.f : 0.f)); };
					sees[q] = make_uint2(two(2 * i), two(2 * i + 1));
				}
#pragma unroll
				for (int x = 0; x < MT; ++x) {
					if (16 * x >= dim) continue;
					uint32_t V[4], up[4], down[4];
					values(i * MT + x, V);
#pragma unroll
					for (int e = 0; e < 4; ++e) V[e] = split2<T>(V[e], up[e], down[e]);
#pragma unroll
					for (int q = 0; q < NQ; ++q) {
						float s_up[4] = {0.f, 0.f, 0.f, 0.f}, s_down[4] = {0.f, 0.f, 0.f, 0.f};
						mma_16<T>(s_up, up, sees[q]), mma_16<T>(s_down, down, sees[q]), mma_16<T>(acc[x][q], V, p[i][q]);
#pragma unroll
						for (int e = 0; e < 4; ++e) // (both: infinity less infinity)
							if (s_up[e] > 0.f || s_down[e] > 0.f) acc[x][q][e] += s_up[e] > 0.f ? s_down[e] > 0.f ? NAN : INFINITY : -INFINITY;
					}
				}
			}
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
	wait(); // the prefixes' shares

	// the warps' sums as one
	float* const sums = reinterpret_cast<float*>(ring); // [warps][TILE][LD]
	float* const own = sums + W * TILE * LD;     // [TILE][D + 2]: what this share of a cluster found
	const int prefix_places = whole && u.lead >= 0 ? a.before : 0;
	__syncthreads();
#pragma unroll
	for (int q = 0; q < NQ; ++q)
#pragma unroll
		for (int e = 0; e < 2; ++e) {
			float* const to = sums + (warp * TILE + 8 * q + 2 * t + e) * LD + g;
#pragma unroll
			for (int i = 0; i < MT; ++i) to[16 * i] = acc[i][q][e], to[16 * i + 8] = acc[i][q][2 + e];
		}
	__syncthreads();
	if (prefix_places) { // with the prefix's shares: a warp a row
#pragma unroll 1
		for (int r = warp; r < rows; r += W) {
			if (row_seq[r] < 0) continue;
			const int token = u.t0 + (row0 + r) / a.group, head = kvh * a.group + (row0 + r) % a.group;
			const size_t place = ((size_t)token * a.heads + head) * a.places;
			float pm = -INFINITY, pl = 0.f, mx = fold_m[0][r], den = 0.f, wt[W];
			if (lane < prefix_places) {
				const float2 st = a.stats[place + lane];
				pm = st.x, pl = st.y;
			}
#pragma unroll
			for (int w = 1; w < W; ++w) mx = fmaxf(mx, fold_m[w][r]);
			const float sk = a.sinks ? a.sinks[head] * A16_LOG2E : -INFINITY, top = fmaxf(fmaxf(mx, sk), warp_max(pm)), pw = pm == -INFINITY ? 0.f : ex2(pm - top);
#pragma unroll
			for (int w = 0; w < W; ++w) wt[w] = fold_m[w][r] == -INFINITY ? 0.f : ex2(fold_m[w][r] - top), den = fmaf(wt[w], fold_l[w][r], den);
			den += warp_sum(pw * pl);
			if (a.sinks) den += at_sink(sk, top); // one more term of the denominator
			const float norm = den > 0.f ? 1.f / den : den == 0.f ? 0.f : den; // (0: nothing was seen; a NaN stays one)
			for (int d0 = 0; d0 < dim; d0 += 128) {
				const int d = min(d0 + 4 * lane, dim - 4); // (every lane has a place's weight)
				float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
				for (int w = 0; w < W; ++w) add4(v, wt[w], *reinterpret_cast<const float4*>(sums + (w * TILE + r) * LD + d));
				add_places(v, a.sums + place * dim + d, dim, prefix_places, pw);
				if (d0 + 4 * lane < dim) put4<T>(a.out + token * a.o_row + head * a.o_head + d, a.out_vec, times4(v, norm));
			}
		}
		return;
	}
	if (tid < rows) { // the warps' weights, with all that multiplies them
		const int token = u.t0 + (row0 + tid) / a.group, head = kvh * a.group + (row0 + tid) % a.group;
		const float sk = whole && a.sinks ? a.sinks[head] * A16_LOG2E : -INFINITY;
		float mx = sk, den = 0.f, wt[W];
#pragma unroll
		for (int w = 0; w < W; ++w) mx = fmaxf(mx, fold_m[w][tid]);
#pragma unroll
		for (int w = 0; w < W; ++w) wt[w] = fold_m[w][tid] == -INFINITY ? 0.f : ex2(fold_m[w][tid] - mx), den = fmaf(wt[w], fold_l[w][tid], den);
		float by = 1.f;
		if (whole) {
			if (a.sinks) den += at_sink(sk, mx); // one more term of the denominator
			by = den > 0.f ? 1.f / den : den == 0.f ? 0.f : den; // (0: nothing was seen; a NaN stays one)
		} else if (a.cluster) own[tid * (D + 2) + D] = mx, own[tid * (D + 2) + D + 1] = den;
		else if (row_seq[tid] >= 0) a.stats[((size_t)token * a.heads + head) * a.places + a.before + share] = make_float2(mx, den);
#pragma unroll
		for (int w = 0; w < W; ++w) fold_m[w][tid] = wt[w] * by;
		row_place[tid] = row_seq[tid] < 0 ? -1 : whole ? token * a.o_row + head * a.o_head : (long long)((((size_t)token * a.heads + head) * a.places + a.before + share) * dim);
	}
	__syncthreads();
	const int quads = dim / 4;
	for (int e = tid; e < rows * quads; e += 32 * W) {
		const int r = e / quads, d = 4 * (e - r * quads);
		float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
		for (int w = 0; w < W; ++w) add4(v, fold_m[w][r], *reinterpret_cast<const float4*>(sums + (w * TILE + r) * LD + d));
		if (!whole && a.cluster) {
			float* const to = own + r * (D + 2) + d; // (8-byte aligned)
			*reinterpret_cast<float2*>(to) = make_float2(v.x, v.y), *reinterpret_cast<float2*>(to + 2) = make_float2(v.z, v.w);
		} else if (row_place[r] >= 0) {
			if (whole) put4<T>(a.out + row_place[r] + d, a.out_vec, v);
			else *reinterpret_cast<float4*>(a.sums + row_place[r] + d) = v;
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
	for (int e = from + tid; e < to; e += 32 * W) {
		const int r = e / dim, d = e - r * dim;
		float v = 0.f;
#pragma unroll 8
		for (int k = 0; k < shares; ++k) v = fmaf(cluster_load_f32(cluster_addr(own + r * (D + 2) + d, k)), wz[k][r], v);
		if (row_seq[r] >= 0) a.out[(u.t0 + (row0 + r) / a.group) * a.o_row + (kvh * a.group + (row0 + r) % a.group) * a.o_head + d] = round16<T>(v * inv[r]);
	}
	cluster_sync(); // no CTA leaves while another reads what it found
}

// ---------------------------------------------------------------- many rows
// Where many rows see the same keys, the products run on the fifth-generation tensor cores: a CTA takes up to 256 rows that read one key head - of a group of sequences over its prefix, or of one sequence over its group's prefix
// and its own keys - and walks tiles of 128 keys.  Two warps, one for keys and one for values, copy tiles with TMA, boxes of 64 channels and as many keys as lie side by side in a page (8 to 64), straight into the layout that the
// products read: keys as rows, values as they lie with the channels as the product's columns.  One thread issues S = Q K^T of the next tile behind O += P V of this one; four warps for each 128 rows, a row a thread, take S from
// tensor memory, form the weights and write them back where the scores stood, the next product's operand.  While one group's weights are formed the other's products run; up to 128 rows are taken by both groups, every other tile
// each, and their sums are added at the end.  O stays in tensor memory; it is rescaled in the rare case that a row's reference moves.  Tiles that some row sees in part go through a slower way of 32 columns at a time in few
// instructions.  Results leave through shared memory, a row a copy.
// Where some row does not see some key of a tile its weight is 0, and 0 times a value that is not finite would be no number: the warp that copies values looks at such tiles and takes those values out, and the rows that see their
// keys add them to their results at the end (add_odd; reached by values that are not finite alone).  Looking takes 0.4 us a tile, which nothing waits for unless most of a block's tiles are of that kind (27 rows over windows' edges, four
// tiles a block, 21.4 -> 24.1 us).  Both functions stay out of line, and the copies' loop rolled: inline 91 us for 82 where up to 128 rows are taken by both groups, unrolled 715 for 710 in the case below.
// Bound: a tile's way through its roles.  256 rows and 128 keys of 128 channels take about 3700 cycles: the products 2048 by the tensor cores' rate (about 2560 as they are, 80 cycles for 64), softmax 1680 to 1800 for a group and
// 110 of hand-over.  16 sequences of up to 300 tokens behind 12000 positions, 32 heads over 8: 711 us where the products alone would be 378 (0.45 of the tensor pipes, 0.47 of the special functions'); its loads alone took 570 us
// from pages of 16 keys, 459 of 32, 416 of 64, 795 of 8.  Tried: tiles of 64 keys with scores ahead 1330 us (N = 64 costs what N = 128 does), weights handed over in halves 905 to 1134, a polynomial for part of the exponentials
// 1085 against 973, a product thread a group 977 to 1017, copying warps with code of their own 820.
constexpr int AW_KEYS = 128, AW_THREADS = 384, AW_MASKS = 8;
constexpr int AW_SOFTMAX_REGS = 176, AW_OTHER_REGS = 144; // 256 x 176 + 128 x 144 = 63488 of the 384 x 168 = 64512 that the block is launched with

struct AwOdd { // where values that are not finite were taken out: the block's tiles of keys, for the rows that see such values
	int found;
	C16 c;
	int kvh, box, lo[2], hi[2], base[2], slot[2], first, begin, tiles; // first: tiles of the prefix
	int wide, least; // every row sees the keys wide .. least
};
template <int D>
struct AwShared { // tiles of rows of 128 bytes, 16-byte pieces swizzled by the row
	static constexpr int PANELS = D / 64, SLOTS = D == 128 ? 5 : 9;
	unsigned char q[2][PANELS][128 * 128];
	unsigned char kv[SLOTS][PANELS][AW_KEYS * 128]; // keys and values in turn
	uint64_t full[SLOTS], empty[SLOTS], mask_full[AW_MASKS], s_full[2], p_full[2], done[2], fix, idle;
	alignas(16) uint32_t seen[AW_MASKS][4]; // keys that are there
	int row_pos[256];
	int span[2]; // the rows' least and largest position
	int found[3], sums[AW_THREADS / 32]; // the task
	uint32_t tmem;
	int lost;
	AwOdd odd;
};
// shared -> global, 16-byte aligned, a multiple of 16 bytes
__device__ __forceinline__ void bulk_store(void* dst, const void* src, uint32_t bytes) {
	asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(src)), "r"(bytes) : "memory");
}
static_assert(sizeof(AwShared<128>) <= 227 * 1024 && sizeof(AwShared<64>) <= 227 * 1024, "shared memory of a CTA");
// a row of scores
__device__ __forceinline__ void tmem_ld128(uint32_t taddr, float (&v)[128]) {
#define AW_R8(b) "=f"(v[b]), "=f"(v[b + 1]), "=f"(v[b + 2]), "=f"(v[b + 3]), "=f"(v[b + 4]), "=f"(v[b + 5]), "=f"(v[b + 6]), "=f"(v[b + 7])
#define AW_R32(b) AW_R8(b), AW_R8(b + 8), AW_R8(b + 16), AW_R8(b + 24)
	asm volatile(
	    "tcgen05.ld.sync.aligned.32x32b.x128.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
	    "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63,"
	    "%64,%65,%66,%67,%68,%69,%70,%71,%72,%73,%74,%75,%76,%77,%78,%79,%80,%81,%82,%83,%84,%85,%86,%87,%88,%89,%90,%91,%92,%93,%94,%95,"
	    "%96,%97,%98,%99,%100,%101,%102,%103,%104,%105,%106,%107,%108,%109,%110,%111,%112,%113,%114,%115,%116,%117,%118,%119,%120,%121,%122,%123,%124,%125,%126,%127}, [%128];\n\t"
	    "tcgen05.wait::ld.sync.aligned;"
	    : AW_R32(0), AW_R32(32), AW_R32(64), AW_R32(96)
	    : "r"(taddr)
	    : "memory");
#undef AW_R8
#undef AW_R32
}
__device__ __forceinline__ float max_nan(float x, float y) { // NaN where one of them is
	float r;
	asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
	return r;
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
	asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
	             : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
	             : "r"(taddr)
	             : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) { // (tcgen05.wait::st is the caller's)
	asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]),
	             "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
	             : "memory");
}
// shared-memory descriptor of values [keys][64 channels], 128-byte swizzle, panels of 64 channels one behind another: the product's columns are the channels, its depth the keys, eight keys 1024 bytes apart
__device__ __forceinline__ uint64_t umma_desc_values(const void* tile) {
	const uint64_t addr = (uint64_t)(smem_u32(tile) & 0x3FFFF) >> 4;
	return addr | ((uint64_t)(AW_KEYS * 128 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// The work of k_c16_tiles: a CTA takes a share of the keys of 256 rows that read one key head.
//   groups (through 0): row tiles and key heads of every group, `shares` of its prefix's keys, `each` tiles of 128 of them; results in the shares' places
//   sequences (through 1): tasks - row tiles and key heads of all sequences, one after another - of which the first `cut` are whole, those from there to `planned` are split into `shares`, so that the last round of
//   CTAs is as long as it has to be, and those behind (where sequences have grown since the plan was made) are whole again.  Whole ones go to out, split ones to places that k_c16_join folds.
struct Wide {
	int through;
	int box;          // keys that a copy brings
	int shares, each;
	int tiles;        // of 256 rows, of the longest unit
	int cut, planned;
};
struct Task {
	int z, kvh, tile;
};
// task t: sequences in order, their key heads, their row tiles from the last (which sees most keys) on.  All of a block's N threads; false: there is none
template <int N>
__device__ __forceinline__ bool task_of(const C16& c, const Attend& a, int t, int (&found)[3], int (&sums)[N / 32], Task& r) { // (both: of shared memory)
	const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
	int before = 0;
	if (tid == 0) found[0] = -1;
	for (int b0 = 0; b0 < c.n; b0 += N) {
		const int b = b0 + tid;
		const int tiles = b < c.n && there(c, a.rows, b) && c.count[b] > -a.families ? (int)(((long long)c.count[b] * a.group + 255) / 256) : 0;
		int sum = tiles;
#pragma unroll
		for (int o = 1; o < 32; o *= 2) {
			const int x = __shfl_up_sync(0xffffffffu, sum, o);
			if (lane >= o) sum += x;
		}
		__syncthreads();
		if (lane == 31) sums[warp] = sum;
		__syncthreads();
		int all = 0;
		for (int w = 0; w < N / 32; ++w) {
			if (w < warp) sum += sums[w];
			all += sums[w];
		}
		const long long from = (long long)(before + sum - tiles) * c.heads, to = (long long)(before + sum) * c.heads;
		if (t >= from && t < to) found[0] = b, found[1] = (int)((t - from) / tiles), found[2] = tiles - 1 - (int)((t - from) % tiles);
		before += all;
		if ((long long)before * c.heads > t) break;
	}
	__syncthreads();
	r.z = found[0], r.kvh = found[1], r.tile = found[2];
	return r.z >= 0;
}

// A tile of values: zeros for those of keys that are not there (`word`: keys 32 lane .. that are, for the first four lanes) and for what is not finite.  True: there was some of that.  A warp.
template <typename T, int PANELS>
__device__ __noinline__ bool clear_values(unsigned char* tile, bool there, uint32_t word) {
	const int lane = threadIdx.x & 31;
	if (!there) {
		for (int k = 0; k < AW_KEYS; ++k)
			if (!(__shfl_sync(0xffffffffu, word, k >> 5) >> (k & 31) & 1) && lane < 8 * PANELS) *reinterpret_cast<uint4*>(tile + (lane >> 3) * AW_KEYS * 128 + k * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
		__syncwarp();
	}
	uint4* const all = reinterpret_cast<uint4*>(tile) + lane;
	uint32_t sums[4] = {0, 0, 0, 0};
#pragma unroll 8
	for (int e = 0; e < AW_KEYS * 8 * PANELS; e += 32) {
		const uint4 x = all[e];
		odd2<T>(x.x, sums[0]), odd2<T>(x.y, sums[1]), odd2<T>(x.z, sums[2]), odd2<T>(x.w, sums[3]);
	}
	const bool found = __any_sync(0xffffffffu, (sums[0] | sums[1] | sums[2] | sums[3]) & 0x7fff7fff);
	if (found)
		for (int e = 0; e < AW_KEYS * 8 * PANELS; e += 32) {
			uint32_t up, down;
			const uint4 x = all[e];
			all[e] = make_uint4(split2<T>(x.x, up, down), split2<T>(x.y, up, down), split2<T>(x.z, up, down), split2<T>(x.w, up, down));
		}
	return found;
}
// What the keys from .. to hold that is not finite, in the tiles whose values were looked at, added to a row of results (32-bit sums or the cache's type).
template <typename T>
__device__ __noinline__ void add_odd(const AwOdd& o, int from, int to, int dim, void* row, bool sums) {
	auto page_of = [&](int part, int pos) {
		const int at = o.c.page_index(pos);
		return pos >= o.lo[part] && pos < o.hi[part] && at < o.c.table_pages ? __ldg(o.c.table + (size_t)o.slot[part] * o.c.table_pages + at) : -1;
	};
	for (int i = 0; i < o.tiles; ++i) {
		const int at = o.begin + i, part = at >= o.first, pos0 = o.base[part] + (at - (part ? o.first : 0)) * AW_KEYS;
		bool looked = pos0 < o.wide || pos0 + AW_KEYS - 1 > o.least || pos0 < o.lo[part] || pos0 + AW_KEYS > o.hi[part];
		for (int k = 0; k < AW_KEYS && !looked; k += o.box) looked = (unsigned)page_of(part, pos0 + k) >= (unsigned)o.c.pages;
		if (!looked) continue;
		for (int pos = max(pos0, from); pos <= min(pos0 + AW_KEYS - 1, to); ++pos) {
			const int id = page_of(part, pos);
			if ((unsigned)id >= (unsigned)o.c.pages) continue;
			const T* const v = reinterpret_cast<const T*>(o.c.v) + (((long long)id * o.c.heads + o.kvh) * o.c.page + o.c.page_row(pos)) * dim;
			for (int d = 0; d < dim; d += 8) {
				const uint4 w = *reinterpret_cast<const uint4*>(v + d);
				uint32_t odd = 0;
				odd2<T>(w.x, odd), odd2<T>(w.y, odd), odd2<T>(w.z, odd), odd2<T>(w.w, odd);
				if (!(odd & 0x7fff7fff)) continue;
				for (int k = d; k < d + 8; ++k) {
					const float x = as_f32(v[k]);
					if (fabsf(x) < INFINITY) continue;
					if (sums) static_cast<float*>(row)[k] += x;
					else static_cast<T*>(row)[k] = from_f32<T>(as_f32(static_cast<T*>(row)[k]) + x);
				}
			}
		}
	}
}

// CAP: soft caps, which all tiles take the slower way for.  (One kernel for both: 731 us for 713 without a cap, 16 sequences of up to 300 tokens behind 12000.)
template <typename T, int D, bool CAP>
__global__ void __launch_bounds__(AW_THREADS, 1) k_c16_tiles(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const C16 c, const Attend a, const Wide w) {
	typedef AwShared<D> Shared;
	constexpr int PANELS = Shared::PANELS, SLOTS = Shared::SLOTS, PIECES = D / 8;
	constexpr uint32_t O_COL = 256;
	extern __shared__ __align__(1024) unsigned char aw_raw[]; // (all of the kernel's shared memory: it starts where the swizzle's pattern does)
	Shared& s = *reinterpret_cast<Shared*>(aw_raw);
	const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
	pdl_launch_next();
	Unit u;
	Task task;
	int share = 0, shares = 1, place0 = -1; // the places of a split task's rows
	if (w.through) {
		const int split = (w.planned - w.cut) * w.shares, x = (int)blockIdx.x - w.cut;
		if (x >= 0 && x < split) share = x % w.shares, shares = w.shares, place0 = x * 256;
		if (!task_of<AW_THREADS>(c, a, x < 0 ? (int)blockIdx.x : x < split ? w.cut + x / w.shares : w.planned + x - split, s.found, s.sums, task) || !own_unit(c, a, task.z, u)) return;
	} else {
		const int per = w.tiles * c.heads;
		share = blockIdx.x / per, shares = w.shares, task.kvh = blockIdx.x % per / w.tiles, task.tile = blockIdx.x % w.tiles;
		if (!group_unit(c, a, blockIdx.z, u)) return;
	}
	const int kvh = task.kvh, tile = task.tile;
	const bool partial = !w.through || shares > 1;
	if ((long long)tile * 256 >= (long long)u.tokens * a.group) return;
	const int row0 = tile * 256, rows = (int)min(256LL, (long long)u.tokens * a.group - row0), groups = rows > 128 ? 2 : 1;
	const bool two = groups == 1; // the same rows twice: each of two groups of warps takes every other tile, and their sums are added at the end

	if (warp == 9) tmem_alloc(&s.tmem, 512);
	if (tid == 0) {
		for (int i = 0; i < SLOTS; ++i) mbar_init(s.full + i, 1), mbar_init(s.empty + i, 1);
		for (int i = 0; i < AW_MASKS; ++i) mbar_init(s.mask_full + i, 1);
		for (int g = 0; g < 2; ++g) mbar_init(s.s_full + g, 1), mbar_init(s.p_full + g, 4), mbar_init(s.done + g, 1);
		mbar_init(&s.fix, 1), mbar_init(&s.idle, 1);
		s.lost = 0, s.odd.found = 0, s.span[0] = INT_MAX, s.span[1] = -1;
		mbar_init_fence();
	}
	if (tid < 256) s.row_pos[tid] = -1;
	const bool alone = u.first == u.last;
	if (alone && !there(c, a.rows, u.first)) u.tokens = 0; // (a group of one that makes no sense: no keys, no rows)
	const int lead_slot = u.lead >= 0 ? c.slot[u.lead] : -1, own_slot = c.slot[u.first], pos0 = c.pos0[u.first];
	// The keys: positions lo .. hi - 1 of the prefix, then of the sequence's own, in tiles that begin where a copy may.  The copies need not wait for the rows' positions where these do not matter for the range.
	const bool ranged = alone || a.window == 0;
	int lo[2], hi[2], base[2], count[2], begin, tiles;
	auto range = [&](int least, int most) {
		lo[0] = low_of(a, least), hi[0] = min(u.prefix, c.reach(lead_slot)), lo[1] = hi[1] = 0;
		if (alone || !ranged) hi[0] = min(hi[0], most + 1);
		if (w.through) lo[1] = max(u.prefix, low_of(a, least)), hi[1] = min(most + 1, c.reach(own_slot));
#pragma unroll
		for (int k = 0; k < 2; ++k) base[k] = lo[k] & ~(w.box - 1), count[k] = u.tokens > 0 && hi[k] > lo[k] ? (hi[k] - base[k] + AW_KEYS - 1) / AW_KEYS : 0;
		const int total = count[0] + count[1];
		const int each = w.through ? (total + shares - 1) / shares : w.each;
		begin = (int)min((long long)total, (long long)share * each), tiles = (share == shares - 1 ? total : min(total, begin + each)) - begin;
	};
	const int low = pos0 + row0 / a.group, high = pos0 + (row0 + rows - 1) / a.group; // of one sequence's rows
	__syncthreads();
	// (the values' copies look at what some row does not see)
	const int waiting = alone ? 0 : ranged ? AW_THREADS - 32 : AW_THREADS;
	if (warp == 8 || warp == 11) {
		if (!ranged) asm volatile("bar.sync 2, %0;" ::"r"(waiting) : "memory");
		range(ranged ? low : s.span[0], ranged ? high : s.span[1]);
	} else {
		for (int b = u.first + (warp < 8 ? tid : tid - 32); b <= u.last; b += AW_THREADS - 64) {
			const int p0 = c.pos0[b], start = c.start[b], n = c.count[b];
			if (!there(c, a.rows, b)) continue;
			const long long r0 = (long long)(start - u.t0) * a.group - row0, r1 = r0 + (long long)n * a.group;
			for (long long r = max(r0, 0LL); r < min(r1, (long long)rows); ++r) s.row_pos[r] = p0 + (int)((unsigned)(r - r0) / (unsigned)a.group);
		}
		// queries, rows of 128 bytes a panel
		const bool vec = ((uintptr_t)a.q | (uintptr_t)(a.q_row * 2) | (uintptr_t)(a.q_head * 2)) % 16 == 0;
		if (warp < 8) {
			constexpr int DEPTH = 8;
#pragma unroll 1
			for (int i0 = tid; i0 < groups * 128 * PIECES; i0 += 256 * DEPTH) {
				uint4 x[DEPTH];
#pragma unroll
				for (int k = 0; k < DEPTH; ++k) {
					const int i = i0 + 256 * k, r = i / PIECES, piece = i % PIECES, rr = row0 + min(r, rows - 1);
					x[k] = make_uint4(0, 0, 0, 0);
					if (r < rows && piece * 8 < c.dim) {
						const uint16_t* const q = a.q + (long long)(u.t0 + rr / a.group) * a.q_row + (long long)(kvh * a.group + rr % a.group) * a.q_head + piece * 8;
						if (vec) x[k] = *reinterpret_cast<const uint4*>(q);
						else x[k] = make_uint4(q[0] | (uint32_t)q[1] << 16, q[2] | (uint32_t)q[3] << 16, q[4] | (uint32_t)q[5] << 16, q[6] | (uint32_t)q[7] << 16);
					}
				}
#pragma unroll
				for (int k = 0; k < DEPTH; ++k) {
					const int i = i0 + 256 * k, r = i / PIECES, piece = i % PIECES;
					if (i < groups * 128 * PIECES) *reinterpret_cast<uint4*>(s.q[r >> 7][piece >> 3] + (r & 127) * 128 + (((piece & 7) ^ (r & 7)) << 4)) = x[k];
				}
			}
			fence_async_smem();
		}
		asm volatile("bar.sync 1, %0;" ::"n"(AW_THREADS - 64) : "memory"); // everybody but the copying warps
		if (warp < 8) {
			const int pos = s.row_pos[tid];
			const int least = __reduce_min_sync(0xffffffffu, pos < 0 ? INT_MAX : pos), most = __reduce_max_sync(0xffffffffu, pos);
			if (lane == 0) atomicMin(&s.span[0], least), atomicMax(&s.span[1], most);
		}
		tc_fence_before();
		asm volatile("bar.sync 1, %0;" ::"n"(AW_THREADS - 64) : "memory");
		tc_fence_after();
		if (waiting) asm volatile("bar.sync 2, %0;" ::"r"(waiting) : "memory");
		range(ranged ? low : s.span[0], ranged ? high : s.span[1]);
	}
	const uint32_t tmem = s.tmem;
	const int least = s.span[0], most = s.span[1];

	if (warp < 8) {
		asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(AW_SOFTMAX_REGS));
		const int group = warp >> 2;
		const int r = two ? tid & 127 : tid, rpos = s.row_pos[r], rlow = low_of(a, rpos), wide = low_of(a, most);
		const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16), scores_at = lanes + 128 * group, sums_at = lanes + O_COL + 128 * group;
		const float qscale = a.scale * A16_LOG2E;
		float m = -INFINITY, l = 0.f;
		if (group < groups || two) {
			int n = 0; // tiles of this group's
			for (int i = two ? group : 0; i < tiles; i += two ? 2 : 1, ++n) {
				const int at = begin + i, part = at >= count[0], pos0 = part ? base[1] + (at - count[0]) * AW_KEYS : base[0] + at * AW_KEYS;
				if (!ap_wait_warp(s.mask_full + i % AW_MASKS, i / AW_MASKS & 1, &s.lost) || !ap_wait_warp(s.s_full + group, n & 1, &s.lost)) break;
				tc_fence_after();
				const uint4 seen = *reinterpret_cast<const uint4*>(s.seen[i % AW_MASKS]);
				const bool all = (seen.x & seen.y & seen.z & seen.w) == 0xffffffffu && pos0 >= wide && pos0 + AW_KEYS - 1 <= least;
				const bool steady = !CAP && __all_sync(0xffffffffu, all && (m != -INFINITY || rpos < 0)) && a.scale > 0.f; // (a row that is not there has scores of zero)
				const float ref = m == -INFINITY ? 0.f : m;
				uint32_t p[64];
				u64 sum = 0;
				bool moves = true;
				if (steady) { // the reference as it stands, unless a score passes it or is no number
					float z[128], tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
					tmem_ld128(scores_at, z);
#pragma unroll
					for (int k = 0; k < 128; k += 2) tops[k / 2 % 4] = max_nan(max_nan(tops[k / 2 % 4], z[k]), z[k + 1]);
					const float top = max_nan(max_nan(tops[0], tops[1]), max_nan(tops[2], tops[3]));
					moves = __any_sync(0xffffffffu, !(fmaf(top, qscale, -ref) <= A16_MOST));
					if (!moves) {
						const u64 by = pair_of(qscale, qscale), off = pair_of(-ref, -ref);
#pragma unroll
						for (int k = 0; k < 128; k += 2) {
							const float2 y = halves(fma2(pair_of(z[k], z[k + 1]), by, off));
							const float w0 = ex2(y.x), w1 = ex2(y.y);
							sum = add2(sum, pair_of(w0, w1));
							p[k / 2] = pack2<T>(w0, w1);
						}
					}
				}
				if (moves) { // 32 columns at a time, in few instructions: most often a block's first and last tiles
					const float most_z = m == -INFINITY ? -INFINITY : A16_MOST;
					const int from = min(max(rlow - pos0, 0), 128), to = min(max(rpos + 1 - pos0, 0), 128); // of this row: keys from .. to - 1
					float top = -INFINITY;
#pragma unroll 1
					for (int x = 0; x < 4; ++x) { // log2 of the weights against the reference (against 0 before there is one), back to where the scores were
						float y[32];
						tmem_ld32(scores_at + 32 * x, y);
						const int f = min(max(from - 32 * x, 0), 32), t = min(max(to - 32 * x, 0), 32);
						const uint32_t see = s.seen[i % AW_MASKS][x] & (t >= 32 ? 0xffffffffu : (1u << t) - 1) & ~(f >= 32 ? 0xffffffffu : (1u << f) - 1);
						if constexpr (CAP) cap_scores(y, cap_of(a), qscale);
#pragma unroll
						for (int k = 0; k < 32; ++k) y[k] = CAP ? y[k] - ref : fmaf(y[k], qscale, -ref);
#pragma unroll
						for (int k = 0; k < 32; ++k) {
							if (!(see >> k & 1)) y[k] = -INFINITY;
							top = fmaxf(top, y[k]);
						}
						tmem_st32(scores_at + 32 * x, reinterpret_cast<const uint32_t(&)[32]>(y));
					}
					float down = 0.f;
					if (__any_sync(0xffffffffu, top > most_z)) { // references move
						const float mn = top > most_z ? ref + top - A16_SET : m, f = m == -INFINITY ? 0.f : ex2(m - mn);
						down = ref - (mn == -INFINITY ? 0.f : mn);
						m = mn, l *= f;
						if (n > 0) { // there are sums; the product that wrote them was issued before these scores'
#pragma unroll 1
							for (int col = 0; col < D; col += 8) tmem_scale8(sums_at + col, f);
						}
					}
					tmem_st_wait();
#pragma unroll 1
					for (int x = 0; x < 4; ++x) {
						float y[32];
						uint32_t w[16];
						tmem_ld32(scores_at + 32 * x, y);
#pragma unroll
						for (int k = 0; k < 32; k += 2) {
							const float w0 = ex2(y[k] + down), w1 = ex2(y[k + 1] + down);
							sum = add2(sum, pair_of(w0, w1));
							w[k / 2] = pack2<T>(w0, w1);
						}
						tmem_st16(scores_at + 16 * x, w); // (where scores were that have been read)
					}
				} else {
					tmem_st32(scores_at, *reinterpret_cast<uint32_t(*)[32]>(p)); // where the scores were
					tmem_st32(scores_at + 32, *reinterpret_cast<uint32_t(*)[32]>(p + 32));
				}
				const float2 both = halves(sum);
				l += both.x + both.y;
				tmem_st_wait();
				tc_fence_before();
				__syncwarp();
				if (lane == 0) mbar_arrive(s.p_full + group);
			}
			if (n > 0) ap_wait_warp(s.done + group, 0, &s.lost);
			tc_fence_after();
			const bool lost = *(volatile int*)&s.lost;
			const int token = u.t0 + (row0 + min(r, rows - 1)) / a.group, head = kvh * a.group + (row0 + min(r, rows - 1)) % a.group;
			const bool writes = r < rows && rpos >= 0 && !(two && group);
			const size_t place = w.through ? (size_t)max(place0, 0) + r : ((size_t)token * a.heads + head) * a.places + share;
			float* const row = reinterpret_cast<float*>(s.kv) + tid * (D + 4);
			asm volatile("bar.sync 4, 288;" ::: "memory"); // (both groups' products have ended, and what the values' copies found is there)
			float f0 = 1.f, f1 = 0.f; // of this group's sums and the other's
			const float* const other = reinterpret_cast<const float*>(s.kv) + (tid ^ 128) * (D + 4);
			if (two) {
				if (group) {
#pragma unroll 1
					for (int col = 0; col < D && n > 0; col += 16) {
						float v[16];
						tmem_ld16(sums_at + col, v);
#pragma unroll
						for (int k = 0; k < 16; k += 4) *reinterpret_cast<float4*>(row + col + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
					}
					row[D] = m, row[D + 1] = l;
				}
				asm volatile("bar.sync 3, 256;" ::: "memory");
				if (!group && tiles > 1) {
					const float m1 = other[D], top = fmaxf(m, m1);
					f0 = m == -INFINITY ? 0.f : ex2(m - top), f1 = m1 == -INFINITY ? 0.f : ex2(m1 - top);
					l = fmaf(l, f0, other[D + 1] * f1), m = top;
				}
			}
			float norm = 1.f;
			if (!partial) {
				const float sk = a.sinks ? a.sinks[head] * A16_LOG2E : -INFINITY, mn = fmaxf(m, sk), down = m == -INFINITY ? 0.f : ex2(m - mn);
				l *= down;
				if (a.sinks) l += at_sink(sk, mn);
				norm = l > 0.f ? down / l : l == 0.f ? 0.f : l; // (0: nothing was seen; a NaN stays one)
			} else if (writes) a.stats[place] = make_float2(lost ? 0.f : m, lost ? NAN : l);
			if (lost) norm = NAN;
			// A thread's row goes to shared memory (where keys and values were: the last product has ended, of the other group's too once both have) and from there as one copy.
			const bool vec = ((uintptr_t)a.out | (uintptr_t)(a.o_row * 2) | (uintptr_t)(a.o_head * 2)) % 16 == 0;
			const bool nothing = partial && m == -INFINITY && !lost; // (the fold leaves out what weighs nothing)
#pragma unroll 1
			for (int col = 0; col < c.dim && !(two && group); col += 16) {
				float v[16];
				__syncwarp(); // (rows behind the last one take part in the load)
				if (n > 0) tmem_ld16(sums_at + col, v);
				else {
#pragma unroll
					for (int k = 0; k < 16; ++k) v[k] = 0.f;
				}
				if (two && tiles > 1) {
#pragma unroll
					for (int k = 0; k < 16; ++k) v[k] = fmaf(v[k], f0, other[col + k] * f1);
				}
				if (partial) {
#pragma unroll
					for (int k = 0; k < 16; k += 4) *reinterpret_cast<float4*>(row + col + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
				} else {
					uint32_t x[8];
#pragma unroll
					for (int k = 0; k < 8; ++k) x[k] = pack2<T>(v[2 * k] * norm, v[2 * k + 1] * norm);
					if (vec) {
						uint4* const to = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(row) + col);
						to[0] = make_uint4(x[0], x[1], x[2], x[3]), to[1] = make_uint4(x[4], x[5], x[6], x[7]);
					} else if (writes) {
						uint16_t* const to = a.out + token * a.o_row + head * a.o_head + col;
#pragma unroll
						for (int k = 0; k < 8; ++k) to[2 * k] = (uint16_t)x[k], to[2 * k + 1] = (uint16_t)(x[k] >> 16);
					}
				}
			}
			if (s.odd.found && writes && !nothing)
				add_odd<T>(s.odd, low_of(a, rpos), rpos, c.dim, partial || vec ? static_cast<void*>(row) : a.out + token * a.o_row + head * a.o_head, partial);
			fence_async_smem();
			if (writes && !nothing && (partial || vec)) {
				if (partial) bulk_store(a.sums + place * c.dim, row, c.dim * 4);
				else bulk_store(a.out + token * a.o_row + head * a.o_head, row, c.dim * 2);
			}
			asm volatile("cp.async.bulk.commit_group;\n\tcp.async.bulk.wait_group 0;" ::: "memory"); // (written: what follows in the stream may read it)
		}
	} else {
		asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(AW_OTHER_REGS));
		if (warp == 8 || warp == 11) {
			// Copies: one warp the keys', one the values'.  Lane l looks up the page of box l of every tile, a tile ahead: nothing waits for the table where it is asked.
			const bool values = warp == 11;
			const CUtensorMap* const map = values ? &tm_v : &tm_k;
			const int boxes = AW_KEYS / w.box, none = c.pages * c.heads * c.page; // (a row past the pool reads as zeros)
			int next = -1;
			auto start = [&](int i, int& part) { // first position of tile i
				const int at = begin + i;
				part = at >= count[0];
				return part ? base[1] + (at - count[0]) * AW_KEYS : base[0] + at * AW_KEYS;
			};
			auto look = [&](int i) { // the page of this lane's box
				int part;
				const int pos = start(i, part) + lane * w.box, at = c.page_index(pos);
				const bool some = lane < boxes && i < tiles && pos < (part ? hi[1] : hi[0]) && at < c.table_pages;
				next = some ? __ldg(c.table + (size_t)(part ? own_slot : lead_slot) * c.table_pages + at) : -1;
			};
			uint32_t fixes = 0;
			int issued = 0; // tiles asked for
			if (tiles > 0) look(0);
			if (values && ranged && waiting) asm volatile("bar.sync 2, %0;" ::"r"(waiting) : "memory");
			const int seen_by_all = alone ? low : s.span[0], wide = low_of(a, alone ? high : s.span[1]); // (of the values' warp)
			if (values && lane == 0) { // for the rows that see values which are taken out
				AwOdd& o = s.odd;
				o.c = c, o.kvh = kvh, o.box = w.box, o.slot[0] = lead_slot, o.slot[1] = own_slot, o.first = count[0], o.begin = begin, o.tiles = tiles, o.wide = wide, o.least = seen_by_all;
				o.lo[0] = lo[0], o.lo[1] = lo[1], o.hi[0] = hi[0], o.hi[1] = hi[1], o.base[0] = base[0], o.base[1] = base[1];
			}
			for (int i = 0; i < tiles; ++i) {
				int part;
				const int pos0 = start(i, part), l0 = (part ? lo[1] : lo[0]) - pos0, h0 = (part ? hi[1] : hi[0]) - pos0;
				const bool some = (unsigned)next < (unsigned)c.pages;
				const int row = some ? (next * c.heads + kvh) * c.page + c.page_row(pos0 + lane * w.box) : none;
				const uint32_t have = __ballot_sync(0xffffffffu, some);
				look(i + 1);
				uint32_t word = 0; // keys 32 lane .. of the tile that are there, for the first four lanes
				if (lane < 4) {
#pragma unroll 4
					for (int k = 0; k < 32; k += 8)
						if (have >> ((32 * lane + k) / w.box) & 1) word |= 0xffu << k;
					const int f = min(max(l0 - 32 * lane, 0), 32), t = min(max(h0 - 32 * lane, 0), 32);
					word &= (t >= 32 ? 0xffffffffu : (1u << t) - 1) & ~(f >= 32 ? 0xffffffffu : (1u << f) - 1);
					if (!values) s.seen[i % AW_MASKS][lane] = word;
				}
				// Values go through this warp where a key is not there or some row does not see some key: 0 times what is not finite would be no number.
				const bool there = __all_sync(0xffffffffu, lane >= 4 || word == 0xffffffffu), whole = !values || (there && pos0 >= wide && pos0 + AW_KEYS - 1 <= seen_by_all);
				__syncwarp();
				if (!values && lane == 0) mbar_arrive(s.mask_full + i % AW_MASKS);
				const int k = 2 * i + values, sl = k % SLOTS;
				if (!ap_wait_warp(s.empty + sl, (k / SLOTS & 1) ^ 1, &s.lost)) break;
				uint64_t* const bar = whole ? s.full + sl : &s.fix;
				if (lane == 0) mbar_expect_tx(bar, PANELS * AW_KEYS * 128);
				unsigned char* to = s.kv[sl][0];
#pragma unroll 1
				for (int x = 0; x < boxes; ++x, to += w.box * 128) {
					const int r = __shfl_sync(0xffffffffu, row, x);
					if (lane == 0) {
#pragma unroll
						for (int pn = 0; pn < PANELS; ++pn) tma_load_2d(to + pn * AW_KEYS * 128, map, pn * 64, r, bar);
					}
				}
				++issued;
				if (!whole) { // values of keys that are not there are zeros, whatever lies there, and so are values that are not finite: rows that see them get them at the end
					if (!ap_wait_warp(&s.fix, fixes & 1, &s.lost)) break;
					++fixes;
					if (clear_values<T, PANELS>(s.kv[sl][0], there, word)) {
						if (lane == 0) s.odd.found = 1;
					}
					fence_async_smem();
					__syncwarp();
					if (lane == 0) mbar_arrive(s.full + sl);
				}
			}
			if (*(volatile int*)&s.lost) // given up: no copy is left in flight when the block's memory goes
				for (int i = max(0, issued - SLOTS); i < issued; ++i) {
					const int k = 2 * i + values;
					mbar_wait_warp(s.full + k % SLOTS, k / SLOTS & 1, 1u << 12);
				}
			if (values) asm volatile("bar.arrive 4, 288;" ::: "memory");
		} else if (warp == 9 && lane == 0) { // the products: the groups take turns
			constexpr uint32_t type = std::is_same<T, bf16>::value ? (1u << 7) | (1u << 10) : 0;
			constexpr uint32_t score = (1u << 4) | type | ((uint32_t)(AW_KEYS >> 3) << 17) | (8u << 24), value = (1u << 4) | type | (1u << 16) | ((uint32_t)(D >> 3) << 17) | (8u << 24); // 128 rows; values: columns side by side
			auto wait_slot = [&](int k) { return ap_wait(s.full + k % SLOTS, k / SLOTS & 1, &s.lost); };
			auto scores = [&](int g, int i) { // of tile i
#pragma unroll
				for (int pn = 0; pn < PANELS; ++pn)
#pragma unroll
					for (int k = 0; k < 4; ++k) umma_f16(tmem + 128 * g, umma_desc_sw128(s.q[two ? 0 : g][pn]) + 2 * k, umma_desc_sw128(s.kv[2 * i % SLOTS][pn]) + 2 * k, score, (pn | k) ? 1u : 0u);
				umma_commit(s.s_full + g);
			};
			auto sums = [&](int g, int i, int n) { // the n-th of the group's
				if (!ap_wait(s.p_full + g, n & 1, &s.lost)) return false;
				tc_fence_after();
#pragma unroll
				for (int x = 0; x < AW_KEYS / 16; ++x) umma_f16_ts(tmem + O_COL + 128 * g, tmem + 128 * g + 8 * x, umma_desc_values(s.kv[(2 * i + 1) % SLOTS]) + 128 * x, value, (n | x) ? 1u : 0u);
				return true;
			};
			// (slots are waited for before the weights and given back after both groups' products: nothing stands between a group's two)
			bool good = true;
			if (two) {
				for (int i = 0; i < min(2, tiles) && good; ++i)
					if ((good = wait_slot(2 * i))) {
						tc_fence_after();
						scores(i, i), umma_commit(s.empty + 2 * i % SLOTS);
					}
				for (int i = 0; i < tiles && good; ++i) {
					const bool more = i + 2 < tiles;
					if (!(good = wait_slot(2 * i + 1) && (!more || wait_slot(2 * i + 4)) && sums(i & 1, i, i >> 1))) break;
					if (more) scores(i & 1, i + 2), umma_commit(s.empty + (2 * i + 4) % SLOTS);
					else umma_commit(s.done + (i & 1));
					umma_commit(s.empty + (2 * i + 1) % SLOTS);
				}
			} else {
				good = tiles > 0 && wait_slot(0);
				if (good) {
					tc_fence_after();
					for (int g = 0; g < groups; ++g) scores(g, 0);
					umma_commit(s.empty);
				}
				for (int i = 0; i < tiles && good; ++i) {
					const bool more = i + 1 < tiles;
					if (!(good = wait_slot(2 * i + 1) && (!more || wait_slot(2 * i + 2)))) break;
					for (int g = 0; g < groups && good; ++g) {
						if (!(good = sums(g, i, i))) break;
						if (more) scores(g, i + 1);
						else umma_commit(s.done + g);
					}
					if (!good) break;
					umma_commit(s.empty + (2 * i + 1) % SLOTS);
					if (more) umma_commit(s.empty + (2 * i + 2) % SLOTS);
				}
			}
			umma_commit(&s.idle); // nothing of this block's is left in the tensor core when its memory goes
			mbar_wait_bounded(&s.idle, 0);
		}
	}
	__syncwarp();
	tc_fence_before();
	__syncthreads();
	tc_fence_after();
	if (warp == 9) tmem_dealloc(tmem, 512);
}

// Folds the shares of a split task (Wide), 32 rows a block, a warp a row.  Bound: latency; 20 tasks of 7 shares (17 MB) 20 us with caches cold, behind a kernel that the split makes 110 us shorter.
template <typename T>
__global__ void __launch_bounds__(128) k_c16_join(const C16 c, const Attend a, const Wide w) {
	pdl_wait_prev();
	Task task;
	Unit u;
	__shared__ int found[3], sums[4];
	if (!task_of<128>(c, a, w.cut + blockIdx.x, found, sums, task) || !own_unit(c, a, task.z, u)) return;
	const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row0 = task.tile * 256, rows = (int)min(256LL, (long long)u.tokens * a.group - row0);
	for (int r = blockIdx.y * 32 + warp; r < min(rows, (int)blockIdx.y * 32 + 32); r += 4) {
		const int token = u.t0 + (row0 + r) / a.group, head = task.kvh * a.group + (row0 + r) % a.group;
		const size_t place = (size_t)blockIdx.x * w.shares * 256 + r;
		const float sk = a.sinks ? a.sinks[head] * A16_LOG2E : -INFINITY;
		const float2 st = lane < w.shares ? a.stats[place + lane * 256] : make_float2(-INFINITY, 0.f);
		const float top = fmaxf(sk, warp_max(st.x)), weight = st.x == -INFINITY ? 0.f : ex2(st.x - top);
		float den = warp_sum(weight * st.y);
		if (a.sinks) den += at_sink(sk, top);
		const float norm = den > 0.f ? 1.f / den : den == 0.f ? 0.f : den; // (0: nothing was seen; a NaN stays one)
		for (int d0 = 0; d0 < c.dim; d0 += 128) {
			const int d = min(d0 + 4 * lane, c.dim - 4);
			float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
			add_places(v, a.sums + place * c.dim + d, (size_t)256 * c.dim, w.shares, weight);
			if (d0 + 4 * lane < c.dim) put4<T>(a.out + token * a.o_row + head * a.o_head + d, a.out_vec, times4(v, norm));
		}
	}
}

// Folds the shares of one (token, head), in the order of their places: a warp for each.  Bound: latency; 18 sequences of 5 tokens with 24 heads 7.8 us, 32 of one token with 32 heads and 11 shares 8.5 us (caches cold, launch included).
template <typename T>
__global__ void __launch_bounds__(128) k_c16_fold(const C16 c, const Attend a) {
	pdl_wait_prev();
	const int b = blockIdx.z, kvh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
	Unit u;
	if (!own_unit(c, a, b, u)) return;
	const int n = u.tokens, start = u.t0, from = u.lead < 0 ? a.before : 0; // (a sequence of no group has no shares of a prefix)
	for (long long row = (long long)blockIdx.x * 4 + warp; row < (long long)n * a.group; row += gridDim.x * 4) {
		const int token = start + (int)(row / a.group), head = kvh * a.group + (int)(row % a.group);
		const size_t place = ((size_t)token * a.heads + head) * a.places;
		const float sk = a.sinks ? a.sinks[head] * A16_LOG2E : -INFINITY;
		float mx = sk, den = 0.f;
		for (int s = from + lane; s < a.places; s += 32) mx = fmaxf(mx, a.stats[place + s].x);
		mx = warp_max(mx);
		float4 v[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
		for (int s0 = from; s0 < a.places; s0 += 32) {
			const float2 st = s0 + lane < a.places ? a.stats[place + s0 + lane] : make_float2(-INFINITY, 0.f);
			const float w = st.x == -INFINITY ? 0.f : ex2(st.x - mx);
			den = fmaf(w, st.y, den);
#pragma unroll
			for (int k = 0; k < 2; ++k) {
				const int d = min(128 * k + 4 * lane, c.dim - 4);
				if (128 * k < c.dim) add_places(v[k], a.sums + (place + s0) * c.dim + d, c.dim, min(a.places - s0, 32), w);
			}
		}
		den = warp_sum(den);
		if (a.sinks) den += at_sink(sk, mx);
		const float norm = den > 0.f ? 1.f / den : den == 0.f ? 0.f : den; // (0: nothing was seen; a NaN stays one)
#pragma unroll
		for (int k = 0; k < 2; ++k)
			if (128 * k + 4 * lane < c.dim) put4<T>(a.out + token * a.o_row + head * a.o_head + 128 * k + 4 * lane, a.out_vec, times4(v[k], norm));
	}
}

// ---------------------------------------------------------------- the host's side
// How the work is cut.  Three ways: few rows of each group or sequence, prefix and own keys in one list (ROWS); the groups' prefixes as tiles of many rows, then every sequence's own keys (PREFIXES); every sequence as tiles of many
// rows (TILES).
enum A16Way { A16_ROWS, A16_PREFIXES, A16_TILES };
struct A16Plan {
	int way;
	int tile, shares, each, cluster; // few rows: rows of a CTA, shares of a tile's keys and the chunks of each, whether a cluster folds the shares
	int warps;                       // of a CTA
	int units;                       // of the grid
	long long rows;                  // of a unit at most
	Wide wide;                       // many rows
	int wide_units;
	int before, places;
	long long tasks, split_places;   // many rows of sequences: CTAs, places of the split ones' rows
	int apart;                       // the rows of those that go apart, at most
};
constexpr int AR_ROOM = 148 * 3; // CTAs of few rows that run at a time
constexpr int AW_ROOM = 148;     // and of many
constexpr int AW_SHARES = 32;    // of a tile's keys at most (a lane for each where they are folded)

int a16_box(int page) { // keys that lie side by side in every page, as a copy's box has them
	int box = 1;
	while (box < 64 && page % (2 * box) == 0) box *= 2;
	return box;
}
// Shares of a tile's keys: folded inside clusters of eight CTAs of eight warps where tiles and keys are few, through memory else.  us, clusters / memory, one sequence of 32 heads over 8 key heads of 128 channels: 1000 keys
// 9.3 / 9.5, 4000 11.2 / 11.7, 16000 19.3 / 16.9, 60000 53 / 48 (over 2 key heads 9.5 / 9.5, 11.4 / 10.9, 19 / 15, 48 / 22); four beams behind 1000 positions 13.1 / 13.5, 4000 14.3 / 16.1, 16000 25 / 23; twice that, which
// clusters of eight do not fit side by side, 21.4 / 19.1.  Clusters of 16 (of four warps) 18.1 and 26.5 for the four beams.
void rows_plan(A16Plan& r, const SeqCache16& c, long long n, long long rows, long long likely, long long keys, bool clusters) { // n: tiles that have rows; rows: of a unit at most, likely: about
	n = std::max(1LL, n), r.rows = rows, r.tile = likely > 8 ? 16 : 8, r.warps = 4;
	const int chunks = (int)std::min<long long>(std::max(keys, 0LL) / AR_KEYS + 2, INT_MAX / 2); // (they begin anywhere)
	const long long room = AR_ROOM;
	r.cluster = clusters && c.dim <= 128 && n <= 12 && chunks > 4 && chunks <= 192;
	if (r.cluster) {
		r.warps = 8, r.shares = AR_CLUSTER, r.each = cdiv(chunks, r.shares);
		return;
	}
	// many CTAs: several rounds, so that the last one is short
	long long shares = n >= room ? 1 : n > room / 2 ? cdiv(6 * room, n) : room / n;
	shares = std::max(1LL, std::min({shares, (long long)cdiv(chunks, n > room / 2 ? 8 : 4), (long long)AR_SHARES}));
	r.each = cdiv(chunks, shares), r.shares = cdiv(chunks, r.each);
}
// Groups: as many shares of their prefixes as CTAs run at a time, of one length for all groups (`lengths`: what each of them shared when the batch was described).
void groups_plan(A16Plan& r, const SeqCache16& c, const SeqShared& s, long long rows, long long likely, long long most) {
	r.wide.box = a16_box(c.page), r.wide.tiles = cdiv(rows, 256), r.wide_units = s.n;
	const int longest = std::max(1, (int)std::min<long long>(cdiv(most, AW_KEYS), INT_MAX / 2));
	const long long per = (long long)cdiv(likely, 256) * c.heads;
	auto ctas = [&](int each) { // that have keys
		long long n = 0;
		for (int g = 0; g < s.n; ++g) n += std::max(1, cdiv(s.lengths ? std::min<long long>(s.lengths[g], most) : most, (long long)each * AW_KEYS));
		return n * per;
	};
	int each = std::max(cdiv(longest, AW_SHARES), std::min(4, longest)); // (two for each group of warps)
	if (s.n * per >= AW_ROOM) each = longest;
	while (each < longest && ctas(each) > AW_ROOM) each += std::max(1, each / 16);
	r.wide.each = std::min(each, longest), r.wide.shares = cdiv(longest, r.wide.each);
}
// Sequences: whole tasks, but for those that a last round of fewer CTAs than run at a time would have.
void tasks_plan(A16Plan& r, const SeqCache16& c, const SeqPortions& p, const SeqAttend16& a, long long rows, long long most) {
	r.wide.box = a16_box(c.page), r.wide.tiles = cdiv(rows, 256), r.wide.through = 1, r.wide_units = 1;
	// As many tasks as there can be, whatever the counts become: no more tiles than the rows fill and one begun for every sequence.  (A prompt of 8192 tokens among 255 single ones behind 2000 positions 1243 us; with as many
	// blocks for each as the prompt has tiles 3318.)
	const long long all = std::min((long long)p.n * r.wide.tiles, (long long)a.q.rows * (a.heads / c.heads) / 256 + p.n) * c.heads, live = a.row_tiles > 0 ? std::min(all, std::max(0LL, a.row_tiles - (r.apart ? a.few : 0)) * c.heads) : all, rest = live % AW_ROOM;
	const int longest = std::max(1, (int)std::min<long long>(cdiv(most, AW_KEYS), INT_MAX / 2));
	const long long shares = rest ? std::min<long long>({AW_ROOM / rest, cdiv(longest, 4), AW_SHARES}) : 1;
	r.wide.shares = (int)std::max(1LL, shares), r.wide.planned = (int)std::min<long long>(live, INT_MAX), r.wide.cut = shares > 1 ? (int)(live - rest) : r.wide.planned;
	r.tasks = all + (long long)(r.wide.planned - r.wide.cut) * (r.wide.shares - 1);
	r.split_places = (long long)(r.wide.planned - r.wide.cut) * r.wide.shares * 256;
}
A16Plan a16_plan(const SeqCache16& c, const SeqPortions& p, const SeqShared* s, const SeqAttend16& a) {
	A16Plan r = {};
	const int group = a.heads / c.heads, groups = s ? s->n : 0;
	// `packed`: rows of a group at most, which the grids have room for; `likely`: about, which times and shares are reckoned from
	const long long rows = (long long)p.longest * group, packed = groups ? (long long)std::min(s->tokens, a.q.rows) * group : 0, likely = groups && s->likely > 0 ? std::min(packed, (long long)s->likely * group) : packed;
	// keys that a row sees at most: of a prefix, behind one, of a sequence of no group
	auto seen = [&](long long keys) { return a.window > 0 ? std::min(keys, (long long)a.window + p.longest) : keys; };
	const long long shared = groups ? seen(s->longest) : 0, own = groups ? seen(s->most_own) : 0, lone = groups ? (s->n_alone ? seen(s->most_alone) : 0) : seen(std::max(a.most_keys, 1));
	const bool wide = (c.dim == 64 || (c.dim > 64 && c.dim <= 128)) && c.page % 8 == 0 && c.pages > 0 && std::max(rows, packed) <= 65535 * 256LL;
	// Each way's time, estimated in us from the work that it does; the least.  Of 129 shapes that were measured in all their ways (1 to 8 groups of 3 to 64 sequences of 1 to 100 tokens behind 600 to 12000 positions, 1 to 8 key
	// heads of 64 and 128 channels) the rule takes one that is 1.4 % slower than the best in the mean.  us, few rows / prefixes / tiles: 8 groups of 8 sequences of 4 heads a key head behind up to 3000 positions 33 / 50, 4 groups of 16
	// behind up to 12000 104 / 79, one of 64 behind 600 25 / 33, behind 3000 37 / 35; 16 sequences of up to 20 tokens behind 600 56 / 43 / 25, behind 12000 253 / 88 / 185; 3 of 60 behind 4000 97 / 47 / 51.
	double prefix = (double)shared; // what the groups share in the mean
	if (groups && s->lengths) {
		prefix = 0.;
		for (int g = 0; g < groups; ++g) prefix += std::min<double>(s->lengths[g], (double)shared) / groups;
	}
	const int alone = groups ? s->n_alone : p.n;
	const long long together = groups ? std::min<long long>(cdiv(16, group), std::max(likely / group, 1LL)) : 0; // sequences of a CTA's rows at most
	const long long most = std::max(shared + own * together, lone), units = groups + alone, tiles_g = (long long)groups * cdiv(likely, 16) * c.heads, tiles_a = (long long)alone * cdiv(rows, 16) * c.heads;
	const double us_rows = 10. + (tiles_g * (prefix + own * together) + tiles_a * lone) / 20000. + 2. * most / (128. * std::max<double>(1., std::min<double>(AR_SHARES, (double)AR_ROOM / std::max(tiles_g + tiles_a, 1LL))));
	const double us_tile = (a.softcap > 0.f ? 6. : 2.) / AW_ROOM / AW_KEYS; // a key of 256 rows, on one of the SMs (a soft cap: a reciprocal and eight products and sums more a score, and every tile takes the slower way)
	const double us_prefixes = 20. + us_tile * groups * c.heads * cdiv(likely, 256) * prefix + cdiv((long long)p.n * c.heads * cdiv(rows, 16), AR_ROOM) * (4. + std::max(own, lone) / 130.);
	const double us_row = us_tile * c.heads * (groups ? prefix + own : lone), us_all = 24. + us_row * (double)(a.row_tiles > 0 ? a.row_tiles : (long long)p.n * cdiv(rows, 256));
	// Single tokens among prompts are a tile each, of which their rows are a small part: they go apart, in CTAs of few rows beside the tiles' last ones.  us, together / apart, 32 heads over 8 of
	// 128 channels: a prompt of 8192 among 255 tokens behind 2000 positions 1243 / 917 (594 and 293 by themselves), of 2048 among 63 262 / 158, of 512 among 31 133 / 86, 8 of 600 among 120 479 / 388, 2 of 900 with 20 that share 1500
	// 154 / 123, one of 500 among 16 behind 20000 395 / 306, one of 300 among 5 42 / 42 (taken together).
	const double us_apart = us_all - us_row * a.few + cdiv((long long)a.few * c.heads, AR_ROOM) * (4. + std::max(shared + own, lone) / 130.);
	const bool apart = a.few > 0 && a.row_tiles > a.few && us_apart < us_all;
	const double us_tiles = apart ? us_apart : us_all;
	if (wide && rows >= 32 && us_tiles < us_rows && (!groups || us_tiles <= us_prefixes)) {
		r.way = A16_TILES;
		if (apart) {
			r.apart = std::max(8, group), r.rows = r.apart, r.tile = r.apart > 8 ? 16 : 8, r.warps = 4, r.shares = 1, r.units = p.n;
			r.each = (int)std::min<long long>(std::max(shared + own, lone) / AR_KEYS + 3, INT_MAX / 2);
		}
		tasks_plan(r, c, p, a, rows, std::max(shared + own, lone));
		return r;
	}
	if (wide && packed > 0 && us_prefixes < us_rows) {
		r.way = A16_PREFIXES;
		groups_plan(r, c, *s, packed, likely, shared);
		r.before = r.wide.shares;
		r.units = p.n;
		rows_plan(r, c, (long long)p.n * cdiv(rows, 16) * c.heads, rows, rows, std::max(own, lone), false);
		r.places = r.before + (r.shares > 1 ? r.shares : 0);
		return r;
	}
	r.way = A16_ROWS, r.units = (int)units;
	rows_plan(r, c, tiles_g + tiles_a, std::max(rows, packed), std::max(rows, likely), most, true);
	r.places = r.shares > 1 && !r.cluster ? r.shares : 0;
	return r;
}
size_t a16_rows(const SeqAttend16& a, const A16Plan& p) { return p.way == A16_TILES ? p.split_places : (size_t)a.q.rows * a.heads * p.places; }
size_t a16_bytes(const SeqCache16& c, const SeqAttend16& a, const A16Plan& p) { return a16_rows(a, p) * (c.dim * sizeof(float) + sizeof(float2)); }

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
		if (s->n < 0 || s->n > p->n || s->longest < 0 || s->tokens < 0 || s->likely < 0 || s->most_own < 0 || s->most_alone < 0) return refuse("attend16: %d groups of %d sequences, longest %d, tokens %d", s->n, p->n, s->longest, s->tokens);
		if (s->n && (!s->first || !s->count || !s->positions || !s->group)) return refuse("attend16: the groups' description is missing");
		if (s->n_alone < 0 || s->n_alone > p->n || (s->n && s->n_alone && !s->alone)) return refuse("attend16: %d sequences of %d in no group of the groups' description", s->n_alone, p->n);
		if (((uintptr_t)s->first | (uintptr_t)s->count | (uintptr_t)s->positions | (uintptr_t)s->group | (uintptr_t)s->alone) % 4) return refuse("attend16: the groups' description is not aligned to 4 bytes");
		if (p->n + s->n > 65535) return refuse("attend16: %d sequences and %d groups: at most 65535", p->n, s->n);
	}
	if (std::max(p->longest, s && s->n ? s->tokens : 0) * group > INT_MAX - 256) return refuse("attend16: %d tokens of %d query heads a key head: at most 2^31 pairs a sequence or group", std::max(p->longest, s ? s->tokens : 0), (int)group);
	if ((uintptr_t)a->sinks % 4) return refuse("attend16: sinks are not aligned to 4 bytes");
	if (!(A16_LOG2E * std::fabs(a->scale) < INFINITY) || a->window < 0 || !(a->softcap >= 0.f && a->softcap < INFINITY) || (a->softcap > 0.f && !(2.f * A16_LOG2E * std::fabs(a->scale) / a->softcap < INFINITY))) return refuse("attend16: scale, window or softcap out of range");
	if (a->row_tiles < 0 || a->few < 0) return refuse("attend16: %lld row tiles, %d sequences of few rows", a->row_tiles, a->few);
	return 0;
}

template <typename T, int D, int NQ, int W, bool CAP>
cudaError_t rows_cap(const C16& c, const Attend& a, dim3 grid, bool after, cudaStream_t st) {
	constexpr size_t smem = ar_smem<D, NQ, W>();
	static std::atomic<uint64_t> done{0};
	cudaError_t e = allow(k_c16_rows<T, D, NQ, W, CAP>, smem, done, true);
	if (e == cudaSuccess) e = launch(st, after, a.cluster ? a.shares : 1, k_c16_rows<T, D, NQ, W, CAP>, grid, dim3(32 * W), smem, c, a);
	return e;
}
template <typename T, int D, int NQ, int W>
cudaError_t rows_launch(const C16& c, const Attend& a, dim3 grid, bool after, cudaStream_t st) {
	return a.softcap > 0.f ? rows_cap<T, D, NQ, W, true>(c, a, grid, after, st) : rows_cap<T, D, NQ, W, false>(c, a, grid, after, st);
}
template <typename T, int D>
cudaError_t rows_tile(const A16Plan& p, const C16& c, const Attend& a, dim3 grid, bool after, cudaStream_t st) {
	if constexpr (D <= 128)
		if (p.warps == 8) return p.tile == 8 ? rows_launch<T, D, 1, 8>(c, a, grid, after, st) : rows_launch<T, D, 2, 8>(c, a, grid, after, st);
	return p.tile == 8 ? rows_launch<T, D, 1, 4>(c, a, grid, after, st) : rows_launch<T, D, 2, 4>(c, a, grid, after, st);
}
// a pool as rows of dim channels; boxes of 64 channels and `box` rows, swizzled by the row
typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                             CUtensorMapFloatOOBfill);
cudaError_t pool_map(CUtensorMap& m, const SeqCache16& c, void* pool, int box) {
	static const EncodeFn encode = [] {
		cudaDriverEntryPointQueryResult found;
		void* fn = nullptr;
		return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &found) == cudaSuccess && found == cudaDriverEntryPointSuccess ? (EncodeFn)fn : nullptr;
	}();
	const cuuint64_t dims[2] = {(cuuint64_t)c.dim, (cuuint64_t)c.pages * c.heads * c.page}, strides[1] = {(cuuint64_t)c.dim * 2};
	const cuuint32_t boxes[2] = {64, (cuuint32_t)box}, steps[2] = {1, 1};
	if (!encode || encode(&m, c.type == SEQ_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, pool, dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
	                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
		return cudaErrorInvalidValue;
	return cudaSuccess;
}
template <typename T, int D, bool CAP>
cudaError_t tiles_launch(const SeqCache16& cache, const C16& c, const Attend& a, const A16Plan& p, cudaStream_t st) {
	static std::atomic<uint64_t> done{0};
	CUtensorMap mk, mv;
	cudaError_t e = pool_map(mk, cache, cache.k, p.wide.box);
	if (e == cudaSuccess) e = pool_map(mv, cache, cache.v, p.wide.box);
	if (e == cudaSuccess) e = allow(k_c16_tiles<T, D, CAP>, sizeof(AwShared<D>), done);
	if (e == cudaSuccess) e = launch(st, false, 1, k_c16_tiles<T, D, CAP>, dim3((unsigned)(p.way == A16_TILES ? p.tasks : (long long)p.wide.tiles * c.heads * p.wide.shares), 1, p.wide_units), dim3(AW_THREADS), sizeof(AwShared<D>), mk, mv, c, a, p.wide);
	return e;
}
template <typename T>
cudaError_t tiles_wide(const SeqCache16& cache, const C16& c, const Attend& a, const A16Plan& p, cudaStream_t st) {
	if (a.softcap > 0.f) return c.dim == 64 ? tiles_launch<T, 64, true>(cache, c, a, p, st) : tiles_launch<T, 128, true>(cache, c, a, p, st);
	return c.dim == 64 ? tiles_launch<T, 64, false>(cache, c, a, p, st) : tiles_launch<T, 128, false>(cache, c, a, p, st);
}
template <typename T>
cudaError_t rows_wide(const A16Plan& p, const C16& c, const Attend& a, dim3 grid, bool after, cudaStream_t st) {
	return c.dim <= 64 ? rows_tile<T, 64>(p, c, a, grid, after, st) : c.dim <= 128 ? rows_tile<T, 128>(p, c, a, grid, after, st) : rows_tile<T, 256>(p, c, a, grid, after, st);
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
	if (shared && shared->n) c.groups = shared->n, c.first = shared->first, c.members = shared->count, c.positions = shared->positions, c.group = shared->group, c.alone = shared->n_alone, c.lonely = shared->alone;
	Attend a = {};
	a.q = (const uint16_t*)q->q.p, a.q_row = q->q.row_stride, a.q_head = q->q.head_stride, a.out = (uint16_t*)q->out.p, a.o_row = q->out.row_stride, a.o_head = q->out.head_stride;
	a.rows = q->q.rows, a.heads = q->heads, a.group = q->heads / cache->heads, a.scale = q->scale, a.softcap = q->softcap, a.window = q->window, a.sinks = q->sinks;
	a.out_vec = ((uintptr_t)a.out | (uintptr_t)(a.o_row * 2) | (uintptr_t)(a.o_head * 2)) % 8 == 0;
	a.families = plan.way == A16_ROWS ? 1 : -plan.apart / a.group, a.shares = plan.shares, a.each = plan.each, a.cluster = plan.cluster, a.before = plan.before, a.places = plan.places;
	a.sums = (float*)q->workspace, a.stats = (float2*)(a.sums + a16_rows(*q, plan) * c.dim);
	const dim3 grid(plan.way == A16_TILES && !plan.apart ? 1 : cdiv(plan.rows, plan.tile), cache->heads * std::max(1, plan.shares), plan.units);
	if (grid.y > 65535) return refuse("attend16: too many key heads");
	if ((long long)plan.wide.tiles * cache->heads * plan.wide.shares > INT_MAX || plan.tasks > INT_MAX || plan.split_places > INT_MAX) return refuse("attend16: too many rows");
	const cudaStream_t st = (cudaStream_t)stream;
	const bool half = cache->type == SEQ_F16;
	cudaError_t e = cudaSuccess;
	if (plan.way != A16_ROWS) e = half ? tiles_wide<__half>(*cache, c, a, plan, st) : tiles_wide<bf16>(*cache, c, a, plan, st);
	const bool after = plan.before > 0 || plan.apart > 0;
	if (e == cudaSuccess && (plan.way != A16_TILES || plan.apart)) e = half ? rows_wide<__half>(plan, c, a, grid, after, st) : rows_wide<bf16>(plan, c, a, grid, after, st);
	if (e == cudaSuccess && plan.split_places)
		e = launch(st, true, 1, half ? k_c16_join<__half> : k_c16_join<bf16>, dim3(plan.wide.planned - plan.wide.cut, 8), dim3(128), 0, c, a, plan.wide);
	if (e == cudaSuccess && plan.places > plan.before) {
		const dim3 fold(std::min(cdiv((long long)batch->longest * a.group, 4), 65535), cache->heads, batch->n);
		e = launch(st, true, 1, half ? k_c16_fold<__half> : k_c16_fold<bf16>, fold, dim3(128), 0, c, a);
	}
	return e == cudaSuccess ? 0 : failed("attend16", e);
}

extern "C" int calm_b200_seq_attend16_way(const struct SeqCache16* cache, const struct SeqPortions* batch, const struct SeqShared* shared, const struct SeqAttend16* args) {
	using namespace seqops;
	if (const int rc = check_attend16(cache, batch, shared, args)) return rc;
	const A16Plan p = a16_plan(*cache, *batch, shared, *args);
	return p.way | (p.way == A16_ROWS && p.cluster ? 4 : 0) | (p.places > p.before || p.split_places ? 8 : 0) | (p.apart ? 16 : 0);
}
