// seqcache8.cu -- a cache of keys and values in 8 bits and attention over it (calm_b200_seq_cache8_store, calm_b200_seq_attend8 in include/calm_b200_seq.h).

#include "seqops.cuh"
#include "tc05.cuh"

#include <limits.h>

#include <algorithm>

namespace seqops {
namespace {

typedef __nv_bfloat16 bf16;

// what the kernels know of the cache and the batch
struct C8 {
	uint8_t *k, *v;
	float *ks, *vs;
	const int* table;
	int pages, heads, page, dim, slots, table_pages;
	int page_shift; // log2 of page, -1: no power of two
	const int *start, *count, *slot, *pos0;
	__device__ __forceinline__ int reach(int slot) const { return (unsigned)slot < (unsigned)slots && pages > 0 ? (int)min((long long)table_pages * page, INT_MAX - 128LL) : 0; } // positions that the table has
};
constexpr int C8_LEAST = -64; // exponent of the smallest scale

__device__ __forceinline__ int pow2_of(float scale) { return max((int)(__float_as_uint(scale) >> 23 & 255) - 127, C8_LEAST); }
// the least e >= C8_LEAST with amax <= 448 * 2^e: amax = m 2^x with 1/2 <= m < 1, 448 = 0.875 * 2^9
__device__ __forceinline__ int scale_exponent(float amax) {
	const uint32_t u = __float_as_uint(amax);
	const int x = (int)(u >> 23) - 126;
	return max(x - ((u & 0x7fffff) <= 0x600000 ? 9 : 8), C8_LEAST);
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
	const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3), hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
	return lo | hi << 16;
}
__device__ __forceinline__ int page_index(const C8& c, int pos) { return c.page_shift >= 0 ? pos >> c.page_shift : pos / c.page; }
__device__ __forceinline__ int page_row(const C8& c, int pos) { return c.page_shift >= 0 ? pos & (c.page - 1) : pos % c.page; }
// four codes as two pairs of fp16
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t codes, uint32_t& lo, uint32_t& hi) {
	asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(codes));
}
// two codes (the lower byte first) as fp16
__device__ __forceinline__ uint32_t e4m3x2_to_f16(uint32_t codes) {
	uint32_t r;
	asm("{\n\t.reg .b16 h, x;\n\tmov.b32 {h, x}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(codes));
	return r;
}

// ---------------------------------------------------------------- storing
// A warp takes one page of a sequence's new rows, one head, keys or values: the largest finite value, the scale, the codes of earlier rows where the scale grew, the codes
// of the new rows.  Pages are independent, so a prompt's run side by side.  Bound: memory for prompts (rows read once from DRAM, once more from L1: 4955 rows of 8 heads of 128
// fp32 channels 11.2 us, 4.5 TB/s), latency for single tokens (32 of them 2.8 us: the page's number, its scale, its rows one after another).
constexpr int ST_WARPS = 4;
struct StoreRows {
	const void* p;
	long long row, head;
	int rows, vec; // vec: four elements at a time
};
template <typename T>
__device__ __forceinline__ float4 store_load(const T* p, bool vec) {
	if constexpr (sizeof(T) == 4) {
		if (vec) return *reinterpret_cast<const float4*>(p);
	} else {
		if (vec) {
			const uint2 w = *reinterpret_cast<const uint2*>(p);
			const T* h = reinterpret_cast<const T*>(&w);
			return make_float4(as_f32(h[0]), as_f32(h[1]), as_f32(h[2]), as_f32(h[3]));
		}
	}
	return make_float4(as_f32(p[0]), as_f32(p[1]), as_f32(p[2]), as_f32(p[3]));
}
template <typename T>
__global__ void __launch_bounds__(32 * ST_WARPS) k_c8_store(const C8 c, const StoreRows rk, const StoreRows rv) {
	const int b = blockIdx.z, unit = blockIdx.y * ST_WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
	if (unit >= 2 * c.heads) return;
	const bool isv = unit >= c.heads;
	const int h = isv ? unit - c.heads : unit, n = c.count[b], p0 = c.pos0[b], start = c.start[b], slot = c.slot[b];
	const StoreRows& r = isv ? rv : rk;
	if (n < 1 || p0 < 0 || p0 > INT_MAX - n || (unsigned)slot >= (unsigned)c.slots || start < 0 || n > r.rows - start) return;
	const long long block = p0 / c.page + (long long)blockIdx.x, page0 = block * c.page;
	if (block >= c.table_pages || page0 >= (long long)p0 + n) return;
	const int id = c.table[(size_t)slot * c.table_pages + block];
	if ((unsigned)id >= (unsigned)c.pages) return;
	const int lo = (int)max((long long)p0 - page0, 0LL), hi = (int)min((long long)p0 + n - page0, (long long)c.page); // rows of the page
	const T* src = (const T*)r.p + (start + (page0 + lo - p0)) * r.row + h * r.head;
	uint8_t* const codes = (isv ? c.v : c.k) + ((size_t)id * c.heads + h) * c.page * c.dim;
	float* const scale = (isv ? c.vs : c.ks) + (size_t)id * c.heads + h;
	const int old = pow2_of(*scale);
	auto mag = [](float x) { const float a = fabsf(x); return a < INFINITY ? a : 0.f; };
	float amax = 0.f;
	for (int d = 4 * lane; d < c.dim; d += 128)
#pragma unroll 4
		for (int i = 0; i < hi - lo; ++i) {
			const float4 x = store_load(src + i * r.row + d, r.vec);
			amax = fmaxf(amax, fmaxf(fmaxf(mag(x.x), mag(x.y)), fmaxf(mag(x.z), mag(x.w))));
		}
	int e = scale_exponent(warp_max(amax));
	if (lo > 0) {
		e = max(e, old);
		if (e > old) { // the earlier rows' codes under the raised scale: exact but for what becomes subnormal
			const float f = pow2f(max(old - e, -126));
			for (int d = 4 * lane; d < c.dim; d += 128)
				for (int i = 0; i < lo; ++i) {
					uint32_t* const w = reinterpret_cast<uint32_t*>(codes + (size_t)i * c.dim + d);
					const uint32_t x = *w, p = e4m3x2_to_f16(x), q = e4m3x2_to_f16(x >> 16);
					const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&p)), v = __half22float2(*reinterpret_cast<const __half2*>(&q));
					*w = e4m3x4(u.x * f, u.y * f, v.x * f, v.y * f);
				}
		}
	}
	const float inv = pow2f(-e);
	auto put = [&](float x) { return x == x ? x * inv : 0.f; };
	for (int d = 4 * lane; d < c.dim; d += 128)
#pragma unroll 4
		for (int i = 0; i < hi - lo; ++i) {
			const float4 x = store_load(src + i * r.row + d, r.vec);
			*reinterpret_cast<uint32_t*>(codes + (size_t)(lo + i) * c.dim + d) = e4m3x4(put(x.x), put(x.y), put(x.z), put(x.w));
		}
	__syncwarp();
	if (lane == 0) *scale = pow2f(e);
}

// ---------------------------------------------------------------- attention
// The rows of a CTA are 8 NQ pairs (token, query head) of one sequence that read one key head, so a key is read once for all of them: row i of a sequence's tile is token
// i / group, head i % group of the group.  Each warp walks its own chunks of 32 keys with running references and sums of its own (no barrier between warps until the end),
// fed by a ring of asynchronous copies; codes become fp16 in registers on their way into m16n8k16 products whose 16 rows are keys (scores: keys x queries) or channels (values:
// channels x queries), so that eight rows of queries fill a product.  An e4m3 code is exact in fp16; scales do not enter the products: a key's scale multiplies its scores,
// a value's scale s joins the exponent, w_j = 2^(z_j - r), z_j = log2(e) score_j + log2 s_j, where r keeps the weights that are rounded to fp16 at 2^15 or less; the denominator sums
// w_j / s_j.  r moves (and the sums are rescaled) when a chunk's largest z passes it by 15, to 10 below that z: almost only in a warp's first chunks.
// 64 tokens of 32 heads over 2000 to 8000 keys of 8 heads of 128 channels (656 MB): 125 us, 5.3 TB/s; one over 4000 keys 11.1 us.  Bound: with many CTAs issue and the latency of
// a warp's chunk (1.7 warp instructions a cycle; 49 million in all), with few the latency of copy, products, softmax and the cluster's fold.
constexpr int AT_WARPS = 4, AT_KEYS = 32;
constexpr int AT_SHARES = 64;  // of a tile's keys at most
constexpr int AT_TILE = 16, AT_CLUSTER = 16; // rows of a CTA at most; shares that a thread-block cluster folds at most
constexpr float AT_LOG2E = 1.4426950408889634f;
constexpr int AT_LIFT = 15;                // the largest query of a tile stands at 2^15 in fp16, so that what rounds as a subnormal is 2^-40 of it
constexpr int AT_ALIKE = 12;               // rows whose largest elements lie further apart (2^this) have a power of two each; nearer ones share the tile's: no factor a score
constexpr int AT_NO_ROW = -1000;           // exponent of a row of zeros
constexpr float AT_MOST = 15.f, AT_SET = 10.f; // weights: at most 2^15, the largest at 2^10 or more

struct Attend {
	const void* q;
	long long q_row, q_head;
	void* out;
	long long o_row, o_head;
	int q_type, out_type;
	int rows, heads, group;
	float scale, softcap;
	int window, keep_first, chunk;
	const float *sinks, *slopes, *gate;
	long long gate_row, gate_head, gate_dim;
	int tile;         // rows of a CTA: 8 NQ
	int shares, each; // shares of a tile's keys at most, chunks of each
	int cluster;      // 1: the shares of a tile are a cluster
	float* part;      // [rows][heads][shares][dim + 2]: sum, reference, denominator
};

template <int D>
struct AtStage { // a warp's chunk: the next one's keys come while its values are used, the next one's values while their keys are
	uint8_t k[AT_KEYS * D], v[AT_KEYS * D];
	float ks[2][AT_KEYS], vs[2][AT_KEYS];
	uint32_t seen[4]; // keys that are there, of this chunk and the next one
};
template <int D>
__host__ __device__ constexpr size_t at_ring() { // (the sums of the warps take its place)
	const size_t a = (size_t)AT_WARPS * sizeof(AtStage<D>), b = (size_t)AT_WARPS * 8 * (8 * (D == 256 ? 52 : 20) + 4) * sizeof(float) + (size_t)AT_TILE * (D + 2) * sizeof(float);
	return a > b ? a : b;
}
template <int D, bool SPLIT, int NQ>
constexpr size_t at_smem() { return (size_t)(SPLIT ? 2 : 1) * 8 * NQ * D * 2 + at_ring<D>(); }

__device__ __forceinline__ void cp4(void* dst, const void* src, bool there) {
	asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint2 b) {
	asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
	             : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
	             : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
}
__device__ __forceinline__ uint32_t pack_f16(float x, float y) {
	const __half2 h = __floats2half2_rn(x, y);
	return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_rest(float x, float y, uint32_t hi) { // what rounding to `hi` left
	const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
	return pack_f16(x - h.x, y - h.y);
}
// 16-byte piece of a row of codes that is stored at place `piece` of row r: rows read together meet different banks
template <int D>
__device__ __forceinline__ int at_place(int r, int piece) { return piece ^ (D == 64 ? (r >> 1) & 3 : r & 7); }
// Queries times 2^-exponent stand at 2^AT_LIFT or less.  What is not finite does not count: it spoils its own row and no other.
__device__ __forceinline__ uint32_t at_size(float x) { // |x| as bits, which are in the order of the values
	const uint32_t a = __float_as_uint(x) & 0x7fffffff;
	return a < 0x7f800000 ? a : 0;
}
__device__ __forceinline__ int at_exponent(uint32_t top) { return top ? min(max((int)(top >> 23) - 126, -85), 115) - AT_LIFT : AT_NO_ROW; } // top = m 2^(result + AT_LIFT)
__device__ __forceinline__ float at_factor(int e) { return pow2f(e >> 1) * pow2f(e - (e >> 1)); } // 2^e, -200 <= e <= 0: under 2^-149 zero

// the positions that a tile of rows sees, in order: [0, kept), then [lo, last]
struct AtSpan {
	int first, last, lo, kept, total, chunks;
};
__device__ __forceinline__ int at_low(const Attend& a, int pos) {
	int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
	return a.chunk > 0 ? max(lo, pos / a.chunk * a.chunk) : lo;
}
__device__ __forceinline__ AtSpan at_span(const Attend& a, int p0, int row0, int rows, int reach) {
	AtSpan s;
	s.first = p0 + row0 / a.group, s.last = p0 + (row0 + rows - 1) / a.group;
	s.lo = at_low(a, s.first), s.kept = min(min(a.keep_first, s.lo), reach);
	s.total = s.kept + max(min(s.last, reach - 1) - s.lo + 1, 0); // (no walk over positions that the table does not have)
	s.chunks = (s.total + AT_KEYS - 1) / AT_KEYS;
	return s;
}
__device__ __forceinline__ void at_finish(const Attend& a, int token, int head, int d, float v) {
	if (a.gate) v *= 1.f / (1.f + expf(-a.gate[token * a.gate_row + head * a.gate_head + d * a.gate_dim]));
	store_f32(a.out, a.out_type, token * a.o_row + head * a.o_head + d, v);
}

template <int D, bool SPLIT, int NQ>
__global__ void __launch_bounds__(32 * AT_WARPS, NQ * D <= 128 ? 4 : NQ * D <= 256 ? 3 : 2) k_c8_attend(const C8 c, const Attend a) {
	constexpr bool KEEP = D * NQ * (SPLIT ? 2 : 1) <= 128; // the queries' fragments stay in registers
	constexpr bool OWN_LATE = SPLIT && D * NQ > 256; // rows' own factors a key at a time: 129 us for 138 where registers are all in use, else all at once (soft-capped prompts 97 for 101)
	constexpr int KS = D / 16, MT = D / 16, PIECES = D / 16;
	constexpr int FS = D == 256 ? 52 : 20, LD = 8 * FS + 4; // sums in shared memory: eight parts of a row FS apart, rows LD: 16-byte stores of eight lanes meet different banks
	extern __shared__ __align__(128) unsigned char at_sm[];
	uint2* const qf = reinterpret_cast<uint2*>(at_sm); // B fragments [KS][NQ][32], then the remainders'
	AtStage<D>* const ring = reinterpret_cast<AtStage<D>*>(at_sm + (size_t)(SPLIT ? 2 : 1) * 8 * NQ * D * 2);
	__shared__ float fold_m[AT_WARPS][8 * NQ], fold_l[AT_WARPS][8 * NQ], qown[8 * NQ];
	__shared__ uint32_t qsize[8 * NQ];
	const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
	const int b = blockIdx.z, n = c.count[b], p0 = c.pos0[b], start = c.start[b], slot = c.slot[b], tile = blockIdx.x;
	const int kvh = blockIdx.y / a.shares, share = blockIdx.y - kvh * a.shares;
	if (n < 1 || p0 < 0 || p0 > INT_MAX - n || start < 0 || n > a.rows - start || (long long)tile * (8 * NQ) >= (long long)n * a.group) return;
	const int row0 = tile * (8 * NQ), rows = (int)min((long long)(8 * NQ), (long long)n * a.group - row0);
	const AtSpan sp = at_span(a, p0, row0, rows, c.reach(slot));
	const int lo = sp.lo, kept = sp.kept, total = sp.total;
	const int begin = min(sp.chunks, share * a.each), end = share == a.shares - 1 ? sp.chunks : min(sp.chunks, begin + a.each); // (more keys than were planned for: the last share's)
	if (share > 0 && begin >= sp.chunks && !a.cluster) return; // (a cluster stays together)
	const int H = c.heads, dim = c.dim;

	auto position = [&](int j) { return j < kept ? j : lo + (j - kept); };
	// The page of this lane's key, as the table has it: a load that nothing waits for here, looked at a chunk later (page_ok: whether there was one to look for).
	bool page_ok = false;
	auto page_of = [&](int chunk) {
		const int j = chunk * AT_KEYS + lane, at = page_index(c, position(min(j, max(total - 1, 0))));
		page_ok = chunk < end && j < total && at < c.table_pages;
		return total > 0 ? __ldg(c.table + (size_t)slot * c.table_pages + min(at, c.table_pages - 1)) : 0;
	};
	AtStage<D>& s = ring[warp];
	int next = begin + warp, next_page = page_of(next), next_row = 0; // the chunk to request, the page and the row of this lane's key
	uint32_t next_seen = 0;
	const int piece = lane % PIECES, prow = lane / PIECES; // which piece of which row of a group of 32 pieces this lane copies
	uint32_t swizzle[2];                                   // where, for even and odd groups (rows of 128 bytes)
#pragma unroll
	for (int i = 0; i < 2; ++i) swizzle[i] = at_place<D>(prow + i * 4, piece) * 16;
	auto copy = [&](uint8_t* to, const uint8_t* from) { // the next chunk's keys or values
		const uint32_t dst = smem_u32(to) + prow * D;
		const uint8_t* const src = from + piece * 16;
		if (next_seen == 0xffffffffu && dim == D) {
#pragma unroll
			for (int i = 0; i < PIECES; ++i) { // 32 rows of PIECES pieces, 32 pieces at a time
				const long long o = (long long)__shfl_sync(0xffffffffu, next_row, i * (32 / PIECES) + prow) * D;
				cp16(dst + i * (32 / PIECES) * D + (D == 128 ? swizzle[i & 1] : at_place<D>(i * (32 / PIECES) + prow, piece) * 16), src + o);
			}
		} else {
#pragma unroll
			for (int i = 0; i < PIECES; ++i) {
				const int r = i * (32 / PIECES) + prow;
				const long long o = (long long)__shfl_sync(0xffffffffu, next_row, r) * dim;
				const bool there = (next_seen >> r & 1) && piece * 16 < dim;
				cp16(dst + i * (32 / PIECES) * D + at_place<D>(r, piece) * 16, there ? src + o : from, there);
			}
		}
	};
	auto request_keys = [&](int half) { // and both scales, in this half of their arrays
		if (next < end) {
			const int id = page_ok && (unsigned)next_page < (unsigned)c.pages ? next_page : -1, unit = max(id, 0) * H + kvh;
			next_seen = __ballot_sync(0xffffffffu, id >= 0);
			next_row = unit * c.page + page_row(c, position(min(next * AT_KEYS + lane, total - 1))); // (rows of a pool: under 2^31)
			if (lane == 0) s.seen[half] = next_seen;
			cp4(s.ks[half] + lane, c.ks + unit, id >= 0), cp4(s.vs[half] + lane, c.vs + unit, id >= 0);
			copy(s.k, c.k);
		}
		asm volatile("cp.async.commit_group;" ::: "memory");
	};
	auto request_values = [&]() { // of the chunk whose keys were requested last
		if (next < end) {
			copy(s.v, c.v);
			next += AT_WARPS, next_page = page_of(next);
		}
		asm volatile("cp.async.commit_group;" ::: "memory");
	};
	request_keys(0), request_values();

	// Queries as B fragments, times a power of two that is the tile's, or a row's own: k index 2t + {0, 1}, 2t + 8 + {0, 1} of step s is channel t * D / 4 + 4 s + {0, 1}, {2, 3} (so that a
	// thread's codes of a key lie side by side).
	float x[2 * NQ][D / 32];
#pragma unroll
	for (int i = 0; i < 2 * NQ; ++i) {
		const int r = i * AT_WARPS + warp, rr = row0 + min(r, rows - 1);
		const long long at = (long long)(start + rr / a.group) * a.q_row + (long long)(kvh * a.group + rr % a.group) * a.q_head;
		uint32_t top = 0;
#pragma unroll
		for (int k = 0; k < D / 32; ++k) {
			const int d = k * 32 + lane;
			x[i][k] = r < rows && d < dim ? load_as_f32(a.q, a.q_type, at + d) : 0.f;
			top = max(top, at_size(x[i][k]));
		}
		top = __reduce_max_sync(0xffffffffu, top);
		if (lane == 0) qsize[r] = top;
	}
	__syncthreads();
	const int row_e = at_exponent(qsize[lane % (8 * NQ)]), tile_e = __reduce_max_sync(0xffffffffu, row_e), qe = tile_e == AT_NO_ROW ? 0 : tile_e;
	const bool alike = __all_sync(0xffffffffu, row_e == AT_NO_ROW || row_e >= qe - AT_ALIKE);
	if (tid < 8 * NQ) qown[tid] = row_e == AT_NO_ROW ? 1.f : at_factor(row_e - qe);
#pragma unroll
	for (int i = 0; i < 2 * NQ; ++i) {
		const int r = i * AT_WARPS + warp, own = __shfl_sync(0xffffffffu, row_e, r);
		const float qdown = pow2f(-(alike || own == AT_NO_ROW ? qe : own));
#pragma unroll
		for (int k = 0; k < D / 32; ++k) {
			const int d = k * 32 + lane, dt = d / (D / 4), ds = d % (D / 4) / 4, de = d & 3;
			const int at = (((ds * NQ + (r >> 3)) * 32 + (r & 7) * 4 + dt) * 2 + (de >> 1)) * 2 + (de & 1);
			const float y = x[i][k] * qdown;
			const __half hi = __float2half_rn(y);
			reinterpret_cast<__half*>(qf)[at] = hi;
			if (SPLIT) reinterpret_cast<__half*>(qf + KS * NQ * 32)[at] = __float2half_rn(y - __half2float(hi));
		}
	}
	__syncthreads();
	const bool extra = a.softcap > 0.f || a.slopes || !alike;
	const float qscale = a.scale * pow2f(qe) * (extra ? 1.f : AT_LOG2E);
	uint2 qr[KEEP ? (SPLIT ? 2 : 1) * KS * NQ : 1];
	if (KEEP) {
#pragma unroll
		for (int i = 0; i < (SPLIT ? 2 : 1) * KS * NQ; ++i) qr[i] = qf[i * 32 + lane];
	}
	auto qfrag = [&](int i) { return KEEP ? qr[i] : qf[i * 32 + lane]; };

	float acc[MT][NQ][4], m[NQ][2], l[NQ][2]; // queries 2t and 2t + 1 of each eight; m: the reference r
	int rpos[NQ][2];
#pragma unroll
	for (int q = 0; q < NQ; ++q) {
#pragma unroll
		for (int i = 0; i < MT; ++i) acc[i][q][0] = acc[i][q][1] = acc[i][q][2] = acc[i][q][3] = 0.f;
#pragma unroll
		for (int e = 0; e < 2; ++e) {
			const int r = 8 * q + 2 * t + e;
			m[q][e] = -INFINITY, l[q][e] = 0.f, rpos[q][e] = r < rows ? p0 + (row0 + r) / a.group : -1;
		}
	}
	const int wide = at_low(a, sp.last); // from here on, and up to `first`, every row sees every key

	int half = 0;
	for (int chunk = begin + warp; chunk < end; chunk += AT_WARPS, half ^= 1) {
		asm volatile("cp.async.wait_group 1;" ::: "memory"); // the keys; the values are the group behind them
		__syncwarp();
		// scores: rows g and g + 8 of product i are keys 16 i + g, + 8
		float z[2][NQ][4];
#pragma unroll
		for (int i = 0; i < 2; ++i) {
#pragma unroll
			for (int q = 0; q < NQ; ++q) z[i][q][0] = z[i][q][1] = z[i][q][2] = z[i][q][3] = 0.f;
#pragma unroll
			for (int k = 0; k < (KS + 3) / 4; ++k) {
				const int r = 16 * i + g;
				const uint4 u = *reinterpret_cast<const uint4*>(s.k + (r * PIECES + at_place<D>(r, t * (PIECES / 4) + k)) * 16);
				const uint4 w = *reinterpret_cast<const uint4*>(s.k + ((r + 8) * PIECES + at_place<D>(r + 8, t * (PIECES / 4) + k)) * 16);
				const uint32_t us[4] = {u.x, u.y, u.z, u.w}, ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
				for (int f = 0; f < 4; ++f) {
					uint32_t A[4];
					e4m3x4_to_f16(us[f], A[0], A[2]), e4m3x4_to_f16(ws[f], A[1], A[3]);
#pragma unroll
					for (int q = 0; q < NQ; ++q) {
						mma_f16(z[i][q], A, qfrag((4 * k + f) * NQ + q));
						if (SPLIT) mma_f16(z[i][q], A, qfrag((KS + 4 * k + f) * NQ + q));
					}
				}
			}
		}
		// with the value's scale in the exponent; this thread's keys are 8 j + g
		__syncwarp(); // every lane has its keys
		request_keys(half ^ 1);
		const uint32_t seen = s.seen[half];
		const int j0 = chunk * AT_KEYS;
		const bool all = seen == 0xffffffffu && j0 >= kept && position(j0) >= wide && position(j0 + AT_KEYS - 1) <= sp.first;
		float over[4]; // 1 / value scale
		if (extra) { // a soft cap, slopes or rows with powers of two of their own
			if (!OWN_LATE && !alike)
#pragma unroll
				for (int i = 0; i < 2 * NQ; ++i) {
					const float f = qown[8 * (i >> 1) + 2 * t + (i & 1)];
					z[0][i >> 1][i & 1] *= f, z[0][i >> 1][2 + (i & 1)] *= f, z[1][i >> 1][i & 1] *= f, z[1][i >> 1][2 + (i & 1)] *= f;
				}
#pragma unroll 1
			for (int j = 0; j < 4; ++j) {
				const int kp = position(j0 + 8 * j + g);
				const float kf = s.ks[half][8 * j + g] * qscale;
#pragma unroll
				for (int q = 0; q < NQ; ++q)
#pragma unroll
					for (int e = 0; e < 2; ++e) {
						float y = (j & 2 ? (j & 1 ? z[1][q][2 + e] : z[1][q][e]) : (j & 1 ? z[0][q][2 + e] : z[0][q][e]));
						if (OWN_LATE && !alike) y *= qown[8 * q + 2 * t + e];
						y *= kf;
						if (a.softcap > 0.f) y = a.softcap * tanhf(y / a.softcap);
						if (a.slopes) y -= a.slopes[kvh * a.group + (row0 + min(8 * q + 2 * t + e, rows - 1)) % a.group] * (float)(rpos[q][e] - kp);
						y *= AT_LOG2E;
						if (j == 0) z[0][q][e] = y;
						else if (j == 1) z[0][q][2 + e] = y;
						else if (j == 2) z[1][q][e] = y;
						else z[1][q][2 + e] = y;
					}
			}
		}
#pragma unroll
		for (int j = 0; j < 4; ++j) {
			const float kf = extra ? 1.f : s.ks[half][8 * j + g] * qscale;
			const int ve = max((int)(__float_as_uint(s.vs[half][8 * j + g]) >> 23) - 127, -126);
			const float lv = (float)ve;
			over[j] = pow2f(-ve);
#pragma unroll
			for (int q = 0; q < NQ; ++q)
#pragma unroll
				for (int e = 0; e < 2; ++e) z[j >> 1][q][(j & 1) * 2 + e] = fmaf(z[j >> 1][q][(j & 1) * 2 + e], kf, lv);
		}
		if (!all) { // some row does not see some key
#pragma unroll
			for (int j = 0; j < 4; ++j) {
				const int kp = position(j0 + 8 * j + g);
				const bool there = seen >> (8 * j + g) & 1, early = kp < a.keep_first;
#pragma unroll
				for (int q = 0; q < NQ; ++q)
#pragma unroll
					for (int e = 0; e < 2; ++e)
						if (!(there && kp <= rpos[q][e] && (early || kp >= at_low(a, rpos[q][e])))) z[j >> 1][q][(j & 1) * 2 + e] = -INFINITY;
			}
		}
		bool move = false;
#pragma unroll
		for (int q = 0; q < NQ; ++q)
#pragma unroll
			for (int e = 0; e < 2; ++e) move |= fmaxf(fmaxf(z[0][q][e], z[0][q][2 + e]), fmaxf(z[1][q][e], z[1][q][2 + e])) > m[q][e] + AT_MOST;
		if (__any_sync(0xffffffffu, move)) { // references move
#pragma unroll
			for (int q = 0; q < NQ; ++q) {
				float f[2];
#pragma unroll
				for (int e = 0; e < 2; ++e) {
					float top = fmaxf(fmaxf(z[0][q][e], z[0][q][2 + e]), fmaxf(z[1][q][e], z[1][q][2 + e]));
#pragma unroll
					for (int o = 4; o < 32; o *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
					const float mn = top > m[q][e] + AT_MOST ? top - AT_SET : m[q][e];
					f[e] = m[q][e] == -INFINITY ? 0.f : ex2(m[q][e] - mn);
					m[q][e] = mn, l[q][e] *= f[e];
				}
#pragma unroll
				for (int i = 0; i < MT; ++i) acc[i][q][0] *= f[0], acc[i][q][1] *= f[1], acc[i][q][2] *= f[0], acc[i][q][3] *= f[1];
			}
		}
		// weights, from keys x queries to the B fragments of queries x keys
		uint2 ph[2][NQ], pl[2][SPLIT ? NQ : 1];
#pragma unroll
		for (int q = 0; q < NQ; ++q) {
			const float base[2] = {m[q][0] == -INFINITY ? 0.f : m[q][0], m[q][1] == -INFINITY ? 0.f : m[q][1]};
#pragma unroll
			for (int i = 0; i < 2; ++i) {
#pragma unroll
				for (int e = 0; e < 4; ++e) {
					z[i][q][e] = ex2(z[i][q][e] - base[e & 1]);
					l[q][e & 1] = fmaf(z[i][q][e], over[2 * i + (e >> 1)], l[q][e & 1]);
				}
				const uint32_t h0 = pack_f16(z[i][q][0], z[i][q][1]), h1 = pack_f16(z[i][q][2], z[i][q][3]);
				ph[i][q] = make_uint2(transposed(h0), transposed(h1));
				if (SPLIT) pl[i][q] = make_uint2(transposed(pack_rest(z[i][q][0], z[i][q][1], h0)), transposed(pack_rest(z[i][q][2], z[i][q][3], h1)));
			}
		}
		asm volatile("cp.async.wait_group 1;" ::: "memory"); // the values; the next keys are the group behind them
		__syncwarp();
		// values: k index 2t + {0, 1}, 2t + 8 + {0, 1} of step kk is key 16 kk + 2t + {0, 1}, + 8; rows g and g + 8 of product i are channels g * D / 8 + 2 i + {0, 1}
#pragma unroll
		for (int kk = 0; kk < 2; ++kk) {
			uint32_t y[4][D / 32]; // this thread's channels of its four keys
#pragma unroll
			for (int u = 0; u < 4; ++u) {
				const int r = 16 * kk + 2 * t + (u & 1) + (u >> 1) * 8;
				if constexpr (D == 64) {
					const uint2 w = *reinterpret_cast<const uint2*>(s.v + (r * PIECES + at_place<D>(r, g >> 1)) * 16 + (g & 1) * 8);
					y[u][0] = w.x, y[u][1] = w.y;
				} else {
#pragma unroll
					for (int i = 0; i < D / 128; ++i) {
						const uint4 w = *reinterpret_cast<const uint4*>(s.v + (r * PIECES + at_place<D>(r, g * (D / 128) + i)) * 16);
						y[u][4 * i] = w.x, y[u][4 * i + 1] = w.y, y[u][4 * i + 2] = w.z, y[u][4 * i + 3] = w.w;
					}
				}
			}
#pragma unroll
			for (int i = 0; i < MT; ++i) { // bytes 2 (i & 1), + 1 of word i / 2
				uint32_t A[4];
				e4m3x4_to_f16(__byte_perm(y[0][i >> 1], y[1][i >> 1], i & 1 ? 0x7362 : 0x5140), A[0], A[1]);
				e4m3x4_to_f16(__byte_perm(y[2][i >> 1], y[3][i >> 1], i & 1 ? 0x7362 : 0x5140), A[2], A[3]);
#pragma unroll
				for (int q = 0; q < NQ; ++q) {
					mma_f16(acc[i][q], A, ph[kk][q]);
					if (SPLIT) mma_f16(acc[i][q], A, pl[kk][q]);
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

	// the warps' sums as one, eight rows at a time
	float* const sums = reinterpret_cast<float*>(ring); // [warps][8][LD]: channel d at d / (D / 8) * FS + d % (D / 8)
	float* const own = sums + AT_WARPS * 8 * LD;              // [16][D + 2]: what this share of a cluster found
	const bool whole = sp.chunks <= a.each || a.shares == 1; // no other share has keys
	if (whole && share > 0) return;                          // (nor does any of the cluster wait)
#pragma unroll
	for (int q = 0; q < NQ; ++q) {
		if (8 * q >= rows) break;
		__syncthreads();
#pragma unroll
		for (int e = 0; e < 2; ++e) {
			float* const to = sums + (warp * 8 + 2 * t + e) * LD + g * FS;
#pragma unroll
			for (int i = 0; i < MT; i += 2) *reinterpret_cast<float4*>(to + 2 * i) = make_float4(acc[i][q][e], acc[i][q][2 + e], acc[i + 1][q][e], acc[i + 1][q][2 + e]);
		}
		__syncthreads();
		for (int rr = warp; rr < min(8, rows - 8 * q); rr += AT_WARPS) {
			const int r = 8 * q + rr;
			float mx = fold_m[0][r], den = 0.f, wt[AT_WARPS];
#pragma unroll
			for (int w = 1; w < AT_WARPS; ++w) mx = fmaxf(mx, fold_m[w][r]);
#pragma unroll
			for (int w = 0; w < AT_WARPS; ++w) wt[w] = fold_m[w][r] == -INFINITY ? 0.f : ex2(fold_m[w][r] - mx), den = fmaf(wt[w], fold_l[w][r], den);
			const int token = start + (row0 + r) / a.group, head = kvh * a.group + (row0 + r) % a.group;
			float* const part = whole ? nullptr : a.cluster ? own + r * (D + 2) : a.part + (((size_t)token * a.heads + head) * a.shares + share) * (dim + 2);
			float norm = 0.f;
			if (whole) {
				if (a.sinks) { // one more term of the denominator
					const float sk = a.sinks[head] * AT_LOG2E, mn = fmaxf(mx, sk), down = mx == -INFINITY ? 0.f : ex2(mx - mn);
					den = den * down + at_sink(sk, mn), norm = down;
				} else norm = 1.f;
				norm = den > 0.f ? norm / den : den == 0.f ? 0.f : den; // (a NaN stays one)
			} else if (lane == 0) part[dim] = mx, part[dim + 1] = den;
			for (int d = lane; d < dim; d += 32) {
				float v = 0.f;
#pragma unroll
				for (int w = 0; w < AT_WARPS; ++w) v = fmaf(wt[w], sums[(w * 8 + rr) * LD + d / (D / 8) * FS + d % (D / 8)], v);
				if (whole) at_finish(a, token, head, d, v * norm);
				else part[d] = v;
			}
		}
	}
	if (whole || !a.cluster) return;
	// A cluster's shares: each CTA finishes its part of the outputs from all of them.
	__shared__ float wz[AT_CLUSTER][AT_TILE], inv[AT_TILE];
	const int shares = min(a.shares, (sp.chunks + a.each - 1) / a.each);
	cluster_sync();
	if (tid < rows) {
		const int head = kvh * a.group + (row0 + tid) % a.group;
		const float sk = a.sinks ? a.sinks[head] * AT_LOG2E : -INFINITY;
		float ms[AT_CLUSTER], ls[AT_CLUSTER], mx = sk, den = 0.f;
#pragma unroll
		for (int k = 0; k < AT_CLUSTER; ++k) {
			ms[k] = -INFINITY, ls[k] = 0.f;
			if (k < shares) ms[k] = cluster_load_f32(cluster_addr(own + tid * (D + 2) + dim, k)), ls[k] = cluster_load_f32(cluster_addr(own + tid * (D + 2) + dim + 1, k));
		}
#pragma unroll
		for (int k = 0; k < AT_CLUSTER; ++k) mx = fmaxf(mx, ms[k]);
#pragma unroll
		for (int k = 0; k < AT_CLUSTER; ++k)
			if (k < shares) {
				const float f = ms[k] == -INFINITY ? 0.f : ex2(ms[k] - mx);
				wz[k][tid] = f, den = fmaf(f, ls[k], den);
			}
		if (a.sinks) den += at_sink(sk, mx);
		inv[tid] = den > 0.f ? 1.f / den : den; // (0: nothing was seen)
	}
	__syncthreads();
	const int all = rows * dim, from = (int)((long long)all * share / a.shares), to = (int)((long long)all * (share + 1) / a.shares);
	for (int e = from + tid; e < to; e += 32 * AT_WARPS) {
		const int r = e / dim, d = e - r * dim;
		float v = 0.f;
#pragma unroll 8
		for (int k = 0; k < shares; ++k) v = fmaf(cluster_load_f32(cluster_addr(own + r * (D + 2) + d, k)), wz[k][r], v);
		at_finish(a, start + (row0 + r) / a.group, kvh * a.group + (row0 + r) % a.group, d, v * inv[r]);
	}
	cluster_sync(); // no CTA leaves while another reads what it found
}

// ---------------------------------------------------------------- attention of prompts
// Where a sequence brings many rows, the products run on the fifth-generation tensor cores: a CTA takes two groups of 128 rows (pairs of token and head, as above; one group where
// queries are pairs) of one key head and walks tiles of 64 keys.  Four warps a group read codes, a tile ahead, and lay them out in fp16 as the products' operands (keys as they are,
// values transposed), once for both groups; one thread issues S = Q K^T of the next tile and O += P V of this one; four warps a group, a row a thread, take S from tensor memory, form
// the weights (exponents, references and denominators as above) and write them back where the scores stood: the next product's operand.  O stays in tensor memory; it is rescaled
// in the rare case that a row's reference moves.
//   warps, in fours: softmax and output of each group; keys and values; a warp for the products
// 1500 and 805 queries of 16 heads behind 700 and 376 keys of 128 channels, 148 CTAs: 78 us (one group a CTA and two CTAs an SM 86, with the weights through shared memory 95).  Bound: the longest CTA, which
// walks 35 tiles where the mean is 19.8, and the way of a tile
// through its roles, about 3900 cycles, of which a softmax warp works 3000 (its exponentials keep the units busy for 1024 of them, the tensor cores are for about 1300); registers
// hold 17 warps.  Not better: values freed apart from keys 93, loads two tiles ahead 84, four warps for keys and values 75 (92 with a cold L2 for 86).
constexpr int AP_KEYS = 64, C8_NONE = -1000;
// Value scales that go through the products together lie within 2^AP_NEAR; a tile whose scales lie further apart comes several times, each time with the keys of one such range.  Codes
// stay exact in units of the largest scale.  Where a row may not see the key that has it, the row's weights would stand as many bits lower as the tile's scales lie apart: references
// are set that much lower there (AT_SET + AP_NEAR is still under AT_MOST).  So what is rounded as a subnormal is 2^-35 of the largest weight times the largest scale that the row sees.
constexpr int AP_NEAR = 4;
static_assert(AP_NEAR < 8 && AT_SET + AP_NEAR < AT_MOST, "three bits; references that are set do not move at once");
constexpr int ap_groups(bool split) { return split ? 1 : 2; } // of 128 rows
constexpr int ap_threads(bool split) { return 256 * ap_groups(split) + 32; }
__device__ __forceinline__ uint32_t mul_f16(uint32_t x, uint32_t y) {
	const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&y));
	return *reinterpret_cast<const uint32_t*>(&r);
}
template <int D, bool SPLIT>
struct ApShared { // tiles of rows of 128 bytes, 16-byte pieces swizzled by the row
	static constexpr int PANELS = D / 64, PAIR = SPLIT ? 2 : 1, GROUPS = ap_groups(SPLIT), STAGES = 2 + (GROUPS > 1);
	unsigned char q[GROUPS][PAIR][PANELS][128 * 128];
	unsigned char k[STAGES][PANELS][AP_KEYS * 128];
	unsigned char v[STAGES][D * 128];
	float factor[STAGES][AP_KEYS]; // of a tile's keys on their scores, in log2
	int units[STAGES]; // 8 times log2 of the largest of the tile's value scales, in units of which its values come, plus that many bits that they lie apart (one number: a register)
	uint32_t seen[STAGES][2];      // keys that are there
	int tile[STAGES], last[STAGES]; // which 64 keys; whether nothing comes behind them
	uint64_t kv_full[STAGES], kv_empty[STAGES], s_full[GROUPS][2], p_full[GROUPS], p_empty[GROUPS], done;
	uint32_t tmem;
	int tops[4 * GROUPS], least[4 * GROUPS]; // exponents of the queries: the largest and the smallest row of a warp's
	int lost;
};
// eight neighbours as floats
__device__ __forceinline__ void load8(const void* p, int type, long long i, bool vec, float (&x)[8]) {
	if (!vec) {
#pragma unroll
		for (int k = 0; k < 8; ++k) x[k] = load_as_f32(p, type, i + k);
	} else if (type == SEQ_F32) {
		const float4 u = *reinterpret_cast<const float4*>((const float*)p + i), w = *reinterpret_cast<const float4*>((const float*)p + i + 4);
		x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = w.x, x[5] = w.y, x[6] = w.z, x[7] = w.w;
	} else {
		const uint4 w = *reinterpret_cast<const uint4*>((const uint16_t*)p + i);
		if (type == SEQ_BF16) unpack16<bf16>(w, x);
		else unpack16<__half>(w, x);
	}
}
template <int N>
__device__ __forceinline__ int ap_tile_exponent(const int (&tops)[N]) {
	int e = tops[0];
#pragma unroll
	for (int i = 1; i < N; ++i) e = max(e, tops[i]);
	return e == AT_NO_ROW ? 0 : e;
}
template <int N>
__device__ __forceinline__ bool ap_alike(const int (&least)[N], int tile_e) {
	int e = least[0];
#pragma unroll
	for (int i = 1; i < N; ++i) e = min(e, least[i]);
	return e >= tile_e - AT_ALIKE;
}
template <int D, bool SPLIT>
__global__ void __launch_bounds__(ap_threads(SPLIT), 1) k_c8_prompt(const C8 c, const Attend a) {
	typedef ApShared<D, SPLIT> Shared;
	constexpr int PANELS = Shared::PANELS, PIECES = D / 16, GROUPS = Shared::GROUPS, STAGES = Shared::STAGES, WARPS = 4 * GROUPS, ROWS = 128 * GROUPS; // WARPS: of the softmax, and as many of the codes
	constexpr uint32_t S_COLS = 64 * GROUPS, O_COL = 2 * S_COLS;
	extern __shared__ __align__(1024) unsigned char ap_raw[]; // (all of the kernel's shared memory: it starts where the swizzle's pattern does)
	Shared& s = *reinterpret_cast<Shared*>(ap_raw);
	const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
	const int b = blockIdx.y, kvh = blockIdx.x, n = c.count[b], p0 = c.pos0[b], start = c.start[b], slot = c.slot[b];
	const int tile = (int)min((long long)gridDim.z, ((long long)n * a.group + ROWS - 1) / ROWS) - 1 - (int)blockIdx.z; // (every sequence's longest rows first)
	if (tile < 0 || n < 1 || p0 < 0 || p0 > INT_MAX - n || start < 0 || n > a.rows - start || (long long)tile * ROWS >= (long long)n * a.group) return;
	const int row0 = tile * ROWS, rows = (int)min((long long)ROWS, (long long)n * a.group - row0);
	const AtSpan sp = at_span(a, p0, row0, rows, c.reach(slot));
	const int tiles = (sp.total + AP_KEYS - 1) / AP_KEYS;
	auto position = [&](int j) { return j < sp.kept ? j : sp.lo + (j - sp.kept); };

	const int groups = rows > 128 ? GROUPS : 1;
	if (warp == 2 * WARPS) tmem_alloc(&s.tmem, 256 * GROUPS);
	if (tid == 0) {
		for (int i = 0; i < STAGES; ++i) mbar_init(s.kv_full + i, WARPS), mbar_init(s.kv_empty + i, 1); // (a warp arrives as one)
		for (int g = 0; g < GROUPS; ++g) mbar_init(s.s_full[g], 1), mbar_init(s.s_full[g] + 1, 1), mbar_init(s.p_full + g, 4), mbar_init(s.p_empty + g, 1);
		mbar_init(&s.done, 1);
		s.lost = 0;
		mbar_init_fence();
	}
	// queries, times the tile's power of two, or the row's own
	int row_e = 0;
	const int token = start + (row0 + min(tid, rows - 1)) / a.group, head = kvh * a.group + (row0 + min(tid, rows - 1)) % a.group;
	if (warp < WARPS) {
		const long long at = token * a.q_row + head * a.q_head;
		const int bytes = a.q_type == SEQ_F32 ? 4 : 2;
		const bool vec = ((uintptr_t)a.q | (uintptr_t)(a.q_row * bytes) | (uintptr_t)(a.q_head * bytes)) % 16 == 0;
		float x[8];
		uint32_t top = 0;
#pragma unroll 4
		for (int piece = 0; piece < D / 8; ++piece) {
			load8(a.q, a.q_type, at + piece * 8, vec, x);
#pragma unroll
			for (int i = 0; i < 8; ++i) top = max(top, at_size(x[i]));
		}
		row_e = at_exponent(top); // (a thread's own row; behind the last one that once more)
		const int most = __reduce_max_sync(0xffffffffu, row_e), least = __reduce_min_sync(0xffffffffu, row_e == AT_NO_ROW ? -AT_NO_ROW : row_e);
		if (lane == 0) s.tops[warp] = most, s.least[warp] = least;
		asm volatile("bar.sync 1, %0;" ::"n"(32 * WARPS) : "memory");
		const int tile_e = ap_tile_exponent(s.tops);
		if (row_e == AT_NO_ROW || ap_alike(s.least, tile_e)) row_e = tile_e;
		const float down = tid < rows ? pow2f(-row_e) : 0.f;
#pragma unroll 2
		for (int piece = 0; piece < D / 8; ++piece) {
			load8(a.q, a.q_type, at + piece * 8, vec, x);
			uint32_t hi[4], rest[4];
#pragma unroll
			for (int i = 0; i < 4; ++i) hi[i] = pack_f16(x[2 * i] * down, x[2 * i + 1] * down), rest[i] = SPLIT ? pack_rest(x[2 * i] * down, x[2 * i + 1] * down, hi[i]) : 0;
			const int place = (tid & 127) * 128 + (((piece & 7) ^ (tid & 7)) << 4);
			*reinterpret_cast<uint4*>(s.q[tid >> 7][0][piece >> 3] + place) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
			if (SPLIT) *reinterpret_cast<uint4*>(s.q[tid >> 7][Shared::PAIR - 1][piece >> 3] + place) = make_uint4(rest[0], rest[1], rest[2], rest[3]);
		}
		fence_async_smem();
	}
	tc_fence_before();
	__syncthreads();
	tc_fence_after();
	const uint32_t tmem = s.tmem; // scores of even tiles, a group's 64 columns beside another's, of odd ones, sums: 128 columns a group
	const int tile_e = ap_tile_exponent(s.tops);
	const float qscale = a.scale * pow2f(tile_e) * AT_LOG2E;
	float m = -INFINITY, l = 0.f;

	// registers go from the warps of keys and values to those of the softmax: 8 x 112 + 8 x 80 + 96 = 17 x 96, what the block was launched with
	if (warp < WARPS) {
		if (!SPLIT) asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
		const int group = warp / 4;
		const int rpos = tid < rows ? p0 + (row0 + tid) / a.group : -1, rlow = tid < rows ? at_low(a, rpos) : 0, wide = at_low(a, sp.last);
		const uint32_t lanes = tmem + ((uint32_t)(warp % 4 * 32) << 16), sums_at = lanes + O_COL + 128 * group;
		const float own = ap_alike(s.least, tile_e) ? 1.f : at_factor(row_e - tile_e);
		int st = 0, i = 0;
		uint32_t round = 0;
		for (bool last = tiles == 0 || group >= groups; !last; ++i) {
			const uint32_t scores_at = lanes + (i & 1) * S_COLS + 64 * group;
			if (!ap_wait_warp(s.kv_full + st, round, &s.lost) || !ap_wait_warp(s.s_full[group] + (i & 1), (i >> 1) & 1, &s.lost)) break; // (the factors; the scores)
			tc_fence_after();
			const int j0 = s.tile[st] * AP_KEYS;
			last = s.last[st];
			const uint32_t seen[2] = {s.seen[st][0], s.seen[st][1]};
			const bool all = (seen[0] & seen[1]) == 0xffffffffu && j0 >= sp.kept && position(j0) >= wide && position(j0 + AP_KEYS - 1) <= sp.first;
			const int units = s.units[st];
			const float base = m == -INFINITY ? 0.f : m, most = m == -INFINITY ? -INFINITY : AT_MOST;
			float z[64], top = -INFINITY; // log2 of the weights against the reference as it stands (against 0 before there is one)
			tmem_ld32(scores_at, *reinterpret_cast<float(*)[32]>(z));
			tmem_ld32(scores_at + 32, *reinterpret_cast<float(*)[32]>(z + 32));
			if (own != 1.f) { // a row with a power of two of its own
#pragma unroll
				for (int k = 0; k < 64; k += 2) {
					const float2 x = halves(mul2(pair_of(z[k], z[k + 1]), pair_of(own, own)));
					z[k] = x.x, z[k + 1] = x.y;
				}
			}
			const float lift = (float)(units >> 3) - base;
			const u64 off = pair_of(lift, lift);
#pragma unroll
			for (int k = 0; k < 64; k += 4) {
				const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(s.factor[st] + k);
				const float2 x = halves(fma2(pair_of(z[k], z[k + 1]), f.x, off)), y = halves(fma2(pair_of(z[k + 2], z[k + 3]), f.y, off));
				z[k] = x.x, z[k + 1] = x.y, z[k + 2] = y.x, z[k + 3] = y.y;
			}
			if (!all) {
#pragma unroll
				for (int k = 0; k < 64; ++k) {
					const int kp = position(j0 + k);
					if (!((seen[k / 32] >> (k & 31) & 1) && kp <= rpos && (kp >= rlow || kp < a.keep_first))) z[k] = -INFINITY;
				}
			}
			float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
			for (int k = 0; k < 64; k += 2) tops[k / 2 % 4] = fmaxf(fmaxf(tops[k / 2 % 4], z[k]), z[k + 1]);
			top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
			if (__any_sync(0xffffffffu, top > most)) { // references move
				const float set = all ? AT_SET : AT_SET + (float)(units & 7), mn = top > most ? base + top - set : m, f = m == -INFINITY ? 0.f : ex2(m - mn), by = base - (mn == -INFINITY ? 0.f : mn);
#pragma unroll
				for (int k = 0; k < 64; ++k) z[k] += by;
				m = mn, l *= f;
				if (i > 0) { // there are sums
					if (!ap_wait_warp(s.p_empty + group, (i - 1) & 1, &s.lost)) break;
					tc_fence_after();
#pragma unroll 1
					for (int col = 0; col < D; col += 8) tmem_scale8(sums_at + col, f);
					tmem_st_wait();
				}
			}
			u64 sum = 0;
			uint32_t hi[32], rest[32];
#pragma unroll
			for (int k = 0; k < 64; k += 2) {
				const float w0 = ex2(z[k]), w1 = ex2(z[k + 1]);
				sum = add2(sum, pair_of(w0, w1));
				hi[k / 2] = pack_f16(w0, w1), rest[k / 2] = SPLIT ? pack_rest(w0, w1, hi[k / 2]) : 0;
			}
			tmem_st32(scores_at, hi); // where the scores were
			if (SPLIT) tmem_st32(scores_at + 32, rest);
			const float2 sums = halves(sum);
			l = fmaf(sums.x + sums.y, pow2f(-(units >> 3)), l); // the weights hold the value scale
			tmem_st_wait();
			if (i > 0 && !ap_wait_warp(s.p_empty + group, (i - 1) & 1, &s.lost)) break; // (long done: the barrier's phases stay in step)
			tc_fence_before();
			__syncwarp();
			if (lane == 0) mbar_arrive(s.p_full + group);
			if (++st == STAGES) st = 0, round ^= 1;
		}
		if (i > 0) ap_wait_warp(s.p_empty + group, (i - 1) & 1, &s.lost);
		tc_fence_after();
		float norm = 1.f;
		if (a.sinks && tid < rows) {
			const float sk = a.sinks[head] * AT_LOG2E, mn = fmaxf(m, sk), down = m == -INFINITY ? 0.f : ex2(m - mn);
			l = l * down + at_sink(sk, mn), norm = down;
		}
		norm = *(volatile int*)&s.lost ? NAN : l > 0.f ? norm / l : l == 0.f ? 0.f : l; // (0: nothing was seen; a NaN stays one)
		const bool wide_store = a.out_type != SEQ_F32 && !a.gate && ((uintptr_t)a.out | (uintptr_t)(a.o_row * 2) | (uintptr_t)(a.o_head * 2)) % 16 == 0;
#pragma unroll 1
		for (int col = 0; col < D && group < groups; col += 32) {
			float z[32];
			__syncwarp(); // (rows behind the last one take part in the load)
			if (tiles > 0) tmem_ld32(sums_at + col, z);
			else {
#pragma unroll
				for (int k = 0; k < 32; ++k) z[k] = 0.f;
			}
			if (tid < rows && wide_store) {
				uint4* to = reinterpret_cast<uint4*>((uint16_t*)a.out + token * a.o_row + head * a.o_head + col);
#pragma unroll
				for (int k = 0; k < 32; k += 8) {
					uint32_t w[4];
#pragma unroll
					for (int e = 0; e < 4; ++e) {
						const float x = z[k + 2 * e] * norm, y = z[k + 2 * e + 1] * norm;
						if (a.out_type == SEQ_BF16) {
							const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
							w[e] = *reinterpret_cast<const uint32_t*>(&h);
						} else w[e] = pack_f16(x, y);
					}
					to[k / 8] = make_uint4(w[0], w[1], w[2], w[3]);
				}
			} else if (tid < rows) {
#pragma unroll
				for (int k = 0; k < 32; ++k) at_finish(a, token, head, col + k, z[k] * norm);
			}
		}
	} else if (warp < 2 * WARPS) {
		if (!SPLIT) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
		// Every thread takes pieces of keys' rows (PIECES lanes read a row) and eight channels of VKEYS keys' values.
		constexpr int KROWS = 32 / PIECES, KEACH = AP_KEYS / (WARPS * KROWS), VKEYS = 8 / GROUPS, VGROUPS = AP_KEYS / VKEYS;
		const int t = tid - 32 * WARPS, own = warp - WARPS, vgroup = t % VGROUPS, dims = t / VGROUPS * 8;
		const bool works = dims < D;
		// Nothing below waits for a load where it asks for it: keys that are not there read row 0 of the pool and the table's last entry, and are sorted out a tile later.
		int ahead[2], exps[2];     // of keys lane and lane + 32: the pages of the tile to load next, as the table has them; the values' scales of the loaded one
		bool asked[2], have[2];    // whether there was a page to look for; whether the key is there
		float scale;               // of key t, the keys'
		uint4 kw[KEACH];
		uint2 vw[VKEYS];
		uint32_t mine = 0;         // this thread's values that are there
		auto look = [&](int i) {
#pragma unroll
			for (int h = 0; h < 2; ++h) {
				const int j = i * AP_KEYS + 32 * h + lane, at = page_index(c, position(min(j, sp.total - 1)));
				asked[h] = j < sp.total && at < c.table_pages;
				ahead[h] = __ldg(c.table + (size_t)slot * c.table_pages + min(at, c.table_pages - 1));
			}
		};
		auto load = [&](int i) {
			int row[2];
#pragma unroll
			for (int h = 0; h < 2; ++h) {
				have[h] = asked[h] && (unsigned)ahead[h] < (unsigned)c.pages;
				const int unit = (have[h] ? ahead[h] : 0) * c.heads + kvh;
				row[h] = have[h] ? unit * c.page + page_row(c, position(i * AP_KEYS + 32 * h + lane)) : -1; // (under 2^31)
				exps[h] = __float_as_int(__ldg(c.vs + unit));
				if (h == (own & 1)) scale = __ldg(c.ks + unit);
			}
#pragma unroll
			for (int k = 0; k < KEACH; ++k) {
				const int key = (k * WARPS + own) * KROWS + lane / PIECES, r = __shfl_sync(0xffffffffu, (k * WARPS + own) * KROWS < 32 ? row[0] : row[1], key & 31);
				kw[k] = ldg_stream(reinterpret_cast<const uint4*>(c.k + (long long)max(r, 0) * D) + lane % PIECES);
			}
			mine = 0;
#pragma unroll
			for (int k = 0; k < VKEYS; ++k) {
				const int key = vgroup * VKEYS + k, r0 = __shfl_sync(0xffffffffu, row[0], key & 31), r1 = __shfl_sync(0xffffffffu, row[1], key & 31), r = key < 32 ? r0 : r1;
				vw[k] = ldg_stream8(reinterpret_cast<const uint2*>(c.v + (long long)max(r, 0) * D + (works ? dims : 0)));
				mine |= (r >= 0 ? 1u : 0u) << k;
			}
			look(i + 1);
		};
		int st = 0;
		uint32_t round = 0;
		if (tiles > 0) look(0), load(0);
		for (int i = 0; i < tiles;) {
			if (!ap_wait_warp(s.kv_empty + st, round ^ 1, &s.lost)) break;
			if (t < AP_KEYS) s.factor[st][t] = (own == 0 ? have[0] : have[1]) ? scale * qscale : 0.f;
#pragma unroll
			for (int k = 0; k < KEACH; ++k) {
				const int key = (k * WARPS + own) * KROWS + lane / PIECES, piece = lane % PIECES;
				uint32_t w[8];
				e4m3x4_to_f16(kw[k].x, w[0], w[1]), e4m3x4_to_f16(kw[k].y, w[2], w[3]), e4m3x4_to_f16(kw[k].z, w[4], w[5]), e4m3x4_to_f16(kw[k].w, w[6], w[7]);
				unsigned char* const to = s.k[st][piece >> 2] + key * 128;
				const bool odd = piece & 4; // (lanes of the second panel store their second half first: eight lanes meet different banks)
				const uint4 lo = make_uint4(w[0], w[1], w[2], w[3]), hi = make_uint4(w[4], w[5], w[6], w[7]);
				const int at = (2 * piece & 7) ^ (key & 7);
				*reinterpret_cast<uint4*>(to + ((odd ? at ^ 1 : at) << 4)) = odd ? hi : lo;
				*reinterpret_cast<uint4*>(to + ((odd ? at : at ^ 1) << 4)) = odd ? lo : hi;
			}
			// values in units of the largest scale, a smaller one's shifted down, exactly; keys whose scales are far smaller are left for the next round
			int e[2];
#pragma unroll
			for (int h = 0; h < 2; ++h) e[h] = have[h] ? max((exps[h] >> 23 & 255) - 127, -126) : C8_NONE;
			int most = __reduce_max_sync(0xffffffffu, max(e[0], e[1]));
			if (most == C8_NONE) most = 0;
			const int least = __reduce_min_sync(0xffffffffu, min(e[0] == C8_NONE ? INT_MAX : e[0], e[1] == C8_NONE ? INT_MAX : e[1]));
			const bool even = least >= most, more = least < most - AP_NEAR;
			have[0] = have[0] && e[0] < most - AP_NEAR, have[1] = have[1] && e[1] < most - AP_NEAR;
			if (t < AP_KEYS) {
				const int own_e = own == 0 ? e[0] : e[1];
				const uint32_t seen = __ballot_sync(0xffffffffu, own_e >= most - AP_NEAR);
				if (lane == 0) s.seen[st][own] = seen;
			}
			if (t == 0) s.units[st] = most * 8 + (more ? AP_NEAR : even ? 0 : most - least), s.tile[st] = i, s.last[st] = i == tiles - 1 && !more;
			if (mine != (1u << VKEYS) - 1) { // (a code that is no number would spoil rows that do not see it)
#pragma unroll
				for (int k = 0; k < VKEYS; ++k)
					if (!(mine >> k & 1)) vw[k] = make_uint2(0, 0);
			}
			uint32_t down[VKEYS / 2]; // of the pairs of this thread's keys, as fp16
			if (!even) {
#pragma unroll
				for (int k = 0; k < VKEYS / 2; ++k) {
					float f[2];
#pragma unroll
					for (int u = 0; u < 2; ++u) {
						const int key = vgroup * VKEYS + 2 * k + u, e0 = __shfl_sync(0xffffffffu, e[0], key & 31), e1 = __shfl_sync(0xffffffffu, e[1], key & 31);
						f[u] = pow2f(max((key < 32 ? e0 : e1) - most, -126));
					}
					down[k] = pack_f16(f[0], f[1]);
				}
			}
			if (works) {
#pragma unroll
				for (int word = 0; word < 2; ++word)
#pragma unroll
					for (int u = 0; u < 2; ++u) { // channels dims + 4 word + 2 u, + 1
						uint32_t lo[VKEYS / 2], hi[VKEYS / 2];
#pragma unroll
						for (int k = 0; k < VKEYS / 2; ++k) {
							const uint32_t x = word ? vw[2 * k].y : vw[2 * k].x, y = word ? vw[2 * k + 1].y : vw[2 * k + 1].x;
							e4m3x4_to_f16(__byte_perm(x, y, u ? 0x7362 : 0x5140), lo[k], hi[k]);
							if (!even) lo[k] = mul_f16(lo[k], down[k]), hi[k] = mul_f16(hi[k], down[k]);
						}
						const int d = dims + 4 * word + 2 * u;
						auto put = [&](int d, const uint32_t (&w)[VKEYS / 2]) {
							unsigned char* const to = s.v[st] + d * 128 + (((vgroup * VKEYS / 8) ^ (d & 7)) << 4) + vgroup * VKEYS % 8 * 2;
							if constexpr (VKEYS == 8) *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
							else *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
						};
						put(d, lo), put(d + 1, hi);
					}
			}
			fence_async_smem();
			__syncwarp();
			if (lane == 0) mbar_arrive(s.kv_full + st);
			if (!more && ++i < tiles) load(i);
			if (++st == STAGES) st = 0, round ^= 1;
		}
	} else if (lane == 0) {
		constexpr uint32_t score = (1u << 4) | ((uint32_t)(AP_KEYS >> 3) << 17) | (8u << 24), value = (1u << 4) | ((uint32_t)(D >> 3) << 17) | (8u << 24); // 128 rows
		int st = 0, behind = 0; // stages of this tile's keys, of the values of the one before
		uint32_t round = 0;
		bool there = tiles > 0, last = false;
		for (int i = 0; there; ++i) {
			if (last) there = false; // the last tile's values are left
			else {
				if (!ap_wait(s.kv_full + st, round, &s.lost)) break; // (the scores' columns: the product of the tile before the last, which read weights there, was issued earlier)
				tc_fence_after();
				last = s.last[st];
				for (int g = 0; g < groups; ++g) {
#pragma unroll
					for (int h = 0; h < Shared::PAIR; ++h)
#pragma unroll
						for (int pn = 0; pn < PANELS; ++pn)
#pragma unroll
							for (int k = 0; k < 4; ++k)
								umma_f16(tmem + (i & 1) * S_COLS + 64 * g, umma_desc_sw128(s.q[g][h][pn]) + 2 * k, umma_desc_sw128(s.k[st][pn]) + 2 * k, score, (h | pn | k) ? 1u : 0u);
					umma_commit(s.s_full[g] + (i & 1));
				}
			}
			if (i > 0) {
				const int j = i - 1;
				for (int g = 0; g < groups; ++g) {
					if (!ap_wait(s.p_full + g, j & 1, &s.lost)) {
						there = false;
						break;
					}
					tc_fence_after();
#pragma unroll
					for (int h = 0; h < Shared::PAIR; ++h)
#pragma unroll
						for (int k = 0; k < 4; ++k)
							umma_f16_ts(tmem + O_COL + 128 * g, tmem + (j & 1) * S_COLS + 64 * g + 32 * h + 8 * k, umma_desc_sw128(s.v[behind]) + 2 * k, value, (j | h | k) ? 1u : 0u);
					umma_commit(s.p_empty + g);
				}
				umma_commit(s.kv_empty + behind);
			}
			behind = st;
			if (++st == STAGES) st = 0, round ^= 1;
		}
		umma_commit(&s.done); // nothing of this block's is left in the tensor core when its memory goes
		mbar_wait_bounded(&s.done, 0);
	}
	__syncwarp();
	tc_fence_before();
	__syncthreads();
	tc_fence_after();
	if (warp == 2 * WARPS) tmem_dealloc(tmem, 256 * GROUPS);
}

// Folds the shares of one (token, head), in share order: a warp for each, all of a lane's shares read at once.  9 us for 2048 rows of 6 shares: latency (the shares do not announce it early, so it starts when the last of them has ended).
__global__ void __launch_bounds__(128) k_c8_fold(const C8 c, const Attend a) {
	pdl_wait_prev();
	const int b = blockIdx.z, kvh = blockIdx.y, n = c.count[b], p0 = c.pos0[b], start = c.start[b], slot = c.slot[b], warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
	if (n < 1 || p0 < 0 || p0 > INT_MAX - n || start < 0 || n > a.rows - start) return;
	for (long long row = (long long)blockIdx.x * 4 + warp; row < (long long)n * a.group; row += gridDim.x * 4) {
		const int row0 = (int)(row / a.tile) * a.tile, rows = (int)min((long long)a.tile, (long long)n * a.group - row0);
		const int shares = min(a.shares, (at_span(a, p0, row0, rows, c.reach(slot)).chunks + a.each - 1) / a.each);
		if (shares <= 1) continue; // its one share has finished it
		const int token = start + (int)(row / a.group), head = kvh * a.group + (int)(row % a.group), stride = c.dim + 2;
		const float* p = a.part + ((size_t)token * a.heads + head) * a.shares * stride;
		const float sk = a.sinks ? a.sinks[head] * AT_LOG2E : -INFINITY;
		float m[AT_SHARES / 32], w[AT_SHARES / 32], mx = sk, den = 0.f; // this lane's shares
#pragma unroll
		for (int i = 0; i < AT_SHARES / 32; ++i) {
			const int s = i * 32 + lane;
			m[i] = s < shares ? p[(size_t)s * stride + c.dim] : -INFINITY, w[i] = s < shares ? p[(size_t)s * stride + c.dim + 1] : 0.f;
			mx = fmaxf(mx, m[i]);
		}
		mx = warp_max(mx);
#pragma unroll
		for (int i = 0; i < AT_SHARES / 32; ++i) {
			const float f = m[i] == -INFINITY ? 0.f : ex2(m[i] - mx);
			den = fmaf(f, w[i], den), w[i] = f;
		}
		den = warp_sum(den);
		if (a.sinks) den += at_sink(sk, mx);
		const float norm = den > 0.f ? 1.f / den : den; // (0: nothing was seen)
		for (int d0 = 0; d0 < c.dim; d0 += 128) {
			float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
			for (int i = 0; i < AT_SHARES / 32; ++i)
#pragma unroll 8
				for (int s = i * 32; s < min(shares, i * 32 + 32); ++s) {
					const float f = __shfl_sync(0xffffffffu, w[i], s & 31);
#pragma unroll
					for (int k = 0; k < 4; ++k) v[k] = fmaf(f, p[(size_t)s * stride + min(d0 + 32 * k + lane, c.dim - 1)], v[k]);
				}
#pragma unroll
			for (int k = 0; k < 4; ++k)
				if (d0 + 32 * k + lane < c.dim) at_finish(a, token, head, d0 + 32 * k + lane, v[k] * norm);
		}
	}
}

int check_cache(const char* what, const SeqCache8* q, const SeqPortions* p) {
	if (!q || !p) return refuse("%s: no cache or no batch", what);
	if (q->pages < 0 || q->heads < 1 || q->page < 1 || q->slots < 0 || q->table_pages < 0) return refuse("%s: a cache of %d pages, %d heads, %d tokens a page", what, q->pages, q->heads, q->page);
	if (q->heads > 4096 || q->page > 65536) return refuse("%s: at most 4096 heads and 65536 tokens a page", what);
	if ((long long)q->pages * q->heads * q->page > INT_MAX) return refuse("%s: a pool of %d pages, %d heads, %d tokens a page has more than 2^31 rows", what, q->pages, q->heads, q->page);
	if (q->dim < 16 || q->dim > 256 || q->dim % 16) return refuse("%s: rows of %d channels: a multiple of 16 up to 256 is served", what, q->dim);
	if (p->n < 0 || p->longest < 0 || p->n > 65535) return refuse("%s: %d sequences (at most 65535), longest %d", what, p->n, p->longest);
	if (p->n && (!p->start || !p->count || !p->slot || !p->pos0)) return refuse("%s: the batch's description is missing", what);
	if (q->pages && (!q->k || !q->v || !q->k_scale || !q->v_scale)) return refuse("%s: the cache has no memory", what);
	if (q->slots > 0 && q->table_pages > 0 && !q->table) return refuse("%s: the page table is missing", what);
	if (((uintptr_t)q->k | (uintptr_t)q->v) % 16) return refuse("%s: codes are not aligned to 16 bytes", what);
	if (((uintptr_t)q->table | (uintptr_t)p->start | (uintptr_t)p->count | (uintptr_t)p->slot | (uintptr_t)p->pos0) % 4) return refuse("%s: the page table or the batch's description is not aligned to 4 bytes", what);
	if (((uintptr_t)q->k_scale | (uintptr_t)q->v_scale) % 4) return refuse("%s: scales are not aligned to 4 bytes", what);
	return 0;
}
C8 describe(const SeqCache8& q, const SeqPortions& p) {
	int shift = 0;
	while (1 << shift < q.page) ++shift;
	return C8{(uint8_t*)q.k, (uint8_t*)q.v, q.k_scale, q.v_scale, q.table, q.pages, q.heads, q.page, q.dim, q.slots, q.table_pages, 1 << shift == q.page ? shift : -1, p.start, p.count, p.slot, p.pos0};
}
StoreRows store_rows(const SeqRows& r) {
	const int bytes = 4 * type_size(r.type);
	return StoreRows{r.p, r.row_stride, r.head_stride, r.rows, (uintptr_t)r.p % bytes == 0 && r.row_stride % 4 == 0 && r.head_stride % 4 == 0};
}

// How the work is cut: rows of a CTA; shares of a tile's keys and the chunks of each (sequences differ in length: shares of one length for all of them, short ones have fewer);
// whether a cluster folds the shares.
struct AtPlan {
	int tile, shares, each, cluster; // tile 128: the prompt kernel
};
constexpr int AT_ROOM = 148 * 3; // CTAs that run at a time
constexpr int AP_TILE = 128;     // stands for the prompt kernel
// 128s of rows from which on the prompt kernel is the faster one (us, and with the other).  Its time is that of a CTA's tiles one after another, whatever the channels; the other's
// work halves with them.  128 channels, 16 bits: 32 46 / 24, 64 42 / 44, 80 21 / 29 and 47 / 30, 100 35 / 41 and 93 / 107, 104 35 / 35, 128 40 / 60 and 31 / 36, 256 43 / 55, 376 76 / 167.
// 64 channels: 64 72 / 33, 128 26 / 18, 200 49 / 66, 224 30 / 33, 256 27 / 31 and 83 / 138.  fp32 (a group of rows a CTA): 80 43 / 34, 104 44 / 38, 128 52 / 67, 224 47 / 37 and
// 74 / 63, 384 52 / 76.
constexpr int ap_least(bool split, int dim) { return split ? 192 : dim > 64 ? 100 : 200; }
// Rows of a CTA: eight fill a product; sixteen read and convert the codes once for all of them, with fewer CTAs an SM.  They pay with many rows a sequence (us with 8 and 16 rows:
// 6000 rows of 80 channels 237 / 176, of 256 438 / 339; 16 and 32 rows, 64 sequences: 60 / 69 and 94 / 108), with 64 channels (64 sequences of 63 rows 46 / 43), and where
// they bring the CTAs down to what clusters serve (1600 rows 31 / 23, 16 sequences of 16 rows 24 / 21); not where CTAs are few (80 of 8 rows 16.5 / 17.4).
int attend_tile(const SeqCache8& c, const SeqPortions& p, const SeqAttend8& a) {
	const long long rows = (long long)p.longest * (a.heads / c.heads);
	auto ctas = [&](int tile) { return (long long)p.n * cdiv(rows, tile) * c.heads; };
	if (rows >= 64 && rows <= 65535 * 128LL && (c.dim == 64 || c.dim == 128) && !(a.softcap > 0.f) && !a.slopes && ctas(128) >= ap_least(a.q.type == SEQ_F32, c.dim)) return AP_TILE;
	return rows > 8 && ctas(8) > AT_ROOM / 2 && (rows >= 64 || c.dim <= 64 || ctas(16) <= AT_ROOM / 2) ? 16 : 8;
}
AtPlan attend_plan(const SeqCache8& c, const SeqPortions& p, const SeqAttend8& a) {
	const int group = a.heads / c.heads, tile = attend_tile(c, p, a);
	if (tile == AP_TILE) return AtPlan{tile, 1, cdiv(std::max(a.most_keys, 1), AT_KEYS), 0};
	const long long ctas = (long long)p.n * cdiv((long long)p.longest * group, tile) * c.heads, room = AT_ROOM;
	long long keys = std::max(a.most_keys, 1);
	if (a.window > 0) keys = std::min(keys, (long long)a.window + a.keep_first + tile / group);
	if (a.chunk > 0) keys = std::min(keys, (long long)a.chunk + a.keep_first + tile / group);
	const int chunks = cdiv(keys, AT_KEYS);
	if (ctas < 1) return AtPlan{tile, 1, chunks, 0};
	// many CTAs: several rounds, so that the last one is short (64 tokens over 2000 to 8000 keys: two rounds 140 us, six 126, eight 126, twelve 139); one where tokens are many, whose
	// shares would be as many rows to write and to fold (us with one and six: 2000 rows 44 / 63, 8 sequences of 400 34 / 53, 4 of 256 24 / 32)
	const int rounds = (long long)p.longest * group >= 64 ? 1 : 6;
	long long shares = ctas >= rounds * room ? 1 : ctas > room / 2 ? cdiv(rounds * room, ctas) : room / ctas;
	shares = std::max(1LL, std::min({shares, (long long)cdiv(chunks, ctas > room / 2 ? 2 * AT_WARPS : AT_WARPS), (long long)AT_SHARES}));
	// one round: a cluster folds them, and the fold's launch is saved (one token over 4000 keys 11.0 us and 32.2 without, four 14.1 and 21.9)
	const bool cluster = shares > 1 && ctas <= room / 2;
	if (cluster) shares = shares >= 16 ? 16 : shares >= 8 ? 8 : shares >= 4 ? 4 : 2;
	const int each = cdiv(chunks, shares);
	return AtPlan{tile, cluster ? (int)shares : cdiv(chunks, each), each, cluster};
}
size_t attend_bytes(const SeqCache8& c, const SeqAttend8& a, const AtPlan& p) { return p.shares > 1 && !p.cluster ? (size_t)a.q.rows * a.heads * p.shares * (c.dim + 2) * sizeof(float) : 0; }

int check_attend(const SeqCache8* c, const SeqPortions* p, const SeqAttend8* a) {
	if (const int rc = check_cache("attend8", c, p)) return rc;
	if (!a) return refuse("attend8: no arguments");
	if (const int rc = check_rows("attend8", "q", a->q)) return rc;
	if (const int rc = check_rows("attend8", "out", a->out)) return rc;
	if (a->heads < 1 || a->heads % c->heads) return refuse("attend8: %d query heads over %d key heads", a->heads, c->heads);
	if (a->heads > 65535) return refuse("attend8: at most 65535 query heads");
	if ((long long)p->longest * (a->heads / c->heads) > INT_MAX - 256) return refuse("attend8: %d tokens of %d query heads a key head: at most 2^31 pairs a sequence", p->longest, a->heads / c->heads);
	if (a->out.type != a->q.type && !(a->q.type == SEQ_F32 && a->out.type == SEQ_BF16)) return refuse("attend8: out has type %d, q %d", a->out.type, a->q.type);
	if (a->out.rows < a->q.rows) return refuse("attend8: out has %d rows, q %d", a->out.rows, a->q.rows);
	if (((uintptr_t)a->sinks | (uintptr_t)a->slopes | (uintptr_t)a->gate) % 4) return refuse("attend8: sinks, slopes or gate are not aligned to 4 bytes");
	if (!(a->scale == a->scale) || a->window < 0 || a->keep_first < 0 || a->chunk < 0 || !(a->softcap >= 0.f)) return refuse("attend8: scale, window, keep_first, chunk or softcap out of range");
	return 0;
}

template <int D, bool SPLIT, int NQ>
cudaError_t attend_launch(const C8& c, const Attend& a, dim3 grid, cudaStream_t st) {
	constexpr size_t smem = at_smem<D, SPLIT, NQ>();
	static std::atomic<uint64_t> done{0};
	cudaError_t e = allow(k_c8_attend<D, SPLIT, NQ>, smem, done, true);
	if (e == cudaSuccess) e = launch(st, false, a.cluster ? a.shares : 1, k_c8_attend<D, SPLIT, NQ>, grid, dim3(32 * AT_WARPS), smem, c, a);
	return e;
}
template <int D, bool SPLIT>
cudaError_t prompt_launch(const C8& c, const Attend& a, dim3 grid, cudaStream_t st) {
	static std::atomic<uint64_t> done{0};
	cudaError_t e = allow(k_c8_prompt<D, SPLIT>, sizeof(ApShared<D, SPLIT>), done);
	if (e == cudaSuccess) e = launch(st, false, 1, k_c8_prompt<D, SPLIT>, dim3(grid.y, grid.z, cdiv(grid.x, ap_groups(SPLIT))), dim3(ap_threads(SPLIT)), sizeof(ApShared<D, SPLIT>), c, a);
	return e;
}
template <int D>
cudaError_t attend_wide(const C8& c, const Attend& a, dim3 grid, cudaStream_t st) {
	const bool split = a.q_type == SEQ_F32;
	if constexpr (D < 256)
		if (a.tile == AP_TILE) return split ? prompt_launch<D, true>(c, a, grid, st) : prompt_launch<D, false>(c, a, grid, st);
	if (a.tile == 8) return split ? attend_launch<D, true, 1>(c, a, grid, st) : attend_launch<D, false, 1>(c, a, grid, st);
	return split ? attend_launch<D, true, 2>(c, a, grid, st) : attend_launch<D, false, 2>(c, a, grid, st);
}
} // namespace

void attend8_plan(const SeqCache8& cache, const SeqPortions& batch, const SeqAttend8& args, int (&plan)[4]) {
	const AtPlan p = attend_plan(cache, batch, args);
	plan[0] = p.tile, plan[1] = p.shares, plan[2] = p.each, plan[3] = p.cluster;
}
} // namespace seqops

extern "C" int calm_b200_seq_cache8_store(const struct SeqCache8* cache, const struct SeqPortions* batch, const struct SeqRows* k, const struct SeqRows* v, void* stream) {
	using namespace seqops;
	if (const int rc = check_cache("store8", cache, batch)) return rc;
	if (!k || !v) return refuse("store8: no rows");
	if (const int rc = check_rows("store8", "k", *k)) return rc;
	if (const int rc = check_rows("store8", "v", *v)) return rc;
	if (k->type != v->type) return refuse("store8: keys have type %d, values %d", k->type, v->type);
	if (batch->n == 0 || batch->longest == 0) return 0;
	const C8 c = describe(*cache, *batch);
	const dim3 grid(cdiv((long long)batch->longest + cache->page - 1, cache->page), cdiv(2 * cache->heads, ST_WARPS), batch->n);
	const StoreRows rk = store_rows(*k), rv = store_rows(*v);
	auto kernel = k->type == SEQ_F32 ? k_c8_store<float> : k->type == SEQ_BF16 ? k_c8_store<bf16> : k_c8_store<__half>;
	const cudaError_t e = launch((cudaStream_t)stream, false, 1, kernel, grid, dim3(32 * ST_WARPS), 0, c, rk, rv);
	return e == cudaSuccess ? 0 : failed("store8", e);
}

extern "C" size_t calm_b200_seq_attend8_workspace(const struct SeqCache8* cache, const struct SeqPortions* batch, const struct SeqAttend8* args) {
	using namespace seqops;
	if (check_attend(cache, batch, args)) return 0;
	return attend_bytes(*cache, *args, attend_plan(*cache, *batch, *args));
}

extern "C" int calm_b200_seq_attend8(const struct SeqCache8* cache, const struct SeqPortions* batch, const struct SeqAttend8* q, void* stream) {
	using namespace seqops;
	if (const int rc = check_attend(cache, batch, q)) return rc;
	if (batch->n == 0 || batch->longest == 0) return 0;
	const AtPlan plan = attend_plan(*cache, *batch, *q);
	const int shares = plan.shares;
	const size_t need = attend_bytes(*cache, *q, plan);
	if (need && (!q->workspace || (uintptr_t)q->workspace % 16 || q->workspace_bytes < need)) return refuse("attend8: the workspace has %zu bytes (16-byte aligned), %zu are needed", q->workspace ? q->workspace_bytes : (size_t)0, need);
	const C8 c = describe(*cache, *batch);
	Attend a;
	a.q = q->q.p, a.q_row = q->q.row_stride, a.q_head = q->q.head_stride, a.out = q->out.p, a.o_row = q->out.row_stride, a.o_head = q->out.head_stride;
	a.rows = q->q.rows, a.heads = q->heads, a.group = q->heads / cache->heads, a.scale = q->scale, a.softcap = q->softcap;
	a.window = q->window, a.keep_first = q->keep_first, a.chunk = q->chunk, a.sinks = q->sinks, a.slopes = q->slopes;
	a.gate = q->gate, a.gate_row = q->gate_row, a.gate_head = q->gate_head, a.gate_dim = q->gate_dim;
	a.shares = shares, a.each = plan.each, a.part = (float*)q->workspace;
	a.q_type = q->q.type, a.out_type = q->out.type, a.tile = plan.tile, a.cluster = plan.cluster;
	const dim3 grid(cdiv((long long)batch->longest * a.group, a.tile), cache->heads * shares, batch->n), fold(std::min(cdiv((long long)batch->longest * a.group, 4), 65535), cache->heads, batch->n);
	if (grid.y > 65535) return refuse("attend8: too many key heads");
	const cudaStream_t st = (cudaStream_t)stream;
	cudaError_t e = cache->dim <= 64 ? attend_wide<64>(c, a, grid, st) : cache->dim <= 128 ? attend_wide<128>(c, a, grid, st) : attend_wide<256>(c, a, grid, st);
	if (e == cudaSuccess && shares > 1 && !plan.cluster) e = launch(st, true, 1, k_c8_fold, fold, dim3(128), 0, c, a);
	return e == cudaSuccess ? 0 : failed("attend8", e);
}
