// seqrotate.cu -- rotary positions, and a step's rows into a paged cache in 16 bits with the rotation on the way (calm_b200_seq_rotate, calm_b200_seq_cache16_store in
// include/calm_b200_seq.h).

#include "seqcache16.cuh"

namespace seqops {
namespace {

typedef __nv_bfloat16 bf16;

// A pair of channels (a, b) of a row at position p becomes (a cos - b sin, b cos + a sin) at the angle 2 pi p turns_i.  The angle is a product in 64 bits of which the whole turns are taken off
// before it becomes fp32: 2^31 positions are as exact as one.  One launch for everything: queries, keys and values are one list of units (U neighbouring channels of a head, with the U
// channels that they turn with where the pairs lie in two halves), a thread takes one unit of TURN_DEPTH tokens, asking for all of them before it uses the first; cosines and sines of the CTA's tokens
// come from shared memory.
constexpr int TURN_THREADS = 256, TURN_DEPTH = 4;
constexpr int TURN_ANGLES = 4096; // cosines and sines of a CTA at most: 32 KB

struct TurnRows {
	const void* p;
	void* out; // queries: where they go
	long long row, head, out_row, out_head;
	int vec, out_vec; // a unit at a time
};
struct Turn {
	TurnRows q, k, v;
	char *kc, *vc; // the pools
	const int* table;
	const int *start, *count, *slot, *pos0;
	const double* turns;
	float gain;
	int rows;                 // of the shortest of the arrays
	int q_heads, heads, dim;  // heads: of the cache, 0 without one
	int pairs;                // pairs of channels
	int page, page_shift, pages, slots, table_pages;
	int turned, rest;         // units of a head that turn and that do not
	int q_units, k_units, units; // units of a token's queries, its queries and keys, all of them
	int q_rest;               // units of a query that are copied (0: in place)
	int groups, step;         // of threads: each takes TURN_DEPTH tokens and every step'th unit
};

template <typename T, int U>
__device__ __forceinline__ void load_unit(const T* p, bool vec, float (&x)[U]) {
	constexpr int BYTES = U * sizeof(T);
	if (!vec || BYTES < 4) {
#pragma unroll
		for (int i = 0; i < U; ++i) x[i] = as_f32(p[i]);
	} else if constexpr (BYTES == 32) {
		const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
		x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
	} else {
		typename std::conditional<BYTES == 16, uint4, typename std::conditional<BYTES == 8, uint2, uint32_t>::type>::type w = *reinterpret_cast<const decltype(w)*>(p);
		const T* h = reinterpret_cast<const T*>(&w);
#pragma unroll
		for (int i = 0; i < U; ++i) x[i] = as_f32(h[i]);
	}
}
template <typename T, int U>
__device__ __forceinline__ void store_unit(T* p, bool vec, const float (&x)[U]) {
	constexpr int BYTES = U * sizeof(T);
	if (!vec || BYTES < 4) {
#pragma unroll
		for (int i = 0; i < U; ++i) p[i] = from_f32<T>(x[i]);
	} else if constexpr (BYTES == 32) {
		reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
		reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
	} else {
		typename std::conditional<BYTES == 16, uint4, typename std::conditional<BYTES == 8, uint2, uint32_t>::type>::type w;
		T* h = reinterpret_cast<T*>(&w);
#pragma unroll
		for (int i = 0; i < U; ++i) h[i] = from_f32<T>(x[i]);
		*reinterpret_cast<decltype(w)*>(p) = w;
	}
}

// T: the rows' type, C: the cache's
template <typename T, typename C, int U, bool NEIGHBOURS>
__global__ void __launch_bounds__(TURN_THREADS) k_turn(const Turn a) {
	extern __shared__ float2 angles[]; // [tokens][pairs]: cosine, sine
	const int b = blockIdx.z, n = a.count[b], p0 = a.pos0[b], start = a.start[b], tokens = a.groups * TURN_DEPTH;
	if (n < 1 || p0 < 0 || p0 > INT_MAX - n || start < 0 || n > a.rows - start) return;
	const long long first = (long long)blockIdx.x * tokens;
	if (first >= n) return;
	const int i0 = (int)first, here = min(tokens, n - i0);
	__shared__ long long place[TURN_THREADS * TURN_DEPTH]; // of each token in a pool, in rows of its first head; -1: nowhere
	for (int i = threadIdx.x; i < here * a.pairs; i += blockDim.x) {
		const int t = i / a.pairs;
		const double turn = (double)(p0 + i0 + t) * a.turns[i - t * a.pairs];
		float s, c;
		sincospif((float)(2.0 * (turn - rint(turn))), &s, &c);
		angles[i] = make_float2(c * a.gain, s * a.gain);
	}
	if (a.heads)
		for (int t = threadIdx.x; t < here; t += blockDim.x) {
			const int pos = p0 + i0 + t, at = a.page_shift >= 0 ? pos >> a.page_shift : pos / a.page, slot = a.slot[b];
			const int id = (unsigned)slot < (unsigned)a.slots && at < a.table_pages ? a.table[(size_t)slot * a.table_pages + at] : -1;
			place[t] = (unsigned)id < (unsigned)a.pages ? (long long)id * a.heads * a.page + (pos - at * a.page) : -1;
		}
	__syncthreads();
	const int group = threadIdx.x / a.step;
	if (group >= a.groups) return;
	const int t0 = group * TURN_DEPTH;
	for (int u = blockIdx.y * a.step + threadIdx.x % a.step; u < a.units; u += gridDim.y * a.step) {
		const bool is_q = u < a.q_units, is_v = u >= a.k_units;
		const TurnRows& r = is_q ? a.q : is_v ? a.v : a.k;
		const int v = is_q ? u : is_v ? u - a.k_units : u - a.q_units, turned = is_v ? 0 : a.turned, each = turned + (is_q ? a.q_rest : is_v ? a.dim / U : a.rest);
		const int head = v / each, w = v - head * each;
		const bool turns = w < turned;
		// the unit's first channel; for pairs that lie in two halves the second half's is `pairs` further
		const int d = (turns || NEIGHBOURS || is_v ? w : w + turned) * U;
		const T* src = (const T*)r.p + (long long)(start + i0 + t0) * r.row + head * r.head + d;
		float x[TURN_DEPTH][U], y[TURN_DEPTH][NEIGHBOURS ? 1 : U];
#pragma unroll
		for (int t = 0; t < TURN_DEPTH; ++t)
			if (t0 + t < here) {
				load_unit<T, U>(src + t * r.row, r.vec, x[t]);
				if constexpr (!NEIGHBOURS)
					if (turns) load_unit<T, U>(src + t * r.row + a.pairs, r.vec, y[t]);
			}
#pragma unroll
		for (int t = 0; t < TURN_DEPTH; ++t) {
			if (t0 + t >= here) break;
			if (turns) {
				const float2* const cs = angles + (t0 + t) * a.pairs + (NEIGHBOURS ? d / 2 : d);
				if constexpr (NEIGHBOURS) {
#pragma unroll
					for (int i = 0; i + 1 < U; i += 2) {
						const float2 f = cs[i / 2];
						const float p = x[t][i], q = x[t][i + 1];
						x[t][i] = p * f.x - q * f.y, x[t][i + 1] = q * f.x + p * f.y;
					}
				} else {
#pragma unroll
					for (int i = 0; i < U; ++i) {
						const float2 f = cs[i];
						const float p = x[t][i], q = y[t][i];
						x[t][i] = p * f.x - q * f.y, y[t][i] = q * f.x + p * f.y;
					}
				}
			}
			if (is_q) {
				T* const to = (T*)r.out + (long long)(start + i0 + t0 + t) * r.out_row + head * r.out_head + d;
				store_unit<T, U>(to, r.out_vec, x[t]);
				if constexpr (!NEIGHBOURS)
					if (turns) store_unit<T, U>(to + a.pairs, r.out_vec, y[t]);
			} else if (place[t0 + t] >= 0) {
				C* const to = (C*)(is_v ? a.vc : a.kc) + (place[t0 + t] + (long long)head * a.page) * a.dim + d;
				store_unit<C, U>(to, true, x[t]); // (rows of a cache are 16-byte aligned)
				if constexpr (!NEIGHBOURS)
					if (turns) store_unit<C, U>(to + a.pairs, true, y[t]);
			}
		}
	}
}

int check_turn(const char* what, const SeqRotation* r, int dim) {
	if (!r) return 0;
	if (r->dims < 2 || r->dims > dim || r->dims % 2) return refuse("%s: a rotation of %d channels in rows of %d: an even number from 2 on", what, r->dims, dim);
	if (!r->turns) return refuse("%s: the rotation has no frequencies", what);
	if ((uintptr_t)r->turns % 8) return refuse("%s: the rotation's frequencies are not aligned to 8 bytes", what);
	return 0;
}
// units of `u` elements can be moved at a time
bool turn_vec(const void* p, long long row, long long head, int type, int u) {
	const int bytes = std::min(16, u * type_size(type)), each = bytes / type_size(type);
	return (uintptr_t)p % bytes == 0 && row % each == 0 && head % each == 0;
}

template <typename T, typename C, int U>
cudaError_t turn_of(bool neighbours, const Turn& a, dim3 grid, int threads, size_t smem, cudaStream_t st) {
	return neighbours ? launch(st, false, 1, k_turn<T, C, U, true>, grid, dim3(threads), smem, a) : launch(st, false, 1, k_turn<T, C, U, false>, grid, dim3(threads), smem, a);
}
template <typename T, typename C>
cudaError_t turn_unit(int unit, bool neighbours, const Turn& a, dim3 grid, int threads, size_t smem, cudaStream_t st) {
	switch (unit) {
	case 8: return turn_of<T, C, 8>(neighbours, a, grid, threads, smem, st);
	case 4: return turn_of<T, C, 4>(neighbours, a, grid, threads, smem, st);
	case 2: return turn_of<T, C, 2>(neighbours, a, grid, threads, smem, st);
	default: return turn_of<T, C, 1>(false, a, grid, threads, smem, st);
	}
}
template <typename T>
cudaError_t turn_type(int cache, int unit, bool neighbours, const Turn& a, dim3 grid, int threads, size_t smem, cudaStream_t st) {
	return cache == SEQ_F16 ? turn_unit<T, __half>(unit, neighbours, a, grid, threads, smem, st) : turn_unit<T, bf16>(unit, neighbours, a, grid, threads, smem, st);
}

TurnRows turn_rows(const SeqRows& r) {
	TurnRows t = {};
	t.p = r.p, t.row = r.row_stride, t.head = r.head_stride;
	return t;
}

// queries into q_out and, with a cache, keys and values into it
int turn(const char* what, const SeqPortions& batch, const SeqRotation* rotation, const SeqRows* q, const SeqRows* q_out, int q_heads, const SeqCache16* cache, const SeqRows* k, const SeqRows* v, int dim,
         cudaStream_t stream) {
	Turn a = {};
	a.rows = INT_MAX;
	int type = 0, unit = 8;
	if (q) {
		a.q = turn_rows(*q), a.q.out = q_out->p, a.q.out_row = q_out->row_stride, a.q.out_head = q_out->head_stride;
		a.q_heads = q_heads, a.rows = std::min(q->rows, q_out->rows), type = q->type;
	}
	if (cache) {
		a.k = turn_rows(*k), a.v = turn_rows(*v), a.heads = cache->heads, a.rows = std::min(a.rows, std::min(k->rows, v->rows)), type = k->type;
		a.kc = (char*)cache->k, a.vc = (char*)cache->v, a.table = cache->table, a.page = cache->page, a.pages = cache->pages, a.slots = cache->slots, a.table_pages = cache->table_pages;
		a.page_shift = log2_of(cache->page);
	}
	const int dims = rotation ? rotation->dims : 0;
	const bool neighbours = rotation && rotation->neighbours;
	a.dim = dim, a.pairs = dims / 2, a.start = batch.start, a.count = batch.count, a.slot = batch.slot, a.pos0 = batch.pos0;
	if (rotation) a.turns = rotation->turns, a.gain = rotation->gain;
	while (unit > 1 && ((neighbours ? dims : dims / 2) % unit || (dim - dims) % unit)) unit /= 2;
	a.turned = (neighbours ? dims : dims / 2) / unit, a.rest = (dim - dims) / unit;
	// Rest units begin behind the turned channels: with two halves these are twice as many as their units
	a.q_rest = q && q->p == q_out->p && q->row_stride == q_out->row_stride && q->head_stride == q_out->head_stride ? 0 : a.rest;
	const long long q_units = (long long)a.q_heads * (a.turned + a.q_rest), k_units = q_units + (long long)a.heads * (a.turned + a.rest), units = k_units + (long long)a.heads * (dim / unit);
	if (units > INT_MAX / 2) return refuse("%s: %d heads of %d channels are too many", what, q_heads, dim);
	if (!units || !batch.n || !batch.longest) return 0;
	a.q_units = (int)q_units, a.k_units = (int)k_units, a.units = (int)units;
	a.q.vec = q && turn_vec(a.q.p, a.q.row, a.q.head, type, unit), a.q.out_vec = q && turn_vec(a.q.out, a.q.out_row, a.q.out_head, type, unit);
	a.k.vec = cache && turn_vec(a.k.p, a.k.row, a.k.head, type, unit), a.v.vec = cache && turn_vec(a.v.p, a.v.row, a.v.head, type, unit);
	// a CTA's threads take all units of TURN_DEPTH tokens in as few rounds as they can, and more tokens where units are few; where tokens are few, several CTAs share a token's units
	const int rounds = cdiv(units, TURN_THREADS);
	a.step = (int)std::min<long long>(TURN_THREADS, cdiv(units, rounds));
	a.groups = std::max(1, std::min({TURN_THREADS / a.step, cdiv(batch.longest, TURN_DEPTH), a.pairs ? TURN_ANGLES / (TURN_DEPTH * a.pairs) : TURN_ANGLES / 8}));
	const int threads = cdiv(a.step * a.groups, 32) * 32, blocks = cdiv(batch.longest, a.groups * TURN_DEPTH);
	const int split = (long long)blocks * batch.n < 2 * 148 ? std::min(rounds, 64) : 1;
	const size_t smem = (size_t)a.groups * TURN_DEPTH * a.pairs * sizeof(float2);
	const dim3 grid(blocks, split, batch.n);
	const int ctype = cache ? cache->type : SEQ_BF16;
	const cudaError_t e = type == SEQ_F32 ? turn_type<float>(ctype, unit, neighbours, a, grid, threads, smem, stream)
	                      : type == SEQ_BF16 ? turn_type<bf16>(ctype, unit, neighbours, a, grid, threads, smem, stream)
	                                         : turn_type<__half>(ctype, unit, neighbours, a, grid, threads, smem, stream);
	return e == cudaSuccess ? 0 : failed(what, e);
}
} // namespace
} // namespace seqops

extern "C" int calm_b200_seq_rotate(const struct SeqPortions* batch, const struct SeqRotation* rotation, const struct SeqRows* x, const struct SeqRows* out, int heads, int dim, void* stream) {
	using namespace seqops;
	if (const int rc = check_batch("rotate", batch)) return rc;
	if (!rotation || !x || !out) return refuse("rotate: no rotation or no rows");
	if (heads < 1 || heads > 65535 || dim < 2 || dim > 1024 || dim % 2) return refuse("rotate: %d heads of %d channels: 1 to 65535 heads of an even number from 2 to 1024", heads, dim);
	if (const int rc = check_turn("rotate", rotation, dim)) return rc;
	if (const int rc = check_rows("rotate", "x", *x)) return rc;
	if (const int rc = check_rows("rotate", "out", *out)) return rc;
	if (x->type != out->type) return refuse("rotate: out has type %d, x %d", out->type, x->type);
	return turn("rotate", *batch, rotation, x, out, heads, nullptr, nullptr, nullptr, dim, (cudaStream_t)stream);
}

extern "C" int calm_b200_seq_cache16_store(const struct SeqCache16* cache, const struct SeqPortions* batch, const struct SeqRows* k, const struct SeqRows* v, const struct SeqRotation* rotation,
                                           const struct SeqRows* q, const struct SeqRows* q_out, int q_heads, void* stream) {
	using namespace seqops;
	if (const int rc = check_cache16("store16", cache, batch)) return rc;
	if (!k || !v) return refuse("store16: no rows");
	if (const int rc = check_rows("store16", "k", *k)) return rc;
	if (const int rc = check_rows("store16", "v", *v)) return rc;
	if (k->type != v->type) return refuse("store16: keys have type %d, values %d", k->type, v->type);
	if (const int rc = check_turn("store16", rotation, cache->dim)) return rc;
	if (q) {
		if (!rotation || !q_out) return refuse("store16: queries come with a rotation and a place to go");
		if (const int rc = check_rows("store16", "q", *q)) return rc;
		if (const int rc = check_rows("store16", "q_out", *q_out)) return rc;
		if (q->type != k->type || q_out->type != q->type) return refuse("store16: queries have types %d and %d, keys %d", q->type, q_out->type, k->type);
		if (q_heads < 1 || q_heads > 65535) return refuse("store16: %d query heads", q_heads);
	}
	return turn("store16", *batch, rotation, q, q_out, q ? q_heads : 0, cache, k, v, cache->dim, (cudaStream_t)stream);
}
