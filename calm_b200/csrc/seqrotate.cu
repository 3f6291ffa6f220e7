// seqrotate.cu -- rotary positions, and a step's rows into a paged cache in 16 bits with the rotation on the way (calm_b200_seq_rotate, calm_b200_seq_cache16_store in
// include/calm_b200_seq.h).

#include "seqcache16.cuh"

namespace seqops {
namespace {

typedef __nv_bfloat16 bf16;

// A pair of channels (a, b) of a row at position p becomes (a cos - b sin, b cos + a sin) at the angle 2 pi p turns_i.  The angle is a product in 64 bits of which the whole turns are taken off
// before it becomes fp32: off by 3 2^-53 of the whole angle beside fp32's pi 2^-25 (7e-7 and 9e-8 at 2^31 positions of a radian each).  A thread keeps one unit of channels (U neighbours of a head, with the U that they turn with where the pairs lie in two halves) of one token: it forms
// the unit's cosines and sines once, in registers, and takes one head after another, asking for TURN_DEPTH of them before it uses the first.  Queries, keys and values are one launch.
// Bound: memory.  11307 rows of 40 heads of 128 bf16 channels (232 MB) 44 us, 5.2 TB/s; 10094 rows of 32 query heads stored with 8 of keys and values (248 MB) 47 us, 5.3 TB/s; one token 2.4 and 2.9 us, a launch's latency.
// (us of the two: blocks of 256 threads 50 and 54, of 64 45 and 46; TURN_DEPTH 4 44 and 51; TURN_HEADS 8 42 and 49, 20 47 and 49; angles through shared memory and a barrier 103 and 127.)
constexpr int TURN_THREADS = 128, TURN_DEPTH = 2;
constexpr int TURN_BLOCKS = 148 * 4; // blocks to keep every SM busy
constexpr int TURN_HEADS = 16;       // heads of a thread at most

struct TurnRows {
	const void* p;
	void* out; // queries: where they go
	long long row, head, out_row, out_head;
	int vec, out_vec; // a unit at a time
};
struct TurnPart { // how the threads of a block share a part's work: columns of units, heads
	int columns, heads, side, each, blocks; // side: threads side by side on one column of a token, each: heads of a thread, blocks: of the grid for a token's heads
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
	int turned;               // columns that turn
	int in_place;             // 1: the columns of a query that do not turn are where they belong
	int tokens;               // of a block
	int spread;               // blocks that share a token's columns
	TurnPart turn, copy;      // queries and keys; values
};

// a unit as it lies in memory, and as floats
template <typename T, int U>
struct Raw {
	static constexpr int BYTES = U * sizeof(T), WORDS = (BYTES + 3) / 4;
	uint32_t w[WORDS];
	__device__ __forceinline__ void load(const T* p, bool vec) {
		if (BYTES < 4 || (!vec && sizeof(T) == 2)) {
			const uint16_t* const h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
			for (int i = 0; i < WORDS; ++i) w[i] = BYTES < 4 ? h[0] : h[2 * i] | (uint32_t)h[2 * i + 1] << 16;
		} else if (!vec || BYTES == 4) {
#pragma unroll
			for (int i = 0; i < WORDS; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
		} else if constexpr (BYTES == 8) {
			const uint2 x = *reinterpret_cast<const uint2*>(p);
			w[0] = x.x, w[1] = x.y;
		} else if constexpr (BYTES >= 16) {
#pragma unroll
			for (int i = 0; i < WORDS; i += 4) {
				const uint4 x = reinterpret_cast<const uint4*>(p)[i / 4];
				w[i] = x.x, w[i + 1] = x.y, w[i + 2] = x.z, w[i + 3] = x.w;
			}
		}
	}
	__device__ __forceinline__ void floats(float (&x)[U]) const {
#pragma unroll
		for (int i = 0; i < U; ++i)
			if constexpr (sizeof(T) == 4) x[i] = __uint_as_float(w[i]);
			else {
				const uint16_t h = (uint16_t)(w[i / 2] >> (i % 2 * 16));
				x[i] = as_f32(*reinterpret_cast<const T*>(&h));
			}
	}
};
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
	constexpr int ANGLES = NEIGHBOURS ? (U + 1) / 2 : U;
	const bool is_v = blockIdx.y >= a.turn.blocks;
	const TurnPart& part = is_v ? a.copy : a.turn;
	const int width = min(part.columns, TURN_THREADS), at = threadIdx.x / width, column = threadIdx.x % width + blockIdx.x % a.spread * TURN_THREADS;
	const unsigned index = blockIdx.x / a.spread * a.tokens + at % a.tokens; // (the last block's threads may pass 2^31)
	const int side = at / a.tokens;
	const int b = blockIdx.z, n = a.count[b], p0 = a.pos0[b], start = a.start[b];
	if (n < 1 || p0 < 0 || p0 > INT_MAX - n || start < 0 || n > a.rows - start || index >= (unsigned)n || side >= part.side || column >= part.columns) return;
	const int token = (int)index;
	const bool turns = !is_v && column < a.turned;
	double step[ANGLES];
	if (turns)
#pragma unroll
		for (int i = 0; i < ANGLES; ++i) step[i] = a.turns[column * ANGLES + i];
	// the unit's first channel; for pairs that lie in two halves the second half's is `pairs` further
	const int d = (NEIGHBOURS || is_v || turns ? column : column + a.turned) * U, pos = p0 + token;
	const int first = (is_v ? blockIdx.y - a.turn.blocks : blockIdx.y) * part.side * part.each + side, last = min(part.heads, first + part.side * part.each);
	long long place = -1; // of the token in a pool, in rows of its first head; -1: nowhere
	if (a.heads && (is_v || last > a.q_heads)) {
		const int page = a.page_shift >= 0 ? pos >> a.page_shift : pos / a.page, slot = a.slot[b];
		const int id = (unsigned)slot < (unsigned)a.slots && page < a.table_pages ? a.table[(size_t)slot * a.table_pages + page] : -1;
		if ((unsigned)id < (unsigned)a.pages) place = (long long)id * a.heads * a.page + (pos - page * a.page);
	}
	float cosine[ANGLES], sine[ANGLES];
	bool formed = false;
	for (int h0 = first; h0 < last; h0 += part.side * TURN_DEPTH) {
		Raw<T, U> x[TURN_DEPTH], y[NEIGHBOURS ? 1 : TURN_DEPTH];
#pragma unroll
		for (int t = 0; t < TURN_DEPTH; ++t) {
			const int h = h0 + t * part.side;
			if (h >= last) break;
			const bool is_q = !is_v && h < a.q_heads;
			if (is_q && a.in_place && !turns) continue;
			const TurnRows& r = is_v ? a.v : is_q ? a.q : a.k;
			const T* const src = (const T*)r.p + (long long)(start + token) * r.row + (is_v || is_q ? h : h - a.q_heads) * r.head + d;
			x[t].load(src, r.vec);
			if constexpr (!NEIGHBOURS)
				if (turns) y[t].load(src + a.pairs, r.vec);
		}
		if (turns && !formed) { // (while the first heads are on their way)
			formed = true;
#pragma unroll
			for (int i = 0; i < ANGLES; ++i) {
				const double turn = (double)pos * step[i];
				sincospif((float)(2.0 * (turn - rint(turn))), sine + i, cosine + i);
				cosine[i] *= a.gain, sine[i] *= a.gain;
			}
		}
#pragma unroll
		for (int t = 0; t < TURN_DEPTH; ++t) {
			const int h = h0 + t * part.side;
			if (h >= last) break;
			const bool is_q = !is_v && h < a.q_heads;
			if (is_q && a.in_place && !turns) continue;
			float u[U], v[NEIGHBOURS ? 1 : U];
			x[t].floats(u);
			if (turns) {
				if constexpr (NEIGHBOURS) {
#pragma unroll
					for (int i = 0; i + 1 < U; i += 2) {
						const float p = u[i], q = u[i + 1];
						u[i] = p * cosine[i / 2] - q * sine[i / 2], u[i + 1] = q * cosine[i / 2] + p * sine[i / 2];
					}
				} else {
					y[t].floats(v);
#pragma unroll
					for (int i = 0; i < U; ++i) {
						const float p = u[i], q = v[i];
						u[i] = p * cosine[i] - q * sine[i], v[i] = q * cosine[i] + p * sine[i];
					}
				}
			}
			if (is_q) {
				T* const to = (T*)a.q.out + (long long)(start + token) * a.q.out_row + h * a.q.out_head + d;
				store_unit<T, U>(to, a.q.out_vec, u);
				if constexpr (!NEIGHBOURS)
					if (turns) store_unit<T, U>(to + a.pairs, a.q.out_vec, v);
			} else if (place >= 0) {
				C* const to = (C*)(is_v ? a.vc : a.kc) + (place + (long long)(is_v ? h : h - a.q_heads) * a.page) * a.dim + d;
				store_unit<C, U>(to, true, u); // (rows of a cache are 16-byte aligned)
				if constexpr (!NEIGHBOURS)
					if (turns) store_unit<C, U>(to + a.pairs, true, v);
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
cudaError_t turn_of(bool neighbours, const Turn& a, dim3 grid, int threads, cudaStream_t st) {
	return neighbours ? launch(st, false, 1, k_turn<T, C, U, true>, grid, dim3(threads), 0, a) : launch(st, false, 1, k_turn<T, C, U, false>, grid, dim3(threads), 0, a);
}
template <typename T, typename C>
cudaError_t turn_unit(int unit, bool neighbours, const Turn& a, dim3 grid, int threads, cudaStream_t st) {
	switch (unit) {
	case 8: return turn_of<T, C, 8>(neighbours, a, grid, threads, st);
	case 4: return turn_of<T, C, 4>(neighbours, a, grid, threads, st);
	case 2: return turn_of<T, C, 2>(neighbours, a, grid, threads, st);
	default: return turn_of<T, C, 1>(false, a, grid, threads, st);
	}
}
template <typename T>
cudaError_t turn_type(int cache, int unit, bool neighbours, const Turn& a, dim3 grid, int threads, cudaStream_t st) {
	return cache == SEQ_F16 ? turn_unit<T, __half>(unit, neighbours, a, grid, threads, st) : turn_unit<T, bf16>(unit, neighbours, a, grid, threads, st);
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
	a.turned = (neighbours ? dims : dims / 2) / unit;
	a.in_place = q && q->p == q_out->p && q->row_stride == q_out->row_stride && q->head_stride == q_out->head_stride;
	if (!(a.q_heads + a.heads) || !batch.n || !batch.longest) return 0;
	a.q.vec = q && turn_vec(a.q.p, a.q.row, a.q.head, type, unit), a.q.out_vec = q && turn_vec(a.q.out, a.q.out_row, a.q.out_head, type, unit);
	a.k.vec = cache && turn_vec(a.k.p, a.k.row, a.k.head, type, unit), a.v.vec = cache && turn_vec(a.v.p, a.v.row, a.v.head, type, unit);
	// a block: as many tokens as its threads have room for, where tokens are few several heads at once; heads go to several blocks while these are few
	a.turn.columns = a.turned + (dim - dims) / unit, a.copy.columns = dim / unit;
	a.turn.heads = a.q_heads + a.heads, a.copy.heads = a.heads;
	const int widest = cache ? a.copy.columns : a.turn.columns; // (of the two)
	a.tokens = std::max(1, std::min(batch.longest, TURN_THREADS / widest));
	a.spread = cdiv(widest, TURN_THREADS);
	const int blocks = cdiv(batch.longest, a.tokens);
	int threads = 32;
	for (TurnPart* p : {&a.turn, &a.copy}) {
		if (!p->heads) continue;
		p->side = std::max(1, std::min(p->heads, TURN_THREADS / (p->columns * a.tokens)));
		const int rounds = cdiv(p->heads, p->side), most = (int)std::max<long long>(1, TURN_BLOCKS / ((long long)blocks * batch.n));
		p->each = cdiv(rounds, std::min(rounds, std::max(most, cdiv(rounds, TURN_HEADS))));
		p->blocks = cdiv(rounds, p->each);
		threads = std::max(threads, cdiv(std::min(p->columns, TURN_THREADS) * a.tokens * p->side, 32) * 32);
	}
	const dim3 grid((unsigned)((long long)blocks * a.spread), a.turn.blocks + a.copy.blocks, batch.n);
	if (grid.y > 65535 || (long long)blocks * a.spread > INT_MAX) return refuse("%s: %d heads of %d channels are too many", what, a.turn.heads, dim);
	const int ctype = cache ? cache->type : SEQ_BF16;
	const cudaError_t e = type == SEQ_F32 ? turn_type<float>(ctype, unit, neighbours, a, grid, threads, stream)
	                      : type == SEQ_BF16 ? turn_type<bf16>(ctype, unit, neighbours, a, grid, threads, stream)
	                                         : turn_type<__half>(ctype, unit, neighbours, a, grid, threads, stream);
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
