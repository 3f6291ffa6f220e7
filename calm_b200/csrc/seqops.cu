// seqops.cu -- what the operators share on the host, and copies of pages and slots (include/calm_b200_seq.h).

#include "seqops.cuh"

#include <stdarg.h>
#include <string.h>

#include <algorithm>
#include <atomic>
#include <new>
#include <vector>

namespace seqops {

namespace {
thread_local char g_message[512] = "";
std::atomic<uint64_t> g_launches{0};
} // namespace

int refuse(const char* fmt, ...) {
	va_list ap;
	va_start(ap, fmt);
	vsnprintf(g_message, sizeof(g_message), fmt, ap);
	va_end(ap);
	return -3;
}
int failed(const char* what, cudaError_t e) {
	snprintf(g_message, sizeof(g_message), "%s: %s (%s)", what, cudaGetErrorString(e), cudaGetErrorName(e));
	(void)cudaGetLastError(); // a launch that was turned down is not found again by the next call
	return -4;
}
void count_launch() { g_launches.fetch_add(1, std::memory_order_relaxed); }
uint64_t launches() { return g_launches.load(std::memory_order_relaxed); }

// ---------------------------------------------------------------- copies of units
// All copies of a call are one launch (a launch per COPY_PAIRS pairs or COPY_POOLS pools): descriptors and lists travel in the kernel's parameters, so nothing is staged, and a captured
// call holds its own lists.  A CTA copies COPY_CHUNK bytes of one unit; CTA index -> pool (by the pools' first CTAs) -> pair -> chunk.  Bound: memory,
// 2 bytes moved for each one copied: 1500 pages of 16 rows in 8 caches (786 MB moved) 126 us, 6.2 TB/s; 96 forks of 17 MB of pages and states each (819 MB) 127 us, 6.5 TB/s, a plain copy's
// rate; three small forks 2.7 us, the latency of one launch.
constexpr int COPY_POOLS = 64, COPY_PAIRS = 1024, COPY_THREADS = 256, COPY_DEPTH = 4;
constexpr int COPY_CHUNK = COPY_THREADS * COPY_DEPTH * 16;

struct CopyPool {
	const char* src;
	char* dst;
	long long unit, row;  // bytes
	unsigned first;       // first CTA of the pool
	unsigned chunks;      // CTAs a unit
	int kind;
};
template <int PAIRS>
struct CopyArgs {
	CopyPool pool[COPY_POOLS];
	int pools, n_pages;           // page pairs come first, slot pairs behind them
	int from[PAIRS], to[PAIRS];
	int rows[PAIRS];              // of the page pairs; -1: the whole unit
};

template <int PAIRS>
__global__ void __launch_bounds__(COPY_THREADS) k_copy_units(const __grid_constant__ CopyArgs<PAIRS> a) {
	int lo = 0, hi = a.pools - 1;
	while (lo < hi) { // the last pool whose first CTA is not behind this one
		const int mid = (lo + hi + 1) / 2;
		if (a.pool[mid].first <= blockIdx.x) lo = mid;
		else hi = mid - 1;
	}
	const CopyPool& p = a.pool[lo];
	const unsigned at = blockIdx.x - p.first, pair = at / p.chunks, chunk = at - pair * p.chunks;
	const int i = p.kind ? a.n_pages + (int)pair : (int)pair;
	long long bytes = p.unit;
	if (!p.kind && p.row > 0 && a.rows[i] >= 0) bytes = min(bytes, p.row * a.rows[i]);
	const long long begin = (long long)chunk * COPY_CHUNK, end = min(bytes, begin + COPY_CHUNK);
	if (begin >= end) return;
	const char* src = p.src + p.unit * a.from[i];
	char* dst = p.dst + p.unit * a.to[i];
	const unsigned align = (unsigned)((uintptr_t)src | (uintptr_t)dst | (uintptr_t)end) & 15;
	if (align == 0) {
		const uint4* s = reinterpret_cast<const uint4*>(src + begin);
		uint4* d = reinterpret_cast<uint4*>(dst + begin);
		const int n = (int)((end - begin) >> 4);
		uint4 v[COPY_DEPTH];
#pragma unroll
		for (int k = 0; k < COPY_DEPTH; ++k)
			if (k * COPY_THREADS + (int)threadIdx.x < n) v[k] = __ldcs(s + k * COPY_THREADS + threadIdx.x);
#pragma unroll
		for (int k = 0; k < COPY_DEPTH; ++k)
			if (k * COPY_THREADS + (int)threadIdx.x < n) d[k * COPY_THREADS + threadIdx.x] = v[k];
	} else if ((align & 3) == 0) {
		for (long long o = begin + 4 * threadIdx.x; o < end; o += 4 * COPY_THREADS) *reinterpret_cast<uint32_t*>(dst + o) = *reinterpret_cast<const uint32_t*>(src + o);
	} else
		for (long long o = begin + threadIdx.x; o < end; o += COPY_THREADS) dst[o] = src[o];
}

namespace {

// one launch of pools [p0, p1) over page pairs [a0, a1) and slot pairs [b0, b1)
template <int PAIRS>
cudaError_t copy_launch(const SeqUnits* pools, int n_pools, const int* pf, const int* pt, const int* pr, int np, const int* sf, const int* st, int ns, cudaStream_t stream) {
	CopyArgs<PAIRS> a;
	a.pools = 0, a.n_pages = np;
	long long ctas = 0;
	for (int i = 0; i < n_pools; ++i) {
		const SeqUnits& u = pools[i];
		const int pairs = u.kind ? ns : np;
		long long most = u.unit_bytes;
		if (!u.kind && u.row_bytes > 0 && pr) { // CTAs only for the longest of the parts
			long long rows = 0;
			for (int k = 0; k < np; ++k) rows = std::max<long long>(rows, pr[k]);
			most = std::min(most, rows * u.row_bytes);
		}
		if (!pairs || !most) continue;
		const long long chunks = (most + COPY_CHUNK - 1) / COPY_CHUNK;
		a.pool[a.pools++] = CopyPool{(const char*)u.src, (char*)u.dst, u.unit_bytes, u.row_bytes, (unsigned)ctas, (unsigned)chunks, u.kind};
		ctas += chunks * pairs;
	}
	if (!ctas) return cudaSuccess;
	if (ctas > 0x7fffffff) return cudaErrorInvalidValue;
	for (int k = 0; k < np; ++k) a.from[k] = pf[k], a.to[k] = pt[k], a.rows[k] = pr ? pr[k] : -1;
	for (int k = 0; k < ns; ++k) a.from[np + k] = sf[k], a.to[np + k] = st[k];
	return launch(stream, false, 1, k_copy_units<PAIRS>, dim3((unsigned)ctas), dim3(COPY_THREADS), 0, a);
}

// a destination named twice, a source among them (same pool only), a unit that is not there
int check_lists(const char* what, int n, const int* from, const int* to, int src_units, int dst_units, bool same) {
	std::vector<unsigned char> seen((size_t)std::max(src_units, dst_units), 0);
	for (int i = 0; i < n; ++i) {
		if (from[i] < 0 || from[i] >= src_units) return refuse("copy: %s %d is not in a pool of %d", what, from[i], src_units);
		if (to[i] < 0 || to[i] >= dst_units) return refuse("copy: %s %d is not in a pool of %d", what, to[i], dst_units);
		if (seen[to[i]] & 1) return refuse("copy: %s %d is written twice", what, to[i]);
		seen[to[i]] |= 1;
	}
	if (same)
		for (int i = 0; i < n; ++i)
			if (seen[from[i]] & 1) return refuse("copy: %s %d is read and written", what, from[i]);
	return 0;
}

int copy_units(int n_pools, const SeqUnits* pools, int np, const int* pf, const int* pt, const int* pr, int ns, const int* sf, const int* st, cudaStream_t stream) {
	if (n_pools < 0 || np < 0 || ns < 0 || (n_pools && !pools) || (np && (!pf || !pt)) || (ns && (!sf || !st))) return refuse("copy: a list is missing");
	for (int i = 0; i < n_pools; ++i) {
		const SeqUnits& u = pools[i];
		const int pairs = u.kind ? ns : np;
		if (u.kind < 0 || u.kind > 1) return refuse("copy: pool %d has kind %d", i, u.kind);
		if (u.unit_bytes < 0 || u.row_bytes < 0 || u.row_bytes > u.unit_bytes || u.src_units < 0 || u.dst_units < 0) return refuse("copy: pool %d has negative sizes, or rows wider than its units", i);
		if (pairs && u.unit_bytes && (!u.src || !u.dst)) return refuse("copy: pool %d has no memory", i);
		if (u.unit_bytes > (1LL << 38)) return refuse("copy: units of pool %d are larger than 256 GB", i);
		const uintptr_t s0 = (uintptr_t)u.src, d0 = (uintptr_t)u.dst;
		const unsigned __int128 sn = (unsigned __int128)u.unit_bytes * u.src_units, dn = (unsigned __int128)u.unit_bytes * u.dst_units; // (units that are not used may be named beyond what 64 bits count)
		if (s0 != d0 && s0 < d0 + dn && d0 < s0 + sn) return refuse("copy: source and destination of pool %d overlap", i);
		bool known = false; // pools of one shape are checked once
		for (int j = 0; j < i && !known; ++j)
			known = pools[j].kind == u.kind && pools[j].src_units == u.src_units && pools[j].dst_units == u.dst_units && (pools[j].src == pools[j].dst) == (u.src == u.dst);
		if (!known)
			if (const int rc = check_lists(u.kind ? "slot" : "page", pairs, u.kind ? sf : pf, u.kind ? st : pt, u.src_units, u.dst_units, u.src == u.dst)) return rc;
	}
	if (pr)
		for (int k = 0; k < np; ++k)
			if (pr[k] < 0) return refuse("copy: page %d has %d rows", pf[k], pr[k]);
	for (int p0 = 0; p0 < n_pools; p0 += COPY_POOLS) {
		const int pn = std::min(COPY_POOLS, n_pools - p0);
		for (int a0 = 0, b0 = 0; a0 < np || b0 < ns;) { // few pairs travel in a small parameter block
			const int an = std::min(COPY_PAIRS, np - a0), bn = std::min(COPY_PAIRS - an, ns - b0);
			cudaError_t e = an + bn <= 64 ? copy_launch<64>(pools + p0, pn, pf + a0, pt + a0, pr ? pr + a0 : nullptr, an, sf + b0, st + b0, bn, stream)
			                              : copy_launch<COPY_PAIRS>(pools + p0, pn, pf + a0, pt + a0, pr ? pr + a0 : nullptr, an, sf + b0, st + b0, bn, stream);
			if (e != cudaSuccess) return failed("copy", e);
			a0 += an, b0 += bn;
		}
	}
	return 0;
}
} // namespace
} // namespace seqops

extern "C" const char* calm_b200_seq_error(void) { return seqops::g_message; }

extern "C" int calm_b200_seq_copy_units(int n_pools, const struct SeqUnits* pools, int n_pages, const int* page_from, const int* page_to, const int* page_rows, int n_slots,
                                        const int* slot_from, const int* slot_to, void* stream) {
	try {
		return seqops::copy_units(n_pools, pools, n_pages, page_from, page_to, page_rows, n_slots, slot_from, slot_to, (cudaStream_t)stream);
	} catch (const std::bad_alloc&) {
		return seqops::refuse("copy: no host memory for the lists");
	}
}
