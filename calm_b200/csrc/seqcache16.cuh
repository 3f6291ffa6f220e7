// seqcache16.cuh -- what storing into a paged cache in 16 bits (seqrotate.cu) and attention over it (seqattend16.cu) share on the host.
#pragma once

#include "seqops.cuh"

#include <limits.h>

#include <algorithm>
#include <type_traits>

namespace seqops {

inline int log2_of(int page) { // -1: no power of two
	int shift = 0;
	while (shift < 30 && 1 << shift < page) ++shift;
	return 1 << shift == page ? shift : -1;
}
inline int check_batch(const char* what, const SeqPortions* p) {
	if (!p) return refuse("%s: no batch", what);
	if (p->n < 0 || p->longest < 0 || p->n > 65535) return refuse("%s: %d sequences (at most 65535), longest %d", what, p->n, p->longest);
	if (p->n && (!p->start || !p->count || !p->slot || !p->pos0)) return refuse("%s: the batch's description is missing", what);
	if (((uintptr_t)p->start | (uintptr_t)p->count | (uintptr_t)p->slot | (uintptr_t)p->pos0) % 4) return refuse("%s: the batch's description is not aligned to 4 bytes", what);
	return 0;
}
inline int check_cache16(const char* what, const SeqCache16* q, const SeqPortions* p) {
	if (!q) return refuse("%s: no cache", what);
	if (q->type != SEQ_BF16 && q->type != SEQ_F16) return refuse("%s: a cache of type %d: bfloat16 or float16", what, q->type);
	if (q->pages < 0 || q->heads < 1 || q->page < 1 || q->slots < 0 || q->table_pages < 0) return refuse("%s: a cache of %d pages, %d heads, %d tokens a page", what, q->pages, q->heads, q->page);
	if (q->heads > 4096 || q->page > 65536) return refuse("%s: at most 4096 heads and 65536 tokens a page", what);
	if ((long long)q->pages * q->heads * q->page > INT_MAX) return refuse("%s: a pool of %d pages, %d heads, %d tokens a page has more than 2^31 rows", what, q->pages, q->heads, q->page);
	if (q->dim < 16 || q->dim > 256 || q->dim % 16) return refuse("%s: rows of %d channels: a multiple of 16 up to 256 is served", what, q->dim);
	if (q->pages && (!q->k || !q->v)) return refuse("%s: the cache has no memory", what);
	if (q->slots > 0 && q->table_pages > 0 && !q->table) return refuse("%s: the page table is missing", what);
	if (((uintptr_t)q->k | (uintptr_t)q->v) % 16) return refuse("%s: keys and values are not aligned to 16 bytes", what);
	if ((uintptr_t)q->table % 4) return refuse("%s: the page table is not aligned to 4 bytes", what);
	return check_batch(what, p);
}

} // namespace seqops
