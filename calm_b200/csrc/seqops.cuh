// seqops.cuh -- what the operators on callers' device memory (seqops.cu, seqbeam.cu, seqcache8.cu; entry points in include/calm_b200_seq.h) share:
// refusals that leave a message instead of ending the process, launches that report their error, element types.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>
#include <stdint.h>

#include <atomic>

#include "../../include/calm_b200_seq.h"
#include "common.cuh"
#include "tc05.cuh"

namespace seqops {

// -3 with a message for calm_b200_seq_error() / -4 for a CUDA error; both leave the process and the context as they were
int refuse(const char* fmt, ...);
int failed(const char* what, cudaError_t e);

void count_launch();
uint64_t launches(); // since the library was loaded

// how calm_b200_seq_attend8 cuts its work (a captured call keeps it): rows of a CTA, shares of the keys, chunks of each, whether clusters fold them
void attend8_plan(const SeqCache8& cache, const SeqPortions& batch, const SeqAttend8& args, int (&plan)[4]);

inline int cdiv(long long a, long long b) { return (int)((a + b - 1) / b); }

// Clusters of cluster_y CTAs along y.  `after`: programmatic dependent launch behind the previous kernel of the stream, which the kernel waits for with pdl_wait_prev()
template <typename... KArgs, typename... Args>
cudaError_t launch(cudaStream_t st, bool after, int cluster_y, void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, Args&&... args) {
	cudaLaunchConfig_t cfg = {};
	cfg.gridDim = grid, cfg.blockDim = block, cfg.dynamicSmemBytes = smem, cfg.stream = st;
	cudaLaunchAttribute at[2];
	int n = 0;
	if (after) at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization, at[n++].val.programmaticStreamSerializationAllowed = 1;
	if (cluster_y > 1) {
		at[n].id = cudaLaunchAttributeClusterDimension;
		at[n].val.clusterDim.x = 1, at[n].val.clusterDim.y = cluster_y, at[n++].val.clusterDim.z = 1;
	}
	cfg.attrs = at, cfg.numAttrs = n;
	count_launch();
	return cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);
}

// More than 48 KB of shared memory (and clusters of more than eight) for a kernel, asked for once on every device.
template <typename... KArgs>
cudaError_t allow(void (*kernel)(KArgs...), size_t smem, std::atomic<uint64_t>& done, bool wide_clusters = false) {
	int dev = 0;
	cudaError_t e = cudaGetDevice(&dev);
	if (e != cudaSuccess || (dev < 64 && (done.load(std::memory_order_acquire) >> dev & 1))) return e;
	e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
	if (e == cudaSuccess && wide_clusters) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
	if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev, std::memory_order_release);
	return e;
}

inline int type_size(int t) { return t == SEQ_F32 ? 4 : 2; }
inline bool type_ok(int t) { return t == SEQ_F32 || t == SEQ_BF16 || t == SEQ_F16; }

inline int check_rows(const char* what, const char* name, const SeqRows& r) {
	if (!type_ok(r.type)) return refuse("%s: %s has type %d", what, name, r.type);
	if (r.rows < 0 || (r.rows && !r.p)) return refuse("%s: %s is missing", what, name);
	if ((uintptr_t)r.p % type_size(r.type)) return refuse("%s: %s is not aligned to its type", what, name);
	return 0;
}

__device__ __forceinline__ float as_f32(float v) { return v; }
__device__ __forceinline__ float as_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float as_f32(__half v) { return __half2float(v); }
typedef unsigned long long u64;
// two fp32 operations in one instruction
__device__ __forceinline__ u64 pair_of(float x, float y) {
	u64 r;
	asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
	return r;
}
__device__ __forceinline__ float2 halves(u64 p) {
	float2 r;
	asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
	return r;
}
__device__ __forceinline__ u64 add2(u64 a, u64 b) {
	u64 r;
	asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
	return r;
}
__device__ __forceinline__ u64 mul2(u64 a, u64 b) {
	u64 r;
	asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
	return r;
}
__device__ __forceinline__ u64 fma2(u64 a, u64 b, u64 c) {
	u64 r;
	asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
	return r;
}
// 2^x to two steps; under 2^-126 zero
__device__ __forceinline__ float ex2(float x) {
	float r;
	asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
	return r;
}

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
// the elements of 16 bytes as floats
template <typename T>
__device__ __forceinline__ void unpack16(const uint4& w, float (&v)[16 / sizeof(T)]) {
	const T* p = reinterpret_cast<const T*>(&w);
#pragma unroll
	for (int i = 0; i < (int)(16 / sizeof(T)); ++i) v[i] = as_f32(p[i]);
}

__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); } // -126 <= e <= 127
__device__ __forceinline__ float load_as_f32(const void* p, int type, long long i) {
	return type == SEQ_F32 ? ((const float*)p)[i] : type == SEQ_BF16 ? as_f32(((const __nv_bfloat16*)p)[i]) : as_f32(((const __half*)p)[i]);
}
__device__ __forceinline__ void store_f32(void* p, int type, long long i, float v) {
	if (type == SEQ_F32) ((float*)p)[i] = v;
	else if (type == SEQ_BF16) ((__nv_bfloat16*)p)[i] = __float2bfloat16_rn(v);
	else ((__half*)p)[i] = __float2half_rn(v);
}
// a sink's term of the denominator against a reference that is no lower: none for -inf, all of it for +inf
__device__ __forceinline__ float at_sink(float sk, float top) { return sk == -INFINITY ? 0.f : sk == top ? 1.f : ex2(sk - top); }
// 16 bytes into shared memory, asynchronously
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
	asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool there) { // zeros where there is nothing to read
	asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
// an 8 x 8 tile of fp16, a row's pair of neighbours a thread, with rows and columns exchanged
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
	uint32_t r;
	asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
	return r;
}
// false: given up, here or by another thread of the block; no thread goes on then, and the rows come out as NaN
__device__ __forceinline__ bool ap_wait(uint64_t* bar, uint32_t parity, int* lost) {
	for (unsigned spins = 0; spins < MBAR_SPINS; ++spins) {
		if (mbar_try_wait(bar, parity)) return true;
		if ((spins & 63) == 63 && *(volatile int*)lost) return false;
	}
	*(volatile int*)lost = 1;
	return false;
}
__device__ __forceinline__ bool ap_wait_warp(uint64_t* bar, uint32_t parity, int* lost) { return __all_sync(0xffffffffu, ap_wait(bar, parity, lost)); }

} // namespace seqops
