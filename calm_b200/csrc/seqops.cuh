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

} // namespace seqops
