// Element types and small device helpers shared by the paged-cache and beam kernels.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace cv3p {

inline int type_size(int64_t type) { return type == CV3_TYPE_F32 ? 4 : 2; }
inline bool type_ok(int64_t type) { return type == CV3_TYPE_F32 || type == CV3_TYPE_F16 || type == CV3_TYPE_BF16; }
inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// element i of an array whose type is known at run time (single elements: queries, outputs)
__device__ __forceinline__ float load_any(const void* p, int type, int64_t i) {
  if (type == CV3_TYPE_F32) return static_cast<const float*>(p)[i];
  if (type == CV3_TYPE_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

__device__ __forceinline__ void store_any(void* p, int type, int64_t i, float x) {
  if (type == CV3_TYPE_F32) static_cast<float*>(p)[i] = x;
  else if (type == CV3_TYPE_F16) static_cast<__half*>(p)[i] = __float2half_rn(x);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
}

// N elements (N * sizeof(T) a multiple of 8, 16-byte pieces where it is one) between memory and fp32 registers
template <typename T, int N>
struct alignas(N * sizeof(T) >= 16 ? 16 : N * sizeof(T)) Vec {
  T v[N];
};

template <typename T, int N>
__device__ __forceinline__ void load_vec(const T* p, float (&x)[N]) {
  const Vec<T, N> r = *reinterpret_cast<const Vec<T, N>*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = to_f32<T>(r.v[i]);
}

template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[N]) {
  Vec<T, N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) r.v[i] = from_f32<T>(x[i]);
  *reinterpret_cast<Vec<T, N>*>(p) = r;
}

// cv3::launch_dep with a cluster of `cluster` CTAs along x
template <typename... KArgs, typename... Args>
cudaError_t launch_cluster(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, unsigned cluster, cudaStream_t st,
                           Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = cv3::dependent_launch_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// a float of another CTA of the cluster: `p` is the place of the same variable in this CTA
__device__ __forceinline__ float cluster_load(const float* p, unsigned rank) {
  uint32_t at;
  float x;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(at) : "memory");
  return x;
}

}  // namespace cv3p
