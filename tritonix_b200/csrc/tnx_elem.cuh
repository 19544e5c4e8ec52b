// Element access shared by the row kernels (norms, routing, combination of expert outputs):
// values of any of the library's three types move as vectors of VEC elements (16 bytes at most)
// and are computed in fp32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace tnx {
namespace elem {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// VEC consecutive elements as they lie in memory.  Vectors of up to 16 bytes are one access;
// longer ones (eight fp32 values next to eight 16-bit ones) are several of 16 bytes.
template <typename T, int VEC>
struct alignas((sizeof(T) * VEC) < 16 ? sizeof(T) * VEC : 16) Pack {
  T v[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ void load(const T* p, float (&out)[VEC]) {
  const Pack<T, VEC> raw = *reinterpret_cast<const Pack<T, VEC>*>(p);
#pragma unroll
  for (int i = 0; i < VEC; ++i) out[i] = to_float(raw.v[i]);
}
template <typename T, int VEC>
__device__ __forceinline__ void store(T* p, const float (&in)[VEC]) {
  Pack<T, VEC> raw;
#pragma unroll
  for (int i = 0; i < VEC; ++i) raw.v[i] = from_float<T>(in[i]);
  *reinterpret_cast<Pack<T, VEC>*>(p) = raw;
}

}  // namespace elem

// Programmatic stream serialization: a kernel launched with it may start while the kernel before
// it in the stream still runs; dependency_wait() returns once that kernel's writes are visible.
// Every kernel that is launched this way calls it before its first global access, so a chain of
// them stays ordered.
__device__ __forceinline__ void dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void dependency_release() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

}  // namespace tnx
