// vec_io.cuh -- element types as vectors of floats: loads and stores of VEC
// consecutive elements (16 bytes where VEC is the type's full vector), values
// widened to fp32 on the way in and rounded once on the way out.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace bevk {
namespace vio {

template <typename T>
struct Full {  // elements in 16 bytes
  static constexpr int value = 16 / sizeof(T);
};

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ float narrow<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// A vector of VEC elements, aligned to its own size.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack(const T *p) {
  return *reinterpret_cast<const Pack<T, VEC> *>(p);
}
template <typename T, int VEC>
__device__ __forceinline__ void unpack(const Pack<T, VEC> &q, float (&f)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) f[i] = widen(q.v[i]);
}
template <typename T, int VEC>
__device__ __forceinline__ void store(T *p, const float (&f)[VEC]) {
  Pack<T, VEC> q;
#pragma unroll
  for (int i = 0; i < VEC; ++i) q.v[i] = narrow<T>(f[i]);
  *reinterpret_cast<Pack<T, VEC> *>(p) = q;
}

// A scalar of the parameter type chosen at run time (fp32, fp16 or bf16).
__device__ __forceinline__ float load_any(const void *p, int64_t i, int dtype) {
  switch (dtype) {
    case 1: return __half2float(static_cast<const __half *>(p)[i]);
    case 2: return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
    default: return static_cast<const float *>(p)[i];
  }
}
__device__ __forceinline__ void store_any(void *p, int64_t i, int dtype, float v) {
  switch (dtype) {
    case 1: static_cast<__half *>(p)[i] = __float2half_rn(v); break;
    case 2: static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v); break;
    default: static_cast<float *>(p)[i] = v;
  }
}

}  // namespace vio
}  // namespace bevk
