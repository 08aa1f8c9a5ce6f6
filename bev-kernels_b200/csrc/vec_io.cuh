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

// VEC elements as the 32-bit words (one 16-bit half where there is only that)
// they are loaded in; at most 16 bytes.
template <typename T, int VEC>
struct Pack {
  static constexpr int kBytes = sizeof(T) * VEC;
  static_assert(kBytes == 2 || kBytes == 4 || kBytes == 8 || kBytes == 16, "one load");
  static constexpr int kWords = kBytes < 4 ? 1 : kBytes / 4;
  uint32_t w[kWords];
};

template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack(const void *p) {
  using P = Pack<T, VEC>;
  P q;
  if constexpr (P::kBytes == 16) {
    const uint4 v = *static_cast<const uint4 *>(p);
    q.w[0] = v.x; q.w[1] = v.y; q.w[2] = v.z; q.w[3] = v.w;
  } else if constexpr (P::kBytes == 8) {
    const uint2 v = *static_cast<const uint2 *>(p);
    q.w[0] = v.x; q.w[1] = v.y;
  } else if constexpr (P::kBytes == 4) {
    q.w[0] = *static_cast<const uint32_t *>(p);
  } else {
    q.w[0] = *static_cast<const uint16_t *>(p);
  }
  return q;
}
template <typename T, int VEC>
__device__ __forceinline__ void store_pack(void *p, const Pack<T, VEC> &q) {
  using P = Pack<T, VEC>;
  if constexpr (P::kBytes == 16)
    *static_cast<uint4 *>(p) = make_uint4(q.w[0], q.w[1], q.w[2], q.w[3]);
  else if constexpr (P::kBytes == 8)
    *static_cast<uint2 *>(p) = make_uint2(q.w[0], q.w[1]);
  else if constexpr (P::kBytes == 4)
    *static_cast<uint32_t *>(p) = q.w[0];
  else
    *static_cast<uint16_t *>(p) = static_cast<uint16_t>(q.w[0]);
}

// The same for data that is not read again soon: it leaves L2 first.
template <typename T, int VEC>
__device__ __forceinline__ void store_pack_streaming(void *p, const Pack<T, VEC> &q) {
  using P = Pack<T, VEC>;
  if constexpr (P::kBytes == 16)
    __stcs(static_cast<uint4 *>(p), make_uint4(q.w[0], q.w[1], q.w[2], q.w[3]));
  else if constexpr (P::kBytes == 8)
    __stcs(static_cast<uint2 *>(p), make_uint2(q.w[0], q.w[1]));
  else
    store_pack<T, VEC>(p, q);
}

__device__ __forceinline__ float2 widen2(uint32_t w, __half) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
__device__ __forceinline__ float2 widen2(uint32_t w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ uint32_t narrow2(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t narrow2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}

template <typename T, int VEC>
__device__ __forceinline__ void unpack(const Pack<T, VEC> &q, float (&f)[VEC]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = __uint_as_float(q.w[i]);
  } else if constexpr (VEC == 1) {
    f[0] = widen2(q.w[0], T()).x;
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      const float2 v = widen2(q.w[i], T());
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
}
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> pack(const float (&f)[VEC]) {
  Pack<T, VEC> q;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) q.w[i] = __float_as_uint(f[i]);
  } else if constexpr (VEC == 1) {
    q.w[0] = narrow2(f[0], 0.f, T());
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) q.w[i] = narrow2(f[2 * i], f[2 * i + 1], T());
  }
  return q;
}
template <typename T, int VEC>
__device__ __forceinline__ void store(T *p, const float (&f)[VEC]) {
  store_pack<T, VEC>(p, pack<T, VEC>(f));
}

// Two fp32 values in one 64-bit register: Blackwell's packed arithmetic does
// both in one instruction, each rounded as on its own.
struct Two {
  unsigned long long v;
};
__device__ __forceinline__ Two two(float a, float b) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ Two two(float a) { return two(a, a); }
__device__ __forceinline__ float2 split(Two a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
// the same with subnormal operands and results taken as zero
__device__ __forceinline__ Two fma2_ftz(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two add2(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

// A vector as pairs; a single element (VEC == 1) has 0 beside it.
template <int VEC>
constexpr int kPairsOf = VEC == 1 ? 1 : VEC / 2;
template <typename T, int VEC>
__device__ __forceinline__ void unpack2(const Pack<T, VEC> &q, Two (&f)[kPairsOf<VEC>]) {
#pragma unroll
  for (int i = 0; i < kPairsOf<VEC>; ++i) {
    if constexpr (sizeof(T) == 4) {
      f[i] = two(__uint_as_float(q.w[2 * i]),
                 VEC == 1 ? 0.f : __uint_as_float(q.w[VEC == 1 ? 0 : 2 * i + 1]));
    } else {
      const float2 v = widen2(q.w[i], T());
      f[i] = two(v.x, VEC == 1 ? 0.f : v.y);
    }
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void store2(T *p, const Two (&f)[kPairsOf<VEC>]) {
  Pack<T, VEC> q;
#pragma unroll
  for (int i = 0; i < kPairsOf<VEC>; ++i) {
    const float2 v = split(f[i]);
    if constexpr (sizeof(T) == 4) {
      q.w[VEC == 1 ? 0 : 2 * i] = __float_as_uint(v.x);
      if constexpr (VEC > 1) q.w[2 * i + 1] = __float_as_uint(v.y);
    } else {
      q.w[i] = narrow2(v.x, v.y, T());
    }
  }
  store_pack<T, VEC>(p, q);
}

// Stores a scalar as the type chosen at run time (fp32, fp16 or bf16).
__device__ __forceinline__ void store_any(void *p, int64_t i, int dtype, float v) {
  switch (dtype) {
    case 1: static_cast<__half *>(p)[i] = __float2half_rn(v); break;
    case 2: static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v); break;
    default: static_cast<float *>(p)[i] = v;
  }
}

// VEC parameters from element i on, as loaded: the conversion waits until they
// are used, so that the loads stay in flight.  With `vectors` p + i is on a
// boundary of 16 bytes (or of all VEC elements, if those are fewer bytes).
template <int VEC>
struct Params {
  uint32_t w[VEC];  // fp32: one each; 16-bit: two each
};
template <int VEC>
__device__ __forceinline__ Params<VEC> load_params(const void *p, int64_t i, int dtype,
                                                   bool vectors) {
  Params<VEC> q;
#pragma unroll
  for (int e = 0; e < VEC; ++e) q.w[e] = 0;
  if (p == nullptr) return q;
  if (dtype == 0) {
    const uint32_t *f = static_cast<const uint32_t *>(p) + i;
    if (VEC >= 4 && vectors) {
#pragma unroll
      for (int e = 0; e + 4 <= VEC; e += 4) {
        const uint4 v = *reinterpret_cast<const uint4 *>(f + e);
        q.w[e] = v.x; q.w[e + 1] = v.y; q.w[e + 2] = v.z; q.w[e + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) q.w[e] = f[e];
    }
  } else {
    const uint16_t *h = static_cast<const uint16_t *>(p) + i;
    if (VEC == 8 && vectors) {
      const uint4 v = *reinterpret_cast<const uint4 *>(h);
      q.w[0] = v.x; q.w[1 % VEC] = v.y; q.w[2 % VEC] = v.z; q.w[3 % VEC] = v.w;
    } else if (VEC == 4 && vectors) {
      const uint2 v = *reinterpret_cast<const uint2 *>(h);
      q.w[0] = v.x; q.w[1 % VEC] = v.y;
    } else {
      uint32_t u[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) u[e] = h[e];
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (e % 2 == 0) q.w[e / 2] = u[e] | (e + 1 < VEC ? u[(e + 1) % VEC] << 16 : 0u);
    }
  }
  return q;
}
template <int VEC>
__device__ __forceinline__ void params_to_float(const Params<VEC> &q, const void *p, int dtype,
                                                float none, float (&f)[VEC]) {
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    const uint32_t pair = q.w[e / 2];
    const uint32_t h = e % 2 ? pair >> 16 : pair & 0xffffu;
    f[e] = p == nullptr ? none
           : dtype == 0 ? __uint_as_float(q.w[e])
           : dtype == 1 ? __half2float(__ushort_as_half(static_cast<uint16_t>(h)))
                        : __uint_as_float(h << 16);
  }
}

// Asynchronous copies of 4, 8 or 16 bytes from global to shared memory, in
// groups that complete in order.
template <int BYTES>
__device__ __forceinline__ void copy_async(void *smem, const void *global) {
  static_assert(BYTES == 4 || BYTES == 8 || BYTES == 16, "one copy");
  const auto to = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(global) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(global), "n"(BYTES)
                 : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Waits until at most `pending` (0 to 7) of the thread's groups are not complete.
__device__ __forceinline__ void copy_wait(int pending) {
  switch (pending) {
    case 0: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
    case 1: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
    case 2: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
    case 3: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
    case 4: asm volatile("cp.async.wait_group 4;" ::: "memory"); break;
    case 5: asm volatile("cp.async.wait_group 5;" ::: "memory"); break;
    case 6: asm volatile("cp.async.wait_group 6;" ::: "memory"); break;
    default: asm volatile("cp.async.wait_group 7;" ::: "memory");
  }
}

}  // namespace vio
}  // namespace bevk
