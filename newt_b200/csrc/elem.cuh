// Element types as fp32 arithmetic sees them, 16-byte vectors of them, and conversions to e4m3.  Used by the norm, cache and log-probability kernels.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace nb200 {

template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static constexpr int kPerVec = 4;
  __device__ static float to_f32(float v) { return v; }
  __device__ static float from_f32(float v) { return v; }
};
template <>
struct Elem<__half> {
  static constexpr int kPerVec = 8;
  __device__ static float to_f32(__half v) { return __half2float(v); }
  __device__ static __half from_f32(float v) { return __float2half_rn(v); }
  __device__ static uint32_t pack2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct Elem<__nv_bfloat16> {
  static constexpr int kPerVec = 8;
  __device__ static float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
  __device__ static __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
  __device__ static uint32_t pack2(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

// One 16-byte vector of T, addressable both ways.
template <typename T>
union alignas(16) Vec {
  uint4 raw;
  T e[Elem<T>::kPerVec];
};

// Read once: no place in L1.  Not the read-only path, so that a kernel may write its result over
// the tensor it read it from.
__device__ __forceinline__ uint4 ld_once(const void* p) {
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}
__device__ __forceinline__ void st_once(void* p, uint4 v) {
  asm volatile("st.global.L1::no_allocate.v4.u32 [%0], {%1,%2,%3,%4};" ::"l"(p), "r"(v.x),
               "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
}

__host__ __device__ __forceinline__ bool at16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// kPerVec fp32 values as one vector of T, each rounded once.
template <typename T>
__device__ __forceinline__ Vec<T> round_elems(const float* v) {
  constexpr int E = Elem<T>::kPerVec;
  Vec<T> o;
  if constexpr (sizeof(T) == 2) {
    uint32_t* words = reinterpret_cast<uint32_t*>(&o.raw);   // two values per conversion
#pragma unroll
    for (int j = 0; j < E; j += 2) words[j / 2] = Elem<T>::pack2(v[j], v[j + 1]);
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j) o.e[j] = v[j];
  }
  return o;
}

// Two fp32 values as e4m3, `lo` in the low byte; beyond +-448 they become +-448, NaN stays NaN.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
      "mov.b32 %0, {lo, hi};\n\t}"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}
// Two e4m3 numbers (low byte first) as fp16, exactly.
__device__ __forceinline__ float2 e4m3x2_values(uint32_t q) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)q));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// Exponent of the smallest power of two s with most <= 448 s, 448 = 1.75 * 2^8 being e4m3's largest
// number: exact, from the bits.  0 and subnormals: -135 or -134.
__device__ __forceinline__ int e4m3_exponent(float most) {
  const uint32_t b = __float_as_uint(most);
  return (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // -126 to 127

// E values times `factor` as e4m3; `to` is E-byte aligned.
template <int E>
__device__ __forceinline__ void store_e4m3(uint8_t* to, const float* v, float factor) {
  uint32_t words[E / 4];
#pragma unroll
  for (int j = 0; j < E; j += 4)
    words[j / 4] = e4m3x4(v[j] * factor, v[j + 1] * factor, v[j + 2] * factor, v[j + 3] * factor);
  if constexpr (E == 8)
    *reinterpret_cast<uint2*>(to) = make_uint2(words[0], words[1]);
  else
    *reinterpret_cast<uint32_t*>(to) = words[0];
}

}  // namespace nb200
