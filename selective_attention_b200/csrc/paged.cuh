// paged.cuh - the 8-bit codes of the paged cache (paged.cu, paged_decode.cu).
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace ssdb200 {
namespace {

struct Int8 {};
struct E4M3 {};

// Eight codes in two words. Packing rounds to the nearest code (ties to even) and saturates at
// the largest one; a NaN becomes 0 as int8 (which has none) and NaN as e4m3.
template <typename C> struct Code;
template <> struct Code<Int8> {
  static constexpr float kPerMost = 1.0f / 127.0f;
  // Whether a quotient that is off by up to 3 * 2^-24 of itself may round to another code.
  static __device__ __forceinline__ bool unsure(float q) { return fabsf(q - rintf(q)) > 0.4999f; }
  static __device__ __forceinline__ unsigned pack1(float x) {
    // fmaxf / fminf would turn a NaN into a bound
    const float y = x == x ? fminf(fmaxf(rintf(x), -127.f), 127.f) : 0.f;
    return (unsigned)(int)y & 0xffu;
  }
  static __device__ __forceinline__ uint2 pack8(const float (&x)[8]) {
    uint2 w;
    w.x = pack1(x[0]) | pack1(x[1]) << 8 | pack1(x[2]) << 16 | pack1(x[3]) << 24;
    w.y = pack1(x[4]) | pack1(x[5]) << 8 | pack1(x[6]) << 16 | pack1(x[7]) << 24;
    return w;
  }
  static __device__ __forceinline__ void unpack8(uint2 w, float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = (float)(signed char)(w.x >> (8 * e));
      x[4 + e] = (float)(signed char)(w.y >> (8 * e));
    }
  }
};
template <> struct Code<E4M3> {
  static constexpr float kPerMost = 1.0f / 448.0f;
  // (codes have three mantissa bits: the middle between two is at bit 19; those below 2^-6 lie evenly)
  static __device__ __forceinline__ bool unsure(float q) {
    return (__float_as_uint(q) & 0xfffffu) - 0x7fff8u <= 16u || fabsf(q) < 0.01563f;
  }
  static __device__ __forceinline__ unsigned pack2c(float a, float b) {
    return (unsigned)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  }
  static __device__ __forceinline__ uint2 pack8(const float (&x)[8]) {
    uint2 w;
    w.x = pack2c(x[0], x[1]) | pack2c(x[2], x[3]) << 16;
    w.y = pack2c(x[4], x[5]) | pack2c(x[6], x[7]) << 16;
    return w;
  }
  static __device__ __forceinline__ void unpack2c(unsigned w, float& a, float& b) {
    const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
    const float2 f = __half22float2(__half2(r));
    a = f.x;
    b = f.y;
  }
  static __device__ __forceinline__ void unpack8(uint2 w, float (&x)[8]) {
    unpack2c(w.x, x[0], x[1]);
    unpack2c(w.x >> 16, x[2], x[3]);
    unpack2c(w.y, x[4], x[5]);
    unpack2c(w.y >> 16, x[6], x[7]);
  }
};

// Eight consecutive values, stored with 16-byte accesses.
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  uint4 w;
  w.x = pack2<T>(x[0], x[1]);
  w.y = pack2<T>(x[2], x[3]);
  w.z = pack2<T>(x[4], x[5]);
  w.w = pack2<T>(x[6], x[7]);
  *reinterpret_cast<uint4*>(p) = w;
}
template <>
__device__ __forceinline__ void store8<float>(float* p, const float (&x)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

// The same, eight fp32 values as one 32-byte sector where the address allows it.
template <typename T>
__device__ __forceinline__ void store8_wide(T* p, const float (&x)[8], bool wide) {
  if constexpr (sizeof(T) == 4) {
    if (wide) {
      asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(x[0]), "f"(x[1]), "f"(x[2]),
                   "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7])
                   : "memory");
      return;
    }
  }
  store8<T>(p, x);
}

}  // namespace
}  // namespace ssdb200
