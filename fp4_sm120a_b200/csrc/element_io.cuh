// Element types of the element-wise kernels (fp32, bf16, fp16): conversion to
// and from fp32, and groups of four moved as one vector where the tensor's
// alignment allows (`full`), else element by element below the end `n`; pairs
// of fp32.
#pragma once

#include <cstdint>
#include <type_traits>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace nvfp4 {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// Two values in one 32-bit word (16-bit types), the first in the low half.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b);
template <>
__device__ __forceinline__ void unpack2<__nv_bfloat16>(uint32_t w, float& a, float& b) {
  a = __uint_as_float(w << 16);
  b = __uint_as_float(w & 0xFFFF0000u);
}
template <>
__device__ __forceinline__ void unpack2<__half>(uint32_t w, float& a, float& b) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  a = f.x;
  b = f.y;
}

// 1 / x and 2^x to a few 2^-23, subnormal arguments and results taken as zero: the
// full-range forms spend more instructions on those than on the result.
__device__ __forceinline__ float fast_rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float fast_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Maximum of the magnitudes of two pairs of 16-bit values, NaN if one is; the
// results' signs mean nothing.
template <typename T>
__device__ __forceinline__ uint32_t max_abs2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (std::is_same_v<T, __half>)
    asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else
    asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Pairs of fp32 in one instruction (add / mul / fma.rn.f32x2).
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void split(uint64_t p, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
template <typename T>
__device__ __forceinline__ void load4(const T* p, uint64_t i, uint64_t n, bool full,
                                      float (&x)[4]) {
  if (full) {
    if constexpr (sizeof(T) == 4) {
      const float4 f = *reinterpret_cast<const float4*>(p + i);
      x[0] = f.x; x[1] = f.y; x[2] = f.z; x[3] = f.w;
    } else {
      const uint2 w = *reinterpret_cast<const uint2*>(p + i);
      unpack2<T>(w.x, x[0], x[1]);
      unpack2<T>(w.y, x[2], x[3]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = i + k < n ? to_f32(p[i + k]) : 0.0f;
  }
}

template <typename T>
__device__ __forceinline__ void store4(T* p, uint64_t i, uint64_t n, bool full,
                                       const float (&x)[4]) {
  if (full) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(p + i) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
      *reinterpret_cast<uint2*>(p + i) = make_uint2(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]));
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i + k < n) p[i + k] = from_f32<T>(x[k]);
  }
}

__device__ __forceinline__ uint32_t load4_bytes(const uint8_t* p, uint64_t i, uint64_t n,
                                                bool full) {
  if (full) return *reinterpret_cast<const uint32_t*>(p + i);
  uint32_t w = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (i + k < n) w |= (uint32_t)p[i + k] << (8 * k);
  return w;
}
__device__ __forceinline__ void store4_bytes(uint8_t* p, uint64_t i, uint64_t n, bool full,
                                             uint32_t w) {
  if (full) {
    *reinterpret_cast<uint32_t*>(p + i) = w;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i + k < n) p[i + k] = (uint8_t)(w >> (8 * k));
  }
}

}  // namespace nvfp4
