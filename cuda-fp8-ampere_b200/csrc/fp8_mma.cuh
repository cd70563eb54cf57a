// FP8 bytes as fp16 operands of mma.sync, shared by the decode-step operators
// (attention over the 8-bit cache, experts' products). Every E4M3FN and E5M2
// value is an fp16 value, so the conversion is exact; scales stay in fp32,
// outside the products.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

namespace fp8imma_dev {

enum { F8_E4M3 = 0, F8_E5M2 = 1 };

// two FP8 bytes (low 16 bits) -> f16x2
template <int FMT>
__device__ __forceinline__ uint32_t f8x2_to_f16x2(uint16_t two) {
  uint32_t r;
  if (FMT == F8_E4M3)
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(two));
  else
    asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(r) : "h"(two));
  return r;
}

// four FP8 bytes -> f16x2 of bytes 0,1 and of bytes 2,3
template <int FMT>
__device__ __forceinline__ void f8x4_to_f16x4(uint32_t x, uint32_t& lo, uint32_t& hi) {
  if (FMT == F8_E4M3) {
    lo = f8x2_to_f16x2<FMT>((uint16_t)(x & 0xFFFFu));
    hi = f8x2_to_f16x2<FMT>((uint16_t)(x >> 16));
  } else {  // E5M2 is the high byte of fp16
    lo = __byte_perm(x, 0u, 0x1404);
    hi = __byte_perm(x, 0u, 0x3424);
  }
}

template <int FMT>
__device__ __forceinline__ float f8_to_f32(uint8_t b) {
  return __half2float(__ushort_as_half((uint16_t)(f8x2_to_f16x2<FMT>(b) & 0xFFFFu)));
}

// fp32 -> FP8, to nearest even, saturating
template <int FMT>
__device__ __forceinline__ uint16_t f32x2_to_f8x2(float lo, float hi) {
  uint16_t two;
  if (FMT == F8_E4M3)
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(two) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(two) : "f"(hi), "f"(lo));
  return two;
}

// 16-bit activation (A_F16 = 0 / A_BF16 = 1) -> fp32
template <int AT>
__device__ __forceinline__ float a16_to_f32(uint16_t b) {
  return AT == 0 ? __half2float(__ushort_as_half(b)) : __uint_as_float((uint32_t)b << 16);
}
template <int AT>
__device__ __forceinline__ uint16_t f32_to_a16(float v) {
  return AT == 0 ? __half_as_ushort(__float2half_rn(v)) : __bfloat16_as_ushort(__float2bfloat16_rn(v));
}

// two fp32 values -> two 16-bit activations, lo in the low half
template <int AT>
__device__ __forceinline__ uint32_t f32x2_to_a16x2(float lo, float hi) {
  uint32_t r;
  if (AT == 0)
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

}  // namespace fp8imma_dev
