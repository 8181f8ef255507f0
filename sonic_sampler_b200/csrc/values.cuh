// Value types of the decode-side kernels (cache, attention, norm): 16-bit and fp32 activations and
// e4m3 rows with an fp32 scale. Arithmetic is fp32; each conversion below rounds once, to nearest
// even.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace sonic {

constexpr float kE4m3Max = 448.0f;
constexpr float kScaleFloor = 8.673617379884035e-19f;  // 2^-60: smallest amax a row is scaled by

template <typename T>
struct Pair;  // packed pairs of a 16-bit type

template <>
struct Pair<__nv_bfloat16> {
  static __device__ __forceinline__ float2 unpack(uint32_t x) {
    return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
  }
};

template <>
struct Pair<__half> {
  static __device__ __forceinline__ float2 unpack(uint32_t x) {
    return __half22float2(*reinterpret_cast<const __half2*>(&x));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
  }
};

// two e4m3 codes (low byte first) of two fp32 values, to nearest even, finite values saturated
__device__ __forceinline__ uint32_t e4m3_pack2(float lo, float hi) {
  uint16_t d;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
  return d;
}

__device__ __forceinline__ uint32_t e4m3_pack4(float a, float b, float c, float d) {
  return e4m3_pack2(a, b) | (e4m3_pack2(c, d) << 16);
}

// two e4m3 codes to packed fp16 (exact)
__device__ __forceinline__ uint32_t e4m3_to_half2(uint16_t codes) {
  uint32_t d;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"(codes));
  return d;
}

// |x| as bits: ordered as the magnitudes are, with NaN above infinity, so that a maximum over
// these bits carries a NaN of the row into its scale
__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Scale of a row whose largest magnitude has these bits, and the factor that maps the row onto
// e4m3's range. Rows below 2^-60 (all-zero rows among them) are scaled as if they reached it.
__device__ __forceinline__ void e4m3_scale(uint32_t amax_bits, float& scale, float& inverse) {
  const uint32_t floor_bits = __float_as_uint(kScaleFloor);
  const float c = __uint_as_float(amax_bits > floor_bits ? amax_bits : floor_bits);
  scale = __fdiv_rn(c, kE4m3Max);
  inverse = __fdiv_rn(kE4m3Max, c);
}

__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_dependency_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

}  // namespace sonic
