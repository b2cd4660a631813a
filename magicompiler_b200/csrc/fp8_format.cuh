// The block-scaled fp8 format that the quantisers write and the products read: e4m3 codes, one fp32 scale for 128 columns of a
// row, scale = max(max|x| / 448, 2^-126), code = e4m3(x / scale).
#pragma once
#include <stdint.h>

#include "ptx_sm100.cuh"

namespace magi {

constexpr float kFp8Max = 448.0f;               // largest e4m3 value
constexpr float kScaleFloor = 1.17549435e-38f;  // 2^-126: a block of zeros (or of subnormals) keeps a normal scale
constexpr float kScaleSmall = 0x1p-80f, kScaleLarge = 0x1p120f;  // see Divisor; no finite block has a larger scale

__device__ __forceinline__ float block_scale(float amax) {
  const float s = __fdiv_rn(amax, kFp8Max);
  return s < kScaleFloor ? kScaleFloor : s;  // a NaN stays
}
__device__ __forceinline__ uint32_t pack4_e4m3(float a, float b, float c, float d) {  // to nearest even, saturating, NaN stays
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}

// Pairs of fp32 values divided by s: x * r with r = 1 / s rounded, corrected by its own remainder (Markstein 1990: q + r * (x -
// q * s) with fused multiply-adds).  The remainder is exact and r off by 2^-24, so what the last step rounds is within 2^-22 of a
// unit in the last place of x / s: the IEEE quotient but for a chance in millions.  That holds for quotients that matter to an
// e4m3 code (above 2^-11) and s above kScaleSmall (the remainder's last bit is then above 2^-149).  s infinite: 0, of an infinity
// NaN.
struct Divisor {
  uint64_t r, minus_s;
  __device__ __forceinline__ explicit Divisor(float s) {
    const float inv = __frcp_rn(s), m = inv == 0.0f ? 0.0f : -s;
    r = pack_f32x2(inv, inv), minus_s = pack_f32x2(m, m);
  }
  __device__ __forceinline__ void divide(float& x0, float& x1) const {
    const uint64_t x = pack_f32x2(x0, x1), q = mul_f32x2(x, r);
    unpack_f32x2(fma_f32x2(r, fma_f32x2(q, minus_s, x), q), x0, x1);
  }
};
// What to multiply a small s and its block with so that s is above kScaleSmall (exact: all of them grow); 1 for any other s.
__device__ __forceinline__ float lift_of(float s) { return s < kScaleSmall ? 0x1p64f : 1.0f; }

}  // namespace magi
