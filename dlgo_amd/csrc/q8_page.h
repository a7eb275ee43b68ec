// The page of the 8-bit cache, shared by the kernel that writes it and the kernels that read it.
//
// A page holds 64 tokens.  Each kv head has 128 * (hd + 1) consecutive bytes of it:
//   keys    64 * hd  e4m3: byte (t * P + p) * 256 + 16 i + e        of token 16 t + i, element 16 p + e   (P = hd / 16)
//   values  64 * hd  e4m3: byte ((c * 4 + g) * 16 + i) * 16 + 4 t + r of token 16 t + 4 g + r, element 16 c + i
//   scales  64 bytes of the keys:   byte 4 i + t        of token 16 t + i
//           64 bytes of the values: byte 16 g + 4 t + r of token 16 t + 4 g + r
// An element is its e4m3 value times 2^(scale - 127), one power for a token's key (value) of a head: e4m3 is a floating
// format, so a finer scale than a power of two would gain nothing but the last half binade, and with a power of two
// every dequantised element is a bfloat16 number exactly (4 significant bits), so that nothing is rounded a second time
// on the way into the matrix instructions.
//
// Why this order: in the matrix product of 16 x 16 x 32, lane 16 g + i of the first operand holds 8 consecutive steps of
// the inner axis of row i.  With keys as rows (inner axis: the head) and with values as rows (inner axis: the tokens,
// in the order in which the product of the scores left them in the lanes), both operands of a page are then what one
// load of 16 bytes a lane, 1 KB in a row per wave, brings: no transposition, no shuffle, no trip through LDS.
//
// The keys' scale 255 (e8m0's NaN) marks a token whose key or value is not finite: whatever sees it becomes NaN, and
// the bytes themselves are never NaN, so that a weight of zero takes nothing from a token that a row must not see.
#pragma once
#include "common.h"

#define Q8_PAGE 64
#define Q8_NAN 255

__host__ __device__ __forceinline__ constexpr long long q8_head_bytes(int hd) { return 128ll * (hd + 1); }

// 2^(b - 127) as a float; b = 0 (2^-127) is written by nobody and reads as 0
__device__ __forceinline__ float q8_scale(uint32_t b) { return __uint_as_float(b << 23); }

// What the writers share.  The largest magnitude of eight elements, as a float's bits.
__device__ __forceinline__ uint32_t q8_top_bits(const float* y) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t b = __float_as_uint(y[e]) & 0x7fffffffu;
    m = b > m ? b : m;
  }
  return m;
}

// the least e with (the float of these bits) <= 448 * 2^e = 1.75 * 2^(8 + e), not below -126
__device__ __forceinline__ int q8_power_for(uint32_t top) {
  const int e = (int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < -126 ? -126 : e;
}

__device__ __forceinline__ uint2 q8_to_e4m3(const float* y, int power) {
  const float f = __uint_as_float((uint32_t)(127 - power) << 23);          // 2^-power: power is -126 to 121
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0] * f, y[1] * f, lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2] * f, y[3] * f, lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4] * f, y[5] * f, hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6] * f, y[7] * f, hi, true);
  return make_uint2((uint32_t)lo, (uint32_t)hi);
}
