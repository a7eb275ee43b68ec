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
