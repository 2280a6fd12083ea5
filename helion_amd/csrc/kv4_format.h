// The 4-bit key/value cache: its number format, its layout and the conversions the kernels share.
//
// Numbers: blocks of 32 consecutive elements of a head share a scale 2^E, E = floor(log2 max|x|) - 2 held as the byte
// E + 127 (E is clamped to -126 .. 125, so the bytes 1 .. 252 occur; a block of zeros has byte 1, a block with an infinity
// or a NaN has byte 255, which stands for NaN throughout).  An element is a 4-bit float (sign, two bits of exponent, one
// of mantissa: 0, 0.5, 1, 1.5, 2, 3, 4, 6) nearest to x / 2^E, ties to the even code; the quotients between 6 and 8 that
// the rule for E leaves become 6.  This is the open MXFP4 format, which the conversion instructions below work on.
//
// Layout (one allocation each, pages of `page` tokens, page a power of two from 16 to 1024):
//   k codes  [pages][heads][page][D/2]            byte b of a token holds elements 2b (low half) and 2b+1
//   k scales [pages][heads][page][D/32]
//   v codes  [pages][heads][page/4][16][4][D/32]  groups of four tokens: piece r of a token is its elements r*D/16 ..
//   v scales [pages][heads][page/4][D/32][4]
// The keys of 16 tokens are the rows of a matrix operand whose lanes hold consecutive elements of one token; the values
// are an operand whose lanes hold consecutive tokens of one element.  With four tokens of a piece side by side a lane
// gets both from wide loads straight into registers, and the lane that holds piece r needs one dword of four scales.
#pragma once
#include "hx_common.h"

typedef __bf16 v2bf __attribute__((ext_vector_type(2)));

// The conversions take a scale from the exponent field of an fp32 number and from nothing else (sign and mantissa measured
// not to matter), so a byte is shifted into place and whatever stands beside it stays.
__device__ __forceinline__ float kv4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }
__device__ __forceinline__ float kv4_scale_of(uint32_t four, int i) {  // byte i of four
  return __uint_as_float(i < 3 ? four << (23 - 8 * i) : four >> 1);
}

// two elements of byte SEL of `codes` times the scale
template <int SEL>
__device__ __forceinline__ v2f kv4_pair_f32(uint32_t codes, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, SEL);
}
template <int SEL>
__device__ __forceinline__ v2bf kv4_pair_bf16(uint32_t codes, float scale) {  // exact: one bit of mantissa
  return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, SEL);
}

// the scale byte of a block whose largest |x| has the pattern `top`
__device__ __forceinline__ uint32_t kv4_scale_byte(uint32_t top) {
  if (top >= 0x7F800000u) return 255;
  const int byte = (int)(top >> 23) - 2;
  return (uint32_t)(byte < 1 ? 1 : byte);
}
