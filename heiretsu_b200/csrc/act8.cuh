// The 8-bit activation format: device-side encoding and decoding.
//
// A row of N values is cut into blocks of 128 columns (the last may be shorter). A block is kept as one
// exponent byte and 128 signed codes:
//   e    = the least whole number >= -126 with max|x| <= 127 * 2^e;  byte = e + 127
//   code = x / 2^e rounded to the nearest whole number, ties to even (|code| <= 127);  value = code * 2^e
// Scaling by a power of two is exact, so the code's rounding is the only error: at most 2^e / 2 <= max|x| / 127
// per value, and the codes of a given input do not depend on the order of any arithmetic. A power of two
// costs up to one bit against a scale of max|x| / 127; in exchange the scale is one byte for 128 values and
// encoding needs no division. The bound goes by the block's largest value: a column 50 times larger than the other
// 127 leaves these off by 15% of their size, one 300 times larger by 70% and more (most codes 0). A block that holds an
// infinity or NaN gets byte 255 and comes back as NaN, so a broken activation still shows in the gradient norm.
#pragma once

#include "common.cuh"

namespace hb {

constexpr int kAct8Block = 128;
constexpr uint32_t kAct8Nan = 255;

// Exponent byte of a block from the bit pattern of max|x| (an unsigned maximum of |x|'s bits: infinity and
// NaN order above every finite value). With max|x| = 1.f * 2^(E - 127), 127 * 2^e = 1.984375 * 2^(e + 6): e + 127 is
// E - 6, plus one when 1.f > 1.984375, i.e. when the fraction field exceeds 0x7E0000 (the addition carries).
__device__ __forceinline__ uint32_t act8_byte(uint32_t max_bits) {
  if (max_bits >= 0x7F800000u) return kAct8Nan;
  const int b = static_cast<int>((max_bits + 0x1FFFFu) >> 23) - 6;
  return static_cast<uint32_t>(b < 1 ? 1 : b);
}
// 2^-e: a normal number for every byte of a finite block (1 .. 249); 0 for byte 255, whose codes are 0.
__device__ __forceinline__ float act8_inv_scale(uint32_t byte) {
  return byte == kAct8Nan ? 0.f : __uint_as_float((254u - byte) << 23);
}
__device__ __forceinline__ float act8_scale(uint32_t byte) {
  return byte == kAct8Nan ? __uint_as_float(0x7FC00000u) : __uint_as_float(byte << 23);
}
// Four codes, the first in the low byte. Rounding by adding 1.5 * 2^23: the sum's low byte is the code in two's
// complement (|x 2^-e| <= 127). Blocks with byte 255 get codes 0 (an infinity or NaN times 0 is NaN).
__device__ __forceinline__ uint32_t act8_codes(const float (&x)[4], uint32_t byte) {
  const float inv = act8_inv_scale(byte);
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = __float_as_uint(__fadd_rn(__fmul_rn(x[i], inv), 12582912.f));
  const uint32_t all = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
  return byte == kAct8Nan ? 0u : all;
}
// The farthest, in steps, that one of four values lies from its code (at most 1/2).
__device__ __forceinline__ float act8_off_code(const float (&x)[4], uint32_t byte) {
  const float inv = act8_inv_scale(byte);
  float off = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float t = __fmul_rn(x[i], inv);
    off = fmaxf(off, fabsf(t - (__fadd_rn(t, 12582912.f) - 12582912.f)));
  }
  return off;
}
// Their values. A byte, with its sign bit flipped, is code + 128; put under the exponent of 2^23 it reads as the
// number 2^23 + 128 + code, so one byte permutation and one subtraction give the code as a float.
__device__ __forceinline__ void act8_values(uint32_t codes, float scale, float (&v)[4]) {
  const uint32_t flipped = codes ^ 0x80808080u;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v[i] = (__uint_as_float(__byte_perm(flipped, 0x4B000000u, 0x7650u + i)) - 8388736.f) * scale;
}

}  // namespace hb
