// How a quantised key or value cache holds a row of `dim` channels.
//
// A group of channels -- the row where codes have 8 bits, 32 channels where they
// have 4 -- shares a scale: the smallest bfloat16 s >= 2^-100 with M s >= the
// group's largest magnitude, M = 127 or 7; a code is x / s rounded to nearest,
// ties to even, and stands for code * s, a product that fp32 holds exactly (but
// where M = 7 and a magnitude lies above 3.396e38: 7 s is then beyond fp32, infinity).
// A group with an infinity or NaN has the scale NaN (and codes 0).
//
// Rows are padded to a pitch P of channels (zeros).  Eight bits: a byte per
// channel, in order.  Four bits: nibbles of code + 8 in the order in which the
// attention kernel's lanes take them, 16 lanes or 4 x 16 lanes to a row:
//   keys: lane group g of 4 holds P/8 bytes, a dword for each 32 channels c, of
//     channels 32c + 8g + j; nibble n of the dword is j = 2 (n % 4) + n / 4;
//   values: lane r of 16 holds P/32 bytes, one for each 32 channels c, of
//     channels 32c + 2r (low nibble) and 32c + 2r + 1.
#pragma once
#include "common.h"

namespace qa {

inline int64_t cache_pitch(int64_t dim) {
  for (const int64_t p : {32, 64, 96, 128, 192, 256})
    if (dim <= p) return p;
  return 0;
}

inline int64_t cache_groups(int64_t pitch, int bits) { return bits == 8 ? 1 : pitch / 32; }
inline int64_t cache_row_bytes(int64_t pitch, int bits) { return pitch * bits / 8; }

// The scale's bfloat16 bits for a largest magnitude; `most` is 127 or 7.
__device__ __forceinline__ uint32_t scale_bits(float amax, float most) {
  if (!(amax <= 3.4028234663852886e38f)) return 0x7fc0u;  // infinity or NaN
  // the rounded quotient upwards; one step more where it was rounded down onto a bfloat16 (M s is exact)
  uint32_t s = (__float_as_uint(amax / most) + 0xffffu) >> 16;
  if (s < 0x0d80u) s = 0x0d80u;  // 2^-100
  if (most * __uint_as_float(s << 16) < amax) s++;
  return s;
}

// x / s rounded to nearest, ties to even, as a float: an estimate, and its exact remainder.
__device__ __forceinline__ float code_of(float x, float s, float inverse) {
  const float q = rintf(x * inverse), rest = fmaf(-q, s, x), twice = 2.f * fabsf(rest);
  const bool off = twice > s || (twice == s && ((int)q & 1));
  return off ? q + copysignf(1.f, rest) : q;
}
// The same where x is a bfloat16: x and s have 8 bits each, so a quotient that is
// no tie lies 2^-9 off it at least, and one step of 2^-11 takes away the estimate's error.
__device__ __forceinline__ float code_of_bf16(float x, float inverse) {
  return rintf(fmaf(x, inverse, 6144.f) - 6144.f);
}
// The low byte of an integer's two's complement, |q| below 2^22, in the low byte of a float's bits.
__device__ __forceinline__ uint32_t low_byte(float q) { return __float_as_uint(q + 12582912.f); }

}  // namespace qa
