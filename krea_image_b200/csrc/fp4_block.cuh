// Rounding of bf16 values to e2m1 with a scale for each block, on packed pairs (two bf16 in a 32-bit word).
//
// e2m1 holds 0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign.  A magnitude becomes the nearest of the eight, a tie the one with
// the even code, 6 at most: its code is how many of the borders 0.25 0.75 1.25 1.75 2.5 3.5 5 it passes, where it has to
// be above the 1st, 3rd, 5th and 7th and may be equal to the others.
//
// MX (block of 32): scale 2^(floor(log2(amax)) - 2), 2^-127 at least, stored as its biased exponent.  x / scale only
// moves the exponent, so it is exact in f32, and the conversion instruction rounds once.
// NV (block of 16): scale s = e4m3(amax / (6 ts)), x / (s ts) is not exact.  A rounded quotient would decide ties and
// values next to a border by its own error, so x is compared with the borders b s ts instead: b s has seven bits, its
// product with ts rounded down (up) to bf16 decides x > border (x >= border) for a bf16 x without any error.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace krea {

constexpr uint32_t FP4_NAN_MX = 0xFFu, FP4_NAN_NV = 0x7Fu;   // scale codes that stand for NaN

// the larger of each 16-bit half, as unsigned integers: orders bf16 magnitudes, and puts NaN above infinity
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// bits of the largest magnitude among W words
template <int W>
__device__ __forceinline__ uint32_t amax_bits(const uint32_t* w) {
  uint32_t m = w[0] & 0x7FFF7FFFu;
#pragma unroll
  for (int i = 1; i < W; i++) m = max_u16x2(m, w[i] & 0x7FFF7FFFu);
  return max(m & 0xFFFFu, m >> 16);
}

// eight f32 -> eight e2m1 codes, the first in the low bits
__device__ __forceinline__ uint32_t cvt_e2m1x8(const float* f) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
  return r;
}

// ---- MX ----
__device__ __forceinline__ uint32_t mx_scale_code(uint32_t amax16) {
  if (amax16 >= 0x7F80u) return FP4_NAN_MX;
  return (uint32_t)max((int)(amax16 >> 7) - 2, 0);
}
// 4 words (8 values) -> 32 bits of codes
__device__ __forceinline__ uint32_t mx_encode8(const uint32_t* w, uint32_t code) {
  if (code == FP4_NAN_MX) return 0u;
  const float m = __uint_as_float((254u - code) << 23);      // 1 / scale
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    f[2 * i] = __uint_as_float(w[i] << 16) * m;
    f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u) * m;
  }
  return cvt_e2m1x8(f);
}

// ---- NV ----
// value of an e4m3 code (no sign, not NaN)
__device__ __forceinline__ float e4m3_value(uint32_t c) {
  return c < 8u ? (float)c * 0x1p-9f : __uint_as_float((c << 20) + (120u << 23));
}
// e4m3 code nearest to amax / (6 ts), 448 at most, a tie to the even code.  inv6: 1 / (6 ts), rounded; it gives a code
// that is at most one off, which the exact remainders at the two borders then put right.
__device__ __forceinline__ uint32_t nv_scale_code(uint32_t amax16, float ts, float inv6) {
  if (amax16 >= 0x7F80u) return FP4_NAN_NV;
  const float a = __uint_as_float(amax16 << 16);
  uint16_t pair;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(pair) : "f"(0.f), "f"(a * inv6));
  uint32_t c = min((uint32_t)pair & 0x7Fu, 0x7Eu);
  const float v = e4m3_value(c);
  if (c < 0x7Eu) {
    const float r = fmaf(-3.f * (v + e4m3_value(c + 1)), ts, a);           // a - 6 ts * border: the sign is exact
    if (r > 0.f || (r == 0.f && (c & 1u))) return c + 1;
  }
  if (c > 0u) {
    const float r = fmaf(-3.f * (v + e4m3_value(c - 1)), ts, a);
    if (r < 0.f || (r == 0.f && (c & 1u))) return c - 1;
  }
  return c;
}
// The seven borders of a block as bf16 bits T, in both halves of a word and with the top bits set: a magnitude is past
// the border exactly when its bits are above T.
struct NvBorders {
  uint32_t t[7];
};
__device__ __forceinline__ NvBorders nv_borders(uint32_t code, float ts) {
  const float s = e4m3_value(code);
  NvBorders b;
  const float above[4] = {0.25f, 1.25f, 2.5f, 5.f}, from[3] = {0.75f, 1.75f, 3.5f};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t u = __float_as_uint(__fmul_rd(above[i] * s, ts)) >> 16;
    b.t[2 * i] = __byte_perm(u, u, 0x1010) | 0x80008000u;
  }
#pragma unroll
  for (int i = 0; i < 3; i++) {
    const uint32_t u = ((__float_as_uint(__fmul_ru(from[i] * s, ts)) + 0xFFFFu) >> 16) - 1u;
    b.t[2 * i + 1] = __byte_perm(u, u, 0x1010) | 0x80008000u;
  }
  return b;
}
// one word (2 values) -> codes in bits 0-3 and 16-19.  t - x keeps the top bit of a half where x is not past the border;
// the passed borders are always the lowest ones, so the bits of their number are parities.
__device__ __forceinline__ uint32_t nv_encode2(uint32_t w, const NvBorders& b) {
  const uint32_t x = w & 0x7FFF7FFFu;
  uint32_t d[7];
#pragma unroll
  for (int i = 0; i < 7; i++) d[i] = b.t[i] - x;
  const uint32_t b0 = ~(d[0] ^ d[1] ^ d[2] ^ d[3] ^ d[4] ^ d[5] ^ d[6]), b1 = ~(d[1] ^ d[3] ^ d[5]), b2 = ~d[3];
  return ((w & 0x80008000u) >> 12) | ((b2 & 0x80008000u) >> 13) | ((b1 & 0x80008000u) >> 14) | ((b0 & 0x80008000u) >> 15);
}
// 4 words (8 values) -> 32 bits of codes
__device__ __forceinline__ uint32_t nv_encode8(const uint32_t* w, uint32_t code, const NvBorders& b) {
  if (code == FP4_NAN_NV || code == 0u) return 0u;
  const uint32_t p = nv_encode2(w[0], b) | (nv_encode2(w[1], b) << 8), q = nv_encode2(w[2], b) | (nv_encode2(w[3], b) << 8);
  return ((p & 0xFFFFu) | (p >> 12)) | (((q & 0xFFFFu) | (q >> 12)) << 16);
}

// ---- storage of the scales: tiles of 128 rows x 256 values, inside a tile groups of four blocks as 512-byte pieces
// [row % 32][row / 32 % 4][block % 4], the order in which the tensor core's scale memory takes them ----
template <bool MX>
__device__ __forceinline__ int64_t scale_offset(int row, int block, int64_t chunks) {
  constexpr int GROUPS = MX ? 2 : 4;          // groups of four blocks in 256 values
  return ((int64_t)(row >> 7) * chunks * GROUPS + (block >> 2)) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}

}  // namespace krea
