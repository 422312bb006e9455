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
__device__ __forceinline__ uint32_t nv_encode8_borders(const uint32_t* w, const NvBorders& b) {
  const uint32_t p = nv_encode2(w[0], b) | (nv_encode2(w[1], b) << 8), q = nv_encode2(w[2], b) | (nv_encode2(w[3], b) << 8);
  return ((p & 0xFFFFu) | (p >> 12)) | (((q & 0xFFFFu) | (q >> 12)) << 16);
}

// Everything that depends on a scale code and ts alone, tabulated in shared memory by 128 threads of the CTA:
//   top[c]  the largest amax (bf16 bits) whose scale code is c or lower: amax / (6 ts) against the border between two e4m3
//           values, by the same directed rounding as above
//   inv[c]  factor of the fast way to encode, below; its sign and zero say which way
// The comparisons with the borders take 9 integer instructions a value, a product and the conversion instruction 2.5.
// The product t = x * inv, inv = 1 / (s ts), is off by less than 4 * 2^-24, so it gives the exact code wherever no bf16
// number is that near to a border.  All borders of a block have one of four mantissas, those of 1, 1.25, 1.5 and 1.75 times
// s ts, so the bf16 numbers next to them are four: where one is within 32 * 2^-24 of its border, its exact side is found
// once, here, and inv is moved by 8 * 2^-24 to that side - 12 * 2^-24 in all cannot carry any other number over a border.
// (With ts = amax / 2688 there are such numbers for two scales in eight: 2688 = 21 * 128, and 1.75 * 1.5 = 21 / 8.)
// Where numbers lie ON borders (ts a power of two), one Newton step makes their quotients exact.  What is left, and every
// scale near the ends of the f32 range, takes the comparisons.
struct NvTable {
  uint2 e[128];          // x: inv as bits - positive: the product, negative: with a Newton step, 0: the comparisons; y: top of c | top of c - 1 << 16
  float ts;
  float pre, inv6;       // their product is 1 / (6 ts); pre, a power of two, brings ts to where that is an f32
};
__device__ __forceinline__ void nv_table_fill(NvTable& t, float ts, int c) {     // c: 0 .. 127, one thread each
  if (c == 0) {
    t.ts = ts;
    // 6 ts passes the largest f32 above 5.67e37, and 1 / (6 ts) below 4.9e-40; amax * pre leaves the range only where the
    // quotient is far beyond the highest or the lowest code
    t.pre = ts < 0x1p-100f ? 0x1p60f : ts > 0x1p100f ? 0x1p-8f : 1.f;
    t.inv6 = 1.f / (6.f * (ts * t.pre));
  }
  // border between a value and the next, times 6: passed from on when its code is odd (a tie goes to the even one), above it else
  const auto top = [&](uint32_t k) -> uint32_t {
    if (k >= 0x7Eu) return 0x7F7Fu;
    const float border = 3.f * (e4m3_value(k) + e4m3_value(k + 1u));
    return k & 1u ? ((__float_as_uint(__fmul_ru(border, ts)) + 0xFFFFu) >> 16) - 1u : __float_as_uint(__fmul_rd(border, ts)) >> 16;
  };
  const uint32_t below = c > 0 ? top((uint32_t)c - 1u) : 0u;      // code 0 has nothing below: its own top is compared
  const float s = e4m3_value((uint32_t)c);
  const float p = s * ts;
  const float m[4] = {1.f, 1.25f, 1.5f, 1.75f};
  bool up = false, down = false, on = false;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t u = __float_as_uint(m[i] * p);
    if (((u + 32u) & 0xFFFFu) <= 64u) {
      const float r = fmaf(-(m[i] * s), ts, __uint_as_float((u + 0x8000u) & 0xFFFF0000u));     // that bf16 number - border, its sign exact
      up = up || r > 0.f;
      down = down || r < 0.f;
      on = on || r == 0.f;
    }
  }
  const uint32_t e = __float_as_uint(ts);
  const bool plain = e - (37u << 23) < (180u << 23);             // 2^-90 <= ts < 2^90
  const float inv = __frcp_rn(p);
  float f = 0.f;
  if (plain && c > 0 && !on && !(up && down)) f = up ? inv * (1.f + 0x1p-21f) : down ? inv * (1.f - 0x1p-21f) : inv;
  else if (plain && c > 0 && c < 0x7E && on && !up && !down) f = -inv;      // not at the top of the scale's range, where x / s has no bound of its own
  t.e[c] = make_uint2(__float_as_uint(f), (top((uint32_t)c) & 0xFFFFu) | (below << 16));
}
// scale code of a block; the product with 1 / (6 ts) gives a code that is at most one off
__device__ __forceinline__ uint32_t nv_scale_code(uint32_t amax16, const NvTable& t) {
  if (amax16 >= 0x7F80u) return FP4_NAN_NV;
  uint16_t pair;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(pair) : "f"(0.f), "f"(__uint_as_float(amax16 << 16) * t.pre * t.inv6));
  const uint32_t c = min((uint32_t)pair & 0x7Fu, 0x7Eu), tops = t.e[c].y;
  if (amax16 > (tops & 0xFFFFu)) return c + 1;
  return c > 0u && amax16 <= (tops >> 16) ? c - 1 : c;
}

// W words (2 W values) of one block (or a part of it) with the block's scale code -> W / 4 words of codes
template <int W>
__device__ __forceinline__ void nv_encode(const uint32_t* w, uint32_t code, const NvTable& t, uint32_t* out) {
  if (code == FP4_NAN_NV || code == 0u) {
#pragma unroll
    for (int i = 0; i < W / 4; i++) out[i] = 0u;
    return;
  }
  const float way = __uint_as_float(t.e[code].x);
  if (way != 0.f) {
    const float inv = fabsf(way), s = e4m3_value(code) * t.ts;
#pragma unroll
    for (int i = 0; i < W / 4; i++) {
      float f[8];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float x0 = __uint_as_float(w[4 * i + j] << 16), x1 = __uint_as_float(w[4 * i + j] & 0xFFFF0000u);
        f[2 * j] = x0 * inv;
        f[2 * j + 1] = x1 * inv;
        if (way < 0.f) {
          f[2 * j] = fmaf(fmaf(f[2 * j], s, -x0), -inv, f[2 * j]);             // in this form -0 stays -0
          f[2 * j + 1] = fmaf(fmaf(f[2 * j + 1], s, -x1), -inv, f[2 * j + 1]);
        }
      }
      out[i] = cvt_e2m1x8(f);
    }
  } else {
    const NvBorders b = nv_borders(code, t.ts);
#pragma unroll
    for (int i = 0; i < W / 4; i++) out[i] = nv_encode8_borders(w + 4 * i, b);
  }
}

// ---- storage of the scales: tiles of 128 rows x 256 values, inside a tile groups of four blocks as 512-byte pieces
// [row % 32][row / 32 % 4][block % 4], the order in which the tensor core's scale memory takes them ----
template <bool MX>
__device__ __forceinline__ int64_t scale_offset(int row, int block, int64_t chunks) {
  constexpr int GROUPS = MX ? 2 : 4;          // groups of four blocks in 256 values
  return ((int64_t)(row >> 7) * chunks * GROUPS + (block >> 2)) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (block & 3);
}

}  // namespace krea
