// Argument checks of the 4-bit entry points and of the gated norm, as plain host functions without CUDA: each returns
// nullptr for a call that may be launched, or what is wrong with it.  A size of zero is no error (the entry points
// return before they launch anything).
#pragma once
#include <math.h>
#include <stdint.h>

#include "../../include/krea_cuda.h"

namespace krea {

inline bool fp4_format_ok(int format) { return format == KREA_CUDA_FP4_MX || format == KREA_CUDA_FP4_NV; }
inline int fp4_block(int format) { return format == KREA_CUDA_FP4_MX ? 32 : 16; }
// bytes of one packed row: two values a byte, whole groups of 32 values
inline int64_t fp4_row_bytes(int64_t K) { return (K + 31) / 32 * 16; }
// bytes of the scales of [rows, K]: tiles of 128 rows x 256 values
inline int64_t fp4_scale_tile_bytes(int format) { return format == KREA_CUDA_FP4_MX ? 1024 : 2048; }
inline int64_t fp4_scale_bytes(int format, int64_t rows, int64_t K) { return (rows + 127) / 128 * ((K + 255) / 256) * fp4_scale_tile_bytes(format); }

// sizes beyond these are refused: rounding them up to whole tiles stays within 32 bits, and the product's longest wait
// (for a whole tile's K) far below the usual limit of two seconds on every wait
constexpr int FP4_MAX_ROWS = 1 << 30, FP4_MAX_K = 1 << 26;

inline bool off16(const void* p) { return ((uintptr_t)p & 15u) != 0; }

// whether the n bytes at a and the m bytes at b have a byte in common
inline bool overlap(const void* a, int64_t n, const void* b, int64_t m) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return a && b && n > 0 && m > 0 && x < y + (uintptr_t)m && y < x + (uintptr_t)n;
}
// bytes that a matrix of `rows` rows of `width` used bytes, `ld` bytes apart, spans
inline int64_t span(int64_t rows, int64_t width, int64_t ld) { return rows > 0 ? (rows - 1) * ld + width : 0; }

// whether two matrices of rows (bytes used of a row, bytes between rows) have a byte in common; rows the same distance apart may
// lie side by side in one buffer
struct Rows {
  const void* p;
  int64_t rows, width, ld;
};
inline bool overlap(const Rows& a, const Rows& b) {
  if (!overlap(a.p, span(a.rows, a.width, a.ld), b.p, span(b.rows, b.width, b.ld))) return false;
  if (a.ld != b.ld) return true;
  const int64_t from = ((intptr_t)b.p - (intptr_t)a.p) % a.ld, at = from < 0 ? from + a.ld : from;      // where b's rows start in a's
  return at < a.width || at + b.width > a.ld;
}

inline const char* check_fp4_quantize(const krea_cuda_fp4_quantize_args* a) {
  if (a->rows < 0 || a->K < 0) return "negative size";
  if (a->rows > FP4_MAX_ROWS || a->K > FP4_MAX_K) return "rows must be 2^30 at most, K 2^26";
  if (!fp4_format_ok(a->format)) return "format must be KREA_CUDA_FP4_MX or KREA_CUDA_FP4_NV";
  if (a->rows == 0 || a->K == 0) return nullptr;
  if (!a->src || !a->q || !a->scales) return "null tensor";
  if (off16(a->src) || off16(a->q) || off16(a->scales)) return "tensors must be 16-byte aligned";
  if (a->tensor_scale && ((uintptr_t)a->tensor_scale & 3u)) return "tensor_scale must be 4-byte aligned";
  if (a->format == KREA_CUDA_FP4_MX && a->tensor_scale) return "the MX format has no tensor scale";
  if (a->ld % 8 || a->ld < (a->transposed ? a->rows : a->K)) return "ld must be a multiple of 8 and cover a row of the source";
  if (a->ldq % 16 || a->ldq < fp4_row_bytes(a->K)) return "ldq must be a multiple of 16 and cover a packed row";
  const int64_t qb = span(a->rows, fp4_row_bytes(a->K), a->ldq), sb = fp4_scale_bytes(a->format, a->rows, a->K);
  const int64_t src = a->transposed ? span(a->K, 2 * (int64_t)a->rows, 2 * (int64_t)a->ld) : span(a->rows, 2 * (int64_t)a->K, 2 * (int64_t)a->ld);
  if (overlap(a->q, qb, a->scales, sb) || overlap(a->q, qb, a->src, src) || overlap(a->scales, sb, a->src, src)) return "tensors overlap";
  if (overlap(a->q, qb, a->tensor_scale, 4) || overlap(a->scales, sb, a->tensor_scale, 4)) return "tensors overlap";
  return nullptr;
}

inline const char* check_fp4_dequantize(const krea_cuda_fp4_dequantize_args* a) {
  if (a->rows < 0 || a->K < 0) return "negative size";
  if (a->rows > FP4_MAX_ROWS || a->K > FP4_MAX_K) return "rows must be 2^30 at most, K 2^26";
  if (!fp4_format_ok(a->format)) return "format must be KREA_CUDA_FP4_MX or KREA_CUDA_FP4_NV";
  if (a->rows == 0 || a->K == 0) return nullptr;
  if (!a->q || !a->scales || !a->out) return "null tensor";
  if (off16(a->q) || off16(a->scales) || off16(a->out)) return "tensors must be 16-byte aligned";
  if (a->tensor_scale && ((uintptr_t)a->tensor_scale & 3u)) return "tensor_scale must be 4-byte aligned";
  if (a->format == KREA_CUDA_FP4_MX && a->tensor_scale) return "the MX format has no tensor scale";
  if (a->ldq % 16 || a->ldq < fp4_row_bytes(a->K)) return "ldq must be a multiple of 16 and cover a packed row";
  if (a->ldo % 8 || a->ldo < a->K) return "ldo must be a multiple of 8 and cover a row";
  const int64_t qb = span(a->rows, fp4_row_bytes(a->K), a->ldq), sb = fp4_scale_bytes(a->format, a->rows, a->K);
  const int64_t ob = span(a->rows, 2 * (int64_t)a->K, 2 * (int64_t)a->ldo);
  if (overlap(a->out, ob, a->q, qb) || overlap(a->out, ob, a->scales, sb) || overlap(a->out, ob, a->tensor_scale, 4)) return "tensors overlap";
  return nullptr;
}

inline bool fp4_epilogue_built(int e) {
  return e == KREA_CUDA_EPI_BF16 || e == KREA_CUDA_EPI_RESID_GATE || e == KREA_CUDA_EPI_SWIGLU || e == KREA_CUDA_EPI_F32 || e == KREA_CUDA_EPI_GELU ||
         e == KREA_CUDA_EPI_BIAS_BF16 || e == KREA_CUDA_EPI_BIAS_F32;
}
inline bool epilogue_f32(int e) { return e == KREA_CUDA_EPI_RESID_GATE || e == KREA_CUDA_EPI_F32 || e == KREA_CUDA_EPI_BIAS_F32; }

inline const char* check_gemm_fp4(const krea_cuda_gemm_fp4_args* a) {
  if (a->M < 0 || a->N < 0 || a->K < 0) return "negative size";
  if (a->M > FP4_MAX_ROWS || a->N > FP4_MAX_ROWS || a->K > FP4_MAX_K) return "M and N must be 2^30 at most, K 2^26";
  if (!fp4_format_ok(a->format)) return "format must be KREA_CUDA_FP4_MX or KREA_CUDA_FP4_NV";
  if (a->M == 0 || a->N == 0) return nullptr;
  if (a->K == 0) return "K must be positive";
  if (!a->A || !a->a_scales || !a->W || !a->w_scales || !a->C) return "null tensor";
  if (off16(a->A) || off16(a->a_scales) || off16(a->W) || off16(a->w_scales) || off16(a->C)) return "tensors must be 16-byte aligned";
  if (((uintptr_t)a->a_tensor_scale & 3u) || ((uintptr_t)a->w_tensor_scale & 3u)) return "tensor scales must be 4-byte aligned";
  if (a->format == KREA_CUDA_FP4_MX && (a->a_tensor_scale || a->w_tensor_scale)) return "the MX format has no tensor scale";
  if (a->lda % 16 || a->ldw % 16 || a->lda < fp4_row_bytes(a->K) || a->ldw < fp4_row_bytes(a->K)) return "lda and ldw must be multiples of 16 bytes and cover a packed row";
  if (a->N % 8 || a->ldc % 8) return "N and ldc must be multiples of 8";
  if (a->epilogue == KREA_CUDA_EPI_SWIGLU && a->N % 64) return "SwiGLU needs N to be a multiple of 64 (32 gate + 32 up columns per group)";
  const int64_t cols = a->epilogue == KREA_CUDA_EPI_SWIGLU ? a->N / 2 : a->N, es = epilogue_f32(a->epilogue) ? 4 : 2;
  if (a->ldc < cols) return "ldc is smaller than a row of C";
  const bool bias = a->epilogue == KREA_CUDA_EPI_BIAS_BF16 || a->epilogue == KREA_CUDA_EPI_BIAS_F32;
  if (bias && !a->vec) return "the bias vector is missing";
  if ((bias || a->epilogue == KREA_CUDA_EPI_RESID_GATE) && off16(a->vec)) return "vec must be 16-byte aligned";
  const int64_t cb = span(a->M, cols * es, (int64_t)a->ldc * es);
  if (overlap(a->C, cb, a->A, span(a->M, fp4_row_bytes(a->K), a->lda)) || overlap(a->C, cb, a->W, span(a->N, fp4_row_bytes(a->K), a->ldw)) ||
      overlap(a->C, cb, a->a_scales, fp4_scale_bytes(a->format, a->M, a->K)) || overlap(a->C, cb, a->w_scales, fp4_scale_bytes(a->format, a->N, a->K)) ||
      overlap(a->C, cb, a->a_tensor_scale, 4) || overlap(a->C, cb, a->w_tensor_scale, 4) ||
      ((bias || a->epilogue == KREA_CUDA_EPI_RESID_GATE) && overlap(a->C, cb, a->vec, (int64_t)a->N * 4)))
    return "C overlaps an operand";
  return nullptr;
}

constexpr int GATED_NORM_MAX_WIDTH = 32768;

inline const char* check_gated_norm(const krea_cuda_gated_norm_args* a) {
  if (a->rows < 0 || a->width < 0) return "negative size";
  if (a->rows > FP4_MAX_ROWS) return "rows must be 2^30 at most";
  if (a->out < KREA_CUDA_OUT_BF16 || a->out > KREA_CUDA_OUT_FP4_NV) return "out must be one of KREA_CUDA_OUT_*";
  if (a->rows == 0 || a->width == 0) return nullptr;
  if (!a->x || !(a->x_out || a->h)) return "null tensor";
  if (a->width % 8 || a->width > GATED_NORM_MAX_WIDTH) return "width must be a multiple of 8, 32768 at most";
  if (a->ld_x % 4 || a->ld_x < a->width) return "ld_x must be a multiple of 4 and cover a row";
  const int64_t R = a->rows, W = a->width;
  if (a->y && (a->ld_y % (a->y_f32 ? 4 : 8) || a->ld_y < W)) return "ld_y must be a multiple of 8 (4 for f32 rows) and cover a row";
  if (a->x_out && (a->ld_xo % 4 || a->ld_xo < W)) return "ld_xo must be a multiple of 4 and cover a row";
  if ((a->post || a->gate) && !a->y) return "post and gate need y";
  const bool q = a->out == KREA_CUDA_OUT_FP4_MX || a->out == KREA_CUDA_OUT_FP4_NV;
  const int fmt = a->out == KREA_CUDA_OUT_FP4_MX ? KREA_CUDA_FP4_MX : KREA_CUDA_FP4_NV;
  const int64_t hb = q ? fp4_row_bytes(W) : W * (a->out == KREA_CUDA_OUT_F32 ? 4 : 2);
  const int64_t hld = q ? (int64_t)a->ld_h : (int64_t)a->ld_h * (a->out == KREA_CUDA_OUT_F32 ? 4 : 2);
  if (a->h) {
    if (!a->mul) return "mul is missing";
    if (hld % 16 || hld < hb) return "rows of h must start 16-byte aligned and ld_h cover a row";
    if (q && !a->h_scales) return "h_scales is missing";
    if (a->h_tensor_scale && a->out != KREA_CUDA_OUT_FP4_NV) return "only the NV format has a tensor scale";
    if ((uintptr_t)a->h_tensor_scale & 3u) return "h_tensor_scale must be 4-byte aligned";
  }
  if (off16(a->x) || off16(a->y) || off16(a->x_out) || off16(a->h) || off16(a->post) || off16(a->gate) || off16(a->mul) || off16(a->add) || off16(a->h_scales))
    return "tensors must be 16-byte aligned";
  if (a->mod_rows < 0) return "mod_rows must not be negative";
  if (a->mod_rows > 0 && (a->mod_ld % 4 || a->mod_ld < 0)) return "mod_ld must be a multiple of 4, not negative";
  if (!(a->eps >= 0.f) || !isfinite(a->x_scale)) return "eps must not be negative, x_scale finite";
  const int64_t es = a->y_f32 ? 4 : 2;
  const Rows x = {a->x, R, W * 4, (int64_t)a->ld_x * 4}, y = {a->y, R, W * es, (int64_t)a->ld_y * es}, xo = {a->x_out, R, W * 4, (int64_t)a->ld_xo * 4}, h = {a->h, R, hb, hld};
  const int64_t xb = span(R, x.width, x.ld), xob = a->x_out ? span(R, xo.width, xo.ld) : 0, yb = a->y ? span(R, y.width, y.ld) : 0;
  const int64_t hs = a->h ? span(R, hb, hld) : 0, sb = a->h && q ? fp4_scale_bytes(fmt, R, W) : 0;
  if (overlap(xo, x) && !((const void*)a->x_out == (const void*)a->x && a->ld_xo == a->ld_x)) return "x_out may be x itself with the same ld, or apart from it";
  if (overlap(xo, y)) return "x_out overlaps y";
  if (overlap(h, x) || overlap(h, y) || overlap(h, xo)) return "h overlaps another tensor";
  if (overlap(a->h_scales, sb, a->x, xb) || overlap(a->h_scales, sb, a->y, yb) || overlap(a->h_scales, sb, a->x_out, xob) || overlap(a->h_scales, sb, a->h, hs))
    return "h_scales overlaps another tensor";
  const int64_t vb = (a->mod_rows > 0 ? (R - 1) / a->mod_rows * a->mod_ld : 0) * 4 + W * 4;      // from the first vector to the end of the last
  const struct { const void* p; int64_t n; } in[] = {{a->post, W * 4}, {a->gate, vb}, {a->mul, vb}, {a->add, vb}, {a->h_tensor_scale, 4}};
  for (const auto& v : in)
    if (overlap(a->x_out, xob, v.p, v.n) || overlap(a->h, hs, v.p, v.n) || overlap(a->h_scales, sb, v.p, v.n)) return "an output overlaps a vector";
  return nullptr;
}

}  // namespace krea
