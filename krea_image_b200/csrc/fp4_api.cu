// The C ABI of the 4-bit operators and of the gated norm (include/krea_cuda.h): argument checks, tensor maps, launches.
#include <cuda.h>
#include <cuda_runtime.h>
#include <string.h>

#include "../../include/krea_cuda.h"
#include "fp4.h"
#include "fp4_checks.h"
#include "handle.h"

using namespace krea;

// packed values [rows, row bytes] in boxes of 128 bytes x box_rows rows, 128-byte swizzle; rows and bytes outside read as zero
static int make_values_map(krea_cuda* h, CUtensorMap* tm, const void* base, int rows, int K, int64_t ld, int box_rows, const char* what) {
  cuuint64_t dims[3] = {(cuuint64_t)fp4_row_bytes(K), (cuuint64_t)rows, 1};
  cuuint64_t strides[2] = {(cuuint64_t)ld, (cuuint64_t)ld * (cuuint64_t)rows};
  cuuint32_t box[3] = {128, (cuuint32_t)box_rows, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = h->encode(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(h, KREA_CUDA_E_CUDA, "gemm_fp4: cuTensorMapEncodeTiled(%s) failed with %d", what, (int)r);
  return KREA_CUDA_OK;
}
// scales as 8-byte words [row tile][chunk of 256 values][chunk words]; row tiles outside read as zero
static int make_scales_map(krea_cuda* h, CUtensorMap* tm, const void* base, int format, int rows, int K, int box_tiles, const char* what) {
  const cuuint64_t words = (cuuint64_t)fp4_scale_tile_bytes(format) / 8, chunks = (cuuint64_t)((K + 255) / 256), tiles = (cuuint64_t)((rows + 127) / 128);
  cuuint64_t dims[3] = {words, chunks, tiles};
  cuuint64_t strides[2] = {words * 8, words * 8 * chunks};
  cuuint32_t box[3] = {(cuuint32_t)words, 1, (cuuint32_t)box_tiles};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = h->encode(tm, CU_TENSOR_MAP_DATA_TYPE_INT64, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(h, KREA_CUDA_E_CUDA, "gemm_fp4: cuTensorMapEncodeTiled(%s) failed with %d", what, (int)r);
  return KREA_CUDA_OK;
}
// C in boxes of 32 rows x 128 bytes, 128-byte swizzle; what a box has outside is not written
static int make_out_map(krea_cuda* h, CUtensorMap* tm, void* base, int rows, int cols, int64_t ld, bool f32) {
  const int es = f32 ? 4 : 2;
  cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, 1};
  cuuint64_t strides[2] = {(cuuint64_t)ld * es, (cuuint64_t)ld * es * (cuuint64_t)rows};
  cuuint32_t box[3] = {(cuuint32_t)(128 / es), 32, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = h->encode(tm, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(h, KREA_CUDA_E_CUDA, "gemm_fp4: cuTensorMapEncodeTiled(C) failed with %d", (int)r);
  return KREA_CUDA_OK;
}

static int sms(const krea_cuda* h) { return h->sm_count > 0 ? h->sm_count : 148; }

extern "C" {

size_t krea_cuda_fp4_row_bytes(int K) { return K > 0 ? (size_t)fp4_row_bytes(K) : 0; }
size_t krea_cuda_fp4_scale_bytes(int format, int rows, int K) { return fp4_format_ok(format) && rows > 0 && K > 0 ? (size_t)fp4_scale_bytes(format, rows, K) : 0; }

int krea_cuda_fp4_quantize(krea_cuda* h, const krea_cuda_fp4_quantize_args* a) {
  if (!h || !a) return fail(h, KREA_CUDA_E_ARG, "fp4_quantize: null handle or arguments");
  if (const char* m = check_fp4_quantize(a)) return fail(h, KREA_CUDA_E_ARG, "fp4_quantize: %s", m);
  if (a->rows == 0 || a->K == 0) return KREA_CUDA_OK;
  Fp4QuantParams p{};
  p.src = (const __nv_bfloat16*)a->src; p.q = (uint8_t*)a->q; p.scales = (uint8_t*)a->scales; p.tensor_scale = a->tensor_scale;
  p.rows = a->rows; p.K = a->K; p.ld = a->ld; p.ldq = a->ldq; p.mx = a->format == KREA_CUDA_FP4_MX;
  CUDA_TRY(h, cudaSetDevice(h->device));
  if (a->transposed) {
    p.status = h->status_dev;
    cuuint64_t dims[3] = {(cuuint64_t)a->rows, (cuuint64_t)a->K, 1};
    cuuint64_t strides[2] = {(cuuint64_t)a->ld * 2, (cuuint64_t)a->ld * 2 * (cuuint64_t)a->K};
    cuuint32_t box[3] = {128, 128, 1}, estr[3] = {1, 1, 1};
    CUtensorMap tm;
    CUresult r = h->encode(&tm, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(a->src), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(h, KREA_CUDA_E_CUDA, "fp4_quantize: cuTensorMapEncodeTiled failed with %d", (int)r);
    CUDA_TRY(h, launch_fp4_quantize_cols(tm, p, sms(h), h->pdl, h->stream));
  } else {
    CUDA_TRY(h, launch_fp4_quantize(p, sms(h), h->pdl, h->stream));
  }
  h->launches++;
  return KREA_CUDA_OK;
}

int krea_cuda_fp4_dequantize(krea_cuda* h, const krea_cuda_fp4_dequantize_args* a) {
  if (!h || !a) return fail(h, KREA_CUDA_E_ARG, "fp4_dequantize: null handle or arguments");
  if (const char* m = check_fp4_dequantize(a)) return fail(h, KREA_CUDA_E_ARG, "fp4_dequantize: %s", m);
  if (a->rows == 0 || a->K == 0) return KREA_CUDA_OK;
  Fp4DequantParams p{};
  p.q = (const uint8_t*)a->q; p.scales = (const uint8_t*)a->scales; p.tensor_scale = a->tensor_scale; p.out = (__nv_bfloat16*)a->out;
  p.rows = a->rows; p.K = a->K; p.ldq = a->ldq; p.ldo = a->ldo; p.mx = a->format == KREA_CUDA_FP4_MX;
  CUDA_TRY(h, cudaSetDevice(h->device));
  CUDA_TRY(h, launch_fp4_dequantize(p, sms(h), h->pdl, h->stream));
  h->launches++;
  return KREA_CUDA_OK;
}

int krea_cuda_gemm_fp4(krea_cuda* h, const krea_cuda_gemm_fp4_args* a) {
  if (!h || !a) return fail(h, KREA_CUDA_E_ARG, "gemm_fp4: null handle or arguments");
  if (!fp4_epilogue_built(a->epilogue)) return fail(h, KREA_CUDA_E_UNSUPPORTED, "gemm_fp4: epilogue %d is not built", a->epilogue);
  if (const char* m = check_gemm_fp4(a)) return fail(h, KREA_CUDA_E_ARG, "gemm_fp4: %s", m);
  if (a->M == 0 || a->N == 0) return KREA_CUDA_OK;
  CUDA_TRY(h, cudaSetDevice(h->device));
  const bool mx = a->format == KREA_CUDA_FP4_MX;
  const Fp4GemmPlan plan = plan_gemm_fp4(a->M, a->N, a->K, mx, sms(h), h->fp4_tile);
  CUtensorMap tmA, tmAs, tmW, tmWs, tmC;
  memset(&tmC, 0, sizeof(tmC));
  int rc;
  // test hook, CTA pairs: boxes that lack rows, so that the bytes that are waited for never all arrive
  const int box_a = plan.pair ? (h->test_drop_last_k ? 64 : 128) : plan.tn;
  if ((rc = make_values_map(h, &tmA, a->A, a->M, a->K, a->lda, box_a, "A"))) return rc;
  if ((rc = make_values_map(h, &tmW, a->W, a->N, a->K, a->ldw, 128, "W"))) return rc;
  if ((rc = make_scales_map(h, &tmAs, a->a_scales, a->format, a->M, a->K, 1, "a_scales"))) return rc;
  if ((rc = make_scales_map(h, &tmWs, a->w_scales, a->format, a->N, a->K, plan.pair ? 2 : 1, "w_scales"))) return rc;
  if (plan.pair && (rc = make_out_map(h, &tmC, a->C, a->M, a->epilogue == KREA_CUDA_EPI_SWIGLU ? a->N / 2 : a->N, a->ldc, epilogue_f32(a->epilogue)))) return rc;
  Fp4GemmParams p{};
  p.C = a->C; p.ldc = a->ldc; p.M = a->M; p.N = a->N; p.K = a->K; p.epi = a->epilogue; p.mx = mx;
  const bool uses_vec = a->epilogue == KREA_CUDA_EPI_RESID_GATE || a->epilogue == KREA_CUDA_EPI_BIAS_BF16 || a->epilogue == KREA_CUDA_EPI_BIAS_F32;
  p.vec = uses_vec ? a->vec : nullptr;
  p.a_ts = a->a_tensor_scale; p.w_ts = a->w_tensor_scale;
  p.status = h->status_dev;
  p.wait_limit_ns = h->wait_limit_ns;
  p.test_drop_load = h->test_drop_last_k;
  CUDA_TRY(h, launch_gemm_fp4(plan, tmA, tmAs, tmW, tmWs, tmC, p, sms(h), h->pdl, h->stream));
  h->launches++;
  return KREA_CUDA_OK;
}

int krea_cuda_gated_norm(krea_cuda* h, const krea_cuda_gated_norm_args* a) {
  if (!h || !a) return fail(h, KREA_CUDA_E_ARG, "gated_norm: null handle or arguments");
  if (const char* m = check_gated_norm(a)) return fail(h, KREA_CUDA_E_ARG, "gated_norm: %s", m);
  if (a->rows == 0 || a->width == 0) return KREA_CUDA_OK;
  GatedNormParams p{};
  p.x = a->x; p.y = a->y; p.x_out = a->x_out; p.h = a->h; p.h_scales = (uint8_t*)a->h_scales; p.h_ts = a->h_tensor_scale;
  p.post = a->post; p.gate = a->gate; p.mul = a->mul; p.add = a->add;
  p.rows = a->rows; p.width = a->width; p.ld_x = a->ld_x; p.ld_y = a->ld_y; p.ld_xo = a->ld_xo; p.ld_h = a->ld_h;
  p.mod_rows = a->mod_rows; p.mod_ld = a->mod_ld; p.x_scale = a->x_scale; p.eps = a->eps; p.y_f32 = a->y_f32 != 0; p.out = a->out;
  CUDA_TRY(h, cudaSetDevice(h->device));
  CUDA_TRY(h, launch_gated_norm(p, sms(h), h->pdl, h->stream));
  h->launches++;
  return KREA_CUDA_OK;
}

}  // extern "C"
