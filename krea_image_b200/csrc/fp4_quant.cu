// bf16 rows -> packed 4-bit rows with block scales, and back (formats and rounding: fp4_block.cuh).
//
// Storage: two values a byte, the lower index in the low bits, rows of whole 16 bytes (32 values; values past K are
// zero); scales as fp4_block.cuh lays them out, zero past K and past the last row.  A block with an infinity or a NaN
// gets the scale code NaN, so that products with it become NaN.
//
// HBM-bound: 2 bytes read and 0.53 (MX) or 0.56 (NV) written per value.  A warp takes the four blocks that share a
// 4-byte word of scales from rows 32 apart, which makes its scale bytes one contiguous piece (16 or 32 bytes) and its
// reads whole 128-byte lines.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "fp4.h"
#include "fp4_block.cuh"
#include "sm100_ptx.cuh"

namespace krea {

constexpr int FQ_THREADS = 256;

// 16 values from `src` (16-byte aligned), zero from index `left` on
__device__ __forceinline__ void load16(const __nv_bfloat16* src, int left, uint32_t* w) {
  if (left >= 16) {
    const uint4 a = __ldg((const uint4*)src), b = __ldg((const uint4*)src + 1);
    w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const uint32_t lo = 2 * i < left ? (uint32_t)__bfloat16_as_ushort(src[2 * i]) : 0u;
      const uint32_t hi = 2 * i + 1 < left ? (uint32_t)__bfloat16_as_ushort(src[2 * i + 1]) : 0u;
      w[i] = lo | (hi << 16);
    }
  }
}

template <bool MX>
__global__ void __launch_bounds__(FQ_THREADS) fp4_quantize_rows_kernel(const Fp4QuantParams p) {
  constexpr int LANES = MX ? 8 : 4;              // lanes of a row: 16 values each, four blocks together
  constexpr int GROUP = LANES * 16;              // values of those four blocks
  constexpr int RUNS = MX ? 32 : 16;             // warp items that cover the 128 rows of a scale tile
  const int64_t chunks = (p.K + 255) / 256;
  const int groups = (int)chunks * (256 / GROUP);
  const int64_t items = (int64_t)((p.rows + 127) / 128) * RUNS * (groups / 2);          // two groups at a time
  const int lane = threadIdx.x & 31, in_row = lane % LANES, rr = lane / LANES;
  griddep_wait();
  __shared__ NvTable nv;
  if constexpr (!MX) {
    if (threadIdx.x < 128) nv_table_fill(nv, p.tensor_scale ? __ldg(p.tensor_scale) : 1.f, threadIdx.x);
    __syncthreads();
  }
  const int64_t step = (int64_t)gridDim.x * (FQ_THREADS / 32);
  for (int64_t it = (int64_t)blockIdx.x * (FQ_THREADS / 32) + (threadIdx.x >> 5); it < items; it += step) {
    const int g = (int)(it % (groups / 2)) * 2;
    const int64_t tr = it / (groups / 2);
    const int run = (int)(tr % RUNS);
    const int row = (int)(tr / RUNS) * 128 + (rr & 3) * 32 + (MX ? run : run * 2 + (rr >> 2));
    const __nv_bfloat16* src = p.src + (int64_t)row * p.ld;
    uint32_t w[2][8];
#pragma unroll
    for (int i = 0; i < 2; i++) {                // both loads are under way before the first is used
      const int k0 = (g + i) * GROUP + in_row * 16;
      load16(src + k0, row < p.rows ? p.K - k0 : 0, w[i]);
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int k0 = (g + i) * GROUP + in_row * 16;
      uint32_t amax = amax_bits<8>(w[i]), code, out[2];
      if constexpr (MX) {
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        code = mx_scale_code(amax);
        out[0] = mx_encode8(w[i], code);
        out[1] = mx_encode8(w[i] + 4, code);
      } else {
        code = nv_scale_code(amax, nv);
        nv_encode<8>(w[i], code, nv, out);
      }
      if (row < p.rows && k0 < ((p.K + 31) & ~31)) *(uint2*)(p.q + (int64_t)row * p.ldq + (k0 >> 1)) = make_uint2(out[0], out[1]);
      const int block = MX ? k0 >> 5 : k0 >> 4;
      if (!MX || (lane & 1) == 0) p.scales[scale_offset<MX>(row, block, chunks)] = (uint8_t)code;
    }
  }
}

// The same for an input-major source [K, ld] (row k holds value k of every output row): a CTA turns a tile of 128 k x 64
// rows.  A lane has two neighbouring output rows and a warp 32 k, read from shared memory as whole 128-byte rows.
constexpr int FT_K = 128, FT_N = 64, FT_THREADS = 128;
template <bool MX>
__global__ void __launch_bounds__(FT_THREADS) fp4_quantize_cols_kernel(const Fp4QuantParams p) {
  __shared__ __align__(16) uint32_t tile[FT_K][FT_N / 2];
  __shared__ __align__(16) uint4 packed[FT_N][FT_K / 32 + 1];
  const int64_t chunks = (p.K + 255) / 256;
  const int n0 = blockIdx.x * FT_N, k0 = blockIdx.y * FT_K;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  griddep_wait();
  __shared__ NvTable nv;
  if constexpr (!MX) nv_table_fill(nv, p.tensor_scale ? __ldg(p.tensor_scale) : 1.f, threadIdx.x);
  for (int i = threadIdx.x; i < FT_K * (FT_N / 8); i += FT_THREADS) {
    const int kr = i / (FT_N / 8), c = (i % (FT_N / 8)) * 8;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (k0 + kr < p.K && n0 + c < p.rows) {
      const __nv_bfloat16* s = p.src + (int64_t)(k0 + kr) * p.ld + n0 + c;
      if (n0 + c + 8 <= p.rows) {
        v = __ldg((const uint4*)s);
      } else {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const uint32_t lo = n0 + c + 2 * j < p.rows ? (uint32_t)__bfloat16_as_ushort(s[2 * j]) : 0u;
          const uint32_t hi = n0 + c + 2 * j + 1 < p.rows ? (uint32_t)__bfloat16_as_ushort(s[2 * j + 1]) : 0u;
          w[j] = lo | (hi << 16);
        }
        v = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    *(uint4*)&tile[kr][c >> 1] = v;
  }
  __syncthreads();
  uint32_t t[32];
#pragma unroll
  for (int i = 0; i < 32; i++) t[i] = tile[warp * 32 + i][lane];
#pragma unroll
  for (int half = 0; half < 2; half++) {
    const int n = n0 + 2 * lane + half, kb = k0 + warp * 32;
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 16; i++) w[i] = __byte_perm(t[2 * i], t[2 * i + 1], half ? 0x7632 : 0x5410);
    uint32_t out[4];
    if constexpr (MX) {
      const uint32_t code = mx_scale_code(amax_bits<16>(w));
#pragma unroll
      for (int j = 0; j < 4; j++) out[j] = mx_encode8(w + 4 * j, code);
      p.scales[scale_offset<MX>(n, kb >> 5, chunks)] = (uint8_t)code;
    } else {
#pragma unroll
      for (int blk = 0; blk < 2; blk++) {
        const uint32_t code = nv_scale_code(amax_bits<8>(w + 8 * blk), nv);
        nv_encode<8>(w + 8 * blk, code, nv, out + 2 * blk);
        p.scales[scale_offset<MX>(n, (kb >> 4) + blk, chunks)] = (uint8_t)code;
      }
    }
    packed[2 * lane + half][warp] = make_uint4(out[0], out[1], out[2], out[3]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < FT_N * (FT_K / 32); i += FT_THREADS) {
    const int r = i / (FT_K / 32), j = i % (FT_K / 32);
    if (n0 + r < p.rows && k0 + j * 32 < p.K) *(uint4*)(p.q + (int64_t)(n0 + r) * p.ldq + (k0 >> 1) + j * 16) = packed[r][j];
  }
}

cudaError_t launch_fp4_quantize(const Fp4QuantParams& p, bool transposed, bool pdl, cudaStream_t stream) {
  if (p.rows <= 0 || p.K <= 0) return cudaSuccess;
  const int64_t tiles = (p.rows + 127) / 128, chunks = (p.K + 255) / 256;
  if (transposed) {
    const dim3 grid((unsigned)(tiles * (128 / FT_N)), (unsigned)(chunks * (256 / FT_K)));      // padding included: its scales are written too
    return launch_kernel(p.mx ? fp4_quantize_cols_kernel<true> : fp4_quantize_cols_kernel<false>, grid, FT_THREADS, 0, stream, pdl, 1, false, p);
  }
  const int64_t items = tiles * (p.mx ? 32 * 1 : 16 * 2) * chunks;
  int64_t blocks = (items + FQ_THREADS / 32 - 1) / (FQ_THREADS / 32);
  if (blocks > 148 * 16) blocks = 148 * 16;          // about two rounds of resident CTAs: each fills its table once
  return launch_kernel(p.mx ? fp4_quantize_rows_kernel<true> : fp4_quantize_rows_kernel<false>, dim3((unsigned)blocks), FQ_THREADS, 0, stream, pdl, 1, false, p);
}

// ---- back to bf16: bf16(e2m1 * block scale * tensor scale), rounded once from f32 ----
__device__ __forceinline__ uint32_t e2m1x2_to_f16x2(uint32_t byte) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b0;\n\t}" : "=r"(r) : "r"(byte));
  return r;
}

template <bool MX>
__global__ void __launch_bounds__(FQ_THREADS) fp4_dequantize_kernel(const Fp4DequantParams p) {
  const int64_t chunks = (p.K + 255) / 256;
  const int per_row = (p.K + 15) / 16;                 // 16 values a thread
  const int64_t items = (int64_t)p.rows * per_row, step = (int64_t)gridDim.x * FQ_THREADS;
  griddep_wait();
  const float ts = MX || !p.tensor_scale ? 1.f : __ldg(p.tensor_scale);
  for (int64_t it = (int64_t)blockIdx.x * FQ_THREADS + threadIdx.x; it < items; it += step) {
    const int row = (int)(it / per_row), k0 = (int)(it - (int64_t)row * per_row) * 16;
    const uint2 q = __ldg((const uint2*)(p.q + (int64_t)row * p.ldq + (k0 >> 1)));
    const uint32_t code = __ldg(p.scales + scale_offset<MX>(row, MX ? k0 >> 5 : k0 >> 4, chunks));
    float s;
    if constexpr (MX) s = code == FP4_NAN_MX ? __uint_as_float(0x7FC00000u) : code == 0u ? 0x1p-127f : __uint_as_float(code << 23);
    else s = (code & 0x7Fu) == FP4_NAN_NV ? __uint_as_float(0x7FC00000u) : e4m3_value(code & 0x7Fu);
    uint32_t out[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const uint32_t byte = ((i < 4 ? q.x : q.y) >> (8 * (i & 3))) & 0xFFu;
      const uint32_t h2 = e2m1x2_to_f16x2(byte);
      const float2 f = __half22float2(*(const __half2*)&h2);
      out[i] = pack_bf16x2(f.x * s * ts, f.y * s * ts);
    }
    __nv_bfloat16* dst = p.out + (int64_t)row * p.ldo + k0;
    if (p.K - k0 >= 16) {
      *(uint4*)dst = make_uint4(out[0], out[1], out[2], out[3]);
      *((uint4*)dst + 1) = make_uint4(out[4], out[5], out[6], out[7]);
    } else {
#pragma unroll
      for (int i = 0; i < 16; i++)
        if (k0 + i < p.K) dst[i] = __ushort_as_bfloat16((unsigned short)(out[i >> 1] >> (16 * (i & 1))));
    }
  }
}

cudaError_t launch_fp4_dequantize(const Fp4DequantParams& p, bool pdl, cudaStream_t stream) {
  if (p.rows <= 0 || p.K <= 0) return cudaSuccess;
  const int64_t items = (int64_t)p.rows * ((p.K + 15) / 16);
  int64_t blocks = (items + FQ_THREADS - 1) / FQ_THREADS;
  if (blocks > 148 * 64) blocks = 148 * 64;
  return launch_kernel(p.mx ? fp4_dequantize_kernel<true> : fp4_dequantize_kernel<false>, dim3((unsigned)blocks), FQ_THREADS, 0, stream, pdl, 1, false, p);
}

}  // namespace krea
