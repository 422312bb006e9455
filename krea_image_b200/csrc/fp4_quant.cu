// bf16 rows -> packed 4-bit rows with block scales, and back (formats and rounding: fp4_block.cuh).
//
// Storage: two values a byte, the lower index in the low bits, rows of whole 16 bytes (32 values; values past K are
// zero); scales as fp4_block.cuh lays them out, zero past K and past the last row.  A block with an infinity or a NaN
// gets the scale code NaN, so that products with it become NaN.
//
// HBM-bound: 2 bytes read and 0.53 (MX) or 0.56 (NV) written per value.  A warp takes the four blocks that share a
// 4-byte word of scales from rows 32 apart, which makes its scale bytes one contiguous piece (16 or 32 bytes) and its
// reads whole 128-byte lines.  Measured at 4608 x 16384: MX 30 us (98 % of the copy bandwidth), NV 39.5 us (76 %: the
// instructions of the scales), back to bf16 32.3 and 33.6 us (92 and 89 %).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "fp4.h"
#include "fp4_block.cuh"
#include "sm100_ptx.cuh"

namespace krea {

constexpr int FQ_THREADS = 256;

// 16 values from `src` (16-byte aligned; `wide`: 32), zero from index `left` on
__device__ __forceinline__ void load16(const __nv_bfloat16* src, int left, bool wide, uint32_t* w) {
  if (left >= 16 && wide) {       // one access a lane and not two, 32 bytes apart, that cost L1 twice the passes
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(src));
  } else if (left >= 16) {
    const uint4 a = ld_global_16B(src), b = ld_global_16B(src + 8);
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

// How a CTA's 8 warps lie on (column, row) items: 2^cols_log2 of them beside one another, the others on further rows.  Row items
// go on in steps of the grid's height, so that no index is divided.
struct Fp4Shape {
  int cols, cols_log2;      // column items; log2 of how many a CTA has
  int row_items;
};

template <bool MX>
__global__ void __launch_bounds__(FQ_THREADS) fp4_quantize_rows_kernel(const Fp4QuantParams p, const Fp4Shape z) {
  constexpr int LANES = MX ? 8 : 4;              // lanes of a row: 16 values each, four blocks together
  constexpr int GROUP = LANES * 16;              // values of those four blocks; a column item is two such groups
  constexpr int RUNS = MX ? 32 : 16;             // row items that cover the 128 rows of a scale tile
  const int64_t chunks = (p.K + 255) / 256;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, in_row = lane % LANES, rr = lane / LANES;
  griddep_wait();
  __shared__ NvTable nv;
  if constexpr (!MX) {
    if (threadIdx.x < 128) nv_table_fill(nv, p.tensor_scale ? ld_global_f1(p.tensor_scale) : 1.f, threadIdx.x);
    __syncthreads();
  }
  const bool wide = (((uintptr_t)p.src | (uintptr_t)(p.ld * 2)) & 31u) == 0;
  const int g = (((int)blockIdx.x << z.cols_log2) + (warp & ((1 << z.cols_log2) - 1))) * 2, rows_cta = 8 >> z.cols_log2;
  if (g >= 2 * z.cols) return;
  for (int tr = (int)blockIdx.y * rows_cta + (warp >> z.cols_log2); tr < z.row_items; tr += (int)gridDim.y * rows_cta) {
    const int run = tr % RUNS;
    const int row = tr / RUNS * 128 + (rr & 3) * 32 + (MX ? run : run * 2 + (rr >> 2));
    const __nv_bfloat16* src = p.src + (int64_t)row * p.ld;
    uint32_t w[2][8];
#pragma unroll
    for (int i = 0; i < 2; i++) {                // both loads are under way before the first is used
      const int k0 = (g + i) * GROUP + in_row * 16;
      load16(src + k0, row < p.rows ? p.K - k0 : 0, wide, w[i]);
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

// The same for an input-major source [K, ld] (row k holds value k of every output row).  CTAs stay and walk over tiles of 128 k x
// 128 rows, which TMA brings into a ring of three (zeros past K and past the last row); a lane has two neighbouring
// output rows and a warp 32 k.  Packed rows and scales are collected in shared memory and leave as whole pieces.
// Measured at 6144 x 15360: NV 54 us (69 % of the copy bandwidth; twice that with a tile a CTA and loads through registers), MX 45 us
// (83 %).
constexpr int FT_K = 128, FT_N = 128, FT_THREADS = 256, FT_STAGES = 3, FT_TILE = FT_K * FT_N * 2;
constexpr int FT_PACKED = FT_K / 2 + 16;             // a packed row's bytes and the step to the next in shared memory
constexpr int FT_SMEM = FT_STAGES * FT_TILE + FT_N * FT_PACKED + FT_N * (FT_K / 16) + 64 + 128;
enum : uint32_t { SITE_QUANT_FULL = 31 };
template <bool MX>
__global__ void __launch_bounds__(FT_THREADS, 2) fp4_quantize_cols_kernel(const __grid_constant__ CUtensorMap tm, const Fp4QuantParams p) {
  constexpr int PIECES = MX ? 1 : 2;                 // 512-byte pieces of scales a tile
  extern __shared__ __align__(128) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((128u - (smem_u32(smem_raw) & 127u)) & 127u);
  uint8_t* packed = smem + FT_STAGES * FT_TILE;
  uint8_t* scales = packed + FT_N * FT_PACKED;
  uint64_t* full = (uint64_t*)(scales + FT_N * (FT_K / 16));
  __shared__ uint32_t abort_word[2];
  __shared__ NvTable nv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kt = (p.K + 255) / 256 * 2, nt = (p.rows + FT_N - 1) / FT_N;       // padding included: its scales are written too
  // tiles in steps of the grid, rows fastest
  struct Place {
    int k, n;
  };
  const int step_k = (int)gridDim.x / nt, step_n = (int)gridDim.x - step_k * nt;
  const auto next = [&](Place& t) {
    t.k += step_k;
    t.n += step_n;
    if (t.n >= nt) t.n -= nt, t.k++;
  };
  Place at = {(int)blockIdx.x / nt, 0}, ahead;
  at.n = (int)blockIdx.x - at.k * nt;
  ahead = at;
  if (threadIdx.x == 0) {
    for (int s = 0; s < FT_STAGES; s++) mbar_init(&full[s], 1);
    abort_word[0] = 0u;
    fence_mbar_init();
  }
  griddep_wait();
  if constexpr (!MX) {
    if (threadIdx.x < 128) nv_table_fill(nv, p.tensor_scale ? ld_global_f1(p.tensor_scale) : 1.f, threadIdx.x);
  }
  __syncthreads();
  const auto request = [&](int s) {                // the next tile not asked for yet, if there is one
    if (ahead.k < kt) {
      mbar_arrive_expect_tx(&full[s], FT_TILE);
      tma_load_3d(smem + s * FT_TILE, &tm, &full[s], ahead.n * FT_N, ahead.k * FT_K, 0);
      next(ahead);
    }
  };
  if (threadIdx.x == 0) {
    for (int s = 0; s < FT_STAGES; s++) request(s);
  }
  const int g = warp & 3, n2 = (warp >> 2) * 32 + lane;       // 32 k from 32 g on, output rows 2 n2 and 2 n2 + 1 of the tile
  int s = 0;
  uint32_t phase = 0;
  for (; at.k < kt; next(at)) {
    const int n0 = at.n * FT_N, k0 = at.k * FT_K;
    if (__syncthreads_or(!mbar_wait(&full[s], phase, abort_word, SITE_QUANT_FULL))) break;
    const uint32_t* tile = (const uint32_t*)(smem + s * FT_TILE);
    uint32_t t[32];
#pragma unroll
    for (int i = 0; i < 32; i++) t[i] = tile[(g * 32 + i) * (FT_N / 2) + n2];
    __syncthreads();                                 // the stage has been read, and the last tile's results have left
    if (threadIdx.x == 0) request(s);
    if (++s == FT_STAGES) s = 0, phase ^= 1u;
#pragma unroll
    for (int half = 0; half < 2; half++) {
      const int n = 2 * n2 + half;
      uint32_t w[16], out[4];
#pragma unroll
      for (int i = 0; i < 16; i++) w[i] = __byte_perm(t[2 * i], t[2 * i + 1], half ? 0x7632 : 0x5410);
      uint8_t* sc = scales + (n & 31) * 16 + (n >> 5) * 4;
      if constexpr (MX) {
        const uint32_t code = mx_scale_code(amax_bits<16>(w));
#pragma unroll
        for (int j = 0; j < 4; j++) out[j] = mx_encode8(w + 4 * j, code);
        sc[g] = (uint8_t)code;
      } else {
#pragma unroll
        for (int blk = 0; blk < 2; blk++) {
          const uint32_t code = nv_scale_code(amax_bits<8>(w + 8 * blk), nv);
          nv_encode<8>(w + 8 * blk, code, nv, out + 2 * blk);
          sc[(g >> 1) * 512 + (g & 1) * 2 + blk] = (uint8_t)code;
        }
      }
      *(uint4*)(packed + n * FT_PACKED + g * 16) = make_uint4(out[0], out[1], out[2], out[3]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < FT_N * (FT_K / 32); i += FT_THREADS) {
      const int r = i / (FT_K / 32), j = i % (FT_K / 32);
      if (n0 + r < p.rows && k0 + j * 32 < p.K) *(uint4*)(p.q + (int64_t)(n0 + r) * p.ldq + (k0 >> 1) + j * 16) = *(const uint4*)(packed + r * FT_PACKED + j * 16);
    }
    if (threadIdx.x < PIECES * 32) {
      uint8_t* dst = p.scales + scale_offset<MX>(n0, MX ? k0 >> 5 : k0 >> 4, (p.K + 255) / 256);
      ((uint4*)dst)[threadIdx.x] = ((const uint4*)scales)[threadIdx.x];
    }
  }
  // after a wait that ran out: nothing may be in flight into this CTA's shared memory when it exits
  if (abort_word[0] != 0u && threadIdx.x == 0) {
    for (int i = 0; i < FT_STAGES; i++) mbar_wait_slow(&full[(s + i) % FT_STAGES], phase ^ (s + i >= FT_STAGES ? 1u : 0u), abort_word + 1, SITE_QUANT_FULL);
    if (p.status) atomicCAS(p.status, 0u, abort_word[0] | ((blockIdx.x & 0xFFFu) << 8));
  }
}

cudaError_t launch_fp4_quantize_cols(const CUtensorMap& tm, const Fp4QuantParams& p, int sms, bool pdl, cudaStream_t stream) {
  if (p.rows <= 0 || p.K <= 0) return cudaSuccess;
  auto* k = p.mx ? fp4_quantize_cols_kernel<true> : fp4_quantize_cols_kernel<false>;
  static ConfiguredOnce once[2];
  const cudaError_t e = once[p.mx].set(k, FT_SMEM);
  if (e != cudaSuccess) return e;
  const int64_t items = (int64_t)((p.K + 255) / 256 * 2) * ((p.rows + FT_N - 1) / FT_N);
  return launch_kernel(k, dim3((unsigned)(items < 2 * sms ? items : 2 * sms)), FT_THREADS, FT_SMEM, stream, pdl, 1, false, tm, p);
}

// the grid for these items, `most` CTAs at most
static dim3 shape_grid(int64_t cols, int64_t row_items, int64_t most, Fp4Shape* z) {
  z->cols = (int)cols;
  z->row_items = (int)row_items;
  z->cols_log2 = 0;
  while (z->cols_log2 < 3 && (1ll << z->cols_log2) < cols) z->cols_log2++;
  const int64_t x = (cols + (1ll << z->cols_log2) - 1) >> z->cols_log2, rows_cta = 8 >> z->cols_log2;
  int64_t y = (row_items + rows_cta - 1) / rows_cta;
  if (x * y > most) y = most / x;
  if (y < 1) y = 1;
  if (y > 65535) y = 65535;
  return dim3((unsigned)x, (unsigned)y);
}

cudaError_t launch_fp4_quantize(const Fp4QuantParams& p, int sms, bool pdl, cudaStream_t stream) {
  if (p.rows <= 0 || p.K <= 0) return cudaSuccess;
  const int64_t tiles = (p.rows + 127) / 128, chunks = (p.K + 255) / 256;
  Fp4Shape z;
  // MX: two rounds of the CTAs that fit.  NV: one round, since each fills its table first (4608 x 16384: 39 us, 45 with MX's)
  const dim3 grid = shape_grid(chunks * (p.mx ? 1 : 2), tiles * (p.mx ? 32 : 16), (int64_t)sms * (p.mx ? 16 : 4), &z);
  return launch_kernel(p.mx ? fp4_quantize_rows_kernel<true> : fp4_quantize_rows_kernel<false>, grid, FQ_THREADS, 0, stream, pdl, 1, false, p, z);
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
  const bool narrow = items <= 0xFFFFFFFFll;            // a 64-bit division costs as much as the rest
  const bool wide = (((uintptr_t)p.out | (uintptr_t)(p.ldo * 2)) & 31u) == 0;
  griddep_wait();
  const float ts = MX || !p.tensor_scale ? 1.f : ld_global_f1(p.tensor_scale);
  for (int64_t it = (int64_t)blockIdx.x * FQ_THREADS + threadIdx.x; it < items; it += step) {
    const int row = narrow ? (int)((uint32_t)it / (uint32_t)per_row) : (int)(it / per_row), k0 = (int)(it - (int64_t)row * per_row) * 16;
    const uint2 q = ld_global_8B(p.q + (int64_t)row * p.ldq + (k0 >> 1));
    const uint32_t code = ld_global_u8(p.scales + scale_offset<MX>(row, MX ? k0 >> 5 : k0 >> 4, chunks));
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
    if (p.K - k0 >= 16 && wide) {
      st_global_32B(dst, out);
    } else if (p.K - k0 >= 16) {
      *(uint4*)dst = make_uint4(out[0], out[1], out[2], out[3]);
      *((uint4*)dst + 1) = make_uint4(out[4], out[5], out[6], out[7]);
    } else {
#pragma unroll
      for (int i = 0; i < 16; i++)
        if (k0 + i < p.K) dst[i] = __ushort_as_bfloat16((unsigned short)(out[i >> 1] >> (16 * (i & 1))));
    }
  }
}

cudaError_t launch_fp4_dequantize(const Fp4DequantParams& p, int sms, bool pdl, cudaStream_t stream) {
  if (p.rows <= 0 || p.K <= 0) return cudaSuccess;
  const int64_t items = (int64_t)p.rows * ((p.K + 15) / 16);
  int64_t blocks = (items + FQ_THREADS - 1) / FQ_THREADS;
  if (blocks > (int64_t)sms * 64) blocks = (int64_t)sms * 64;
  return launch_kernel(p.mx ? fp4_dequantize_kernel<true> : fp4_dequantize_kernel<false>, dim3((unsigned)blocks), FQ_THREADS, 0, stream, pdl, 1, false, p);
}

}  // namespace krea
