// 4-bit GEMM for B200 (sm_100a): C[M, N] = (A . sA) x (W . sW)^T on packed e2m1 rows with block scales, both operands
// with K innermost, fp32 accumulation, the epilogues of the bf16 GEMM.
//
// tcgen05.mma kind::mxf4nvf4 (NV, a scale each 16 values) and kind::mxf4 (MX, each 32) multiply 64 values of K an
// instruction and take the scales from tensor memory: 32 lanes x 4 columns of words for 128 rows, repeated in the four
// lane quarters.  The scale storage (fp4_block.cuh) is that order, so a 512-byte piece goes from memory to shared memory by
// TMA and to tensor memory by one tcgen05.cp, untouched.
//
// Two kernels:
//   gemm_fp4_rows_sm100   few rows of A: the 128 tensor-core rows are columns of C (rows of W), the rows of A (16 to 128)
//                         are its columns, so the weights stream through once and no tensor-core row idles; the CTAs of a
//                         cluster share K and add their parts through shared memory, in a fixed order.  HBM-bound:
//                         1 x 15360 x 6144 NV 12 us, of which the 53 MB take 8.2 at the copy bandwidth.
//   gemm_fp4_pair_sm100   many rows: 256 x 256 tiles on CTA pairs (cta_group::2), persistent, like the bf16 kernel.  A stage
//                         moves 38 KB (NV) into each SM for 512 clocks of products, about what L2 delivers, and the clock falls under the
//                         power cap, to 1.55 GHz in a short run and 1.35 in a long one: 4608 x 15360 x 6144 NV 184 us in a run of two
//                         seconds (4.7 PFLOP/s), 156 us among single launches.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/krea_cuda.h"
#include "fp4.h"
#include "sm100_pair.cuh"
#include "sm100_ptx.cuh"

namespace krea {

namespace fp4g {
enum : uint32_t { SITE_FULL = 21, SITE_EMPTY = 22, SITE_ACC_FULL = 23, SITE_ACC_EMPTY = 24, SITE_PARTS = 25 };
constexpr int KB = 256;                              // values of K a stage: one 128-byte row of packed values
constexpr int ROW_TILE_BYTES = 128 * 128;            // 128 rows of a stage
__host__ __device__ constexpr int scale_chunk(bool mx) { return mx ? 1024 : 2048; }   // scale bytes of 128 rows x 256 values
__host__ __device__ constexpr int scale_pieces(bool mx) { return mx ? 2 : 4; }        // 512-byte pieces (4 columns of tensor memory) among them

// instruction descriptor of the block-scaled kinds: e2m1 x e2m1, fp32 accumulator, both operands K-major
__host__ __device__ constexpr uint32_t idesc(bool mx, int M, int N) {
  return (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((mx ? 1u : 0u) << 23) | ((uint32_t)(M >> 4) << 24);
}
// which bytes of the scale words an MX instruction takes: 0 the lower two, 2 the upper two (bits 29-30: A, 4-5: B)
__host__ __device__ constexpr uint32_t idesc_sf(uint32_t id) { return (id << 29) | (id << 4); }

template <bool MX, int CTAS>
__device__ __forceinline__ void mma(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc_, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  if constexpr (MX && CTAS == 1)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\ttcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                 ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc_), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
  else if constexpr (MX)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\ttcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                 ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc_), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
  else if constexpr (CTAS == 1)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\ttcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                 ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc_), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\ttcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
                 ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc_), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}
// 512 bytes of scales, shared -> tensor memory: 32 lanes x 16 bytes, repeated in the four lane quarters
template <int CTAS>
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint32_t saddr16) {
  // no swizzle, groups of 8 rows x 16 bytes 128 bytes apart
  const uint64_t desc = make_desc(saddr16, (128u >> 4) | (1u << 14));
  if constexpr (CTAS == 1) asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
  else asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}

// Both tensor scales, and whether an earlier kernel gave up on a wait (then nothing is stored).  Asked for at the kernel's start
// and not where the compiler would put it, next to the use: a memory latency at the end of every launch.  Looked at only
// at the use: before that nobody waits for them.  The status says only what is stored: loads and products run to their end
// either way, since CTAs of a cluster that stopped after different stages would leave loads and signals under way to one another.
struct Early {
  float a = 1.f, w = 1.f;
  uint32_t status = 0u;
  __device__ __forceinline__ explicit Early(const Fp4GemmParams& p) {
    if (p.a_ts) asm volatile("ld.global.f32 %0, [%1];" : "=f"(a) : "l"(p.a_ts));
    if (p.w_ts) asm volatile("ld.global.f32 %0, [%1];" : "=f"(w) : "l"(p.w_ts));
    if (p.status) asm volatile("ld.volatile.global.u32 %0, [%1];" : "=r"(status) : "l"(p.status));
  }
};
// The factor of a sum is the product of both tensor scales.  Where that is below the normal f32 numbers (digits would be lost) or
// beyond the largest (a sum of zero would become NaN), sums are first multiplied by a power of two that the factor then lacks:
// exact wherever the result is neither zero nor infinite.  That happens in tensor memory and out of line, since no ordinary
// tensors come here (and MX has no such scales): a second product for each value cost 0.45 us on 600 x 6144 x 2048 with GELU.
__device__ __forceinline__ bool is_normal(float positive) { return __float_as_uint(positive) - 0x00800000u < 0x7F000000u; }
// such scales: this warp's lanes of the accumulator, `cols` columns (a multiple of 32) from `src` on, times that power; returns the factor
__device__ __noinline__ float scale_sums(uint32_t src, int cols, float a, float w) {
  const float small = a < w ? a : w, large = a < w ? w : a;
  const bool low = small * large < 1.f;
  const float pre = low ? 0x1p-64f : 0x1p100f;
#pragma unroll 1
  for (int c0 = 0; c0 < cols; c0 += 32) {
    uint32_t v[32];
    tmem_ld32(src + (uint32_t)c0, v);
    tmem_wait_ld();
#pragma unroll
    for (int e = 0; e < 32; e++) v[e] = __float_as_uint(__uint_as_float(v[e]) * pre);
    tmem_st32(src + (uint32_t)c0, v);
    tmem_wait_st();
  }
  const float alpha = low ? small * 0x1p64f * large : large * 0x1p-100f * small;
  return alpha > 3.402823466e38f ? 3.402823466e38f : alpha;      // a sum that is not zero becomes infinite all the same
}
__device__ __forceinline__ float gelu_tanh(float x) { return 0.5f * x * (1.0f + tanhf(0.7978845608028654f * (x + 0.044715f * x * x * x))); }

// Everything after the sum for 8 columns of one row (SwiGLU apart), and their store.  vec: p.vec, from after_wait()
__device__ __forceinline__ void finish8(const Fp4GemmParams& p, const float* vec, float* f, int row, int col) {
  if (p.epi == KREA_CUDA_EPI_BIAS_BF16 || p.epi == KREA_CUDA_EPI_BIAS_F32) {
    const float4 a = ld_global_f4(vec + col), b = ld_global_f4(vec + col + 4);
    f[0] += a.x; f[1] += a.y; f[2] += a.z; f[3] += a.w; f[4] += b.x; f[5] += b.y; f[6] += b.z; f[7] += b.w;
  } else if (p.epi == KREA_CUDA_EPI_GELU) {
#pragma unroll
    for (int e = 0; e < 8; e++) f[e] = gelu_tanh(f[e]);
  }
  const int64_t at = (int64_t)row * p.ldc + col;
  if (p.epi == KREA_CUDA_EPI_RESID_GATE) {
    float4* o = (float4*)((float*)p.C + at);
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const float4 gt = vec ? ld_global_f4(vec + col + 4 * e) : make_float4(1.f, 1.f, 1.f, 1.f);
      float4 x = o[e];
      x.x = fmaf(gt.x, f[4 * e], x.x); x.y = fmaf(gt.y, f[4 * e + 1], x.y); x.z = fmaf(gt.z, f[4 * e + 2], x.z); x.w = fmaf(gt.w, f[4 * e + 3], x.w);
      o[e] = x;
    }
  } else if (p.epi == KREA_CUDA_EPI_F32 || p.epi == KREA_CUDA_EPI_BIAS_F32) {
    float4* o = (float4*)((float*)p.C + at);
    o[0] = make_float4(f[0], f[1], f[2], f[3]);
    o[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    *(uint4*)((__nv_bfloat16*)p.C + at) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  }
}

// Epilogue of a warp of the pair kernel: rows [row0, row0 + 32), a lane each, columns [col0, col0 + 128).  The results leave
// through shared memory as boxes of 32 rows x 128 bytes by TMA, which writes whole lines and stops at the last row and
// column by itself.  Stored from registers, 32 bytes of 32 rows at a time, a tile took 5000 clocks and held up the loads of
// the next one (3800 clocks a tile lost at 4608 x 15360 x 6144).  box: one box, used again and again, or `many` in a row.
__device__ __forceinline__ void pair_store(const Fp4GemmParams& p, const float* vec, const CUtensorMap& tmC, const uint32_t* v, int row0, int col0, float alpha, uint8_t* box, bool many, int lane) {
  const bool swiglu = p.epi == KREA_CUDA_EPI_SWIGLU, f32 = p.epi == KREA_CUDA_EPI_F32 || p.epi == KREA_CUDA_EPI_BIAS_F32;
  uint32_t dst = smem_u32(box) + lane * 128;
  // 16 bytes at place q of the lane's row, swizzled as the tensor map has it
  const auto put = [&](int q, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + (uint32_t)((q ^ (lane & 7)) << 4)), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
  };
  const auto acc = [&](int i) { return __uint_as_float(v[i]) * alpha; };
  const auto begin = [&] {                       // the box before this one has been read
    if (many) return;
    if (lane == 0) tma_store_wait_read();
    __syncwarp();
  };
  const auto send = [&](int col) {
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      tma_store_3d(&tmC, box, col, row0, 0);
      tma_store_commit();
    }
    if (many) {
      box += 32 * 128;
      dst += 32 * 128;
    }
  };
  if (swiglu) {                                  // 32 gate columns, then the 32 they gate: 64 columns of C
    begin();
#pragma unroll
    for (int q = 0; q < 8; q++) {
      uint32_t pk[4];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int c = (q >> 2) * 64 + (q & 3) * 8 + 2 * e;
        const float g0 = acc(c), g1 = acc(c + 1);
        pk[e] = pack_bf16x2(g0 * sigmoid_approx(g0) * acc(c + 32), g1 * sigmoid_approx(g1) * acc(c + 33));
      }
      put(q, pk[0], pk[1], pk[2], pk[3]);
    }
    send(col0 >> 1);
    return;
  }
  if (f32) {
#pragma unroll
    for (int c0 = 0; c0 < 128; c0 += 32) {
      if (col0 + c0 >= p.N) break;
      begin();
#pragma unroll
      for (int q = 0; q < 8; q++) {
        const int c = c0 + q * 4;
        float4 b = make_float4(0.f, 0.f, 0.f, 0.f);
        if (p.epi == KREA_CUDA_EPI_BIAS_F32 && col0 + c < p.N) b = ld_global_f4(vec + col0 + c);
        put(q, __float_as_uint(acc(c) + b.x), __float_as_uint(acc(c + 1) + b.y), __float_as_uint(acc(c + 2) + b.z), __float_as_uint(acc(c + 3) + b.w));
      }
      send(col0 + c0);
    }
    return;
  }
  // one path a kind, each without the others' instructions between its own: a cold launch fetches them once, in order
  const auto bf16_boxes = [&](auto after) {
#pragma unroll
    for (int c0 = 0; c0 < 128; c0 += 64) {
      if (col0 + c0 >= p.N) break;
      begin();
#pragma unroll
      for (int q = 0; q < 8; q++) {
        const int c = c0 + q * 8;
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; e++) f[e] = acc(c + e);
        after(f, col0 + c);
        put(q, pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
      }
      send(col0 + c0);
    }
  };
  if (p.epi == KREA_CUDA_EPI_BF16) {
    bf16_boxes([](float*, int) {});
  } else if (p.epi == KREA_CUDA_EPI_BIAS_BF16) {
    bf16_boxes([&](float* f, int col) {
      if (col < p.N) {
        const float4 a = ld_global_f4(vec + col), b = ld_global_f4(vec + col + 4);
        f[0] += a.x; f[1] += a.y; f[2] += a.z; f[3] += a.w; f[4] += b.x; f[5] += b.y; f[6] += b.z; f[7] += b.w;
      }
    });
  } else {
    bf16_boxes([](float* f, int) {
#pragma unroll
      for (int e = 0; e < 8; e++) f[e] = gelu_tanh(f[e]);
    });
  }
}
// C (f32) += vec * acc for a warp's 32 rows, a lane each, and 128 columns.  The vector's piece waits in shared memory (`piece`, 512
// bytes): a load of it from global memory stays behind every store to C before it (367 us at 4608 x 6144 x 16384, not 196).
__device__ __forceinline__ void pair_add(const Fp4GemmParams& p, const float* vec, const uint32_t* v, int row0, int col0, float alpha, uint8_t* piece, int lane) {
  const uint32_t gates = smem_u32(piece);
  float4 g = make_float4(1.f, 1.f, 1.f, 1.f);
  if (vec && col0 + 4 * lane < p.N) g = ld_global_f4(vec + col0 + 4 * lane);
  __syncwarp();                                  // the last tile's piece has been read
  asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(gates + lane * 16), "f"(g.x), "f"(g.y), "f"(g.z), "f"(g.w) : "memory");
  __syncwarp();
  if (row0 + lane >= p.M) return;
  float* row = (float*)p.C + (int64_t)(row0 + lane) * p.ldc + col0;
#pragma unroll
  for (int c = 0; c < 128; c += 8) {
    if (col0 + c >= p.N) break;
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      float4 gt, x = *(const float4*)(row + c + e);
      asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(gt.x), "=f"(gt.y), "=f"(gt.z), "=f"(gt.w) : "r"(gates + (c + e) * 4));
      x.x = fmaf(gt.x, __uint_as_float(v[c + e]) * alpha, x.x);
      x.y = fmaf(gt.y, __uint_as_float(v[c + e + 1]) * alpha, x.y);
      x.z = fmaf(gt.z, __uint_as_float(v[c + e + 2]) * alpha, x.z);
      x.w = fmaf(gt.w, __uint_as_float(v[c + e + 3]) * alpha, x.w);
      *(float4*)(row + c + e) = x;
    }
  }
}

// ---------------------------------------------------------------------------------------------- few rows
// A stage: 128 rows of W, tn rows of A (a multiple of 16), the scales of the row tiles that hold them
__host__ __device__ constexpr int rows_stage_bytes(bool mx, int tn) { return ROW_TILE_BYTES + tn * 128 + 2 * scale_chunk(mx); }
__host__ __device__ constexpr int rows_sf_cols(bool mx) { return 2 * 4 * scale_pieces(mx); }      // tensor-memory columns of a stage's scales
__host__ __device__ constexpr int rows_acc_cols(int tn) { return (tn + 31) & ~31; }
__host__ __device__ constexpr int rows_tmem_cols(bool mx, int tn, int stages) {
  const int used = rows_acc_cols(tn) + stages * rows_sf_cols(mx);
  return used <= 128 ? 128 : used <= 256 ? 256 : 512;
}
// The tile and the other CTAs' parts lie over the stages, (2 tn + 8) * 512 bytes at most.  They fit in every plan that shares K: a stage
// has tn * 128 bytes and 18 KB more, and there are six stages, or three and 64 rows at most (two CTAs an SM).
constexpr int ROWS_MAX_STAGES = 8;
constexpr int ROWS_THREADS = 192;   // warp 0 TMA, warp 1 MMA, warps 2-5 epilogue
}  // namespace fp4g

template <bool MX>
__global__ void __launch_bounds__(fp4g::ROWS_THREADS)
gemm_fp4_rows_sm100(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmAs, const __grid_constant__ CUtensorMap tmW,
                    const __grid_constant__ CUtensorMap tmWs, const Fp4GemmParams p) {
  using namespace fp4g;
  constexpr int PIECES = scale_pieces(MX), S_BYTES = scale_chunk(MX), SF_COLS = rows_sf_cols(MX);
  const int TN = p.tn, STAGES = p.stages, STAGE_BYTES = rows_stage_bytes(MX, TN), Y_BYTES = TN * 128;
  const uint32_t TMEM_COLS = (uint32_t)rows_tmem_cols(MX, TN, STAGES);
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = (uint64_t*)(smem + STAGES * STAGE_BYTES);
  uint64_t* empty = full + ROWS_MAX_STAGES;
  uint64_t* acc_full = empty + ROWS_MAX_STAGES;
  uint64_t* received = acc_full + 1;                     // the other CTAs' parts of this CTA's rows have arrived
  uint32_t* tmem_slot = (uint32_t*)(received + 1);
  volatile uint32_t* abort_word = (volatile uint32_t*)(tmem_slot + 1);      // [0] a wait ran out; [1], [2] the same, while what is under way is awaited
  const uint64_t limit = p.wait_limit_ns;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t split = gridDim.z, rank = blockIdx.z;       // the cluster is the grid's z axis
  const int n0 = blockIdx.x * 128, m0 = blockIdx.y * TN;
  const int kblocks = (p.K + KB - 1) / KB;
  const int kb0 = (int)((int64_t)kblocks * rank / split), kb1 = (int)((int64_t)kblocks * (rank + 1) / split);

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmWs);
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmAs);
    for (int s = 0; s < STAGES; s++) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(received, 1);
    abort_word[0] = abort_word[1] = abort_word[2] = 0u;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot, sf_base = tmem_base + (uint32_t)rows_acc_cols(TN);
  griddep_wait();
  griddep_launch();
  const Early early(p);
  const float* vec = after_wait(p.vec);

  if (warp == 0) {
    if (lane == 0) {
      int s = 0, done = 0;
      uint32_t phase = 0;
      const int asked = kb1 - (p.test_drop_load && rank == split - 1 ? 1 : 0);
      for (int kb = kb0; kb < asked && *abort_word == 0u; kb++, done++) {
        if (!mbar_wait(&empty[s], phase ^ 1u, abort_word, SITE_EMPTY, limit)) break;
        uint8_t* st = smem + s * STAGE_BYTES;
        mbar_arrive_expect_tx(&full[s], STAGE_BYTES);
        tma_load_3d(st, &tmW, &full[s], kb * 128, n0, 0);
        tma_load_3d(st + ROW_TILE_BYTES, &tmA, &full[s], kb * 128, m0, 0);
        tma_load_3d(st + ROW_TILE_BYTES + Y_BYTES, &tmWs, &full[s], 0, kb, n0 >> 7);
        tma_load_3d(st + ROW_TILE_BYTES + Y_BYTES + S_BYTES, &tmAs, &full[s], 0, kb, m0 >> 7);
        if (++s == STAGES) s = 0, phase ^= 1u;
      }
      // nothing may still be in flight into this CTA's shared memory when it exits
      if (*abort_word != 0u) {
        for (int i = done > STAGES ? done - STAGES : 0; i < done; i++) mbar_wait_slow(&full[i % STAGES], (uint32_t)(i / STAGES) & 1u, abort_word + 1, SITE_FULL, limit);
      }
    }
  } else if (warp == 1) {
    const bool leader = elect_one();
    constexpr uint32_t HI = desc_hi(1024);
    const uint32_t ID = idesc(MX, 128, TN);
    const uint32_t smem16 = smem_u32(smem) >> 4;
    int s = 0, kb = kb0;
    uint32_t phase = 0;
    for (; kb < kb1; kb++) {
      if (!__all_sync(0xffffffffu, mbar_wait(&full[s], phase, abort_word, SITE_FULL, limit))) break;      // the warp decides as one
      tc_fence_after();
      const uint32_t x = smem16 + s * (STAGE_BYTES >> 4), y = x + (ROW_TILE_BYTES >> 4), sx = y + (Y_BYTES >> 4), sy = sx + (S_BYTES >> 4);
      const uint32_t tx = sf_base + s * SF_COLS, ty = tx + 4 * PIECES;
      if (leader) {
#pragma unroll
        for (int j = 0; j < PIECES; j++) {
          copy_scales<1>(tx + 4 * j, sx + j * 32);
          copy_scales<1>(ty + 4 * j, sy + j * 32);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int piece = MX ? j >> 1 : j;
          mma<MX, 1>(tmem_base, make_desc(x + j * 2, HI), make_desc(y + j * 2, HI), ID | idesc_sf(MX ? (j & 1) * 2 : 0), tx + 4 * piece, ty + 4 * piece, (kb > kb0 || j > 0) ? 1u : 0u);
        }
        umma_commit(&empty[s]);
      }
      __syncwarp();
      if (++s == STAGES) s = 0, phase ^= 1u;
    }
    if (kb == kb1) {                         // a sum that lacks a part is never announced
      if (leader) umma_commit(acc_full);
    } else {                                 // products under way still read the stages
      for (int i = max(0, kb - kb0 - STAGES); i < kb - kb0; i++) mbar_wait_slow(&empty[i % STAGES], (uint32_t)(i / STAGES) & 1u, abort_word + 2, SITE_EMPTY, limit);
    }
    __syncwarp();
  }
  // Each CTA of the cluster finishes an equal share of the tile's rows.  The tile goes from tensor memory to this CTA's shared
  // memory, over the stages, as [row][128 columns of C] f32; bulk copies take the other CTAs' rows to them, into
  // [CTA they come from][row][128 columns] behind their own tile.
  float* part = (float*)smem;
  float* parts = part + TN * 128;
  const int rows = min(TN, p.M - m0), share = (rows + (int)split - 1) / (int)split;
  const auto rows_of = [&](int q) { return max(0, min(rows - q * share, share)); };
  const int r0 = (int)rank * share, mine = rows_of((int)rank);
  if (split > 1 && threadIdx.x == 0 && mine > 0) mbar_arrive_expect_tx(received, (split - 1) * (uint32_t)mine * 512u);
  bool done = true;
  if (warp >= 2) {
    done = __all_sync(0xffffffffu, mbar_wait(acc_full, 0, abort_word, SITE_ACC_FULL, limit));      // what follows takes whole warps
    tc_fence_after();
  }
  __syncwarp();
  if (split > 1) cluster_arrive_relaxed();   // nothing uses this CTA's stages any more
  if (warp >= 2) {
    const int quarter = warp & 3;
    if (done) {
      if (!MX && !is_normal(early.a * early.w)) scale_sums(tmem_base + ((uint32_t)(quarter * 32) << 16), rows_acc_cols(TN), early.a, early.w);
#pragma unroll 1
      for (int c0 = 0; c0 < rows; c0 += 32) {
        uint32_t v[32];
        tmem_ld32(tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)c0, v);
        tmem_wait_ld();
        const uint32_t at = smem_u32(part + c0 * 128 + quarter * 32 + lane);
#pragma unroll
        for (int e = 0; e < 32; e++)
          if (c0 + e < rows) asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + e * 512), "r"(v[e]) : "memory");
      }
    }
    fence_proxy_async_smem();                // the copies read what was stored
    tc_fence_before();
  }
  __syncwarp();
  __syncthreads();
  const bool whole = *abort_word == 0u;
  bool live = whole && early.status == 0u;
  if (split > 1) {
    cluster_wait();
    if (threadIdx.x == 0 && whole) {         // an incomplete part is not sent: those who need it give up on it and store nothing
      for (uint32_t q = 0; q < split; q++) {
        const int n = rows_of((int)q);
        if (q != rank && n > 0) {
          const uint32_t dst = mapa(smem_u32(parts + (int)(rank < q ? rank : rank - 1) * share * 128), q);
          bulk_copy_cluster(dst, smem_u32(part + (int)q * share * 128), (uint32_t)n * 512u, mapa(smem_u32(received), q));
        }
      }
    }
    if (mine > 0 && !mbar_wait(received, 0, abort_word, SITE_PARTS, limit)) {
      live = false;
      // what the others may have sent all the same has to land before this CTA says that it may leave
      if (threadIdx.x == 0) mbar_wait_slow(received, 0, abort_word + 2, SITE_PARTS, limit);
    }
    __syncwarp();
    cluster_arrive_relaxed();                // this CTA has what the others sent
  }

  // parts added in rank order, 8 columns of a row at a time
  const bool swiglu = p.epi == KREA_CUDA_EPI_SWIGLU;
  const int units_log2 = swiglu ? 3 : 4;
  float alpha = MX ? 1.f : early.a * early.w;
  if (!MX && !is_normal(alpha)) alpha = scale_sums(0, 0, early.a, early.w);
  const float *own = part + r0 * 128, *before = parts, *after = parts + (int)rank * share * 128;      // parts of CTAs below and above this one
#pragma unroll 2
  for (int u = threadIdx.x; u < (live ? mine << units_log2 : 0); u += ROWS_THREADS) {
    const int r = u >> units_log2, uc = u & ((1 << units_log2) - 1);
    const int c = swiglu ? (uc >> 2) * 64 + (uc & 3) * 8 : uc * 8;       // first of the tile's columns (SwiGLU: of the gate's)
    if (n0 + c >= p.N) continue;
    float f[8], g[8];
    const auto sum = [&](int col, float* o) {
      const int at = r * 128 + col;
#pragma unroll
      for (int e = 0; e < 8; e++) o[e] = 0.f;
      const auto add = [&](const float* from) {
        const float4 x = *(const float4*)(from + at), y = *(const float4*)(from + at + 4);
        o[0] += x.x; o[1] += x.y; o[2] += x.z; o[3] += x.w; o[4] += y.x; o[5] += y.y; o[6] += y.z; o[7] += y.w;
      };
      for (uint32_t q = 0; q < rank; q++) add(before + q * share * 128);
      add(own);
      for (uint32_t q = rank + 1; q < split; q++) add(after + (q - rank - 1) * share * 128);
#pragma unroll
      for (int e = 0; e < 8; e++) o[e] *= alpha;
    };
    sum(c, f);
    int col = n0 + c;
    if (swiglu) {
      sum(c + 32, g);
#pragma unroll
      for (int e = 0; e < 8; e++) f[e] = f[e] * sigmoid_approx(f[e]) * g[e];
      col = ((n0 + c) >> 6) * 32 + (uc & 3) * 8;
    }
    finish8(p, vec, f, m0 + r0 + r, col);
  }
  if (!done) mbar_wait_slow(acc_full, 0, abort_word + 2, SITE_ACC_FULL, limit);      // products that are late may not meet a CTA that has left
  __syncwarp();
  __syncthreads();
  if (split > 1) cluster_wait();             // the others have what this CTA sent
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
  if (threadIdx.x == 0 && p.status != nullptr) {
    const uint32_t a = *abort_word;
    if (a != 0u) atomicCAS(p.status, 0u, a | ((blockIdx.x & 0xFFFu) << 8));
  }
}

// ---------------------------------------------------------------------------------------------- many rows
namespace fp4g {
template <bool MX>
struct PairCfg {
  static constexpr int S_BYTES = scale_chunk(MX);
  // this CTA's 128 rows of A and of W (half of the tile's columns), the scales of its rows of A and of all 256 columns
  static constexpr int STAGE_BYTES = 2 * ROW_TILE_BYTES + 3 * S_BYTES;
  static constexpr int STAGES = 5;
  static constexpr int OUT_BYTES = 32 * 128;               // a warp's output box: 32 rows x 128 bytes
  static constexpr int SF_COLS = 3 * 4 * scale_pieces(MX);
  static constexpr int ACC_COLS = 256;
  static constexpr int TMEM_COLS = 512;
  static constexpr int SMEM = STAGES * STAGE_BYTES + 8 * OUT_BYTES + 256 + 1024;
  static_assert(8 * 4 * OUT_BYTES <= STAGES * STAGE_BYTES, "the last tile's boxes lie over the stages");
  static_assert(ACC_COLS + STAGES * SF_COLS <= TMEM_COLS && SMEM <= 227 * 1024, "tile does not fit");
};
// ns between the output of one epilogue warp and the next, for each stage of K (340 ns of products): seven such steps, twice as
// long at worst, end before the next tile does
constexpr int PACE_NS = 22;
constexpr int PAIR_THREADS = 384;   // warp 0 TMA, warp 1 MMA, warps 4-11 epilogue (two for each quarter of the tensor-memory lanes)
}  // namespace fp4g

template <bool MX>
__global__ void __launch_bounds__(fp4g::PAIR_THREADS, 1)
gemm_fp4_pair_sm100(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmAs, const __grid_constant__ CUtensorMap tmW,
                    const __grid_constant__ CUtensorMap tmWs, const __grid_constant__ CUtensorMap tmC, const Fp4GemmParams p) {
  using namespace fp4g;
  using C = PairCfg<MX>;
  constexpr int STAGES = C::STAGES, STAGE_BYTES = C::STAGE_BYTES, PIECES = scale_pieces(MX), BN = 256, TILE_M = 256;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* out_smem = smem + STAGES * STAGE_BYTES;
  uint64_t* full = (uint64_t*)(out_smem + 8 * C::OUT_BYTES);   // [STAGES] TMA landed (the leader's count both CTAs' bytes)
  uint64_t* empty = full + STAGES;                             // [STAGES] MMAs that read the stage have finished
  uint64_t* acc_full = empty + STAGES;                         // accumulator complete
  uint64_t* acc_empty = acc_full + 1;                          // accumulator in registers (the leader's, by both CTAs' epilogue warps)
  uint32_t* tmem_slot = (uint32_t*)(acc_empty + 1);
  // [0] a wait ran out; [1] the loading warp's; [2] the same, while what is under way is awaited
  volatile uint32_t* abort_word = (volatile uint32_t*)(tmem_slot + 1);
  const uint64_t limit = p.wait_limit_ns;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();     // 0 = leader
  const int worker = blockIdx.x >> 1, workers = gridDim.x >> 1;
  const int mt = (p.M + TILE_M - 1) / TILE_M, nt = (p.N + BN - 1) / BN;
  const int kblocks = (p.K + KB - 1) / KB, tiles = mt * nt;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmWs);
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmAs);
    tma_prefetch_desc(&tmC);
    for (int s = 0; s < STAGES; s++) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, 16);      // one arrival a warp: 512 threads' would take longer than the loads they report
    abort_word[0] = abort_word[1] = abort_word[2] = 0u;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc2(tmem_slot, C::TMEM_COLS);
    tmem_relinquish2();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();       // the peer's barriers are initialised, both allocations are done
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot, sf_base = tmem_base + C::ACC_COLS;

  // tile t -> origin: groups of group_m row blocks x all column blocks, row block fastest, so that the pairs running
  // together share a few rows of both operands and a group's slice of A stays in L2
  auto tile_origin = [&](int t, int& m0, int& n0) {
    const int per_group = p.group_m * nt;
    const int g = t / per_group, first = g * p.group_m;
    const int gm = min(p.group_m, mt - first);
    const int local = t - g * per_group;
    m0 = (first + local % gm) * TILE_M + (int)rank * 128;     // this CTA's rows of the tile
    n0 = (local / gm) * BN;
  };
  int m0 = 0, n0 = 0;
  tile_origin(worker, m0, n0);       // the divisions of the first tile are done before the wait
  griddep_wait();
  griddep_launch();
  if (warp == 0) {
    if (lane == 0) {
      // The two CTAs have to stop behind the same stage, or loads of one would be awaited by neither: so nothing but the
      // stages' own barriers, which the products free in both, ends this loop, and its waits are longer than the two that the
      // products' warp can spend between one stage and the next.
      const uint64_t long_limit = 3 * limit;
      uint32_t n = 0;
      bool ok = true;
      for (int t = worker; t < tiles && ok; t += workers) {
        if (t != worker) tile_origin(t, m0, n0);
        for (int kb = 0; kb < kblocks; kb++, n++) {
          const int s = n % STAGES;
          ok = mbar_wait(&empty[s], ((n / STAGES) & 1) ^ 1, abort_word + 1, SITE_EMPTY, long_limit);
          if (!ok) break;
          uint8_t* st = smem + s * STAGE_BYTES;
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * STAGE_BYTES);
          const uint32_t bar = mapa(smem_u32(&full[s]), 0);
          tma_load_3d_pair(st, &tmA, bar, kb * 128, m0, 0);
          tma_load_3d_pair(st + ROW_TILE_BYTES, &tmW, bar, kb * 128, n0 + (int)rank * 128, 0);
          tma_load_3d_pair(st + 2 * ROW_TILE_BYTES, &tmAs, bar, 0, kb, m0 >> 7);
          tma_load_3d_pair(st + 2 * ROW_TILE_BYTES + C::S_BYTES, &tmWs, bar, 0, kb, n0 >> 7);
        }
      }
      // the leader's products signal this CTA's barriers: the last ones are waited for here
      for (uint32_t i = n > STAGES ? n - STAGES : 0; i < n && ok; i++) ok = mbar_wait(&empty[i % STAGES], (i / STAGES) & 1, abort_word + 1, SITE_EMPTY, long_limit);
      if (!ok) atomicCAS((uint32_t*)abort_word, 0u, SITE_EMPTY);
      // nothing may still be in flight into either CTA's shared memory when it exits, loads (the leader's barriers count both
      // CTAs') or the last tile's signal
      if (*abort_word != 0u) {
        if (!ok && rank == 0)
          for (uint32_t i = (n > STAGES ? n - STAGES : 0); i < n; i++) mbar_wait_slow(&full[i % STAGES], (i / STAGES) & 1, abort_word + 2, SITE_FULL, limit);
        mbar_wait_slow(acc_full, (uint32_t)((tiles - 1 - worker) / workers) & 1u, abort_word + 2, SITE_ACC_FULL, limit);
      }
    }
  } else if (warp == 1 && rank == 0) {
    const bool leader = elect_one();
    constexpr uint32_t HI = desc_hi(1024), ID = idesc(MX, 256, BN);
    const uint32_t smem16 = smem_u32(smem) >> 4;
    uint32_t n = 0;
    int it = 0;
    for (int t = worker; t < tiles; t += workers, it++) {
      if (it >= 1) {
        if (!__all_sync(0xffffffffu, mbar_wait(acc_empty, (it - 1) & 1, abort_word, SITE_ACC_EMPTY, limit))) break;      // the warp decides as one
        tc_fence_after();
      }
      int kb = 0;
      for (; kb < kblocks; kb++, n++) {
        const int s = n % STAGES;
        if (!__all_sync(0xffffffffu, mbar_wait(&full[s], (n / STAGES) & 1, abort_word, SITE_FULL, limit))) break;
        tc_fence_after();
        const uint32_t a = smem16 + s * (STAGE_BYTES >> 4), w = a + (ROW_TILE_BYTES >> 4), sa = w + (ROW_TILE_BYTES >> 4), sw = sa + (C::S_BYTES >> 4);
        const uint32_t ta = sf_base + s * C::SF_COLS, tw = ta + 4 * PIECES;
        if (leader) {
#pragma unroll
          for (int j = 0; j < PIECES; j++) {
            copy_scales<2>(ta + 4 * j, sa + j * 32);
            copy_scales<2>(tw + 8 * j, sw + j * 32);                                // columns 0-127 of the tile
            copy_scales<2>(tw + 8 * j + 4, sw + (C::S_BYTES >> 4) + j * 32);        // columns 128-255
          }
#pragma unroll
          for (int j = 0; j < 4; j++) {
            const int piece = MX ? j >> 1 : j;
            mma<MX, 2>(tmem_base, make_desc(a + j * 2, HI), make_desc(w + j * 2, HI), ID | idesc_sf(MX ? (j & 1) * 2 : 0), ta + 4 * piece, tw + 8 * piece, (kb > 0 || j > 0) ? 1u : 0u);
          }
          umma_commit2(mapa(smem_u32(&empty[s]), 0));
          umma_commit2(mapa(smem_u32(&empty[s]), 1));
        }
        __syncwarp();
      }
      if (kb < kblocks) break;               // a sum that lacks a part is never announced
      if (leader) {
        umma_commit2(mapa(smem_u32(acc_full), 0));
        umma_commit2(mapa(smem_u32(acc_full), 1));
      }
      __syncwarp();
    }
  } else if (warp >= 4) {
    // A thread takes one row and 128 columns into registers and hands the accumulator back before it does anything else
    // with them: the tensor cores go on while the stores are under way.
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const uint32_t src = tmem_base + ((uint32_t)(quarter * 32) << 16) + half * 128;
    const Early early(p);
    const float* vec = after_wait(p.vec);
    float alpha = MX ? 1.f : early.a * early.w;
    const bool normal = is_normal(alpha);
    int it = 0;
    bool arrived = false;
    for (int t = worker; t < tiles; t += workers, it++) {
      if (t != worker) tile_origin(t, m0, n0);
      if (!__all_sync(0xffffffffu, mbar_wait(acc_full, it & 1, abort_word, SITE_ACC_FULL, limit))) break;      // what follows takes whole warps
      tc_fence_after();
      if (!MX && !normal) alpha = scale_sums(src, 128, early.a, early.w);
      uint32_t v[128];
#pragma unroll
      for (int c = 0; c < 128; c += 32) tmem_ld32(src + c, v + c);
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      const bool last = t + workers >= tiles;
      if (last) {                  // nobody waits for the accumulator any more, and this warp has no more business with the other CTA
        cluster_arrive_relaxed();
        arrived = true;
      } else if (lane == 0) {
        mbar_arrive_cluster_relaxed(mapa(smem_u32(acc_empty), 0));
      }
      const int row0 = m0 + quarter * 32, col0 = n0 + half * 128;
      if (row0 >= p.M || col0 >= p.N || __any_sync(0xffffffffu, early.status != 0u)) continue;
      if (p.epi == KREA_CUDA_EPI_RESID_GATE) {
        pair_add(p, vec, v, row0, col0, alpha, out_smem + (warp - 4) * C::OUT_BYTES, lane);
      } else {
        // All pairs end their tiles at about the same time, and 64 KB from every SM at once hold up the loads of the next ones:
        // the warps take turns over the next tile's products (4608 x 15360 x 6144: 183 -> 177 us NV, 176 -> 170 us MX)
        if (!last) __nanosleep((uint32_t)((warp - 4) * kblocks * PACE_NS));
        // after a worker's last tile the stages are free: every box of a warp has a place of its own there
        pair_store(p, vec, tmC, v, row0, col0, alpha, last ? smem + (warp - 4) * 4 * C::OUT_BYTES : out_smem + (warp - 4) * C::OUT_BYTES, last, lane);
      }
    }
    if (lane == 0) tma_store_wait_read();      // the last box has left shared memory
    __syncwarp();
    if (!arrived) cluster_arrive_relaxed();
  }
  if (warp < 4) {
    __syncwarp();
    cluster_arrive_relaxed();
  }

  // nobody leaves or frees tensor memory while the peer may still read this CTA's shared memory, signal its barriers or
  // write its accumulator
  tc_fence_before();
  __syncwarp();
  __syncthreads();
  cluster_wait();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc2(tmem_base, C::TMEM_COLS);
  }
  if (threadIdx.x == 0 && p.status != nullptr) {
    const uint32_t a = *abort_word;
    if (a != 0u) atomicCAS(p.status, 0u, a | ((blockIdx.x & 0xFFFu) << 8));
  }
}

template <bool MX>
static cudaError_t launch_rows_variant(const CUtensorMap& tmA, const CUtensorMap& tmAs, const CUtensorMap& tmW, const CUtensorMap& tmWs, const Fp4GemmParams& p, int split, bool pdl,
                                       cudaStream_t stream) {
  using namespace fp4g;
  static ConfiguredOnce once;
  cudaError_t e = once.set(gemm_fp4_rows_sm100<MX>, 227 * 1024);
  if (e != cudaSuccess) return e;
  const dim3 grid((unsigned)((p.N + 127) / 128), (unsigned)((p.M + p.tn - 1) / p.tn), (unsigned)split);
  const size_t smem = (size_t)p.stages * rows_stage_bytes(MX, p.tn) + 256 + 1024;
  return launch_kernel(gemm_fp4_rows_sm100<MX>, grid, ROWS_THREADS, smem, stream, pdl, split, false, tmA, tmAs, tmW, tmWs, p);
}

template <bool MX>
static cudaError_t launch_pair_variant(const CUtensorMap& tmA, const CUtensorMap& tmAs, const CUtensorMap& tmW, const CUtensorMap& tmWs, const CUtensorMap& tmC, Fp4GemmParams p, int sms, bool pdl,
                                       cudaStream_t stream) {
  using namespace fp4g;
  static ConfiguredOnce once;
  cudaError_t e = once.set(gemm_fp4_pair_sm100<MX>, PairCfg<MX>::SMEM);
  if (e != cudaSuccess) return e;
  const int mt = (p.M + 255) / 256, tiles = mt * ((p.N + 255) / 256);
  int workers = sms / 2 < tiles ? sms / 2 : tiles;
  const int waves = (tiles + workers - 1) / workers;
  workers = (tiles + waves - 1) / waves;
  // row blocks per group: 32 MB of packed A at most, groups of equal size
  int64_t gmax = (32ll << 20) / ((int64_t)(p.K / 2 + 1) * 256);
  if (gmax < 1) gmax = 1;
  const int groups = (int)((mt + gmax - 1) / gmax);
  p.group_m = (mt + groups - 1) / groups;
  return launch_kernel(gemm_fp4_pair_sm100<MX>, dim3((unsigned)workers * 2), PAIR_THREADS, PairCfg<MX>::SMEM, stream, pdl, 2, true, tmA, tmAs, tmW, tmWs, tmC, p);
}

Fp4GemmPlan plan_gemm_fp4(int M, int N, int K, int mx, int sms, int force) {
  Fp4GemmPlan plan{};
  plan.split = 1;
  // rows of A a CTA of the few-rows kernel: all of them up to 128, in whole sixteens; above, tiles of 128 (a tile starts where its
  // scales do)
  const int shares = (M + 127) / 128;
  plan.tn = M < 128 ? (M + 15) & ~15 : 128;
  const int64_t tiles = (int64_t)((N + 127) / 128) * shares;
  const int kblocks = (K + fp4g::KB - 1) / fp4g::KB;
  // Pairs above 128 rows, unless so few tiles would leave them idle through a long K that the few-rows kernel can share.  us, NV,
  // few rows | pairs: 128 x 6144 x 6144 10.7 | 12.4, 256 x 6144 x 6144 14.2 | 12.7, 256 x 15360 x 6144 19.7 | 15.6; with tiles for
  // half of the SMs: 512 x 2048 x 2048 8.2 | 7.2, 256 x 2504 x 2500 8.9 | 9.5, 512 x 2048 x 6144 10.9 | 11.9, 160 x 1024 x 16384 11.6 | 23.8
  plan.pair = force == 2 || (force == 0 && M > 128 && !(tiles * 2 <= sms && kblocks >= 10));
  if (plan.pair) return plan;
  // How K is shared: clusters of up to four CTAs (eight where a few tiles are all there is).  One CTA an SM with a deep ring
  // moves the most while clusters find room side by side: pairs on all SMs, larger ones on five in six (48 clusters of three
  // on 148 SMs ran in two rounds).  Where that leaves a quarter of the SMs idle and a CTA has at most 64 rows to finish, two
  // CTAs an SM with short rings.  us, MX: 64 x 6144 x 6144 deep 2 x 48 CTAs 9.0, deep 3 x 48 13.9, short 4 x 48 8.8;
  // 64 x 2504 x 2500 deep 3 x 20 6.1, short 4 x 20 5.9; 96 x 6144 x 6144 deep 2 x 48 9.5; 1 x 15360 x 6144 deep 120 11.3, short
  // 240 11.5; 64 x 8192 x 2048 deep 1 x 64 7.0, 2 x 64 6.3; 1 x 1024 x 8192 short 4 x 8 5.7, 8 x 8 4.5.
  const int top = tiles * 16 <= sms ? 8 : 4;
  const auto most = [&](auto room) {
    int c = 1;
    while (c < top && tiles * (c + 1) <= room(c + 1) && kblocks > c) c++;
    return c;
  };
  plan.split = most([&](int c) { return c == 2 ? sms : sms * 5 / 6; });
  int ctas = tiles * plan.split > sms ? 2 : 1;      // a SM
  if (ctas == 1 && plan.tn <= 64 && tiles * plan.split * 4 < 3 * (int64_t)sms) {
    plan.split = most([&](int) { return sms * 4 / 3; });
    ctas = 2;
  }
  const int room = 228 * 1024 / ctas - 1024 - 256 - 1024;
  plan.stages = room / fp4g::rows_stage_bytes(mx != 0, plan.tn);
  if (plan.stages > fp4g::ROWS_MAX_STAGES) plan.stages = fp4g::ROWS_MAX_STAGES;
  while (fp4g::rows_tmem_cols(mx != 0, plan.tn, plan.stages) > 512 / ctas) plan.stages--;
  return plan;
}

cudaError_t launch_gemm_fp4(const Fp4GemmPlan& plan, const CUtensorMap& tmA, const CUtensorMap& tmAs, const CUtensorMap& tmW, const CUtensorMap& tmWs, const CUtensorMap& tmC, const Fp4GemmParams& p,
                            int sms, bool pdl, cudaStream_t stream) {
  if (p.M <= 0 || p.N <= 0 || p.K <= 0) return cudaSuccess;
  if (plan.pair) return p.mx ? launch_pair_variant<true>(tmA, tmAs, tmW, tmWs, tmC, p, sms, pdl, stream) : launch_pair_variant<false>(tmA, tmAs, tmW, tmWs, tmC, p, sms, pdl, stream);
  Fp4GemmParams q = p;
  q.tn = plan.tn;
  q.stages = plan.stages;
  return p.mx ? launch_rows_variant<true>(tmA, tmAs, tmW, tmWs, q, plan.split, pdl, stream) : launch_rows_variant<false>(tmA, tmAs, tmW, tmWs, q, plan.split, pdl, stream);
}

}  // namespace krea
