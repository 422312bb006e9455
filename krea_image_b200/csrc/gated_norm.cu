// The end of one sublayer and the start of the next in one pass over the row:
//   r  = post ? y * rsqrt(mean(y^2) + eps) * post : y
//   x' = x_scale * x + gate * r
//   h  = x' * rsqrt(mean(x'^2) + eps) * mul + add,   stored as bf16, f32, or 4-bit values with block scales
// (the DiT block's gated residual, engine/kernels/gemm.metal:262-264, with the norm that follows it, norm.metal:28-55,
// and the post-sublayer norm of blocks that have one).  The 4-bit forms round h to bf16 first, so that they equal the
// quantisation of the bf16 form bit for bit.
//
// HBM-bound: x and y are read once, x' and h written once; a group of threads keeps its row in registers through both
// sums.  Sums of squares are fp32, 8 values a thread at a time, then a tree over the threads.
//
// What counts is how much is under way at once, and how few instructions a value takes.  CTAs stay for many rows, one row
// each at a time: a thread has HOLD pieces of 8 columns and asks for its pieces of the next row as soon as those of this one
// are in x', so that they are under way through the sum, the norm and the stores; the arithmetic is on packed pairs.
// HOLD = 1 with 40 registers up to 6144 columns, 2 up to 16384, 4 above (whose 64 registers do not hold all of the row: it spills).
// Fewer rows than two an SM, of 8192 columns at most, take HOLD = 1 with 64 registers and load the vectors a step before their use
// (AHEAD): there the time is one row's chain of accesses.
// Measured at 4608 x 6144: bf16 57 us (93 % of the copy bandwidth), MX 52 us (88 %), NV 58 us (80 %); f32 with a
// post-norm at 4748 x 2560 31-34 us (78-85 %); one row of 6144 3.4 us; 4608 x 20480 bf16 376 us (47 %), NV 425 us (36 %).  Measured slower: vectors kept in shared memory instead of
// L1 (f32 43.6 us), one row a CTA without the loop (NV 75.7 us), rows brought by bulk copies into a ring in shared memory
// (f32 35.0 us, NV 67 us: L1 is what the ring takes).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/krea_cuda.h"
#include "fp4.h"
#include "fp4_block.cuh"
#include "sm100_ptx.cuh"

namespace krea {

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// sum over the CTA; `part`: a float a warp, not written again before the CTA's next barrier
__device__ __forceinline__ float cta_sum(float v, float* part) {
  v = warp_sum(v);
  if (blockDim.x == 32) return v;
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  return warp_sum(lane < (int)(blockDim.x >> 5) ? part[lane] : 0.f);
}

// ---- 8 values as four packed pairs ----
struct F8 {
  uint64_t p[4];
};
__device__ __forceinline__ F8 splat(float v) {
  const uint64_t u = pack_f32x2(v, v);
  return {{u, u, u, u}};
}
__device__ __forceinline__ F8 mul8(const F8& a, const F8& b) {
  F8 r;
#pragma unroll
  for (int i = 0; i < 4; i++) r.p[i] = mul_f32x2(a.p[i], b.p[i]);
  return r;
}
__device__ __forceinline__ F8 fma8(const F8& a, const F8& b, const F8& c) {
  F8 r;
#pragma unroll
  for (int i = 0; i < 4; i++) r.p[i] = fma_f32x2(a.p[i], b.p[i], c.p[i]);
  return r;
}
__device__ __forceinline__ F8 add8(const F8& a, const F8& b) {
  F8 r;
#pragma unroll
  for (int i = 0; i < 4; i++) r.p[i] = add_f32x2(a.p[i], b.p[i]);
  return r;
}
__device__ __forceinline__ F8 from_bf16(uint4 u) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  F8 r;
#pragma unroll
  for (int i = 0; i < 4; i++) r.p[i] = pack_f32x2(bf16lo_to_f32(w[i]), bf16hi_to_f32(w[i]));
  return r;
}

// 8 floats in one access where every row starts on 32 bytes (V8), in two else.  One access a thread makes a warp's a
// whole kilobyte; two of 16 bytes, 32 apart, cost twice the passes through L1.  NC: by the read-only path, which is only for kernels
// that start when their predecessor has ended (4748 x 2560 f32 with post-norm 33.8 us, 34.5 without).
template <bool V8, bool NC>
__device__ __forceinline__ F8 load8(const float* s) {
  F8 r;
  if constexpr (V8 && NC) {
    asm volatile("ld.global.nc.v4.b64 {%0, %1, %2, %3}, [%4];" : "=l"(r.p[0]), "=l"(r.p[1]), "=l"(r.p[2]), "=l"(r.p[3]) : "l"(s));
  } else if constexpr (V8) {
    asm volatile("ld.global.v4.b64 {%0, %1, %2, %3}, [%4];" : "=l"(r.p[0]), "=l"(r.p[1]), "=l"(r.p[2]), "=l"(r.p[3]) : "l"(s));
  } else if constexpr (NC) {
    asm volatile("ld.global.nc.v2.b64 {%0, %1}, [%2];" : "=l"(r.p[0]), "=l"(r.p[1]) : "l"(s));
    asm volatile("ld.global.nc.v2.b64 {%0, %1}, [%2];" : "=l"(r.p[2]), "=l"(r.p[3]) : "l"(s + 4));
  } else {
    asm volatile("ld.global.v2.b64 {%0, %1}, [%2];" : "=l"(r.p[0]), "=l"(r.p[1]) : "l"(s));
    asm volatile("ld.global.v2.b64 {%0, %1}, [%2];" : "=l"(r.p[2]), "=l"(r.p[3]) : "l"(s + 4));
  }
  return r;
}
// rows that pass through once: not kept in L1, where the vectors of the modulation stay.  x may be the same memory as
// x_out (a thread reads a piece before it writes it), so no read-only path.
template <bool V8>
__device__ __forceinline__ F8 stream8(const float* s) {
  F8 r;
  if constexpr (V8) {
    asm volatile("ld.global.L1::no_allocate.v4.b64 {%0, %1, %2, %3}, [%4];" : "=l"(r.p[0]), "=l"(r.p[1]), "=l"(r.p[2]), "=l"(r.p[3]) : "l"(s) : "memory");
  } else {
    asm volatile("ld.global.L1::no_allocate.v2.b64 {%0, %1}, [%2];" : "=l"(r.p[0]), "=l"(r.p[1]) : "l"(s) : "memory");
    asm volatile("ld.global.L1::no_allocate.v2.b64 {%0, %1}, [%2];" : "=l"(r.p[2]), "=l"(r.p[3]) : "l"(s + 4) : "memory");
  }
  return r;
}
template <bool V8>
__device__ __forceinline__ void store8(float* d, const F8& v) {
  if constexpr (V8) {
    asm volatile("st.global.v4.b64 [%0], {%1, %2, %3, %4};" ::"l"(d), "l"(v.p[0]), "l"(v.p[1]), "l"(v.p[2]), "l"(v.p[3]) : "memory");
  } else {
    asm volatile("st.global.v2.b64 [%0], {%1, %2};" ::"l"(d), "l"(v.p[0]), "l"(v.p[1]) : "memory");
    asm volatile("st.global.v2.b64 [%0], {%1, %2};" ::"l"(d + 4), "l"(v.p[2]), "l"(v.p[3]) : "memory");
  }
}
__device__ __forceinline__ uint4 stream_bf16x8(const void* s) {
  uint4 u;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(s) : "memory");
  return u;
}

// The thread's pieces of one row, as they come from memory
template <int HOLD, bool Y32>
struct RowPieces {
  F8 x[HOLD];
  uint4 yb[Y32 ? 1 : HOLD];
  F8 yf[Y32 ? HOLD : 1];
  template <bool V8>
  __device__ __forceinline__ void fetch(const GatedNormParams& p, int row) {
#pragma unroll
    for (int k = 0; k < HOLD; k++) {
      const int c = (threadIdx.x + k * blockDim.x) * 8;
      const bool in = c < p.width;
      if constexpr (Y32) {
        yf[k] = splat(0.f);
        if (in) yf[k] = stream8<V8>((const float*)p.y + (int64_t)row * p.ld_y + c);
      } else {
        yb[k] = make_uint4(0u, 0u, 0u, 0u);
        if (in && p.y) yb[k] = stream_bf16x8((const __nv_bfloat16*)p.y + (int64_t)row * p.ld_y + c);
      }
      x[k] = splat(0.f);
      if (in) x[k] = stream8<V8>(p.x + (int64_t)row * p.ld_x + c);
    }
  }
};

// A CTA takes rows blockIdx.x, blockIdx.x + gridDim.x, ...  V8: every row and vector starts on 32 bytes.
template <int HOLD, int REGS, bool AHEAD, bool V8, bool Y32, int OUT>
__global__ void __maxnreg__(REGS) gated_norm_kernel(const GatedNormParams p) {
  constexpr bool FP4 = OUT == KREA_CUDA_OUT_FP4_MX || OUT == KREA_CUDA_OUT_FP4_NV, MX = OUT == KREA_CUDA_OUT_FP4_MX;
  __shared__ float part[2][2][32];        // [row parity][which sum][warp]
  __shared__ NvTable nv;
  griddep_wait();
  const int t = threadIdx.x;
  unsigned row = blockIdx.x;                 // unsigned: row + gridDim.x passes 2^31 at the end of the longest inputs
  RowPieces<HOLD, Y32> in;
  in.template fetch<V8>(p, (int)min(row, (unsigned)p.rows - 1u));      // not under a condition: the compiler would move it into the loop, to where it is used
  if constexpr (OUT == KREA_CUDA_OUT_FP4_NV) {       // read after the sums' barriers; a CTA of one warp has none
    for (int c = t; c < 128; c += blockDim.x) nv_table_fill(nv, p.h_ts ? ld_global_f1(p.h_ts) : 1.f, c);
    if (blockDim.x == 32) __syncwarp();
  }
  const float inv_w = 1.0f / (float)p.width;
  const int chunks = (p.width + 255) / 256;
  const F8 xs = splat(p.x_scale);
  // piece k of one of the vectors, `none` where there is none
  const auto vec = [&](const float* base, int k, float none) {
    const int c = (t + k * (int)blockDim.x) * 8;
    F8 r = splat(none);
    if (base && c < p.width) r = load8<V8, !AHEAD>(base + c);
    return r;
  };
  const auto total = [](const F8& s) {
    float a, b, r = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      unpack_f32x2(s.p[i], a, b);
      r += a + b;
    }
    return r;
  };
  int64_t mod = 0;                 // where the row's vectors start
  unsigned until = p.mod_rows > 0 ? 0u : 0xFFFFFFFFu;      // first row that has others
  for (int it = 0; row < (unsigned)p.rows; it ^= 1) {
    if (row >= until) {
      const unsigned sample = row / (unsigned)p.mod_rows;
      mod = (int64_t)sample * p.mod_ld;
      until = (sample + 1u) * (unsigned)p.mod_rows;
    }
    const float *gate = p.gate ? p.gate + mod : nullptr, *mul = p.h ? p.mul + mod : nullptr, *add = p.add ? p.add + mod : nullptr;
    F8 v[HOLD], w[AHEAD ? HOLD : 1], w2[AHEAD ? HOLD : 1];
    if constexpr (AHEAD) {
#pragma unroll
      for (int k = 0; k < HOLD; k++) {
        w[k] = vec(gate, k, 1.f);
        if (p.post) w2[k] = vec(p.post, k, 1.f);
      }
    }
#pragma unroll
    for (int k = 0; k < HOLD; k++) {
      if constexpr (Y32) v[k] = in.yf[k];
      else v[k] = from_bf16(in.yb[k]);
    }
    if (p.post) {
      F8 ss = splat(0.f);
#pragma unroll
      for (int k = 0; k < HOLD; k++) ss = fma8(v[k], v[k], ss);
      const F8 rr = splat(rsqrtf(cta_sum(total(ss), part[it][0]) * inv_w + p.eps));
#pragma unroll
      for (int k = 0; k < HOLD; k++) v[k] = mul8(mul8(v[k], rr), AHEAD ? w2[k] : vec(p.post, k, 1.f));
    }
    F8 ss = splat(0.f);
#pragma unroll
    for (int k = 0; k < HOLD; k++) {
      const int c = (t + k * blockDim.x) * 8;
      if (p.gate) v[k] = mul8(v[k], AHEAD ? w[k] : vec(gate, k, 1.f));
      v[k] = add8(mul8(xs, in.x[k]), v[k]);          // each product rounded by itself, as the formula is written
      if (c < p.width && p.x_out) store8<V8>(p.x_out + (int64_t)row * p.ld_xo + c, v[k]);
      ss = fma8(v[k], v[k], ss);
    }
    const int now = (int)row;
    row += gridDim.x;
    if (row < (unsigned)p.rows) in.template fetch<V8>(p, (int)row);
    else griddep_launch();       // not before the last row: a successor that waits on the SM would take L1 away
    if (!p.h) continue;
    if constexpr (AHEAD) {
#pragma unroll
      for (int k = 0; k < HOLD; k++) w[k] = vec(mul, k, 0.f);
    }
    const F8 rr = splat(rsqrtf(cta_sum(total(ss), part[it][1]) * inv_w + p.eps));
#pragma unroll
    for (int k = 0; k < HOLD; k++) {
      const int c = (t + k * blockDim.x) * 8;
      if (!FP4 && c >= p.width) continue;
      if (FP4 && (int)(k * blockDim.x) * 8 >= chunks * 256) continue;     // the same for every thread: whole warps meet the exchanges below
      F8 f = mul8(mul8(v[k], rr), AHEAD ? w[k] : vec(mul, k, 0.f));
      if (p.add) f = add8(f, vec(add, k, 0.f));
      if constexpr (OUT == KREA_CUDA_OUT_F32) {
        store8<V8>((float*)p.h + (int64_t)now * p.ld_h + c, f);
      } else {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          float a, b;
          unpack_f32x2(f.p[i], a, b);
          u[i] = pack_bf16x2(a, b);
        }
        if constexpr (!FP4) {
          *(uint4*)((__nv_bfloat16*)p.h + (int64_t)now * p.ld_h + c) = make_uint4(u[0], u[1], u[2], u[3]);
        } else {
          uint32_t amax = amax_bits<4>(u);                       // a block is two (NV) or four (MX) neighbouring threads
          amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
          if (MX) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
          uint32_t code, q;
          if constexpr (MX) {
            code = mx_scale_code(amax);
            q = mx_encode8(u, code);
          } else {
            code = nv_scale_code(amax, nv);
            nv_encode<4>(u, code, nv, &q);
          }
          if (c < ((p.width + 31) & ~31)) *(uint32_t*)((uint8_t*)p.h + (int64_t)now * p.ld_h + (c >> 1)) = q;
          // Blocks past the width get 0, whatever the row's factor made of their zeros (NaN, where it is not finite).  In a block that
          // the width ends in, such a factor leaves no value finite before the width either.
          if (c >= p.width) code = 0u;
          if ((t & (MX ? 3 : 1)) == 0 && c < chunks * 256) p.h_scales[scale_offset<MX>(now, MX ? c >> 5 : c >> 4, chunks)] = (uint8_t)code;
        }
      }
    }
  }
  if constexpr (FP4) {
    // zero scales for the rows that fill up the last tile of 128
    const int64_t words = p.h && p.rows % 128 ? (int64_t)chunks * (MX ? 2 : 4) * 128 : 0;
    uint32_t* tile = (uint32_t*)p.h_scales + (int64_t)(p.rows / 128) * words;
    for (int64_t w = (int64_t)blockIdx.x * blockDim.x + t; w < words; w += (int64_t)gridDim.x * blockDim.x)
      if ((int)(w & 3) * 32 + (int)((w & 127) >> 2) >= p.rows % 128) tile[w] = 0u;
  }
}

template <int HOLD, int REGS, bool AHEAD, bool V8, bool Y32>
static cudaError_t launch_rows_as(const GatedNormParams& p, int block, int sms, bool pdl, cudaStream_t stream) {
  auto* k = gated_norm_kernel<HOLD, REGS, AHEAD, V8, Y32, KREA_CUDA_OUT_BF16>;
  if (p.out == KREA_CUDA_OUT_F32) k = gated_norm_kernel<HOLD, REGS, AHEAD, V8, Y32, KREA_CUDA_OUT_F32>;
  if (p.out == KREA_CUDA_OUT_FP4_MX) k = gated_norm_kernel<HOLD, REGS, AHEAD, V8, Y32, KREA_CUDA_OUT_FP4_MX>;
  if (p.out == KREA_CUDA_OUT_FP4_NV) k = gated_norm_kernel<HOLD, REGS, AHEAD, V8, Y32, KREA_CUDA_OUT_FP4_NV>;
  // CTAs an SM holds: each of its four parts has 512 registers for a lane
  int resident = 4 * (512 / REGS) / (block / 32);
  resident = resident < 1 ? 1 : resident > 32 ? 32 : resident;
  // with a dozen rows or more for each of them, two rounds of CTAs: the second evens out the ends (4608 x 6144 bf16: 57 us
  // against 63); with fewer, setting up twice costs more than that (4748 x 2560: 37 us against 35)
  const int64_t slots = (int64_t)sms * resident, want = p.rows >= 12 * slots ? 2 * slots : slots;
  const int grid = (int)(p.rows < want ? p.rows : want);
  // Programmatic only with few rows (AHEAD).  CTAs that start on an SM as the kernel before leaves it keep that kernel's split of L1
  // and shared memory, and after a GEMM the vectors have no L1 to stay in (norm + 4-bit product at 4608 x 6144: 134 us against 116)
  return launch_kernel(k, dim3((unsigned)grid), block, 0, stream, AHEAD && pdl, 1, false, p);
}
template <int HOLD, int REGS, bool AHEAD, bool V8>
static cudaError_t launch_rows(const GatedNormParams& p, int block, int sms, bool pdl, cudaStream_t stream) {
  return p.y && p.y_f32 ? launch_rows_as<HOLD, REGS, AHEAD, V8, true>(p, block, sms, pdl, stream) : launch_rows_as<HOLD, REGS, AHEAD, V8, false>(p, block, sms, pdl, stream);
}

cudaError_t launch_gated_norm(const GatedNormParams& p, int sms, bool pdl, cudaStream_t stream) {
  if (p.rows <= 0 || p.width <= 0) return cudaSuccess;
  const int padded = (p.width + 255) & ~255;           // the 4-bit forms also write the scales of the padding
  const auto threads = [&](int hold) { return (padded / 8 / hold + 31) & ~31; };
  const uintptr_t rows32 = (uintptr_t)p.x | (uintptr_t)p.x_out | (uintptr_t)(p.ld_x * 4) | (uintptr_t)(p.x_out ? p.ld_xo * 4 : 0) |
                           (p.y_f32 ? (uintptr_t)p.y | (uintptr_t)(p.ld_y * 4) : 0) | (p.out == KREA_CUDA_OUT_F32 ? (uintptr_t)p.h | (uintptr_t)(p.ld_h * 4) : 0);
  const uintptr_t vec32 = (uintptr_t)p.post | (uintptr_t)p.gate | (uintptr_t)p.mul | (uintptr_t)p.add | (uintptr_t)(p.mod_rows > 0 ? p.mod_ld * 4 : 0);
  const bool v8 = ((rows32 | vec32) & 31u) == 0;
  if (p.rows < 2 * sms && padded <= 8192) return launch_rows<1, 64, true, false>(p, threads(1), sms, pdl, stream);
  // Many thin threads hide the chain of a row's sums better than half as many with two pieces each (2560 columns, f32, post-norm:
  // 34 us against 37; 4608 x 6144 NV 55.4 against 59.5, MX 51 against 55.5), as long as two rows fit side by side:
  // at 8192 columns, where one does, NV takes 63 us against 56
  if (padded <= 6144) return v8 ? launch_rows<1, 40, false, true>(p, threads(1), sms, pdl, stream) : launch_rows<1, 40, false, false>(p, threads(1), sms, pdl, stream);
  if (padded <= 16384) return v8 ? launch_rows<2, 64, false, true>(p, threads(2), sms, pdl, stream) : launch_rows<2, 64, false, false>(p, threads(2), sms, pdl, stream);
  return launch_rows<4, 64, false, false>(p, threads(4), sms, pdl, stream);
}

}  // namespace krea
