// Layout of 4-bit weights and what the kernels that multiply them share (w4.cu: up
// to 16 token rows, w4_sm100.cu: more).
//
// Weights [N, K] are laid out once for the kernels that stream them: int32
// q [ceil(N/16), ceil(K/128), 2, 32, 4] and fp16 scales
// [ceil(N/16), ceil(K/128) * 128 / group, 8, 2]. Tile (n, k) holds rows 16 n ..
// and columns 128 k ..; [h, l, j] of it is row 8 h + l / 4, and element e of
// its eight is column 16 (2 j + e / 4) + 4 (l % 4) + e % 4, in bits
// {0, 16, 4, 20, 8, 24, 12, 28}[e]. scales[n, g, r, h] belongs to row 8 h + r.
// Rows and columns past N and K are padding (code 8, scale 0).
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace aether {
namespace w4 {

struct Weight {
  const uint32_t* q;
  const __half* s;
  int N, K, kt, groups, gshift;  // kt: column tiles; groups: scales of a row; gshift: log2(group)
};

__device__ __forceinline__ float scale_at(const Weight& w, int n, int k) {
  return __half2float(w.s[(((int64_t)(n >> 4) * w.groups + (k >> w.gshift)) * 8 + (n & 7)) * 2 + ((n >> 3) & 1)]);
}
__device__ __forceinline__ int code_at(uint32_t word, int e) {
  return (int)((word >> (4 * (e >> 1) + 16 * (e & 1))) & 15u) - 8;
}

struct LinearParams {
  Weight w;
  const __nv_bfloat16* x;
  int64_t xs;
  const __nv_bfloat16* bias;
  const __nv_bfloat16* res;
  int64_t rs;
  __nv_bfloat16* y;
  int64_t ys;
  int M, n_out, swiglu;
  int outs, tiles, S, per;  // outputs of a CTA and how many such; parts of the columns and their column tiles
  int* status;
};

// A constant that stays in a register: written as an immediate, it is moved into one again for each use.
__device__ __forceinline__ uint32_t in_register(uint32_t c) {
  uint32_t r;
  asm volatile("mov.u32 %0, %1;" : "=r"(r) : "r"(c));
  return r;
}
struct Consts {
  uint32_t mask, bias, minus;  // 0x000f000f, 0x43004300 (128), 0xc308c308 (-136)
};
// bf16 pair of two weight codes (nibbles i and i + 4 of w), exact
template <int i>
__device__ __forceinline__ uint32_t codes2(uint32_t w, const Consts& k) {
  uint32_t x, r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(x) : "r"(w >> (4 * i)), "r"(k.mask), "r"(k.bias));  // (a & b) | c
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(k.minus));
  return r;
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, bool in) {  // zeros where not `in`
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}

// A CTA's share of a cluster's outputs, four rows to a thread: `sums`
// [part][token][kLd] in the shared memory of each of the S CTAs, in the order
// of the columns, then bias, SwiGLU (up rows `up` rows into their tiles, which
// start at kUpAt) and residual.
template <int KH, int kLd, int kUpAt>
__device__ __forceinline__ void finish(const LinearParams& p, const float* sums, int S, int rank, int n0, int up,
                                       int tid, int nthreads) {
  const uint32_t own = smem_u32(sums);
  auto sum_at = [&](int tok, int row) {  // four rows, all parts of all ranks
    float4 v[8], w = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int h = 0; h < KH; ++h) {
      const int at = (h * p.M + tok) * kLd + row;
      if (S == 1) {
        v[0] = *reinterpret_cast<const float4*>(sums + at);
        w.x += v[0].x, w.y += v[0].y, w.z += v[0].z, w.w += v[0].w;
        continue;
      }
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        v[c] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (c < S) v[c] = ld_cluster4(mapa_shared(own + at * 4, c));
      }
#pragma unroll
      for (int c = 0; c < 8; ++c) w.x += v[c].x, w.y += v[c].y, w.z += v[c].z, w.w += v[c].w;
    }
    return w;
  };
  // outputs and residuals as 8 bytes of four where their rows allow it
  const bool wide = p.ys % 4 == 0 && reinterpret_cast<uintptr_t>(p.y) % 8 == 0 &&
                    (p.res == nullptr || (p.rs % 4 == 0 && reinterpret_cast<uintptr_t>(p.res) % 8 == 0));
  const int per = p.outs / 4, quads = p.M * per, share = (quads + S - 1) / S;
  const int end = min(quads, (rank + 1) * share);
  int e = rank * share + tid, tok = e / per, q = e - tok * per;
  const int step_tok = nthreads / per, step_q = nthreads - step_tok * per;
#pragma unroll 2
  for (; e < end; e += nthreads, tok += step_tok, q += step_q) {
    if (q >= per) q -= per, ++tok;
    const int i = q * 4, n = n0 + i;
    if (n >= p.n_out) continue;
    const float4 v4 = sum_at(tok, i);
    float v[4] = {v4.x, v4.y, v4.z, v4.w};
    float u[4] = {0.f, 0.f, 0.f, 0.f};
    if (p.swiglu) {  // up rows start `up` rows into their tiles: from the two aligned quads around them
      const int o = up & 3;
      const float4 a = sum_at(tok, kUpAt + ((up + i) & ~3));
      float4 c = a;
      if (o) c = sum_at(tok, kUpAt + ((up + i) & ~3) + 4);
      u[0] = o == 0 ? a.x : o == 1 ? a.y : o == 2 ? a.z : a.w;
      u[1] = o == 0 ? a.y : o == 1 ? a.z : o == 2 ? a.w : c.x;
      u[2] = o == 0 ? a.z : o == 1 ? a.w : o == 2 ? c.x : c.y;
      u[3] = o == 0 ? a.w : o == 1 ? c.x : o == 2 ? c.y : c.z;
    }
    const bool whole = wide && n + 4 <= p.n_out;
    float r[4] = {0.f, 0.f, 0.f, 0.f};
    if (p.res && whole) {
      const uint2 w = *reinterpret_cast<const uint2*>(p.res + tok * p.rs + n);
      r[0] = bf16lo(w.x), r[1] = bf16hi(w.x), r[2] = bf16lo(w.y), r[3] = bf16hi(w.y);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (n + k >= p.n_out) break;
      if (p.bias) v[k] += __bfloat162float(p.bias[n + k]);
      if (p.swiglu) {
        if (p.bias) u[k] += __bfloat162float(p.bias[p.n_out + n + k]);
        v[k] = __fdividef(v[k], 1.f + __expf(-v[k])) * u[k];
      }
      if (p.res && !whole) r[k] = __bfloat162float(p.res[tok * p.rs + n + k]);
      v[k] += r[k];
      if (!whole) p.y[tok * p.ys + n + k] = __float2bfloat16(v[k]);
    }
    if (whole) *reinterpret_cast<uint2*>(p.y + tok * p.ys + n) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
  }
}

}  // namespace w4

// w4_sm100.cu
void linear_w4_tc(w4::LinearParams& p, cudaStream_t st);

}  // namespace aether
