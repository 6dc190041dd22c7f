// Products of a few token rows with 4-bit weights and group scales.
//
//   y[m, n] = sum_g s[n, g] * sum_{k in group g} (c[n, k] - 8) * x[m, k]
//
// Weights [N, K] are laid out once for the kernel that streams them: int32
// q [ceil(N/16), ceil(K/128), 2, 32, 4] and fp16 scales
// [ceil(N/16), ceil(K/128) * 128 / group, 8, 2]. Tile (n, k) holds rows 16 n ..
// and columns 128 k ..; [h, l, j] of it is row 8 h + l / 4, and element e of
// its eight is column 16 (2 j + e / 4) + 4 (l % 4) + e % 4, in bits
// {0, 16, 4, 20, 8, 24, 12, 28}[e]. scales[n, g, r, h] belongs to row 8 h + r.
// Rows and columns past N and K are padding (code 8, scale 0).
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "host_utils.h"

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
  int M, n_out, swiglu, x_aligned, stage;  // stage: column tiles of x in shared memory at a time
};

// A CTA of eight warps owns 128 rows (SwiGLU: 64 gate rows and the 64 up rows
// they meet) and, in a cluster of S, the S-th part of the columns. A warp
// streams 16 rows: one column tile is two 16-byte loads a thread, kept kAhead
// tiles ahead in registers, and its nibbles become the A operand of m16n8k16
// steps without a shuffle -- (w >> 4 i) & 0xf | 0x4300 is bf16 128 + code, minus
// 136 the exact weight code. The token rows (B operand, eight to a step) sit in
// shared memory, whose rows are 32 bytes apart modulo 128, so that a quad's
// 8-byte reads of four rows meet no bank twice. A group's sum of exact
// products stays in fp32 and is scaled once. The CTAs of a cluster add their
// sums over distributed shared memory, each its share of the outputs in the
// order of the columns, so no workspace is needed and the result is the same
// on every run.
constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = kWarps * 16;
constexpr int kSumLd = kRows + 4;  // floats of one token's sums
constexpr int kStageBytes = 72 * 1024;

__device__ __forceinline__ uint4 ld_stream16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
// bf16 pair of two weight codes (nibbles i and i + 4 of w), exact
template <int i>
__device__ __forceinline__ uint32_t codes2(uint32_t w) {
  uint32_t x, r;
  asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;" : "=r"(x) : "r"(w >> (4 * i)));  // (a & b) | c
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(0x43084308u));
  return r;
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}

// MT: tiles of eight token rows; GS: k16 steps of a scale group (2, 4 or 8)
template <int MT, int GS>
__global__ void __launch_bounds__(kThreads, MT <= 2 ? 2 : 1) linear_kernel(LinearParams p) {
  constexpr int kAhead = MT <= 2 ? 4 : 2;
  extern __shared__ __align__(16) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, t = lane & 3;
  const int S = (int)cluster_size(), rank = (int)cluster_ctarank();
  const int tile = blockIdx.x / S;
  const int outs = p.swiglu ? kRows / 2 : kRows;  // outputs of this CTA
  const int n0 = tile * outs;
  const int per = (p.w.kt + S - 1) / S;
  const int kt0 = rank * per, n_kt = max(0, min(p.w.kt, kt0 + per) - kt0);

  // this lane's two weight rows (past the last row: the last row again, its sums are dropped)
  const int warp_row = p.swiglu ? (warp < kWarps / 2 ? n0 + warp * 16 : p.n_out + n0 + (warp - kWarps / 2) * 16) : n0 + warp * 16;
  const int ra = min(warp_row + r, p.w.N - 1), rb = min(warp_row + r + 8, p.w.N - 1);
  auto row_q = [&](int n) {
    return p.w.q + ((((int64_t)(n >> 4) * p.w.kt + kt0) * 2 + ((n >> 3) & 1)) * 32 + (n & 7) * 4 + t) * 4;
  };
  constexpr int kGroups = 8 / GS;  // of a column tile
  auto row_s = [&](int n) {
    return p.w.s + (((int64_t)(n >> 4) * p.w.groups + (int64_t)kt0 * kGroups) * 8 + (n & 7)) * 2 + ((n >> 3) & 1);
  };
  const uint32_t *qa = row_q(ra), *qb = row_q(rb);
  const __half *sa = row_s(ra), *sb = row_s(rb);

  uint4 ba[kAhead], bb[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; ++u)
    if (u < n_kt) {
      ba[u] = ld_stream16(qa + u * 256);
      bb[u] = ld_stream16(qb + u * 256);
    }
  float acc[MT][4];
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[m][0] = acc[m][1] = acc[m][2] = acc[m][3] = 0.f;

  // column tiles staged at a time; one row of them is ld bytes
  const int stage = min(per, p.stage);
  const uint32_t ld = (uint32_t)stage * 256 + 32;
  const uint32_t xb = smem_u32(smem) + t * 8;
  uint32_t xrow[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) xrow[m] = xb + (uint32_t)min(m * 8 + r, p.M - 1) * ld;

  int staged = 0;  // tiles before the ones in shared memory
  for (int i0 = 0; i0 < n_kt; i0 += kAhead) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + u;
      if (i < n_kt) {
        if (i % stage == 0) {
          if (i > 0) __syncthreads();
          staged = i;
          const int cols = min(stage, n_kt - i) * 128, k0 = (kt0 + i) * 128;
          const int units = cols / 8;
          for (int e = tid; e < p.M * units; e += kThreads) {
            const int m = e / units, c = e % units * 8;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (k0 + c < p.w.K) {
              const __nv_bfloat16* src = p.x + m * p.xs + k0 + c;
              if (p.x_aligned) {
                v = __ldg(reinterpret_cast<const uint4*>(src));
              } else {
                const uint16_t* h = reinterpret_cast<const uint16_t*>(src);
                v.x = h[0] | (uint32_t)h[1] << 16;
                v.y = h[2] | (uint32_t)h[3] << 16;
                v.z = h[4] | (uint32_t)h[5] << 16;
                v.w = h[6] | (uint32_t)h[7] << 16;
              }
            }
            *reinterpret_cast<uint4*>(smem + (uint32_t)m * ld + c * 2) = v;
          }
          __syncthreads();
        }
        const uint32_t wa[4] = {ba[u].x, ba[u].y, ba[u].z, ba[u].w}, wb[4] = {bb[u].x, bb[u].y, bb[u].z, bb[u].w};
        if (i + kAhead < n_kt) {
          ba[u] = ld_stream16(qa + (int64_t)(i + kAhead) * 256);
          bb[u] = ld_stream16(qb + (int64_t)(i + kAhead) * 256);
        }
        float fa[kGroups], fb[kGroups];
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          fa[g] = __half2float(sa[(int64_t)(i * kGroups + g) * 16]);
          fb[g] = __half2float(sb[(int64_t)(i * kGroups + g) * 16]);
        }
        const uint32_t xoff = (uint32_t)(i - staged) * 256;
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          float c[MT][4];
#pragma unroll
          for (int m = 0; m < MT; ++m) c[m][0] = c[m][1] = c[m][2] = c[m][3] = 0.f;
#pragma unroll
          for (int s = g * GS; s < (g + 1) * GS; ++s) {
            const uint32_t a[4] = {s & 1 ? codes2<2>(wa[s >> 1]) : codes2<0>(wa[s >> 1]),
                                   s & 1 ? codes2<2>(wb[s >> 1]) : codes2<0>(wb[s >> 1]),
                                   s & 1 ? codes2<3>(wa[s >> 1]) : codes2<1>(wa[s >> 1]),
                                   s & 1 ? codes2<3>(wb[s >> 1]) : codes2<1>(wb[s >> 1])};
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              uint32_t b0, b1;
              asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(b0), "=r"(b1) : "r"(xrow[m] + xoff + s * 32));
              mma_bf16(c[m], a, b0, b1);
            }
          }
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            acc[m][0] += fa[g] * c[m][0];
            acc[m][1] += fa[g] * c[m][1];
            acc[m][2] += fb[g] * c[m][2];
            acc[m][3] += fb[g] * c[m][3];
          }
        }
      }
    }
  }
  // sums [token][row] in shared memory, then this CTA's share of the outputs
  __syncthreads();
  float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int tok = m * 8 + 2 * t + (e & 1);
      if (tok < p.M) sums[tok * kSumLd + warp * 16 + r + 8 * (e >> 1)] = acc[m][e];
    }
  if (S > 1) cluster_sync(); else __syncthreads();
  const uint32_t own = smem_u32(smem);
  auto sum_at = [&](int tok, int row) {
    if (S == 1) return sums[tok * kSumLd + row];
    float v = 0.f;
    for (int c = 0; c < S; ++c) v += ld_cluster(mapa_shared(own + (tok * kSumLd + row) * 4, c));
    return v;
  };
  const int share = (p.M * outs + S - 1) / S;
  for (int e = rank * share + tid; e < min(p.M * outs, (rank + 1) * share); e += kThreads) {
    const int tok = e / outs, i = e % outs, n = n0 + i;
    if (n >= p.n_out) continue;
    float v = sum_at(tok, i);
    if (p.bias) v += __bfloat162float(p.bias[n]);
    if (p.swiglu) {
      float u = sum_at(tok, kRows / 2 + i);
      if (p.bias) u += __bfloat162float(p.bias[p.n_out + n]);
      v = v / (1.f + __expf(-v)) * u;
    }
    if (p.res) v += __bfloat162float(p.res[tok * p.rs + n]);
    p.y[tok * p.ys + n] = __float2bfloat16(v);
  }
  if (S > 1) cluster_sync();  // every CTA's sums are read before its shared memory goes
}

template <int MT, int GS>
static void launch_linear(LinearParams& p, cudaStream_t st) {
  const int sms = num_sms(current_device());
  const int outs = p.swiglu ? kRows / 2 : kRows;
  const int tiles = (p.n_out + outs - 1) / outs;
  // columns are split until two CTAs an SM have work, while each keeps two column tiles
  int S = 1;
  while (S < 8 && tiles * S < 2 * sms && p.w.kt >= 4 * S) S *= 2;
  const int per = (p.w.kt + S - 1) / S;
  p.stage = std::max(1, std::min(per, (kStageBytes / p.M - 32) / 256));
  const int smem = std::max(p.M * (p.stage * 256 + 32), p.M * kSumLd * 4);
  static bool set[64] = {};
  const int dev = current_device();
  if (!set[dev]) {
    AETHER_CUDA_CHECK(cudaFuncSetAttribute(linear_kernel<MT, GS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kStageBytes));
    set[dev] = true;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(tiles * S));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim = {(unsigned)S, 1, 1};
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  AETHER_CUDA_CHECK(cudaLaunchKernelEx(&cfg, linear_kernel<MT, GS>, p));
}
template <int MT>
static void launch_group(LinearParams& p, cudaStream_t st) {
  if (p.w.gshift == 7)
    launch_linear<MT, 8>(p, st);
  else if (p.w.gshift == 6)
    launch_linear<MT, 4>(p, st);
  else
    launch_linear<MT, 2>(p, st);
}

// out [N, K] bf16 = code * scale, for products of more rows than a decode
// batch: one thread a word of eight elements.
__global__ void __launch_bounds__(256) dequant_kernel(Weight w, int64_t words, __nv_bfloat16* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= words) return;
  const int j = (int)(i & 3), l = (int)(i >> 2) & 31, h = (int)(i >> 7) & 1;
  const int64_t tile = i >> 8;
  const int kt = (int)(tile % w.kt);
  const int n = (int)(tile / w.kt) * 16 + 8 * h + (l >> 2);
  if (n >= w.N) return;
  const uint32_t word = w.q[i];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int k = kt * 128 + 16 * (2 * j + s) + 4 * (l & 3);
    if (k >= w.K) return;  // K is a multiple of 32: the four columns are in or out together
    const float f = scale_at(w, n, k);
    uint2 v;
    v.x = pack_bf16(code_at(word, 4 * s) * f, code_at(word, 4 * s + 1) * f);
    v.y = pack_bf16(code_at(word, 4 * s + 2) * f, code_at(word, 4 * s + 3) * f);
    *reinterpret_cast<uint2*>(out + (int64_t)n * w.K + k) = v;
  }
}

static Weight make_weight(const at::Tensor& q, const at::Tensor& s, int64_t N, int64_t K, int64_t group,
                          const char* what) {
  TORCH_CHECK(group == 32 || group == 64 || group == 128, what, ": groups of 32, 64 or 128");
  TORCH_CHECK(N >= 1 && N < (int64_t(1) << 30) && K >= group && K < (int64_t(1) << 30) && K % group == 0, what,
              ": K is a multiple of the group");
  const int64_t nt = (N + 15) / 16, kt = (K + 127) / 128;
  TORCH_CHECK(q.is_cuda() && q.scalar_type() == at::kInt && q.is_contiguous() && q.numel() == nt * kt * 256 &&
                  reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0,
              what, ": q is contiguous CUDA int32 [ceil(N/16), ceil(K/128), 2, 32, 4]");
  TORCH_CHECK(s.device() == q.device() && s.scalar_type() == at::kHalf && s.is_contiguous() &&
                  s.numel() == nt * (kt * 128 / group) * 16 && reinterpret_cast<uintptr_t>(s.data_ptr()) % 4 == 0,
              what, ": scales are contiguous float16 [ceil(N/16), ceil(K/128) * 128 / group, 8, 2] beside q");
  Weight w{};
  w.q = reinterpret_cast<const uint32_t*>(q.data_ptr<int>());
  w.s = reinterpret_cast<const __half*>(s.data_ptr());
  w.N = (int)N;
  w.K = (int)K;
  w.kt = (int)kt;
  w.groups = (int)(kt * 128 / group);
  w.gshift = group == 32 ? 5 : group == 64 ? 6 : 7;
  return w;
}

}  // namespace w4

void linear_w4(at::Tensor x, at::Tensor q, at::Tensor s, int64_t N, int64_t K, int64_t group,
               std::optional<at::Tensor> bias, std::optional<at::Tensor> residual, bool swiglu, at::Tensor y) {
  using namespace w4;
  LinearParams p{};
  p.w = make_weight(q, s, N, K, group, "linear_w4");
  const int64_t M = x.size(0), n_out = swiglu ? N / 2 : N;
  TORCH_CHECK(!swiglu || N % 2 == 0, "linear_w4: SwiGLU takes an even number of rows (gate, then up)");
  TORCH_CHECK(x.device() == q.device() && x.scalar_type() == at::kBFloat16 && x.dim() == 2 && x.size(1) == K &&
                  x.stride(1) == 1,
              "linear_w4: x is bf16 [M, K] with unit inner stride, beside the weights");
  TORCH_CHECK(y.device() == q.device() && y.scalar_type() == at::kBFloat16 && y.dim() == 2 && y.size(0) == M &&
                  y.size(1) == n_out && (n_out == 1 || y.stride(1) == 1),
              "linear_w4: out is bf16 [M, N] (SwiGLU: [M, N / 2]) with unit inner stride, beside the weights");
  TORCH_CHECK(M <= 64, "linear_w4: at most 64 rows");
  if (bias && bias->defined()) {
    TORCH_CHECK(bias->device() == q.device() && bias->scalar_type() == at::kBFloat16 && bias->is_contiguous() &&
                    bias->numel() == N,
                "linear_w4: bias is contiguous bf16 [N]");
    p.bias = reinterpret_cast<const __nv_bfloat16*>(bias->data_ptr());
  }
  if (residual && residual->defined()) {
    TORCH_CHECK(residual->device() == q.device() && residual->scalar_type() == at::kBFloat16 &&
                    residual->sizes() == y.sizes() && (n_out == 1 || residual->stride(1) == 1),
                "linear_w4: residual is bf16 in the shape of out, unit inner stride");
    p.res = reinterpret_cast<const __nv_bfloat16*>(residual->data_ptr());
    p.rs = residual->stride(0);
  }
  if (M == 0) return;
  c10::cuda::CUDAGuard g(q.device());
  p.x = reinterpret_cast<const __nv_bfloat16*>(x.data_ptr());
  p.xs = x.stride(0);
  p.y = reinterpret_cast<__nv_bfloat16*>(y.data_ptr());
  p.ys = y.stride(0);
  p.M = (int)M;
  p.n_out = (int)n_out;
  p.swiglu = swiglu;
  p.x_aligned = reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && p.xs % 8 == 0;
  auto st = at::cuda::getCurrentCUDAStream();
  if (M <= 8)
    launch_group<1>(p, st);
  else if (M <= 16)
    launch_group<2>(p, st);
  else if (M <= 32)
    launch_group<4>(p, st);
  else
    launch_group<8>(p, st);
}

void dequant_w4(at::Tensor q, at::Tensor s, int64_t N, int64_t K, int64_t group, at::Tensor out) {
  using namespace w4;
  const Weight w = make_weight(q, s, N, K, group, "dequant_w4");
  TORCH_CHECK(out.device() == q.device() && out.scalar_type() == at::kBFloat16 && out.is_contiguous() &&
                  out.numel() == N * K && reinterpret_cast<uintptr_t>(out.data_ptr()) % 8 == 0,
              "dequant_w4: out is contiguous bf16 [N, K] beside the weights");
  c10::cuda::CUDAGuard g(q.device());
  const int64_t words = q.numel();
  dequant_kernel<<<(unsigned)((words + 255) / 256), 256, 0, at::cuda::getCurrentCUDAStream()>>>(
      w, words, reinterpret_cast<__nv_bfloat16*>(out.data_ptr()));
  AETHER_CUDA_CHECK(cudaGetLastError());
}

}  // namespace aether
