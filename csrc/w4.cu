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
  int M, n_out, swiglu;
};

// sum over k of row n's weights with token m, on one warp: a lane takes one
// 8-element word of the row, two column tiles at a time.
__device__ __forceinline__ float row_dot(const LinearParams& p, int n, int m, int lane) {
  float acc = 0.f;
  for (int kt = lane >> 4; kt < p.w.kt; kt += 2) {
    const int t = (lane >> 2) & 3, j = lane & 3;
    const uint32_t word =
        p.w.q[((((int64_t)(n >> 4) * p.w.kt + kt) * 2 + ((n >> 3) & 1)) * 32 + (n & 7) * 4 + t) * 4 + j];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int k = kt * 128 + 16 * (2 * j + (e >> 2)) + 4 * t + (e & 3);
      if (k < p.w.K) acc += (code_at(word, e) * scale_at(p.w, n, k)) * __bfloat162float(p.x[m * p.xs + k]);
    }
  }
  return warp_sum(acc);
}

__global__ void __launch_bounds__(128) linear_kernel(LinearParams p) {
  const int lane = threadIdx.x & 31;
  const int n = blockIdx.x * 4 + (threadIdx.x >> 5), m = blockIdx.y;
  if (n >= p.n_out) return;
  float v = row_dot(p, n, m, lane);
  if (p.bias) v += __bfloat162float(p.bias[n]);
  if (p.swiglu) {
    float u = row_dot(p, p.n_out + n, m, lane);
    if (p.bias) u += __bfloat162float(p.bias[p.n_out + n]);
    v = v / (1.f + __expf(-v)) * u;
  }
  if (p.res) v += __bfloat162float(p.res[m * p.rs + n]);
  if (lane == 0) p.y[m * p.ys + n] = __float2bfloat16(v);
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
  linear_kernel<<<dim3((unsigned)((n_out + 3) / 4), (unsigned)M), 128, 0, at::cuda::getCurrentCUDAStream()>>>(p);
  AETHER_CUDA_CHECK(cudaGetLastError());
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
