// Products of a few token rows with 4-bit weights and group scales.
//
//   y[m, n] = sum_g s[n, g] * sum_{k in group g} (c[n, k] - 8) * x[m, k]
//
// (layout in w4.cuh)
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "common.cuh"
#include "host_utils.h"
#include "w4.cuh"

namespace aether {
namespace w4 {

// A CTA's eight multiplying warps own 128 / KH rows, a tile of 16 each (SwiGLU:
// gate tiles and the up tiles they meet), and, in a cluster of S, the S-th part
// of the columns, in KH parts that warps take side by side. Each streams its
// codes and scales through its own ring in shared memory, six of eight column
// tiles ahead (16-byte asynchronous copies: 16 warps keep about 100 KB in flight
// on an SM, and half of that reads at two thirds of the rate). A ninth warp
// brings the token rows, 4 / KH column tiles at a time, into one of two buffers
// that the eight share (bulk copies of its 512-byte rows took 65 ns each). A lane's 16 bytes of a weight row become
// the A operand of m16n8k16 steps without a shuffle -- (w >> 4 i) & 0xf | 0x4300
// is bf16 128 + code, minus 136 the exact weight code. Token rows (B operand,
// eight to a step) lie 32 bytes apart modulo 128, so that a quad's 8-byte reads
// of four rows meet no bank twice. A group's sum of exact products stays in fp32
// and is scaled once. The CTAs of a cluster add their sums over distributed
// shared memory, each its share of the outputs in the order of the columns, so
// no workspace is needed and the result is the same on every run.
// No unit is at its limit: 16 multiplying warps an SM leave 40 % of the issue slots
// empty (11 unpacking instructions for eight weights, about 125 for a warp's column
// tile, wait for one another), and 59 % with 16 rows. Measured, groups of 128:
// 1 x 3584 -> 37888 (SwiGLU) in 17.9 us, 70.0 MB at 3.92 TB/s (0.60 of a copy's
// rate); 16 rows 24.7 us; 16 x 18944 -> 3584, groups of 64, in 18.8 us;
// 1 x 1536 -> 2048 in 3.9 us.
constexpr int kWarps = 8;                   // that multiply
constexpr int kThreads = kWarps * 32 + 32;
constexpr int kPair = 2;                    // column tiles of a ring stage
constexpr int kRing = 4;                    // stages of a warp's ring

// MT: tiles of eight token rows; GS: k16 steps of a scale group (2, 4 or 8); KH: parts of the columns side by side
template <int MT, int GS, int KH>
__global__ void __launch_bounds__(kThreads, 2) linear_kernel(LinearParams p) {
  constexpr int kGroups = 8 / GS;  // of a column tile
  constexpr int kRowTiles = kWarps / KH;
  constexpr int kTileBytes = 1024 + kGroups * 32;
  constexpr int kXTiles = 4 / KH;                 // column tiles of a token buffer
  constexpr int kRowBytes = kXTiles * 256 + 32;   // a token row of it
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t s_full[2], s_empty[2];
  __shared__ int s_abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, t = lane & 3;
  if (tid == 0) {
    s_abort = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i, 32);
      mbar_init(s_empty + i, kWarps);
    }
    fence_mbar_init();
  }
  const int S = p.S, rank = S > 1 ? (int)cluster_ctarank() : 0;
  const int tile = S > 1 ? blockIdx.x / S : blockIdx.x;
  const int n0 = tile * p.outs;                           // first output of this CTA
  const int up = p.swiglu ? (p.n_out + n0) & 15 : 0;      // SwiGLU: where the first up row sits in its tile
  const int c0 = rank * p.per, n_cta = max(0, min(p.w.kt, c0 + p.per) - c0);  // this CTA's column tiles
  const int mid = KH == 1 ? n_cta : (n_cta + 1) / 2;      // of which the first part takes so many
  const uint32_t x_at = kWarps * kRing * kPair * kTileBytes, x_bytes = KH * p.M * kRowBytes;
  auto give_up = [&]() {
    s_abort = 1;
    atomicExch(p.status, kStatusTimeoutProducer);
  };
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  __syncthreads();
  float acc[MT][4];
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[m][0] = acc[m][1] = acc[m][2] = acc[m][3] = 0.f;
  if (warp == kWarps) {
    int buf = 0, parity = 1;  // a barrier that nothing has passed lets parity 1 through
    for (int i = 0; i < mid; i += kXTiles) {
      if (!mbar_wait(s_empty + buf, parity, &s_abort)) give_up();
#pragma unroll
      for (int h = 0; h < KH; ++h) {
        const int n = min(kXTiles, (h == 0 ? mid : n_cta - mid) - i);
        const int k0 = (c0 + h * mid + i) * 128;
        const uint32_t dst = smem_u32(smem) + x_at + buf * x_bytes + h * p.M * kRowBytes + lane * 16;
        for (int m = 0; m < p.M; ++m)
#pragma unroll
          for (int c = 0; c < kXTiles / 2; ++c) {  // 256 columns a step, zeros past K
            const int k = k0 + c * 256 + lane * 8;
            if (c * 2 + (lane >> 4) < n)
              cp_async16_zfill(dst + m * kRowBytes + c * 512, p.x + m * p.xs + (k < p.w.K ? k : 0), k < p.w.K);
          }
      }
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(s_full + buf)) : "memory");
      if (++buf == 2) buf = 0, parity ^= 1;
    }
  } else {
    const Consts k{in_register(0x000f000fu), in_register(0x43004300u), in_register(0xc308c308u)};
    const int kh = warp / kRowTiles, rt = warp % kRowTiles;
    const int kt0 = c0 + kh * mid, n_kt = kh == 0 ? mid : n_cta - mid;
    int wt = (n0 >> 4) + rt;  // packed row tile (past the last: the last, its sums are dropped)
    if (p.swiglu && rt >= kRowTiles / 2) wt = ((p.n_out + n0) >> 4) + rt - kRowTiles / 2;
    wt = min(wt, (p.w.N + 15) / 16 - 1);
    const uint8_t* q = reinterpret_cast<const uint8_t*>(p.w.q) + ((int64_t)wt * p.w.kt + kt0) * 1024 + lane * 16;
    const uint8_t* sc = reinterpret_cast<const uint8_t*>(p.w.s) + ((int64_t)wt * p.w.groups + (int64_t)kt0 * kGroups) * 32 + lane * 16;
    const uint32_t ring = smem_u32(smem) + warp * (kRing * kPair * kTileBytes);
    int fetched = 0;
    uint32_t into = ring;
    auto fetch = [&]() {  // the next stage: codes of its column tiles, then their scales
      if (fetched < n_kt) {
        cp_async16(into + lane * 16, q);
        cp_async16(into + lane * 16 + 512, q + 512);
        const bool two = fetched + 1 < n_kt;
        if (two) {
          cp_async16(into + lane * 16 + 1024, q + 1024);
          cp_async16(into + lane * 16 + 1536, q + 1536);
        }
        if (lane < (two ? 4 : 2) * kGroups) cp_async16(into + kPair * 1024 + lane * 16, sc);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      fetched += kPair;
      q += kPair * 1024;
      sc += kPair * kGroups * 32;
      into = into == ring + (kRing - 1) * kPair * kTileBytes ? ring : into + kPair * kTileBytes;
    };
#pragma unroll
    for (int i = 0; i < kRing - 1; ++i) fetch();
    uint32_t xoff[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) xoff[m] = smem_u32(smem) + x_at + (kh * p.M + min(m * 8 + r, p.M - 1)) * kRowBytes + t * 8;
    // one column tile: u of the stage at `at`, xo bytes into the token rows
    auto column_tile = [&](uint32_t at, int u, uint32_t xo) {
      const uint4 va = lds128(at + u * 1024 + lane * 16), vb = lds128(at + u * 1024 + lane * 16 + 512);
      const uint32_t wa[4] = {va.x, va.y, va.z, va.w}, wb[4] = {vb.x, vb.y, vb.z, vb.w};
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const uint32_t s2 = lds32(at + kPair * 1024 + (u * kGroups + g) * 32 + r * 4);  // rows r and r + 8
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&s2));
        float c[MT][4];
#pragma unroll
        for (int m = 0; m < MT; ++m) c[m][0] = c[m][1] = c[m][2] = c[m][3] = 0.f;
#pragma unroll
        for (int s = g * GS; s < (g + 1) * GS; ++s) {
          const uint32_t a[4] = {s & 1 ? codes2<2>(wa[s >> 1], k) : codes2<0>(wa[s >> 1], k),
                                 s & 1 ? codes2<2>(wb[s >> 1], k) : codes2<0>(wb[s >> 1], k),
                                 s & 1 ? codes2<3>(wa[s >> 1], k) : codes2<1>(wa[s >> 1], k),
                                 s & 1 ? codes2<3>(wb[s >> 1], k) : codes2<1>(wb[s >> 1], k)};
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            uint32_t b0, b1;
            asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(b0), "=r"(b1) : "r"(xoff[m] + xo + s * 32) : "memory");
            mma_bf16(c[m], a, b0, b1);
          }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          acc[m][0] += f.x * c[m][0];
          acc[m][1] += f.x * c[m][1];
          acc[m][2] += f.y * c[m][2];
          acc[m][3] += f.y * c[m][3];
        }
      }
    };
    int buf = 0, parity = 0;
    uint32_t at = ring;
    for (int i0 = 0; i0 < mid; i0 += kXTiles) {
      if (!mbar_wait(s_full + buf, parity, &s_abort)) give_up();
      const uint32_t xo = buf * x_bytes;
#pragma unroll
      for (int j = 0; j < kXTiles; j += kPair) {
        const int i = i0 + j;
        if (i < n_kt) {
          asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory");
          __syncwarp();  // the stage is there for every lane, and the one before it is free
          fetch();
#pragma unroll
          for (int u = 0; u < kPair; ++u) {
            if (i + u < n_kt) column_tile(at, u, xo + (j + u) * 256);
          }
          at = at == ring + (kRing - 1) * kPair * kTileBytes ? ring : at + kPair * kTileBytes;
        }
      }
      __syncwarp();  // every lane has read the token rows
      if (lane == 0) mbar_arrive(s_empty + buf);
      if (++buf == 2) buf = 0, parity ^= 1;
    }
  }
  // sums [part][token][row] in shared memory, then this CTA's share of the outputs, four rows to a thread
  __syncthreads();
  constexpr int kLd = kRowTiles * 16 + 4;
  if (warp < kWarps) {
    float* sums = reinterpret_cast<float*>(smem) + warp / kRowTiles * p.M * kLd + warp % kRowTiles * 16 + r;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int tok = m * 8 + 2 * t + (e & 1);
        if (tok < p.M) sums[tok * kLd + 8 * (e >> 1)] = acc[m][e];
      }
  }
  if (S > 1) cluster_sync(); else __syncthreads();
  finish<KH, kLd, kRowTiles * 8>(p, reinterpret_cast<const float*>(smem), S, rank, n0, up, tid, kThreads);
  if (S > 1) cluster_sync();  // every CTA's sums are read before its shared memory goes
}

template <int MT, int GS, int KH>
static void launch_linear(LinearParams& p, cudaStream_t st) {
  constexpr int kRingBytes = kWarps * kRing * kPair * (1024 + 8 / GS * 32);
  constexpr int kRowBytes = 4 / KH * 256 + 32;
  static_assert(kRingBytes >= 128 * (MT * 8) * 4 + KH * MT * 8 * 16, "the sums fit the rings");
  const int smem = kRingBytes + 2 * KH * p.M * kRowBytes;
  constexpr int kSmem = kRingBytes + 2 * KH * MT * 8 * kRowBytes;
  static bool set[64] = {};
  const int dev = current_device();
  if (!set[dev]) {
    AETHER_CUDA_CHECK(cudaFuncSetAttribute(linear_kernel<MT, GS, KH>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    set[dev] = true;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.tiles * p.S));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2] = {};
  int n = 0;
  if (p.S > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n++].val.clusterDim = {(unsigned)p.S, 1, 1};
  }
  // A launch of at most a CTA an SM may begin while the kernel before it drains (this one waits for it before it touches
  // memory): 1 x 2048 x 1536 takes 3.9 us instead of 4.4. More CTAs would take what slots come free first and load the
  // SMs unevenly: 1 x 37888 x 3584 back to back 23.7 us instead of 20.5.
  if (p.tiles * p.S <= num_sms(dev)) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  AETHER_CUDA_CHECK(cudaLaunchKernelEx(&cfg, linear_kernel<MT, GS, KH>, p));
}
// Rows of a CTA and parts of the columns. An SM's fullest load is n CTAs of (column tiles + 4 for their start and end)
// each; one alone leaves issue slots empty, two hide each other's waits.
static int plan(LinearParams& p) {
  const int sms = num_sms(current_device());
  float best = 0.f;
  int kh = 1;
  for (int h = 1; h <= 2; ++h) {
    const int rows = 128 / h;
    const int outs = !p.swiglu ? rows : p.n_out % 16 == 0 ? rows / 2 : rows / 2 - 16;  // (see row_tile: one tile more)
    const int tiles = (p.n_out + outs - 1) / outs;
    for (int c = 1; c <= 8 && c <= p.w.kt; ++c) {
      const int n = (tiles * c + sms - 1) / sms;
      const float cost = (((p.w.kt + c - 1) / c + h - 1) / h + 4) * (n == 1 ? 0.7f : 0.5f * n);
      if ((h == 1 && c == 1) || cost < best) best = cost, kh = h, p.S = c, p.outs = outs, p.tiles = tiles;
    }
  }
  p.per = (p.w.kt + p.S - 1) / p.S;
  return kh;
}
template <int MT, int GS>
static void launch_parts(LinearParams& p, cudaStream_t st) {
  if (plan(p) == 1)
    launch_linear<MT, GS, 1>(p, st);
  else
    launch_linear<MT, GS, 2>(p, st);
}
template <int MT>
static void launch_group(LinearParams& p, cudaStream_t st) {
  if (p.w.gshift == 7)
    launch_parts<MT, 8>(p, st);
  else if (p.w.gshift == 6)
    launch_parts<MT, 4>(p, st);
  else
    launch_parts<MT, 2>(p, st);
}

// out [N, K] bf16 = code * scale, for products of more rows than a decode
// batch: one thread a word of eight elements. Bound by bytes written in pieces of
// eight, two of a row to a thread. Measured, groups of 128: 37888 x 3584 in 87 us
// (339 MB at 3.9 TB/s, 0.59 of a copy's rate).
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
                  s.numel() == nt * (kt * 128 / group) * 16 && reinterpret_cast<uintptr_t>(s.data_ptr()) % 16 == 0,
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

namespace w4 {
// Checks the arguments of a product of any number of rows and fills p with them; returns the output, made where none is
// given.
static at::Tensor arguments(LinearParams& p, const at::Tensor& x, const at::Tensor& q, const at::Tensor& s, int64_t N,
                            int64_t K, int64_t group, const std::optional<at::Tensor>& bias,
                            const std::optional<at::Tensor>& residual, bool swiglu, const std::optional<at::Tensor>& out) {
  p.w = make_weight(q, s, N, K, group, "linear_w4");
  TORCH_CHECK(x.dim() == 2, "linear_w4: x is [M, K]");
  const int64_t M = x.size(0), n_out = swiglu ? N / 2 : N;
  TORCH_CHECK(!swiglu || N % 2 == 0, "linear_w4: SwiGLU takes an even number of rows (gate, then up)");
  TORCH_CHECK(x.device() == q.device() && x.scalar_type() == at::kBFloat16 && x.size(1) == K && x.stride(1) == 1,
              "linear_w4: x is bf16 [M, K] with unit inner stride, beside the weights");
  TORCH_CHECK(M < (int64_t(1) << 31), "linear_w4: fewer than 2^31 rows");
  const at::Tensor y = out && out->defined() ? *out : at::empty({M, n_out}, x.options());
  TORCH_CHECK(y.device() == q.device() && y.scalar_type() == at::kBFloat16 && y.dim() == 2 && y.size(0) == M &&
                  y.size(1) == n_out && (n_out == 1 || y.stride(1) == 1),
              "linear_w4: out is bf16 [M, N] (SwiGLU: [M, N / 2]) with unit inner stride, beside the weights");
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
  p.y = reinterpret_cast<__nv_bfloat16*>(y.data_ptr());
  p.ys = y.stride(0);
  p.M = (int)M;
  p.n_out = (int)n_out;
  p.swiglu = swiglu;
  return y;
}
}  // namespace w4

at::Tensor linear_w4_output(at::Tensor x, at::Tensor q, at::Tensor s, int64_t N, int64_t K, int64_t group,
                            std::optional<at::Tensor> bias, std::optional<at::Tensor> residual, bool swiglu,
                            std::optional<at::Tensor> out) {
  w4::LinearParams p{};
  return w4::arguments(p, x, q, s, N, K, group, bias, residual, swiglu, out);
}

at::Tensor linear_w4(at::Tensor x, at::Tensor q, at::Tensor s, int64_t N, int64_t K, int64_t group,
                     std::optional<at::Tensor> bias, std::optional<at::Tensor> residual, bool swiglu,
                     std::optional<at::Tensor> out) {
  using namespace w4;
  LinearParams p{};
  const at::Tensor y = arguments(p, x, q, s, N, K, group, bias, residual, swiglu, out);
  const int64_t M = x.size(0);
  TORCH_CHECK(M <= 64, "linear_w4: at most 64 rows");
  if (M == 0) return y;
  c10::cuda::CUDAGuard g(q.device());
  // 16-byte copies: rows on 16-byte boundaries; a tensor map (more than 16 rows) wants rows that do not overlap
  if (reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 != 0 || (M > 1 && x.stride(0) % 8 != 0) || (M > 16 && x.stride(0) < K))
    x = x.clone(at::MemoryFormat::Contiguous);
  p.x = reinterpret_cast<const __nv_bfloat16*>(x.data_ptr());
  p.xs = x.stride(0);
  p.status = device_status_word();
  auto st = at::cuda::getCurrentCUDAStream();
  // Here every group of eight rows costs its products and sums again; on tcgen05 32 rows cost what one does (17 or 24
  // rows there; 16 and 24 here): 3584 -> 3584 8.3 us; 7.5 and 13.5; 18944 -> 3584, groups of 64, 28; 18 and 41;
  // 3584 -> 37888 SwiGLU 30.5; 24.9 and 36 (groups of 32, the one that would gain from a later change: 52; 26 and 39).
  if (M <= 8)
    launch_group<1>(p, st);
  else if (M <= 16)
    launch_group<2>(p, st);
  else
    linear_w4_tc(p, st);
  return y;
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
