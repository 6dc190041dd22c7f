// 8-bit paged KV cache: append with the rotation and the quantisation on the
// way, attention of single tokens over it, and the way back to bf16.
//
// Layout per layer, K and V alike: codes uint8 [pages, Hkv, page, D] (code + 128,
// codes -127..127) and scales fp32 [pages, Hkv, page / 16]: the value of a code
// is code * scale, and 16 consecutive positions of a sequence (a "block") share
// one scale for each KV head. A page's rows of one head are contiguous, so a
// block is one run of 16 * D bytes. Key t of the sequence in page-table row
// `slot` is row t % page of page table[slot, t / page].
//
// Positions, slots and lengths are read from device memory, so a captured CUDA
// graph replays the same launch for any step. A table row, page or position out
// of range is skipped (appends) or taken as an empty sequence / page 0 (reads)
// and reported in the device status word, never dereferenced.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "common.cuh"
#include "decode_common.cuh"
#include "host_utils.h"

namespace aether {
namespace kv8 {

constexpr int kBlock = 16;  // positions that share a scale

// One pool (K or V) of a layer.
struct Pool {
  uint8_t* codes;
  float* scale;
};

// Where positions live; `pages` and `cols` bound every lookup.
struct Map {
  const int* table;  // [rows, cols]
  int rows, cols, pages, shift;
  int64_t stride;
  int Hkv, D;
};

// Physical page of position t of table row `slot`, or -1 (reported).
__device__ __forceinline__ int page_of(const Map& m, int slot, int t, int* status) {
  const int c = t >> m.shift;
  if ((unsigned)slot >= (unsigned)m.rows || (unsigned)c >= (unsigned)m.cols) {
    atomicExch(status, kStatusKvRange);
    return -1;
  }
  const int p = m.table[(int64_t)slot * m.stride + c];
  if ((unsigned)p >= (unsigned)m.pages) {
    atomicExch(status, kStatusKvRange);
    return -1;
  }
  return p;
}
// First code byte of (page, head, row); the block's scale is at the row / 16.
__device__ __forceinline__ int64_t code_offset(const Map& m, int page, int h, int row) {
  return ((((int64_t)page * m.Hkv + h) << m.shift) + row) * m.D;
}
__device__ __forceinline__ int64_t scale_offset(const Map& m, int page, int h, int row) {
  return ((((int64_t)page * m.Hkv + h) << m.shift) + row) >> 4;
}

__device__ __forceinline__ float code_of(uint32_t w, int i) { return (float)((int)((w >> (8 * i)) & 255u) - 128); }

// ------------------------------------------------------------------ append
struct AppendParams {
  const __nv_bfloat16* qkv;  // [T, rs]: q heads, k heads, v heads
  __nv_bfloat16* out;        // [T, os]: rotated q and k heads
  int64_t rs, os;
  const int* pos;        // [B] first new position of each sequence
  const int* slot;       // [B] page-table row (negative: the sequence is skipped)
  const int* row_start;  // [B + 1] rows of qkv of each sequence, or null: one each
  const float* cos_t;    // [max_pos, D / 2]
  const float* sin_t;
  Pool k, v;
  Map m;
  int B, Hq, max_pos;
  int64_t T;
  int* status;
};

// A warp owns one (block of 16 positions, head), so a block's scale has one
// writer and the result depends on no order:
//   y = rope(x) (k heads) or x (v heads), each product rounded by itself
//   s = max(s_old if the block holds older tokens, max |y| / 127)
//   code = rint(y * (1 / s)); older codes c become rint(c * (s_old / s))
// max |y| is taken on the bit patterns, so that a NaN wins and the block reads
// as NaN. With row_start, unit u belongs to the sequence b whose first unit
// row_start[b] / 16 + 2 b is the last one not after u: a sequence of n rows
// touches at most n / 16 + 1.875 blocks, so these ranges never overlap.
template <int D>
__global__ void __launch_bounds__(128) append_kernel(AppendParams p) {
  constexpr int kLanes = D / 16;            // lanes of one token: 8 + 8 dims each
  constexpr int kTok = 32 / kLanes;         // tokens side by side
  constexpr int kIt = kBlock / kTok;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int H = p.Hq + 2 * p.m.Hkv;
  const int h = blockIdx.y * 4 + warp;
  int b, j, r0, n;
  if (p.row_start == nullptr) {
    b = blockIdx.x;
    j = 0;
    r0 = b;
    n = 1;
  } else {
    const int u = blockIdx.x;
    int cnt = 0;
    for (int i = 0; i < p.B; i += 32) {
      const bool in = i + lane < p.B && (p.row_start[i + lane] >> 4) + 2 * (i + lane) <= u;
      cnt += __popc(__ballot_sync(0xffffffffu, in));
    }
    if (cnt == 0) return;
    b = cnt - 1;
    r0 = p.row_start[b];
    n = p.row_start[b + 1] - r0;
    j = u - ((r0 >> 4) + 2 * b);
  }
  if (h >= H) return;
  const int pos = p.pos[b], slot = p.slot[b];
  const int base = ((pos >> 4) + j) << 4;  // first position of the block
  const int lo = max(pos, base), hi = min(pos + n, base + kBlock);
  if (slot < 0 || lo >= hi) return;
  if (pos < 0 || r0 < 0 || r0 + (int64_t)n > p.T || hi > p.max_pos) {
    if (lane == 0) atomicExch(p.status, kStatusKvRange);
    return;
  }
  const int page = page_of(p.m, slot, base, p.status);
  if (page < 0) return;
  const int c = (lane % kLanes) * 8, sub = lane / kLanes;
  const bool is_q = h < p.Hq, is_v = h >= p.Hq + p.m.Hkv;
  float y[kIt][16];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kIt; ++i) {
    const int t = base + i * kTok + sub;
    if (t < lo || t >= hi) continue;
    const int64_t r = r0 + (t - pos);
    const __nv_bfloat16* x = p.qkv + r * p.rs + (int64_t)h * D + c;
    float a[8], bb[8];
    dec::unpack8(*reinterpret_cast<const uint4*>(x), a);
    dec::unpack8(*reinterpret_cast<const uint4*>(x + D / 2), bb);
    if (!is_v) {
      const float* cp = p.cos_t + (int64_t)t * (D / 2) + c;
      const float* sp = p.sin_t + (int64_t)t * (D / 2) + c;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x1 = a[e], x2 = bb[e];
        a[e] = __fsub_rn(__fmul_rn(x1, cp[e]), __fmul_rn(x2, sp[e]));
        bb[e] = __fadd_rn(__fmul_rn(x2, cp[e]), __fmul_rn(x1, sp[e]));
      }
      __nv_bfloat16* o = p.out + r * p.os + (int64_t)h * D + c;
      *reinterpret_cast<uint4*>(o) = dec::pack8(a);
      *reinterpret_cast<uint4*>(o + D / 2) = dec::pack8(bb);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      y[i][e] = a[e];
      y[i][8 + e] = bb[e];
      top = max(top, max(__float_as_uint(a[e]) & 0x7fffffffu, __float_as_uint(bb[e]) & 0x7fffffffu));
    }
  }
  if (is_q) return;
  top = __reduce_max_sync(0xffffffffu, top);
  const Pool& pool = is_v ? p.v : p.k;
  const int hk = h - p.Hq - (is_v ? p.m.Hkv : 0);
  const int row = base & ((1 << p.m.shift) - 1);
  uint8_t* codes = pool.codes + code_offset(p.m, page, hk, row);
  float* scale = pool.scale + scale_offset(p.m, page, hk, row);
  // 2^-100: a block of zeros gets a tiny scale, and 1 / s stays finite
  const float s_new = __fdiv_rn(__uint_as_float(max(top, 0x0d800000u)), 127.f);
  float s = s_new;
  if (lo > base) {
    const float s_old = *scale;
    s = __uint_as_float(max(__float_as_uint(s_old), __float_as_uint(s_new)));
    const float f = __fdiv_rn(s_old, s);
    for (int i = lane; i < (lo - base) * (D / 4); i += 32) {
      uint32_t w = reinterpret_cast<uint32_t*>(codes)[i], o = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) o |= (uint32_t)(__float2int_rn(__fmul_rn(code_of(w, e), f)) + 128) << (8 * e);
      reinterpret_cast<uint32_t*>(codes)[i] = o;
    }
  }
  __syncwarp();
  if (lane == 0) *scale = s;
  const float inv = __fdiv_rn(1.f, s);
#pragma unroll
  for (int i = 0; i < kIt; ++i) {
    const int t = base + i * kTok + sub;
    if (t < lo || t >= hi) continue;
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int q = min(127, max(-127, __float2int_rn(__fmul_rn(y[i][e], inv))));
      w[e >> 2] |= (uint32_t)(q + 128) << (8 * (e & 3));
    }
    uint8_t* d = codes + (t - base) * D + c;
    *reinterpret_cast<uint2*>(d) = make_uint2(w[0], w[1]);
    *reinterpret_cast<uint2*>(d + D / 2) = make_uint2(w[2], w[3]);
  }
}

// ------------------------------------------------------------------ gather
// out [B, n, Hkv, D] bf16 = code * scale of positions first[b] .. first[b] + n:
// a thread turns 16 codes into two 16-byte stores. Bound by the bytes moved.
__global__ void __launch_bounds__(256) gather_kernel(Pool c, Map m, const int* __restrict__ slot,
                                                     const int* __restrict__ first, int first0, int64_t n, int64_t total,
                                                     __nv_bfloat16* __restrict__ out, int* status) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= total) return;
  const int per = m.D / 16;
  const int ch = (int)(i % per) * 16;
  const int64_t r = i / per;  // (b, position, head)
  const int h = (int)(r % m.Hkv);
  const int64_t bt = r / m.Hkv;
  const int b = (int)(bt / n);
  const int t = (first ? first[b] : first0) + (int)(bt % n);
  uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
  const int page = page_of(m, slot[b], t, status);
  if (page >= 0) {
    const int row = t & ((1 << m.shift) - 1);
    const uint4 w = *reinterpret_cast<const uint4*>(c.codes + code_offset(m, page, h, row) + ch);
    const float s = c.scale[scale_offset(m, page, h, row)];
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
    float v[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = code_of(ws[e >> 2], e & 3) * s;
    lo = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    hi = make_uint4(pack_bf16(v[8], v[9]), pack_bf16(v[10], v[11]), pack_bf16(v[12], v[13]), pack_bf16(v[14], v[15]));
  }
  uint4* o = reinterpret_cast<uint4*>(out + r * m.D + ch);
  o[0] = lo;
  o[1] = hi;
}

// ------------------------------------------------------------------ attention
constexpr float kLog2e = 1.4426950408889634f;

struct AttnParams {
  const __nv_bfloat16* q;
  int64_t q_rs;
  __nv_bfloat16* out;
  int64_t o_rs;
  Pool k, v;
  Map m;
  const int* slot;
  const int* seqlen;
  int B, Hq, window;
  float scale, softcap;
  int* status;
};

// One CTA of 128 threads for each (sequence, query head): 128 keys at a time, a
// thread a key for the logits, a thread a dimension for the sum, running
// maximum and sum in fp32.
__global__ void __launch_bounds__(128) attn_kernel(AttnParams p) {
  __shared__ float sq[128], sp[128], red[4];
  __shared__ int64_t srow[128];
  const int b = blockIdx.y, h = blockIdx.x, tid = threadIdx.x;
  const int D = p.m.D, hk = h / (p.Hq / p.m.Hkv);
  const int slot = p.slot[b];
  const int len = slot < 0 ? 0 : min(max(p.seqlen[b], 0), p.m.cols << p.m.shift);
  const int first = p.window > 0 ? max(0, len - p.window) : 0;
  if (tid < D) sq[tid] = __bfloat162float(p.q[(int64_t)b * p.q_rs + (int64_t)h * D + tid]);
  float mx = -INFINITY, sum = 0.f, acc = 0.f;
  for (int k0 = first; k0 < len; k0 += 128) {
    const int t = k0 + tid;
    float x = -INFINITY;
    int64_t row = -1;
    __syncthreads();
    if (t < len) {
      const int page = page_of(p.m, slot, t, p.status);
      if (page >= 0) {
        const int r = t & ((1 << p.m.shift) - 1);
        row = (((int64_t)page * p.m.Hkv + hk) << p.m.shift) + r;
        const uint32_t* kc = reinterpret_cast<const uint32_t*>(p.k.codes + row * D);
        float d = 0.f;
        for (int i = 0; i < D / 4; ++i) {
          const uint32_t w = kc[i];
#pragma unroll
          for (int e = 0; e < 4; ++e) d += sq[4 * i + e] * code_of(w, e);
        }
        x = d * p.k.scale[row >> 4] * p.scale;
        if (p.softcap > 0.f) x = p.softcap * tanhf(x / p.softcap);
      }
    }
    float m = warp_max(x);
    if ((tid & 31) == 0) red[tid >> 5] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float mn = fmaxf(mx, m), base = mn == -INFINITY ? 0.f : mn;
    const float alpha = exp2f((mx - base) * kLog2e);
    const float e = exp2f((x - base) * kLog2e);
    sp[tid] = e;
    srow[tid] = row;
    float s = warp_sum(e);
    __syncthreads();
    if ((tid & 31) == 0) red[tid >> 5] = s;
    __syncthreads();
    sum = sum * alpha + (red[0] + red[1] + red[2] + red[3]);
    acc *= alpha;
    mx = mn;
    if (tid < D)
      for (int i = 0; i < min(128, len - k0); ++i) {
        const int64_t r = srow[i];
        if (r >= 0) acc += sp[i] * (p.v.scale[r >> 4] * (float)((int)p.v.codes[r * D + tid] - 128));
      }
  }
  if (tid < D) p.out[(int64_t)b * p.o_rs + (int64_t)h * D + tid] = __float2bfloat16(sum == 0.f ? 0.f : acc / sum);
}

// ------------------------------------------------------------------ host
static void check_pool(const at::Tensor& codes, const at::Tensor& scale, const at::Tensor& table, const char* what) {
  TORCH_CHECK(codes.is_cuda() && codes.scalar_type() == at::kByte && codes.dim() == 4 && codes.is_contiguous(), what,
              ": codes are contiguous CUDA uint8 [pages, Hkv, page, D]");
  const int64_t P = codes.size(2), D = codes.size(3);
  TORCH_CHECK(P >= kBlock && (P & (P - 1)) == 0 && P <= 65536, what, ": page is a power of two of at least 16");
  TORCH_CHECK(D == 64 || D == 128, what, ": head_dim 64 or 128");
  TORCH_CHECK(codes.size(0) < (int64_t(1) << 31) && codes.size(1) >= 1, what, ": pages and KV heads");
  TORCH_CHECK(scale.device() == codes.device() && scale.scalar_type() == at::kFloat && scale.dim() == 3 &&
                  scale.is_contiguous() && scale.size(0) == codes.size(0) && scale.size(1) == codes.size(1) &&
                  scale.size(2) == P / kBlock,
              what, ": scales are contiguous float32 [pages, Hkv, page / 16] beside the codes");
  TORCH_CHECK(table.device() == codes.device() && table.scalar_type() == at::kInt && table.dim() == 2 &&
                  (table.size(1) <= 1 || table.stride(1) == 1),
              what, ": page_table is int32 [rows, max_pages] with unit inner stride, beside the codes");
  TORCH_CHECK(table.size(1) * P < (int64_t(1) << 31), what, ": page_table holds fewer than 2^31 positions");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(codes.data_ptr()) % 16 == 0, what, ": codes start on a 16-byte boundary");
}
static Map make_map(const at::Tensor& codes, const at::Tensor& table) {
  Map m{};
  m.table = table.data_ptr<int>();
  m.rows = (int)table.size(0);
  m.cols = (int)table.size(1);
  m.stride = table.stride(0);
  m.pages = (int)codes.size(0);
  m.Hkv = (int)codes.size(1);
  m.D = (int)codes.size(3);
  while ((int64_t(1) << m.shift) < codes.size(2)) ++m.shift;
  return m;
}
static Pool pool_of(const at::Tensor& codes, const at::Tensor& scale) {
  return Pool{codes.data_ptr<uint8_t>(), scale.data_ptr<float>()};
}
static void check_ints(const at::Tensor& t, const at::Tensor& like, int64_t n, const char* what) {
  TORCH_CHECK(t.device() == like.device() && t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous() &&
                  t.size(0) >= n,
              what, " int32 on the cache's device");
}
static void check_same(const at::Tensor& kc, const at::Tensor& vc, const char* what) {
  TORCH_CHECK(kc.sizes() == vc.sizes() && kc.device() == vc.device(), what, ": k and v pools of one shape and device");
}

}  // namespace kv8

void rope_kv8_append(at::Tensor qkv, at::Tensor pos, at::Tensor slot, std::optional<at::Tensor> row_start,
                     at::Tensor cos_t, at::Tensor sin_t, at::Tensor kc, at::Tensor ks, at::Tensor vc, at::Tensor vs,
                     at::Tensor page_table, int64_t Hq, at::Tensor out) {
  using namespace kv8;
  check_pool(kc, ks, page_table, "rope_kv8_append");
  check_pool(vc, vs, page_table, "rope_kv8_append");
  check_same(kc, vc, "rope_kv8_append");
  const int64_t Hkv = kc.size(1), D = kc.size(3), T = qkv.size(0), B = pos.size(0);
  TORCH_CHECK(Hq >= 1 && Hq + 2 * Hkv <= 4 * 65535, "rope_kv8_append: heads");
  TORCH_CHECK(qkv.device() == kc.device() && qkv.dim() == 2 && qkv.scalar_type() == at::kBFloat16 &&
                  qkv.size(1) >= (Hq + 2 * Hkv) * D && qkv.stride(1) == 1 && qkv.stride(0) % 8 == 0 &&
                  reinterpret_cast<uintptr_t>(qkv.data_ptr()) % 16 == 0,
              "rope_kv8_append: qkv is bf16 [T, >= (Hq + 2 Hkv) D], rows on 16-byte boundaries");
  TORCH_CHECK(out.device() == kc.device() && out.dim() == 2 && out.scalar_type() == at::kBFloat16 &&
                  out.size(0) == T && out.size(1) >= (Hq + Hkv) * D && out.stride(1) == 1 && out.stride(0) % 8 == 0 &&
                  reinterpret_cast<uintptr_t>(out.data_ptr()) % 16 == 0,
              "rope_kv8_append: out is bf16 [T, >= (Hq + Hkv) D], rows on 16-byte boundaries");
  check_ints(pos, kc, B, "rope_kv8_append: pos [B]");
  check_ints(slot, kc, B, "rope_kv8_append: slot [B]");
  TORCH_CHECK(T < (int64_t(1) << 31), "rope_kv8_append: fewer than 2^31 rows");
  int64_t units = B;
  if (row_start && row_start->defined()) {
    check_ints(*row_start, kc, B + 1, "rope_kv8_append: row_start [B + 1]");
    units = T / kBlock + 2 * B;
  } else {
    TORCH_CHECK(T == B, "rope_kv8_append: without row_start, one row of qkv for each sequence");
  }
  for (const at::Tensor* t : {&cos_t, &sin_t})
    TORCH_CHECK(t->device() == kc.device() && t->scalar_type() == at::kFloat && t->dim() == 2 && t->is_contiguous() &&
                    t->size(1) == D / 2 && t->size(0) == cos_t.size(0) && reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0,
                "rope_kv8_append: cos / sin are contiguous float32 [max_pos, D / 2]");
  if (T == 0 || B == 0) return;
  c10::cuda::CUDAGuard g(kc.device());
  AppendParams p{};
  p.qkv = reinterpret_cast<const __nv_bfloat16*>(qkv.data_ptr());
  p.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  p.rs = qkv.stride(0);
  p.os = out.stride(0);
  p.pos = pos.data_ptr<int>();
  p.slot = slot.data_ptr<int>();
  p.row_start = row_start && row_start->defined() ? row_start->data_ptr<int>() : nullptr;
  p.cos_t = cos_t.data_ptr<float>();
  p.sin_t = sin_t.data_ptr<float>();
  p.k = pool_of(kc, ks);
  p.v = pool_of(vc, vs);
  p.m = make_map(kc, page_table);
  p.B = (int)B;
  p.Hq = (int)Hq;
  p.max_pos = (int)std::min<int64_t>(cos_t.size(0), (int64_t(1) << 31) - 1);
  p.T = T;
  p.status = device_status_word();
  const dim3 grid((unsigned)units, (unsigned)((Hq + 2 * Hkv + 3) / 4));
  auto st = at::cuda::getCurrentCUDAStream();
  if (D == 128)
    append_kernel<128><<<grid, 128, 0, st>>>(p);
  else
    append_kernel<64><<<grid, 128, 0, st>>>(p);
  AETHER_CUDA_CHECK(cudaGetLastError());
}

void gather_kv8(at::Tensor codes, at::Tensor scale, at::Tensor page_table, at::Tensor slot,
                std::optional<at::Tensor> first, int64_t first0, at::Tensor out) {
  using namespace kv8;
  check_pool(codes, scale, page_table, "gather_kv8");
  TORCH_CHECK(out.device() == codes.device() && out.scalar_type() == at::kBFloat16 && out.dim() == 4 &&
                  out.is_contiguous() && out.size(2) == codes.size(1) && out.size(3) == codes.size(3) &&
                  reinterpret_cast<uintptr_t>(out.data_ptr()) % 16 == 0,
              "gather_kv8: out is contiguous bf16 [B, n, Hkv, D]");
  const int64_t B = out.size(0), n = out.size(1);
  check_ints(slot, codes, B, "gather_kv8: slot [B]");
  const bool each = first && first->defined();
  if (each) check_ints(*first, codes, B, "gather_kv8: first [B]");
  TORCH_CHECK(n < (int64_t(1) << 31) && first0 >= 0 && first0 + n < (int64_t(1) << 31), "gather_kv8: positions");
  const int64_t total = out.numel() / 16;
  if (total == 0) return;
  c10::cuda::CUDAGuard g(codes.device());
  TORCH_CHECK((total + 255) / 256 < (int64_t(1) << 31), "gather_kv8: output too large");
  gather_kernel<<<(unsigned)((total + 255) / 256), 256, 0, at::cuda::getCurrentCUDAStream()>>>(
      pool_of(codes, scale), make_map(codes, page_table), slot.data_ptr<int>(), each ? first->data_ptr<int>() : nullptr,
      (int)first0, n, total, reinterpret_cast<__nv_bfloat16*>(out.data_ptr()), device_status_word());
  AETHER_CUDA_CHECK(cudaGetLastError());
}

void kv8_decode_attention(at::Tensor q, at::Tensor kc, at::Tensor ks, at::Tensor vc, at::Tensor vs,
                          at::Tensor page_table, at::Tensor slot, at::Tensor seqlen, at::Tensor out, int64_t Hq,
                          double scale, int64_t window, double softcap) {
  using namespace kv8;
  check_pool(kc, ks, page_table, "kv8_decode_attention");
  check_pool(vc, vs, page_table, "kv8_decode_attention");
  check_same(kc, vc, "kv8_decode_attention");
  const int64_t Hkv = kc.size(1), D = kc.size(3), B = q.size(0);
  TORCH_CHECK(Hq >= Hkv && Hq % Hkv == 0, "kv8_decode_attention: query heads are a multiple of the KV heads");
  for (const at::Tensor* t : {&q, &out})
    TORCH_CHECK(t->device() == kc.device() && t->dim() == 2 && t->scalar_type() == at::kBFloat16 && t->size(0) == B &&
                    t->size(1) >= Hq * D && t->stride(1) == 1 && t->stride(0) % 8 == 0 &&
                    reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0,
                "kv8_decode_attention: q and out are bf16 [B, >= Hq D], rows on 16-byte boundaries");
  check_ints(slot, kc, B, "kv8_decode_attention: slot [B]");
  check_ints(seqlen, kc, B, "kv8_decode_attention: seqlen [B]");
  TORCH_CHECK(window >= 0 && window < (int64_t(1) << 31) && softcap >= 0, "kv8_decode_attention: window and softcap");
  TORCH_CHECK(B <= 65535, "kv8_decode_attention: at most 65535 sequences");
  if (B == 0) return;
  c10::cuda::CUDAGuard g(kc.device());
  AttnParams p{};
  p.q = reinterpret_cast<const __nv_bfloat16*>(q.data_ptr());
  p.q_rs = q.stride(0);
  p.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  p.o_rs = out.stride(0);
  p.k = pool_of(kc, ks);
  p.v = pool_of(vc, vs);
  p.m = make_map(kc, page_table);
  p.slot = slot.data_ptr<int>();
  p.seqlen = seqlen.data_ptr<int>();
  p.B = (int)B;
  p.Hq = (int)Hq;
  p.window = (int)window;
  p.scale = (float)scale;
  p.softcap = (float)softcap;
  p.status = device_status_word();
  attn_kernel<<<dim3((unsigned)Hq, (unsigned)B), 128, 0, at::cuda::getCurrentCUDAStream()>>>(p);
  AETHER_CUDA_CHECK(cudaGetLastError());
}

}  // namespace aether
