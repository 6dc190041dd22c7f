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
// of range is reported in the device status word and never dereferenced: an
// append skips the block, a gather reads zeros, attention takes a bad table row
// for an empty sequence, stops at the table's end and gives the keys of a bad
// page no weight.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp16.h>

#include <cmath>

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

// A warp owns one (block of 16 positions, head) at a time, so a block's scale
// has one writer and the result depends on no order:
//   y = rope(x) (k heads) or x (v heads), each product rounded by itself
//   s = max(s_old if the block holds older tokens, max |y| / 127)
//   code = rint(y * (1 / s)); older codes c become rint(c * (s_old / s))
// max |y| is taken on the bit patterns, so that a NaN wins and the block reads
// as NaN. With row_start, unit u belongs to the sequence b whose first unit
// row_start[b] / 16 + 2 b is the last one not after u: a sequence of n rows
// touches at most n / 16 + 1.875 blocks, so these ranges never overlap.
// q heads need no block: a warp turns kTok tokens of one head after another and
// keeps the tokens' angles in registers. Bound by the bytes of qkv and out while
// blocks are many; a few tokens are spread over more CTAs (latency is all there
// is). Measured, 28 + 2 * 4 heads of D 128: 8 x 2048 tokens in 54.5 us (285 MB at
// 5.2 TB/s, 0.80 of a copy's rate; 64 x 4096: 6.1 TB/s), 64 single tokens in 5.6.
constexpr int kAppendWarps = 8;

template <int D>
__global__ void __launch_bounds__(kAppendWarps * 32, 2) append_kernel(AppendParams p) {
  constexpr int kLanes = D / 16;            // lanes of one token: 8 + 8 dims each
  constexpr int kTok = 32 / kLanes;         // tokens side by side
  constexpr int kIt = kBlock / kTok;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
  const int row = base & ((1 << p.m.shift) - 1);
  const int gw = blockIdx.y * kAppendWarps + warp, W = gridDim.y * kAppendWarps;
  // y = x rotated by position t's angles, dims c .. and D / 2 + c ..
  auto angles = [&](int t, float (&cs)[8], float (&sn)[8]) {
    const float4* cp = reinterpret_cast<const float4*>(p.cos_t + (int64_t)t * (D / 2) + c);
    const float4* sp = reinterpret_cast<const float4*>(p.sin_t + (int64_t)t * (D / 2) + c);
    const float4 c0 = __ldg(cp), c1 = __ldg(cp + 1), s0 = __ldg(sp), s1 = __ldg(sp + 1);
    cs[0] = c0.x, cs[1] = c0.y, cs[2] = c0.z, cs[3] = c0.w, cs[4] = c1.x, cs[5] = c1.y, cs[6] = c1.z, cs[7] = c1.w;
    sn[0] = s0.x, sn[1] = s0.y, sn[2] = s0.z, sn[3] = s0.w, sn[4] = s1.x, sn[5] = s1.y, sn[6] = s1.z, sn[7] = s1.w;
  };
  auto rotate = [&](float (&a)[8], float (&bb)[8], const float (&cs)[8], const float (&sn)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x1 = a[e], x2 = bb[e];
      a[e] = __fsub_rn(__fmul_rn(x1, cs[e]), __fmul_rn(x2, sn[e]));
      bb[e] = __fadd_rn(__fmul_rn(x2, cs[e]), __fmul_rn(x1, sn[e]));
    }
  };
  // k and v heads: the whole block at once
  for (int h = gw; h < 2 * p.m.Hkv; h += W) {
    const bool is_v = h >= p.m.Hkv;
    const Pool& pool = is_v ? p.v : p.k;
    const int hk = is_v ? h - p.m.Hkv : h;
    uint8_t* codes = pool.codes + code_offset(p.m, page, hk, row);
    float* scale = pool.scale + scale_offset(p.m, page, hk, row);
    const float s_old = lo > base ? *scale : 0.f;
    uint4 xa[kIt], xb[kIt];
#pragma unroll
    for (int i = 0; i < kIt; ++i) {
      const int t = base + i * kTok + sub;
      if (t >= lo && t < hi) {
        const __nv_bfloat16* x = p.qkv + (int64_t)(r0 + (t - pos)) * p.rs + (int64_t)(p.Hq + h) * D + c;
        xa[i] = *reinterpret_cast<const uint4*>(x);
        xb[i] = *reinterpret_cast<const uint4*>(x + D / 2);
      }
    }
    auto value = [&](int i, int t, float (&a)[8], float (&bb)[8]) {
      dec::unpack8(xa[i], a);
      dec::unpack8(xb[i], bb);
      if (is_v) return;
      float cs[8], sn[8];
      angles(t, cs, sn);
      rotate(a, bb, cs, sn);
    };
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kIt; ++i) {
      const int t = base + i * kTok + sub;
      if (t < lo || t >= hi) continue;
      float a[8], bb[8];
      value(i, t, a, bb);
      if (!is_v) {
        __nv_bfloat16* o = p.out + (int64_t)(r0 + (t - pos)) * p.os + (int64_t)(p.Hq + h) * D + c;
        *reinterpret_cast<uint4*>(o) = dec::pack8(a);
        *reinterpret_cast<uint4*>(o + D / 2) = dec::pack8(bb);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e)
        top = max(top, max(__float_as_uint(a[e]) & 0x7fffffffu, __float_as_uint(bb[e]) & 0x7fffffffu));
    }
    top = __reduce_max_sync(0xffffffffu, top);
    // 2^-100: a block of zeros gets a tiny scale, and 1 / s stays finite
    const float s_new = __fdiv_rn(__uint_as_float(max(top, 0x0d800000u)), 127.f);
    float s = s_new;
    if (lo > base) {
      s = __uint_as_float(max(__float_as_uint(s_old), __float_as_uint(s_new)));
      const float f = __fdiv_rn(s_old, s);
      if (f != 1.f)  // the scale has grown (or is no number)
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
      float a[8], bb[8];
      value(i, t, a, bb);  // again: cheaper than 64 registers to keep it
      uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int q = min(127, max(-127, __float2int_rn(__fmul_rn(e < 8 ? a[e] : bb[e - 8], inv))));
        w[e >> 2] |= (uint32_t)(q + 128) << (8 * (e & 3));
      }
      uint8_t* d = codes + (t - base) * D + c;
      *reinterpret_cast<uint2*>(d) = make_uint2(w[0], w[1]);
      *reinterpret_cast<uint2*>(d + D / 2) = make_uint2(w[2], w[3]);
    }
  }
  // q heads: kTok tokens of a head at a time, seven heads in flight, the tokens' angles kept from head to head
  const int i_lo = (lo - base) / kTok, ni = (hi - 1 - base) / kTok - i_lo + 1, step = W / ni;
  if (gw >= step * ni) return;
  const int t = base + (i_lo + gw % ni) * kTok + sub;
  const bool in = t >= lo && t < hi;
  const int64_t tok = r0 + (in ? t - pos : lo - pos);
  float cs[8], sn[8];
  angles(in ? t : lo, cs, sn);
  const __nv_bfloat16* x = p.qkv + tok * p.rs + c;
  __nv_bfloat16* o = p.out + tok * p.os + c;
  constexpr int kHeads = 7;
  for (int h = gw / ni; h < p.Hq; h += kHeads * step) {
    uint4 xa[kHeads], xb[kHeads];
#pragma unroll
    for (int k = 0; k < kHeads; ++k)
      if (h + k * step < p.Hq) {
        xa[k] = *reinterpret_cast<const uint4*>(x + (h + k * step) * D);
        xb[k] = *reinterpret_cast<const uint4*>(x + (h + k * step) * D + D / 2);
      }
#pragma unroll
    for (int k = 0; k < kHeads; ++k)
      if (h + k * step < p.Hq) {
        float a[8], bb[8];
        dec::unpack8(xa[k], a);
        dec::unpack8(xb[k], bb);
        rotate(a, bb, cs, sn);
        if (in) {
          *reinterpret_cast<uint4*>(o + (h + k * step) * D) = dec::pack8(a);
          *reinterpret_cast<uint4*>(o + (h + k * step) * D + D / 2) = dec::pack8(bb);
        }
      }
  }
}

// ------------------------------------------------------------------ gather
struct GatherParams {
  Pool c;
  Map m;
  const int* slot;
  const int* first;  // [B], or null: first0 for all
  int first0, n, heads;  // heads of one CTA
  __nv_bfloat16* out;    // [B, n, Hkv, D]
  int* status;
};

// out = code * scale, rounded once: a thread keeps its head and its 16 dims and
// turns kGatherRows positions, all loaded before the first is stored. Bound by
// the bytes moved; a position's heads are one run of the output, and 128 bytes
// of a head's row one line of the pool. Measured, 4 heads of D 128: 64 x 4096
// positions in 75 us (403 MB at 5.4 TB/s, 0.82 of a copy's rate).
constexpr int kGatherThreads = 256;
constexpr int kGatherRows = 2;

// four codes of w times s
__device__ __forceinline__ uint2 four(uint32_t w, float s) {
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e)  // 2^23 + u, minus 2^23 + 128, exact
    v[e] = __fmul_rn(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7650 + e)) - 8388736.f, s);
  return make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
}

__global__ void __launch_bounds__(kGatherThreads) gather_kernel(GatherParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const int per = p.m.D / 16;  // threads of a row
  const int side = kGatherThreads / (per * p.heads);  // positions side by side
  const int ch = (threadIdx.x % per) * 16, hs = threadIdx.x / per;
  const int h = blockIdx.z * p.heads + hs % p.heads, sub = hs / p.heads;
  const int b = blockIdx.y;
  if (sub >= side || h >= p.m.Hkv) return;
  const int i0 = blockIdx.x * side * kGatherRows + sub;
  const int slot = p.slot[b], f = p.first ? p.first[b] : p.first0;
  int page[kGatherRows];
#pragma unroll
  for (int k = 0; k < kGatherRows; ++k) page[k] = i0 + k * side < p.n ? page_of(p.m, slot, f + i0 + k * side, p.status) : -1;
  uint4 w[kGatherRows];
  float s[kGatherRows];
#pragma unroll
  for (int k = 0; k < kGatherRows; ++k) {
    w[k] = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
    s[k] = 0.f;
    if (page[k] >= 0) {
      const int row = (f + i0 + k * side) & ((1 << p.m.shift) - 1);
      w[k] = *reinterpret_cast<const uint4*>(p.c.codes + code_offset(p.m, page[k], h, row) + ch);
      s[k] = p.c.scale[scale_offset(p.m, page[k], h, row)];
    }
  }
#pragma unroll
  for (int k = 0; k < kGatherRows; ++k) {
    const int i = i0 + k * side;
    if (i >= p.n) continue;
    uint4* o = reinterpret_cast<uint4*>(p.out + (((int64_t)b * p.n + i) * p.m.Hkv + h) * p.m.D + ch);
    const uint2 a = four(w[k].x, s[k]), bb = four(w[k].y, s[k]), c = four(w[k].z, s[k]), d = four(w[k].w, s[k]);
    o[0] = make_uint4(a.x, a.y, bb.x, bb.y);
    o[1] = make_uint4(c.x, c.y, d.x, d.y);
  }
}

// ------------------------------------------------------------------ attention
// x_j = scale * s_k[j / 16] * sum_d q_d c_jd, p = softmax(x), o = sum_j p_j s_v[j / 16] c'_j
//
// Codes are exact in fp16, so both products run on the tensor cores with the
// codes as they are and the scales outside: S^T = K q^T (16 keys x 8 query
// heads of one KV head) and O^T = V^T w^T, as m16n8k16 steps whose operands come
// straight from 16-byte global loads -- the order of the contraction is free, so
// a thread's 16 consecutive codes are the k slots it owns, and no shared memory
// is needed. q (8 significant bits) is exact in fp16 after a power-of-two scaling
// of its row; the weight w_j = 2^(x_j + log2 s_v - M) carries the value scale, so
// that fp16 (2^-11, range 2^-24 .. 2^14 around the running reference M) rounds
// it relative to what it adds to the output. The denominator sums w_j / s_v in
// fp32. M moves only when a weight would pass 2^4, so the accumulators are
// rescaled a few times per sequence and not at every step.
//
// Bound by the cache's bytes. The 16-key blocks of all (sequence, KV head, eight
// query heads) segments are laid end to end and cut into equal ranges, one for
// each CTA (two of eight warps on an SM), so ragged batches fill the GPU; a
// segment that one CTA holds whole is written at once, the parts of a cut one go
// through the workspace to a second kernel, which joins them in order; it has its
// prefix sums ready when the first one ends (joined by the last CTA to arrive,
// 37 parts took 8 us of fences, waits and loads).
//
// Measured, 28 query heads of 4 KV heads, D 128, pages of 64: 64 x 4096 keys in
// 50.5 us (5.34 TB/s, 0.81 of a copy's rate: 16 warps a SM with a step of K and V
// each in registers keep 64 KB in flight, and the tensor pipe is busy for a sixth
// of the time); 1 x 100001 keys, 8 KV heads, in 45 us (0.69: a range more or less
// of 128 keys is 4 % of a CTA's work, and the join adds 3 us); 16 ragged sequences
// of up to 2304 keys in 14.5 us and 1 x 97 keys (12 heads of 2) in 4.5 us, the chain
// page -> codes -> products -> sums of eight warps; 6.3 us with a page table of 4096
// positions, which takes ranges and the join. 64 x 4096 with a softcap 55.2 us, with
// a window of 2048 31.8 (134 MB, 4.2 TB/s), with D 64 34.4 (135 MB, 3.9 TB/s). A ring of asynchronous copies in shared
// memory adds instructions and was slower (63 us for 64 x 4096, this form then 55).
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxCtas = 512;       // parts: two for each CTA
constexpr int kMaxSeqs = 8192;
constexpr int kMinSteps = 2;        // of kWarps blocks: shorter ranges cost more to join than they save
// Page tables (or windows) of at most so many positions: a CTA for each segment, none cut. The host knows the table's
// width and not the lengths, so short sequences in a wide table, as a server's, go the other way. 1, 16, 64 and 256 full sequences of 4 KV
// heads, whole / in ranges: 512 keys 6.8 / 8.1, 7.2 / 10.4, 9.6 / 11.5, 36.2 / 37.5 us; 1024 keys 9.4 / 8.8, 9.8 / 11.9,
// 13.9 / 20.1, 57.0 / 56.1; 2048 keys 14.6 / 9.3, 14.9 / 14.2, 26.4 / 30.9, 100.5 / 94.2.
constexpr int kWholeKeys = 1024;
constexpr float kWeightBits = 10.f; // weights are at most 2^(10 + 4) in fp16
constexpr int kPartFloats = 8 * 128 + 16;
constexpr int64_t kWorkspaceBytes = (int64_t)kMaxCtas * 2 * kPartFloats * 4;
// dynamic shared memory: [8 warps][D / 16][32 lanes] 16-byte sums, their M and l, block records, prefix of steps
constexpr int kSmemSums = kWarps * 8 * 128 * 4;
constexpr int kSmemFixed = kSmemSums + 2 * kWarps * 8 * 4 + kWarps * 32 * 16;

struct AttnParams {
  const __nv_bfloat16* q;
  int64_t q_rs;
  __nv_bfloat16* out;
  int64_t o_rs;
  Pool k, v;
  Map m;
  const int* slot;
  const int* seqlen;
  float* parts;   // [CTAs][2][kPartFloats]: a CTA's first segment's and its last one's, where they are cut
  int B, Hq, G, hg, window;  // G: query heads of a KV head; hg: groups of eight of them
  int ctas;                  // of the attention kernel where segments are cut; 0: a CTA for each segment
  float scale_log2, cap_in, cap_out;  // cap_in = scale / softcap, cap_out = softcap * log2 e
  int* status;
};

__device__ __forceinline__ uint4 ld_stream16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ld_stream8(const void* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
// A constant that stays in a register: written as an immediate, it is moved into one again for each use.
__device__ __forceinline__ uint32_t in_register(uint32_t c) {
  uint32_t r;
  asm volatile("mov.u32 %0, %1;" : "=r"(r) : "r"(c));
  return r;
}
struct Consts {
  uint32_t high, minus;  // 0x64646464 (the high bytes of fp16 1024 + u), 0xe480e480 (-1152)
};
// fp16 pair of two biased codes: bytes (sel) of w become 1024 + u, minus 1152
template <int kSel>
__device__ __forceinline__ uint32_t half2_of(uint32_t w, const Consts& k) {
  uint32_t x = __byte_perm(w, k.high, kSel), r;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(k.minus));
  return r;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float ex2(float x) {  // 2^x to 2^-22, 0 below 2^-126
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}

// Blocks [first, first + count) that sequence b attends to.
__device__ __forceinline__ void blocks_of(const AttnParams& p, int b, int& len, int& lo, int& first, int& count) {
  const int slot = p.slot[b];
  len = p.seqlen[b];
  if (slot >= p.m.rows || len > (p.m.cols << p.m.shift)) atomicExch(p.status, kStatusKvRange);
  len = (unsigned)slot < (unsigned)p.m.rows ? min(max(len, 0), p.m.cols << p.m.shift) : 0;
  lo = p.window > 0 ? max(0, len - p.window) : 0;
  first = lo >> 4;
  count = len > 0 ? ((len + kBlock - 1) >> 4) - first : 0;
}

// s_pre[b]: steps (of kWarps blocks) before sequence b, for one KV head and group; returns their number. The host has
// checked that all of them fit 30 bits.
// kSides: of kThreads threads; each sequence's steps rounded up to a multiple of `unit`.
template <int kSides = 1>
__device__ __forceinline__ int prefix_steps(const AttnParams& p, int unit, int* s_pre, int* s_warp) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int carry = 0;
  for (int b0 = 0; b0 < p.B; b0 += kThreads * kSides) {
    int n = 0;
    if (b0 + tid < p.B) {
      int len, lo, first, count;
      blocks_of(p, b0 + tid, len, lo, first, count);
      n = (count + kWarps - 1) / kWarps;
      if (unit > 1) n = (n + unit - 1) / unit * unit;
    }
    int x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    int before = carry;
#pragma unroll
    for (int w = 0; w < kWarps * kSides; ++w) {
      if (w < warp) before += s_warp[w];
      carry += s_warp[w];
    }
    if (b0 + tid < p.B) s_pre[b0 + tid] = before + x - n;
    if (b0 + tid == p.B - 1) s_pre[p.B] = before + x;
    __syncthreads();
  }
  return carry;
}
// The ranges: `per` steps for each CTA; returns how many steps all segments take. Where segments are few beside the
// CTAs, each starts a range of its own (its steps count as a multiple of `per`): a CTA that ends one segment and
// begins another waits twice for page, scales and codes, 3 of 16 us for 16 x 2304.
template <int kSides = 1>
__device__ __forceinline__ int cut_ranges(const AttnParams& p, int V, int* s_pre, int* s_warp, int& per) {
  int total = prefix_steps<kSides>(p, 1, s_pre, s_warp) * V;
  const int segments = p.B * V;
  const bool own = 3 * segments <= p.ctas;
  const int ranges = own ? p.ctas - segments : p.ctas;
  per = max((total + ranges - 1) / ranges, kMinSteps);
  if (own) total = prefix_steps<kSides>(p, per, s_pre, s_warp) * V;
  return total;
}
// The last sequence that starts at or before step `at` of all.
__device__ __forceinline__ int sequence_at(const int* s_pre, int B, int V, int at) {
  int b = 0, hi = B;
  while (hi - b > 1) {
    const int mid = (b + hi) >> 1;
    if (s_pre[mid] * V <= at) b = mid; else hi = mid;
  }
  while (s_pre[b + 1] == s_pre[b] || s_pre[b + 1] * V <= at) ++b;  // (not one without a key)
  return b;
}
// The weight of a sum whose reference is m beside the largest reference: 0 for one of masked keys alone (l = 0).
__device__ __forceinline__ float factor(float m, float l, float top) {
  return m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : ex2(m - top);
}
// Dims d and d + 1 of heads h and h + 1 (where there are so many) of an output row.
__device__ __forceinline__ void write_out(__nv_bfloat16* y, int D, int h, int heads, const float4& a, float inv0, float inv1) {
  if (h < heads) *reinterpret_cast<uint32_t*>(y) = pack_bf16(a.x * inv0, a.z * inv0);
  if (h + 1 < heads) *reinterpret_cast<uint32_t*>(y + D) = pack_bf16(a.y * inv1, a.w * inv1);
}

template <int D, bool CAP>
__global__ void __launch_bounds__(kThreads, 2) attn_kernel(AttnParams p) {
  constexpr int kKs = D / 16;   // k steps of S, m tiles of O
  constexpr int kKl = D / 64;   // 16-byte loads of a key's row by a quad
  extern __shared__ __align__(16) uint8_t smem[];
  float* s_o = reinterpret_cast<float*>(smem);
  float* s_m = s_o + kWarps * 8 * 128;  // [warps][8]
  float* s_l = s_m + kWarps * 8;
  int4* s_rec = reinterpret_cast<int4*>(s_l + kWarps * 8) + (threadIdx.x >> 5) * 32;  // this warp's
  int* s_pre = reinterpret_cast<int*>(smem + kSmemFixed);  // [B + 1] steps before each sequence (one KV head)
  __shared__ int s_warp[kWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int r = lane >> 2, t = lane & 3;
  const int V = p.m.Hkv * p.hg;
  const Consts konst{in_register(0x64646464u), in_register(0xe480e480u)};
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");

  int at = 0, end = 1, per = 1, b = blockIdx.x / V;
  if (p.ctas > 0) {
    const int total = cut_ranges(p, V, s_pre, s_warp, per);
    at = blockIdx.x * per;
    end = min(total, at + per);
    if (at < end) b = sequence_at(s_pre, p.B, V, at);
  }
  while (at < end) {
    int len, lo, first, count, steps, v, st0, st1;
    if (p.ctas > 0) {
      while (s_pre[b + 1] == s_pre[b] || s_pre[b + 1] * V <= at) ++b;
      steps = s_pre[b + 1] - s_pre[b];
      const int off = at - s_pre[b] * V;
      v = off / steps;
      st0 = off - v * steps;
      st1 = min(steps, st0 + (end - at));
      blocks_of(p, b, len, lo, first, count);
    } else {
      v = blockIdx.x - b * V;
      blocks_of(p, b, len, lo, first, count);
      if (count == 0) break;
      steps = (count + kWarps - 1) / kWarps;
      st0 = 0;
      st1 = steps;
    }
    const int hk = v / p.hg, h0 = hk * p.G + (v - hk * p.hg) * 8;
    const int heads = min(8, p.G - (v - hk * p.hg) * 8);
    const int slot = p.slot[b];
    const int blk0 = first + st0 * kWarps + warp;              // this warp's blocks: blk0, blk0 + kWarps, ...
    const int blk1 = min(first + count, first + st1 * kWarps);
    const int n_blk = blk1 > blk0 ? (blk1 - blk0 + kWarps - 1) / kWarps : 0;

    uint4 kr[2 * kKl];   // rows r and r + 8
    uint4 vr[4];         // rows 2 t, 2 t + 1, 2 t + 8, 2 t + 9 (D = 64: the low half of each)
    const uint32_t koff = (uint32_t)(r * D + t * 16), voff = (uint32_t)(2 * t * D + r * (D / 8));
    auto block_base = [&](int page, int blk) {
      return code_offset(p.m, page, hk, (blk << 4) & ((1 << p.m.shift) - 1));
    };
    auto load_k = [&](int64_t base) {
      const uint8_t* c = p.k.codes + base + koff;
#pragma unroll
      for (int i = 0; i < kKl; ++i) {
        kr[i] = ld_stream16(c + i * 64);
        kr[kKl + i] = ld_stream16(c + 8 * D + i * 64);
      }
    };
    auto load_v = [&](int64_t base) {
      const uint8_t* c = p.v.codes + base + voff;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint8_t* a = c + ((i & 1) + (i >> 1) * 8) * D;
        if constexpr (D == 128) {
          vr[i] = ld_stream16(a);
        } else {
          const uint2 h = ld_stream8(a);
          vr[i].x = h.x;
          vr[i].y = h.y;
        }
      }
    };
    // Records of this warp's next 32 blocks: page, key scale, log2 and inverse of the value scale. The first block's
    // codes are asked for as soon as its page is known, beside the scales.
    int rpage;
    float rks, rvs;
    auto fetch_records = [&](int i0) {
      rpage = -1;
      const int pos = (blk0 + (i0 + lane) * kWarps) << 4;
      if (i0 + lane < n_blk) rpage = page_of(p.m, slot, pos, p.status);
      const int64_t base = block_base(max(__shfl_sync(0xffffffffu, rpage, 0), 0), blk0 + i0 * kWarps);
      load_k(base);
      load_v(base);
      rks = rvs = 0.f;
      if (rpage >= 0) {
        const int64_t so = scale_offset(p.m, rpage, hk, pos & ((1 << p.m.shift) - 1));
        rks = p.k.scale[so];
        rvs = p.v.scale[so];
      }
    };
    auto store_records = [&]() {
      const float vs = rvs < 6.2e-33f ? 6.2e-33f : rvs;  // (a NaN stays)
      __syncwarp();
      // an unusable page has weights of zero
      s_rec[lane] = make_int4(max(rpage, 0), __float_as_int(rks), __float_as_int(rpage >= 0 ? log2f(vs) : -INFINITY),
                              __float_as_int(rpage >= 0 ? 1.f / vs : 0.f));
      __syncwarp();
    };
    uint4 qraw[kKl][2];  // head r, dims 16 t .. of each 64
    {
      const __nv_bfloat16* qr = p.q + (int64_t)b * p.q_rs + (int64_t)(h0 + (r < heads ? r : 0)) * D + t * 16;
#pragma unroll
      for (int i = 0; i < kKl; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) qraw[i][j] = *reinterpret_cast<const uint4*>(qr + i * 64 + j * 8);
    }
    if (n_blk > 0) fetch_records(0);

    // q as the B operand
    uint32_t qb[kKs][2];
    float fac0, fac1;
    {
      const bool ok = r < heads;
      float f[kKs * 4];
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < kKl; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float e8[8];
          dec::unpack8(qraw[i][j], e8);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            f[i * 16 + j * 8 + e] = ok ? e8[e] : 0.f;
            top = max(top, __float_as_uint(f[i * 16 + j * 8 + e]) & 0x7fffffffu);
          }
        }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      int k = top == 0 || top >= 0x7f800000u ? 0 : 13 + 127 - (int)(top >> 23);  // largest |q| into [2^13, 2^14)
      k = min(k, 100);
      const float up = __uint_as_float((uint32_t)(127 + k) << 23), down = __uint_as_float((uint32_t)(127 - k) << 23);
#pragma unroll
      for (int i = 0; i < kKs; ++i) {
        qb[i][0] = pack_f16(f[4 * i] * up, f[4 * i + 1] * up);
        qb[i][1] = pack_f16(f[4 * i + 2] * up, f[4 * i + 3] * up);
      }
      const float fac = (CAP ? p.cap_in : p.scale_log2) * down;
      fac0 = __shfl_sync(0xffffffffu, fac, 8 * t);  // heads 2 t and 2 t + 1
      fac1 = __shfl_sync(0xffffffffu, fac, 8 * t + 4);
    }
    float o[kKs][4];
#pragma unroll
    for (int i = 0; i < kKs; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

    for (int i0 = 0; i0 < n_blk; i0 += 32) {
      const int nb = min(32, n_blk - i0);
      if (i0 > 0) fetch_records(i0);
      store_records();
      for (int i = 0; i < nb; ++i) {
        const int4 rec = s_rec[i];
        const int pos = (blk0 + (i0 + i) * kWarps) << 4;
        const int nx = min(i + 1, nb - 1);
        const int64_t base = block_base(s_rec[nx].x, blk0 + (i0 + nx) * kWarps);
        float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < kKl; ++j) {
          const uint32_t wl[4] = {kr[j].x, kr[j].y, kr[j].z, kr[j].w};
          const uint32_t wh[4] = {kr[kKl + j].x, kr[kKl + j].y, kr[kKl + j].z, kr[kKl + j].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t a[4] = {half2_of<0x4140>(wl[e], konst), half2_of<0x4140>(wh[e], konst), half2_of<0x4342>(wl[e], konst),
                                   half2_of<0x4342>(wh[e], konst)};
            mma_f16(c, a, qb[4 * j + e][0], qb[4 * j + e][1]);
          }
        }
        if (i + 1 < nb) load_k(base);  // in flight behind the rest of this block
        const float ks = __int_as_float(rec.y), lv = __int_as_float(rec.z), inv = __int_as_float(rec.w);
        const float f0 = fac0 * ks, f1 = fac1 * ks;
        float x[4] = {c[0] * f0, c[1] * f1, c[2] * f0, c[3] * f1};  // keys r, r, r + 8, r + 8; heads 2 t, 2 t + 1
        if constexpr (CAP) {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = p.cap_out * tanhf(x[e]);
        }
        if (pos < lo || pos + kBlock > len) {
          const bool a = pos + r >= lo && pos + r < len, bb = pos + r + 8 >= lo && pos + r + 8 < len;
          x[0] = a ? x[0] : -INFINITY;
          x[1] = a ? x[1] : -INFINITY;
          x[2] = bb ? x[2] : -INFINITY;
          x[3] = bb ? x[3] : -INFINITY;
        }
        // M covers x + log2 s_v; scales below 2^-60 count as 2^-60, so that l (the sum of 2^(x - M)) stays in range
        const float lm = fmaxf(lv, -60.f);
        float n0 = fmaxf(x[0], x[2]) + lm, n1 = fmaxf(x[1], x[3]) + lm;
        if (__any_sync(0xffffffffu, n0 > m0 + 4.f || n1 > m1 + 4.f)) {
#pragma unroll
          for (int s = 4; s < 32; s <<= 1) {
            n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, s));
            n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, s));
          }
          n0 = fmaxf(n0, m0);
          n1 = fmaxf(n1, m1);
          const float a0 = n0 == -INFINITY ? 1.f : ex2(m0 - n0), a1 = n1 == -INFINITY ? 1.f : ex2(m1 - n1);
          m0 = n0;
          m1 = n1;
          l0 *= a0;
          l1 *= a1;
#pragma unroll
          for (int k = 0; k < kKs; ++k) {
            o[k][0] *= a0;
            o[k][1] *= a1;
            o[k][2] *= a0;
            o[k][3] *= a1;
          }
        }
        const float d0 = lv + kWeightBits - (m0 == -INFINITY ? 0.f : m0);
        const float d1 = lv + kWeightBits - (m1 == -INFINITY ? 0.f : m1);
        const float w0 = ex2(x[0] + d0), w1 = ex2(x[1] + d1), w2 = ex2(x[2] + d0), w3 = ex2(x[3] + d1);
        l0 = fmaf(w0 + w2, inv, l0);
        l1 = fmaf(w1 + w3, inv, l1);
        const uint32_t pb0 = transpose8x8(pack_f16(w0, w1)), pb1 = transpose8x8(pack_f16(w2, w3));
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
          const uint32_t wa = j == 0 ? vr[0].x : j == 1 ? vr[0].y : j == 2 ? vr[0].z : vr[0].w;
          const uint32_t wb = j == 0 ? vr[1].x : j == 1 ? vr[1].y : j == 2 ? vr[1].z : vr[1].w;
          const uint32_t wc = j == 0 ? vr[2].x : j == 1 ? vr[2].y : j == 2 ? vr[2].z : vr[2].w;
          const uint32_t wd = j == 0 ? vr[3].x : j == 1 ? vr[3].y : j == 2 ? vr[3].z : vr[3].w;
#pragma unroll
          for (int e = 0; e < 2; ++e) {  // dims (D / 8) r + 4 j + 2 e (rows r) and the next (rows r + 8)
            const uint32_t ab = __byte_perm(wa, wb, e ? 0x7362 : 0x5140), cd = __byte_perm(wc, wd, e ? 0x7362 : 0x5140);
            const uint32_t a[4] = {half2_of<0x4140>(ab, konst), half2_of<0x4342>(ab, konst), half2_of<0x4140>(cd, konst), half2_of<0x4342>(cd, konst)};
            mma_f16(o[2 * j + e], a, pb0, pb1);
          }
        }
        if (i + 1 < nb) load_v(base);
      }
    }
    // Join the warps. o[k] is dims (D / 8) r + 2 k and the next (elements 0, 1 and 2, 3) of heads 2 t and 2 t + 1; sums
    // and parts keep that order, [k][lane] 16 bytes each, and warp k joins its slice.
#pragma unroll
    for (int s = 4; s < 32; s <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, s);
      l1 += __shfl_xor_sync(0xffffffffu, l1, s);
    }
    if (r == 0) {
      *reinterpret_cast<float2*>(s_m + warp * 8 + 2 * t) = make_float2(m0, m1);
      *reinterpret_cast<float2*>(s_l + warp * 8 + 2 * t) = make_float2(l0, l1);
    }
    float4* sums = reinterpret_cast<float4*>(s_o);
#pragma unroll
    for (int k = 0; k < kKs; ++k) sums[(warp * kKs + k) * 32 + lane] = make_float4(o[k][0], o[k][1], o[k][2], o[k][3]);
    __syncthreads();
    const bool whole = st0 == 0 && st1 == steps;
    if (warp < kKs) {
      float mm0 = -INFINITY, mm1 = -INFINITY, ll0 = 0.f, ll1 = 0.f;
      float2 mw[kWarps];
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        mw[w] = *reinterpret_cast<const float2*>(s_m + w * 8 + 2 * t);
        mm0 = fmaxf(mm0, mw[w].x);
        mm1 = fmaxf(mm1, mw[w].y);
      }
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 lw = *reinterpret_cast<const float2*>(s_l + w * 8 + 2 * t);
        const float f0 = factor(mw[w].x, lw.x, mm0), f1 = factor(mw[w].y, lw.y, mm1);
        const float4 x = sums[(w * kKs + warp) * 32 + lane];
        ll0 += f0 * lw.x;
        ll1 += f1 * lw.y;
        acc.x += f0 * x.x;
        acc.y += f1 * x.y;
        acc.z += f0 * x.z;
        acc.w += f1 * x.w;
      }
      const int h = 2 * t;
      if (whole) {
        write_out(p.out + (int64_t)b * p.o_rs + (int64_t)(h0 + h) * D + (D / 8) * r + 2 * warp, D, h, heads, acc,
                  ll0 == 0.f ? 0.f : 1.f / ll0, ll1 == 0.f ? 0.f : 1.f / ll1);
      } else {
        const bool begins = s_pre[b] * V + v * steps >= (int)blockIdx.x * per;  // the segment's first part
        float* part = p.parts + ((int64_t)blockIdx.x * 2 + begins) * kPartFloats;
        reinterpret_cast<float4*>(part)[warp * 32 + lane] = acc;
        if (warp == 0 && r == 0) {
          *reinterpret_cast<float2*>(part + 8 * D + h) = make_float2(mm0, mm1);
          *reinterpret_cast<float2*>(part + 8 * D + 8 + h) = make_float2(ll0, ll1);
        }
      }
    }
    if (p.ctas == 0) break;
    __syncthreads();  // the sums are free again
    at += st1 - st0;
  }
  // sequences without a key: zero rows
  const int nb = p.ctas > 0 ? p.B : (blockIdx.x % V == 0 ? blockIdx.x / V + 1 : 0);
  for (b = p.ctas > 0 ? blockIdx.x : blockIdx.x / V; b < nb; b += gridDim.x) {
    int len, lo, first, count;
    blocks_of(p, b, len, lo, first, count);
    if (count > 0) continue;
    for (int i = tid; i < p.Hq * D / 8; i += kThreads)
      *reinterpret_cast<uint4*>(p.out + (int64_t)b * p.o_rs + i * 8) = make_uint4(0, 0, 0, 0);
  }
}

// Joins the segment that the boundary between CTAs blockIdx.x and the next cuts, if it is that segment's first one:
// o = sum_i 2^(M_i - M) o_i / sum_i 2^(M_i - M) l_i, the parts in order. Latency is all there is: everything but the
// parts is known before the attention kernel ends (which has waited for the inputs to be complete before it let
// this one begin), and a batch of parts is in flight at once.
// kSides: halves of the parts, side by side
template <int D, int kSides>
__global__ void __launch_bounds__(kThreads * kSides) join_kernel(AttnParams p) {
  constexpr int kKs = D / 16;
  extern __shared__ __align__(16) uint8_t smem[];
  int* s_pre = reinterpret_cast<int*>(smem);
  __shared__ int s_warp[kWarps * kSides];
  __shared__ float4 s_acc[kSides == 2 ? kThreads : 1], s_ml[kSides == 2 ? kThreads : 1];
  const int tid = threadIdx.x, side = tid / kThreads, warp = tid / 32 % kWarps, lane = tid & 31, r = lane >> 2, t = lane & 3;
  const int V = p.m.Hkv * p.hg;
  int per;
  const int total = cut_ranges<kSides>(p, V, s_pre, s_warp, per);
  const int cut = ((int)blockIdx.x + 1) * per;
  bool mine = cut < total;
  int b = 0, v = 0, np = 0;
  if (mine) {
    b = sequence_at(s_pre, p.B, V, cut);
    const int steps = s_pre[b + 1] - s_pre[b];
    v = (cut - s_pre[b] * V) / steps;
    const int seg0 = s_pre[b] * V + v * steps;
    mine = seg0 < cut && seg0 / per == (int)blockIdx.x;
    np = (seg0 + steps - 1) / per - (int)blockIdx.x + 1;
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  if (!mine) return;
  // part i: this CTA's last segment, then each following CTA's first; a side takes its half of them
  const float* parts = p.parts + (int64_t)blockIdx.x * 2 * kPartFloats;
  const int half = (np + kSides - 1) / kSides, n0 = side * half, n1 = min(np, n0 + half);
  constexpr int kBatch = kSides == 2 ? 10 : 8;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = n0; i0 < n1 && warp < kKs; i0 += kBatch) {
    float2 pm[kBatch], pl[kBatch];
    float4 po[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int n = min(i0 + i, n1 - 1);
      const float* part = parts + (2 * n + (n == 0 ? 1 : 0)) * kPartFloats;
      pm[i] = *reinterpret_cast<const float2*>(part + 8 * D + 2 * t);
      pl[i] = *reinterpret_cast<const float2*>(part + 8 * D + 8 + 2 * t);
      po[i] = reinterpret_cast<const float4*>(part)[warp * 32 + lane];
    }
    float t0 = m0, t1 = m1;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      t0 = fmaxf(t0, pm[i].x);
      t1 = fmaxf(t1, pm[i].y);
    }
    const float a0 = factor(m0, l0, t0), a1 = factor(m1, l1, t1);
    l0 *= a0;
    l1 *= a1;
    acc.x *= a0;
    acc.y *= a1;
    acc.z *= a0;
    acc.w *= a1;
    m0 = t0;
    m1 = t1;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (i0 + i >= n1) break;
      const float f0 = factor(pm[i].x, pl[i].x, t0), f1 = factor(pm[i].y, pl[i].y, t1);
      l0 += f0 * pl[i].x;
      l1 += f1 * pl[i].y;
      acc.x += f0 * po[i].x;
      acc.y += f1 * po[i].y;
      acc.z += f0 * po[i].z;
      acc.w += f1 * po[i].w;
    }
  }
  if constexpr (kSides == 2) {
    if (side == 1) {
      s_acc[tid - kThreads] = acc;
      s_ml[tid - kThreads] = make_float4(m0, m1, l0, l1);
    }
    __syncthreads();
    if (side == 1) return;
    const float4 o = s_acc[tid], ml = s_ml[tid];
    const float t0 = fmaxf(m0, ml.x), t1 = fmaxf(m1, ml.y);
    const float a0 = factor(m0, l0, t0), a1 = factor(m1, l1, t1), c0 = factor(ml.x, ml.z, t0), c1 = factor(ml.y, ml.w, t1);
    l0 = l0 * a0 + ml.z * c0;
    l1 = l1 * a1 + ml.w * c1;
    acc = make_float4(acc.x * a0 + o.x * c0, acc.y * a1 + o.y * c1, acc.z * a0 + o.z * c0, acc.w * a1 + o.w * c1);
  }
  if (warp >= kKs) return;
  const int hk = v / p.hg, g0 = (v - hk * p.hg) * 8, h = 2 * t;
  write_out(p.out + (int64_t)b * p.o_rs + (int64_t)(hk * p.G + g0 + h) * D + (D / 8) * r + 2 * warp, D, h, min(8, p.G - g0),
            acc, l0 == 0.f ? 0.f : 1.f / l0, l1 == 0.f ? 0.f : 1.f / l1);
}

// ------------------------------------------------------------------ host
// Launch that may begin while the kernel before it in the stream drains; every kernel here waits for that one to
// complete (griddepcontrol.wait) before it touches memory, and only then lets its own successor begin.
template <typename P>
static void launch_pdl(void (*kernel)(P), dim3 grid, dim3 block, int smem, cudaStream_t st, const P& p) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  AETHER_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, p));
}
static void check_pool(const at::Tensor& codes, const at::Tensor& scale, const at::Tensor& table, const char* what) {
  TORCH_CHECK(codes.is_cuda() && codes.scalar_type() == at::kByte && codes.dim() == 4 && codes.is_contiguous(), what,
              ": codes are contiguous CUDA uint8 [pages, Hkv, page, D]");
  const int64_t P = codes.size(2), D = codes.size(3);
  TORCH_CHECK(P >= kBlock && (P & (P - 1)) == 0 && P <= 65536, what, ": page is a power of two of at least 16");
  TORCH_CHECK(D == 64 || D == 128, what, ": head_dim 64 or 128");
  TORCH_CHECK(codes.size(0) >= 1 && codes.size(0) < (int64_t(1) << 31) && codes.size(1) >= 1, what, ": pages and KV heads");
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
  // a warp for each head while there are few blocks; a CTA that walks over the heads once they fill the GPU
  const int64_t all = (Hq + 2 * Hkv + kAppendWarps - 1) / kAppendWarps;
  const int64_t spread = std::max<int64_t>(1, std::min<int64_t>(all, 8 * num_sms(current_device()) / units));
  const dim3 grid((unsigned)units, (unsigned)spread);
  auto st = at::cuda::getCurrentCUDAStream();
  launch_pdl(D == 128 ? append_kernel<128> : append_kernel<64>, grid, dim3(kAppendWarps * 32), 0, st, p);
}

at::Tensor gather_kv8(at::Tensor codes, at::Tensor scale, at::Tensor page_table, at::Tensor slot,
                      std::optional<at::Tensor> first, int64_t first0, int64_t n, std::optional<at::Tensor> into) {
  using namespace kv8;
  check_pool(codes, scale, page_table, "gather_kv8");
  TORCH_CHECK(slot.dim() == 1 && n >= 0, "gather_kv8: slot [B] and a length");
  const int64_t B = slot.size(0);
  const at::Tensor out = into && into->defined()
                             ? *into
                             : at::empty({B, n, codes.size(1), codes.size(3)}, codes.options().dtype(at::kBFloat16));
  TORCH_CHECK(out.device() == codes.device() && out.scalar_type() == at::kBFloat16 && out.dim() == 4 &&
                  out.is_contiguous() && out.size(0) == B && out.size(1) == n && out.size(2) == codes.size(1) && out.size(3) == codes.size(3) &&
                  reinterpret_cast<uintptr_t>(out.data_ptr()) % 16 == 0,
              "gather_kv8: out is contiguous bf16 [B, n, Hkv, D]");
  check_ints(slot, codes, B, "gather_kv8: slot [B]");
  const bool each = first && first->defined();
  if (each) check_ints(*first, codes, B, "gather_kv8: first [B]");
  TORCH_CHECK(n < (int64_t(1) << 31) && first0 >= 0 && first0 + n < (int64_t(1) << 31), "gather_kv8: positions");
  TORCH_CHECK(B <= 65535, "gather_kv8: at most 65535 sequences");
  if (out.numel() == 0) return out;
  c10::cuda::CUDAGuard g(codes.device());
  GatherParams p{};
  p.c = pool_of(codes, scale);
  p.m = make_map(codes, page_table);
  p.slot = slot.data_ptr<int>();
  p.first = each ? first->data_ptr<int>() : nullptr;
  p.first0 = (int)first0;
  p.n = (int)n;
  p.heads = std::min(p.m.Hkv, kGatherThreads / (p.m.D / 16));
  p.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  p.status = device_status_word();
  const int rows = kGatherThreads / (p.m.D / 16 * p.heads) * kGatherRows;
  launch_pdl(gather_kernel, dim3((unsigned)((n + rows - 1) / rows), (unsigned)B, (unsigned)((p.m.Hkv + p.heads - 1) / p.heads)),
             dim3(kGatherThreads), 0, at::cuda::getCurrentCUDAStream(), p);
  return out;
}

namespace kv8 {
// The most keys that a call can see of one sequence (with a window: that and the rest of its first block).
static int64_t most_keys(const at::Tensor& kc, const at::Tensor& page_table, int64_t window) {
  const int64_t keys = page_table.size(1) * kc.size(2);
  return window > 0 ? std::min<int64_t>(keys, window + kBlock) : keys;
}
}  // namespace kv8

// Kernels that kv8_decode_attention launches for these shapes.
int64_t kv8_decode_kernels(at::Tensor q, at::Tensor kc, at::Tensor page_table, int64_t window) {
  return q.size(0) == 0 ? 0 : kv8::most_keys(kc, page_table, window) <= kv8::kWholeKeys ? 1 : 2;
}

at::Tensor kv8_decode_attention(at::Tensor q, at::Tensor kc, at::Tensor ks, at::Tensor vc, at::Tensor vs,
                                at::Tensor page_table, at::Tensor slot, at::Tensor seqlen,
                                std::optional<at::Tensor> into, int64_t Hq, double scale, at::Tensor workspace,
                                int64_t window, double softcap) {
  using namespace kv8;
  check_pool(kc, ks, page_table, "kv8_decode_attention");
  check_pool(vc, vs, page_table, "kv8_decode_attention");
  check_same(kc, vc, "kv8_decode_attention");
  TORCH_CHECK(q.dim() == 2, "kv8_decode_attention: q is [B, >= Hq D]");
  const int64_t Hkv = kc.size(1), D = kc.size(3), B = q.size(0);
  TORCH_CHECK(Hq >= Hkv && Hq % Hkv == 0, "kv8_decode_attention: query heads are a multiple of the KV heads");
  const at::Tensor out = into && into->defined() ? *into : at::empty({B, Hq * D}, q.options());
  for (const at::Tensor* t : std::initializer_list<const at::Tensor*>{&q, &out})
    TORCH_CHECK(t->device() == kc.device() && t->dim() == 2 && t->scalar_type() == at::kBFloat16 && t->size(0) == B &&
                    t->size(1) >= Hq * D && t->stride(1) == 1 && t->stride(0) % 8 == 0 &&
                    reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0,
                "kv8_decode_attention: q and out are bf16 [B, >= Hq D], rows on 16-byte boundaries");
  check_ints(slot, kc, B, "kv8_decode_attention: slot [B]");
  check_ints(seqlen, kc, B, "kv8_decode_attention: seqlen [B]");
  TORCH_CHECK(window >= 0 && window < (int64_t(1) << 31) && softcap >= 0 && std::isfinite(softcap),
              "kv8_decode_attention: window and softcap");
  const int64_t G = Hq / Hkv, hg = (G + 7) / 8;
  TORCH_CHECK(B <= kMaxSeqs, "kv8_decode_attention: at most 8192 sequences");
  TORCH_CHECK(workspace.device() == kc.device() && workspace.scalar_type() == at::kByte && workspace.is_contiguous() &&
                  workspace.numel() >= kWorkspaceBytes && reinterpret_cast<uintptr_t>(workspace.data_ptr()) % 16 == 0,
              "kv8_decode_attention: workspace from kv8_workspace on the cache's device");
  if (B == 0) return out;
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
  p.parts = reinterpret_cast<float*>(workspace.data_ptr());
  p.B = (int)B;
  p.Hq = (int)Hq;
  p.G = (int)G;
  p.hg = (int)hg;
  p.window = (int)window;
  p.scale_log2 = (float)scale * kLog2e;
  if (softcap > 0) {
    p.cap_in = (float)(scale / softcap);
    p.cap_out = (float)softcap * kLog2e;
  }
  p.status = device_status_word();
  const int64_t keys = most_keys(kc, page_table, window);
  const int64_t most = B * Hkv * hg * std::max<int64_t>(1, (keys + kWarps * kBlock - 1) / (kWarps * kBlock));
  TORCH_CHECK(most < (int64_t(1) << 30), "kv8_decode_attention: the page table's positions times sequences and heads");
  // short tables: a CTA for each segment; else equal ranges for two CTAs an SM
  const int grid = keys <= kWholeKeys ? (int)(B * Hkv * hg)
                                      : (int)std::min<int64_t>(std::min(2 * num_sms(current_device()), kMaxCtas), most);
  p.ctas = keys <= kWholeKeys ? 0 : grid;
  const int smem = kSmemFixed + ((int)B + 1) * 4;
  auto st = at::cuda::getCurrentCUDAStream();
  // many parts a segment: two halves of them side by side (37 parts: 3 us less); else the smaller CTA, which finds room
  // as soon as one of the attention kernel's ends (64 x 4096: 3 us less)
  const int sides = p.ctas > 12 * B * Hkv * hg ? 2 : 1;
  auto launch = [&](auto kernel, auto join, bool* set) {
    const int dev = current_device();
    if (!set[dev]) {
      AETHER_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             kSmemFixed + (kMaxSeqs + 1) * 4));
      set[dev] = true;
    }
    launch_pdl(kernel, dim3(grid), dim3(kThreads), smem, st, p);
    if (p.ctas > 1) launch_pdl(join, dim3(grid - 1), dim3(kThreads * sides), ((int)B + 1) * 4, st, p);
  };
  static bool set[4][64] = {};
  if (D == 128 && softcap > 0)
    launch(attn_kernel<128, true>, sides == 2 ? join_kernel<128, 2> : join_kernel<128, 1>, set[0]);
  else if (D == 128)
    launch(attn_kernel<128, false>, sides == 2 ? join_kernel<128, 2> : join_kernel<128, 1>, set[1]);
  else if (softcap > 0)
    launch(attn_kernel<64, true>, sides == 2 ? join_kernel<64, 2> : join_kernel<64, 1>, set[2]);
  else
    launch(attn_kernel<64, false>, sides == 2 ? join_kernel<64, 2> : join_kernel<64, 1>, set[3]);
  return out;
}

}  // namespace aether
