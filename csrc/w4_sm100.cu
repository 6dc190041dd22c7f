// Products of more token rows than a few (17 to 64) with 4-bit weights, on the
// 5th-generation tensor cores (layout in w4.cuh):
//
//   y[m, n] = sum_g s[n, g] * sum_{k in group g} (c[n, k] - 8) * x[m, k]
//
// A CTA owns 128 weight rows -- the 128 lanes of TMEM -- and, in a cluster of S,
// the S-th part of the columns. Sixteen warps unpack: each streams the codes of 16
// rows and every other column tile through its own ring (16-byte asynchronous
// copies, 12 column tiles ahead, 10 for groups of 32) and writes exact bf16 codes
// straight into TMEM, where a lane's registers are already in the order that a
// 16 x 256-bit store wants, so the unpacked weights never pass through shared
// memory. (With eight warps the way of one column tile -- ring, unpacking, barrier,
// store, barrier, about 1000 cycles -- set the pace: 64 x 3584 -> 37888 took 38.8
// us.) One thread issues tcgen05.mma with the codes as the A operand from TMEM and
// the token rows (TMA, 128-byte swizzle, zeros past K and M) as B, a scale group at
// a time into one of four accumulators; eight warps read each accumulator back and
// add it, times the row's scale of that group (from a ring of their own, eight
// column tiles ahead), to fp32 sums in registers. Without a cluster a CTA walks
// over several row tiles and its pipelines run on from one to the next.
// Bound by the hand-offs: with neither unpacking, products nor scaling the same
// pipeline takes 27.6 of the 35.4 us of 64 x 3584 -> 37888 (SwiGLU, groups of 128:
// 493 TFLOP/s); groups of 64 and 32 hand over twice and four times as often, 47.7
// and 64 us. 32 rows of it 30.6 us; 64 x 3584 -> 3584 in 9.5 and, groups of 32, in
// 13.1 us. More accumulators, more stages of token rows or one warp that brings the
// scales for all did not help (30.6 -> 30.7, 35.4 -> 36.5 and 37.8 us).
#include <ATen/ATen.h>

#include "common.cuh"
#include "host_utils.h"
#include "w4.cuh"

namespace aether {
namespace w4 {
namespace tc {

constexpr int kUnpack = 16;                  // warps that unpack: a row tile and every other column tile each
constexpr int kScale = 8;                    // warps that scale: 32 rows and half of the tokens each
constexpr int kLoader = kUnpack + kScale;    // warp of the token rows
constexpr int kIssuer = kLoader + 1;         // first warp of the tensor cores
constexpr int kIssuers = 2;                  // take column tiles in turn: one spends as long on its waits as on its products
constexpr int kThreads = (kIssuer + kIssuers) * 32;
constexpr int ring(int groups) { return groups == 4 ? 6 : 7; }  // column tiles of an unpacking warp's ring
constexpr int kStages = 4;                   // column tiles of codes in TMEM (64 columns each) and of token rows
constexpr int kD = 4;                        // accumulators in TMEM, 64 columns each
constexpr int kFar = 3;                      // stages of a scaling warp's ring of scales, four column tiles each
constexpr int kLd = 128 + 4;                 // floats of one token's sums
constexpr int kColsA = kD * 64;              // first TMEM column of the codes (all 512 are in use)

// 16 lanes x 64 columns: a thread's registers 4 i .. are (lane l / 4, columns 8 i + 2 (l % 4) and the next), then lane
// l / 4 + 8
__device__ __forceinline__ void tmem_st_16x256b_x8(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x8.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}

struct Pipe {  // place and phase in a ring of N
  int at = 0;
  uint32_t phase = 0;
  template <int N>
  __device__ __forceinline__ void next() {
    if (++at == N) at = 0, phase ^= 1;
  }
};

// NP: token rows, padded; GS: k16 steps of a scale group (2, 4 or 8)
template <int NP, int GS>
__global__ void __launch_bounds__(kThreads, 1) linear_kernel(const __grid_constant__ CUtensorMap xmap, LinearParams p) {
  constexpr int kGroups = 8 / GS;  // of a column tile
  // The issuers take turns by groups where a column tile's groups use every accumulator, else by column tiles: each
  // always meets the same accumulators and stages, so that no phase of theirs passes it by.
  constexpr bool kByGroup = kGroups == kD;
  static_assert(kStages % kIssuers == 0 && kD % kIssuers == 0 && (kByGroup || kD % (kGroups * kIssuers) == 0), "turns");
  constexpr int kXBytes = 2 * NP * 128;
  constexpr int kRing = ring(kGroups);
  constexpr int kScaleBytes = 2 * 4 * kGroups * 32;  // of a ring's stage
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_x = smem;                                        // [kStages][2][NP][128 bytes]
  uint8_t* s_ring = s_x + kStages * kXBytes;                  // [kUnpack][kRing][1024]
  uint8_t* s_scales = s_ring + kUnpack * kRing * 1024;        // [kScale][kFar][2 row tiles][4][kGroups][32 bytes]
  float* s_sums = reinterpret_cast<float*>(s_scales + kScale * kFar * kScaleBytes);  // [M][kLd]
  // full: a column tile's codes are in TMEM and its token rows in shared memory; free: its products are done
  __shared__ __align__(8) uint64_t full[kStages], free_[kStages], d_full[kD], d_empty[kD], drain[kIssuers];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    s_abort = 0;
    for (int i = 0; i < kStages; ++i) mbar_init(full + i, 8 + 1), mbar_init(free_ + i, kByGroup ? kIssuers : 1);
    for (int i = 0; i < kD; ++i) mbar_init(d_full + i, 1), mbar_init(d_empty + i, kScale);
    for (int i = 0; i < kIssuers; ++i) mbar_init(drain + i, 1);
    fence_mbar_init();
    fence_async_smem();
  }
  const int S = p.S, rank = S > 1 ? (int)cluster_ctarank() : 0;
  const int c0 = rank * p.per, n_kt = max(0, min(p.w.kt, c0 + p.per) - c0);  // this CTA's column tiles
  const int tile0 = S > 1 ? blockIdx.x / S : blockIdx.x, tile_step = S > 1 ? p.tiles : gridDim.x;
  auto row_tile = [&](int tile, int rt) {  // packed row tile (past the last: the last, its sums are dropped)
    const int n0 = tile * p.outs;
    return min(p.swiglu && rt >= 4 ? ((p.n_out + n0) >> 4) + rt - 4 : (n0 >> 4) + rt, (p.w.N + 15) / 16 - 1);
  };
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (warp == kIssuer) {
    tmem_alloc(&s_tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // Not before TMEM is held: a kernel that begins now may take TMEM and then wait for this one to end.
  asm volatile("griddepcontrol.launch_dependents;");
  const uint32_t tmem = s_tmem;
  bool ok = true;
  auto wait = [&](uint64_t* bar, uint32_t phase) {
    if (ok && !mbar_wait(bar, phase, &s_abort)) {
      ok = false;
      s_abort = 1;
    }
    return ok;
  };

  if (warp < kUnpack) {
    // ------------------------------------------------------------ codes -> TMEM
    // a warp reaches the 32 lanes of its number modulo 4: row tiles 2 (warp % 4) and the next
    const int rt = 2 * (warp & 3) + ((warp >> 2) & 1), turn = warp >> 3;
    const Consts k{in_register(0x000f000fu), in_register(0x43004300u), in_register(0xc308c308u)};
    const uint32_t ring = smem_u32(s_ring) + warp * (kRing * 1024) + lane * 16;
    const uint32_t to = tmem + ((uint32_t)(rt * 16) << 16) + kColsA;
    const uint8_t* const q0 = reinterpret_cast<const uint8_t*>(p.w.q) + (int64_t)c0 * 1024 + lane * 16;
    // This warp's column tiles are every other one of all its row tiles' laid end to end.
    const int tiles = tile0 < p.tiles ? (p.tiles - tile0 + tile_step - 1) / tile_step : 0;
    int f_tile = tile0, f_first = turn, f_left = (n_kt - turn + 1) / 2, f_to = 0;
    const uint8_t* q = q0 + ((int64_t)row_tile(min(f_tile, p.tiles - 1), rt) * p.w.kt + f_first) * 1024;
    auto fetch = [&]() {
      while (f_left == 0 && f_tile < p.tiles) {  // the next row tile
        f_tile += tile_step;
        f_first ^= n_kt & 1;
        f_left = (n_kt - f_first + 1) / 2;
        if (f_tile < p.tiles) q = q0 + ((int64_t)row_tile(f_tile, rt) * p.w.kt + f_first) * 1024;
      }
      if (f_tile < p.tiles) {
        cp_async16(ring + f_to, q);
        cp_async16(ring + f_to + 512, q + 512);
        q += 2048;
        --f_left;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      if ((f_to += 1024) == kRing * 1024) f_to = 0;
    };
    for (int i = 0; i < kRing - 1; ++i) fetch();
    Pipe a;
    if (turn) a.next<kStages>();
    int at = 0;
    for (int left = (tiles * n_kt - turn + 1) / 2; left > 0; --left) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory");
      __syncwarp();  // the tile is there for every lane, and the one before it is free
      fetch();
      const uint4 va = lds128(ring + at), vb = lds128(ring + at + 512);
      if ((at += 1024) == kRing * 1024) at = 0;
      const uint32_t wa[4] = {va.x, va.y, va.z, va.w}, wb[4] = {vb.x, vb.y, vb.z, vb.w};
      uint32_t out[32];
#pragma unroll
      for (int s = 0; s < 8; s += 2) {
        out[4 * s + 0] = codes2<0>(wa[s >> 1], k);
        out[4 * s + 1] = codes2<1>(wa[s >> 1], k);
        out[4 * s + 2] = codes2<0>(wb[s >> 1], k);
        out[4 * s + 3] = codes2<1>(wb[s >> 1], k);
        out[4 * s + 4] = codes2<2>(wa[s >> 1], k);
        out[4 * s + 5] = codes2<3>(wa[s >> 1], k);
        out[4 * s + 6] = codes2<2>(wb[s >> 1], k);
        out[4 * s + 7] = codes2<3>(wb[s >> 1], k);
      }
      if (!wait(free_ + a.at, a.phase ^ 1)) break;
      __syncwarp();
      tc_fence_after();
      tmem_st_16x256b_x8(to + a.at * 64, out);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(full + a.at);
      a.next<kStages>();
      a.next<kStages>();
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp < kLoader) {
    // ------------------------------------------------------------ scales and sums
    constexpr int kTok = NP / 2;
    const int quad = warp & 3, row = quad * 32 + lane, tok0 = (warp - kUnpack) / 4 * kTok;
    const uint32_t from = tmem + ((uint32_t)(quad * 32) << 16) + tok0;
    const uint32_t ring = smem_u32(s_scales) + (warp - kUnpack) * (kFar * kScaleBytes);
    const uint32_t mine = ring + (lane >> 4) * (kScaleBytes / 2) + (row & 7) * 4 + ((row >> 3) & 1) * 2;
    int f_tile = tile0, f_i = 0, f_at = 0, at = 0;
    auto fetch = [&]() {  // the scales of four column tiles
      if (f_tile < p.tiles && n_kt > 0) {
#pragma unroll
        for (int e = lane; e < kScaleBytes / 16; e += 32) {
          const int piece = e % (8 * kGroups);
          if (f_i + piece / (2 * kGroups) < n_kt)
            cp_async16(ring + f_at * kScaleBytes + e * 16,
                       reinterpret_cast<const uint8_t*>(p.w.s) + piece * 16 +
                           ((int64_t)row_tile(f_tile, 2 * quad + e / (8 * kGroups)) * p.w.groups + (c0 + f_i) * kGroups) * 32);
        }
        if ((f_i += 4) >= n_kt) f_i = 0, f_tile += tile_step;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      if (++f_at == kFar) f_at = 0;
    };
    for (int i = 0; i < kFar - 1; ++i) fetch();
    Pipe d;
    for (int tile = tile0; tile < p.tiles; tile += tile_step) {  // (all of them: the eight warps meet at a barrier)
      float acc[kTok];
#pragma unroll
      for (int n = 0; n < kTok; ++n) acc[n] = 0.f;
      for (int i = 0; i < n_kt; ++i) {
        if ((i & 3) == 0) {
          if (i > 0 && ++at == kFar) at = 0;
          asm volatile("cp.async.wait_group %0;" ::"n"(kFar - 2) : "memory");
          __syncwarp();  // the scales are there for every lane, and those before them are free
          fetch();
        }
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          uint16_t h;
          asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(mine + at * kScaleBytes + ((i & 3) * kGroups + g) * 32) : "memory");
          const float s = __half2float(__ushort_as_half(h));
          wait(d_full + d.at, d.phase);
          __syncwarp();
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < kTok; c += 16) {
            uint32_t v[16];
            tmem_ld16(from + d.at * 64 + c, v);
            tmem_ld_wait();
            if (c + 16 == kTok) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(d_empty + d.at);
            }
#pragma unroll
            for (int n = 0; n < 16; ++n) acc[c + n] += s * __uint_as_float(v[n]);
          }
          d.next<kD>();
        }
      }
      if (++at == kFar) at = 0;
#pragma unroll
      for (int n = 0; n < kTok; ++n)
        if (tok0 + n < p.M) s_sums[(tok0 + n) * kLd + row] = acc[n];
      if (S == 1) {
        const int n0 = tile * p.outs;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        finish<1, kLd, 64>(p, s_sums, 1, 0, n0, p.swiglu ? (p.n_out + n0) & 15 : 0, tid - kUnpack * 32, kScale * 32);
        asm volatile("bar.sync 1, 256;" ::: "memory");  // the sums are free again
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp == kLoader) {
    // ------------------------------------------------------------ token rows
    Pipe x;
    for (int tile = tile0; tile < p.tiles && ok; tile += tile_step)
      for (int i = 0; i < n_kt; ++i) {
        if (!wait(free_ + x.at, x.phase ^ 1)) break;
        __syncwarp();
        if (lane == 0) {
          mbar_arrive_expect_tx(full + x.at, kXBytes);
          tma_load_2d(s_x + x.at * kXBytes, &xmap, full + x.at, (c0 + i) * 128, 0);
          tma_load_2d(s_x + x.at * kXBytes + kXBytes / 2, &xmap, full + x.at, (c0 + i) * 128 + 64, 0);
        }
        x.next<kStages>();
      }
  } else {
    // ------------------------------------------------------------ tensor cores
    // The whole warp goes through the waits and one lane issues: what the products need is the same in all lanes and
    // stays in uniform registers.
    constexpr uint32_t idesc = idesc_bf16_f32(128, NP, false, false);
    const int who = __shfl_sync(0xffffffffu, warp, 0) - kIssuer;
    const uint32_t d0 = __shfl_sync(0xffffffffu, tmem, 0);
    const uint64_t x0 = sdesc_sw128(smem_u32(s_x), 16, 1024);
    const bool lead = elect_one();
    auto ready = [&](uint64_t* bar, uint32_t phase) { return __all_sync(0xffffffffu, wait(bar, phase)); };
    Pipe a, d;
    int turn = 0;
    bool go = true;
    for (int tile = tile0; tile < p.tiles && go; tile += tile_step)
      for (int i = 0; i < n_kt && go; ++i) {
        if (kByGroup || turn == who) {
          go = ready(full + a.at, a.phase);
          const uint64_t b = x0 + a.at * (kXBytes >> 4);
          const uint32_t codes = d0 + kColsA + a.at * 64;
#pragma unroll
          for (int g = 0; g < kGroups; ++g) {
            if (kByGroup && g % kIssuers != who) {
              d.next<kD>();
              continue;
            }
            go = go && ready(d_empty + d.at, d.phase ^ 1);
            if (!go) break;
            tc_fence_after();
            if (lead) {
#pragma unroll
              for (int s = g * GS; s < (g + 1) * GS; ++s)
                umma_f16_ts(d0 + d.at * 64, codes + s * 8, b + (((s >> 2) * (kXBytes / 2) + (s & 3) * 32) >> 4), idesc,
                            s != g * GS ? 1u : 0u);
              umma_commit(d_full + d.at);
            }
            d.next<kD>();
          }
          if (!go) break;
          if (lead) umma_commit(free_ + a.at);
        } else {
#pragma unroll
          for (int g = 0; g < kGroups; ++g) d.next<kD>();
        }
        a.next<kStages>();
        if (++turn == kIssuers) turn = 0;
      }
    volatile int never = 0;
    if (lead) umma_commit(drain + who);
    mbar_wait(drain + who, 0, &never);
  }
  if (!ok) atomicExch(p.status, kStatusTimeoutMma);
  __syncwarp();
  __syncthreads();
  if (S > 1) {
    cluster_sync();
    const int n0 = tile0 * p.outs;
    finish<1, kLd, 64>(p, s_sums, S, rank, n0, p.swiglu ? (p.n_out + n0) & 15 : 0, tid, kThreads);
    cluster_sync();  // every CTA's sums are read before its shared memory goes
  }
  if (warp == kIssuer) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int NP, int GS>
static void launch(LinearParams& p, cudaStream_t st) {
  const int sms = num_sms(current_device());
  // SwiGLU: four gate tiles meet four up tiles, or three gate tiles four, where the up rows start inside a tile
  p.outs = !p.swiglu ? 128 : p.n_out % 16 == 0 ? 64 : 48;
  p.tiles = (p.n_out + p.outs - 1) / p.outs;
  constexpr int kFixed = kStages * 2 * NP * 128 + kUnpack * ring(8 / GS) * 1024 + kScale * kFar * (8 / GS) * 256 + 1024;
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[2] = {};
  static bool set[64] = {};
  static int clusters[64][9];  // clusters of so many CTAs that run at once
  const int dev = current_device();
  if (!set[dev]) {
    AETHER_CUDA_CHECK(cudaFuncSetAttribute(linear_kernel<NP, GS>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFixed + NP * kLd * 4));
    cfg.dynamicSmemBytes = kFixed + NP * kLd * 4;
    for (int c = 2; c <= 8; ++c) {
      cfg.gridDim = dim3((unsigned)(c * sms));
      at[0].id = cudaLaunchAttributeClusterDimension;
      at[0].val.clusterDim = {(unsigned)c, 1, 1};
      cfg.attrs = at;
      cfg.numAttrs = 1;
      AETHER_CUDA_CHECK(cudaOccupancyMaxActiveClusters(&clusters[dev][c], linear_kernel<NP, GS>, &cfg));
    }
    set[dev] = true;
  }
  // Parts of the columns: the fewest column tiles for an SM, and six for a CTA's start and end. Alone a CTA walks over
  // its row tiles; in clusters each round starts anew.
  p.S = 1;
  float best = 0.f;
  for (int c = 1; c <= 8 && c <= p.w.kt; ++c) {
    const int at_once = c == 1 ? sms : clusters[dev][c];
    if (at_once < 1) continue;
    const int rounds = (p.tiles + at_once - 1) / at_once;
    const float cost = c == 1 ? (float)rounds * p.w.kt + 6 : rounds * ((p.w.kt + c - 1) / c + 6.f) + 2.f;
    if (c == 1 || cost < best) best = cost, p.S = c;
  }
  p.per = (p.w.kt + p.S - 1) / p.S;
  const CUtensorMap xmap = make_tmap_2d_bf16(p.x, p.w.K, p.M, (uint64_t)p.xs * 2, 64, NP);
  cfg.gridDim = dim3((unsigned)(p.S > 1 ? p.tiles * p.S : std::min(p.tiles, sms)));
  cfg.dynamicSmemBytes = kFixed + p.M * kLd * 4;
  // the launch may begin while the kernel before it drains; this one waits for it before it touches memory
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim = {(unsigned)p.S, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = p.S > 1 ? 2 : 1;
  AETHER_CUDA_CHECK(cudaLaunchKernelEx(&cfg, linear_kernel<NP, GS>, xmap, p));
}

template <int NP>
static void launch_group(LinearParams& p, cudaStream_t st) {
  if (p.w.gshift == 7)
    launch<NP, 8>(p, st);
  else if (p.w.gshift == 6)
    launch<NP, 4>(p, st);
  else
    launch<NP, 2>(p, st);
}

}  // namespace tc
}  // namespace w4

void linear_w4_tc(w4::LinearParams& p, cudaStream_t st) {
  if (p.M <= 32)
    w4::tc::launch_group<32>(p, st);
  else
    w4::tc::launch_group<64>(p, st);
}

}  // namespace aether
