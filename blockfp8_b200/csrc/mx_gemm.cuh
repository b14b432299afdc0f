// MXFP4 GEMM on the block-scaled tensor cores (tcgen05.mma.kind::mxf4):
//
//   C[m, n] = sum_b 2^(ea[m, b] + eb[n, b]) sum_{k in block b of 32} A[m, k] B[n, k]
//
// The scales go into tensor memory beside the accumulator and the MMA applies
// them, so there is no promotion step between K blocks: a tile's whole K
// range accumulates in fp32 in TMEM, and the epilogue rounds once to bf16.
//
// The 128 MMA rows are weight rows and the BN columns are tokens (BN = 16 to
// 128), so a decode batch pays for no padding rows.  One CTA per (tile, K
// part): a cluster of up to 8 CTAs along K splits a tile's K range where there
// are few tiles, and its CTAs sum their parts over distributed shared memory,
// always in rank order -- no workspace, no counters, nothing shared between
// launches.  Two CTAs fit on an SM, so one's epilogue overlaps another's loop.
//
// Stages of K = 256: 128 bytes of codes per row (one 128-byte-swizzled TMA
// box for the weights, one for the tokens) and 512 bytes of scales per 128
// rows per 128 of K (bulk copies).  The epilogue's warps, which have nothing
// else to do in the loop, carry the scales on into TMEM: row r of a tile lies
// in lane r % 32, column r / 32, the same in each warp's 32 lanes, and the
// layout in memory is that order, so a warp needs one 16-byte load a lane and
// tile.  (tcgen05.cp would do the same on the tensor pipe, where a copy of
// 512 bytes costs about 170 clocks and does not overlap MMAs.)  One thread
// issues four MMAs of K = 64 a stage.
//
// QUANT (up to 16 tokens): the activations arrive as bf16 or fp16, and the same
// four warps quantize them into the stage's token tile and scales (the
// quantization kernel's arithmetic: identical codes), which saves its launch:
// at N = 6144, K = 4096 7.0 against 8.2 us for one token and 8.1 against 8.6 for
// 16.  Every weight tile quantizes again, so with 192 of them (N = 24576) the
// two kernels win from four tokens on (18.0 and 15.4 us for 16).
//
// Measured (device time in a graph, quantization included): one token, N = 6144,
// K = 4096 6.8 us for 13 MB of weights; 24 tokens, N = 4096, K = 12288 12 us for
// 27 MB.  What is left is launch, set-up and the sum over the cluster: the
// stream itself is 2 and 4 us.
//
// Warps: 0 TMA producer, 1 MMA issuer and TMEM owner, 2-5 scales, epilogue.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "mxfp4.cuh"
#include "ptx.cuh"

namespace bfp8 {

struct MxGemmParams {
  CUtensorMap map_w;  // weight codes [N, K / 2] bytes: [128 x 128] boxes, 128-byte swizzle
  CUtensorMap map_x;  // token codes [M, K / 2] bytes: [BN x 128] boxes; QUANT: 16-bit x [M, K]: [M x 256] boxes
  const uint8_t* sw;  // weight scales [ceil(N / 128), k_tiles, 512]
  const uint8_t* sx;  // token scales [ceil(M / 128), k_tiles, 512]
  __nv_bfloat16* c;   // [M, N], row stride ldc
  int64_t ldc;
  int M, N, K;
  int n_tiles;   // weight tiles (128 rows)
  int m_tiles;   // token tiles (BN)
  int k_tiles;   // 128-wide scale tiles
  int k_stages;  // 256-wide stages
  int splits;    // CTAs of a cluster along K
  int early;     // weights may be requested before griddepcontrol.wait
  int stages, stage_bytes, raw_bytes;  // ring; QUANT: bytes of a stage's 16-bit activations
  int half;                            // QUANT: x is fp16
};

enum MxWaitSite : uint32_t {
  kMxWaitEmpty = 33,
  kMxWaitFull = 34,
  kMxWaitDone = 35,
  kMxWaitDrain = 36,
  kMxWaitAcc = 37,
  kMxWaitScales = 38,
  kMxLayout = 39,
};

template <int BN_, bool QUANT_>
struct MxCfg {
  static constexpr int BN = BN_;
  static constexpr bool QUANT = QUANT_;
  static constexpr int THREADS = 192;
  static constexpr int W_BYTES = 128 * 128, X_BYTES = BN * 128, S_BYTES = 1024;  // per stage
  static constexpr int TILE_BYTES = W_BYTES + X_BYTES + 2 * S_BYTES;             // and QUANT's activations
  static constexpr int ACC_COLS = BN < 32 ? 32 : BN;
  // behind the accumulator every stage's scales: 2 K tiles x (4 weight + 4 token) columns
  static constexpr int TMEM_COLS = BN <= 64 ? 128 : 256;
  static constexpr int MAX_STAGES = (TMEM_COLS - ACC_COLS) / 16 < 6 ? (TMEM_COLS - ACC_COLS) / 16 : 6;
  static constexpr int SUM_BYTES = 128 * BN * 4;  // the tile's fp32 sums, over the ring
  static constexpr int BAR_BYTES = (3 * MAX_STAGES + 1) * 8 + 16;
};

template <class Cfg>
__global__ void __launch_bounds__(Cfg::THREADS) mx_gemm_kernel(const __grid_constant__ MxGemmParams p) {
  constexpr int BN = Cfg::BN;
  constexpr bool QUANT = Cfg::QUANT;
  const int S = p.stages;
  griddep_launch_dependents();
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);
  auto w_tile = [&](int s) { return base + uint32_t(s * p.stage_bytes); };
  auto x_tile = [&](int s) { return w_tile(s) + Cfg::W_BYTES; };
  auto sw_tile = [&](int s) { return x_tile(s) + Cfg::X_BYTES; };
  auto sx_tile = [&](int s) { return sw_tile(s) + Cfg::S_BYTES; };
  auto raw_tile = [&](int s) { return sx_tile(s) + Cfg::S_BYTES; };
  const uint32_t off_bars = uint32_t(max(S * p.stage_bytes, Cfg::SUM_BYTES)), bars = base + off_bars;
  auto full = [&](int s) { return bars + 8u * uint32_t(s); };
  auto empty = [&](int s) { return bars + 8u * uint32_t(S + s); };
  auto scaled = [&](int s) { return bars + 8u * uint32_t(2 * S + s); };  // the stage's scales are in TMEM
  const uint32_t done = bars + 8u * uint32_t(3 * S);
  uint32_t* misc = reinterpret_cast<uint32_t*>(smem + off_bars + 8 * (3 * S + 1));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(misc + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = p.splits > 1 ? int(cluster_rank()) : 0;
  const int tile = int(blockIdx.x) / p.splits;
  const int nt = tile % p.n_tiles, mt = tile / p.n_tiles;
  // this CTA's stages of the tile's K range
  const int s0 = p.k_stages * rank / p.splits, s1 = p.k_stages * (rank + 1) / p.splits;
  const int L = s1 - s0;

  if (warp == 0 && lane == 0) {
    for (int i = 0; i < 3 * S + 1; ++i) mbar_init(bars + 8u * uint32_t(i), i >= 2 * S && i < 3 * S ? 4u : 1u);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&p.map_w);
    tma_prefetch_desc(&p.map_x);
  }
  if (warp == 1) {
    tmem_alloc<1>(smem_u32(misc), Cfg::TMEM_COLS);
    tmem_relinquish<1>();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = misc[0];

  if (warp == 0) {
    if (lane == 0) {
      const uint64_t pol_w = p.m_tiles > 1 ? policy_evict_normal() : policy_evict_first();
      const uint64_t pol_x = policy_evict_last();
      auto kts = [&](int i) { return min(2, p.k_tiles - 2 * (s0 + i)); };  // scale tiles of stage i
      auto load_w = [&](int i) {
        const int s = i % S, k = s0 + i;
        mbar_arrive_expect_tx(full(s), QUANT ? uint32_t(Cfg::W_BYTES + 512 * kts(i) + p.raw_bytes)
                                             : uint32_t(Cfg::W_BYTES + Cfg::X_BYTES + 2 * 512 * kts(i)));
        tma_load_2d(w_tile(s), &p.map_w, k * 128, nt * 128, full(s), pol_w);
        bulk_load(sw_tile(s), p.sw + (int64_t(nt) * p.k_tiles + 2 * k) * 512, uint32_t(512 * kts(i)), full(s), pol_w);
      };
      auto load_x = [&](int i) {
        const int s = i % S, k = s0 + i;
        if constexpr (QUANT) {
          tma_load_2d(raw_tile(s), &p.map_x, k * 256, 0, full(s), pol_x);
          return;
        }
        tma_load_2d(x_tile(s), &p.map_x, k * 128, mt * BN, full(s), pol_x);
        bulk_load(sx_tile(s), p.sx + (int64_t(mt * BN / 128) * p.k_tiles + 2 * k) * 512, uint32_t(512 * kts(i)),
                  full(s), pol_x);
      };
      int pre = 0;
      if (p.early)
        for (; pre < S && pre < L; ++pre) load_w(pre);
      griddep_wait();
      for (int i = 0; i < pre; ++i) load_x(i);
      int issued = pre;
      for (int i = pre; i < L; ++i) {
        if (i >= S && !mbar_wait(empty(i % S), uint32_t(i / S - 1) & 1u, abort_flag, kMxWaitEmpty)) break;
        load_w(i);
        load_x(i);
        ++issued;
      }
      for (int i = issued - S > 0 ? issued - S : 0; i < issued; ++i)
        mbar_wait(full(i % S), uint32_t(i / S) & 1u, nullptr, kMxWaitDrain);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_mxf4(128, BN);
      const uint32_t scales = tmem + Cfg::ACC_COLS;
      for (int i = 0; i < L; ++i) {
        const int s = i % S;
        if (!mbar_wait(full(s), uint32_t(i / S) & 1u, abort_flag, kMxWaitFull)) break;
        if (!mbar_wait(scaled(s), uint32_t(i / S) & 1u, abort_flag, kMxWaitScales)) break;
        tc_fence_after();
        const int left = p.K - (s0 + i) * 256;  // values of K from this stage on
        const int steps = left >= 256 ? 4 : (left + 63) / 64;
        const uint32_t sf = scales + uint32_t(16 * s);  // [kt][4 weight + 4 token] columns
        const uint64_t a = smem_desc_k128_sw128(w_tile(s)), b = smem_desc_k128_sw128(x_tile(s));
#pragma unroll
        for (int k = 0; k < 4; ++k)  // K = 64 codes = 32 bytes = 2 descriptor units
          if (k < steps)
            mma_mxf4<1>(tmem, a + 2 * k, b + 2 * k, idesc | idesc_scale_half(k & 1), sf + uint32_t(8 * (k >> 1)),
                        sf + uint32_t(8 * (k >> 1) + 4), (i > 0 || k > 0) ? 1u : 0u);
        mma_commit<1>(empty(s));
      }
      mma_commit<1>(done);
      if (!mbar_wait(done, 0, nullptr, kMxWaitDone)) *abort_flag = 1;
    }
    __syncwarp();
  } else {
    // Scales of stage i: its TMEM columns were last read by the MMAs whose end
    // let the producer refill the stage.
    const uint32_t t_lane = tmem + (uint32_t(32 * (warp & 3)) << 16) + uint32_t(Cfg::ACC_COLS);
    bool ok = true;
    for (int i = 0; i < L; ++i) {
      const int s = i % S;
      // After a wait that gave up (the MMA thread's next one then does, too) a warp
      // still meets the others at the barrier below.
      if (ok) ok = mbar_wait_warp(full(s), uint32_t(i / S) & 1u, abort_flag, kMxWaitFull);
      if constexpr (QUANT) {
        // A thread takes 32 values of one token; tokens past M are zeros.
        for (int task = ok ? threadIdx.x - 64 : BN * 8; task < BN * 8; task += 128) {
          const int t = task >> 3, b = task & 7;
          uint32_t codes[4] = {0u, 0u, 0u, 0u}, byte = 0u;
          if (t < p.M) {
            float v[4][8];
            uint32_t m = 0u;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint4 u = ld_shared_v4(raw_tile(s) + uint32_t(t * 512 + b * 64 + j * 16));
              if (p.half) {
                const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
                  v[j][2 * e] = f.x, v[j][2 * e + 1] = f.y;
                }
              } else {
                bf16x8_to_float(u, v[j]);
              }
#pragma unroll
              for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(v[j][e]) & 0x7FFFFFFFu);
            }
            byte = mxfp4_scale_byte(m);
            const float inv = byte == 255u ? 0.f : e8m0_inverse(byte);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
#pragma unroll
              for (int e = 0; e < 8; ++e) v[j][e] = byte == 255u ? 0.f : v[j][e] * inv;
              codes[j] = e2m1x8(v[j]);
            }
          }
          st_shared_v4(x_tile(s) + uint32_t(t * 128 + ((b ^ (t & 7)) << 4)), codes[0], codes[1], codes[2], codes[3]);
          st_shared_u8(sx_tile(s) + uint32_t(512 * (b >> 2) + (t & 31) * 16 + (t >> 5) * 4 + (b & 3)), byte);
        }
        fence_proxy_async_smem();  // the MMAs read the codes through the async proxy
        named_bar_sync(1, 128);
      }
      if (!ok) continue;
      tc_fence_after();  // those MMAs' reads come before the stores below
      uint32_t r[16];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const uint4 w = ld_shared_v4(sw_tile(s) + uint32_t(512 * kt + 16 * lane));
        const uint4 x = ld_shared_v4(sx_tile(s) + uint32_t(512 * kt + 16 * lane));
        r[8 * kt] = w.x, r[8 * kt + 1] = w.y, r[8 * kt + 2] = w.z, r[8 * kt + 3] = w.w;
        r[8 * kt + 4] = x.x, r[8 * kt + 5] = x.y, r[8 * kt + 6] = x.z, r[8 * kt + 7] = x.w;
      }
      tmem_st16(t_lane + uint32_t(16 * s), r);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(scaled(s));
    }
  }
  // Every load has landed and every MMA is done: the ring is free.
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  // Sums to shared memory, [token][weight row] fp32: lanes hold consecutive rows.
  // After a wait that gave up they are NaN, and with them the tile (the other
  // CTAs of the cluster see it without a flag to fetch: 0.4 us of 7 for one token).
  float* sums = reinterpret_cast<float*>(smem);
  if (warp >= 2) {
    const int q = warp & 3;  // the TMEM lanes this warp may read
    const int row = 32 * q + lane;
    const uint32_t t_lane = tmem + (uint32_t(32 * q) << 16);
    const bool gave_up = *abort_flag;
#pragma unroll 1
    for (int c = 0; c < BN; c += 16) {
      float v[16];
      tmem_ld16(t_lane + uint32_t(c), v);
#pragma unroll
      for (int j = 0; j < 16; ++j) sums[(c + j) * 128 + row] = gave_up ? NAN : L > 0 ? v[j] : 0.f;
    }
  }
  tc_fence_before();
  if (p.splits > 1) cluster_sync();
  else __syncthreads();
  tc_fence_after();

  // This CTA's share of the tile's tokens: two weight rows a thread, the parts
  // in rank order.
  {
    griddep_wait();
    const int c0 = BN * rank / p.splits, c1 = BN * (rank + 1) / p.splits;
    for (int idx = threadIdx.x; idx < (c1 - c0) * 64; idx += Cfg::THREADS) {
      const int col = c0 + idx / 64, r2 = (idx & 63) * 2;
      const int m = mt * BN + col, n = nt * 128 + r2;
      if (m >= p.M || n >= p.N) continue;
      float2 v = make_float2(0.f, 0.f);
      if (p.splits == 1) {
        v = *reinterpret_cast<const float2*>(sums + col * 128 + r2);
      } else {
        for (int r = 0; r < p.splits; ++r) {
          const float2 w = ld_cluster_f32x2(map_shared_rank(base + uint32_t((col * 128 + r2) * 4), uint32_t(r)));
          v.x += w.x;
          v.y += w.y;
        }
      }
      *reinterpret_cast<__nv_bfloat162*>(p.c + int64_t(m) * p.ldc + n) = __floats2bfloat162_rn(v.x, v.y);
    }
  }
  // A CTA's sums stay until every CTA of the cluster has read them.
  if (p.splits > 1) cluster_sync();
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<1>(tmem, Cfg::TMEM_COLS);
  }
}

// ---- prompts: CTA pairs ------------------------------------------------------------
//
// A cluster of two CTAs computes 256 tokens x 256 weight rows with
// cta_group::2 MMAs (M = 256, N = 256, K = 64): each CTA holds 128 token rows
// and 128 of the weight rows, so a stage of K = 256 costs an SM 35 KB of
// shared-memory fill for 512 clocks of MMA (70 B per clock while MMAs run).  Token
// rows are the MMA rows: a thread of the epilogue holds one row's consecutive
// columns.
//
// TMEM: 256 accumulator columns and every stage's scales (each CTA its token
// rows', and all 256 weight rows').
// There is no room for a second accumulator, so the epilogue first empties it
// into registers as bf16 (eight warps, about 500 clocks of a tile's 8,192 at
// K = 4096), frees it, and stores while the next tile runs: through shared
// memory and TMA, 32 columns at a time.  Persistent, one pair on two SMs;
// tiles go to the pairs in groups of eight token tiles, so that concurrent
// tiles share operands in L2.
//
// Measured: 8192 x 24576 x 4096 in 322 us (5.1 PFLOP/s; the MMAs alone, without
// loads, 231 us).  Over the whole kernel the tensor pipe is busy for 0.66 of the
// clocks, an SM receives 44 B per clock and L2 is at 0.47 of its peak: what is left
// is loads that come late to the K loop and the epilogue between tiles.  One thread
// that issues everything is what held it back: 507 us with the scales' copies in
// the MMA thread, 340 with a thread of their own.  That is at 1.6 GHz or more;
// calls without a pause run into the power limit, at 1.45 to 1.5 GHz and 405 to
// 415 us, from a graph as from Python.
//
// Warps: TMA producers 0 (weights), 12 (tokens) and 2 (scales), 1 MMA issuer and
// TMEM owner, 3 issuer of the scales' copies into TMEM (1 and 3 the leader's),
// 4-11 epilogue.
struct MxPairParams {
  CUtensorMap map_x, map_w;    // codes [rows, K / 2] bytes: [128 x 128] boxes, 128-byte swizzle
  CUtensorMap map_sx, map_sw;  // scale tiles [row tiles, k_tiles * 512 bytes]: 1 and 2 x 1024 bytes
  CUtensorMap map_c;           // C [M, N]: [128 x 32] boxes, 64-byte swizzle
  int K, k_stages, m_tiles, n_tiles;  // tiles of 256
  int early;
};

struct MxPairCfg {
  static constexpr int STAGES = 6;
  static constexpr int THREADS = 416;
  static constexpr int TILE_BYTES = 128 * 128, S_BYTES = 1024;
  static constexpr int SCALE_COLS = 24;  // of a stage: [K tile][4 token, 8 weight columns]
  static constexpr int OUT_BYTES = 2 * 128 * 64;  // [column half][128 rows][32 bf16]
  static constexpr int TMEM_COLS = 512;
  // tiles stay 1024-byte aligned, scales behind all of them
  static constexpr int OFF_SCALES = STAGES * 2 * TILE_BYTES;
  static constexpr int OFF_OUT = OFF_SCALES + STAGES * 3 * S_BYTES;
  static_assert(OFF_OUT % 1024 == 0, "alignment");
  static_assert(256 + STAGES * SCALE_COLS <= TMEM_COLS, "TMEM");
  // barriers in front, in what aligning the tiles to 1024 bytes leaves
  static constexpr int BAR_BYTES = (4 * STAGES + 4) * 8 + 16;
  static constexpr int SMEM_BYTES = 1024 + OFF_OUT + OUT_BYTES;
};

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(MxPairCfg::THREADS, 1)
    mx_pair_kernel(const __grid_constant__ MxPairParams p) {
  using Cfg = MxPairCfg;
  constexpr int S = Cfg::STAGES;
  griddep_launch_dependents();
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + uint32_t(Cfg::BAR_BYTES) + 1023u) & ~1023u;
  auto x_tile = [&](int s) { return base + uint32_t(s * 2 * Cfg::TILE_BYTES); };
  auto w_tile = [&](int s) { return x_tile(s) + Cfg::TILE_BYTES; };
  auto sx_tile = [&](int s) { return base + uint32_t(Cfg::OFF_SCALES + s * 3 * Cfg::S_BYTES); };
  const uint32_t bars = raw;
  auto full = [&](int s) { return bars + 8u * uint32_t(s); };  // the leader's: both CTAs' copies
  auto empty = [&](int s) { return bars + 8u * uint32_t(S + s); };
  auto sfull = [&](int s) { return bars + 8u * uint32_t(2 * S + s); };   // the leader's: both CTAs' scales
  auto scaled = [&](int s) { return bars + 8u * uint32_t(3 * S + s); };  // the leader's: they are in TMEM
  const uint32_t leader_bars = map_shared_rank(bars, 0);
  const uint32_t acc_full = bars + 8u * uint32_t(4 * S), acc_empty = acc_full + 8u, done = acc_full + 16u;
  const uint32_t copied = acc_full + 24u;
  uint32_t* misc = reinterpret_cast<uint32_t*>(smem_raw + 8 * (4 * S + 4));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(misc + 1);

  if (base - raw > 1024u) {  // dynamic shared memory starts 1024-byte aligned: no static arrays here
    record_status((0x5Bull << 56) | (uint64_t(kMxLayout) << 32));
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const bool leader = rank == 0;
  const int pair = int(blockIdx.x >> 1), pairs = int(gridDim.x >> 1);
  const int tiles = p.m_tiles * p.n_tiles;
  auto place = [&](int t, int& mt, int& nt) {  // groups of 8 token tiles, token tiles first
    const int group = t / (8 * p.n_tiles), rest = t - group * 8 * p.n_tiles;
    const int rows = min(8, p.m_tiles - group * 8);
    nt = rest / rows;
    mt = group * 8 + rest - nt * rows;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
      mbar_init(sfull(s), 1);
      mbar_init(scaled(s), 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, 16);  // the eight epilogue warps of both CTAs
    mbar_init(done, 1);
    mbar_init(copied, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&p.map_x);
    tma_prefetch_desc(&p.map_w);
    tma_prefetch_desc(&p.map_c);
  }
  if (warp == 1) {
    tmem_alloc<2>(smem_u32(misc), Cfg::TMEM_COLS);
    tmem_relinquish<2>();
  }
  tc_fence_before();
  cluster_sync();  // the peer's barriers are initialised before any remote use
  tc_fence_after();
  const uint32_t tmem = misc[0];

  if (warp == 0 || warp == 12) {
    // Weights (warp 0) and tokens (warp 12): a copy and the wait before it cost
    // a thread about 250 clocks.
    if (lane == 0) {
      const bool weights = warp == 0;
      const uint64_t pol = policy_evict_normal();
      auto load = [&](int s, int k, int mt, int nt) {
        const uint32_t bar = leader_bars + 8u * uint32_t(s);
        if (weights) {
          if (leader) mbar_arrive_expect_tx(full(s), 4u * Cfg::TILE_BYTES);
          tma_load_2d_pair(w_tile(s), &p.map_w, k * 128, nt * 256 + int(rank) * 128, bar, pol);
        } else {
          tma_load_2d_pair(x_tile(s), &p.map_x, k * 128, mt * 256 + int(rank) * 128, bar, pol);
        }
      };
      int pre = 0;
      if (weights && p.early && pair < tiles) {
        int mt, nt;
        place(pair, mt, nt);
        for (; pre < S && pre < p.k_stages; ++pre) load(pre, pre, mt, nt);
      }
      griddep_wait();
      int i = 0;
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += pairs) {
        int mt, nt;
        place(t, mt, nt);
        for (int k = 0; k < p.k_stages; ++k, ++i) {
          const int s = i % S;
          if (i >= S && !(ok = mbar_wait(empty(s), uint32_t(i / S - 1) & 1u, abort_flag, kMxWaitEmpty))) break;
          if (i >= pre) load(s, k, mt, nt);
        }
      }
      // The leader's MMAs read what was loaded last; every copy has landed once
      // they are done.  (A CTA stays until its peer gets here, so that no
      // commit arrives on a barrier that is gone.)  After a wait that gave up the
      // leader waits for the copies themselves.
      for (int k = i > S ? i - S : 0; k < i; ++k) {
        if (ok) ok = mbar_wait(empty(k % S), uint32_t(k / S) & 1u, abort_flag, kMxWaitDrain);
        if (!ok && leader) mbar_wait(full(k % S), uint32_t(k / S) & 1u, nullptr, kMxWaitDrain);
      }
    }
    __syncwarp();
  } else if (warp == 2) {
    if (lane == 0) {
      const uint64_t pol = policy_evict_normal();
      griddep_wait();
      int i = 0;
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += pairs) {
        int mt, nt;
        place(t, mt, nt);
        for (int k = 0; k < p.k_stages; ++k, ++i) {
          const int s = i % S;
          if (i >= S && !(ok = mbar_wait(empty(s), uint32_t(i / S - 1) & 1u, abort_flag, kMxWaitEmpty))) break;
          if (leader) mbar_arrive_expect_tx(sfull(s), 6u * Cfg::S_BYTES);
          const uint32_t bar = leader_bars + 8u * uint32_t(2 * S + s);
          tma_load_2d_pair(sx_tile(s), &p.map_sx, k * 256, mt * 2 + int(rank), bar, pol);
          tma_load_2d_pair(sx_tile(s) + Cfg::S_BYTES, &p.map_sw, k * 256, nt * 2, bar, pol);
        }
      }
      if (leader)
        for (int k = i > S ? i - S : 0; k < i; ++k) mbar_wait(sfull(k % S), uint32_t(k / S) & 1u, nullptr, kMxWaitDrain);
    }
    __syncwarp();
  } else if (warp == 3) {
    // Scales into TMEM, by a thread of their own: issuing six copies takes one
    // thread about 500 clocks a stage, as long as the MMAs run.  A stage's
    // columns were last read by the MMAs whose end let it be refilled.
    if (leader && lane == 0) {
      int i = 0;
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += pairs) {
        for (int k = 0; k < p.k_stages; ++k, ++i) {
          const int s = i % S;
          if (!(ok = mbar_wait(sfull(s), uint32_t(i / S) & 1u, abort_flag, kMxWaitFull))) break;
          if (!(ok = mbar_wait(full(s), uint32_t(i / S) & 1u, abort_flag, kMxWaitFull))) break;  // for the MMAs
          tc_fence_after();
          const uint32_t sf = tmem + 256u + uint32_t(Cfg::SCALE_COLS * s);  // [kt][4 token, 8 weight columns]
          const uint64_t desc = smem_desc_scales(sx_tile(s));
#pragma unroll
          for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int h = 0; h < 3; ++h)  // token rows, weight rows 0-127, 128-255
              tmem_cp_scales_pair(sf + uint32_t(12 * kt + 4 * h), desc + uint64_t((h * Cfg::S_BYTES + 512 * kt) >> 4));
          mma_commit<2>(scaled(s));
        }
      }
      mma_commit<2>(copied);
      mbar_wait(copied, 0, nullptr, kMxWaitDone);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (leader && lane == 0) {
      constexpr uint32_t idesc = idesc_mxf4(256, 256);
      const uint64_t desc_a = smem_desc_k128_sw128(x_tile(0)), desc_b = smem_desc_k128_sw128(w_tile(0));
      int n = 0, s = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += pairs, ++n) {
        if (n > 0 && !mbar_wait(acc_empty, uint32_t(n - 1) & 1u, abort_flag, kMxWaitAcc)) break;
        for (int left = p.K, first = 1; left > 0; left -= 256, first = 0) {
          // (scaled: the codes have landed, too)
          if (!(ok = mbar_wait(scaled(s), phase, abort_flag, kMxWaitScales))) break;
          tc_fence_after();
          const uint32_t sf = tmem + 256u + uint32_t(Cfg::SCALE_COLS * s);
          const uint64_t a = desc_a + uint64_t(s * (2 * Cfg::TILE_BYTES >> 4)), b = desc_b + uint64_t(s * (2 * Cfg::TILE_BYTES >> 4));
          auto mma = [&](int j) {  // K = 64 codes
            mma_mxf4<2>(tmem, a + 2 * j, b + 2 * j, idesc | idesc_scale_half(j & 1), sf + uint32_t(12 * (j >> 1)),
                        sf + uint32_t(12 * (j >> 1) + 4), j > 0 || !first);
          };
          if (left >= 256) {
#pragma unroll
            for (int j = 0; j < 4; ++j) mma(j);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (64 * j < left) mma(j);
          }
          mma_commit_pair(empty(s));
          if (++s == S) s = 0, phase ^= 1u;
        }
        if (ok) mma_commit_pair(acc_full);  // a part of a sum is not stored, not by the peer either
      }
      mma_commit<2>(done);
      mbar_wait(done, 0, nullptr, kMxWaitDone);
    }
    __syncwarp();
  } else {
    griddep_wait();  // C
    const int q = warp & 3, half = (warp - 4) >> 2;  // lanes 32 q .., columns 128 half ..
    const int row = 32 * q + lane;
    const uint32_t t_lane = tmem + (uint32_t(32 * q) << 16) + uint32_t(128 * half);
    const uint32_t out = base + uint32_t(Cfg::OFF_OUT + half * 128 * 64);
    const uint32_t empty_bar = leader_bars + 8u * uint32_t(4 * S + 1);
    int n = 0;
    bool ok = true;
    for (int t = pair; t < tiles; t += pairs, ++n) {
      // After a wait that gave up nothing is stored (the abort flag is up), but a
      // warp still meets the others at the barriers below.
      if (ok) ok = mbar_wait_warp(acc_full, uint32_t(n) & 1u, abort_flag, kMxWaitAcc);
      tc_fence_after();
      uint32_t packed[64];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float v[32];
        tmem_ld32(t_lane + uint32_t(32 * c), v);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
          packed[c * 16 + j] = *reinterpret_cast<const uint32_t*>(&b);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0 && ok) mbar_arrive_cluster(empty_bar);  // the next tile's MMAs may start
      int mt, nt;
      place(t, mt, nt);
#pragma unroll
      for (int c = 0; c < 4; ++c) {  // 32 columns: 64 bytes a row, in the 64-byte swizzle
        // the store that read this buffer last is done
        if ((warp & 3) == 0 && lane == 0) bulk_wait_read0();
        named_bar_sync(1 + half, 128);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          st_shared_v4(out + uint32_t(row * 64 + ((j ^ ((row >> 1) & 3)) << 4)), packed[c * 16 + 4 * j],
                       packed[c * 16 + 4 * j + 1], packed[c * 16 + 4 * j + 2], packed[c * 16 + 4 * j + 3]);
        fence_proxy_async_smem();
        named_bar_sync(1 + half, 128);
        const int col = nt * 256 + half * 128 + c * 32;
        if ((warp & 3) == 0 && lane == 0 && !*abort_flag) {
          tma_store_2d(&p.map_c, col, mt * 256 + int(rank) * 128, out);
          bulk_commit();
        }
      }
    }
    if ((warp & 3) == 0 && lane == 0) bulk_wait0();
  }
  tc_fence_before();
  // The leader's MMAs and both CTAs' remote arrivals are over before either
  // frees TMEM or exits.
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<2>(tmem, Cfg::TMEM_COLS);
  }
}

}  // namespace bfp8
