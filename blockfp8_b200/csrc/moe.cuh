// A mixture-of-experts layer for a few tokens, in two kernels:
//
//   moe_kernel<GATE>  ids, p = router(logits)            (every CTA, from the logits)
//                     h[t, j] = silu(W1[e] x[t]) * (W3[e] x[t]),  e = ids[t, j]
//   moe_kernel<DOWN>  z[t, j] = W2[e] h[t, j],  y[t] = sum_j p[t, j] z[t, j]
//
// Expert weights are block FP8 (e4m3, one fp32 scale per 128 x 128) or MXFP4
// (e2m1, one power-of-two scale per 32); activations are not quantized.  At
// these sizes the weights of the chosen experts are the only traffic that
// counts, so the kernels are built to stream them:
//
// - Work: (token, expert) pairs are grouped by expert into chunks of up to
//   8 NT tokens, in token order.  A unit is 16 weight rows (GATE: 8 gate rows
//   and the 8 up rows beside them, so that one thread ends with both) of one
//   chunk over a whole K range, and CTA b of G takes units [U b / G, U (b+1) / G).
//   16 rows keep the last wave short (one token, 8 experts of I = 768: 768
//   units over 148 CTAs) and need no sums across CTAs.
// - A ring of shared-memory stages, 16 rows x up to 1 KB each, filled by one
//   warp with one bulk copy per row; it runs across units, so the memory
//   system sees one stream per SM.  Rows are padded by 16 bytes, which makes
//   ldmatrix conflict-free.
// - Eight consumer warps take the 128-wide K blocks of a stage in turn:
//   ldmatrix, codes to f16 (exact: cvt, 128 codes per clock and SM), mma.sync
//   m16n8k16 with fp32 accumulation, then the block's scales in fp32.  The
//   legacy MMA is no bound here (one 8-token MMA per 256 weights is 0.09 of
//   its 0.5 per clock at the HBM rate) and takes the dequantized registers
//   directly; tcgen05 would need them written back to shared memory.
// - Activations are held in shared memory as f16 in MMA fragment order with
//   one power-of-two scale per token and 128 values, which puts the largest
//   at 2^14: bf16 values are exact down to 2^-28 of it, and h (fp32) keeps 11
//   bits, 8 times finer than a bf16 h would.
// - A last warp finishes units: it adds the eight warps' sums in warp order
//   and, DOWN, the last unit to arrive at an output row tile (a counter)
//   adds its pairs in j order.  No result depends on the order of arrival.
//
// Warps: 0-7 consumers, 8 producer, 9 finisher.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "mxfp4.cuh"
#include "producers.cuh"
#include "ptx.cuh"

namespace bfp8 {

constexpr int kMoeMaxTokens = 64;
constexpr int kMoeMaxTopK = 16;
constexpr int kMoeMaxExperts = 512;
constexpr int kMoeConsumers = 8;
constexpr int kMoeThreads = 32 * (kMoeConsumers + 2);
constexpr int kMoeBatch = 16;  // units whose arrival DOWN counts together

struct MoeParams {
  const void* x;  // [T, H] bf16 or fp16
  int64_t ldx;
  // routing: logits [T, E], or ids and weights [T, top_k]
  const void* logits;
  int64_t ld_logits;
  int logits_type;  // 0 fp32, 1 bf16, 2 fp16
  const int* ids;
  const float* weights;
  int renormalize;
  const uint8_t* w;          // this kernel's weights
  int64_t w_expert, w_row;   // bytes
  const void* ws;            // their scales: fp32 [E, rb, kb], or E8M0 tiles [E, rb, kb, 32, 16]
  int rb, kb;
  float* h;       // [T top_k, I]
  float* z;       // [T top_k, segments, H]
  int* counters;  // [H / 16], zeroed by GATE
  void* y;        // [T, H]
  int64_t ldy;
  int T, H, I, E, top_k;
  int segments, seg_len;  // K ranges of DOWN (multiples of 128)
  int stages, stage_row;  // ring: stages, bytes of a row per stage
  uint32_t off_b, off_ts, off_red, off_route, off_bars;  // shared memory
};

enum MoeWaitSite : uint32_t {
  kMoeWaitEmpty = 49,
  kMoeWaitFull = 50,
  kMoeWaitRedEmpty = 51,
  kMoeWaitRedFull = 52,
  kMoeWaitDrain = 53,
};

struct MoeRoute {  // shared-memory tables, P = T top_k pairs
  short* expert;        // [P] -1: none
  float* weight;        // [P]
  short* list;          // [P] pairs by expert, then by index
  short* chunk_expert;  // [P]
  short* chunk_first;   // [P] into list
  short* chunk_count;   // [P]
  int* totals;          // [1] chunks
};
constexpr int moe_route_bytes(int P) { return P * (2 + 4 + 2 + 2 + 2 + 2) + 16; }

__device__ __forceinline__ MoeRoute moe_route_at(uint8_t* base, int P) {
  MoeRoute r;
  r.totals = reinterpret_cast<int*>(base);
  r.weight = reinterpret_cast<float*>(base + 16);
  r.expert = reinterpret_cast<short*>(base + 16 + 4 * P);
  r.list = r.expert + P;
  r.chunk_expert = r.list + P;
  r.chunk_first = r.chunk_expert + P;
  r.chunk_count = r.chunk_first + P;
  return r;
}

// Larger floats get larger keys; NaN and -inf get 0 (never chosen); -0 = +0.
__device__ __forceinline__ uint32_t moe_key(float v) {
  if (!(v > -INFINITY)) return 0u;
  const uint32_t u = __float_as_uint(v + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float moe_key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

// The router and the chunk tables, by all threads of the CTA.  scratch: room
// for E * ceil(P / 32) words and E ints.
__device__ void moe_route(const MoeParams& p, const MoeRoute& r, uint32_t* scratch, int chunk_cap) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int P = p.T * p.top_k, words = (P + 31) / 32;
  uint32_t* masks = scratch;                               // [E][words]
  int* offsets = reinterpret_cast<int*>(scratch + p.E * words);  // [E]: (first pair << 16) | first chunk
  for (int i = tid; i < p.E * words; i += kMoeThreads) masks[i] = 0u;
  if (p.logits) {
    for (int t = warp; t < p.T; t += kMoeThreads / 32) {
      uint32_t key[kMoeMaxExperts / 32];
#pragma unroll
      for (int i = 0; i < kMoeMaxExperts / 32; ++i) {
        key[i] = 0u;
        const int e = i * 32 + lane;
        if (e < p.E) {
          const int64_t at = int64_t(t) * p.ld_logits + e;
          float v;
          if (p.logits_type == 0) v = static_cast<const float*>(p.logits)[at];
          else if (p.logits_type == 1) v = __bfloat162float(static_cast<const __nv_bfloat16*>(p.logits)[at]);
          else v = __half2float(static_cast<const __half*>(p.logits)[at]);
          key[i] = moe_key(v);
        }
      }
      float all = 0.f, top = 0.f, chosen = 0.f;
      float mine = 0.f;  // lane j keeps exp(l_j - l_0) of the j-th choice
      for (int j = 0; j < p.top_k; ++j) {
        uint32_t best = 0u;
#pragma unroll
        for (int i = 0; i < kMoeMaxExperts / 32; ++i) best = max(best, key[i]);
        best = __reduce_max_sync(~0u, best);
        int id = -1;
        float ex = 0.f;
        if (best) {
          uint32_t at = ~0u;
#pragma unroll
          for (int i = kMoeMaxExperts / 32 - 1; i >= 0; --i)
            if (key[i] == best) at = uint32_t(i * 32 + lane);
          id = int(__reduce_min_sync(~0u, at));
          const float v = moe_key_value(best);
          if (j == 0) {
            top = v;
            if (!p.renormalize) {
#pragma unroll
              for (int i = 0; i < kMoeMaxExperts / 32; ++i)
                if (key[i]) all += expf(moe_key_value(key[i]) - top);
#pragma unroll
              for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(~0u, all, o);
            }
          }
          ex = expf(v - top);
          chosen += ex;
#pragma unroll
          for (int i = 0; i < kMoeMaxExperts / 32; ++i)
            if (id == i * 32 + lane) key[i] = 0u;
        }
        if (lane == 0) r.expert[t * p.top_k + j] = short(id);
        if (lane == j) mine = ex;
      }
      if (lane < p.top_k) r.weight[t * p.top_k + lane] = mine / (p.renormalize ? chosen : all);
    }
  } else {
    for (int i = tid; i < P; i += kMoeThreads) {
      const int e = p.ids[i];
      r.expert[i] = short(e >= 0 && e < p.E ? e : -1);
      r.weight[i] = p.weights[i];
    }
  }
  __syncthreads();
  for (int i = tid; i < P; i += kMoeThreads) {
    const int e = r.expert[i];
    if (e >= 0) atomicOr(masks + e * words + i / 32, 1u << (i & 31));
  }
  __syncthreads();
  if (warp == 0) {  // first pair and first chunk of every expert
    const int per = (p.E + 31) / 32;
    int pairs = 0, chunks = 0;
    for (int k = 0; k < per; ++k) {
      const int e = lane * per + k;
      if (e >= p.E) break;
      int n = 0;
      for (int w = 0; w < words; ++w) n += __popc(masks[e * words + w]);
      pairs += n;
      chunks += (n + chunk_cap - 1) / chunk_cap;
    }
    int pi = pairs, ci = chunks;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(~0u, pi, o), b = __shfl_up_sync(~0u, ci, o);
      if (lane >= o) pi += a, ci += b;
    }
    if (lane == 31) r.totals[0] = ci;
    pi -= pairs;
    ci -= chunks;
    for (int k = 0; k < per; ++k) {
      const int e = lane * per + k;
      if (e >= p.E) break;
      int n = 0;
      for (int w = 0; w < words; ++w) n += __popc(masks[e * words + w]);
      offsets[e] = (pi << 16) | ci;
      pi += n;
      ci += (n + chunk_cap - 1) / chunk_cap;
    }
  }
  __syncthreads();
  for (int e = tid; e < p.E; e += kMoeThreads) {
    const int first = offsets[e] >> 16, chunk = offsets[e] & 0xFFFF;
    int n = 0;
    for (int w = 0; w < words; ++w) {
      uint32_t m = masks[e * words + w];
      while (m) {
        r.list[first + n++] = short(w * 32 + __ffs(m) - 1);
        m &= m - 1;
      }
    }
    for (int c = 0; c * chunk_cap < n; ++c) {
      r.chunk_expert[chunk + c] = short(e);
      r.chunk_first[chunk + c] = short(first + c * chunk_cap);
      r.chunk_count[chunk + c] = short(min(chunk_cap, n - c * chunk_cap));
    }
  }
  fence_proxy_async_smem();  // the ring's copies overwrite the scratch next
  __syncthreads();
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Four e4m3 codes to two f16 pairs (exact).
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\t"
      "mov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(codes));
}
// The powers of two of four E8M0 bytes (exact; 255 is NaN).
__device__ __forceinline__ void e8m0x4_to_float(uint32_t bytes, float (&f)[4]) {
  uint32_t lo, hi;
  asm("{\n\t.reg .b16 a, b;\n\t"
      "mov.b32 {a, b}, %2;\n\t"
      "cvt.rn.bf16x2.ue8m0x2 %0, a;\n\t"
      "cvt.rn.bf16x2.ue8m0x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(bytes));
  f[0] = __uint_as_float(lo << 16);
  f[1] = __uint_as_float(lo & 0xFFFF0000u);
  f[2] = __uint_as_float(hi << 16);
  f[3] = __uint_as_float(hi & 0xFFFF0000u);
}
__device__ __forceinline__ uint32_t pack_f16x2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// 2^(14 - floor(log2 amax)), kept finite, and its inverse.
__device__ __forceinline__ void moe_act_scale(uint32_t amax_bits, float& to, float& back) {
  const int e = int(amax_bits >> 23);  // biased; 0: zero or subnormal, 255: inf or NaN
  const int f = amax_bits == 0u ? 127 : min(127 + 14 + 127 - e, 253);  // biased exponent of `to`
  to = __uint_as_float(uint32_t(f) << 23);
  back = __uint_as_float(uint32_t(254 - f) << 23);
}

// y of the row tiles in list[1 .. list[0]]: a thread takes four rows of one
// token and adds its pairs in order (and each pair's K ranges in order).
template <class T>
__device__ void moe_combine(const MoeParams& p, const MoeRoute& route, const int* list, int thread, int threads) {
  const int tasks = list[0] * p.T * 4;
  for (int task = thread; task < tasks; task += threads) {
    const int t = (task >> 2) % p.T, r0 = list[1 + (task >> 2) / p.T] * 16 + (task & 3) * 4;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int j = 0; j < p.top_k; ++j) {
      const int pair = t * p.top_k + j;
      if (route.expert[pair] < 0) continue;
      const float* z = p.z + int64_t(pair) * p.segments * p.H + r0;
      float4 v = __ldcg(reinterpret_cast<const float4*>(z));
      for (int sg = 1; sg < p.segments; ++sg) {
        const float4 a = __ldcg(reinterpret_cast<const float4*>(z + int64_t(sg) * p.H));
        v.x += a.x, v.y += a.y, v.z += a.z, v.w += a.w;
      }
      const float w = route.weight[pair];
      sum.x = fmaf(w, v.x, sum.x), sum.y = fmaf(w, v.y, sum.y);
      sum.z = fmaf(w, v.z, sum.z), sum.w = fmaf(w, v.w, sum.w);
    }
    T* y = static_cast<T*>(p.y) + int64_t(t) * p.ldy + r0;
    uint2 out;
    if constexpr (std::is_same_v<T, __nv_bfloat16>)
      out = make_uint2(pack_bf16x2(sum.x, sum.y), pack_bf16x2(sum.z, sum.w));
    else
      out = make_uint2(pack_f16x2(sum.x, sum.y), pack_f16x2(sum.z, sum.w));
    *reinterpret_cast<uint2*>(y) = out;
  }
}

template <bool GATE_, bool MX_, int NT_, class T_>
struct MoeCfg {
  static constexpr bool GATE = GATE_, MX = MX_;
  static constexpr int NT = NT_;  // 8-token MMA tiles of a chunk
  using T = T_;                   // x and y
  static constexpr int BLOCK_BYTES = MX ? 64 : 128;  // 128 values of K of one row
};

template <class Cfg>
__global__ void __launch_bounds__(kMoeThreads, 1) moe_kernel(const __grid_constant__ MoeParams p) {
  constexpr bool GATE = Cfg::GATE, MX = Cfg::MX;
  constexpr int NT = Cfg::NT, BB = Cfg::BLOCK_BYTES;
  using T = typename Cfg::T;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int S = p.stages, row_pitch = p.stage_row + 16;
  const uint32_t stage_bytes = uint32_t(16 * row_pitch + (MX ? p.stage_row / BB * 256 : 0));
  auto full = [&](int s) { return base + p.off_bars + 8u * uint32_t(s); };
  auto empty = [&](int s) { return base + p.off_bars + 8u * uint32_t(S + s); };
  auto red_full = [&](int b) { return base + p.off_bars + 8u * uint32_t(2 * S + b); };
  auto red_empty = [&](int b) { return base + p.off_bars + 8u * uint32_t(2 * S + 2 + b); };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + p.off_bars + 8 * (2 * S + 4));
  int* finished = reinterpret_cast<int*>(smem + p.off_bars + 8 * (2 * S + 4) + 16);  // [1 + kMoeBatch]
  const MoeRoute route = moe_route_at(smem + p.off_route, p.T * p.top_k);

  if (tid == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(full(s), 1u);
      mbar_init(empty(s), kMoeConsumers);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(red_full(b), kMoeConsumers);
      mbar_init(red_empty(b), 1u);
    }
    *abort_flag = 0;
    finished[0] = 0;
    fence_barrier_init();
  }
  if constexpr (GATE) {
    griddep_wait();
    griddep_launch_dependents();  // DOWN may start: what earlier kernels wrote is visible to it
    for (int i = blockIdx.x * kMoeThreads + tid; i < p.H / 16; i += gridDim.x * kMoeThreads) p.counters[i] = 0;
  }
  // The routing tables (scratch: the ring, before its first copy).
  moe_route(p, route, reinterpret_cast<uint32_t*>(smem), 8 * NT);

  const int chunks = route.totals[0];
  const int tiles = GATE ? p.I / 8 : p.H / 16, per_chunk = tiles * p.segments;
  const int K = GATE ? p.H : p.I;
  const int64_t units = int64_t(chunks) * per_chunk;
  const int u0 = int(units * blockIdx.x / gridDim.x), u1 = int(units * (blockIdx.x + 1) / gridDim.x);
  // A unit's place: chunk, K range, rows.
  auto place = [&](int u, int& chunk, int& seg, int& tile) {
    chunk = u / per_chunk;
    const int rest = u - chunk * per_chunk;
    seg = rest / tiles;
    tile = rest - seg * tiles;
  };
  const int stage_blocks = p.stage_row / BB;  // 128-wide blocks of a stage

  if (warp == kMoeConsumers) {
    // ---------------------------------------------------------------- producer
    const uint64_t policy = policy_evict_first(), scale_policy = policy_evict_normal();
    int n = 0;
    bool ok = true;
    for (int u = u0; u < u1 && ok; ++u) {
      int chunk, seg, tile;
      place(u, chunk, seg, tile);
      const int row = GATE ? (lane & 8 ? p.I : 0) + tile * 8 + (lane & 7) : tile * 16 + (lane & 15);
      const uint8_t* src = p.w + int64_t(route.chunk_expert[chunk]) * p.w_expert + int64_t(row) * p.w_row +
                           int64_t(seg) * p.seg_len / 128 * BB;
      const int k_len = min(p.seg_len, K - seg * p.seg_len);
      const int bytes = MX ? k_len / 2 : k_len;
      for (int at = 0; at < bytes; at += p.stage_row, ++n) {
        const int s = n % S;
        if (n >= S) ok = mbar_wait(empty(s), uint32_t(n / S - 1) & 1u, abort_flag, kMoeWaitEmpty);
        ok = __all_sync(~0u, ok);
        if (!ok) break;
        const uint32_t len = uint32_t(min(p.stage_row, bytes - at));
        const int nb = (int(len) + BB - 1) / BB;
        const uint32_t stage = base + uint32_t(s) * stage_bytes;
        if (lane == 0) mbar_arrive_expect_tx(full(s), 16u * len + (MX ? uint32_t(nb) * 256u : 0u));
        __syncwarp();
        if (lane < 16) bulk_load(stage + uint32_t(lane * row_pitch), src + at, len, full(s), policy);
        if constexpr (MX) {
          // A block's scale words of 8 rows are 8 x 16 contiguous bytes of its
          // tile, each with the words of the rows 32, 64 and 96 further on:
          // a fourth of it is used here, the rest by the CTA's next units (from L2).
          const int half = lane >> 4;  // rows 0-7 and 8-15 of the unit
          const int r = GATE ? half * p.I + tile * 8 : tile * 16 + 8 * half;
          const uint8_t* sc = static_cast<const uint8_t*>(p.ws) +
                              ((int64_t(route.chunk_expert[chunk]) * p.rb + (r >> 7)) * p.kb + seg * (p.seg_len / 128) + at / BB) * 512 +
                              (r & 31) * 16;
          for (int i = lane & 15; i < nb; i += 16)
            bulk_load(stage + uint32_t(16 * row_pitch + i * 256 + half * 128), sc + i * 512, 128u, full(s), scale_policy);
        }
      }
    }
    for (int k = n > S ? n - S : 0; k < n; ++k) mbar_wait(full(k % S), uint32_t(k / S) & 1u, nullptr, kMoeWaitDrain);
  } else if (warp < kMoeConsumers) {
    // ---------------------------------------------------------------- consumers
    const int g = lane >> 2, t4 = lane & 3;
    uint8_t* bfrag = smem + p.off_b;
    float* ts = reinterpret_cast<float*>(smem + p.off_ts);  // [block][8 NT]
    if constexpr (!GATE) griddep_wait();                    // h
    int n = 0, q = 0, have = -1, count = 0;
    bool ok = true;
    // Block FP8 scales: lane l holds those of K blocks l and l + 32 of the
    // unit's two 8-row halves, requested a unit ahead.
    float sc[2][2], sc_next[2][2];
    auto load_scales = [&](int u, float (&v)[2][2]) {
      int chunk, seg, tile;
      place(u, chunk, seg, tile);
      const float* e = static_cast<const float*>(p.ws) + int64_t(route.chunk_expert[chunk]) * p.rb * p.kb;
      const int kb = seg * (p.seg_len / 128);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int r = GATE ? half * p.I + tile * 8 : tile * 16 + 8 * half;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int b = kb + lane + 32 * j;
          v[half][j] = b < p.kb ? ldg_pinned(e + int64_t(r >> 7) * p.kb + b) : 0.f;
        }
      }
    };
    if (!MX && u0 < u1) load_scales(u0, sc_next);
    for (int u = u0; u < u1; ++u) {
      int chunk, seg, tile;
      place(u, chunk, seg, tile);
      if constexpr (!MX) {
#pragma unroll
        for (int half = 0; half < 2; ++half) sc[half][0] = sc_next[half][0], sc[half][1] = sc_next[half][1];
        if (u + 1 < u1) load_scales(u + 1, sc_next);
      }
      const int k_len = min(p.seg_len, K - seg * p.seg_len);
      const int blocks = (k_len + 127) / 128;
      if (have != chunk * p.segments + seg) {
        // ---- the chunk's activations to f16 fragments
        have = chunk * p.segments + seg;
        count = route.chunk_count[chunk];
        named_bar_sync(1, 32 * kMoeConsumers);
        const int half = tid >> 4, l16 = tid & 15;  // 16 half-warps; a task is one token's block
        const int tasks = count * blocks;
        for (int task0 = 0; task0 < tasks; task0 += 16) {
          const int task = task0 + half;
          const int tok = task / blocks, b = task - tok * blocks;
          const int k = b * 128 + l16 * 8;
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = 0.f;
          if (task < tasks && k < k_len) {
            const int pair = route.list[route.chunk_first[chunk] + tok];
            if constexpr (GATE)
              load8(static_cast<const T*>(p.x) + int64_t(pair / p.top_k) * p.ldx + k, v);
            else
              load8(p.h + int64_t(pair) * p.I + seg * p.seg_len + k, v);
          }
          uint32_t m = 0u;
#pragma unroll
          for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
#pragma unroll
          for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(~0u, m, o));
          float to, back;
          moe_act_scale(m, to, back);
          if (task < tasks) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = pack_f16x2(v[2 * i] * to, v[2 * i + 1] * to);
            const int nt = tok >> 3;
            // 32 values of K make one 512-byte piece: [token of 8][lane quarter][16 bytes]
            uint8_t* piece = bfrag + ((b * 4 + (l16 >> 2)) * NT + nt) * 512 + (tok & 7) * 64;
            if constexpr (MX) {
              // a lane's codes are 8 consecutive values
              *reinterpret_cast<uint4*>(piece + (l16 & 3) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
              // a lane's codes are 4 consecutive values of each 16
              uint8_t* at = piece + ((l16 >> 1) & 1) * 8 + (l16 & 1) * 32;
              *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[1]);
              *reinterpret_cast<uint2*>(at + 16) = make_uint2(w[2], w[3]);
            }
            if (l16 == 0) ts[b * 8 * NT + tok] = back;
          }
        }
        named_bar_sync(1, 32 * kMoeConsumers);
      }
      float acc[NT][4];
#pragma unroll
      for (int i = 0; i < NT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
      for (int b0 = 0; b0 < blocks; b0 += stage_blocks, ++n) {
        const int s = n % S;
        ok = mbar_wait(full(s), uint32_t(n / S) & 1u, abort_flag, kMoeWaitFull) && ok;
        const int nb = min(stage_blocks, blocks - b0);
        for (int i = (warp - q) & (kMoeConsumers - 1); i < nb; i += kMoeConsumers) {
          const int b = b0 + i;  // block of this K range
          float sa = 1.f, sb = 1.f;
          float fa4[4], fb4[4];
          if constexpr (MX) {
            // the word of this row: 32-row quarter of its tile
            const int ra = (GATE ? tile * 8 : tile * 16), rb = GATE ? p.I + tile * 8 : tile * 16 + 8;
            const uint32_t at = base + uint32_t(s) * stage_bytes + uint32_t(16 * row_pitch + i * 256 + g * 16);
            e8m0x4_to_float(ld_shared_u32(at + uint32_t((ra >> 5) & 3) * 4u), fa4);
            e8m0x4_to_float(ld_shared_u32(at + 128u + uint32_t((rb >> 5) & 3) * 4u), fb4);
          } else {
            sa = __shfl_sync(~0u, b < 32 ? sc[0][0] : sc[0][1], b & 31);
            sb = GATE ? __shfl_sync(~0u, b < 32 ? sc[1][0] : sc[1][1], b & 31) : sa;
          }
          // ldmatrix rows: lanes 0-7 / 8-15 the two row halves of one 16-byte
          // column, lanes 16-31 of the next
          const uint32_t a_addr = base + uint32_t(s) * stage_bytes + uint32_t((lane & 15) * row_pitch + i * BB + (lane >> 4) * 16);
          const uint8_t* bp = bfrag + b * 4 * NT * 512 + lane * 16;
          const int pairs = min(4, (k_len - b * 128) / 32);  // 32-wide steps of the block
          float part[NT][4];
#pragma unroll
          for (int c = 0; c < NT; ++c) part[c][0] = part[c][1] = part[c][2] = part[c][3] = 0.f;
          if constexpr (MX) {
#pragma unroll
            for (int pp = 0; pp < 4; pp += 2) {
              if (pp < pairs) {
                uint32_t r[4];
                ldmatrix_x4(a_addr + uint32_t(pp * 16), r);
#pragma unroll
                for (int h2 = 0; h2 < 2; ++h2) {
                  if (pp + h2 < pairs) {
                    uint32_t ha[4], hb[4];
                    e2m1x8_to_f16(r[2 * h2], ha);
                    e2m1x8_to_f16(r[2 * h2 + 1], hb);
                    const float fa = fa4[pp + h2], fb = fb4[pp + h2];
#pragma unroll
                    for (int c = 0; c < NT; ++c) {
                      if (c == 0 || c * 8 < count) {
                        const uint4 bv = *reinterpret_cast<const uint4*>(bp + ((pp + h2) * NT + c) * 512);
                        float d[4] = {0.f, 0.f, 0.f, 0.f};
                        mma_f16(d, ha[0], hb[0], ha[1], hb[1], bv.x, bv.y);
                        mma_f16(d, ha[2], hb[2], ha[3], hb[3], bv.z, bv.w);
                        part[c][0] = fmaf(d[0], fa, part[c][0]);
                        part[c][1] = fmaf(d[1], fa, part[c][1]);
                        part[c][2] = fmaf(d[2], fb, part[c][2]);
                        part[c][3] = fmaf(d[3], fb, part[c][3]);
                      }
                    }
                  }
                }
              }
            }
          } else {
#pragma unroll
            for (int pp = 0; pp < 4; ++pp) {
              if (pp < pairs) {
                uint32_t r[4], lo[4], hi[4];
                ldmatrix_x4(a_addr + uint32_t(pp * 32), r);
#pragma unroll
                for (int k = 0; k < 4; ++k) e4m3x4_to_f16(r[k], lo[k], hi[k]);
#pragma unroll
                for (int c = 0; c < NT; ++c) {
                  if (c == 0 || c * 8 < count) {
                    const uint4 bv = *reinterpret_cast<const uint4*>(bp + (pp * NT + c) * 512);
                    mma_f16(part[c], lo[0], lo[1], hi[0], hi[1], bv.x, bv.y);
                    mma_f16(part[c], lo[2], lo[3], hi[2], hi[3], bv.z, bv.w);
                  }
                }
              }
            }
          }
#pragma unroll
          for (int c = 0; c < NT; ++c) {
            if (c == 0 || c * 8 < count) {
              const float2 tsc = *reinterpret_cast<const float2*>(ts + b * 8 * NT + c * 8 + 2 * t4);
              acc[c][0] = fmaf(part[c][0], tsc.x * sa, acc[c][0]);
              acc[c][1] = fmaf(part[c][1], tsc.y * sa, acc[c][1]);
              acc[c][2] = fmaf(part[c][2], tsc.x * sb, acc[c][2]);
              acc[c][3] = fmaf(part[c][3], tsc.y * sb, acc[c][3]);
            }
          }
        }
        q += nb;
        __syncwarp();
        if (lane == 0) mbar_arrive(empty(s));
      }
      // ---- this warp's sums of the unit
      const int i = u - u0, buf = i & 1;
      if (i >= 2) ok = mbar_wait(red_empty(buf), uint32_t(i / 2 - 1) & 1u, abort_flag, kMoeWaitRedEmpty) && ok;
      float4* red = reinterpret_cast<float4*>(smem + p.off_red) + (buf * kMoeConsumers + warp) * NT * 32 + lane;
#pragma unroll
      for (int c = 0; c < NT; ++c) red[c * 32] = make_float4(acc[c][0], acc[c][1], acc[c][2], acc[c][3]);
      __syncwarp();
      if (lane == 0) mbar_arrive(red_full(buf));
    }
  } else {
    // ---------------------------------------------------------------- finisher
    const int g = lane >> 2, t4 = lane & 3;
    if constexpr (!GATE) griddep_wait();  // the counters, y
    const bool none = !GATE && units == 0;
    if (none) {  // no pair has an expert: y = 0
      T* y = static_cast<T*>(p.y);
      for (int64_t i = int64_t(blockIdx.x) * 32 + lane; i < int64_t(p.T) * p.H; i += int64_t(gridDim.x) * 32)
        y[i / p.H * p.ldy + i % p.H] = T(0.f);
    }
    int flushed = u0;  // units whose arrival is counted
    for (int u = u0; u < u1; ++u) {
      int chunk, seg, tile;
      place(u, chunk, seg, tile);
      const int i = u - u0, buf = i & 1;
      if (!mbar_wait(red_full(buf), uint32_t(i / 2) & 1u, abort_flag, kMoeWaitRedFull)) break;
      const int count = route.chunk_count[chunk], first = route.chunk_first[chunk];
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        if (c > 0 && c * 8 >= count) break;
        const float4* red = reinterpret_cast<const float4*>(smem + p.off_red) + (buf * kMoeConsumers * NT + c) * 32 + lane;
        float4 v = red[0];
#pragma unroll
        for (int w = 1; w < kMoeConsumers; ++w) {
          const float4 a = red[w * NT * 32];
          v.x += a.x, v.y += a.y, v.z += a.z, v.w += a.w;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {  // columns 2 t4 and 2 t4 + 1
          const int tok = c * 8 + 2 * t4 + k;
          if (tok >= count) continue;
          const int pair = route.list[first + tok];
          const float a = k ? v.y : v.x, b = k ? v.w : v.z;
          if constexpr (GATE) {
            p.h[int64_t(pair) * p.I + tile * 8 + g] = a / (1.f + expf(-a)) * b;
          } else {
            float* z = p.z + (int64_t(pair) * p.segments + seg) * p.H + tile * 16 + g;
            z[0] = a;
            z[8] = b;
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(red_empty(buf));
      if constexpr (!GATE) {
        // Arrivals are counted a batch of units at a time: a fence and an
        // atomic cost as much as streaming two to four units.
        if (u + 1 - flushed == kMoeBatch || u + 1 == u1) {
          __threadfence();
          __syncwarp();
          bool last = false;
          int tile_l = 0;
          if (lane < u + 1 - flushed) {
            int c_l, s_l;
            place(flushed + lane, c_l, s_l, tile_l);
            last = atomicAdd(p.counters + tile_l, 1) == chunks * p.segments - 1;
          }
          __threadfence();
          const uint32_t lasts = __ballot_sync(~0u, last);
          if (last) finished[1 + __popc(lasts & ((1u << lane) - 1u))] = tile_l;
          if (lane == 0) finished[0] = __popc(lasts);
          __syncwarp();
          flushed = u + 1;
          if (u + 1 < u1) moe_combine<T>(p, route, finished, lane, 32);
        }
      }
    }
  }
  if constexpr (!GATE) {
    __syncthreads();
    // the last batch's row tiles, by every warp
    if (!*abort_flag) moe_combine<T>(p, route, finished, tid, kMoeThreads);
  }
}

}  // namespace bfp8
