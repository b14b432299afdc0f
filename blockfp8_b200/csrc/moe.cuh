// A mixture-of-experts layer for a few tokens, in two kernels that stream the
// weights and a small sum:
//
//   moe_kernel<GATE>  ids, p = router(logits)            (every CTA, from the logits)
//                     h[t, j] = silu(W1[e] x[t]) * (W3[e] x[t]),  e = ids[t, j]
//   moe_kernel<DOWN>  z[t, j] = W2[e] h[t, j]
//   moe_sum_kernel    y[t] = sum_j p[t, j] z[t, j]
//
// Expert weights are block FP8 (e4m3, one fp32 scale per 128 x 128) or MXFP4
// (e2m1, one power-of-two scale per 32); activations are not quantized.  At
// these sizes the weights of the chosen experts are the only traffic that
// counts, so the kernels are built to stream them:
//
// Measured (B200, device time of a call in a graph): 64 tokens, 128 experts, top
// 8, H = 4096, I = 1280 in block FP8: 350 to 380 us for the 1.5 to 1.6 GB of the
// 96 to 104 experts that they meet; 13 tokens, 64 experts, top 6, I = 1408: 125 to
// 132 us for 37 to 43 of them; one token, 128 experts, top 8, H = 2048, I = 768: 27
// us for 38 MB (6 us at the measured copy rate): there the router (3 us), the
// hand-over between the kernels and their ends count, not the stream.  MXFP4, 40
// tokens, 64 experts, top 4, I = 2048: 188 to 191 us for 0.6 GB.  (Batches run into
// the power limit: 1.7 to 1.9 GHz; the lower figures are the first calls'.)
//
// - Work: (token, expert) pairs are grouped by expert into chunks of up to
//   8, in token order (busier experts are read again, mostly from L2: chunks of 16
//   with two MMA tiles and half the ring took 1.4 to 2.2 times as long for 5 to
//   25 tokens an expert).  A unit is 16 weight rows (GATE: 8 gate rows
//   and the 8 up rows beside them, so that one thread ends with both) of one
//   chunk over a whole K range, and CTA b of G takes units [U b / G, U (b+1) / G).
//   16 rows keep the last wave short (one token, 8 experts of I = 768: 768
//   units over 148 CTAs) and need no sums across CTAs.
// - A ring of shared-memory stages, 16 rows x up to 1 KB each; it runs across
//   units, so the memory system sees one stream per SM.  A stage is one 5-D TMA
//   box [128 bytes, 8 rows, up to 8 columns of 128 bytes, 2 halves, 1 expert]
//   in the 128-byte swizzle, which ldmatrix reads without conflicts.  (One
//   bulk copy per row took the issuing warp about 60 clocks each, 1,000 a
//   stage: more than the 700 that HBM takes to deliver it.)
// - Consumer warps (8 or 16) work in groups, each with a unit and a ring of its
//   own, and take the 128-wide K blocks of a stage in turn inside a group:
//   ldmatrix, codes to f16 (exact: cvt, 128 codes per clock and SM), mma.sync
//   m16n8k16 with fp32 accumulation, then the block's scales in fp32.  The
//   legacy MMA is no bound here (one 8-token MMA per 256 weights is 0.09 of
//   its 0.5 per clock at the HBM rate) and takes the dequantized registers
//   directly; tcgen05 would need them written back to shared memory.
// - Activations are held in shared memory as f16 in MMA fragment order with
//   one power-of-two scale per token and 128 values, which puts the largest
//   at 2^14: bf16 values are exact down to 2^-28 of it.  h (fp32) takes two
//   f16 parts, the value rounded and what that leaves: 22 bits of each value,
//   at worst 2^-39 of the largest.  Up to four pairs have their upper parts in
//   the MMA's columns 0-3 and the lower ones in 4-7.  Batches beyond 8 tokens have
//   chunks of up to eight, whose parts lie in two planes of eight columns and
//   take MMAs of their own (and a unit of them more time: the CTAs' shares count
//   it a quarter more).
// - A last warp finishes units: it adds the consumers' sums in warp order.
//   z goes to memory and a small third kernel adds each token's pairs in j
//   order.  (Counting arrivals and letting the last unit of an output row tile
//   add them makes the slowest CTA do nearly all of it: 2.4 times the median
//   CTA's time at 64 tokens.)  No result depends on the order of arrival.
//
// Warps: consumers, then one or two producers, then the finisher.
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
constexpr int kMoeBeside = 4;  // most pairs whose h has both parts in one MMA's columns

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
  // This kernel's weights, rows of `columns` full 128-byte columns (map_w: box
  // columns of 8 rows and of the 8 rows of the unit's other half) and perhaps
  // one shorter (map_tail: 128 bytes of 8 rows).
  CUtensorMap map_w, map_tail;
  int columns, rows, tail_reads_on;
  CUtensorMap map_s;    // MXFP4: scale tiles, [128 bytes = 8 rows] x 2 box K blocks,
  int scales_together;  // of both halves at once where they are a fixed distance apart
  const void* ws;     // block FP8: scales fp32 [E, rb, kb]
  int rb, kb;
  float* h;       // [T top_k, I]
  float* z;       // [T top_k, segments, H]
  float2* routed;  // [T top_k] (weight, expert or -1), written by GATE
  int T, H, I, E, top_k;
  int segments, seg_len;  // K ranges of DOWN
  int stages, box;        // ring: stages, 128-byte columns of a stage
  int unit_stages;        // stages of a unit
  int cols;               // token columns held
  int resident;           // every token (GATE) or pair (DOWN) has its own
  uint32_t off_b, off_ts, off_red, off_route, off_bars;  // shared memory
  uint32_t plane;  // DOWN: bytes of a plane of columns
};

struct MoeSumParams {
  const float* z;
  const float2* routed;
  void* y;
  int64_t ldy;
  int T, H, top_k, segments;
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

// The top_k of one token by one warp: E <= 32 NE logits.
template <int NE>
__device__ __forceinline__ void moe_top_k(const MoeParams& p, const MoeRoute& r, int t, int lane) {
  uint32_t key[NE];
#pragma unroll
  for (int i = 0; i < NE; ++i) {
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
  float all = 0.f, top = 0.f, mine = 0.f;  // lane j keeps exp(l_j - l_0) of the j-th choice
  int id = -1, my_id = -1;
  for (int j = 0; j < p.top_k; ++j) {
    uint32_t best = 0u, at = ~0u;
#pragma unroll
    for (int i = NE - 1; i >= 0; --i)  // the lane's largest, the lowest index of equals
      if (key[i] >= best) best = key[i], at = uint32_t(i * 32 + lane);
    const uint32_t most = __reduce_max_sync(~0u, best);
    if (most == 0u) break;  // nothing left to choose
    const uint32_t who = __ballot_sync(~0u, best == most);
    id = who & (who - 1u) ? int(__reduce_min_sync(~0u, best == most ? at : ~0u))  // equals: the lowest index
                          : int(__shfl_sync(~0u, at, __ffs(who) - 1));
    const float v = moe_key_value(most);
    if (j == 0) {
      top = v;
      if (!p.renormalize) {
#pragma unroll
        for (int i = 0; i < NE; ++i)
          if (key[i]) all += expf(moe_key_value(key[i]) - top);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(~0u, all, o);
      }
    }
    if (lane == j) mine = v, my_id = id;
#pragma unroll
    for (int i = 0; i < NE; ++i)
      if (id == i * 32 + lane) key[i] = 0u;
  }
  mine = my_id >= 0 ? expf(mine - top) : 0.f;
  if (p.renormalize) {
    all = mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(~0u, all, o);
  }
  if (lane < p.top_k) {
    r.expert[t * p.top_k + lane] = short(my_id);
    r.weight[t * p.top_k + lane] = my_id >= 0 ? mine / all : 0.f;
  }
}

// Each pair's expert and weight.  Tokens go to warps from the last one down:
// the first ones have other work at that time.
template <int THREADS>
__device__ __forceinline__ void moe_select(const MoeParams& p, const MoeRoute& r) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (p.logits) {
    for (int t = THREADS / 32 - 1 - warp; t < p.T; t += THREADS / 32) {
      if (p.E <= 128) moe_top_k<4>(p, r, t, lane);
      else moe_top_k<kMoeMaxExperts / 32>(p, r, t, lane);
    }
  } else {
    for (int i = tid; i < p.T * p.top_k; i += THREADS) {
      const int e = p.ids[i];
      r.expert[i] = short(e >= 0 && e < p.E ? e : -1);
      r.weight[i] = p.weights[i];
    }
  }
}

// The chunk tables, by all threads of the CTA; at most cap pairs a chunk, and
// (P <= 8) all of one half of the pairs where `halves` says so.
// scratch: room for E (ceil(P / 32) + 1) words.
template <int THREADS>
__device__ __forceinline__ void moe_group(const MoeParams& p, const MoeRoute& r, uint32_t* scratch, int cap, bool halves) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int P = p.T * p.top_k, words = (P + 31) / 32;
  uint32_t* masks = scratch;                                     // [E][words] pairs of each expert
  int* offsets = reinterpret_cast<int*>(scratch + p.E * words);  // [E]
  if (P > 32)
    for (int i = tid; i < p.E * words; i += THREADS) masks[i] = 0u;
  __syncthreads();
  if (P <= 32) {
    // One warp, a pair a lane; an expert's chunks stand where its first pair does.
    if (warp == 0) {
      const int e = lane < P ? r.expert[lane] : -1;
      const uint32_t same = __match_any_sync(~0u, halves && e >= 0 ? 2 * e + lane / kMoeBeside : e);
      const int n = e >= 0 ? __popc(same) : 0, at = __popc(same & ((1u << lane) - 1u));
      const bool first = n > 0 && at == 0;
      int pairs = first ? n : 0, chunks = first ? (n + cap - 1) / cap : 0;
      const int own_pairs = pairs, own_chunks = chunks;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(~0u, pairs, o), y = __shfl_up_sync(~0u, chunks, o);
        if (lane >= o) pairs += x, chunks += y;
      }
      if (lane == 31) r.totals[0] = chunks;
      const int pair0 = __shfl_sync(~0u, pairs - own_pairs, __ffs(same) - 1);
      if (n > 0) r.list[pair0 + at] = short(lane);
      for (int c = 0; c < own_chunks; ++c) {
        const int k = chunks - own_chunks + c;
        r.chunk_expert[k] = short(e);
        r.chunk_first[k] = short(pair0 + c * cap);
        r.chunk_count[k] = short(min(cap, n - c * cap));
      }
    }
  } else {
    for (int i = tid; i < P; i += THREADS) {
      const int e = r.expert[i];
      if (e >= 0) atomicOr(masks + e * words + i / 32, 1u << (i & 31));
    }
    __syncthreads();
    for (int e = tid; e < p.E; e += THREADS) {
      int n = 0;
      for (int w = 0; w < words; ++w) n += __popc(masks[e * words + w]);
      offsets[e] = n;
    }
    __syncthreads();
    if (warp == 0) {  // first pair and first chunk of every expert
      int pairs = 0, chunks = 0;
      for (int e0 = 0; e0 < p.E; e0 += 32) {
        const int e = e0 + lane, n = e < p.E ? offsets[e] : 0;
        int pi = n, ci = (n + cap - 1) / cap;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int x = __shfl_up_sync(~0u, pi, o), y = __shfl_up_sync(~0u, ci, o);
          if (lane >= o) pi += x, ci += y;
        }
        if (e < p.E) offsets[e] = ((pairs + pi - n) << 16) | (chunks + ci - (n + cap - 1) / cap);
        pairs += __shfl_sync(~0u, pi, 31);
        chunks += __shfl_sync(~0u, ci, 31);
      }
      if (lane == 0) r.totals[0] = chunks;
    }
    __syncthreads();
    for (int e = tid; e < p.E; e += THREADS) {
      const int first = offsets[e] >> 16, chunk = offsets[e] & 0xFFFF;
      int n = 0;
      for (int w = 0; w < words; ++w) {
        uint32_t m = masks[e * words + w];
        while (m) {
          r.list[first + n++] = short(w * 32 + __ffs(m) - 1);
          m &= m - 1;
        }
      }
      for (int c = 0; c * cap < n; ++c) {
        r.chunk_expert[chunk + c] = short(e);
        r.chunk_first[chunk + c] = short(first + c * cap);
        r.chunk_count[chunk + c] = short(min(cap, n - c * cap));
      }
    }
    fence_proxy_async_smem();  // the ring's copies overwrite the scratch next
  }
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

// What rounding a and b to the f16 pair `upper` leaves (exact), as a pair.
__device__ __forceinline__ uint32_t f16x2_rest(float a, float b, uint32_t upper) {
  const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&upper));
  return pack_f16x2(a - u.x, b - u.y);
}

// 2^(14 - floor(log2 amax)), kept finite, and its inverse.
__device__ __forceinline__ void moe_act_scale(uint32_t amax_bits, float& to, float& back) {
  const int e = int(amax_bits >> 23);  // biased; 0: zero or subnormal, 255: inf or NaN
  const int f = amax_bits == 0u ? 127 : min(127 + 14 + 127 - e, 253);  // biased exponent of `to`
  to = __uint_as_float(uint32_t(f) << 23);
  back = __uint_as_float(uint32_t(254 - f) << 23);
}

// y[t] = sum_j p[t, j] z[t, j]: a thread takes four columns of one token and
// adds its pairs in order (and each pair's K ranges in order).
constexpr int kMoeSumThreads = 128;
template <class T>
__global__ void __launch_bounds__(kMoeSumThreads) moe_sum_kernel(const MoeSumParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int task = blockIdx.x * kMoeSumThreads + threadIdx.x;
  const int t = task / (p.H / 4), col = task % (p.H / 4) * 4;
  if (t >= p.T) return;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int j = 0; j < p.top_k; ++j) {
    const int pair = t * p.top_k + j;
    const float2 r = p.routed[pair];
    if (__float_as_int(r.y) < 0) continue;
    const float* z = p.z + int64_t(pair) * p.segments * p.H + col;
    float4 v = __ldcg(reinterpret_cast<const float4*>(z));
    for (int sg = 1; sg < p.segments; ++sg) {
      const float4 a = __ldcg(reinterpret_cast<const float4*>(z + int64_t(sg) * p.H));
      v.x += a.x, v.y += a.y, v.z += a.z, v.w += a.w;
    }
    sum.x = fmaf(r.x, v.x, sum.x), sum.y = fmaf(r.x, v.y, sum.y);
    sum.z = fmaf(r.x, v.z, sum.z), sum.w = fmaf(r.x, v.w, sum.w);
  }
  uint2 out;
  if constexpr (std::is_same_v<T, __nv_bfloat16>)
    out = make_uint2(pack_bf16x2(sum.x, sum.y), pack_bf16x2(sum.z, sum.w));
  else
    out = make_uint2(pack_f16x2(sum.x, sum.y), pack_f16x2(sum.z, sum.w));
  *reinterpret_cast<uint2*>(static_cast<T*>(p.y) + int64_t(t) * p.ldy + col) = out;
}

constexpr int kMoeChunk = 8;       // most pairs of a chunk: the MMA's columns
constexpr int kMoeGroupWarps = 4;  // consumer warps of a group, which works on a unit of its own
constexpr int kMoeRedBufs = 2;     // buffers of the warps' sums (512 bytes a warp)

template <bool GATE_, bool MX_, int WARPS_, class T_>
struct MoeCfg {
  static constexpr bool GATE = GATE_, MX = MX_;
  static constexpr int WARPS = WARPS_;  // consumers
  static constexpr int GROUPS = WARPS / kMoeGroupWarps;
  static constexpr int PRODUCERS = WARPS == 16 ? 2 : 1;
  static constexpr int THREADS = 32 * (WARPS + PRODUCERS + 1);
  static constexpr int CTAS_PER_SM = WARPS == 8 ? 2 : 1;
  // DOWN's chunks may have more than four pairs; otherwise all pairs may have
  // columns of their own.
  static constexpr bool BUSY = !GATE && WARPS == 16;
  using T = T_;                   // x and y
  static constexpr int BLOCK_BYTES = MX ? 64 : 128;  // 128 values of K of one row
};

// acc += one 128-wide K block of 16 weight rows times the chunk's 8 columns.
// a_row, chunk0: this lane's ldmatrix row and first 16-byte chunk in it;
// b_addr: its piece of the tokens' fragments, piece bytes apart per 32 values
// of K; LOW: as much again `low` further on, for the same columns; ts: the scales of this lane's two columns.  FULL: all four 32-wide steps, so
// that every load can go out first; else `steps` of them.
template <class Cfg, bool FULL, bool LOW>
__device__ __forceinline__ void moe_block(float (&acc)[4], uint32_t a_row, uint32_t chunk0, uint32_t b_addr,
                                          uint32_t piece, uint32_t low, int steps, const float (&fa)[4],
                                          const float (&fb)[4], const float* ts) {
  // the 128-byte swizzle: chunk XOR row inside 8 rows
  auto chunk_at = [&](uint32_t c) { return a_row + (((chunk0 + c) ^ (threadIdx.x & 7u)) << 4); };
  float part[2][4] = {};
  if constexpr (Cfg::MX) {
    uint32_t r[4][2];  // [step][8-row half]: eight codes
#pragma unroll
    for (int s = 0; s < 4; s += 2)
      if (FULL || s < steps) {
        uint32_t v[4];
        ldmatrix_x4(chunk_at(uint32_t(s)), v);
        r[s][0] = v[0], r[s][1] = v[1], r[s + 1][0] = v[2], r[s + 1][1] = v[3];
      }
#pragma unroll
    for (int s = 0; s < 4; ++s)
      if (FULL || s < steps) {
        uint32_t ha[4], hb[4];
        e2m1x8_to_f16(r[s][0], ha);
        e2m1x8_to_f16(r[s][1], hb);
        const uint4 b = ld_shared_v4(b_addr + uint32_t(s) * piece);
        float d[4] = {0.f, 0.f, 0.f, 0.f};
        mma_f16(d, ha[0], hb[0], ha[1], hb[1], b.x, b.y);
        mma_f16(d, ha[2], hb[2], ha[3], hb[3], b.z, b.w);
        if constexpr (LOW) {
          const uint4 l = ld_shared_v4(b_addr + low + uint32_t(s) * piece);
          mma_f16(d, ha[0], hb[0], ha[1], hb[1], l.x, l.y);
          mma_f16(d, ha[2], hb[2], ha[3], hb[3], l.z, l.w);
        }
        float(&q)[4] = part[s & 1];
        q[0] = fmaf(d[0], fa[s], q[0]);
        q[1] = fmaf(d[1], fa[s], q[1]);
        q[2] = fmaf(d[2], fb[s], q[2]);
        q[3] = fmaf(d[3], fb[s], q[3]);
      }
  } else {
    uint32_t r[4][4];
#pragma unroll
    for (int s = 0; s < 4; ++s)
      if (FULL || s < steps) ldmatrix_x4(chunk_at(uint32_t(2 * s)), r[s]);
#pragma unroll
    for (int s = 0; s < 4; ++s)
      if (FULL || s < steps) {
        uint32_t lo[4], hi[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) e4m3x4_to_f16(r[s][k], lo[k], hi[k]);
        const uint4 b = ld_shared_v4(b_addr + uint32_t(s) * piece);
        mma_f16(part[0], lo[0], lo[1], hi[0], hi[1], b.x, b.y);
        mma_f16(part[1], lo[2], lo[3], hi[2], hi[3], b.z, b.w);
        if constexpr (LOW) {
          const uint4 l = ld_shared_v4(b_addr + low + uint32_t(s) * piece);
          mma_f16(part[0], lo[0], lo[1], hi[0], hi[1], l.x, l.y);
          mma_f16(part[1], lo[2], lo[3], hi[2], hi[3], l.z, l.w);
        }
      }
  }
  const float sa = Cfg::MX ? 1.f : fa[0], sb = Cfg::MX ? 1.f : fb[0];
  const float2 t = *reinterpret_cast<const float2*>(ts);
  acc[0] = fmaf(part[0][0] + part[1][0], t.x * sa, acc[0]);
  acc[1] = fmaf(part[0][1] + part[1][1], t.y * sa, acc[1]);
  acc[2] = fmaf(part[0][2] + part[1][2], t.x * sb, acc[2]);
  acc[3] = fmaf(part[0][3] + part[1][3], t.y * sb, acc[3]);
}

// A stage as a consumer warp sees it, and one of its 128-wide K blocks: the
// block's scales of rows g and g + 8, this lane's ldmatrix row (lanes 0-7 / 8-15
// the two halves' rows in one 16-byte chunk, lanes 16-31 in the next), its
// token fragments and scales.
struct MoeStage {
  uint32_t base, words, word_a, word_b;  // MXFP4: of the scales, and in them the halves' words
  uint32_t a_lane, b_cols, piece, low;
  const float* ts;
  int b0;  // its first block's place in the K range
};
template <class Cfg, bool FULL, bool LOW, int SC>
__device__ __forceinline__ void moe_stage_block(const MoeStage& st, int i, int steps, const float (&sc)[SC][SC], float (&acc)[4]) {
  const int lane = threadIdx.x & 31, b = st.b0 + i;
  float fa[4], fb[4];
  if constexpr (Cfg::MX) {
    const uint32_t word = st.base + st.words + uint32_t(i * 128 + (lane >> 2) * 16);
    e8m0x4_to_float(ld_shared_u32(word + st.word_a), fa);
    e8m0x4_to_float(ld_shared_u32(word + st.word_b), fb);
  } else {
    fa[0] = __shfl_sync(~0u, b < 32 ? sc[0][0] : sc[0][SC - 1], b & 31);
    fb[0] = Cfg::GATE ? __shfl_sync(~0u, b < 32 ? sc[SC - 1][0] : sc[SC - 1][SC - 1], b & 31) : fa[0];
  }
  const uint32_t a_row = st.base + st.a_lane + uint32_t(Cfg::MX ? i >> 1 : i) * 1024u;
  const uint32_t chunk0 = (Cfg::MX ? (i & 1) * 4u : 0u) + (lane >> 4);
  moe_block<Cfg, FULL, LOW>(acc, a_row, chunk0, st.b_cols + uint32_t(b * 4) * st.piece, st.piece, st.low, steps, fa, fb,
                            st.ts + b * kMoeChunk);
}

// The producer that fills a slot: a ring belongs to one group, a group to one
// producer.  It alone may drain the slot: to another one its passes are still
// running, and a parity tells a pass only from its neighbours.
__host__ __device__ constexpr int moe_producer_of(int slot, int ring, int producers) { return slot / ring % producers; }
constexpr bool moe_producers_agree(int groups, int producers) {
  for (int ring = 2; ring * groups <= 16; ++ring)
    for (int slot = 0; slot < ring * groups; ++slot) {
      int owners = 0;
      for (int w = 0; w < producers; ++w)
        for (int k = 0; k < groups / producers; ++k) {  // as the producers walk them
          const int g = w + k * producers;
          if (slot >= g * ring && slot < (g + 1) * ring) {
            if (moe_producer_of(slot, ring, producers) != w) return false;
            ++owners;
          }
        }
      if (owners != 1) return false;
    }
  return true;
}
static_assert(moe_producers_agree(2, 1) && moe_producers_agree(4, 2), "a slot has one producer");

template <class Cfg>
__global__ void __launch_bounds__(Cfg::THREADS, Cfg::CTAS_PER_SM) moe_kernel(const __grid_constant__ MoeParams p) {
  constexpr bool GATE = Cfg::GATE, MX = Cfg::MX;
  constexpr int BB = Cfg::BLOCK_BYTES, W = Cfg::WARPS, G = Cfg::GROUPS, RB = kMoeRedBufs;
  constexpr int THREADS = Cfg::THREADS, PRODUCERS = Cfg::PRODUCERS;
  using T = typename Cfg::T;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int S = p.stages;
  const bool resident = !Cfg::BUSY && p.resident;
  // a stage: [half][column][8 rows][128 bytes], MXFP4: then [half][K block][8 rows][16 bytes] of scales
  const uint32_t half_bytes = uint32_t(p.box) * 1024u;
  const uint32_t scale_copy = MX ? uint32_t(p.box) * 256u : 0u;  // of a half
  const uint32_t stage_bytes = (2u * (half_bytes + scale_copy) + 1023u) & ~1023u;
  auto full = [&](int s) { return base + p.off_bars + 8u * uint32_t(s); };
  auto empty = [&](int s) { return base + p.off_bars + 8u * uint32_t(S + s); };
  // of a group's buffer b
  auto red_full = [&](int g, int b) { return base + p.off_bars + 8u * uint32_t(2 * S + g * RB + b); };
  auto red_empty = [&](int g, int b) { return base + p.off_bars + 8u * uint32_t(2 * S + (G + g) * RB + b); };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + p.off_bars + 8 * (2 * S + 2 * G * RB));
  volatile int* issued = abort_flag + 4;  // [S] passes of each slot whose copies went out
  const MoeRoute route = moe_route_at(smem + p.off_route, p.T * p.top_k);

  if (tid == 0) {
    for (int s = 0; s < S; ++s) {
      issued[s] = 0;
      mbar_init(full(s), 1u);
      mbar_init(empty(s), kMoeGroupWarps);
    }
    for (int g = 0; g < G; ++g)
      for (int b = 0; b < RB; ++b) {
        mbar_init(red_full(g, b), kMoeGroupWarps);
        mbar_init(red_empty(g, b), 1u);
      }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if constexpr (GATE) {
    griddep_wait();
    griddep_launch_dependents();  // DOWN may start: what earlier kernels wrote is visible to it
  }
  // Activations in shared memory as f16 in MMA fragment order,
  // [32 values of K][token column][lane quarter][16 bytes], and one power of
  // two per column and 128-wide block.  A column past the batch reads some
  // other token's values and is not used.  DOWN: upper parts in the first half of
  // a plane's columns and lower ones in the second, four pairs a plane; or, for a
  // chunk of more, upper and lower ones in a plane each.
  uint8_t* bfrag = smem + p.off_b;
  float* ts = reinterpret_cast<float*>(smem + p.off_ts);  // [block][8]
  const uint32_t piece = uint32_t(p.cols) * 64u;
  auto fragments = [&](int columns, int k_len, auto row_of) {  // by the consumer warps
    const int blocks = (k_len + 127) / 128, tasks = columns * blocks;
    const int half = tid >> 4, l16 = tid & 15;  // a half-warp's task is one column's block
    constexpr int U = 2;  // tasks whose loads are in flight together
    for (int task0 = 0; task0 < tasks; task0 += 2 * W * U) {
      float v[U][8];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int task = task0 + u * 2 * W + half;
        const int col = task / blocks, k = (task - col * blocks) * 128 + l16 * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[u][i] = 0.f;
        if (task < tasks && k < k_len) load8(row_of(col) + k, v[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int task = task0 + u * 2 * W + half;
        const int col = task / blocks, b = task - col * blocks;
        uint32_t m = 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[u][i]) & 0x7FFFFFFFu);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(~0u, m, o));
        float to, back;
        moe_act_scale(m, to, back);
        if (task < tasks) {
          uint8_t* block = bfrag + uint32_t(b * 4 + (l16 >> 2)) * piece;
          const bool planes = Cfg::BUSY && columns > kMoeBeside;
          const int at = GATE || planes ? col : col % kMoeBeside;
          uint8_t* to16 = block + at * 64 + (GATE || planes ? 0u : col / kMoeBeside * p.plane);
          auto put = [&](uint8_t* row, const uint32_t (&w)[4]) {
            if constexpr (MX) {
              // a lane's codes are 8 consecutive values
              *reinterpret_cast<uint4*>(row + (l16 & 3) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
              // a lane's codes are 4 consecutive values of each 16
              uint8_t* at = row + ((l16 >> 1) & 1) * 8 + (l16 & 1) * 32;
              *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[1]);
              *reinterpret_cast<uint2*>(at + 16) = make_uint2(w[2], w[3]);
            }
          };
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = pack_f16x2(v[u][2 * i] * to, v[u][2 * i + 1] * to);
          put(to16, w);
          if constexpr (!GATE) {  // (beside an infinity or a NaN nothing else counts)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              w[i] = m < 0x7F800000u ? f16x2_rest(v[u][2 * i] * to, v[u][2 * i + 1] * to, w[i]) : 0u;
            put(to16 + (planes ? p.plane : piece / 2), w);
          }
          if (l16 == 0) ts[b * kMoeChunk + col] = back;
        }
      }
    }
  };

  // Resident: all tokens (GATE) or pairs (DOWN) have a column of their own, laid
  // out once, and a chunk uses its pairs' columns; else a chunk's pairs are laid
  // out when a unit of it comes up.
  moe_select<THREADS>(p, route);
  if (GATE && resident && warp < W)
    fragments(p.T, p.H, [&](int t) { return static_cast<const T*>(p.x) + int64_t(t) * p.ldx; });
  // (scratch: the ring, before its first copy)
  moe_group<THREADS>(p, route, reinterpret_cast<uint32_t*>(smem),
                     resident ? p.T * p.top_k : GATE || Cfg::BUSY ? p.cols : kMoeBeside, !GATE && resident);

  if (GATE && blockIdx.x == 0)
    for (int i = tid; i < p.T * p.top_k; i += THREADS)
      p.routed[i] = make_float2(route.weight[i], __int_as_float(route.expert[i]));
  const int chunks = route.totals[0];
  const int tiles = GATE ? p.I / 8 : p.H / 16, per_chunk = tiles * p.segments;
  const int K = GATE ? p.H : p.I;
  // CTA b of G has units [x b / G, x (b + 1) / G) of all x = chunks * per_chunk;
  // with BUSY, places where a unit of five pairs or more counts 5 and others 4
  // (DOWN of MXFP4, 40 tokens, 10 of 52 chunks busy: 79 us, with 9 : 8 84, with 6 : 4
  // 81; block FP8 within 3% between 9 : 8 and 11 : 8).
  auto first_unit = [&](int b) {
    if constexpr (!Cfg::BUSY) {
      return int(int64_t(chunks) * per_chunk * b / gridDim.x);
    } else {
      auto busy_of = [&](int c) { return __ballot_sync(~0u, c < chunks && route.chunk_count[c] > kMoeBeside); };
      int total = 4 * chunks;
      for (int c = 0; c < chunks; c += 32) total += __popc(busy_of(c + lane));
      const int64_t place = int64_t(total) * per_chunk * b / gridDim.x;
      int64_t before = 0;
      for (int c = 0; c < chunks; c += 32) {
        const uint32_t busy = busy_of(c + lane);
        const int n = min(32, chunks - c), own = busy >> lane & 1u ? 5 : 4;
        const int64_t at = before + int64_t(4 * lane + __popc(busy & ((1u << lane) - 1u))) * per_chunk;
        const uint32_t mine = __ballot_sync(~0u, lane < n && place >= at && place < at + int64_t(own) * per_chunk);
        const int u = (c + lane) * per_chunk + int((place - at) / own);
        if (mine) return __shfl_sync(~0u, u, __ffs(mine) - 1);
        before += int64_t(4 * n + __popc(busy)) * per_chunk;
      }
      return chunks * per_chunk;
    }
  };
  const int u0 = first_unit(blockIdx.x), u1 = first_unit(blockIdx.x + 1);
  // The walk over this CTA's units, a row of up to G of them (one a group) with
  // the same chunk and K range at a time.
  struct Walk {
    int u, chunk, seg, tile, count;  // first unit, its place, units of the row
  };
  auto begin = [&]() {
    Walk w = {u0, u0 / per_chunk, u0 % per_chunk / tiles, u0 % per_chunk % tiles, 0};
    w.count = min(G, min(u1 - w.u, tiles - w.tile));
    return w;
  };
  auto next = [&](Walk& w) {
    w.u += w.count;
    w.tile += w.count;
    if (w.tile == tiles) {
      w.tile = 0;
      if (++w.seg == p.segments) w.seg = 0, ++w.chunk;
    }
    w.count = min(G, min(u1 - w.u, tiles - w.tile));
  };
  // Every group has a ring of S / G slots of its own.  (In one ring for all, a
  // slot would change groups from pass to pass, and a group ahead of another
  // could take the parity of the pass before last for its own.)
  const int ring = S / G, unit_stages = p.unit_stages;
  const int stage_blocks = p.box * (128 / BB);  // 128-wide K blocks of a stage

  if (warp >= W && warp < W + PRODUCERS) {
    // ---------------------------------------------------------------- producer
    // One lane issues, for every PRODUCERS-th group: a stage costs it several
    // hundred clocks of waits, addresses and the copy itself, and HBM delivers
    // one in 700.
    if (lane == 0) {
      const uint64_t policy = policy_evict_first(), scale_policy = policy_evict_normal();
      bool ok = true;
      int slot[G / PRODUCERS] = {};
      uint32_t pass[G / PRODUCERS] = {};
      for (Walk w = begin(); w.u < u1 && ok; next(w)) {
        const int expert = route.chunk_expert[w.chunk];
        const int first = w.seg * (p.seg_len / 128) * BB / 128;  // 128-byte columns
        const int last = first + (min(p.seg_len, K - w.seg * p.seg_len) * BB / 128 + 127) / 128;
        for (int i = 0, c = first; i < unit_stages && ok; ++i, c += p.box) {
          const int end = min(c + p.box, last);
#pragma unroll
          for (int k = 0; k < G / PRODUCERS; ++k) {
            const int g = warp - W + k * PRODUCERS;
            if (g >= w.count) break;
            const int s = g * ring + slot[k];
            if (pass[k] > 0 && !(ok = mbar_wait(empty(s), (pass[k] - 1) & 1u, abort_flag, kMoeWaitEmpty))) break;
            issued[s] = int(pass[k]) + 1;
            if (++slot[k] == ring) slot[k] = 0, ++pass[k];
            const int row = (w.tile + g) * (GATE ? 8 : 16), row_b = row + (GATE ? p.I : 8);
            const uint32_t to = base + uint32_t(s) * stage_bytes;
            if (end <= c) {  // a shorter last K range: nothing left
              mbar_arrive(full(s));
              continue;
            }
            // A short last column is read past the row's end, into the next
            // row: consumers stop at K.  Behind the stack's last row there may
            // be nothing to read.
            if (end <= p.columns || (p.tail_reads_on && (expert < p.E - 1 || row_b + 8 < p.rows))) {
              mbar_arrive_expect_tx(full(s), 2u * (half_bytes + scale_copy));
              tma_load_5d(to, &p.map_w, 0, row, c, 0, expert, full(s), policy);
            } else {  // column by column, zeros past the row
              mbar_arrive_expect_tx(full(s), uint32_t(end - c) * 2048u + 2u * scale_copy);
              for (int j = c; j < end; ++j) {
                tma_load_3d(to + uint32_t(j - c) * 1024u, &p.map_tail, j * 128, row, expert, full(s), policy);
                tma_load_3d(to + half_bytes + uint32_t(j - c) * 1024u, &p.map_tail, j * 128, row_b, expert, full(s), policy);
              }
            }
            if constexpr (MX) {
              // A K block's scale words of 8 rows are 128 contiguous bytes of
              // its tile, each next to the words of the rows 32, 64 and 96
              // further on: a fourth is used here, the rest by the units that
              // follow (from L2).
              tma_load_5d(to + 2u * half_bytes, &p.map_s, (row & 31) * 16, 2 * c, row >> 7, 0, expert, full(s), scale_policy);
              if (!p.scales_together)
                tma_load_5d(to + 2u * half_bytes + scale_copy, &p.map_s, (row_b & 31) * 16, 2 * c, row_b >> 7, 0, expert,
                            full(s), scale_policy);
            }
          }
        }
      }
    }
    __syncwarp();
    // Every copy this warp issued lands before the CTA may exit (the consumers
    // have waited for them all, unless a wait gave up).
    if (lane < S && moe_producer_of(lane, ring, PRODUCERS) == warp - W && issued[lane] > 0)
      mbar_wait(full(lane), uint32_t(issued[lane] - 1) & 1u, nullptr, kMoeWaitDrain);
    __syncwarp();
  } else if (warp < W) {
    // ---------------------------------------------------------------- consumers
    const int g = lane >> 2, t4 = lane & 3;
    auto column = [&](int n) { return min(g % kMoeBeside, n - 1) + (g < kMoeBeside ? 0 : n); };  // n and n, upper and lower
    const uint32_t b_lane = base + p.off_b + uint32_t((GATE ? min(g, p.cols - 1) : column(p.cols / 2)) * 64 + t4 * 16);
    constexpr int kStep = kMoeGroupWarps;
    const int group = warp / kStep, warp_in_group = warp % kStep;
    const uint32_t a_lane = ((lane >> 3) & 1) * half_bytes + (lane & 7) * 128u;
    int have = -1, count = 0, done = 0, slot = 0;
    uint32_t phase = 0u;
    bool ok = true;
    // Block FP8 scales: lane l holds those of K blocks l and l + 32 of the
    // unit's two 8-row halves, requested a unit ahead where they change.  (DOWN:
    // both halves have the same, and a K range at most 32 blocks.)
    constexpr int SC = GATE ? 2 : 1;
    float sc[SC][SC] = {}, sc_next[SC][SC] = {};
    auto load_scales = [&](int chunk, int seg, int tile) {
      const float* e = static_cast<const float*>(p.ws) + int64_t(route.chunk_expert[chunk]) * p.rb * p.kb;
      const int kb = seg * (p.seg_len / 128);
#pragma unroll
      for (int half = 0; half < SC; ++half) {
        const int r = GATE ? half * p.I + tile * 8 : tile * 16;
#pragma unroll
        for (int j = 0; j < SC; ++j) {
          const int b = kb + lane + 32 * j;
          sc_next[half][j] = b < p.kb ? ldg_pinned(e + int64_t(r >> 7) * p.kb + b) : 0.f;
        }
      }
    };
    MoeStage st;
    st.words = 2u * half_bytes;
    st.a_lane = a_lane, st.piece = piece, st.low = p.plane;
    st.b_cols = b_lane, st.ts = ts + 2 * t4;
    bool busy = false;
    int columns_of = -1;
    Walk w = begin();
    if (!MX && w.u < u1 && group < w.count) load_scales(w.chunk, w.seg, w.tile + group);
    for (; w.u < u1; next(w)) {
      const int chunk = w.chunk, seg = w.seg, tile = w.tile + group;
      const int k_len = min(p.seg_len, K - seg * p.seg_len);
      const int blocks = (k_len + 127) / 128;
      const int key = resident ? seg : chunk * p.segments + seg;
      if (have != key) {
        count = resident ? p.T * p.top_k : route.chunk_count[chunk];
        if (!GATE || !resident) {
          if constexpr (!GATE) griddep_wait();  // h
          named_bar_sync(1, 32 * W);  // every warp is done with the last ones
          fragments(count, k_len, [&](int col) {
            const int pair = resident ? col : route.list[route.chunk_first[chunk] + col];
            if constexpr (GATE) return static_cast<const T*>(p.x) + int64_t(pair / p.top_k) * p.ldx;
            else return p.h + int64_t(pair) * p.I + seg * p.seg_len;
          });
          named_bar_sync(1, 32 * W);
        }
        have = key;
      }
      if constexpr (!MX) {
#pragma unroll
        for (int half = 0; half < SC; ++half)
#pragma unroll
          for (int j = 0; j < SC; ++j) sc[half][j] = sc_next[half][j];
        // the next row's unit of this group (if it has none, what is loaded is not used)
        Walk v = w;
        next(v);
        if (v.u < u1) {
          const int t = v.tile + min(group, v.count - 1);
          const bool same = group < w.count && v.chunk == chunk && v.seg == seg &&
                            (GATE ? t >> 4 == tile >> 4 && (p.I + t * 8) >> 7 == (p.I + tile * 8) >> 7 : t >> 3 == tile >> 3);
          if (!same) load_scales(v.chunk, v.seg, t);
        }
      }
      if (group >= w.count) continue;
      if (!GATE && columns_of != chunk) {  // which four pairs' plane, and the scales of columns 2 t4 mod 4
        columns_of = chunk;
        busy = Cfg::BUSY && count > kMoeBeside;
        const int set = resident ? route.list[route.chunk_first[chunk]] / kMoeBeside : 0;
        st.b_cols = b_lane + set * p.plane;
        st.ts = ts + (busy ? 2 * t4 : 2 * (t4 & 1) + kMoeBeside * set);
      }
      // MXFP4: the 32-row quarter of the rows' scale tiles
      const uint32_t word_a = uint32_t(((GATE ? tile * 8 : tile * 16) >> 5) & 3) * 4u;
      const uint32_t word_b = scale_copy + uint32_t(((GATE ? p.I + tile * 8 : tile * 16 + 8) >> 5) & 3) * 4u;
      st.word_a = word_a, st.word_b = word_b;
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      for (int b0 = 0; b0 < unit_stages * stage_blocks; b0 += stage_blocks) {
        const int s = group * ring + slot;
        ok = mbar_wait(full(s), phase, abort_flag, kMoeWaitFull) && ok;
        const int nb = min(stage_blocks, blocks - b0);
        st.base = base + uint32_t(s) * stage_bytes;
        st.b0 = b0;
        // Blocks are dealt over the whole unit, so that no warp has two more than
        // another.
        int i = (warp_in_group - b0) & (kStep - 1);
        if (Cfg::BUSY && busy) {
          for (; i < nb; i += kStep) {
            const int steps = (k_len - (b0 + i) * 128) / 32;
            if (steps >= 4) moe_stage_block<Cfg, true, Cfg::BUSY>(st, i, 4, sc, acc);
            else moe_stage_block<Cfg, false, Cfg::BUSY>(st, i, steps, sc, acc);
          }
        } else {
          // Whole blocks two at a time (their loads and MMA chains overlap),
          // then what is left; the last block of K may be short.
          const int whole = min(nb, (k_len - b0 * 128) / 128);
          for (; i + kStep < whole; i += 2 * kStep) {
            moe_stage_block<Cfg, true, false>(st, i, 4, sc, acc);
            moe_stage_block<Cfg, true, false>(st, i + kStep, 4, sc, acc);
          }
          for (; i < nb; i += kStep) {
            if (i < whole) moe_stage_block<Cfg, true, false>(st, i, 4, sc, acc);
            else moe_stage_block<Cfg, false, false>(st, i, (k_len - (b0 + i) * 128) / 32, sc, acc);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty(s));
        if (++slot == ring) slot = 0, phase ^= 1u;
      }
      // ---- this warp's sums of the unit
      const int buf = done % RB;
      if (done >= RB) ok = mbar_wait(red_empty(group, buf), uint32_t(done / RB - 1) & 1u, abort_flag, kMoeWaitRedEmpty) && ok;
      ++done;
      reinterpret_cast<float4*>(smem + p.off_red)[(buf * W + warp) * 32 + lane] =
          make_float4(acc[0], acc[1], acc[2], acc[3]);
      __syncwarp();
      if (lane == 0) mbar_arrive(red_full(group, buf));
    }
  } else {
    // ---------------------------------------------------------------- finisher
    const int g = lane >> 2, t4 = lane & 3;
    if constexpr (!GATE) {
      griddep_wait();  // z
      griddep_launch_dependents();
    }
    uint32_t done[G] = {};
    Walk w = begin();
    bool ok = true;
    for (; w.u < u1 && ok; next(w)) {
#pragma unroll
      for (int group = 0; group < G; ++group) {
        if (group >= w.count) break;
        const int chunk = w.chunk, seg = w.seg, tile = w.tile + group;
        const int buf = int(done[group] % RB);
        ok = mbar_wait(red_full(group, buf), done[group] / RB & 1u, abort_flag, kMoeWaitRedFull);
        ++done[group];
        const int count = route.chunk_count[chunk];
        const short* pairs = route.list + route.chunk_first[chunk];
        const float4* red =
            reinterpret_cast<const float4*>(smem + p.off_red) + (buf * W + group * kMoeGroupWarps) * 32 + lane;
        float4 v = red[0];
#pragma unroll
        for (int j = 1; j < kMoeGroupWarps; ++j) {
          const float4 a = red[j * 32];
          v.x += a.x, v.y += a.y, v.z += a.z, v.w += a.w;
        }
        auto store = [&](int pair, float a, float b) {  // row g of either half
          if constexpr (GATE) {
            p.h[int64_t(pair) * p.I + tile * 8 + g] = a / (1.f + expf(-a)) * b;
          } else {
            float* z = p.z + (int64_t(pair) * p.segments + seg) * p.H + tile * 16 + g;
            z[0] = a;
            z[8] = b;
          }
        };
        // this lane has columns 2 t4 and the next
        if (!GATE && (!Cfg::BUSY || count <= kMoeBeside)) {  // the lower parts are four columns further on
          v.x += __shfl_down_sync(~0u, v.x, 2), v.y += __shfl_down_sync(~0u, v.y, 2);
          v.z += __shfl_down_sync(~0u, v.z, 2), v.w += __shfl_down_sync(~0u, v.w, 2);
        }
        if (resident) {
          for (int k = 0; k < count; ++k) {
            const int col = GATE ? pairs[k] / p.top_k : pairs[k] % kMoeBeside;
            if (col >> 1 == t4) store(pairs[k], col & 1 ? v.y : v.x, col & 1 ? v.w : v.z);
          }
        } else {
          if (2 * t4 < count) store(pairs[2 * t4], v.x, v.z);
          if (2 * t4 + 1 < count) store(pairs[2 * t4 + 1], v.y, v.w);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(red_empty(group, buf));
        // (The lanes agree on a wait that gave up here, off the path to the stores:
        // a vote behind the wait took 0.6 of 28 us for one token.)
        if (!(ok = __all_sync(~0u, ok))) break;
      }
    }
  }
}

}  // namespace bfp8
