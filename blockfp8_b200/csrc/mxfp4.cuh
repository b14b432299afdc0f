// MXFP4 (OCP microscaling, 4 bit): e2m1 codes with one power-of-two scale
// (E8M0: a biased exponent byte) per 32 consecutive values of a row.
//
//   e    = max(floor(log2(amax of the 32)) - 2, -127)     byte = e + 127
//   code = e2m1(x * 2^-e), to nearest even, at most 6 in magnitude
//
// so the largest value of a block lands in [4, 8).  x * 2^-e is exact (a
// product with a power of two), so the one rounding is the conversion's own.
// A block that holds an infinity or a NaN gets the byte 255 (E8M0's NaN) and
// zero codes: all of it reads back as NaN.
//
// Operands:
//   codes   [R, K / 2] bytes, value 2j in the low nibble of byte j
//   scales  [ceil(R / 128), ceil(K / 128), 32, 16] bytes: the 512 bytes of a
//           128-row x 128-column tile are what one tcgen05.cp.32x128b.warpx4
//           brings into tensor memory, row r of the tile at [r % 32], its four
//           bytes (four 32-wide blocks) at 4 (r / 32).  Rows and blocks past
//           the matrix hold zeros.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "ptx.cuh"
#include "quant_math.cuh"

namespace bfp8 {

struct Mxfp4QuantParams {
  const void* x;  // [M, K] bf16, fp16 or fp32
  int64_t ldx;
  uint8_t* q;  // [M, K / 2], row stride ldq
  int64_t ldq;
  uint8_t* s;  // [m_tiles, k_tiles, 32, 16]
  int M, K;
  int m_tiles, k_tiles;
  int trigger;  // let the dependent kernel start early (it waits before it reads q and s)
};

struct Mxfp4DequantParams {
  const uint8_t* q;
  int64_t ldq;
  const uint8_t* s;
  void* y;  // [M, K] bf16 or fp32
  int64_t ldy;
  int M, K;
  int m_tiles, k_tiles;
};

// 2^(127 - byte) for byte <= 253 (a normal float).
__device__ __forceinline__ float e8m0_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
// 2^(byte - 127); 2^-127 is subnormal, 255 is NaN.
__device__ __forceinline__ float e8m0_value(uint32_t byte) {
  return byte == 255u ? __uint_as_float(0x7FC00000u) : __uint_as_float(byte ? byte << 23 : 0x00400000u);
}

// Four e2m1 pairs to a 32-bit word, value 0 in the lowest nibble.
__device__ __forceinline__ uint32_t e2m1x8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
// The eight values of a 32-bit word of codes, as f16 pairs (exact).
__device__ __forceinline__ void e2m1x8_to_f16(uint32_t codes, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(codes));
}

// Eight consecutive values as floats.
template <class T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      bf16x8_to_float(u, v);
    } else {
      const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(h[i]);
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
      }
    }
  }
}

// The scale byte of a block from the bits of its largest magnitude.
__device__ __forceinline__ uint32_t mxfp4_scale_byte(uint32_t amax_bits) {
  const uint32_t ef = amax_bits >> 23;  // floor(log2) + 127; 0 for subnormals
  return ef == 255u ? 255u : (ef > 2u ? ef - 2u : 0u);
}

constexpr int kMxThreads = 256;

// A warp takes rows r, r + 32, r + 64, r + 96 of a 128-row tile over 256
// columns: lane l holds values 8 l .. 8 l + 7 of each, a block is four lanes,
// and the four rows' scale bytes of a K tile are 16 contiguous bytes.  Four
// independent loads per lane.  24576 x 4096 bf16: 54 us (4.7 TB/s), where the
// schedulers issue in 0.72 of the clocks (maxima, scaling, conversion) and HBM is at
// 0.52 of its peak; and 39 us (6.5 TB/s) back.  A warp a task: a grid of resident
// CTAs that loop took 3 us longer for the two.
template <class T>
__global__ void __launch_bounds__(kMxThreads) mxfp4_quantize_kernel(const Mxfp4QuantParams p) {
  // The wait comes first: a dependent that has started may then read whatever
  // earlier kernels wrote (the GEMM of linear_mxfp4 its weights) at once.  As
  // this kernel may be the one that writes such weights, it triggers only
  // inside linear_mxfp4.
  griddep_wait();
  if (p.trigger) griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int chunks = (p.k_tiles + 1) / 2;
  const uint32_t tasks = uint32_t(p.m_tiles) * 32u * uint32_t(chunks);
  const uint32_t task = blockIdx.x * (kMxThreads / 32) + (threadIdx.x >> 5);
  if (task < tasks) {
    const int rows = int(task / uint32_t(chunks)), chunk = int(task) - rows * chunks;  // (row tile, r)
    const int r = rows & 31, mt = rows >> 5;
    const int col = chunk * 256 + lane * 8;
    const bool col_ok = col < p.K;
    float v[4][8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = mt * 128 + r + 32 * j;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[j][i] = 0.f;
      if (col_ok && row < p.M) load8(static_cast<const T*>(p.x) + int64_t(row) * p.ldx + col, v[j]);
    }
    uint32_t bytes[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // the largest magnitude by its bits: a NaN stays the largest
      uint32_t m = 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[j][i]) & 0x7FFFFFFFu);
      m = max(m, __shfl_xor_sync(~0u, m, 1));
      m = max(m, __shfl_xor_sync(~0u, m, 2));
      bytes[j] = mxfp4_scale_byte(m);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = mt * 128 + r + 32 * j;
      const float inv = e8m0_inverse(min(bytes[j], 253u));
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = v[j][i] * inv;
      if (col_ok && row < p.M)
        *reinterpret_cast<uint32_t*>(p.q + int64_t(row) * p.ldq + col / 2) = bytes[j] == 255u ? 0u : e2m1x8(w);
    }
    // 16 scale bytes of a K tile from its 16 lanes: lane 4 b holds block b.
    uint32_t word[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t w = bytes[j] << (8 * ((lane >> 2) & 3));
      w |= __shfl_xor_sync(~0u, w, 4);
      w |= __shfl_xor_sync(~0u, w, 8);
      word[j] = w;
    }
    const int kt = chunk * 2 + (lane >> 4);
    if ((lane & 15) == 0 && kt < p.k_tiles)
      *reinterpret_cast<uint4*>(p.s + ((int64_t(mt) * p.k_tiles + kt) * 32 + r) * 16) =
          make_uint4(word[0], word[1], word[2], word[3]);
  }
}

// The values the codes stand for: the same walk, backwards.  A code times a
// power of two is exact in both output types.
template <class T>
__global__ void __launch_bounds__(kMxThreads) mxfp4_dequantize_kernel(const Mxfp4DequantParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int chunks = (p.k_tiles + 1) / 2;
  const uint32_t tasks = uint32_t(p.m_tiles) * 32u * uint32_t(chunks);
  const uint32_t task = blockIdx.x * (kMxThreads / 32) + (threadIdx.x >> 5);
  if (task < tasks) {
    const int rows = int(task / uint32_t(chunks)), chunk = int(task) - rows * chunks;
    const int r = rows & 31, mt = rows >> 5;
    const int col = chunk * 256 + lane * 8;
    if (col >= p.K) return;
    const int kt = col >> 7, shift = 8 * ((lane >> 2) & 3);
    const uint4 words = *reinterpret_cast<const uint4*>(p.s + ((int64_t(mt) * p.k_tiles + kt) * 32 + r) * 16);
    const uint32_t word[4] = {words.x, words.y, words.z, words.w};
    uint32_t codes[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = mt * 128 + r + 32 * j;
      codes[j] = row < p.M ? *reinterpret_cast<const uint32_t*>(p.q + int64_t(row) * p.ldq + col / 2) : 0u;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = mt * 128 + r + 32 * j;
      if (row >= p.M) continue;
      const float scale = e8m0_value((word[j] >> shift) & 255u);
      uint32_t h[4];
      e2m1x8_to_f16(codes[j], h);
      float f[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 pair = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        f[2 * i] = pair.x * scale, f[2 * i + 1] = pair.y * scale;
      }
      T* y = static_cast<T*>(p.y) + int64_t(row) * p.ldy + col;
      if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(y)[0] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4*>(y)[1] = make_float4(f[4], f[5], f[6], f[7]);
      } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&b);
        }
        *reinterpret_cast<uint4*>(y) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
}

}  // namespace bfp8
