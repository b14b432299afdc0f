// Host side of the MXFP4 operators and the expert layer: checks, launch
// shapes and the C ABI (include/blockfp8_b200.h).  Included by capi.cu.
#pragma once

namespace bfp8 {
namespace {

// Raise a kernel's shared-memory limit once per device.
int allow_smem(const void* kernel, int bytes, int dev, std::atomic<uint64_t>& done) {
  const uint64_t bit = dev < 64 ? (uint64_t(1) << dev) : 0;
  if (bit && (done.load(std::memory_order_acquire) & bit)) return BFP8_OK;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
  if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute");
  done.fetch_or(bit, std::memory_order_release);
  return BFP8_OK;
}

int element_size(int type) { return type == 0 ? 4 : 2; }

int round_up(int x, int m) { return cdiv(x, m) * m; }

// Sizes whose rounding up to tiles stays in 32 bits.
constexpr int kMxMaxSize = INT32_MAX / 2;

// ---- MXFP4 quantization -----------------------------------------------------------

int check_codes(const void* q, int64_t ldq, const void* s, int M, int K) {
  if (M < 0 || K <= 0 || K % 32 != 0) return fail(BFP8_EINVAL, "K must be a positive multiple of 32");
  if (M > kMxMaxSize || K > kMxMaxSize) return fail(BFP8_EINVAL, "too large");
  if (M == 0) return BFP8_OK;
  if (!q || !s) return fail(BFP8_EINVAL, "null operand pointer");
  if (!aligned16(q) || !aligned16(s) || ldq < K / 2 || ldq % 16 != 0)
    return fail(BFP8_EINVAL, "codes must be row-major with 16-byte aligned rows, scales 16-byte aligned");
  return BFP8_OK;
}

int launch_mx(const void* kernel, int m_tiles, int k_tiles, void** args, cudaStream_t stream, const char* what) {
  const int64_t tasks = int64_t(m_tiles) * 32 * cdiv(k_tiles, 2);
  if (tasks > INT32_MAX) return fail(BFP8_EINVAL, "too many rows x columns for one launch");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned((tasks + kMxThreads / 32 - 1) / (kMxThreads / 32)));
  cfg.blockDim = dim3(kMxThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  set_pdl(cfg, attr);
  cudaError_t e = cudaLaunchKernelExC(&cfg, kernel, args);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, what);
  return BFP8_OK;
}

// ---- MXFP4 GEMM -------------------------------------------------------------------

constexpr int kMxPairSmem = 112 * 1024;  // two CTAs on an SM

// K parts of a tile: more while the CTAs still fit two to an SM and each has
// two stages.
int mx_splits(int64_t tiles, int k_stages, int num_sms) {
  int splits = 1;
  while (splits < 8 && tiles * splits <= num_sms && k_stages >= splits * 4) splits *= 2;
  return splits;
}

template <class Cfg>
int launch_mx_gemm(const bfp8_mxfp4_gemm_problem& p, int x_type, int dev, int num_sms, cudaStream_t stream) {
  static std::atomic<uint64_t> done{0};
  const void* kernel = reinterpret_cast<const void*>(&mx_gemm_kernel<Cfg>);
  if (int r = allow_smem(kernel, kMxPairSmem, dev, done)) return r;
  MxGemmParams gp;
  std::memset(&gp, 0, sizeof(gp));
  if (int r = make_map(&gp.map_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.b, uint64_t(p.K / 2), uint64_t(p.N), uint64_t(p.ldb),
                       128, 128, CU_TENSOR_MAP_SWIZZLE_128B))
    return r;
  if (Cfg::QUANT) {
    if (int r = make_map(&gp.map_x, CU_TENSOR_MAP_DATA_TYPE_UINT16, p.a, uint64_t(p.K), uint64_t(p.M),
                         uint64_t(p.lda) * 2, 256, uint32_t(p.M), CU_TENSOR_MAP_SWIZZLE_NONE))
      return r;
  } else {
    if (int r = make_map(&gp.map_x, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.a, uint64_t(p.K / 2), uint64_t(p.M),
                         uint64_t(p.lda), 128, Cfg::BN, CU_TENSOR_MAP_SWIZZLE_128B))
      return r;
  }
  gp.sw = static_cast<const uint8_t*>(p.sb);
  gp.sx = static_cast<const uint8_t*>(p.sa);
  gp.c = static_cast<__nv_bfloat16*>(p.c);
  gp.ldc = p.ldc;
  gp.M = p.M;
  gp.N = p.N;
  gp.K = p.K;
  gp.n_tiles = cdiv(p.N, 128);
  gp.m_tiles = cdiv(p.M, Cfg::BN);
  gp.k_tiles = cdiv(p.K, 128);
  gp.k_stages = cdiv(p.K, 256);
  gp.early = p.weights_ready && g_weight_prefetch.load(std::memory_order_relaxed);
  gp.half = x_type == 2;
  gp.raw_bytes = Cfg::QUANT ? p.M * 512 : 0;
  gp.stage_bytes = round_up(Cfg::TILE_BYTES + gp.raw_bytes, 1024);
  gp.stages = std::min(Cfg::MAX_STAGES, (kMxPairSmem - 1024 - Cfg::BAR_BYTES) / gp.stage_bytes);
  const int smem = 1024 + std::max(gp.stages * gp.stage_bytes, Cfg::SUM_BYTES) + Cfg::BAR_BYTES;
  const int64_t tiles = int64_t(gp.n_tiles) * gp.m_tiles;
  gp.splits = mx_splits(tiles, gp.k_stages, num_sms);
  if (tiles * gp.splits > INT32_MAX) return fail(BFP8_EINVAL, "too many tiles for one launch");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(tiles * gp.splits));
  cfg.blockDim = dim3(Cfg::THREADS);
  cfg.dynamicSmemBytes = size_t(smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  set_pdl(cfg, attr);
  if (gp.splits > 1) {
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = unsigned(gp.splits);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  }
  cudaError_t e = cudaLaunchKernelEx(&cfg, mx_gemm_kernel<Cfg>, gp);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "MXFP4 GEMM launch");
  return BFP8_OK;
}

// 256 x 256 tiles by CTA pairs.
int launch_mx_pair(const bfp8_mxfp4_gemm_problem& p, int dev, int num_sms, cudaStream_t stream) {
  static std::atomic<uint64_t> done{0};
  if (int r = allow_smem(reinterpret_cast<const void*>(&mx_pair_kernel), MxPairCfg::SMEM_BYTES, dev, done)) return r;
  MxPairParams gp;
  std::memset(&gp, 0, sizeof(gp));
  const uint64_t scale_row = uint64_t(cdiv(p.K, 128)) * 512;
  const auto u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8, i32 = CU_TENSOR_MAP_DATA_TYPE_INT32;
  const auto sw128 = CU_TENSOR_MAP_SWIZZLE_128B, plain = CU_TENSOR_MAP_SWIZZLE_NONE;
  int r = make_map(&gp.map_x, u8, p.a, uint64_t(p.K / 2), uint64_t(p.M), uint64_t(p.lda), 128, 128, sw128);
  if (!r) r = make_map(&gp.map_w, u8, p.b, uint64_t(p.K / 2), uint64_t(p.N), uint64_t(p.ldb), 128, 128, sw128);
  if (!r) r = make_map(&gp.map_sx, i32, p.sa, scale_row / 4, uint64_t(cdiv(p.M, 128)), scale_row, 256, 1, plain);
  if (!r) r = make_map(&gp.map_sw, i32, p.sb, scale_row / 4, uint64_t(cdiv(p.N, 128)), scale_row, 256, 2, plain);
  if (!r) r = make_map(&gp.map_c, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, p.c, uint64_t(p.N), uint64_t(p.M), uint64_t(p.ldc) * 2, 32, 128, CU_TENSOR_MAP_SWIZZLE_64B);
  if (r) return r;
  gp.K = p.K;
  gp.k_stages = cdiv(p.K, 256);
  gp.m_tiles = cdiv(p.M, 256);
  gp.n_tiles = cdiv(p.N, 256);
  gp.early = p.weights_ready && g_weight_prefetch.load(std::memory_order_relaxed);
  const int64_t tiles = int64_t(gp.m_tiles) * gp.n_tiles;
  if (tiles > INT32_MAX / 8) return fail(BFP8_EINVAL, "too many tiles for one launch");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2 * unsigned(std::min<int64_t>(tiles, num_sms / 2)));
  cfg.blockDim = dim3(MxPairCfg::THREADS);
  cfg.dynamicSmemBytes = MxPairCfg::SMEM_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  set_pdl(cfg, attr);
  cudaError_t e = cudaLaunchKernelEx(&cfg, mx_pair_kernel, gp);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "MXFP4 GEMM launch");
  return BFP8_OK;
}

// ---- the expert layer ---------------------------------------------------------------

constexpr int kMoeMaxHidden = 8192;
constexpr int kMoeMaxInner = 1 << 24;
constexpr int kMoeSegment = 4096;  // most K values whose activations DOWN keeps in shared memory
constexpr int kMoeBusySegment = 2048;  // the same in two planes: 64 KB, which leaves the ring its depth
constexpr int kMoeHalfSmem = 113 * 1024;
constexpr int kMoeSharedSmem = 226 * 1024;  // of two CTAs on an SM, without what the system takes

// How one kernel's units (segments of seg_len values of K) and shared memory
// are laid out.
struct MoeLayout {
  int segments, seg_len, box, unit_stages, stages, smem, cols, resident;
  uint32_t off_b, off_ts, off_red, off_route, off_bars, plane;
};

// K of `k` values in `segments` ranges, `entries` tokens or pairs that could
// have a column of their own (DOWN: two), in stages of up to max_box 128-byte
// columns and within `limit` bytes of shared memory.
bool moe_layout(const bfp8_moe_problem& p, int k, int segments, int entries, bool down, int warps, int max_box, int limit,
                MoeLayout* out) {
  const int P = p.T * p.top_k, per_column = p.format ? 256 : 128;  // values of a 128-byte column
  const int columns = cdiv(cdiv(k, per_column), segments), unit_stages = cdiv(columns, max_box);
  out->box = cdiv(columns, unit_stages);
  out->unit_stages = unit_stages;
  out->seg_len = segments == 1 ? columns * per_column : unit_stages * out->box * per_column;
  out->segments = cdiv(k, out->seg_len);
  // (DOWN's second four pairs take a plane of their own: beyond 64 KB that costs
  // the ring more than laying out each chunk's pairs: MXFP4, 2 tokens, 64 experts,
  // top 4, H = I = 2880: 55 us against 47.)
  out->resident = entries <= kMoeChunk && (!down || (warps == 8 && (entries <= kMoeBeside || k <= kMoeBusySegment)));
  out->cols = down ? (out->resident ? 2 * std::min(entries, kMoeBeside) : kMoeChunk)
                   : out->resident ? entries : std::min(P, kMoeChunk);
  const int planes = !down ? 1 : out->resident ? cdiv(entries, kMoeBeside) : warps == 8 ? 1 : 2;
  const int blocks = cdiv(std::min(k, out->seg_len), 128);
  const int stage = round_up(out->box * (2048 + (p.format ? 512 : 0)), 1024);
  const int b = blocks * 256 * out->cols * planes, ts = blocks * kMoeChunk * 4;
  const int red = kMoeRedBufs * warps * 512, route = round_up(moe_route_bytes(P), 16);
  const int scratch = P > 32 ? p.E * (cdiv(P, 32) + 1) * 4 : 0;
  auto end_of = [&](int stages) { return 8 * (2 * stages + 2 * warps / kMoeGroupWarps * kMoeRedBufs) + 16 + 4 * stages; };
  const int fixed = 1024 + b + ts + red + route + end_of(16);
  const int groups = warps / kMoeGroupWarps;
  const int stages = std::min(16, (limit - fixed) / stage) / groups * groups;
  if (stages < 2 * groups) return false;
  // the routing scratch lies where the ring and, unless they come first, the activations do
  const int ring = std::max(stages * stage, round_up(scratch - (out->resident ? 0 : b), 128));
  if (fixed + ring > limit) return false;
  out->stages = stages;
  out->off_b = uint32_t(ring);
  out->plane = uint32_t(b / planes);
  out->off_ts = out->off_b + uint32_t(b);
  out->off_red = out->off_ts + uint32_t(ts);
  out->off_route = out->off_red + uint32_t(red);
  out->off_bars = out->off_route + uint32_t(route);
  out->smem = 1024 + int(out->off_bars) + end_of(stages);
  return true;
}

struct MoeShape {
  int warps;  // consumers
  MoeLayout gate, down;
};

bool moe_layouts(const bfp8_moe_problem& p, MoeShape* s) {
  const int P = p.T * p.top_k;
  auto one = [&](int k, int ranges, int entries, bool down, int warps, int limit, MoeLayout* lay) {
    s->warps = warps;
    for (int box = 8; box >= 1; box /= 2)
      if (moe_layout(p, k, ranges, entries, down, warps, box, limit, lay)) return true;
    return false;
  };
  // Up to 8 tokens: GATE in half an SM's shared memory and DOWN in what it
  // leaves, so that DOWN starts beside GATE and requests its weights while GATE
  // runs.
  if (p.T <= 8 && one(p.H, 1, p.T, false, 8, kMoeHalfSmem, &s->gate) &&
      one(p.I, cdiv(p.I, kMoeSegment), P, true, 8, kMoeSharedSmem - s->gate.smem, &s->down))
    return true;
  return one(p.H, 1, p.T, false, 16, kMaxSmem, &s->gate) && one(p.I, cdiv(p.I, kMoeBusySegment), P, true, 16, kMaxSmem, &s->down);
}

int moe_shape(const bfp8_moe_problem& p, MoeShape* s) {
  if (!moe_layouts(p, s)) return fail(BFP8_EINVAL, "this expert layer's activations do not fit shared memory");
  // every pair could be a chunk of its own
  const int64_t units = int64_t(p.T) * p.top_k * std::max<int64_t>(p.I / 8, int64_t(p.H / 16) * s->down.segments);
  if (units > INT32_MAX) return fail(BFP8_EINVAL, "too many units for one launch: fewer tokens or choices for an I this large");
  return BFP8_OK;
}

// Tensor maps of one stack of expert weights [E, rows, k] and its scales.
// A unit takes 8 rows and the 8 rows `half` further on.
int moe_maps(MoeParams& mp, const MoeLayout& lay, int format, const void* w, int64_t w_expert, int64_t w_row,
             const void* scales, int E, int rows, int half, int k) {
  const uint64_t bytes = uint64_t(format ? k / 2 : k), full = bytes / 128;
  mp.columns = int(full);
  mp.rows = rows;
  if (E == 1) w_expert = w_row * rows;  // one expert's stride says nothing
  auto fn = encode_fn();
  if (!fn) return fail(BFP8_ECUDA, "cuTensorMapEncodeTiled is not available from the driver");
  auto encode = [&](CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
                    const cuuint32_t* box, CUtensorMapSwizzle swizzle) {
    const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, cuuint32_t(rank), const_cast<void*>(base), dims, strides, box, ones,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(BFP8_ECUDA, "cuTensorMapEncodeTiled failed (" + std::to_string(int(r)) + ")");
    return int(BFP8_OK);
  };
  // A short last column may be read past a row's end: another row of the stack
  // follows in memory, but for the last one.
  mp.tail_reads_on = bytes % 128 != 0;
  const uint64_t columns = full + (mp.tail_reads_on ? 1 : 0);
  if (columns > 0) {  // [128 bytes][rows][columns][halves][experts]
    const cuuint64_t dims[5] = {128, cuuint64_t(rows - half), columns, 2, cuuint64_t(E)};
    const cuuint64_t strides[4] = {cuuint64_t(w_row), 128, cuuint64_t(w_row) * half, cuuint64_t(w_expert)};
    const cuuint32_t box[5] = {128, 8, cuuint32_t(lay.box), 2, 1};
    if (int r = encode(&mp.map_w, w, 5, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return r;
  }
  if (bytes % 128) {
    const cuuint64_t dims[3] = {bytes, cuuint64_t(rows), cuuint64_t(E)};
    const cuuint64_t strides[2] = {cuuint64_t(w_row), cuuint64_t(w_expert)};
    const cuuint32_t box[3] = {128, 8, 1};
    if (int r = encode(&mp.map_tail, w, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B)) return r;
  }
  mp.rb = cdiv(rows, 128);
  mp.kb = cdiv(k, 128);
  mp.ws = scales;
  if (format) {  // [512 bytes of a tile][K blocks][row tiles][halves][experts]
    mp.scales_together = half == 8 || half % 128 == 0;
    const uint64_t tiles = uint64_t(mp.kb) * 512;  // bytes of a row of tiles
    const cuuint64_t dims[5] = {512, cuuint64_t(mp.kb), cuuint64_t(mp.rb), mp.scales_together ? 2u : 1u, cuuint64_t(E)};
    const cuuint64_t strides[4] = {512, tiles, half == 8 ? 128 : std::max(1, half / 128) * tiles, tiles * mp.rb};
    const cuuint32_t box[5] = {128, cuuint32_t(2 * lay.box), 1, mp.scales_together ? 2u : 1u, 1};
    if (int r = encode(&mp.map_s, scales, 5, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE)) return r;
  }
  return BFP8_OK;
}

int check_moe(const bfp8_moe_problem& p) {
  if (p.T < 1 || p.T > kMoeMaxTokens) return fail(BFP8_EINVAL, "the expert layer takes 1 to 64 tokens");
  if (p.H < 32 || p.H % 32 || p.H > kMoeMaxHidden)
    return fail(BFP8_EINVAL, "H must be a multiple of 32, at most 8192");
  if (p.I < 32 || p.I % 32 || p.I > kMoeMaxInner) return fail(BFP8_EINVAL, "I must be a positive multiple of 32, at most 2^24");
  if (p.E < 1 || p.E > kMoeMaxExperts) return fail(BFP8_EINVAL, "1 to 512 experts");
  if (p.top_k < 1 || p.top_k > kMoeMaxTopK || p.top_k > p.E)
    return fail(BFP8_EINVAL, "top_k must be at least 1 and at most min(16, E)");
  if (p.x_type != 1 && p.x_type != 2) return fail(BFP8_EINVAL, "x must be bf16 or fp16");
  if (p.format != 0 && p.format != 1) return fail(BFP8_EINVAL, "unknown weight format");
  if (!p.x || !p.y || !p.w13 || !p.s13 || !p.w2 || !p.s2) return fail(BFP8_EINVAL, "null operand pointer");
  if (p.logits ? (p.ids || p.weights) : (!p.ids || !p.weights))
    return fail(BFP8_EINVAL, "either logits, or ids and weights");
  if (p.logits && (p.ld_logits < p.E || p.logits_type < 0 || p.logits_type > 2))
    return fail(BFP8_EINVAL, "logits must be row-major fp32, bf16 or fp16");
  if (!aligned16(p.x) || p.ldx < p.H || p.ldx % 8 || !aligned16(p.y) || p.ldy < p.H || p.ldy % 8)
    return fail(BFP8_EINVAL, "x and y must be row-major with 16-byte aligned rows");
  const int64_t k13 = p.format ? p.H / 2 : p.H, k2 = p.format ? p.I / 2 : p.I;
  if (!aligned16(p.w13) || !aligned16(p.w2) || p.w13_row < k13 || p.w13_row % 16 || p.w2_row < k2 || p.w2_row % 16 ||
      p.w13_expert % 16 || p.w2_expert % 16)
    return fail(BFP8_EINVAL, "expert weights must be row-major with 16-byte aligned rows");
  if (p.E > 1 && (p.w13_expert < 2 * p.I * p.w13_row || p.w2_expert < p.H * p.w2_row))
    return fail(BFP8_EINVAL, "experts must not overlap or interleave");
  if (!aligned16(p.s13) || !aligned16(p.s2)) return fail(BFP8_EINVAL, "scales must be 16-byte aligned");
  return BFP8_OK;
}

template <class Cfg>
int launch_moe_kernel(MoeParams& mp, const MoeLayout& lay, int dev, int num_sms, cudaStream_t stream) {
  static std::atomic<uint64_t> done{0};
  if (int r = allow_smem(reinterpret_cast<const void*>(&moe_kernel<Cfg>), kMaxSmem, dev, done)) return r;
  mp.segments = lay.segments;
  mp.seg_len = lay.seg_len;
  mp.stages = lay.stages;
  mp.box = lay.box;
  mp.unit_stages = lay.unit_stages;
  mp.off_b = lay.off_b;
  mp.off_ts = lay.off_ts;
  mp.off_red = lay.off_red;
  mp.off_route = lay.off_route;
  mp.off_bars = lay.off_bars;
  mp.plane = lay.plane;
  mp.cols = lay.cols;
  mp.resident = lay.resident;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(num_sms));
  cfg.blockDim = dim3(Cfg::THREADS);
  cfg.dynamicSmemBytes = size_t(lay.smem);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  set_pdl(cfg, attr);
  cudaError_t e = cudaLaunchKernelEx(&cfg, moe_kernel<Cfg>, mp);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "expert layer launch");
  return BFP8_OK;
}

template <bool GATE>
int launch_moe_any(MoeParams& mp, const MoeLayout& lay, int format, const MoeShape& s, int x_type, int dev, int num_sms,
                   cudaStream_t stream) {
  auto go = [&](auto mx, auto warps, auto t) {
    return launch_moe_kernel<MoeCfg<GATE, decltype(mx)::value, decltype(warps)::value, decltype(t)>>(mp, lay, dev, num_sms,
                                                                                                   stream);
  };
  auto by_type = [&](auto mx, auto warps) {
    return x_type == 1 ? go(mx, warps, __nv_bfloat16()) : go(mx, warps, __half());
  };
  auto by_shape = [&](auto mx) {
    return s.warps == 16 ? by_type(mx, std::integral_constant<int, 16>()) : by_type(mx, std::integral_constant<int, 8>());
  };
  return format ? by_shape(std::true_type()) : by_shape(std::false_type());
}

}  // namespace
}  // namespace bfp8

extern "C" {

int bfp8_launch_mxfp4_quantize(const bfp8_mxfp4_quant_problem* pp, void* stream) {
  if (!pp) return fail(BFP8_EINVAL, "null problem");
  const bfp8_mxfp4_quant_problem& p = *pp;
  if (p.x_type < 0 || p.x_type > 2) return fail(BFP8_EINVAL, "x must be fp32, bf16 or fp16");
  if (int r = check_codes(p.q, p.ldq, p.s, p.M, p.K)) return r;
  if (p.M == 0) return BFP8_OK;
  if (!p.x || !aligned16(p.x) || p.ldx < p.K || (p.ldx * element_size(p.x_type)) % 16)
    return fail(BFP8_EINVAL, "x must be row-major with 16-byte aligned rows");
  Mxfp4QuantParams k{p.x, p.ldx, static_cast<uint8_t*>(p.q), p.ldq, static_cast<uint8_t*>(p.s), p.M, p.K,
                     cdiv(p.M, 128), cdiv(p.K, 128), p.trigger ? 1 : 0};
  void* args[] = {&k};
  const void* kernel = p.x_type == 0   ? reinterpret_cast<const void*>(&mxfp4_quantize_kernel<float>)
                       : p.x_type == 1 ? reinterpret_cast<const void*>(&mxfp4_quantize_kernel<__nv_bfloat16>)
                                       : reinterpret_cast<const void*>(&mxfp4_quantize_kernel<__half>);
  return launch_mx(kernel, k.m_tiles, k.k_tiles, args, static_cast<cudaStream_t>(stream),
                   "MXFP4 quantization launch");
}

int bfp8_launch_mxfp4_dequantize(const bfp8_mxfp4_dequant_problem* pp, void* stream) {
  if (!pp) return fail(BFP8_EINVAL, "null problem");
  const bfp8_mxfp4_dequant_problem& p = *pp;
  if (p.y_type < 0 || p.y_type > 1) return fail(BFP8_EINVAL, "y must be fp32 or bf16");
  if (int r = check_codes(p.q, p.ldq, p.s, p.M, p.K)) return r;
  if (p.M == 0) return BFP8_OK;
  if (!p.y || !aligned16(p.y) || p.ldy < p.K || (p.ldy * element_size(p.y_type)) % 16)
    return fail(BFP8_EINVAL, "y must be row-major with 16-byte aligned rows");
  Mxfp4DequantParams k{static_cast<const uint8_t*>(p.q), p.ldq, static_cast<const uint8_t*>(p.s), p.y, p.ldy, p.M, p.K,
                       cdiv(p.M, 128), cdiv(p.K, 128)};
  void* args[] = {&k};
  const void* kernel = p.y_type == 0 ? reinterpret_cast<const void*>(&mxfp4_dequantize_kernel<float>)
                                     : reinterpret_cast<const void*>(&mxfp4_dequantize_kernel<__nv_bfloat16>);
  return launch_mx(kernel, k.m_tiles, k.k_tiles, args, static_cast<cudaStream_t>(stream),
                   "MXFP4 dequantization launch");
}

int bfp8_launch_mxfp4_gemm(const bfp8_mxfp4_gemm_problem* pp, void* stream) {
  if (!pp) return fail(BFP8_EINVAL, "null problem");
  const bfp8_mxfp4_gemm_problem& p = *pp;
  const bool quant = p.a_type != 0;  // 16-bit activations
  if (p.N <= 0 || p.N % 8) return fail(BFP8_EINVAL, "N must be a positive multiple of 8");
  if (p.a_type < 0 || p.a_type > 2) return fail(BFP8_EINVAL, "a must be MXFP4 codes, bf16 or fp16");
  if (quant) {
    if (p.M < 0 || p.M > BFP8_MXFP4_QUANT_MAX_M || p.K <= 0 || p.K % 32)
      return fail(BFP8_EINVAL, "16-bit activations: at most 16 rows, K a positive multiple of 32");
    if (p.K > kMxMaxSize) return fail(BFP8_EINVAL, "too large");
    if (p.M && (!p.a || !aligned16(p.a) || p.lda < p.K || p.lda % 8))
      return fail(BFP8_EINVAL, "a must be row-major with 16-byte aligned rows");
  } else if (int r = check_codes(p.a, p.lda, p.sa, p.M, p.K)) {
    return r;
  }
  if (p.M == 0) return BFP8_OK;
  if (int r = check_codes(p.b, p.ldb, p.sb, p.N, p.K)) return r;
  if (!p.c || !aligned16(p.c) || p.ldc < p.N || p.ldc % 8)
    return fail(BFP8_EINVAL, "c must be row-major with 8-element aligned rows");
  int dev = 0;
  const int num_sms = current_device_sms(&dev);
  if (num_sms < 0) return fail(BFP8_ECUDA, "no CUDA device");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (quant) return launch_mx_gemm<MxCfg<16, true>>(p, p.a_type, dev, num_sms, s);
  if (p.M <= 16) return launch_mx_gemm<MxCfg<16, false>>(p, 0, dev, num_sms, s);
  if (p.M <= 32) return launch_mx_gemm<MxCfg<32, false>>(p, 0, dev, num_sms, s);
  if (p.M <= 64) return launch_mx_gemm<MxCfg<64, false>>(p, 0, dev, num_sms, s);
  // Beyond a token tile: pairs, or single CTAs with K split, whichever this
  // fit to measured times (us) puts ahead.  Measured, single and pairs: 256 x
  // 6144 x 4096 14.3 and 11.9, 256 x 24576 x 4096 31.9 and 20.6, 256 x 4096 x
  // 12288 14.9 and 25.0, 512 x 6144 x 4096 15.6 and 12.9.
  const int k_stages = cdiv(p.K, 256);
  const int64_t tiles = int64_t(cdiv(p.N, 128)) * cdiv(p.M, 128), splits = mx_splits(tiles, k_stages, num_sms);
  const int64_t rounds = (int64_t(cdiv(p.N, 256)) * cdiv(p.M, 256) + num_sms / 2 - 1) / (num_sms / 2);
  const double single = 4 + 1.35 * double(cdiv(k_stages, int(splits))) * std::max(0.65, double(tiles * splits) / (2 * num_sms));
  const double paired = 2.4 + double(rounds) * (0.55 * k_stages + 0.7);
  if (p.M > 128 && paired < single) return launch_mx_pair(p, dev, num_sms, s);
  return launch_mx_gemm<MxCfg<128, false>>(p, 0, dev, num_sms, s);
}

int64_t bfp8_moe_workspace_bytes(const bfp8_moe_problem* pp) {
  if (!pp) return fail(BFP8_EINVAL, "null problem");
  const bfp8_moe_problem& p = *pp;
  if (int r = check_moe(p)) return r;
  MoeShape s;
  if (int r = moe_shape(p, &s)) return r;
  const int64_t pairs = int64_t(p.T) * p.top_k;
  return align256(pairs * p.I * 4) + align256(pairs * s.down.segments * p.H * 4) + align256(pairs * 8);
}

int bfp8_launch_moe(const bfp8_moe_problem* pp, void* workspace, void* stream) {
  if (!pp) return fail(BFP8_EINVAL, "null problem");
  const bfp8_moe_problem& p = *pp;
  if (int r = check_moe(p)) return r;
  if (!workspace || !aligned16(workspace)) return fail(BFP8_EINVAL, "the workspace must be 16-byte aligned");
  MoeShape s;
  if (int r = moe_shape(p, &s)) return r;
  int dev = 0;
  const int num_sms = current_device_sms(&dev);
  if (num_sms < 0) return fail(BFP8_ECUDA, "no CUDA device");
  const int64_t pairs = int64_t(p.T) * p.top_k;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  MoeParams mp;
  std::memset(&mp, 0, sizeof(mp));
  mp.x = p.x;
  mp.ldx = p.ldx;
  mp.logits = p.logits;
  mp.ld_logits = p.ld_logits;
  mp.logits_type = p.logits_type;
  mp.ids = p.ids;
  mp.weights = p.weights;
  mp.renormalize = p.renormalize;
  mp.h = reinterpret_cast<float*>(ws);
  mp.z = reinterpret_cast<float*>(ws + align256(pairs * p.I * 4));
  mp.routed = reinterpret_cast<float2*>(ws + align256(pairs * p.I * 4) + align256(pairs * s.down.segments * p.H * 4));
  mp.T = p.T;
  mp.H = p.H;
  mp.I = p.I;
  mp.E = p.E;
  mp.top_k = p.top_k;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int r = moe_maps(mp, s.gate, p.format, p.w13, p.w13_expert, p.w13_row, p.s13, p.E, 2 * p.I, p.I, p.H)) return r;
  if (int r = launch_moe_any<true>(mp, s.gate, p.format, s, p.x_type, dev, num_sms, st)) return r;
  if (int r = moe_maps(mp, s.down, p.format, p.w2, p.w2_expert, p.w2_row, p.s2, p.E, p.H, 8, p.I)) return r;
  if (int r = launch_moe_any<false>(mp, s.down, p.format, s, p.x_type, dev, num_sms, st)) return r;
  const MoeSumParams sp{mp.z, mp.routed, p.y, p.ldy, p.T, p.H, p.top_k, s.down.segments};
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(cdiv(p.T * (p.H / 4), kMoeSumThreads)));
  cfg.blockDim = dim3(kMoeSumThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  set_pdl(cfg, attr);
  cudaError_t e = p.x_type == 1 ? cudaLaunchKernelEx(&cfg, moe_sum_kernel<__nv_bfloat16>, sp)
                                : cudaLaunchKernelEx(&cfg, moe_sum_kernel<__half>, sp);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "expert layer sum launch");
  return BFP8_OK;
}

}  // extern "C"
