// torch.ops.blockfp8: the seven operators of the reference's extension
// (simon-jd/blockfp8 csrc/ops.cpp:213-232) -- the same schemas, defaults and
// CUDA dispatch -- implemented over the C ABI of libblockfp8_b200.so
// (include/blockfp8_b200.h).  This file is glue: tensor checks, output
// allocation, plan resolution and scratch; the kernels, planner and launch
// logic live behind the ABI.
//
// Conventions:
// - outputs are allocated on the input's device (C; q and M-major scales);
//   inputs are borrowed, never copied;
// - everything is enqueued on the current CUDA stream under a device guard
//   and nothing synchronises;
// - split-K workspace comes from the caching allocator per call (so it is
//   graph-pool memory under capture); arrival counters come from a
//   per-device pool that is zero between launches (the kernels reset what
//   they use) and is never freed, because captured graphs keep pointing at
//   it.  Two calls running at once on different streams of one device must
//   not share a pool: the ops assume one stream per device, as vLLM uses.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <deque>
#include <map>
#include <mutex>
#include <string>
#include <tuple>

#include "blockfp8_b200.h"

namespace {

constexpr double kDefaultEps = 1e-10;

// ---- checks ------------------------------------------------------------------
// Messages read "blockfp8[.op]: what"; callers (and the tests) match on the
// `what` part.

[[noreturn]] void reject(const char* op, const std::string& what) {
  TORCH_CHECK(false, op, ": ", what);
}

void require(bool ok, const char* op, const char* what) {
  if (!ok) reject(op, what);
}

void require_abi(int status) {
  if (status < 0) TORCH_CHECK(false, bfp8_last_error());
}

bool aligned16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

bool row_major(const at::Tensor& t, int64_t row_multiple) {
  return t.stride(1) == 1 && t.stride(0) % row_multiple == 0;
}

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Weights and their 128x128 block scales, for a reduction length K.
void check_weights(const at::Tensor& b, const at::Tensor& b_scales, int64_t K) {
  const char* op = "blockfp8";
  require(b.is_cuda() && b_scales.is_cuda(), op, "all operands must be CUDA tensors");
  require(b.scalar_type() == at::kFloat8_e4m3fn, op, "b must be float8_e4m3fn");
  require(b_scales.scalar_type() == at::kFloat, op, "scales must be float32");
  require(b.dim() == 2 && b.size(1) == K, op, "bad shapes");
  require(K > 0 && K % 16 == 0, op, "K must be a positive multiple of 16");
  require(b.size(0) > 0 && b.size(0) % 8 == 0, op, "N must be a positive multiple of 8");
  require(row_major(b, 16), op, "b must be row-major with 16-element aligned rows");
  require(aligned16(b), op, "b must be 16-byte aligned");
  require(b_scales.dim() == 2 && b_scales.size(0) == cdiv(b.size(0), 128) && b_scales.size(1) == cdiv(K, 128), op,
          "b_scales must be [ceil(N/128), ceil(K/128)]");
  require(b.device() == b_scales.device(), op, "all operands must be on one device");
  require(b.size(0) <= INT32_MAX && K <= INT32_MAX, op, "too large");
}

// bf16 activations of linear / quantize.
void check_activations(const at::Tensor& x, const char* op) {
  require(x.is_cuda() && x.scalar_type() == at::kBFloat16 && x.dim() == 2, op,
          "x must be a 2-D bfloat16 CUDA tensor");
  require(row_major(x, 8) && aligned16(x), op, "x must be row-major with 16-byte aligned rows");
  require(x.size(1) > 0 && x.size(1) % 16 == 0, op, "K must be a positive multiple of 16");
  require(x.size(0) <= INT32_MAX && x.size(1) <= INT32_MAX, op, "too large");
}

// ---- split-K arrival counters --------------------------------------------------

class CounterPool {
 public:
  // At least `needed` zeroed ints on `device`.
  int* get(const at::Device& device, int needed) {
    std::lock_guard<std::mutex> lock(mu_);
    at::Tensor& live = live_[device.index()];
    if (!live.defined() || live.numel() < needed) {
      if (live.defined()) kept_.push_back(live);  // a captured graph may still use it
      int64_t size = int64_t(1) << 16;
      while (size < needed) size *= 2;
      live = at::zeros({size}, at::TensorOptions().dtype(at::kInt).device(device));
    }
    return live.data_ptr<int>();
  }

 private:
  std::mutex mu_;
  std::map<int, at::Tensor> live_;
  std::deque<at::Tensor> kept_;
};

CounterPool& counter_pool() {
  static CounterPool pool;
  return pool;
}

// ---- plans and launches ----------------------------------------------------------

int sm_count() { return at::cuda::getCurrentDeviceProperties()->multiProcessorCount; }

// The plan a call runs: the library's choice, unless the caller names a
// configuration (then split_k defaults to one split) and/or a split count
// (> 0: K splits; < 0: stream-K over -split_k CTAs).
bfp8_plan resolve(bfp8_plan chosen, int64_t config, int64_t split_k, int num_configs) {
  if (config >= 0) {
    TORCH_CHECK(config < num_configs, "blockfp8: config out of range");
    chosen.config = int(config);
    if (split_k == 0) split_k = 1;
  }
  if (split_k != 0) chosen.splits = int(split_k);
  return chosen;
}

// Scratch for one launch (workspace from the caching allocator, counters
// from the pool), then the launch on the current stream.
void launch(const bfp8_gemm_problem& p, const bfp8_plan& plan, const at::Tensor& like) {
  const int64_t ws_bytes = bfp8_workspace_bytes(&p, plan);
  require_abi(int(std::min<int64_t>(ws_bytes, 0)));
  const int n_counters = bfp8_counters_needed(&p, plan);
  require_abi(std::min(n_counters, 0));
  at::Tensor ws;
  if (ws_bytes > 0) ws = at::empty({cdiv(ws_bytes, 4)}, like.options().dtype(at::kFloat));
  int* counters = n_counters > 0 ? counter_pool().get(like.device(), n_counters) : nullptr;
  require_abi(bfp8_launch_gemm(&p, plan, ws.defined() ? ws.data_ptr<float>() : nullptr, counters,
                               at::cuda::getCurrentCUDAStream().stream()));
}

// The weight side and output of a problem; the caller fills in A.
bfp8_gemm_problem weight_problem(const at::Tensor& b, const at::Tensor& b_scales, const at::Tensor& c) {
  bfp8_gemm_problem p{};
  p.b = b.data_ptr();
  p.ldb = b.stride(0);
  p.sb = b_scales.data_ptr<float>();
  p.sb_n = b_scales.stride(0);
  p.sb_k = b_scales.stride(1);
  p.c = c.data_ptr();
  p.ldc = c.stride(0);
  p.M = int(c.size(0));
  p.N = int(b.size(0));
  p.K = int(b.size(1));
  p.eps = float(kDefaultEps);
  return p;
}

// ---- the operators -------------------------------------------------------------

// C = (a, a_scales) x (b, b_scales)^T: e4m3 activations with per-row 1x128
// scales (any strides) against 128x128-block-scaled e4m3 weights, bf16 out.
at::Tensor gemm(const at::Tensor& a, const at::Tensor& a_scales, const at::Tensor& b, const at::Tensor& b_scales,
                int64_t config, int64_t split_k) {
  const char* op = "blockfp8.gemm";
  require(a.is_cuda() && a_scales.is_cuda(), op, "all operands must be CUDA tensors");
  require(a.scalar_type() == at::kFloat8_e4m3fn, op, "a must be float8_e4m3fn");
  require(a_scales.scalar_type() == at::kFloat, op, "scales must be float32");
  require(a.dim() == 2, op, "bad shapes");
  check_weights(b, b_scales, a.size(1));
  require(row_major(a, 16), op, "a must be row-major with 16-element aligned rows");
  require(aligned16(a), op, "a must be 16-byte aligned");
  require(a_scales.dim() == 2 && a_scales.size(0) == a.size(0) && a_scales.size(1) == cdiv(a.size(1), 128), op,
          "a_scales must be [M, ceil(K/128)]");
  require(a.device() == b.device() && a.device() == a_scales.device(), op, "all operands must be on one device");
  require(a.size(0) <= INT32_MAX, op, "too large");

  const at::cuda::CUDAGuard guard(a.device());
  at::Tensor c = at::empty({a.size(0), b.size(0)}, a.options().dtype(at::kBFloat16));
  if (c.size(0) == 0) return c;
  bfp8_gemm_problem p = weight_problem(b, b_scales, c);
  p.a = a.data_ptr();
  p.lda = a.stride(0);
  p.sa = a_scales.data_ptr<float>();
  p.sa_m = a_scales.stride(0);
  p.sa_k = a_scales.stride(1);
  launch(p, resolve(bfp8_choose_plan(p.M, p.N, p.K, sm_count()), config, split_k, bfp8_num_configs()), a);
  return c;
}

// The same product from bf16 activations, quantized as part of the call
// (bitwise gemm(quantize(x))).
at::Tensor gemm_bf16(const at::Tensor& x, const at::Tensor& b, const at::Tensor& b_scales, int64_t config,
                     int64_t split_k, double eps) {
  const char* op = "blockfp8.gemm_bf16";
  require(x.is_cuda(), op, "all operands must be CUDA tensors");
  require(x.scalar_type() == at::kBFloat16, op, "x must be bfloat16");
  require(x.dim() == 2, op, "bad shapes");
  check_weights(b, b_scales, x.size(1));
  require(row_major(x, 8), op, "x must be row-major with 8-element aligned rows");
  require(aligned16(x), op, "x must be 16-byte aligned");
  require(x.device() == b.device(), op, "all operands must be on one device");
  require(x.size(0) <= INT32_MAX, op, "too large");
  require(eps > 0, op, "eps must be positive");

  const at::cuda::CUDAGuard guard(x.device());
  at::Tensor c = at::empty({x.size(0), b.size(0)}, x.options().dtype(at::kBFloat16));
  if (c.size(0) == 0) return c;
  bfp8_gemm_problem p = weight_problem(b, b_scales, c);
  p.a = x.data_ptr();
  p.lda = x.stride(0);
  p.eps = float(eps);
  launch(p, resolve(bfp8_choose_fused_plan(p.M, p.N, p.K, sm_count()), config, split_k, bfp8_num_fused_configs()),
         x);
  return c;
}

// x [M, K] bf16 -> (q [M, K] e4m3, scales [M, ceil(K/128)] float32 stored
// M-contiguous, strides (1, M)).
std::tuple<at::Tensor, at::Tensor> quantize(const at::Tensor& x, double eps) {
  const char* op = "blockfp8.quantize";
  check_activations(x, op);
  require(eps > 0, op, "eps must be positive");
  const at::cuda::CUDAGuard guard(x.device());
  const int64_t M = x.size(0), K = x.size(1);
  at::Tensor q = at::empty({M, K}, x.options().dtype(at::kFloat8_e4m3fn));
  at::Tensor s = at::empty({cdiv(K, 128), M}, x.options().dtype(at::kFloat)).t();
  const bfp8_quant_problem p{x.data_ptr(), x.stride(0), q.data_ptr(), q.stride(0), s.data_ptr<float>(),
                             s.stride(0),  s.stride(1), int(M),     int(K),      float(eps)};
  require_abi(bfp8_launch_quantize(&p, at::cuda::getCurrentCUDAStream().stream()));
  return {q, s};
}

bool prefers_fused(int64_t M, int64_t N, int64_t K) { return bfp8_prefers_fused(int(M), int(N), int(K)) != 0; }

// A linear layer on bf16 activations: the fused path where the library
// prefers it (everywhere today), else quantize() then gemm().
at::Tensor linear(const at::Tensor& x, const at::Tensor& b, const at::Tensor& b_scales) {
  check_activations(x, "blockfp8.linear");
  if (prefers_fused(x.size(0), b.size(0), x.size(1))) return gemm_bf16(x, b, b_scales, -1, 0, kDefaultEps);
  const auto qs = quantize(x, kDefaultEps);
  return gemm(std::get<0>(qs), std::get<1>(qs), b, b_scales, -1, 0);
}

// ";"-joined configuration names.
std::string joined(int count, const char* (*name_of)(int)) {
  std::string out;
  for (int i = 0; i < count; ++i) out.append(i ? ";" : "").append(name_of(i));
  return out;
}

std::string config_names() { return joined(bfp8_num_configs(), bfp8_config_name); }
std::string fused_config_names() { return joined(bfp8_num_fused_configs(), bfp8_fused_config_name); }

// ---- producers that emit the linear's operand (torch.ops.blockfp8_b200) ---------
// Not in the reference's extension: an RMSNorm and a SiLU-and-mul whose
// outputs are the e4m3 codes and M-major scales blockfp8.gemm takes, so the
// linear after them needs no quantization launch.

std::tuple<at::Tensor, at::Tensor> quant_outputs(const at::Tensor& like, int64_t M, int64_t cols) {
  at::Tensor q = at::empty({M, cols}, like.options().dtype(at::kFloat8_e4m3fn));
  at::Tensor s = at::empty({cdiv(cols, 128), M}, like.options().dtype(at::kFloat)).t();
  return {q, s};
}

// (q, scales, h): h = x + residual in bf16 when a residual is given (the
// next layer's residual), else an empty tensor.
std::tuple<at::Tensor, at::Tensor, at::Tensor> rms_norm_quant(const at::Tensor& x, const at::Tensor& weight,
                                                              double variance_epsilon,
                                                              const c10::optional<at::Tensor>& residual, double eps) {
  const char* op = "blockfp8_b200.rms_norm_quant";
  check_activations(x, op);
  const int64_t M = x.size(0), H = x.size(1);
  require(H % 128 == 0 && H <= 16384, op, "hidden size must be a multiple of 128, at most 16384");
  require(weight.is_cuda() && weight.scalar_type() == at::kBFloat16 && weight.dim() == 1 && weight.size(0) == H &&
              weight.stride(0) == 1 && aligned16(weight) && weight.device() == x.device(),
          op, "weight must be a contiguous bfloat16 [H] tensor on x's device");
  require(eps > 0 && variance_epsilon >= 0, op, "eps must be positive");
  const at::cuda::CUDAGuard guard(x.device());
  auto [q, s] = quant_outputs(x, M, H);
  at::Tensor h;
  bfp8_rmsnorm_quant_problem p{};
  p.x = x.data_ptr();
  p.ldx = x.stride(0);
  if (residual.has_value()) {
    const at::Tensor& r = *residual;
    check_activations(r, op);
    require(r.sizes() == x.sizes() && r.device() == x.device(), op, "residual must match x");
    h = at::empty({M, H}, x.options());
    p.residual = r.data_ptr();
    p.ldr = r.stride(0);
    p.residual_out = h.data_ptr();
    p.ldro = h.stride(0);
  } else {
    h = at::empty({0}, x.options());
  }
  if (M == 0) return {q, s, h};
  p.weight = weight.data_ptr();
  p.q = q.data_ptr();
  p.ldq = q.stride(0);
  p.s = s.data_ptr<float>();
  p.s_m = s.stride(0);
  p.s_k = s.stride(1);
  p.M = int(M);
  p.H = int(H);
  p.variance_epsilon = float(variance_epsilon);
  p.eps = float(eps);
  require_abi(bfp8_launch_rmsnorm_quant(&p, at::cuda::getCurrentCUDAStream().stream()));
  return {q, s, h};
}

std::tuple<at::Tensor, at::Tensor> silu_mul_quant(const at::Tensor& x, double eps) {
  const char* op = "blockfp8_b200.silu_mul_quant";
  check_activations(x, op);
  const int64_t M = x.size(0), I = x.size(1) / 2;
  require(x.size(1) % 256 == 0, op, "x must be [M, 2I] with I a multiple of 128");
  require(M <= 65535, op, "at most 65535 rows");
  require(eps > 0, op, "eps must be positive");
  const at::cuda::CUDAGuard guard(x.device());
  auto [q, s] = quant_outputs(x, M, I);
  if (M == 0) return {q, s};
  bfp8_silu_mul_quant_problem p{};
  p.x = x.data_ptr();
  p.ldx = x.stride(0);
  p.q = q.data_ptr();
  p.ldq = q.stride(0);
  p.s = s.data_ptr<float>();
  p.s_m = s.stride(0);
  p.s_k = s.stride(1);
  p.M = int(M);
  p.I = int(I);
  p.eps = float(eps);
  require_abi(bfp8_launch_silu_mul_quant(&p, at::cuda::getCurrentCUDAStream().stream()));
  return {q, s};
}

// ---- MXFP4 and the expert layer (torch.ops.blockfp8_b200) -------------------------
// Every argument is checked here, once; refusals are ValueErrors.  The
// operators are registered for CPU tensors too, so that a call on them is
// refused with its reason (shapes and types first, then the device) rather
// than by the dispatcher.

#define CHECK_VALUE(cond, ...) TORCH_CHECK_VALUE(cond, __VA_ARGS__)

void require_valid(int status) {
  CHECK_VALUE(status != BFP8_EINVAL, bfp8_last_error());
  require_abi(status);
}

int float_type(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default: return -1;
  }
}

bool aligned_rows(const at::Tensor& t) {  // 2-D, contiguous 16-byte aligned rows
  return t.stride(1) == 1 && (t.size(0) <= 1 || t.stride(0) >= t.size(1)) &&
         (t.size(0) <= 1 || (t.stride(0) * t.element_size()) % 16 == 0) && aligned16(t);
}

// The row stride handed to the kernels; a single row's says nothing.
int64_t row_stride(const at::Tensor& t) {
  const int64_t unit = 16 / t.element_size();
  return t.size(-2) > 1 ? t.stride(-2) : cdiv(t.size(-1), unit) * unit;
}

void check_mxfp4(const at::Tensor& q, const at::Tensor& s, const char* op, const char* name) {
  CHECK_VALUE(q.scalar_type() == at::kByte && q.dim() == 2, op, ": ", name, " must be 2-D uint8 codes [rows, K / 2]");
  const int64_t rows = q.size(0), K = 2 * q.size(1);
  CHECK_VALUE(K > 0 && K % 32 == 0, op, ": K must be a positive multiple of 32, got ", K);
  CHECK_VALUE(rows <= INT32_MAX / 2 && K <= INT32_MAX / 2, op, ": too large");
  CHECK_VALUE(aligned_rows(q), op, ": ", name, " must be row-major with 16-byte aligned rows");
  CHECK_VALUE(s.scalar_type() == at::kByte && s.dim() == 4 && s.size(0) == cdiv(rows, 128) && s.size(1) == cdiv(K, 128) &&
                  s.size(2) == 32 && s.size(3) == 16,
              op, ": the scales of ", name, " must be uint8 [", cdiv(rows, 128), ", ", cdiv(K, 128),
              ", 32, 16] (tile_mxfp4_scales), got ", s.sizes());
  CHECK_VALUE(s.is_contiguous() && aligned16(s), op, ": the scales of ", name, " must be contiguous");
}

void check_cuda(std::initializer_list<const at::Tensor*> tensors, const char* op) {
  const at::Tensor& first = **tensors.begin();
  for (const at::Tensor* t : tensors) {
    CHECK_VALUE(t->device() == first.device(), op, ": all operands must be on one device");
    CHECK_VALUE(t->is_cuda(), op, ": runs on CUDA tensors only");
  }
}

std::tuple<at::Tensor, at::Tensor> empty_mxfp4(const at::Tensor& like, int64_t rows, int64_t K) {
  const auto bytes = like.options().dtype(at::kByte);
  return {at::empty({rows, K / 2}, bytes), at::empty({cdiv(rows, 128), cdiv(K, 128), 32, 16}, bytes)};
}

void check_mxfp4_input(const at::Tensor& x, const char* op) {
  CHECK_VALUE(x.dim() == 2, op, ": x must be 2-D [M, K], got shape ", x.sizes());
  CHECK_VALUE(x.size(1) > 0 && x.size(1) % 32 == 0, op, ": K must be a positive multiple of 32, got ", x.size(1));
  CHECK_VALUE(x.size(0) <= INT32_MAX / 2 && x.size(1) <= INT32_MAX / 2, op, ": too large");
  CHECK_VALUE(aligned_rows(x), op, ": x must be row-major with 16-byte aligned rows, got strides ", x.strides());
}

void launch_mxfp4_quantize(const at::Tensor& x, const at::Tensor& q, const at::Tensor& s, bool trigger) {
  const bfp8_mxfp4_quant_problem p{x.data_ptr(),  row_stride(x), float_type(x),  q.data_ptr(),
                                   row_stride(q), s.data_ptr(),  int(x.size(0)), int(x.size(1)), trigger ? 1 : 0};
  require_valid(bfp8_launch_mxfp4_quantize(&p, at::cuda::getCurrentCUDAStream().stream()));
}

// x [M, K] -> (codes [M, K / 2], scale tiles).
std::tuple<at::Tensor, at::Tensor> quantize_mxfp4(const at::Tensor& x) {
  const char* op = "blockfp8_b200.quantize_mxfp4";
  CHECK_VALUE(float_type(x) >= 0, op, ": x must be bfloat16, float16 or float32, got ", x.scalar_type());
  check_mxfp4_input(x, op);
  check_cuda({&x}, op);
  const at::cuda::CUDAGuard guard(x.device());
  auto out = empty_mxfp4(x, x.size(0), x.size(1));
  if (x.size(0) > 0) launch_mxfp4_quantize(x, std::get<0>(out), std::get<1>(out), false);
  return out;
}

at::Tensor dequantize_mxfp4(const at::Tensor& q, const at::Tensor& s, at::ScalarType dtype) {
  const char* op = "blockfp8_b200.dequantize_mxfp4";
  check_mxfp4(q, s, op, "q");
  CHECK_VALUE(dtype == at::kBFloat16 || dtype == at::kFloat, op, ": dtype must be bfloat16 or float32, got ", dtype);
  check_cuda({&q, &s}, op);
  const at::cuda::CUDAGuard guard(q.device());
  at::Tensor y = at::empty({q.size(0), 2 * q.size(1)}, q.options().dtype(dtype));
  if (y.size(0) == 0) return y;
  const bfp8_mxfp4_dequant_problem p{q.data_ptr(), row_stride(q),  s.data_ptr(), y.data_ptr(), y.stride(0),
                                     float_type(y), int(y.size(0)), int(y.size(1))};
  require_valid(bfp8_launch_mxfp4_dequantize(&p, at::cuda::getCurrentCUDAStream().stream()));
  return y;
}

// a: codes with their scales, or (sa null) 16-bit activations.
at::Tensor launch_mxfp4_gemm(const at::Tensor& a, const at::Tensor* sa, const at::Tensor& b, const at::Tensor& sb,
                             bool weights_ready) {
  at::Tensor c = at::empty({a.size(0), b.size(0)}, a.options().dtype(at::kBFloat16));
  const bfp8_mxfp4_gemm_problem p{a.data_ptr(),   row_stride(a),
                                  sa ? sa->data_ptr() : nullptr,
                                  b.data_ptr(),   row_stride(b),  sb.data_ptr(),      c.data_ptr(),
                                  c.stride(0),    int(a.size(0)), int(b.size(0)),     int(2 * b.size(1)),
                                  weights_ready ? 1 : 0, sa ? 0 : float_type(a)};
  require_valid(bfp8_launch_mxfp4_gemm(&p, at::cuda::getCurrentCUDAStream().stream()));
  return c;
}

void check_mxfp4_weights(const at::Tensor& b, const at::Tensor& b_scales, int64_t K, const char* op) {
  check_mxfp4(b, b_scales, op, "b_q");
  CHECK_VALUE(2 * b.size(1) == K, op, ": K mismatch: ", K, " and ", 2 * b.size(1));
  CHECK_VALUE(b.size(0) > 0 && b.size(0) % 8 == 0, op, ": N must be a positive multiple of 8, got ", b.size(0));
}

at::Tensor gemm_mxfp4(const at::Tensor& a, const at::Tensor& a_scales, const at::Tensor& b, const at::Tensor& b_scales) {
  const char* op = "blockfp8_b200.gemm_mxfp4";
  check_mxfp4(a, a_scales, op, "a_q");
  check_mxfp4_weights(b, b_scales, 2 * a.size(1), op);
  check_cuda({&a, &a_scales, &b, &b_scales}, op);
  const at::cuda::CUDAGuard guard(a.device());
  if (a.size(0) == 0) return at::empty({0, b.size(0)}, a.options().dtype(at::kBFloat16));
  // b may have been written by the kernel right before this one
  return launch_mxfp4_gemm(a, &a_scales, b, b_scales, false);
}

// quantize_mxfp4 then gemm_mxfp4; in one kernel for up to 16 tokens while the
// weight tiles are no more than the SMs (each quantizes again).  The GEMM
// may request its weights as soon as it starts: the quantization kernel lets it
// start only after every earlier kernel has finished, and quantize_mxfp4 (which
// may just have written them) not before its own end.
at::Tensor linear_mxfp4(const at::Tensor& x, const at::Tensor& b, const at::Tensor& b_scales) {
  const char* op = "blockfp8_b200.linear_mxfp4";
  CHECK_VALUE(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, op,
              ": x must be bfloat16 or float16, got ", x.scalar_type());
  check_mxfp4_input(x, op);
  check_mxfp4_weights(b, b_scales, x.size(1), op);
  check_cuda({&x, &b, &b_scales}, op);
  const at::cuda::CUDAGuard guard(x.device());
  if (x.size(0) == 0) return at::empty({0, b.size(0)}, x.options().dtype(at::kBFloat16));
  if (x.size(0) <= BFP8_MXFP4_QUANT_MAX_M && cdiv(b.size(0), 128) <= sm_count())
    return launch_mxfp4_gemm(x, nullptr, b, b_scales, true);
  const auto [q, s] = empty_mxfp4(x, x.size(0), x.size(1));
  launch_mxfp4_quantize(x, q, s, true);
  return launch_mxfp4_gemm(q, &s, b, b_scales, true);
}

// One of the layer's two weight stacks: [E, rows, K] in either format.
void check_experts(const at::Tensor& w, const at::Tensor& s, int64_t E, int64_t rows, int64_t K, bool mx, const char* op,
                   const char* name) {
  const int64_t cols = mx ? K / 2 : K;
  CHECK_VALUE(w.dim() == 3 && w.size(0) == E && w.size(1) == rows && w.size(2) == cols, op, ": ", name, " must be [", E, ", ", rows, ", ",
              cols, "], got ", w.sizes());
  CHECK_VALUE(E == 1 || w.stride(0) >= rows * w.stride(1), op, ": the experts of ", name,
              " must not overlap or interleave, got strides ", w.strides());
  CHECK_VALUE(w.stride(2) == 1 && w.stride(1) >= cols && w.stride(1) % 16 == 0 && w.stride(0) % 16 == 0 && aligned16(w),
              op, ": ", name, " must have contiguous, 16-byte aligned rows, got strides ", w.strides());
  if (mx) {
    CHECK_VALUE(s.scalar_type() == at::kByte && s.dim() == 5 && s.size(0) == E && s.size(1) == cdiv(rows, 128) &&
                    s.size(2) == cdiv(K, 128) && s.size(3) == 32 && s.size(4) == 16,
                op, ": the scales of ", name, " must be uint8 [", E, ", ", cdiv(rows, 128), ", ", cdiv(K, 128),
                ", 32, 16] (tile_mxfp4_scales), got ", s.sizes());
  } else {
    CHECK_VALUE(s.scalar_type() == at::kFloat && s.dim() == 3 && s.size(0) == E && s.size(1) == cdiv(rows, 128) &&
                    s.size(2) == cdiv(K, 128),
                op, ": the scales of ", name, " must be float32 [", E, ", ", cdiv(rows, 128), ", ", cdiv(K, 128), "], got ",
                s.sizes());
  }
  CHECK_VALUE(s.is_contiguous() && aligned16(s), op, ": the scales of ", name, " must be contiguous");
}

at::Tensor launch_moe(const char* op, const at::Tensor& x, const at::Tensor& w13, const at::Tensor& w13_scales,
                      const at::Tensor& w2, const at::Tensor& w2_scales, int64_t E, int64_t top_k,
                      bfp8_moe_problem p, std::initializer_list<const at::Tensor*> all) {
  CHECK_VALUE(x.dim() == 2 && (x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf), op,
              ": x must be 2-D bfloat16 or float16 [T, H]");
  const int64_t T = x.size(0), H = x.size(1);
  CHECK_VALUE(T <= 64, op, ": at most 64 tokens, got ", T);
  CHECK_VALUE(H >= 32 && H % 32 == 0 && H <= 8192, op, ": H must be a multiple of 32, at most 8192, got ", H);
  CHECK_VALUE(aligned_rows(x), op, ": x must be row-major with 16-byte aligned rows, got strides ", x.strides());
  CHECK_VALUE(E >= 1 && E <= 512, op, ": 1 to 512 experts, got ", E);
  CHECK_VALUE(top_k >= 1 && top_k <= std::min<int64_t>(16, E), op, ": top_k must be at least 1 and at most min(16, E), got ",
              top_k);
  const bool mx = w13.scalar_type() == at::kByte;
  CHECK_VALUE(w2.dim() == 3 && w2.scalar_type() == w13.scalar_type() && (mx || w13.scalar_type() == at::kFloat8_e4m3fn), op,
              ": w13 and w2 must both be float8_e4m3fn [E, rows, K] or both uint8 MXFP4 codes [E, rows, K / 2]");
  const int64_t I = w2.size(2) * (mx ? 2 : 1);
  CHECK_VALUE(I >= 32 && I % 32 == 0 && I <= (1 << 24), op, ": I must be a positive multiple of 32, got ", I);
  check_experts(w13, w13_scales, E, 2 * I, H, mx, op, "w13");
  check_experts(w2, w2_scales, E, H, I, mx, op, "w2");
  check_cuda(all, op);
  const at::cuda::CUDAGuard guard(x.device());
  at::Tensor y = at::empty({T, H}, x.options());
  if (T == 0) return y;
  p.x = x.data_ptr();
  p.ldx = row_stride(x);
  p.x_type = float_type(x);
  p.format = mx ? 1 : 0;
  p.w13 = w13.data_ptr();
  p.w13_expert = w13.stride(0);
  p.w13_row = w13.stride(1);
  p.s13 = w13_scales.data_ptr();
  p.w2 = w2.data_ptr();
  p.w2_expert = w2.stride(0);
  p.w2_row = w2.stride(1);
  p.s2 = w2_scales.data_ptr();
  p.y = y.data_ptr();
  p.ldy = y.stride(0);
  p.T = int(T);
  p.H = int(H);
  p.I = int(I);
  p.E = int(E);
  p.top_k = int(top_k);
  const int64_t bytes = bfp8_moe_workspace_bytes(&p);
  require_valid(int(std::min<int64_t>(bytes, 0)));
  const at::Tensor ws = at::empty({bytes}, x.options().dtype(at::kByte));
  require_valid(bfp8_launch_moe(&p, ws.data_ptr(), at::cuda::getCurrentCUDAStream().stream()));
  return y;
}

at::Tensor moe(const at::Tensor& x, const at::Tensor& router_logits, const at::Tensor& w13, const at::Tensor& w13_scales,
               const at::Tensor& w2, const at::Tensor& w2_scales, int64_t top_k, bool renormalize) {
  const char* op = "blockfp8_b200.moe";
  CHECK_VALUE(router_logits.dim() == 2 && float_type(router_logits) >= 0 && x.dim() == 2 &&
                  router_logits.size(0) == x.size(0) && router_logits.stride(1) == 1 &&
                  (x.size(0) <= 1 || router_logits.stride(0) >= router_logits.size(1)),
              op, ": router_logits must be row-major float32, bfloat16 or float16 [T, E]");
  bfp8_moe_problem p{};
  p.logits = router_logits.data_ptr();
  p.ld_logits = x.size(0) > 1 ? router_logits.stride(0) : router_logits.size(1);
  p.logits_type = float_type(router_logits);
  p.renormalize = renormalize ? 1 : 0;
  return launch_moe(op, x, w13, w13_scales, w2, w2_scales, router_logits.size(1), top_k, p,
                    {&x, &router_logits, &w13, &w13_scales, &w2, &w2_scales});
}

at::Tensor moe_experts(const at::Tensor& x, const at::Tensor& topk_ids, const at::Tensor& topk_weights,
                       const at::Tensor& w13, const at::Tensor& w13_scales, const at::Tensor& w2,
                       const at::Tensor& w2_scales) {
  const char* op = "blockfp8_b200.moe_experts";
  CHECK_VALUE(topk_ids.dim() == 2 && topk_ids.scalar_type() == at::kInt && topk_weights.scalar_type() == at::kFloat &&
                  topk_weights.sizes() == topk_ids.sizes() && x.dim() == 2 && topk_ids.size(0) == x.size(0) &&
                  topk_ids.is_contiguous() && topk_weights.is_contiguous(),
              op, ": topk_ids must be contiguous int32 [T, top_k] and topk_weights contiguous float32 of the same shape");
  CHECK_VALUE(w13.dim() == 3, op, ": w13 must be 3-D");
  bfp8_moe_problem p{};
  p.ids = topk_ids.data_ptr<int>();
  p.weights = topk_weights.data_ptr<float>();
  return launch_moe(op, x, w13, w13_scales, w2, w2_scales, w13.size(0), topk_ids.size(1), p,
                    {&x, &topk_ids, &topk_weights, &w13, &w13_scales, &w2, &w2_scales});
}

}  // namespace

TORCH_LIBRARY(blockfp8_b200, m) {
  m.def("quantize_mxfp4(Tensor x) -> (Tensor, Tensor)");
  m.def("dequantize_mxfp4(Tensor q, Tensor scales, ScalarType dtype=bfloat16) -> Tensor");
  m.def("gemm_mxfp4(Tensor a, Tensor a_scales, Tensor b, Tensor b_scales) -> Tensor");
  m.def("linear_mxfp4(Tensor x, Tensor b, Tensor b_scales) -> Tensor");
  m.def("moe(Tensor x, Tensor router_logits, Tensor w13, Tensor w13_scales, Tensor w2, Tensor w2_scales, int top_k, "
        "bool renormalize=True) -> Tensor");
  m.def("moe_experts(Tensor x, Tensor topk_ids, Tensor topk_weights, Tensor w13, Tensor w13_scales, Tensor w2, "
        "Tensor w2_scales) -> Tensor");
  m.def("rms_norm_quant(Tensor x, Tensor weight, float variance_epsilon, Tensor? residual=None, "
        "float eps=1e-10) -> (Tensor, Tensor, Tensor)");
  m.def("silu_mul_quant(Tensor x, float eps=1e-10) -> (Tensor, Tensor)");
}

void impl_experts(torch::Library& m) {
  m.impl("quantize_mxfp4", &quantize_mxfp4);
  m.impl("dequantize_mxfp4", &dequantize_mxfp4);
  m.impl("gemm_mxfp4", &gemm_mxfp4);
  m.impl("linear_mxfp4", &linear_mxfp4);
  m.impl("moe", &moe);
  m.impl("moe_experts", &moe_experts);
}

TORCH_LIBRARY_IMPL(blockfp8_b200, CPU, m) { impl_experts(m); }

TORCH_LIBRARY_IMPL(blockfp8_b200, CUDA, m) {
  impl_experts(m);
  m.impl("rms_norm_quant", &rms_norm_quant);
  m.impl("silu_mul_quant", &silu_mul_quant);
}

TORCH_LIBRARY(blockfp8, m) {
  m.def("gemm(Tensor a, Tensor a_scales, Tensor b, Tensor b_scales, int config=-1, int split_k=0) -> Tensor");
  m.def(
      "gemm_bf16(Tensor x, Tensor b, Tensor b_scales, int config=-1, int split_k=0, float eps=1e-10) -> Tensor");
  m.def("quantize(Tensor x, float eps=1e-10) -> (Tensor, Tensor)");
  m.def("linear(Tensor x, Tensor b, Tensor b_scales) -> Tensor");
  m.def("prefers_fused(int m, int n, int k) -> bool", &prefers_fused);
  m.def("config_names() -> str", &config_names);
  m.def("fused_config_names() -> str", &fused_config_names);
}

TORCH_LIBRARY_IMPL(blockfp8, CUDA, m) {
  m.impl("gemm", &gemm);
  m.impl("gemm_bf16", &gemm_bf16);
  m.impl("quantize", &quantize);
  m.impl("linear", &linear);
}
