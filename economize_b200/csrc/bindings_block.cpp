// PyTorch bindings of the 4-bit operators (fp4.cu, gemm_fp4.cu) and of the norms around a block (block_norm.cu):
// argument checks, workspaces from PyTorch's caching allocator, tensor maps, launches on the current stream.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/CUDAGraphsUtils.cuh>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>

#include <cmath>
#include <cstring>
#include <tuple>
#include <vector>

#include "bindings.h"
#include "launchers.h"

namespace {

using at::Tensor;

constexpr int64_t kMaxRows = int64_t{1} << 30;

// Rows a kernel reads in place: unit stride along the row; others are copied.
Tensor rows_of(const Tensor& x) {
  const bool ok = (x.size(1) <= 1 || x.stride(1) == 1) && (x.size(0) <= 1 || x.stride(0) >= x.size(1));
  return ok ? x : x.contiguous();
}

int64_t row_stride(const Tensor& x) { return x.size(0) > 1 ? x.stride(0) : x.size(1); }

// Whether every row starts on a boundary of `bytes`.
bool aligned(const Tensor& x, int64_t bytes = 16) {
  return !x.defined() || (reinterpret_cast<uintptr_t>(x.data_ptr()) % bytes == 0 &&
                          (x.dim() < 2 || row_stride(x) * x.element_size() % bytes == 0));
}

// x, or a copy whose rows start on boundaries of 16 bytes (rows of whole 16-byte groups).
Tensor on_boundary(const Tensor& x) { return aligned(x) ? x : x.clone(at::MemoryFormat::Contiguous); }

// x, or a copy: 16-bit rows that start in the middle of a word where those of a tensor without gaps do, which are read in
// words.
Tensor on_words(const Tensor& x) {
  const bool ok = !x.defined() || (reinterpret_cast<uintptr_t>(x.data_ptr()) % 4 == 0 &&
                                   (x.size(0) <= 1 || (x.stride(0) - x.size(1)) % 2 == 0));
  return ok ? x : x.clone(at::MemoryFormat::Contiguous);
}

// x as the norms' kernels read it.
Tensor norm_rows(const Tensor& x, bool vec) { return vec ? on_boundary(x) : x.element_size() == 2 ? on_words(x) : x; }

// [..., C] as rows [R, C].
Tensor as_rows(const Tensor& x) { return x.dim() == 2 ? x : x.reshape({-1, x.size(-1)}); }

// The sizes of x with another last dimension.
std::vector<int64_t> sizes_with(const Tensor& x, int64_t last) {
  std::vector<int64_t> sizes = x.sizes().vec();
  sizes.back() = last;
  return sizes;
}

// ---- 4-bit operands ------------------------------------------------------------------------------------------------
// Where an operand's codes, scales and row scales lie.
struct Fp4 {
  uint8_t* codes = nullptr;
  uint8_t* scales = nullptr;
  float* row_scale = nullptr;
  int64_t rows = 0, K = 0, tiles = 0;
  int fmt = 0;
};

void check_format(int64_t fmt) { TORCH_CHECK_VALUE(fmt == 1 || fmt == 2, "unknown 4-bit format ", fmt); }

void check_columns(int64_t K, const char* what) {
  TORCH_CHECK_VALUE(K >= 32 && K % 32 == 0 && K <= ecz::kFp4MaxK, what, ": columns must be a multiple of 32, up to ",
                    ecz::kFp4MaxK, " (got ", K, ")");
}

// Rows of activations in one buffer of bytes: scales, codes, row scales, each from a multiple of 256 bytes on.
struct Fp4Layout {
  int64_t scales, codes, row_scale, bytes;
};

Fp4Layout fp4_layout(const Fp4& x) {
  Fp4Layout l;
  l.scales = 0;
  l.codes = (x.rows + 127) / 128 * x.tiles * 512;
  l.row_scale = l.codes + (x.rows * x.K / 2 + 255) / 256 * 256;
  l.bytes = l.row_scale + (x.fmt == 1 ? 4 * x.rows : 0);
  return l;
}

Fp4 fp4_shape(int64_t rows, int64_t K, int64_t fmt) {
  Fp4 x;
  x.rows = rows;
  x.K = K;
  x.fmt = static_cast<int>(fmt);
  x.tiles = ecz::fp4_scale_tiles(x.fmt, static_cast<int>(K));
  return x;
}

void fp4_place(Fp4& x, void* data) {
  const Fp4Layout l = fp4_layout(x);
  uint8_t* p = static_cast<uint8_t*>(data);
  x.scales = p;
  x.codes = p + l.codes;
  x.row_scale = x.fmt == 1 ? reinterpret_cast<float*>(p + l.row_scale) : nullptr;
}

Tensor fp4_buffer(Fp4& x, const Tensor& like) {
  Tensor data = at::empty({fp4_layout(x).bytes}, like.options().dtype(at::kByte));
  fp4_place(x, data.data_ptr());
  return data;
}

// x [M, K] into `to`. pad: scales of the rows up to a multiple of 128 become zeros; early: see launch_fp4_quantize.
void quantize_into(Tensor x, const Fp4& to, bool pad, bool early) {
  if (to.rows == 0) return;
  x = rows_of(x);
  if (!aligned(x, 32)) x = x.clone(at::MemoryFormat::Contiguous);
  const int rc = ecz::launch_fp4_quantize(x.data_ptr(), row_stride(x), to.fmt, to.codes, to.scales, to.row_scale,
                                          static_cast<int>(to.rows), static_cast<int>(to.K), pad, early,
                                          ecz::device_sms(x.get_device()), at::cuda::getCurrentCUDAStream());
  TORCH_CHECK(rc == 0, "fp4_quantize: launch failed");
}

// x [..., K] in 4 bits (a buffer as in Fp4Layout).
Tensor fp4_quantize(const Tensor& x, int64_t fmt) {
  CHECK_CUDA(x);
  CHECK_BF16(x);
  check_format(fmt);
  TORCH_CHECK_VALUE(x.dim() >= 1, "fp4_quantize expects x [..., K]");
  check_columns(x.size(-1), "fp4_quantize");
  c10::cuda::CUDAGuard guard(x.device());
  const Tensor rows = as_rows(x);
  TORCH_CHECK_VALUE(rows.size(0) <= kMaxRows, "fp4_quantize: too many rows");
  Fp4 to = fp4_shape(rows.size(0), x.size(-1), fmt);
  Tensor data = fp4_buffer(to, x);
  // any kernel may come next, those among them that fetch weights ahead of their wait: no early start
  quantize_into(rows, to, true, false);
  return data;
}

Fp4 check_buffer(const Tensor& data, int64_t rows, int64_t K, int64_t fmt, const char* what) {
  check_format(fmt);
  check_columns(K, what);
  TORCH_CHECK_VALUE(rows >= 0 && rows <= kMaxRows, what, ": ", rows, " rows");
  Fp4 x = fp4_shape(rows, K, fmt);
  TORCH_CHECK_VALUE(data.is_cuda() && data.scalar_type() == at::kByte && data.dim() == 1 && data.is_contiguous() &&
                        data.size(0) == fp4_layout(x).bytes && reinterpret_cast<uintptr_t>(data.data_ptr()) % 256 == 0,
                    what, ": not a buffer of ", rows, " x ", K, " 4-bit values");
  fp4_place(x, data.data_ptr());
  return x;
}

// Codes, scales and row scales of one operand belong together and lie on the device of ref.
Fp4 check_operand(const Tensor& codes, const Tensor& scales, const Tensor& row_scale, int64_t fmt, const Tensor& ref,
                  const char* what) {
  check_format(fmt);
  TORCH_CHECK(codes.is_cuda() && codes.get_device() == ref.get_device() && scales.is_cuda() &&
                  scales.get_device() == ref.get_device(),
              what, ": codes and scales must be on the device of the call");
  TORCH_CHECK(codes.scalar_type() == at::kByte && scales.scalar_type() == at::kByte && codes.dim() == 2 &&
                  codes.is_contiguous() && scales.is_contiguous(),
              what, ": codes [rows, K / 2] and scales must be contiguous uint8");
  Fp4 o;
  o.fmt = static_cast<int>(fmt);
  o.rows = codes.size(0);
  o.K = codes.size(1) * 2;
  check_columns(o.K, what);
  TORCH_CHECK(o.rows <= kMaxRows, what, ": too many rows");
  o.tiles = ecz::fp4_scale_tiles(o.fmt, static_cast<int>(o.K));
  TORCH_CHECK(scales.dim() == 3 && scales.size(0) == (o.rows + 127) / 128 && scales.size(1) == o.tiles &&
                  scales.size(2) == 512,
              what, ": scales must be [", (o.rows + 127) / 128, ", ", o.tiles, ", 512], got ", scales.sizes());
  o.codes = codes.data_ptr<uint8_t>();
  o.scales = scales.data_ptr<uint8_t>();
  if (fmt == 1) {
    TORCH_CHECK(row_scale.is_cuda() && row_scale.get_device() == ref.get_device() &&
                    row_scale.scalar_type() == at::kFloat && row_scale.dim() == 1 && row_scale.size(0) == o.rows &&
                    row_scale.is_contiguous(),
                what, ": nvfp4 has an fp32 scale per row");
    o.row_scale = row_scale.data_ptr<float>();
  }
  TORCH_CHECK(reinterpret_cast<uintptr_t>(o.codes) % 16 == 0 && reinterpret_cast<uintptr_t>(o.scales) % 16 == 0,
              what, ": codes and scales must start on 16-byte boundaries");
  return o;
}

Tensor dequantize(const Fp4& x, const Tensor& like) {
  c10::cuda::CUDAGuard guard(like.device());
  Tensor out = at::empty({x.rows, x.K}, like.options().dtype(at::kBFloat16));
  if (x.rows == 0) return out;
  const int rc = ecz::launch_fp4_dequantize(x.codes, x.scales, x.row_scale, x.fmt, out.data_ptr(),
                                            static_cast<int>(x.rows), static_cast<int>(x.K),
                                            ecz::device_sms(like.get_device()), at::cuda::getCurrentCUDAStream());
  TORCH_CHECK(rc == 0, "fp4_dequantize: launch failed");
  return out;
}

Tensor fp4_dequantize(const Tensor& codes, const Tensor& scales, const Tensor& row_scale, int64_t fmt) {
  CHECK_CUDA(codes);
  return dequantize(check_operand(codes, scales, row_scale, fmt, codes, "fp4_dequantize"), codes);
}

Tensor fp4_values(const Tensor& data, int64_t rows, int64_t K, int64_t fmt) {
  return dequantize(check_buffer(data, rows, K, fmt, "fp4_values"), data);
}

CUtensorMap codes_map(const Fp4& x, int box_rows) {
  CUtensorMap map;
  std::memset(&map, 0, sizeof(map));
  const int rc = ecz::make_tmap_2d(&map, 1, x.codes, x.rows, x.K / 2, x.K / 2, 128, box_rows, 128);
  TORCH_CHECK(rc == 0, "cuTensorMapEncodeTiled failed (code ", rc, ") for codes of ", x.rows, " x ", x.K);
  return map;
}

// Scales as rows of 128 bytes, one box the K block of 128 rows.
CUtensorMap scales_map(const Fp4& x) {
  CUtensorMap map;
  std::memset(&map, 0, sizeof(map));
  const int rc = ecz::make_tmap_2d(&map, 1, x.scales, (x.rows + 127) / 128 * x.tiles * 4, 128, 128, 128,
                                   x.fmt == 1 ? 16 : 8, 0);
  TORCH_CHECK(rc == 0, "cuTensorMapEncodeTiled failed (code ", rc, ") for scales of ", x.rows, " x ", x.K);
  return map;
}

// y [M, N] of operands [M, K] and [N, K] of one format. path: 0 by the sizes, 1 gemm_fp4.cu, 2 gemm_fp4_pair.cu.
void multiply(const Fp4& x, const Fp4& w, const Tensor& y, const at::Device& device, int64_t path = 0) {
  TORCH_CHECK_VALUE(path >= 0 && path <= 2, "fp4 product: path must be 0, 1 or 2");
  TORCH_CHECK_VALUE(x.K == w.K, "fp4 product: activations have ", x.K, " columns, the weight ", w.K);
  TORCH_CHECK_VALUE(w.rows >= 1, "fp4 product: the weight has no rows");
  if (x.rows == 0) return;
  const int M = static_cast<int>(x.rows), N = static_cast<int>(w.rows), K = static_cast<int>(x.K);
  const int sms = ecz::device_sms(device.index());
  unsigned* status = ecz::device_status(device);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  int rc;
  if (path == 2 || (path == 0 && M > 128)) {
    ecz::Fp4PairMaps maps{codes_map(x, 128), codes_map(w, 128), scales_map(x), scales_map(w), {}};
    if (N % 8 == 0)
      TORCH_CHECK(ecz::make_tmap_2d(&maps.y, 2, y.data_ptr(), M, N, int64_t{2} * N, 32, 32, 64) == 0,
                  "cuTensorMapEncodeTiled failed for a ", M, " x ", N, " result");
    rc = ecz::launch_gemm_fp4_pair(maps, x.row_scale, w.row_scale, x.fmt, y.data_ptr(), M, N, K, sms, status, stream);
  } else {
    const CUtensorMap tw = codes_map(w, 128), tx = codes_map(x, ecz::fp4_block_rows(M));
    rc = ecz::launch_gemm_fp4(&tw, &tx, w.scales, x.scales, w.row_scale, x.row_scale, x.fmt, y.data_ptr(), M, N, K, sms,
                              status, stream);
  }
  TORCH_CHECK(rc == 0, "fp4 product: launch failed");
}

// 4-bit activations (a buffer) times a 4-bit weight.
Tensor fp4_matmul(const Tensor& data, int64_t rows, int64_t K, const Tensor& w, const Tensor& ws, const Tensor& wr,
                  int64_t fmt, int64_t path) {
  const Fp4 a = check_buffer(data, rows, K, fmt, "fp4_matmul"), b = check_operand(w, ws, wr, fmt, data, "fp4_matmul: weight");
  c10::cuda::CUDAGuard guard(data.device());
  Tensor y = at::empty({a.rows, b.rows}, data.options().dtype(at::kBFloat16));
  multiply(a, b, y, data.device(), path);
  return y;
}

// Activations [..., K] times a 4-bit weight [N, K]: quantised first, in a workspace. The result has x's type.
Tensor linear_fp4(const Tensor& x, const Tensor& w, const Tensor& ws, const Tensor& wr, int64_t fmt) {
  CHECK_CUDA(x);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.is_floating_point(), "linear_fp4 expects floating point x [..., K]");
  const Fp4 b = check_operand(w, ws, wr, fmt, x, "linear_fp4: weight");
  TORCH_CHECK_VALUE(x.size(-1) == b.K, "linear_fp4: x has ", x.size(-1), " columns, the weight ", b.K);
  c10::cuda::CUDAGuard guard(x.device());
  const bool cast = x.scalar_type() != at::kBFloat16;
  const Tensor rows = as_rows(cast ? x.detach().to(at::kBFloat16) : x.detach());
  Fp4 a = fp4_shape(rows.size(0), b.K, fmt);
  TORCH_CHECK_VALUE(a.rows <= kMaxRows, "linear_fp4: too many rows");
  // scales of the rows that complete a tile stay as they are: they reach only sums that nothing reads
  Tensor work = fp4_buffer(a, w);
  Tensor y = at::empty(sizes_with(x, b.rows), rows.options());
  quantize_into(rows, a, false, true);  // the product waits before it reads
  multiply(a, b, y, x.device());
  return cast ? y.to(x.scalar_type()) : y;
}

// ---- norms around a block ------------------------------------------------------------------------------------------
ecz::NormType norm_type(const Tensor& x) {
  switch (x.scalar_type()) {
    case at::kBFloat16: return ecz::kNormBf16;
    case at::kHalf: return ecz::kNormFp16;
    case at::kFloat: return ecz::kNormFp32;
    default: TORCH_CHECK_VALUE(false, "block_norm takes bfloat16, float16 or float32, got ", x.scalar_type());
  }
}

struct NormOperands {
  Tensor x, residual, weight, post, gate;
  int gate_mode = ecz::kGateNone;
  bool vec = false;
};

// Checked operands, rows readable in place. Undefined: residual, post and gate that are not given.
NormOperands norm_operands(const Tensor& x, const Tensor& residual, const Tensor& weight, const Tensor& post,
                           const Tensor& gate, double scale, double eps) {
  const int64_t T = x.size(0), H = x.size(1);
  TORCH_CHECK_VALUE(H >= 1 && H <= ecz::kBlockNormMaxHidden, "block_norm: 1 to ", ecz::kBlockNormMaxHidden,
                    " columns (got ", H, ")");
  TORCH_CHECK_VALUE(T <= kMaxRows, "block_norm: too many rows");
  TORCH_CHECK_VALUE(std::isfinite(scale) && std::isfinite(eps) && eps >= 0,
                    "block_norm: scale and eps must be finite, eps >= 0");
  for (const Tensor* t : {&residual, &weight, &post, &gate}) {
    if (!t->defined()) continue;
    TORCH_CHECK_VALUE(t->scalar_type() == x.scalar_type() && t->is_cuda() && t->get_device() == x.get_device(),
                      "block_norm: all operands must have one type and device, got ", x.scalar_type(), " on ", x.device(),
                      " and ", t->scalar_type(), " on ", t->device());
  }
  TORCH_CHECK_VALUE(weight.defined() && weight.dim() == 1 && weight.size(0) == H, "block_norm: weight must be [", H, "]");
  TORCH_CHECK_VALUE(!post.defined() || (post.dim() == 1 && post.size(0) == H), "block_norm: post_weight must be [", H, "]");
  TORCH_CHECK_VALUE(!residual.defined() || residual.sizes() == x.sizes(), "block_norm: the residual does not match x");
  NormOperands o;
  o.x = rows_of(x);
  o.weight = weight.contiguous();
  if (residual.defined()) o.residual = rows_of(residual);
  if (post.defined()) o.post = post.contiguous();
  if (gate.defined()) {
    TORCH_CHECK_VALUE(gate.dim() == 2 && gate.size(0) == T && (gate.size(1) == 1 || gate.size(1) == H),
                      "block_norm: the gate must have one value per token or per element");
    o.gate_mode = gate.size(1) == 1 ? ecz::kGateToken : ecz::kGateFull;
    o.gate = o.gate_mode == ecz::kGateFull ? rows_of(gate) : gate;
  }
  // rows of whole 16-byte groups are read in such groups, from copies where they do not start on a boundary (a token's
  // gate is read by itself): a row's sums then do not depend on where it lies
  o.vec = H * x.element_size() % 16 == 0;
  for (Tensor* t : {&o.x, &o.residual, &o.gate})
    if (t->defined() && !(t == &o.gate && o.gate_mode == ecz::kGateToken)) *t = norm_rows(*t, o.vec);
  if (o.vec)
    for (Tensor* t : {&o.weight, &o.post}) *t = on_boundary(*t);
  return o;
}

const void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

ecz::BlockNormArgs norm_args(const NormOperands& o, double scale, double eps) {
  ecz::BlockNormArgs a;
  a.x = ptr(o.x);
  a.residual = ptr(o.residual);
  a.weight = ptr(o.weight);
  a.post = ptr(o.post);
  a.gate = ptr(o.gate);
  a.x_stride = row_stride(o.x);
  a.r_stride = o.residual.defined() ? row_stride(o.residual) : 0;
  a.gate_stride = o.gate.defined() ? (o.gate.size(0) > 1 ? o.gate.stride(0) : 0) : 0;
  a.gate_mode = o.gate_mode;
  a.rows = static_cast<int>(o.x.size(0));
  a.hidden = static_cast<int>(o.x.size(1));
  a.scale = static_cast<float>(scale);
  a.eps = static_cast<float>(eps);
  return a;
}

struct NormResult {
  Tensor normed, stream, inv_s, inv_x;
};

NormResult norm_forward(const Tensor& x, const Tensor& residual, const Tensor& weight, const Tensor& post,
                        const Tensor& gate, double scale, double eps, bool training) {
  c10::cuda::CUDAGuard guard(x.device());
  const NormOperands o = norm_operands(x, residual, weight, post, gate, scale, eps);
  const auto f32 = x.options().dtype(at::kFloat);
  NormResult r;
  r.normed = at::empty(x.sizes(), x.options());
  r.stream = at::empty(x.sizes(), x.options());
  if (training) {
    r.inv_s = at::empty({x.size(0)}, f32);
    r.inv_x = at::empty({post.defined() ? x.size(0) : 0}, f32);
  }
  if (x.size(0) == 0) return r;
  ecz::BlockNormArgs a = norm_args(o, scale, eps);
  a.normed = r.normed.data_ptr();
  a.stream = r.stream.data_ptr();
  if (training) {
    a.inv_s = r.inv_s.data_ptr<float>();
    if (post.defined()) a.inv_x = r.inv_x.data_ptr<float>();
  }
  TORCH_CHECK(ecz::launch_block_norm(a, norm_type(x), o.vec, 0, ecz::device_sms(x.get_device()),
                                     at::cuda::getCurrentCUDAStream()) == 0,
              "block_norm: launch failed");
  return r;
}

Tensor value(const c10::optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }

// The operands [..., H] of a call as rows.
struct NormCall {
  Tensor x, residual, post, gate;
};

NormCall norm_call(const Tensor& x, const c10::optional<Tensor>& residual, const c10::optional<Tensor>& post,
                   const c10::optional<Tensor>& gate) {
  CHECK_CUDA(x);
  norm_type(x);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "block_norm expects x [..., H]");
  NormCall c{x, value(residual), value(post), value(gate)};
  TORCH_CHECK_VALUE(!c.residual.defined() || c.residual.sizes() == x.sizes(), "block_norm: residual ", c.residual.sizes(),
                    " does not match x ", x.sizes());
  TORCH_CHECK_VALUE(!c.gate.defined() || c.gate.sizes() == x.sizes() || c.gate.sizes() == at::IntArrayRef(sizes_with(x, 1)),
                    "block_norm: gate ", c.gate.sizes(), " must be like x ", x.sizes(), " or have a last dimension of 1");
  if (x.dim() != 2) {
    c.x = as_rows(x);
    if (c.residual.defined()) c.residual = as_rows(c.residual);
    if (c.gate.defined()) c.gate = as_rows(c.gate);
  }
  return c;
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// A tensor that the forward pass saved is what it was: saved-tensor hooks may return anything, and kernels read it by its
// pointer.
void check_saved(const Tensor& x, const Tensor& like, at::ScalarType type, at::IntArrayRef sizes, const char* what) {
  TORCH_CHECK(x.defined() && x.is_cuda() && x.get_device() == like.get_device() && x.scalar_type() == type &&
                  x.sizes() == sizes && x.is_contiguous(),
              "block_norm: the saved ", what, " did not come back as it was saved (device, type, sizes, contiguous)");
}

// Without a norm behind the block and a gate the backward pass needs the stream alone, half of what x and the residual are
// to read. In fp32 it takes the one that the forward pass returned. One that was rounded to 16 bits would double the error
// of dweight, which sums its values over the tokens (8192 rows of 4096 in bf16: 0.0024 of itself, of which 0.0016 are its
// own rounding), so there the stream is formed again from x and the residual.
bool from_stream(const Tensor& weight, const Tensor& post, const Tensor& gate) {
  return weight.scalar_type() == at::kFloat && !post.defined() && !gate.defined();
}

struct BlockNormFunction : torch::autograd::Function<BlockNormFunction> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const c10::optional<Tensor>& residual_,
                               const Tensor& weight, const c10::optional<Tensor>& post_,
                               const c10::optional<Tensor>& gate_, double scale, double eps) {
    const Tensor residual = value(residual_), post = value(post_), gate = value(gate_);
    NormResult r = norm_forward(x, residual, weight, post, gate, scale, eps, true);
    const bool whole = from_stream(weight, post, gate);
    ctx->save_for_backward({whole ? Tensor() : x, whole ? Tensor() : residual, weight, post, gate,
                            whole ? r.stream : Tensor(), r.inv_s, r.inv_x});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["residual"] = residual.defined();
    ctx->set_materialize_grads(false);
    return {r.normed, r.stream};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "block_norm cannot be differentiated twice");
    const auto s = ctx->get_saved_variables();
    const Tensor &weight = s[2], &post = s[3], &gate = s[4], &stream = s[5], &inv_s = s[6], &inv_x = s[7];
    const double scale = ctx->saved_data["scale"].toDouble(), eps = ctx->saved_data["eps"].toDouble();
    const bool whole = from_stream(weight, post, gate);
    size_t input = 0;  // tensors that were not given have no place among the inputs
    auto needs = [&](bool given) { return given && ctx->needs_input_grad(input++); };
    const bool need_x = needs(true), need_r = needs(ctx->saved_data["residual"].toBool()), need_w = needs(true);
    const bool need_p = needs(post.defined()), need_g = needs(gate.defined());
    variable_list out(7);
    Tensor dn = grads[0], up = grads[1];
    if (!dn.defined() && !up.defined()) return out;
    const Tensor& like = dn.defined() ? dn : up;
    const int64_t T = like.size(0), H = like.size(1);
    if (whole) check_saved(stream, weight, weight.scalar_type(), {T, H}, "stream");
    c10::cuda::CUDAGuard guard(weight.device());
    // the operands as in the forward pass (the stream in x's place where it alone was saved)
    norm_type(weight);
    const NormOperands o = norm_operands(whole ? stream : s[0], whole ? Tensor() : s[1], weight, post, gate, scale, eps);
    for (const Tensor* t : {&dn, &up})
      TORCH_CHECK(!t->defined() || (t->is_cuda() && t->get_device() == o.x.get_device() &&
                                    t->scalar_type() == o.x.scalar_type() && t->sizes() == o.x.sizes()),
                  "block_norm: a gradient does not match its output");
    check_saved(inv_s, o.x, at::kFloat, {T}, "norms");
    check_saved(inv_x, o.x, at::kFloat, {post.defined() ? T : 0}, "norms of the block's output");
    const auto opts = o.x.options();
    const bool shared = !post.defined() && !gate.defined() && scale == 1.0;  // both gradients are the same values
    Tensor dx, dr, dw, dp, dg;
    if (need_x && !shared) dx = at::empty({T, H}, opts);
    if (need_r || (need_x && shared)) dr = at::empty({T, H}, opts);
    if (need_w) dw = at::empty({H}, opts);
    if (need_p) dp = at::empty({H}, opts);
    if (need_g) dg = at::empty(gate.sizes(), opts);
    if (T == 0) {
      if (need_w) dw.zero_();
      if (need_p) dp.zero_();
    } else {
      if (dn.defined()) dn = norm_rows(rows_of(dn), o.vec);
      if (up.defined()) up = norm_rows(rows_of(up), o.vec);
      const ecz::NormType type = norm_type(o.x);
      const int sms = ecz::device_sms(o.x.get_device());
      ecz::BlockNormGrads a;
      a.dnormed = ptr(dn);
      a.dstream = ptr(up);
      a.dn_stride = dn.defined() ? row_stride(dn) : 0;
      a.ds_stride = up.defined() ? row_stride(up) : 0;
      const ecz::BlockNormArgs f = norm_args(o, scale, eps);
      a.x = f.x;
      a.residual = f.residual;
      a.stream = whole ? f.x : nullptr;
      a.weight = f.weight;
      a.post = f.post;
      a.gate = f.gate;
      a.x_stride = f.x_stride;
      a.r_stride = f.r_stride;
      a.gate_stride = f.gate_stride;
      a.gate_mode = f.gate_mode;
      a.inv_s = inv_s.data_ptr<float>();
      a.inv_x = post.defined() ? inv_x.data_ptr<float>() : nullptr;
      a.dx = const_cast<void*>(ptr(dx));
      a.dresidual = const_cast<void*>(ptr(dr));
      a.dgate = const_cast<void*>(ptr(dg));
      a.dweight = const_cast<void*>(ptr(dw));
      a.dpost = const_cast<void*>(ptr(dp));
      a.rows = f.rows;
      a.hidden = f.hidden;
      a.scale = f.scale;
      Tensor parts;
      if (need_w || need_p) {
        const int n = ecz::block_norm_parts(type, a.rows, a.hidden, o.vec, whole, sms);
        parts = at::empty({(need_w ? 1 : 0) + (need_p ? 1 : 0), n, H}, opts.dtype(at::kFloat));
        float* p = parts.data_ptr<float>();
        if (need_w) a.dw_part = p;
        if (need_p) a.dpost_part = p + (need_w ? static_cast<int64_t>(n) * H : 0);
      }
      TORCH_CHECK(ecz::launch_block_norm_grads(a, type, o.vec, sms, at::cuda::getCurrentCUDAStream()) == 0,
                  "block_norm: backward launch failed");
    }
    if (need_x) out[0] = shared ? dr : dx;
    if (need_r) out[1] = dr;
    if (need_w) out[2] = dw;
    if (need_p) out[3] = dp;
    if (need_g) out[4] = dg;
    return out;
  }
};

// A leaf's gradients are added up on the stream of the first graph that holds the leaf. Where that is the default stream,
// which cannot join a capture, and that graph still lives, the engine would break off the captured backward pass, and the
// process with it. An operand is often not the leaf itself but its rows, a view or a cast of it (as_rows, autocast): its
// history is followed as long as it has one input.
void check_captured_leaf(const Tensor& t) {
  if (!t.defined() || !t.requires_grad()) return;
  auto node = t.is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(t) : t.grad_fn();
  while (node && node->num_outputs() == 1) node = node->next_edge(0).function;
  if (!node || dynamic_cast<torch::autograd::AccumulateGrad*>(node.get()) == nullptr) return;
  const auto stream = node->stream();
  TORCH_CHECK(!stream.has_value() || c10::cuda::CUDAStream(*stream) != c10::cuda::getDefaultCUDAStream(t.get_device()),
              "block_norm: a graph made on the default stream still holds a leaf of this captured call, whose backward "
              "pass could not be captured; drop that graph, or make it on a side stream");
}

// Whether the call becomes part of a graph.
bool differentiated(const NormCall& c, const Tensor& weight) {
  bool grad = false;
  for (const Tensor* t : {&c.x, &c.residual, &weight, &c.post, &c.gate}) {
    if (!t->defined()) continue;
    grad |= t->requires_grad();
    // the kernels carry no tangents: refused, or a dual number's would be dropped without a word
    TORCH_CHECK(!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t->_fw_grad(0).defined(),
                "block_norm has no forward-mode derivative on CUDA");
  }
  return grad && at::GradMode::is_enabled();
}

std::tuple<Tensor, Tensor> block_norm(const Tensor& x, const c10::optional<Tensor>& residual, const Tensor& weight,
                                      const c10::optional<Tensor>& post, const c10::optional<Tensor>& gate, double scale,
                                      double eps) {
  const NormCall c = norm_call(x, residual, post, gate);
  Tensor normed, stream;
  if (differentiated(c, weight)) {
    c10::cuda::CUDAGuard guard(x.device());
    if (at::cuda::currentStreamCaptureStatus() != at::cuda::CaptureStatus::None)
      for (const Tensor* t : {&c.x, &c.residual, &weight, &c.post, &c.gate}) check_captured_leaf(*t);
    auto given = [](const Tensor& t) { return t.defined() ? c10::optional<Tensor>(t) : c10::nullopt; };
    auto out = BlockNormFunction::apply(c.x, given(c.residual), weight, given(c.post), given(c.gate), scale, eps);
    normed = out[0];
    stream = out[1];
  } else {
    NormResult out = norm_forward(c.x, c.residual, weight, c.post, c.gate, scale, eps, false);
    normed = out.normed;
    stream = out.stream;
  }
  if (x.dim() != 2) return {normed.view(x.sizes()), stream.view(x.sizes())};
  return {normed, stream};
}

// normed in 4 bits (a buffer), and the stream. The 4-bit result has no gradient; where the call is differentiated the
// stream keeps its own, and the two operators run one after the other, with the same bits.
std::tuple<Tensor, Tensor> block_norm_fp4(const Tensor& x, const c10::optional<Tensor>& residual, const Tensor& weight,
                                          const c10::optional<Tensor>& post, const c10::optional<Tensor>& gate,
                                          double scale, double eps, int64_t fmt) {
  check_format(fmt);
  CHECK_CUDA(x);
  TORCH_CHECK_VALUE(x.scalar_type() == at::kBFloat16, "block_norm in 4 bits takes bfloat16, got ", x.scalar_type());
  const NormCall c = norm_call(x, residual, post, gate);
  check_columns(x.size(-1), "block_norm in 4 bits");
  c10::cuda::CUDAGuard guard(x.device());
  if (differentiated(c, weight)) {
    const auto [normed, stream] = block_norm(x, residual, weight, post, gate, scale, eps);
    return {fp4_quantize(normed.detach(), fmt), stream};
  }
  const NormOperands o = norm_operands(c.x, c.residual, weight, c.post, c.gate, scale, eps);
  Fp4 to = fp4_shape(c.x.size(0), c.x.size(1), fmt);
  Tensor data = fp4_buffer(to, x), stream = at::empty(x.sizes(), x.options());
  if (to.rows == 0) return {data, stream};
  ecz::BlockNormArgs a = norm_args(o, scale, eps);
  a.stream = stream.data_ptr();
  a.codes = to.codes;
  a.scales = to.scales;
  a.row_scale = to.row_scale;
  a.tiles = static_cast<int>(to.tiles);
  TORCH_CHECK(ecz::launch_block_norm(a, ecz::kNormBf16, true, static_cast<int>(fmt), ecz::device_sms(x.get_device()),
                                     at::cuda::getCurrentCUDAStream()) == 0,
              "block_norm: launch failed");
  return {data, stream};
}

}  // namespace

namespace ecz {

void bind_block(pybind11::module_& m) {
  namespace py = pybind11;
  m.def("fp4_quantize", &fp4_quantize, "bf16 rows in 4 bits, one buffer (fmt 1 nvfp4, 2 mxfp4)", py::arg("x"),
        py::arg("fmt"));
  m.def("fp4_values", &fp4_values, "the bf16 values of such a buffer", py::arg("data"), py::arg("rows"), py::arg("K"),
        py::arg("fmt"));
  m.def("fp4_dequantize", &fp4_dequantize, "the bf16 values of a 4-bit weight", py::arg("codes"), py::arg("scales"),
        py::arg("row_scale"), py::arg("fmt"));
  m.def("fp4_matmul", &fp4_matmul, "4-bit activations times a 4-bit weight (tcgen05 block-scaled MMA)", py::arg("data"),
        py::arg("rows"), py::arg("K"), py::arg("w"), py::arg("w_scales"), py::arg("w_row_scale"), py::arg("fmt"),
        py::arg("path") = 0);
  m.def("linear_fp4", &linear_fp4, "bf16 activations quantised and multiplied with a 4-bit weight", py::arg("x"),
        py::arg("w"), py::arg("w_scales"), py::arg("w_row_scale"), py::arg("fmt"));
  m.def("block_norm", &block_norm, "norm after a block, gate, residual scale and sum, norm before the next (autograd)",
        py::arg("x"), py::arg("residual"), py::arg("weight"), py::arg("post_weight"), py::arg("gate"), py::arg("scale"),
        py::arg("eps"));
  m.def("block_norm_fp4", &block_norm_fp4, "block_norm with its result in 4 bits", py::arg("x"), py::arg("residual"),
        py::arg("weight"), py::arg("post_weight"), py::arg("gate"), py::arg("scale"), py::arg("eps"), py::arg("fmt"));
}

}  // namespace ecz
