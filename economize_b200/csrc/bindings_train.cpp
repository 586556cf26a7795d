// PyTorch bindings of the training operators (readout.cu, packed_attention.cu): argument checks, workspaces from
// PyTorch's caching allocator, tensor maps, and the launches on the current stream.
#include <ATen/cuda/CUDAContext.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/graph_task.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <tuple>

#include "bindings.h"
#include "launchers.h"

namespace {

using at::Tensor;

// bf16 [rows, cols] (row stride in elements), 128-byte swizzle, box {64, box_rows}.
CUtensorMap map_2d(const void* base, int64_t rows, int64_t cols, int64_t stride, int box_rows) {
  CUtensorMap map;
  std::memset(&map, 0, sizeof(map));
  const int rc = ecz::make_tmap_2d(&map, 2, base, rows, cols, stride * 2, 64, box_rows, 128);
  TORCH_CHECK(rc == 0, "cuTensorMapEncodeTiled failed (code ", rc, ") for rows=", rows, " cols=", cols);
  return map;
}

// Elements from one row to the next (a single row's stride says nothing).
int64_t row_stride(const Tensor& x) { return x.size(0) > 1 ? x.stride(0) : x.size(1); }

// A row-major operand the kernels read in 16-byte groups: rows may be further apart than they are long.
Tensor rows_of(const Tensor& x) {
  const bool ok = x.stride(1) == 1 && row_stride(x) >= x.size(1) && row_stride(x) % 8 == 0 &&
                  reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
  if (ok) return x;
  Tensor y = x.contiguous();
  return reinterpret_cast<uintptr_t>(y.data_ptr()) % 16 == 0 ? y : y.clone();
}

// A tensor that the forward pass saved is what it was: saved-tensor hooks may return anything, and kernels read it by its
// pointer.
void check_saved(const Tensor& x, const Tensor& like, at::ScalarType type, at::IntArrayRef sizes, const char* what) {
  TORCH_CHECK(x.defined() && x.is_cuda() && x.get_device() == like.get_device() && x.scalar_type() == type &&
                  x.sizes() == sizes && x.is_contiguous() && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0,
              "the saved ", what, " did not come back as it was saved (device, type, sizes, contiguous)");
}

// What a chunk of rows may hold of unnormalised probabilities (2 bytes each).
constexpr int64_t kChunkBytes = int64_t{1} << 30;

// Losses and, where asked for, gradients of the readout (see ops.linear_cross_entropy). reduction 0: per-row losses
// [T]; 1 / 2: their mean / sum as a scalar. grad_rows: the per-row upstream gradient of reduction 0 (then no loss is
// returned); reductions 1 and 2 compute the gradients of the scalar itself.
std::tuple<Tensor, c10::optional<Tensor>, c10::optional<Tensor>> readout(
    Tensor hidden, Tensor weight, Tensor targets, int64_t ignore_index, double logit_scale, int64_t reduction,
    bool need_dx, bool need_dw, c10::optional<Tensor> grad_rows, int64_t chunk_rows) {
  CHECK_CUDA(hidden);
  CHECK_BF16(hidden);
  CHECK_BF16(weight);
  CHECK_I64(targets);
  CHECK_ON(weight, hidden);
  CHECK_ON(targets, hidden);
  TORCH_CHECK(hidden.dim() == 2 && weight.dim() == 2 && targets.dim() == 1,
              "readout expects hidden [T, H], weight [V, H] and targets [T]");
  const int64_t T = hidden.size(0), H = hidden.size(1), V = weight.size(0);
  TORCH_CHECK(weight.size(1) == H, "hidden has ", H, " columns, weight ", weight.size(1));
  TORCH_CHECK(targets.size(0) == T, "hidden has ", T, " rows, targets ", targets.size(0));
  TORCH_CHECK(H >= 8 && H % 8 == 0, "readout: the hidden size must be a multiple of 8 (got ", H, ")");
  TORCH_CHECK(V >= 1 && V <= (int64_t{1} << 22), "readout: 1 to 4194304 vocabulary rows (got ", V, ")");
  TORCH_CHECK(H <= (int64_t{1} << 17) && T <= (int64_t{1} << 30), "readout: hidden size or row count too large");
  TORCH_CHECK(reduction >= 0 && reduction <= 2, "unknown reduction ", reduction);
  c10::cuda::CUDAGuard guard(hidden.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  const int sms = ecz::device_sms(hidden.get_device());
  unsigned* status = ecz::device_status(hidden.device());
  Tensor x = T > 0 ? rows_of(hidden) : hidden, w = rows_of(weight);
  targets = targets.contiguous();
  const auto f32 = hidden.options().dtype(at::kFloat);
  const bool per_row = reduction == ecz::kReduceNone;
  const bool want_loss = !grad_rows.has_value();
  Tensor loss = want_loss ? (per_row ? at::empty({T}, f32) : at::empty({}, f32)) : Tensor();
  c10::optional<Tensor> dx, dw;
  if (need_dx) dx = at::empty({T, H}, hidden.options());
  if (need_dw) dw = at::empty({V, H}, weight.options());
  if (grad_rows.has_value()) {
    TORCH_CHECK(per_row && grad_rows->scalar_type() == at::kFloat && grad_rows->dim() == 1 && grad_rows->size(0) == T,
                "grad_rows must be fp32 [T] of a per-row loss");
    CHECK_ON(*grad_rows, hidden);
    grad_rows = grad_rows->contiguous();
  }
  if (T == 0) {
    if (want_loss && !per_row) loss.zero_();
    if (dw) dw->zero_();
    return {loss, dx, dw};
  }
  const bool grads = need_dx || need_dw;
  // rows of e and of the packed states start on 128-byte lines, or every row of a TMA box would touch two
  const int64_t ld = (V + 63) / 64 * 64, xld = (H + 63) / 64 * 64;
  // Rows of a chunk: 1 GiB of e; with dW as much as the fp32 sum of several chunks would take (4 V H bytes).
  int64_t chunk = T;
  if (chunk_rows > 0) {
    chunk = chunk_rows;
  } else if (grads) {
    const int64_t budget = std::max(kChunkBytes, need_dw ? 4 * V * H : int64_t{0});
    chunk = std::max<int64_t>(256, budget / (2 * ld) / 256 * 256);
  } else {
    chunk = std::max<int64_t>(256, kChunkBytes / (8 * ecz::readout_pieces(V)) / 256 * 256);
  }
  chunk = std::min((T + 63) / 64 * 64, (chunk + 63) / 64 * 64);
  const int64_t chunks = (T + chunk - 1) / chunk;

  // One workspace: row lists, losses, target logits, statistics, packed states, e, partial products.
  const int64_t pieces = ecz::readout_pieces(static_cast<int>(V));
  int64_t bytes = 0;
  auto place = [&](int64_t n) {
    const int64_t at = bytes;
    bytes += (n + 255) / 256 * 256;
    return at;
  };
  const bool planned = ecz::readout_needs_plan(static_cast<int>(T));
  const int64_t o_rows = place(4 * T), o_target = place(4 * T), o_pos = place(planned ? 4 * T : 0), o_count = place(8);
  const int64_t o_picked = place(4 * T), o_nll = place(4 * T), o_stats = place(8 * chunk * pieces);
  const int64_t o_xs = place(2 * (T + 64) * xld), o_e = place(grads ? 2 * chunk * ld : 0);
  const int64_t o_part = place(grads ? ecz::readout_part_bytes(sms) : 0);
  const int64_t o_sum = place(need_dw && chunks > 1 ? 4 * V * H : 0);
  Tensor workspace = at::empty({bytes}, hidden.options().dtype(at::kByte));
  uint8_t* ws = workspace.data_ptr<uint8_t>();
  int *rows = reinterpret_cast<int*>(ws + o_rows), *target_of = reinterpret_cast<int*>(ws + o_target);
  int *pos = planned ? reinterpret_cast<int*>(ws + o_pos) : nullptr, *count = reinterpret_cast<int*>(ws + o_count);
  float *picked = reinterpret_cast<float*>(ws + o_picked), *nll = reinterpret_cast<float*>(ws + o_nll);
  uint8_t* xs = ws + o_xs;
  void* e = grads ? ws + o_e : nullptr;

  auto check = [](int rc, const char* what) { TORCH_CHECK(rc == 0, "readout: ", what, " launch failed"); };
  ecz::ReadoutRows r;
  r.x = x.data_ptr();
  r.w = w.data_ptr();
  r.x_stride = row_stride(x);
  r.w_stride = row_stride(w);
  r.xs_stride = xld;
  r.targets = targets.data_ptr<int64_t>();
  r.T = static_cast<int>(T);
  r.H = static_cast<int>(H);
  r.V = static_cast<int>(V);
  r.ignore = ignore_index;
  r.logit_scale = static_cast<float>(logit_scale);
  if (planned)
    check(ecz::launch_readout_plan(r.targets, r.T, r.V, ignore_index, pos, count, status, stream), "plan");
  check(ecz::launch_readout_gather(r, pos, rows, target_of, count, picked, xs, need_dx ? dx->data_ptr() : nullptr,
                                   want_loss && per_row ? loss.data_ptr<float>() : nullptr, status, stream),
        "gather");
  const CUtensorMap w_rows = map_2d(w.data_ptr(), V, H, row_stride(w), 128);
  CUtensorMap w_cols;
  if (need_dx) w_cols = map_2d(w.data_ptr(), V, H, row_stride(w), 64);
  for (int64_t i = 0; i < chunks; ++i) {
    ecz::ReadoutChunk c;
    c.row0 = static_cast<int>(i * chunk);
    c.chunk = static_cast<int>(std::min(chunk, T - i * chunk));
    c.H = r.H;
    c.V = r.V;
    c.rows = rows;
    c.target = target_of;
    c.count = count;
    c.stats = ws + o_stats;
    c.picked = picked;
    c.e = e;
    c.ld = ld;
    c.logit_scale = r.logit_scale;
    c.reduction = static_cast<int>(reduction);
    c.grad_rows = grad_rows.has_value() ? grad_rows->data_ptr<float>() : nullptr;
    const int64_t padded = (c.chunk + 63) / 64 * 64;  // rows of xs and e that the maps may read
    uint8_t* xs0 = xs + static_cast<int64_t>(c.row0) * xld * 2;
    const CUtensorMap x_rows = map_2d(xs0, padded, H, xld, 128);
    check(ecz::launch_readout_logits(&x_rows, &w_rows, c, sms, status, stream), "logits");
    const bool sums = want_loss && !per_row;
    check(ecz::launch_readout_finish(c, sums ? nll : nullptr, want_loss && per_row ? loss.data_ptr<float>() : nullptr,
                                     sums && i == chunks - 1 ? loss.data_ptr<float>() : nullptr, count + 1, sms, stream),
          "finish");
    if (need_dx) {
      const CUtensorMap dz = map_2d(e, padded, V, ld, 128);
      check(ecz::launch_readout_dx(&dz, &w_cols, c, reinterpret_cast<float*>(ws + o_part), dx->data_ptr(), sms,
                                   status, stream),
            "dx");
    }
    if (need_dw) {
      const CUtensorMap dz = map_2d(e, padded, V, ld, 64);
      const CUtensorMap x_cols = map_2d(xs0, padded, H, xld, 64);
      check(ecz::launch_readout_dw(&dz, &x_cols, c, reinterpret_cast<float*>(ws + o_part),
                                   chunks > 1 ? reinterpret_cast<float*>(ws + o_sum) : nullptr, i == 0,
                                   i == chunks - 1, dw->data_ptr(), sms, status, stream),
            "dw");
    }
  }
  return {loss, dx, dw};
}

// A [T, heads, D] operand as TMA reads it: unit stride along D, 16-byte strides and base.
Tensor heads_of(const Tensor& x) {
  const auto step = [&](int d) { return x.size(d) > 1 ? x.stride(d) : int64_t{8}; };
  const bool ok = x.stride(2) == 1 && step(0) > 0 && step(1) > 0 && step(0) % 8 == 0 && step(1) % 8 == 0 &&
                  reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
  if (ok) return x;
  Tensor y = x.contiguous();
  return reinterpret_cast<uintptr_t>(y.data_ptr()) % 16 == 0 ? y : y.clone();
}

CUtensorMap map_heads(const Tensor& x, int box_heads, int box_tokens) {
  CUtensorMap map;
  std::memset(&map, 0, sizeof(map));
  const auto step = [&](int d, int64_t one) { return x.size(d) > 1 ? x.stride(d) : one; };
  const int rc = ecz::make_tmap_heads(&map, x.data_ptr(), x.size(0), x.size(1), x.size(2),
                                      step(0, x.size(1) * x.size(2)), step(1, x.size(2)), box_heads, box_tokens);
  TORCH_CHECK(rc == 0, "cuTensorMapEncodeTiled failed (code ", rc, ") for a [", x.size(0), ", ", x.size(1), ", ",
              x.size(2), "] operand");
  return map;
}

void check_operands(const Tensor& q, const Tensor& k, const Tensor& v) {
  CHECK_CUDA(q);
  CHECK_BF16(q);
  CHECK_BF16(k);
  CHECK_BF16(v);
  CHECK_ON(k, q);
  CHECK_ON(v, q);
  TORCH_CHECK(q.dim() == 3 && k.dim() == 3 && v.dim() == 3, "packed_attention expects q [T, H, D], k / v [T, Hkv, D]");
  TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == q.size(0) && k.size(2) == q.size(2),
              "packed_attention: q ", q.sizes(), ", k ", k.sizes(), " and v ", v.sizes(), " do not match");
  const int64_t T = q.size(0), H = q.size(1), Hkv = k.size(1), D = q.size(2);
  TORCH_CHECK(Hkv >= 1 && H >= 1 && H % Hkv == 0, "packed_attention: ", H, " query heads over ", Hkv, " K/V heads");
  TORCH_CHECK(D >= 8 && D <= 128 && D % 8 == 0, "packed_attention: head dimensions 8 to 128 in steps of 8 (got ", D,
              ")");
  TORCH_CHECK(T <= (int64_t{1} << 26), "packed_attention: too many tokens");
}

void check_packed(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu, double scale) {
  check_operands(q, k, v);
  CHECK_I32(cu);
  CHECK_ON(cu, q);
  TORCH_CHECK(cu.dim() == 1 && cu.size(0) >= 1, "packed_attention: cu_seqlens must be [B + 1]");
  TORCH_CHECK(cu.size(0) <= (int64_t{1} << 24), "packed_attention: too many sequences");
  TORCH_CHECK(scale > 0 && std::isfinite(scale), "packed_attention: the scale must be positive (got ", scale, ")");
}

// Shapes and the places of the tile tables of `count` kernels (1: the forward pass, 3: the gradients' too) in `buf`.
ecz::PackedArgs packed_args(const Tensor& q, const Tensor& k, int64_t B, double scale, int tiles, int count,
                            const Tensor& buf) {
  ecz::PackedArgs a;
  a.T = static_cast<int>(q.size(0));
  a.H = static_cast<int>(q.size(1));
  a.Hkv = static_cast<int>(k.size(1));
  a.D = static_cast<int>(q.size(2));
  a.lp = ecz::packed_heads_log2(a.H, a.Hkv);
  a.num_sms = ecz::device_sms(q.get_device());
  a.scale = static_cast<float>(scale);
  int* at = buf.defined() ? buf.data_ptr<int>() : nullptr;
  ecz::PackedTable* tables[3] = {&a.fwd, &a.dq, &a.dkv};
  const int rows[3] = {(128 >> a.lp) * tiles, 128 >> a.lp, 128};
  for (int i = 0; i < count; ++i) {
    tables[i]->rows = rows[i];
    tables[i]->max_tiles = std::max(1, ecz::packed_max_tiles(a.T, static_cast<int>(B), rows[i]));
    if (at == nullptr) continue;
    tables[i]->entries = at;
    tables[i]->head = at + int64_t{4} * tables[i]->max_tiles;
    tables[i]->scratch = tables[i]->head + 4;
    at = tables[i]->scratch + (2 * (B + 1) + 3) / 4 * 4;
  }
  return a;
}

// Ints of the tile tables of PackedArgs, and of the forward pass's alone (count 1).
int64_t plan_ints(const ecz::PackedArgs& a, int64_t B) {
  int64_t ints = 0;
  for (const auto* t : {&a.fwd, &a.dq, &a.dkv})
    ints += t->max_tiles > 0 ? int64_t{4} * t->max_tiles + 4 + (2 * (B + 1) + 3) / 4 * 4 : 0;
  return ints;
}

// Output [T, H, D] and, for a backward pass, what its rounding left, the log2-domain log-sum-exp of every row [H, T] and
// the tile tables.
// tiles: query tiles a CTA works on (0: by the mean length).
std::tuple<Tensor, Tensor, Tensor, Tensor> packed_forward(Tensor q, Tensor k, Tensor v, Tensor cu, double scale,
                                                          bool training, int64_t tiles) {
  check_packed(q, k, v, cu, scale);
  TORCH_CHECK(tiles >= 0 && tiles <= 2, "packed_attention: tiles must be 0, 1 or 2");
  c10::cuda::CUDAGuard guard(q.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  Tensor out = at::empty(q.sizes(), q.options()), rest, lse, plan;
  if (training) {
    rest = at::empty(q.sizes(), q.options());
    lse = at::empty({q.size(1), q.size(0)}, q.options().dtype(at::kFloat));
  }
  if (q.size(0) == 0) return {out, rest, lse, plan};
  q = heads_of(q);
  k = heads_of(k);
  v = heads_of(v);
  cu = cu.contiguous();
  const int T = static_cast<int>(q.size(0)), B = static_cast<int>(cu.size(0)) - 1;
  if (tiles == 0) tiles = ecz::packed_single_tiles(T, B, static_cast<int>(q.size(2))) ? 1 : 2;
  const int count = training ? 3 : 1;
  ecz::PackedArgs a = packed_args(q, k, B, scale, static_cast<int>(tiles), count, Tensor());
  plan = at::empty({plan_ints(a, B)}, cu.options());
  a = packed_args(q, k, B, scale, static_cast<int>(tiles), count, plan);
  unsigned* status = ecz::device_status(q.device());
  const ecz::PackedTable tables[3] = {a.fwd, a.dq, a.dkv};
  TORCH_CHECK(ecz::launch_packed_plan(cu.data_ptr<int>(), B, T, tables, count, status, stream) == 0,
              "packed_attention: plan launch failed");
  ecz::PackedMaps maps;
  maps.q = map_heads(q, 1 << a.lp, 128 >> a.lp);
  maps.k = map_heads(k, 1, 128);
  maps.v = map_heads(v, 1, 128);
  maps.k32 = map_heads(k, 1, 32);
  maps.v32 = map_heads(v, 1, 32);
  const int rc = ecz::launch_packed_forward(maps, a, out.data_ptr(), training ? rest.data_ptr() : nullptr,
                                            training ? lse.data_ptr<float>() : nullptr,
                                            static_cast<int>(tiles), status, stream);
  TORCH_CHECK(rc == 0, "packed_attention: forward launch failed (", rc, ")");
  return {out, rest, lse, plan};
}

// Gradients of q, k and v (those asked for; undefined otherwise) given the output's. plan, tiles: of the forward pass
// over B sequences.
std::tuple<Tensor, Tensor, Tensor> packed_backward(Tensor dout, Tensor q, Tensor k, Tensor v, const Tensor& out,
                                                   const Tensor& rest, const Tensor& lse, const Tensor& plan,
                                                   int64_t B, double scale, int64_t tiles, bool need_dq, bool need_dkv) {
  CHECK_BF16(dout);
  CHECK_ON(dout, q);
  TORCH_CHECK(dout.sizes() == q.sizes(), "packed_attention: the output's gradient has the queries' shape");
  check_operands(q, k, v);
  c10::cuda::CUDAGuard guard(q.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  Tensor dq, dk, dv;
  if (need_dq) dq = at::empty(q.sizes(), q.options());
  if (need_dkv) {
    dk = at::empty(k.sizes(), k.options());
    dv = at::empty(v.sizes(), v.options());
  }
  if (q.size(0) == 0 || (!need_dq && !need_dkv)) return {dq, dk, dv};
  check_saved(out, q, at::kBFloat16, q.sizes(), "output");
  check_saved(rest, q, at::kBFloat16, q.sizes(), "rounding rest of the output");
  check_saved(lse, q, at::kFloat, {q.size(1), q.size(0)}, "log-sum-exps");
  check_saved(plan, q, at::kInt,
              {plan_ints(packed_args(q, k, B, scale, static_cast<int>(tiles), 3, Tensor()), B)}, "plan");
  q = heads_of(q);
  k = heads_of(k);
  v = heads_of(v);
  dout = heads_of(dout);
  const ecz::PackedArgs a = packed_args(q, k, B, scale, static_cast<int>(tiles), 3, plan);
  // delta [H, T] and the two kernels' item counters
  const int64_t rows = q.size(1) * q.size(0);
  Tensor delta = at::empty({rows + 2}, q.options().dtype(at::kFloat));
  int* taken = reinterpret_cast<int*>(delta.data_ptr<float>() + rows);
  const int splits = need_dkv ? ecz::packed_dkv_splits(a, static_cast<int>(B)) : 1;
  Tensor part;
  if (splits > 1) part = at::empty({splits, 2, k.size(0), k.size(1), k.size(2)}, delta.options());
  TORCH_CHECK(ecz::launch_packed_delta(a, out.data_ptr(), rest.data_ptr(), dout.data_ptr(), dout.stride(0),
                                       dout.stride(1), delta.data_ptr<float>(), taken, stream) == 0,
              "packed_attention: delta launch failed");
  ecz::PackedMaps maps;
  maps.q = map_heads(q, 1 << a.lp, 128 >> a.lp);
  maps.dout = map_heads(dout, 1 << a.lp, 128 >> a.lp);
  maps.k = map_heads(k, 1, 128);
  maps.v = map_heads(v, 1, 128);
  maps.k32 = map_heads(k, 1, 32);
  maps.v32 = map_heads(v, 1, 32);
  const int rc = ecz::launch_packed_backward(maps, a, lse.data_ptr<float>(), delta.data_ptr<float>(),
                                             need_dq ? dq.data_ptr() : nullptr, need_dkv ? dk.data_ptr() : nullptr,
                                             need_dkv ? dv.data_ptr() : nullptr, splits,
                                             splits > 1 ? part.data_ptr<float>() : nullptr, taken,
                                             ecz::device_status(q.device()), stream);
  TORCH_CHECK(rc == 0, "packed_attention: backward launch failed (", rc, ")");
  return {dq, dk, dv};
}

// The gradients times a scalar on the device, in place (one launch; undefined ones are skipped).
void scale_both(const Tensor& dx, const Tensor& dw, const Tensor& g) {
  const Tensor& any = dx.defined() ? dx : dw;
  if (!any.defined()) return;
  c10::cuda::CUDAGuard guard(any.device());
  TORCH_CHECK(ecz::launch_scale_by(dx.defined() ? dx.data_ptr() : nullptr, dx.defined() ? dx.numel() : 0,
                                   dw.defined() ? dw.data_ptr() : nullptr, dw.defined() ? dw.numel() : 0,
                                   g.data_ptr<float>(), ecz::device_sms(any.get_device()),
                                   at::cuda::getCurrentCUDAStream()) == 0,
              "linear_cross_entropy: scaling launch failed");
}

// ---- autograd ------------------------------------------------------------------------------------------------------
// In C++: a training step's small calls would otherwise spend more time in Python's autograd hooks than on the GPU
// (a forward and backward pair of either operator took 100 to 120 us on the host as Python functions).
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void once(const char* name) {
  TORCH_CHECK(!at::GradMode::is_enabled(), name, " cannot be differentiated twice");
}

// The kernels carry no tangents: refused, or a dual number's would be dropped without a word.
template <class... Operands>
void no_tangent(const char* name, const Operands&... x) {
  TORCH_CHECK(!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !(x._fw_grad(0).defined() || ...), name,
              " has no forward-mode derivative on CUDA");
}

// Losses of the readout. A scalar loss computes its gradients in the forward pass, where the unnormalised probabilities
// are at hand, saves them (and nothing else), and its backward pass scales them by the upstream gradient; per-row losses,
// whose upstream gradients are not known by then, save the operands and run the products in the backward pass.
struct ReadoutFunction : torch::autograd::Function<ReadoutFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight, const Tensor& targets,
                        int64_t ignore_index, double logit_scale, int64_t reduction, int64_t chunk_rows) {
    const bool per_row = reduction == ecz::kReduceNone;
    auto r = readout(hidden, weight, targets, ignore_index, logit_scale, reduction, !per_row && hidden.requires_grad(),
                     !per_row && weight.requires_grad(), c10::nullopt, chunk_rows);
    ctx->saved_data["reduction"] = reduction;
    if (per_row) {
      ctx->save_for_backward({hidden, weight, targets});
      ctx->saved_data["ignore"] = ignore_index;
      ctx->saved_data["scale"] = logit_scale;
      ctx->saved_data["chunk"] = chunk_rows;
    } else {
      ctx->save_for_backward({std::get<1>(r).value_or(Tensor()), std::get<2>(r).value_or(Tensor())});
    }
    return std::get<0>(r);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("linear_cross_entropy");
    auto& data = ctx->saved_data;
    const bool need_dx = ctx->needs_input_grad(0), need_dw = ctx->needs_input_grad(1);
    const int64_t reduction = data["reduction"].toInt();
    const auto saved = ctx->get_saved_variables();
    variable_list out(7);
    Tensor g = grads[0].to(at::kFloat).contiguous();
    if (reduction == ecz::kReduceNone) {
      auto r = readout(saved[0], saved[1], saved[2], data["ignore"].toInt(), data["scale"].toDouble(), reduction,
                       need_dx, need_dw, c10::optional<Tensor>(g), data["chunk"].toInt());
      if (need_dx) out[0] = *std::get<1>(r);
      if (need_dw) out[1] = *std::get<2>(r);
      return out;
    }
    // scaled in place and given away; a graph that is kept for another pass keeps its own
    const bool keep = torch::autograd::get_current_graph_task_keep_graph();
    for (int i = 0; i < 2; ++i) {
      if (!(i == 0 ? need_dx : need_dw)) continue;
      check_saved(saved[i], g, at::kBFloat16, saved[i].sizes(), "gradient");
      out[i] = keep ? saved[i].clone() : saved[i];
    }
    scale_both(out[0], out[1], g);
    return out;
  }
};

Tensor linear_cross_entropy(const Tensor& hidden, const Tensor& weight, const Tensor& targets, int64_t ignore_index,
                            double logit_scale, int64_t reduction, int64_t chunk_rows) {
  no_tangent("linear_cross_entropy", hidden, weight);
  if (at::GradMode::is_enabled() && (hidden.requires_grad() || weight.requires_grad()))
    return ReadoutFunction::apply(hidden, weight, targets, ignore_index, logit_scale, reduction, chunk_rows);
  return std::get<0>(
      readout(hidden, weight, targets, ignore_index, logit_scale, reduction, false, false, c10::nullopt, chunk_rows));
}

struct PackedFunction : torch::autograd::Function<PackedFunction> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu,
                        double scale, int64_t tiles) {
    const int64_t B = cu.dim() == 1 ? cu.size(0) - 1 : 0;
    if (tiles == 0 && q.dim() == 3)
      tiles = ecz::packed_single_tiles(static_cast<int>(q.size(0)), static_cast<int>(B), static_cast<int>(q.size(2)))
                  ? 1 : 2;
    auto r = packed_forward(q, k, v, cu, scale, true, tiles);
    // all of it as saved variables: saved_data would keep the output's rest until the graph itself goes, past the
    // backward pass and unseen by saved-tensor hooks
    ctx->save_for_backward({q, k, v, std::get<0>(r), std::get<1>(r), std::get<2>(r), std::get<3>(r)});
    ctx->saved_data["B"] = B;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["tiles"] = tiles;
    return std::get<0>(r);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("packed_attention");
    const auto s = ctx->get_saved_variables();
    auto& data = ctx->saved_data;
    const bool need_dq = ctx->needs_input_grad(0);
    const bool need_dk = ctx->needs_input_grad(1), need_dv = ctx->needs_input_grad(2);
    auto r = packed_backward(grads[0], s[0], s[1], s[2], s[3], s[4], s[5], s[6], data["B"].toInt(),
                             data["scale"].toDouble(), data["tiles"].toInt(), need_dq, need_dk || need_dv);
    variable_list out(6);
    if (need_dq) out[0] = std::get<0>(r);
    if (need_dk) out[1] = std::get<1>(r);
    if (need_dv) out[2] = std::get<2>(r);
    return out;
  }
};

Tensor packed_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu, double scale,
                        int64_t tiles) {
  no_tangent("packed_attention", q, k, v);
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad()))
    return PackedFunction::apply(q, k, v, cu, scale, tiles);
  return std::get<0>(packed_forward(q, k, v, cu, scale, false, tiles));
}

}  // namespace

namespace ecz {

void bind_training(pybind11::module_& m) {
  namespace py = pybind11;
  m.def("linear_cross_entropy", &linear_cross_entropy,
        "softmax cross-entropy of hidden @ weight.T without keeping the logits (autograd)", py::arg("hidden"),
        py::arg("weight"), py::arg("targets"), py::arg("ignore_index"), py::arg("logit_scale"), py::arg("reduction"),
        py::arg("chunk_rows") = 0);
  m.def("packed_attention", &packed_attention, "causal attention over packed sequences (tcgen05, autograd)",
        py::arg("q"), py::arg("k"), py::arg("v"), py::arg("cu_seqlens"), py::arg("scale"),
        py::arg("tiles") = 0);
}

}  // namespace ecz
