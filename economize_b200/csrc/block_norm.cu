// What stands between two blocks of a decoder: the norm after a block, its gate and residual scale, the residual sum and
// the norm before the next block, in one pass over the data, and its gradients.
//
//   b = x rsqrt(mean x^2 + eps) post       (or x)
//   s = residual + scale gate b            (stream; the residual and the gate may be missing)
//   n = s rsqrt(mean s^2 + eps) weight     (normed; as bf16 / fp16 / fp32, or from bf16 on to 4 bits, fp4_common.cuh)
//
// Everything is held in fp32; n and s are rounded once each, n is taken from the unrounded s. Bound by HBM: forward two
// rows read and two written per token, backward up to four read and two written. A team of warps keeps a row in
// registers; rows are read in 16-byte vectors where bases and strides allow it, else element by element.
//
// Backward, with g = dn weight, sh = s is (is = rsqrt(mean s^2 + eps), xh = x ix likewise):
//   ds = dstream + is (g - sh mean(g sh)),  dweight = sum_t dn sh,  dresidual = ds
//   dgate = scale b . ds (summed over the columns where the gate has one value a token),  db = scale gate ds
//   dx = ix (h - xh mean(h xh)) with h = db post,  dpost = sum_t db xh      (dx = db without a norm behind the block)
// The forward pass saves is and ix. Sums over tokens: every team adds up its rows in registers, in order, and a second
// kernel adds up the teams in order, so results do not depend on timing.
#include <algorithm>
#include <type_traits>

#include "fp4_common.cuh"
#include "launchers.h"

namespace ecz {

namespace {

constexpr int kMaxWarps = 32;

template <typename T>
struct Cast;
template <>
struct Cast<float> {
  static __device__ __forceinline__ float to(float v) { return v; }
  static __device__ __forceinline__ float from(float v) { return v; }
};
template <>
struct Cast<bf16> {
  static __device__ __forceinline__ float to(bf16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ bf16 from(float v) { return __float2bfloat16(v); }
};
template <>
struct Cast<__half> {
  static __device__ __forceinline__ float to(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half from(float v) { return __float2half(v); }
};

// VEC consecutive elements (VEC sizeof(T) = 16 bytes, aligned, or VEC = 1).
template <typename T, int VEC>
struct Pack {
  T v[VEC];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (VEC == 1) v[0] = *p;
    else *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(p);
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (VEC == 1) *p = v[0];
    else *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(v);
  }
  __device__ __forceinline__ float get(int i) const { return Cast<T>::to(v[i]); }
  __device__ __forceinline__ void set(int i, float f) { v[i] = Cast<T>::from(f); }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = Cast<T>::from(0.f);
  }
};

// A team's place: `warps` consecutive warps of the block, and its reductions. Two buffers in turn: a warp writes one again
// only behind a barrier that all warps reach after reading it.
struct Team {
  int warps, index, first, step, lane, warp;
  float2* scratch;  // [2][kMaxWarps]
  int turn = 0;
  __device__ __forceinline__ Team(int warps_, float2* buf) : warps(warps_), scratch(buf) {
    const int w = threadIdx.x >> 5;
    lane = threadIdx.x & 31;
    index = w / warps;
    warp = w - index * warps;
    first = warp * 32 + lane;
    step = warps * 32;
  }
  __device__ __forceinline__ void barrier() const {
    asm volatile("bar.sync %0, %1;" ::"r"(index + 1), "r"(warps * 32) : "memory");
  }
  __device__ __forceinline__ float2 sum(float2 v) {
    v.x = warp_sum(v.x);
    v.y = warp_sum(v.y);
    if (warps == 1) return v;
    float2* buf = scratch + turn * kMaxWarps + index * warps;
    turn ^= 1;
    if (lane == 0) buf[warp] = v;
    barrier();
    float2 out = make_float2(0.f, 0.f);
    for (int w = 0; w < warps; ++w) {
      out.x += buf[w].x;
      out.y += buf[w].y;
    }
    return out;
  }
  __device__ __forceinline__ float sum(float v) {
    v = warp_sum(v);
    if (warps == 1) return v;
    float2* buf = scratch + turn * kMaxWarps + index * warps;
    turn ^= 1;
    if (lane == 0) buf[warp].x = v;
    barrier();
    float out = 0.f;
    for (int w = 0; w < warps; ++w) out += buf[w].x;
    return out;
  }
  __device__ __forceinline__ float max(float v) {
    v = warp_max(v);
    if (warps == 1) return v;
    float2* buf = scratch + turn * kMaxWarps + index * warps;
    turn ^= 1;
    if (lane == 0) buf[warp].x = v;
    barrier();
    float out = buf[0].x;
    for (int w = 1; w < warps; ++w) out = fmaxf(out, buf[w].x);
    return out;
  }
};

// FMT 0: normed as T; else as 4-bit codes (VEC = 8 elements of bf16).
template <typename T, int VEC, int NV, int FMT>
__global__ void __launch_bounds__(1024) block_norm_kernel(const __grid_constant__ BlockNormArgs a, int warps) {
  __shared__ float2 scratch[2 * kMaxWarps];
  pdl_trigger();
  Team team(warps, scratch);
  pdl_wait();
  const int teams = blockDim.x / (32 * warps);
  const T* weight = static_cast<const T*>(a.weight);
  const T* post = static_cast<const T*>(a.post);
  const int vecs = (a.hidden + VEC - 1) / VEC;
  const float mean = 1.f / static_cast<float>(a.hidden);
  const int row = blockIdx.x * teams + team.index;
  if (FMT == 0 && row >= a.rows) return;
  if (FMT != 0 && row >= (a.rows + 127) / 128 * 128) return;
  const bool real = row < a.rows;
  Pack<T, VEC> x[NV], r[NV];
  float s[NV][VEC];
  const T* xr = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* rr = static_cast<const T*>(a.residual) + row * a.r_stride;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = team.first + i * team.step;
    x[i].zero();
    r[i].zero();
    if (real && v < vecs) {
      x[i].load(xr + static_cast<size_t>(v) * VEC);
      if (a.residual != nullptr) r[i].load(rr + static_cast<size_t>(v) * VEC);
    }
  }
  float factor = a.scale;
  if (a.gate_mode == kGateToken && real) factor *= Cast<T>::to(static_cast<const T*>(a.gate)[row * a.gate_stride]);
  float ix = 1.f;
  if (post != nullptr) {
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) q = fmaf(x[i].get(j), x[i].get(j), q);
    ix = rsqrtf(team.sum(q) * mean + a.eps);
    if (a.inv_x != nullptr && team.first == 0 && real) a.inv_x[row] = ix;
  }
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = team.first + i * team.step;
    Pack<T, VEC> p, g;
    if (post != nullptr && v < vecs) p.load(post + static_cast<size_t>(v) * VEC);
    if (a.gate_mode == kGateFull && real && v < vecs)
      g.load(static_cast<const T*>(a.gate) + row * a.gate_stride + static_cast<size_t>(v) * VEC);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      float b = x[i].get(j);
      if (post != nullptr && v < vecs) b = b * ix * p.get(j);
      if (a.gate_mode == kGateFull && real && v < vecs) b *= g.get(j);
      s[i][j] = fmaf(factor, b, r[i].get(j));
      q = fmaf(s[i][j], s[i][j], q);
    }
    if (real && v < vecs) {
      Pack<T, VEC> out;
#pragma unroll
      for (int j = 0; j < VEC; ++j) out.set(j, s[i][j]);
      out.store(static_cast<T*>(a.stream) + static_cast<size_t>(row) * a.hidden + static_cast<size_t>(v) * VEC);
    }
  }
  const float is = rsqrtf(team.sum(q) * mean + a.eps);
  if (a.inv_s != nullptr && team.first == 0 && real) a.inv_s[row] = is;
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = team.first + i * team.step;
    if (FMT != 0 || v < vecs) {
      Pack<T, VEC> w, out;
      w.zero();
      if (v < vecs) w.load(weight + static_cast<size_t>(v) * VEC);
#pragma unroll
      for (int j = 0; j < VEC; ++j) out.set(j, real ? s[i][j] * is * w.get(j) : 0.f);
      if constexpr (FMT == 0) {
        out.store(static_cast<T*>(a.normed) + static_cast<size_t>(row) * a.hidden + static_cast<size_t>(v) * VEC);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) s[i][j] = out.get(j);  // what quantising the rounded result takes
        bool bad;
        if (FMT == fp4::kNv) top = fmaxf(top, fp4::finite_max8(s[i], bad));
      }
    }
  }
  if constexpr (FMT != 0) {
    float mul = 1.f;
    if constexpr (FMT == fp4::kNv) {
      const int e = fp4::row_exponent(team.max(top));
      mul = fp4::pow2(-e);
      if (real && team.first == 0) a.row_scale[row] = fp4::pow2(e);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int base = (team.warp + i * warps) * 32;
      if (base >= a.tiles * fp4::Format<FMT>::kWordLanes) break;
      fp4::store8<FMT>(s[i], mul, row, base + team.lane, real ? vecs : 0, a.tiles, a.codes, a.scales);
    }
  }
}

// Persistent over rows: team t of all takes rows t, t + teams, ...; its sums for dweight and dpost go to row t of
// a.dw_part / a.dpost_part (fp32 [teams, hidden]).
template <typename T, int VEC, int NV, bool POST>
__global__ void __launch_bounds__(NV * VEC > 16 ? 512 : 1024)
    block_norm_bwd_kernel(const __grid_constant__ BlockNormGrads a, int warps) {
  __shared__ float2 scratch[2 * kMaxWarps];
  pdl_trigger();
  Team team(warps, scratch);
  pdl_wait();
  const int per_block = blockDim.x / (32 * warps);
  const int teams = gridDim.x * per_block, self = blockIdx.x * per_block + team.index;
  const int vecs = (a.hidden + VEC - 1) / VEC;
  const float mean = 1.f / static_cast<float>(a.hidden);
  const T* weight = static_cast<const T*>(a.weight);
  const T* post = static_cast<const T*>(a.post);
  float dw[NV][VEC], dp[NV][POST ? VEC : 1];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      dw[i][j] = 0.f;
      if (POST) dp[i][j] = 0.f;
    }
  for (int row = self; row < a.rows; row += teams) {
    const float is = a.inv_s[row], ix = POST ? a.inv_x[row] : 1.f;
    float gate = a.scale;  // scale times the token's gate
    if (a.gate_mode == kGateToken) gate *= Cast<T>::to(static_cast<const T*>(a.gate)[row * a.gate_stride]);
    // sh: the normalised stream; ds: the upstream gradient of the stream
    float sh[NV][VEC], g[NV][VEC], ds[NV][VEC];
    Pack<T, VEC> x[NV];
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = team.first + i * team.step;
      const size_t at = static_cast<size_t>(v) * VEC;
      Pack<T, VEC> dn, up, r, w, p, fg;
      x[i].zero();
      dn.zero();
      up.zero();
      r.zero();
      w.zero();
      if (v < vecs) {
        if (a.dnormed != nullptr) dn.load(static_cast<const T*>(a.dnormed) + row * a.dn_stride + at);
        if (a.dstream != nullptr) up.load(static_cast<const T*>(a.dstream) + row * a.ds_stride + at);
        if (a.stream != nullptr) r.load(static_cast<const T*>(a.stream) + static_cast<size_t>(row) * a.hidden + at);
        else if (a.residual != nullptr) r.load(static_cast<const T*>(a.residual) + row * a.r_stride + at);
        if (a.stream == nullptr) x[i].load(static_cast<const T*>(a.x) + row * a.x_stride + at);
        w.load(weight + at);
      }
      if (POST && v < vecs) p.load(post + at);
      if (a.gate_mode == kGateFull && v < vecs) fg.load(static_cast<const T*>(a.gate) + row * a.gate_stride + at);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        float s = r.get(j);
        if (a.stream == nullptr) {
          float b = x[i].get(j);
          if (POST) b *= ix * (v < vecs ? p.get(j) : 0.f);
          if (a.gate_mode == kGateFull) b *= v < vecs ? fg.get(j) : 0.f;
          s = fmaf(gate, b, s);
        }
        sh[i][j] = s * is;
        dw[i][j] = fmaf(dn.get(j), sh[i][j], dw[i][j]);
        g[i][j] = dn.get(j) * w.get(j);
        dot = fmaf(g[i][j], sh[i][j], dot);
        ds[i][j] = up.get(j);
      }
    }
    dot = team.sum(dot) * mean;
    float2 sums = make_float2(0.f, 0.f);  // h . xh and the token gate's gradient
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = team.first + i * team.step;
      const size_t at = static_cast<size_t>(v) * VEC;
      Pack<T, VEC> p, fg, out, dg;
      if (POST && v < vecs) p.load(post + at);
      if (a.gate_mode == kGateFull && v < vecs) fg.load(static_cast<const T*>(a.gate) + row * a.gate_stride + at);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        ds[i][j] += is * (g[i][j] - sh[i][j] * dot);
        out.set(j, ds[i][j]);
        const float xh = x[i].get(j) * ix;
        const float pw = POST ? (v < vecs ? p.get(j) : 0.f) : 1.f;
        const float b = xh * pw;  // without POST ix is 1
        float db = gate * ds[i][j];
        if (a.gate_mode == kGateFull) {
          dg.set(j, db * b);
          db *= v < vecs ? fg.get(j) : 0.f;
        } else if (a.gate_mode == kGateToken) {
          sums.y = fmaf(b, ds[i][j], sums.y);
        }
        if (POST) {
          dp[i][j] = fmaf(db, xh, dp[i][j]);
          g[i][j] = db * pw;  // h
          sums.x = fmaf(g[i][j], xh, sums.x);
        } else {
          g[i][j] = db;
        }
      }
      if (v < vecs) {
        if (a.dresidual != nullptr)
          out.store(static_cast<T*>(a.dresidual) + static_cast<size_t>(row) * a.hidden + at);
        if (a.gate_mode == kGateFull && a.dgate != nullptr)
          dg.store(static_cast<T*>(a.dgate) + static_cast<size_t>(row) * a.hidden + at);
      }
    }
    if (POST || a.gate_mode == kGateToken) {
      sums = team.sum(sums);
      if (a.gate_mode == kGateToken && a.dgate != nullptr && team.first == 0)
        static_cast<T*>(a.dgate)[row] = Cast<T>::from(a.scale * sums.y);
    }
    if (a.dx != nullptr) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = team.first + i * team.step;
        if (v < vecs) {
          Pack<T, VEC> out;
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            out.set(j, POST ? ix * (g[i][j] - x[i].get(j) * ix * (sums.x * mean)) : g[i][j]);
          out.store(static_cast<T*>(a.dx) + static_cast<size_t>(row) * a.hidden + static_cast<size_t>(v) * VEC);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = team.first + i * team.step;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int c = v * VEC + j;
      if (v < vecs && c < a.hidden) {
        if (a.dw_part != nullptr) a.dw_part[static_cast<size_t>(self) * a.hidden + c] = dw[i][j];
        if (POST && a.dpost_part != nullptr) a.dpost_part[static_cast<size_t>(self) * a.hidden + c] = dp[i][j];
      }
    }
  }
}

// Columns of `parts` rows of fp32 added up in order: eight threads per column take every eighth row each.
template <typename T>
__global__ void __launch_bounds__(256) block_norm_sum_kernel(const float* __restrict__ dw_part,
                                                             const float* __restrict__ dpost_part, T* dw, T* dpost,
                                                             int parts, int hidden) {
  __shared__ float sums[8][32];
  pdl_trigger();
  pdl_wait();
  const float* part = blockIdx.y == 0 ? dw_part : dpost_part;
  T* out = blockIdx.y == 0 ? dw : dpost;
  if (out == nullptr) return;
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), lane = threadIdx.x >> 5;
  float s = 0.f;
  if (c < hidden)
    for (int p = lane; p < parts; p += 8) s += part[static_cast<size_t>(p) * hidden + c];
  sums[lane][threadIdx.x & 31] = s;
  __syncthreads();
  if (threadIdx.x < 32 && c < hidden) {
#pragma unroll
    for (int i = 1; i < 8; ++i) s += sums[i][threadIdx.x];
    out[c] = Cast<T>::from(s);
  }
}

struct Grid {
  int warps, nv, teams;  // warps of a team, vectors a lane, teams of a block
};

// Teams that hold a row of `vecs` vectors with about `target` vectors a lane.
Grid teams_of(int vecs, int target, int block_warps) {
  const int all = (vecs + 31) / 32;
  Grid g;
  g.warps = std::min(kMaxWarps, std::max(1, (all + target - 1) / target));
  if (g.warps <= block_warps) {
    int p = 1;
    while (p < g.warps) p *= 2;
    g.warps = p;
  }
  g.nv = (all + g.warps - 1) / g.warps;
  g.teams = g.warps < block_warps ? block_warps / g.warps : 1;
  return g;
}

template <typename T, int VEC, int FMT>
int run_forward(const BlockNormArgs& a, int sms, cudaStream_t stream) {
  const int vecs = FMT == 0 ? (a.hidden + VEC - 1) / VEC : a.tiles * fp4::Format<FMT == 0 ? fp4::kNv : FMT>::kWordLanes;
  const bool many = a.rows >= 4 * sms;
  const Grid g = teams_of(vecs, many ? 4 : 1, many ? 8 : 1);
  const int rows = FMT == 0 ? a.rows : (a.rows + 127) / 128 * 128;
  const dim3 grid((rows + g.teams - 1) / g.teams), block(32 * g.warps * g.teams);
  auto go = [&](auto kernel) { return launch_pdl(kernel, grid, block, 0, stream, a, g.warps) == cudaSuccess ? 0 : -1; };
  if (g.nv <= 1) return go(block_norm_kernel<T, VEC, 1, FMT>);
  if (g.nv <= 2) return go(block_norm_kernel<T, VEC, 2, FMT>);
  if (g.nv <= 4) return go(block_norm_kernel<T, VEC, 4, FMT>);
  if constexpr (VEC == 1) {
    if (g.nv <= 8) return go(block_norm_kernel<T, VEC, 8, FMT>);
    if (g.nv <= 16) return go(block_norm_kernel<T, VEC, 16, FMT>);
  }
  return -1;
}

template <typename T>
int run_forward_type(const BlockNormArgs& a, bool vec, int sms, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  return vec ? run_forward<T, V, 0>(a, sms, stream) : run_forward<T, 1, 0>(a, sms, stream);
}

constexpr int kBwdBlockWarps = 8;

template <typename T, int VEC>
Grid backward_grid(int hidden) {
  return teams_of((hidden + VEC - 1) / VEC, VEC == 8 ? 2 : 4, kBwdBlockWarps);
}

int backward_blocks(const Grid& g, int rows, int sms) {
  const int resident = std::max(1, 16 / (g.warps * g.teams));
  return std::min((rows + g.teams - 1) / g.teams, sms * resident);
}

template <typename T, int VEC>
int run_backward(const BlockNormGrads& a, int sms, cudaStream_t stream) {
  const Grid g = backward_grid<T, VEC>(a.hidden);
  const dim3 grid(backward_blocks(g, a.rows, sms)), block(32 * g.warps * g.teams);
  auto go = [&](auto kernel) { return launch_pdl(kernel, grid, block, 0, stream, a, g.warps) == cudaSuccess ? 0 : -1; };
  int rc = -1;
  auto pick = [&](auto post) {
    constexpr bool P = decltype(post)::value;
    if (g.nv <= 1) return go(block_norm_bwd_kernel<T, VEC, 1, P>);
    if (g.nv <= 2) return go(block_norm_bwd_kernel<T, VEC, 2, P>);
    if constexpr (VEC <= 4) {
      if (g.nv <= 4) return go(block_norm_bwd_kernel<T, VEC, 4, P>);
    }
    if constexpr (VEC == 1) {
      if (g.nv <= 8) return go(block_norm_bwd_kernel<T, VEC, 8, P>);
      if (g.nv <= 16) return go(block_norm_bwd_kernel<T, VEC, 16, P>);
    }
    return -1;
  };
  rc = a.post != nullptr ? pick(std::true_type{}) : pick(std::false_type{});
  if (rc != 0 || (a.dweight == nullptr && a.dpost == nullptr)) return rc;
  return launch_pdl(block_norm_sum_kernel<T>, dim3((a.hidden + 31) / 32, a.dpost != nullptr ? 2 : 1), dim3(256), 0, stream,
                    static_cast<const float*>(a.dw_part), static_cast<const float*>(a.dpost_part),
                    static_cast<T*>(a.dweight), static_cast<T*>(a.dpost), static_cast<int>(grid.x) * g.teams,
                    a.hidden) == cudaSuccess ? 0 : -1;
}

template <typename T>
int run_backward_type(const BlockNormGrads& a, bool vec, int sms, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  return vec ? run_backward<T, V>(a, sms, stream) : run_backward<T, 1>(a, sms, stream);
}

template <typename T>
int parts_type(int rows, int hidden, bool vec, int sms) {
  constexpr int V = 16 / sizeof(T);
  const Grid g = vec ? backward_grid<T, V>(hidden) : backward_grid<T, 1>(hidden);
  return backward_blocks(g, rows, sms) * g.teams;
}

}  // namespace

int launch_block_norm(const BlockNormArgs& a, NormType type, bool vec, int fmt, int sms, cudaStream_t stream) {
  if (a.rows < 1 || a.hidden < 1 || a.hidden > kBlockNormMaxHidden) return -1;
  if (fmt != 0) {
    if (type != kNormBf16 || !vec || a.hidden % 32 != 0) return -1;
    return fmt == fp4::kNv ? run_forward<bf16, 8, fp4::kNv>(a, sms, stream) : run_forward<bf16, 8, fp4::kMx>(a, sms, stream);
  }
  switch (type) {
    case kNormBf16: return run_forward_type<bf16>(a, vec, sms, stream);
    case kNormFp16: return run_forward_type<__half>(a, vec, sms, stream);
    default: return run_forward_type<float>(a, vec, sms, stream);
  }
}

int block_norm_parts(NormType type, int rows, int hidden, bool vec, int sms) {
  switch (type) {
    case kNormBf16: return parts_type<bf16>(rows, hidden, vec, sms);
    case kNormFp16: return parts_type<__half>(rows, hidden, vec, sms);
    default: return parts_type<float>(rows, hidden, vec, sms);
  }
}

int launch_block_norm_grads(const BlockNormGrads& a, NormType type, bool vec, int sms, cudaStream_t stream) {
  if (a.rows < 1 || a.hidden < 1 || a.hidden > kBlockNormMaxHidden) return -1;
  switch (type) {
    case kNormBf16: return run_backward_type<bf16>(a, vec, sms, stream);
    case kNormFp16: return run_backward_type<__half>(a, vec, sms, stream);
    default: return run_backward_type<float>(a, vec, sms, stream);
  }
}

}  // namespace ecz
