// Softmax cross-entropy of a vocabulary readout without keeping the logits, with its gradient.
//
//   z_tv = s x_t . w_v     L_t = log sum_v exp z_tv     nll_t = L_t - z_{t, y_t}
//   dz_tv = g_t (exp(z_tv - L_t) - [v = y_t])     dx_t = s sum_v dz_tv w_v     dW_v = s sum_t dz_tv x_t
//
// Rows whose target is the ignored index are left out before the first product: the plan kernel lists the other rows
// in order and the gather kernel packs their states, so a prompt mask saves its share of all three products and
// nothing that stands in a masked row (not even NaN) reaches a result. Packed rows are processed in chunks:
//
//   logits    256 x 256 tiles of X . W^T (gemm_pair.cuh); the epilogue reduces each row's 128-column piece to its
//             maximum m and sum of exp(z - m), picks the target's logit and, when gradients follow, stores
//             e = exp(z - m) in fp16. e lies in (0, 1] with its piece's largest at 1, so fp16 keeps 11 bits of
//             everything that counts (bf16 would add a second 8-bit rounding to the gradients); the logits
//             themselves are never stored.
//   finish    joins a row's pieces to L_t and nll_t and rewrites e in place as dz = g s (e exp(m - L)) in bf16, the
//             one rounding of the gradient's left factor. The target's entry is g s expm1(-nll), which keeps its
//             digits where the probability is near one.
//   products  dX = dz . W (K = V, W read MN-major) and dW = dz^T . X (K = rows, both operands MN-major), no
//             transposes. Over several chunks dW is summed in an fp32 buffer in chunk order.
//
// Without gradients only the statistics of the pieces are written (8 bytes per 128 logits).
#include <algorithm>

#include "gemm_pair.cuh"
#include "launchers.h"

namespace ecz {

namespace {

constexpr int kPiece = 128;  // columns a row statistic covers
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ---- plan ------------------------------------------------------------------------------------------------------
// One CTA: rows[i] = the i-th row with a target, pos[t] = its place or -1, target_of[i] = its target, *count = how
// many. A target outside [0, V) that is not the ignored index counts as ignored and sets kStatusBadIndex.
__global__ void __launch_bounds__(1024) readout_plan_kernel(const int64_t* __restrict__ targets, int T, int V,
                                                            int64_t ignore, int* __restrict__ rows,
                                                            int* __restrict__ pos, int* __restrict__ target_of,
                                                            int* __restrict__ count, unsigned* status) {
  __shared__ int warp_count[32];
  __shared__ int base;
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) base = 0;
  __syncthreads();
  for (int t0 = 0; t0 < T; t0 += 1024) {
    const int t = t0 + threadIdx.x;
    int64_t y = t < T ? targets[t] : ignore;
    bool keep = t < T && y != ignore;
    if (keep && (y < 0 || y >= V)) {
      atomicOr(status, kStatusBadIndex);
      keep = false;
    }
    const unsigned ballot = __ballot_sync(0xffffffffu, keep);
    if (lane == 0) warp_count[warp] = __popc(ballot);
    __syncthreads();
    int before = base;
    int total = 0;
#pragma unroll
    for (int w = 0; w < 32; ++w) {
      const int c = warp_count[w];
      if (w < warp) before += c;
      total += c;
    }
    const int at = before + __popc(ballot & ((1u << lane) - 1u));
    if (keep) {
      rows[at] = t;
      target_of[at] = static_cast<int>(y);
    }
    if (t < T) pos[t] = keep ? at : -1;
    __syncthreads();
    if (threadIdx.x == 0) base += total;
    __syncthreads();
  }
  if (threadIdx.x == 0) *count = base;
}

// ---- gather ----------------------------------------------------------------------------------------------------
// Warp per row t: its state to xs[pos[t]], or zeros to dx[t] (and losses[t]) where it is ignored. The rows behind
// the last packed one are zeroed up to the K block that reads them.
__global__ void __launch_bounds__(256) readout_gather_kernel(const bf16* __restrict__ x, long x_stride, int T, int H,
                                                             const int* __restrict__ pos,
                                                             const int* __restrict__ count, bf16* __restrict__ xs,
                                                             bf16* __restrict__ dx, float* __restrict__ losses) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int t = blockIdx.x * 8 + (threadIdx.x >> 5);
  const uint4 zero = make_uint4(0, 0, 0, 0);
  if (t >= T) {
    const int n = *count;
    const int r = n + (t - T);
    if (t - T < pair::kBK && r < (n + pair::kBK - 1) / pair::kBK * pair::kBK)
      for (int c = lane * 8; c < H; c += 256) *reinterpret_cast<uint4*>(xs + static_cast<size_t>(r) * H + c) = zero;
    return;
  }
  const int p = pos[t];
  if (p >= 0) {
    for (int c = lane * 8; c < H; c += 256)
      *reinterpret_cast<uint4*>(xs + static_cast<size_t>(p) * H + c) =
          *reinterpret_cast<const uint4*>(x + static_cast<size_t>(t) * x_stride + c);
  } else {
    if (dx != nullptr)
      for (int c = lane * 8; c < H; c += 256) *reinterpret_cast<uint4*>(dx + static_cast<size_t>(t) * H + c) = zero;
    if (losses != nullptr && lane == 0) losses[t] = 0.f;
  }
}

// ---- logits: statistics (and e) of a tile's rows -----------------------------------------------------------------
struct LogitsEpi {
  float2* stats;      // [rows of the chunk, pieces]: (max, sum of exp2(z - max)), log2 units
  float* picked;      // [rows]: the target's logit, log2 units
  const int* target;  // [rows] of the chunk
  __half* e;          // [rows, ld] or null
  long ld;
  int V, pieces;
  float scale2;  // logit scale times log2(e)

  __device__ __forceinline__ void operator()(const pair::Unit&, int M, int row0, int col0, uint32_t taddr, bool,
                                             uint8_t* patch, int lane) const {
    if (row0 >= M || col0 >= V) return;  // uniform over the warp
    const int row = row0 + lane;
    const int cols = min(kPiece, V - col0);
    const int mine = row < M ? target[row] - col0 : -1;
    float top = -INFINITY;
#pragma unroll 1
    for (int c = 0; c < kPiece; c += 32) {
      float v[32];
      tmem_ld32(taddr + c, v);
      if (c + 32 <= cols) {
#pragma unroll
        for (int j = 0; j < 32; ++j) top = fmaxf(top, v[j] * scale2);
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (c + j < cols) top = fmaxf(top, v[j] * scale2);
      }
    }
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
#pragma unroll 1
    for (int c = 0; c < kPiece; c += 32) {
      float v[32];
      tmem_ld32(taddr + c, v);
      if (mine >= c && mine < c + 32) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (c + j == mine) picked[row] = v[j] * scale2;
      }
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        v[j] = c + j < cols ? ex2(fmaf(v[j], scale2, -ref)) : 0.f;
        sum += v[j];
      }
      if (e != nullptr) {
#pragma unroll
        for (int j = 0; j < 32; j += 8) {
          uint4 w;
          __half2 h0 = __floats2half2_rn(v[j], v[j + 1]), h1 = __floats2half2_rn(v[j + 2], v[j + 3]);
          __half2 h2 = __floats2half2_rn(v[j + 4], v[j + 5]), h3 = __floats2half2_rn(v[j + 6], v[j + 7]);
          w.x = *reinterpret_cast<uint32_t*>(&h0);
          w.y = *reinterpret_cast<uint32_t*>(&h1);
          w.z = *reinterpret_cast<uint32_t*>(&h2);
          w.w = *reinterpret_cast<uint32_t*>(&h3);
          *reinterpret_cast<uint4*>(patch + lane * pair::kPatchStride + (c & 32) * 2 + j * 2) = w;
        }
        if (c & 32) {  // 64 columns staged: 8 lanes write a row's 128 bytes
          __syncwarp();
          const int col = col0 + (c & ~63) + (lane & 7) * 8;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = i * 4 + (lane >> 3);
            if (row0 + r < M && col < V)  // ld is a multiple of 8: a started group of 8 fits
              *reinterpret_cast<uint4*>(e + static_cast<size_t>(row0 + r) * ld + col) =
                  *reinterpret_cast<const uint4*>(patch + r * pair::kPatchStride + (lane & 7) * 16);
          }
          __syncwarp();
        }
      }
    }
    if (row < M) stats[static_cast<size_t>(row) * pieces + col0 / kPiece] = make_float2(top, sum);
  }
};

// ---- finish ------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float block_reduce(float v, float* red, bool want_max) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  v = want_max ? warp_max(v) : warp_sum(v);
  if (lane == 0) red[warp] = v;
  __syncthreads();
  float r = red[0];
  for (int w = 1; w < warps; ++w) r = want_max ? fmaxf(r, red[w]) : r + red[w];
  __syncthreads();
  return r;
}

// One CTA per packed row of the chunk: joins its pieces, writes nll, and (with e) turns e into dz in place. NaN
// statistics give NaN, as the plain formula does.
constexpr int kFinishThreads = 256;

__global__ void __launch_bounds__(kFinishThreads)
    readout_finish_kernel(const float2* __restrict__ stats, const float* __restrict__ picked,
                          const int* __restrict__ target, const int* __restrict__ rows,
                          const int* __restrict__ count, int row0, int chunk, int V, int pieces, void* e_dz, long ld,
                          float logit_scale, int reduction, const float* __restrict__ grad_rows,
                          float* __restrict__ nll, float* __restrict__ losses) {
  extern __shared__ float factor[];  // [pieces]: exp2(m - L) g s
  __shared__ float red[kFinishThreads / 32];
  pdl_trigger();
  pdl_wait();
  const int total = *count;
  const int n = min(chunk, total - row0);
  const int r = blockIdx.x;
  if (n <= 0) return;
  if (r >= n) {  // zero rows up to the K block of dz^T . X that reads them
    if (e_dz != nullptr && r < (n + pair::kBK - 1) / pair::kBK * pair::kBK) {
      uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(e_dz) + static_cast<size_t>(r) * ld);
      for (int c = threadIdx.x; c < ld / 8; c += kFinishThreads) dst[c] = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  const float2* st = stats + static_cast<size_t>(r) * pieces;
  float top = -INFINITY;
  bool nan = false;
  for (int j = threadIdx.x; j < pieces; j += kFinishThreads) {
    top = fmaxf(top, st[j].x);
    nan |= st[j].y != st[j].y;
  }
  top = block_reduce(top, red, true);
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  for (int j = threadIdx.x; j < pieces; j += kFinishThreads) {
    const float2 v = st[j];
    sum += v.y * exp2f(v.x - ref);
  }
  sum = block_reduce(sum, red, false);
  if (nan) sum = NAN;
  const float lse2 = ref + log2f(sum);
  const float loss = (lse2 - picked[r]) * kLn2;
  const int orig = rows[row0 + r];
  if (threadIdx.x == 0) {
    if (nll != nullptr) nll[row0 + r] = loss;
    if (losses != nullptr) losses[orig] = loss;
  }
  if (e_dz == nullptr) return;
  float g = logit_scale;
  if (grad_rows != nullptr) g *= grad_rows[orig];
  else if (reduction == kReduceMean) g /= static_cast<float>(total);
  for (int j = threadIdx.x; j < pieces; j += kFinishThreads) factor[j] = exp2f(st[j].x - lse2) * g;
  __syncthreads();
  const int tgt = target[r];
  const float at_target = g * expm1f(-loss);
  uint16_t* row = static_cast<uint16_t*>(e_dz) + static_cast<size_t>(r) * ld;
  for (int c = threadIdx.x * 8; c < V; c += kFinishThreads * 8) {
    uint4 v = *reinterpret_cast<const uint4*>(row + c);
    const float f = factor[c / kPiece];
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 ev = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
      float a = ev.x * f, b = ev.y * f;
      if (c + 2 * k == tgt) a = at_target;
      if (c + 2 * k + 1 == tgt) b = at_target;
      __nv_bfloat162 o = __floats2bfloat162_rn(a, b);
      w[k] = *reinterpret_cast<uint32_t*>(&o);
    }
    *reinterpret_cast<uint4*>(row + c) = v;
  }
}

// loss = sum of nll (in a fixed order: thread t sums rows t, t + 1024, ..., then a tree) / count, 0 without rows.
__global__ void __launch_bounds__(1024) readout_loss_kernel(const float* __restrict__ nll,
                                                            const int* __restrict__ count, int reduction,
                                                            float* __restrict__ loss) {
  __shared__ float red[32];
  pdl_trigger();
  pdl_wait();
  const int n = *count;
  float v = 0.f;
  for (int i = threadIdx.x; i < n; i += 1024) v += nll[i];
  v = block_reduce(v, red, false);
  if (threadIdx.x == 0) *loss = reduction == kReduceMean ? (n > 0 ? v / static_cast<float>(n) : 0.f) : v;
}

// ---- product epilogues ---------------------------------------------------------------------------------------------
// Stores a warp's 32 x 128 accumulators: bf16 rows (through the patch, 128-byte row segments), fp32 partials of a K
// split, or an fp32 running sum over the chunks whose last chunk stores bf16.
struct StoreEpi {
  bf16* out;        // [.., N] or null
  float* part;      // [splits, M, N] fp32 partials, or the running sum [M, N] (splits == 1), or null
  const int* rows;  // destination row of row m (null: m)
  int N;
  long part_rows;   // rows of a split's partials
  bool add, last;   // running sum: add to what is there; store the sum as bf16

  __device__ __forceinline__ void operator()(const pair::Unit& u, int M, int row0, int col0, uint32_t taddr, bool zero,
                                             uint8_t* patch, int lane) const {
    if (row0 >= M || col0 >= N) return;
    const int cols = min(128, N - col0);
    float* prow = part == nullptr
                      ? nullptr
                      : part + (static_cast<size_t>(u.split) * part_rows + row0 + lane) * static_cast<size_t>(N) + col0;
    const bool row_ok = row0 + lane < M;
#pragma unroll 1
    for (int c = 0; c < cols; c += 32) {
      float v[32];
      if (zero) {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = 0.f;
      } else {
        tmem_ld32(taddr + c, v);
      }
      if (prow != nullptr && row_ok) {
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          if (c + j >= cols) break;  // N is a multiple of 8
          float4* p = reinterpret_cast<float4*>(prow + c + j);
          if (add) {
            const float4 o = *p;
            v[j] += o.x;
            v[j + 1] += o.y;
            v[j + 2] += o.z;
            v[j + 3] += o.w;
          }
          if (!last) *p = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
        }
      }
      if (!last) continue;
#pragma unroll
      for (int j = 0; j < 32; j += 8) {
        uint4 w;
        __nv_bfloat162 h0 = __floats2bfloat162_rn(v[j], v[j + 1]), h1 = __floats2bfloat162_rn(v[j + 2], v[j + 3]);
        __nv_bfloat162 h2 = __floats2bfloat162_rn(v[j + 4], v[j + 5]), h3 = __floats2bfloat162_rn(v[j + 6], v[j + 7]);
        w.x = *reinterpret_cast<uint32_t*>(&h0);
        w.y = *reinterpret_cast<uint32_t*>(&h1);
        w.z = *reinterpret_cast<uint32_t*>(&h2);
        w.w = *reinterpret_cast<uint32_t*>(&h3);
        *reinterpret_cast<uint4*>(patch + lane * pair::kPatchStride + (c & 32) * 2 + j * 2) = w;
      }
      if ((c & 32) || c + 32 >= cols) {
        __syncwarp();
        const int off = (c & ~63) + (lane & 7) * 8;
        const bool staged = off < cols && off < c + 32;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = i * 4 + (lane >> 3);
          if (staged && row0 + r < M) {
            const long dst = rows != nullptr ? rows[row0 + r] : row0 + r;
            *reinterpret_cast<uint4*>(out + dst * N + col0 + off) =
                *reinterpret_cast<const uint4*>(patch + r * pair::kPatchStride + (lane & 7) * 16);
          }
        }
        __syncwarp();
      }
    }
  }
};

// out[rows[m]] = bf16(sum over splits, in order, of part[s, m]).
__global__ void __launch_bounds__(256) readout_join_kernel(const float* __restrict__ part, int splits, long part_rows,
                                                           int N, const int* __restrict__ rows,
                                                           const int* __restrict__ count, int row0, int chunk,
                                                           bf16* __restrict__ out) {
  pdl_trigger();
  pdl_wait();
  const int n = min(chunk, *count - row0);
  const long i = (static_cast<long>(blockIdx.x) * 256 + threadIdx.x) * 4;
  const long m = i / N, c = i % N;
  if (m >= n) return;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = 0; s < splits; ++s) {
    const float4 v = *reinterpret_cast<const float4*>(part + (s * part_rows + m) * N + c);
    acc.x += v.x;
    acc.y += v.y;
    acc.z += v.z;
    acc.w += v.w;
  }
  __nv_bfloat162 lo = __floats2bfloat162_rn(acc.x, acc.y), hi = __floats2bfloat162_rn(acc.z, acc.w);
  uint2 w;
  w.x = *reinterpret_cast<uint32_t*>(&lo);
  w.y = *reinterpret_cast<uint32_t*>(&hi);
  *reinterpret_cast<uint2*>(out + static_cast<long>(rows[m]) * N + c) = w;
}

// x and y times *g in place (bf16, sizes in groups of 8); reads nothing more when *g is 1, what a loss's own backward
// passes.
__global__ void __launch_bounds__(256) scale_by_kernel(uint4* __restrict__ x, long nx, uint4* __restrict__ y, long ny,
                                                       const float* __restrict__ g) {
  pdl_trigger();
  pdl_wait();
  const float s = *g;
  if (s == 1.f) return;
  for (long i = static_cast<long>(blockIdx.x) * 256 + threadIdx.x; i < nx + ny;
       i += static_cast<long>(gridDim.x) * 256) {
    uint4* at = i < nx ? x + i : y + (i - nx);
    uint4 v = *at;
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float2 f = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&w[k]));
      __nv_bfloat162 o = __floats2bfloat162_rn(f.x * s, f.y * s);
      w[k] = *reinterpret_cast<uint32_t*>(&o);
    }
    *at = v;
  }
}

}  // namespace

int readout_pieces(int V) { return (V + kPiece - 1) / kPiece; }

// Splits of K for a product of `tiles` 256 x 256 tiles and `kblocks` K blocks: as many as fill the pairs of SMs once,
// each with eight K blocks at least (a shorter one is all prologue).
int readout_splits(long tiles, long kblocks, int num_sms) {
  const long pairs = num_sms / 2;
  if (tiles >= pairs) return 1;
  return static_cast<int>(std::max(1l, std::min(pairs / std::max(1l, tiles), kblocks / 8)));
}

int launch_readout_plan(const int64_t* targets, int T, int V, int64_t ignore, int* rows, int* pos, int* target_of,
                        int* count, unsigned* status, cudaStream_t stream) {
  return launch_pdl(readout_plan_kernel, dim3(1), dim3(1024), 0, stream, targets, T, V, ignore, rows, pos, target_of,
                    count, status) == cudaSuccess ? 0 : -1;
}

int launch_readout_gather(const void* x, long x_stride, int T, int H, const int* pos, const int* count, void* xs,
                          void* dx, float* losses, cudaStream_t stream) {
  return launch_pdl(readout_gather_kernel, dim3((T + pair::kBK + 7) / 8), dim3(256), 0, stream,
                    static_cast<const bf16*>(x), x_stride, T, H, pos, count, static_cast<bf16*>(xs),
                    static_cast<bf16*>(dx), losses) == cudaSuccess ? 0 : -1;
}

int launch_readout_logits(const CUtensorMap* xs, const CUtensorMap* w, const ReadoutChunk& c, int num_sms,
                          unsigned* status, cudaStream_t stream) {
  LogitsEpi epi{static_cast<float2*>(c.stats), c.picked, c.target + c.row0, static_cast<__half*>(c.e), c.ld, c.V,
                readout_pieces(c.V), c.logit_scale * kLog2e};
  const pair::Shape shape{c.chunk, c.V, c.H, c.count, c.row0, true, false, 1, false};
  return pair::launch_pair<false, false>(*xs, *w, shape, epi, num_sms, status, stream);
}

int launch_readout_finish(const ReadoutChunk& c, int reduction, const float* grad_rows, float* nll, float* losses,
                          cudaStream_t stream) {
  const int pieces = readout_pieces(c.V);
  const int smem = c.e != nullptr ? pieces * 4 : 0;
  if (smem > 48 * 1024 && set_max_smem(readout_finish_kernel, smem) != cudaSuccess) return -1;
  return launch_pdl(readout_finish_kernel, dim3((c.chunk + pair::kBK - 1) / pair::kBK * pair::kBK),
                    dim3(kFinishThreads), smem, stream, static_cast<const float2*>(c.stats), c.picked,
                    c.target + c.row0, c.rows, c.count, c.row0, c.chunk, c.V, pieces, c.e, c.ld, c.logit_scale,
                    reduction, grad_rows, nll, losses) == cudaSuccess ? 0 : -1;
}

int launch_readout_loss(const float* nll, const int* count, int reduction, float* loss, cudaStream_t stream) {
  return launch_pdl(readout_loss_kernel, dim3(1), dim3(1024), 0, stream, nll, count, reduction, loss) == cudaSuccess
             ? 0 : -1;
}

int launch_readout_dx(const CUtensorMap* dz, const CUtensorMap* w, const ReadoutChunk& c, int splits, float* part,
                      void* dx, int num_sms, unsigned* status, cudaStream_t stream) {
  StoreEpi epi{static_cast<bf16*>(dx), splits > 1 ? part : nullptr, c.rows + c.row0, c.H, c.chunk, false, splits == 1};
  const pair::Shape shape{c.chunk, c.H, c.V, c.count, c.row0, true, false, splits, false};
  int rc = pair::launch_pair<false, true>(*dz, *w, shape, epi, num_sms, status, stream);
  if (rc != 0 || splits == 1) return rc;
  const long groups = static_cast<long>(c.chunk) * c.H / 4;
  return launch_pdl(readout_join_kernel, dim3(static_cast<unsigned>((groups + 255) / 256)), dim3(256), 0, stream, part,
                    splits, static_cast<long>(c.chunk), c.H, c.rows + c.row0, c.count, c.row0, c.chunk,
                    static_cast<bf16*>(dx)) == cudaSuccess ? 0 : -1;
}

int launch_readout_dw(const CUtensorMap* dz, const CUtensorMap* xs, const ReadoutChunk& c, float* sum, bool first,
                      bool last, void* dw, int num_sms, unsigned* status, cudaStream_t stream) {
  StoreEpi epi{static_cast<bf16*>(dw), first && last ? nullptr : sum, nullptr, c.H, 0, !first, last};
  const pair::Shape shape{c.V, c.H, c.chunk, c.count, c.row0, false, true, 1, true};
  return pair::launch_pair<true, true>(*dz, *xs, shape, epi, num_sms, status, stream);
}

int launch_scale_by(void* x, long nx, void* y, long ny, const float* g, int num_sms, cudaStream_t stream) {
  const long blocks = std::min(((nx + ny) / 8 + 255) / 256, static_cast<long>(num_sms) * 8);
  if (blocks <= 0) return 0;
  return launch_pdl(scale_by_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, static_cast<uint4*>(x),
                    nx / 8, static_cast<uint4*>(y), ny / 8, g) == cudaSuccess ? 0 : -1;
}

}  // namespace ecz
