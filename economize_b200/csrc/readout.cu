// Softmax cross-entropy of a vocabulary readout without keeping the logits, with its gradient.
//
//   z_tv = s x_t . w_v     L_t = log sum_v exp z_tv     nll_t = L_t - z_{t, y_t}
//   dz_tv = g_t (exp(z_tv - L_t) - [v = y_t])     dx_t = s sum_v dz_tv w_v     dW_v = s sum_t dz_tv x_t
//
// Rows whose target is the ignored index are left out before the first product: the gather kernel packs the other rows'
// states in order, so a prompt mask saves its share of all three products and nothing that stands in a masked row (not
// even NaN) reaches a result. It also computes each row's target logit on the CUDA cores, in fp32 with rounding: the
// tensor cores' accumulation of 4096 products is off by up to 1e-5 of a logit of 10, and the target's is the large one.
// Packed rows are processed in chunks:
//
//   logits    256 x 256 tiles of X . W^T (gemm_pair.cuh); the epilogue reduces each row's 128-column piece, without the
//             target's column, to its maximum m and sum of exp(z - m) and, when gradients follow, stores e = exp(z - m)
//             in fp16. e lies in (0, 1] with its piece's largest at 1, so fp16 keeps 11 bits of everything that counts
//             (bf16 would add a second 8-bit rounding to the gradients); the logits themselves are never stored.
//   finish    joins a row's pieces to S, the sum over the other tokens. nll = log(1 + S exp(-z_y)) and the target's
//             gradient -S / (S + exp(z_y)) keep their digits where the target's probability is near one. Rewrites e in
//             place as dz = g (e exp(m - L)) in bf16, the one rounding of the gradient's left factor. What all rows share
//             (s, 1 / count of a mean, the first row's g of losses by row) stays out of dz and is multiplied in at the
//             end, in fp32: near -1 / count, most targets' entries were rounded the same way, and the whole gradient was
//             off by up to 0.4%. The last CTA of the last chunk adds the losses up in row order.
//   products  dX = dz . W (K = V, W read MN-major) and dW = dz^T . X (K = rows, both operands MN-major), no
//             transposes. Over several chunks dW is summed in an fp32 buffer in chunk order.
//
// Without gradients only the statistics of the pieces are written (8 bytes per 128 logits).
//
// Measured on one B200, 4096 rows x 4096 x 32000: logits 681 us (1580 TFLOP/s), finish 101 us (e read and dz written
// once, 5.2 TB/s), dX 683 us, dW 687 us (1570 each), one by one; 2.55 to 2.65 ms in a row, at the clock that the power
// limit leaves. 1024 rows x 4096 x 128256, losses only: 860 us in a row, 1250 TFLOP/s. 16 rows x 1024 x 32000 with both
// gradients: 87 us, of which the two reads of W and the write of dW need 30: 17 to 25 for each of the three products,
// whose tiles of 256 rows stand almost empty, and the launches of a training step's call.
//
// The tensor cores cut off, not round, what their fp32 sums cannot hold, so the logits are summed in parts (LogitsEpi).
// The target's logit does not share what is left of it (see the gather kernel). The gradients' products do: over K =
// 128256 a sum is up to 1.2e-4 of itself too small by the same measure, a twentieth of the rounding to bf16 that follows.
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

// ---- plan and gather -------------------------------------------------------------------------------------------
__device__ __forceinline__ bool has_target(int64_t y, int V, int64_t ignore, unsigned* status) {
  if (y == ignore) return false;
  if (y >= 0 && y < V) return true;
  atomicOr(status, kStatusBadIndex);  // counts as ignored
  return false;
}

// One CTA, for many rows: pos[t] = the place of row t among those with a target, or -1; *count = how many.
__global__ void __launch_bounds__(1024) readout_plan_kernel(const int64_t* __restrict__ targets, int T, int V,
                                                            int64_t ignore, int* __restrict__ pos,
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
    const bool keep = t < T && has_target(targets[t], V, ignore, status);
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
    if (t < T) pos[t] = keep ? before + __popc(ballot & ((1u << lane) - 1u)) : -1;
    __syncthreads();
    if (threadIdx.x == 0) base += total;
    __syncthreads();
  }
  if (threadIdx.x == 0) *count = base;
}

// Warp per row t, eight to a CTA: its state to xs, its target's logit to picked, or zeros to dx (and losses[t]) where it
// is ignored. The rows behind the last packed one are zeroed up to the K block that reads them. Without a plan (pos
// null, few rows) every CTA counts the rows before its own itself, which saves a launch.
// Rows up to which every CTA counts. Losses of T rows x 256 x 1000 from a CUDA graph, us counted / planned: 1024 18.0 /
// 18.7, 2048 21.3 / 23.7, 4096 30.6 / 32.7, 16384 95.8 / 98.1, 32768 206 / 182, 131072 1483 / 771 (every CTA reads all
// targets: T^2 / 8 of them). Between 2048 and about 20000 the rule is 2 to 4 us on the safe side.
constexpr int kPlanRows = 2048;

struct GatherArgs {
  const bf16 *x, *w;
  long x_stride, w_stride, xs_stride;
  const int64_t* targets;
  int T, H, V;
  int64_t ignore;
  float scale2;      // logit scale times log2(e)
  const int* pos;
  int *rows, *target_of, *count;  // packed row -> row, target; how many, and the finish kernel's counter
  float* picked;
  bf16 *xs, *dx;
  float* losses;
};

__global__ void __launch_bounds__(256) readout_gather_kernel(const __grid_constant__ GatherArgs a, unsigned* status) {
  __shared__ int before, total;
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t0 = blockIdx.x * 8, t = t0 + warp;
  int p = -1, n = 0;
  if (a.pos == nullptr) {
    if (threadIdx.x == 0) before = total = 0;
    __syncthreads();
    int mine = 0, all = 0;
    for (int i = threadIdx.x; i < a.T; i += 256) {
      const int64_t y = a.targets[i];
      const bool keep = y != a.ignore && y >= 0 && y < a.V;
      all += keep;
      mine += keep && i < t0;
    }
    mine = __reduce_add_sync(0xffffffffu, mine);
    all = __reduce_add_sync(0xffffffffu, all);
    if (lane == 0) {
      atomicAdd(&before, mine);
      atomicAdd(&total, all);
    }
    __syncthreads();
    n = total;
    if (t < a.T && has_target(a.targets[t], a.V, a.ignore, status)) {
      p = before;
      for (int i = t0; i < t; ++i) {
        const int64_t y = a.targets[i];
        p += y != a.ignore && y >= 0 && y < a.V;
      }
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.count = n;
  } else {
    n = *a.count;
    if (t < a.T) p = a.pos[t];
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) a.count[1] = 0;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  if (t >= a.T) {
    const int r = n + (t - a.T);
    if (t - a.T < pair::kBK && r < (n + pair::kBK - 1) / pair::kBK * pair::kBK)
      for (int c = lane * 8; c < a.H; c += 256)
        *reinterpret_cast<uint4*>(a.xs + static_cast<size_t>(r) * a.xs_stride + c) = zero;
    return;
  }
  if (p < 0) {
    if (a.dx != nullptr)
      for (int c = lane * 8; c < a.H; c += 256)
        *reinterpret_cast<uint4*>(a.dx + static_cast<size_t>(t) * a.H + c) = zero;
    if (a.losses != nullptr && lane == 0) a.losses[t] = 0.f;
    return;
  }
  const int y = static_cast<int>(a.targets[t]);
  const bf16 *x = a.x + static_cast<size_t>(t) * a.x_stride, *w = a.w + static_cast<size_t>(y) * a.w_stride;
  float acc[2] = {0.f, 0.f};
  for (int c = lane * 8; c < a.H; c += 256) {
    const uint4 u = *reinterpret_cast<const uint4*>(x + c), v = *reinterpret_cast<const uint4*>(w + c);
    *reinterpret_cast<uint4*>(a.xs + static_cast<size_t>(p) * a.xs_stride + c) = u;
    const uint32_t l[4] = {u.x, u.y, u.z, u.w}, r[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&l[k]));
      const float2 g = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&r[k]));
      acc[0] = fmaf(f.x, g.x, acc[0]);
      acc[1] = fmaf(f.y, g.y, acc[1]);
    }
  }
  const float z = warp_sum(acc[0] + acc[1]);
  if (lane == 0) {
    a.rows[p] = t;
    a.target_of[p] = y;
    a.picked[p] = z * a.scale2;
  }
}

// ---- logits: statistics (and e) of a tile's rows -----------------------------------------------------------------
// kSums: of logits in registers, added up from parts of at most kPartBlocks K blocks (see gemm_pair.cuh), else read twice
// from TMEM. One sum was 3.9e-6 of itself too small at H = 4096, and a mean loss of 4.2 by 1.1e-6 of itself; parts of
// 1024 leave 1.0e-6 and 2.5e-7, of 512 half of that. What parts cost, us of the logits with e, one sum / 1024 / 512:
// 4096 x 4096 x 32000 669 / 680 / 756, 2048 x 1088 x 50257 (losses) 141 / 152 / 179. Where H takes one part there is
// nothing to add up, and the shorter form serves (16 x 1024 x 32000 with both gradients: 90, in registers 96).
constexpr int kPartBlocks = 16;

template <bool kSums>
struct LogitsEpi {
  static constexpr bool kParts = kSums;
  float2* stats;      // [rows of the chunk, pieces]: (max, sum of exp2(z - max)) without the target, log2 units
  const int* target;  // [rows] of the chunk
  __half* e;          // [rows, ld] or null
  long ld;
  int V, pieces;
  float scale2;  // logit scale times log2(e)

  __device__ __forceinline__ void operator()(const pair::Unit&, int M, int row0, int col0, uint32_t taddr, bool,
                                             uint8_t* patch, int lane) const {
    piece(M, row0, col0, patch, lane, [&](int c, float* v) {
      tmem_ld32(taddr + c, v);
      return v;
    });
  }

  __device__ __forceinline__ void operator()(const pair::Unit&, int M, int row0, int col0, float (&z)[kPiece],
                                             uint8_t* patch, int lane) const {
    piece(M, row0, col0, patch, lane, [&](int c, float*) { return z + c; });
  }

  // `fetch`: the logits of 32 columns from c on, in the given place or one of their own, to be written over.
  template <class Fetch>
  __device__ __forceinline__ void piece(int M, int row0, int col0, uint8_t* patch, int lane, Fetch fetch) const {
    constexpr int kUnroll = kSums ? kPiece / 32 : 1;
    if (row0 >= M || col0 >= V) return;  // uniform over the warp
    const int row = row0 + lane;
    const int cols = V - col0;
    const int mine = row < M ? target[row] - col0 : -1;
    // the columns of 32 from c on that count: inside the vocabulary and not the row's target
    auto counted = [&](int c) {
      const uint32_t inside = cols - c >= 32 ? ~0u : (1u << max(0, cols - c)) - 1u;
      return (mine >> 5) == (c >> 5) ? inside & ~(1u << (mine & 31)) : inside;
    };
    float top = -INFINITY;
#pragma unroll kUnroll
    for (int c = 0; c < kPiece; c += 32) {
      float here[32];
      float* v = fetch(c, here);
      const uint32_t bits = counted(c);
      if (__all_sync(0xffffffffu, bits == ~0u)) {
#pragma unroll
        for (int j = 0; j < 32; ++j) top = fmaxf(top, v[j] * scale2);
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j) top = (bits >> j) & 1u ? fmaxf(top, v[j] * scale2) : top;
      }
    }
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
#pragma unroll kUnroll
    for (int c = 0; c < kPiece; c += 32) {
      float here[32];
      float* v = fetch(c, here);
      const uint32_t bits = counted(c);
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] = ex2(fmaf(v[j], scale2, -ref));
      if (!__all_sync(0xffffffffu, bits == ~0u)) {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = (bits >> j) & 1u ? v[j] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < 32; ++j) sum += v[j];
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

// The factor that the gradients' products leave to their end.
struct Shared {
  float logit_scale;
  bool mean;
  const float* grad_rows;   // of losses by row, or null
  const int *rows, *count;  // all packed rows
  // the first row's gradient: rows of one gradient, as a mean of the losses gives them, have entries as a sum's
  __device__ __forceinline__ float grad() const {
    const float g = grad_rows != nullptr && *count > 0 ? fabsf(grad_rows[rows[0]]) : 1.f;
    return g > 0x1p-40f && g < 0x1p40f ? g : 1.f;  // a quotient of another row's, below 2^87, does not overflow
  }
  __device__ __forceinline__ float value() const {
    const float f = logit_scale * grad();
    return mean ? f / static_cast<float>(max(1, *count)) : f;
  }
};

// CTAs (row, part) of the packed rows of a chunk: every part joins the row's pieces and turns its columns of e into dz
// in place; part 0 writes nll. NaN statistics give NaN, as the plain formula does. Counts itself on *done where a loss
// is wanted of the last chunk: the last CTA adds up.
constexpr int kFinishThreads = 256;

struct FinishArgs {
  const float2* stats;
  const float* picked;  // of the chunk's rows
  const int *target, *rows, *count;
  int row0, chunk, V, pieces;
  void* e_dz;
  long ld;
  Shared shared;
  float *nll, *losses;
  float* loss;  // null but for the last chunk of a scalar loss
  int* done;
};

// loss = the sum of nll in a fixed order (thread t sums rows t, t + 256, ..., then a tree), / count, 0 without rows.
__device__ __forceinline__ void add_up(const FinishArgs& a, float* red) {
  __shared__ bool last;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(a.done, 1) == static_cast<int>(gridDim.x * gridDim.y) - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  const int n = *a.count;
  float v = 0.f;
  for (int i = threadIdx.x; i < n; i += kFinishThreads) v += __ldcg(a.nll + i);
  v = block_reduce(v, red, false);
  if (threadIdx.x == 0) *a.loss = a.shared.mean ? (n > 0 ? v / static_cast<float>(n) : 0.f) : v;
}

__device__ __forceinline__ void finish_row(const FinishArgs& a, int r, float* factor, float* red) {
  const float2* st = a.stats + static_cast<size_t>(r) * a.pieces;
  const float z = a.picked[r];
  float top = z;
  bool nan = false;
  for (int j = threadIdx.x; j < a.pieces; j += kFinishThreads) {
    top = fmaxf(top, st[j].x);
    nan |= st[j].y != st[j].y;
  }
  top = block_reduce(top, red, true);
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  for (int j = threadIdx.x; j < a.pieces; j += kFinishThreads) {
    const float2 v = st[j];
    sum += v.y * exp2f(v.x - ref);
  }
  if (nan) sum = NAN;
  sum = block_reduce(sum, red, false);
  const float own = exp2f(z - ref);
  const float lse2 = ref + log2f(sum + own);
  const float loss = z >= ref ? log1pf(sum) : (lse2 - z) * kLn2;
  const int orig = a.rows[a.row0 + r];
  if (threadIdx.x == 0 && blockIdx.y == 0) {
    if (a.nll != nullptr) a.nll[a.row0 + r] = loss;
    if (a.losses != nullptr) a.losses[orig] = loss;
  }
  if (a.e_dz == nullptr) return;
  const float g = a.shared.grad_rows != nullptr ? a.shared.grad_rows[orig] / a.shared.grad() : 1.f;
  for (int j = threadIdx.x; j < a.pieces; j += kFinishThreads) factor[j] = exp2f(st[j].x - lse2) * g;
  __syncthreads();
  const int tgt = a.target[r];
  const float at_target = -g * (sum / (sum + own));
  uint16_t* row = static_cast<uint16_t*>(a.e_dz) + static_cast<size_t>(r) * a.ld;
  const int step = kFinishThreads * 8, begin = blockIdx.y * step;
  for (int c = begin + threadIdx.x * 8; c < a.V; c += step * gridDim.y) {
    uint4 v = *reinterpret_cast<const uint4*>(row + c);
    const float f = factor[c / kPiece];
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 ev = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
      float p = ev.x * f, q = ev.y * f;
      if (c + 2 * k == tgt) p = at_target;
      if (c + 2 * k + 1 == tgt) q = at_target;
      __nv_bfloat162 o = __floats2bfloat162_rn(p, q);
      w[k] = *reinterpret_cast<uint32_t*>(&o);
    }
    *reinterpret_cast<uint4*>(row + c) = v;
  }
}

__global__ void __launch_bounds__(kFinishThreads) readout_finish_kernel(const __grid_constant__ FinishArgs a) {
  extern __shared__ float factor[];  // [pieces]: exp2(m - L) g
  __shared__ float red[kFinishThreads / 32];
  pdl_trigger();
  pdl_wait();
  const int total = *a.count;
  const int n = min(a.chunk, total - a.row0);
  const int r = blockIdx.x;
  if (r < n) {
    finish_row(a, r, factor, red);
  } else if (n > 0 && a.e_dz != nullptr && r < (n + pair::kBK - 1) / pair::kBK * pair::kBK) {
    // zero rows up to the K block of dz^T . X that reads them
    uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.e_dz) + static_cast<size_t>(r) * a.ld);
    for (int c = blockIdx.y * kFinishThreads + threadIdx.x; c < a.ld / 8; c += kFinishThreads * gridDim.y)
      dst[c] = make_uint4(0, 0, 0, 0);
  }
  if (a.loss != nullptr) add_up(a, red);
}

// ---- product epilogues ---------------------------------------------------------------------------------------------
// Where a split tile's partial keeps columns 32 cb + 4 q .. + 3 of row 32 rb + lane, in floats: a warp's lanes hold a
// row each and write side by side.
__device__ __forceinline__ int partial_at(int rb, int cb, int q, int lane) {
  return (((rb * (pair::kTile / 32) + cb) * 8 + q) * 32 + lane) * 4;
}

// Stores a warp's 32 x 128 accumulators: bf16 rows (through the patch, 128-byte row segments), a split tile's fp32
// partial, or an fp32 running sum over the chunks whose last chunk stores bf16.
struct StoreEpi {
  static constexpr bool kParts = false;
  bf16* out;        // [.., N]
  float* part;      // partials of split tiles, [tile, split] and see partial_at
  float* sum;       // running sum [M, N], or null
  const int* rows;  // destination row of row m (null: m)
  int N;
  bool add, last;   // running sum: add to what is there; store the sum as bf16
  Shared shared;    // what bf16 results are multiplied by

  __device__ __forceinline__ void operator()(const pair::Unit& u, int M, int row0, int col0, uint32_t taddr, bool zero,
                                             uint8_t* patch, int lane) const {
    if (row0 >= M || col0 >= N) return;
    const int cols = min(128, N - col0);
    const bool split = u.splits > 1;
    float* prow = sum == nullptr ? nullptr : sum + static_cast<size_t>(row0 + lane) * N + col0;
    float* tile = part + (static_cast<size_t>(u.tail) * u.splits + u.split) * pair::kTile * pair::kTile;
    const bool row_ok = row0 + lane < M;
    const float factor = last ? shared.value() : 1.f;
#pragma unroll 1
    for (int c = 0; c < cols; c += 32) {
      float v[32];
      if (zero) {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = 0.f;
      } else {
        tmem_ld32(taddr + c, v);
      }
      if (split) {
#pragma unroll
        for (int j = 0; j < 32; j += 4)
          *reinterpret_cast<float4*>(tile + partial_at((row0 - u.m0) / 32, (col0 - u.n0 + c) / 32, j / 4, lane)) =
              make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
        continue;
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
      for (int j = 0; j < 32; ++j) v[j] *= factor;
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

constexpr int kJoinThreads = 256;

// The split tiles of a product: out[rows[m]] = bf16(the shared factor times the sum of the partials, in order). A thread
// adds up eight columns of a row; CTAs (32 rows, tile, place of the eight in every 32 columns).
__global__ void __launch_bounds__(kJoinThreads)
    readout_join_kernel(const __grid_constant__ pair::Shape shape, const float* __restrict__ part, const int* rows,
                        Shared shared, bf16* __restrict__ out) {
  pdl_trigger();
  pdl_wait();
  const pair::Schedule sched(shape);
  const int u = sched.whole + blockIdx.y * sched.splits;
  if (sched.splits == 1 || u >= sched.units) return;
  const pair::Unit t = sched.unit(u);
  const int rb = blockIdx.x, cb = threadIdx.x / 32, lane = threadIdx.x & 31;
  const int m = t.m0 + rb * 32 + lane;
  if (m >= sched.M) return;
  const float* tile = part + static_cast<size_t>(t.tail) * t.splits * pair::kTile * pair::kTile;
  const float f = shared.value();
  bf16* row = out + static_cast<long>(rows != nullptr ? rows[m] : m) * shape.N;
  const int q = blockIdx.z * 2, n = t.n0 + cb * 32 + q * 4;
  if (n >= shape.N) return;
  float acc[8] = {};
#pragma unroll 4
  for (int i = 0; i < t.splits; ++i) {
    const float* from = tile + static_cast<size_t>(i) * pair::kTile * pair::kTile;
    const float4 a = *reinterpret_cast<const float4*>(from + partial_at(rb, cb, q, lane));
    const float4 b = *reinterpret_cast<const float4*>(from + partial_at(rb, cb, q + 1, lane));
    acc[0] += a.x;
    acc[1] += a.y;
    acc[2] += a.z;
    acc[3] += a.w;
    acc[4] += b.x;
    acc[5] += b.y;
    acc[6] += b.z;
    acc[7] += b.w;
  }
  uint32_t w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(acc[2 * k] * f, acc[2 * k + 1] * f);
    w[k] = *reinterpret_cast<const uint32_t*>(&h);
  }
  *reinterpret_cast<uint4*>(row + n) = make_uint4(w[0], w[1], w[2], w[3]);
}

// x and y times *g in place (bf16, sizes in groups of 8); reads nothing more when *g is 1, what a loss's own backward
// passes. Unless *g is a power of two this is a second rounding to bf16 of the gradients of a mean or sum, which were
// rounded before *g was known: as much again as the first at most. Keeping what the first rounding left would write
// every gradient twice (65 MB more for 16 rows x 1024 x 32000: 10 of 90 us) for a case that is not the usual one.
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

bool readout_needs_plan(int T) { return T > kPlanRows; }

int launch_readout_plan(const int64_t* targets, int T, int V, int64_t ignore, int* pos, int* count, unsigned* status,
                        cudaStream_t stream) {
  return launch_pdl(readout_plan_kernel, dim3(1), dim3(1024), 0, stream, targets, T, V, ignore, pos, count, status) ==
                 cudaSuccess ? 0 : -1;
}

int launch_readout_gather(const ReadoutRows& r, const int* pos, int* rows, int* target_of, int* count, float* picked,
                          void* xs, void* dx, float* losses, unsigned* status, cudaStream_t stream) {
  const GatherArgs a{static_cast<const bf16*>(r.x), static_cast<const bf16*>(r.w), r.x_stride, r.w_stride, r.xs_stride,
                     r.targets, r.T, r.H, r.V, r.ignore, r.logit_scale * kLog2e, pos, rows, target_of, count, picked,
                     static_cast<bf16*>(xs), static_cast<bf16*>(dx), losses};
  return launch_pdl(readout_gather_kernel, dim3((r.T + pair::kBK + 7) / 8), dim3(256), 0, stream, a, status) ==
                 cudaSuccess ? 0 : -1;
}

int launch_readout_logits(const CUtensorMap* xs, const CUtensorMap* w, const ReadoutChunk& c, int num_sms,
                          unsigned* status, cudaStream_t stream) {
  const int blocks = (c.H + pair::kBK - 1) / pair::kBK, parts = (blocks + kPartBlocks - 1) / kPartBlocks;
  const pair::Shape shape{c.chunk, c.V, c.H, c.count, c.row0, true, false, num_sms / 2, false, false,
                          (blocks + parts - 1) / parts};
  auto launch = [&](auto epi) { return pair::launch_pair<false, false>(*xs, *w, shape, epi, status, stream); };
  float2* stats = static_cast<float2*>(c.stats);
  __half* e = static_cast<__half*>(c.e);
  const int pieces = readout_pieces(c.V);
  const float scale2 = c.logit_scale * kLog2e;
  return parts > 1 ? launch(LogitsEpi<true>{stats, c.target + c.row0, e, c.ld, c.V, pieces, scale2})
                   : launch(LogitsEpi<false>{stats, c.target + c.row0, e, c.ld, c.V, pieces, scale2});
}

static Shared shared_of(const ReadoutChunk& c) {
  return Shared{c.logit_scale, c.reduction == kReduceMean, c.grad_rows, c.rows, c.count};
}

int launch_readout_finish(const ReadoutChunk& c, float* nll, float* losses, float* loss, int* done, int num_sms,
                          cudaStream_t stream) {
  const int pieces = readout_pieces(c.V);
  const int smem = c.e != nullptr ? pieces * 4 : 0;
  if (smem > 40 * 1024 && set_max_smem(readout_finish_kernel, smem) != cudaSuccess) return -1;
  const FinishArgs a{static_cast<const float2*>(c.stats), c.picked + c.row0, c.target + c.row0, c.rows, c.count, c.row0,
                     c.chunk, c.V, pieces, c.e, c.ld, shared_of(c), nll, losses, loss, done};
  const int rows = (c.chunk + pair::kBK - 1) / pair::kBK * pair::kBK;
  // few rows: several CTAs to a row, so that eight on every SM share the columns
  const int most = c.e == nullptr ? 1 : (c.V + kFinishThreads * 8 - 1) / (kFinishThreads * 8);
  const int parts = std::max(1, std::min(most, num_sms * 8 / rows));
  return launch_pdl(readout_finish_kernel, dim3(rows, parts), dim3(kFinishThreads), smem, stream, a) == cudaSuccess ? 0
                                                                                                                   : -1;
}

static int launch_join(const pair::Shape& shape, const float* part, const int* rows, const ReadoutChunk& c, void* out,
                       cudaStream_t stream) {
  const int tail = pair::most_tail(shape);
  if (tail == 0) return 0;
  return launch_pdl(readout_join_kernel, dim3(pair::kTile / 32, tail, 4), dim3(kJoinThreads), 0,
                    stream, shape, part, rows, shared_of(c), static_cast<bf16*>(out)) == cudaSuccess ? 0 : -1;
}

long readout_part_bytes(int num_sms) { return static_cast<long>(num_sms / 2) * pair::kTile * pair::kTile * 4; }

int launch_readout_dx(const CUtensorMap* dz, const CUtensorMap* w, const ReadoutChunk& c, float* part, void* dx,
                      int num_sms, unsigned* status, cudaStream_t stream) {
  const int* rows = c.rows + c.row0;
  const StoreEpi epi{static_cast<bf16*>(dx), part, nullptr, rows, c.H, false, true, shared_of(c)};
  const pair::Shape shape{c.chunk, c.H, c.V, c.count, c.row0, true, false, num_sms / 2, true, false, 0};
  const int rc = pair::launch_pair<false, true>(*dz, *w, shape, epi, status, stream);
  return rc != 0 ? rc : launch_join(shape, part, rows, c, dx, stream);
}

int launch_readout_dw(const CUtensorMap* dz, const CUtensorMap* xs, const ReadoutChunk& c, float* part, float* sum,
                      bool first, bool last, void* dw, int num_sms, unsigned* status, cudaStream_t stream) {
  const bool once = first && last;
  const StoreEpi epi{static_cast<bf16*>(dw), part, once ? nullptr : sum, nullptr, c.H, !first, last, shared_of(c)};
  const pair::Shape shape{c.V, c.H, c.chunk, c.count, c.row0, false, true, num_sms / 2, once, true, 0};
  const int rc = pair::launch_pair<true, true>(*dz, *xs, shape, epi, status, stream);
  return rc != 0 ? rc : launch_join(shape, part, nullptr, c, dw, stream);
}

int launch_scale_by(void* x, long nx, void* y, long ny, const float* g, int num_sms, cudaStream_t stream) {
  const long blocks = std::min(((nx + ny) / 8 + 255) / 256, static_cast<long>(num_sms) * 8);
  if (blocks <= 0) return 0;
  return launch_pdl(scale_by_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, static_cast<uint4*>(x),
                    nx / 8, static_cast<uint4*>(y), ny / 8, g) == cudaSuccess ? 0 : -1;
}

}  // namespace ecz
