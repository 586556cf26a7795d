// Quantisation of bf16 rows to 4-bit floating point (fp4_common.cuh describes the formats) and back.
//
// fp4_quantize_kernel: a team of warps per row, its values in registers. nvfp4 first takes the row's largest magnitude
// (the row's power of two); a group's largest magnitude comes from 2 or 4 neighbouring lanes, 8 columns each.
// Bound by HBM: 2 bytes read and 0.56 (nvfp4) or 0.53 (mxfp4) written per column.
#include <algorithm>

#include "fp4_common.cuh"
#include "launchers.h"

namespace ecz {

namespace {

using namespace fp4;

// x [rows, 8 vecs], row stride x_stride; rows from `rows` on up to a multiple of 128 get zero scales. Teams of `warps`
// warps take the rows; NV vectors of 8 columns a lane cover the row and the scales' padding.
template <int FMT, int NV>
__global__ void __launch_bounds__(1024) fp4_quantize_kernel(const bf16* __restrict__ x, size_t x_stride,
                                                            uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                            float* __restrict__ row_scale, int rows, int vecs, int tiles,
                                                            int warps, bool early) {
  __shared__ float scratch[32];
  if (early) pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int team = warp / warps, wt = warp - team * warps;
  const int row = blockIdx.x * (blockDim.x / (32 * warps)) + team;
  const int first = wt * 32 + lane, step = warps * 32;
  const bool real = row < rows;
  uint4 raw[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int vec = first + i * step;
    raw[i] = real && vec < vecs ? *reinterpret_cast<const uint4*>(x + row * x_stride + static_cast<size_t>(vec) * 8)
                                : make_uint4(0, 0, 0, 0);
  }
  float mul = 1.f;
  if constexpr (FMT == kNv) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float v[8];
      unpack8(raw[i], v);
      bool bad;
      m = fmaxf(m, finite_max8(v, bad));
    }
    m = warp_max(m);
    if (warps > 1) {
      if (lane == 0) scratch[warp] = m;
      __syncthreads();
      for (int w = 0; w < warps; ++w) m = fmaxf(m, scratch[team * warps + w]);
    }
    const int e = row_exponent(m);
    mul = pow2(-e);
    if (real && first == 0) row_scale[row] = pow2(e);
  }
  if (row >= (rows + 127) / 128 * 128) return;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int base = (wt + i * warps) * 32;
    if (base >= tiles * Format<FMT>::kWordLanes) break;
    float v[8];
    unpack8(raw[i], v);
    store8<FMT>(v, mul, row, base + lane, real ? vecs : 0, tiles, codes, scales);
  }
}

// One thread per 8 columns: the values of their codes, exact in bf16.
template <int FMT>
__global__ void __launch_bounds__(256) fp4_dequantize_kernel(const uint8_t* __restrict__ codes,
                                                             const uint8_t* __restrict__ scales,
                                                             const float* __restrict__ row_scale,
                                                             bf16* __restrict__ out, int rows, int vecs, int tiles) {
  using F = Format<FMT>;
  pdl_wait();
  const size_t total = static_cast<size_t>(rows) * vecs;
  for (size_t i = blockIdx.x * static_cast<size_t>(blockDim.x) + threadIdx.x; i < total;
       i += static_cast<size_t>(gridDim.x) * blockDim.x) {
    const int row = static_cast<int>(i / vecs), vec = static_cast<int>(i - static_cast<size_t>(row) * vecs);
    const uint32_t c = *reinterpret_cast<const uint32_t*>(codes + i * 4);
    const int group = vec / F::kLanes;
    const float s = scale_value<FMT>(scales[scale_word(row, group >> 2, tiles) + (group & 3)]) *
                    (FMT == kNv ? row_scale[row] : 1.f);
    *reinterpret_cast<uint4*>(out + i * 8) = values8(c, s);
  }
}

template <int FMT>
int run_quantize(const void* x, size_t x_stride, uint8_t* codes, uint8_t* scales, float* row_scale, int rows, int K,
                 bool early, int sms, cudaStream_t stream) {
  const int vecs = K / 8, tiles = fp4_scale_tiles(FMT, K);
  const int padded = tiles * Format<FMT>::kWordLanes;
  // few rows: as many warps as there are vectors, for the shortest chain; many: four vectors a lane and several teams a
  // block (more loads in flight per barrier)
  const int all = (padded + 31) / 32;
  const bool many = rows >= 4 * sms;
  int warps = std::min(32, std::max(1, many ? (all + 3) / 4 : all));
  if (warps <= 8) {
    int p = 1;
    while (p < warps) p *= 2;
    warps = p;
  }
  const int nv = (all + warps - 1) / warps;
  const int teams = warps < 8 && many ? 8 / warps : 1;
  const int padded_rows = (rows + 127) / 128 * 128;
  const dim3 grid((padded_rows + teams - 1) / teams), block(32 * warps * teams);
  auto go = [&](auto kernel) {
    return launch_pdl(kernel, grid, block, 0, stream, static_cast<const bf16*>(x), x_stride, codes, scales, row_scale,
                      rows, vecs, tiles, warps, early) == cudaSuccess ? 0 : -1;
  };
  if (nv <= 1) return go(fp4_quantize_kernel<FMT, 1>);
  if (nv <= 2) return go(fp4_quantize_kernel<FMT, 2>);
  if (nv <= 4) return go(fp4_quantize_kernel<FMT, 4>);
  if (nv <= 8) return go(fp4_quantize_kernel<FMT, 8>);
  return -1;
}

}  // namespace

int fp4_scale_tiles(int fmt, int K) {
  return (K + kBlockK - 1) / kBlockK * (fmt == kNv ? Format<kNv>::kTilesPerBlock : Format<kMx>::kTilesPerBlock);
}

int launch_fp4_quantize(const void* x, size_t x_stride, int fmt, void* codes, void* scales, float* row_scale, int rows,
                        int K, bool early, int sms, cudaStream_t stream) {
  if (K % 32 != 0 || K < 32 || K > kFp4MaxK || rows < 1) return -1;
  auto* c = static_cast<uint8_t*>(codes);
  auto* s = static_cast<uint8_t*>(scales);
  return fmt == kNv ? run_quantize<kNv>(x, x_stride, c, s, row_scale, rows, K, early, sms, stream)
                    : run_quantize<kMx>(x, x_stride, c, s, row_scale, rows, K, early, sms, stream);
}

int launch_fp4_dequantize(const void* codes, const void* scales, const float* row_scale, int fmt, void* out, int rows,
                          int K, int sms, cudaStream_t stream) {
  if (K % 32 != 0 || rows < 1) return -1;
  const int vecs = K / 8, tiles = fp4_scale_tiles(fmt, K);
  const size_t total = static_cast<size_t>(rows) * vecs;
  const dim3 grid(static_cast<unsigned>(std::min<size_t>((total + 255) / 256, static_cast<size_t>(sms) * 32)));
  auto kernel = fmt == kNv ? fp4_dequantize_kernel<kNv> : fp4_dequantize_kernel<kMx>;
  return launch_pdl(kernel, grid, dim3(256), 0, stream, static_cast<const uint8_t*>(codes),
                    static_cast<const uint8_t*>(scales), row_scale, static_cast<bf16*>(out), rows, vecs, tiles) ==
                 cudaSuccess ? 0 : -1;
}

}  // namespace ecz
