// Quantisation of bf16 rows to 4-bit floating point (fp4_common.cuh describes the formats) and back.
//
// fp4_quantize_kernel: a team of warps per row, its values in registers as they were loaded, 16 columns to a lane (one
// 32-byte load), so a lane holds a whole group of nvfp4 and two lanes one of mxfp4. nvfp4 first takes the row's largest
// magnitude, for the row's power of two. Bound by HBM: 2 bytes read and 0.56 (nvfp4) or 0.53 (mxfp4) written per column.
// 8192 rows of 14336 in mxfp4 take 45 us (6.5 TB/s) and 48 back to bf16 (6.2 TB/s); a row of 4096 takes 3.6, one dependent
// load, maximum and store behind a launch.
#include <algorithm>

#include "fp4_common.cuh"
#include "launchers.h"

namespace ecz {

namespace {

using namespace fp4;

// x [rows, 16 vecs], row stride x_stride. Teams of `warps` warps take the rows; NV vectors of 16 columns a lane cover the
// row and the scales' padding. Blocks beyond `rows` write zero scales.
template <int FMT, int NV>
__global__ void __launch_bounds__(1024) fp4_quantize_kernel(const bf16* __restrict__ x, size_t x_stride,
                                                            uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                            float* __restrict__ row_scale, int rows, int vecs, int tiles,
                                                            int warps, bool early) {
  __shared__ uint32_t scratch[32];
  if (early) pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int team = warp / warps, first = (warp - team * warps) * 32 + lane, step = warps * 32;
  const int row = blockIdx.x * (blockDim.x / step) + team;
  const bool real = row < rows;
  uint32_t raw[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int vec = first + i * step;
#pragma unroll
    for (int j = 0; j < 8; ++j) raw[i][j] = 0;
    if (real && vec < vecs) load32(x + row * x_stride + static_cast<size_t>(vec) * 16, raw[i]);
  }
  float mul = 1.f;
  if constexpr (FMT == kNv) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) top = max(top, max_bits<8>(raw[i]));
    if (top >= 0x7f80u) {  // infinities and NaN do not count
      top = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) top = max(top, finite_bits<8>(raw[i]));
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if (warps > 1) {
      if (lane == 0) scratch[warp] = top;
      __syncthreads();
      for (int w = 0; w < warps; ++w) top = max(top, scratch[team * warps + w]);
    }
    const int e = row_exponent(bits_value(top));
    mul = pow2(-e);
    if (real && first == 0) row_scale[row] = pow2(e);
  }
  if (row >= (rows + 127) / 128 * 128) return;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int vec = first + i * step;
    if (vec - lane >= tiles * (Format<FMT>::kGroup / 4)) break;  // the whole warp is past the padding
    store16<FMT>(raw[i], mul, row, vec, real ? vecs : 0, tiles, codes, scales);
  }
}

// One thread per 16 columns: the values of their codes.
template <int FMT>
__global__ void __launch_bounds__(256) fp4_dequantize_kernel(const uint8_t* __restrict__ codes,
                                                             const uint8_t* __restrict__ scales,
                                                             const float* __restrict__ row_scale,
                                                             bf16* __restrict__ out, int rows, int vecs, int tiles) {
  pdl_wait();
  const size_t total = static_cast<size_t>(rows) * vecs;
  for (size_t i = blockIdx.x * static_cast<size_t>(blockDim.x) + threadIdx.x; i < total;
       i += static_cast<size_t>(gridDim.x) * blockDim.x) {
    const int row = static_cast<int>(total <= 0xffffffffu ? static_cast<uint32_t>(i) / static_cast<uint32_t>(vecs) : i / vecs);
    const int vec = static_cast<int>(i - static_cast<size_t>(row) * vecs);
    const uint2 c = *reinterpret_cast<const uint2*>(codes + i * 8);
    const int group = vec / (Format<FMT>::kGroup / 16);
    float s = scale_value<FMT>(scales[scale_word(row, group >> 2, tiles) + (group & 3)]);
    if constexpr (FMT == kNv) s *= row_scale[row];
    uint32_t v[8];
    values8(c.x, s, v);
    values8(c.y, s, v + 4);
    store32(out + i * 16, v);
  }
}

template <int FMT>
int run_quantize(const void* x, size_t x_stride, uint8_t* codes, uint8_t* scales, float* row_scale, int rows, int K,
                 bool pad, bool early, int sms, cudaStream_t stream) {
  const int vecs = K / 16, tiles = fp4_scale_tiles(FMT, K);
  // few rows: as many warps as there are vectors, for the shortest chain; many: four vectors a lane and several teams a
  // block (more loads in flight per barrier)
  const int all = (tiles * (Format<FMT>::kGroup / 4) + 31) / 32;
  const bool many = rows >= 4 * sms;
  int warps = std::min(32, std::max(1, many ? (all + 3) / 4 : all));
  if (warps <= 8) {
    int p = 1;
    while (p < warps) p *= 2;
    warps = p;
  }
  const int nv = (all + warps - 1) / warps;
  const int teams = warps < 8 && many ? 8 / warps : 1;
  const int last = pad ? (rows + 127) / 128 * 128 : rows;
  const dim3 grid((last + teams - 1) / teams), block(32 * warps * teams);
  auto go = [&](auto kernel) {
    return launch_pdl(kernel, grid, block, 0, stream, static_cast<const bf16*>(x), x_stride, codes, scales, row_scale,
                      rows, vecs, tiles, warps, early) == cudaSuccess ? 0 : -1;
  };
  if (nv <= 1) return go(fp4_quantize_kernel<FMT, 1>);
  if (nv <= 2) return go(fp4_quantize_kernel<FMT, 2>);
  if (nv <= 4) return go(fp4_quantize_kernel<FMT, 4>);
  return -1;
}

}  // namespace

int fp4_scale_tiles(int fmt, int K) {
  return (K + kBlockK - 1) / kBlockK * (fmt == kNv ? Format<kNv>::kTilesPerBlock : Format<kMx>::kTilesPerBlock);
}

int launch_fp4_quantize(const void* x, size_t x_stride, int fmt, void* codes, void* scales, float* row_scale, int rows,
                        int K, bool pad, bool early, int sms, cudaStream_t stream) {
  if (K % 32 != 0 || K < 32 || K > kFp4MaxK || rows < 1) return -1;
  auto* c = static_cast<uint8_t*>(codes);
  auto* s = static_cast<uint8_t*>(scales);
  return fmt == kNv ? run_quantize<kNv>(x, x_stride, c, s, row_scale, rows, K, pad, early, sms, stream)
                    : run_quantize<kMx>(x, x_stride, c, s, row_scale, rows, K, pad, early, sms, stream);
}

int launch_fp4_dequantize(const void* codes, const void* scales, const float* row_scale, int fmt, void* out, int rows,
                          int K, int sms, cudaStream_t stream) {
  if (K % 32 != 0 || rows < 1) return -1;
  const int vecs = K / 16, tiles = fp4_scale_tiles(fmt, K);
  const size_t total = static_cast<size_t>(rows) * vecs;
  const dim3 grid(static_cast<unsigned>(std::min<size_t>((total + 255) / 256, static_cast<size_t>(sms) * 32)));
  auto kernel = fmt == kNv ? fp4_dequantize_kernel<kNv> : fp4_dequantize_kernel<kMx>;
  return launch_pdl(kernel, grid, dim3(256), 0, stream, static_cast<const uint8_t*>(codes),
                    static_cast<const uint8_t*>(scales), row_scale, static_cast<bf16*>(out), rows, vecs, tiles) ==
                 cudaSuccess ? 0 : -1;
}

}  // namespace ecz
