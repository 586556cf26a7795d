// The 4-bit product for hundreds to thousands of rows (gemm_fp4.cu serves fewer): a cluster of two CTAs computes a tile of
// 256 rows x 256 output features with cta_group::2 MMAs, 128 rows of activations and 128 of the 256 weight rows in either
// CTA's shared memory. Per K block of 256 columns a CTA loads 32 KB of codes, its rows' scales and all 256 features'
// (every CTA's tensor memory holds the scales of both operands for its half), and computes 128 x 256 x 256 products in
// 512 cycles at the tensor cores' nominal rate: 64 + 12 bytes a cycle from L2, where a tile of one CTA would need 96 + 12.
//
//   warp 0      TMA producer (both CTAs; completion counted on the even CTA's barrier)
//   warp 1      even CTA: copies a block's scales to tensor memory of both CTAs, issues its four MMAs of 64 columns
//   warps 2-9   epilogue: warp w holds TMEM lanes 32 (w % 4) .. + 31 (rows) and 128 of the 256 columns
//
// The accumulators take 256 of the 512 TMEM columns and the scales' places 3 x 48, so there is no room for a second tile:
// the epilogue first brings its columns to registers, scaled and rounded to bf16, gives the accumulators back, and stores
// under the next tile's MMAs. The grid is persistent over tiles, in strips of kStrip row tiles so that the tiles in flight
// share operands in L2. Every wait is bounded (common.cuh).
#include <algorithm>

#include "fp4_common.cuh"
#include "gemm_pair.cuh"
#include "launchers.h"

namespace ecz {

namespace {

using namespace fp4;

constexpr int kTile = 256, kHalf = 128;
constexpr int kOperandBytes = kHalf * kBlockK / 2;
constexpr int kThreads = 320;
constexpr int kEpiWarps = 8;
constexpr int kPatchStride = 144;  // bytes per row of an epilogue warp's [32 rows, 64 bf16] patch
constexpr int kPatchBytes = 32 * kPatchStride + 512;
constexpr int kSlots = 3;  // places for scales in tensor memory
constexpr int kStrip = 8;

template <int FMT>
struct PairCfg {
  static constexpr int kScaleBytes = Format<FMT>::kBlockBytes;              // of 128 rows
  static constexpr int kStageBytes = 2 * kOperandBytes + 3 * kScaleBytes;
  static constexpr int kStages = 4;
  static constexpr int kSmem = kStages * kStageBytes + kEpiWarps * kPatchBytes + 1024 + 256;
  static constexpr int kSlotCols = 3 * 4 * Format<FMT>::kTilesPerBlock;     // 128 rows of A, 256 of B
  static_assert(kSmem <= 232448, "227 KB of shared memory");
  static_assert(kTile + kSlots * kSlotCols <= 512, "tensor memory");
  static_assert(kStages >= kSlots, "a slot of scales is waited for by its stage's barrier");
};

struct PairArgs {
  const float* w_row;  // nvfp4
  const float* x_row;
  bf16* y;
  int M, N, kblocks;
  unsigned* status;
};

template <int FMT>
__device__ __forceinline__ void umma_fp4_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa,
                                              uint32_t sfb, uint32_t accumulate) {
  if constexpr (FMT == kNv) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  }
}

// In both CTAs: 512 bytes of scales of its shared memory to four columns of its tensor memory.
__device__ __forceinline__ void copy_scales_pair(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

struct Tiles {
  int m_tiles, n_tiles, total;
  __device__ __forceinline__ Tiles(int M, int N)
      : m_tiles((M + kTile - 1) / kTile), n_tiles((N + kTile - 1) / kTile), total(m_tiles * n_tiles) {}
  // strips of kStrip row tiles; within a strip the rows vary fastest
  __device__ __forceinline__ void at(int t, int& m0, int& n0) const {
    const int strip = t / (kStrip * n_tiles), first = strip * kStrip, height = min(kStrip, m_tiles - first);
    const int in = t - strip * kStrip * n_tiles;
    m0 = (first + in % height) * kTile;
    n0 = in / height * kTile;
  }
};

template <int FMT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    gemm_fp4_pair_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                         const __grid_constant__ CUtensorMap tm_sx, const __grid_constant__ CUtensorMap tm_sw,
                         const __grid_constant__ PairArgs args) {
  using C = PairCfg<FMT>;
  constexpr int S = C::kStages;
  constexpr int kT = Format<FMT>::kTilesPerBlock;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* scales = smem + S * 2 * kOperandBytes;
  uint8_t* patches = smem + S * C::kStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(patches + kEpiWarps * kPatchBytes);
  uint64_t* empty = full + S;
  uint64_t* acc_full = empty + S;
  uint64_t* acc_empty = acc_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = packed::uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, 2 * kEpiWarps);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_w);
    tma_prefetch_desc(&tm_sx);
    tma_prefetch_desc(&tm_sw);
  }
  __syncwarp();
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the peer's barriers are initialised before anything is counted on them
  tc_fence_after();
  const uint32_t tmem = packed::uniform(*tmem_slot);
  pdl_trigger();
  pdl_wait();

  const Tiles tiles(args.M, args.N);
  const int pairs = gridDim.x >> 1, pair_id = blockIdx.x >> 1;
  if (warp == 0 && lane == 0) {
    // ---- producer ----
    const uint32_t base = smem_u32(smem), sbase = smem_u32(scales);
    uint32_t it = 0;
    bool ok = true;
    for (int t = pair_id; ok && t < tiles.total; t += pairs) {
      int m0, n0;
      tiles.at(t, m0, n0);
      const int m = m0 + static_cast<int>(rank) * kHalf, n = n0 + static_cast<int>(rank) * kHalf;
      constexpr int kRows = C::kScaleBytes / 128;  // of 128 bytes, per K block and 128 rows of scales
      const int sx = (m / kHalf) * args.kblocks * kRows, sw = (n0 / kHalf) * args.kblocks * kRows;
      for (int kb = 0; kb < args.kblocks; ++kb, ++it) {
        const int s = it % S;
        if (!mbar_wait(&empty[s], ((it / S) & 1u) ^ 1u, args.status, kStatusWaitEmpty, abort_flag)) {
          ok = false;
          break;
        }
        const uint32_t bar = pair::mapa_u32(smem_u32(&full[s]), 0);
        if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * C::kStageBytes);
        const uint32_t dst = base + s * 2 * kOperandBytes, sdst = sbase + s * 3 * C::kScaleBytes;
        pair::tma_load_pair(dst, &tm_x, bar, kb * (kBlockK / 2), m);
        pair::tma_load_pair(dst + kOperandBytes, &tm_w, bar, kb * (kBlockK / 2), n);
        pair::tma_load_pair(sdst, &tm_sx, bar, 0, sx + kb * kRows);
        pair::tma_load_pair(sdst + C::kScaleBytes, &tm_sw, bar, 0, sw + kb * kRows);
        pair::tma_load_pair(sdst + 2 * C::kScaleBytes, &tm_sw, bar, 0, sw + (args.kblocks + kb) * kRows);
      }
    }
    if (!ok) {  // copies in flight get time to land
      const unsigned long long t0 = global_timer_ns();
      while (global_timer_ns() - t0 < 1000000ull) {
      }
    }
  } else if (warp == 1 && rank == 0) {
    // ---- MMA issuer: the whole warp walks, one lane issues, from descriptors in uniform registers ----
    const uint32_t base = smem_u32(smem);
    const uint64_t a0 = desc_kmajor_sw128(base), b0 = desc_kmajor_sw128(base + kOperandBytes);
    const uint64_t s0 = desc_scales(smem_u32(scales));
    const bool leader = packed::elect_one();
    uint32_t tile = 0, it = 0;
    bool ok = true;
    for (int t = pair_id; ok && t < tiles.total; t += pairs, ++tile) {
      ok = packed::warp_wait(acc_empty, (tile & 1u) ^ 1u, args.status, kStatusWaitAccum, abort_flag);
      if (!ok) break;
      tc_fence_after();
      for (int kb = 0; kb < args.kblocks; ++kb, ++it) {
        const uint32_t s = it % S;
        if (it >= kSlots) {  // the MMAs that read this slot's last scales have completed
          const uint32_t old = it - kSlots;
          ok = packed::warp_wait(&empty[old % S], (old / S) & 1u, args.status, kStatusWaitEmpty, abort_flag);
          if (!ok) break;
        }
        ok = packed::warp_wait(&full[s], (it / S) & 1u, args.status, kStatusWaitFull, abort_flag);
        if (!ok) break;
        tc_fence_after();
        if (leader) {
          const uint32_t sfa = tmem + kTile + (it % kSlots) * C::kSlotCols, sfb = sfa + 4 * kT;
          const uint64_t a = packed::desc_step(a0, s * 2 * kOperandBytes), b = packed::desc_step(b0, s * 2 * kOperandBytes);
          const uint64_t sd = packed::desc_step(s0, s * 3 * C::kScaleBytes);
          // B's scales of rows 128 .. 255 lie four columns behind those of rows 0 .. 127
#pragma unroll
          for (int i = 0; i < kT; ++i) {
            copy_scales_pair(sfa + 4 * i, packed::desc_step(sd, i * kTileBytes));
            copy_scales_pair(sfb + 8 * i, packed::desc_step(sd, C::kScaleBytes + i * kTileBytes));
            copy_scales_pair(sfb + 8 * i + 4, packed::desc_step(sd, 2 * C::kScaleBytes + i * kTileBytes));
          }
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const int i = FMT == kNv ? kk : kk / 2;
            const uint32_t idesc =
                FMT == kNv ? idesc_fp4<FMT>(kTile, kTile) : idesc_fp4<FMT>(kTile, kTile, (kk & 1) * 2);
            umma_fp4_pair<FMT>(tmem, packed::desc_step(a, kk * 32), packed::desc_step(b, kk * 32), idesc, sfa + 4 * i,
                               sfb + 8 * i, (kb | kk) != 0 ? 1u : 0u);
          }
          pair::commit_pair(&empty[s]);
        }
        __syncwarp();
      }
      if (leader) pair::commit_pair(acc_full);
      __syncwarp();
    }
  } else if (warp >= 2) {
    // ---- epilogue ----
    const int ew = warp - 2, quad = warp & 3, half = ew >> 2;
    uint8_t* patch = patches + ew * kPatchBytes;
    float* features = reinterpret_cast<float*>(patch + 32 * kPatchStride);  // row scales of this warp's 128 features
    const uint32_t taddr = tmem + (static_cast<uint32_t>(quad * 32) << 16) + half * 128u;
    const bool wide = args.N % 8 == 0;  // 16-byte rows of y
    uint32_t tile = 0;
    for (int t = pair_id; t < tiles.total; t += pairs, ++tile) {
      int m0, n0;
      tiles.at(t, m0, n0);
      const int row0 = m0 + static_cast<int>(rank) * kHalf + quad * 32, col0 = n0 + half * 128;
      float rx = 1.f;
      if constexpr (FMT == kNv) {  // the rows' powers of two, at hand before the sums are
        if (row0 + lane < args.M) rx = args.x_row[row0 + lane];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int n = col0 + i * 32 + lane;
          features[i * 32 + lane] = n < args.N ? args.w_row[n] : 1.f;
        }
        __syncwarp();
      }
      const bool ok = mbar_wait(acc_full, tile & 1u, args.status, kStatusWaitAccum, abort_flag);
      if (__any_sync(0xffffffffu, !ok)) break;
      tc_fence_after();
      uint32_t out[64];
#pragma unroll
      for (int c = 0; c < 128; c += 32) {
        float v[32];
        tmem_ld32(taddr + c, v);
        if constexpr (FMT == kNv) {
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 w = *reinterpret_cast<const float4*>(features + c + j);
            v[j] *= rx * w.x;
            v[j + 1] *= rx * w.y;
            v[j + 2] *= rx * w.z;
            v[j + 3] *= rx * w.w;
          }
        }
#pragma unroll
        for (int j = 0; j < 32; j += 2) out[(c + j) / 2] = packed::pack_bf16(v[j], v[j + 1]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) pair::arrive_cluster(pair::mapa_u32(smem_u32(acc_empty), 0));
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        // a lane's 64 columns into its row of the patch, then rows out in whole 128-byte lines
#pragma unroll
        for (int j = 0; j < 8; ++j)
          *reinterpret_cast<uint4*>(patch + lane * kPatchStride + j * 16) =
              make_uint4(out[p * 32 + 4 * j], out[p * 32 + 4 * j + 1], out[p * 32 + 4 * j + 2], out[p * 32 + 4 * j + 3]);
        __syncwarp();
        const int n = col0 + p * 64;
        if (wide) {
          const int c = (lane & 7) * 8;
          for (int r = lane >> 3; r < 32 && row0 + r < args.M; r += 4)
            if (n + c < args.N)
              *reinterpret_cast<uint4*>(args.y + static_cast<size_t>(row0 + r) * args.N + n + c) =
                  *reinterpret_cast<const uint4*>(patch + r * kPatchStride + c * 2);
        } else {
          for (int r = 0; r < 32 && row0 + r < args.M; ++r)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int c = h * 32 + lane;
              if (n + c < args.N)
                args.y[static_cast<size_t>(row0 + r) * args.N + n + c] =
                    *reinterpret_cast<const bf16*>(patch + r * kPatchStride + c * 2);
            }
        }
        __syncwarp();
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs are done with each other's barriers and with the accumulators
  tc_fence_after();
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

template <int FMT>
int run(const CUtensorMap* x, const CUtensorMap* w, const CUtensorMap* sx, const CUtensorMap* sw, const PairArgs& args,
        int sms, cudaStream_t stream) {
  const long tiles = static_cast<long>((args.M + kTile - 1) / kTile) * ((args.N + kTile - 1) / kTile);
  auto kernel = gemm_fp4_pair_kernel<FMT>;
  if (tiles > (1 << 30) || set_max_smem(kernel, PairCfg<FMT>::kSmem) != cudaSuccess) return -1;
  const int pairs = static_cast<int>(std::min<long>(tiles, sms / 2));
  return launch_pdl(kernel, dim3(2 * pairs), dim3(kThreads), PairCfg<FMT>::kSmem, stream, *x, *w, *sx, *sw, args) ==
                 cudaSuccess ? 0 : -1;
}

}  // namespace

int launch_gemm_fp4_pair(const CUtensorMap* x, const CUtensorMap* w, const CUtensorMap* sx, const CUtensorMap* sw,
                         const float* x_row, const float* w_row, int fmt, void* y, int M, int N, int K, int sms,
                         unsigned* status, cudaStream_t stream) {
  if (M < 1 || N < 1 || K < 32 || K % 32 != 0 || K > kFp4MaxK) return -1;
  PairArgs args{};
  args.x_row = x_row;
  args.w_row = w_row;
  args.y = static_cast<bf16*>(y);
  args.M = M;
  args.N = N;
  args.kblocks = (K + kBlockK - 1) / kBlockK;
  args.status = status;
  return fmt == kNv ? run<kNv>(x, w, sx, sw, args, sms, stream) : run<kMx>(x, w, sx, sw, args, sms, stream);
}

}  // namespace ecz
