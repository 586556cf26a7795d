// The 4-bit product for hundreds to thousands of rows (gemm_fp4.cu serves fewer): a cluster of two CTAs computes a tile of
// 256 rows x 256 or 384 output features with cta_group::2 MMAs; a CTA holds 128 rows of activations and half of the
// tile's weight rows in shared memory, and the scales of its rows and of all the tile's features (every CTA's tensor
// memory holds the scales of both operands for its half).
//
// What bounds it is bringing the operands in: per K block of 256 columns a CTA of a 256-wide tile loads 38 KB for 128 x 256
// x 256 products, 512 cycles at the tensor cores' nominal rate. Loads alone took 690 cycles (16 TB/s from L2 to all SMs),
// MMAs alone 590, both 810. A 384-wide tile loads 48 KB for half as many products again. Its sums are two accumulators of
// 256 and 128 columns; with the scales' places they fill tensor memory, so neither width has room for a second tile: the
// epilogue first brings its columns to registers, scaled and rounded to bf16, gives the accumulators back, and stores
// under the next tile's MMAs.
//
//   warp 0      TMA producer of the codes (both CTAs; completion counted on the even CTA's barrier)
//   warp 1      even CTA: copies a block's scales to tensor memory of both CTAs, issues its MMAs of 64 columns
//   warps 2-9   epilogue: warp w holds TMEM lanes 32 (w % 4) .. + 31 (rows) and half of each accumulator's columns
//   warp 10     TMA producer of the scales (both CTAs)
//
// The grid is persistent over tiles, in strips of kStrip row tiles so that the tiles in flight share operands in L2. Every
// wait is bounded (common.cuh).
#include <algorithm>
#include <type_traits>

#include "fp4_common.cuh"
#include "gemm_pair.cuh"
#include "launchers.h"

namespace ecz {

namespace {

using namespace fp4;

constexpr int kTileM = 256, kHalf = 128;
constexpr int kABytes = kHalf * kBlockK / 2;  // 128 rows of codes
constexpr int kThreads = 352;
constexpr int kEpiWarps = 8;
constexpr int kScaleWarp = 2 + kEpiWarps;
constexpr int kPatchStride = 80;  // bytes per row of an epilogue warp's [32 rows, 32 bf16] patch
constexpr int kStrip = 8;

template <int FMT, bool WIDE>
struct PairCfg {
  static constexpr int kTileN = WIDE ? 384 : 256;
  static constexpr int kBBytes = kTileN / 2 * kBlockK / 2;
  static constexpr int kScaleBytes = Format<FMT>::kBlockBytes;  // of 128 rows
  static constexpr int kScaleTiles = 1 + kTileN / 128;          // of A and of B
  static constexpr int kStageBytes = kABytes + kBBytes + kScaleTiles * kScaleBytes;
  static constexpr int kStages = WIDE ? 4 : 5;
  static constexpr int kWarpCols = kTileN / 2;                  // of an epilogue warp
  static constexpr int kPatchBytes = 32 * kPatchStride + kWarpCols * 4;
  static constexpr int kSmem = kStages * kStageBytes + kEpiWarps * kPatchBytes + 1024 + 256;
  static constexpr int kSlotCols = kScaleTiles * 4 * Format<FMT>::kTilesPerBlock;
  static constexpr int kSlots = WIDE && FMT == kNv ? 2 : kStages;  // places for scales in tensor memory
  static_assert(kSmem <= 232448, "227 KB of shared memory");
  static_assert(kTileN + kSlots * kSlotCols <= 512, "tensor memory");
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

// Whether the phase has completed, without waiting.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok)
               : "r"(smem_u32(bar)), "r"(parity)
               : "memory");
  return ok != 0;
}

template <int TILE_N>
struct Tiles {
  int m_tiles, n_tiles, total;
  __device__ __forceinline__ Tiles(int M, int N)
      : m_tiles((M + kTileM - 1) / kTileM), n_tiles((N + TILE_N - 1) / TILE_N), total(m_tiles * n_tiles) {}
  // strips of kStrip row tiles; within a strip the rows vary fastest
  __device__ __forceinline__ void at(int t, int& m0, int& n0) const {
    const int strip = t / (kStrip * n_tiles), first = strip * kStrip, height = min(kStrip, m_tiles - first);
    const int in = t - strip * kStrip * n_tiles;
    m0 = (first + in % height) * kTileM;
    n0 = in / height * TILE_N;
  }
};

template <int FMT, bool WIDE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    gemm_fp4_pair_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                         const __grid_constant__ CUtensorMap tm_w64, const __grid_constant__ CUtensorMap tm_sx,
                         const __grid_constant__ CUtensorMap tm_sw, const __grid_constant__ PairArgs args) {
  using C = PairCfg<FMT, WIDE>;
  constexpr int S = C::kStages, kAccs = WIDE ? 2 : 1;
  constexpr int kT = Format<FMT>::kTilesPerBlock;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* scales = smem + S * (kABytes + C::kBBytes);
  uint8_t* patches = smem + S * C::kStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(patches + kEpiWarps * C::kPatchBytes);
  uint64_t* empty = full + S;
  uint64_t* acc_full = empty + S;       // [kAccs]
  uint64_t* acc_empty = acc_full + 2;   // [kAccs]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = packed::uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < kAccs; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 2 * kEpiWarps);
    }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_w);
    if (WIDE) tma_prefetch_desc(&tm_w64);
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

  const Tiles<C::kTileN> tiles(args.M, args.N);
  const int pairs = gridDim.x >> 1, pair_id = blockIdx.x >> 1;
  if ((warp == 0 || warp == kScaleWarp) && lane == 0) {
    // ---- producers: one of the codes, one of the scales (a thread takes 70 cycles to issue a copy) ----
    const bool codes = warp == 0;
    const uint32_t base = codes ? smem_u32(smem) : smem_u32(scales);
    const uint32_t step = codes ? kABytes + C::kBBytes : C::kScaleTiles * C::kScaleBytes;
    const uint32_t bars = pair::mapa_u32(smem_u32(full), 0);
    constexpr int kRows = C::kScaleBytes / 128;  // of 128 bytes, per K block and 128 rows of scales
    uint32_t s = 0, turn = 1;
    bool ok = true;
    for (int t = pair_id; ok && t < tiles.total; t += pairs) {
      int m0, n0;
      tiles.at(t, m0, n0);
      const int m = m0 + static_cast<int>(rank) * kHalf;
      // of the first 256 weight rows this CTA's 128, of the other 128 its 64
      const int n = n0 + static_cast<int>(rank) * kHalf, far = n0 + 256 + static_cast<int>(rank) * 64;
      int sx = (m / kHalf) * args.kblocks * kRows, sw = (n0 / kHalf) * args.kblocks * kRows, k = 0;
      for (int kb = 0; kb < args.kblocks; ++kb) {
        if (!mbar_wait(&empty[s], turn, args.status, kStatusWaitEmpty, abort_flag)) {
          ok = false;
          break;
        }
        const uint32_t bar = bars + s * 8, to = base + s * step;
        if (codes) {
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * C::kStageBytes);
          pair::tma_load_pair(to, &tm_x, bar, k, m);
          pair::tma_load_pair(to + kABytes, &tm_w, bar, k, n);
          if (WIDE) pair::tma_load_pair(to + 2 * kABytes, &tm_w64, bar, k, far);
          k += kBlockK / 2;
        } else {
          pair::tma_load_pair(to, &tm_sx, bar, 0, sx);
#pragma unroll
          for (int i = 0; i < C::kTileN / 128; ++i)
            pair::tma_load_pair(to + (1 + i) * C::kScaleBytes, &tm_sw, bar, 0, sw + i * args.kblocks * kRows);
          sx += kRows;
          sw += kRows;
        }
        if (++s == S) {
          s = 0;
          turn ^= 1u;
        }
      }
    }
    if (!ok) {  // copies in flight get time to land
      const unsigned long long t0 = global_timer_ns();
      while (global_timer_ns() - t0 < 1000000ull) {
      }
    }
  } else if (warp == 1 && rank == 0) {
    // ---- MMA issuer: the whole warp walks, one lane issues, from descriptors in uniform registers ----
    // Its instructions one after another have to take less than the MMAs (590 cycles a block of a 256-wide tile): with a
    // wait for the scales' place, a wait for the stage and two warp synchronisations they took 760.
    const uint32_t base = smem_u32(smem);
    const uint64_t a0 = desc_kmajor_sw128(base), b0 = desc_kmajor_sw128(base + kABytes);
    const uint64_t s0 = desc_scales(smem_u32(scales));
    const bool leader = packed::elect_one();
    constexpr int kBTiles = C::kTileN / 128;
    uint32_t tile = 0, s = 0, turn = 0;        // stage and its phase
    uint32_t slot = 0, old = 0, old_turn = 0;  // place of the scales; the stage whose MMAs read that place last
    int filled = 0;                            // places that have been used
    bool ok = true, ready = false;
    for (int t = pair_id; ok && t < tiles.total; t += pairs, ++tile) {
      for (int kb = 0; kb < args.kblocks; ++kb) {
        if (kb == 0) {
          ok = packed::warp_wait(&acc_empty[0], (tile & 1u) ^ 1u, args.status, kStatusWaitAccum, abort_flag);
          if (!ok) break;
        }
        if constexpr (C::kSlots < S) {
          if (filled == C::kSlots) {  // the MMAs that read this place's last scales have completed
            ok = packed::warp_wait(&empty[old], old_turn, args.status, kStatusWaitEmpty, abort_flag);
            if (!ok) break;
            if (++old == S) {
              old = 0;
              old_turn ^= 1u;
            }
          } else {
            ++filled;
          }
        }  // with a place per stage the stage itself was waited for, by the producer, before it was filled again
        if (!__all_sync(0xffffffffu, ready)) {
          ok = packed::warp_wait(&full[s], turn, args.status, kStatusWaitFull, abort_flag);
          if (!ok) break;
        }
        tc_fence_after();
        const uint32_t next = s + 1 == S ? 0 : s + 1;
        ready = mbar_test(&full[next], next == 0 ? turn ^ 1u : turn);  // asked while the block is issued
        const uint32_t sfa = tmem + C::kTileN + slot * C::kSlotCols, sfb = sfa + 4 * kT;
        const uint64_t a = packed::desc_step(a0, s * (kABytes + C::kBBytes));
        const uint64_t b = packed::desc_step(b0, s * (kABytes + C::kBBytes));
        auto multiply = [&](auto which) {
          constexpr int acc = decltype(which)::value, kCols = acc == 0 ? 256 : 128;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const int i = FMT == kNv ? kk : kk / 2;
            const uint32_t idesc =
                FMT == kNv ? idesc_fp4<FMT>(kTileM, kCols) : idesc_fp4<FMT>(kTileM, kCols, (kk & 1) * 2);
            umma_fp4_pair<FMT>(tmem + acc * 256, packed::desc_step(a, kk * 32), packed::desc_step(b, acc * kABytes + kk * 32),
                               idesc, sfa + 4 * i, sfb + 4 * (kBTiles * i + 2 * acc), (kb | kk) != 0 ? 1u : 0u);
          }
          if (kb == args.kblocks - 1) pair::commit_pair(&acc_full[acc]);
        };
        if (leader) {
          const uint64_t sd = packed::desc_step(s0, s * C::kScaleTiles * C::kScaleBytes);
          // the scales of B's 128-row tiles lie four columns behind one another
#pragma unroll
          for (int i = 0; i < kT; ++i) {
            copy_scales_pair(sfa + 4 * i, packed::desc_step(sd, i * kTileBytes));
#pragma unroll
            for (int j = 0; j < kBTiles; ++j)
              copy_scales_pair(sfb + 4 * (kBTiles * i + j), packed::desc_step(sd, (1 + j) * C::kScaleBytes + i * kTileBytes));
          }
          multiply(std::integral_constant<int, 0>{});
        }
        if constexpr (WIDE) {
          if (kb == 0) {
            __syncwarp();
            ok = packed::warp_wait(&acc_empty[1], (tile & 1u) ^ 1u, args.status, kStatusWaitAccum, abort_flag);
            if (!ok) break;
            tc_fence_after();
          }
          if (leader) multiply(std::integral_constant<int, 1>{});
        }
        if (leader) pair::commit_pair(&empty[s]);
        if (next == 0) turn ^= 1u;
        s = next;
        slot = slot + 1 == C::kSlots ? 0 : slot + 1;
      }
    }
    __syncwarp();
  } else if (warp >= 2 && warp < kScaleWarp) {
    // ---- epilogue ----
    const int ew = warp - 2, quad = warp & 3, half = ew >> 2;
    uint8_t* patch = patches + ew * C::kPatchBytes;
    float* features = reinterpret_cast<float*>(patch + 32 * kPatchStride);  // row scales of this warp's features
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const bool whole_rows = args.N % 8 == 0;  // 16-byte rows of y
    uint32_t tile = 0;
    for (int t = pair_id; t < tiles.total; t += pairs, ++tile) {
      int m0, n0;
      tiles.at(t, m0, n0);
      const int row0 = m0 + static_cast<int>(rank) * kHalf + quad * 32;
      // this warp's columns in groups of 32: four of the first accumulator, two of the second
      auto column = [&](int g) { return g < 4 ? half * 128 + g * 32 : 256 + half * 64 + (g - 4) * 32; };
      constexpr int kGroups = C::kWarpCols / 32;
      float rx = 1.f;
      if constexpr (FMT == kNv) {  // the rows' powers of two, at hand before the sums are
        if (row0 + lane < args.M) rx = args.x_row[row0 + lane];
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          const int n = n0 + column(g) + lane;
          features[g * 32 + lane] = n < args.N ? args.w_row[n] : 1.f;
        }
        __syncwarp();
      }
      uint32_t out[kGroups * 16];
      auto drain = [&](auto which) {
        constexpr int acc = decltype(which)::value;
        const bool ok = mbar_wait(&acc_full[acc], tile & 1u, args.status, kStatusWaitAccum, abort_flag);
        if (__any_sync(0xffffffffu, !ok)) return false;
        tc_fence_after();
#pragma unroll
        for (int i = 0; i < (acc == 0 ? 4 : 2); ++i) {
          const int g = acc * 4 + i;
          float v[32];
          tmem_ld32(lanes + column(g), v);
          if constexpr (FMT == kNv) {
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              const float4 w = *reinterpret_cast<const float4*>(features + g * 32 + j);
              v[j] *= rx * w.x;
              v[j + 1] *= rx * w.y;
              v[j + 2] *= rx * w.z;
              v[j + 3] *= rx * w.w;
            }
          }
#pragma unroll
          for (int j = 0; j < 32; j += 2) out[g * 16 + j / 2] = packed::pack_bf16(v[j], v[j + 1]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) pair::arrive_cluster(pair::mapa_u32(smem_u32(&acc_empty[acc]), 0));
        return true;
      };
      if (!drain(std::integral_constant<int, 0>{})) break;
      if constexpr (WIDE) {
        if (!drain(std::integral_constant<int, 1>{})) break;
      }
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        // a lane's 32 columns into its row of the patch, then rows out in 64-byte pieces
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<uint4*>(patch + lane * kPatchStride + j * 16) =
              make_uint4(out[g * 16 + 4 * j], out[g * 16 + 4 * j + 1], out[g * 16 + 4 * j + 2], out[g * 16 + 4 * j + 3]);
        __syncwarp();
        const int n = n0 + column(g);
        if (whole_rows) {
          const int c = (lane & 3) * 8;
          if (n + c < args.N) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = i * 8 + (lane >> 2);
              if (row0 + r < args.M)
                *reinterpret_cast<uint4*>(args.y + static_cast<size_t>(row0 + r) * args.N + n + c) =
                    *reinterpret_cast<const uint4*>(patch + r * kPatchStride + c * 2);
            }
          }
        } else if (n + lane < args.N) {
          for (int r = 0; r < 32 && row0 + r < args.M; ++r)
            args.y[static_cast<size_t>(row0 + r) * args.N + n + lane] =
                *reinterpret_cast<const bf16*>(patch + r * kPatchStride + lane * 2);
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

long tiles_of(int M, int N, int tile_n) {
  return static_cast<long>((M + kTileM - 1) / kTileM) * ((N + tile_n - 1) / tile_n);
}

template <int FMT, bool WIDE>
int run(const Fp4PairMaps& maps, const PairArgs& args, int sms, cudaStream_t stream) {
  using C = PairCfg<FMT, WIDE>;
  const long tiles = tiles_of(args.M, args.N, C::kTileN);
  auto kernel = gemm_fp4_pair_kernel<FMT, WIDE>;
  if (tiles > (1 << 30) || set_max_smem(kernel, C::kSmem) != cudaSuccess) return -1;
  const int pairs = static_cast<int>(std::min<long>(tiles, sms / 2));
  return launch_pdl(kernel, dim3(2 * pairs), dim3(kThreads), C::kSmem, stream, maps.x, maps.w, maps.w64, maps.sx, maps.sw,
                    args) == cudaSuccess ? 0 : -1;
}

}  // namespace

int launch_gemm_fp4_pair(const Fp4PairMaps& maps, const float* x_row, const float* w_row, int fmt, void* y, int M, int N,
                         int K, int width, int sms, unsigned* status, cudaStream_t stream) {
  if (M < 1 || N < 1 || K < 32 || K % 32 != 0 || K > kFp4MaxK) return -1;
  PairArgs args{};
  args.x_row = x_row;
  args.w_row = w_row;
  args.y = static_cast<bf16*>(y);
  args.M = M;
  args.N = N;
  args.kblocks = (K + kBlockK - 1) / kBlockK;
  args.status = status;
  // A round of 384-wide tiles takes as long as 1.2 of 256-wide ones: whichever needs less in whole rounds.
  const long pairs = sms / 2;
  const long narrow_rounds = (tiles_of(M, N, 256) + pairs - 1) / pairs, wide_rounds = (tiles_of(M, N, 384) + pairs - 1) / pairs;
  const bool wide = width == 384 || (width == 0 && 6 * wide_rounds < 5 * narrow_rounds);
  if (fmt == kNv)
    return wide ? run<kNv, true>(maps, args, sms, stream) : run<kNv, false>(maps, args, sms, stream);
  return wide ? run<kMx, true>(maps, args, sms, stream) : run<kMx, false>(maps, args, sms, stream);
}

}  // namespace ecz
