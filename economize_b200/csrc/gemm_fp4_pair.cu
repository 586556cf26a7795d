// The 4-bit product for hundreds to thousands of rows (gemm_fp4.cu serves fewer): a cluster of two CTAs computes a tile of
// 256 rows x 256 output features with cta_group::2 MMAs, 128 rows of activations and 128 of the 256 weight rows in either
// CTA's shared memory. Per K block of 256 columns a CTA loads 32 KB of codes, its rows' scales and all 256 features'
// (every CTA's tensor memory holds the scales of both operands for its half).
//
//   warp 0      TMA producer of the codes (both CTAs; completion counted on the even CTA's barrier)
//   warp 1      even CTA: copies a block's scales to tensor memory of both CTAs, issues its four MMAs of 64 columns
//   warps 2-9   epilogue: warp w holds TMEM lanes 32 (w % 4) .. + 31 (rows) and 128 of the 256 columns; TMA stores them
//   warp 10     TMA producer of the scales (both CTAs): a thread takes 70 cycles to issue a copy, and the five of a block
//               from one thread took longer than its MMAs
//
// The four MMAs of a block take 590 cycles (512 at the nominal rate), the loads alone 690 from one thread and less from two.
// The accumulators and a place for the scales of every stage fill 496 of 512 TMEM columns; the places being as many as the
// stages, a stage that has been filled again is proof that its place is free. There is no room for a second tile's sums:
// the epilogue brings its columns to registers as they are, gives the accumulators back, and scales, rounds and stores
// under the next tile's MMAs. (Tiles of 384 features, 18% fewer bytes per product, were no faster: the MMAs bound them too,
// and they fill whole rounds of the pairs less often.)
//
// 8192 x 4096 x 28672 takes 386 us in a burst (5.0 PFLOP/s) and 453 at the clock that 1 kW sustains (1.45 GHz); zeros, which
// cost less power, reach 7.1 PFLOP/s.
//
// The grid is persistent over tiles, in strips of kStrip row tiles so that the tiles in flight share operands in L2. Every
// wait is bounded (common.cuh).
#include <algorithm>

#include "fp4_common.cuh"
#include "gemm_pair.cuh"
#include "launchers.h"

namespace ecz {

namespace {

using namespace fp4;

constexpr int kTile = 256, kHalf = 128;
constexpr int kOperandBytes = kHalf * kBlockK / 2;
constexpr int kThreads = 352;
constexpr int kEpiWarps = 8;
constexpr int kScaleWarp = 2 + kEpiWarps;
constexpr int kPatchBytes = 32 * 64;  // [32 rows, 32 bf16], 64-byte swizzle; an epilogue warp has two
constexpr int kEpiBytes = 2 * kPatchBytes + 128 * 2;  // and the row scales of its 128 features
constexpr int kStages = 5;  // and places for scales in tensor memory
constexpr int kStrip = 8;

template <int FMT>
struct PairCfg {
  static constexpr int kScaleBytes = Format<FMT>::kBlockBytes;              // of 128 rows
  static constexpr int kStageBytes = 2 * kOperandBytes + 3 * kScaleBytes;
  static constexpr int kSmem = kStages * kStageBytes + kEpiWarps * kEpiBytes + 1024 + 256;
  static constexpr int kSlotCols = 3 * 4 * Format<FMT>::kTilesPerBlock;     // 128 rows of A, 256 of B
  static_assert(kSmem <= 232448, "227 KB of shared memory");
  static_assert(kTile + kStages * kSlotCols <= 512, "tensor memory");
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
                         const __grid_constant__ CUtensorMap tm_y, const __grid_constant__ PairArgs args) {
  using C = PairCfg<FMT>;
  constexpr int kT = Format<FMT>::kTilesPerBlock;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* scales = smem + kStages * 2 * kOperandBytes;
  uint8_t* patches = smem + kStages * C::kStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(patches + kEpiWarps * kEpiBytes);
  uint64_t* empty = full + kStages;
  uint64_t* acc_full = empty + kStages;
  uint64_t* acc_empty = acc_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = packed::uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
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
    if (args.N % 8 == 0) tma_prefetch_desc(&tm_y);
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
  if ((warp == 0 || warp == kScaleWarp) && lane == 0) {
    // ---- producers ----
    const bool codes = warp == 0;
    const uint32_t base = codes ? smem_u32(smem) : smem_u32(scales);
    const uint32_t step = codes ? 2 * kOperandBytes : 3 * C::kScaleBytes;
    const uint32_t bars = pair::mapa_u32(smem_u32(full), 0);
    constexpr int kRows = C::kScaleBytes / 128;  // of 128 bytes, per K block and 128 rows of scales
    uint32_t s = 0, turn = 1;
    bool ok = true;
    for (int t = pair_id; ok && t < tiles.total; t += pairs) {
      int m0, n0;
      tiles.at(t, m0, n0);
      const int m = m0 + static_cast<int>(rank) * kHalf, n = n0 + static_cast<int>(rank) * kHalf;
      int sx = (m / kHalf) * args.kblocks * kRows, sw = (n0 / kHalf) * args.kblocks * kRows;
      for (int kb = 0; kb < args.kblocks; ++kb) {
        if (!mbar_wait(&empty[s], turn, args.status, kStatusWaitEmpty, abort_flag)) {
          ok = false;
          break;
        }
        const uint32_t bar = bars + s * 8, to = base + s * step;
        if (codes) {
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * C::kStageBytes);
          pair::tma_load_pair(to, &tm_x, bar, kb * (kBlockK / 2), m);
          pair::tma_load_pair(to + kOperandBytes, &tm_w, bar, kb * (kBlockK / 2), n);
        } else {
          pair::tma_load_pair(to, &tm_sx, bar, 0, sx);
          pair::tma_load_pair(to + C::kScaleBytes, &tm_sw, bar, 0, sw);
          pair::tma_load_pair(to + 2 * C::kScaleBytes, &tm_sw, bar, 0, sw + args.kblocks * kRows);
          sx += kRows;
          sw += kRows;
        }
        if (++s == kStages) {
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
    // What it does for a block, one instruction after another, has to take less than the block's MMAs: with a wait for the
    // scales' place and warp synchronisations it took 760 cycles.
    const uint32_t base = smem_u32(smem);
    const uint64_t a0 = desc_kmajor_sw128(base), b0 = desc_kmajor_sw128(base + kOperandBytes);
    const uint64_t s0 = desc_scales(smem_u32(scales));
    const bool leader = packed::elect_one();
    uint32_t tile = 0, s = 0, turn = 0;  // stage (and place of its scales), its phase
    bool ok = true, ready = false;
    for (int t = pair_id; ok && t < tiles.total; t += pairs, ++tile) {
      ok = packed::warp_wait(acc_empty, (tile & 1u) ^ 1u, args.status, kStatusWaitAccum, abort_flag);
      if (!ok) break;
      for (int kb = 0; kb < args.kblocks; ++kb) {
        if (!__all_sync(0xffffffffu, ready)) {
          ok = packed::warp_wait(&full[s], turn, args.status, kStatusWaitFull, abort_flag);
          if (!ok) break;
        }
        tc_fence_after();
        const uint32_t next = s + 1 == kStages ? 0 : s + 1;
        ready = mbar_test(&full[next], next == 0 ? turn ^ 1u : turn);  // asked while the block is issued
        if (leader) {
          const uint32_t sfa = tmem + kTile + s * C::kSlotCols, sfb = sfa + 4 * kT;
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
          if (kb == args.kblocks - 1) pair::commit_pair(acc_full);
        }
        if (next == 0) turn ^= 1u;
        s = next;
      }
    }
    __syncwarp();
  } else if (warp >= 2 && warp < kScaleWarp) {
    // ---- epilogue ----
    const int ew = warp - 2, quad = warp & 3, half = ew >> 2;
    uint8_t* patch = patches + ew * 2 * kPatchBytes;
    bf16* features = reinterpret_cast<bf16*>(patches + kEpiWarps * 2 * kPatchBytes) + ew * 128;
    const uint32_t taddr = tmem + (static_cast<uint32_t>(quad * 32) << 16) + half * 128u;
    const bool whole_rows = args.N % 8 == 0;  // 16-byte rows of y, which TMA stores
    int row0, col0;
    float rx = 1.f, rw[4] = {1.f, 1.f, 1.f, 1.f};  // powers of two of this lane's row and of features 32 i + lane
    auto locate = [&](int t) {
      int m0, n0;
      tiles.at(t, m0, n0);
      row0 = m0 + static_cast<int>(rank) * kHalf + quad * 32;
      col0 = n0 + half * 128;
    };
    auto row_scales = [&]() {
      if constexpr (FMT == kNv) {
        rx = row0 + lane < args.M ? args.x_row[row0 + lane] : 1.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) rw[i] = col0 + i * 32 + lane < args.N ? args.w_row[col0 + i * 32 + lane] : 1.f;
      }
    };
    if (pair_id < tiles.total) {
      locate(pair_id);
      row_scales();
    }
    uint32_t tile = 0;
    for (int t = pair_id; t < tiles.total; t += pairs, ++tile) {
      const RowFactors rf = row_factors(rx);
      const uint64_t rx_first = pair_of(rf.first, rf.first), rx_last = pair_of(rf.last, rf.last);
      if constexpr (FMT == kNv) {
#pragma unroll
        for (int i = 0; i < 4; ++i) features[i * 32 + lane] = __float2bfloat16(rw[i]);
        __syncwarp();
      }
      const bool ok = mbar_wait(acc_full, tile & 1u, args.status, kStatusWaitAccum, abort_flag);
      if (__any_sync(0xffffffffu, !ok)) break;
      tc_fence_after();
      float v[128];
      tmem_load64(taddr, v);
      tmem_load64(taddr + 64, v + 64);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) pair::arrive_cluster(pair::mapa_u32(smem_u32(acc_empty), 0));
      const int row = row0, col = col0;
      if (t + pairs < tiles.total) {  // the next tile's scales are fetched under this one's stores
        locate(t + pairs);
        row_scales();
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        // a lane's 32 columns, times the powers of two and rounded once, into its row of a patch
        uint8_t* to = patch + (g & 1) * kPatchBytes;
        if (whole_rows) {
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
          __syncwarp();
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          __nv_bfloat162 out[4];
          uint4 w = make_uint4(0, 0, 0, 0);
          if constexpr (FMT == kNv) w = *reinterpret_cast<const uint4*>(features + g * 32 + j * 8);
          const uint32_t* w2 = reinterpret_cast<const uint32_t*>(&w);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float lo = v[g * 32 + j * 8 + 2 * i], hi = v[g * 32 + j * 8 + 2 * i + 1];
            if constexpr (FMT == kNv) {
              const uint64_t y = mul2(mul2(pair_of(lo, hi), rx_first), pair_of(low_bf16(w2[i]), high_bf16(w2[i])));
              packed::unpair(mul2(y, rx_last), lo, hi);
            }
            out[i] = __floats2bfloat162_rn(lo, hi);
          }
          *reinterpret_cast<uint4*>(to + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) = *reinterpret_cast<uint4*>(out);
        }
        const int n = col + g * 32;
        if (whole_rows) {
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (row < args.M && n < args.N)
              asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                               reinterpret_cast<uint64_t>(&tm_y)),
                           "r"(n), "r"(row), "r"(smem_u32(to))
                           : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        } else {
          __syncwarp();
          // rows that TMA does not store, a column a lane: eight rows' values first, then their stores
          bf16* out = args.y + static_cast<size_t>(row) * args.N + n + lane;
          const int rows = n + lane < args.N ? args.M - row : 0;
#pragma unroll
          for (int r = 0; r < 32; r += 8) {
            bf16 column[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
              column[i] = *reinterpret_cast<const bf16*>(to + (r + i) * 64 + (((lane >> 3) ^ (((r + i) >> 1) & 3)) << 4) +
                                                         (lane & 7) * 2);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (r + i < rows) out[static_cast<size_t>(r + i) * args.N] = column[i];
          }
          __syncwarp();
        }
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs are done with each other's barriers and with the accumulators
  tc_fence_after();
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

template <int FMT>
int run(const Fp4PairMaps& maps, const PairArgs& args, int sms, cudaStream_t stream) {
  const long tiles = static_cast<long>((args.M + kTile - 1) / kTile) * ((args.N + kTile - 1) / kTile);
  auto kernel = gemm_fp4_pair_kernel<FMT>;
  if (tiles > (1 << 30) || set_max_smem(kernel, PairCfg<FMT>::kSmem) != cudaSuccess) return -1;
  const int pairs = static_cast<int>(std::min<long>(tiles, sms / 2));
  return launch_pdl(kernel, dim3(2 * pairs), dim3(kThreads), PairCfg<FMT>::kSmem, stream, maps.x, maps.w, maps.sx, maps.sw,
                    maps.y, args) == cudaSuccess ? 0 : -1;
}

}  // namespace

int launch_gemm_fp4_pair(const Fp4PairMaps& maps, const float* x_row, const float* w_row, int fmt, void* y, int M, int N,
                         int K, int sms, unsigned* status, cudaStream_t stream) {
  if (M < 1 || N < 1 || K < 32 || K % 32 != 0 || K > kFp4MaxK) return -1;
  PairArgs args{};
  args.x_row = x_row;
  args.w_row = w_row;
  args.y = static_cast<bf16*>(y);
  args.M = M;
  args.N = N;
  args.kblocks = (K + kBlockK - 1) / kBlockK;
  args.status = status;
  return fmt == kNv ? run<kNv>(maps, args, sms, stream) : run<kMx>(maps, args, sms, stream);
}

}  // namespace ecz
