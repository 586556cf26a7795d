// Large-tile GEMM core of the training operators: D[M, N] = A . B^T with either operand K-major ([M, K] / [N, K]
// rows) or MN-major ([K, M] / [K, N] rows), bf16 in, fp32 accumulation, for products with thousands of rows (the
// decode GEMMs of gemm_tc.cu swap the operands instead, for a few dozen rows).
//
// A cluster of two CTAs computes one 256 x 256 tile with cta_group::2 MMAs (M = 256, N = 256): each CTA holds its
// own 128 rows of A and half of the columns of B in shared memory (32 KB per 64-element K step) and 128 x 256 fp32
// accumulators in TMEM, so per 128 x 256 outputs a CTA reads 32 KB from L2 where a one-CTA tile of the same shape
// reads 48 KB. The accumulators are double-buffered (2 x 256 TMEM columns): the epilogue of a tile runs under the
// next tile's MMAs.
//
// A product whose sums may not shrink takes them in parts of `part` K blocks, an accumulator buffer each, and its epilogue
// adds the parts up in registers: the tensor cores cut off, towards zero, what an accumulator cannot hold, at every 16
// products, so sums of 4096 came out 3.9e-6 of themselves too small. Parts of 1024 bring that to 1e-6, whatever K is.
//
//   warp 0      TMA producer (both CTAs; completion counted on the even CTA's barrier)
//   warp 1      MMA issuer (even CTA only): the whole warp walks the K blocks, an elected lane issues from descriptors in
//               uniform registers; issued by a branch of one lane, the MMAs came so slowly that every change of
//               accumulators, a part's or a tile's, left the tensor pipes idle for 600 cycles
//   warps 2-9   epilogue: warp w reads TMEM lanes 32 (w % 4) .. + 31 and 128 of the 256 columns
//
// The grid is persistent over tiles. Tiles beyond whole rounds of all pairs are split along K where that fills the pairs
// (Schedule): their units leave fp32 partial tiles that a joining kernel adds up in order. Every wait is bounded
// (common.cuh).
//
// Measured on one B200, 4096 x 4096 x 32000, single launches: both operands K-major with sums in one part 1600 to 1680
// TFLOP/s, in parts of 1024 (logits) 1580 to 1670, the tensor pipes busy 98% of the cycles; in a long step the power limit
// of 1 kW and the clock that it leaves are what bounds it.
#pragma once

#include "common.cuh"
#include "packed_common.cuh"

namespace ecz {
namespace pair {

constexpr int kTile = 256;    // output tile (both dimensions) of a CTA pair
constexpr int kHalf = 128;    // A rows and B rows (columns of the output) a CTA loads
constexpr int kBK = 64;       // K elements per stage
constexpr int kOperandBytes = kHalf * kBK * 2;
constexpr int kStageBytes = 2 * kOperandBytes;
constexpr int kStages = 5;
constexpr int kThreads = 320;
constexpr int kEpiWarps = 8;
constexpr int kPatchStride = 144;                 // bytes per row of an epilogue warp's [32 rows, 64 bf16] patch
constexpr int kPatchBytes = 32 * kPatchStride;
constexpr int kSmem = kStages * kStageBytes + kEpiWarps * kPatchBytes + 1024 + 256;
static_assert(kSmem <= 232448, "227 KB of shared memory");

constexpr int kSplitBlocks = 8, kTailBlocks = 64;  // see Schedule

// What a launch computes. Counts on the device (rows_dev) clip M (clip_m) or K (clip_k) of a chunk of rows that
// starts at row0: limit = clamp(*rows_dev - row0, 0, M or K).
struct Shape {
  int M, N, K;
  const int* rows_dev;
  int row0;
  bool clip_m, clip_k;
  int pairs;       // CTA pairs of the device
  bool split;      // tiles beyond whole rounds may be split along K
  bool n_fastest;  // order of the tiles: N varies fastest (else M)
  int part;        // K blocks of a part of a sum, for epilogues with kParts (no such product is split or clipped in K)
};

__device__ __forceinline__ uint32_t mapa_u32(uint32_t addr, uint32_t rank) {
  uint32_t out;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(out) : "r"(addr), "r"(rank));
  return out;
}

// TMA load into this CTA's shared memory whose bytes are counted on barrier `bar` (a shared::cluster address, of the
// pair's even CTA).
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, "
      "%4}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
      : "memory");
}

__device__ __forceinline__ void umma_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Arrive on barrier `bar` (same offset) of both CTAs once every MMA issued so far by this thread has completed.
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  const uint16_t mask = 3;
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"(mask)
      : "memory");
}

__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// An operand stage of 128 MN rows x 64 K: K-major, one {64 (K), 128} box; MN-major, two {64 (MN), 64 (K)} boxes.
template <bool MN>
__device__ __forceinline__ void load_operand(uint32_t dst, const CUtensorMap* map, uint32_t bar, int mn, int k) {
  if (MN) {
    tma_load_pair(dst, map, bar, mn, k);
    tma_load_pair(dst + kOperandBytes / 2, map, bar, mn + 64, k);
  } else {
    tma_load_pair(dst, map, bar, k, mn);
  }
}

template <bool MN>
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, int kk) {
  return MN ? desc_mnmajor_sw128(addr + kk * 16 * 128, kOperandBytes / 2) : desc_kmajor_sw128(addr + kk * 32);
}

// A unit of the persistent grid: tile (m0, n0) and the K blocks [kb0, kb0 + nkb) of its split; `tail`: the tile's place
// among the split ones.
struct Unit {
  int m0, n0, split, splits, tail, kb0, nkb;
};

// Tiles in order of units, the first `whole` in one piece. The rest (fewer than the pairs) in as many as fill the pairs
// once, each with eight K blocks at least (a shorter one is all prologue) and, behind whole rounds, of 64 K blocks or
// more: a round of those takes 18 us, the joining kernel 5.
struct Schedule {
  int m_tiles, n_tiles, whole, splits, units, kblocks;
  const Shape& s;
  int M, K;
  __device__ __forceinline__ explicit Schedule(const Shape& shape) : s(shape) {
    int rows = 0;
    if (s.rows_dev != nullptr) rows = max(0, *s.rows_dev - s.row0);
    M = s.clip_m ? min(s.M, rows) : s.M;
    K = s.clip_k ? min(s.K, rows) : s.K;
    m_tiles = (M + kTile - 1) / kTile;
    n_tiles = (s.N + kTile - 1) / kTile;
    kblocks = (K + kBK - 1) / kBK;
    const int tiles = m_tiles * n_tiles, rest = tiles % s.pairs;
    splits = s.split && rest > 0 && (rest == tiles || kblocks >= kTailBlocks)
                 ? max(1, min(s.pairs / rest, kblocks / kSplitBlocks)) : 1;
    whole = splits > 1 ? tiles - rest : tiles;
    units = whole + (tiles - whole) * splits;
  }
  __device__ __forceinline__ Unit unit(int u) const {
    Unit r;
    const bool part = u >= whole;
    r.splits = part ? splits : 1;
    r.tail = part ? (u - whole) / splits : 0;
    r.split = part ? (u - whole) - r.tail * splits : 0;
    const int t = part ? whole + r.tail : u;
    const int mt = s.n_fastest ? t / n_tiles : t % m_tiles;
    const int nt = s.n_fastest ? t % n_tiles : t / m_tiles;
    r.m0 = mt * kTile;
    r.n0 = nt * kTile;
    const int per = part ? (kblocks + splits - 1) / splits : kblocks;
    r.kb0 = min(kblocks, r.split * per);
    r.nkb = min(per, kblocks - r.kb0);
    return r;
  }
};

// Most split tiles of a launch, and whether it may have any.
inline int most_tail(const Shape& s) {
  const int tiles = ((s.M + kTile - 1) / kTile) * ((s.N + kTile - 1) / kTile);
  const int kblocks = (s.K + kBK - 1) / kBK;
  if (!s.split || kblocks < 2 * kSplitBlocks) return 0;
  if (s.clip_m) return tiles < s.pairs / 2 ? tiles : s.pairs / 2;
  const int rest = tiles % s.pairs;
  return 2 * rest <= s.pairs && (rest == tiles || kblocks >= kTailBlocks) ? rest : 0;
}

// Epi: a functor `void operator()(const Unit&, int M, int row0, int col0, uint32_t taddr, bool zero, uint8_t* patch,
// int lane)` of one warp: rows row0 + lane (of the whole output), columns [col0, col0 + 128), accumulators at TMEM
// address taddr (this warp's lanes), or zeros where the unit has no K block. With Epi::kParts the sums in registers, z[j]
// of column col0 + j, in place of taddr and zero.
template <bool A_MN, bool B_MN, class Epi>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    gemm_pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                     const __grid_constant__ Shape shape, const __grid_constant__ Epi epi, unsigned* status) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* patches = smem + kStages * kStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(patches + kEpiWarps * kPatchBytes);
  uint64_t* empty = full + kStages;
  uint64_t* acc_full = empty + kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = packed::uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 2 * kEpiWarps);
    }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tm_a);
    tma_prefetch_desc(&tm_b);
  }
  __syncwarp();
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(512)
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

  const Schedule sched(shape);
  const int pairs = gridDim.x >> 1, pair_id = blockIdx.x >> 1;
  if (warp == 0 && lane == 0) {
    // ---- producer ----
    const uint32_t base = smem_u32(smem);
    uint32_t it = 0;
    bool ok = true;
    for (int u = pair_id; ok && u < sched.units; u += pairs) {
      const Unit t = sched.unit(u);
      for (int kb = 0; kb < t.nkb; ++kb, ++it) {
        const int s = it % kStages;
        if (!mbar_wait(&empty[s], ((it / kStages) & 1u) ^ 1u, status, kStatusWaitEmpty, abort_flag)) {
          ok = false;
          break;
        }
        const uint32_t bar = mapa_u32(smem_u32(&full[s]), 0);
        if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * kStageBytes);
        const uint32_t dst = base + s * kStageBytes;
        const int k = (t.kb0 + kb) * kBK;
        load_operand<A_MN>(dst, &tm_a, bar, t.m0 + static_cast<int>(rank) * kHalf, k);
        load_operand<B_MN>(dst + kOperandBytes, &tm_b, bar, t.n0 + static_cast<int>(rank) * kHalf, k);
      }
    }
    // every copy in flight has landed before the pair leaves (its barriers' phases have been consumed, or a wait gave
    // up): the last stages' loads were waited for by the MMA issuer; after an abort, give them time
    if (!ok) {
      const unsigned long long t0 = global_timer_ns();
      while (global_timer_ns() - t0 < 1000000ull) {
      }
    }
  } else if (warp == 1 && rank == 0) {
    // ---- MMA issuer: the whole warp walks, one lane issues, from descriptors in uniform registers ----
    constexpr uint32_t idesc = idesc_bf16_f32(256, 256, B_MN) | ((A_MN ? 1u : 0u) << 15);
    const uint32_t base = smem_u32(smem);
    const uint64_t a0 = operand_desc<A_MN>(base, 0), b0 = operand_desc<B_MN>(base + kOperandBytes, 0);
    const bool leader = packed::elect_one();
    uint32_t tile = 0, s = 0, turn = 0;  // stage, its phase
    bool ok = true;
    for (int u = pair_id; ok && u < sched.units; u += pairs) {
      const Unit t = sched.unit(u);
      const int part = Epi::kParts ? shape.part : t.nkb;
      for (int kb0 = 0; ok && kb0 < t.nkb; kb0 += part) {
        const uint32_t buf = tile & 1u;
        ok = packed::warp_wait(&acc_empty[buf], ((tile >> 1) & 1u) ^ 1u, status, kStatusWaitAccum, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const uint32_t d = tmem + buf * 256u;
        const int blocks = min(part, t.nkb - kb0);
        for (int kb = 0; kb < blocks; ++kb) {
          ok = packed::warp_wait(&full[s], turn, status, kStatusWaitFull, abort_flag);
          if (!ok) break;
          tc_fence_after();
          if (leader) {
            const uint64_t a = packed::desc_step(a0, s * kStageBytes), b = packed::desc_step(b0, s * kStageBytes);
#pragma unroll
            for (int kk = 0; kk < kBK / 16; ++kk)
              umma_pair(d, packed::desc_step(a, kk * (A_MN ? 16 * 128 : 32)),
                        packed::desc_step(b, kk * (B_MN ? 16 * 128 : 32)), idesc, (kb | kk) != 0 ? 1u : 0u);
            commit_pair(&empty[s]);
          }
          __syncwarp();
          if (++s == kStages) {
            s = 0;
            turn ^= 1u;
          }
        }
        if (leader) commit_pair(&acc_full[buf]);
        __syncwarp();
        ++tile;
      }
    }
  } else if (warp >= 2) {
    // ---- epilogue ----
    const int ew = warp - 2;
    const int quad = warp & 3, half = ew >> 2;
    uint8_t* patch = patches + ew * kPatchBytes;
    uint32_t tile = 0;
    for (int u = pair_id; u < sched.units; u += pairs) {
      const Unit t = sched.unit(u);
      const int row0 = t.m0 + static_cast<int>(rank) * kHalf + quad * 32, col0 = t.n0 + half * 128;
      const uint32_t taddr = tmem + (static_cast<uint32_t>(quad * 32) << 16) + half * 128u;
      // waits for the accumulators that come next, hands them to `take`, and gives their buffer back
      auto accumulators = [&](auto&& take) {
        const uint32_t buf = tile & 1u;
        const bool ok = mbar_wait(&acc_full[buf], (tile >> 1) & 1u, status, kStatusWaitAccum, abort_flag);
        if (__any_sync(0xffffffffu, !ok)) return false;
        tc_fence_after();
        take(taddr + buf * 256u);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_cluster(mapa_u32(smem_u32(&acc_empty[buf]), 0));
        ++tile;
        return true;
      };
      if constexpr (Epi::kParts) {
        float z[kHalf];  // the first part's sums, then the others' added
        bool ok = accumulators([&](uint32_t at) {
#pragma unroll
          for (int c = 0; c < kHalf; c += 16) tmem_ld16(at + c, z + c);
        });
#pragma unroll 1
        for (int kb = shape.part; ok && kb < t.nkb; kb += shape.part)
          ok = accumulators([&](uint32_t at) {
#pragma unroll
            for (int c = 0; c < kHalf; c += 16) {
              float v[16];
              tmem_ld16(at + c, v);
#pragma unroll
              for (int j = 0; j < 16; ++j) z[c + j] += v[j];
            }
          });
        if (!ok) break;
        epi(t, sched.M, row0, col0, z, patch, lane);
      } else if (t.nkb <= 0) {
        epi(t, sched.M, row0, col0, 0u, true, patch, lane);
      } else if (!accumulators([&](uint32_t at) { epi(t, sched.M, row0, col0, at, false, patch, lane); })) {
        break;
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

template <bool A_MN, bool B_MN, class Epi>
inline int launch_pair(const CUtensorMap& a, const CUtensorMap& b, const Shape& shape, const Epi& epi,
                       unsigned* status, cudaStream_t stream) {
  const long tiles = static_cast<long>((shape.M + kTile - 1) / kTile) * ((shape.N + kTile - 1) / kTile);
  if (tiles <= 0) return 0;
  const int pairs = shape.split || tiles > shape.pairs ? shape.pairs : static_cast<int>(tiles);
  auto kernel = gemm_pair_kernel<A_MN, B_MN, Epi>;
  if (set_max_smem(kernel, kSmem) != cudaSuccess) return -1;
  return launch_pdl(kernel, dim3(2 * pairs), dim3(kThreads), kSmem, stream, a, b, shape, epi, status) == cudaSuccess ? 0
                                                                                                                    : -1;
}

}  // namespace pair
}  // namespace ecz
