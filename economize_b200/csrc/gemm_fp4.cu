// Products of 4-bit operands with block scales on tcgen05 (kind::mxf4nvf4 with e4m3 scales per 16 columns, kind::mxf4
// with E8M0 scales per 32): Y[m, n] = rx[m] rw[n] sum_k (qx fx)[m, k] (qw fw)[n, k], fp32 sums, rounded to bf16 once.
// The tensor cores multiply the scales in; rx and rw are the rows' powers of two of nvfp4. Layouts: fp4_common.cuh.
//
// gemm_fp4_kernel, for up to 128 rows of activations: weights are the MMA's 128 rows (A), activations its BN columns
// (B), so a tile streams 128 rows of weights once. A K block is 256 columns (128 bytes of codes a row, one swizzle row).
//
//   warp 0      TMA: codes of the weights [128 x 128 B] and of the activations [BN x 128 B], both blocks' scales as bulk
//               copies
//   warp 1      copies a block's scales to tensor memory (tcgen05.cp, in one of kSlots places, reused once the MMAs that
//               read it have completed) and issues its four MMAs of 64 columns
//   warps 2-5   epilogue: TMEM lane = output feature
//
// Few tiles are split along K over the CTAs of a cluster; the partial sums are added up through distributed shared
// memory in the order of the splits.
//
// Bound by HBM where the weights are large (times in a CUDA graph of calls over several weights): one row x 28672 x 4096
// takes 14.6 us, 10 of them its bytes, the rest launch, first loads and the last sums; 61 rows take 17.3 there, since every
// tile reads the activations and their scales again (10 KB beside a K block's 18 of weights). 4096 x 4096 takes 5.3 us, of
// which 1.5 are its bytes. At 128 rows it is level with the pairs of gemm_fp4_pair.cu (4096 x 4096: both 10.8 us) and behind
// from there on (192 rows: 17.6 against 10.8), which is where that kernel takes over.
#include <algorithm>

#include "fp4_common.cuh"
#include "launchers.h"

namespace ecz {

namespace {

using namespace fp4;

constexpr int kBM = 128;
constexpr int kRowBytes = kBlockK / 2;  // a K block of codes
constexpr int kABytes = kBM * kRowBytes;
constexpr int kThreads = 192;
constexpr int kSlots = 3;  // places for scales in tensor memory
constexpr int kMaxSplits = 8;

template <int FMT>
__device__ __forceinline__ void umma_fp4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                         uint32_t accumulate) {
  if constexpr (FMT == kNv) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  }
}

// 512 bytes of scales (32 rows of 16 bytes) to four TMEM columns, the same in all four groups of 32 lanes.
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// Weights and their scales to L2. Unlike a load this may run before the kernel that writes them has ended: all SMs share L2's
// copy of a line, so a load behind the wait finds what was written meanwhile.
__device__ __forceinline__ void prefetch_tile(const CUtensorMap* map, int x, int y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ void prefetch_bulk(const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src), "r"(bytes) : "memory");
}

// Four of CTA `rank`'s sums, at the address `local` has in this CTA's shared memory.
__device__ __forceinline__ float4 ld_sums(uint32_t local, uint32_t rank) {
  uint32_t remote;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(remote) : "memory");
  return v;
}

__device__ __forceinline__ void wait_ns(unsigned long long ns) {
  const unsigned long long start = global_timer_ns();
  while (global_timer_ns() - start < ns) {
  }
}

template <int FMT, int BN>
struct Cfg {
  static constexpr int kBBytes = BN * kRowBytes;
  static constexpr int kScaleBytes = Format<FMT>::kBlockBytes;
  static constexpr int kStageBytes = kABytes + kBBytes + 2 * kScaleBytes;
  // two CTAs to an SM: with one of five stages at BN = 128, 224 tiles took two rounds
  static constexpr int kOcc = 2;
  static constexpr int kStages = std::min(8, 110 * 1024 / kStageBytes);
  static constexpr int kSmem = kStages * kStageBytes + 1024 + 256 + BN * 4;
  static_assert(kSmem <= 113 * 1024, "two CTAs to an SM");
  static constexpr int kAccCols = BN < 32 ? 32 : BN;
  static constexpr int kSlotCols = 2 * 4 * Format<FMT>::kTilesPerBlock;
  static constexpr int kCols = kAccCols + kSlots * kSlotCols;
  static constexpr int kTmemCols = kCols <= 128 ? 128 : kCols <= 256 ? 256 : 512;
  static_assert(kStages >= kSlots, "a slot of scales is waited for by its stage's barrier");
  static_assert(kStages * kStageBytes >= BN * kBM * 4, "the partial sums reuse the stages");
};

struct Fp4Args {
  const uint8_t* w_scales;
  const uint8_t* x_scales;
  const float* w_row;  // nvfp4
  const float* x_row;
  bf16* y;
  int M, N, kblocks, per_split;
  unsigned* status;
};

template <int FMT, int BN>
__global__ void __launch_bounds__(kThreads, Cfg<FMT, BN>::kOcc)
    gemm_fp4_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                    const __grid_constant__ Fp4Args args) {
  using C = Cfg<FMT, BN>;
  constexpr int S = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* a_tiles = smem;
  uint8_t* b_tiles = a_tiles + S * kABytes;
  uint8_t* sa_tiles = b_tiles + S * C::kBBytes;
  uint8_t* sb_tiles = sa_tiles + S * C::kScaleBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(sb_tiles + S * C::kScaleBytes);
  uint64_t* empty = full + S;
  uint64_t* acc_full = empty + S;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* x_row = reinterpret_cast<float*>(tmem_slot + 2);  // [BN]

  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * kBM, m0 = blockIdx.y * BN, split = blockIdx.z, splits = gridDim.z;
  const int kb0 = split * args.per_split;
  const int nkb = max(0, min(args.per_split, args.kblocks - kb0));
  const size_t wide = static_cast<size_t>(args.kblocks) * C::kScaleBytes;  // scales of 128 rows
  const uint8_t* ws = args.w_scales + blockIdx.x * wide;
  // tiles that are not split begin at different K blocks: in step they would all read the same activations at once
  // (61 x 4096 x 28672 takes 0.8 us more in step; split tiles, fewer, lose 0.1 of 5 by it)
  const int turn = splits == 1 ? static_cast<int>(blockIdx.x) % args.kblocks : 0;
  auto place = [&](int kb) { return kb0 + (kb + turn < nkb ? kb + turn : kb + turn - nkb); };
  auto weights = [&](int kb) {
    const int s = kb % S, k = place(kb);
    mbar_arrive_expect_tx(&full[s], C::kStageBytes);
    tma_load_2d(a_tiles + s * kABytes, &tm_w, &full[s], k * kRowBytes, n0);
    bulk_load(sa_tiles + s * C::kScaleBytes, ws + static_cast<size_t>(k) * C::kScaleBytes, C::kScaleBytes, &full[s]);
  };
  const int pre = min(nkb, S);
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    *abort_flag = 0;
    fence_mbar_init();
    // The weights of the first stages go to L2 before the previous kernel ends and the block is ready, and to shared memory
    // behind the wait alone: nothing else orders them after a kernel that has just written them. (Loaded to shared memory
    // here, one row x 4096 x 4096 took 5.8 us with its quantisation in front, where this takes 6.2; ordered by kernels in
    // front that let this one start behind their own wait only, 6.7.)
    for (int kb = 0; kb < pre; ++kb) {
      const int k = place(kb);
      prefetch_tile(&tm_w, k * kRowBytes, n0);
      prefetch_bulk(ws + static_cast<size_t>(k) * C::kScaleBytes, C::kScaleBytes);
    }
    tma_prefetch_desc(&tm_x);
  }
  __syncwarp();
  if (warp == 1) tmem_alloc(tmem_slot, C::kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0 && lane == 0) {
    const uint8_t* xs = args.x_scales + (m0 / 128) * wide;
    auto activations = [&](int kb) {
      const int s = kb % S, k = place(kb);
      tma_load_2d(b_tiles + s * C::kBBytes, &tm_x, &full[s], k * kRowBytes, m0);
      bulk_load(sb_tiles + s * C::kScaleBytes, xs + static_cast<size_t>(k) * C::kScaleBytes, C::kScaleBytes, &full[s]);
    };
    pdl_wait();
    for (int kb = 0; kb < pre; ++kb) {
      weights(kb);
      activations(kb);
    }
    for (int kb = pre; kb < nkb; ++kb) {
      const int s = kb % S;
      if (!mbar_wait(&empty[s], ((kb / S) & 1u) ^ 1u, args.status, kStatusWaitEmpty, abort_flag)) break;
      weights(kb);
      activations(kb);
    }
  } else if (warp == 1 && lane == 0) {
    for (int kb = 0; kb < nkb; ++kb) {
      const int s = kb % S;
      if (kb >= kSlots) {  // the MMAs that read this slot's last scales have completed
        const int old = kb - kSlots;
        if (!mbar_wait(&empty[old % S], (old / S) & 1u, args.status, kStatusWaitAccum, abort_flag)) break;
      }
      if (!mbar_wait(&full[s], (kb / S) & 1u, args.status, kStatusWaitFull, abort_flag)) break;
      tc_fence_after();
      const uint32_t sfa = tmem + C::kAccCols + (kb % kSlots) * C::kSlotCols;
      const uint32_t sfb = sfa + 4 * Format<FMT>::kTilesPerBlock;
      const uint32_t sa = smem_u32(sa_tiles + s * C::kScaleBytes), sb = smem_u32(sb_tiles + s * C::kScaleBytes);
#pragma unroll
      for (int t = 0; t < Format<FMT>::kTilesPerBlock; ++t) {
        copy_scales(sfa + 4 * t, desc_scales(sa + t * kTileBytes));
        copy_scales(sfb + 4 * t, desc_scales(sb + t * kTileBytes));
      }
      const uint32_t a = smem_u32(a_tiles + s * kABytes), b = smem_u32(b_tiles + s * C::kBBytes);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        const int t = FMT == kNv ? kk : kk / 2;
        const uint32_t idesc = FMT == kNv ? idesc_fp4<FMT>(kBM, BN) : idesc_fp4<FMT>(kBM, BN, (kk & 1) * 2);
        umma_fp4<FMT>(tmem, desc_kmajor_sw128(a + kk * 32), desc_kmajor_sw128(b + kk * 32), idesc, sfa + 4 * t,
                      sfb + 4 * t, (kb | kk) != 0 ? 1u : 0u);
      }
      umma_commit(&empty[s]);
    }
    umma_commit(acc_full);
  }
  __syncwarp();
  pdl_wait();
  if (warp < 2 && *abort_flag) wait_ns(1000000);  // a wait gave up: copies in flight get time to land
  bool ok = true;
  const int quarter = warp & 3;
  const uint32_t taddr = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
  const int cols = min(BN, args.M - m0), n = n0 + lane * 4;
  float4 rw = make_float4(1.f, 1.f, 1.f, 1.f);
  if (warp >= 2) {
    if constexpr (FMT == kNv) {  // at hand before the sums are
      for (int j = threadIdx.x - 64; j < cols; j += 128) x_row[j] = args.x_row[m0 + j];
    }
    ok = mbar_wait(acc_full, 0, args.status, kStatusWaitAccum, abort_flag);
    ok = __all_sync(0xffffffffu, ok) && !*abort_flag;
    tc_fence_after();
  }
  // This CTA's sums [BN][128] go where its stages were (every copy has landed and was read); each CTA of the cluster then
  // adds up and stores a share of the columns, four features a thread.
  float* part = reinterpret_cast<float*>(smem);
  if constexpr (FMT == kNv) {
    if (n < args.N) rw.x = args.w_row[n];
    if (n + 1 < args.N) rw.y = args.w_row[n + 1];
    if (n + 2 < args.N) rw.z = args.w_row[n + 2];
    if (n + 3 < args.N) rw.w = args.w_row[n + 3];
  }
  if (warp >= 2) {
#pragma unroll
    for (int c = 0; c < BN; c += 16) {
      if (c < cols) {
        float v[16];
        if (ok && nkb > 0) tmem_ld16(taddr + c, v);
#pragma unroll
        for (int j = 0; j < 16; ++j) part[(c + j) * kBM + quarter * 32 + lane] = ok && nkb > 0 ? v[j] : 0.f;
      }
    }
  }
  if (splits > 1) cluster_sync();
  else __syncthreads();
  {
    const uint32_t at = smem_u32(part) + lane * 16;
    for (int j = split + warp * splits; j < cols; j += splits * (kThreads / 32)) {
      float4 p[kMaxSplits];
#pragma unroll
      for (int r = 0; r < kMaxSplits; ++r)
        if (r < splits) p[r] = splits > 1 ? ld_sums(at + j * kBM * 4, r)
                                          : *reinterpret_cast<const float4*>(part + j * kBM + lane * 4);
      float4 sum = p[0];
#pragma unroll
      for (int r = 1; r < kMaxSplits; ++r) {
        if (r < splits) {
          sum.x += p[r].x;
          sum.y += p[r].y;
          sum.z += p[r].z;
          sum.w += p[r].w;
        }
      }
      if constexpr (FMT == kNv) {
        const RowFactors rx = row_factors(x_row[j]);
        sum.x = sum.x * rx.first * rw.x * rx.last;
        sum.y = sum.y * rx.first * rw.y * rx.last;
        sum.z = sum.z * rx.first * rw.z * rx.last;
        sum.w = sum.w * rx.first * rw.w * rx.last;
      }
      const __nv_bfloat162 lo = __floats2bfloat162_rn(sum.x, sum.y);
      const __nv_bfloat162 hi = __floats2bfloat162_rn(sum.z, sum.w);
      bf16* out = args.y + static_cast<size_t>(m0 + j) * args.N + n;
      if (args.N % 4 == 0) {
        if (n < args.N)
          *reinterpret_cast<uint2*>(out) =
              make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
      } else {
        if (n < args.N) out[0] = lo.x;
        if (n + 1 < args.N) out[1] = lo.y;
        if (n + 2 < args.N) out[2] = hi.x;
        if (n + 3 < args.N) out[3] = hi.y;
      }
    }
  }
  if (splits > 1) cluster_sync();  // the others have read this CTA's sums
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, C::kTmemCols);
}

template <int FMT, int BN>
int run(const CUtensorMap& w, const CUtensorMap& x, Fp4Args args, int splits, cudaStream_t stream) {
  using C = Cfg<FMT, BN>;
  auto kernel = gemm_fp4_kernel<FMT, BN>;
  if (set_max_smem(kernel, C::kSmem) != cudaSuccess) return -1;
  args.per_split = (args.kblocks + splits - 1) / splits;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((args.N + kBM - 1) / kBM, (args.M + BN - 1) / BN, splits);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = splits;
  cfg.attrs = attr;
  cfg.numAttrs = splits > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, w, x, args) == cudaSuccess ? 0 : -1;
}

template <int FMT>
int run_fmt(const CUtensorMap& w, const CUtensorMap& x, const Fp4Args& args, int bn, int splits, cudaStream_t stream) {
  switch (bn) {
    case 16: return run<FMT, 16>(w, x, args, splits, stream);
    case 32: return run<FMT, 32>(w, x, args, splits, stream);
    case 64: return run<FMT, 64>(w, x, args, splits, stream);
    default: return run<FMT, 128>(w, x, args, splits, stream);
  }
}

}  // namespace

int fp4_block_rows(int M) { return M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128; }

int launch_gemm_fp4(const CUtensorMap* w, const CUtensorMap* x, const void* w_scales, const void* x_scales,
                    const float* w_row, const float* x_row, int fmt, void* y, int M, int N, int K, int sms,
                    unsigned* status, cudaStream_t stream) {
  if (M < 1 || N < 1 || K < 32 || K % 32 != 0 || K > kFp4MaxK) return -1;
  Fp4Args args{};
  args.w_scales = static_cast<const uint8_t*>(w_scales);
  args.x_scales = static_cast<const uint8_t*>(x_scales);
  args.w_row = w_row;
  args.x_row = x_row;
  args.y = static_cast<bf16*>(y);
  args.M = M;
  args.N = N;
  args.kblocks = (K + kBlockK - 1) / kBlockK;
  args.status = status;
  const int bn = fp4_block_rows(M);
  // splits by the weights' size alone, so that a row's sums do not depend on how many rows there are
  const int tiles = (N + kBM - 1) / kBM;
  int splits = 1;
  while (splits < kMaxSplits && tiles * splits < sms && 2 * splits <= args.kblocks) splits *= 2;
  return fmt == kNv ? run_fmt<kNv>(*w, *x, args, bn, splits, stream) : run_fmt<kMx>(*w, *x, args, bn, splits, stream);
}

}  // namespace ecz
