// What the forward and backward kernels of the packed attention share: tile loads, MMAs over 128-row tiles in shared
// memory and TMEM, and the zeroing of rows outside the sequences.
#pragma once

#include "common.cuh"
#include "tmem_wide.cuh"

namespace ecz {
namespace packed {

constexpr int kRowsT = 128;  // rows of a query tile, keys of a chunk
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// 3-D tiled load: box {64 (d), 1 (head), 128 (tokens)} at (d, head, token). d is a multiple of 64.
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int d, int head,
                                            int token) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(d), "r"(head), "r"(token)
      : "memory");
}

// [128 rows, DP] as DP / 64 atoms of 128 rows x 128 bytes.
template <int DP>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int head, int token) {
#pragma unroll
  for (int a = 0; a < DP / 64; ++a) tma_load_3d(dst + a * kRowsT * 128, map, bar, a * 64, head, token);
}

// Zero rows [from, to) of a [128, DP] tile (the swizzle permutes 16-byte groups inside a row only); one warp.
template <int DP>
__device__ __forceinline__ void zero_rows(uint8_t* tile, int from, int to, int lane) {
  const int per_row = DP / 8;
  for (int i = lane; i < (to - from) * per_row; i += 32) {
    const int row = from + i / per_row, c = i % per_row;
    *reinterpret_cast<uint4*>(tile + (c >> 3) * kRowsT * 128 + row * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_async_smem();
  __syncwarp();
}

// The MMA loops below are unrolled around one descriptor per operand and constant steps, added to its low word (the
// address field, which does not overflow); the issuing warp's tile fields are broadcast from lane 0 (uniform()) so that
// descriptors live in uniform registers. With descriptors built in a run-time loop a 128 x 128 x 16 MMA took 115 cycles
// to issue (64 to execute).
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

// True in one lane of the (converged) warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xffffffff;\n\tselp.u32 %0, 1, 0, P;\n\t}" : "=r"(p));
  return p != 0;
}

__device__ __forceinline__ uint64_t desc_step(uint64_t desc, uint32_t bytes) {
  const uint32_t lo = static_cast<uint32_t>(desc) + (bytes >> 4), hi = static_cast<uint32_t>(desc >> 32);
  return (static_cast<uint64_t>(hi) << 32) | lo;
}

// D[128, n] = A[128, :16 ksteps] . B[n, :16 ksteps]^T, both K-major tiles of [128, DP] (K the head dimension).
template <int DP>
__device__ __forceinline__ void mma_dims(uint32_t d, uint32_t a, uint32_t b, int n, int ksteps) {
  const uint32_t idesc = idesc_bf16_f32(128, n);
  const uint64_t da = desc_kmajor_sw128(a), db = desc_kmajor_sw128(b);
#pragma unroll
  for (int kk = 0; kk < DP / 16; ++kk) {
    const uint32_t off = (kk >> 2) * kRowsT * 128 + (kk & 3) * 32;
    if (kk < ksteps) umma_bf16(d, desc_step(da, off), desc_step(db, off), idesc, kk != 0 ? 1u : 0u);
  }
}

// D[128, n] (+)= P[128, :16 ksteps] . B[:16 ksteps, n], P packed bf16 in TMEM (kPer K steps of 8 columns side by side in
// every group of kStride columns), B's rows along K (MN-major).
template <int kPer, int kStride>
__device__ __forceinline__ void mma_rows(uint32_t d, uint32_t p, uint32_t b, int n, int ksteps, bool accumulate) {
  const uint32_t idesc = idesc_bf16_f32(128, n, true);
  const uint64_t db = desc_mnmajor_sw128(b, kRowsT * 128);
#pragma unroll
  for (int kk = 0; kk < 8; ++kk) {
    const uint32_t pc = p + (kk / kPer) * kStride + (kk % kPer) * 8;
    if (kk < ksteps) umma_bf16_ta(d, pc, desc_step(db, kk * 16 * 128), idesc, kk != 0 ? 1u : (accumulate ? 1u : 0u));
  }
}

// Zero the rows of x [T, width] outside the sequences (16-byte groups), shared by the grid.
__device__ __forceinline__ void zero_padding(bf16* x, int T, long width, const int* head) {
  const int first = head[1], last = head[2];
  const long groups = (static_cast<long>(first) + (T - last)) * (width / 8);
  for (long i = static_cast<long>(blockIdx.x) * blockDim.x + threadIdx.x; i < groups;
       i += static_cast<long>(gridDim.x) * blockDim.x) {
    long row = i / (width / 8);
    if (row >= first) row += last - first;
    *reinterpret_cast<uint4*>(x + row * width + (i % (width / 8)) * 8) = make_uint4(0, 0, 0, 0);
  }
}

// The end of a CTA whose waits may have given up: copies in flight land before the shared memory goes.
__device__ __forceinline__ void settle(bool aborted) {
  if (!aborted) return;
  const unsigned long long t0 = global_timer_ns();
  while (global_timer_ns() - t0 < 1000000ull) {
  }
}

// mbar_wait of a whole warp.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, unsigned* status, unsigned code,
                                          volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, status, code, abort_flag));
}

}  // namespace packed
}  // namespace ecz
