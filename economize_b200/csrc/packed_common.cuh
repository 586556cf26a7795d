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

// What packing a and b into `packed` rounded away, packed the same way.
__device__ __forceinline__ uint32_t rest_of(uint32_t packed, float a, float b) {
  const float2 kept = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&packed));
  return pack_bf16(a - kept.x, b - kept.y);
}

// Two fp32 values in a 64-bit register and the operations on both at once, and the maximum of three.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// The low n bits (0 <= n <= 32 after clamping).
__device__ __forceinline__ uint32_t low_bits(int n) {
  return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
}

// 3-D tiled load of the map's box at (d, head, token). d is a multiple of 64.
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int d, int head,
                                            int token) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(d), "r"(head), "r"(token)
      : "memory");
}

// A tile of 128 rows, [128, DP] as DP / 64 atoms of 128 rows x 128 bytes, with one box per atom. Rows are tokens of one
// head, or (token, head) with the heads varying fastest: `1 << lp` heads of 128 >> lp tokens.
template <int DP>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int head, int token) {
#pragma unroll
  for (int a = 0; a < DP / 64; ++a) tma_load_3d(dst + a * kRowsT * 128, map, bar, a * 64, head, token);
}

// A chunk of keys or values of which `rows` are needed: whole, or by boxes of 32 rows (map32), so that a short
// sequence does not fetch a hundred rows of its successors. Counts the bytes on `bar` first.
template <int DP>
__device__ __forceinline__ void load_chunk(uint32_t dst, const CUtensorMap* map, const CUtensorMap* map32, uint64_t* bar,
                                           int head, int token, int rows) {
  if (rows > 64) {
    mbar_arrive_expect_tx(bar, kRowsT * DP * 2);
    load_tile<DP>(dst, map, bar, head, token);
    return;
  }
  const int boxes = (rows + 31) >> 5;
  mbar_arrive_expect_tx(bar, boxes * 32 * DP * 2);
  for (int b = 0; b < boxes; ++b)
#pragma unroll
    for (int a = 0; a < DP / 64; ++a)
      tma_load_3d(dst + a * kRowsT * 128 + b * 32 * 128, map32, bar, a * 64, head, token + b * 32);
}

// Zero rows [from, to) of a [128, DP] tile (the swizzle permutes 16-byte groups inside a row only); one warp.
template <int DP>
__device__ __forceinline__ void zero_rows(uint8_t* tile, int from, int to, int lane) {
  constexpr int kPerRow = DP / 8;
  for (int i = lane; i < (to - from) * kPerRow; i += 32) {
    const int row = from + i / kPerRow, c = i % kPerRow;
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
// every group of kStride columns), B's rows along K (MN-major); K steps kFrom, kFrom + kStep, ... < kTo of them.
template <int kPer, int kStride, int kFrom = 0, int kTo = 8, int kStep = 1>
__device__ __forceinline__ void mma_rows(uint32_t d, uint32_t p, uint32_t b, int n, int ksteps, bool accumulate) {
  const uint32_t idesc = idesc_bf16_f32(128, n, true);
  const uint64_t db = desc_mnmajor_sw128(b, kRowsT * 128);
#pragma unroll
  for (int kk = kFrom; kk < kTo; kk += kStep) {
    const uint32_t pc = p + (kk / kPer) * kStride + (kk % kPer) * 8;
    if (kk < ksteps) umma_bf16_ta(d, pc, desc_step(db, kk * 16 * 128), idesc, kk != 0 ? 1u : (accumulate ? 1u : 0u));
  }
}

// Zero the rows of x [T, width] outside the sequences (16-byte groups), shared by `threads` threads of every CTA, this
// one the `tid`-th of them.
__device__ __forceinline__ void zero_padding(bf16* x, int T, long width, const int* head, int tid, int threads) {
  const int first = head[1], last = head[2];
  const long groups = (static_cast<long>(first) + (T - last)) * (width / 8);
  for (long i = static_cast<long>(blockIdx.x) * threads + tid; i < groups; i += static_cast<long>(gridDim.x) * threads) {
    long row = i / (width / 8);
    if (row >= first) row += last - first;
    *reinterpret_cast<uint4*>(x + row * width + (i % (width / 8)) * 8) = make_uint4(0, 0, 0, 0);
  }
}

// ---- the work of persistent CTAs --------------------------------------------------------------------------------
// Items (table entry, sub) with sub < per varying fastest, heaviest first. A CTA's first item is its own index; the next
// ones it takes from a counter when its loading warp comes to the last chunk of an item, so that no CTA is left with a
// heavy item at the end (dealt out beforehand, the busiest CTA had 12 to 50% more than the mean). The loading warp
// publishes an item in a ring in shared memory from which the other warps read it. CTAs are persistent because an item
// of a short sequence is one or two tiles: with a CTA for each, set-up, first loads and last stores took two thirds of
// the time.
struct WorkItem {
  int4 tile;  // (first token, end, tile, tiles of its sequence)
  int sub, valid;
  int pad[2];
};

constexpr int kWorkRing = 4;

struct WorkRing {
  WorkItem* slots;         // [kWorkRing]
  uint64_t *full, *empty;  // [kWorkRing] each
  static constexpr int kBytes = kWorkRing * (static_cast<int>(sizeof(WorkItem)) + 16);
  __device__ __forceinline__ explicit WorkRing(void* base)
      : slots(static_cast<WorkItem*>(base)), full(reinterpret_cast<uint64_t*>(slots + kWorkRing)),
        empty(full + kWorkRing) {}
  __device__ __forceinline__ void init(int readers) const {
    for (int i = 0; i < kWorkRing; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], readers);
    }
  }
};

// The loading warp's side; lane 0 holds the item to come.
struct Feed {
  WorkRing ring;
  const int4* table;
  int* taken;
  int per, count, n, index;
  int4 ahead, tile;
  int sub;
  // The first tile is read along with the number of items: a CTA's first entry is inside the table.
  __device__ __forceinline__ Feed(const WorkRing& r, const int4* t, const int* head, int* counter, int per_entry)
      : ring(r), table(t), taken(counter), per(per_entry), count(head[0] * per_entry), n(0), index(blockIdx.x),
        ahead(t[blockIdx.x / per_entry]) {}
  // Lane 0, once for every item, at its last chunk: the next item's index is on its way ...
  __device__ __forceinline__ void reserve() { index = static_cast<int>(gridDim.x) + atomicAdd(taken, 1); }
  // ... and a load later its entry.
  __device__ __forceinline__ void fetch() {
    if (index < count) ahead = table[index / per];
  }
  // Publishes the next item; false when there is none (published too) or a wait gave up.
  __device__ __forceinline__ bool next(int lane, unsigned* status, volatile int* abort_flag) {
    int valid = 0;
    const int slot = n % kWorkRing;
    if (lane == 0 && mbar_wait(&ring.empty[slot], ((n / kWorkRing) & 1) ^ 1, status, kStatusWaitEmpty, abort_flag)) {
      valid = index < count;
      WorkItem item;
      item.tile = tile = ahead;
      item.sub = sub = index % per;
      item.valid = valid;
      ring.slots[slot] = item;
      mbar_arrive(&ring.full[slot]);
    }
    ++n;
    valid = uniform(valid);
    tile = make_int4(uniform(tile.x), uniform(tile.y), uniform(tile.z), uniform(tile.w));
    sub = uniform(sub);
    return valid != 0;
  }
};

// A reading warp's side; a warp that follows the items twice counts as two readers.
struct Items {
  WorkRing ring;
  int n;
  int4 tile;
  int sub;
  __device__ __forceinline__ explicit Items(const WorkRing& r) : ring(r), n(0) {}
  // Moves to the next item; false when there is none or a wait gave up.
  __device__ __forceinline__ bool next(unsigned* status, volatile int* abort_flag) {
    const int slot = n % kWorkRing;
    if (!__all_sync(0xffffffffu,
                    mbar_wait(&ring.full[slot], (n / kWorkRing) & 1, status, kStatusWaitFull, abort_flag)))
      return false;
    const WorkItem& item = ring.slots[slot];
    tile = make_int4(uniform(item.tile.x), uniform(item.tile.y), uniform(item.tile.z), uniform(item.tile.w));
    sub = uniform(item.sub);
    const int valid = uniform(item.valid);
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&ring.empty[slot]);
    ++n;
    return valid != 0;
  }
};

// Where the rows of a tile go: row r (< rows) to dst + (r >> lp) token + (r & ((1 << lp) - 1)) head, its columns below
// `cols`.
struct TileOut {
  bf16* dst;
  long token, head;  // strides in elements
  int lp, rows, cols;
  __device__ __forceinline__ bf16* row(int r) const {
    return dst + (r >> lp) * token + (r & ((1 << lp) - 1)) * head;
  }
};

// Stores 8 kG columns of a warp's 32 rows, from `row0` of the tile on: lane r holds row r's as kG 16-byte groups. A kG x
// kG transpose over groups of kG lanes (log2 kG exchanges) first, so that kG lanes write a row's segment at once: rows
// written by their own lanes touch 32 lines per store and took 3900 cycles for a 128 x 128 tile.
template <int kG>
__device__ __forceinline__ void store_rows(uint4 (&c)[kG], const TileOut& to, int row0, int lane) {
#pragma unroll
  for (int m = kG / 2; m > 0; m >>= 1) {
    const bool up = (lane & m) != 0;
#pragma unroll
    for (int i = 0; i < kG; ++i) {
      if (i & m) continue;
      uint4 out = up ? c[i] : c[i | m];
      out.x = __shfl_xor_sync(0xffffffffu, out.x, m);
      out.y = __shfl_xor_sync(0xffffffffu, out.y, m);
      out.z = __shfl_xor_sync(0xffffffffu, out.z, m);
      out.w = __shfl_xor_sync(0xffffffffu, out.w, m);
      if (up) c[i] = out;
      else c[i | m] = out;
    }
  }
  const int col = (lane & (kG - 1)) * 8;
#pragma unroll
  for (int j = 0; j < kG; ++j) {
    const int row = row0 + (lane & (32 - kG)) + j;
    if (row < to.rows && col < to.cols) *reinterpret_cast<uint4*>(to.row(row) + col) = c[j];
  }
}

// 8 kG fp32 columns of a lane's TMEM row, times f, as kG groups of eight bf16.
template <int kG>
__device__ __forceinline__ void load_packed(uint32_t taddr, float f, uint4 (&c)[kG]) {
  static_assert(kG == 2 || kG % 4 == 0, "TMEM is read by 16 or 32 columns");
  constexpr int kCols = kG == 2 ? 16 : 32;
  const uint64_t ff = pair_of(f, f);
#pragma unroll
  for (int h = 0; h < 8 * kG / kCols; ++h) {
    float o[kCols];
    if constexpr (kG == 2) tmem_ld16(taddr, o);
    else tmem_load32(taddr + h * 32, o);
#pragma unroll
    for (int j = 0; j < kCols / 8; ++j) {
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float a, b;
        unpair(mul2(pair_of(o[8 * j + 2 * k], o[8 * j + 2 * k + 1]), ff), a, b);
        w[k] = pack_bf16(a, b);
      }
      c[h * 4 + j] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// 64 columns of the warp's TMEM lanes, times each lane's f, as bf16 rows through 4 KB of shared memory (16-byte groups
// swizzled by the row, so that neither side conflicts). kRest: what bf16 rounds away of the values instead (itself
// rounded to bf16).
template <bool kRest>
__device__ __forceinline__ void stage_tmem64(uint32_t taddr, float f, uint8_t* stage, const TileOut& to, int row0,
                                             int lane) {
  const uint64_t ff = pair_of(f, f);
  uint8_t* mine = stage + lane * 128;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float o[32];
    tmem_load32(taddr + h * 32, o);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float a, b;
        unpair(mul2(pair_of(o[8 * j + 2 * k], o[8 * j + 2 * k + 1]), ff), a, b);
        w[k] = pack_bf16(a, b);
        if (kRest) w[k] = rest_of(w[k], a, b);
      }
      *reinterpret_cast<uint4*>(mine + (((h * 4 + j) ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  __syncwarp();
  const int g = lane & 7;
  if (g * 8 < to.cols) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = i * 4 + (lane >> 3);
      if (row0 + r < to.rows)
        *reinterpret_cast<uint4*>(to.row(row0 + r) + g * 8) =
            *reinterpret_cast<const uint4*>(stage + r * 128 + ((g ^ (r & 7)) << 4));
    }
  }
  __syncwarp();
}

// Tiles need 1024-byte boundaries, and there is no room to align them: dynamic shared memory starts on such a boundary
// where nothing static precedes it. Should it not, every thread leaves and the status says so.
__device__ __forceinline__ bool misplaced(const uint8_t* smem, unsigned* status) {
  if ((smem_u32(smem) & 1023u) == 0) return false;
  if (threadIdx.x == 0) atomicOr(status, kStatusBadShape);
  return true;
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
