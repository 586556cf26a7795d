// Causal attention over packed sequences with grouped heads: the forward pass (training and scoring prompts).
//
//   s_ij = scale q_i . k_j (a <= j <= i < b for the sequence [a, b) of token i)     L_i = log sum_j exp s_ij
//   o_i = sum_j exp(s_ij - L_i) v_j
//
// Tokens of all sequences lie one after another, q [T, H, D], k / v [T, Hkv, D]; sequence n holds the tokens
// [cu[n], cu[n + 1]). A tile of queries is 128 rows of one sequence: (token, head) pairs of 1, 2, 4 or 8 heads of a group
// (the largest of these that divides it) and 128, 64, 32 or 16 tokens. All heads of a pack read the same K / V chunk, a
// short sequence fills its tiles better (85 tokens of four heads are three tiles, not four), and less of the diagonal
// chunk is computed in vain. The plan kernel cuts every sequence into tiles from its first token on, so a tile never
// mixes sequences, and lists them heaviest first: the last ones dealt to the persistent CTAs (see Feed) are short.
//
// A CTA works on one or two neighbouring query tiles over the same K / V chunks. One warp loads (TMA, a ring of 128-key
// K and V chunks), one issues the MMAs, and a warpgroup per tile runs its softmax, one thread per row, so the tensor
// cores work on one tile while the other's exponentials run. S and P share TMEM columns (P overwrites S as bf16 and is
// the A operand of P . V), O accumulates in TMEM. A row's reference maximum moves only when a chunk raises it by more
// than 2^8 (lazy rescaling), so O is rarely read back before the end.
//
// The running reference and sum are those of the online softmax (Milakov and Gimelshein, 2018), the recomputation of P
// from the log-sum-exp in the backward pass is that of Dao et al. (2022).
//
// P is rounded to bf16 for P . V: one rounding of the output's left factor, as its result's is of the whole. Over many
// keys these errors average out; a tile of one chunk multiplies what the rounding leaves of P as well (eight MMAs more),
// so that the output's rows of few keys, and the backward pass's delta, where dp - delta cancels, do not carry it.
//
// A chunk that reaches past its sequence's end holds other rows (the next sequence's, or unwritten padding): their
// scores are replaced, not multiplied, and the at most 15 V rows that P . V reads in its last K step beyond the end
// are zeroed in shared memory, so NaN or infinities there reach nothing.
#include <algorithm>

#include "launchers.h"
#include "packed_common.cuh"

namespace ecz {

using namespace packed;

namespace {

constexpr float kLazy = 8.f;  // log2 units
constexpr float kFar = 60.f;

// ---- plan ----------------------------------------------------------------------------------------------------------
// One CTA per table: a list of tiles of `rows` tokens, heaviest first: entry = (first token, end, tile, tiles of its
// sequence); head = (tiles, first token of the first sequence, end of the last, items taken). Offsets outside [0, T] or
// falling are clamped (a sequence starts where the one before it ended at the earliest) and reported. Latency bounds it:
// scans and a search per tile, 4.0 us for the tables of all three kernels of 8192 tokens in 5 sequences, 32 heads over 8
// (6.0 with scans in which every thread read the 32 warps' results).
constexpr int kPlanThreads = 1024;
constexpr int kPlanTables = 3;

struct PlanArgs {
  PackedTable tables[kPlanTables];
};

__device__ __forceinline__ int warp_scan(int v) {  // inclusive
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  return v;
}

__device__ __forceinline__ int warp_scan_max(int v) {  // inclusive
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v = max(v, y);
  }
  return v;
}

// Over the block's 32 warps: every warp scans the warps' results again.
__device__ __forceinline__ int scan_add(int v, int* warp_sums, int& total) {  // exclusive
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int x = warp_scan(v);
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  const int sum = warp_sums[lane], upto = warp_scan(sum);
  const int before = __shfl_sync(0xffffffffu, upto - sum, warp);
  total = __shfl_sync(0xffffffffu, upto, 31);
  __syncthreads();
  return before + x - v;
}

__device__ __forceinline__ int scan_max(int v, int* warp_max) {  // inclusive, of values from 0 on
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = warp_scan_max(v);
  if (lane == 31) warp_max[warp] = v;
  __syncthreads();
  const int upto = warp_scan_max(warp_max[lane]);
  const int before = __shfl_sync(0xffffffffu, upto, max(warp - 1, 0));
  __syncthreads();
  return warp > 0 ? max(v, before) : v;
}

__global__ void __launch_bounds__(kPlanThreads)
    packed_plan_kernel(const int* __restrict__ cu, int B, int T, const __grid_constant__ PlanArgs args,
                       unsigned* status) {
  // Tiles are sorted by bins of their weight (tile i reads i + 1 times as many keys as tile 0), a thread per bin:
  // `change` counts how many tiles a bin has more than the one before, `rest` those of sequences that end in it.
  __shared__ int change[kPlanThreads], rest[kPlanThreads], near_lo[kPlanThreads + 1], near_base[kPlanThreads + 1];
  __shared__ int sums[32];
  __shared__ int carry_max, carry_tiles;
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x;
  const PackedTable& table = args.tables[blockIdx.x];
  int4* entries = static_cast<int4*>(table.entries);
  const int rows = table.rows, max_tiles = table.max_tiles;
  // searched per tile, in shared memory where they fit
  int* lo = B <= kPlanThreads ? near_lo : table.scratch;
  int* base = B <= kPlanThreads ? near_base : table.scratch + B + 1;
  const int per = (max_tiles + kPlanThreads - 2) / (kPlanThreads - 1);  // weights of a bin
  change[tid] = 0;
  rest[tid] = 0;
  if (tid == 0) {
    carry_max = 0;
    carry_tiles = 0;
  }
  __syncthreads();
  for (int s0 = 0; s0 <= B; s0 += kPlanThreads) {
    const int s = s0 + tid;
    const int raw = s <= B ? cu[s] : 0;
    int edge = max(0, min(T, raw));
    const int before = carry_max;
    edge = max(before, scan_max(edge, sums));
    if (s <= B) {
      if (edge != raw) atomicOr(status, kStatusBadIndex);
      lo[s] = edge;
    }
    __syncthreads();
    if (tid == kPlanThreads - 1) carry_max = edge;
    __syncthreads();
  }
  for (int s0 = 0; s0 < B; s0 += kPlanThreads) {
    const int s = s0 + tid;
    const int n = s < B ? (lo[s + 1] - lo[s] + rows - 1) / rows : 0;
    int total;
    const int at = carry_tiles + scan_add(n, sums, total);
    if (s < B) base[s] = at;
    if (n > 0) {  // `per` tiles in each of the first n / per bins, the rest in the next
      atomicAdd(&change[0], per);
      atomicSub(&change[n / per], per);
      atomicAdd(&rest[n / per], n % per);
    }
    __syncthreads();
    if (tid == 0) carry_tiles += total;
    __syncthreads();
  }
  const int tiles = min(carry_tiles, max_tiles);
  if (tid == 0) {
    table.head[0] = tiles;
    table.head[1] = lo[0];
    table.head[2] = lo[B];
    table.head[3] = 0;
  }
  int total;
  const int own = change[tid], more = rest[tid];  // read before the scan's barriers: both are overwritten after it
  const int mine = scan_add(own, sums, total) + own + more;
  change[kPlanThreads - 1 - tid] = mine;  // heaviest bin first
  __syncthreads();
  const int place = scan_add(change[tid], sums, total);
  rest[kPlanThreads - 1 - tid] = place;  // of the bin's next tile
  __syncthreads();
  for (int t = tid; t < tiles; t += kPlanThreads) {
    int a = 0, b = B - 1;  // the last sequence whose first tile is t or earlier
    while (a < b) {
      const int m = (a + b + 1) >> 1;
      if (base[m] <= t) a = m; else b = m - 1;
    }
    const int i = t - base[a];
    const int at = atomicAdd(&rest[i / per], 1);
    if (at < max_tiles) entries[at] = make_int4(lo[a], lo[a + 1], i, (lo[a + 1] - lo[a] + rows - 1) / rows);
  }
}

// ---- forward -------------------------------------------------------------------------------------------------------
// kTiles 2: a CTA per SM works on two tiles that share the K / V chunks. kTiles 1: two CTAs per SM work on a tile each,
// with half the shared memory and TMEM: they load K and V twice, but are not tied to one another's phases, which is what
// counts where an item is a chunk or two (see packed_single_tiles).
// One thread per row: with two (sixteen softmax warps that exchange their maxima) a document of 16384 tokens, 16 heads
// over 4, took 973 us instead of 885.
//
// Measured on one B200, D = 128: that document 830 us, 1320 TFLOP/s of its 4 D n (n + 1) / 2 useful operations, bound by
// the tensor cores at the clock that 1 kW leaves them; 8192 tokens in 8 sequences of 364 to 1587, 32 heads over 8, 97 us,
// 830 TFLOP/s: the diagonal chunks' hidden half and seven or eight items to a CTA cost the rest (49% of the tensor pipes'
// cycles at 1638 tokens in the mean); 4096 tokens in 48 sequences 33 us, 3.7 TB/s: an item is a chunk or two, and the
// latency of its loads, softmax and store bounds it.
template <int DP, int kTiles>
struct FwdCfg {
  static constexpr int kTileBytes = kRowsT * DP * 2;
  static constexpr int kRing = (DP == 64 ? 4 : 2) * kTiles;  // K and V chunks in turn
  static constexpr int kStage = kTiles * 4 * 4096;           // 4 KB for each softmax warp's output rows
  static constexpr int kSmem = (kTiles + kRing) * kTileBytes + kStage + 512;  // and barriers, WorkRing
  static constexpr int kSoftmaxWarps = 4 * kTiles;
  static constexpr int kThreads = 32 * (kSoftmaxWarps + 2);  // and a warp each for loads and MMAs
  static constexpr int kTmem = 256 * kTiles;                 // S of every tile, then O of every tile
  static_assert(kSmem + 1024 <= 233472 / (3 - kTiles), "the CTAs of an SM fit its 228 KB, 1 KB each reserved");
};

struct FwdArgs {
  bf16* out;   // [T, H, D]
  bf16* rest;  // [T, H, D] what out's rounding left of the output, for the backward pass, or null
  float* lse;  // [H, T] log2-domain log-sum-exp, or null
  const int4* table;  // entries of kTiles query tiles
  const int* head;
  int* taken;  // items given out
  int T, H, Hkv, D, lp;
  float scale2;  // scale times log2(e)
};

template <int DP, int kTiles>
__global__ void __launch_bounds__((FwdCfg<DP, kTiles>::kThreads), (3 - kTiles))
    packed_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_k32,
                      const __grid_constant__ CUtensorMap tm_v32, const __grid_constant__ FwdArgs p, unsigned* status) {
  using Cfg = FwdCfg<DP, kTiles>;
  constexpr int kRing = Cfg::kRing, kTileBytes = Cfg::kTileBytes;
  constexpr int kLoadWarp = Cfg::kSoftmaxWarps, kMmaWarp = kLoadWarp + 1;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* q_tiles = smem;
  uint8_t* ring = smem + kTiles * kTileBytes;
  uint8_t* stages = ring + kRing * kTileBytes;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(stages + Cfg::kStage);
  uint64_t* q_empty = q_full + 1;
  uint64_t* kv_full = q_empty + 1;
  uint64_t* kv_empty = kv_full + kRing;
  uint64_t* s_full = kv_empty + kRing;   // [2] scores of a tile's chunk are in TMEM
  uint64_t* p_ready = s_full + 2;        // [2][2] its probabilities are, by halves of the chunk's keys
  uint64_t* o_done = p_ready + 4;        // [2] P . V of the chunk is complete
  const WorkRing work(o_done + 2);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(work.empty + kWorkRing);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (misplaced(smem, status)) return;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[2 * i], 4);
      mbar_init(&p_ready[2 * i + 1], 4);
      mbar_init(&o_done[i], 1);
    }
    work.init(Cfg::kSoftmaxWarps + 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  __syncwarp();
  if (warp == 0) tmem_alloc(tmem_slot, Cfg::kTmem);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);
  pdl_trigger();
  pdl_wait();

  zero_padding(p.out, p.T, static_cast<long>(p.H) * p.D, p.head, threadIdx.x, Cfg::kThreads);
  const int group = p.H / p.Hkv;
  const int ksteps = (p.D + 15) / 16;
  const int tokens = kRowsT >> p.lp;  // of a query tile
  const int per = p.H >> p.lp;        // items of a table entry: one for every 1 << lp heads
  // an item's query tile i: its first token, its number of key chunks (the last one holds the diagonal), and the keys it
  // needs of chunk c
  auto token_of = [&](const auto& items, int i) { return items.tile.x + (items.tile.z * kTiles + i) * tokens; };
  auto chunks_of = [&](const auto& items, int i) {
    const int first = token_of(items, i);
    return i < kTiles && first < items.tile.y ? (first - items.tile.x) / kRowsT + 1 : 0;
  };
  auto keys_of = [&](const auto& items, int i, int c) {
    return min(kRowsT, min(items.tile.y, token_of(items, i) + tokens) - (items.tile.x + c * kRowsT));
  };

  if (warp == kLoadWarp) {
    // ---- loads: an item's Q, then its K and V chunks in turn ----
    Feed items(work, p.table, p.head, p.taken, per);
    const uint32_t qa = smem_u32(q_tiles), ra = smem_u32(ring);
    int it = 0;
    bool ok = true;
    for (int n_items = 0; ok && items.next(lane, status, abort_flag); ++n_items) {
      const int lo = items.tile.x, c1 = chunks_of(items, 1), n = max(chunks_of(items, 0), c1);
      const int head = items.sub << p.lp, kvh = head / group;
      const int first = token_of(items, 0), last_keys = keys_of(items, c1 > 0 ? 1 : 0, n - 1);
      if (lane == 0) {
        auto chunk = [&](int x) {  // K (even) or V (odd) of a chunk
          const int s = (it + x) % kRing, c = x >> 1;
          if (x == 2 * n - 2) items.reserve();
          if (x == 2 * n - 1) items.fetch();
          if (!mbar_wait(&kv_empty[s], (((it + x) / kRing) & 1) ^ 1, status, kStatusWaitEmpty, abort_flag)) return false;
          load_chunk<DP>(ra + s * kTileBytes, (x & 1) ? &tm_v : &tm_k, (x & 1) ? &tm_v32 : &tm_k32, &kv_full[s], kvh,
                         lo + c * kRowsT, c + 1 < n ? kRowsT : last_keys);
          return true;
        };
        // the first K does not wait for the previous item's queries to be read, nor the queries for its last V
        ok = chunk(0) && mbar_wait(q_empty, (n_items & 1) ^ 1, status, kStatusWaitEmpty, abort_flag);
        if (ok) {
          mbar_arrive_expect_tx(q_full, (c1 > 0 ? 2 : 1) * kTileBytes);
          load_tile<DP>(qa, &tm_q, q_full, head, first);
          if (c1 > 0) load_tile<DP>(qa + kTileBytes, &tm_q, q_full, head, first + tokens);
        }
        for (int x = 1; ok && x < 2 * n; ++x) ok = chunk(x);
      }
      it += 2 * n;
      ok = uniform(ok);
    }
  } else if (warp == kMmaWarp) {
    // ---- MMAs ----
    Items items(work);
    const bool leader = elect_one();
    const uint32_t qa = smem_u32(q_tiles), ra = smem_u32(ring);
    int base = 0;            // ring position of the item's first chunk
    uint32_t used[2] = {0, 0};  // chunks of tile i so far, over all items
    bool ok = true;
    auto wait_ring = [&](int it) {
      return warp_wait(&kv_full[it % kRing], (it / kRing) & 1, status, kStatusWaitFull, abort_flag);
    };
    for (int n_items = 0; ok && items.next(status, abort_flag); ++n_items) {
      const int chunks[2] = {chunks_of(items, 0), chunks_of(items, 1)};
      const int n_chunks = max(chunks[0], chunks[1]);
      const int left = items.tile.y - items.tile.x;  // keys of the sequence
      const int first0 = token_of(items, 0) - items.tile.x;
      // columns of S and rows of V that tile i takes of chunk c, in steps of 16
      auto width = [&](int i, int c) {
        return (min(kRowsT, min(left, first0 + (i + 1) * tokens) - c * kRowsT) + 15) & ~15;
      };
      ok = warp_wait(q_full, n_items & 1, status, kStatusWaitFull, abort_flag) && wait_ring(base);
      if (!ok) break;
      tc_fence_after();
      if (leader) {
        for (int i = 0; i < kTiles; ++i) {
          if (chunks[i] == 0) continue;
          mma_dims<DP>(tmem + i * 128, qa + i * kTileBytes, ra + (base % kRing) * kTileBytes, width(i, 0), ksteps);
          umma_commit(&s_full[i]);
        }
        umma_commit(&kv_empty[base % kRing]);
        if (n_chunks == 1) umma_commit(q_empty);
      }
      __syncwarp();
      for (int c = 0; ok && c < n_chunks; ++c) {
        const int v_it = base + 2 * c + 1, k_it = v_it + 1;
        const bool more = c + 1 < n_chunks;
        ok = wait_ring(v_it) && (!more || wait_ring(k_it));
        if (!ok) break;
        uint8_t* v_tile = ring + (v_it % kRing) * kTileBytes;
        if (!more) {  // rows past the sequence's end that a K step of P . V reads
          const int keys = left - c * kRowsT, widest = width(chunks[1] > 0 ? 1 : 0, c);
          if (keys < widest) zero_rows<DP>(v_tile, keys, widest, lane);
        }
        for (int i = 0; ok && i < kTiles; ++i) {
          if (c >= chunks[i]) continue;
          // the first half of P . V runs under the exponentials of the second
          ok = warp_wait(&p_ready[2 * i], (used[i] + c) & 1, status, kStatusWaitAccum, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const int vsteps = width(i, c) / 16;
          const uint32_t t_o = tmem + kTiles * 128 + i * DP, t_p = tmem + i * 128;
          const bool single = chunks[i] == 1;  // P and its rest, 16 columns each in turn
          if (leader) {
            if (single) {
              mma_rows<2, 32, 0, 4>(t_o, t_p, smem_u32(v_tile), ksteps * 16, vsteps, false);
              mma_rows<2, 32, 0, 4>(t_o, t_p + 16, smem_u32(v_tile), ksteps * 16, vsteps, true);
            } else {
              mma_rows<8, 64, 0, 4>(t_o, t_p, smem_u32(v_tile), ksteps * 16, vsteps, c > 0);
            }
          }
          __syncwarp();
          ok = warp_wait(&p_ready[2 * i + 1], (used[i] + c) & 1, status, kStatusWaitAccum, abort_flag);
          if (!ok) break;
          tc_fence_after();
          if (leader) {
            if (single) {
              mma_rows<2, 32, 4, 8>(t_o, t_p, smem_u32(v_tile), ksteps * 16, vsteps, true);
              mma_rows<2, 32, 4, 8>(t_o, t_p + 16, smem_u32(v_tile), ksteps * 16, vsteps, true);
            } else {
              mma_rows<8, 64, 4, 8>(t_o, t_p, smem_u32(v_tile), ksteps * 16, vsteps, true);
            }
            umma_commit(&o_done[i]);
            if (c + 1 < chunks[i]) {
              mma_dims<DP>(tmem + i * 128, qa + i * kTileBytes, ra + (k_it % kRing) * kTileBytes, width(i, c + 1),
                           ksteps);
              umma_commit(&s_full[i]);
            }
          }
          __syncwarp();
        }
        if (leader) {
          umma_commit(&kv_empty[v_it % kRing]);
          if (more) umma_commit(&kv_empty[k_it % kRing]);
          if (c + 2 == n_chunks) umma_commit(q_empty);  // the last scores are under way
        }
        __syncwarp();
      }
      base += 2 * n_chunks;
      used[0] += chunks[0];
      used[1] += chunks[1];
    }
  } else {
    // ---- softmax: one thread per row ----
    const int i = warp >> 2, quad = warp & 3;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const uint32_t s_addr = lane_base + i * 128, o_addr = lane_base + kTiles * 128 + i * DP;
    Items items(work);
    uint32_t used = 0;  // chunks of this tile so far, over all items
    bool ok = true;
    while (ok && items.next(status, abort_flag)) {
      const int n_mine = chunks_of(items, i);
      const int first = token_of(items, i), token = first + ((quad * 32 + lane) >> p.lp);
      // Exponentials are taken against a reference that is settled beforehand (0 for a row's first chunk): the chunk's
      // maximum is reduced beside them, and only where it lies more than kLazy above (or far below, in the first chunk,
      // where small sums would underflow) does the row take it as its reference and repeat.
      float ref = 0.f, sum = 0.f;
      auto publish = [&](int h) {
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[2 * i + h]);
      };
      if (n_mine == 1) {
        // The only chunk: its maximum first, and what P's rounding leaves beside P. 32 columns at a time, read twice.
        ok = warp_wait(&s_full[i], used & 1, status, kStatusWaitAccum, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const int limit = min(items.tile.y, token + 1) - items.tile.x, blocks = (keys_of(items, i, 0) + 31) >> 5;
        float top = -INFINITY;
#pragma unroll 1
        for (int b = 0; b < blocks; ++b) {
          float v[32];
          tmem_load32(s_addr + b * 32, v);
          const uint32_t bits = low_bits(limit - b * 32);
#pragma unroll
          for (int j = 0; j < 32; ++j) top = (bits >> j) & 1u ? fmaxf(top, v[j]) : top;
        }
        ref = top * p.scale2;
        const float shift = ref == -INFINITY ? 0.f : ref;
#pragma unroll 1
        for (int b = 0; b < blocks; ++b) {
          float v[32];
          uint32_t w[16], rest[16];
          tmem_load32(s_addr + b * 32, v);
          const uint32_t bits = low_bits(limit - b * 32);
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float x = (bits >> j) & 1u ? ex2(fmaf(v[j], p.scale2, -shift)) : 0.f;
            const float y = (bits >> (j + 1)) & 1u ? ex2(fmaf(v[j + 1], p.scale2, -shift)) : 0.f;
            sum += x + y;
            w[j / 2] = pack_bf16(x, y);
            rest[j / 2] = rest_of(w[j / 2], x, y);
          }
          tmem_st_u32x16(s_addr + b * 32, w);
          tmem_st_u32x16(s_addr + b * 32 + 16, rest);
          if (b == 1) publish(0);
        }
        if (blocks < 2) publish(0);
        publish(1);
      }
      for (int c = n_mine == 1 ? 1 : 0; c < n_mine; ++c) {
        ok = warp_wait(&s_full[i], (used + c) & 1, status, kStatusWaitAccum, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const bool masked = c == n_mine - 1;  // the diagonal and the sequence's end
        const int limit = min(items.tile.y, token + 1) - (items.tile.x + c * kRowsT);
        const bool both = !masked || keys_of(items, i, c) > 64;  // the second half of the columns holds scores
        float v[64];
        float high;
        auto scores = [&](int h) {  // 64 columns, those of hidden keys replaced, to v; their maximum to high
          tmem_load64(s_addr + h * 64, v);
          if (masked) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              const uint32_t bits = low_bits(limit - h * 64 - g * 32);
#pragma unroll
              for (int j = 0; j < 32; ++j) v[g * 32 + j] = (bits >> j) & 1u ? v[g * 32 + j] : -INFINITY;
            }
          }
          float m0 = max3(v[0], v[1], v[2]), m1 = max3(v[3], v[4], v[5]);
#pragma unroll
          for (int j = 6; j < 62; j += 4) {
            m0 = max3(m0, v[j], v[j + 1]);
            m1 = max3(m1, v[j + 2], v[j + 3]);
          }
          high = max3(fmaxf(m0, m1), v[62], v[63]);
        };
        uint32_t w[32];
        auto exponentials = [&]() {  // of v, packed to w; their sum
          const float shift = ref == -INFINITY ? 0.f : ref;
          const uint64_t scale2 = pair_of(p.scale2, p.scale2), minus = pair_of(-shift, -shift);
          uint64_t a = 0, b = 0;
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            float x0, x1, y0, y1;
            unpair(fma2(pair_of(v[2 * j], v[2 * j + 1]), scale2, minus), x0, x1);
            unpair(fma2(pair_of(v[2 * j + 2], v[2 * j + 3]), scale2, minus), y0, y1);
            x0 = ex2(x0);
            x1 = ex2(x1);
            y0 = ex2(y0);
            y1 = ex2(y1);
            a = add2(a, pair_of(x0, x1));
            b = add2(b, pair_of(y0, y1));
            w[j] = pack_bf16(x0, x1);
            w[j + 1] = pack_bf16(y0, y1);
          }
          float x, y;
          unpair(add2(a, b), x, y);
          return x + y;
        };
        scores(0);
        float top = high, part = exponentials();
        if (both) {
          scores(1);
          top = fmaxf(top, high);
        }
        top *= p.scale2;
        const bool move = top > ref + kLazy || (c == 0 && top < -kFar);
        if (__any_sync(0xffffffffu, move)) {
          const float f = move ? ex2(ref - top) : 1.f;
          if (move) ref = top;
          if (c > 0) {
            ok = warp_wait(&o_done[i], (used + c - 1) & 1, status, kStatusWaitAccum, abort_flag);
            if (!ok) break;
            tc_fence_after();
            sum *= f;
#pragma unroll 1
            for (int d = 0; d < DP; d += 16) {
              float o[16];
              tmem_ld16(o_addr + d, o);
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] *= f;
              tmem_st16(o_addr + d, o);
            }
          }
          scores(0);  // P has not overwritten them yet
          part = exponentials();
          if (both) scores(1);
        }
        tmem_store32(s_addr, w);
        publish(0);
        if (both) {
          part += exponentials();
          tmem_store32(s_addr + 32, w);
        }
        publish(1);
        sum += part;
      }
      if (!ok) break;
      if (n_mine > 0) {
        used += n_mine;
        ok = warp_wait(&o_done[i], (used - 1) & 1, status, kStatusWaitAccum, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const float inv = 1.f / sum;
        const int head = items.sub << p.lp;
        if (token < items.tile.y && p.lse != nullptr)
          p.lse[static_cast<long>(head + (lane & ((1 << p.lp) - 1))) * p.T + token] = ref + log2f(sum);
        TileOut to{p.out + (static_cast<long>(first) * p.H + head) * p.D, static_cast<long>(p.H) * p.D, p.D, p.lp,
                   (items.tile.y - first) << p.lp, p.D};
#pragma unroll 1
        for (int d = 0; d < p.D; d += 64, to.dst += 64, to.cols -= 64)
          stage_tmem64<false>(o_addr + d, inv, stages + warp * 4096, to, quad * 32, lane);
        if (p.rest != nullptr) {
          to.dst += p.rest - p.out - (p.D + 63) / 64 * 64;
          to.cols = p.D;
#pragma unroll 1
          for (int d = 0; d < p.D; d += 64, to.dst += 64, to.cols -= 64)
            stage_tmem64<true>(o_addr + d, inv, stages + warp * 4096, to, quad * 32, lane);
        }
        tc_fence_before();  // the next item's first P . V overwrites O after this warp's next p_ready
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  settle(*abort_flag != 0);
  if (warp == 0) tmem_dealloc(tmem, Cfg::kTmem);
}

template <int DP, int kTiles>
int run_fwd(const PackedMaps& maps, const PackedArgs& a, void* out, void* rest, float* lse, unsigned* status,
            cudaStream_t stream) {
  using Cfg = FwdCfg<DP, kTiles>;
  auto kernel = packed_fwd_kernel<DP, kTiles>;
  if (set_max_smem(kernel, Cfg::kSmem) != cudaSuccess) return -1;
  const FwdArgs args{static_cast<bf16*>(out), static_cast<bf16*>(rest), lse, static_cast<const int4*>(a.fwd.entries),
                     a.fwd.head, a.fwd.head + 3, a.T, a.H, a.Hkv, a.D, a.lp, a.scale * kLog2e};
  const long most = static_cast<long>(a.fwd.max_tiles) * (a.H >> a.lp);
  if (most > 0x7fff0000l) return -2;
  const long grid = std::min(most, static_cast<long>(a.num_sms) * (3 - kTiles));
  return launch_pdl(kernel, dim3(static_cast<unsigned>(grid)), dim3(Cfg::kThreads), Cfg::kSmem, stream, maps.q, maps.k,
                    maps.v, maps.k32, maps.v32, args, status) == cudaSuccess ? 0 : -1;
}

}  // namespace

int packed_max_tiles(int T, int B, int rows) {
  return static_cast<int>(std::min<long>(T, static_cast<long>(T) / rows + B));
}

int packed_heads_log2(int H, int Hkv) {
  int lp = 0;
  while (lp < 3 && (H / Hkv) % (2 << lp) == 0) ++lp;
  return lp;
}

int launch_packed_plan(const int* cu, int B, int T, const PackedTable* tables, int count, unsigned* status,
                       cudaStream_t stream) {
  if (count < 1 || count > kPlanTables) return -2;
  PlanArgs args;
  for (int i = 0; i < count; ++i) args.tables[i] = tables[i];
  return launch_pdl(packed_plan_kernel, dim3(count), dim3(kPlanThreads), 0, stream, cu, B, T, args, status) ==
                 cudaSuccess ? 0 : -1;
}

// Measured on one B200 with the plan, us for one / two tiles of 8192 tokens. D = 64, 12 heads of their own, in sequences
// of 16: 60 / 113, of 128: 20.5 / 27.0, of 1024: 32.3 / 35.7, one of 8192: 148 / 161. D = 128, 32 heads over 8, of 16: 51 /
// 95, of 64: 39.0 / 38.1, of 96: 41.7 / 44.3, of 128: 44.2 / 42.4, of 256: 49.2 / 45.0, of 384: 56.7 / 51.1, of 512: 65.3 /
// 58.2, of 1024: 91.4 / 79.7, one of 8192: 500 / 450. At D = 128 they cross near 100 tokens; the rule keeps one tile up to
// a mean of 511, at a cost of 4 to 11%. The mean says little of mixed lengths: one sequence of 8000 beside 24 of 8 counts
// as short ones and takes 530 us where two tiles take 475; one of 4096 beside 256 of 16 is even (181 / 185).
bool packed_single_tiles(int T, int B, int D) { return D <= 64 || static_cast<long>(T) < 512l * B; }

int launch_packed_forward(const PackedMaps& maps, const PackedArgs& a, void* out, void* rest, float* lse, int tiles,
                          unsigned* status, cudaStream_t stream) {
  if (tiles == 1)
    return a.D <= 64 ? run_fwd<64, 1>(maps, a, out, rest, lse, status, stream)
                     : run_fwd<128, 1>(maps, a, out, rest, lse, status, stream);
  return a.D <= 64 ? run_fwd<64, 2>(maps, a, out, rest, lse, status, stream)
                   : run_fwd<128, 2>(maps, a, out, rest, lse, status, stream);
}

}  // namespace ecz
