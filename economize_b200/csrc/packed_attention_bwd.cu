// Gradients of the packed causal attention (packed_attention.cu).
//
//   d_i = do_i . o_i      p_ij = exp(s_ij - L_i)      ds_ij = p_ij (do_i . v_j - d_i)
//   dv_j = sum_i p_ij do_i      dk_j = scale sum_i ds_ij q_i      dq_i = scale sum_j ds_ij k_j
//
// Two kernels, one per reduction axis, so every sum has one owner and a fixed order: no atomics, the same bits every
// time, and the shared heads of a group add up inside a CTA. The price is that s and do . v are computed twice (seven
// tile products instead of five).
//
// dkv  CTA: 128 keys of one K/V head; walks the query tiles from the diagonal to the sequence's end for every query
//      head of the group. S^T = K Q^T and dP^T = V dO^T put keys on the TMEM lanes, so P^T and dS^T are the A operands
//      of dV += P^T dO and dK += dS^T Q where they lie (bf16 over the fp32 scores they came from): nothing of a
//      128 x 128 tile passes through shared memory. TMEM: S, dP, dV, dK of 128 columns each, all 512. The tensor cores
//      run dV and the next S while the threads turn dP into dS, and dK and the next dP while they turn S into P.
// dq   CTA: a tile of queries, as in the forward pass; walks the key chunks up to the diagonal. S (two buffers), dP and
//      dQ in TMEM; dS is dQ's A operand where S was.
//
// P^T and dS^T (dS) are rounded to bf16 once, as operands: the other factor of their products is bf16, and kind::f16 takes
// both of one type. Those roundings are independent from entry to entry, so over a row's keys they add up to less than
// the rounding of the bf16 result: gradients are 0.0024 of themselves from their 64-bit values where products of 32-bit
// operands are 0.0017 from them. The rest of P that the forward pass multiplies for tiles of one chunk would cost a product
// more here. The log-sum-exp, delta and all sums are fp32.
//
// Measured on one B200, D = 128. One sequence of 16384 tokens, 16 heads over 4: dkv 1600 us, 1370 TFLOP/s of its four
// products' useful operations, dq 1340 us, 1230 of its three: the tensor cores at the clock that 1 kW leaves them (the
// forward pass's S once more, computed by both, is the price of the fixed order). 8192 tokens in 5 sequences, 32 heads
// over 8: dkv 336 us with the tensor pipes busy 67% of the cycles, dq 303 us and 52%: the exponentials (16 a cycle and
// SM) and, in dq, the end of every item. 4096 tokens in 48 sequences: 42 and 36 us, an item being a chunk or two whose
// loads, two products deep, and stores stand one after another. delta: 16 and 33 us, the copy bandwidth.
#include <algorithm>

#include "launchers.h"
#include "packed_common.cuh"

namespace ecz {

using namespace packed;

namespace {

// Warp 0 loads, 1 issues, 2 fetches row statistics (dkv) or loads Q and dO (dq); sixteen compute warps, so that four per
// scheduler hide the latencies of the tile's short phases (eight with twice the columns each spent 3000 of 4700 cycles
// per tile in them).
constexpr int kComputeWarps = 16;
constexpr int kBwdThreads = 128 + 32 * kComputeWarps;

struct BwdArgs {
  bf16 *dq, *dk, *dv;
  const float *lse, *delta;  // [H, T]
  const int4 *dq_table, *dkv_table;  // tiles of queries, tiles of 128 keys
  const int *dq_head, *dkv_head;
  int* taken;  // [2] items given out: key tiles, query tiles
  int T, H, Hkv, D, lp;
  float scale, scale2;
  int splits;   // CTAs that share the query tiles of a key tile
  float* part;  // [splits, 2 (dV, dK), T, Hkv, D] their sums where splits > 1
};

// delta[h, t] = dout[t, h] . (out[t, h] + rest[t, h]); 16 lanes per row. dp - delta cancels where a row attends few keys:
// with the output rounded to bf16 alone, dQ and dK of sequences of a few tokens were off by 0.8% (5 times their own
// rounding), so the forward pass keeps what its rounding leaves.
__global__ void __launch_bounds__(256) packed_delta_kernel(const bf16* __restrict__ out, const bf16* __restrict__ rest,
                                                           const bf16* __restrict__ dout, int* __restrict__ taken,
                                                           long stride_t, long stride_h, int T, int H, int D,
                                                           float* __restrict__ delta) {
  pdl_trigger();
  pdl_wait();
  if (blockIdx.x == 0 && threadIdx.x < 2) taken[threadIdx.x] = 0;  // by the kernels that follow
  const long row = (static_cast<long>(blockIdx.x) * 256 + threadIdx.x) >> 4;
  const int c = (threadIdx.x & 15) * 8;
  const bool real = row < static_cast<long>(T) * H;
  const long t = real ? row / H : 0;
  const int h = real ? static_cast<int>(row % H) : 0;
  float acc = 0.f;
  if (real && c < D) {
    const uint4 a = *reinterpret_cast<const uint4*>(out + row * D + c);
    const uint4 b = *reinterpret_cast<const uint4*>(dout + t * stride_t + h * stride_h + c);
    const uint4 r = *reinterpret_cast<const uint4*>(rest + row * D + c);
    const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w}, z[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 u = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x[k]));
      const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&y[k]));
      const float2 l = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&z[k]));
      acc = fmaf(u.x + l.x, v.x, acc);
      acc = fmaf(u.y + l.y, v.y, acc);
    }
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  if (real && c == 0) delta[static_cast<long>(h) * T + t] = acc;
}

template <int DP>
struct BwdCfg {
  static constexpr int kTileBytes = kRowsT * DP * 2;
  static constexpr int kRing = DP == 64 ? 10 : 5;  // streamed tiles
  static constexpr int kStatRing = 3;
  static constexpr int kStats = 2 * 128 * 4;  // -lse and -delta of a query tile
  static constexpr int kSmem = (2 + kRing) * kTileBytes + (DP == 64 ? kStatRing : 2) * kStats + 512;
  static_assert(kSmem <= 232448, "227 KB of shared memory");
};

// The stream of tiles of a backward kernel: item 2 i + which, ring slot item % kRing.
template <int DP>
struct Stream {
  static constexpr int kRing = BwdCfg<DP>::kRing;
  uint8_t* tiles;
  uint64_t *full, *empty;
  __device__ __forceinline__ uint8_t* tile(int item) const { return tiles + (item % kRing) * BwdCfg<DP>::kTileBytes; }
  __device__ __forceinline__ uint64_t* full_of(int item) const { return &full[item % kRing]; }
  __device__ __forceinline__ uint64_t* empty_of(int item) const { return &empty[item % kRing]; }
  __device__ __forceinline__ uint32_t use(int item) const { return (item / kRing) & 1; }
};

// The query tiles that see a key tile, in order: `tiles` of one pack of heads, then the next pack's. Counters instead of
// a division of the iteration: that took the issuing warp a tenth of a tile's time.
struct Walk {
  int head, token;  // first head of the pack, first token of the tile
  int left, tiles, token0, tokens, heads;
  __device__ __forceinline__ Walk(int first_head, int first_token, int n, int lp)
      : head(first_head), token(first_token), left(n), tiles(n), token0(first_token), tokens(kRowsT >> lp),
        heads(1 << lp) {}
  __device__ __forceinline__ void skip(int n) {
    head += n / tiles * heads;
    token += n % tiles * tokens;
    left -= n % tiles;
  }
  __device__ __forceinline__ void next() {
    token += tokens;
    if (--left == 0) {
      left = tiles;
      token = token0;
      head += heads;
    }
  }
};

// ---- dK and dV -----------------------------------------------------------------------------------------------------
// kSplit: p.splits CTAs share the query tiles of a key tile and leave their sums, in fp32, to packed_join_kernel.
template <int DP, bool kSplit>
__global__ void __launch_bounds__(kBwdThreads, 1)
    packed_dkv_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
                      const __grid_constant__ BwdArgs p, unsigned* status) {
  using Cfg = BwdCfg<DP>;
  constexpr int kRing = Cfg::kRing, kTileBytes = Cfg::kTileBytes, kStatRing = DP == 64 ? Cfg::kStatRing : 2;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t *k_tile = smem, *v_tile = smem + kTileBytes;
  float* stats = reinterpret_cast<float*>(smem + (2 + kRing) * kTileBytes);  // stage s: -lse [128], -delta [128]
  uint64_t* kv_full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(stats) + kStatRing * Cfg::kStats);
  Stream<DP> ring{smem + 2 * kTileBytes, kv_full + 1, kv_full + 1 + kRing};
  uint64_t* st_full = kv_full + 1 + 2 * kRing;
  uint64_t* st_empty = st_full + kStatRing;
  uint64_t* s_full = st_empty + kStatRing;
  uint64_t* p_ready = s_full + 1;  // [2], by halves of every warp's queries
  uint64_t* dp_full = p_ready + 2;
  uint64_t* ds_ready = dp_full + 1;
  uint64_t* done = ds_ready + 1;
  uint64_t* kv_empty = done + 1;
  const WorkRing work(kv_empty + 1);  // an even number of barriers: on 16 bytes
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(work.empty + kWorkRing);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (misplaced(smem, status)) return;
  if (threadIdx.x == 0) {
    mbar_init(kv_full, 1);
    mbar_init(kv_empty, 1);
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&ring.full[i], 1);
      mbar_init(&ring.empty[i], 1);
    }
    for (int i = 0; i < kStatRing; ++i) {
      mbar_init(&st_full[i], 1);
      mbar_init(&st_empty[i], kComputeWarps);
    }
    mbar_init(s_full, 1);
    mbar_init(&p_ready[0], kComputeWarps);
    mbar_init(&p_ready[1], kComputeWarps);
    mbar_init(dp_full, 1);
    mbar_init(ds_ready, kComputeWarps);
    mbar_init(done, 1);
    work.init(kComputeWarps + 2);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    tma_prefetch_desc(&tm_do);
  }
  __syncwarp();
  if (warp == 0) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);
  const uint32_t t_s = tmem, t_dp = tmem + 128, t_dv = tmem + 256, t_dk = tmem + 384;
  pdl_trigger();
  pdl_wait();

  if (!kSplit && warp >= 4) {
    zero_padding(p.dk, p.T, static_cast<long>(p.Hkv) * p.D, p.dkv_head, threadIdx.x - 128, kComputeWarps * 32);
    zero_padding(p.dv, p.T, static_cast<long>(p.Hkv) * p.D, p.dkv_head, threadIdx.x - 128, kComputeWarps * 32);
  }
  const int splits = kSplit ? p.splits : 1;
  const int group = p.H / p.Hkv;
  const int ksteps = (p.D + 15) / 16;
  const int tokens = kRowsT >> p.lp, packs = group >> p.lp;
  // What an item stands for: its K/V head and split, first key (the entry's weight counts from the sequence's end), the
  // query tiles that see it, and its iterations over them (of every pack of heads).
  struct Keys {
    int kvh, split, key0, end, tiles, first, total;
    __device__ __forceinline__ Keys(const int4& tile, int sub, int splits, int tokens, int packs) {
      kvh = sub / splits;
      split = sub - kvh * splits;
      end = tile.y;
      key0 = tile.x + (tile.w - tile.z - 1) * kRowsT;
      tiles = (end - key0 + tokens - 1) / tokens;
      first = 0;
      total = packs * tiles;
      if (kSplit) {
        const long all = total;
        first = static_cast<int>(all * split / splits);
        total = static_cast<int>(all * (split + 1) / splits) - first;
      }
    }
    __device__ __forceinline__ Walk walk(int group, int lp) const {
      Walk at(kvh * group, key0, tiles, lp);
      if (kSplit) at.skip(first);
      return at;
    }
  };

  if (warp == 0) {
    int x = 0;  // ring item
    bool ok = true;
    Feed items(work, p.dkv_table, p.dkv_head, p.taken, p.Hkv * splits);
    int n_loaded = 0;  // items with anything to load
    while (ok && items.next(lane, status, abort_flag)) {
      const Keys keys(items.tile, items.sub, splits, tokens, packs);
      const int total = keys.total;
      if (kSplit && total == 0) {
        if (lane == 0) {
          items.reserve();
          items.fetch();
        }
        continue;
      }
      if (lane == 0) {
        Walk at = keys.walk(group, p.lp);
        auto load = [&](int i) {  // Q (even) or dO (odd) of an iteration
          if (i == 2 * total - 2) items.reserve();
          if (i == 2 * total - 1) items.fetch();
          if (!mbar_wait(ring.empty_of(x + i), ring.use(x + i) ^ 1, status, kStatusWaitEmpty, abort_flag)) return false;
          mbar_arrive_expect_tx(ring.full_of(x + i), kTileBytes);
          load_tile<DP>(smem_u32(ring.tile(x + i)), (i & 1) ? &tm_do : &tm_q, ring.full_of(x + i), at.head, at.token);
          if (i & 1) at.next();
          return true;
        };
        // the first query tile does not wait for the previous item's keys to be read
        ok = load(0) && load(1) && mbar_wait(kv_empty, (n_loaded & 1) ^ 1, status, kStatusWaitEmpty, abort_flag);
        if (ok) {
          mbar_arrive_expect_tx(kv_full, 2 * kTileBytes);
          load_tile<DP>(smem_u32(k_tile), &tm_k, kv_full, keys.kvh, keys.key0);
          load_tile<DP>(smem_u32(v_tile), &tm_v, kv_full, keys.kvh, keys.key0);
        }
        for (int i = 2; ok && i < 2 * total; ++i) ok = load(i);
      }
      x += 2 * total;
      ++n_loaded;
      ok = uniform(ok);
    }
  } else if (warp == 1) {
    const bool leader = elect_one();
    const uint32_t ka = smem_u32(k_tile), va = smem_u32(v_tile);
    int base = 0;  // iterations before the item
    bool ok = true;
    Items items(work);
    int n_items = 0;  // with anything to multiply
    while (ok && items.next(status, abort_flag)) {
      const Keys keys(items.tile, items.sub, splits, tokens, packs);
      const int hi = keys.end, total = keys.total;
      if (kSplit && total == 0) continue;
      // rows of the query tile at `token`, all 128 or up to the sequence's end
      auto rows_of = [&](int token) { return min(kRowsT, (hi - token) << p.lp); };
      // ring item x, of the query tile at `token`, is in shared memory and its rows past the sequence's end are zeroed
      auto ready = [&](int x, int token) {
        if (!warp_wait(ring.full_of(x), ring.use(x), status, kStatusWaitFull, abort_flag)) return false;
        const int n = rows_of(token), n16 = (n + 15) & ~15;
        if (n != n16) zero_rows<DP>(ring.tile(x), n, n16, lane);
        return true;
      };
      Walk at = keys.walk(group, p.lp);
      int rows16 = (rows_of(at.token) + 15) & ~15;  // of the current iteration's query tile
      ok = ready(2 * base, at.token) && ready(2 * base + 1, at.token) &&
           warp_wait(kv_full, n_items & 1, status, kStatusWaitFull, abort_flag);
      tc_fence_after();
      if (ok && leader) {
        mma_dims<DP>(t_s, ka, smem_u32(ring.tile(2 * base)), rows16, ksteps);
        umma_commit(s_full);
        mma_dims<DP>(t_dp, va, smem_u32(ring.tile(2 * base + 1)), rows16, ksteps);
        umma_commit(dp_full);
        if (total == 1) umma_commit(kv_empty);
      }
      __syncwarp();
      for (int it = base; ok && it < base + total; ++it) {
        const bool more = it + 1 < base + total;
        const int xq = 2 * it, xd = xq + 1;
        at.next();
        const int next16 = (rows_of(at.token) + 15) & ~15;
        if (more) ok = ready(xq + 2, at.token);
        // the first half of dV runs under the exponentials of the second
        ok = ok && warp_wait(&p_ready[0], it & 1, status, kStatusWaitAccum, abort_flag);
        if (!ok) break;
        tc_fence_after();
        if (leader)
          mma_rows<2, 32, 0, 8, 2>(t_dv, t_s, smem_u32(ring.tile(xd)), ksteps * 16, rows16 / 16, it > base);
        __syncwarp();
        ok = warp_wait(&p_ready[1], it & 1, status, kStatusWaitAccum, abort_flag);
        if (!ok) break;
        tc_fence_after();
        if (leader) {
          mma_rows<2, 32, 1, 8, 2>(t_dv, t_s, smem_u32(ring.tile(xd)), ksteps * 16, rows16 / 16, true);
          umma_commit(ring.empty_of(xd));
          if (more) {
            mma_dims<DP>(t_s, ka, smem_u32(ring.tile(xq + 2)), next16, ksteps);
            umma_commit(s_full);
          }
        }
        __syncwarp();
        if (more) ok = ready(xd + 2, at.token);
        ok = ok && warp_wait(ds_ready, it & 1, status, kStatusWaitAccum, abort_flag);
        if (!ok) break;
        tc_fence_after();
        if (leader) {
          mma_rows<2, 32>(t_dk, t_dp, smem_u32(ring.tile(xq)), ksteps * 16, rows16 / 16, it > base);
          umma_commit(ring.empty_of(xq));
          if (more) {
            mma_dims<DP>(t_dp, va, smem_u32(ring.tile(xd + 2)), next16, ksteps);
            umma_commit(dp_full);
            if (it + 2 == base + total) umma_commit(kv_empty);  // the last use of K and V is under way
          } else {
            umma_commit(done);
          }
        }
        __syncwarp();
        rows16 = next16;
      }
      base += total;
      ++n_items;
    }
  } else if (warp == 2) {
    // ---- -lse and -delta of the query tiles ----
    int base = 0;
    bool ok = true;
    Items items(work);
    while (ok && items.next(status, abort_flag)) {
      const Keys keys(items.tile, items.sub, splits, tokens, packs);
      const int hi = keys.end, total = keys.total;
      Walk at = keys.walk(group, p.lp);
      for (int it = base; it < base + total; ++it, at.next()) {
        const int s = it % kStatRing;
        ok = warp_wait(&st_empty[s], ((it / kStatRing) & 1) ^ 1, status, kStatusWaitEmpty, abort_flag);
        if (!ok) break;
        float* dst = stats + s * 256;
#pragma unroll
        for (int j = lane; j < kRowsT; j += 32) {
          const int token = at.token + (j >> p.lp);
          const long from = static_cast<long>(at.head + (j & ((1 << p.lp) - 1))) * p.T + token;
          dst[j] = token < hi ? -p.lse[from] : 0.f;
          dst[128 + j] = token < hi ? -p.delta[from] : 0.f;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&st_full[s]);
      }
      base += total;
    }
  } else if (warp >= 4) {
    // ---- P^T and dS^T: one thread per key and quarter of the queries ----
    const int part = (warp - 4) >> 2, quad = warp & 3;
    const int key = quad * 32 + lane;  // relative to key0
    const uint32_t lane_base = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t s_addr = t_s + lane_base + part * 32, dp_addr = t_dp + lane_base + part * 32;
    int base = 0;
    bool ok = true;
    Items items(work);
    int n_items = 0;  // with anything summed
    while (ok && items.next(status, abort_flag)) {
      const Keys keys(items.tile, items.sub, splits, tokens, packs);
      const int hi = keys.end, key0 = keys.key0, kvh = keys.kvh, total = keys.total;
      Walk at = keys.walk(group, p.lp);
      for (int it = base; it < base + total; ++it, at.next()) {
        const int s = it % kStatRing;
        const float* lse = stats + s * 256 + part * 32;
        const float* delta = lse + 128;
        ok = warp_wait(&st_full[s], (it / kStatRing) & 1, status, kStatusWaitFull, abort_flag) &&
             warp_wait(s_full, it & 1, status, kStatusWaitAccum, abort_flag);
        if (!ok) break;
        tc_fence_after();
        float v[32];
        tmem_load32(s_addr, v);
        // rows [from, to) of this part see the key: from its own token on, up to the sequence's end
        const int from = ((key0 + key - at.token) << p.lp) - part * 32, to = ((hi - at.token) << p.lp) - part * 32;
        const bool masked = at.token < key0 + kRowsT || to < 32;
        const uint32_t seen = low_bits(to) & ~low_bits(from);
        const uint64_t scale2 = pair_of(p.scale2, p.scale2);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t w[8];
#pragma unroll
          for (int j = h * 16; j < h * 16 + 16; j += 4) {
            const float4 l = *reinterpret_cast<const float4*>(lse + j);
            unpair(fma2(pair_of(v[j], v[j + 1]), scale2, pair_of(l.x, l.y)), v[j], v[j + 1]);
            unpair(fma2(pair_of(v[j + 2], v[j + 3]), scale2, pair_of(l.z, l.w)), v[j + 2], v[j + 3]);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[j + e] = ex2(v[j + e]);
          }
          if (masked) {
#pragma unroll
            for (int j = h * 16; j < h * 16 + 16; ++j) v[j] = (seen >> j) & 1u ? v[j] : 0.f;
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) w[j] = pack_bf16(v[h * 16 + 2 * j], v[h * 16 + 2 * j + 1]);
          tmem_st_u32x8(s_addr + h * 8, w);
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_ready[h]);
        }
        ok = warp_wait(dp_full, it & 1, status, kStatusWaitAccum, abort_flag);
        if (!ok) break;
        tc_fence_after();
        float g[32];
        tmem_load32(dp_addr, g);
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          const float4 d = *reinterpret_cast<const float4*>(delta + j);
          unpair(mul2(pair_of(v[j], v[j + 1]), add2(pair_of(g[j], g[j + 1]), pair_of(d.x, d.y))), g[j], g[j + 1]);
          unpair(mul2(pair_of(v[j + 2], v[j + 3]), add2(pair_of(g[j + 2], g[j + 3]), pair_of(d.z, d.w))), g[j + 2],
                 g[j + 3]);
        }
        uint32_t w[16];
        if (masked) {
#pragma unroll
          for (int j = 0; j < 32; ++j) g[j] = (seen >> j) & 1u ? g[j] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) w[j] = pack_bf16(g[2 * j], g[2 * j + 1]);
        tmem_st_u32x16(dp_addr, w);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(ds_ready);
          mbar_arrive(&st_empty[s]);
        }
      }
      base += total;
      if (!kSplit || total > 0) {
        ok = ok && warp_wait(done, n_items & 1, status, kStatusWaitAccum, abort_flag);
        ++n_items;
      }
      if (!ok) break;
      tc_fence_after();
      constexpr int kCols = DP / 2;  // of a warp
      const int col = (part & 1) * kCols;
      if (col < p.D) {
        const bool values = part < 2;
        const uint32_t t_sum = (values ? t_dv : t_dk) + lane_base + col;
        const long stride = static_cast<long>(p.Hkv) * p.D;
        const long at0 = key0 * stride + static_cast<long>(kvh) * p.D + col;
        if (!kSplit) {
#pragma unroll
          for (int d = 0; d < kCols; d += 32) {
            const TileOut to{(values ? p.dv : p.dk) + at0 + d, stride, 0, 0, hi - key0, p.D - col - d};
            uint4 c[4];
            load_packed(t_sum + d, values ? 1.f : p.scale, c);
            store_rows(c, to, quad * 32, lane);
          }
        } else {  // this split's sum, fp32, or zeros of a split without query tiles
          const long sums = static_cast<long>(keys.split) * 2 + (values ? 0 : 1);
          float* dst = p.part + sums * p.T * stride + at0 + key * stride;
#pragma unroll 1
          for (int d = 0; d < kCols; d += 16) {
            float o[16];
            if (total > 0) tmem_ld16(t_sum + d, o);
#pragma unroll
            for (int j = 0; j < 16; j += 4)
              if (key0 + key < hi && col + d + j < p.D)
                *reinterpret_cast<float4*>(dst + d + j) =
                    total > 0 ? make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]) : make_float4(0.f, 0.f, 0.f, 0.f);
          }
        }
      }
      tc_fence_before();  // the next item's first dV overwrites this one's after this warp's next p_ready
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  settle(*abort_flag != 0);
  if (warp == 0) tmem_dealloc(tmem, 512);
}

// dV and dK from the splits' sums, in split order; rows outside the sequences are zero.
__global__ void __launch_bounds__(256) packed_join_kernel(const __grid_constant__ BwdArgs p) {
  pdl_trigger();
  pdl_wait();
  const long stride = static_cast<long>(p.Hkv) * p.D, size = p.T * stride;
  const long i = (static_cast<long>(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (i >= size) return;
  const int token = static_cast<int>(i / stride);
  const bool inside = token >= p.dkv_head[1] && token < p.dkv_head[2];
  const int which = blockIdx.y;  // 0: dV, 1: dK
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (inside) {
    for (int s = 0; s < p.splits; ++s) {
      const float4 v = *reinterpret_cast<const float4*>(p.part + (static_cast<long>(s) * 2 + which) * size + i);
      acc.x += v.x;
      acc.y += v.y;
      acc.z += v.z;
      acc.w += v.w;
    }
  }
  const float f = which ? p.scale : 1.f;
  *reinterpret_cast<uint2*>((which ? p.dk : p.dv) + i) =
      make_uint2(pack_bf16(acc.x * f, acc.y * f), pack_bf16(acc.z * f, acc.w * f));
}

// ---- dQ --------------------------------------------------------------------------------------------------------------
// The chunks of a persistent CTA's items in one row: `chunk` of the item's `n`, counted over all items by `k`. The
// issuing warp follows them twice, scores one chunk ahead of dP and dQ, across items.
struct ChunkWalk {
  Items items;
  int chunk, n, k, item, lp;
  bool valid;
  unsigned* status;
  volatile int* abort_flag;
  __device__ __forceinline__ ChunkWalk(const WorkRing& work, int lp_, unsigned* st, volatile int* ab)
      : items(work), k(0), item(-1), lp(lp_), status(st), abort_flag(ab) {
    take();
  }
  __device__ __forceinline__ void take() {
    valid = items.next(status, abort_flag);
    chunk = 0;
    ++item;
    n = items.tile.z * (kRowsT >> lp) / kRowsT + 1;  // key chunks, the last one on the diagonal
  }
  __device__ __forceinline__ void step() {
    ++k;
    if (++chunk == n) take();
  }
  __device__ __forceinline__ bool first() const { return chunk == 0; }
  __device__ __forceinline__ bool last() const { return chunk + 1 == n; }
  __device__ __forceinline__ int lo() const { return items.tile.x; }
  __device__ __forceinline__ int hi() const { return items.tile.y; }
  __device__ __forceinline__ int token() const { return items.tile.x + items.tile.z * (kRowsT >> lp); }
  __device__ __forceinline__ int head() const { return items.sub << lp; }
  // keys of the sequence from the chunk on, and those the tile needs of it, in steps of 16
  __device__ __forceinline__ int keys() const { return hi() - (lo() + chunk * kRowsT); }
  __device__ __forceinline__ int width() const {
    return (min(kRowsT, min(hi(), token() + (kRowsT >> lp)) - (lo() + chunk * kRowsT)) + 15) & ~15;
  }
};

template <int DP>
__global__ void __launch_bounds__(kBwdThreads, 1)
    packed_dq_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
                     const __grid_constant__ CUtensorMap tm_k32, const __grid_constant__ CUtensorMap tm_v32,
                     const __grid_constant__ BwdArgs p, unsigned* status) {
  using Cfg = BwdCfg<DP>;
  constexpr int kRing = Cfg::kRing, kTileBytes = Cfg::kTileBytes;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t *q_tile = smem, *do_tile = smem + kTileBytes;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + (2 + kRing) * kTileBytes);
  Stream<DP> ring{smem + 2 * kTileBytes, q_full + 1, q_full + 1 + kRing};
  uint64_t* s_full = q_full + 1 + 2 * kRing;  // [2], of the S buffer of even and odd chunks
  uint64_t* dp_full = s_full + 2;
  uint64_t* ds_ready = dp_full + 1;
  uint64_t* dq_full = ds_ready + 1;  // an item's dQ is complete
  uint64_t* dq_free = dq_full + 1;   // and in registers
  uint64_t* q_empty = dq_free + 1;   // an item's last scores are computed: Q may be overwritten, some time before dO
  uint64_t* do_full = q_empty + 1;
  uint64_t* do_empty = do_full + 1;
  const WorkRing work(do_empty + 1);  // an even number of barriers: on 16 bytes
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(work.empty + kWorkRing);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (misplaced(smem, status)) return;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&ring.full[i], 1);
      mbar_init(&ring.empty[i], 1);
    }
    mbar_init(&s_full[0], 1);
    mbar_init(&s_full[1], 1);
    mbar_init(dp_full, 1);
    mbar_init(ds_ready, kComputeWarps);
    mbar_init(dq_full, 1);
    mbar_init(dq_free, kComputeWarps);
    mbar_init(q_empty, 1);
    mbar_init(do_full, 1);
    mbar_init(do_empty, 1);
    work.init(kComputeWarps + 3);  // the issuing warp follows the items twice
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    tma_prefetch_desc(&tm_do);
    tma_prefetch_desc(&tm_k32);
    tma_prefetch_desc(&tm_v32);
  }
  __syncwarp();
  if (warp == 0) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(*tmem_slot);
  const uint32_t t_s = tmem, t_dp = tmem + 256, t_dq = tmem + 384;  // S: two buffers of 128 columns
  pdl_trigger();
  pdl_wait();

  if (warp >= 4)
    zero_padding(p.dq, p.T, static_cast<long>(p.H) * p.D, p.dq_head, threadIdx.x - 128, kComputeWarps * 32);
  const int group = p.H / p.Hkv;
  const int ksteps = (p.D + 15) / 16;

  if (warp == 0) {
    // ---- loads of K and V ----
    Feed items(work, p.dq_table, p.dq_head, p.taken + 1, p.H >> p.lp);
    const int tokens = kRowsT >> p.lp;
    int x = 0;  // ring item
    bool ok = true;
    while (ok && items.next(lane, status, abort_flag)) {
      const int lo = items.tile.x, n = items.tile.z * tokens / kRowsT + 1, kvh = (items.sub << p.lp) / group;
      const int token = lo + items.tile.z * tokens;
      const int last = min(items.tile.y, token + tokens) - (lo + (n - 1) * kRowsT);  // keys of the last chunk
      if (lane == 0) {
        for (int i = 0; ok && i < 2 * n; ++i) {  // K (even) or V (odd) of a chunk
          if (i == 2 * n - 2) items.reserve();
          if (i == 2 * n - 1) items.fetch();
          ok = mbar_wait(ring.empty_of(x + i), ring.use(x + i) ^ 1, status, kStatusWaitEmpty, abort_flag);
          if (ok)
            load_chunk<DP>(smem_u32(ring.tile(x + i)), (i & 1) ? &tm_v : &tm_k, (i & 1) ? &tm_v32 : &tm_k32,
                           ring.full_of(x + i), kvh, lo + (i >> 1) * kRowsT, (i >> 1) + 1 < n ? kRowsT : last);
        }
      }
      x += 2 * n;
      ok = uniform(ok);
    }
  } else if (warp == 2) {
    // ---- loads of Q and dO: not behind a K or V that waits for its place ----
    Items items(work);
    const int tokens = kRowsT >> p.lp;
    bool ok = true;
    for (int n_items = 0; ok && items.next(status, abort_flag); ++n_items) {
      const int head = items.sub << p.lp, token = items.tile.x + items.tile.z * tokens;
      if (lane == 0) {
        const uint32_t turn = (n_items & 1) ^ 1;
        ok = mbar_wait(q_empty, turn, status, kStatusWaitEmpty, abort_flag);
        if (ok) {
          mbar_arrive_expect_tx(q_full, kTileBytes);
          load_tile<DP>(smem_u32(q_tile), &tm_q, q_full, head, token);
        }
        ok = ok && mbar_wait(do_empty, turn, status, kStatusWaitEmpty, abort_flag);
        if (ok) {
          mbar_arrive_expect_tx(do_full, kTileBytes);
          load_tile<DP>(smem_u32(do_tile), &tm_do, do_full, head, token);
        }
      }
      ok = uniform(ok);
    }
  } else if (warp == 1) {
    const bool leader = elect_one();
    const uint32_t qa = smem_u32(q_tile), da = smem_u32(do_tile);
    auto scores = [&](ChunkWalk& a) {  // S of a chunk into its buffer; K rows past the end zeroed
      if (!a.valid) return true;
      if (a.first() && !warp_wait(q_full, a.item & 1, status, kStatusWaitFull, abort_flag)) return false;
      const int x = 2 * a.k;
      if (!warp_wait(ring.full_of(x), ring.use(x), status, kStatusWaitFull, abort_flag)) return false;
      if (a.keys() < a.width()) zero_rows<DP>(ring.tile(x), a.keys(), a.width(), lane);
      tc_fence_after();
      if (leader) {
        mma_dims<DP>(t_s + (a.k & 1) * 128, qa, smem_u32(ring.tile(x)), a.width(), ksteps);
        umma_commit(&s_full[a.k & 1]);
        if (a.last()) umma_commit(q_empty);
      }
      __syncwarp();
      a.step();
      return true;
    };
    ChunkWalk a(work, p.lp, status, abort_flag), c(work, p.lp, status, abort_flag);
    bool ok = scores(a);
    if (ok && c.valid) {
      ok = warp_wait(do_full, 0, status, kStatusWaitFull, abort_flag) &&
           warp_wait(ring.full_of(1), 0, status, kStatusWaitFull, abort_flag);
      tc_fence_after();
      if (ok && leader) {
        mma_dims<DP>(t_dp, da, smem_u32(ring.tile(1)), c.width(), ksteps);
        umma_commit(dp_full);
        umma_commit(ring.empty_of(1));
        if (c.last()) umma_commit(do_empty);
      }
      __syncwarp();
    }
    while (ok && c.valid) {
      const int k = c.k, width = c.width();
      const bool first = c.first(), last = c.last();
      const int item = c.item;
      c.step();
      // while the threads work on chunk k: S of the next, and its V is waited for
      if (c.valid) {
        ok = scores(a) && warp_wait(ring.full_of(2 * k + 3), ring.use(2 * k + 3), status, kStatusWaitFull, abort_flag);
        if (ok && c.first()) ok = warp_wait(do_full, c.item & 1, status, kStatusWaitFull, abort_flag);
      }
      if (ok && first && item > 0) ok = warp_wait(dq_free, (item - 1) & 1, status, kStatusWaitAccum, abort_flag);
      ok = ok && warp_wait(ds_ready, k & 1, status, kStatusWaitAccum, abort_flag);
      if (!ok) break;
      tc_fence_after();
      if (leader) {
        if (c.valid) {
          mma_dims<DP>(t_dp, da, smem_u32(ring.tile(2 * k + 3)), c.width(), ksteps);
          umma_commit(dp_full);
          umma_commit(ring.empty_of(2 * k + 3));
          if (c.last()) umma_commit(do_empty);
        }
        mma_rows<2, 32>(t_dq, t_s + (k & 1) * 128, smem_u32(ring.tile(2 * k)), ksteps * 16, width / 16, !first);
        umma_commit(ring.empty_of(2 * k));
        if (last) umma_commit(dq_full);
      }
      __syncwarp();
    }
  } else if (warp >= 4) {
    // ---- dS: one thread per query and quarter of the chunk's keys ----
    const int part = (warp - 4) >> 2, quad = warp & 3;
    const uint32_t lane_base = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t dp_addr = t_dp + lane_base + part * 32;
    ChunkWalk at(work, p.lp, status, abort_flag);
    bool ok = true;
    float lse = 0.f, delta = 0.f;
    // An item's dQ is stored after the first chunk of the next: the product has ended by then, and the next one waits
    // for these loads at most. A quarter of the columns to a warp (by halves of the warps it took twice as long).
    constexpr int kCols = DP / 4;
    int done_item = -1, done_first = 0, done_hi = 0, done_head = 0;
    auto store = [&]() {
      if (!warp_wait(dq_full, done_item & 1, status, kStatusWaitAccum, abort_flag)) return false;
      tc_fence_after();
      const int col = part * kCols;
      uint4 c[kCols / 8];
      if (col < p.D) load_packed(t_dq + lane_base + col, p.scale, c);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(dq_free);
      if (col < p.D) {
        const TileOut to{p.dq + (static_cast<long>(done_first) * p.H + done_head) * p.D + col,
                         static_cast<long>(p.H) * p.D, p.D, p.lp, (done_hi - done_first) << p.lp, p.D - col};
        store_rows(c, to, quad * 32, lane);
      }
      return true;
    };
    while (ok && at.valid) {
      const uint32_t s_addr = t_s + (at.k & 1) * 128 + lane_base + part * 32;
      const int first = at.token(), token = first + ((quad * 32 + lane) >> p.lp), hi = at.hi();
      const bool last = at.last();
      const int limit = min(hi, token + 1) - (at.lo() + at.chunk * kRowsT) - part * 32;  // visible keys, last chunk
      if (at.first()) {
        lse = delta = 0.f;
        if (token < hi) {
          const long from = static_cast<long>(at.head() + (lane & ((1 << p.lp) - 1))) * p.T + token;
          lse = p.lse[from];
          delta = p.delta[from];
        }
      }
      ok = warp_wait(&s_full[at.k & 1], (at.k >> 1) & 1, status, kStatusWaitAccum, abort_flag);
      if (!ok) break;
      tc_fence_after();
      float v[32], g[32];
      tmem_load32(s_addr, v);
      const uint64_t scale2 = pair_of(p.scale2, p.scale2), minus_lse = pair_of(-lse, -lse);
#pragma unroll
      for (int j = 0; j < 32; j += 2) {
        unpair(fma2(pair_of(v[j], v[j + 1]), scale2, minus_lse), v[j], v[j + 1]);
        v[j] = ex2(v[j]);
        v[j + 1] = ex2(v[j + 1]);
      }
      ok = warp_wait(dp_full, at.k & 1, status, kStatusWaitAccum, abort_flag);
      if (!ok) break;
      tc_fence_after();
      tmem_load32(dp_addr, g);
      const uint64_t minus_delta = pair_of(-delta, -delta);
#pragma unroll
      for (int j = 0; j < 32; j += 2)
        unpair(mul2(pair_of(v[j], v[j + 1]), add2(pair_of(g[j], g[j + 1]), minus_delta)), g[j], g[j + 1]);
      if (last) {
        const uint32_t seen = low_bits(limit);
#pragma unroll
        for (int j = 0; j < 32; ++j) g[j] = (seen >> j) & 1u ? g[j] : 0.f;
      }
      uint32_t w[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) w[j] = pack_bf16(g[2 * j], g[2 * j + 1]);
      tmem_st_u32x16(s_addr, w);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(ds_ready);
      if (at.first() && at.item > 0) ok = store();
      if (last) {
        done_item = at.item;
        done_first = first;
        done_hi = hi;
        done_head = at.head();
      }
      at.step();
    }
    if (ok && done_item >= 0) ok = store();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  settle(*abort_flag != 0);
  if (warp == 0) tmem_dealloc(tmem, 512);
}

template <int DP>
int run_bwd(const PackedMaps& m, const PackedArgs& a, const BwdArgs& args, bool want_dq, bool want_dkv,
            unsigned* status, cudaStream_t stream) {
  const long items_kv = static_cast<long>(a.dkv.max_tiles) * a.Hkv * args.splits;
  const long items_q = static_cast<long>(a.dq.max_tiles) * (a.H >> a.lp);
  if (items_q > 0x7fff0000l || items_kv > 0x7fff0000l) return -2;
  const long grid_kv = std::min(items_kv, static_cast<long>(a.num_sms));
  const long grid_q = std::min(items_q, static_cast<long>(a.num_sms));
  if (want_dkv) {
    const bool split = args.splits > 1;
    auto kernel = split ? packed_dkv_kernel<DP, true> : packed_dkv_kernel<DP, false>;
    if (set_max_smem(kernel, BwdCfg<DP>::kSmem) != cudaSuccess) return -1;
    if (launch_pdl(kernel, dim3(static_cast<unsigned>(grid_kv)), dim3(kBwdThreads), BwdCfg<DP>::kSmem, stream, m.q,
                   m.k, m.v, m.dout, args, status) != cudaSuccess)
      return -1;
    if (args.splits > 1) {
      const long groups = static_cast<long>(a.T) * a.Hkv * a.D / 4;
      if (launch_pdl(packed_join_kernel, dim3(static_cast<unsigned>((groups + 255) / 256), 2), dim3(256), 0, stream,
                     args) != cudaSuccess)
        return -1;
    }
  }
  if (want_dq) {
    auto kernel = packed_dq_kernel<DP>;
    if (set_max_smem(kernel, BwdCfg<DP>::kSmem) != cudaSuccess) return -1;
    if (launch_pdl(kernel, dim3(static_cast<unsigned>(grid_q)), dim3(kBwdThreads), BwdCfg<DP>::kSmem, stream, m.q, m.k,
                   m.v, m.dout, m.k32, m.v32, args, status) != cudaSuccess)
      return -1;
  }
  return 0;
}

}  // namespace

// Splits of a key tile's query tiles, where the key tiles are too few for the SMs (a sequence's first tile has twice the
// mean work, so two per SM are wanted), each of eight iterations of the mean tile at least. Measured with delta, us
// for 1 / 2 / 4 / 8 splits, D = 128, by key tiles x iterations of the mean one: 16 x 64 194 / 129 / 75 / 53, 64 x 32
// 110 / 85 / 69 / 93, 64 x 16 68 / 55 / 55 / 75, 128 x 128 427 / 277 / 280 / 349, 8 x 8 51 / 54 / 53 / 53,
// 256 x 128 471 / 536 / 619 / 711. Both numbers go by the mean length, which says little of mixed ones: a sequence of 2048
// (8 heads over 2) beside 100 of 8 tokens gets no splits and takes 184 us with the forward pass, alone 123; one of 4096 (8
// heads over 1) beside 200 of 4 tokens 523, alone 212.
int packed_dkv_splits(const PackedArgs& a, int B) {
  const long items = static_cast<long>(std::max(1, a.T / 128)) * a.Hkv;
  const long mean = (static_cast<long>(a.T) / std::max(1, B)) * (a.H / a.Hkv) / 256;  // iterations of 128 rows
  return static_cast<int>(std::max(1l, std::min({2l * a.num_sms / items, mean / 8, 8l})));
}

int launch_packed_delta(const PackedArgs& a, const void* out, const void* rest, const void* dout, long stride_t,
                        long stride_h, float* delta, int* taken, cudaStream_t stream) {
  const long rows = static_cast<long>(a.T) * a.H;
  return launch_pdl(packed_delta_kernel, dim3(static_cast<unsigned>((rows + 15) / 16)), dim3(256), 0, stream,
                    static_cast<const bf16*>(out), static_cast<const bf16*>(rest), static_cast<const bf16*>(dout),
                    taken, stride_t, stride_h, a.T, a.H, a.D, delta) == cudaSuccess ? 0 : -1;
}

int launch_packed_backward(const PackedMaps& maps, const PackedArgs& a, const float* lse, const float* delta, void* dq,
                           void* dk, void* dv, int splits, float* part, int* taken, unsigned* status,
                           cudaStream_t stream) {
  const BwdArgs args{static_cast<bf16*>(dq), static_cast<bf16*>(dk), static_cast<bf16*>(dv), lse, delta,
                     static_cast<const int4*>(a.dq.entries), static_cast<const int4*>(a.dkv.entries), a.dq.head,
                     a.dkv.head, taken, a.T, a.H, a.Hkv, a.D, a.lp, a.scale, a.scale * kLog2e, splits, part};
  const bool want_dkv = dk != nullptr;
  return a.D <= 64 ? run_bwd<64>(maps, a, args, dq != nullptr, want_dkv, status, stream)
                   : run_bwd<128>(maps, a, args, dq != nullptr, want_dkv, status, stream);
}

}  // namespace ecz
