// What stands between two blocks of a decoder: the norm after a block, its gate and residual scale, the residual sum and
// the norm before the next block, in one pass over the data, and its gradients.
//
//   b = x rsqrt(mean x^2 + eps) post       (or x)
//   s = residual + scale gate b            (stream; the residual and the gate may be missing)
//   n = s rsqrt(mean s^2 + eps) weight     (normed; as bf16 / fp16 / fp32, or from bf16 on to 4 bits, fp4_common.cuh)
//
// Everything is held in fp32; n and s are rounded once each, n is taken from the unrounded s. A team of warps keeps a row
// in registers. Rows are read in 16-byte vectors, two a lane (16 columns, in fp32 8, beyond 8192 columns 16); 16-bit rows that
// are no multiple of 16 bytes in words, up to eight a lane (16 columns); other fp32 rows element by element, four a lane forward
// and eight backward, up to 16 beyond 4096 columns.
//
// Forward two rows are read and two written per token: 8192 rows of 4096 in bf16 take 39 us, 6.9 TB/s, bound by HBM (6.3 at
// 8192 columns). Backward four are read and up to two written. In a CUDA graph, with the 6 us that add up the blocks' sums:
// 69 us where x's and the residual's gradients are one tensor (5.3 TB/s without the sums), 77 where they are two, 101 with
// both norms (4.2 TB/s), where half of all issue slots and two barriers a row stand against 16 warps an SM.
// In 4 bits the quantisation's instructions bound it: 4096 rows of 4096 with both norms take 29 us, 3.8 TB/s, 65% of the
// issue slots. Sums, products and roundings work on pairs of columns (f32x2): with single ones the last took 34 us.
//
// Backward, with g = dn weight, sh = s is (is = rsqrt(mean s^2 + eps), xh = x ix likewise):
//   ds = dstream + is (g - sh mean(g sh)),  dweight = sum_t dn sh,  dresidual = ds
//   dgate = scale b . ds (summed over the columns where the gate has one value a token),  db = scale gate ds
//   dx = ix (h - xh mean(h xh)) with h = db post,  dpost = sum_t db xh      (dx = db without a norm behind the block)
// The forward pass saves is and ix. Sums over tokens: every team adds up its rows in registers, a block its teams, a second
// kernel the blocks, each in order, so results do not depend on timing.
#include <algorithm>
#include <type_traits>

#include "fp4_common.cuh"
#include "launchers.h"

namespace ecz {

namespace {

using packed::fma2;
using packed::mul2;
using packed::pair_of;
using packed::unpair;

constexpr int kMaxWarps = 32;
constexpr int kMostSmem = 227 * 1024 - 2 * kMaxWarps * 8;  // beside the teams' scratch

template <typename T>
struct Cast;
template <>
struct Cast<float> {
  static __device__ __forceinline__ float to(float v) { return v; }
  static __device__ __forceinline__ float from(float v) { return v; }
};
template <>
struct Cast<bf16> {
  static __device__ __forceinline__ float to(bf16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ bf16 from(float v) { return __float2bfloat16(v); }
  static __device__ __forceinline__ uint32_t from(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};
template <>
struct Cast<__half> {
  static __device__ __forceinline__ float to(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half from(float v) { return __float2half(v); }
  static __device__ __forceinline__ uint32_t from(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};

// What arithmetic works on: two fp32 values in a 64-bit register, both at once, or the one of VEC = 1.
template <int VEC>
using Vals = std::conditional_t<VEC == 1, float, uint64_t>;
__device__ __forceinline__ float mul2(float a, float b) { return a * b; }
__device__ __forceinline__ float fma2(float a, float b, float c) { return fmaf(a, b, c); }
template <int VEC>
__device__ __forceinline__ Vals<VEC> vals(float v) {
  if constexpr (VEC == 1) return v;
  else return pair_of(v, v);
}
__device__ __forceinline__ float one_of(float v, int) { return v; }
__device__ __forceinline__ float one_of(uint64_t pair, int k) {
  float v[2];
  unpair(pair, v[0], v[1]);
  return v[k];
}
__device__ __forceinline__ float total(float v) { return v; }
__device__ __forceinline__ float total(uint64_t pair) {
  float lo, hi;
  unpair(pair, lo, hi);
  return lo + hi;
}

// A lane's VEC consecutive elements, from element `at` of a row of `hidden` on: 16 bytes, or one element, or (16-bit rows
// that are no multiple of 16 bytes) a word. Odd rows of an odd length start in the middle of a word: `at` is odd there, and
// -1 in the word that the row shares with the row before. (With 32 bytes a lane, two loads or stores of 16, every access
// would touch half of each sector: 66 us where this took 45 for 8192 rows of 4096.)
template <typename T, int VEC>
struct Pack {
  static constexpr int kWords = (VEC * static_cast<int>(sizeof(T)) + 3) / 4;
  union {
    T v[VEC];
    uint32_t words[kWords];
  };
  __device__ __forceinline__ Pack() {}
  __device__ __forceinline__ float get(int i) const { return Cast<T>::to(v[i]); }
  __device__ __forceinline__ void set(int i, float f) { v[i] = Cast<T>::from(f); }
  // elements 2 k and 2 k + 1 (Vals)
  __device__ __forceinline__ Vals<VEC> get2(int k) const {
    if constexpr (VEC == 1) return get(0);
    else return pair_of(get(2 * k), get(2 * k + 1));
  }
  __device__ __forceinline__ void set2(int k, Vals<VEC> f) {
    if constexpr (VEC == 1) {
      set(0, f);
    } else {
      float lo, hi;
      unpair(f, lo, hi);
      if constexpr (sizeof(T) == 4) {
        set(2 * k, lo);
        set(2 * k + 1, hi);
      } else {
        words[k] = Cast<T>::from(lo, hi);
      }
    }
  }
  // row[at ..] of a row that starts like the others do (Team::shift), zeros where it has ended or has not begun
  __device__ __forceinline__ void fetch_row(const T* row, int at, int hidden) {
    if constexpr (VEC == 2) {
      if (row != nullptr && at >= 0 && at + 1 < hidden) {
        words[0] = *reinterpret_cast<const uint32_t*>(row + at);
        return;
      }
    }
    fetch(row, at, hidden);
  }
  // row[at ..], zeros where the row is null, has ended or has not begun
  __device__ __forceinline__ void fetch(const T* row, int at, int hidden) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) words[i] = 0;
    if (row == nullptr || at >= hidden) return;
    if constexpr (VEC == 1) {
      v[0] = row[at];
    } else if constexpr (VEC == 2) {
      if (at >= 0) v[0] = row[at];
      if (at + 1 < hidden) v[1] = row[at + 1];
    } else {
      *reinterpret_cast<uint4*>(words) = *reinterpret_cast<const uint4*>(row + at);
    }
  }
  __device__ __forceinline__ void store(T* row, int at, int hidden) const {
    if (at >= hidden) return;
    if constexpr (VEC == 1) {
      row[at] = v[0];
    } else if constexpr (VEC == 2) {
      if (at >= 0 && at + 1 < hidden) *reinterpret_cast<uint32_t*>(row + at) = words[0];
      else if (at >= 0) row[at] = v[0];
      else row[0] = v[1];
    } else {
      *reinterpret_cast<uint4*>(row + at) = *reinterpret_cast<const uint4*>(words);
    }
  }
};

// Threads of a block: 256, or (longer rows) fewer than the 1024 that the kernel allows.
template <int THREADS>
__device__ __forceinline__ int block_threads() {
  if constexpr (THREADS == 256) return 256;
  else return static_cast<int>(blockDim.x);
}

// Rows on their way: every thread copies the vectors that it will work on itself into shared memory (cp.async), DEPTH rows
// ahead, so nothing is shared, no barrier is needed and no register is held. Operand k, vector i of a thread in slot s
// lies in a plane of one entry (16 bytes, a word of two 16-bit elements or an fp32 element) per thread. DEPTH 0 (fp32 rows
// beyond 8192 columns): operands are read when they are needed.
template <typename T, int VEC, int NV, int OPS, int DEPTH, int THREADS>
struct Rows {
  using P = Pack<T, VEC>;
  static constexpr bool kAhead = DEPTH > 0;
  static constexpr int kEntry = VEC * static_cast<int>(sizeof(T));
  static_assert(!kAhead || kEntry == 16 || kEntry == 4, "what cp.async copies");
  static constexpr int kSlotPlanes = OPS * NV;
  static constexpr int bytes(int threads) { return DEPTH * kSlotPlanes * threads * kEntry; }
  uint32_t base;
  int slot = 0;
  const T* ptr[OPS];  // rows being worked on (DEPTH 0)
  __device__ __forceinline__ Rows(void* smem) : base(smem_u32(smem) + threadIdx.x * kEntry) {}
  __device__ __forceinline__ uint32_t plane(int s, int op, int i) const {
    return base + static_cast<uint32_t>((s * kSlotPlanes + op * NV + i) * block_threads<THREADS>() * kEntry);
  }
  // start the copy of operand op's row (zeros for null) into slot s. Where nothing is copied the source is `spare`, a row of
  // the call: an address behind a row's end, or counted from a null row (in words an odd one), would not be a valid one.
  template <class Place>
  __device__ __forceinline__ void start(int s, int op, const T* row, const Place& place, int hidden, const T* spare) {
    if constexpr (kAhead) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int at = place.template at<VEC>(i);
        const uint32_t to = plane(s, op, i);
        int bytes = row != nullptr && at < hidden ? kEntry : 0;  // the rest of the entry becomes zero
        if constexpr (VEC == 2) bytes = at + 1 == hidden ? bytes / 2 : bytes;
        const T* from = bytes > 0 ? row + at : spare;
        if constexpr (kEntry == 16)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
        else
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
      }
    } else {
      ptr[op] = row;
    }
  }
  __device__ __forceinline__ static void commit() {
    if constexpr (kAhead) asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // the oldest slot's copies have landed
  __device__ __forceinline__ static void wait() {
    if constexpr (kAhead) asm volatile("cp.async.wait_group %0;" ::"n"(kAhead ? DEPTH - 1 : 0) : "memory");
  }
  __device__ __forceinline__ void get(P& out, int op, int i, int at, int hidden) const {
    if constexpr (kAhead) {
      if constexpr (kEntry == 16)
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(out.words[0]), "=r"(out.words[1]), "=r"(out.words[2]), "=r"(out.words[3])
                     : "r"(plane(slot, op, i))
                     : "memory");
      else
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(out.words[0]) : "r"(plane(slot, op, i)) : "memory");
      if (VEC == 2 && i == 0 && at < 0) out.words[0] &= 0xffff0000u;  // the low half is the row before's
    } else {
      out.fetch(ptr[op], at, hidden);
    }
  }
};

// This lane's part of a weight: in registers, or (SHARED) in planes of shared memory like Rows', where two weights or the
// sums over tokens would spill.
template <typename T, int VEC, int NV, bool SHARED, int THREADS>
struct Lanes {
  using P = Pack<T, VEC>;
  static constexpr int kEntry = VEC * static_cast<int>(sizeof(T));
  static constexpr int bytes(int threads) { return SHARED ? NV * threads * kEntry : 0; }
  P held[SHARED ? 1 : NV];
  P* plane;
  template <class Place>
  __device__ __forceinline__ void fetch(void* smem, const T* row, const Place& place, int hidden) {
    plane = static_cast<P*>(smem) + threadIdx.x;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      P v;
      v.fetch(row, place.template at<VEC>(i), hidden);
      if constexpr (SHARED) plane[i * block_threads<THREADS>()] = v;
      else held[i] = v;
    }
  }
  __device__ __forceinline__ P get(int i) const {
    if constexpr (SHARED) return plane[i * block_threads<THREADS>()];
    else return held[i];
  }
};

// A team's place: `warps` (at most MOST) consecutive warps of the block, and its reductions. Two buffers in turn: a warp writes one again
// only behind a barrier that all warps reach after reading it.
template <int MOST>
struct Team {
  int warps, index, first, step, lane, warp;
  float2* scratch;  // [2][kMaxWarps]
  int turn = 0;
  int shift = 0;  // 1: this team's rows start in the middle of a word (and are added up in another order than with 0)
  __device__ __forceinline__ Team(int warps_, float2* buf) : warps(warps_), scratch(buf) {
    const int w = threadIdx.x >> 5;
    lane = threadIdx.x & 31;
    index = w / warps;
    warp = w - index * warps;
    first = warp * 32 + lane;
    step = warps * 32;
  }
  // the column of this lane's i-th vector
  template <int VEC>
  __device__ __forceinline__ int at(int i) const {
    return (first + i * step) * VEC - (VEC == 2 ? shift : 0);
  }
  __device__ __forceinline__ void barrier() const {
    asm volatile("bar.sync %0, %1;" ::"r"(index + 1), "r"(warps * 32) : "memory");
  }
  // every lane: the part of warp lane % MOST of the team, or `neutral`
  template <class V>
  __device__ __forceinline__ V parts(V v, V neutral) {
    V* buf = reinterpret_cast<V*>(scratch + turn * kMaxWarps + index * warps);
    turn ^= 1;
    if (lane == 0) buf[warp] = v;
    barrier();
    const int of = lane % MOST;
    return of < warps ? buf[of] : neutral;
  }
  __device__ __forceinline__ float sum(float v) {
    v = warp_sum(v);
    if (warps == 1) return v;
    v = parts(v, 0.f);
#pragma unroll
    for (int o = 1; o < MOST; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
  __device__ __forceinline__ float2 sum(float2 v) {
    v.x = warp_sum(v.x);
    v.y = warp_sum(v.y);
    if (warps == 1) return v;
    v = parts(v, make_float2(0.f, 0.f));
#pragma unroll
    for (int o = 1; o < MOST; o <<= 1) {
      v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
      v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    return v;
  }
  __device__ __forceinline__ uint32_t max(uint32_t v) {
    v = __reduce_max_sync(0xffffffffu, v);
    return warps == 1 ? v : __reduce_max_sync(0xffffffffu, parts(v, 0u));
  }
};

// Whether the forward kernel's weights lie in shared memory (Lanes).
template <int VEC, int FMT, bool POST>
constexpr bool kForwardShared = VEC > 1 && (POST || FMT != 0);

// FMT 0: normed as T; else as 4-bit codes (bf16). POST: there may be a norm behind the block. Persistent over
// rows: team t of all takes rows t, t + teams, ...
template <typename T, int VEC, int NV, int FMT, bool POST, int THREADS, int BLOCKS, int DEPTH>
__global__ void __launch_bounds__(THREADS, BLOCKS)
    block_norm_kernel(const __grid_constant__ BlockNormArgs a, int warps) {
  __shared__ float2 scratch[2 * kMaxWarps];
  extern __shared__ uint8_t ring[];
  pdl_trigger();
  Team<THREADS == 256 ? 8 : kMaxWarps> team(warps, scratch);
  Rows<T, VEC, NV, 2, DEPTH, THREADS> rows(ring);
  const int per_block = blockDim.x / (32 * warps);
  const int teams = gridDim.x * per_block;
  const bool post = POST && (VEC > 1 || a.post != nullptr);
  const int hidden = a.hidden;
  const float mean = 1.f / static_cast<float>(hidden);
  const int last = FMT == 0 ? a.rows : (a.rows + 127) / 128 * 128;
  const T* xp = static_cast<const T*>(a.x);
  const T* rp = static_cast<const T*>(a.residual);
  const T* gp = static_cast<const T*>(a.gate);
  constexpr int kPairs = (VEC + 1) / 2;
  auto start = [&](int slot, int row) {
    const bool on = row < a.rows;
    rows.start(slot, 0, on ? xp + row * a.x_stride : nullptr, team, hidden, xp);
    rows.start(slot, 1, on && rp != nullptr ? rp + row * a.r_stride : nullptr, team, hidden, xp);
    rows.commit();
  };
  pdl_wait();
  int row = blockIdx.x * per_block + team.index;
  if constexpr (VEC == 2) team.shift = row & hidden & 1;
#pragma unroll
  for (int d = 0; d < DEPTH; ++d) start(d, row + d * teams);
  Lanes<T, VEC, NV, kForwardShared<VEC, FMT, POST>, THREADS> w, p;
  uint8_t* behind = ring + Rows<T, VEC, NV, 2, DEPTH, THREADS>::bytes(blockDim.x);
  w.fetch(behind, static_cast<const T*>(a.weight), team, hidden);
  if constexpr (POST)
    p.fetch(behind + w.bytes(blockDim.x), static_cast<const T*>(a.post), team, hidden);
  for (; row < last; row += teams) {
    const bool real = row < a.rows;
    float factor = a.scale;
    if (a.gate_mode == kGateToken && real) factor *= Cast<T>::to(gp[row * a.gate_stride]);
    if constexpr (DEPTH == 0) start(0, row);
    rows.wait();
    Vals<VEC> s[NV][kPairs];
    float ix = 1.f;
    if (post) {
      Vals<VEC> q = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        Pack<T, VEC> x;
        rows.get(x, 0, i, team.template at<VEC>(i), hidden);
#pragma unroll
        for (int k = 0; k < kPairs; ++k) {
          s[i][k] = x.get2(k);
          q = fma2(s[i][k], s[i][k], q);
        }
      }
      ix = rsqrtf(team.sum(total(q)) * mean + a.eps);
      if (a.inv_x != nullptr && team.first == 0 && real) a.inv_x[row] = ix;
    }
    const Vals<VEC> ix2 = vals<VEC>(ix), factor2 = vals<VEC>(factor);
    Vals<VEC> q = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = team.template at<VEC>(i);
      Pack<T, VEC> r;
      if (post) {
        const Pack<T, VEC> pi = p.get(i);
#pragma unroll
        for (int k = 0; k < kPairs; ++k) s[i][k] = mul2(s[i][k], mul2(ix2, pi.get2(k)));
      } else {
        Pack<T, VEC> x;
        rows.get(x, 0, i, at, hidden);
#pragma unroll
        for (int k = 0; k < kPairs; ++k) s[i][k] = x.get2(k);
      }
      if (a.gate_mode == kGateFull) {
        Pack<T, VEC> g;
        g.fetch_row(real ? gp + row * a.gate_stride : nullptr, at, hidden);
#pragma unroll
        for (int k = 0; k < kPairs; ++k) s[i][k] = mul2(s[i][k], g.get2(k));
      }
      rows.get(r, 1, i, at, hidden);
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        s[i][k] = fma2(factor2, s[i][k], r.get2(k));
        q = fma2(s[i][k], s[i][k], q);
      }
    }
    if constexpr (DEPTH > 0) {  // this row's slot is read: the row DEPTH further
      start(rows.slot, row + DEPTH * teams);
      rows.slot = rows.slot + 1 == DEPTH ? 0 : rows.slot + 1;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      Pack<T, VEC> out;
#pragma unroll
      for (int k = 0; k < kPairs; ++k) out.set2(k, s[i][k]);
      if (real)
        out.store(static_cast<T*>(a.stream) + static_cast<size_t>(row) * hidden, team.template at<VEC>(i), hidden);
    }
    const float is = rsqrtf(team.sum(total(q)) * mean + a.eps);
    const Vals<VEC> is2 = vals<VEC>(is);
    if (a.inv_s != nullptr && team.first == 0 && real) a.inv_s[row] = is;
    Pack<T, VEC> out[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const Pack<T, VEC> wi = w.get(i);
#pragma unroll
      for (int k = 0; k < kPairs; ++k) out[i].set2(k, mul2(mul2(s[i][k], is2), wi.get2(k)));
      if (FMT == 0)
        out[i].store(static_cast<T*>(a.normed) + static_cast<size_t>(row) * hidden, team.template at<VEC>(i),
                     hidden);
    }
    if constexpr (FMT != 0) {
      float mul = 1.f;
      if constexpr (FMT == fp4::kNv) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) top = max(top, fp4::max_bits<4>(out[i].words));
        if (top >= 0x7f80u) {
          top = 0;
#pragma unroll
          for (int i = 0; i < NV; ++i) top = max(top, fp4::finite_bits<4>(out[i].words));
        }
        const int e = fp4::row_exponent(fp4::bits_value(team.max(top)));
        mul = fp4::pow2(-e);
        if (real && team.first == 0) a.row_scale[row] = fp4::pow2(e);
      }
#pragma unroll
      for (int i = 0; i < NV; ++i)
        fp4::store8<FMT>(out[i].words, mul, row, team.first + i * team.step, real ? hidden / 8 : 0, a.tiles, a.codes,
                         a.scales);
    }
  }
}

// Where the backward kernel's weights lie (Lanes): in shared memory beside x and the residual.
template <int VEC, bool WHOLE>
struct SharedWeights {
  static constexpr bool value = VEC > 1 && !WHOLE;
};

// Persistent like the forward kernel. A block's sums for dweight and dpost go to its row of a.dw_part / a.dpost_part (fp32
// [blocks, hidden]). WHOLE: the stream is given in place of x and the residual (fp32).
template <typename T, int VEC, int NV, bool POST, bool WHOLE, int THREADS, int BLOCKS, int DEPTH>
__global__ void __launch_bounds__(THREADS, BLOCKS)
    block_norm_bwd_kernel(const __grid_constant__ BlockNormGrads a, int warps) {
  __shared__ float2 scratch[2 * kMaxWarps];
  extern __shared__ uint8_t ring[];
  pdl_trigger();
  Team<THREADS == 256 ? 8 : kMaxWarps> team(warps, scratch);
  Rows<T, VEC, NV, WHOLE ? 3 : 4, DEPTH, THREADS> rows(ring);
  const int per_block = blockDim.x / (32 * warps);
  const int teams = gridDim.x * per_block, self = blockIdx.x * per_block + team.index;
  if constexpr (VEC == 2) team.shift = self & a.hidden & 1;
  const bool post = POST && (VEC > 1 || a.post != nullptr);
  const int gate_mode = WHOLE ? kGateNone : a.gate_mode;
  const int hidden = a.hidden;
  const float mean = 1.f / static_cast<float>(hidden);
  const T* np = static_cast<const T*>(a.dnormed);
  const T* up = static_cast<const T*>(a.dstream);
  const T* xp = static_cast<const T*>(a.x);
  const T* rp = static_cast<const T*>(WHOLE ? a.stream : a.residual);
  const T* gp = static_cast<const T*>(a.gate);
  const int64_t r_stride = WHOLE ? hidden : a.r_stride;
  auto start = [&](int slot, int row) {
    const bool on = row < a.rows;
    const T* spare = WHOLE ? rp : xp;
    rows.start(slot, 0, on && np != nullptr ? np + row * a.dn_stride : nullptr, team, hidden, spare);
    rows.start(slot, 1, on && up != nullptr ? up + row * a.ds_stride : nullptr, team, hidden, spare);
    rows.start(slot, 2, on && rp != nullptr ? rp + row * r_stride : nullptr, team, hidden, spare);
    if constexpr (!WHOLE) rows.start(slot, 3, on ? xp + row * a.x_stride : nullptr, team, hidden, spare);
    rows.commit();
  };
  pdl_wait();
#pragma unroll
  for (int d = 0; d < DEPTH; ++d) start(d, self + d * teams);
  constexpr bool kShared = SharedWeights<VEC, WHOLE>::value;
  Lanes<T, VEC, NV, kShared, THREADS> w, p;
  uint8_t* behind = ring + Rows<T, VEC, NV, WHOLE ? 3 : 4, DEPTH, THREADS>::bytes(blockDim.x);
  w.fetch(behind, static_cast<const T*>(a.weight), team, hidden);
  if constexpr (POST)
    p.fetch(behind + w.bytes(blockDim.x), static_cast<const T*>(a.post), team, hidden);
  constexpr int kPairs = (VEC + 1) / 2;
  Vals<VEC> dw[NV][kPairs], dp[POST ? NV : 1][kPairs];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < kPairs; ++k) {
      dw[i][k] = 0;
      if constexpr (POST) dp[i][k] = 0;
    }
  for (int row = self; row < a.rows; row += teams) {
    const float is = a.inv_s[row], ix = post ? a.inv_x[row] : 1.f;
    float gate = a.scale;  // scale times the token's gate
    if (gate_mode == kGateToken) gate *= Cast<T>::to(gp[row * a.gate_stride]);
    if constexpr (DEPTH == 0) start(0, row);
    rows.wait();
    const Vals<VEC> is2 = vals<VEC>(is), ix2 = vals<VEC>(ix), gate2 = vals<VEC>(gate);
    Vals<VEC> sh[NV][kPairs];  // the normalised stream
    Vals<VEC> dots = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = team.template at<VEC>(i);
      Pack<T, VEC> dn, r, x, fg;
      rows.get(dn, 0, i, at, hidden);
      rows.get(r, 2, i, at, hidden);
      if constexpr (!WHOLE) rows.get(x, 3, i, at, hidden);
      if (gate_mode == kGateFull) fg.fetch_row(gp + row * a.gate_stride, at, hidden);
      const Pack<T, VEC> wi = w.get(i);
      Pack<T, VEC> pi;
      if constexpr (POST) pi = p.get(i);
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        Vals<VEC> s = r.get2(k);
        if constexpr (!WHOLE) {
          Vals<VEC> b = x.get2(k);
          if (POST && post) b = mul2(b, mul2(ix2, pi.get2(k)));
          if (gate_mode == kGateFull) b = mul2(b, fg.get2(k));
          s = fma2(gate2, b, s);
        }
        sh[i][k] = mul2(s, is2);
        dw[i][k] = fma2(dn.get2(k), sh[i][k], dw[i][k]);
        dots = fma2(mul2(dn.get2(k), wi.get2(k)), sh[i][k], dots);
      }
    }
    const float dot = -team.sum(total(dots)) * mean;
    const Vals<VEC> dot2 = vals<VEC>(dot), scale2 = vals<VEC>(a.scale);
    Vals<VEC> hx = 0, gx = 0;  // h . xh and the token gate's gradient
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = team.template at<VEC>(i);
      Pack<T, VEC> dn, u, x, fg, out, dg;
      rows.get(dn, 0, i, at, hidden);
      rows.get(u, 1, i, at, hidden);
      if constexpr (!WHOLE) rows.get(x, 3, i, at, hidden);
      if (gate_mode == kGateFull) fg.fetch_row(gp + row * a.gate_stride, at, hidden);
      const Pack<T, VEC> wi = w.get(i);
      Pack<T, VEC> pi;
      if constexpr (POST) pi = p.get(i);
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        const Vals<VEC> ds = fma2(is2, fma2(sh[i][k], dot2, mul2(dn.get2(k), wi.get2(k))), u.get2(k));
        out.set2(k, ds);
        Vals<VEC> db = mul2(gate2, ds);
        if constexpr (!WHOLE) {
          const Vals<VEC> xh = mul2(x.get2(k), ix2);  // without a norm behind the block ix is 1
          const Vals<VEC> pw = POST && post ? pi.get2(k) : vals<VEC>(1.f);
          if (gate_mode == kGateFull) {
            dg.set2(k, mul2(mul2(scale2, ds), mul2(xh, pw)));
            db = mul2(db, fg.get2(k));
          } else if (gate_mode == kGateToken) {
            gx = fma2(mul2(xh, pw), ds, gx);
          }
          if (POST && post) {
            dp[POST ? i : 0][k] = fma2(db, xh, dp[POST ? i : 0][k]);
            db = mul2(db, pw);  // h
            hx = fma2(db, xh, hx);
          }
        }
        sh[i][k] = db;
      }
      if (a.dresidual != nullptr) out.store(static_cast<T*>(a.dresidual) + static_cast<size_t>(row) * hidden, at, hidden);
      if (gate_mode == kGateFull && a.dgate != nullptr)
        dg.store(static_cast<T*>(a.dgate) + static_cast<size_t>(row) * hidden, at, hidden);
    }
    float2 sums = make_float2(total(hx), total(gx));
    if constexpr (!WHOLE) {
      if ((POST && post) || gate_mode == kGateToken) {
        sums = team.sum(sums);
        if (gate_mode == kGateToken && a.dgate != nullptr && team.first == 0)
          static_cast<T*>(a.dgate)[row] = Cast<T>::from(a.scale * sums.y);
      }
    }
    if (a.dx != nullptr) {
      const float m = -ix * sums.x * mean;
      const Vals<VEC> m2 = vals<VEC>(m);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int at = team.template at<VEC>(i);
        Pack<T, VEC> x, out;
        if (POST && post) rows.get(x, WHOLE ? 0 : 3, i, at, hidden);
#pragma unroll
        for (int k = 0; k < kPairs; ++k)
          out.set2(k, POST && post ? mul2(ix2, fma2(x.get2(k), m2, sh[i][k])) : sh[i][k]);
        out.store(static_cast<T*>(a.dx) + static_cast<size_t>(row) * hidden, at, hidden);
      }
    }
    if constexpr (DEPTH > 0) {
      start(rows.slot, row + DEPTH * teams);
      rows.slot = rows.slot + 1 == DEPTH ? 0 : rows.slot + 1;
    }
  }
  // A block's teams add their sums up in order, in the rows' place; a block's are its row of the parts.
  const bool several = per_block > 1;
  if (several) {
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
  }
  static_assert(THREADS > 256 || DEPTH * (WHOLE ? 3 : 4) * sizeof(T) >= sizeof(float), "the sums fit in the rows' place");
  float* sums = reinterpret_cast<float*>(ring);  // [teams of the block][hidden]
#pragma unroll
  for (int which = 0; which < (POST ? 2 : 1); ++which) {
    float* part = which == 0 ? a.dw_part : a.dpost_part;
    if (part == nullptr) continue;
    part += static_cast<size_t>(blockIdx.x) * hidden;
    float* to = several ? sums + team.index * hidden : part;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = team.template at<VEC>(i);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if (at + j < 0 || at + j >= hidden) continue;
        to[at + j] = one_of(which == 0 ? dw[i][j / 2] : dp[POST ? i : 0][j / 2], j % 2);
      }
    }
    if (several) {
      __syncthreads();
      for (int c = threadIdx.x; c < hidden; c += blockDim.x) {
        float v = sums[c];
        for (int t = 1; t < per_block; ++t) v += sums[t * hidden + c];
        part[c] = v;
      }
      __syncthreads();
    }
  }
}

// Columns of `parts` rows of fp32 added up in order: 32 threads a column take every 32nd row each, then one adds theirs.
template <typename T>
__global__ void __launch_bounds__(1024) block_norm_sum_kernel(const float* __restrict__ dw_part,
                                                              const float* __restrict__ dpost_part, T* dw, T* dpost,
                                                              int parts, int hidden) {
  __shared__ float sums[32][33];
  pdl_trigger();
  const float* part = blockIdx.y == 0 ? dw_part : dpost_part;
  T* out = blockIdx.y == 0 ? dw : dpost;
  const int lane = threadIdx.x & 31, c = blockIdx.x * 32 + lane, group = threadIdx.x >> 5;
  pdl_wait();
  if (out == nullptr) return;
  float s = 0.f;
  if (c < hidden) {
#pragma unroll 4
    for (int p = group; p < parts; p += 32) s += part[static_cast<size_t>(p) * hidden + c];
  }
  sums[group][lane] = s;
  __syncthreads();
  if (group == 0 && c < hidden) {
#pragma unroll
    for (int i = 1; i < 32; ++i) s += sums[i][lane];
    out[c] = Cast<T>::from(s);
  }
}

// The layout depends on the row's length alone, so a row's sums do not depend on how many rows there are. In words they do
// depend on whether the row starts in the middle of one (Team::shift): odd rows of an odd length are added up in another
// order than even ones.
struct Grid {
  int warps, nv, teams, threads;  // warps of a team, vectors a lane, teams and threads of a block
};

// `target` vectors a lane, more where that would take more than 32 warps; several teams to a block of 256 threads, or one.
template <int VEC>
Grid grid_of(int hidden, int target) {
  const int all = (hidden + (VEC == 2 ? hidden % 2 : 0) + 32 * VEC - 1) / (32 * VEC);
  Grid g;
  g.warps = std::min(kMaxWarps, (all + target - 1) / target);
  if (g.warps <= 8) {
    int p = 1;
    while (p < g.warps) p *= 2;
    g.warps = p;
  }
  g.nv = (all + g.warps - 1) / g.warps;
  g.teams = g.warps <= 8 ? 8 / g.warps : 1;
  g.threads = 32 * g.warps * g.teams;
  return g;
}

// Blocks for `rows`, at most `most`. In words, a team's rows start all in the middle of one or none does (Team::shift): where
// it has more than one, the number of teams is even.
int blocks_for(const Grid& g, int rows, int most, bool words) {
  const int all = (rows + g.teams - 1) / g.teams;
  if (all <= most) return all;
  return words ? std::max(2, most & ~1) : most;
}

template <typename T>
constexpr int vec_of() { return 16 / static_cast<int>(sizeof(T)); }

template <class Kernel, class Args>
int go(Kernel kernel, int smem, int blocks, const Grid& g, const Args& a, cudaStream_t stream) {
  if (set_max_smem(kernel, smem) != cudaSuccess) return -1;
  return launch_pdl(kernel, dim3(blocks), dim3(g.threads), smem, stream, a, g.warps) == cudaSuccess ? 0 : -1;
}

template <typename T, int VEC, int NV, int FMT, bool POST, int THREADS, int BLOCKS, int DEPTH>
int go_forward(const BlockNormArgs& a, const Grid& g, int sms, cudaStream_t stream) {
  const int rows = FMT == 0 ? a.rows : (a.rows + 127) / 128 * 128;
  const int resident = THREADS <= 256 ? BLOCKS : 1024 / g.threads;
  using R = Rows<T, VEC, NV, 2, DEPTH, THREADS>;
  using L = Lanes<T, VEC, NV, kForwardShared<VEC, FMT, POST>, THREADS>;
  static_assert(R::bytes(THREADS) + 2 * L::bytes(THREADS) <= kMostSmem, "227 KB of shared memory");
  const int smem = R::bytes(g.threads) + 2 * L::bytes(g.threads);
  return go(block_norm_kernel<T, VEC, NV, FMT, POST, THREADS, BLOCKS, DEPTH>, smem,
            blocks_for(g, rows, sms * resident, VEC == 2), g, a, stream);
}

// Blocks of 256 threads, two rows ahead: three to an SM, or four where the norm behind the block or the 4-bit result make
// the chain from a row's arrival to its end longer.
template <typename T, int FMT, bool POST>
int run_forward(const BlockNormArgs& a, int sms, cudaStream_t stream) {
  constexpr int V = vec_of<T>();
  // 4-bit results: lanes cover the scales' padding too
  const Grid g = grid_of<V>(FMT == 0 ? a.hidden : (a.hidden + fp4::kBlockK - 1) / fp4::kBlockK * fp4::kBlockK, 2);
  if (g.threads <= 256) return go_forward<T, V, 2, FMT, POST, 256, POST || FMT != 0 ? 4 : 3, 2>(a, g, sms, stream);
  if (g.nv <= 2) return go_forward<T, V, 2, FMT, POST, 1024, 1, 2>(a, g, sms, stream);
  if constexpr (sizeof(T) == 4) return go_forward<T, V, 4, FMT, POST, 1024, 1, 0>(a, g, sms, stream);
  return -1;
}

// 16-bit rows in words: as many columns a lane as above. 8192 rows of 4095 take 104 us where vectors take 49 for 4096 (four
// times the accesses); single elements, which cp.async does not copy ahead, took 289.
template <typename T, bool POST>
int run_forward_words(const BlockNormArgs& a, int sms, cudaStream_t stream) {
  const Grid g = grid_of<2>(a.hidden, 8);
  if (g.threads > 256) return go_forward<T, 2, 8, 0, POST, 1024, 1, 2>(a, g, sms, stream);
  if (g.nv > 4) return go_forward<T, 2, 8, 0, POST, 256, 4, 2>(a, g, sms, stream);
  return go_forward<T, 2, 4, 0, POST, 256, 4, 2>(a, g, sms, stream);
}

template <typename T>
int run_forward_type(const BlockNormArgs& a, bool vec, int sms, cudaStream_t stream) {
  if (vec) return a.post != nullptr ? run_forward<T, 0, true>(a, sms, stream) : run_forward<T, 0, false>(a, sms, stream);
  if constexpr (sizeof(T) == 2) {
    return a.post != nullptr ? run_forward_words<T, true>(a, sms, stream) : run_forward_words<T, false>(a, sms, stream);
  } else {
    // single elements: four a lane, more beyond 4096 columns (32768 rows of 1001: 113 us, with eight 117)
    const Grid g = grid_of<1>(a.hidden, 4);
    if (g.threads <= 256) return go_forward<T, 1, 4, 0, true, 256, 4, 2>(a, g, sms, stream);
    if (g.nv <= 4) return go_forward<T, 1, 4, 0, true, 1024, 1, 2>(a, g, sms, stream);
    if (g.nv <= 8) return go_forward<T, 1, 8, 0, true, 1024, 1, 2>(a, g, sms, stream);
    return go_forward<T, 1, 16, 0, true, 1024, 1, 0>(a, g, sms, stream);
  }
}

template <int FMT>
int run_forward_fp4(const BlockNormArgs& a, int sms, cudaStream_t stream) {
  return a.post != nullptr ? run_forward<bf16, FMT, true>(a, sms, stream) : run_forward<bf16, FMT, false>(a, sms, stream);
}

template <typename T>
Grid backward_grid(int hidden, bool vec) {
  if (vec) return grid_of<vec_of<T>()>(hidden, 2);
  // eight single elements a lane (32768 rows of 1001 in fp32: 121 us, with four 160)
  return sizeof(T) == 2 ? grid_of<2>(hidden, 8) : grid_of<1>(hidden, 8);
}

// Three blocks of 256 threads to an SM from the stream, two from x and the residual, which takes more registers.
template <typename T>
int backward_blocks(const Grid& g, int rows, int sms, bool vec, bool whole) {
  const int resident = g.threads > 256 ? 1 : vec && whole ? 3 : 2;
  return blocks_for(g, rows, sms * resident, !vec && sizeof(T) == 2);
}

template <typename T, int VEC, int NV, bool POST, bool WHOLE, int THREADS, int BLOCKS, int DEPTH>
int go_backward(const BlockNormGrads& a, const Grid& g, int blocks, cudaStream_t stream) {
  using R = Rows<T, VEC, NV, WHOLE ? 3 : 4, DEPTH, THREADS>;
  using L = Lanes<T, VEC, NV, SharedWeights<VEC, WHOLE>::value, THREADS>;
  static_assert(R::bytes(THREADS) + 2 * L::bytes(THREADS) <= kMostSmem, "227 KB of shared memory");
  const int smem = R::bytes(g.threads) + 2 * L::bytes(g.threads);
  return go(block_norm_bwd_kernel<T, VEC, NV, POST, WHOLE, THREADS, BLOCKS, DEPTH>, smem, blocks, g, a, stream);
}

template <typename T>
int run_backward_whole(const BlockNormGrads& a, const Grid& g, int blocks, cudaStream_t stream) {
  constexpr int V = vec_of<T>();
  if (g.threads <= 256) return go_backward<T, V, 2, false, true, 256, 3, 2>(a, g, blocks, stream);
  if (g.threads <= 512) return go_backward<T, V, 2, false, true, 512, 1, 2>(a, g, blocks, stream);
  if (g.nv <= 2) return go_backward<T, V, 2, false, true, 1024, 1, 2>(a, g, blocks, stream);
  return go_backward<T, V, 4, false, true, 1024, 1, 1>(a, g, blocks, stream);
}

template <typename T, bool POST>
int run_backward(const BlockNormGrads& a, const Grid& g, int blocks, cudaStream_t stream) {
  constexpr int V = vec_of<T>();
  if (g.threads <= 256) return go_backward<T, V, 2, POST, false, 256, 2, 2>(a, g, blocks, stream);
  if (g.threads <= 512) return go_backward<T, V, 2, POST, false, 512, 1, 2>(a, g, blocks, stream);
  if (g.nv <= 2) return go_backward<T, V, 2, POST, false, 1024, 1, 1>(a, g, blocks, stream);
  if constexpr (sizeof(T) == 4) return go_backward<T, V, 4, POST, false, 1024, 1, 0>(a, g, blocks, stream);
  return -1;
}

template <typename T, bool WHOLE>
int run_backward_single(const BlockNormGrads& a, const Grid& g, int blocks, cudaStream_t stream) {
  if (g.threads <= 256) return go_backward<T, 1, 8, !WHOLE, WHOLE, 256, 2, 2>(a, g, blocks, stream);
  if (g.threads <= 512) return go_backward<T, 1, 8, !WHOLE, WHOLE, 512, 1, 2>(a, g, blocks, stream);
  if (g.nv <= 8) return go_backward<T, 1, 8, !WHOLE, WHOLE, 1024, 1, 1>(a, g, blocks, stream);
  return go_backward<T, 1, 16, !WHOLE, WHOLE, 1024, 1, 0>(a, g, blocks, stream);
}

template <typename T, bool POST>
int run_backward_words(const BlockNormGrads& a, const Grid& g, int blocks, cudaStream_t stream) {
  if (g.threads > 512) return go_backward<T, 2, 8, POST, false, 1024, 1, 1>(a, g, blocks, stream);
  if (g.threads > 256) return go_backward<T, 2, 8, POST, false, 512, 1, 2>(a, g, blocks, stream);
  if (g.nv > 4) return go_backward<T, 2, 8, POST, false, 256, 2, 2>(a, g, blocks, stream);
  return go_backward<T, 2, 4, POST, false, 256, 2, 2>(a, g, blocks, stream);
}

template <typename T>
int run_backward_type(const BlockNormGrads& a, bool vec, int sms, cudaStream_t stream) {
  const bool whole = a.stream != nullptr;
  if (whole && sizeof(T) != 4) return -1;
  const Grid g = backward_grid<T>(a.hidden, vec);
  const int blocks = backward_blocks<T>(g, a.rows, sms, vec, whole);
  int rc;
  if constexpr (sizeof(T) == 2) {
    if (vec)
      rc = a.post != nullptr ? run_backward<T, true>(a, g, blocks, stream) : run_backward<T, false>(a, g, blocks, stream);
    else
      rc = a.post != nullptr ? run_backward_words<T, true>(a, g, blocks, stream)
                             : run_backward_words<T, false>(a, g, blocks, stream);
  } else if (vec) {
    rc = whole               ? run_backward_whole<T>(a, g, blocks, stream)
         : a.post != nullptr ? run_backward<T, true>(a, g, blocks, stream)
                             : run_backward<T, false>(a, g, blocks, stream);
  } else {
    rc = whole ? run_backward_single<T, true>(a, g, blocks, stream) : run_backward_single<T, false>(a, g, blocks, stream);
  }
  if (rc != 0 || (a.dweight == nullptr && a.dpost == nullptr)) return rc;
  return launch_pdl(block_norm_sum_kernel<T>, dim3((a.hidden + 31) / 32, a.dpost != nullptr ? 2 : 1), dim3(1024), 0, stream,
                    static_cast<const float*>(a.dw_part), static_cast<const float*>(a.dpost_part),
                    static_cast<T*>(a.dweight), static_cast<T*>(a.dpost), blocks, a.hidden) == cudaSuccess ? 0
                                                                                                                    : -1;
}

template <typename T>
int parts_type(int rows, int hidden, bool vec, bool whole, int sms) {
  const Grid g = backward_grid<T>(hidden, vec);
  return backward_blocks<T>(g, rows, sms, vec, whole);
}

}  // namespace

int launch_block_norm(const BlockNormArgs& a, NormType type, bool vec, int fmt, int sms, cudaStream_t stream) {
  if (a.rows < 1 || a.hidden < 1 || a.hidden > kBlockNormMaxHidden) return -1;
  if (fmt != 0) {
    if (type != kNormBf16 || !vec || a.hidden % 32 != 0) return -1;
    return fmt == fp4::kNv ? run_forward_fp4<fp4::kNv>(a, sms, stream) : run_forward_fp4<fp4::kMx>(a, sms, stream);
  }
  switch (type) {
    case kNormBf16: return run_forward_type<bf16>(a, vec, sms, stream);
    case kNormFp16: return run_forward_type<__half>(a, vec, sms, stream);
    default: return run_forward_type<float>(a, vec, sms, stream);
  }
}

int block_norm_parts(NormType type, int rows, int hidden, bool vec, bool whole, int sms) {
  switch (type) {
    case kNormBf16: return parts_type<bf16>(rows, hidden, vec, whole, sms);
    case kNormFp16: return parts_type<__half>(rows, hidden, vec, whole, sms);
    default: return parts_type<float>(rows, hidden, vec, whole, sms);
  }
}

int launch_block_norm_grads(const BlockNormGrads& a, NormType type, bool vec, int sms, cudaStream_t stream) {
  if (a.rows < 1 || a.hidden < 1 || a.hidden > kBlockNormMaxHidden) return -1;
  switch (type) {
    case kNormBf16: return run_backward_type<bf16>(a, vec, sms, stream);
    case kNormFp16: return run_backward_type<__half>(a, vec, sms, stream);
    default: return run_backward_type<float>(a, vec, sms, stream);
  }
}

}  // namespace ecz
