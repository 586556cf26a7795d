// 4-bit floating point (E2M1) with scales per group of columns, as the block-scaled MMAs of sm_100a read it.
//
// Codes: [rows, K] E2M1, two per byte, column 2b in the low nibble of byte b. Scales: one byte per group of 16 columns
// (nvfp4, e4m3) or 32 (mxfp4, E8M0), stored in tiles of 128 rows x 4 groups, 512 bytes each, in the order in which
// tcgen05.cp.32x128b.warpx4 copies them into tensor memory: row r, group g of a tile at (r % 32) 16 + (r / 32) 4 + g.
// The tiles of 128 rows follow one another along K, padded with zeros to whole K blocks of 256 columns, so one bulk copy
// brings a K block's scales. nvfp4 has an fp32 power of two per row besides.
#pragma once

#include "common.cuh"

namespace ecz {
namespace fp4 {

constexpr int kNv = 1, kMx = 2;   // formats
constexpr int kBlockK = 256;      // columns of a K block (a 128-byte row of codes)
constexpr int kTileBytes = 512;   // scales of 128 rows x 4 groups

template <int FMT>
struct Format {
  static constexpr int kGroup = FMT == kNv ? 16 : 32;
  static constexpr int kTilesPerBlock = kBlockK / (4 * kGroup);           // 4 (nvfp4), 2 (mxfp4)
  static constexpr int kBlockBytes = kTilesPerBlock * kTileBytes;         // scales of 128 rows x 256 columns
  static constexpr int kLanes = kGroup / 8;                               // lanes of 8 columns that share a scale
  static constexpr int kWordLanes = 4 * kLanes;                           // ... that share a 4-byte word of scales
};

// Byte offset of the word that holds the scales of row `row`, groups 4 t .. 4 t + 3; `tiles` of them along K.
__device__ __forceinline__ size_t scale_word(int row, int t, int tiles) {
  return (static_cast<size_t>(row >> 7) * tiles + t) * kTileBytes + (row & 31) * 16 + ((row >> 5) & 3) * 4;
}

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

// The power of two of a row of nvfp4 with largest (finite) magnitude `amax`: the smallest that is no less than
// amax / 2688 (= 6 x 448, the largest value times the largest scale). Its exponent.
__device__ __forceinline__ int row_exponent(float amax) {
  if (amax == 0.f) return 0;
  const uint32_t bits = __float_as_uint(__fdiv_rn(amax, 2688.f));
  const int e = static_cast<int>((bits + 0x7fffffu) >> 23) - 127;  // rounded up
  return min(max(e, -100), 120);
}

// Eight e2m1 codes of v * r, the first in the lowest nibble. r is the rounded reciprocal of the scale, so v * r misses the
// quotient by 2^-23 of it at most; the quotient of a bf16 value by an e4m3 scale (or a power of two) is either a tie
// between two codes or at least 2^-10 away from it, so rounding the product to multiples of 2^-14 first (adding and
// subtracting 1.5 * 2^9) lands on ties where they are and moves nothing else across. Beyond
// 6 all become 6.
__device__ __forceinline__ uint32_t codes8(const float* v, float r) {
  float q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] = __fsub_rn(__fmaf_rn(v[i], r, 768.f), 768.f);
  uint32_t out;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(out)
      : "f"(q[0]), "f"(q[1]), "f"(q[2]), "f"(q[3]), "f"(q[4]), "f"(q[5]), "f"(q[6]), "f"(q[7]));
  return out;
}

__device__ __forceinline__ void unpack8(const uint4& raw, float* v) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(h[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// The value of a scale byte.
template <int FMT>
__device__ __forceinline__ float scale_value(uint32_t byte) {
  if constexpr (FMT == kMx) {
    return byte == 0xffu ? __int_as_float(0x7fc00000) : byte == 0 ? 5.877471754111438e-39f : __int_as_float(byte << 23);
  } else {
    uint32_t halves;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(halves) : "h"(static_cast<uint16_t>(byte)));
    return __low2float(*reinterpret_cast<const __half2*>(&halves));
  }
}

// Eight codes times s, as bf16.
__device__ __forceinline__ uint4 values8(uint32_t codes, float s) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(codes));
  uint4 out;
  uint32_t* o = reinterpret_cast<uint32_t*>(&out);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    const __nv_bfloat162 b = __floats2bfloat162_rn(f.x * s, f.y * s);
    o[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  return out;
}

// Largest magnitude of the finite ones of eight values, and whether any is not finite.
__device__ __forceinline__ float finite_max8(const float* v, bool& bad) {
  float m = 0.f;
  bad = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = fabsf(v[i]);
    const bool fin = a < __int_as_float(0x7f800000);
    bad |= !fin;
    m = fmaxf(m, fin ? a : 0.f);
  }
  return m;
}

// Maximum over the lanes of a group (aligned lanes).
template <int FMT>
__device__ __forceinline__ float group_max(float m) {
#pragma unroll
  for (int o = 1; o < Format<FMT>::kLanes; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

// The scale byte of a group with largest finite magnitude `m` (nvfp4: in units of the row's power of two) and the
// reciprocal that its values are multiplied with. A group with a value that is not finite has the format's NaN as its
// scale, which makes every product that reads it NaN.
template <int FMT>
__device__ __forceinline__ uint32_t group_scale(float m, bool bad, float& recip) {
  if constexpr (FMT == kMx) {
    // exponent of m, one more from a mantissa of 1.75 on, less 2; 2^-126 <= scale <= 2^125
    int e = static_cast<int>((__float_as_uint(m) + 0x200000u) >> 23) - 127 - 2;
    e = min(max(e, -126), 125);
    recip = pow2(-e);
    return bad ? 0xffu : static_cast<uint32_t>(e + 127);
  } else {
    const float t = fmaxf(__fdiv_rn(m, 6.f), 0.001953125f);
    uint16_t pair;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(pair) : "f"(0.f), "f"(t));
    uint32_t halves;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(halves) : "h"(pair));
    const __half2 h = *reinterpret_cast<const __half2*>(&halves);
    recip = __frcp_rn(__low2float(h));
    return bad ? 0x7fu : static_cast<uint32_t>(pair & 0xffu);
  }
}

// Quantise the eight columns of this lane and store them: lane l of the warp holds vector `vec` (columns 8 vec ..) of
// row `row`, consecutive lanes consecutive vectors from a multiple of 32; `live`: vec < vecs (others hold zeros and are
// padding of the scales). mul (nvfp4): the reciprocal of the row's power of two. All lanes take part.
template <int FMT>
__device__ __forceinline__ void store8(const float* v, float mul, int row, int vec, int vecs, int tiles,
                                       uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  using F = Format<FMT>;
  const bool live = vec < vecs;
  bool bad;
  const float m = group_max<FMT>(finite_max8(v, bad));
  const unsigned votes = __ballot_sync(0xffffffffu, bad);
  const int lane = threadIdx.x & 31;
  const unsigned mates = ((1u << F::kLanes) - 1u) << (lane & ~(F::kLanes - 1));
  float recip;
  uint32_t byte = group_scale<FMT>(FMT == kNv ? m * mul : m, (votes & mates) != 0, recip);
  if (!live) byte = 0;  // groups do not straddle the end: K is a multiple of 32
  if (live) {
    if constexpr (FMT == kNv) {
      float scaled[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) scaled[i] = v[i] * mul;  // exact: a power of two
      *reinterpret_cast<uint32_t*>(codes + (static_cast<size_t>(row) * vecs + vec) * 4) = codes8(scaled, recip);
    } else {
      *reinterpret_cast<uint32_t*>(codes + (static_cast<size_t>(row) * vecs + vec) * 4) = codes8(v, recip);
    }
  }
  // four groups' bytes to one word, stored by the first of their lanes
  uint32_t word = byte << (8 * ((lane / F::kLanes) & 3));
#pragma unroll
  for (int o = F::kLanes; o < F::kWordLanes; o <<= 1) word |= __shfl_xor_sync(0xffffffffu, word, o);
  const int t = vec / F::kWordLanes;
  if ((lane & (F::kWordLanes - 1)) == 0 && t < tiles)
    *reinterpret_cast<uint32_t*>(scales + scale_word(row, t, tiles)) = word;
}

// ---- block-scaled MMAs ---------------------------------------------------------------------------------------------
// Instruction descriptor of the block-scaled kinds: e2m1 operands, K-major, shape m x n, scales of type e4m3 (nvfp4) or
// E8M0 (mxfp4); sf: which bytes of the 32-bit scale words the MMA's two scales per row are (kind::mxf4: 0 or 2).
template <int FMT>
__host__ __device__ constexpr uint32_t idesc_fp4(int m, int n, int sf = 0) {
  return (static_cast<uint32_t>(sf) << 4)          // scale id of B
         | (1u << 7) | (1u << 10)                  // A, B: e2m1
         | (static_cast<uint32_t>(n >> 3) << 17)   // N >> 3
         | ((FMT == kMx ? 1u : 0u) << 23)          // scale type
         | (static_cast<uint32_t>(m >> 7) << 27)   // M >> 7
         | (static_cast<uint32_t>(sf) << 29);      // scale id of A
}

// Descriptor of such a tile: no swizzle, 8-row groups of 16-byte rows 128 bytes apart.
__device__ __forceinline__ uint64_t desc_scales(uint32_t addr) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(128u >> 4) << 32) |
         (static_cast<uint64_t>(1u) << 46);
}

}  // namespace fp4
}  // namespace ecz
