// 4-bit floating point (E2M1) with scales per group of columns, as the block-scaled MMAs of sm_100a read it.
//
// Codes: [rows, K] E2M1, two per byte, column 2b in the low nibble of byte b. Scales: one byte per group of 16 columns
// (nvfp4, e4m3) or 32 (mxfp4, E8M0), stored in tiles of 128 rows x 4 groups, 512 bytes each, in the order in which
// tcgen05.cp.32x128b.warpx4 copies them into tensor memory: row r, group g of a tile at (r % 32) 16 + (r / 32) 4 + g.
// The tiles of 128 rows follow one another along K, padded with zeros to whole K blocks of 256 columns, so one bulk copy
// brings a K block's scales. nvfp4 has an fp32 power of two per row besides.
#pragma once

#include "common.cuh"
#include "packed_common.cuh"

namespace ecz {
namespace fp4 {

using packed::add2;
using packed::fma2;
using packed::mul2;
using packed::pair_of;

constexpr int kNv = 1, kMx = 2;   // formats
constexpr int kBlockK = 256;      // columns of a K block (a 128-byte row of codes)
constexpr int kTileBytes = 512;   // scales of 128 rows x 4 groups

template <int FMT>
struct Format {
  static constexpr int kGroup = FMT == kNv ? 16 : 32;
  static constexpr int kTilesPerBlock = kBlockK / (4 * kGroup);           // 4 (nvfp4), 2 (mxfp4)
  static constexpr int kBlockBytes = kTilesPerBlock * kTileBytes;         // scales of 128 rows x 256 columns
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

// A row's power of two r as two factors, for a product with another row's power of two w: (sum first) w last. Sums lie
// between 2^-20 (the smallest product) and 2^40 (6 x 448 squared, 65536 columns), r and w between 2^-100 and 2^120, so r w
// may leave fp32's range on either side, and sum r beyond 2^127, where the result does not. Nothing in between does here:
// with r up to 2^64, sum r is between 2^-120 and 2^104; a larger r comes after w and moves up what is at least 2^-120.
struct RowFactors {
  float first, last;
};
__device__ __forceinline__ RowFactors row_factors(float r) {
  const bool large = r > 18446744073709551616.f;  // 2^64
  return {large ? 1.f : r, large ? r : 1.f};
}

// ---- vectors of packed bf16 ----------------------------------------------------------------------------------------
// 32 bytes (16 bf16) from a 32-byte boundary.
__device__ __forceinline__ void load32(const void* p, uint32_t* v) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "l"(p));
}
__device__ __forceinline__ void store32(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

__device__ __forceinline__ float low_bf16(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float high_bf16(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

// Largest magnitude of 2 W packed bf16, as the bits of a bf16: they order like the magnitudes, 0x7f80 and above are not
// finite.
template <int W>
__device__ __forceinline__ uint32_t max_bits(const uint32_t* v) {
  uint32_t m = v[0] & 0x7fff7fffu;
#pragma unroll
  for (int i = 1; i < W; ++i) m = __vmaxu2(m, v[i] & 0x7fff7fffu);
  return max(m & 0xffffu, m >> 16);
}

// The same of the finite ones alone.
template <int W>
__device__ __forceinline__ uint32_t finite_bits(const uint32_t* v) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const uint32_t lo = v[i] & 0x7fffu, hi = (v[i] >> 16) & 0x7fffu;
    m = max(m, max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u));
  }
  return m;
}

__device__ __forceinline__ float bits_value(uint32_t bf16_bits) { return __uint_as_float(bf16_bits << 16); }

// ---- scales --------------------------------------------------------------------------------------------------------
// The scale byte of a group with largest magnitude `bits` (max_bits) and the factor that its values are multiplied with
// to become codes; mul (nvfp4): the reciprocal of the row's power of two, exact. A group with a value that is not finite
// has the format's NaN as its scale, which makes every product that reads it NaN.
template <int FMT>
__device__ __forceinline__ uint32_t group_scale(uint32_t bits, float mul, float& factor) {
  const bool bad = bits >= 0x7f80u;
  const float m = bits_value(bits);
  if constexpr (FMT == kMx) {
    // exponent of m, one more from a mantissa of 1.75 on, less 2; 2^-126 <= scale <= 2^125
    int e = static_cast<int>((__float_as_uint(m) + 0x200000u) >> 23) - 127 - 2;
    e = min(max(e, -126), 125);
    factor = pow2(-e);
    return bad ? 0xffu : static_cast<uint32_t>(e + 127);
  } else {
    // m / 6, off by 2^-23 of itself, then rounded to 12 bits (t (2^12 + 1) less its own low part): ties between e4m3
    // values, which have 5 bits, land where they are, and other quotients of an 8-bit number are 2^-8 of themselves away
    const float t = m * mul * 0.166666671633720398f, c = __fmul_rn(t, 4097.f);
    const float q = fmaxf(__fsub_rn(c, __fsub_rn(c, t)), 0.001953125f);
    uint16_t pair;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(pair) : "f"(0.f), "f"(q));
    uint32_t halves;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(halves) : "h"(pair));
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(__low2float(*reinterpret_cast<const __half2*>(&halves))));
    factor = r * mul;
    return bad ? 0x7fu : static_cast<uint32_t>(pair & 0xffu);
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

// ---- codes ---------------------------------------------------------------------------------------------------------
// Codes of eight packed bf16 times f, the first in the lowest nibble. f is the reciprocal of the scale, so the product
// misses the quotient by 2^-22 of it at most; the quotient of a bf16 value by an e4m3 scale (or a power of two) is either
// a tie between two codes or at least 2^-10 away from it, so rounding the product to multiples of 2^-14 first (adding and
// subtracting 768) lands on ties where they are and moves nothing else across. With the power of two of mxfp4 the product
// is the quotient. Beyond 6 all become 6.
template <int FMT>
__device__ __forceinline__ uint32_t codes8(const uint32_t* v, float f) {
  uint64_t q[4];
  const uint64_t ff = pair_of(f, f), up = pair_of(768.f, 768.f), down = pair_of(-768.f, -768.f);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t x = pair_of(low_bf16(v[i]), high_bf16(v[i]));
    q[i] = FMT == kMx ? mul2(x, ff) : add2(fma2(x, ff, up), down);
  }
  uint32_t out;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t.reg .f32 l, h;\n\t"
      "mov.b64 {l, h}, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 a, h, l;\n\t"
      "mov.b64 {l, h}, %2;\n\tcvt.rn.satfinite.e2m1x2.f32 b, h, l;\n\t"
      "mov.b64 {l, h}, %3;\n\tcvt.rn.satfinite.e2m1x2.f32 c, h, l;\n\t"
      "mov.b64 {l, h}, %4;\n\tcvt.rn.satfinite.e2m1x2.f32 d, h, l;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(out)
      : "l"(q[0]), "l"(q[1]), "l"(q[2]), "l"(q[3]));
  return out;
}

// Eight codes times s, as packed bf16.
__device__ __forceinline__ void values8(uint32_t codes, float s, uint32_t* out) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(codes));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    const __nv_bfloat162 b = __floats2bfloat162_rn(f.x * s, f.y * s);
    out[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
}

// ---- a lane's 16 columns -------------------------------------------------------------------------------------------
// Quantises the 16 columns (v: packed bf16) at 16 `vec` of row `row` and stores codes and scale; mxfp4: two neighbouring
// lanes hold a group, and both lanes of the pair call. Columns from 16 `vecs` on are padding of the scales (v zero).
template <int FMT>
__device__ __forceinline__ void store16(const uint32_t* v, float mul, int row, int vec, int vecs, int tiles,
                                        uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  uint32_t bits = max_bits<8>(v);
  if constexpr (FMT == kMx) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 1));
  float factor;
  uint32_t byte = group_scale<FMT>(bits, mul, factor);
  if (vec < vecs) {
    *reinterpret_cast<uint2*>(codes + (static_cast<size_t>(row) * vecs + vec) * 8) =
        make_uint2(codes8<FMT>(v, factor), codes8<FMT>(v + 4, factor));
  } else {
    byte = 0;
  }
  constexpr int kLanes = Format<FMT>::kGroup / 16;
  const int g = vec / kLanes;
  if ((kLanes == 1 || (vec & 1) == 0) && (g >> 2) < tiles) scales[scale_word(row, g >> 2, tiles) + (g & 3)] = byte;
}

// The same of 8 columns a lane: two (nvfp4) or four (mxfp4) neighbouring lanes hold a group; the whole warp calls.
template <int FMT>
__device__ __forceinline__ void store8(const uint32_t* v, float mul, int row, int vec, int vecs, int tiles,
                                       uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  constexpr int kLanes = Format<FMT>::kGroup / 8;
  uint32_t bits = max_bits<4>(v);
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
  float factor;
  uint32_t byte = group_scale<FMT>(bits, mul, factor);
  if (vec < vecs) *reinterpret_cast<uint32_t*>(codes + (static_cast<size_t>(row) * vecs + vec) * 4) = codes8<FMT>(v, factor);
  else byte = 0;
  const int g = vec / kLanes;
  if (vec % kLanes == 0 && (g >> 2) < tiles) scales[scale_word(row, g >> 2, tiles) + (g & 3)] = byte;
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
