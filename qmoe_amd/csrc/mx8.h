// Device side of the microscaled 8-bit format, for activations.
//
// Blocks of 32 values along a row: 32 bytes of codes, each an e4m3 (a sign, four bits of exponent,
// three of mantissa, up to 448, no infinities), and one byte of scale, 2^(byte - 127), 255 for a block
// that is no number.  Rows as in the 4-bit format: ceil(W / 32) blocks back to back, zeros behind W.
#ifndef MX8_H_
#define MX8_H_

#include "mx4.h"

namespace mx8 {

using mx4::blocks_of;
using mx4::f32x2;
using mx4::kBlock;
using mx4::u32x2;
using mx4::u32x4;

typedef short s16x2 __attribute__((ext_vector_type(2)));

// DPP: a lane's neighbour and the lane two further (quad_perm), halves of a row of 16 and rows backwards
constexpr int kDppSwap1 = 0xb1, kDppSwap2 = 0x4e, kDppHalfMirror = 0x141, kDppMirror = 0x140;
template <int kCtrl>
__device__ __forceinline__ uint32_t of_lane(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), kCtrl, 0xf, 0xf, true));
}

// The op of v over kLanes lanes that lie together (16 or 64), in all of them.
template <int kLanes, class Op>
__device__ __forceinline__ uint32_t over_lanes(uint32_t v, Op op) {
  v = op(v, of_lane<kDppSwap1>(v));
  v = op(v, of_lane<kDppSwap2>(v));
  v = op(v, of_lane<kDppHalfMirror>(v));
  v = op(v, of_lane<kDppMirror>(v));
  if constexpr (kLanes == 64) {
    const auto rows = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = op(rows[0], rows[1]);
    const auto halves = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = op(halves[0], halves[1]);
  }
  return v;
}

__device__ __forceinline__ double double_of(uint32_t high, uint32_t low) {
  return __longlong_as_double(static_cast<unsigned long long>(high) << 32 | low);
}
// Sums over kLanes lanes, in all of them, the same bits in each.
template <int kLanes>
__device__ __forceinline__ double sum_over(double v) {
  auto add = [&](auto control) {
    const unsigned long long u = __double_as_longlong(v);
    v += double_of(of_lane<decltype(control)::value>(static_cast<uint32_t>(u >> 32)), of_lane<decltype(control)::value>(static_cast<uint32_t>(u)));
  };
  add(std::integral_constant<int, kDppSwap1>{});
  add(std::integral_constant<int, kDppSwap2>{});
  add(std::integral_constant<int, kDppHalfMirror>{});
  add(std::integral_constant<int, kDppMirror>{});
  if constexpr (kLanes == 64) {
    unsigned long long u = __double_as_longlong(v);
    auto high = __builtin_amdgcn_permlane16_swap(static_cast<uint32_t>(u >> 32), static_cast<uint32_t>(u >> 32), false, false);
    auto low = __builtin_amdgcn_permlane16_swap(static_cast<uint32_t>(u), static_cast<uint32_t>(u), false, false);
    v = double_of(high[0], low[0]) + double_of(high[1], low[1]);
    u = __double_as_longlong(v);
    high = __builtin_amdgcn_permlane32_swap(static_cast<uint32_t>(u >> 32), static_cast<uint32_t>(u >> 32), false, false);
    low = __builtin_amdgcn_permlane32_swap(static_cast<uint32_t>(u), static_cast<uint32_t>(u), false, false);
    v = double_of(high[0], low[0]) + double_of(high[1], low[1]);
  }
  return v;
}

__device__ __forceinline__ uint32_t largest_of(const float (&v)[8]) {
  uint32_t largest = 0;   // magnitudes compare as their bits do, and what is no number is above all
#pragma unroll
  for (int i = 0; i < 8; i++) largest = max(largest, __float_as_uint(v[i]) & 0x7fffffffu);
  return largest;
}

// The scale's byte by the bits of a block's largest magnitude: the smallest power of two, not below 2^-127, under
// which that is at most 448 = 1.75 * 2^8.  (By the exponent alone, values between 1.75 and 2 times a power
// of two would be up to an eighth too small.)
__device__ __forceinline__ uint32_t scale_byte(uint32_t largest) {
  const int exponent = static_cast<int>(largest >> 23);
  if (exponent == 255) return 255;
  return static_cast<uint32_t>(max(exponent - 8 + ((largest & 0x7fffffu) > 0x600000u ? 1 : 0), 0));
}

// As a float, 2^-127 too, for the instructions that divide by it.
__device__ __forceinline__ float divisor_of(uint32_t byte) { return __uint_as_float(byte ? byte << 23 : 0x00400000u); }

// Eight values as codes under a scale: exact division, to nearest, ties to even.  None of them is past 448 scales (what is
// would be no number: the instruction does not saturate).
__device__ __forceinline__ u32x2 pack8(const float (&v)[8], uint32_t byte) {
  if (byte == 255) return u32x2{0, 0};
  const float scale = divisor_of(byte);
  u32x2 out;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    s16x2 four = {0, 0};
    four = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(four, v[4 * i], v[4 * i + 1], scale, false);
    four = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(four, v[4 * i + 2], v[4 * i + 3], scale, true);
    out[i] = __builtin_bit_cast(uint32_t, four);
  }
  return out;
}

// Eight values of a lane, which with its three neighbours' are a block, to codes + 8 chunk and scales + chunk / 4, where `chunk` counts
// the eights of all rows; all lanes of the four come here.
__device__ __forceinline__ void store_block(const float (&v)[8], uint8_t *codes, uint8_t *scales, int64_t chunk, bool there) {
  uint32_t largest = largest_of(v);
  largest = max(largest, of_lane<kDppSwap1>(largest));
  largest = max(largest, of_lane<kDppSwap2>(largest));
  const uint32_t byte = scale_byte(largest);
  if (!there) return;
  *reinterpret_cast<u32x2 *>(codes + 8 * chunk) = pack8(v, byte);
  if ((chunk & 3) == 0) scales[chunk >> 2] = static_cast<uint8_t>(byte);
}

// Four codes as values.
__device__ __forceinline__ void unpack4(uint32_t codes, float scale, float *v) {
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, scale, false);
  const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes, scale, true);
  v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1];
}

// Eight values rounded to T.
template <class T>
__device__ __forceinline__ void round8(uint8_t *row, int first, int width, const float (&v)[8]) {
  mx4::Eight<T>::store(row, first, width, v);
}
template <>
__device__ __forceinline__ void round8<__bf16>(uint8_t *row, int first, int width, const float (&v)[8]) {
  uint16_t *p = reinterpret_cast<uint16_t *>(row) + first;
  uint32_t two[4];
#pragma unroll
  for (int i = 0; i < 4; i++) two[i] = mx4::two_bf16(v[2 * i], v[2 * i + 1]);
  if (first + 8 <= width) {
    __builtin_memcpy(p, two, 16);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (first + i < width) p[i] = static_cast<uint16_t>(two[i / 2] >> (16 * (i & 1)));
  }
}

// torch's types as the entry points number them
constexpr int kTypes = 3;
constexpr int64_t kTypeBytes[kTypes] = {2, 2, 4};

}  // namespace mx8

#endif  // MX8_H_
