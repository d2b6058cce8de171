// origami_element.h -- 16-bit, 8-bit and 4-bit element types of the operators on the paged cache
// (origami_append.hip, origami_attention.hip, origami_evict.hip): vectors, loads and conversions.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "origami_layout.h"

namespace origami_element {

using bf16 = __bf16;
using f16 = _Float16;

template <typename T>
using Vec2 = T __attribute__((ext_vector_type(2)));
template <typename T>
using Vec4 = T __attribute__((ext_vector_type(4)));
template <typename T>
using Vec8 = T __attribute__((ext_vector_type(8)));
using Float4 = float __attribute__((ext_vector_type(4)));
using U32x2 = uint32_t __attribute__((ext_vector_type(2)));
using U32x4 = uint32_t __attribute__((ext_vector_type(4)));

// Two e4m3 values, the low (HIGH = false) or high half of `word`, as two T; exact, since T
// has every value of e4m3.
template <bool HIGH>
__device__ __forceinline__ Vec2<bf16> fp8_pair(uint32_t word, bf16) {
  return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, 1.0f, HIGH);
}
template <bool HIGH>
__device__ __forceinline__ Vec2<f16> fp8_pair(uint32_t word, f16) {
  return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, 1.0f, HIGH);
}

// Eight e4m3 values as eight T (16 bytes).
template <typename T>
__device__ __forceinline__ U32x4 fp8_expand(U32x2 raw) {
  U32x4 out;
  out[0] = __builtin_bit_cast(uint32_t, fp8_pair<false>(raw[0], T()));
  out[1] = __builtin_bit_cast(uint32_t, fp8_pair<true>(raw[0], T()));
  out[2] = __builtin_bit_cast(uint32_t, fp8_pair<false>(raw[1], T()));
  out[3] = __builtin_bit_cast(uint32_t, fp8_pair<true>(raw[1], T()));
  return out;
}

// x as it is stored in e4m3: at most 448 in size (the conversion makes NaN of what is larger),
// NaN kept, rounded to nearest even.
__device__ __forceinline__ float fp8_clamp(float x) {
  const float y = fminf(fmaxf(x, -448.0f), 448.0f);
  return x != x ? x : y;
}

// How a cache holds its rows: in the 16-bit type of the queries, in e4m3, or in 4 bits.
//
// A row of D channels in 4 bits is D / 2 bytes of e2m1 values (a sign, two exponent bits and one
// mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4 and 6), channel 2 i in the low half of byte i, and then one
// byte s for each 32 channels, whose values are multiplied with 2^(s - 127) (255: NaN), filled up
// to whole dwords with zeros.  Appending keeps s - 127 within kLeastScale and kMostScale, so that
// bfloat16 and float16 have every value of the cache: nothing is rounded when it is read.
enum Cell { kWide = 0, kFp8 = 1, kFp4 = 2 };

constexpr int kLeastScale = -23, kMostScale = 13;

__host__ __device__ constexpr int fp4_row_bytes(int head_dim) {
  return head_dim / 2 + (head_dim + 127) / 128 * 4;
}

inline Cell cell_of(int64_t cache_dtype) {
  return cache_dtype == ORIGAMI_DTYPE_FLOAT4_E2M1     ? kFp4
         : cache_dtype == ORIGAMI_DTYPE_FLOAT8_E4M3FN ? kFp8
                                                      : kWide;
}

// Bytes of one row of a cache.
__host__ __device__ constexpr int row_bytes_of(Cell cell, int head_dim) {
  return cell == kFp4 ? fp4_row_bytes(head_dim) : (cell == kFp8 ? head_dim : 2 * head_dim);
}

// 2^(s - 127) of a scale's byte, as the conversions take it (by its exponent alone; of 0 it is
// 2^-127, and 255 makes everything NaN).
__device__ __forceinline__ float fp4_scale(uint32_t s) {
  return __builtin_bit_cast(float, s << 23);
}

// Byte BYTE of `codes` as two T; exact where T has the values.
template <int BYTE>
__device__ __forceinline__ Vec2<bf16> fp4_pair(uint32_t codes, float scale, bf16) {
  return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, BYTE);
}
template <int BYTE>
__device__ __forceinline__ Vec2<f16> fp4_pair(uint32_t codes, float scale, f16) {
  return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, BYTE);
}

// Eight 4-bit values as eight T (16 bytes).
template <typename T>
__device__ __forceinline__ U32x4 fp4_expand(uint32_t codes, float scale) {
  U32x4 out;
  out[0] = __builtin_bit_cast(uint32_t, fp4_pair<0>(codes, scale, T()));
  out[1] = __builtin_bit_cast(uint32_t, fp4_pair<1>(codes, scale, T()));
  out[2] = __builtin_bit_cast(uint32_t, fp4_pair<2>(codes, scale, T()));
  out[3] = __builtin_bit_cast(uint32_t, fp4_pair<3>(codes, scale, T()));
  return out;
}

// The scale's byte for values of at most `most` in size (the bits of a binary32): the least power
// of two at which none is further from its 4 bits than half a step, which is 7 2^e >= most, since
// what rounds to 6 reaches up to 7.  Larger than any that is kept, infinity too, becomes
// 6 2^kMostScale; NaN makes the 32 values NaN.
__device__ __forceinline__ uint32_t fp4_scale_byte(uint32_t most) {
  if (most > 0x7f800000u) return 255;
  // up by one past a mantissa of 1.75
  const int s = static_cast<int>((most + 0x1fffffu) >> 23) - 2;
  return static_cast<uint32_t>(min(max(s, 127 + kLeastScale), 127 + kMostScale));
}

// Eight values over `scale`, rounded to nearest even and limited to 6.
__device__ __forceinline__ uint32_t fp4_pack(const float (&x)[8], float scale) {
  uint32_t v = 0;
  v = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(v, x[0], x[1], scale, 0);
  v = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(v, x[2], x[3], scale, 1);
  v = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(v, x[4], x[5], scale, 2);
  v = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(v, x[6], x[7], scale, 3);
  return v;
}

// x of another lane of the same 16, moved without LDS.
template <int CTRL>
__device__ __forceinline__ float lane_moved(float x) {
  return __builtin_bit_cast(
      float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, false));
}

template <int CTRL>
__device__ __forceinline__ uint32_t lane_moved(uint32_t x) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, 0xf, 0xf, false));
}

// x folded over 8 or 16 neighbouring lanes, the same bits in each of them for a commutative fold.
template <int LANES, typename Fold>
__device__ __forceinline__ float fold_lanes(float x, Fold fold) {
  x = fold(x, lane_moved<0xb1>(x));   // quad_perm 1 0 3 2
  x = fold(x, lane_moved<0x4e>(x));   // quad_perm 2 3 0 1
  x = fold(x, lane_moved<0x141>(x));  // the other way round in 8 lanes
  if constexpr (LANES == 16) x = fold(x, lane_moved<0x140>(x));  // and in 16
  return x;
}

// Division of 0 <= x < 2^31 by a divisor that the host knows: x / d = mulhi(x, mul) >> shift, with
// mul the ceiling of 2^(32 + shift) / d and 2^shift < d <= 2^(shift + 1) (d = 1: shift -1).
struct Divisor {
  uint32_t mul;
  int32_t d, shift;
};

__device__ __forceinline__ int divide(int x, const Divisor& by) {
  return by.shift < 0 ? x : static_cast<int>(__umulhi(x, by.mul) >> by.shift);
}

inline Divisor divisor(int64_t d) {
  int shift = -1;
  while ((int64_t(1) << (shift + 1)) < d) ++shift;
  const uint64_t mul = d == 1 ? 0 : ((uint64_t(1) << (32 + shift)) + d - 1) / d;
  return Divisor{static_cast<uint32_t>(mul), static_cast<int32_t>(d), shift};
}

}  // namespace origami_element
