// origami_element.h -- 16-bit and 8-bit element types of the operators on the paged cache
// (origami_append.hip, origami_attention.hip): vectors, loads and conversions.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

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

// x of another lane of the same 16, moved without LDS.
template <int CTRL>
__device__ __forceinline__ float lane_moved(float x) {
  return __builtin_bit_cast(
      float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, false));
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
