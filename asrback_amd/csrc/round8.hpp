// Rounding of rows to 8 bits with a scale each, shared by the 8-bit layers
// (linear8.hip) and the 8-bit cache (cache8.hip).
//
// A row's scale is the 127th part of its largest magnitude, rounded to float32 as the
// division rounds, and a value its quotient by that scale, rounded to a whole
// number, ties to even.  The quotient is not divided out: x times the scale's
// reciprocal lies within one of it, and the remainder x - q s, which float32
// holds exactly (both terms are multiples of half the scale's last place, and it is
// below the scale), says on which side of the border x lies.
#pragma once

#include "common.hpp"

namespace asrattn {
namespace {

// The magnitude's bits: larger for larger magnitudes, and NaN above infinity, so
// that the largest of a row carries a NaN where fmaxf would drop it.
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The largest over aligned groups of W lanes (W a power of two from 2 to 64).
template <int W>
__device__ __forceinline__ uint32_t group_umax(uint32_t x) {
  if constexpr (W >= 2) x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xF, 0xF, false));
  if constexpr (W >= 4) x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xF, 0xF, false));
  if constexpr (W >= 8) x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x141, 0xF, 0xF, false));
  if constexpr (W >= 16) x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x140, 0xF, 0xF, false));
  if constexpr (W >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max(r[0], r[1]);
  }
  if constexpr (W >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    x = max(r[0], r[1]);
  }
  return x;
}

struct Scale8 {
  float scale;    // NaN for a row that holds an infinity or a NaN
  float inverse;  // 0 where values are not found by it: such rows, 0, and tiny
  bool tiny;      // the reciprocal would overflow: divide
};

__device__ __forceinline__ Scale8 scale8(uint32_t largest) {
  Scale8 s;
  const bool finite = largest < 0x7f800000u;
  s.scale = finite ? __uint_as_float(largest) / 127.f : __uint_as_float(0x7fc00000u);
  s.tiny = s.scale > 0.f && s.scale < 0x1p-120f;
  s.inverse = s.scale >= 0x1p-120f ? 1.f / s.scale : 0.f;
  return s;
}

// x / scale rounded to a whole number, for any scale.
__device__ __forceinline__ float round8_any(float x, const Scale8& s) {
  if (s.inverse == 0.f && !s.tiny) return 0.f;
  float q = __builtin_rintf(s.tiny ? x / s.scale : x * s.inverse);
  const float two = 2.f * fmaf(-q, s.scale, x);  // twice the remainder
  if (fabsf(two) > s.scale)
    q += two > 0.f ? 1.f : -1.f;
  else if (fabsf(two) == s.scale && ((int)q & 1))
    q += two > 0.f ? 1.f : -1.f;
  return fminf(fmaxf(q, -127.f), 127.f);
}

// Four values x / scale rounded to whole numbers, the first in the low byte.
__device__ __forceinline__ uint32_t round8x4(const float* x, const Scale8& s) {
  // Added to 3 2^22, a number this small is rounded to a whole one, which is the low bits.
  constexpr float kWhole = 0x1.8p23f;
  float q[4], most = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    q[e] = fmaf(x[e], s.inverse, kWhole);
    most = fmaxf(most, fabsf(fmaf(kWhole - q[e], s.scale, x[e])));
  }
  // Some value at a border, or none found by the reciprocal.
  if (!(most < 0.5f * s.scale)) {
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e] = round8_any(x[e], s) + kWhole;
  }
  const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(q[1]), __float_as_uint(q[0]), 0x0c0c0400u);
  const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(q[3]), __float_as_uint(q[2]), 0x0c0c0400u);
  return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}

// The largest magnitude of a vector of elements.
__device__ __forceinline__ uint32_t largest_of(const uint4& raw, float) {
  auto bits = [](uint32_t x) { return x & 0x7fffffffu; };
  return max(max(bits(raw.x), bits(raw.y)), max(bits(raw.z), bits(raw.w)));
}
__device__ __forceinline__ uint32_t largest_of(const uint4& raw, bf16_raw) {
  typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
  auto bits = [](uint32_t x) { return __builtin_bit_cast(u16x2_t, x & 0x7fff7fffu); };
  const u16x2_t a = __builtin_elementwise_max(bits(raw.x), bits(raw.y)), b = __builtin_elementwise_max(bits(raw.z), bits(raw.w)),
                c = __builtin_elementwise_max(a, b);
  return (uint32_t)max(c[0], c[1]) << 16;
}

}  // namespace
}  // namespace asrattn
