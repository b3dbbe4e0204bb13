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
__device__ __forceinline__ float whole_of(float x, const Scale8& s) {
  if (s.inverse == 0.f && !s.tiny) return 0.f;
  float q = __builtin_rintf(s.tiny ? x / s.scale : x * s.inverse);
  const float two = 2.f * fmaf(-q, s.scale, x);  // twice the remainder
  if (fabsf(two) > s.scale || (fabsf(two) == s.scale && ((int)q & 1))) q += two > 0.f ? 1.f : -1.f;
  return fminf(fmaxf(q, -127.f), 127.f);
}

// N values x / scale of elements T rounded to whole numbers, the first in the low byte of
// w[0].
//
// A row of bf16 has values next to a border all the time (254 x / largest is odd for many
// numbers of eight bits), so they are taken without a branch: the remainder times the
// reciprocal is added to the whole number found first, rounded with it.  With the scale
// S 2^k, S below 2^24, twice the remainder is a multiple of 2^k, so that it differs from the
// scale by one S-th of it or is equal; the reciprocal is off by at most S 2^-48 of
// itself, and S (S + 1) < 2^48, so the sum falls on the side of the border that x
// lies on.  Equal it is only where (2 q + 1) S has as few bits as x.  With eight that
// takes a scale of a power of two, whose reciprocal is exact, and then the even one is
// taken (a scale that is the 127th part of a number of eight bits is that or has no such S).
// In float32 a loop over one value at a time decides, as for tiny and non-finite rows: written
// out for all it would be most of a kernel's instructions, which come from memory
// anew at each launch (16 rows of 2048 and a product 7.3 us, so written 8.3).
template <typename T, int N>
__device__ __forceinline__ void bytes_of(const float (&x)[N], const Scale8& s, uint32_t (&w)[N / 4]) {
  // Added to 3 2^22, a number this small is rounded to a whole one, which is the low bits.
  constexpr float kWhole = 0x1.8p23f;
  constexpr bool kShort = sizeof(T) == 2;
  const float half = 0.5f * s.scale;
  float q[N];
  bool tie = false;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    q[e] = fmaf(x[e], s.inverse, kWhole);
    const float rest = fmaf(kWhole - q[e], s.scale, x[e]);
    q[e] = fmaf(rest, s.inverse, q[e]);
    if constexpr (!kShort) tie = tie || fabsf(rest) == half;
  }
#pragma unroll
  for (int e = 0; e < N; e += 4) {
    const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(q[e + 1]), __float_as_uint(q[e]), 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(q[e + 3]), __float_as_uint(q[e + 2]), 0x0c0c0400u);
    w[e / 4] = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
  }
  if (__builtin_expect(s.scale != 0.f && (s.inverse == 0.f || tie), 0)) {
#pragma unroll 1
    for (int e = 0; e < N; ++e) {
      float one = x[0];
#pragma unroll
      for (int i = 1; i < N; ++i) one = i == e ? x[i] : one;
      const uint32_t byte = (uint32_t)(int)whole_of(one, s) & 0xff;
#pragma unroll
      for (int i = 0; i < N / 4; ++i)
        w[i] = i == e / 4 ? (w[i] & ~(0xffu << (e % 4 * 8))) | byte << (e % 4 * 8) : w[i];
    }
  }
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
