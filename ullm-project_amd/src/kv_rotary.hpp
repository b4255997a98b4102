// kv_rotary.hpp -- rotation of queries and keys by their positions, in 64 bits.
//
// The angle of position p and frequency f is p * f / (2 pi) turns.  The
// quotient f / (2 pi) is held in two doubles, so that the whole turns of the
// product fall away exactly (one fused multiply-add) at any 32-bit position; what
// remains is taken to an eighth of a turn of an axis, where Taylor's series of
// sine and cosine end after x^15 and x^16 below 2^-53.  Products of bf16 and a
// cosine are rounded to a float whose last bit says "and a bit more", which
// rounds further, to bf16 or to a code, as the unrounded value would: a key on
// the border of two codes goes to the same one in every implementation.
#pragma once

#include "device_common.hpp"

namespace ullm {

struct Turn {
  double c, s;
};

// Cosine and sine of p * f.
__device__ __forceinline__ Turn turn_of(int32_t p, float f) {
  constexpr double kHi = 0x1.45f306dc9c883p-3, kLo = -0x1.6b01ec5417056p-57;  // 1 / (2 pi)
  const double hi = double(f) * kHi;
  const double lo = fma(double(f), kHi, -hi) + double(f) * kLo;
  const double turns = fma(double(p), hi, -rint(double(p) * hi)) + double(p) * lo;
  const double quarter = rint(turns * 4);
  const double x = fma(quarter, -0.25, turns) * 0x1.921fb54442d18p+2, z = x * x;
  double s = -1.0 / 1307674368000;
  s = fma(s, z, 1.0 / 6227020800);
  s = fma(s, z, -1.0 / 39916800);
  s = fma(s, z, 1.0 / 362880);
  s = fma(s, z, -1.0 / 5040);
  s = fma(s, z, 1.0 / 120);
  s = fma(s, z, -1.0 / 6);
  s = fma(s * z, x, x);
  double c = 1.0 / 20922789888000;
  c = fma(c, z, -1.0 / 87178291200);
  c = fma(c, z, 1.0 / 479001600);
  c = fma(c, z, -1.0 / 3628800);
  c = fma(c, z, 1.0 / 40320);
  c = fma(c, z, -1.0 / 720);
  c = fma(c, z, 1.0 / 24);
  c = fma(c, z, -0.5);
  c = fma(c, z, 1.0);
  const int q = int(quarter);
  const double a = q % 2 != 0 ? s : c, b = q % 2 != 0 ? c : s;
  return {(q + 1) & 2 ? -a : a, q & 2 ? -b : b};
}

// A double as a float, towards zero with the last bit set where that is not
// exact; magnitudes past the largest float become it.
__device__ __forceinline__ float to_odd(double v) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, v);
  const uint32_t hi = uint32_t(bits >> 32), lo = uint32_t(bits), e = hi >> 20 & 0x7ff;
  const uint32_t odd = (hi & 0x80000000u) | (((hi & 0x7fffffffu) - (896u << 20)) << 3) |
                       lo >> 29 | ((lo & 0x1fffffffu) != 0 ? 1u : 0u);
  const uint32_t past = (hi & 0x80000000u) | 0x7f7fffffu;
  return e == 0x7ff || e <= 896 ? float(v) : bits_f32(e > 896 + 254 ? past : odd);
}

// The dims of pair j of a head: rotated for j < rotary / 2, as they are past it.
struct PairDims {
  uint32_t first, second;
};
__device__ __forceinline__ PairDims pair_dims(uint32_t j, uint32_t rotary, bool interleaved) {
  return interleaved || j >= rotary / 2 ? PairDims{2 * j, 2 * j + 1}
                                        : PairDims{j, j + rotary / 2};
}

}  // namespace ullm
