// kv_store.hpp -- what the kernels that write tokens into a cache share: rows of
// bf16, codes of 8 bits, and the end of an append of 8 bits.
#pragma once

#include "kv_cache.hpp"

namespace ullm {

constexpr uint32_t kThreads = 256;

// 16 bf16 of a row, two to a word (two 16-byte loads, or 16 loads where rows
// are unaligned).
struct Bf16x16 {
  u32x4 w[2];
};
__device__ __forceinline__ Bf16x16 load16(const uint16_t *p, bool vec) {
  Bf16x16 r;
  if (vec) {
    r.w[0] = reinterpret_cast<const u32x4 *>(p)[0];
    r.w[1] = reinterpret_cast<const u32x4 *>(p)[1];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      r.w[i / 4][i % 4] = p[2 * i] | uint32_t(p[2 * i + 1]) << 16;
    }
  }
  return r;
}

// The larger magnitude bits in each half of a word, of what was found so far
// and two bf16.
__device__ __forceinline__ uint32_t max_magnitudes(uint32_t top, uint32_t w) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t,
                            __builtin_elementwise_max(__builtin_bit_cast(u16x2, top),
                                                      __builtin_bit_cast(u16x2, w & 0x7fff7fffu)));
}
// Two bf16 with infinities and NaN as 0, or with magnitudes past 448 * 2^119
// as that.
__device__ __forceinline__ uint32_t each_half(uint32_t w, bool finite) {
  const auto one = [&](uint32_t h) {
    const uint32_t m = h & 0x7fffu;
    return finite ? (m < 0x7f80u ? h : 0u) : (m > 0x7f60u && m < 0x7f80u ? h - m + 0x7f60u : h);
  };
  return one(w & 0xffffu) | one(w >> 16) << 16;
}
// Magnitude bits of the largest finite one of N rows' pieces.
template <uint32_t N>
__device__ __forceinline__ uint32_t largest_magnitude(const Bf16x16 (&x)[N]) {
  uint32_t top = 0;
#pragma unroll
  for (uint32_t i = 0; i < 8 * N; ++i) {
    top = max_magnitudes(top, x[i / 8].w[i / 4 % 2][i % 4]);
  }
  if (max(top & 0xffffu, top >> 16) >= 0x7f80u) {  // once more, past infinities and NaN
    top = 0;
#pragma unroll
    for (uint32_t i = 0; i < 8 * N; ++i) {
      top = max_magnitudes(top, each_half(x[i / 8].w[i / 4 % 2][i % 4], true));
    }
  }
  return max(top & 0xffffu, top >> 16);
}
// Smallest exponent e with a <= 448 * 2^e = 1.75 * 2^(e + 8), clamped, of
// magnitude bits of a bf16.
__device__ __forceinline__ int exponent_for(uint32_t a) {
  const int e = int(a >> 7) - 127 - 8 + ((a & 0x7fu) > 0x60u ? 1 : 0);
  return e < kKvExpMin ? kKvExpMin : e > kKvExpMax ? kKvExpMax : e;
}

// Codes of 16 bf16 over 2^e, of magnitudes that 448 * 2^e reaches: rounded to
// nearest even, infinities and NaN to NaN (checked for every bf16).  Only the
// largest exponent leaves finite elements past its reach.
__device__ __forceinline__ u32x4 encode16(Bf16x16 x, int e) {
  typedef short s16x2v __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  if (e == kKvExpMax) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x.w[i / 4][i % 4] = each_half(x.w[i / 4][i % 4], false);
    }
  }
  const float power = exp2_int(e);
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const auto pair = [&](int j) {
      return __builtin_bit_cast(bf16x2, uint32_t(x.w[i / 2][i % 2 * 2 + j]));
    };
    s16x2v r = {0, 0};
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, pair(0), power, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, pair(1), power, true);
    w[i] = __builtin_bit_cast(uint32_t, r);
  }
  return w;
}
// Exponent of a magnitude's f32 bits, likewise.
__device__ __forceinline__ int exponent_for_f32(uint32_t a) {
  const int e = int(a >> 23) - 127 - 8 + ((a & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < kKvExpMin ? kKvExpMin : e > kKvExpMax ? kKvExpMax : e;
}
// Codes of sixteen numbers over 2^e, likewise.
__device__ __forceinline__ u32x4 encode16(const float (&x)[16], int e) {
  typedef short s16x2v __attribute__((ext_vector_type(2)));
  const float power = exp2_int(e);
  const auto fit = [&](float v) {  // past the largest exponent's reach, infinities, NaN
    const float m = __builtin_fabsf(v), most = 448.f * exp2_int(kKvExpMax);
    return m <= most ? v : m < INFINITY ? __builtin_copysignf(most, v) : __builtin_nanf("");
  };
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s16x2v r = {0, 0};
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, fit(x[4 * i]), fit(x[4 * i + 1]), power, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, fit(x[4 * i + 2]), fit(x[4 * i + 3]), power,
                                                 true);
    w[i] = __builtin_bit_cast(uint32_t, r);
  }
  return w;
}
// Codes times powers of two, rounded to codes again; products that 448 does
// not reach are not asked for.  Four codes of four tokens in f32, sixteen of
// one by way of bf16, where every product is exact or rounds to code 0.
__device__ __forceinline__ uint32_t rescale4(uint32_t w, f32x4 f) {
  typedef short s16x2v __attribute__((ext_vector_type(2)));
  typedef float f2 __attribute__((ext_vector_type(2)));
  const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), false);
  const f2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), true);
  s16x2v r = {0, 0};
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, lo[0] * f[0], lo[1] * f[1], 1.0f, false);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, hi[0] * f[2], hi[1] * f[3], 1.0f, true);
  return __builtin_bit_cast(uint32_t, r);
}
__device__ __forceinline__ u32x4 rescale16(u32x4 w, float f) {
  typedef short s16x2v __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const auto lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], f, false);
    const auto hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], f, true);
    s16x2v r = {0, 0};
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, lo, 1.0f, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, hi, 1.0f, true);
    w[i] = __builtin_bit_cast(uint32_t, r);
  }
  return w;
}

__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const uint32_t o = __shfl_xor(v, off, kWave);
    v = o > v ? o : v;
  }
  return v;
}
// Maxima of two values over the workgroup.
template <uint32_t THREADS = kThreads>
__device__ __forceinline__ void block_umax2(uint32_t &a, uint32_t &b) {
  __shared__ uint32_t red[2][THREADS / kWave];
  a = wave_umax(a);
  b = wave_umax(b);
  if (threadIdx.x % kWave == 0) {
    red[0][threadIdx.x / kWave] = a;
    red[1][threadIdx.x / kWave] = b;
  }
  __syncthreads();
  for (uint32_t i = 0; i < THREADS / kWave; ++i) {
    a = red[0][i] > a ? red[0][i] : a;
    b = red[1][i] > b ? red[1][i] : b;
  }
  __syncthreads();
}

// Token j (0..7) of the 8 that lane group g of a 32-token value tile holds.
__device__ __forceinline__ uint32_t value_token(uint32_t g, uint32_t j) {
  return 4 * g + j % 4 + 16 * (j / 4);
}

// The append of a block in 8 bits: the keys of its first `lo` tokens times a
// factor.
template <int D, uint32_t THREADS = kThreads>
__device__ __forceinline__ void rescale_keys(uint8_t *kc, uint32_t lo, float f) {
  if (f != 1.f) {
    for (uint32_t u = threadIdx.x; u < lo * (D / 16); u += THREADS) {
      u32x4 *at =
          reinterpret_cast<u32x4 *>(kc + kv_key_unit<D>(u / (D / 16), threadIdx.x % (D / 16)));
      *at = rescale16(*at, f);
    }
  }
}
// A token's codes (dims 16c ..) to their places among the values.
template <int D>
__device__ __forceinline__ void place_value(uint8_t *image, uint32_t t, uint32_t c, u32x4 w) {
  uint8_t *at = image + kv_value_byte<D>(t, c * 16);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    at[i * 16] = uint8_t(w[i / 4] >> (8 * (i % 4)));
  }
}
// New values lo .. hi - 1 of the image to memory, beside those before them times
// a factor.
template <int D, uint32_t THREADS = kThreads>
__device__ __forceinline__ void store_values(const uint8_t *image, uint8_t *vc, uint32_t lo,
                                             uint32_t hi, float fv) {
  const uint32_t tid = threadIdx.x;
  // Units of 8 tokens x 2 dims: unit u of the block's has tokens t .. t + 3 and
  // t + 16 .. t + 19.
  const uint32_t vfrom = fv != 1.f ? 0u : lo / 32 * 32;
  for (uint32_t u = vfrom * (D / 16) + tid; u < (hi + 31) / 32 * (2 * D); u += THREADS) {
    const uint32_t t = u / (2 * D) * 32 + u % 64 / 16 * 4;
    // Bytes of the new ones among four tokens from t0 on.  (Signed differences:
    // of an unsigned one that a condition guards the compiler has concluded
    // that the condition always holds.)
    const auto bytes = [&](uint32_t t0) {
      const auto below = [&](uint32_t end) {
        const int n = min(max(int(end) - int(t0), 0), 4);
        return uint32_t((uint64_t(1) << (8 * n)) - 1);
      };
      return below(hi) & ~below(lo);
    };
    const uint32_t new0 = bytes(t), new1 = bytes(t + 16);
    const bool kept = t < lo;
    if ((new0 | new1) == 0 && (fv == 1.f || !kept)) {
      continue;
    }
    u32x4 *at = reinterpret_cast<u32x4 *>(vc) + u;
    const u32x4 now = reinterpret_cast<const u32x4 *>(image)[u];
    u32x4 w = {0u, 0u, 0u, 0u};
    if (kept) {
      w = fv != 1.f ? rescale16(*at, fv) : *at;
    }
    *at = u32x4{(now.x & new0) | (w.x & ~new0), (now.y & new1) | (w.y & ~new1),
                (now.z & new0) | (w.z & ~new0), (now.w & new1) | (w.w & ~new1)};
  }
}

}  // namespace ullm
