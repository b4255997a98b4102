// kv_cache4.hpp -- HBM layout of the 4-bit key/value cache, and its launchers.
//
// A block of a head is a run of chunks of 32 tokens, each whole: codes of keys,
// codes of values, exponents of keys, scales of values, so that a wave finds
// all it needs of 32 tokens at constant offsets from one address.
//
//   keys, D / 64 KiB.  Lane l = t % 16 + 16 * g of a wave holds dims D / 4 * g ..
//     of tokens t and t + 16, low nibble first: 16 bytes of each in tiles of
//     1 KiB (128 dims; the 16 bytes are one scale's 32 dims), or 8 bytes of each
//     side by side (64 dims).  Eight codes in order are a lane's part of the A
//     operand of S^T = K Q^T, for any order of dims that the queries share.
//   values, D / 64 KiB, 64 dims each: lane l = d % 16 + 16 * g holds a dword for
//     each of dims d, d + 16, d + 32, d + 48: nibble j is token
//     4g + j % 4 + 16 * (j / 4), the order of a lane's softmax weights as S^T
//     leaves them (kv_cache.hpp).
//   exponents, D bytes: of tokens t, t + 16 side by side, at
//     (t % 16 + 16 * (d / 32)) * 2; the exponent plus 127, or 255 for NaN.
//   scales, 64 bytes: f16, in the order of the values' nibbles: 8 for each g.
#pragma once

#include "kv_cache.hpp"
#include "ullm/kv_cache4.h"
#include "ullm/kv_rotary.h"

namespace ullm {

template <int D>
struct Kv4Chunk {
  static constexpr uint32_t kSide = 16 * D;  // codes of one side
  static constexpr uint32_t kExps = 2 * kSide, kScales = kExps + D, kBytes = kScales + 64;
};
constexpr uint64_t kv4_chunk_bytes(uint32_t dim) { return 33 * uint64_t(dim) + 64; }

// Chunk `in_block` / 32 of a block and head.
template <int D>
__device__ __forceinline__ uint8_t *kv4_chunk(const KvPool &p, uint64_t unit, uint32_t in_block) {
  return p.codes + ((unit << p.shift) + in_block) / 32 * Kv4Chunk<D>::kBytes;
}

// Byte of (token t of 32, dim d) of the keys, an even d in the low nibble.
template <int D>
__host__ __device__ constexpr uint32_t kv4_key_byte(uint32_t t, uint32_t d) {
  return D == 128 ? t / 16 * 1024 + (t % 16 + 16 * (d / 32)) * 16 + d % 32 / 2
                  : (t % 16 + 16 * (d / 16)) * 16 + t / 16 * 8 + d % 16 / 2;
}
// Number of token t of 32 among the 8 of its lane group.
__host__ __device__ constexpr uint32_t kv4_value_slot(uint32_t t) { return t % 4 + 4 * (t / 16); }
__host__ __device__ constexpr uint32_t kv4_value_group(uint32_t t) { return t % 16 / 4; }
// Byte of the dword that dim d has for the tokens of lane group g.
__host__ __device__ constexpr uint32_t kv4_value_dword(uint32_t g, uint32_t d) {
  return d / 64 * 1024 + (d % 16 + 16 * g) * 16 + d % 64 / 16 * 4;
}
__host__ __device__ constexpr uint32_t kv4_exp_byte(uint32_t t, uint32_t d) {
  return (t % 16 + 16 * (d / 32)) * 2 + t / 16;
}
__host__ __device__ constexpr uint32_t kv4_scale_byte(uint32_t t) {
  return (8 * kv4_value_group(t) + kv4_value_slot(t)) * 2;
}

constexpr uint32_t kKv4ExpNan = 255;
constexpr float kScaleLeast = 0x1p-19f, kScaleMost = 64512.f;  // of values
constexpr uint16_t kScaleMostBits = 0x7be0;                    // in f16

// Eight codes as bf16 operands, times a power of two (NaN where its exponent is
// that of infinity); as f16 operands.
__device__ __forceinline__ bf16x8 codes4_to_bf16(uint32_t w, float power) {
  u32x4 r;
  r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, power, 0));
  r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, power, 1));
  r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, power, 2));
  r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, power, 3));
  return __builtin_bit_cast(bf16x8, r);
}
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ f16x8 codes4_to_f16(uint32_t w) {
  u32x4 r;
  r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.f, 0));
  r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.f, 1));
  r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.f, 2));
  r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.f, 3));
  return __builtin_bit_cast(f16x8, r);
}

// How queries and keys are rotated on the way; dims = 0: not at all.
struct KvRotary {
  const float *inv_freq;
  const int32_t *positions;  // null: places in the sequence
  uint64_t position_stride;
  const uint8_t *pair_axes;  // null: axis 0
  uint32_t dims, axes;
  bool interleaved;
};
struct KvRotateArgs {
  KvAppendArgs append;
  KvRotary rotary;
  const uint16_t *q;
  uint16_t *q_out;
  uint64_t q_row, q_head, out_row, out_head;  // strides, elements
  bool q_vec;                                 // rows of q and q_out 16-byte aligned
  uint32_t group;                             // query heads of a key/value head
};

// Into a cache of 4 bits, rotated if rotary.dims != 0; into one of 8, rotated.
hipError_t launch_kv4_append(const KvRotateArgs &a, uint32_t dim, hipStream_t s);
hipError_t launch_kv8_append_rotary(const KvRotateArgs &a, uint32_t dim, hipStream_t s);
// Threads of these launches, which count them in 32 bits.
uint64_t kv4_append_threads(const KvAppendArgs &a);
uint64_t kv8_append_rotary_threads(const KvAppendArgs &a, uint32_t dim);
hipError_t launch_kv4_gather(const KvGatherArgs &a, uint32_t dim, hipStream_t s);
hipError_t launch_kv4_evict(const KvEvictArgs &a, uint32_t dim, hipStream_t s);
KvAttendPlan plan_kv4_attend(const KvAttendArgs &a, uint32_t dim);
hipError_t launch_kv4_attend(const KvAttendArgs &a, uint32_t dim, const KvAttendPlan &p,
                             void *workspace, hipStream_t s);

}  // namespace ullm
