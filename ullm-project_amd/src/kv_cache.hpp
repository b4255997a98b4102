// kv_cache.hpp -- HBM layout of the 8-bit key/value cache, and its launchers.
//
// A block of bt tokens holds, for each key/value head, bt * D bytes of key
// codes followed by bt * D bytes of value codes, as 1 KiB wave tiles that one
// wave fetches with a 16-byte-per-lane load and feeds to the matrix cores as
// they are:
//
//   keys, tile (t / 16, d / 64): lane l holds token l % 16, dims
//     16 * (l / 16) .. +15 of the 64, the order of the FP8 weight tiles
//     (layout.hpp): the A operand of S^T = K Q^T.
//   values, tile (t / 32, d / 32): lane l = d % 16 + 16 * g holds, for dim
//     d % 16 (bytes 0..7) and d % 16 + 16 (bytes 8..15), the tokens
//     4g .. 4g + 3 and 16 + 4g .. 16 + 4g + 3 of the 32: the A operand of
//     O^T = V^T P^T when the softmax weights stay in the registers that
//     S^T left them in (lane group g of a 16 x 16 result holds rows 4g .. 4g + 3).
//
// exps: int8 [blocks][kv_heads][2], the exponents of keys and values.
// weights: f32 [blocks][kv_heads][bt], or null.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "device_common.hpp"
#include "ullm/kv_cache.h"

struct ullm_kv_cache_t {
  uint64_t blocks = 0;
  uint32_t block_tokens = 0, kv_heads = 0, head_dim = 0, flags = 0;
  int device = 0;
  uint8_t *codes = nullptr;
  int8_t *exps = nullptr;
  float *weights = nullptr;
  uint64_t device_bytes = 0;
};

namespace ullm {

constexpr int kKvExpMin = -100, kKvExpMax = 119;

struct KvPool {
  uint8_t *codes;
  int8_t *exps;
  float *weights;
  uint32_t blocks;
  uint32_t shift;  // log2 of the block's tokens
  uint32_t heads;  // key/value heads
};

struct KvSeqs {
  const int32_t *tables;
  uint64_t stride;
  uint32_t max_blocks;
  const int32_t *lengths;
  const int32_t *starts;  // null: `each` rows per sequence
  uint32_t batch, rows, each;
};

struct KvAppendArgs {
  KvPool pool;
  KvSeqs seqs;
  const uint16_t *k, *v;
  uint64_t k_row, k_head, v_row, v_head;  // strides, elements
  bool vec;  // rows 16-byte aligned
  const float *weights;
};
struct KvGatherArgs {
  KvPool pool;
  KvSeqs seqs;
  uint16_t *k, *v;
  float *weights;
};
struct KvEvictArgs {
  KvPool pool;
  KvSeqs seqs;
  const int32_t *new_tables;
  uint64_t new_stride;
  int32_t *new_lengths;
  int32_t *kept;
  uint32_t keep, sink, recent;
};
struct KvAttendArgs {
  KvPool pool;
  KvSeqs seqs;
  const uint16_t *q;
  uint16_t *out;
  uint64_t q_row, q_head, out_row, out_head;  // strides, elements
  bool vec;      // query rows 16-byte aligned
  bool out_vec;  // output rows 8-byte aligned
  float *lse;    // [rows][heads] or null
  uint32_t heads, group;
  uint32_t window;
  float scale_log2;  // |scale| * log2(e), not 0
  uint32_t q_sign;   // 0x80008000 if the scale is negative: two queries' signs
  bool accumulate;
};
struct KvAttendPlan {
  uint32_t kernel = 0, row_tile = 0, parts = 1, part_tokens = 0;
  uint32_t waves = 4;
  bool keep_scores = false;  // weights from stored scores
  bool one_tile = false;     // sequences have one tile of rows, on average
  uint64_t grid = 0, workspace = 0;
};

hipError_t launch_kv_append(const KvAppendArgs &a, uint32_t dim, hipStream_t s);
hipError_t launch_kv_gather(const KvGatherArgs &a, uint32_t dim, hipStream_t s);
hipError_t launch_kv_evict(const KvEvictArgs &a, uint32_t dim, hipStream_t s);
KvAttendPlan plan_kv_attend(const KvAttendArgs &a, uint32_t dim);
hipError_t launch_kv_attend(const KvAttendArgs &a, uint32_t dim, const KvAttendPlan &p,
                            void *workspace, hipStream_t s);

// ---------------------------------------------------------------- device side

// Byte offset of the 16-byte unit (token t, dims 16c .. 16c + 15) of a block
// and head's keys.
template <int D>
__host__ __device__ constexpr uint32_t kv_key_unit(uint32_t t, uint32_t c) {
  return ((t / 16) * (D / 64) + c / 4) * 1024 + (t % 16 + 16 * (c % 4)) * 16;
}
// Byte offset of (token t, dim d) of its values.
template <int D>
__host__ __device__ constexpr uint32_t kv_value_byte(uint32_t t, uint32_t d) {
  return ((t / 32) * (D / 32) + d / 32) * 1024 + (d % 16 + 16 * ((t % 16) / 4)) * 16 +
         8 * ((d % 32) / 16) + t % 4 + 4 * ((t % 32) / 16);
}

// 2^e for e in -126 .. 127.
__device__ __forceinline__ float exp2_int(int e) {
  return bits_f32(uint32_t(e + 127) << 23);
}

__device__ __forceinline__ uint32_t kv_length(const KvSeqs &s, uint32_t shift, uint32_t b) {
  const int64_t n = s.lengths[b], most = int64_t(s.max_blocks) << shift;
  return uint32_t(n < 0 ? 0 : n < most ? n : most);
}
// Rows first .. first + count - 1 of sequence b.
struct KvRows {
  uint32_t first, count;
};
__device__ __forceinline__ uint32_t kv_start(const KvSeqs &s, uint32_t b) {
  const int32_t v = s.starts[b];
  return v < 0 ? 0u : uint32_t(v) < s.rows ? uint32_t(v) : s.rows;
}
__device__ __forceinline__ KvRows kv_rows(const KvSeqs &s, uint32_t b) {
  if (s.starts == nullptr) {
    return {b * s.each, s.each};
  }
  const uint32_t lo = kv_start(s, b), hi = kv_start(s, b + 1);
  return {lo, hi > lo ? hi - lo : 0u};
}
// Pool block of column j of a sequence's table, or -1.
__device__ __forceinline__ int32_t kv_block(const int32_t *table, const KvSeqs &s,
                                            uint32_t blocks, uint32_t j) {
  const int32_t id = j < s.max_blocks ? table[j] : -1;
  return id >= 0 && uint32_t(id) < blocks ? id : -1;
}

// Slots of work over ragged sequences without a host-side plan: sequence b
// owns the slots from starts[b] * mult / tile + extra * b on.  Since
// floor(x + y) + 1 >= floor(x) + ceil(y), `extra` = 1 leaves it room for
// ceil(count * mult / tile) slots.  Returns the sequence of slot `id` (every
// lane of a wave calls it with the same one), its rows and the slot's number
// within it; seq >= batch when there is none.  64 offsets are looked at with
// one load.
struct KvSlot {
  uint32_t seq, local;
  KvRows rows;
};
__device__ __forceinline__ KvSlot kv_find_slot(const KvSeqs &s, uint32_t id, uint32_t mult,
                                               uint32_t tile, uint32_t extra,
                                               uint32_t each_slots) {
  if (s.starts == nullptr) {
    const uint32_t b = id / each_slots;
    return {b, id % each_slots, {b * s.each, s.each}};
  }
  const uint32_t lane = threadIdx.x % kWave;
  KvSlot r{s.batch, 0, {0, 0}};
  for (uint32_t c = 0; c < s.batch; c += kWave) {
    const uint32_t b = c + lane;
    const uint32_t at = kv_start(s, b < s.batch ? b : s.batch);
    const uint64_t slot0 = uint64_t(at) * mult / tile + uint64_t(extra) * b;
    const uint32_t n = uint32_t(__popcll(__ballot(b < s.batch && slot0 <= id)));
    if (n != 0) {
      r.seq = c + n - 1;
      r.local = id - uint32_t(__builtin_amdgcn_readlane(int(slot0), n - 1));
      r.rows.first = uint32_t(__builtin_amdgcn_readlane(int(at), n - 1));
      const uint32_t next = n < kWave ? uint32_t(__builtin_amdgcn_readlane(int(at), n & 63))
                                      : kv_start(s, c + kWave);
      r.rows.count = next > r.rows.first ? next - r.rows.first : 0u;
    }
    if (n < kWave) {
      break;
    }
  }
  return r;
}
// The most tokens of a part that touches at most `blocks` blocks of 2^shift
// tokens, wherever it starts: with a window the first part of a tile starts at
// any 32-token group, so that up to a block less 32 tokens precede it in its
// first block; without one parts start at multiples of their size, which is
// one of 64.
constexpr uint64_t kv_part_limit(uint32_t blocks, uint32_t shift, uint32_t window) {
  return (uint64_t(blocks) << shift) - (window != 0 ? (1u << shift) - 32u : 0u);
}

// Keys from .. from + width, cut into at most 4096 bins of 2^shift keys, and
// the keys of one of the bins that has any: its end is the range's where it
// reaches past that, for past 2^32 keys begin again at 0.
struct KvKeyRange {
  uint32_t from, width;
};
constexpr uint32_t kKvBinBits = 12;
__host__ __device__ constexpr uint32_t kv_bin_shift(KvKeyRange r) {
  const uint32_t bits = 32 - uint32_t(__builtin_clz(r.width | 1));
  return bits > kKvBinBits ? bits - kKvBinBits : 0;
}
__host__ __device__ constexpr KvKeyRange kv_bin_keys(KvKeyRange r, uint32_t shift, uint32_t bin) {
  const uint32_t skipped = bin << shift, most = (1u << shift) - 1;
  return {r.from + skipped, r.width - skipped < most ? r.width - skipped : most};
}

inline uint64_t kv_slots(const KvSeqs &s, uint64_t mult, uint64_t tile, uint64_t extra,
                         uint64_t each_slots) {
  return s.starts == nullptr ? uint64_t(s.batch) * each_slots
                             : uint64_t(s.rows) * mult / tile + extra * s.batch;
}

}  // namespace ullm
