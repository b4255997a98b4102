// kv_attend.hpp -- what the attention kernels of the 8-bit and the 4-bit cache
// share: tiles of rows, the softmax's scratch, the end of a kernel, and the
// launches that work on scratch alone.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kernels.hpp"
#include "kv_cache.hpp"

namespace ullm {

constexpr uint32_t kRows = 16;  // rows of a tile
constexpr uint32_t kWaves = 4;
constexpr float kLn2 = 0.693147180559945309f;
constexpr int kOff = 11;             // weights are at most 2^kOff in f16

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mfma_f16(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ uint32_t f32x2_to_f16x2(float lo, float hi) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{lo, hi}, h2));
}
// Results below 2^-126 become 0.
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Softmax statistics of a row: scores are in units of log2, weight =
// exp2(score - top) * inv_sum.
struct RowStats {
  float top, inv_sum;
};

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 mfma32_bf16(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32_f16(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// Eight elements of a query, negated if the scale is negative (so that scores
// and products have one order and a maximum can be taken before scaling).
__device__ __forceinline__ bf16x8 flip(bf16x8 v, uint32_t sign) {
  const u32x4 w = __builtin_bit_cast(u32x4, v);
  return __builtin_bit_cast(bf16x8, u32x4{w.x ^ sign, w.y ^ sign, w.z ^ sign, w.w ^ sign});
}
__device__ __forceinline__ bf16x8 load_query8(const uint16_t *p, bool vec, uint32_t sign) {
  u32x4 w;
  if (vec) {
    w = *reinterpret_cast<const u32x4 *>(p);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = p[2 * i] | uint32_t(p[2 * i + 1]) << 16;
    }
  }
  return flip(__builtin_bit_cast(bf16x8, w), sign);
}

// Codes that one workgroup alone reads pass the caches by (nontemporal: 47
// against 53 us for 131072 tokens of 8 heads); with several tiles of rows to a
// sequence the later ones find them there.
template <bool NT>
__device__ __forceinline__ u32x4 load_codes(const u32x4 *p) {
  return NT ? __builtin_nontemporal_load(p) : *p;
}

__device__ __forceinline__ uint32_t uniform(uint32_t v) {
  return uint32_t(__builtin_amdgcn_readfirstlane(int(v)));
}

// Rows of a tile: positions of the queries, the tokens they can see.
struct Tile {
  uint32_t seq, length, first_row, count;  // the sequence, its rows
  uint32_t r0, live;                       // the tile's rows in the sequence's list
  int64_t origin;                          // position of the sequence's first query
  int64_t low, high;                       // positions of the tile's first and last query
  uint32_t begin, end;                     // tokens that some row sees
};

// The rows of a slot or of tile `id`; false if it has none.
__device__ __forceinline__ bool slot_rows(const KvAttendArgs &a, const KvSlot &slot, uint32_t rows,
                                          Tile *t) {
  const uint32_t all = slot.rows.count * a.group;
  t->seq = slot.seq;
  t->first_row = slot.rows.first;
  t->count = slot.rows.count;
  t->r0 = slot.local * rows;
  t->live = all - t->r0 < rows ? all - t->r0 : rows;
  return slot.seq < a.seqs.batch && t->r0 < all;
}
__device__ __forceinline__ bool tile_rows(const KvAttendArgs &a, uint32_t id, uint32_t rows,
                                          uint32_t each_slots, Tile *t) {
  return slot_rows(a, kv_find_slot(a.seqs, id, a.group, rows, 1, each_slots), rows, t);
}
// The tiles of all sequences by their number in the sequence, highest first:
// of prompts that see themselves the last tiles take longest, so they start
// first (prompts of 4096 and 3001 tokens: 229 us; sequence by sequence 243).
// Lane i looks at 64 numbers at once, one walk over the sequences for each
// factor of 64 in the tiles; of more than 64 sequences none takes long, and
// they are left in their order.  `slots`: ids in the grid.
__device__ __forceinline__ bool tile_rows_last_first(const KvAttendArgs &a, uint32_t id,
                                                     uint32_t slots, uint32_t rows,
                                                     uint32_t each_slots, Tile *t) {
  const uint32_t batch = a.seqs.batch;
  if (a.seqs.starts == nullptr) {
    const uint32_t b = id % batch;
    return slot_rows(a, {b, each_slots - 1 - id / batch, {b * a.seqs.each, a.seqs.each}}, rows, t);
  }
  if (batch > kWave) {
    return tile_rows(a, slots - 1 - id, rows, each_slots, t);
  }
  const uint32_t lane = threadIdx.x % kWave;
  const KvRows mine = kv_rows(a.seqs, lane < batch ? lane : 0);
  const uint32_t tiles =
      lane < batch ? uint32_t((uint64_t(mine.count) * a.group + rows - 1) / rows) : 0u;
  uint32_t step = 1;
  while (__any(tiles > kWave * step)) {
    step *= kWave;
  }
  // The lowest number that at most `id` tiles are above of lies in
  // [number, number + 64 step): lane i looks at the end of its 64th of that.
  uint32_t number = 0, above = 0;
  for (; step != 0; step /= kWave) {
    const uint32_t next = number + (lane + 1) * step;
    uint32_t n = 0;
    for (uint32_t b = 0; b < batch; ++b) {
      const uint32_t of_b = uint32_t(__builtin_amdgcn_readlane(int(tiles), int(b)));
      n += of_b > next ? of_b - next : 0u;
    }
    const uint32_t first = uint32_t(__builtin_ctzll(__ballot(n <= id)));
    number += first * step;
    above = uint32_t(__builtin_amdgcn_readlane(int(n), int(first)));
  }
  // Of the tiles of this number, the one of the (id - above)-th sequence.
  const bool has = tiles > number;
  const uint64_t with = __ballot(has);
  const uint64_t mask = __ballot(
      has && uint32_t(__popcll(with & ((uint64_t(1) << lane) - 1))) == id - above);
  if (mask == 0) {
    return false;
  }
  const uint32_t b = uint32_t(__builtin_ctzll(mask));
  return slot_rows(a,
                   {b, number,
                    {uint32_t(__builtin_amdgcn_readlane(int(mine.first), int(b))),
                     uint32_t(__builtin_amdgcn_readlane(int(mine.count), int(b)))}},
                   rows, t);
}
// Their positions, from the sequence's length.
__device__ __forceinline__ void tile_tokens(const KvAttendArgs &a, uint32_t length, Tile *t) {
  t->length = length;
  t->origin = int64_t(length) - t->count;
  t->low = t->origin + t->r0 / a.group;
  t->high = t->origin + (t->r0 + t->live - 1) / a.group;
  const int64_t begin = a.window != 0 ? t->low - int64_t(a.window) + 1 : 0;
  t->begin = begin > 0 ? uint32_t(begin) : 0u;
  t->end = t->high >= 0 ? uint32_t(t->high + 1) : 0u;
}

// Where a group lies and which of its tokens the lane's row sees.
struct Place {
  int32_t pos, oldest;  // the row's query, and the newest token that it no longer sees
  int32_t low;          // first query of the tile
  int32_t hidden;       // newest token that the tile's last query no longer sees
};

// The newest token that a query at `pos` no longer sees, -1 if it sees all.
__device__ __forceinline__ int32_t oldest_hidden(int64_t pos, uint32_t window) {
  const int64_t t = window != 0 ? pos - int64_t(window) : -1;
  return t > -1 ? int32_t(t) : -1;
}

// Maximum over the four lane groups of a column.
__device__ __forceinline__ float max_groups(float v) {
  const auto half = __builtin_amdgcn_permlane32_swap(f32_bits(v), f32_bits(v), false, false);
  v = fmaxf(bits_f32(half[0]), bits_f32(half[1]));
  const auto row = __builtin_amdgcn_permlane16_swap(f32_bits(v), f32_bits(v), false, false);
  return fmaxf(bits_f32(row[0]), bits_f32(row[1]));
}

// Results of a part of a row's tokens: the mean of the values by weight, and
// what joins it with the other parts.
struct PartSum {
  float m, l;
};

// Scratch of a call: partial results [row][head][part], row statistics
// [row][head] and scores [row][head][token].
struct Scratch {
  float *part_o;
  PartSum *part_s;
  RowStats *stats;
  float *scores;
  uint64_t score_stride;
  uint32_t parts, part_tokens;
};

__device__ __forceinline__ uint32_t part_count(const Tile &t, uint32_t part_tokens) {
  const uint32_t from = t.begin / 32 * 32;
  return t.end > from ? (t.end - from + part_tokens - 1) / part_tokens : 0u;
}

// Place of the first of a row's statistics for a key/value head: rows and the
// heads of the group run on in the order of a tile's rows.
__device__ __forceinline__ uint64_t stats_at(const KvAttendArgs &a, uint32_t kvh, uint64_t row) {
  return (uint64_t(kvh) * a.seqs.rows + row) * a.group;
}

// Log-sum and statistics of a row.
__device__ __forceinline__ void store_stats(const KvAttendArgs &a, const Scratch &x, uint64_t row,
                                            uint32_t head, float top, float sum) {
  const uint64_t at = row * a.heads + head;
  if (a.lse != nullptr) {
    a.lse[at] = sum == 0.f ? -INFINITY : (top + (log2f(sum) - float(kOff))) * kLn2;
  }
  if (x.stats != nullptr) {
    x.stats[stats_at(a, head / a.group, row) + head % a.group] = RowStats{(top == -INFINITY ? 0.f : top) - float(kOff),
                           sum == 0.f ? 0.f : 1.0f / sum};
  }
}

// Final results of a row: `n` elements of the output from dim d0 on, log-sum
// and statistics.
template <int N>
__device__ __forceinline__ void store_row(const KvAttendArgs &a, const Scratch &x, uint64_t row,
                                          uint32_t head, uint32_t d0, const float (&v)[N],
                                          float top, float sum) {
  const float join = sum == 0.f ? 0.f : 1.0f / sum;
  uint16_t *to = a.out + row * a.out_row + head * a.out_head + d0;
  uint32_t packed[N / 2];
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    packed[i] = f32x2_to_bf16x2(v[2 * i] * join, v[2 * i + 1] * join);
  }
  if (N % 4 == 0 && a.out_vec) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      reinterpret_cast<u32x2 *>(to)[i] = u32x2{packed[2 * i], packed[2 * i + 1]};
    }
  } else {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      to[2 * i] = uint16_t(packed[i]);
      to[2 * i + 1] = uint16_t(packed[i] >> 16);
    }
  }
  if (d0 == 0) {
    store_stats(a, x, row, head, top, sum);
  }
}

// Where a row's result goes: its part, or the output itself.
struct RowSink {
  uint64_t row;
  uint32_t head;
  bool live, whole;
  uint64_t slot;
};
__device__ __forceinline__ void store4(const KvAttendArgs &a, const Scratch &x, const RowSink &to,
                                       uint32_t dim, uint32_t d0, f32x4 v) {
  if (!to.live) {
    return;
  }
  if (!to.whole) {
    *reinterpret_cast<f32x4 *>(x.part_o + to.slot * dim + d0) = v;
    return;
  }
  uint16_t *p = a.out + to.row * a.out_row + to.head * a.out_head + d0;
  const u32x2 w = {f32x2_to_bf16x2(v[0], v[1]), f32x2_to_bf16x2(v[2], v[3])};
  if (a.out_vec) {
    *reinterpret_cast<u32x2 *>(p) = w;
  } else {
    p[0] = uint16_t(w.x);
    p[1] = uint16_t(w.x >> 16);
    p[2] = uint16_t(w.y);
    p[3] = uint16_t(w.y >> 16);
  }
}
__device__ __forceinline__ void store_sums(const KvAttendArgs &a, const Scratch &x,
                                           const RowSink &to, float top, float sum) {
  if (to.live && to.whole) {
    store_stats(a, x, to.row, to.head, top, sum);
  } else if (to.live) {
    x.part_s[to.slot] = PartSum{top, sum};
  }
}

// The end of a kernel whose W waves each met some of a part's tokens for a tile
// of 16 rows: wave w's running maximum and sum of a row in lane r and the lanes
// 16, 32 and 48 after it (of the sum each a part), its accumulators over `power`
// as a product of 16 dims and the rows leaves them.  Joined in LDS, stored as
// the result or as a part of it.
template <int D, int W>
struct JoinLds {
  alignas(16) float o[W][kRows][D + 4];
  float m[W][kRows], l[W][kRows];
};
template <int D, int W>
__device__ __forceinline__ void join_waves(JoinLds<D, W> &lds, const KvAttendArgs &a, const Scratch &x, const Tile &t,
                                           uint32_t kvh, uint32_t part, uint32_t parts, float m,
                                           float lane_sum, const f32x4 (&o)[D / 16],
                                           float power) {
  auto &part_o = lds.o;
  auto &part_m = lds.m;
  auto &part_l = lds.l;
  const uint32_t lane = threadIdx.x % kWave;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const uint32_t g = lane / 16, col = lane % 16;
  float l = lane_sum + __shfl_xor(lane_sum, 16, kWave);
  l += __shfl_xor(l, 32, kWave);
  if (g == 0) {
    part_m[wave][col] = m;
    part_l[wave][col] = l;
  }
  // Means of the wave's tokens, to be joined by their sums.
  const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    *reinterpret_cast<f32x4 *>(&part_o[wave][col][16 * i + 4 * g]) = o[i] * inv * power;
  }
  __syncthreads();
  constexpr int kPer = D / (4 * W);  // dims of a thread: 4 W threads to a row
  const uint32_t own = threadIdx.x / (4 * W);
  if (own >= t.live) {
    return;
  }
  const uint32_t rr = t.r0 + own;
  const uint64_t out_row = t.first_row + rr / a.group;
  const uint32_t out_head = kvh * a.group + rr % a.group;
  float top = part_m[0][own];
#pragma unroll
  for (int w = 1; w < W; ++w) {
    top = fmaxf(top, part_m[w][own]);
  }
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f, f[W];
#pragma unroll
  for (int w = 0; w < W; ++w) {
    f[w] = exp2_fast(part_m[w][own] - ref) * part_l[w][own];
    sum += f[w];
  }
  const uint32_t d0 = threadIdx.x % (4 * W) * kPer;
  float v[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    v[i] = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      v[i] += part_o[w][own][d0 + i] * f[w];
    }
  }
  if (parts <= 1) {
    store_row(a, x, out_row, out_head, d0, v, top, sum);
    return;
  }
  const uint64_t slot = (out_row * a.heads + out_head) * x.parts + part;
  const float join = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    x.part_o[slot * D + d0 + i] = v[i] * join;
  }
  if (d0 == 0) {
    x.part_s[slot] = PartSum{top, sum};
  }
}

// 16 bytes per lane from memory into LDS at the wave's base.
__device__ __forceinline__ void copy_to_lds(const uint8_t *from, uint8_t *to) {
  __builtin_amdgcn_global_load_lds(
      reinterpret_cast<const __attribute__((address_space(1))) void *>(
          reinterpret_cast<uintptr_t>(from)),
      (__attribute__((address_space(3))) void *)(to), 16, 0, 0);
}
template <int N>
__device__ __forceinline__ void wait_copies() {
  __builtin_amdgcn_s_waitcnt((N & 0xf) | ((N >> 4) << 14) | (0x7 << 4) | (0xf << 8));
}
// Workgroup barrier that waits for this wave's LDS reads only.
__device__ __forceinline__ void step_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Host side (kv_attend.hip).

// Scratch of a plan in its order: partial results, row statistics, scores.
Scratch scratch_of(const KvAttendArgs &a, uint32_t dim, const KvAttendPlan &p, void *ws,
                   uint64_t *bytes);
// Tiles of `rows` rows of a sequence, where each has as many rows.
inline uint64_t each_tiles(const KvAttendArgs &a, uint32_t rows) {
  return (uint64_t(a.seqs.each) * a.group + rows - 1) / rows;
}
// Joins the parts of all rows, adds the weights of stored scores.
void launch_join_parts(const KvAttendArgs &a, uint32_t dim, const KvAttendPlan &p,
                       const Scratch &x, hipStream_t s);
void launch_add_scores(const KvAttendArgs &a, const Scratch &x, hipStream_t s);

}  // namespace ullm
