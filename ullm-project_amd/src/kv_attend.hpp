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
    // A whole reference and the sum's exponent cancel exactly where the log-sum is
    // small and they are not (values of small or large scales).
    const float log2_sum =
        a.whole_refs ? (top + float(__builtin_amdgcn_frexp_expf(sum) - kOff)) +
                           log2f(__builtin_amdgcn_frexp_mantf(sum))
                     : top + (log2f(sum) - float(kOff));
    a.lse[at] = sum == 0.f ? -INFINITY : log2_sum * kLn2;
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
__device__ __forceinline__ void join_waves(JoinLds<D, W> &lds, const KvAttendArgs &a,
                                           const Scratch &x, const Tile &t,
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

// Adds the weights that tokens receive from all rows of their sequence, by a
// second product of keys and queries: a wave owns 32 tokens, whose keys it
// holds as operands, and the rows pass by in tiles of 64 that the workgroup
// stages in LDS, the next tile on its way meanwhile.  Each token's sum has a
// fixed order; the addition is atomic for blocks that several sequences of a
// call share.  Bound as the products above are: 8 products and 48 other vector
// instructions for 32 rows and 32 tokens.  (509 queries of 32 heads at 16384
// tokens: 86 us; with four offsets a lane to move on and rows on their way in
// registers, 125.)
//
// Keys: how a cache's codes become the A operands, and which dims those are.
//
// LDS holds a tile as D / 32 planes of 64 bytes of each row; 16-byte chunk k of
// row r is at place k ^ r / 4 % 4 of the 64, so that 16 neighbours read 16
// groups of banks and a wave copies 16 rows at once, a lane always the same.
constexpr uint32_t kWeightTokens = 32 * kWaves, kWeightRows = 64;

template <class Keys>
__global__ __launch_bounds__(kWaves * kWave, 4) void add_weights_kernel(KvAttendArgs a,
                                                                        const RowStats *stats) {
  constexpr int D = Keys::kDim;
  constexpr uint32_t kPlane = kWeightRows * 64;
  static_assert(kWeightRows == 16 * kWaves, "a wave copies 16 rows of each plane");
  extern __shared__ __align__(1024) uint8_t weight_rows[];
  const auto rows_lds = [](uint32_t stage) { return weight_rows + stage * (D / 32 * kPlane); };
  const uint32_t kvh = blockIdx.y, b = blockIdx.z;
  const uint32_t lane = threadIdx.x % kWave;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const uint32_t h = lane / 32, i = lane % 32;
  const uint32_t first = blockIdx.x * kWeightTokens;
  const uint32_t length = kv_length(a.seqs, a.pool.shift, b);
  if (first >= length) {
    return;
  }
  const KvRows rows = kv_rows(a.seqs, b);
  const int64_t origin = int64_t(length) - rows.count;
  const uint32_t all = rows.count * a.group;
  // Queries before the first token, or past the last one's window, see none.
  const int64_t from = int64_t(first) - origin;
  const uint32_t begin = from <= 0 ? 0u
                         : from < int64_t(rows.count) ? uint32_t(from) * a.group / kWeightRows * kWeightRows
                                                      : all;
  const int64_t past = a.window != 0 ? int64_t(first) + kWeightTokens - 1 + a.window - origin
                                     : int64_t(rows.count);
  const uint32_t end = past <= 0 ? 0u
                       : past < int64_t(rows.count) ? uint32_t(past) * a.group
                                                    : all;

  const uint32_t t0 = first + 32 * wave;
  const int32_t id = t0 < length ? kv_block(a.seqs.tables + b * a.seqs.stride, a.seqs,
                                            a.pool.blocks, t0 >> a.pool.shift)
                                 : -1;
  const uint64_t unit = uint64_t(id < 0 ? 0 : id) * a.pool.heads + kvh;
  const uint32_t in_block = t0 & ((1u << a.pool.shift) - 1);
  bf16x8 k[D / 16];
  Keys::load(a.pool, unit, in_block, lane, k);
#pragma unroll
  for (int c = 0; c < D / 16; ++c) {
    k[c] = flip(k[c], a.q_sign);
  }

  // A row's query, head of the group and offset, moved on by whole tiles
  // without a division or product; rows past the end are the last one's.
  const uint32_t tile_queries = kWeightRows / a.group, tile_heads = kWeightRows % a.group;
  const uint64_t tile_step = tile_queries * a.q_row + tile_heads * a.q_head;
  const uint64_t wrap_step = a.q_row - a.group * a.q_head;
  const uint64_t last_row = (rows.count - 1) * a.q_row + (a.group - 1) * a.q_head;
  struct RowAt {
    uint32_t query, head;
    uint64_t offset;
  };
  const auto row_at = [&](uint32_t r) {
    return RowAt{r / a.group, r % a.group, r / a.group * a.q_row + r % a.group * a.q_head};
  };
  const auto next_tile = [&](RowAt &r) {
    r.head += tile_heads;
    const bool carry = r.head >= a.group;
    r.head -= carry ? a.group : 0u;
    r.query += tile_queries + (carry ? 1u : 0u);
    r.offset += tile_step + (carry ? wrap_step : 0u);
  };
  RowAt mine = row_at(begin + 16 * wave + lane / 4);
  const uint16_t *q_rows = a.q + rows.first * a.q_row + uint64_t(kvh) * a.group * a.q_head +
                           (lane % 4 ^ lane / 16) * 8;
  const auto start_tile = [&](uint8_t *to) {
    const uint16_t *from = q_rows + (mine.query < rows.count ? mine.offset : last_row);
    to += wave * 1024;
    next_tile(mine);
    if (a.vec) {
#pragma unroll
      for (uint32_t c = 0; c < D / 32; ++c) {
        copy_to_lds(reinterpret_cast<const uint8_t *>(from + c * 32), to + c * kPlane);
      }
    } else {
#pragma unroll
      for (uint32_t c = 0; c < D / 32; ++c) {
        *reinterpret_cast<bf16x8 *>(to + c * kPlane + lane * 16) =
            load_query8(from + c * 32, false, 0);
      }
    }
  };
  const RowStats *row_stats = stats + stats_at(a, kvh, rows.first);
  RowStats next[2];
  const auto load_stats = [&](uint32_t r0) {
#pragma unroll
    for (uint32_t u = 0; u < 2; ++u) {
      next[u] = row_stats[min(r0 + 32 * u + i, all - 1)];
    }
  };
  // Rows that see some of the wave's tokens, and all of them.
  struct Range {
    uint32_t first, end;
  };
  const auto range = [&](int64_t from, int64_t past) {
    const auto row = [&](int64_t query) {
      return uint32_t(min(max(query - origin, int64_t(0)), int64_t(rows.count))) * a.group;
    };
    return Range{uniform(row(from)), a.window != 0 ? uniform(row(past + a.window)) : all};
  };
  const Range seen = range(t0, int64_t(t0) + 31), whole = range(int64_t(t0) + 31, t0);
  float sum[16] = {};
  uint32_t stage = 0;
  if (begin < end) {
    load_stats(begin);
    start_tile(rows_lds(0));
  }
  for (uint32_t r0 = begin; r0 < end; r0 += kWeightRows, stage ^= 1) {
    wait_copies<0>();
    step_barrier();
    const RowStats now[2] = {next[0], next[1]};
    if (r0 + kWeightRows < end) {
      load_stats(r0 + kWeightRows);
      start_tile(rows_lds(stage ^ 1));
    }
    if (id < 0 || r0 + kWeightRows <= seen.first || r0 >= seen.end) {
      continue;
    }
    const bool edge = r0 < whole.first || r0 + kWeightRows > whole.end;
    const uint8_t *tile = rows_lds(stage) + i * 64;
#pragma unroll
    for (uint32_t u = 0; u < 2; ++u) {
      bf16x8 q[D / 16];
#pragma unroll
      for (uint32_t c = 0; c < D / 16; ++c) {
        const uint32_t place = Keys::chunk(h, c) ^ i / 4 % 4;
        q[c] = *reinterpret_cast<const bf16x8 *>(tile + Keys::plane(h, c) * kPlane + 32 * u * 64 +
                                                 place * 16);
      }
      f32x16 s = f32x16{};
#pragma unroll
      for (uint32_t c = 0; c < D / 16; ++c) {
        s = mfma32_bf16(k[c], q[c], s);
      }
      float inv_sum = now[u].inv_sum;
      if (edge) {
        // A row of NaN gives it to what it sees, and nothing to the rest.
        const bool bad = inv_sum != inv_sum;
        const float add = bad ? inv_sum : 0.f;
        inv_sum = bad ? 1.f : inv_sum;
        const uint32_t r = r0 + 32 * u + i;
        const int32_t pos = int32_t(origin + r / a.group);
        const int32_t oldest = oldest_hidden(pos, a.window);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int32_t tok = int32_t(t0) + e / 4 * 8 + 4 * int32_t(h) + e % 4;
          s[e] = r < all && tok <= pos && tok > oldest ? s[e] + add : -INFINITY;
        }
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        sum[e] = __builtin_fmaf(exp2_fast(__builtin_fmaf(s[e], a.scale_log2, -now[u].top)),
                                inv_sum, sum[e]);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) {
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      sum[e] += __shfl_xor(sum[e], off, kWave);
    }
    const uint32_t t = e / 4 * 8 + 4 * h + e % 4;
    if (i == uint32_t(e) && id >= 0 && t0 + t < length) {
      unsafeAtomicAdd(&a.pool.weights[(unit << a.pool.shift) + in_block + t], sum[e]);
    }
  }
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
template <typename K>
void launch_add_weights(K kernel, const KvAttendArgs &a, uint32_t dim, const RowStats *stats,
                        hipStream_t s) {
  const uint64_t tokens = uint64_t(a.seqs.max_blocks) << a.pool.shift;
  const dim3 grid(uint32_t((tokens + kWeightTokens - 1) / kWeightTokens), a.pool.heads,
                  a.seqs.batch);
  kernel<<<grid, kWaves * kWave, 2 * kWeightRows * dim * 2, s>>>(a, stats);
}

}  // namespace ullm
