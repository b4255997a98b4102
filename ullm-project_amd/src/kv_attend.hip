// kv_attend.hip -- softmax attention over the 8-bit key/value cache.
//
// Rows.  The queries of a sequence and the heads that share a key/value head
// form one list of rows r = i * group + h (query i, head h of the group); a
// tile of them meets the keys and values of that head once.
//
// Scores.  S^T = K Q^T on v_mfma_f32_16x16x32_bf16, the keys converted to
// bf16 in registers (exact, scale included: v_cvt_scalef32_pk_bf16_fp8 takes
// the power of two).  The FP8 matrix instructions would need no conversion,
// with q as the sum of two E4M3 parts, at the same matrix time; but their sums
// keep only about 16 bits below the largest product (measured: error 1.7e-5
// of the norm of 128 products, any FP8 shape, against 8e-9 in bf16), which is
// an error of 1e-5 and more in a row's log-sum.
//
// Softmax.  A lane of the S^T result holds 4 keys of one row in each 16-key
// tile, so the running maximum and sum of a row live in the lanes of its
// column, and the weights of 32 keys are the B operand of O^T = V^T P^T in
// the registers that S^T left them in (the value tiles are laid out for
// that).  Sums and accumulators are f32.
//
// Weights enter that product in f16, 2^kOff for the largest score: relative
// error 2^-11 each (bf16's 2^-8 would be the largest error of rows that see
// few tokens), absolute 2^-36 of the largest weight.  Values enter as f16 too,
// code * 2^d with d = (block's exponent) - (accumulator's exponent) in -15 .. 7,
// where every E4M3 code is exact.  A block outside of that moves the
// accumulator's exponent to its own, which is exact in f32; but no further than
// kSpread below the highest so far, where the accumulators end.  The exponents
// are those of whole blocks, of tokens too that a row does not see: its own
// values keep their precision beside any of up to 2^kSpread times their size.
#include <algorithm>

#include "kernels.hpp"
#include "kv_cache.hpp"

namespace ullm {
namespace {

constexpr uint32_t kRows = 16;  // rows of a tile
constexpr uint32_t kWaves = 4;
constexpr float kLn2 = 0.693147180559945309f;
constexpr int kOff = 11;             // weights are at most 2^kOff in f16
constexpr int kDown = -15, kUp = 7;  // exponents at which codes are exact in f16
// Sums of 2^20 codes of 448 * 2^kUp with weights of 2^15 stay below 2^51, and
// below 2^111 where their exponent is 60 lower.
constexpr int kSpread = 60;

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

// A row's query as B operands: lane group g holds dims 64c + 16g .. + 15 in
// q[2c] and q[2c + 1], the order of the key tiles.
template <int D>
struct Query {
  bf16x8 q[D / 32];
};

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

template <int D>
__device__ __forceinline__ Query<D> load_query(const uint16_t *row, bool vec, uint32_t sign,
                                               uint32_t g) {
  Query<D> r;
#pragma unroll
  for (int c = 0; c < D / 32; ++c) {
    r.q[c] = load_query8(row + 64 * (c / 2) + 16 * g + 8 * (c % 2), vec, sign);
  }
  return r;
}

// Eight codes as bf16 operands, times a power of two.
__device__ __forceinline__ bf16x8 codes_to_bf16(uint32_t a, uint32_t b, float power) {
  u32x4 r;
  r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, power, false));
  r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, power, true));
  r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, power, false));
  r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, power, true));
  return __builtin_bit_cast(bf16x8, r);
}

// Eight codes as f16 operands, times a power of two in 2^kDown .. 2^kUp.
__device__ __forceinline__ f16x8 codes_to_f16(uint32_t a, uint32_t b, float power) {
  u32x4 r;
  r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, power, false));
  r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, power, true));
  r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, power, false));
  r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, power, true));
  return __builtin_bit_cast(f16x8, r);
}

// Codes that one workgroup alone reads pass the caches by (nontemporal: 47
// against 53 us for 131072 tokens of 8 heads); with several tiles of rows to a
// sequence the later ones find them there.
template <bool NT>
__device__ __forceinline__ u32x4 load_codes(const u32x4 *p) {
  return NT ? __builtin_nontemporal_load(p) : *p;
}

// The codes of 16 keys: tile `tile` (of 16 tokens) of a block and head.
template <int D>
struct Keys {
  u32x4 w[D / 64];
};
template <int D, bool NT>
__device__ __forceinline__ Keys<D> load_keys(const uint8_t *keys, uint32_t tile, uint32_t lane) {
  Keys<D> r;
#pragma unroll
  for (int c = 0; c < D / 64; ++c) {
    r.w[c] = load_codes<NT>(reinterpret_cast<const u32x4 *>(keys + tile * (D * 16)) + c * 64 + lane);
  }
  return r;
}

// Products of 16 keys and the rows: lane l holds row l % 16, keys
// 4 (l / 16) + 0..3.
template <int D>
__device__ __forceinline__ f32x4 products(const Keys<D> &k, float power, const Query<D> &q) {
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < D / 64; ++c) {
    s = mfma_bf16(codes_to_bf16(k.w[c].x, k.w[c].y, power), q.q[2 * c], s);
    s = mfma_bf16(codes_to_bf16(k.w[c].z, k.w[c].w, power), q.q[2 * c + 1], s);
  }
  return s;
}

// High bit of each byte that is an E4M3 NaN (0x7f or 0xff).
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
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

// The 32 tokens of a group: keys and values of one head, 16 bytes per lane
// and load.
template <int D>
struct Group {
  Keys<D> k[2];
  u32x4 v[D / 32];
};
template <int D, bool NT>
__device__ __forceinline__ void load_group_keys(Group<D> &x, const uint8_t *unit,
                                                uint32_t in_block, uint32_t lane) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    x.k[i] = load_keys<D, NT>(unit, in_block / 16 + i, lane);
  }
}
template <int D, bool NT>
__device__ __forceinline__ void load_group_values(Group<D> &x, const uint8_t *unit,
                                                  uint32_t shift, uint32_t in_block,
                                                  uint32_t lane) {
  const u32x4 *p = reinterpret_cast<const u32x4 *>(unit + (uint64_t(D) << shift) +
                                                   in_block / 32 * (D * 32)) + lane;
#pragma unroll
  for (int c = 0; c < D / 32; ++c) {
    x.v[c] = load_codes<NT>(p + c * 64);
  }
}

// The exponent of accumulators, sums over 2^now; `top`: the highest so far.
struct SumExponent {
  int now = kKvExpMin, top = kKvExpMin;

  __device__ bool holds(int block) const { return block <= now + kUp && block >= now + kDown; }
  // Towards that of a block; returns what the accumulators are multiplied by.
  __device__ float move(int block) {
    top = max(top, block);
    const int to = max(block, top - kSpread);
    const float f = exp2_int(max(now - to, -126));
    now = to;
    return f;
  }
  // Power of two of a block's codes as they enter the product.
  __device__ float power(int block) const { return exp2_int(max(block - now, -126)); }
};

// What a row has met so far: the running maximum and the sum of 2^kOff
// exp2(score - m) (this lane's part of it), and its accumulators with their
// exponent.
template <int D>
struct RowState {
  float m, l;
  SumExponent exp;
  f32x4 o[D / 16];
};

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

// A NaN in a token that some rows do not see must not reach them through a
// weight of zero: it is taken out of the group's values, and the rows that do
// see it become NaN.  Bit i of `seen`: the lane's row sees its i-th token.
template <int D>
__device__ __forceinline__ void confine_nan(RowState<D> &st, Group<D> &x, uint32_t seen) {
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < D / 8; ++i) {
    any |= nan_bytes(x.v[i / 4][i % 4]);
  }
  if (!__any(any)) {
    return;
  }
  u32x4 sv;
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    sv[h] = (seen >> (2 * h) & 1u ? 0x3c00u : 0u) | (seen >> (2 * h + 1) & 1u ? 0x3c000000u : 0u);
  }
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    u32x4 nv;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t w = x.v[i / 2][i % 2 * 2 + h], bad = nan_bytes(w);
      x.v[i / 2][i % 2 * 2 + h] = w & ~(bad | (bad - (bad >> 7)));
      nv[2 * h] = (bad & 0x80u ? 0x3c00u : 0u) | (bad & 0x8000u ? 0x3c000000u : 0u);
      nv[2 * h + 1] = (bad & 0x800000u ? 0x3c00u : 0u) | (bad >> 31 ? 0x3c000000u : 0u);
    }
    const f32x4 hit = mfma_f16(__builtin_bit_cast(f16x8, nv), __builtin_bit_cast(f16x8, sv),
                               f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      st.o[i][j] = hit[j] > 0.f ? __builtin_nanf("") : st.o[i][j];
    }
  }
}

// One group for the 16 rows of a wave.  `scores_to`: where the scores of the
// lane's row start (token 0; SCORES).  `more_keys` and `more_values`
// issue the next group's loads as soon as the registers of this one are used.
template <int D, bool SCORES, typename FK, typename FV>
__device__ __forceinline__ void attend_group(RowState<D> &st, Group<D> &x, const Query<D> &q,
                                             const Place &at, uint32_t t0, bool present, float pk,
                                             int ev, float scale_log2, uint32_t g,
                                             float *scores_to, FK more_keys, FV more_values) {
  f32x4 s[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    s[i] = products(x.k[i], pk, q) * scale_log2;
  }
  __builtin_amdgcn_sched_barrier(0);
  more_keys();
  __builtin_amdgcn_sched_barrier(0);
  const bool edge = !present || int32_t(t0) + 31 > at.low || int32_t(t0) <= at.hidden;
  if (edge) {
    uint32_t seen = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int32_t tok = int32_t(t0 + 16 * (i / 4) + 4 * g + i % 4);
      const bool see = present && tok <= at.pos && tok > at.oldest;
      seen |= see ? 1u << i : 0u;
      s[i / 4][i % 4] = see ? s[i / 4][i % 4] : -INFINITY;
    }
    confine_nan(st, x, seen);
  }
  if constexpr (SCORES) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      *reinterpret_cast<f32x4 *>(scores_to + t0 + 16 * i + 4 * g) = s[i];
    }
  }
  // A block out of the pool has no say: its codes are those of another one.
  ev = present ? ev : st.exp.now;
  if (!st.exp.holds(ev)) {
    const float f = st.exp.move(ev);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      st.o[i] *= f;
    }
  }
  const float pv = st.exp.power(ev);
  float top = s[0][0];  // fmaxf passes NaN over: it makes the sum below NaN
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    top = fmaxf(top, s[i / 4][i % 4]);
  }
  top = max_groups(top);
  if (__any(top > st.m)) {  // rare once a row has met its largest scores
    const float now = fmaxf(st.m, top);
    const float keep = now == -INFINITY ? 1.f : exp2_fast(st.m - now);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      st.o[i] *= keep;
    }
    st.l *= keep;
    st.m = now;
  }
  const float ref = st.m == -INFINITY ? 0.f : st.m;
  float p[8], sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    p[i] = exp2_fast(s[i / 4][i % 4] - (ref - float(kOff)));
    sum += p[i];
  }
  st.l += sum;
  u32x4 pw;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    pw[i] = f32x2_to_f16x2(p[2 * i], p[2 * i + 1]);
  }
  const f16x8 pb = __builtin_bit_cast(f16x8, pw);
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    const u32x4 &w = x.v[i / 2];
    st.o[i] = mfma_f16(codes_to_f16(w[i % 2 * 2], w[i % 2 * 2 + 1], pv), pb, st.o[i]);
  }
  __builtin_amdgcn_sched_barrier(0);
  more_values();
  __builtin_amdgcn_sched_barrier(0);
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

// One workgroup owns a part of the tokens of a tile of 16 rows of one
// key/value head.  Its waves take the 32-token groups in turn, each with a
// softmax of its own, and join them at the end.  Block numbers and exponents
// of the part's blocks are fetched by one load of the wave, so that a group
// costs no dependent load; the next group's codes are under way while one is
// computed.  Bound by reading the codes: 131072 tokens of 8 heads 41 us, 6.6
// TB/s, what a plain read of them reaches (16 sequences of up to 8192 tokens
// 33 us, 6.0 TB/s).
template <int D, int W, bool NT, bool SCORES>
__global__ __launch_bounds__(W * kWave, 3) void few_rows_kernel(KvAttendArgs a, Scratch x,
                                                             uint32_t each_slots) {
  __shared__ float part_o[W][kRows][D + 4];
  __shared__ float part_m[W][kRows], part_l[W][kRows];
  const uint32_t kvh = blockIdx.x % a.pool.heads;
  const uint32_t part = blockIdx.x / a.pool.heads % x.parts;
  Tile t;
  if (!tile_rows(a, blockIdx.x / a.pool.heads / x.parts, kRows, each_slots, &t)) {
    return;
  }
  const uint32_t lane = threadIdx.x % kWave;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const uint32_t g = lane / 16, col = lane % 16;
  // Rows past the end see what the last one does; their results are not stored.
  const uint32_t r = t.r0 + (col < t.live ? col : t.live - 1);
  const uint32_t head = kvh * a.group + r % a.group;
  const uint64_t row = t.first_row + r / a.group;
  // Three loads that wait for none: the query, the block numbers of the part
  // (with a window they depend on the length) and the length.  Lane i: block i
  // of the part, which touches at most 64 (kv_part_limit).
  const Query<D> q = load_query<D>(a.q + row * a.q_row + head * a.q_head, a.vec, a.q_sign, g);
  const int32_t *table = a.seqs.tables + t.seq * a.seqs.stride;
  uint32_t block0 = part * x.part_tokens >> a.pool.shift;
  int32_t mine = a.window == 0 ? kv_block(table, a.seqs, a.pool.blocks, block0 + lane) : -1;
  tile_tokens(a, kv_length(a.seqs, a.pool.shift, t.seq), &t);
  const uint32_t parts = part_count(t, x.part_tokens);
  if (part != 0 && part >= parts) {
    return;
  }
  Place at;
  at.pos = int32_t(t.origin + r / a.group);
  at.oldest = oldest_hidden(at.pos, a.window);
  at.low = int32_t(t.low);
  at.hidden = oldest_hidden(t.high, a.window);
  float *scores_to = SCORES ? x.scores + (row * a.heads + head) * x.score_stride : nullptr;

  RowState<D> st;
  st.m = -INFINITY;
  st.l = 0.f;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    st.o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const uint32_t from = t.begin / 32 + part * (x.part_tokens / 32);
  const uint32_t all = (t.end + 31) / 32;
  const uint32_t to = __builtin_amdgcn_readfirstlane(
      all < from + x.part_tokens / 32 ? all : from + x.part_tokens / 32);
  uint32_t grp = __builtin_amdgcn_readfirstlane(from + wave);
  if (grp < to) {
    if (a.window != 0) {
      block0 = from * 32 >> a.pool.shift;
      mine = kv_block(table, a.seqs, a.pool.blocks, block0 + lane);
    }
    block0 = __builtin_amdgcn_readfirstlane(block0);
    const uint64_t my_unit = uint64_t(mine < 0 ? 0 : mine) * a.pool.heads + kvh;
    const int my_exps = *reinterpret_cast<const uint16_t *>(a.pool.exps + my_unit * 2);
    const auto unit_of = [&](uint32_t group) {
      const int id = __builtin_amdgcn_readlane(mine, (group * 32 >> a.pool.shift) - block0);
      return a.pool.codes + (uint64_t(id < 0 ? 0 : id) * a.pool.heads + kvh) *
                                (uint64_t(2 * D) << a.pool.shift);
    };
    const uint32_t in_mask = (1u << a.pool.shift) - 1;
    Group<D> x32;
    // Keys first, as in the loop: a wait for them then leaves the values' loads
    // in flight.
    load_group_keys<D, NT>(x32, unit_of(grp), grp * 32 & in_mask, lane);
    __builtin_amdgcn_sched_barrier(0);
    load_group_values<D, NT>(x32, unit_of(grp), a.pool.shift, grp * 32 & in_mask, lane);
    __builtin_amdgcn_sched_barrier(0);
    while (grp < to) {
      // The last group is loaded again past the end: no load is conditional.
      const uint32_t ahead = grp + W < to ? grp + W : grp;
      const uint32_t i = (grp * 32 >> a.pool.shift) - block0;
      const int exps = __builtin_amdgcn_readlane(my_exps, i);
      attend_group<D, SCORES>(
          st, x32, q, at, grp * 32, __builtin_amdgcn_readlane(mine, i) >= 0, exp2_int(int8_t(exps)),
          int8_t(exps >> 8), a.scale_log2, g, scores_to,
          [&] { load_group_keys<D, NT>(x32, unit_of(ahead), ahead * 32 & in_mask, lane); },
          [&] { load_group_values<D, NT>(x32, unit_of(ahead), a.pool.shift, ahead * 32 & in_mask, lane); });
      grp += W;
    }
  }
  float l = st.l + __shfl_xor(st.l, 16, kWave);
  l += __shfl_xor(l, 32, kWave);
  if (g == 0) {
    part_m[wave][col] = st.m;
    part_l[wave][col] = l;
  }
  // Means of the wave's tokens, to be joined by their sums.
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  const float power = exp2_int(st.exp.now);
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    *reinterpret_cast<f32x4 *>(&part_o[wave][col][16 * i + 4 * g]) = st.o[i] * inv * power;
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

// ------------------------------------------------------------- many rows
//
// 128 rows to a workgroup, 32 to a wave, in the same transposed form with
// 32 x 32 x 16 products: each byte of a block serves 32 rows where the small
// tiles serve 16, and a lane's column holds half of a row's scores.  Steps of
// 64 tokens go through a ring of two stages in LDS, filled by copies that
// no register waits for; every wave converts what it reads.
//
// Bound by instructions and by the clock they leave: a SIMD issues one in four
// cycles, and the conversions, powers and reads beside the 16 products of 32
// rows and 32 tokens (512 cycles of the matrix core) fill 1000; on zeros,
// which switch less, the same launch runs a quarter faster.  (Prompts of 4096
// and 3001 tokens, 32 heads over 8: 221 us, 0.95 PFLOP/s.  Measured against
// this, both slower: codes converted once for the workgroup into operands in
// LDS, 227; 64 rows to a wave, 285.)
//
// Order of the operands (lane l, half h = l / 32, i = l % 32), all read with
// 16 bytes to a lane, which 16 neighbours find in one row of banks:
//   keys: row i of the product is token i with bits 3 and 4 exchanged, so that
//     element e of a result is token {0, 16, 8, 24}[e / 4] + 4h + e % 4 and
//     elements 8c .. 8c + 7 are the 8 tokens of pair 2c + h of a value tile;
//   values: row i is dim 32 (i / 16) + i % 16 of 64 (first 8 bytes) or that
//     plus 16 (last 8 bytes).
constexpr uint32_t kManyRows = 128, kStep = 64, kStages = 2, kManyBlocks = 512;
// A maximum may grow by this much before accumulators are scaled to it: the
// weights then reach 2^(kOff + kSlack) = 2^15 in f16.
constexpr float kSlack = 4.f;

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 mfma32_bf16(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32_f16(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
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

template <int D>
struct ManyState {
  float m, l;
  f32x16 o[D / 32];  // [2 pair + p]
};

// A block of a workgroup's range, as LDS holds it: where its codes start, 2^e
// of its keys, and the exponent of its values plus kExpCode; a block out of
// the pool reads the first one's codes and has the bit kAbsent.
struct BlockEntry {
  uint64_t codes;
  float power;
  uint32_t exp_code;
};
constexpr uint32_t kExpCode = 256, kAbsent = 1u << 31;

__device__ __forceinline__ uint32_t uniform(uint32_t v) {
  return uint32_t(__builtin_amdgcn_readfirstlane(int(v)));
}

// The values' 16 bytes of a lane for 64 dims and the tokens of pair 2c + h.
__device__ __forceinline__ u32x4 value_unit(const uint8_t *values, uint32_t lane, uint32_t c,
                                            uint32_t pair) {
  const uint32_t i = lane % 32, h = lane / 32;
  return *reinterpret_cast<const u32x4 *>(values + (2 * pair + i / 16) * 1024 +
                                          (i % 16 + 16 * (2 * c + h)) * 16);
}

// O^T += V^T P^T for 32 tokens.  The barriers keep later conversions out of the
// registers that a third wave needs.
template <int D>
__device__ __forceinline__ void add_values(ManyState<D> &st, const u32x4 (&v)[D / 32],
                                           const u32x4 (&p)[2], float power) {
#pragma unroll
  for (uint32_t c = 0; c < 2; ++c) {
#pragma unroll
    for (uint32_t pair = 0; pair < D / 64; ++pair) {
      const u32x4 w = v[c * (D / 64) + pair];
      f32x16 *acc = st.o + 2 * pair;
      const f16x8 b = __builtin_bit_cast(f16x8, p[c]);
      acc[0] = mfma32_f16(codes_to_f16(w.x, w.y, power), b, acc[0]);
      acc[1] = mfma32_f16(codes_to_f16(w.z, w.w, power), b, acc[1]);
      __builtin_amdgcn_sched_barrier(0);
    }
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

// LONG: a part may have more blocks than LDS holds entries of, which are then
// replaced on the way.  (Where it has not, that costs 229 against 221 us.)
template <int D, bool LONG>
__global__ __launch_bounds__(kWaves * kWave, 3) void many_rows_kernel(KvAttendArgs a, Scratch x,
                                                                      uint32_t each_slots) {
  constexpr uint32_t kGroup = 64 * D;  // bytes of 32 tokens: keys, then values
  // Dynamic, so that its reads are not taken to depend on every copy under way
  // (as those of a static array are).
  extern __shared__ __align__(1024) uint8_t many_ring[];
  const auto ring = [](uint32_t stage) { return many_ring + stage * 2 * kGroup; };
  __shared__ BlockEntry entries[kManyBlocks];
  const uint32_t kvh = blockIdx.x % a.pool.heads;
  const uint32_t rest = blockIdx.x / a.pool.heads, slots = gridDim.x / a.pool.heads / x.parts;
  const uint32_t part = rest % x.parts;
  Tile t;
  if (!tile_rows_last_first(a, rest / x.parts, slots, kManyRows, each_slots, &t)) {
    return;
  }
  tile_tokens(a, kv_length(a.seqs, a.pool.shift, t.seq), &t);
  const uint32_t parts = part_count(t, x.part_tokens);
  if (part != 0 && part >= parts) {
    return;
  }
  const uint32_t lane = threadIdx.x % kWave;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const uint32_t h = lane / 32, i = lane % 32;
  // The wave's rows; rows past the end see what the last one does.
  const uint32_t last = t.live - 1;
  const uint32_t w0 = min(32 * wave, last), w1 = min(32 * wave + 31, last);
  const uint32_t r = t.r0 + min(32 * wave + i, last);
  const uint32_t head = kvh * a.group + r % a.group;
  const uint64_t row = t.first_row + r / a.group;
  const int32_t pos = int32_t(t.origin + r / a.group), oldest = oldest_hidden(pos, a.window);
  const int32_t low = int32_t(t.origin + (t.r0 + w0) / a.group);
  const int32_t high = int32_t(t.origin + (t.r0 + w1) / a.group);
  bf16x8 q[D / 16];
#pragma unroll
  for (int c = 0; c < D / 16; ++c) {
    q[c] = load_query8(a.q + row * a.q_row + head * a.q_head + 16 * (2 * (c / 2) + h) + 8 * (c % 2),
                       a.vec, a.q_sign);
  }
  const uint32_t from = t.begin / 32 + part * (x.part_tokens / 32);
  const uint32_t all = (t.end + 31) / 32;
  const uint32_t to = min(all, from + x.part_tokens / 32);
  const int32_t *table = a.seqs.tables + t.seq * a.seqs.stride;
  const auto entry_of = [&](uint32_t block) {
    const int32_t id = kv_block(table, a.seqs, a.pool.blocks, block);
    const uint64_t unit = uint64_t(id < 0 ? 0 : id) * a.pool.heads + kvh;
    const int e = *reinterpret_cast<const uint16_t *>(a.pool.exps + unit * 2);
    return BlockEntry{
        reinterpret_cast<uint64_t>(a.pool.codes) + unit * (uint64_t(2 * D) << a.pool.shift),
        exp2_int(int8_t(e)), uint32_t(int8_t(e >> 8) + int(kExpCode)) | (id < 0 ? kAbsent : 0u)};
  };
  // LDS holds the blocks `held` .. held + kManyBlocks - 1 of the sequence, as
  // far as the part goes.
  uint32_t held = from * 32 >> a.pool.shift;
  const auto hold_blocks = [&] {
    const uint32_t end = to > from ? ((to * 32 - 1) >> a.pool.shift) + 1 : held;
    for (uint32_t b = threadIdx.x; b < kManyBlocks && held + b < end; b += kWaves * kWave) {
      entries[b] = entry_of(held + b);
    }
  };
  hold_blocks();
  ManyState<D> st;
  st.m = -INFINITY;
  st.l = 0.f;
#pragma unroll
  for (int c = 0; c < D / 32; ++c) {
    st.o[c] = f32x16{};
  }
  __syncthreads();

  // What a step needs of its two groups (one past the end is the last one
  // again), looked up a step ahead.
  struct Step {
    float power[2];
    uint32_t exp_code[2];
  };
  const uint32_t in_mask = (1u << a.pool.shift) - 1;
  const uint32_t copy_at = (D == 128 ? wave : wave % 2) * 1024 + lane * 16;
  const auto start_step = [&](uint32_t grp0, uint8_t *stage) {
    Step s;
#pragma unroll
    for (uint32_t u = 0; u < 2; ++u) {
      const uint32_t tok = min(grp0 + u, to - 1) * 32;
      const u32x4 e =
          *reinterpret_cast<const u32x4 *>(&entries[(tok >> a.pool.shift) - held]);
      s.power[u] = bits_f32(uniform(e.z));
      s.exp_code[u] = uniform(e.w);
      const uint8_t *keys =
          reinterpret_cast<const uint8_t *>(uint64_t(uniform(e.y)) << 32 | uniform(e.x)) +
          (tok & in_mask) * D;
      const uint8_t *values = keys + (uint64_t(D) << a.pool.shift);
      uint8_t *to_lds = stage + u * kGroup + wave * 1024;
      if (D == 128) {
        copy_to_lds(keys + copy_at, to_lds);
        copy_to_lds(values + copy_at, to_lds + 32 * D);
      } else {
        copy_to_lds((wave < 2 ? keys : values) + copy_at, to_lds);
      }
    }
    return s;
  };
  // Groups that some of the wave's rows see, and of those the ones that every
  // row sees whole: [first, first + count) each.
  struct Range {
    uint32_t first, count;
  };
  const auto range = [](int64_t first, int64_t end) {
    return Range{uniform(uint32_t(first)), uniform(uint32_t(end > first ? end - first : 0))};
  };
  const Range some = range((int64_t(oldest_hidden(low, a.window)) + 1) / 32,
                           high < 0 ? 0 : min(int64_t(high / 32 + 1), int64_t(to)));
  const Range whole = range((int64_t(oldest_hidden(high, a.window)) + 1 + 31) / 32,
                            low < 0 ? 0 : (int64_t(low) + 1) / 32);
  const uint32_t steps = to > from ? (to - from + 1) / 2 : 0;
  Step next{};
  if (steps != 0) {
    next = start_step(from, ring(0));
  }
  // Lane's place in a key tile pair: token i with bits 3 and 4 exchanged.
  const uint32_t tok = (i & 7) | (i & 8) << 1 | (i & 16) >> 1;
  const uint32_t key_at = tok / 16 * (D / 64) * 1024 + tok % 16 * 16 + h * 256;
  // The instructions of a group are what bounds this loop (a SIMD issues one
  // in four cycles, whatever its kind): what changes rarely is kept ready and
  // changed under a branch.  bias: kOff - m, what a scaled score becomes a
  // power of two with; limit: the unscaled score past which m grows; power:
  // that of the last exponent code.
  SumExponent exp;
  uint32_t code = ~0u;
  float bias = float(kOff), limit = -INFINITY, power = 1.f;
  bool dirty = false;  // a NaN value in a group that some rows do not see
  for (uint32_t step = 0; step < steps; ++step) {
    wait_copies<0>();
    step_barrier();
    const Step now = next;
    const uint8_t *stage = ring(step % kStages);
    if (step + 1 < steps) {
      const uint32_t grp0 = from + 2 * step + 2;
      if (LONG && (min(grp0 + 1, to - 1) * 32 >> a.pool.shift) - held >= kManyBlocks) {
        // No wave is past this step's barrier without the entries it read.
        held = grp0 * 32 >> a.pool.shift;
        hold_blocks();
        __syncthreads();
      }
      next = start_step(grp0, ring((step + 1) % kStages));
    }
#pragma unroll
    for (uint32_t u = 0; u < 2; ++u) {
      const uint32_t grp = from + 2 * step + u;
      if (grp - some.first >= some.count) {
        continue;
      }
      const uint8_t *keys = stage + u * kGroup + key_at, *values = stage + u * kGroup + 32 * D;
      // All of a product's LDS reads are under way before its first use, those
      // of the values during the softmax.
      u32x4 units[D / 32];
#pragma unroll
      for (uint32_t c = 0; c < D / 32; ++c) {
        units[c] = *reinterpret_cast<const u32x4 *>(keys + c / 2 * 1024 + c % 2 * 512);
      }
      __builtin_amdgcn_sched_barrier(0);
      f32x16 s = f32x16{};
#pragma unroll
      for (uint32_t c = 0; c < D / 32; ++c) {
        const u32x4 w = units[c];
        s = mfma32_bf16(codes_to_bf16(w.x, w.y, now.power[u]), q[2 * c], s);
        s = mfma32_bf16(codes_to_bf16(w.z, w.w, now.power[u]), q[2 * c + 1], s);
      }
#pragma unroll
      for (uint32_t c = 0; c < D / 32; ++c) {
        units[c] = value_unit(values, lane, c / (D / 64), c % (D / 64));
      }
      if (now.exp_code[u] != code) {
        code = now.exp_code[u];
        // A block out of the pool has no say: its codes are those of another one.
        const int ev = (code & kAbsent) != 0 ? exp.now : int(code & 0xffffu) - int(kExpCode);
        if (!exp.holds(ev)) {
          const float f = exp.move(ev);
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            st.o[c] *= f;
          }
        }
        power = exp.power(ev);
      }
      if (((grp - whole.first) | (code & kAbsent)) >= whole.count) {
        const int32_t t0 = int32_t(grp * 32);
        const bool present = (code & kAbsent) == 0;
        uint32_t any = 0;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int32_t at = t0 + int32_t((e / 4 % 2) * 16 + e / 8 * 8 + 4 * h + e % 4);
          const bool see = present && at <= pos && at > oldest;
          s[e] = see ? s[e] : -INFINITY;
        }
#pragma unroll
        for (uint32_t c = 0; c < D / 32; ++c) {
          const u32x4 w = units[c];
          any |= nan_bytes(w.x) | nan_bytes(w.y) | nan_bytes(w.z) | nan_bytes(w.w);
        }
        dirty = dirty || __any(any);
      }
      float top = s[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) {
        top = fmaxf(top, s[e]);
      }
      if (__any(top > limit)) {
        const auto both =
            __builtin_amdgcn_permlane32_swap(f32_bits(top), f32_bits(top), false, false);
        top = fmaxf(bits_f32(both[0]), bits_f32(both[1])) * a.scale_log2;
        const float m = fmaxf(st.m, top);
        const float keep = m == -INFINITY ? 1.f : exp2_fast(st.m - m);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          st.o[c] *= keep;
        }
        st.l *= keep;
        st.m = m;
        limit = (m + kSlack) / a.scale_log2;
        bias = float(kOff) - (m == -INFINITY ? 0.f : m);
      }
      float sum = 0.f;
      u32x4 p[2];
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const float p0 = exp2_fast(__builtin_fmaf(s[e], a.scale_log2, bias));
        const float p1 = exp2_fast(__builtin_fmaf(s[e + 1], a.scale_log2, bias));
        sum += p0;
        sum += p1;
        p[e / 8][e % 8 / 2] = f32x2_to_f16x2(p0, p1);
      }
      st.l += sum;
      add_values<D>(st, units, p, power);
    }
  }
  wait_copies<0>();  // none may land after the workgroup has gone

  const auto sink = [&](uint32_t r_of_tile) {
    const uint32_t rr = t.r0 + min(r_of_tile, last);
    RowSink to;
    to.row = t.first_row + rr / a.group;
    to.head = kvh * a.group + rr % a.group;
    to.live = r_of_tile <= last;
    to.whole = parts <= 1;
    to.slot = (to.row * a.heads + to.head) * x.parts + part;
    return to;
  };
  if (!dirty) {
    const auto half =
        __builtin_amdgcn_permlane32_swap(f32_bits(st.l), f32_bits(st.l), false, false);
    const float sum = bits_f32(half[0]) + bits_f32(half[1]);
    const float join = sum == 0.f ? 0.f : 1.0f / sum, unit = exp2_int(exp.now);
    const RowSink out = sink(32 * wave + i);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f32x4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[j] = st.o[c][4 * e + j] * join * unit;
        }
        store4(a, x, out, D, 64 * (c / 2) + 32 * (e / 2) + 16 * (c % 2) + 8 * (e % 2) + 4 * h, v);
      }
    }
    if (h == 0) {
      store_sums(a, x, out, st.m, sum);
    }
    return;
  }
  // The NaN must reach the rows that see it and no others: the wave's rows go
  // through the small tiles' code, which sees to that, 16 at a time.  (In the
  // loop above it would cost the registers of a third wave.)
  for (uint32_t part16 = 0; part16 < 2; ++part16) {
    const uint32_t first = 32 * wave + 16 * part16, g = lane / 16;
    if (first > last) {
      return;
    }
    const RowSink out = sink(first + lane % 16);
    Place at;
    at.pos = int32_t(t.origin + (t.r0 + min(first + lane % 16, last)) / a.group);
    at.oldest = oldest_hidden(at.pos, a.window);
    at.low = int32_t(t.origin + (t.r0 + first) / a.group);
    at.hidden =
        oldest_hidden(t.origin + (t.r0 + min(first + 15, last)) / a.group, a.window);
    const Query<D> q16 =
        load_query<D>(a.q + out.row * a.q_row + out.head * a.q_head, a.vec, a.q_sign, g);
    RowState<D> rs;
    rs.m = -INFINITY;
    rs.l = 0.f;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      rs.o[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (uint32_t grp = from; grp < to; ++grp) {
      const uint32_t in_block = grp * 32 & in_mask;
      const BlockEntry e = entry_of(grp * 32 >> a.pool.shift);
      const uint8_t *unit = reinterpret_cast<const uint8_t *>(e.codes);
      const uint32_t exp_code = uniform(e.exp_code);
      Group<D> x32;
      load_group_keys<D, false>(x32, unit, in_block, lane);
      load_group_values<D, false>(x32, unit, a.pool.shift, in_block, lane);
      attend_group<D, false>(
          rs, x32, q16, at, grp * 32, (exp_code & kAbsent) == 0, bits_f32(uniform(f32_bits(e.power))),
          int(exp_code & 0xffffu) - int(kExpCode), a.scale_log2, g, nullptr, [] {}, [] {});
    }
    float l = rs.l + __shfl_xor(rs.l, 16, kWave);
    l += __shfl_xor(l, 32, kWave);
    const float join = l == 0.f ? 0.f : 1.0f / l, power = exp2_int(rs.exp.now);
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      store4(a, x, out, D, 16 * c + 4 * g, rs.o[c] * join * power);
    }
    if (g == 0) {
      store_sums(a, x, out, rs.m, l);
    }
  }
}

// Joins the parts of a row: one workgroup of J waves, which take the parts in
// turn, kJoinAhead of them under way at once (the sums of a part are small:
// the time goes into waiting for them).
constexpr uint32_t kJoinAhead = 4;
template <int D, uint32_t J>
__global__ __launch_bounds__(J * kWave) void join_parts_kernel(KvAttendArgs a, Scratch x,
                                                               uint32_t tile,
                                                               uint32_t rows_of_tile,
                                                               uint32_t each_slots) {
  __shared__ float part_o[J][D];
  __shared__ float part_m[J], part_l[J];
  constexpr int kPer = D / kWave;
  Tile t;
  const uint32_t index = blockIdx.x / rows_of_tile;
  if (!tile_rows(a, index / a.pool.heads, tile, each_slots, &t) ||
      blockIdx.x % rows_of_tile >= t.live) {
    return;
  }
  tile_tokens(a, kv_length(a.seqs, a.pool.shift, t.seq), &t);
  const uint32_t parts = part_count(t, x.part_tokens), r = t.r0 + blockIdx.x % rows_of_tile;
  if (parts <= 1) {
    return;
  }
  const uint64_t row = t.first_row + r / a.group;
  const uint32_t head = index % a.pool.heads * a.group + r % a.group;
  const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint64_t slot = (row * a.heads + head) * x.parts;
  float m = -INFINITY, l = 0.f, v[kPer] = {};
  for (uint32_t p0 = wave; p0 < parts; p0 += J * kJoinAhead) {
    PartSum s[kJoinAhead];
    float o[kJoinAhead][kPer];
#pragma unroll
    for (uint32_t j = 0; j < kJoinAhead; ++j) {
      const uint32_t p = p0 + j * J;
      const uint64_t at = slot + (p < parts ? p : p0);
      s[j] = x.part_s[at];
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        o[j][i] = x.part_o[at * D + lane * kPer + i];
      }
      s[j].l = p < parts ? s[j].l : 0.f;
    }
    float now = m;
#pragma unroll
    for (uint32_t j = 0; j < kJoinAhead; ++j) {
      now = fmaxf(now, s[j].m);
    }
    const float ref = now == -INFINITY ? 0.f : now, keep = exp2_fast(m - ref);
    m = now;
    l *= keep;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      v[i] *= keep;
    }
#pragma unroll
    for (uint32_t j = 0; j < kJoinAhead; ++j) {
      const float f = exp2_fast(s[j].m - ref) * s[j].l;
      const bool none = p0 + j * J >= parts;
      l += f;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        v[i] += none ? 0.f : o[j][i] * f;
      }
    }
  }
  if (lane == 0) {
    part_m[wave] = m;
    part_l[wave] = l;
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    part_o[wave][lane * kPer + i] = v[i];
  }
  __syncthreads();
  if (threadIdx.x * 2 >= D) {
    return;
  }
  float top = part_m[0], sum = 0.f, out[2] = {0.f, 0.f};
#pragma unroll
  for (uint32_t w = 1; w < J; ++w) {
    top = fmaxf(top, part_m[w]);
  }
  const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
  for (uint32_t w = 0; w < J; ++w) {
    const float f = exp2_fast(part_m[w] - ref);
    sum += part_l[w] * f;
    out[0] += part_o[w][threadIdx.x * 2] * f;
    out[1] += part_o[w][threadIdx.x * 2 + 1] * f;
  }
  store_row(a, x, row, head, threadIdx.x * 2, out, top, sum);
}

// Adds each token's weights from the scores that few_rows_kernel stored: a
// thread owns a token and sums its rows in order.  Bound by reading the scores
// (8 sequences of 16384 tokens, 32 heads: 6.7 us for 17 MB and 1 M additions).
__global__ __launch_bounds__(256) void add_scores_kernel(KvAttendArgs a, Scratch x) {
  const uint32_t kvh = blockIdx.y, b = blockIdx.z;
  const uint32_t t = blockIdx.x * 256 + threadIdx.x;
  const uint32_t length = kv_length(a.seqs, a.pool.shift, b);
  if (t >= length) {
    return;
  }
  const int32_t id = kv_block(a.seqs.tables + b * a.seqs.stride, a.seqs, a.pool.blocks,
                              t >> a.pool.shift);
  if (id < 0) {
    return;
  }
  const KvRows rows = kv_rows(a.seqs, b);
  const int64_t origin = int64_t(length) - rows.count;
  const int64_t from = int64_t(t) - origin;  // the first query that sees the token
  uint32_t i = from > 0 ? uint32_t(from) : 0u;
  const int64_t past = a.window != 0 ? from + int64_t(a.window) : int64_t(rows.count);
  const uint32_t end = past < int64_t(rows.count) ? uint32_t(past < 0 ? 0 : past) : rows.count;
  float sum = 0.f;
  for (; i < end; ++i) {
    const uint64_t at = uint64_t(rows.first + i) * a.heads + kvh * a.group;
    const RowStats *stats = x.stats + stats_at(a, kvh, rows.first + i);
    for (uint32_t h0 = 0; h0 < a.group; h0 += 4) {  // four on their way at once
      float s[4];
      RowStats st[4];
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) {
        const uint32_t h = min(h0 + j, a.group - 1);
        s[j] = x.scores[(at + h) * x.score_stride + t];
        st[j] = stats[h];
      }
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) {
        const float p = exp2_fast(s[j] - st[j].top) * st[j].inv_sum;
        sum += h0 + j < a.group ? p : 0.f;
      }
    }
  }
  const uint64_t unit = uint64_t(id) * a.pool.heads + kvh;
  unsafeAtomicAdd(&a.pool.weights[(unit << a.pool.shift) + (t & ((1u << a.pool.shift) - 1))], sum);
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
// LDS holds a tile as D / 32 planes of 64 bytes of each row; 16-byte chunk k of
// row r is at place k ^ r / 4 % 4 of the 64, so that 16 neighbours read 16
// groups of banks and a wave copies 16 rows at once, a lane always the same.
constexpr uint32_t kWeightTokens = 32 * kWaves, kWeightRows = 64;

template <int D>
__global__ __launch_bounds__(kWaves * kWave, 4) void add_weights_kernel(KvAttendArgs a,
                                                                        const RowStats *stats) {
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
  const uint8_t *keys =
      a.pool.codes + unit * (uint64_t(2 * D) << a.pool.shift) + uint64_t(in_block) * D;
  const float power = exp2_int(a.pool.exps[unit * 2]);
  bf16x8 k[D / 16];
#pragma unroll
  for (int c = 0; c < D / 32; ++c) {
    const u32x4 w = *reinterpret_cast<const u32x4 *>(
        keys + (i / 16 * (D / 64) + c / 2) * 1024 + (i % 16 + 16 * (c % 2 * 2 + h)) * 16);
    k[2 * c] = flip(codes_to_bf16(w.x, w.y, power), a.q_sign);
    k[2 * c + 1] = flip(codes_to_bf16(w.z, w.w, power), a.q_sign);
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
        const uint32_t place = (2 * h + c % 2) ^ i / 4 % 4;
        q[c] = *reinterpret_cast<const bf16x8 *>(tile + c / 2 * kPlane + 32 * u * 64 + place * 16);
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

}  // namespace

// Scratch of a plan in its order: partial results, row statistics, scores.
static Scratch scratch_of(const KvAttendArgs &a, uint32_t dim, const KvAttendPlan &p, void *ws,
                          uint64_t *bytes) {
  Scratch x{};
  x.parts = p.parts;
  x.part_tokens = p.part_tokens;
  const uint64_t rows = uint64_t(a.seqs.rows) * a.heads;
  uint64_t at = 0;
  const auto take = [&](uint64_t n) {
    char *r = ws == nullptr ? nullptr : static_cast<char *>(ws) + at;
    at += (n + 255) / 256 * 256;
    return r;
  };
  if (p.parts > 1) {
    x.part_o = reinterpret_cast<float *>(take(rows * p.parts * dim * sizeof(float)));
    x.part_s = reinterpret_cast<PartSum *>(take(rows * p.parts * sizeof(PartSum)));
  }
  if (a.accumulate) {
    x.stats = reinterpret_cast<RowStats *>(take(rows * sizeof(RowStats)));
    if (p.keep_scores) {
      x.score_stride = uint64_t(a.seqs.max_blocks) << a.pool.shift;
      x.scores = reinterpret_cast<float *>(take(rows * x.score_stride * sizeof(float)));
    }
  }
  *bytes = at;
  return x;
}

static uint64_t each_tiles(const KvAttendArgs &a, uint32_t rows) {
  return (uint64_t(a.seqs.each) * a.group + rows - 1) / rows;
}

// Tokens are split where the tiles alone leave compute units idle, into parts
// that together give each a workgroup: more and smaller parts cost their start
// and the join (131072 tokens of 8 heads: 32 parts each 46.7 us, 64 50.1, 128
// 53.2).  With many rows two of them, three at 64 dims, run at once (twice 128
// queries at 8000 tokens 56 us, three 76; 64 dims, 28 heads over 4, 500 queries
// at 8000: 70, three 68).  Many rows that fill the units by themselves are
// split in two if they are long (8 times 128 queries at 16000 tokens: 327 us,
// whole 343; 4 times 300: 406, whole 488), and not if they are short (16 times
// 64 at 2000: 51, in three 64; 1024 at 1024: 30, in two 45).  A part has at least kPartLeast
// tokens (333 tokens of 8 heads: whole 5.7 us, in two parts 7.8), with few rows
// those of at most 64 blocks, what a wave looks up with one load.
constexpr uint32_t kPartLeast = 512, kPartLong = 8192;
// Small tiles serve up to kFewMost rows of a sequence and key/value head, on
// average, and more where all their tiles run at about once and the tokens are
// not many (us, 32 heads over 8, small tiles against large ones): 512 queries
// at 512 tokens 13 / 18, 4 times 128 at 2000 37 / 41, 8 times 64 at 1000 23 /
// 28; past that 8 times 128 at 1000 39 / 30, 32 at 30000 42 / 37.  64 times 16
// at 4000 tokens: 157 / 164, 64 times 24 206 / 167.
constexpr uint32_t kFewMost = 64, kFewTilesOfUnit = 4, kFewTokens = 4096;
// Stored scores cost 8 bytes for each row and token, a second pass over the keys
// `dim` bytes for each token.  Scores have a place for each token of the tables,
// in use or not: past kMostScores bytes, under a hundredth of the memory, the
// second pass is taken (64 sequences of 2000 tokens, 32 heads, tables of 131072
// tokens: 1.1 GB of scores and 190 us, second pass 303; tables of 2048 tokens:
// 61 and 111).
constexpr uint64_t kMostScores = uint64_t(1) << 31;

KvAttendPlan plan_kv_attend(const KvAttendArgs &a, uint32_t dim) {
  KvAttendPlan p;
  if (a.seqs.rows == 0 || a.seqs.batch == 0) {
    return p;
  }
  const uint32_t cus = device_cu_count();
  const uint64_t rows_of_head = uint64_t(a.seqs.rows) * a.group;
  const auto tiles_of = [&](uint32_t rows) {
    return kv_slots(a.seqs, a.group, rows, 1, each_tiles(a, rows)) * a.pool.heads;
  };
  // The most tokens that a tile's rows see, from the start of a 32-token group.
  const auto span_of = [&](uint32_t rows) {
    const uint64_t all = uint64_t(a.seqs.max_blocks) << a.pool.shift;
    return a.window == 0 ? all
                         : std::min<uint64_t>(all, uint64_t(a.window) + rows / a.group + 32);
  };
  const bool many = rows_of_head > uint64_t(kFewMost) * a.seqs.batch &&
                    (tiles_of(kRows) > uint64_t(kFewTilesOfUnit) * cus ||
                     span_of(kRows) > kFewTokens);
  p.kernel = many ? ULLM_KV_KERNEL_MANY_ROWS : ULLM_KV_KERNEL_FEW_ROWS;
  p.row_tile = many ? kManyRows : kRows;
  const uint64_t tiles = tiles_of(p.row_tile), span = span_of(p.row_tile);
  const uint64_t split = tiles < cus ? (!many ? 1 : dim == 64 ? 3 : 2) * cus / tiles
                         : many && span > kPartLong && tiles < 2 * cus ? 2
                                                                       : 1;
  const uint64_t part = std::max<uint64_t>((span + split - 1) / split, kPartLeast);
  const uint64_t most =
      many ? uint64_t(1) << 31 : kv_part_limit(kWave, a.pool.shift, a.window) / kStep * kStep;
  p.part_tokens = uint32_t(std::min<uint64_t>((part + kStep - 1) / kStep * kStep, most));
  p.parts = uint32_t((span + p.part_tokens - 1) / p.part_tokens);
  const uint64_t scores = uint64_t(a.seqs.rows) * a.heads * sizeof(float) *
                          (uint64_t(a.seqs.max_blocks) << a.pool.shift);
  p.keep_scores = a.accumulate && !many && rows_of_head <= uint64_t(dim) / 8 * a.seqs.batch &&
                  scores <= kMostScores;
  p.one_tile = rows_of_head <= uint64_t(kRows) * a.seqs.batch;
  p.grid = tiles * p.parts;
  // Eight waves shorten the walk of a lone workgroup (333 tokens: 5.7 against
  // 6.2 us) and keep enough bytes on their way where a workgroup has a unit to
  // itself and 64 dims (131072 tokens of 8 heads: 27.4 against 32.2 us); four
  // have less to join and do better beyond that (128 dims, 32 sequences of 2000
  // tokens: 24.4 against 26.4; 64 dims, 64 of them: 24.5 against 27.1).
  p.waves = p.grid <= uint64_t(cus) * 64 / dim ? 8 : 4;
  scratch_of(a, dim, p, nullptr, &p.workspace);
  return p;
}

template <int D>
static hipError_t launch_attend(const KvAttendArgs &a, const KvAttendPlan &p, void *workspace,
                                hipStream_t s) {
  uint64_t bytes = 0;
  const Scratch x = scratch_of(a, D, p, workspace, &bytes);
  const uint32_t each = uint32_t(each_tiles(a, p.row_tile));
  const auto few = [&](auto kernel8, auto kernel4) {
    if (p.waves == 8) {
      kernel8<<<uint32_t(p.grid), 8 * kWave, 0, s>>>(a, x, each);
    } else {
      kernel4<<<uint32_t(p.grid), 4 * kWave, 0, s>>>(a, x, each);
    }
  };
  if (p.kernel == ULLM_KV_KERNEL_MANY_ROWS) {
    constexpr uint32_t lds = kStages * 2 * 64 * D;
    const auto many = [&](auto kernel) {
      const hipError_t e = raise_lds_limit(reinterpret_cast<const void *>(kernel), lds);
      if (e == hipSuccess) {
        kernel<<<uint32_t(p.grid), kWaves * kWave, lds, s>>>(a, x, each);
      }
      return e;
    };
    const bool longer = p.part_tokens > kv_part_limit(kManyBlocks, a.pool.shift, a.window);
    const hipError_t e = longer ? many(many_rows_kernel<D, true>) : many(many_rows_kernel<D, false>);
    if (e != hipSuccess) {
      return e;
    }
  } else if (x.scores != nullptr) {
    few(few_rows_kernel<D, 8, true, true>, few_rows_kernel<D, 4, true, true>);
  } else if (p.one_tile) {
    few(few_rows_kernel<D, 8, true, false>, few_rows_kernel<D, 4, true, false>);
  } else {
    few(few_rows_kernel<D, 8, false, false>, few_rows_kernel<D, 4, false, false>);
  }
  if (p.parts > 1) {
    const uint32_t rows =
        a.seqs.starts == nullptr ? std::min(a.seqs.each * a.group, p.row_tile) : p.row_tile;
    const uint32_t grid = uint32_t(p.grid / p.parts) * rows;
    if (p.parts > 2 * kJoinAhead) {
      join_parts_kernel<D, 8><<<grid, 8 * kWave, 0, s>>>(a, x, p.row_tile, rows, each);
    } else {
      join_parts_kernel<D, 1><<<grid, kWave, 0, s>>>(a, x, p.row_tile, rows, each);
    }
  }
  if (a.accumulate) {
    const uint64_t tokens = uint64_t(a.seqs.max_blocks) << a.pool.shift;
    if (x.scores != nullptr) {
      add_scores_kernel<<<dim3(uint32_t((tokens + 255) / 256), a.pool.heads, a.seqs.batch), 256, 0,
                          s>>>(a, x);
    } else {
      const dim3 grid(uint32_t((tokens + kWeightTokens - 1) / kWeightTokens), a.pool.heads,
                      a.seqs.batch);
      add_weights_kernel<D>
          <<<grid, kWaves * kWave, 2 * kWeightRows * D * 2, s>>>(a, x.stats);
    }
  }
  return hipGetLastError();
}

hipError_t launch_kv_attend(const KvAttendArgs &a, uint32_t dim, const KvAttendPlan &p,
                            void *workspace, hipStream_t s) {
  return dim == 64 ? launch_attend<64>(a, p, workspace, s)
                   : launch_attend<128>(a, p, workspace, s);
}

}  // namespace ullm
