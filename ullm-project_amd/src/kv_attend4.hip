// kv_attend4.hip -- softmax attention over the 4-bit key/value cache.
//
// Rows, tiles, parts and their joins are those of the 8-bit cache
// (kv_attend.hip); the products are the same too: S^T = K Q^T in bf16, O^T = V^T
// P^T in f16, with keys and values converted in registers, exactly.
//
// Keys.  A lane's codes of a token belong to one exponent, which the conversion
// to bf16 takes.
//
// Values.  A token's scale s enters its weight: the operand is p' = p * s in f16
// beside the bare codes, while the row's sum takes p in f32.  Powers are taken
// over a reference M that follows the largest of score + log2(s) (not of the
// score alone), so that the largest p' is near 2^kOff: what a token adds to the
// result decides how exactly it enters, whatever the scales of the others.  M is
// left alone while the largest sum (few rows: (largest score) + log2(largest s) of a
// lane's tokens, which no sum passes) stays within kSlack of it; else it moves to the
// largest, rounded down to a whole number: what is added to a score before its power
// is then exact, and so is what earlier sums are multiplied by.  With scales from
// 2^-19 to 2^16 the p of a row's sum stay within 2^-28 and 2^34 of what they would be
// over the largest score, far inside f32.
//
// NaN.  Codes are finite, NaN is in a key's exponent or a value's scale.  A key's
// reaches a row through its score, and -infinity takes the place of the scores that
// a row does not see.  A value's makes the row's result NaN, but neither its log-sum
// nor the weights that its tokens receive, which are of scores alone: with few rows
// it enters the operand p' (scale 0 takes the place of hidden ones), with many the
// quotient at the end.
#include <algorithm>

#include "kv_attend.hpp"
#include "kv_cache4.hpp"

namespace ullm {
namespace {

// A reference may lag by this much: weights then reach 2^(kOff + kSlack) = 2^15
// in f16.
constexpr float kSlack = 4.f;

// A row's query as B operands: lane group g holds dims D / 4 * g + 8c .. + 7 in
// q[c], the order of the keys' codes.
template <int D>
struct Query4 {
  bf16x8 q[D / 32];
};
template <int D>
__device__ __forceinline__ Query4<D> load_query4(const uint16_t *row, bool vec, uint32_t sign,
                                                 uint32_t g) {
  Query4<D> r;
#pragma unroll
  for (int c = 0; c < D / 32; ++c) {
    r.q[c] = load_query8(row + D / 4 * g + 8 * c, vec, sign);
  }
  return r;
}

// What a lane needs of a chunk: codes of keys (16 bytes each: of tokens t, t +
// 16, or both) and their two exponents, of values, and eight scales in f16.
template <int D>
struct Group4 {
  u32x4 k[D / 64], v[D / 64], scales;
  uint32_t exps;
};
template <int D, bool NT>
__device__ __forceinline__ void load_keys4(Group4<D> &x, const uint8_t *chunk, uint32_t lane) {
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    x.k[i] = load_codes<NT>(reinterpret_cast<const u32x4 *>(chunk) + i * 64 + lane);
  }
  const uint32_t at = D == 128 ? lane : lane % 16 + 16 * (lane / 32);
  x.exps = reinterpret_cast<const uint16_t *>(chunk + Kv4Chunk<D>::kExps)[at];
}
template <int D, bool NT>
__device__ __forceinline__ void load_values4(Group4<D> &x, const uint8_t *chunk, uint32_t lane) {
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    x.v[i] = load_codes<NT>(
        reinterpret_cast<const u32x4 *>(chunk + Kv4Chunk<D>::kSide) + i * 64 + lane);
  }
  x.scales = reinterpret_cast<const u32x4 *>(chunk + Kv4Chunk<D>::kScales)[lane / 16];
}

// Products of the chunk's tokens 16 i .. + 15 and the rows: lane l holds row
// l % 16, tokens 16 i + 4 (l / 16) + 0..3.
template <int D>
__device__ __forceinline__ f32x4 products4(const Group4<D> &x, int i, const Query4<D> &q) {
  const float power = bits_f32((i == 0 ? x.exps & 0xffu : x.exps >> 8) << 23);
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < D / 32; ++c) {
    const uint32_t w = D == 128 ? x.k[i % (D / 64)][c] : x.k[0][2 * i + c % 2];
    s = mfma_bf16(codes4_to_bf16(w, power), q.q[c], s);
  }
  return s;
}

// Two weights times two scales, in f16.
__device__ __forceinline__ uint32_t scaled_weights(float p0, float p1, uint32_t scales) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  const h2 s = __builtin_bit_cast(h2, scales);
  return __builtin_bit_cast(uint32_t, h2{_Float16(__builtin_fmaf(p0, float(s[0]), 0.f)),
                                         _Float16(__builtin_fmaf(p1, float(s[1]), 0.f))});
}
// The larger of two pairs of scales, of which NaN is the largest.
__device__ __forceinline__ uint32_t max_scales(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a),
                                                                __builtin_bit_cast(u16x2, b)));
}
// log2 of the larger of two scales, at least of the smallest there is; of NaN
// that of the largest.
__device__ __forceinline__ float largest_log2(uint32_t scales) {
  const uint32_t most = min(max(scales & 0xffffu, scales >> 16), uint32_t(kScaleMostBits));
  return __builtin_amdgcn_logf(fmaxf(f16_to_f32(uint16_t(most)), kScaleLeast));
}
// log2 of a scale in a word's lower or upper half.  Also of what has none: the
// zero of a token that was never written, NaN; their tokens have a score and a
// share of the sum like any other.
__device__ __forceinline__ float scale_log2_of(uint32_t scales, int half) {
  const float s = f16_to_f32(uint16_t(half == 0 ? scales : scales >> 16));
  return __builtin_amdgcn_logf(fmaxf(s, kScaleLeast));
}

// What a row has met so far: the reference M, this lane's part of the sum of
// 2^kOff exp2(score - M), and its accumulators.
template <int D>
struct RowState4 {
  float m, l;
  f32x4 o[D / 16];
};

// One chunk for the 16 rows of a wave.  `scores_to`: where the scores of the
// lane's row start (token 0; SCORES).  `more_keys` and `more_values` issue the
// next chunk's loads as soon as the registers of this one are used.
template <int D, bool SCORES, typename FK, typename FV>
__device__ __forceinline__ void attend_group4(RowState4<D> &st, Group4<D> &x, const Query4<D> &q,
                                              const Place &at, uint32_t t0, bool present,
                                              float scale_log2, uint32_t g, float *scores_to,
                                              FK more_keys, FV more_values) {
  f32x4 s[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    s[i] = products4<D>(x, i, q) * scale_log2;
  }
  __builtin_amdgcn_sched_barrier(0);
  more_keys();
  __builtin_amdgcn_sched_barrier(0);
  const bool edge = !present || int32_t(t0) + 31 > at.low || int32_t(t0) <= at.hidden;
  if (edge) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int32_t tok = int32_t(t0 + 16 * (i / 4) + 4 * g + i % 4);
      const bool see = present && tok <= at.pos && tok > at.oldest;
      s[i / 4][i % 4] = see ? s[i / 4][i % 4] : -INFINITY;
      x.scales[i / 2] = see ? x.scales[i / 2]
                            : x.scales[i / 2] & (i % 2 == 0 ? 0xffff0000u : 0x0000ffffu);
    }
  }
  if constexpr (SCORES) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      *reinterpret_cast<f32x4 *>(scores_to + t0 + 16 * i + 4 * g) = s[i];
    }
  }
  float top = s[0][0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    top = fmaxf(top, s[i / 4][i % 4]);
  }
  const uint32_t most =
      max_scales(max_scales(x.scales.x, x.scales.y), max_scales(x.scales.z, x.scales.w));
  if (__any(top + largest_log2(most) > st.m + kSlack)) {
    float now = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      now = fmaxf(now, s[i / 4][i % 4] + scale_log2_of(x.scales[i / 2], i % 2));
    }
    now = fmaxf(st.m, floorf(max_groups(now)));
    const float keep = now == -INFINITY ? 1.f : exp2_fast(st.m - now);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      st.o[i] *= keep;
    }
    st.l *= keep;
    st.m = now;
  }
  const float bias = float(kOff) - (st.m == -INFINITY ? 0.f : st.m);
  float p[8], sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    p[i] = exp2_fast(s[i / 4][i % 4] + bias);
    sum += p[i];
  }
  st.l += sum;
  u32x4 pw;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    pw[i] = scaled_weights(p[2 * i], p[2 * i + 1], x.scales[i]);
  }
  const f16x8 pb = __builtin_bit_cast(f16x8, pw);
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    st.o[i] = mfma_f16(codes4_to_f16(x.v[i / 4][i % 4]), pb, st.o[i]);
  }
  __builtin_amdgcn_sched_barrier(0);
  more_values();
  __builtin_amdgcn_sched_barrier(0);
}

// One workgroup owns a part of the tokens of a tile of 16 rows of one
// key/value head, as few_rows_kernel does: its waves take the 32-token chunks
// in turn, each with a softmax of its own, and join them at the end.
//
// What bounds it: the read, and some 5.7 us of start and end.  131072 tokens of 8
// heads of 128 (140 MB) 24 to 25 us, the loads alone, nothing computed, 24.8; 16
// sequences of 4000 14.4, of 8000 23; 128 of 4000 88 (6.2 TB/s).  With caches of 1.2
// GB in turn, so that none is found in the card's last cache, 24.8, 15.6, 25 and 90:
// 7.4 TB/s beyond the 5.7.  Two chunks on their way to a wave 31 (of 131072 tokens),
// two workgroups to a compute unit 27, loads through the caches 27.  333 tokens, 5.7:
// launch, three loads that wait for each other, the join of the waves.
template <int D, int W, bool NT, bool SCORES>
__global__ __launch_bounds__(W * kWave, 3) void few_rows4_kernel(KvAttendArgs a, Scratch x,
                                                              uint32_t each_slots) {
  __shared__ JoinLds<D, W> join;
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
  const Query4<D> q = load_query4<D>(a.q + row * a.q_row + head * a.q_head, a.vec, a.q_sign, g);
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

  RowState4<D> st;
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
    const uint32_t in_mask = (1u << a.pool.shift) - 1;
    const auto chunk_of = [&](uint32_t group) {
      const int id = __builtin_amdgcn_readlane(mine, (group * 32 >> a.pool.shift) - block0);
      return kv4_chunk<D>(a.pool, uint64_t(id < 0 ? 0 : id) * a.pool.heads + kvh,
                          group * 32 & in_mask);
    };
    Group4<D> x32;
    // Keys first, as in the loop: a wait for them then leaves the values' loads
    // in flight.
    load_keys4<D, NT>(x32, chunk_of(grp), lane);
    __builtin_amdgcn_sched_barrier(0);
    load_values4<D, NT>(x32, chunk_of(grp), lane);
    __builtin_amdgcn_sched_barrier(0);
    while (grp < to) {
      // The last chunk is loaded again past the end: no load is conditional.
      const uint32_t ahead = grp + W < to ? grp + W : grp;
      const uint32_t i = (grp * 32 >> a.pool.shift) - block0;
      const uint8_t *next = chunk_of(ahead);
      attend_group4<D, SCORES>(
          st, x32, q, at, grp * 32, __builtin_amdgcn_readlane(mine, i) >= 0, a.scale_log2, g,
          scores_to, [&] { load_keys4<D, NT>(x32, next, lane); },
          [&] { load_values4<D, NT>(x32, next, lane); });
      grp += W;
    }
  }
  join_waves<D, W>(join, a, x, t, kvh, part, parts, st.m, st.l, st.o, 1.f);
}

// ------------------------------------------------------------- many rows
//
// 128 rows to a workgroup, 32 to a wave, with 32 x 32 x 16 products, as
// many_rows_kernel does: steps of 64 tokens go through a ring of two stages in
// LDS, filled by copies that no register waits for; every wave converts what it
// reads.
//
// Order of the operands (lane l, half h = l / 32, i = l % 32):
//   keys: row i of the product is token i with bits 3 and 4 exchanged, so that
//     element e of a result is token {0, 16, 8, 24}[e / 4] + 4h + e % 4 and
//     elements 8c .. 8c + 7 are the 8 tokens of group 2c + h of the values; half
//     h has dims D / 2 * h .. of the contraction, so two exponents at most;
//   values: accumulator m, row i is dim D / 2 * (i / 16) + 16 m + i % 16: a lane's
//     run of dims, read at once, serves all accumulators.
constexpr uint32_t kManyRows = 128, kStages = 2, kManyBlocks = 512;

template <int D>
struct Many4 {
  // A chunk's place in LDS: codes, then exponents and scales, copied by 64 lanes.
  static constexpr uint32_t kCodes = 2 * Kv4Chunk<D>::kSide, kTail = Kv4Chunk<D>::kBytes - kCodes;
  static constexpr uint32_t kSlot = kCodes + 1024, kLds = kStages * 2 * kSlot;
};

// Scales.  Token t's scale s_t enters where the matrix instructions take it for
// nothing: a score starts as log2(s_t) / scale, so that its power is p' = p * s_t at
// once and the largest of what the row has is the reference; the sum takes p' / s_t.
// A wave makes both numbers for a step, a token to a lane, and reads them back as
// the 16 of each lane's results.  A large score rounds log2(s_t) with its own last
// bits: tokens of equal keys and different scales then get weights as far apart.  A
// scale of NaN counts as the least; that there was one is noted, and which rows see
// it found at the end.  (Against the product p * s in f16, with the reference checked
// by a bound: 14 instructions fewer of 158 for 32 x 32, prompts of 4096 and 3001
// tokens of 32 and 8 heads 5 % less time; 218 us now, in a row of such launches.)
//
// What bounds it: 16 matrix instructions of 32 cycles and 144 others of 4 and more
// for 32 rows x 32 tokens, at the clock that they leave the card: 990 TFLOP/s in long
// parts (1024 rows at 140000 tokens, 2.37 ms), 800 to 920 where tiles are few or end
// early.  The next chunk's scores beside this one's powers, in two waves to a SIMD:
// level in parts, 9 % slower in prompts.  A fourth wave with 64 dims: level.
//
// LONG: a part may have more blocks than LDS holds entries of, which are then
// replaced on the way; two waves to a SIMD then have their registers (1 % faster
// than three that spill).
template <int D, bool LONG>
__global__ __launch_bounds__(kWaves * kWave, LONG ? 2 : 3) void many_rows4_kernel(
    KvAttendArgs a, Scratch x, uint32_t each_slots) {
  using Chunk = Kv4Chunk<D>;
  constexpr uint32_t kSlot = Many4<D>::kSlot;
  extern __shared__ __align__(1024) uint8_t many_ring4[];
  const auto ring = [](uint32_t stage) { return many_ring4 + stage * 2 * kSlot; };
  // Where a block's chunks start; one out of the pool has the first one's, plus 1.
  __shared__ uint64_t entries[kManyBlocks];
  // Of a wave and the 64 tokens of a step: log2(scale) in units of scores, and
  // 1 / scale.
  __shared__ __align__(16) float tables[kWaves][2][64];
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
    q[c] = load_query8(a.q + row * a.q_row + head * a.q_head + D / 2 * h + 8 * c, a.vec, a.q_sign);
  }
  const uint32_t from = t.begin / 32 + part * (x.part_tokens / 32);
  const uint32_t all = (t.end + 31) / 32;
  const uint32_t to = min(all, from + x.part_tokens / 32);
  const int32_t *table = a.seqs.tables + t.seq * a.seqs.stride;
  // LDS holds the blocks `held` .. held + kManyBlocks - 1 of the sequence, as
  // far as the part goes.
  uint32_t held = from * 32 >> a.pool.shift;
  const auto hold_blocks = [&] {
    const uint32_t end = to > from ? ((to * 32 - 1) >> a.pool.shift) + 1 : held;
    for (uint32_t b = threadIdx.x; b < kManyBlocks && held + b < end; b += kWaves * kWave) {
      const int32_t id = kv_block(table, a.seqs, a.pool.blocks, held + b);
      const uint8_t *first =
          kv4_chunk<D>(a.pool, uint64_t(id < 0 ? 0 : id) * a.pool.heads + kvh, 0);
      entries[b] = reinterpret_cast<uint64_t>(first) | (id < 0 ? 1u : 0u);
    }
  };
  hold_blocks();
  // bias: what a scaled score becomes a power of two with.
  // dirty: not 0 if a value of NaN was met, in a token that some row sees or not.
  float m = -INFINITY, l = 0.f, limit = -INFINITY, bias = float(kOff);
  uint64_t dirty = 0;
  f32x16 o[D / 32];
#pragma unroll
  for (int c = 0; c < D / 32; ++c) {
    o[c] = f32x16{};
  }
  __syncthreads();

  const uint32_t in_mask = (1u << a.pool.shift) - 1;
  // Copies a step's two chunks (one past the end is the last one again); returns
  // which of them are of no block.
  const auto start_step = [&](uint32_t grp0, uint8_t *stage) {
    uint32_t absent = 0;
#pragma unroll
    for (uint32_t u = 0; u < 2; ++u) {
      const uint32_t tok = min(grp0 + u, to - 1) * 32;
      const u32x2 e =
          *reinterpret_cast<const u32x2 *>(&entries[(tok >> a.pool.shift) - held]);
      const uint32_t low_bits = uniform(e.x);
      absent |= (low_bits & 1u) << u;
      const uint8_t *chunk =
          reinterpret_cast<const uint8_t *>(uint64_t(uniform(e.y)) << 32 | (low_bits & ~1u)) +
          (tok & in_mask) / 32 * Chunk::kBytes;
      uint8_t *slot = stage + u * kSlot;
      if (D == 128) {
        copy_to_lds(chunk + wave * 1024 + lane * 16, slot + wave * 1024);
      } else if (wave / 2 == u) {
        copy_to_lds(chunk + wave % 2 * 1024 + lane * 16, slot + wave % 2 * 1024);
      }
      if (wave == 2 + u) {
        constexpr uint32_t kLanes = Many4<D>::kTail / 16;
        copy_to_lds(chunk + Many4<D>::kCodes + lane % kLanes * 16, slot + Many4<D>::kCodes);
      }
    }
    return absent;
  };
  // Chunks that some of the wave's rows see, and of those the ones that every
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
  uint32_t next = 0;
  if (steps != 0) {
    next = start_step(from, ring(0));
  }
  // Lane's token in a chunk of keys: i with bits 3 and 4 exchanged.
  const uint32_t tok = (i & 7) | (i & 8) << 1 | (i & 16) >> 1;
  // (A register each: taken apart again in the loop they would not fit.)
  const uint32_t key_at = opaque_u32(kv4_key_byte<D>(tok, D / 2 * h));
  const uint32_t exp_at = opaque_u32(Chunk::kExps + kv4_exp_byte(tok, D / 2 * h));
  const uint32_t value_at =
      opaque_u32(Chunk::kSide + kv4_value_dword(h, D / 2 * (i / 16) + i % 16));
  const float per_score = 1.0f / a.scale_log2;
  const uint32_t table_at = opaque_u32(wave * 512 + 32 * h);
  // Four entries, of the tokens of elements e .. e + 3 in chunk u of the step.
  const auto token_table = [&](uint32_t side, uint32_t u, uint32_t e) {
    return *reinterpret_cast<const f32x4 *>(reinterpret_cast<const uint8_t *>(tables) + table_at +
                                            256 * side + 128 * u + 64 * (e / 8) + 4 * (e % 8));
  };
  for (uint32_t step = 0; step < steps; ++step) {
    wait_copies<0>();
    step_barrier();
    const uint32_t absent = next;
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
    {  // each lane's token of the step's 64
      const float scale = f16_to_f32(*reinterpret_cast<const uint16_t *>(
          stage + lane / 32 * kSlot + Chunk::kScales + 2 * (lane % 32)));
      dirty |= __ballot(scale != scale);
      // Of a token that was never written, 0, and of NaN as of the least.
      const float sure = fmaxf(scale, kScaleLeast);
      float *const to = &tables[wave][0][lane];
      to[0] = __builtin_amdgcn_logf(sure) * per_score;
      to[64] = __builtin_amdgcn_rcpf(sure);
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
#pragma unroll
    for (uint32_t u = 0; u < 2; ++u) {
      const uint32_t grp = from + 2 * step + u;
      if (grp - some.first >= some.count) {
        continue;
      }
      const uint8_t *chunk = stage + u * kSlot;
      // Keys: with 128 dims two runs of 32 dims, with 64 of 16.
      u32x4 keys[D / 64];
      float power[D / 64];
      if constexpr (D == 128) {
#pragma unroll
        for (uint32_t c = 0; c < 2; ++c) {
          keys[c] = *reinterpret_cast<const u32x4 *>(chunk + key_at + c * 256);
          power[c] = bits_f32(uint32_t(chunk[exp_at + c * 32]) << 23);
        }
      } else {
        const u32x2 w0 = *reinterpret_cast<const u32x2 *>(chunk + key_at);
        const u32x2 w1 = *reinterpret_cast<const u32x2 *>(chunk + key_at + 256);
        keys[0] = u32x4{w0.x, w0.y, w1.x, w1.y};
        power[0] = bits_f32(uint32_t(chunk[exp_at]) << 23);
      }
      f32x16 s;
#pragma unroll
      for (uint32_t e = 0; e < 16; e += 4) {
        const f32x4 w = token_table(0, u, e);
        s[e] = w[0], s[e + 1] = w[1], s[e + 2] = w[2], s[e + 3] = w[3];
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (uint32_t c = 0; c < D / 16; ++c) {
        s = mfma32_bf16(codes4_to_bf16(keys[c / 4][c % 4], power[c / 4]), q[c], s);
      }
      u32x4 values[2];
#pragma unroll
      for (uint32_t c = 0; c < 2; ++c) {
        if constexpr (D == 128) {
          values[c] = *reinterpret_cast<const u32x4 *>(chunk + value_at + c * 512);
        } else {
          const u32x2 w = *reinterpret_cast<const u32x2 *>(chunk + value_at + c * 512);
          values[c] = u32x4{w.x, w.y, 0u, 0u};
        }
      }
      const uint32_t gone = absent >> u << 31;
      if (((grp - whole.first) | gone) >= whole.count) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int32_t at =
              int32_t(grp * 32) + int32_t((e / 4 % 2) * 16 + e / 8 * 8 + 4 * h + e % 4);
          s[e] = gone == 0 && at <= pos && at > oldest ? s[e] : -INFINITY;
        }
      }
      float top = s[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) {
        top = fmaxf(top, s[e]);
      }
      top *= a.scale_log2;
      if (__any(top > limit)) {
        const auto both =
            __builtin_amdgcn_permlane32_swap(f32_bits(top), f32_bits(top), false, false);
        const float now = fmaxf(m, floorf(fmaxf(bits_f32(both[0]), bits_f32(both[1]))));
        const float keep = now == -INFINITY ? 1.f : exp2_fast(m - now);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          o[c] *= keep;
        }
        l *= keep;
        m = now;
        limit = m + kSlack;
        bias = float(kOff) - (m == -INFINITY ? 0.f : m);
      }
      u32x4 p[2];
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const f32x4 per = token_table(1, u, e);
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          const float p0 = exp2_fast(__builtin_fmaf(s[e + j], a.scale_log2, bias));
          const float p1 = exp2_fast(__builtin_fmaf(s[e + j + 1], a.scale_log2, bias));
          sum = __builtin_fmaf(p0, per[j], sum);
          sum = __builtin_fmaf(p1, per[j + 1], sum);
          p[e / 8][e % 8 / 2 + j / 2] = f32x2_to_f16x2(p0, p1);
        }
      }
      l += sum;
#pragma unroll
      for (uint32_t c = 0; c < 2; ++c) {
        const f16x8 b = __builtin_bit_cast(f16x8, p[c]);
#pragma unroll
        for (uint32_t n = 0; n < D / 32; ++n) {
          o[n] = mfma32_f16(codes4_to_f16(values[c][n]), b, o[n]);
        }
      }
    }
  }
  wait_copies<0>();  // none may land after the workgroup has gone

  // Whether the lane's row sees a value of NaN: the scales once more, a chunk to a
  // lane (rare; the same question in the loop cost prompts 2 % without any NaN).
  bool spoilt = false;
  for (uint32_t grp0 = from; dirty != 0 && grp0 < to; grp0 += kWave) {
    const uint32_t grp = grp0 + lane;
    const int32_t id =
        grp < to ? kv_block(table, a.seqs, a.pool.blocks, grp * 32 >> a.pool.shift) : -1;
    uint32_t bad = 0;  // bit n: scale n is NaN
    if (id >= 0) {
      const uint8_t *chunk =
          kv4_chunk<D>(a.pool, uint64_t(id) * a.pool.heads + kvh, grp * 32 & in_mask);
      const uint16_t *scales = reinterpret_cast<const uint16_t *>(chunk + Chunk::kScales);
      for (uint32_t n = 0; n < 32; ++n) {
        bad |= (scales[n] & 0x7fffu) > 0x7c00u ? 1u << n : 0u;
      }
    }
    for (uint64_t with = __ballot(bad != 0); with != 0; with &= with - 1) {
      const uint32_t of = uint32_t(__builtin_ctzll(with));
      uint32_t rest = uint32_t(__builtin_amdgcn_readlane(int(bad), int(of)));
      for (; rest != 0; rest &= rest - 1) {
        const uint32_t n = uint32_t(__builtin_ctz(rest));
        const int32_t at = int32_t((grp0 + of) * 32 + n / 8 * 4 + n % 4 + n % 8 / 4 * 16);
        spoilt = spoilt || (at <= pos && at > oldest);
      }
    }
  }
  // (The row once more: kept through the loop it would cost it registers.)
  const uint32_t mine = opaque_u32(32 * wave + i), rr = t.r0 + min(mine, last);
  RowSink out;
  out.row = t.first_row + rr / a.group;
  out.head = kvh * a.group + rr % a.group;
  out.live = mine <= last;
  out.whole = parts <= 1;
  out.slot = (out.row * a.heads + out.head) * x.parts + part;
  const auto half = __builtin_amdgcn_permlane32_swap(f32_bits(l), f32_bits(l), false, false);
  const float total = bits_f32(half[0]) + bits_f32(half[1]);
  const float join = spoilt ? __builtin_nanf("") : total == 0.f ? 0.f : 1.0f / total;
#pragma unroll
  for (int n = 0; n < D / 32; ++n) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] = o[n][4 * e + j] * join;
      }
      store4(a, x, out, D, D / 2 * (e / 2) + 16 * n + 8 * (e % 2) + 4 * h, v);
    }
  }
  if (h == 0) {
    store_sums(a, x, out, m, total);
  }
}

// The keys of add_weights_kernel: lane l's part of the A operands of 32 tokens,
// dims D / 2 * (l / 32) + 8 c .. + 7 in operand c.
template <int D>
struct WeightKeys4 {
  static constexpr int kDim = D;
  static __device__ __forceinline__ void load(const KvPool &pool, uint64_t unit, uint32_t in_block,
                                              uint32_t lane, bf16x8 (&k)[D / 16]) {
    const uint32_t h = lane / 32, i = lane % 32;
    const uint8_t *chunk = kv4_chunk<D>(pool, unit, in_block);
#pragma unroll
    for (uint32_t c = 0; c < D / 16; ++c) {
      const uint32_t d = D / 2 * h + 8 * c;
      const uint32_t w = *reinterpret_cast<const uint32_t *>(chunk + kv4_key_byte<D>(i, d));
      const uint32_t e = chunk[Kv4Chunk<D>::kExps + kv4_exp_byte(i, d)];
      k[c] = codes4_to_bf16(w, bits_f32(e << 23));
    }
  }
  static __device__ __forceinline__ uint32_t plane(uint32_t h, uint32_t c) {
    return (D / 2 * h + 8 * c) / 32;
  }
  static __device__ __forceinline__ uint32_t chunk(uint32_t, uint32_t c) { return c % 4; }
};

}  // namespace

KvAttendPlan plan_kv4_attend(const KvAttendArgs &a, uint32_t dim) {
  KvAttendPlan p = plan_kv_attend(a, dim);
  // Small tiles also for more rows than with 8 bits, where all their workgroups run
  // at once (us with the join, small tiles against large ones: 32 heads over 8, 17
  // queries at 16000 tokens 20 / 26, 32 26 / 29; 14 over 2 of 64 dims, 10 queries 10 /
  // 19, 64 20 / 24; 2 over 2, 400 queries 22 / 30), and not past that (17 queries at
  // 30000 38 / 34, 8 times 32 at 8000 70 / 59).
  if (p.kernel == ULLM_KV_KERNEL_MANY_ROWS) {
    const KvAttendPlan few = plan_kv_tiles(a, dim, false);
    if (few.grid <= uint64_t(device_cu_count())) {
      p = few;
    }
  }
  // A wave has half the bytes on their way that it has with 8 bits: eight waves
  // where a workgroup has a compute unit to itself, for 128 dims too (131072
  // tokens of 8 heads: 25.5 us, four waves 31.9; 16 sequences of up to 8192
  // 22.6, 30.6).  Beyond that level: 40 sequences of 4000 35.0 against 35.6, 64 43.4
  // against 41.4, 128 87.9 against 88.7; 160 with 14 and 2 heads of 64 25.3 against
  // 29.0, 256 of 1000 11.6 against 11.3.
  p.waves = p.grid <= device_cu_count() ? 8 : 4;
  return p;
}

template <int D>
static hipError_t launch_attend4(const KvAttendArgs &a, const KvAttendPlan &p, void *workspace,
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
    const bool longer = p.part_tokens > kv_part_limit(kManyBlocks, a.pool.shift, a.window);
    const auto kernel = longer ? many_rows4_kernel<D, true> : many_rows4_kernel<D, false>;
    kernel<<<uint32_t(p.grid), kWaves * kWave, Many4<D>::kLds, s>>>(a, x, each);
  } else if (x.scores != nullptr) {
    few(few_rows4_kernel<D, 8, true, true>, few_rows4_kernel<D, 4, true, true>);
  } else if (p.one_tile) {
    few(few_rows4_kernel<D, 8, true, false>, few_rows4_kernel<D, 4, true, false>);
  } else {
    few(few_rows4_kernel<D, 8, false, false>, few_rows4_kernel<D, 4, false, false>);
  }
  launch_join_parts(a, D, p, x, s);
  if (a.accumulate && x.scores != nullptr) {
    launch_add_scores(a, x, s);
  } else if (a.accumulate) {
    launch_add_weights(add_weights_kernel<WeightKeys4<D>>, a, D, x.stats, s);
  }
  return hipGetLastError();
}

hipError_t launch_kv4_attend(const KvAttendArgs &a, uint32_t dim, const KvAttendPlan &p,
                             void *workspace, hipStream_t s) {
  return dim == 64 ? launch_attend4<64>(a, p, workspace, s)
                   : launch_attend4<128>(a, p, workspace, s);
}

}  // namespace ullm
