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
// result decides how exactly it enters, whatever the scales of the others.  M
// moves when some p' passes 2^15: the weights of a group are computed first and
// looked at after.  With scales from 2^-19 to 2^16 the p of a row's sum stay
// within 2^-28 and 2^52 of what they would be over the largest score, far inside
// f32.
//
// NaN.  Codes are finite, NaN is in a key's exponent or a value's scale, so that
// it can reach a row only through its score or its weight: tokens that a row
// does not see have score -infinity and scale 0 put in their place.
#include <algorithm>

#include "kv_attend.hpp"
#include "kv_cache4.hpp"

namespace ullm {
namespace {

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
// The larger of two pairs of f16, NaN passed over.
__device__ __forceinline__ uint32_t max_f16(uint32_t a, uint32_t b) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(h2, a),
                                                                __builtin_bit_cast(h2, b)));
}
// Whether one of two weights (not negative, or NaN) has passed 2^15; infinity has.
__device__ __forceinline__ bool past_limit(uint32_t w) {
  const auto past = [](uint32_t h) { return h > 0x7800u && h <= 0x7c00u; };
  return past(w & 0xffffu) || past(w >> 16);
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
  float p[8];
  u32x4 pw;
  const auto weigh = [&] {
    const float bias = float(kOff) - (st.m == -INFINITY ? 0.f : st.m);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[i] = exp2_fast(s[i / 4][i % 4] + bias);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      pw[i] = scaled_weights(p[2 * i], p[2 * i + 1], x.scales[i]);
      top = max_f16(top, pw[i]);
    }
    return past_limit(top);
  };
  // The first tokens that a row sees always set its reference.
  bool grow = st.m == -INFINITY;
  grow = weigh() || grow;
  if (__any(grow)) {
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float y = s[i / 4][i % 4] + scale_log2_of(x.scales[i / 2], i % 2);
      top = fmaxf(top, y);  // passes NaN over: it makes the sum below NaN
    }
    top = max_groups(top);
    const float now = fmaxf(st.m, top);
    const float keep = st.m == -INFINITY ? 1.f : exp2_fast(st.m - now);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      st.o[i] *= keep;
    }
    st.l *= keep;
    st.m = now;
    weigh();
  }
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    sum += p[i];
  }
  st.l += sum;
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

// Adds the weights that tokens receive from all rows of their sequence, by a
// second product of keys and queries: a wave owns 32 tokens and walks the rows,
// 16 at a time.
template <int D>
__global__ __launch_bounds__(kWaves * kWave) void add_weights4_kernel(KvAttendArgs a,
                                                                      const RowStats *stats) {
  const uint32_t kvh = blockIdx.y, b = blockIdx.z;
  const uint32_t lane = threadIdx.x % kWave, g = lane / 16, col = lane % 16;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const uint32_t length = kv_length(a.seqs, a.pool.shift, b);
  const uint32_t t0 = (blockIdx.x * kWaves + wave) * 32;
  if (t0 >= length) {
    return;
  }
  const int32_t id = kv_block(a.seqs.tables + b * a.seqs.stride, a.seqs, a.pool.blocks,
                              t0 >> a.pool.shift);
  const KvRows rows = kv_rows(a.seqs, b);
  const uint32_t all = rows.count * a.group;
  if (id < 0 || all == 0) {
    return;
  }
  const int64_t origin = int64_t(length) - rows.count;
  const uint64_t unit = uint64_t(id) * a.pool.heads + kvh;
  const uint32_t in_block = t0 & ((1u << a.pool.shift) - 1);
  Group4<D> x;
  load_keys4<D, false>(x, kv4_chunk<D>(a.pool, unit, in_block), lane);
  float sum[8] = {};
  for (uint32_t r0 = 0; r0 < all; r0 += kRows) {
    const uint32_t r = r0 + col < all ? r0 + col : all - 1, head = kvh * a.group + r % a.group;
    const uint64_t row = rows.first + r / a.group;
    const Query4<D> q = load_query4<D>(a.q + row * a.q_row + head * a.q_head, a.vec, a.q_sign, g);
    const RowStats st = stats[stats_at(a, kvh, rows.first) + r];
    const int32_t pos = int32_t(origin + r / a.group), oldest = oldest_hidden(pos, a.window);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f32x4 s = products4<D>(x, i, q);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int32_t tok = int32_t(t0 + 16 * i + 4 * g + j);
        const bool see = r0 + col < all && tok <= pos && tok > oldest;
        // A row of NaN gives it to what it sees, and nothing to the rest.
        const float p = exp2_fast(s[j] * a.scale_log2 - st.top) * st.inv_sum;
        sum[4 * i + j] += see ? p : 0.f;
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) {
      sum[e] += __shfl_xor(sum[e], off, kWave);
    }
    const uint32_t t = 16 * (e / 4) + 4 * g + e % 4;
    if (col == uint32_t(e) && t0 + t < length) {
      unsafeAtomicAdd(&a.pool.weights[(unit << a.pool.shift) + in_block + t], sum[e]);
    }
  }
}

// Workgroups for each compute unit: tokens are split into that many parts.
constexpr uint32_t kPartLeast4 = 512;

}  // namespace

KvAttendPlan plan_kv4_attend(const KvAttendArgs &a, uint32_t dim) {
  KvAttendPlan p;
  if (a.seqs.rows == 0 || a.seqs.batch == 0) {
    return p;
  }
  const uint32_t cus = device_cu_count();
  const uint64_t rows_of_head = uint64_t(a.seqs.rows) * a.group;
  p.kernel = ULLM_KV_KERNEL_FEW_ROWS;
  p.row_tile = kRows;
  const uint64_t tiles =
      kv_slots(a.seqs, a.group, kRows, 1, each_tiles(a, kRows)) * a.pool.heads;
  const uint64_t tokens = uint64_t(a.seqs.max_blocks) << a.pool.shift;
  const uint64_t span =
      a.window == 0 ? tokens : std::min<uint64_t>(tokens, uint64_t(a.window) + kRows / a.group + 32);
  const uint64_t split = tiles < cus ? cus / tiles : 1;
  const uint64_t part = std::max<uint64_t>((span + split - 1) / split, kPartLeast4);
  const uint64_t most = kv_part_limit(kWave, a.pool.shift, a.window) / 64 * 64;
  p.part_tokens = uint32_t(std::min<uint64_t>((part + 63) / 64 * 64, most));
  p.parts = uint32_t((span + p.part_tokens - 1) / p.part_tokens);
  p.one_tile = rows_of_head <= uint64_t(kRows) * a.seqs.batch;
  p.grid = tiles * p.parts;
  p.waves = p.grid <= uint64_t(cus) * 64 / dim ? 8 : 4;
  uint64_t bytes = 0;
  scratch_of(a, dim, p, nullptr, &bytes);
  p.workspace = bytes;
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
  if (p.one_tile) {
    few(few_rows4_kernel<D, 8, true, false>, few_rows4_kernel<D, 4, true, false>);
  } else {
    few(few_rows4_kernel<D, 8, false, false>, few_rows4_kernel<D, 4, false, false>);
  }
  launch_join_parts(a, D, p, x, s);
  if (a.accumulate) {
    const uint64_t tokens = uint64_t(a.seqs.max_blocks) << a.pool.shift;
    const dim3 grid(uint32_t((tokens + 32 * kWaves - 1) / (32 * kWaves)), a.pool.heads,
                    a.seqs.batch);
    add_weights4_kernel<D><<<grid, kWaves * kWave, 0, s>>>(a, x.stats);
  }
  return hipGetLastError();
}

hipError_t launch_kv4_attend(const KvAttendArgs &a, uint32_t dim, const KvAttendPlan &p,
                             void *workspace, hipStream_t s) {
  return dim == 64 ? launch_attend4<64>(a, p, workspace, s)
                   : launch_attend4<128>(a, p, workspace, s);
}

}  // namespace ullm
