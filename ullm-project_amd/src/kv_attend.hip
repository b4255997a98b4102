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
// where every E4M3 code is exact.  A block further below shifts its weights
// down instead (kept exact in the sum, which is f32), one further above raises
// the accumulator's exponent: blocks of any exponents meet in one product with
// an error below 2^-60 of the largest value.
#include "kv_cache.hpp"

namespace ullm {
namespace {

constexpr uint32_t kRows = 16;  // rows of a tile
constexpr uint32_t kWaves = 4;
constexpr float kLn2 = 0.693147180559945309f;
constexpr int kOff = 11;             // weights are at most 2^kOff in f16
constexpr int kDown = -15, kUp = 7;  // exponents at which codes are exact in f16

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

template <int D>
__device__ __forceinline__ Query<D> load_query(const uint16_t *row, bool vec, uint32_t g) {
  Query<D> r;
#pragma unroll
  for (int c = 0; c < D / 64; ++c) {
    const uint16_t *p = row + 64 * c + 16 * g;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (vec) {
        r.q[2 * c + h] = reinterpret_cast<const bf16x8 *>(p)[h];
      } else {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[i] = p[8 * h + 2 * i] | uint32_t(p[8 * h + 2 * i + 1]) << 16;
        }
        r.q[2 * c + h] = __builtin_bit_cast(bf16x8, w);
      }
    }
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

// The codes of 16 keys: tile `tile` (of 16 tokens) of a block and head.
template <int D>
struct Keys {
  u32x4 w[D / 64];
};
template <int D>
__device__ __forceinline__ Keys<D> load_keys(const uint8_t *keys, uint32_t tile, uint32_t lane) {
  Keys<D> r;
#pragma unroll
  for (int c = 0; c < D / 64; ++c) {
    r.w[c] = reinterpret_cast<const u32x4 *>(keys + tile * (D * 16))[c * 64 + lane];
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
  uint32_t seq, length, first_row, live;  // live rows of the tile
  uint32_t r0;                            // first row's index in the sequence's list
  int64_t origin;                         // position of the sequence's first query
  int64_t low, high;                      // positions of the tile's first and last query
  uint32_t begin, end;                    // tokens that some row sees
};

__device__ __forceinline__ bool make_tile(const KvAttendArgs &a, uint32_t id, uint32_t rows,
                                          uint32_t each_slots, Tile *t) {
  const KvSlot slot = kv_find_slot(a.seqs, id, a.group, rows, 1, each_slots);
  if (slot.seq >= a.seqs.batch) {
    return false;
  }
  const KvRows r = kv_rows(a.seqs, slot.seq);
  t->seq = slot.seq;
  t->first_row = r.first;
  t->r0 = slot.local * rows;
  const uint32_t all = r.count * a.group;
  if (t->r0 >= all) {
    return false;
  }
  t->live = all - t->r0 < rows ? all - t->r0 : rows;
  t->length = kv_length(a.seqs, a.pool.shift, slot.seq);
  t->origin = int64_t(t->length) - r.count;
  t->low = t->origin + t->r0 / a.group;
  t->high = t->origin + (t->r0 + t->live - 1) / a.group;
  const int64_t begin = a.window != 0 ? t->low - int64_t(a.window) + 1 : 0;
  t->begin = begin > 0 ? uint32_t(begin) : 0u;
  t->end = t->high >= 0 ? uint32_t(t->high + 1) : 0u;
  return true;
}

// One workgroup owns a tile of 16 rows of one key/value head; its waves take
// the 32-token groups in turn, each with a softmax of its own, and join them
// at the end.
template <int D>
__global__ __launch_bounds__(kWaves * kWave) void few_rows_kernel(KvAttendArgs a,
                                                                 RowStats *stats,
                                                                 uint32_t each_slots) {
  __shared__ float part_o[kWaves][kRows][D + 4];
  __shared__ float part_m[kWaves][kRows], part_l[kWaves][kRows];
  Tile t;
  if (!make_tile(a, blockIdx.x / a.pool.heads, kRows, each_slots, &t)) {
    return;
  }
  const uint32_t kvh = blockIdx.x % a.pool.heads;
  const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint32_t g = lane / 16, col = lane % 16;
  // Rows past the end see what the last one does; their results are not stored.
  const uint32_t r = t.r0 + (col < t.live ? col : t.live - 1);
  const uint32_t head = kvh * a.group + r % a.group;
  const uint64_t row = t.first_row + r / a.group;
  const int64_t pos = t.origin + r / a.group;
  const int64_t oldest = a.window != 0 ? pos - int64_t(a.window) : -1;  // not seen
  const Query<D> q = load_query<D>(a.q + row * a.q_row + head * a.q_head, a.vec, g);
  const int32_t *table = a.seqs.tables + t.seq * a.seqs.stride;

  float m = -INFINITY, l = 0.f;  // running maximum; sum of 2^kOff exp2(score - m)
  int acc_exp = kKvExpMin;       // o holds sums over 2^(acc_exp)
  f32x4 o[D / 16];
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  for (uint32_t grp = t.begin / 32 + wave; grp < (t.end + 31) / 32; grp += kWaves) {
    const uint32_t t0 = grp * 32;
    const int32_t id = kv_block(table, a.seqs, a.pool.blocks, t0 >> a.pool.shift);
    if (id < 0) {
      continue;
    }
    const uint64_t unit = uint64_t(id) * a.pool.heads + kvh;
    const uint8_t *keys = a.pool.codes + unit * (uint64_t(2 * D) << a.pool.shift);
    const uint8_t *values = keys + (uint64_t(D) << a.pool.shift);
    const uint32_t in_block = t0 & ((1u << a.pool.shift) - 1);
    const float pk = exp2_int(a.pool.exps[unit * 2]);
    const int ev = a.pool.exps[unit * 2 + 1];
    if (ev > acc_exp + kUp) {
      const float f = exp2_int(max(acc_exp - ev, -126));
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        o[i] *= f;
      }
      acc_exp = ev;
    }
    const int d = ev - acc_exp;
    const float pv = exp2_int(d < kDown ? kDown : d);
    const int shift = d < kDown ? max(d - kDown, -100) : 0;
    f32x4 s[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s[i] = products(load_keys<D>(keys, in_block / 16 + i, lane), pk, q) * a.scale_log2;
    }
    const bool edge = int64_t(t0) + 31 > t.low ||
                      (a.window != 0 && int64_t(t0) <= t.high - int64_t(a.window));
    uint32_t seen = 0xffu;
    if (edge) {
      seen = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int64_t tok = int64_t(t0) + 16 * (i / 4) + 4 * g + i % 4;
        const bool see = tok <= pos && tok > oldest;
        seen |= see ? 1u << i : 0u;
        s[i / 4][i % 4] = see ? s[i / 4][i % 4] : -INFINITY;
      }
    }
    float top = s[0][0];  // fmaxf passes NaN over: it makes the sum below NaN
#pragma unroll
    for (int i = 1; i < 8; ++i) {
      top = fmaxf(top, s[i / 4][i % 4]);
    }
    top = fmaxf(top, __shfl_xor(top, 16, kWave));
    top = fmaxf(top, __shfl_xor(top, 32, kWave));
    const float now = fmaxf(m, top);
    const float ref = now == -INFINITY ? 0.f : now;
    const float keep = exp2_fast(m - ref);
    m = now;
    float p[8], sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      p[i] = exp2_fast(s[i / 4][i % 4] - (ref - float(kOff + shift)));
      sum += p[i];
    }
    l = l * keep + sum * exp2_int(-shift);
    u32x4 pw;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      pw[i] = f32x2_to_f16x2(p[2 * i], p[2 * i + 1]);
    }
    const f16x8 pb = __builtin_bit_cast(f16x8, pw);
    const u32x4 *vt =
        reinterpret_cast<const u32x4 *>(values + in_block / 32 * (D * 32)) + lane;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      u32x4 w = vt[c * 64];
      u32x4 bad_v = {0u, 0u, 0u, 0u};
      if (edge) {
        // A NaN in a token that some rows do not see must not reach them
        // through a weight of zero: it is taken out of the product, and the
        // rows that see it become NaN.
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          bad_v[i] = nan_bytes(w[i]);
          w[i] &= ~(bad_v[i] | (bad_v[i] - (bad_v[i] >> 7)));
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        f32x4 &acc = o[2 * c + h];
        acc = mfma_f16(codes_to_f16(w[2 * h], w[2 * h + 1], pv), pb, acc * keep);
        if (edge && __any(bad_v[2 * h] | bad_v[2 * h + 1])) {
          u32x4 nv, sv;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t two = bad_v[2 * h + i / 2] >> (16 * (i % 2));
            nv[i] = (two & 0x80u ? 0x3c00u : 0u) | (two & 0x8000u ? 0x3c000000u : 0u);
            sv[i] = (seen >> (2 * i) & 1u ? 0x3c00u : 0u) |
                    (seen >> (2 * i + 1) & 1u ? 0x3c000000u : 0u);
          }
          const f32x4 hit =
              mfma_f16(__builtin_bit_cast(f16x8, nv), __builtin_bit_cast(f16x8, sv),
                       f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            acc[i] = hit[i] > 0.f ? __builtin_nanf("") : acc[i];
          }
        }
      }
    }
  }
  l += __shfl_xor(l, 16, kWave);
  l += __shfl_xor(l, 32, kWave);
  if (g == 0) {
    part_m[wave][col] = m;
    part_l[wave][col] = l;
  }
  // Means of the wave's tokens, to be joined by their sums.
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  const float power = exp2_int(acc_exp);
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {
    *reinterpret_cast<f32x4 *>(&part_o[wave][col][16 * i + 4 * g]) = o[i] * inv * power;
  }
  __syncthreads();
  // 16 threads to a row, D / 16 dims each.
  const uint32_t mine = threadIdx.x / 16;
  if (mine >= t.live) {
    return;
  }
  const uint32_t rr = t.r0 + mine;
  const uint64_t out_row = t.first_row + rr / a.group;
  const uint32_t out_head = kvh * a.group + rr % a.group;
  float top = part_m[0][mine];
#pragma unroll
  for (uint32_t w = 1; w < kWaves; ++w) {
    top = fmaxf(top, part_m[w][mine]);
  }
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f, f[kWaves];
#pragma unroll
  for (uint32_t w = 0; w < kWaves; ++w) {
    f[w] = exp2_fast(part_m[w][mine] - ref) * part_l[w][mine];
    sum += f[w];
  }
  const float join = sum == 0.f ? 0.f : 1.0f / sum;
  const uint32_t d0 = threadIdx.x % 16 * (D / 16);
  uint32_t packed[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    float v[2] = {0.f, 0.f};
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) {
      v[0] += part_o[w][mine][d0 + 2 * i] * f[w];
      v[1] += part_o[w][mine][d0 + 2 * i + 1] * f[w];
    }
    packed[i] = f32x2_to_bf16x2(v[0] * join, v[1] * join);
  }
  uint16_t *to = a.out + out_row * a.out_row + out_head * a.out_head + d0;
  if (a.out_vec) {
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      reinterpret_cast<u32x2 *>(to)[i] = u32x2{packed[2 * i], packed[2 * i + 1]};
    }
  } else {
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      to[2 * i] = uint16_t(packed[i]);
      to[2 * i + 1] = uint16_t(packed[i] >> 16);
    }
  }
  if (threadIdx.x % 16 == 0) {
    const uint64_t at = out_row * a.heads + out_head;
    if (a.lse != nullptr) {
      a.lse[at] = sum == 0.f ? -INFINITY : (top + (log2f(sum) - float(kOff))) * kLn2;
    }
    if (stats != nullptr) {
      stats[at] = RowStats{ref - float(kOff), join};
    }
  }
}

// Adds the weights that the tokens of a 32-token group receive from all rows
// of their sequence: a wave owns the group, so its sums have a fixed order;
// the addition is atomic for blocks that several sequences of a call share.
template <int D>
__global__ __launch_bounds__(kWaves * kWave) void add_weights_kernel(KvAttendArgs a,
                                                                    const RowStats *stats) {
  const uint32_t kvh = blockIdx.y, b = blockIdx.z;
  const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint32_t g = lane / 16, col = lane % 16;
  const uint32_t t0 = (blockIdx.x * kWaves + wave) * 32;
  const uint32_t length = kv_length(a.seqs, a.pool.shift, b);
  if (t0 >= length) {
    return;
  }
  const int32_t id = kv_block(a.seqs.tables + b * a.seqs.stride, a.seqs, a.pool.blocks,
                              t0 >> a.pool.shift);
  if (id < 0) {
    return;
  }
  const KvRows rows = kv_rows(a.seqs, b);
  const uint64_t unit = uint64_t(id) * a.pool.heads + kvh;
  const uint8_t *keys = a.pool.codes + unit * (uint64_t(2 * D) << a.pool.shift);
  const uint32_t in_block = t0 & ((1u << a.pool.shift) - 1);
  const float power = exp2_int(a.pool.exps[unit * 2]);
  Keys<D> k[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    k[i] = load_keys<D>(keys, in_block / 16 + i, lane);
  }
  const int64_t origin = int64_t(length) - rows.count;
  const uint32_t all = rows.count * a.group;
  // Queries before the group's first token, or past its last one's window,
  // see none of it.
  const int64_t from = int64_t(t0) - origin;
  uint32_t r0 = from <= 0 ? 0u
                : from < int64_t(rows.count) ? uint32_t(from) * a.group / kRows * kRows
                                             : all;
  const int64_t past = a.window != 0 ? int64_t(t0) + 31 + a.window - origin : rows.count;
  const uint32_t r1 = past <= 0 ? 0u
                      : past < int64_t(rows.count) ? uint32_t(past) * a.group
                                                   : all;
  float sum[8] = {};
  for (; r0 < r1; r0 += kRows) {
    const uint32_t r = r0 + col;
    const bool live = r < all;
    const uint32_t head = kvh * a.group + (live ? r % a.group : 0u);
    const uint64_t row = rows.first + (live ? r / a.group : 0u);
    const int64_t pos = origin + r / a.group;
    const int64_t oldest = a.window != 0 ? pos - int64_t(a.window) : -1;
    const Query<D> q = load_query<D>(a.q + row * a.q_row + head * a.q_head, a.vec, g);
    const RowStats st = stats[row * a.heads + head];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f32x4 s = products(k[i], power, q) * a.scale_log2;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t tok = int64_t(t0) + 16 * i + 4 * g + j;
        const float p = exp2_fast(s[j] - st.top) * st.inv_sum;
        sum[4 * i + j] += live && tok <= pos && tok > oldest ? p : 0.f;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) {
      sum[i] += __shfl_xor(sum[i], off, kWave);
    }
  }
  if (col == 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t t = 16 * (i / 4) + 4 * g + i % 4;
      if (t0 + t < length) {
        unsafeAtomicAdd(&a.pool.weights[(unit << a.pool.shift) + in_block + t], sum[i]);
      }
    }
  }
}

}  // namespace

KvAttendPlan plan_kv_attend(const KvAttendArgs &a, uint32_t dim) {
  KvAttendPlan p;
  if (a.seqs.rows == 0 || a.seqs.batch == 0) {
    return p;
  }
  p.kernel = ULLM_KV_KERNEL_FEW_ROWS;
  p.row_tile = kRows;
  p.part_tokens = a.seqs.max_blocks << a.pool.shift;
  const uint64_t each = (uint64_t(a.seqs.each) * a.group + kRows - 1) / kRows;
  p.grid = kv_slots(a.seqs, a.group, kRows, 1, each) * a.pool.heads;
  if (a.accumulate) {
    p.workspace = uint64_t(a.seqs.rows) * a.heads * sizeof(RowStats);
  }
  return p;
}

template <int D>
static hipError_t launch_attend(const KvAttendArgs &a, const KvAttendPlan &p, void *workspace,
                                hipStream_t s) {
  RowStats *stats = a.accumulate ? static_cast<RowStats *>(workspace) : nullptr;
  const uint32_t each = (a.seqs.each * a.group + kRows - 1) / kRows;
  few_rows_kernel<D><<<uint32_t(p.grid), kWaves * kWave, 0, s>>>(a, stats, each);
  if (a.accumulate) {
    const uint64_t tokens = uint64_t(a.seqs.max_blocks) << a.pool.shift;
    const dim3 grid(uint32_t((tokens + 32 * kWaves - 1) / (32 * kWaves)), a.pool.heads,
                    a.seqs.batch);
    add_weights_kernel<D><<<grid, kWaves * kWave, 0, s>>>(a, stats);
  }
  return hipGetLastError();
}

hipError_t launch_kv_attend(const KvAttendArgs &a, uint32_t dim, const KvAttendPlan &p,
                            void *workspace, hipStream_t s) {
  return dim == 64 ? launch_attend<64>(a, p, workspace, s)
                   : launch_attend<128>(a, p, workspace, s);
}

}  // namespace ullm
