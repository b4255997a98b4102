// kv_store4.hip -- what writes and moves the tokens of the 4-bit key/value
// cache, and the appends that rotate: append, gather and evict.  All are bound
// by HBM and launches.
#include "kernels.hpp"
#include "kv_cache4.hpp"
#include "kv_rotary.hpp"
#include "kv_store.hpp"

namespace ullm {
namespace {

// ------------------------------------------------------------- 4-bit codes

// Smallest exponent e with a <= 6 * 2^e = 1.5 * 2^(e + 2), clamped, plus 127, of
// the largest magnitude's f32 bits; of infinities and NaN kKv4ExpNan.
__device__ __forceinline__ uint32_t key_exp4(uint32_t a) {
  const int e = int(a >> 23) - 127 - 2 + ((a & 0x7fffffu) > 0x400000u ? 1 : 0);
  const int c = e < kKvExpMin ? kKvExpMin : e > kKvExpMax ? kKvExpMax : e;
  return a >= 0x7f800000u ? kKv4ExpNan : uint32_t(c + 127);
}
__device__ __forceinline__ float exp4_power(uint32_t e) { return bits_f32(e << 23); }

// Smallest number of 6 significant bits, within the f16 ones that are allowed,
// whose 6-fold reaches a magnitude.  Products by 6 of such numbers are exact, so
// the comparisons decide; the quotient before them only has to be near.
__device__ __forceinline__ float value_scale4(float a) {
  constexpr uint32_t kStep = 1u << 18;
  float s = bits_f32(f32_bits(a * (0.999999f / 6.f)) & ~(kStep - 1));
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    s = 6.f * s < a ? bits_f32(f32_bits(s) + kStep) : s;
  }
  return fminf(fmaxf(s, kScaleLeast), kScaleMost);
}

// Sixteen codes, low nibble first, of sixteen numbers over a power of two.
__device__ __forceinline__ u32x2 encode4(const float (&x)[16], float power) {
  u32x2 r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[8 * i], x[8 * i + 1], power, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[8 * i + 2], x[8 * i + 3], power, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[8 * i + 4], x[8 * i + 5], power, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[8 * i + 6], x[8 * i + 7], power, 3);
    r[i] = w;
  }
  return r;
}
// Of sixteen bf16 over any scale s.  The quotient is exact where it is a border
// of two codes (a number of at most 4 significant bits): x / s rounded, and once
// more by its remainder.
__device__ __forceinline__ u32x2 encode4_scaled(const float (&x)[16], float s) {
  const float inv = 1.f / s;
  float y[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    y[i] = x[i] * inv;
    y[i] = __builtin_fmaf(__builtin_fmaf(-y[i], s, x[i]), inv, y[i]);
  }
  return encode4(y, 1.f);
}
// Four codes, a byte each in w, as bf16 times a scale.
__device__ __forceinline__ u32x2 decode4_bytes(uint32_t w, float s) {
  const uint32_t t = w | w >> 4;  // bytes 0 and 2: two codes each
  const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(t, 1.f, 0);
  const auto hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(t, 1.f, 2);
  return {f32x2_to_bf16x2(lo[0] * s, lo[1] * s), f32x2_to_bf16x2(hi[0] * s, hi[1] * s)};
}

__device__ __forceinline__ void unpack16(const Bf16x16 &x, float (&f)[16]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t w = x.w[i / 4][i % 4];
    f[2 * i] = bits_f32(w << 16);
    f[2 * i + 1] = bits_f32(w & 0xffff0000u);
  }
}
// Bits of the largest magnitude of sixteen numbers (NaN above all) over the
// lanes that differ in the bits of `lanes`.
template <uint32_t LANES>
__device__ __forceinline__ uint32_t largest16(const float (&f)[16]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    top = max(top, f32_bits(f[i]) & 0x7fffffffu);
  }
#pragma unroll
  for (uint32_t off = 1; off < LANES; off <<= 1) {
    top = max(top, uint32_t(__shfl_xor(int(top), off, kWave)));
  }
  return top;
}

// ----------------------------------------------------------------- rotation

// Up to T tokens of a sequence, of which lo .. hi - 1 are rows of the call: row
// `row0` + t is token t, at place `base` + t.
struct Span {
  int64_t row0, base;
  uint32_t lo, hi;
};
// That of a sequence's slot; false if it has no rows.
template <uint32_t T>
__device__ __forceinline__ bool span_of(const KvSlot &slot, uint32_t length, Span *s) {
  const int64_t origin = int64_t(length) - slot.rows.count;  // place of the first row
  // Rounded down, places before the first token too.
  s->base = (origin >= 0 ? origin / T : -((T - 1 - origin) / int64_t(T))) * T +
            int64_t(slot.local) * T;
  s->lo = origin > s->base ? uint32_t(origin - s->base) : 0u;
  s->hi = uint32_t(min(max(int64_t(length) - s->base, int64_t(0)), int64_t(T)));
  s->row0 = int64_t(slot.rows.first) + (s->base - origin);
  return s->lo < s->hi;
}

// Threads of a workgroup for T tokens: one for each unit of 16 dims at least.
template <int D, uint32_t T>
constexpr uint32_t kSpanThreads = T * (D / 16) > kThreads ? T * (D / 16) : kThreads;

// A thread's part of a span's rows: token t, pairs 8u .. 8u + 7, of heads `head`,
// `head` + step and so on; none where `head` is kNoHead.
constexpr uint32_t kNoHead = ~0u;
struct Lot {
  uint32_t t, row, u, head, step;  // row: t counted from lo
};
template <int D, uint32_t T>
__device__ __forceinline__ Lot lot_of(const Span &s) {
  constexpr uint32_t kUnits = D / 16;
  const uint32_t n = (s.hi - s.lo) * kUnits, step = kSpanThreads<D, T> / n;
  const uint32_t head = threadIdx.x / n, i = threadIdx.x % n;
  return {s.lo + i / kUnits, i / kUnits, i % kUnits, head < step ? head : kNoHead, step};
}

// Cosines and sines of a span, those of token t from t * D / 2 on: where pair 8u + i
// is there keeps both the threads that write a token's pairs in order and those that
// read pair i of eight apart, some tokens at a time, on banks of their own.
template <int D, uint32_t T>
struct SpanTurns {
  Turn at[T][D / 2];
};
__device__ __forceinline__ uint32_t turn_slot(uint32_t t, uint32_t u, uint32_t i) {
  return 8 * (u ^ (t & 1)) + (i ^ (u & 7) ^ 2 * (t & 2));
}
// Pair j's frequency, and its axis' positions from the span's token 0 on.
struct PairTurns {
  float f;
  const int32_t *at;
};
__device__ __forceinline__ PairTurns pair_turns(const KvRotary &r, const Span &s, uint32_t j) {
  const uint32_t axis = r.pair_axes == nullptr ? 0u : min(uint32_t(r.pair_axes[j]), r.axes - 1);
  return {r.inv_freq[j],
          r.positions == nullptr ? nullptr : r.positions + axis * r.position_stride + s.row0};
}
__device__ __forceinline__ int32_t place_of(const PairTurns &p, const Span &s, uint32_t t) {
  return p.at == nullptr ? int32_t(s.base + t) : p.at[t];
}
template <int D, uint32_t T>
__device__ __forceinline__ void span_turns(const KvRotary &r, const Span &s,
                                           SpanTurns<D, T> *turns) {
  constexpr uint32_t kAtOnce = kSpanThreads<D, T> / (D / 2), kRounds = T / kAtOnce;
  const uint32_t j = threadIdx.x % (D / 2), first = s.lo + threadIdx.x / (D / 2);
  if (j >= r.dims / 2) {
    return;
  }
  const PairTurns p = pair_turns(r, s, j);
  // A thread's positions are on their way at once, not each a load to wait for
  // (7300 tokens with positions of three axes: 20.0 us, one by one 21.7).
  int32_t place[kRounds];
#pragma unroll
  for (uint32_t i = 0; i < kRounds; ++i) {
    const uint32_t t = first + i * kAtOnce;
    place[i] = t < s.hi ? place_of(p, s, t) : 0;
  }
  for (uint32_t t = first; t < s.hi; t += kAtOnce) {
    turns->at[t][turn_slot(t, j / 8, j % 8)] = turn_of(place[0], p.f);
#pragma unroll
    for (uint32_t i = 0; i + 1 < kRounds; ++i) {
      place[i] = place[i + 1];
    }
  }
}

// Eight pairs of a row as they lie in memory: two runs of eight dims, or one of
// sixteen (`side`: a pair's elements side by side).
struct RawPairs {
  u32x4 a, b;
};
// Where that is so: pairs of neighbours, dims past the rotated ones among them.
__device__ __forceinline__ bool side_by_side(const KvRotary &r, uint32_t u, bool runs) {
  return runs && (r.interleaved || 8 * u >= r.dims / 2);
}
__device__ __forceinline__ RawPairs load_pairs(const uint16_t *row, const KvRotary &r, uint32_t u,
                                               bool runs) {
  RawPairs p;
  if (runs) {
    const PairDims d = pair_dims(8 * u, r.dims, r.interleaved);
    p.a = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(row + d.first));
    p.b = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(
        row + (side_by_side(r, u, runs) ? d.first + 8 : d.second)));
  } else {
#pragma unroll
    for (uint32_t i = 0; i < 8; i += 2) {
      const PairDims d = pair_dims(8 * u + i, r.dims, r.interleaved);
      const PairDims e = pair_dims(8 * u + i + 1, r.dims, r.interleaved);
      p.a[i / 2] = row[d.first] | uint32_t(row[e.first]) << 16;
      p.b[i / 2] = row[d.second] | uint32_t(row[e.second]) << 16;
    }
  }
  return p;
}
// The elements of pair i.
struct PairXY {
  float x, y;
};
__device__ __forceinline__ PairXY raw_pair(const RawPairs &p, bool side, int i) {
  const uint32_t near = i < 4 ? p.a[i % 4] : p.b[i % 4];
  const uint32_t fx = p.a[i / 2], fy = p.b[i / 2];
  return {bits_f32(side ? near << 16 : i % 2 == 0 ? fx << 16 : fx & 0xffff0000u),
          bits_f32(side ? near & 0xffff0000u : i % 2 == 0 ? fy << 16 : fy & 0xffff0000u)};
}

// A thread's eight turns, and which of its pairs they are for.
struct Turns8 {
  Turn w[8];
  uint32_t live;
};
// The same in f32, for queries.
struct QueryTurns8 {
  float c[8], s[8];
  uint32_t live;
};
template <int D, uint32_t T>
__device__ __forceinline__ Turns8 load_turns(const SpanTurns<D, T> &turns, const KvRotary &r,
                                             const Lot &lot) {
  Turns8 v;
  const uint32_t pairs = r.dims / 2, first = 8 * lot.u;
  v.live = first >= pairs ? 0u : pairs - first >= 8 ? 0xffu : (1u << (pairs - first)) - 1;
#pragma unroll
  for (uint32_t i = 0; i < 8; ++i) {
    v.w[i] = turns.at[lot.t][turn_slot(lot.t, lot.u, i)];
  }
  return v;
}

// A query's eight pairs, rotated in f32, to their place.  Rows of q are read
// once, and their results next by another kernel: both pass the caches by (14006
// tokens of 32 and 8 heads: 64 us, through them 75).
__device__ __forceinline__ void rotate_query(uint16_t *row, const RawPairs &p, const KvRotary &r,
                                             const QueryTurns8 &v, uint32_t u, bool runs) {
  const bool side = side_by_side(r, u, runs);
  float x[8], y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const PairXY e = raw_pair(p, side, i);
    const float c = v.c[i], s = v.s[i];
    const bool live = (v.live >> i & 1u) != 0;
    x[i] = live ? __builtin_fmaf(e.x, c, -(e.y * s)) : e.x;
    y[i] = live ? __builtin_fmaf(e.y, c, e.x * s) : e.y;
  }
  if (runs) {
    const PairDims d = pair_dims(8 * u, r.dims, r.interleaved);
    u32x4 a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = side ? f32x2_to_bf16x2(x[i], y[i]) : f32x2_to_bf16x2(x[2 * i], x[2 * i + 1]);
      b[i] = side ? f32x2_to_bf16x2(x[4 + i], y[4 + i]) : f32x2_to_bf16x2(y[2 * i], y[2 * i + 1]);
    }
    __builtin_nontemporal_store(a, reinterpret_cast<u32x4 *>(row + d.first));
    __builtin_nontemporal_store(
        b, reinterpret_cast<u32x4 *>(row + (side ? d.first + 8 : d.second)));
  } else {
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      const PairDims d = pair_dims(8 * u + i, r.dims, r.interleaved);
      row[d.first] = f32_to_bf16(x[i]);
      row[d.second] = f32_to_bf16(y[i]);
    }
  }
}

// Rows of a span's rotated keys in LDS, its first new token's first.
template <int D, uint32_t T>
struct KeyImage {
  alignas(16) float x[T][D + 4];
};
// A key's eight pairs, rotated in 64 bits.
template <int D, uint32_t T>
__device__ __forceinline__ void rotate_key(KeyImage<D, T> *to, const RawPairs &p,
                                           const KvRotary &r, const Turns8 &v, const Lot &lot,
                                           bool runs) {
  const bool side = side_by_side(r, lot.u, runs);
  float a[8], b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const PairXY e = raw_pair(p, side, i);
    const double x = e.x, y = e.y, c = v.w[i].c, s = v.w[i].s;
    const bool live = (v.live >> i & 1u) != 0;
    a[i] = live ? to_odd(fma(x, c, -(y * s))) : e.x;
    b[i] = live ? to_odd(fma(y, c, x * s)) : e.y;
  }
  float *const row = to->x[lot.row];
  if (runs) {
    const PairDims d = pair_dims(8 * lot.u, r.dims, r.interleaved);
    f32x4 *const near = reinterpret_cast<f32x4 *>(row + d.first);
    f32x4 *const far = reinterpret_cast<f32x4 *>(row + (side ? d.first + 8 : d.second));
    near[0] = side ? f32x4{a[0], b[0], a[1], b[1]} : f32x4{a[0], a[1], a[2], a[3]};
    near[1] = side ? f32x4{a[2], b[2], a[3], b[3]} : f32x4{a[4], a[5], a[6], a[7]};
    far[0] = side ? f32x4{a[4], b[4], a[5], b[5]} : f32x4{b[0], b[1], b[2], b[3]};
    far[1] = side ? f32x4{a[6], b[6], a[7], b[7]} : f32x4{b[4], b[5], b[6], b[7]};
  } else {
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      const PairDims d = pair_dims(8 * lot.u + i, r.dims, r.interleaved);
      row[d.first] = a[i];
      row[d.second] = b[i];
    }
  }
}

// The rotation of a span: the first loads of keys and of AHEAD heads of queries are
// on their way before their turns are known.  (14006 tokens of 32 and 8 heads, an
// earlier state: queries in 64 bits 78 us, in 32 76; heads of a span side by side in
// the grid 72.)
template <int D, uint32_t T, uint32_t AHEAD>
struct Rotation {
  const KvRotateArgs &a;
  const Span &s;
  uint32_t head;  // key/value head
  Lot lot;
  bool k_runs, q_runs;
  RawPairs key, query[AHEAD];

  __device__ __forceinline__ Rotation(const KvRotateArgs &args, const Span &span, uint32_t kvh,
                                      bool keys, bool any)
      : a(args), s(span), head(kvh), lot(lot_of<D, T>(span)) {
    const bool runs = a.rotary.interleaved || a.rotary.dims % 16 == 0;
    k_runs = runs && a.append.vec;
    q_runs = runs && a.q_vec;
    if (!any) {
      return;
    }
    if (keys && lot.head == 0) {
      key = load_pairs(a.append.k + row() * a.append.k_row + head * a.append.k_head, a.rotary,
                       lot.u, k_runs);
    }
    load_queries(lot.head);
  }
  __device__ __forceinline__ uint64_t row() const { return uint64_t(s.row0 + lot.t); }
  __device__ __forceinline__ uint64_t query_head(uint32_t h) const { return head * a.group + h; }
  __device__ __forceinline__ void load_queries(uint32_t h) {
#pragma unroll
    for (uint32_t i = 0; i < AHEAD; ++i, h += lot.step) {
      if (lot.head != kNoHead && h < a.group) {
        query[i] = load_pairs(a.q + row() * a.q_row + query_head(h) * a.q_head, a.rotary, lot.u,
                              q_runs);
      }
    }
  }
  // Turns by way of `turns` in LDS; keys (if the span has any) to `keys`, which may
  // lie in the same place.
  __device__ __forceinline__ QueryTurns8 turn_keys(SpanTurns<D, T> *turns, KeyImage<D, T> *keys) {
    span_turns<D, T>(a.rotary, s, turns);
    __syncthreads();
    const Turns8 v = load_turns<D, T>(*turns, a.rotary, lot);
    __syncthreads();
    if (keys != nullptr && lot.head == 0) {
      rotate_key<D, T>(keys, key, a.rotary, v, lot, k_runs);
    }
    __syncthreads();
    QueryTurns8 q;
    q.live = v.live;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      q.c[i] = float(v.w[i].c);
      q.s[i] = float(v.w[i].s);
    }
    return q;
  }
  __device__ __forceinline__ void turn_queries(const QueryTurns8 &v) {
    for (uint32_t h = lot.head; lot.head != kNoHead && h < a.group;) {
#pragma unroll
      for (uint32_t i = 0; i < AHEAD; ++i, h += lot.step) {
        if (h < a.group) {
          rotate_query(a.q_out + row() * a.out_row + query_head(h) * a.out_head, query[i],
                       a.rotary, v, lot.u, q_runs);
        }
      }
      load_queries(h);
    }
  }
};
// The same of a span so short that each pair of a row has a thread: a thread makes
// its turn itself and rotates one pair of each row (the key's first, if there are
// `keys`, then the queries').  A token then takes a tenth of the instructions in a
// row that a thread with eight pairs has: what a single token waits for.
template <int D, uint32_t THREADS>
constexpr uint32_t kFewTokens = THREADS / (D / 2);  // most tokens of such a span
template <int D, uint32_t THREADS, uint32_t T>
__device__ __forceinline__ void rotate_pairs(const KvRotateArgs &a, const Span &s, uint32_t head,
                                             KeyImage<D, T> *keys) {
  const uint32_t n = (s.hi - s.lo) * (D / 2), step = THREADS / n;
  const uint32_t lot = threadIdx.x / n, i = threadIdx.x % n;
  const uint32_t t = i / (D / 2), j = i % (D / 2);  // the span's token t, pair j
  uint32_t m = lot < step ? lot : kNoHead;  // row 0: the key
  if (keys == nullptr && m == 0) {
    m = step;
  }
  const PairDims d = pair_dims(j, a.rotary.dims, a.rotary.interleaved);
  const uint64_t row = uint64_t(s.row0 + s.lo + t);
  uint32_t x = 0, y = 0;
  const auto load = [&] {
    if (m <= a.group) {
      const uint16_t *from = m == 0 ? a.append.k + row * a.append.k_row + head * a.append.k_head
                                    : a.q + row * a.q_row +
                                          (uint64_t(head) * a.group + m - 1) * a.q_head;
      x = from[d.first];
      y = from[d.second];
    }
  };
  load();
  const bool live = j < a.rotary.dims / 2;
  Turn w = {1.0, 0.0};
  if (live) {
    const PairTurns p = pair_turns(a.rotary, s, j);
    w = turn_of(place_of(p, s, s.lo + t), p.f);
  }
  const float c = float(w.c), sn = float(w.s);
  while (m <= a.group) {
    const float u = bits_f32(x << 16), v = bits_f32(y << 16);
    if (m == 0) {
      keys->x[t][d.first] = live ? to_odd(fma(double(u), w.c, -(double(v) * w.s))) : u;
      keys->x[t][d.second] = live ? to_odd(fma(double(v), w.c, double(u) * w.s)) : v;
    } else {
      uint16_t *to = a.q_out + row * a.out_row + (uint64_t(head) * a.group + m - 1) * a.out_head;
      to[d.first] = f32_to_bf16(live ? __builtin_fmaf(u, c, -(v * sn)) : u);
      to[d.second] = f32_to_bf16(live ? __builtin_fmaf(v, c, u * sn) : v);
    }
    m += step;
    load();
  }
  __syncthreads();
}
// A span's keys (if it has any) to an image in `lds` that `store` takes them from,
// and its queries to memory: before that or after it, as the caller's workgroups are
// served best.  In 4 bits two heads ahead and before (14006 tokens of 32 and 8 heads
// with the gather 76 us, 7300 of 28 and 4 of 64 dims with positions of three axes 24;
// after it 77 and 26, four heads ahead and after it 79 and 24); in 8, whose exponents
// cost more barriers, four and after (82 us; two and before 86, two and after 84).
template <int D, uint32_t T, uint32_t AHEAD, bool AFTER, typename F>
__device__ __forceinline__ void rotate_span(const KvRotateArgs &a, const Span &s, uint32_t head,
                                            uint8_t *lds, bool has_keys, F store) {
  KeyImage<D, T> *const keys = has_keys ? reinterpret_cast<KeyImage<D, T> *>(lds) : nullptr;
  const bool few = s.hi - s.lo <= kFewTokens<D, kSpanThreads<D, T>>;
  Rotation<D, T, AHEAD> r(a, s, head, has_keys, !few);
  QueryTurns8 v{};
  if (few) {
    rotate_pairs<D, kSpanThreads<D, T>>(a, s, head, keys);
  } else {
    v = r.turn_keys(reinterpret_cast<SpanTurns<D, T> *>(lds), keys);
  }
  if (!AFTER && !few) {
    r.turn_queries(v);
  }
  if (has_keys) {
    store();
  }
  if (AFTER && !few) {
    r.turn_queries(v);
  }
}
// Sixteen elements of a rotated row.
template <int D, uint32_t T>
__device__ __forceinline__ void read_row(const KeyImage<D, T> &keys, uint32_t row, uint32_t c,
                                         float (&k)[16]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const f32x4 w = *reinterpret_cast<const f32x4 *>(&keys.x[row][c * 16 + 4 * j]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      k[4 * j + e] = w[e];
    }
  }
}
constexpr size_t larger(size_t a, size_t b) { return a > b ? a : b; }

// What an append rotates: nothing, spans of any size, or such as kFewTokens names.
enum Turning { kTurnNone, kTurnAny, kTurnFew };

// --------------------------------------------------------------- append, 4 bits

// One workgroup stores the new tokens among 32 of one head, and rotates the
// queries of its group.  A thread has the same eight pairs of the same token in
// all heads, so that it reads their turns once.  Keys go from memory, or rotated
// from LDS, to their codes and memory; values' codes are brought into dwords of
// eight tokens in LDS.  A dword that new tokens share with earlier ones is read
// and written by this workgroup alone.
//
// What bounds it: with many tokens the memory (32768 tokens of 8 heads of 128,
// nothing rotated, 35 us: 4.8 TB/s; 14006 with 32 heads of queries 65 us: 4.6; with
// 7300 of 28 and 4 heads of 64, 20 us, each workgroup's chain of loads, all of them
// running at once); with few the chain alone (one token 4.5 us, rotated 5.2).
template <int D, Turning MODE>
__global__ __launch_bounds__(kThreads) void append4_kernel(KvRotateArgs ra, uint32_t each_slots) {
  using Chunk = Kv4Chunk<D>;
  using Image = KeyImage<D, MODE == kTurnFew ? kFewTokens<D, kThreads> : 32>;
  constexpr uint32_t kUnits = D / 16, kPitch = D + 16;
  static_assert(kSpanThreads<D, 32> == kThreads, "a thread for each unit");
  // Turns, and when all threads have theirs, keys and values.
  constexpr uint32_t kImage = MODE != kTurnNone ? sizeof(Image) : 0;
  __shared__ __align__(16) uint8_t
      lds[larger(MODE == kTurnAny ? sizeof(SpanTurns<D, 32>) : 0, kImage + 32 * kPitch)];
  uint8_t *const values = lds + kImage;  // a code to a byte
  const KvAppendArgs &a = ra.append;
  const uint32_t head = blockIdx.x % a.pool.heads, tid = threadIdx.x;
  const KvSlot slot = kv_find_slot(a.seqs, blockIdx.x / a.pool.heads, 1, 32, 2, each_slots);
  Span s;
  if (slot.seq >= a.seqs.batch ||
      !span_of<32>(slot, kv_length(a.seqs, a.pool.shift, slot.seq), &s)) {
    return;
  }
  // Places before the first token have no block, but queries.
  const int32_t id = s.base < 0 ? -1
                                : kv_block(a.seqs.tables + slot.seq * a.seqs.stride, a.seqs,
                                           a.pool.blocks, uint32_t(s.base) >> a.pool.shift);
  // This thread's unit, of at most 256: token t, dims 16c .. 16c + 15.
  const uint32_t t = s.lo + tid / kUnits, c = tid % kUnits;
  const bool live = t < s.hi && id >= 0;
  const uint64_t row = uint64_t(s.row0 + (live ? t : s.lo));
  const Bf16x16 raw_value = load16(a.v + head * a.v_head + row * a.v_row + c * 16, a.vec);
  const uint32_t in_block = uint32_t(s.base) & ((1u << a.pool.shift) - 1);
  const uint64_t unit = uint64_t(id < 0 ? 0 : id) * a.pool.heads + head;
  uint8_t *const chunk = kv4_chunk<D>(a.pool, unit, in_block);
  // At the end a thread has two dwords of a lane's four: dims d and d + 16 of the
  // eight tokens of group g.  What they hold is on its way from here.
  const uint32_t g = tid / (D / 2), d = tid % (D / 2) / 16 * 32 + tid % 16;
  u32x2 *const value_at =
      reinterpret_cast<u32x2 *>(chunk + Chunk::kSide + kv4_value_dword(g % 4, d));
  uint32_t fresh = 0;  // nibbles of new tokens
#pragma unroll
  for (uint32_t j = 0; j < 8; ++j) {
    const uint32_t of = 4 * g + j % 4 + 16 * (j / 4);
    fresh |= g < 4 && of >= s.lo && of < s.hi ? 15u << (4 * j) : 0u;
  }
  u32x2 held = {0u, 0u};
  if (fresh != 0 && fresh != ~0u) {
    held = *value_at;
  }
  const auto store = [&] {
    float k[16], v[16];
    if constexpr (MODE == kTurnNone) {
      unpack16(load16(a.k + head * a.k_head + row * a.k_row + c * 16, a.vec), k);
    } else if (live) {
      read_row(*reinterpret_cast<const Image *>(lds), t - s.lo, c, k);
    }
    if (live) {
      unpack16(raw_value, v);
      const uint32_t e = key_exp4(largest16<2>(k));
      *reinterpret_cast<u32x2 *>(chunk + kv4_key_byte<D>(t, c * 16)) = encode4(k, exp4_power(e));
      if (c % 2 == 0) {
        chunk[Chunk::kExps + kv4_exp_byte(t, c * 16)] = uint8_t(e);
      }
      const uint32_t top = largest16<kUnits>(v);
      const float scale = value_scale4(bits_f32(top));
      const u32x2 w = encode4_scaled(v, scale);
      u32x4 bytes;
#pragma unroll
      for (int j = 0; j < 4; ++j) {  // four codes of w to four bytes
        const uint32_t h = w[j / 2] >> (16 * (j % 2)) & 0xffffu;
        const uint32_t b = (h | h << 8) & 0x00ff00ffu;
        bytes[j] = (b | b << 4) & 0x0f0f0f0fu;
      }
      *reinterpret_cast<u32x4 *>(values + t * kPitch + c * 16) = bytes;
      if (c == 0) {
        *reinterpret_cast<uint16_t *>(chunk + Chunk::kScales + kv4_scale_byte(t)) =
            top >= 0x7f800000u ? uint16_t(0x7e00) : f32_to_f16(scale);
      }
    }
    __syncthreads();
    if (fresh != 0) {
      u32x2 w = {held.x & ~fresh, held.y & ~fresh};
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) {
        const uint8_t *from = values + (4 * g + j % 4 + 16 * (j / 4)) * kPitch + d;
        const bool is_new = (fresh >> (4 * j) & 1u) != 0;
        w.x |= (is_new ? from[0] : 0u) << (4 * j);
        w.y |= (is_new ? from[16] : 0u) << (4 * j);
      }
      *value_at = w;
    }
    if (a.pool.weights != nullptr) {
      for (uint32_t i = s.lo + tid; i < s.hi; i += kThreads) {
        a.pool.weights[(unit << a.pool.shift) + in_block + i] =
            a.weights != nullptr ? a.weights[uint64_t(s.row0 + i) * a.pool.heads + head] : 0.f;
      }
    }
  };
  if constexpr (MODE == kTurnAny) {
    rotate_span<D, 32, 2, false>(ra, s, head, lds, id >= 0, store);
  } else {
    if constexpr (MODE == kTurnFew) {
      rotate_pairs<D, kThreads>(ra, s, head, id >= 0 ? reinterpret_cast<Image *>(lds) : nullptr);
    }
    if (id >= 0) {
      store();
    }
  }
}

// ------------------------------------------------------- append, 8 bits, rotated

// One workgroup stores the new tokens of one block and head, as append_kernel
// does, with keys that come rotated from LDS, and rotates the queries of its
// group: a thread has one unit of 16 dims of the block.  Bound as append4_kernel is,
// with fewer workgroups at once (turns of a whole block in LDS): 14006 tokens of 32
// and 8 heads 70 us in blocks of 32, 69 to 75 of 64 (4.5 TB/s), 88 of 128 (one
// workgroup to a compute unit); one token 5.4.
template <int D, uint32_t bt, bool FEW>
struct Append8 {
  static constexpr uint32_t kAll = FEW ? kThreads : kSpanThreads<D, bt>;
  using Image = KeyImage<D, FEW ? kFewTokens<D, kThreads> : bt>;
  static constexpr size_t kLds =
      larger(larger(FEW ? 0 : sizeof(SpanTurns<D, bt>), sizeof(Image)), bt * D);
};
template <int D, uint32_t bt, bool FEW>
__global__ __launch_bounds__((Append8<D, bt, FEW>::kAll)) void append8_rotary_kernel(
    KvRotateArgs ra, uint32_t each_slots) {
  using Image = typename Append8<D, bt, FEW>::Image;
  constexpr uint32_t kUnits = D / 16, kAll = Append8<D, bt, FEW>::kAll;
  // Turns, and when all threads have theirs, rotated keys; at the end values.
  extern __shared__ __align__(16) uint8_t append8_lds[];
  Image *const rotated = reinterpret_cast<Image *>(append8_lds);
  const KvAppendArgs &a = ra.append;
  const uint32_t head = blockIdx.x % a.pool.heads, tid = threadIdx.x;
  const KvSlot slot = kv_find_slot(a.seqs, blockIdx.x / a.pool.heads, 1, bt, 2, each_slots);
  Span s;
  if (slot.seq >= a.seqs.batch ||
      !span_of<bt>(slot, kv_length(a.seqs, a.pool.shift, slot.seq), &s)) {
    return;
  }
  const int32_t id = s.base < 0 ? -1
                                : kv_block(a.seqs.tables + slot.seq * a.seqs.stride, a.seqs,
                                           a.pool.blocks, uint32_t(s.base) >> a.pool.shift);
  const uint64_t unit = uint64_t(id < 0 ? 0 : id) * a.pool.heads + head;
  const int ek0 = a.pool.exps[unit * 2], ev0 = a.pool.exps[unit * 2 + 1];
  // This thread's unit: token t, dims 16c .. 16c + 15.
  const uint32_t t = s.lo + tid / kUnits, c = tid % kUnits;
  const bool live = t < s.hi && id >= 0;
  Bf16x16 y[1] = {};
  if (live) {
    y[0] = load16(a.v + head * a.v_head + uint64_t(s.row0 + t) * a.v_row + c * 16, a.vec);
  }
  const auto store = [&] {
    float x[16];
    uint32_t ak = 0, av = largest_magnitude(y);
    if (live) {
      read_row(*rotated, t - s.lo, c, x);
#pragma unroll
      for (int i = 0; i < 16; ++i) {  // infinities and NaN do not count
        const uint32_t m = f32_bits(x[i]) & 0x7fffffffu;
        ak = max(ak, m < 0x7f800000u ? m : 0u);
      }
    }
    block_umax2<kAll>(ak, av);
    int ek = exponent_for_f32(ak), ev = exponent_for(av);
    float fk = 1.f, fv = 1.f;  // factor of the codes that were there
    if (s.lo > 0) {
      ek = max(ek, ek0);
      ev = max(ev, ev0);
      fk = exp2_int(max(ek0 - ek, -126));
      fv = exp2_int(max(ev0 - ev, -126));
    }
    if (tid == 0) {  // all have read the old ones
      a.pool.exps[unit * 2] = int8_t(ek);
      a.pool.exps[unit * 2 + 1] = int8_t(ev);
    }
    uint8_t *kc = a.pool.codes + unit * (uint64_t(2 * D) << a.pool.shift);
    uint8_t *vc = kc + (uint64_t(D) << a.pool.shift);
    rescale_keys<D, kAll>(kc, s.lo, fk);
    if (live) {
      *reinterpret_cast<u32x4 *>(kc + kv_key_unit<D>(t, c)) = encode16(x, ek);
      place_value<D>(append8_lds, t, c, encode16(y[0], ev));
    }
    __syncthreads();
    store_values<D, kAll>(append8_lds, vc, s.lo, s.hi, fv);
    if (a.pool.weights != nullptr) {
      for (uint32_t i = s.lo + tid; i < s.hi; i += kAll) {
        a.pool.weights[(unit << a.pool.shift) + i] =
            a.weights != nullptr ? a.weights[uint64_t(s.row0 + i) * a.pool.heads + head] : 0.f;
      }
    }
  };
  if constexpr (FEW) {
    rotate_pairs<D, kThreads>(ra, s, head, id >= 0 ? rotated : nullptr);
    if (id >= 0) {
      store();
    }
  } else {
    rotate_span<D, bt, 4, true>(ra, s, head, append8_lds, id >= 0, store);
  }
}

// ------------------------------------------------------------------- gather

// One workgroup reads 32 tokens of one head; values are brought into rows in
// LDS, a code to a byte.  Bound by its writes, four times what it reads (14006
// tokens of 8 heads of 128 16 us: 4.5 TB/s), and by the chain of loads where tokens
// are few (64 sequences of one: 6.4).
template <int D>
__global__ __launch_bounds__(kThreads) void gather4_kernel(KvGatherArgs a, uint32_t each_slots) {
  using Chunk = Kv4Chunk<D>;
  constexpr uint32_t kUnits = D / 16, kPitch = D + 16;
  __shared__ __align__(16) uint8_t values[32 * kPitch];
  const uint32_t head = blockIdx.y, tid = threadIdx.x;
  const KvSlot slot = kv_find_slot(a.seqs, blockIdx.x, 1, 32, 2, each_slots);
  if (slot.seq >= a.seqs.batch) {
    return;
  }
  const KvRows rows = slot.rows;
  const uint32_t length = kv_length(a.seqs, a.pool.shift, slot.seq);
  const int64_t origin = int64_t(length) - rows.count;  // place of the first row
  const int64_t base = (origin >> 5) * 32 + int64_t(slot.local) * 32;
  const uint32_t lo = origin > base ? uint32_t(origin - base) : 0u;  // tokens lo .. hi - 1
  const uint32_t hi = uint32_t(min(max(length - base, int64_t(0)), int64_t(32)));
  if (lo >= hi) {
    return;
  }
  // Rows before the first token, and those of no block, are zeros.
  const int32_t id = base < 0 ? -1
                              : kv_block(a.seqs.tables + slot.seq * a.seqs.stride, a.seqs,
                                         a.pool.blocks, uint32_t(base) >> a.pool.shift);
  const uint32_t in_block = uint32_t(base) & ((1u << a.pool.shift) - 1);
  const uint64_t unit = uint64_t(id < 0 ? 0 : id) * a.pool.heads + head;
  const uint8_t *chunk = kv4_chunk<D>(a.pool, unit, in_block);
  const int64_t row0 = int64_t(rows.first) + (base - origin);
  if (a.v != nullptr) {
    // Unit i: a lane's 16 bytes, dims d + 16 * 0 .. 3 of eight tokens.
    for (uint32_t i = tid; i < D; i += kThreads) {
      const uint32_t g = i % 64 / 16, d = i / 64 * 64 + i % 16;
      const u32x4 w = *reinterpret_cast<const u32x4 *>(chunk + Chunk::kSide + i * 16);
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) {
        uint8_t *to = values + (4 * g + j % 4 + 16 * (j / 4)) * kPitch + d;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          to[16 * n] = uint8_t(w[n] >> (4 * j) & 15u);
        }
      }
    }
    __syncthreads();
  }
  for (uint32_t i = tid; i < (hi - lo) * kUnits; i += kThreads) {
    const uint32_t t = lo + i / kUnits, c = i % kUnits;
    const uint64_t to = (uint64_t(row0 + t) * a.pool.heads + head) * D + c * 16;
    u32x4 o[2] = {};
    if (a.k != nullptr) {
      if (id >= 0) {
        const u32x2 w = *reinterpret_cast<const u32x2 *>(chunk + kv4_key_byte<D>(t, c * 16));
        const float power = exp4_power(chunk[Chunk::kExps + kv4_exp_byte(t, c * 16)]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          o[j] = __builtin_bit_cast(u32x4, codes4_to_bf16(w[j], power));
        }
      }
      reinterpret_cast<u32x4 *>(a.k + to)[0] = o[0];
      reinterpret_cast<u32x4 *>(a.k + to)[1] = o[1];
    }
    if (a.v != nullptr) {
      o[0] = o[1] = u32x4{};
      if (id >= 0) {
        const float s = f16_to_f32(
            *reinterpret_cast<const uint16_t *>(chunk + Chunk::kScales + kv4_scale_byte(t)));
        const u32x4 w = *reinterpret_cast<const u32x4 *>(values + t * kPitch + c * 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const u32x2 b = decode4_bytes(w[j], s);
          o[j / 2][j % 2 * 2] = b.x;
          o[j / 2][j % 2 * 2 + 1] = b.y;
        }
      }
      reinterpret_cast<u32x4 *>(a.v + to)[0] = o[0];
      reinterpret_cast<u32x4 *>(a.v + to)[1] = o[1];
    }
  }
  if (a.weights != nullptr && tid >= lo && tid < hi) {
    a.weights[uint64_t(row0 + tid) * a.pool.heads + head] =
        id < 0 ? 0.f : a.pool.weights[(unit << a.pool.shift) + in_block + tid];
  }
}

// -------------------------------------------------------------------- evict

// One workgroup fills 32 tokens of one head of the new tables with those that
// stay.  Tokens have their own scales, so codes move as they are: keys whole,
// of values' dwords a token's nibble to its new place among eight.  Bound by the
// chain of loads and by what the layout makes it read, a value's line for eight
// tokens (4096 of 32768 tokens of 8 heads 6.8 us, in 8 bits 13; 16 times 1536 of
// 4096 21, in 8 bits 36).
template <int D>
__global__ __launch_bounds__(kThreads) void evict4_move_kernel(KvEvictArgs a) {
  using Chunk = Kv4Chunk<D>;
  constexpr uint32_t kKeyBytes = D / 8;  // of a lane's run: 16, or 8 with 64 dims
  constexpr uint64_t kNone = ~uint64_t(0);
  __shared__ uint64_t from[32];   // offset of the token's chunk, kNone: it has no block
  __shared__ uint32_t place[32];  // its number there
  const uint32_t head = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const uint32_t base = blockIdx.x * 32;
  const uint32_t length = kv_length(a.seqs, a.pool.shift, b);
  const uint32_t stay = length < a.keep ? length : a.keep;
  const int32_t raw =
      base < stay ? a.new_tables[b * a.new_stride + (base >> a.pool.shift)] : -1;
  if (raw < 0 || uint32_t(raw) >= a.pool.blocks) {
    return;
  }
  const uint32_t n = min(stay - base, 32u), mask = (1u << a.pool.shift) - 1;
  const uint64_t dst = uint64_t(raw) * a.pool.heads + head;
  uint8_t *to = kv4_chunk<D>(a.pool, dst, base & mask);
  if (tid < 32) {
    uint64_t at = kNone;
    uint32_t t = 0;
    if (tid < n) {
      t = uint32_t(a.kept[(uint64_t(b) * a.pool.heads + head) * a.keep + base + tid]);
      const int32_t id = kv_block(a.seqs.tables + b * a.seqs.stride, a.seqs, a.pool.blocks,
                                  t >> a.pool.shift);
      float weight = 0.f;
      if (id >= 0) {
        const uint64_t src = uint64_t(id) * a.pool.heads + head;
        at = uint64_t(kv4_chunk<D>(a.pool, src, t & mask) - a.pool.codes);
        weight = a.pool.weights[(src << a.pool.shift) + (t & mask)];
      }
      a.pool.weights[(dst << a.pool.shift) + (base & mask) + tid] = weight;
    }
    from[tid] = at;
    place[tid] = t % 32;
    // A token of no block is zeros, as if appended.
    *reinterpret_cast<uint16_t *>(to + Chunk::kScales + kv4_scale_byte(tid)) =
        at != kNone ? *reinterpret_cast<const uint16_t *>(a.pool.codes + at + Chunk::kScales +
                                                          kv4_scale_byte(t % 32))
                    : f32_to_f16(kScaleLeast);
  }
  __syncthreads();
  if (tid < 128) {  // keys: token tid / 4, run g of four
    const uint32_t i = tid / 4, g = tid % 4;
    const uint64_t at = from[i];
    const uint32_t d = D / 4 * g;
    const uint8_t *src = a.pool.codes + (at != kNone ? at : 0);
    u32x4 w = {};
    uint8_t e = uint8_t(kKvExpMin + 127);
    if (at != kNone) {
      if constexpr (kKeyBytes == 16) {
        w = *reinterpret_cast<const u32x4 *>(src + kv4_key_byte<D>(place[i], d));
      } else {
        const u32x2 half = *reinterpret_cast<const u32x2 *>(src + kv4_key_byte<D>(place[i], d));
        w.x = half.x;
        w.y = half.y;
      }
      e = src[Chunk::kExps + kv4_exp_byte(place[i], d)];
    }
    if constexpr (kKeyBytes == 16) {
      *reinterpret_cast<u32x4 *>(to + kv4_key_byte<D>(i, d)) = w;
    } else {
      *reinterpret_cast<u32x2 *>(to + kv4_key_byte<D>(i, d)) = u32x2{w.x, w.y};
    }
    if (d % 32 == 0) {
      to[Chunk::kExps + kv4_exp_byte(i, d)] = e;
    }
  } else if (tid - 128 < D) {  // values: the 16 bytes of a lane for eight new tokens
    const uint32_t l = tid - 128, g = l % 64 / 16;
    u32x4 w = {};
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
      const uint32_t i = 4 * g + j % 4 + 16 * (j / 4), p = place[i];
      const uint64_t at = from[i];
      if (at != kNone) {
        const u32x4 x = *reinterpret_cast<const u32x4 *>(
            a.pool.codes + at + Chunk::kSide + l / 64 * 1024 +
            (l % 16 + 16 * kv4_value_group(p)) * 16);
        const uint32_t shift = 4 * kv4_value_slot(p);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          w[k] |= (x[k] >> shift & 15u) << (4 * j);
        }
      }
    }
    reinterpret_cast<u32x4 *>(to + Chunk::kSide)[l] = w;
  }
}

}  // namespace

// Slots that n rows of every sequence need: they touch at most (n + t - 2) / t + 1
// spans of t tokens.
static uint32_t each_slots(const KvSeqs &q, uint32_t t) {
  return q.each == 0 ? 1 : (q.each + t - 2) / t + 1;
}
// Workgroups: the heads of a span lie side by side, so that whole rows are on
// their way at a time.
static uint64_t append_grid(const KvAppendArgs &a, uint32_t t) {
  return kv_slots(a.seqs, 1, t, 2, each_slots(a.seqs, t)) * a.pool.heads;
}
uint64_t kv4_append_threads(const KvAppendArgs &a) { return append_grid(a, 32) * kThreads; }
// Whether a workgroup of kThreads has a thread for each pair of the rows that a
// sequence appends.  A kernel for such calls alone has half the registers and less
// LDS, so that more of it runs at once (32 and 8 heads of 128; 256 sequences of one
// token: 9.7 us against 11.2 in 4 bits, 10.6 against 18.6 in 8; 400 of four 28
// against 39, 30 against 66; a single one: level).
static bool few_each(const KvSeqs &q, uint32_t dim) {
  return q.each != 0 && q.each <= kThreads / (dim / 2);
}
uint64_t kv8_append_rotary_threads(const KvAppendArgs &a, uint32_t dim) {
  const uint32_t bt = 1u << a.pool.shift;
  return append_grid(a, bt) *
         (few_each(a.seqs, dim) ? kThreads : larger(bt * (dim / 16), kThreads));
}

hipError_t launch_kv4_append(const KvRotateArgs &a, uint32_t dim, hipStream_t s) {
  const uint32_t each = each_slots(a.append.seqs, 32), grid = uint32_t(append_grid(a.append, 32));
  const auto launch = [&](auto kernel) { kernel<<<grid, kThreads, 0, s>>>(a, each); };
  if (a.rotary.dims == 0) {
    launch(dim == 64 ? append4_kernel<64, kTurnNone> : append4_kernel<128, kTurnNone>);
  } else if (few_each(a.append.seqs, dim)) {
    launch(dim == 64 ? append4_kernel<64, kTurnFew> : append4_kernel<128, kTurnFew>);
  } else {
    launch(dim == 64 ? append4_kernel<64, kTurnAny> : append4_kernel<128, kTurnAny>);
  }
  return hipGetLastError();
}

template <int D, uint32_t bt, bool FEW>
static hipError_t launch_append8(const KvRotateArgs &a, hipStream_t s) {
  using Form = Append8<D, bt, FEW>;
  const uint32_t each = each_slots(a.append.seqs, bt), grid = uint32_t(append_grid(a.append, bt));
  const auto kernel = append8_rotary_kernel<D, bt, FEW>;
  if constexpr (Form::kLds > 32768) {
    const hipError_t e = raise_lds_limit(reinterpret_cast<const void *>(kernel), Form::kLds);
    if (e != hipSuccess) {
      return e;
    }
  }
  kernel<<<grid, Form::kAll, Form::kLds, s>>>(a, each);
  return hipGetLastError();
}
template <int D, uint32_t bt>
static hipError_t launch_append8(const KvRotateArgs &a, hipStream_t s) {
  return few_each(a.append.seqs, D) ? launch_append8<D, bt, true>(a, s)
                                    : launch_append8<D, bt, false>(a, s);
}
hipError_t launch_kv8_append_rotary(const KvRotateArgs &a, uint32_t dim, hipStream_t s) {
  switch (dim + a.append.pool.shift) {
    case 64 + 5: return launch_append8<64, 32>(a, s);
    case 64 + 6: return launch_append8<64, 64>(a, s);
    case 64 + 7: return launch_append8<64, 128>(a, s);
    case 128 + 5: return launch_append8<128, 32>(a, s);
    case 128 + 6: return launch_append8<128, 64>(a, s);
    default: return launch_append8<128, 128>(a, s);
  }
}

hipError_t launch_kv4_gather(const KvGatherArgs &a, uint32_t dim, hipStream_t s) {
  if (a.k == nullptr && a.v == nullptr) {
    launch_kv_gather_weights(a, s);
    return hipGetLastError();
  }
  const uint32_t each = each_slots(a.seqs, 32);
  const dim3 grid(uint32_t(kv_slots(a.seqs, 1, 32, 2, each)), a.pool.heads);
  if (dim == 64) {
    gather4_kernel<64><<<grid, kThreads, 0, s>>>(a, each);
  } else {
    gather4_kernel<128><<<grid, kThreads, 0, s>>>(a, each);
  }
  return hipGetLastError();
}

hipError_t launch_kv4_evict(const KvEvictArgs &a, uint32_t dim, hipStream_t s) {
  launch_kv_evict_select(a, s);
  const dim3 grid((a.keep + 31) / 32, a.pool.heads, a.seqs.batch);
  if (dim == 64) {
    evict4_move_kernel<64><<<grid, kThreads, 0, s>>>(a);
  } else {
    evict4_move_kernel<128><<<grid, kThreads, 0, s>>>(a);
  }
  return hipGetLastError();
}

}  // namespace ullm
