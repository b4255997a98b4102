// kv_store.hip -- what writes and moves the tokens of the 8-bit key/value
// cache: append, gather and evict.  All are bound by HBM and launches.
#include "kv_store.hpp"

namespace ullm {
namespace {

// One workgroup stores the new tokens of one block and head.  The new rows are
// read once, into registers; with their largest magnitudes the exponents are
// known.  Keys are written from there, values go through LDS, where a token's
// bytes take their places among the others' of a 16-byte unit.  Codes that
// were there are touched only when the exponent grows, or where they share a
// unit with a new one.  Bound by reading and writing: 12000 tokens of 8 heads
// 16 us, 4.6 TB/s (with 32-token blocks, whose workgroups have half the work
// for the same start, 18.6; a token encoded with 18 vector instructions per
// element instead of 4: 21; rows read twice and values two bytes at a time 33).
template <int D, uint32_t bt>
__global__ __launch_bounds__(kThreads) void append_kernel(KvAppendArgs a, uint32_t each_slots) {
  constexpr uint32_t kUnits = (bt * (D / 16) + kThreads - 1) / kThreads;  // of a thread
  __shared__ __align__(16) uint8_t image[bt * D];  // the block's values
  const uint32_t head = blockIdx.y, tid = threadIdx.x;
  const KvSlot slot = kv_find_slot(a.seqs, blockIdx.x, 1, bt, 2, each_slots);
  if (slot.seq >= a.seqs.batch) {
    return;
  }
  const KvRows rows = slot.rows;
  const uint32_t length = kv_length(a.seqs, a.pool.shift, slot.seq);
  const int64_t origin = int64_t(length) - rows.count;  // position of the first row
  const uint32_t first = origin < 0 ? 0u : uint32_t(origin);
  const uint32_t j = (first >> a.pool.shift) + slot.local;
  const uint32_t base = j << a.pool.shift;
  const uint32_t lo = first > base ? first - base : 0u;       // new tokens lo .. hi - 1
  const uint32_t hi = uint32_t(min(max(int64_t(length) - base, int64_t(0)), int64_t(bt)));
  if (j >= a.seqs.max_blocks || lo >= hi) {
    return;
  }
  const int32_t id = kv_block(a.seqs.tables + slot.seq * a.seqs.stride, a.seqs, a.pool.blocks, j);
  const uint64_t row0 = uint64_t(rows.first + (int64_t(base) - origin));  // row of token 0
  const uint16_t *k = a.k + head * a.k_head, *v = a.v + head * a.v_head;
  // Unit r of this thread: token t, dims 16c .. 16c + 15.
  const auto token = [&](uint32_t r) { return lo + (tid + r * kThreads) / (D / 16); };
  const uint32_t c = tid % (D / 16);
  Bf16x16 x[kUnits], y[kUnits];
#pragma unroll
  for (uint32_t r = 0; r < kUnits; ++r) {
    x[r] = Bf16x16{};
    y[r] = Bf16x16{};
    if (token(r) < hi) {
      const uint64_t row = row0 + token(r);
      x[r] = load16(k + row * a.k_row + c * 16, a.vec);
      y[r] = load16(v + row * a.v_row + c * 16, a.vec);
    }
  }
  if (id < 0) {
    return;
  }
  const uint64_t unit = uint64_t(id) * a.pool.heads + head;
  const int ek0 = a.pool.exps[unit * 2], ev0 = a.pool.exps[unit * 2 + 1];
  uint32_t ak = largest_magnitude(x), av = largest_magnitude(y);
  block_umax2(ak, av);
  int ek = exponent_for(ak), ev = exponent_for(av);
  float fk = 1.f, fv = 1.f;  // factor of the codes that were there
  if (lo > 0) {
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
  rescale_keys<D>(kc, lo, fk);
#pragma unroll
  for (uint32_t r = 0; r < kUnits; ++r) {
    const uint32_t t = token(r);
    if (t < hi) {
      *reinterpret_cast<u32x4 *>(kc + kv_key_unit<D>(t, c)) = encode16(x[r], ek);
      place_value<D>(image, t, c, encode16(y[r], ev));
    }
  }
  __syncthreads();
  store_values<D>(image, vc, lo, hi, fv);
  if (a.pool.weights != nullptr) {
    for (uint32_t t = lo + tid; t < hi; t += kThreads) {
      a.pool.weights[(unit << a.pool.shift) + t] =
          a.weights != nullptr ? a.weights[(row0 + t) * a.pool.heads + head] : 0.f;
    }
  }
}

// 16 codes as bf16, times a power of two: exact.
__device__ __forceinline__ void store_decoded(uint16_t *to, u32x4 w, float f) {
  u32x4 o[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    o[i / 2][i % 2 * 2] = __builtin_bit_cast(
        uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], f, false));
    o[i / 2][i % 2 * 2 + 1] = __builtin_bit_cast(
        uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], f, true));
  }
  reinterpret_cast<u32x4 *>(to)[0] = o[0];
  reinterpret_cast<u32x4 *>(to)[1] = o[1];
}

// One workgroup reads 32 tokens of one head, from a multiple of 32 on: 16
// bytes to a thread and load; values are brought into rows in LDS.  (12000
// tokens of 8 heads: 15 us, 4.9 TB/s; a workgroup for each row, which fetches all it
// needs to know for 4 KiB, 36.)
template <int D>
__global__ __launch_bounds__(kThreads) void gather_kernel(KvGatherArgs a, uint32_t each_slots) {
  constexpr uint32_t kUnits = 32 * (D / 16);  // of a side
  constexpr uint32_t kPitch = D + 16;
  __shared__ __align__(16) uint8_t values[32 * kPitch];
  const uint32_t head = blockIdx.y, tid = threadIdx.x;
  const KvSlot slot = kv_find_slot(a.seqs, blockIdx.x, 1, 32, 2, each_slots);
  if (slot.seq >= a.seqs.batch) {
    return;
  }
  const KvRows rows = slot.rows;
  const uint32_t length = kv_length(a.seqs, a.pool.shift, slot.seq);
  const int64_t origin = int64_t(length) - rows.count;  // position of the first row
  const int64_t base = (origin >> 5) * 32 + int64_t(slot.local) * 32;
  const uint32_t lo = origin > base ? uint32_t(origin - base) : 0u;  // tokens lo .. hi - 1
  const uint32_t hi = uint32_t(min(max(length - base, int64_t(0)), int64_t(32)));
  if (lo >= hi) {
    return;
  }
  // Rows before the first position, and those of no block, are zeros.
  const int32_t id = base < 0 ? -1
                              : kv_block(a.seqs.tables + slot.seq * a.seqs.stride, a.seqs,
                                         a.pool.blocks, uint32_t(base) >> a.pool.shift);
  const uint32_t in_block = uint32_t(base) & ((1u << a.pool.shift) - 1);
  const uint64_t unit = uint64_t(id < 0 ? 0 : id) * a.pool.heads + head;
  const int64_t row0 = int64_t(rows.first) + (base - origin);
  const uint8_t *keys =
      a.pool.codes + unit * (uint64_t(2 * D) << a.pool.shift) + uint64_t(in_block) * D;
  const uint8_t *side1 = keys + (uint64_t(D) << a.pool.shift);
  const float fk = exp2_int(a.pool.exps[unit * 2]), fv = exp2_int(a.pool.exps[unit * 2 + 1]);
  // Threads take the keys' units, then the values'.
  constexpr uint32_t kTurns = 2 * kUnits / kThreads;
  u32x4 w[kTurns];
#pragma unroll
  for (uint32_t r = 0; r < kTurns; ++r) {
    const uint32_t u = tid + r * kThreads;
    w[r] = u32x4{0u, 0u, 0u, 0u};
    if (id >= 0 && (u < kUnits ? a.k : a.v) != nullptr) {
      w[r] = u < kUnits ? *reinterpret_cast<const u32x4 *>(
                              keys + kv_key_unit<D>(u / (D / 16), u % (D / 16)))
                        : reinterpret_cast<const u32x4 *>(side1)[u - kUnits];
    }
  }
  const auto row_of = [&](uint16_t *to, uint32_t u) {
    return to + (uint64_t(row0 + u / (D / 16)) * a.pool.heads + head) * D + u % (D / 16) * 16;
  };
  const auto live = [&](uint32_t u) { return u / (D / 16) >= lo && u / (D / 16) < hi; };
#pragma unroll
  for (uint32_t r = 0; r < kTurns; ++r) {
    const uint32_t u = tid + r * kThreads;
    if (u < kUnits) {
      if (a.k != nullptr && live(u)) {
        store_decoded(row_of(a.k, u), w[r], fk);
      }
    } else {
      const uint32_t l = (u - kUnits) % 64, d = (u - kUnits) / 64 * 32 + l % 16;
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i) {
        values[value_token(l / 16, i % 8) * kPitch + d + 16 * (i / 8)] =
            uint8_t(w[r][i / 4] >> (8 * (i % 4)));
      }
    }
  }
  __syncthreads();
  if (a.v != nullptr) {
    for (uint32_t u = tid; u < kUnits; u += kThreads) {
      if (live(u)) {
        store_decoded(row_of(a.v, u),
                      *reinterpret_cast<const u32x4 *>(values + u / (D / 16) * kPitch +
                                                       u % (D / 16) * 16),
                      fv);
      }
    }
  }
  if (a.weights != nullptr && tid >= lo && tid < hi) {
    a.weights[uint64_t(row0 + tid) * a.pool.heads + head] =
        id < 0 ? 0.f : a.pool.weights[(unit << a.pool.shift) + in_block + tid];
  }
}

constexpr uint32_t kWeightRows = 128;

// Weights alone: one workgroup reads 128 rows of all heads.  (131072 tokens of
// 8 heads: 4.4 us; by the kernel above, whose workgroups fetch all they need to
// know for 128 bytes, 43.)
__global__ __launch_bounds__(kThreads) void gather_weights_kernel(KvGatherArgs a,
                                                                  uint32_t each_slots) {
  const KvSlot slot = kv_find_slot(a.seqs, blockIdx.x, 1, kWeightRows, 1, each_slots);
  if (slot.seq >= a.seqs.batch) {
    return;
  }
  const KvRows rows = slot.rows;
  const uint32_t first = slot.local * kWeightRows;
  if (first >= rows.count) {
    return;
  }
  const uint32_t n = min(rows.count - first, kWeightRows);
  const int64_t at =
      int64_t(kv_length(a.seqs, a.pool.shift, slot.seq)) - rows.count + first;
  const int32_t *table = a.seqs.tables + slot.seq * a.seqs.stride;
  float *to = a.weights + uint64_t(rows.first + first) * a.pool.heads;
  for (uint32_t u = threadIdx.x; u < n * a.pool.heads; u += kThreads) {
    const int64_t t = at + u / a.pool.heads;
    const int32_t id =
        t < 0 ? -1 : kv_block(table, a.seqs, a.pool.blocks, uint32_t(t) >> a.pool.shift);
    const uint64_t unit = uint64_t(id < 0 ? 0 : id) * a.pool.heads + u % a.pool.heads;
    const float w =
        a.pool.weights[(unit << a.pool.shift) + (uint32_t(t) & ((1u << a.pool.shift) - 1))];
    to[u] = id < 0 ? 0.f : w;
  }
}

// ------------------------------------------------------------------- evict

// A weight as an unsigned key of the same order, NaN above all, -0 as 0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  const uint32_t b = f32_bits(w + 0.f);  // -0 becomes 0
  const uint32_t key = b ^ (uint32_t(int32_t(b) >> 31) | 0x80000000u);
  return w != w ? 0xffffffffu : key;
}

constexpr uint32_t kSelectThreads = 1024, kSelectWaves = kSelectThreads / kWave;
constexpr uint32_t kSelectBins = 1u << kKvBinBits;

// Exclusive sums over the workgroup in the order of the threads; `sums`: one
// per wave.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t *sums) {
  const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  uint32_t upto = v;
#pragma unroll
  for (uint32_t off = 1; off < kWave; off <<= 1) {
    const uint32_t o = __shfl_up(upto, off, kWave);
    upto += lane >= off ? o : 0u;
  }
  if (lane == kWave - 1) {
    sums[wave] = upto;
  }
  __syncthreads();
#pragma unroll
  for (uint32_t w = 0; w < kSelectWaves; ++w) {
    upto += w < wave ? sums[w] : 0u;
  }
  return upto - v;
}

// One workgroup selects the tokens of one sequence and head.  A thread holds K
// keys in registers, 1024 K for the workgroup, so that a pass costs no memory.
// (ONE: the tables hold no more.  Longer sequences read theirs again, as many
// at a time, in each pass.)
//
// First the key of the last token that stays: the range of the keys in
// question, at first their smallest to their largest, is cut into 4096 bins,
// and the bin that it falls into is the next range, until all keys of a bin
// stay or they are equal.  Bins that follow the keys' own range keep the lanes
// of a wave on different counters, which fixed digits do not (weights share
// most of their exponent).  Then the positions, in order: a wave holds 64 K
// tokens on end and counts its own, the waves' counts are joined once.
//
// Bound by the instructions of a lone workgroup per head.  (32768 tokens of 8
// heads: 16 us; by bytes of the key, each pass reading the weights again, 128.)
template <uint32_t K, bool ONE>
__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(KvEvictArgs a) {
  constexpr uint32_t kSpan = K * kSelectThreads;
  __shared__ uint32_t hist[kSelectBins];
  __shared__ uint32_t sums[kSelectWaves], ties[kSelectWaves], pick[3], range[2];
  const uint32_t b = blockIdx.y, head = blockIdx.x, tid = threadIdx.x;
  const uint32_t lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const uint32_t length = kv_length(a.seqs, a.pool.shift, b);
  int32_t *kept = a.kept + (uint64_t(b) * a.pool.heads + head) * a.keep;
  const uint32_t stay = length < a.keep ? length : a.keep;
  if (head == 0 && tid == 0) {
    a.new_lengths[b] = int32_t(stay);
  }
  if (length <= a.keep) {
    for (uint32_t i = tid; i < a.keep; i += kSelectThreads) {
      kept[i] = i < length ? int32_t(i) : -1;
    }
    return;
  }
  const uint32_t lo = a.sink, hi = length - a.recent;  // candidates lo .. hi - 1
  uint32_t want = a.keep - a.sink - a.recent;
  for (uint32_t i = tid; i < a.sink + a.recent; i += kSelectThreads) {
    kept[i < lo ? i : i + want] = int32_t(i < lo ? i : i - lo + hi);
  }
  if (want == 0) {
    return;
  }
  const int32_t *table = a.seqs.tables + b * a.seqs.stride;
  const uint32_t mask = (1u << a.pool.shift) - 1;
  const uint32_t spans = ONE ? 1 : (length + kSpan - 1) / kSpan;
  const uint32_t mine = wave * K * kWave + lane;  // this thread's first token of a span

  uint32_t keys[K];
  // Keys of a span: 0 is no candidate, 1 a token of no block, which is less
  // than any weight.  Lane i looks up where the wave's 32 tokens from 32 i on
  // lie: two waits serve for all, and a key costs its load and little else.
  const auto load = [&](uint32_t span) __attribute__((always_inline)) {
    static_assert(2 * K <= kWave, "a lane for each 32 tokens");
    const uint32_t first = span * kSpan + wave * K * kWave;
    const uint32_t t32 = first + 32 * lane, block = t32 >> a.pool.shift;
    const uint32_t id = uint32_t(table[min(block, a.seqs.max_blocks - 1)]);
    const bool there = id < a.pool.blocks && block < a.seqs.max_blocks;
    const uint64_t at = (((there ? id : 0u) * uint64_t(a.pool.heads) + head) << a.pool.shift) +
                        (t32 & mask);
    const auto at_lane = [&](uint32_t from) {
      return uint64_t(uint32_t(__builtin_amdgcn_readlane(int(at >> 32), int(from)))) << 32 |
             uint32_t(__builtin_amdgcn_readlane(int(at), int(from)));
    };
    float w[K];
    if (a.pool.shift >= 6) {  // 64 tokens of a block at a time
#pragma unroll
      for (uint32_t k = 0; k < K; ++k) {
        w[k] = a.pool.weights[at_lane(2 * k) + lane];
      }
    } else {
#pragma unroll
      for (uint32_t k = 0; k < K; ++k) {
        const uint64_t low = at_lane(2 * k), high = at_lane(2 * k + 1);
        w[k] = a.pool.weights[(lane < 32 ? low : high) + lane % 32];
      }
    }
    const uint32_t from_lo = first + lane - lo, candidates = hi - lo;
#pragma unroll
    for (uint32_t k = 0; k < K; ++k) {
      keys[k] = from_lo + k * kWave < candidates ? weight_key(w[k]) : 0u;
    }
    if (__any(!there && lane < 2 * K && t32 < hi)) {
#pragma unroll
      for (uint32_t k = 0; k < K; ++k) {
        const bool none = __shfl(int(there), int(2 * k + lane / 32), kWave) == 0;
        keys[k] = none && keys[k] != 0u ? 1u : keys[k];
      }
    }
  };
  const auto each_span = [&](const auto &f) __attribute__((always_inline)) {
    for (uint32_t span = 0; span < spans; ++span) {
      if (!ONE) {
        load(span);
      }
      f(span);
    }
  };
  if (ONE) {
    load(0);
  }

  if (tid == 0) {
    range[0] = ~0u;
    range[1] = 0u;
  }
  __syncthreads();
  uint32_t least = ~0u, most = 0;
  each_span([&](uint32_t) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t k = 0; k < K; ++k) {
      least = min(least, keys[k] - 1u);  // no candidate: the largest
      most = max(most, keys[k]);
    }
  });
  least = ~wave_umax(~least);
  most = wave_umax(most);
  if (lane == 0) {
    atomicMin(&range[0], least);
    atomicMax(&range[1], most);
  }
  __syncthreads();
  KvKeyRange cut{range[0] + 1, range[1] - (range[0] + 1)};
  uint32_t last;  // tokens of keys above it stay, and of this one `want`
  for (;;) {
    last = cut.from;
    if (cut.width == 0) {
      break;
    }
    for (uint32_t i = tid; i < kSelectBins; i += kSelectThreads) {
      hist[i] = 0;
    }
    __syncthreads();
    const uint32_t shift = kv_bin_shift(cut);
    each_span([&](uint32_t) __attribute__((always_inline)) {
#pragma unroll
      for (uint32_t k = 0; k < K; ++k) {
        const uint32_t off = keys[k] - cut.from;
        if (off <= cut.width) {
          atomicAdd(&hist[kSelectBins - 1 - (off >> shift)], 1u);
        }
      }
    });
    __syncthreads();
    // The first bin, from the highest on, that reaches `want` keys.
    constexpr uint32_t kMine = kSelectBins / kSelectThreads;
    uint32_t n[kMine], sum = 0;
#pragma unroll
    for (uint32_t i = 0; i < kMine; ++i) {
      n[i] = hist[tid * kMine + i];
      sum += n[i];
    }
    uint32_t upto = block_scan(sum, sums);
#pragma unroll
    for (uint32_t i = 0; i < kMine; ++i) {
      if (upto < want && upto + n[i] >= want) {
        pick[0] = kSelectBins - 1 - (tid * kMine + i);
        pick[1] = want - upto;
        pick[2] = n[i];
      }
      upto += n[i];
    }
    __syncthreads();
    cut = kv_bin_keys(cut, shift, pick[0]);
    want = pick[1];
    if (want == pick[2]) {
      last = cut.from - 1;
      want = 0;
      break;
    }
  }

  // Lanes below this one among those of a mask, from `base` on.
  const auto rank = [](uint64_t lanes, uint32_t base) {
    return __builtin_amdgcn_mbcnt_hi(uint32_t(lanes >> 32),
                                     __builtin_amdgcn_mbcnt_lo(uint32_t(lanes), base));
  };
  uint32_t at = a.sink, equal = 0;  // where the next goes, tokens of key `last` so far
  each_span([&](uint32_t span) __attribute__((always_inline)) {
    uint32_t n = 0, m = 0;
#pragma unroll
    for (uint32_t k = 0; k < K; ++k) {
      n += uint32_t(__popcll(__ballot(keys[k] > last)));
    }
    if (want != 0) {
#pragma unroll
      for (uint32_t k = 0; k < K; ++k) {
        m += uint32_t(__popcll(__ballot(keys[k] == last)));
      }
    }
    __syncthreads();  // the sums of the last span are read
    if (lane == 0) {
      sums[wave] = n;
      ties[wave] = m;
    }
    __syncthreads();
    uint32_t next = at, same = equal;
#pragma unroll
    for (uint32_t w = 0; w < kSelectWaves; ++w) {
      next += w < wave ? sums[w] : 0u;
      same += w < wave ? ties[w] : 0u;
      at += sums[w];
      equal += ties[w];
    }
    const uint32_t t0 = span * kSpan + mine;
    if (want == 0) {
#pragma unroll
      for (uint32_t k = 0; k < K; ++k) {
        const uint64_t above = __ballot(keys[k] > last);
        if (keys[k] > last) {
          kept[rank(above, next)] = int32_t(t0 + k * kWave);
        }
        next += uint32_t(__popcll(above));
      }
    } else {
#pragma unroll
      for (uint32_t k = 0; k < K; ++k) {
        const uint64_t above = __ballot(keys[k] > last), tie = __ballot(keys[k] == last);
        const uint32_t before = rank(tie, same);
        if (keys[k] > last || (keys[k] == last && before < want)) {
          kept[rank(above, next) + min(before, want)] = int32_t(t0 + k * kWave);
        }
        next += uint32_t(__popcll(above));
        same += uint32_t(__popcll(tie));
      }
    }
  });
}

// Magnitudes of four codes without the sign, those of NaN as 0.
__device__ __forceinline__ uint32_t finite_codes(uint32_t w) {
  w &= 0x7f7f7f7fu;
  const uint32_t nan = (w + 0x01010101u) & 0x80808080u;
  return w & ~(nan - (nan >> 7));
}
// The largest of sixteen such magnitudes, two at a time.
__device__ __forceinline__ uint32_t largest_code(u32x4 w) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  u16x2 top = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t m = finite_codes(w[i]);
    top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, m & 0x00ff00ffu));
    top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, m >> 8 & 0x00ff00ffu));
  }
  return top[0] > top[1] ? top[0] : top[1];
}
// Factor of codes that go from one exponent to another.  Only codes of zero
// and NaN meet a difference past the clamp upwards.
__device__ __forceinline__ float code_factor(int from, int to) {
  const int by = from - to;
  return exp2_int(by < -126 ? -126 : by > 126 ? 126 : by);
}

// One workgroup fills one block and head of the new tables with the tokens
// that stay.  All codes are read once: the keys' 16 bytes stay in registers,
// and of the values' units, which a token shares with seven others, its two
// bytes go to their new places in LDS.  Then the exponents are known, and
// codes whose exponent does not change are written as they are.  Bound by what
// the layout makes it read: a value's cache line holds eight tokens' bytes, and
// where a third of the tokens stays nearly all lines are read.  (16 sequences
// to 1536 tokens of 8 heads: 42 us for 187 MB, 4.5 TB/s; with loads of single
// bytes, twice, 86.)
template <int D, uint32_t bt>
__global__ __launch_bounds__(kThreads) void evict_move_kernel(KvEvictArgs a) {
  constexpr uint32_t kKeyUnits = (bt * (D / 16) + kThreads - 1) / kThreads;  // of a thread
  constexpr uint32_t kLanes = D / 2;                                // of a token's values
  constexpr uint32_t kTokens = kThreads / kLanes, kAhead = 8;
  __shared__ __align__(16) uint8_t image[bt * D];  // the new block's values
  // Of each token: where its part of the keys' units starts (kNone: it has no
  // block), where that of the values' does, with its byte of the eight in the
  // low bits, and the exponents there.
  __shared__ uint64_t key_from[bt], value_from[bt];
  __shared__ int power[2][bt];
  __shared__ __align__(16) float factor[bt];
  constexpr uint64_t kNone = ~uint64_t(0);
  const uint32_t j = blockIdx.x, head = blockIdx.y, b = blockIdx.z;
  const uint32_t tid = threadIdx.x;
  const uint32_t base = j << a.pool.shift;
  // Loads that do not depend on each other first: the kernel is a chain of
  // them (position, block, exponents beside codes).
  const uint32_t place = base + tid < a.keep ? base + tid : base;
  const uint32_t t = uint32_t(a.kept[(uint64_t(b) * a.pool.heads + head) * a.keep + place]);
  const int32_t raw = a.new_tables[b * a.new_stride + j];
  const uint32_t length = kv_length(a.seqs, a.pool.shift, b);
  const uint32_t stay = length < a.keep ? length : a.keep;
  if (base >= stay || raw < 0 || uint32_t(raw) >= a.pool.blocks) {
    return;
  }
  const uint32_t n = stay - base < bt ? stay - base : bt, padded = (n + 31) / 32 * 32;
  const uint64_t dst = uint64_t(raw) * a.pool.heads + head;
  const uint64_t side = uint64_t(D) << a.pool.shift;
  int exp_key = 0, exp_value = 0;
  float weight = 0.f;
  if (tid < padded) {
    const int32_t id = tid < n ? kv_block(a.seqs.tables + b * a.seqs.stride, a.seqs,
                                          a.pool.blocks, t >> a.pool.shift)
                               : -1;
    const uint64_t src = uint64_t(id < 0 ? 0 : id) * a.pool.heads + head;
    const uint32_t at = t & (bt - 1);
    key_from[tid] = id < 0 ? kNone : src * 2 * side + kv_key_unit<D>(at, 0);
    value_from[tid] = src * 2 * side + side + kv_value_byte<D>(at, 0);
    exp_key = a.pool.exps[src * 2];
    exp_value = a.pool.exps[src * 2 + 1];
    if (id >= 0) {
      weight = a.pool.weights[(src << a.pool.shift) + at];
    }
  }
  __syncthreads();

  // Largest finite magnitudes, as f32 bits; a token of no block is zeros.
  uint32_t ak = 0, av = 0;
  const auto magnitude = [](uint32_t code, int e) {
    return f32_bits(__builtin_amdgcn_cvt_f32_fp8(int(code), 0) * exp2_int(e));
  };
  u32x4 keys[kKeyUnits];
#pragma unroll
  for (uint32_t r = 0; r < kKeyUnits; ++r) {
    const uint32_t u = tid + r * kThreads, i = u / (D / 16), c = u % (D / 16);
    keys[r] = u32x4{0u, 0u, 0u, 0u};
    if (i < n && key_from[i] != kNone) {
      keys[r] = *reinterpret_cast<const u32x4 *>(a.pool.codes + key_from[i] +
                                                 kv_key_unit<D>(0, c));
    }
  }
  const uint32_t vd = tid % kLanes / 16 * 32 + tid % 16;  // this lane's dims: vd, vd + 16
  u32x4 unit[kAhead];
  const auto load_values = [&](uint32_t i0) {
#pragma unroll
    for (uint32_t r = 0; r < kAhead; ++r) {
      const uint32_t i = i0 + r * kTokens + tid / kLanes;
      unit[r] = u32x4{0u, 0u, 0u, 0u};
      if (i < padded && key_from[i] != kNone) {
        unit[r] = *reinterpret_cast<const u32x4 *>(
            a.pool.codes + (value_from[i] & ~uint64_t(7)) + kv_value_byte<D>(0, vd));
      }
    }
  };
  load_values(0);
  if (tid < padded) {
    power[0][tid] = exp_key;
    power[1][tid] = exp_value;
  }
  __syncthreads();
  for (uint32_t i0 = 0; i0 < padded; i0 += kAhead * kTokens) {
    if (i0 != 0) {
      load_values(i0);
    }
#pragma unroll
    for (uint32_t r = 0; r < kAhead; ++r) {
      const uint32_t i = i0 + r * kTokens + tid / kLanes;
      if (i < padded) {
        // Its byte of each half, the others 0.
        const uint32_t pick = 0x0c0c0c00u | (uint32_t(value_from[i]) & 7u);
        const u32x4 w = unit[r];
        const uint32_t x = __builtin_amdgcn_perm(w.y, w.x, pick);
        const uint32_t y = __builtin_amdgcn_perm(w.w, w.z, pick);
        uint8_t *to = image + kv_value_byte<D>(i, vd);
        to[0] = uint8_t(x);
        to[8] = uint8_t(y);
        const uint32_t both = finite_codes(x | y << 8);
        av = max(av, magnitude(max(both & 0xffu, both >> 8), power[1][i]));
      }
    }
  }
#pragma unroll
  for (uint32_t r = 0; r < kKeyUnits; ++r) {
    const uint32_t i = (tid + r * kThreads) / (D / 16);
    if (i < n) {
      ak = max(ak, magnitude(largest_code(keys[r]), power[0][i]));
    }
  }
  block_umax2(ak, av);
  // Products of a code and a power of two are exact in bf16: their bits are
  // the upper half.
  const int ek = exponent_for(ak >> 16), ev = exponent_for(av >> 16);
  if (tid == 0) {
    a.pool.exps[dst * 2] = int8_t(ek);
    a.pool.exps[dst * 2 + 1] = int8_t(ev);
  }
  if (tid < padded) {
    factor[tid] = code_factor(power[1][tid], ev);
  }
  if (tid < n) {
    a.pool.weights[(dst << a.pool.shift) + tid] = weight;
  }
  uint8_t *to = a.pool.codes + dst * 2 * side;
#pragma unroll
  for (uint32_t r = 0; r < kKeyUnits; ++r) {
    const uint32_t u = tid + r * kThreads, i = u / (D / 16), c = u % (D / 16);
    if (i < n) {
      const float f = code_factor(power[0][i], ek);
      *reinterpret_cast<u32x4 *>(to + kv_key_unit<D>(i, c)) =
          f == 1.f ? keys[r] : rescale16(keys[r], f);
    }
  }
  __syncthreads();
  for (uint32_t u = tid; u < padded * (D / 16); u += kThreads) {
    // Unit u of the image: tokens t .. t + 3 and t + 16 .. t + 19.
    const uint32_t t = u / (2 * D) * 32 + u % 64 / 16 * 4;
    u32x4 w = reinterpret_cast<const u32x4 *>(image)[u];
    const f32x4 f0 = *reinterpret_cast<const f32x4 *>(factor + t);
    const f32x4 f1 = *reinterpret_cast<const f32x4 *>(factor + t + 16);
    bool same = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      same = same && f0[i] == 1.f && f1[i] == 1.f;
    }
    if (!same) {
      w.x = rescale4(w.x, f0);
      w.y = rescale4(w.y, f1);
      w.z = rescale4(w.z, f0);
      w.w = rescale4(w.w, f1);
    }
    reinterpret_cast<u32x4 *>(to + side)[u] = w;
  }
}

}  // namespace

hipError_t launch_kv_append(const KvAppendArgs &a, uint32_t dim, hipStream_t s) {
  const uint32_t bt = 1u << a.pool.shift;
  // A sequence's n rows touch at most (n + bt - 2) / bt + 1 blocks.
  const uint32_t each = a.seqs.each == 0 ? 1 : (a.seqs.each + bt - 2) / bt + 1;
  const dim3 grid(uint32_t(kv_slots(a.seqs, 1, bt, 2, each)), a.pool.heads);
  const auto launch = [&](auto kernel) { kernel<<<grid, kThreads, 0, s>>>(a, each); };
  if (dim == 64) {
    launch(bt == 32 ? append_kernel<64, 32> : bt == 64 ? append_kernel<64, 64>
                                                       : append_kernel<64, 128>);
  } else {
    launch(bt == 32 ? append_kernel<128, 32> : bt == 64 ? append_kernel<128, 64>
                                                        : append_kernel<128, 128>);
  }
  return hipGetLastError();
}

void launch_kv_gather_weights(const KvGatherArgs &a, hipStream_t s) {
  const uint32_t each = (a.seqs.each + kWeightRows - 1) / kWeightRows;
  gather_weights_kernel<<<uint32_t(kv_slots(a.seqs, 1, kWeightRows, 1, each)), kThreads, 0, s>>>(
      a, each);
}

hipError_t launch_kv_gather(const KvGatherArgs &a, uint32_t dim, hipStream_t s) {
  if (a.k == nullptr && a.v == nullptr) {
    launch_kv_gather_weights(a, s);
    return hipGetLastError();
  }
  const uint32_t each = a.seqs.each == 0 ? 1 : (a.seqs.each + 30) / 32 + 1;
  const dim3 grid(uint32_t(kv_slots(a.seqs, 1, 32, 2, each)), a.pool.heads);
  if (dim == 64) {
    gather_kernel<64><<<grid, kThreads, 0, s>>>(a, each);
  } else {
    gather_kernel<128><<<grid, kThreads, 0, s>>>(a, each);
  }
  return hipGetLastError();
}

void launch_kv_evict_select(const KvEvictArgs &a, hipStream_t s) {
  const dim3 units(a.pool.heads, a.seqs.batch);
  // Keys of a thread: what the tables' size needs.  (16 sequences of up to
  // 4500 tokens: 8 keys 9.5 us, 32 16, 32 read in spans 32; one of 32768: 16,
  // in spans 27.)
  const uint64_t tokens = uint64_t(a.seqs.max_blocks) << a.pool.shift;
  if (tokens <= 8 * kSelectThreads) {
    evict_select_kernel<8, true><<<units, kSelectThreads, 0, s>>>(a);
  } else if (tokens <= 32 * kSelectThreads) {
    evict_select_kernel<32, true><<<units, kSelectThreads, 0, s>>>(a);
  } else {
    evict_select_kernel<32, false><<<units, kSelectThreads, 0, s>>>(a);
  }
}

hipError_t launch_kv_evict(const KvEvictArgs &a, uint32_t dim, hipStream_t s) {
  const uint32_t bt = 1u << a.pool.shift;
  launch_kv_evict_select(a, s);
  const dim3 grid((a.keep + bt - 1) / bt, a.pool.heads, a.seqs.batch);
  const auto move = [&](auto kernel) { kernel<<<grid, kThreads, 0, s>>>(a); };
  if (dim == 64) {
    move(bt == 32 ? evict_move_kernel<64, 32> : bt == 64 ? evict_move_kernel<64, 64>
                                                         : evict_move_kernel<64, 128>);
  } else {
    move(bt == 32 ? evict_move_kernel<128, 32> : bt == 64 ? evict_move_kernel<128, 64>
                                                          : evict_move_kernel<128, 128>);
  }
  return hipGetLastError();
}

}  // namespace ullm
