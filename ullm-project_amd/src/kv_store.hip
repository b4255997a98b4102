// kv_store.hip -- what writes and moves the tokens of the 8-bit key/value
// cache: append, gather and evict.  All are bound by HBM and launches.
#include "kv_cache.hpp"

namespace ullm {
namespace {

constexpr uint32_t kThreads = 256;

// 16 bf16 of a row (two 16-byte loads, or 16 loads where rows are unaligned).
struct alignas(16) Bf16x16 {
  uint16_t v[16];
};
__device__ __forceinline__ Bf16x16 load16(const uint16_t *p, bool vec) {
  Bf16x16 r;
  if (vec) {
    u32x4 *o = reinterpret_cast<u32x4 *>(&r);
    o[0] = reinterpret_cast<const u32x4 *>(p)[0];
    o[1] = reinterpret_cast<const u32x4 *>(p)[1];
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      r.v[i] = p[i];
    }
  }
  return r;
}

// Magnitude bits of a bf16, 0 for infinities and NaN.
__device__ __forceinline__ uint32_t finite_magnitude(uint16_t h) {
  const uint32_t a = h & 0x7fffu;
  return a < 0x7f80u ? a : 0u;
}
// Smallest exponent e with a <= 448 * 2^e = 1.75 * 2^(e + 8), clamped, of
// magnitude bits of a bf16.
__device__ __forceinline__ int exponent_for(uint32_t a) {
  const int e = int(a >> 7) - 127 - 8 + ((a & 0x7fu) > 0x60u ? 1 : 0);
  return e < kKvExpMin ? kKvExpMin : e > kKvExpMax ? kKvExpMax : e;
}

// Four E4M3 codes of four f32, saturated to 448 (which only the largest
// exponent needs) and with NaN kept.
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  typedef short s16x2v __attribute__((ext_vector_type(2)));
  const auto clip = [](float x) { return x != x ? x : fminf(fmaxf(x, -448.f), 448.f); };
  s16x2v r = {0, 0};
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, clip(a), clip(b), 1.0f, false);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, clip(c), clip(d), 1.0f, true);
  return __builtin_bit_cast(uint32_t, r);
}
// A bf16 to encode, over 2^e: infinities become NaN.
__device__ __forceinline__ float scaled(uint16_t h, float inv) {
  return (h & 0x7f80u) == 0x7f80u ? __builtin_nanf("") : bf16_to_f32(h) * inv;
}
// Four codes times a power of two, rounded to codes again.
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float f) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), false);
  const f2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), true);
  return encode4(lo[0] * f, lo[1] * f, hi[0] * f, hi[1] * f);
}
__device__ __forceinline__ u32x4 rescale16(u32x4 w, float f) {
  return u32x4{rescale4(w.x, f), rescale4(w.y, f), rescale4(w.z, f), rescale4(w.w, f)};
}

__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const uint32_t o = __shfl_xor(v, off, kWave);
    v = o > v ? o : v;
  }
  return v;
}
// Maxima of two values over the workgroup.
__device__ __forceinline__ void block_umax2(uint32_t &a, uint32_t &b) {
  __shared__ uint32_t red[2][kThreads / kWave];
  a = wave_umax(a);
  b = wave_umax(b);
  if (threadIdx.x % kWave == 0) {
    red[0][threadIdx.x / kWave] = a;
    red[1][threadIdx.x / kWave] = b;
  }
  __syncthreads();
  for (uint32_t i = 0; i < kThreads / kWave; ++i) {
    a = red[0][i] > a ? red[0][i] : a;
    b = red[1][i] > b ? red[1][i] : b;
  }
  __syncthreads();
}

// Token j (0..7) of the 8 that lane group g of a 32-token value tile holds.
__device__ __forceinline__ uint32_t value_token(uint32_t g, uint32_t j) {
  return 4 * g + j % 4 + 16 * (j / 4);
}

// One workgroup stores the new tokens of one block and head.  It reads the
// new rows twice (the second time from L2): for the largest magnitude, then
// to encode them.  Codes that were there are touched only when the exponent
// grows, or where they share a 16-byte unit of values with a new one.
template <int D>
__global__ __launch_bounds__(kThreads) void append_kernel(KvAppendArgs a, uint32_t each_slots) {
  const uint32_t bt = 1u << a.pool.shift, head = blockIdx.y, tid = threadIdx.x;
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
  const uint32_t hi = length > base ? (length - base < bt ? length - base : bt) : 0u;
  if (j >= a.seqs.max_blocks || lo >= hi) {
    return;
  }
  const int32_t id = kv_block(a.seqs.tables + slot.seq * a.seqs.stride, a.seqs, a.pool.blocks, j);
  if (id < 0) {
    return;
  }
  const uint64_t unit = uint64_t(id) * a.pool.heads + head;
  const uint64_t row0 = uint64_t(rows.first + (int64_t(base) - origin));  // row of token 0
  const uint16_t *k = a.k + head * a.k_head, *v = a.v + head * a.v_head;

  uint32_t ak = 0, av = 0;
  for (uint32_t u = tid; u < (hi - lo) * (D / 16); u += kThreads) {
    const uint64_t row = row0 + lo + u / (D / 16);
    const uint32_t c = u % (D / 16) * 16;
    const Bf16x16 x = load16(k + row * a.k_row + c, a.vec);
    const Bf16x16 y = load16(v + row * a.v_row + c, a.vec);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      ak = max(ak, finite_magnitude(x.v[i]));
      av = max(av, finite_magnitude(y.v[i]));
    }
  }
  block_umax2(ak, av);
  int ek = exponent_for(ak), ev = exponent_for(av);
  float fk = 1.f, fv = 1.f;  // factor of the codes that were there
  if (lo > 0) {
    const int ek0 = a.pool.exps[unit * 2], ev0 = a.pool.exps[unit * 2 + 1];
    ek = max(ek, ek0);
    ev = max(ev, ev0);
    fk = exp2_int(max(ek0 - ek, -126));
    fv = exp2_int(max(ev0 - ev, -126));
  }
  __syncthreads();  // the old exponents are read
  if (tid == 0) {
    a.pool.exps[unit * 2] = int8_t(ek);
    a.pool.exps[unit * 2 + 1] = int8_t(ev);
  }
  const float ik = exp2_int(-ek), iv = exp2_int(-ev);
  uint8_t *kc = a.pool.codes + unit * (uint64_t(2 * D) << a.pool.shift);
  uint8_t *vc = kc + (uint64_t(D) << a.pool.shift);

  const uint32_t kfrom = fk != 1.f ? 0u : lo;
  for (uint32_t u = tid; u < (hi - kfrom) * (D / 16); u += kThreads) {
    const uint32_t t = kfrom + u / (D / 16), c = u % (D / 16);
    u32x4 *at = reinterpret_cast<u32x4 *>(kc + kv_key_unit<D>(t, c));
    if (t < lo) {
      *at = rescale16(*at, fk);
    } else {
      const Bf16x16 x = load16(k + (row0 + t) * a.k_row + c * 16, a.vec);
      u32x4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = encode4(scaled(x.v[4 * i], ik), scaled(x.v[4 * i + 1], ik),
                       scaled(x.v[4 * i + 2], ik), scaled(x.v[4 * i + 3], ik));
      }
      *at = w;
    }
  }

  // Units of 8 tokens x 2 dims, D / 2 of them for each lane group of 32 tokens.
  const uint32_t vfrom = fv != 1.f ? 0u : lo;
  const uint32_t s0 = vfrom / 32 * 4, s1 = (hi + 31) / 32 * 4;
  for (uint32_t u = tid; u < (s1 - s0) * (D / 2); u += kThreads) {
    const uint32_t set = s0 + u / (D / 2), r = u % (D / 2);
    const uint32_t t32 = set / 4 * 32, g = set % 4, d = r / 16 * 32 + r % 16;
    uint32_t fresh = 0;  // new tokens of the eight
    bool kept = false;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
      const uint32_t t = t32 + value_token(g, i);
      fresh |= t >= lo && t < hi ? 1u << i : 0u;
      kept = kept || t < lo;
    }
    if (fresh == 0 && (fv == 1.f || !kept)) {
      continue;
    }
    u32x4 *at = reinterpret_cast<u32x4 *>(vc + kv_value_byte<D>(t32 + 4 * g, d));
    u32x4 w = {0u, 0u, 0u, 0u};
    if (kept) {
      w = fv != 1.f ? rescale16(*at, fv) : *at;
    }
#pragma unroll
    for (uint32_t half = 0; half < 4; ++half) {  // dim d or d + 16, tokens 0..3 or 4..7
      const uint32_t dd = d + 16 * (half / 2), i0 = 4 * (half % 2);
      float x[4];
      uint32_t mask = 0;
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) {
        const bool is = (fresh >> (i0 + i)) & 1u;
        const uint64_t row = row0 + t32 + value_token(g, i0 + i);
        x[i] = is ? scaled(v[row * a.v_row + dd], iv) : 0.f;
        mask |= is ? 0xffu << (8 * i) : 0u;
      }
      const uint32_t now = encode4(x[0], x[1], x[2], x[3]);
      w[half] = (now & mask) | (w[half] & ~mask);
    }
    *at = w;
  }
  if (a.pool.weights != nullptr) {
    for (uint32_t t = lo + tid; t < hi; t += kThreads) {
      a.pool.weights[(unit << a.pool.shift) + t] =
          a.weights != nullptr ? a.weights[(row0 + t) * a.pool.heads + head] : 0.f;
    }
  }
}

// One workgroup reads one row: all heads of a token.
template <int D>
__global__ __launch_bounds__(kThreads) void gather_kernel(KvGatherArgs a) {
  const KvSlot slot = kv_find_slot(a.seqs, blockIdx.x, 1, 1, 0, a.seqs.each);
  if (slot.seq >= a.seqs.batch) {
    return;
  }
  const KvRows rows = slot.rows;
  if (slot.local >= rows.count) {
    return;
  }
  const uint64_t row = rows.first + slot.local;
  const int64_t at =
      int64_t(kv_length(a.seqs, a.pool.shift, slot.seq)) - rows.count + slot.local;
  const uint32_t t = uint32_t(at) & ((1u << a.pool.shift) - 1);
  const int32_t id = at < 0 ? -1
                            : kv_block(a.seqs.tables + slot.seq * a.seqs.stride, a.seqs,
                                       a.pool.blocks, uint32_t(at) >> a.pool.shift);
  const uint32_t per = D / 16;
  for (uint32_t u = threadIdx.x; u < a.pool.heads * per; u += kThreads) {
    const uint32_t head = u / per, c = u % per;
    const uint64_t unit = uint64_t(id < 0 ? 0 : id) * a.pool.heads + head;
    const uint8_t *codes = a.pool.codes + unit * (uint64_t(2 * D) << a.pool.shift);
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      uint16_t *to = side == 0 ? a.k : a.v;
      if (to == nullptr) {
        continue;
      }
      u32x4 w = {0u, 0u, 0u, 0u};
      float f = 1.f;
      if (id >= 0) {
        f = exp2_int(a.pool.exps[unit * 2 + side]);
        if (side == 0) {
          w = *reinterpret_cast<const u32x4 *>(codes + kv_key_unit<D>(t, c));
        } else {
          const uint8_t *vc = codes + (uint64_t(D) << a.pool.shift) + kv_value_byte<D>(t, c * 16);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            w[i / 4] |= uint32_t(vc[i * 16]) << (8 * (i % 4));
          }
        }
      }
      u32x4 o[2];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        typedef float f2 __attribute__((ext_vector_type(2)));
        const f2 x = __builtin_amdgcn_cvt_pk_f32_fp8(int(w[i]), false);
        const f2 y = __builtin_amdgcn_cvt_pk_f32_fp8(int(w[i]), true);
        o[i / 2][i % 2 * 2] = f32x2_to_bf16x2(x[0] * f, x[1] * f);
        o[i / 2][i % 2 * 2 + 1] = f32x2_to_bf16x2(y[0] * f, y[1] * f);
      }
      u32x4 *p = reinterpret_cast<u32x4 *>(to + (row * a.pool.heads + head) * D + c * 16);
      p[0] = o[0];
      p[1] = o[1];
    }
    if (a.weights != nullptr && c == 0) {
      a.weights[row * a.pool.heads + head] =
          id < 0 ? 0.f : a.pool.weights[(unit << a.pool.shift) + t];
    }
  }
}

// ------------------------------------------------------------------- evict

// A weight as an unsigned key of the same order, NaN above all, -0 as 0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  const uint32_t b = f32_bits(w);
  if ((b & 0x7fffffffu) > 0x7f800000u) {
    return 0xffffffffu;
  }
  return (b & 0x80000000u) ? (b == 0x80000000u ? 0x80000000u : ~b) : (b | 0x80000000u);
}

constexpr uint32_t kSelectThreads = 1024;

// One workgroup selects the tokens of one sequence and head: the key that the
// last selected token has, by its bytes from the highest (a histogram each),
// then the selected positions in order.
__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(KvEvictArgs a) {
  __shared__ uint32_t hist[256];
  __shared__ uint32_t pick[2];
  __shared__ uint32_t counts[2][kSelectThreads / kWave];
  const uint32_t b = blockIdx.y, head = blockIdx.x, tid = threadIdx.x;
  const uint32_t lane = tid % kWave, wave = tid / kWave;
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
  const int32_t *table = a.seqs.tables + b * a.seqs.stride;
  const uint32_t mask = (1u << a.pool.shift) - 1;
  const auto key_of = [&](uint32_t t) {
    const int32_t id = kv_block(table, a.seqs, a.pool.blocks, t >> a.pool.shift);
    return id < 0 ? 0u
                  : weight_key(a.pool.weights[((uint64_t(id) * a.pool.heads + head)
                                               << a.pool.shift) + (t & mask)]);
  };
  const uint32_t lo = a.sink, hi = length - a.recent;  // candidates lo .. hi - 1
  uint32_t want = a.keep - a.sink - a.recent;
  uint32_t prefix = 0;  // the bytes of the last selected key found so far
  if (want != 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (uint32_t i = tid; i < 256; i += kSelectThreads) {
        hist[i] = 0;
      }
      __syncthreads();
      for (uint32_t t = lo + tid; t < hi; t += kSelectThreads) {
        const uint32_t key = key_of(t);
        if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) {
          atomicAdd(&hist[(key >> shift) & 255u], 1u);
        }
      }
      __syncthreads();
      if (tid == 0) {
        uint32_t above = 0, bin = 255;
        while (above + hist[bin] < want) {  // the bins hold at least `want` keys
          above += hist[bin--];
        }
        pick[0] = bin;
        pick[1] = above;
      }
      __syncthreads();
      prefix |= pick[0] << shift;
      want -= pick[1];
      __syncthreads();
    }
  }
  // `want` tokens of key `prefix` stay, the lowest positions first.
  const bool none = a.keep == a.sink + a.recent;
  uint32_t done = 0, equal = 0;
  for (uint32_t t0 = 0; t0 < length; t0 += kSelectThreads) {
    const uint32_t t = t0 + tid;
    const bool free = t >= lo && t < hi;
    const uint32_t key = free && !none ? key_of(t) : 0u;
    const bool tie = free && !none && key == prefix;
    const uint64_t ties = __ballot(tie);
    const uint64_t below = (uint64_t(1) << lane) - 1;
    if (lane == 0) {
      counts[0][wave] = uint32_t(__popcll(ties));
    }
    __syncthreads();
    uint32_t rank = equal + uint32_t(__popcll(ties & below));
    for (uint32_t i = 0; i < kSelectThreads / kWave; ++i) {
      rank += i < wave ? counts[0][i] : 0u;
      equal += counts[0][i];
    }
    const bool stays =
        t < length && (!free || (!none && (key > prefix || (tie && rank < want))));
    const uint64_t all = __ballot(stays);
    if (lane == 0) {
      counts[1][wave] = uint32_t(__popcll(all));
    }
    __syncthreads();
    uint32_t at = done + uint32_t(__popcll(all & below));
    for (uint32_t i = 0; i < kSelectThreads / kWave; ++i) {
      at += i < wave ? counts[1][i] : 0u;
      done += counts[1][i];
    }
    if (stays && at < a.keep) {
      kept[at] = int32_t(t);
    }
  }
}

constexpr int kNoToken = -128;

// One workgroup fills one block and head of the new tables with the tokens
// that stay.
template <int D>
__global__ __launch_bounds__(kThreads) void evict_move_kernel(KvEvictArgs a) {
  __shared__ uint64_t from[128];   // byte offset of the token's block and head
  __shared__ uint32_t slot[128];   // its place in that block
  __shared__ int power[2][128];    // the exponents there, kNoToken: no block
  const uint32_t bt = 1u << a.pool.shift, j = blockIdx.x, head = blockIdx.y, b = blockIdx.z;
  const uint32_t tid = threadIdx.x;
  const uint32_t length = kv_length(a.seqs, a.pool.shift, b);
  const uint32_t stay = length < a.keep ? length : a.keep;
  const uint32_t base = j << a.pool.shift;
  if (base >= stay) {
    return;
  }
  const uint32_t n = stay - base < bt ? stay - base : bt;
  const int32_t raw = a.new_tables[b * a.new_stride + j];
  if (raw < 0 || uint32_t(raw) >= a.pool.blocks) {
    return;
  }
  const uint64_t dst = uint64_t(raw) * a.pool.heads + head;
  const int32_t *kept = a.kept + (uint64_t(b) * a.pool.heads + head) * a.keep + base;
  const int32_t *table = a.seqs.tables + b * a.seqs.stride;
  for (uint32_t i = tid; i < n; i += kThreads) {
    const uint32_t t = uint32_t(kept[i]);
    const int32_t id = kv_block(table, a.seqs, a.pool.blocks, t >> a.pool.shift);
    const uint64_t src = uint64_t(id < 0 ? 0 : id) * a.pool.heads + head;
    from[i] = src * (uint64_t(2 * D) << a.pool.shift);
    slot[i] = t & (bt - 1);
    power[0][i] = id < 0 ? kNoToken : int(a.pool.exps[src * 2]);
    power[1][i] = id < 0 ? kNoToken : int(a.pool.exps[src * 2 + 1]);
    if (a.pool.weights != nullptr) {
      a.pool.weights[(dst << a.pool.shift) + i] =
          id < 0 ? 0.f : a.pool.weights[(src << a.pool.shift) + slot[i]];
    }
  }
  __syncthreads();
  const uint64_t side = uint64_t(D) << a.pool.shift;
  // A token of no block is moved as zeros.
  const auto value = [](uint32_t code, int e) {
    return e == kNoToken ? 0.f : __builtin_amdgcn_cvt_f32_fp8(int(code), 0) * exp2_int(e);
  };
  // Largest finite magnitudes, as f32 bits.
  uint32_t ak = 0, av = 0;
  for (uint32_t u = tid; u < n * D; u += kThreads) {
    const uint32_t i = u / D, d = u % D;
    const uint8_t *src = a.pool.codes + from[i];
    const uint32_t ck = src[kv_key_unit<D>(slot[i], d / 16) + d % 16] & 0x7fu;
    const uint32_t cv = src[side + kv_value_byte<D>(slot[i], d)] & 0x7fu;
    ak = max(ak, ck == 0x7fu ? 0u : f32_bits(value(ck, power[0][i])));
    av = max(av, cv == 0x7fu ? 0u : f32_bits(value(cv, power[1][i])));
  }
  block_umax2(ak, av);
  // Products of a code and a power of two are exact in bf16: their bits are
  // the upper half.
  const int ek = exponent_for(ak >> 16), ev = exponent_for(av >> 16);
  if (tid == 0) {
    a.pool.exps[dst * 2] = int8_t(ek);
    a.pool.exps[dst * 2 + 1] = int8_t(ev);
  }
  const float iv = exp2_int(-ev);
  uint8_t *to = a.pool.codes + dst * 2 * side;
  for (uint32_t u = tid; u < n * (D / 16); u += kThreads) {
    const uint32_t i = u / (D / 16), c = u % (D / 16);
    const u32x4 w = *reinterpret_cast<const u32x4 *>(a.pool.codes + from[i] +
                                                     kv_key_unit<D>(slot[i], c));
    // Only codes of zero and NaN meet a difference past the clamp upwards.
    const int by = power[0][i] - ek;
    const float f = exp2_int(by < -126 ? -126 : by > 126 ? 126 : by);
    *reinterpret_cast<u32x4 *>(to + kv_key_unit<D>(i, c)) =
        power[0][i] == kNoToken ? u32x4{0u, 0u, 0u, 0u} : rescale16(w, f);
  }
  for (uint32_t u = tid; u < (n + 31) / 32 * 4 * (D / 2); u += kThreads) {
    const uint32_t set = u / (D / 2), r = u % (D / 2);
    const uint32_t t32 = set / 4 * 32, g = set % 4, d = r / 16 * 32 + r % 16;
    u32x4 w;
#pragma unroll
    for (uint32_t half = 0; half < 4; ++half) {
      const uint32_t dd = d + 16 * (half / 2), i0 = 4 * (half % 2);
      float x[4];
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t t = t32 + value_token(g, i0 + i);
        x[i] = 0.f;
        if (t < n) {
          const uint8_t code = a.pool.codes[from[t] + side + kv_value_byte<D>(slot[t], dd)];
          x[i] = value(code, power[1][t]) * iv;
        }
      }
      w[half] = encode4(x[0], x[1], x[2], x[3]);
    }
    *reinterpret_cast<u32x4 *>(to + side + kv_value_byte<D>(t32 + 4 * g, d)) = w;
  }
}

}  // namespace

hipError_t launch_kv_append(const KvAppendArgs &a, uint32_t dim, hipStream_t s) {
  const uint32_t bt = 1u << a.pool.shift;
  // A sequence's n rows touch at most (n + bt - 2) / bt + 1 blocks.
  const uint32_t each = a.seqs.each == 0 ? 1 : (a.seqs.each + bt - 2) / bt + 1;
  const dim3 grid(uint32_t(kv_slots(a.seqs, 1, bt, 2, each)), a.pool.heads);
  if (dim == 64) {
    append_kernel<64><<<grid, kThreads, 0, s>>>(a, each);
  } else {
    append_kernel<128><<<grid, kThreads, 0, s>>>(a, each);
  }
  return hipGetLastError();
}

hipError_t launch_kv_gather(const KvGatherArgs &a, uint32_t dim, hipStream_t s) {
  if (dim == 64) {
    gather_kernel<64><<<a.seqs.rows, kThreads, 0, s>>>(a);
  } else {
    gather_kernel<128><<<a.seqs.rows, kThreads, 0, s>>>(a);
  }
  return hipGetLastError();
}

hipError_t launch_kv_evict(const KvEvictArgs &a, uint32_t dim, hipStream_t s) {
  evict_select_kernel<<<dim3(a.pool.heads, a.seqs.batch), kSelectThreads, 0, s>>>(a);
  const uint32_t bt = 1u << a.pool.shift;
  const dim3 grid((a.keep + bt - 1) / bt, a.pool.heads, a.seqs.batch);
  if (dim == 64) {
    evict_move_kernel<64><<<grid, kThreads, 0, s>>>(a);
  } else {
    evict_move_kernel<128><<<grid, kThreads, 0, s>>>(a);
  }
  return hipGetLastError();
}

}  // namespace ullm
