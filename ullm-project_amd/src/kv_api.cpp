// kv_api.cpp -- C entry points of the 8-bit key/value cache.
//
// Validation order per entry, as in linear_api.cpp: sink, descriptor header
// (size, version), reserved words, handle, sizes and enums, pointers; only
// then is the device touched.  Block tables, lengths and row offsets are
// device memory and cannot be checked here: the kernels take them within
// their bounds.
#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <cmath>
#include <mutex>
#include <string>
#include <unordered_set>

#include "abi_common.hpp"
#include "host_common.hpp"
#include "kv_cache.hpp"

namespace {

using ullm::check_device;
using ullm::DeviceScope;
using ullm::hip_fail;
using ullm::write_error;
using ullm::write_errorf;

constexpr uint64_t kMaxCount = (uint64_t(1) << 31) - 1;
constexpr uint64_t kMaxGridYz = 65535;

std::mutex g_caches_mutex;
std::unordered_set<const ullm_kv_cache_t *> g_caches;

ullm_status_t lookup_cache(const ullm_kv_cache_t *c, ullm_error_sink_t *sink) {
  if (c == nullptr) {
    return write_error(sink, ULLM_STATUS_INVALID_ARGUMENT, "cache handle is null");
  }
  std::lock_guard<std::mutex> lock(g_caches_mutex);
  if (g_caches.count(c) == 0) {
    return write_error(sink, ULLM_STATUS_HIP_INVALID_HANDLE, "cache handle is not live");
  }
  return ULLM_STATUS_OK;
}

ullm_status_t fail(ullm_error_sink_t *sink, const char *message) {
  return write_error(sink, ULLM_STATUS_INVALID_ARGUMENT, message);
}

// Header, reserved words and handle of a call on a cache.
template <typename D>
ullm_status_t validate_call(const D *d, ullm_error_sink_t *sink, const char *null_message) {
  const ullm_status_t st = ullm::validate_header(d, sink, null_message);
  if (st != ULLM_STATUS_OK) {
    return st;
  }
  if (!ullm::all_zero(d->reserved)) {
    return write_error(sink, ULLM_STATUS_RESERVED_NONZERO,
                       "descriptor reserved fields must be zero");
  }
  return lookup_cache(d->cache, sink);
}

// `per_row`: the most heads a row has in this call.
ullm_status_t validate_seqs(const ullm_kv_cache_t *c, const ullm_kv_sequences_t &s, bool rows,
                            uint64_t per_row, ullm_error_sink_t *sink) {
  if (s.batch > kMaxGridYz) {
    return write_error(sink, ULLM_STATUS_UNSUPPORTED, "batch exceeds 65535 sequences");
  }
  if (!rows && (s.rows != 0 || s.starts != nullptr)) {
    return fail(sink, "this call takes no rows: rows must be 0 and starts null");
  }
  if (s.rows > kMaxCount / per_row) {
    return write_error(sink, ULLM_STATUS_UNSUPPORTED, "rows x heads exceeds 2^31 - 1");
  }
  if (s.max_blocks > kMaxCount / c->block_tokens) {
    return write_error(sink, ULLM_STATUS_UNSUPPORTED,
                       "max_blocks x block_tokens exceeds 2^31 - 1");
  }
  if (s.table_stride != 0 && s.table_stride < s.max_blocks) {
    return fail(sink, "table_stride is smaller than max_blocks");
  }
  if (rows && s.rows != 0 && s.starts == nullptr && (s.batch == 0 || s.rows % s.batch != 0)) {
    return fail(sink, "without starts, rows must be a multiple of batch");
  }
  const bool work = s.batch != 0 && (!rows || s.rows != 0);
  if (work && s.max_blocks == 0) {
    return fail(sink, "max_blocks must be at least 1");
  }
  if (work && (s.tables == nullptr || s.lengths == nullptr)) {
    return fail(sink, "tables or lengths pointer is null");
  }
  return ULLM_STATUS_OK;
}

bool no_work(const ullm_kv_sequences_t &s) { return s.batch == 0 || s.rows == 0; }

ullm::KvPool pool_of(const ullm_kv_cache_t *c) {
  ullm::KvPool p{};
  p.codes = c->codes;
  p.exps = c->exps;
  p.weights = c->weights;
  p.blocks = uint32_t(c->blocks);
  p.shift = c->block_tokens == 32 ? 5 : c->block_tokens == 64 ? 6 : 7;
  p.heads = c->kv_heads;
  return p;
}

ullm::KvSeqs seqs_of(const ullm_kv_sequences_t &s) {
  ullm::KvSeqs r{};
  r.tables = s.tables;
  r.stride = s.table_stride != 0 ? s.table_stride : s.max_blocks;
  r.max_blocks = uint32_t(s.max_blocks);
  r.lengths = s.lengths;
  r.starts = s.starts;
  r.batch = uint32_t(s.batch);
  r.rows = uint32_t(s.rows);
  r.each = s.starts == nullptr && s.batch != 0 ? uint32_t(s.rows / s.batch) : 0;
  return r;
}

// Strides of [rows][heads][dim] elements, 0 = contiguous.
struct Strides {
  uint64_t row, head;
};
Strides strides_of(uint64_t row, uint64_t head, uint64_t heads, uint64_t dim) {
  return {row != 0 ? row : heads * dim, head != 0 ? head : dim};
}
bool aligned(const void *p, const Strides &s, uint64_t bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && s.row * 2 % bytes == 0 &&
         s.head * 2 % bytes == 0;
}

ullm_status_t validate_append(const ullm_kv_cache_append_desc_t *d, ullm_error_sink_t *sink) {
  ullm_status_t st = validate_call(d, sink, "append descriptor is null");
  if (st != ULLM_STATUS_OK) {
    return st;
  }
  const ullm_kv_cache_t *c = d->cache;
  st = validate_seqs(c, d->seqs, true, c->kv_heads, sink);
  if (st != ULLM_STATUS_OK) {
    return st;
  }
  for (const uint64_t s : {d->k_row_stride, d->k_head_stride, d->v_row_stride, d->v_head_stride}) {
    if (s != 0 && s < c->head_dim) {
      return fail(sink, "a k or v stride is smaller than head_dim");
    }
  }
  if (d->weights != nullptr && c->weights == nullptr) {
    return fail(sink, "weights are given but the cache does not track weights");
  }
  if (!no_work(d->seqs) && (d->k == nullptr || d->v == nullptr)) {
    return fail(sink, "k or v pointer is null");
  }
  return ULLM_STATUS_OK;
}

// A scale in units of log2.
float log2_scale(float scale) { return float(double(scale) * 1.44269504088896340736); }

ullm_status_t validate_attend(const ullm_kv_cache_attend_desc_t *d, ullm_error_sink_t *sink) {
  ullm_status_t st = validate_call(d, sink, "attend descriptor is null");
  if (st != ULLM_STATUS_OK) {
    return st;
  }
  const ullm_kv_cache_t *c = d->cache;
  if (d->heads == 0 || d->heads % c->kv_heads != 0) {
    return fail(sink, "heads must be a multiple of the cache's kv_heads");
  }
  st = validate_seqs(c, d->seqs, true, d->heads, sink);
  if (st != ULLM_STATUS_OK) {
    return st;
  }
  if ((d->flags & ~ULLM_KV_ATTEND_ACCUMULATE) != 0) {
    return fail(sink, "unknown attend flags");
  }
  if ((d->flags & ULLM_KV_ATTEND_ACCUMULATE) != 0 && c->weights == nullptr) {
    return fail(sink, "ACCUMULATE needs a cache that tracks weights");
  }
  if (!std::isfinite(log2_scale(d->scale))) {
    return fail(sink, "scale must be finite, and in units of log2 too");
  }
  for (const uint64_t s :
       {d->q_row_stride, d->q_head_stride, d->out_row_stride, d->out_head_stride}) {
    if (s != 0 && s < c->head_dim) {
      return fail(sink, "a q or out stride is smaller than head_dim");
    }
  }
  const Strides o = strides_of(d->out_row_stride, d->out_head_stride, d->heads, c->head_dim);
  const bool rows_outer = o.row >= (d->heads - 1) * o.head + c->head_dim;
  const bool heads_outer =
      d->seqs.rows == 0 || o.head >= (d->seqs.rows - 1) * o.row + c->head_dim;
  if (!rows_outer && !heads_outer) {
    return fail(sink, "out strides make rows overlap");
  }
  if (!no_work(d->seqs) && (d->q == nullptr || d->out == nullptr)) {
    return fail(sink, "q or out pointer is null");
  }
  return ULLM_STATUS_OK;
}

ullm::KvAttendArgs attend_args(const ullm_kv_cache_attend_desc_t *d) {
  const ullm_kv_cache_t *c = d->cache;
  const Strides q = strides_of(d->q_row_stride, d->q_head_stride, d->heads, c->head_dim);
  const Strides o = strides_of(d->out_row_stride, d->out_head_stride, d->heads, c->head_dim);
  ullm::KvAttendArgs a{};
  a.pool = pool_of(c);
  a.seqs = seqs_of(d->seqs);
  a.q = static_cast<const uint16_t *>(d->q);
  a.out = static_cast<uint16_t *>(d->out);
  a.q_row = q.row;
  a.q_head = q.head;
  a.out_row = o.row;
  a.out_head = o.head;
  a.vec = aligned(d->q, q, 16);
  a.out_vec = aligned(d->out, o, 8);
  a.lse = d->lse;
  a.heads = d->heads;
  a.group = d->heads / c->kv_heads;
  a.window = d->window;
  // A scale of 0 becomes one that leaves every score at 0 but a token that is
  // not seen at -infinity.
  a.scale_log2 = std::max(std::fabs(log2_scale(d->scale)), 0x1p-120f);
  a.q_sign = d->scale < 0.f ? 0x80008000u : 0u;
  a.accumulate = (d->flags & ULLM_KV_ATTEND_ACCUMULATE) != 0;
  return a;
}

}  // namespace

extern "C" ULLM_HIP_API ullm_status_t ullm_kv_cache_create(const ullm_kv_cache_desc_t *desc,
                                                           ullm_kv_cache_t **cache,
                                                           ullm_error_sink_t *error_sink) {
  ULLM_ENTRY(error_sink, "cache create", {
    ullm_status_t st = ullm::validate_header(desc, error_sink, "cache descriptor is null");
    if (st != ULLM_STATUS_OK) {
      return st;
    }
    if (!ullm::all_zero(desc->reserved) || desc->reserved0 != 0) {
      return write_error(error_sink, ULLM_STATUS_RESERVED_NONZERO,
                         "cache descriptor reserved fields must be zero");
    }
    if (desc->blocks == 0 || desc->kv_heads == 0) {
      return fail(error_sink, "blocks and kv_heads must be at least 1");
    }
    if (desc->blocks > kMaxCount || desc->kv_heads > kMaxGridYz) {
      return write_error(error_sink, ULLM_STATUS_UNSUPPORTED,
                         "blocks exceed 2^31 - 1 or kv_heads 65535");
    }
    if (desc->block_tokens != 32 && desc->block_tokens != 64 && desc->block_tokens != 128) {
      return write_error(error_sink, ULLM_STATUS_UNSUPPORTED,
                         "block_tokens must be 32, 64 or 128");
    }
    if (desc->head_dim != 64 && desc->head_dim != 128) {
      return write_error(error_sink, ULLM_STATUS_UNSUPPORTED, "head_dim must be 64 or 128");
    }
    if ((desc->flags & ~ULLM_KV_CACHE_TRACK_WEIGHTS) != 0) {
      return fail(error_sink, "unknown cache flags");
    }
    if (cache == nullptr) {
      return fail(error_sink, "cache output pointer is null");
    }
    *cache = nullptr;
    st = check_device(desc->device, error_sink);
    if (st != ULLM_STATUS_OK) {
      return st;
    }
    DeviceScope scope(desc->device);
    HIP_TRY(error_sink, "hipSetDevice", scope.error());
    struct Owner {
      ullm_kv_cache_t *c;
      ~Owner() {
        if (c != nullptr) {
          (void)hipFree(c->codes);
          (void)hipFree(c->exps);
          (void)hipFree(c->weights);
          delete c;
        }
      }
    } owner{new ullm_kv_cache_t()};
    ullm_kv_cache_t *c = owner.c;
    c->blocks = desc->blocks;
    c->block_tokens = desc->block_tokens;
    c->kv_heads = desc->kv_heads;
    c->head_dim = desc->head_dim;
    c->flags = desc->flags;
    c->device = desc->device;
    const uint64_t units = desc->blocks * desc->kv_heads;
    const uint64_t code_bytes = units * 2 * desc->head_dim * desc->block_tokens;
    const uint64_t weight_bytes = (desc->flags & ULLM_KV_CACHE_TRACK_WEIGHTS) != 0
                                      ? units * desc->block_tokens * sizeof(float)
                                      : 0;
    HIP_TRY(error_sink, "hipMalloc (cache codes)", hipMalloc(&c->codes, code_bytes));
    HIP_TRY(error_sink, "hipMalloc (cache exponents)", hipMalloc(&c->exps, units * 2));
    HIP_TRY(error_sink, "hipMemset", hipMemset(c->codes, 0, code_bytes));
    HIP_TRY(error_sink, "hipMemset", hipMemset(c->exps, 0, units * 2));
    if (weight_bytes != 0) {
      HIP_TRY(error_sink, "hipMalloc (cache weights)", hipMalloc(&c->weights, weight_bytes));
      HIP_TRY(error_sink, "hipMemset", hipMemset(c->weights, 0, weight_bytes));
    }
    HIP_TRY(error_sink, "hipStreamSynchronize", hipStreamSynchronize(nullptr));
    c->device_bytes = code_bytes + units * 2 + weight_bytes;
    {
      std::lock_guard<std::mutex> lock(g_caches_mutex);
      g_caches.insert(c);
    }
    *cache = c;
    owner.c = nullptr;
    return ULLM_STATUS_OK;
  });
}

extern "C" ULLM_HIP_API ullm_status_t ullm_kv_cache_destroy(ullm_kv_cache_t **cache,
                                                            ullm_error_sink_t *error_sink) {
  ULLM_ENTRY(error_sink, "cache destroy", {
    if (cache == nullptr) {
      return fail(error_sink, "cache handle pointer is null");
    }
    ullm_kv_cache_t *c = *cache;
    if (c == nullptr) {
      return fail(error_sink, "cache handle is null");
    }
    {
      std::lock_guard<std::mutex> lock(g_caches_mutex);
      if (g_caches.erase(c) == 0) {
        return write_error(error_sink, ULLM_STATUS_HIP_INVALID_HANDLE,
                           "cache handle is not live");
      }
    }
    *cache = nullptr;
    DeviceScope scope(c->device);
    // hipFree synchronizes with outstanding work on the device.
    hipError_t first = hipSuccess;
    for (void *p : {static_cast<void *>(c->codes), static_cast<void *>(c->exps),
                    static_cast<void *>(c->weights)}) {
      const hipError_t e = hipFree(p);
      first = first == hipSuccess ? e : first;
    }
    delete c;
    HIP_TRY(error_sink, "hipFree", first);
    return ULLM_STATUS_OK;
  });
}

extern "C" ULLM_HIP_API ullm_status_t ullm_kv_cache_query(const ullm_kv_cache_t *cache,
                                                          ullm_kv_cache_info_t *info,
                                                          ullm_error_sink_t *error_sink) {
  ULLM_ENTRY(error_sink, "cache query", {
    ullm_status_t st = lookup_cache(cache, error_sink);
    if (st != ULLM_STATUS_OK) {
      return st;
    }
    st = ullm::validate_header(info, error_sink, "cache info output is null");
    if (st != ULLM_STATUS_OK) {
      return st;
    }
    if (!ullm::all_zero(info->reserved) || info->reserved0 != 0) {
      return write_error(error_sink, ULLM_STATUS_RESERVED_NONZERO,
                         "cache info reserved fields must be zero");
    }
    info->blocks = cache->blocks;
    info->block_tokens = cache->block_tokens;
    info->kv_heads = cache->kv_heads;
    info->head_dim = cache->head_dim;
    info->flags = cache->flags;
    info->device = cache->device;
    info->device_bytes = cache->device_bytes;
    return ULLM_STATUS_OK;
  });
}

extern "C" ULLM_HIP_API ullm_status_t ullm_kv_cache_append(
    const ullm_kv_cache_append_desc_t *desc, ullm_error_sink_t *error_sink) {
  ULLM_ENTRY(error_sink, "cache append", {
    const ullm_status_t st = validate_append(desc, error_sink);
    if (st != ULLM_STATUS_OK || no_work(desc->seqs)) {
      return st;
    }
    const ullm_kv_cache_t *c = desc->cache;
    DeviceScope scope(c->device);
    HIP_TRY(error_sink, "hipSetDevice", scope.error());
    const Strides k = strides_of(desc->k_row_stride, desc->k_head_stride, c->kv_heads,
                                 c->head_dim);
    const Strides v = strides_of(desc->v_row_stride, desc->v_head_stride, c->kv_heads,
                                 c->head_dim);
    ullm::KvAppendArgs a{};
    a.pool = pool_of(c);
    a.seqs = seqs_of(desc->seqs);
    a.k = static_cast<const uint16_t *>(desc->k);
    a.v = static_cast<const uint16_t *>(desc->v);
    a.k_row = k.row;
    a.k_head = k.head;
    a.v_row = v.row;
    a.v_head = v.head;
    a.vec = aligned(desc->k, k, 16) && aligned(desc->v, v, 16);
    a.weights = desc->weights;
    HIP_TRY(error_sink, "cache append kernel",
            ullm::launch_kv_append(a, c->head_dim, static_cast<hipStream_t>(desc->stream)));
    return ULLM_STATUS_OK;
  });
}

extern "C" ULLM_HIP_API ullm_status_t ullm_kv_cache_gather(
    const ullm_kv_cache_gather_desc_t *desc, ullm_error_sink_t *error_sink) {
  ULLM_ENTRY(error_sink, "cache gather", {
    ullm_status_t st = validate_call(desc, error_sink, "gather descriptor is null");
    if (st != ULLM_STATUS_OK) {
      return st;
    }
    const ullm_kv_cache_t *c = desc->cache;
    st = validate_seqs(c, desc->seqs, true, c->kv_heads, error_sink);
    if (st != ULLM_STATUS_OK) {
      return st;
    }
    if (desc->weights != nullptr && c->weights == nullptr) {
      return fail(error_sink, "weights are asked for but the cache does not track weights");
    }
    if (no_work(desc->seqs)) {
      return ULLM_STATUS_OK;
    }
    if (desc->k == nullptr && desc->v == nullptr && desc->weights == nullptr) {
      return fail(error_sink, "k, v and weights pointers are all null");
    }
    if ((reinterpret_cast<uintptr_t>(desc->k) | reinterpret_cast<uintptr_t>(desc->v)) % 16 != 0) {
      return fail(error_sink, "k and v must be 16-byte aligned");
    }
    DeviceScope scope(c->device);
    HIP_TRY(error_sink, "hipSetDevice", scope.error());
    ullm::KvGatherArgs a{};
    a.pool = pool_of(c);
    a.seqs = seqs_of(desc->seqs);
    a.k = static_cast<uint16_t *>(desc->k);
    a.v = static_cast<uint16_t *>(desc->v);
    a.weights = desc->weights;
    HIP_TRY(error_sink, "cache gather kernel",
            ullm::launch_kv_gather(a, c->head_dim, static_cast<hipStream_t>(desc->stream)));
    return ULLM_STATUS_OK;
  });
}

extern "C" ULLM_HIP_API ullm_status_t ullm_kv_cache_attend_plan(
    const ullm_kv_cache_attend_desc_t *desc, ullm_kv_attend_plan_t *plan,
    ullm_error_sink_t *error_sink) {
  ULLM_ENTRY(error_sink, "attend plan", {
    ullm_status_t st = validate_attend(desc, error_sink);
    if (st != ULLM_STATUS_OK) {
      return st;
    }
    st = ullm::validate_header(plan, error_sink, "plan output is null");
    if (st != ULLM_STATUS_OK) {
      return st;
    }
    if (!ullm::all_zero(plan->reserved)) {
      return write_error(error_sink, ULLM_STATUS_RESERVED_NONZERO,
                         "plan reserved fields must be zero");
    }
    ullm::KvAttendPlan p;
    if (!no_work(desc->seqs)) {
      DeviceScope scope(desc->cache->device);
      HIP_TRY(error_sink, "hipSetDevice", scope.error());
      p = ullm::plan_kv_attend(attend_args(desc), desc->cache->head_dim);
    }
    plan->kernel = p.kernel;
    plan->row_tile = p.row_tile;
    plan->parts = p.parts;
    plan->part_tokens = p.part_tokens;
    plan->grid = p.grid;
    plan->workspace_bytes = p.workspace;
    return ULLM_STATUS_OK;
  });
}

extern "C" ULLM_HIP_API ullm_status_t ullm_kv_cache_attend(
    const ullm_kv_cache_attend_desc_t *desc, ullm_error_sink_t *error_sink) {
  ULLM_ENTRY(error_sink, "cache attend", {
    ullm_status_t st = validate_attend(desc, error_sink);
    if (st != ULLM_STATUS_OK || no_work(desc->seqs)) {
      return st;
    }
    const ullm_kv_cache_t *c = desc->cache;
    const ullm::KvAttendArgs a = attend_args(desc);
    if (desc->out == desc->q) {
      // A workgroup reads its queries before it writes their results; the
      // second pass for the weights comes after all results.
      if (a.accumulate) {
        return fail(error_sink, "out must not be q with ACCUMULATE");
      }
      if ((a.seqs.rows > 1 && a.out_row != a.q_row) || (a.heads > 1 && a.out_head != a.q_head)) {
        return fail(error_sink, "out in place of q needs the strides of q");
      }
    }
    DeviceScope scope(c->device);
    HIP_TRY(error_sink, "hipSetDevice", scope.error());
    const ullm::KvAttendPlan p = ullm::plan_kv_attend(a, c->head_dim);
    // A launch counts its threads in 32 bits; the join has a wave for each row.
    if (p.grid > UINT32_MAX / 512 ||
        (p.parts > 1 && p.grid / p.parts > UINT32_MAX / 512 / p.row_tile)) {
      return write_error(error_sink, ULLM_STATUS_UNSUPPORTED,
                         "too many tiles of rows for one launch");
    }
    void *ws = desc->workspace;
    if (p.workspace != 0 && ws != nullptr) {
      if (desc->workspace_size < p.workspace) {
        return write_errorf(error_sink, ULLM_STATUS_BUFFER_TOO_SMALL,
                            "workspace needs " + std::to_string(p.workspace) + " bytes");
      }
      if (reinterpret_cast<uintptr_t>(ws) % 16 != 0) {
        return fail(error_sink, "workspace must be 16-byte aligned");
      }
    } else if (p.workspace != 0) {
      // Sizes grow with the sequences: whole powers of two keep the buffers
      // that growth retires few.
      uint64_t need = uint64_t(1) << 20;
      while (need < p.workspace) {
        need *= 2;
      }
      st = ullm::library_workspace(c->device, desc->stream, false, need, &ws, error_sink);
      if (st != ULLM_STATUS_OK) {
        return st;
      }
    }
    HIP_TRY(error_sink, "cache attend kernel",
            ullm::launch_kv_attend(a, c->head_dim, p, ws,
                                   static_cast<hipStream_t>(desc->stream)));
    return ULLM_STATUS_OK;
  });
}

extern "C" ULLM_HIP_API ullm_status_t ullm_kv_cache_evict(
    const ullm_kv_cache_evict_desc_t *desc, ullm_error_sink_t *error_sink) {
  ULLM_ENTRY(error_sink, "cache evict", {
    ullm_status_t st = validate_call(desc, error_sink, "evict descriptor is null");
    if (st != ULLM_STATUS_OK) {
      return st;
    }
    const ullm_kv_cache_t *c = desc->cache;
    st = validate_seqs(c, desc->seqs, false, c->kv_heads, error_sink);
    if (st != ULLM_STATUS_OK) {
      return st;
    }
    if (c->weights == nullptr) {
      return fail(error_sink, "evict needs a cache that tracks weights");
    }
    if (desc->keep == 0) {
      return fail(error_sink, "keep must be at least 1");
    }
    if (desc->keep > kMaxCount) {
      return write_error(error_sink, ULLM_STATUS_UNSUPPORTED, "keep exceeds 2^31 - 1");
    }
    if (desc->sink > desc->keep || desc->recent > desc->keep - desc->sink) {
      return fail(error_sink, "sink + recent exceeds keep");
    }
    const uint64_t columns = (desc->keep + c->block_tokens - 1) / c->block_tokens;
    if (desc->new_table_stride != 0 && desc->new_table_stride < columns) {
      return fail(error_sink, "new_table_stride is smaller than keep needs");
    }
    if (desc->seqs.batch == 0) {
      return ULLM_STATUS_OK;
    }
    if (desc->new_tables == nullptr || desc->new_lengths == nullptr || desc->kept == nullptr) {
      return fail(error_sink, "new_tables, new_lengths or kept pointer is null");
    }
    if (desc->new_lengths == desc->seqs.lengths || desc->new_tables == desc->seqs.tables) {
      return fail(error_sink, "new_lengths and new_tables must not be the old ones");
    }
    DeviceScope scope(c->device);
    HIP_TRY(error_sink, "hipSetDevice", scope.error());
    ullm::KvEvictArgs a{};
    a.pool = pool_of(c);
    a.seqs = seqs_of(desc->seqs);
    a.new_tables = desc->new_tables;
    a.new_stride = desc->new_table_stride != 0 ? desc->new_table_stride : columns;
    a.new_lengths = desc->new_lengths;
    a.kept = desc->kept;
    a.keep = uint32_t(desc->keep);
    a.sink = uint32_t(desc->sink);
    a.recent = uint32_t(desc->recent);
    HIP_TRY(error_sink, "cache evict kernels",
            ullm::launch_kv_evict(a, c->head_dim, static_cast<hipStream_t>(desc->stream)));
    return ULLM_STATUS_OK;
  });
}
