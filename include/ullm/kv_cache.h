/*
 * ullm/kv_cache.h -- key/value cache in 8 bits and its attention (gfx950 build).
 *
 * The reference has no attention: its tests describe where a cached token
 * lies (tests/reference/oracles.py:46-115) and no numerics.  These functions
 * are the part of a layer between the qkv and the output projection of
 * ullm/linear.h, under the same ABI v1 conventions: {struct_size,
 * abi_version} headers, zero reserved words, caller-owned error sinks, opaque
 * handles checked against a live-handle table, and no C++ exception across
 * the boundary.
 *
 * The cache is a pool of blocks of `block_tokens` tokens.  A block holds, for
 * each key/value head, E4M3FN codes of keys and of values and two exponents:
 * an element's value is code * 2^e, with e the smallest exponent (at least
 * -100, at most 119) for which 448 * 2^e reaches every finite element of that
 * block, head and side.  E4M3 is a floating format, so a power of two loses
 * nothing against a free scale but the use of the last binade, and it lets a
 * block take in a larger token later without rounding the others again
 * (codes that become subnormal aside).  E4M3FN has no infinity: infinite and
 * NaN elements are stored as NaN and do not count for the exponent.
 *
 * Which blocks a sequence owns is the caller's: row b of `tables` names the
 * block of tokens j * block_tokens .. of sequence b in column j.  Entries
 * outside the pool name no block: tokens there are not seen, and what is
 * written there is dropped.  Sequences may share blocks, but append and the
 * new tables of evict need blocks that no other sequence of the call uses.
 *
 * Rows.  Calls take the new tokens or queries of all sequences in one array
 * of `rows` rows; sequence b owns rows starts[b] .. starts[b + 1] - 1, or
 * rows / batch rows each when `starts` is null.  lengths[b] counts the
 * sequence's tokens with its new ones, so that append and attend take the
 * same lengths: the n rows of a sequence are its tokens (queries) at
 * positions lengths[b] - n .. lengths[b] - 1.  Rows at negative positions
 * name no token.  `tables`, `lengths` and `starts` are device memory, read in
 * stream order; lengths past max_blocks * block_tokens and starts outside
 * 0 .. rows are taken as those bounds.  Results of rows that no sequence owns
 * are left as they are.
 */
#ifndef ULLM_KV_CACHE_H
#define ULLM_KV_CACHE_H

#include "ullm/hip.h"
#include "ullm/linear.h"

/* ullm_kv_cache_desc_t.flags: keep a weight (f32) for each token and head,
 * which attend can add to and evict selects by. */
#define ULLM_KV_CACHE_TRACK_WEIGHTS UINT32_C(1)

/* ullm_kv_cache_attend_desc_t.flags: add to each token's weight, per
 * key/value head, the softmax weights that it receives from all queries of
 * the call and all query heads of the group. */
#define ULLM_KV_ATTEND_ACCUMULATE UINT32_C(1)

typedef struct ullm_kv_cache_t ullm_kv_cache_t;

typedef struct ullm_kv_cache_desc_t {
  uint32_t struct_size;
  uint32_t abi_version;
  uint64_t blocks;       /* blocks of the pool, >= 1 */
  uint32_t block_tokens; /* 32, 64 or 128 */
  uint32_t kv_heads;     /* >= 1 */
  uint32_t head_dim;     /* 64 or 128 */
  uint32_t flags;        /* ULLM_KV_CACHE_* */
  int32_t device;        /* HIP device ordinal that will own the pool */
  uint32_t reserved0;
  uint64_t reserved[4];
} ullm_kv_cache_desc_t;

typedef struct ullm_kv_cache_info_t {
  uint32_t struct_size;
  uint32_t abi_version;
  uint64_t blocks;
  uint32_t block_tokens;
  uint32_t kv_heads;
  uint32_t head_dim;
  uint32_t flags;
  int32_t device;
  uint32_t reserved0;
  uint64_t device_bytes; /* bytes the pool holds in HBM */
  uint64_t reserved[3];
} ullm_kv_cache_info_t;

/* Sequences of a call (see "Rows" above). */
typedef struct ullm_kv_sequences_t {
  uint64_t batch;
  uint64_t rows;
  const int32_t *tables;  /* device [batch][table_stride] */
  uint64_t table_stride;  /* elements, 0 = max_blocks */
  uint64_t max_blocks;    /* columns of a row; the split of long sequences
                             goes by it, so pass no more than are in use */
  const int32_t *lengths; /* device [batch] */
  const int32_t *starts;  /* device [batch + 1], or null: rows / batch each */
} ullm_kv_sequences_t;

/* New tokens of each sequence are quantized and stored.  A block whose first
 * token is among them starts anew; another one keeps its earlier tokens and
 * raises its exponent if a new one needs it. */
typedef struct ullm_kv_cache_append_desc_t {
  uint32_t struct_size;
  uint32_t abi_version;
  ullm_kv_cache_t *cache;
  ullm_kv_sequences_t seqs;
  const void *k;           /* device bf16 [rows][kv_heads][head_dim] */
  uint64_t k_row_stride;   /* elements, 0 = kv_heads * head_dim */
  uint64_t k_head_stride;  /* elements, 0 = head_dim */
  const void *v;           /* likewise */
  uint64_t v_row_stride;
  uint64_t v_head_stride;
  const float *weights;    /* device [rows][kv_heads], or null: weights are 0;
                              only for a cache that tracks weights */
  void *stream;
  uint64_t reserved[4];
} ullm_kv_cache_append_desc_t;

/* The values of each sequence's last rows, exact in bf16: the inverse of
 * append, whose result on them is the same values again.  Rows that name no
 * token are written as zeros. */
typedef struct ullm_kv_cache_gather_desc_t {
  uint32_t struct_size;
  uint32_t abi_version;
  const ullm_kv_cache_t *cache;
  ullm_kv_sequences_t seqs;
  void *k;        /* device bf16 [rows][kv_heads][head_dim], or null */
  void *v;        /* likewise */
  float *weights; /* device f32 [rows][kv_heads], or null */
  void *stream;
  uint64_t reserved[4];
} ullm_kv_cache_gather_desc_t;

/* Causal softmax attention of each sequence's rows over its cached tokens:
 * the query at position p sees the tokens at max(0, p - window + 1) .. p,
 *   out = sum_t exp(scale * q.k_t - lse) * v_t,
 *   lse = log(sum_t exp(scale * q.k_t));
 * a query that sees no token gives zeros and lse = -infinity.  Query head h
 * reads key/value head h / (heads / kv_heads).  Scores, sums and accumulators
 * are f32, the softmax weights enter the product with V in f16, 2^11 for the
 * largest of a row: each with a relative error of 2^-11, and those below 2^-25
 * of the largest with an absolute one of 2^-36 of it.  So it is for values
 * beside blocks with exponents up to 60 above theirs; next to larger ones they
 * may be lost. */
typedef struct ullm_kv_cache_attend_desc_t {
  uint32_t struct_size;
  uint32_t abi_version;
  ullm_kv_cache_t *cache;
  ullm_kv_sequences_t seqs;
  const void *q;            /* device bf16 [rows][heads][head_dim] */
  uint64_t q_row_stride;    /* elements, 0 = heads * head_dim */
  uint64_t q_head_stride;   /* elements, 0 = head_dim */
  void *out;                /* device bf16 [rows][heads][head_dim]: q itself,
                               with its strides and without ACCUMULATE, or
                               memory that does not overlap q */
  uint64_t out_row_stride;  /* elements, 0 = heads * head_dim */
  uint64_t out_head_stride; /* elements, 0 = head_dim */
  float *lse;               /* device f32 [rows][heads], or null */
  uint32_t heads;           /* a multiple of kv_heads */
  uint32_t window;          /* tokens a query sees, 0 = all up to its own */
  float scale;              /* finite, as is scale * log2(e); 0 and magnitudes
                               below count as 2^-120 / log2(e) */
  uint32_t flags;           /* ULLM_KV_ATTEND_* */
  void *stream;
  /* Device scratch of ullm_kv_attend_plan_t.workspace_bytes; null =
   * library-owned, one buffer per device and stream, allocated or grown by
   * the first call that needs it: make that call outside stream capture. */
  void *workspace;
  uint64_t workspace_size;
  uint64_t reserved[4];
} ullm_kv_cache_attend_desc_t;

/* Kernels reported by ullm_kv_cache_attend_plan. */
#define ULLM_KV_KERNEL_FEW_ROWS UINT32_C(1)  /* one wave's tile: 16 rows */
#define ULLM_KV_KERNEL_MANY_ROWS UINT32_C(2) /* tiles of many rows through LDS */

/* The launch an attend call with a given descriptor makes. */
typedef struct ullm_kv_attend_plan_t {
  uint32_t struct_size;
  uint32_t abi_version;
  uint32_t kernel;       /* ULLM_KV_KERNEL_* (0: nothing runs) */
  uint32_t row_tile;     /* (query, head of the group) rows of a tile */
  uint32_t parts;        /* parts of the longest sequence's tokens (1: no split) */
  uint32_t part_tokens;  /* tokens of a part */
  uint64_t grid;         /* workgroups */
  uint64_t workspace_bytes;
  uint64_t reserved[2];
} ullm_kv_attend_plan_t;

/* Cuts each sequence to its heaviest tokens.  Per key/value head of a
 * sequence longer than `keep`: the first `sink` and the last `recent` tokens
 * stay, and of the others those of the largest weight, the lower position
 * first among equal ones (NaN counts as larger than any number).  Shorter
 * sequences stay whole.  The tokens that stay are stored in their order, as
 * if gathered and appended with their weights, in the blocks that row b of
 * new_tables names: blocks that `seqs.tables` does not use.  seqs.rows and
 * seqs.starts are not used (0 and null). */
typedef struct ullm_kv_cache_evict_desc_t {
  uint32_t struct_size;
  uint32_t abi_version;
  ullm_kv_cache_t *cache;
  ullm_kv_sequences_t seqs;
  const int32_t *new_tables; /* device [batch][new_table_stride] */
  uint64_t new_table_stride; /* elements, 0 = ceil(keep / block_tokens) */
  int32_t *new_lengths;      /* device [batch]: min(length, keep); not `lengths` */
  int32_t *kept;             /* device [batch][kv_heads][keep]: positions that
                                stay, ascending, then -1 */
  uint64_t keep;             /* >= 1 */
  uint64_t sink;
  uint64_t recent;           /* sink + recent <= keep */
  void *stream;
  uint64_t reserved[4];
} ullm_kv_cache_evict_desc_t;

#ifdef __cplusplus
extern "C" {
#endif

/* Create a cache of zeroed blocks.  Blocks until it is ready. */
ULLM_HIP_API ullm_status_t ullm_kv_cache_create(
    const ullm_kv_cache_desc_t *desc, ullm_kv_cache_t **cache,
    ullm_error_sink_t *error_sink);

/* Destroy and null *cache.  Waits for the device to finish using it. */
ULLM_HIP_API ullm_status_t ullm_kv_cache_destroy(ullm_kv_cache_t **cache,
                                                 ullm_error_sink_t *error_sink);

ULLM_HIP_API ullm_status_t ullm_kv_cache_query(const ullm_kv_cache_t *cache,
                                               ullm_kv_cache_info_t *info,
                                               ullm_error_sink_t *error_sink);

/* The calls below are asynchronous in stream order. */
ULLM_HIP_API ullm_status_t ullm_kv_cache_append(
    const ullm_kv_cache_append_desc_t *desc, ullm_error_sink_t *error_sink);

ULLM_HIP_API ullm_status_t ullm_kv_cache_gather(
    const ullm_kv_cache_gather_desc_t *desc, ullm_error_sink_t *error_sink);

ULLM_HIP_API ullm_status_t ullm_kv_cache_attend(
    const ullm_kv_cache_attend_desc_t *desc, ullm_error_sink_t *error_sink);

/* The launch and the workspace of an attend call.  Launches nothing. */
ULLM_HIP_API ullm_status_t ullm_kv_cache_attend_plan(
    const ullm_kv_cache_attend_desc_t *desc, ullm_kv_attend_plan_t *plan,
    ullm_error_sink_t *error_sink);

ULLM_HIP_API ullm_status_t ullm_kv_cache_evict(
    const ullm_kv_cache_evict_desc_t *desc, ullm_error_sink_t *error_sink);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* ULLM_KV_CACHE_H */
