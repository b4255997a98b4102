/*
 * ullm/kv_rotary.h -- rotary positions on the way into the cache (gfx950 build).
 *
 * ullm_kv_cache_append_rotary is ullm_kv_cache_append for keys that a
 * position still has to rotate, and rotates the queries of the same rows: the
 * step between the qkv projection and ullm_kv_cache_attend in one launch.  Of
 * each head the first `rotary_dims` dims are rotated in pairs, the others stay
 * as they are.  Pair j has dims j and j + rotary_dims / 2, or 2j and 2j + 1
 * with ULLM_KV_ROTARY_INTERLEAVED; its elements x, y become
 *
 *   x * cos(a) - y * sin(a),  y * cos(a) + x * sin(a),  a = p * inv_freq[j],
 *
 * p the row's position on the pair's axis.  Positions are whole numbers: by
 * default the row's place in its sequence (that of lengths, as in
 * ullm/kv_cache.h), else those of `positions`, one for each axis and row, for
 * example the time, height and width of an image's patch.  `pair_axes` names
 * each pair's axis.
 *
 * Angles are reduced to a turn, and their cosines and sines taken, in 64 bits:
 * position 2^31 - 1 is as exact as position 1 (for frequencies up to 2^16).
 * Queries are then rotated in f32 and rounded to bf16.  Keys are rotated in 64
 * bits and rounded once, to their codes (in caches of 8 and of 4 bits), so that a
 * key between two codes does not depend on the last bits of an f32.
 *
 * Every row that a sequence owns has its queries rotated, rows that name no
 * token among them (their place is negative); rows that no sequence owns are
 * left as they are.
 */
#ifndef ULLM_KV_ROTARY_H
#define ULLM_KV_ROTARY_H

#include "ullm/kv_cache.h"

/* ullm_kv_cache_append_rotary_desc_t.flags: pairs of neighbouring dims. */
#define ULLM_KV_ROTARY_INTERLEAVED UINT32_C(1)

typedef struct ullm_kv_cache_append_rotary_desc_t {
  uint32_t struct_size;
  uint32_t abi_version;
  ullm_kv_cache_t *cache;
  ullm_kv_sequences_t seqs;
  const void *q;            /* device bf16 [rows][heads][head_dim] */
  uint64_t q_row_stride;    /* elements, 0 = heads * head_dim */
  uint64_t q_head_stride;   /* elements, 0 = head_dim */
  void *q_out;              /* device bf16 [rows][heads][head_dim]: q itself,
                               with its strides, or memory that does not
                               overlap q, k and v */
  uint64_t q_out_row_stride;  /* elements, 0 = heads * head_dim */
  uint64_t q_out_head_stride; /* elements, 0 = head_dim */
  const void *k;            /* device bf16 [rows][kv_heads][head_dim] */
  uint64_t k_row_stride;    /* elements, 0 = kv_heads * head_dim */
  uint64_t k_head_stride;   /* elements, 0 = head_dim */
  const void *v;            /* likewise */
  uint64_t v_row_stride;
  uint64_t v_head_stride;
  const float *weights;     /* device [rows][kv_heads], or null: weights are 0;
                               only for a cache that tracks weights */
  const float *inv_freq;    /* device [rotary_dims / 2], angle of a position */
  const int32_t *positions; /* device [axes][rows], or null: places (1 axis) */
  uint64_t position_stride; /* elements from axis to axis, 0 = rows */
  const uint8_t *pair_axes; /* device [rotary_dims / 2], or null: axis 0; an
                               axis past the last is taken as the last */
  uint32_t heads;           /* query heads: 0 (no q) or a multiple of kv_heads */
  uint32_t rotary_dims;     /* even, 2 .. head_dim */
  uint32_t axes;            /* 1 .. 4 */
  uint32_t flags;           /* ULLM_KV_ROTARY_* */
  void *stream;
  uint64_t reserved[4];
} ullm_kv_cache_append_rotary_desc_t;

#ifdef __cplusplus
extern "C" {
#endif

/* Rotate and store new tokens; asynchronous in stream order. */
ULLM_HIP_API ullm_status_t ullm_kv_cache_append_rotary(
    const ullm_kv_cache_append_rotary_desc_t *desc, ullm_error_sink_t *error_sink);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* ULLM_KV_ROTARY_H */
