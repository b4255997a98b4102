/*
 * ullm/kv_cache4.h -- key/value cache in 4 bits (gfx950 build).
 *
 * A cache that ullm_kv_cache_create makes with the flag
 * ULLM_KV_CACHE_4_BITS holds keys and values as E2M1 codes (0, 0.5, 1, 1.5,
 * 2, 3, 4, 6 and their negatives); every call of ullm/kv_cache.h and
 * ullm/kv_rotary.h takes it.  A token takes head_dim * 33 / 32 + 2 bytes for
 * each head, 0.53 of what it takes in 8 bits.
 *
 * Scales.  A token has scales of its own, so that an append changes no earlier
 * token's codes.  They follow the products that read them:
 *
 *   keys: one exponent e for each 32 dims, the smallest (at least -100, at
 *     most 119) for which 6 * 2^e reaches every element of the 32.  The
 *     product with a query runs over dims, and converting a code to bf16 takes
 *     a power of two for free.
 *   values: one scale s for all dims, the smallest of the numbers n * 2^k, n
 *     = 32 .. 63, from 2^-19 to 63 * 2^10, for which 6 * s reaches every
 *     element.  The product with the softmax weights runs over tokens, where a
 *     token's scale enters its weight.
 *
 * Codes are rounded to nearest, ties to the even code; elements past 6 * 2^119
 * (keys) or 6 * 63 * 2^10 = 387072 (values) are stored as that.  Stored values
 * are exact in bf16: gather's result, appended again, is stored as the same
 * values.  E2M1 has neither infinities nor NaN: 32 dims of a key, or a whole
 * value, with an infinite or NaN element are NaN as a whole.
 *
 * Attention as in ullm/kv_cache.h.  A token's weight times its scale enters
 * the product with the values in f16: with a relative error of 2^-11, and where
 * it is below 2^-25 of the row's largest, with an absolute one of 2^-36 of that.
 * Calls of many rows (ULLM_KV_KERNEL_MANY_ROWS) add log2 of the value's scale to
 * the score, in f32: tokens of equal keys and values of different scales have
 * weights that are equal within the rounding of such a sum (2^-20 of its
 * magnitudes) there.
 * A value of NaN makes the results of the queries that see it NaN, not their
 * lse nor the weights that tokens receive from them.
 * The scale of the scores must not pass 2^100 / log2(e), 2^100 in units of log2.
 *
 * Evict moves codes and scales as they are.
 */
#ifndef ULLM_KV_CACHE4_H
#define ULLM_KV_CACHE4_H

#include "ullm/kv_cache.h"

/* ullm_kv_cache_desc_t.flags: hold keys and values in 4 bits. */
#define ULLM_KV_CACHE_4_BITS UINT32_C(4)

#endif /* ULLM_KV_CACHE4_H */
