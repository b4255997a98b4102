/* ullm/ullm.h -- umbrella header (reference include/ullm/ullm.h:1-6), extended
 * with the linear-layer, key/value-cache and weight-file entry points of this library. */
#ifndef ULLM_ULLM_H
#define ULLM_ULLM_H

#include "ullm/hip.h"
#include "ullm/kv_cache.h"
#include "ullm/kv_cache4.h"
#include "ullm/kv_rotary.h"
#include "ullm/linear.h"
#include "ullm/weights_io.h"

#endif /* ULLM_ULLM_H */
