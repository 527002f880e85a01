// What the kernels of the paged 4-bit cache share: vector types and the checks of a cache's arguments.
#pragma once

#include <stdint.h>

#include "dkv_host.h"
#include "dimmerkv.h"

typedef float floatx2 __attribute__((ext_vector_type(2)));
struct dkv_bf16 { uint16_t bits; };

namespace dkv {

// log2 of a page's tokens; -1 for a page that is not a power of two from 16 (an attention tile) to 4096.
inline int page_shift(int32_t page) {
  for (int s = 4; s <= 12; ++s)
    if (page == 1 << s) return s;
  return -1;
}

inline int check_fp4_cache(const dkv_fp4_cache_t* c, const char* what) {
  if (!c || !c->key_codes || !c->key_scales || !c->value_codes || !c->value_scales) {
    set_error("%s: null cache pointer", what);
    return DKV_EINVAL;
  }
  if ((((uintptr_t)c->key_codes | (uintptr_t)c->value_codes) & 15) || (((uintptr_t)c->key_scales | (uintptr_t)c->value_scales) & 15)) {
    set_error("%s: the cache's arrays must be 16-byte aligned", what);
    return DKV_EINVAL;
  }
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) {
    set_error("%s: head_dim %d is not 64, 128 or 256", what, c->head_dim);
    return DKV_ESHAPE;
  }
  if (c->pages <= 0 || c->kv_heads <= 0 || c->kv_heads > 65535 || page_shift(c->page) < 0) {
    set_error("%s: bad cache (pages=%d kv_heads=%d page=%d, a power of two from 16 to 4096)", what, c->pages, c->kv_heads, c->page);
    return DKV_ESHAPE;
  }
  return DKV_OK;
}

}  // namespace dkv
