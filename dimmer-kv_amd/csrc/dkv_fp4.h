// What the kernels of the paged 4-bit cache share: vector types and the checks of a cache's arguments.
#pragma once

#include <stdint.h>

#include "dkv_device.h"
#include "dkv_host.h"
#include "dimmerkv.h"

typedef float floatx2 __attribute__((ext_vector_type(2)));
struct dkv_bf16 { uint16_t bits; };

#ifdef __HIPCC__
// Results that one workgroup leaves for another of the same launch, on whatever die.  They are written and read at the
// device's scope, past the dies' own caches, so that neither side has to flush or drop a cache; `left_behind` waits until a
// wave's are there, and after a barrier one thread of the workgroup may announce them.
DKV_DEVICE void leave(uint64_t* at, uint64_t v) { __hip_atomic_store(at, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
DKV_DEVICE uint64_t pick_up(const uint64_t* at) {
  return __hip_atomic_load((uint64_t*)at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
DKV_DEVICE void leave2(float* at, float a, float b) {
  leave((uint64_t*)at, (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a));
}
DKV_DEVICE float2 pick_up2(const float* at) {
  const uint64_t v = pick_up((const uint64_t*)at);
  return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}
DKV_DEVICE void left_behind() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// Whether this is the last of `all` announcements on a word that is 0 before the first one, and 0 again after the last.
DKV_DEVICE bool last_of(uint32_t* word, uint32_t all) {
  if (__hip_atomic_fetch_add(word, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != all - 1) return false;
  __hip_atomic_store(word, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return true;
}
#endif

namespace dkv {

// Tokens a request may have: what the kernels round up to whole chunks stays below 2^31.
constexpr int64_t kMostTokens = (1L << 31) - (1 << 16);

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
