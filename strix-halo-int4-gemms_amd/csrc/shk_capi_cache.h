// Checks of a cache that the C ABI's files share.
#pragma once

#include <climits>
#include <string>

#include "../../include/strix_halo_gfx950.h"
#include "shk_capi.h"

namespace shk {

inline bool on(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// 0, or the rc of a message about the cache.
inline int check_cache(const shk_kv_cache* c) {
  if (c == nullptr) return capi_fail("cache must be non-null");
  if (c->bits != 4 && c->bits != 8) return capi_fail("cache bits must be 4 or 8; got " + std::to_string(c->bits));
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return capi_fail("cache head_dim must be 64, 128 or 256; got " + std::to_string(c->head_dim));
  if (c->page_size < 16 || c->page_size > 1024 || (c->page_size & (c->page_size - 1)) != 0)
    return capi_fail("cache page_size must be a power of two from 16 to 1024; got " + std::to_string(c->page_size));
  if (c->kv_heads < 1 || c->kv_heads > 65535 || c->pages < 1 || c->pages > INT_MAX)
    return capi_fail("cache needs 1 to 65535 heads and 1 to 2147483647 pages");
  if (c->pages * c->kv_heads > INT_MAX) return capi_fail("the cache holds more than 2147483647 pages of a head");
  if (!c->key_codes || !c->value_codes || !c->key_scales || !c->value_scales)
    return capi_fail("cache pointers must be non-null");
  if (!on(c->key_codes, 16) || !on(c->value_codes, 16)) return capi_fail("cache codes must be aligned to 16 bytes");
  if (!on(c->key_scales, 8) || !on(c->value_scales, 8)) return capi_fail("cache scales must be aligned to 8 bytes");
  return 0;
}

}  // namespace shk
