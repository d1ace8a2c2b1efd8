// Paged key/value cache in int8 or int4 (k_kvcache.hip, k_kvattn.hip), shared
// with the C ABI.
//
// A page holds `page` tokens of every key head: codes [pages, kv_heads, page,
// head_dim * bits / 8] and one bf16 scale per row, [pages, kv_heads, page].
// A head's rows of a page are contiguous, so a workgroup that serves one key
// head streams whole pieces of page * row bytes.  int4 rows hold pairs along
// head_dim, the even element in the low nibble, as pack_int4_k_major writes.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/strix_halo_gfx950.h"

namespace shk {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));

// A launch holds fewer than 2^32 work-items: the tokens of a write or read, and
// whether an attention's query rows fit.
constexpr int64_t kMostWorkgroups = 0xFFFFFF;  // of 256
int64_t kv_rows_most(bool write, const shk_kv_cache& c);
bool kv_attention_fits(const shk_kv_cache& c, const shk_kv_attention& a);
hipError_t launch_kv_write(const shk_kv_cache& c, const shk_kv_rows& r, hipStream_t s);
hipError_t launch_kv_read(const shk_kv_cache& c, const shk_kv_rows& r, hipStream_t s);
int64_t kv_attention_workspace(const shk_kv_cache& c, const shk_kv_attention& a);
hipError_t launch_kv_attention(const shk_kv_cache& c, const shk_kv_attention& a, hipStream_t s);

}  // namespace shk
