// C ABI of the decode step's operators: argument validation and launches.
// Declarations are in include/strix_halo_gfx950.h.
#include <climits>
#include <cmath>
#include <string>

#include "shk_capi.h"
#include "shk_capi_cache.h"
#include "shk_kvcache.h"
#include "shk_moe.h"

namespace {

using shk::check_cache;
using shk::on;
using shk::capi_entry;
using shk::capi_fail;
using shk::capi_fail_hip;

int check_rows(const shk_kv_rows* r) {
  if (r == nullptr) return capi_fail("rows must be non-null");
  if (r->type != SHK_SRC_F32 && r->type != SHK_SRC_F16 && r->type != SHK_SRC_BF16)
    return capi_fail("unknown row type " + std::to_string(r->type));
  if (r->slot_bytes != 4 && r->slot_bytes != 8) return capi_fail("slots are int32 or int64");
  if (r->tokens < 0) return capi_fail("tokens must not be negative");
  if (r->tokens > 0 && (!r->keys || !r->values || !r->slots))
    return capi_fail("keys, values and slots pointers must be non-null");
  return 0;
}

int rows_entry(bool write, int device_index, uintptr_t stream, const shk_kv_cache* cache, const shk_kv_rows* rows) {
  return capi_entry([&] {
    if (int rc = check_cache(cache)) return rc;
    if (int rc = check_rows(rows)) return rc;
    if (rows->tokens == 0) return 0;
    if (rows->tokens > shk::kv_rows_most(write, *cache)) return capi_fail("too many tokens for one launch");
    shk::DeviceGuard guard(device_index);
    if (guard.error() != hipSuccess) return capi_fail_hip("hipSetDevice", guard.error());
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const hipError_t err = write ? shk::launch_kv_write(*cache, *rows, s) : shk::launch_kv_read(*cache, *rows, s);
    if (err != hipSuccess) return capi_fail_hip(write ? "kv_write launch" : "kv_read launch", err);
    return 0;
  });
}

int check_attention(const shk_kv_cache* c, const shk_kv_attention* a) {
  if (int rc = check_cache(c)) return rc;
  if (a == nullptr) return capi_fail("attention arguments must be non-null");
  if (a->type != SHK_SRC_F16 && a->type != SHK_SRC_BF16) return capi_fail("q is float16 or bfloat16");
  if (a->batch < 0 || a->queries < 0 || a->heads < 0) return capi_fail("batch, queries and heads must not be negative");
  if (a->heads == 0 || a->heads % c->kv_heads != 0)
    return capi_fail("heads must be a multiple of the cache's kv_heads; got " + std::to_string(a->heads) + " and " +
                     std::to_string(c->kv_heads));
  if (a->batch > INT_MAX || a->queries > INT_MAX || a->heads > INT_MAX ||
      (__int128)a->batch * a->queries * a->heads > INT_MAX / 32)
    return capi_fail("too many query rows for one launch");
  // tokens are counted in 32 bits, and rounded up to pieces of 256 there
  constexpr int64_t most = INT_MAX - 256;
  if (a->table_pages < 0 || (__int128)a->table_pages * c->page_size > most)
    return capi_fail("a sequence holds at most 2147483391 tokens");
  if ((__int128)a->batch * ((a->table_pages * c->page_size + 255) / 256) > most)
    return capi_fail("too many tokens in the page table");
  if (!std::isfinite((float)a->scale))
    return capi_fail("the softmax scale must be finite in 32 bits; got " + std::to_string(a->scale));
  if (a->prefix_length < 0 || a->prefix_length > most)
    return capi_fail("prefix_length must be from 0 to 2147483391; got " + std::to_string(a->prefix_length));
  if (a->batch * a->queries > 0 && !shk::kv_attention_fits(*c, *a)) return capi_fail("too many query rows for one launch");
  return 0;
}

int check_moe(const shk_moe* a) {
  if (a == nullptr) return capi_fail("moe arguments must be non-null");
  if (a->type != SHK_SRC_F16 && a->type != SHK_SRC_BF16) return capi_fail("x is float16 or bfloat16");
  if (a->layout != SHK_LAYOUT_NN && a->layout != SHK_LAYOUT_NT) return capi_fail("moe layouts are NN and NT");
  if (a->group != 0 && a->group != 32 && a->group != 64 && a->group != 128 && a->group != 256)
    return capi_fail("the scale group is 0, 32, 64, 128 or 256; got " + std::to_string(a->group));
  if (a->tokens < 0 || a->tokens > 64)
    return capi_fail("at most 64 tokens a call; got " + std::to_string(a->tokens));
  if (a->top < 0 || (a->tokens > 0 && a->top > 1024 / a->tokens)) return capi_fail("at most 1024 (token, expert) pairs a call");
  if (a->experts < 1 || a->experts > 1024) return capi_fail("1 to 1024 experts; got " + std::to_string(a->experts));
  if (a->hidden < 1 || a->inner < 1 || a->hidden > (1 << 20) || a->inner > (1 << 20))
    return capi_fail("hidden and inner must be from 1 to 1048576");
  // codes are read a dword at a time, the last one from the matrix's end
  if (a->experts * 2 * a->inner * ((a->hidden + 1) / 2) < 4 || a->experts * a->hidden * ((a->inner + 1) / 2) < 4)
    return capi_fail("up_gate and down must hold at least 4 bytes each");
  if (a->id_bytes != 4 && a->id_bytes != 8) return capi_fail("ids are int32 or int64");
  return 0;
}

}  // namespace

extern "C" {

int amd_strix_halo_kernels_kv_write(int device_index, uintptr_t stream, const shk_kv_cache* cache,
                                    const shk_kv_rows* rows) {
  return rows_entry(true, device_index, stream, cache, rows);
}

int amd_strix_halo_kernels_kv_read(int device_index, uintptr_t stream, const shk_kv_cache* cache,
                                   const shk_kv_rows* rows) {
  return rows_entry(false, device_index, stream, cache, rows);
}

int64_t amd_strix_halo_kernels_kv_attention_workspace(const shk_kv_cache* cache, const shk_kv_attention* args) {
  int64_t bytes = -1;
  (void)capi_entry([&] {
    if (int rc = check_attention(cache, args)) return rc;
    bytes = args->batch * args->queries == 0 ? 0 : shk::kv_attention_workspace(*cache, *args);
    return 0;
  });
  return bytes;
}

int amd_strix_halo_kernels_kv_attention(int device_index, uintptr_t stream, const shk_kv_cache* cache,
                                        const shk_kv_attention* args) {
  return capi_entry([&] {
    if (int rc = check_attention(cache, args)) return rc;
    const shk_kv_attention& a = *args;
    if (a.batch * a.queries == 0) return 0;
    if (!a.q || !a.out || !a.lengths) return capi_fail("q, out and lengths pointers must be non-null");
    if (a.table_pages > 0 && !a.page_table) return capi_fail("the page_table pointer must be non-null");
    if (a.prefix_length > 0 && !a.prefix_pages) return capi_fail("the prefix_pages pointer must be non-null");
    if (!on(a.q, 16) || a.q_batch_stride % 8 || a.q_query_stride % 8 || a.q_head_stride % 8)
      return capi_fail("rows of q must be aligned to 16 bytes");
    if (!on(a.out, 8)) return capi_fail("out must be aligned to 8 bytes");
    const int64_t need = shk::kv_attention_workspace(*cache, a);
    if (need > 0 && (a.workspace == nullptr || a.workspace_bytes < need || !on(a.workspace, 16)))
      return capi_fail("the workspace must hold " + std::to_string(need) + " bytes, aligned to 16");
    shk::DeviceGuard guard(device_index);
    if (guard.error() != hipSuccess) return capi_fail_hip("hipSetDevice", guard.error());
    const hipError_t err = shk::launch_kv_attention(*cache, a, reinterpret_cast<hipStream_t>(stream));
    if (err != hipSuccess) return capi_fail_hip("kv_attention launch", err);
    return 0;
  });
}

int64_t amd_strix_halo_kernels_moe_workspace(const shk_moe* args) {
  int64_t bytes = -1;
  (void)capi_entry([&] {
    if (int rc = check_moe(args)) return rc;
    bytes = shk::moe_workspace(*args);
    return 0;
  });
  return bytes;
}

int amd_strix_halo_kernels_moe(int device_index, uintptr_t stream, const shk_moe* args) {
  return capi_entry([&] {
    if (int rc = check_moe(args)) return rc;
    const shk_moe& a = *args;
    if (a.tokens == 0) return 0;
    if (!a.x || !a.out || !a.up_gate || !a.up_gate_scale || !a.down || !a.down_scale)
      return capi_fail("x, out, weight and scale pointers must be non-null");
    if (a.top > 0 && (!a.ids || !a.share)) return capi_fail("ids and share pointers must be non-null");
    if (!on(a.x, 2) || !on(a.out, 2) || !on(a.up_gate_scale, 2) || !on(a.down_scale, 2) ||
        !on(a.ids, (uintptr_t)a.id_bytes) || !on(a.share, 4))
      return capi_fail("x, out, scales, ids and share must be aligned to their elements");
    const int64_t need = shk::moe_workspace(a);
    if (need > 0 && (a.workspace == nullptr || a.workspace_bytes < need || !on(a.workspace, 16)))
      return capi_fail("the workspace must hold " + std::to_string(need) + " bytes, aligned to 16");
    shk::DeviceGuard guard(device_index);
    if (guard.error() != hipSuccess) return capi_fail_hip("hipSetDevice", guard.error());
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const hipError_t err = a.layout == SHK_LAYOUT_NT ? shk::launch_moe_nt(a, s) : shk::launch_moe_nn(a, s);
    if (err != hipSuccess) return capi_fail_hip("moe launch", err);
    return 0;
  });
}

}  // extern "C"
