// C ABI of a step's operators around its cached attention: argument validation
// and launches.  Declarations are in include/strix_halo_gfx950.h.
#include <climits>
#include <cmath>
#include <cstdlib>
#include <string>

#include "shk_capi.h"
#include "shk_capi_cache.h"
#include "shk_step.h"

namespace {

using shk::capi_entry;
using shk::capi_fail;
using shk::capi_fail_hip;
using shk::check_cache;
using shk::on;

bool source(int64_t t) { return t == SHK_SRC_F32 || t == SHK_SRC_F16 || t == SHK_SRC_BF16; }

int check_rotate(const shk_kv_cache* c, const shk_rotate* args) {
  if (args == nullptr) return capi_fail("rotation arguments must be non-null");
  const shk_rotate& a = *args;
  if (!source(a.type) || !source(a.weight_type)) return capi_fail("unknown value type");
  if (a.tokens < 0 || a.heads < 1 || a.kv_heads < 1 || a.heads > 65535 || a.kv_heads > 65535)
    return capi_fail("q and k need 1 to 65535 heads");
  if (a.head_dim < 2 || a.head_dim > 256 || a.head_dim % 2)
    return capi_fail("head_dim must be even, from 2 to 256; got " + std::to_string(a.head_dim));
  if (a.rotated < 0 || a.rotated > a.head_dim || a.rotated % 2)
    return capi_fail("rotated must be even, from 0 to head_dim; got " + std::to_string(a.rotated));
  if (a.position_bytes != 4 && a.position_bytes != 8) return capi_fail("positions are int32 or int64");
  if (!std::isfinite((float)a.amplitude)) return capi_fail("the amplitude must be finite in 32 bits");
  if (!(a.eps >= 0.0) || !std::isfinite((float)a.eps)) return capi_fail("eps must be finite and not negative");
  if ((a.q_weight == nullptr) != (a.k_weight == nullptr)) return capi_fail("q and k have weights both or neither");
  // a launch holds fewer than 2^32 work-items, and rows are counted in 32 bits
  const int64_t lanes = a.head_dim <= 64 ? 8 : a.head_dim <= 128 ? 16 : 32;
  if ((__int128)a.tokens * (a.heads + (c != nullptr ? 2 : 1) * a.kv_heads) > (0xFFFFFFFFLL / lanes) - 4096)
    return capi_fail("too many rows for one launch");
  if (c != nullptr) {
    if (int rc = check_cache(c)) return rc;
    if (c->head_dim != a.head_dim || c->kv_heads != a.kv_heads)
      return capi_fail("head_dim and kv_heads must be the cache's, " + std::to_string(c->head_dim) + " and " +
                       std::to_string(c->kv_heads));
    if (a.slot_bytes != 4 && a.slot_bytes != 8) return capi_fail("slots are int32 or int64");
  }
  const auto apart = [&](int64_t token_stride, int64_t head_stride, int64_t heads) {
    return (a.tokens <= 1 || std::llabs(token_stride) >= a.head_dim) &&
           (heads <= 1 || std::llabs(head_stride) >= a.head_dim);
  };
  if (!apart(a.q_out_token_stride, a.q_out_head_stride, a.heads) ||
      (c == nullptr && !apart(a.k_out_token_stride, a.k_out_head_stride, a.kv_heads)))
    return capi_fail("rows of q_out and k_out must not overlap");
  return 0;
}

int check_verify(const shk_verify* args) {
  if (args == nullptr) return capi_fail("verification arguments must be non-null");
  const shk_verify& a = *args;
  if (!source(a.type)) return capi_fail("unknown value type");
  if (a.batch < 0 || a.batch > 65535) return capi_fail("0 to 65535 sequences a call; got " + std::to_string(a.batch));
  if (a.drafts < 0 || a.drafts >= shk::kMostDrafts)
    return capi_fail("0 to 63 drafts a sequence; got " + std::to_string(a.drafts));
  if (a.vocab < 1 || a.vocab > INT_MAX / 2) return capi_fail("the vocabulary has 1 to 1073741823 tokens");
  if (a.token_bytes != 4 && a.token_bytes != 8) return capi_fail("tokens are int32 or int64");
  return 0;
}

}  // namespace

extern "C" {

int amd_strix_halo_kernels_rotate(int device_index, uintptr_t stream, const shk_kv_cache* cache,
                                  const shk_rotate* args) {
  return capi_entry([&] {
    if (int rc = check_rotate(cache, args)) return rc;
    const shk_rotate& a = *args;
    if (a.tokens == 0) return 0;
    if (!a.q || !a.k || !a.positions || !a.q_out || (a.rotated > 0 && !a.turns))
      return capi_fail("q, k, positions, turns and q_out pointers must be non-null");
    if (cache != nullptr ? !a.values || !a.slots : !a.k_out)
      return capi_fail(cache != nullptr ? "values and slots pointers must be non-null"
                                        : "the k_out pointer must be non-null");
    const uintptr_t size = a.type == SHK_SRC_F32 ? 4 : 2, weight = a.weight_type == SHK_SRC_F32 ? 4 : 2;
    if (!on(a.q, size) || !on(a.k, size) || !on(a.q_out, size) || !on(a.k_out, size) || !on(a.values, size) ||
        !on(a.q_weight, weight) || !on(a.k_weight, weight) || !on(a.positions, (uintptr_t)a.position_bytes) ||
        !on(a.turns, 8) || (cache != nullptr && !on(a.slots, (uintptr_t)a.slot_bytes)))
      return capi_fail("tensors must be aligned to their elements");
    shk::DeviceGuard guard(device_index);
    if (guard.error() != hipSuccess) return capi_fail_hip("hipSetDevice", guard.error());
    const hipError_t err = shk::launch_rotate(cache, a, reinterpret_cast<hipStream_t>(stream));
    if (err != hipSuccess) return capi_fail_hip("rotate launch", err);
    return 0;
  });
}

int amd_strix_halo_kernels_kv_plan(int device_index, uintptr_t stream, const shk_kv_plan* args) {
  return capi_entry([&] {
    if (args == nullptr) return capi_fail("plan arguments must be non-null");
    const shk_kv_plan& a = *args;
    if (a.batch < 1 || a.batch > shk::kPlanBatch)
      return capi_fail("1 to 4096 sequences a step; got " + std::to_string(a.batch));
    if (a.page_size < 16 || a.page_size > 1024 || (a.page_size & (a.page_size - 1)) != 0)
      return capi_fail("page_size must be a power of two from 16 to 1024; got " + std::to_string(a.page_size));
    if (a.width < 1 || a.width > INT_MAX / a.page_size)
      return capi_fail("a sequence holds at most 2147483647 tokens, in at least one page");
    if (a.free_total < 0 || a.free_total >= INT_MAX) return capi_fail("0 to 2147483646 places for free pages");
    if (a.capacity < 0 || a.capacity > INT_MAX) return capi_fail("capacity must be from 0 to 2147483647");
    if (!a.page_table || !a.lengths || !a.owned || !a.free_count || !a.new_tokens || !a.starts || !a.taken || !a.ticket ||
        (a.free_total > 0 && !a.free_pages) || (a.capacity > 0 && (!a.slots || !a.positions || !a.sequences)))
      return capi_fail("plan pointers must be non-null");
    if (!on(a.page_table, 4) || !on(a.lengths, 4) || !on(a.owned, 4) || !on(a.free_pages, 4) || !on(a.free_count, 4) ||
        !on(a.new_tokens, 4) || !on(a.slots, 8) || !on(a.positions, 4) || !on(a.sequences, 4) || !on(a.starts, 4) ||
        !on(a.taken, 4) || !on(a.ticket, 4))
      return capi_fail("tensors must be aligned to their elements");
    shk::DeviceGuard guard(device_index);
    if (guard.error() != hipSuccess) return capi_fail_hip("hipSetDevice", guard.error());
    const hipError_t err = shk::launch_kv_plan(a, reinterpret_cast<hipStream_t>(stream));
    if (err != hipSuccess) return capi_fail_hip("kv_plan launch", err);
    return 0;
  });
}

int64_t amd_strix_halo_kernels_verify_workspace(const shk_verify* args) {
  int64_t bytes = -1;
  (void)capi_entry([&] {
    if (int rc = check_verify(args)) return rc;
    bytes = shk::verify_workspace(*args);
    return 0;
  });
  return bytes;
}

int amd_strix_halo_kernels_verify(int device_index, uintptr_t stream, const shk_verify* args) {
  return capi_entry([&] {
    if (int rc = check_verify(args)) return rc;
    const shk_verify& a = *args;
    if (a.batch == 0) return 0;
    if (!a.target || !a.uniforms || !a.out || !a.kept || (a.drafts > 0 && !a.tokens))
      return capi_fail("target, tokens, uniforms, out and kept pointers must be non-null");
    const uintptr_t size = a.type == SHK_SRC_F32 ? 4 : 2;
    if (!on(a.target, size) || !on(a.draft, size) || !on(a.tokens, (uintptr_t)a.token_bytes) || !on(a.uniforms, 4) ||
        !on(a.counts, 4) || !on(a.out, 8) || !on(a.kept, 4) || !on(a.lengths, 4))
      return capi_fail("tensors must be aligned to their elements");
    const int64_t need = shk::verify_workspace(a);
    if (need > 0 && (a.workspace == nullptr || a.workspace_bytes < need || !on(a.workspace, 16)))
      return capi_fail("the workspace must hold " + std::to_string(need) + " bytes, aligned to 16");
    shk::DeviceGuard guard(device_index);
    if (guard.error() != hipSuccess) return capi_fail_hip("hipSetDevice", guard.error());
    const hipError_t err = shk::launch_verify(a, reinterpret_cast<hipStream_t>(stream));
    if (err != hipSuccess) return capi_fail_hip("verify launch", err);
    return 0;
  });
}

}  // extern "C"
