// C ABI of the 8-bit floating-point products: argument validation and launches.
// Declarations are in include/strix_halo_gfx950.h.
#include <algorithm>
#include <climits>
#include <string>

#include "shk_capi.h"
#include "shk_fp8.h"

namespace {

using shk::capi_entry;
using shk::capi_fail;
using shk::capi_fail_hip;

bool on(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
bool kind(int64_t k) { return k == SHK_FP8_E4M3 || k == SHK_FP8_E5M2; }
bool source(int64_t t) { return t == SHK_SRC_F32 || t == SHK_SRC_F16 || t == SHK_SRC_BF16; }
int64_t blocks(int64_t n) { return (n + shk::kFp8Block - 1) / shk::kFp8Block; }

// Bytes that `rows` rows of `cols` scales span.
bool scales_fit(int64_t rows, int64_t row_stride, int64_t cols, int64_t block_stride) {
  return row_stride >= 0 && block_stride >= 0 &&
         ((__int128)(rows - 1) * row_stride + (__int128)(cols - 1) * block_stride + 1) * 4 < (1LL << 31);
}

int check_mm(const shk_fp8_mm* a) {
  if (a == nullptr) return capi_fail("product arguments must be non-null");
  if (!kind(a->a_kind) || !kind(a->b_kind)) return capi_fail("operands are e4m3 or e5m2");
  if (!source(a->out_type)) return capi_fail("unknown output type " + std::to_string(a->out_type));
  if (a->b_rows != 1 && a->b_rows != shk::kFp8Block)
    return capi_fail("b_rows is 1 or 128; got " + std::to_string(a->b_rows));
  if (a->m < 0 || a->n < 0 || a->k < 0 || a->m > INT_MAX / 4 || a->n > INT_MAX / 4 || a->k >= (1 << 23))
    return capi_fail("m and n are from 0 to 536870911, k to 8388607");
  if (a->m * a->n == 0) return 0;
  // a launch holds fewer than 2^32 work-items: 256 for 64 x 128 results (64 x 64 where
  // K has no values), 512 for 64 columns of few rows, and one for 16 bytes of an
  // operand that is copied
  const int64_t columns = a->k == 0 ? 64 : 128;
  if ((__int128)((a->m + 63) / 64) * ((a->n + columns - 1) / columns) > 0xFFFFFF || (a->m <= 32 && a->n > (1LL << 29) - 64) ||
      (a->k > 0 && std::max(a->m, a->n) > 0xFFFFFF00LL / ((a->k + 15) / 16)))
    return capi_fail("too many outputs for one launch");
  if (a->a_pitch < a->k || a->b_pitch < a->k || a->a_pitch >= (1 << 24) || a->b_pitch >= (1 << 24))
    return capi_fail("row pitches are from k to 16777215 bytes");
  if (a->out_stride < a->n) return capi_fail("rows of out must not overlap");
  if (a->k > 0 && (!scales_fit(a->m, a->a_scale_row_stride, blocks(a->k), a->a_scale_block_stride) ||
                   !scales_fit((a->n + a->b_rows - 1) / a->b_rows, a->b_scale_row_stride, blocks(a->k),
                               a->b_scale_block_stride)))
    return capi_fail("scales have strides that are not negative and span less than 2147483648 bytes");
  return 0;
}

}  // namespace

extern "C" {

int amd_strix_halo_kernels_fp8_quantize(int device_index, uintptr_t stream, const shk_fp8_quantize* args) {
  return capi_entry([&] {
    if (args == nullptr) return capi_fail("conversion arguments must be non-null");
    const shk_fp8_quantize& a = *args;
    if (!source(a.type)) return capi_fail("unknown source type " + std::to_string(a.type));
    if (!kind(a.kind)) return capi_fail("codes are e4m3 or e5m2");
    if (a.block_rows != 1 && a.block_rows != shk::kFp8Block)
      return capi_fail("block_rows is 1 or 128; got " + std::to_string(a.block_rows));
    if (a.rows < 0 || a.cols < 0 || a.rows > INT_MAX || a.cols > INT_MAX)
      return capi_fail("rows and cols are from 0 to 2147483647");
    if (a.rows * a.cols == 0) return 0;
    // a launch holds fewer than 2^32 work-items
    const bool tiles = a.transpose || a.block_rows != 1;
    if (tiles ? blocks(a.rows) > 65535 || blocks(a.rows) * blocks(a.cols) > 0xFFFFFF
              : (a.rows * blocks(a.cols) + 15) / 16 > 0xFFFFFF)
      return capi_fail("too many blocks for one launch");
    if (a.x_stride < a.cols && a.rows > 1) return capi_fail("rows of x must not overlap");
    if (a.code_pitch < (a.transpose ? a.rows : a.cols)) return capi_fail("rows of codes must not overlap");
    if (!a.x || !a.codes || !a.scales) return capi_fail("x, codes and scales pointers must be non-null");
    if (!on(a.x, a.type == SHK_SRC_F32 ? 4 : 2) || !on(a.scales, 4))
      return capi_fail("x and scales must be aligned to their elements");
    shk::DeviceGuard guard(device_index);
    if (guard.error() != hipSuccess) return capi_fail_hip("hipSetDevice", guard.error());
    const hipError_t err = shk::launch_fp8_quantize(a, reinterpret_cast<hipStream_t>(stream));
    if (err != hipSuccess) return capi_fail_hip("fp8_quantize launch", err);
    return 0;
  });
}

int64_t amd_strix_halo_kernels_fp8_mm_workspace(const shk_fp8_mm* args) {
  int64_t bytes = -1;
  (void)capi_entry([&] {
    if (int rc = check_mm(args)) return rc;
    bytes = shk::fp8_mm_workspace(*args);
    return 0;
  });
  return bytes;
}

int amd_strix_halo_kernels_fp8_mm(int device_index, uintptr_t stream, const shk_fp8_mm* args) {
  return capi_entry([&] {
    if (int rc = check_mm(args)) return rc;
    const shk_fp8_mm& a = *args;
    if (a.m * a.n == 0) return 0;
    if (!a.out || (a.k > 0 && (!a.a || !a.b || !a.a_scale || !a.b_scale)))
      return capi_fail("operand, scale and out pointers must be non-null");
    if (!on(a.a_scale, 4) || !on(a.b_scale, 4) || !on(a.out, a.out_type == SHK_SRC_F32 ? 4 : 2))
      return capi_fail("scales and out must be aligned to their elements");
    const int64_t need = shk::fp8_mm_workspace(a);
    if (need > 0 && (a.workspace == nullptr || a.workspace_bytes < need || !on(a.workspace, 16)))
      return capi_fail("the workspace must hold " + std::to_string(need) + " bytes, aligned to 16");
    shk::DeviceGuard guard(device_index);
    if (guard.error() != hipSuccess) return capi_fail_hip("hipSetDevice", guard.error());
    const hipError_t err = shk::launch_fp8_mm(a, reinterpret_cast<hipStream_t>(stream));
    if (err != hipSuccess) return capi_fail_hip("fp8_mm launch", err);
    return 0;
  });
}

}  // extern "C"
