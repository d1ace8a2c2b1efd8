// Products in 8-bit floating point with a scale for each block of 128 values of
// K (k_fp8.hip), and the conversion that makes the operands (k_fp8quant.hip),
// shared with the C ABI.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/strix_halo_gfx950.h"

namespace shk {

constexpr int kFp8Block = 128;  // values of K that share a scale

hipError_t launch_fp8_quantize(const shk_fp8_quantize& a, hipStream_t s);

// Bytes of workspace of a product: rows that do not start on 16 bytes are laid
// out there, and the partial sums of a K that several workgroups share.
int64_t fp8_mm_workspace(const shk_fp8_mm& a);
hipError_t launch_fp8_mm(const shk_fp8_mm& a, hipStream_t s);

}  // namespace shk
