// The gated mixture-of-experts layer for a few tokens (k_moe.hip), shared
// with the C ABI.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/strix_halo_gfx950.h"

namespace shk {

int64_t moe_workspace(const shk_moe& a);
hipError_t launch_moe(const shk_moe& a, hipStream_t s);

}  // namespace shk
