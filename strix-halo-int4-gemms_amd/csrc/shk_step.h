// What a step of a serving loop needs around its cached attention, shared with
// the C ABI: k_rotate.hip, k_kvplan.hip, k_verify.hip.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/strix_halo_gfx950.h"

namespace shk {

constexpr int kPlanBatch = 4096;  // sequences of a step
constexpr int kMostDrafts = 64;   // of a sequence: one lane tests each

hipError_t launch_rotate(const shk_kv_cache* c, const shk_rotate& a, hipStream_t s);
hipError_t launch_kv_plan(const shk_kv_plan& a, hipStream_t s);
int64_t verify_workspace(const shk_verify& a);
hipError_t launch_verify(const shk_verify& a, hipStream_t s);

}  // namespace shk
