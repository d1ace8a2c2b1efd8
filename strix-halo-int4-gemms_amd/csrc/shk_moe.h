// The gated mixture-of-experts layer for a few tokens (k_moe.hip), shared
// with the C ABI.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/strix_halo_gfx950.h"

namespace shk {

constexpr int kMoeColumns = 128;  // columns of a workgroup's tile
constexpr int kMoePiece = 128;    // K values a wave takes at a time

// h's rows are whole pieces of K, the rest zero.
inline int64_t moe_inner_pad(const shk_moe& a) { return (a.inner + kMoePiece - 1) / kMoePiece * kMoePiece; }
inline int64_t moe_down_tiles(const shk_moe& a) { return (a.hidden + kMoeColumns - 1) / kMoeColumns; }
// h and the results of each pair, and a counter for each tile of the output.
inline int64_t moe_workspace(const shk_moe& a) {
  return a.tokens * a.top * (moe_inner_pad(a) + a.hidden) * 4 + moe_down_tiles(a) * 4;
}

hipError_t launch_moe_nn(const shk_moe& a, hipStream_t s);
hipError_t launch_moe_nt(const shk_moe& a, hipStream_t s);

}  // namespace shk
