// Values of other lanes of a wave.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace shk {

// The value of another lane whose step of a reduction over 1, 2, 4.. lanes was the
// same but for the bit `d`: inside 16 lanes a move, not a way through LDS.
__device__ __forceinline__ uint32_t across(uint32_t v, int d) {
  const int i = (int)v;
  switch (d) {
    case 1: return (uint32_t)__builtin_amdgcn_update_dpp(0, i, 0xB1, 0xF, 0xF, false);   // lanes 1 0 3 2
    case 2: return (uint32_t)__builtin_amdgcn_update_dpp(0, i, 0x4E, 0xF, 0xF, false);   // lanes 2 3 0 1
    case 4: return (uint32_t)__builtin_amdgcn_update_dpp(0, i, 0x141, 0xF, 0xF, false);  // eights reversed
    case 8: return (uint32_t)__builtin_amdgcn_update_dpp(0, i, 0x140, 0xF, 0xF, false);  // sixteens reversed
    default: return (uint32_t)__shfl_xor(i, d, 64);
  }
}

}  // namespace shk
