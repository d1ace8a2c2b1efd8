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

// v plus the value of 8 bytes that CTRL moves to this lane, in the rows of ROWS (else
// plus 0).
template <int CTRL, int ROWS, class T>
__device__ __forceinline__ T plus_moved(T v) {
  static_assert(sizeof(T) == 8, "");
  const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xF, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xF, false);
  return v + __builtin_bit_cast(T, ((unsigned long long)hi << 32) | lo);
}

// Inclusive sum over a wave's lanes, all of them active: within rows of 16 by 1, 2, 4
// and 8 lanes up, then the last lane of rows 0 and 2 to the rows above them, and lane
// 31 to both rows behind it.
template <class T>
__device__ __forceinline__ T wave_inclusive(T v) {
  v = plus_moved<0x111, 0xF>(v);
  v = plus_moved<0x112, 0xF>(v);
  v = plus_moved<0x114, 0xF>(v);
  v = plus_moved<0x118, 0xF>(v);
  v = plus_moved<0x142, 0xA>(v);
  return plus_moved<0x143, 0xC>(v);
}

}  // namespace shk
