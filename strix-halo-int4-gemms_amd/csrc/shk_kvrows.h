// Rows of the quantized cache in a lane's registers: 8 values in, 8 codes out
// (k_kvcache.hip, k_rotate.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/strix_halo_gfx950.h"
#include "shk_common.h"

namespace shk {

// Row of the cache, counted in rows, of (slot, head).
__device__ __forceinline__ long cache_row(long slot, int head, unsigned heads, int page_shift) {
  const long page = slot >> page_shift;
  return (((page * heads + head) << page_shift) | (slot & ((1L << page_shift) - 1)));
}

template <int TYPE>
constexpr int kSize = TYPE == SHK_SRC_F32 ? 4 : 2;

__device__ __forceinline__ float half_bits(uint32_t h) { return (float)__builtin_bit_cast(_Float16, (uint16_t)h); }

// 8 values starting at element address p; VEC: p is 16-byte aligned.
template <int TYPE, bool VEC>
__device__ __forceinline__ void load8(const uint8_t* p, float (&v)[8]) {
  if constexpr (TYPE == SHK_SRC_F32) {
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (VEC) {
        const uint4 w = reinterpret_cast<const uint4*>(p)[i];
        u[4 * i] = w.x, u[4 * i + 1] = w.y, u[4 * i + 2] = w.z, u[4 * i + 3] = w.w;
      } else {
        for (int j = 0; j < 4; ++j) u[4 * i + j] = reinterpret_cast<const uint32_t*>(p)[4 * i + j];
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(u[i]);
  } else {
    uint32_t u[4];
    if constexpr (VEC) {
      const uint4 w = *reinterpret_cast<const uint4*>(p);
      u[0] = w.x, u[1] = w.y, u[2] = w.z, u[3] = w.w;
    } else {
      const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = h[2 * i] | ((uint32_t)h[2 * i + 1] << 16);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = TYPE == SHK_SRC_BF16 ? __uint_as_float(u[i] << 16) : half_bits(u[i] & 0xFFFFu);
      v[2 * i + 1] = TYPE == SHK_SRC_BF16 ? __uint_as_float(u[i] & 0xFFFF0000u) : half_bits(u[i] >> 16);
    }
  }
}

// fl32(x / s) for 8 values.  With inv = fl32(1 / s), q = fl32(x * inv) is
// within one unit of x / s, its remainder x - q * s is exact in one fused
// multiply-add, and q + remainder * inv rounds to fl32(x / s) (Markstein's
// theorem) as long as nothing on the way leaves the normal range.  That
// holds for the scales between the bounds, where codes matter (|x / s| of 2^-30
// rounds to 0 either way); rows outside them divide.
template <int BITS>
__device__ __forceinline__ void codes8(const float (&v)[8], float s, int (&c)[8]) {
  constexpr float Q = BITS == 4 ? 7.0f : 127.0f;
  const bool usable = s > 0.0f && s < __builtin_inff();
  float q[8];
  if (s > 0x1p-60f && s < 0x1p60f) {
    const float inv = 1.0f / s;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float q0 = v[i] * inv;
      q[i] = __builtin_fmaf(__builtin_fmaf(-q0, s, v[i]), inv, q0);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = v[i] / s;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float r = __builtin_fminf(__builtin_fmaxf(__builtin_rintf(q[i]), -Q), Q);
    c[i] = usable ? (int)r : 0;
  }
}

// The 8 codes at dst, packed.
template <int BITS>
__device__ __forceinline__ void store_codes(uint8_t* dst, const int (&c)[8]) {
  if constexpr (BITS == 4) {
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) w |= ((uint32_t)c[e] & 0xFu) << (4 * e);
    *reinterpret_cast<uint32_t*>(dst) = w;
  } else {
    uint32_t lo = 0, hi = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      lo |= ((uint32_t)c[e] & 0xFFu) << (8 * e);
      hi |= ((uint32_t)c[e + 4] & 0xFFu) << (8 * e);
    }
    *reinterpret_cast<uint2*>(dst) = make_uint2(lo, hi);
  }
}

}  // namespace shk
