// What the kernels of the 8-bit floating-point products share (k_fp8.hip,
// k_fp8big.hip, k_fp8few.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "shk_common.h"
#include "shk_dma.h"
#include "shk_fp8.h"
#include "shk_loads.h"

namespace shk {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

struct Fp8Product {
  const uint8_t* a;
  const uint8_t* b;
  long a_pitch, b_pitch;
  const float* sa;
  const float* sb;
  long sa_row, sa_block, sb_row, sb_block;  // elements
  void* out;
  long out_stride;
  float* partial;   // [splits][m][n] where splits > 1
  int m, n, k;
  int tiles_m, tiles_n;
  int splits, per_split;  // blocks of K
  int out_type, b_shift;  // rows of b >> b_shift: its row of scales
};

// One block of K.  Rows of the result are b's (four of a lane group's), columns
// a's (lane % 16).
template <int KIND_A, int KIND_B>
__device__ __forceinline__ v4f mfma128(const v8i& b, const v8i& a) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, v4f{0.f, 0.f, 0.f, 0.f}, KIND_B, KIND_A, 0, 0, 0, 0);
}

// (A NaN keeps its payload, in whichever of these forms a column is stored.)
__device__ __forceinline__ void store_value(const Fp8Product& p, long at, float v) {
  if (p.out_type == SHK_SRC_F32) static_cast<float*>(p.out)[at] = v;
  else if (p.out_type == SHK_SRC_BF16) static_cast<uint16_t*>(p.out)[at] = (uint16_t)pack_bf16x2_nonan(v, 0.f);
  else static_cast<_Float16*>(p.out)[at] = (_Float16)v;
}

// Four neighbouring values of a row, in one store where they lie inside (rows of
// out start where they will: the memory unit takes vectors of any alignment).
__device__ __forceinline__ void store_four(const Fp8Product& p, int m, int n, const v4f& v) {
  const long at = (long)m * p.out_stride + n;
  if (n + 3 < p.n) {
    if (p.out_type == SHK_SRC_F32) {
      *reinterpret_cast<any_u4*>(static_cast<float*>(p.out) + at) =
          u4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
    } else {
      u2 u;
      if (p.out_type == SHK_SRC_BF16) {
        u = u2{pack_bf16x2_nonan(v[0], v[1]), pack_bf16x2_nonan(v[2], v[3])};
      } else {
        u[0] = __builtin_bit_cast(uint16_t, (_Float16)v[0]) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[1]) << 16);
        u[1] = __builtin_bit_cast(uint16_t, (_Float16)v[2]) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[3]) << 16);
      }
      *reinterpret_cast<any_u2*>(static_cast<uint16_t*>(p.out) + at) = u;
    }
    return;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (n + r < p.n) store_value(p, at + r, v[r]);
}

// The tile of a workgroup: each of the 8 XCDs takes a run of neighbours (its L2
// then holds what they share), which fills `high` tiles along M before it moves
// along N.
__device__ __forceinline__ void tile_of(const Fp8Product& p, int high, int& tm, int& tn) {
  const int tiles = p.tiles_m * p.tiles_n, xcd = blockIdx.x & 7, each = tiles >> 3, more = tiles & 7;
  const int id = xcd * each + min(xcd, more) + (int)(blockIdx.x >> 3);
  const int group = id / (high * p.tiles_n), in = id - group * high * p.tiles_n;
  const int rows = min(high, p.tiles_m - group * high);
  tm = group * high + in % rows, tn = in / rows;
}

hipError_t launch_fp8_big(Fp8Product& p, bool e5_a, bool e5_b, hipStream_t s);  // k_fp8big.hip
hipError_t launch_fp8_wide(Fp8Product& p, bool e5_a, bool e5_b, hipStream_t s);  // k_fp8wide.hip
hipError_t launch_fp8_few(Fp8Product& p, bool e5_a, bool e5_b, hipStream_t s);  // k_fp8few.hip

}  // namespace shk
