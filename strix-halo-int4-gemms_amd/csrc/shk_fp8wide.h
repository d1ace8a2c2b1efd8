// A block of K through the f16 matrix unit, whose sums are f32 ones.
#pragma once

#include "shk_fp8product.h"

namespace shk {

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

// Eight codes of one operand as f16, which holds every one of them exactly.
template <int KIND>
__device__ __forceinline__ v8h widen(int lo, int hi) {
  v2h h[4];
  if constexpr (KIND == SHK_FP8_E4M3) {
    h[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false);
    h[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true);
    h[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false);
    h[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true);
  } else {  // the upper bytes of f16
    h[0] = __builtin_bit_cast(v2h, perm_b32(0u, lo, 0x010C000Cu));
    h[1] = __builtin_bit_cast(v2h, perm_b32(0u, lo, 0x030C020Cu));
    h[2] = __builtin_bit_cast(v2h, perm_b32(0u, hi, 0x010C000Cu));
    h[3] = __builtin_bit_cast(v2h, perm_b32(0u, hi, 0x030C020Cu));
  }
  return v8h{h[0][0], h[0][1], h[1][0], h[1][1], h[2][0], h[2][1], h[3][0], h[3][1]};
}

template <int KIND>
struct Wide {
  v8h part[4];
  __device__ __forceinline__ explicit Wide(const v8i& f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) part[i] = widen<KIND>(f[2 * i], f[2 * i + 1]);
  }
};

// One block of K, rows of the result b's, columns a's.  WIDE: by the f16 unit.
template <int KIND_A, int KIND_B, bool WIDE>
__device__ __forceinline__ v4f product128(const v8i& b, const v8i& a) {
  if constexpr (!WIDE) return mfma128<KIND_A, KIND_B>(b, a);
  const Wide<KIND_A> wa(a);
  const Wide<KIND_B> wb(b);
  v4f t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i) t = __builtin_amdgcn_mfma_f32_16x16x32_f16(wb.part[i], wa.part[i], t, 0, 0, 0);
  return t;
}

}  // namespace shk
