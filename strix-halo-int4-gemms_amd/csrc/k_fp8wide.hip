// 8-bit floating-point products with f32 results on tiles of 128 x 128, through
// the f16 matrix unit (k_fp8.hip says why).
//
// A stage is one block of K as the copy brings it, 8 bits a value, in one of two
// LDS slots; two workgroups share a CU and fill each other's waits.  Four waves
// hold 64 x 64 each.  A wave widens b's half of the stage to f16 registers once
// and a's as it goes (128 conversions of two values, exact), multiplies with
// v_mfma_f32_32x32x16_f16 (2060 TFLOP/s from registers; the 16x16x32 form reaches
// 1215), and folds each 32 x 32 result of a block into its sums.  Bound by the
// vector unit: conversions and, where every row of b has its own scale, two
// operations a value and block make as many cycles as the MFMAs, and by power.
// 4096 x 4096 x 8064: 258 to 313 us from box to box, 1050 TFLOP/s at most, clock
// 1.75 GHz, matrix unit 48%.  Power is what holds it: with operands of one value
// 204 to 218 us, and an order fixed step by step, folds and conversions under the
// next MFMAs, took those to 193 but random ones from 246 to 250 only, and spilled
// where rows of b have scales.  Dropped too: copies spread over the stage.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "shk_fp8product.h"
#include "shk_fp8wide.h"

namespace shk {
namespace {

typedef float v16f __attribute__((ext_vector_type(16)));

constexpr int kB = 128 * 128;
constexpr int kScales = 256 * 128;
constexpr int kStage = kScales + 1024;

// Unit u of row r of a stage lies at r * 128 + 16 * (u ^ swizzle(r)): a fragment's
// 32 rows meet no bank twice in a step (with r % 8 alone, 40% of the LDS's cycles).
__device__ __forceinline__ int swizzle(int row) { return (row ^ (row >> 3)) & 7; }

template <int KIND_A, int KIND_B, bool BROW>
__global__ __launch_bounds__(256, 2) void fp8_wide_kernel(const Fp8Product p) {
  __shared__ __align__(16) uint8_t lds[2 * kStage];  // 64 KiB of it for the results, too
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int tm, tn;
  tile_of(p, 8, tm, tn);
  const int m0 = tm * 128, n0 = tn * 128;
  const int count = (p.k + 127) >> 7;
  const int rows_a = min(128, p.m - m0), rows_b = min(128, p.n - n0);
  const long row_bytes = (p.k + 15) & ~15;

  // waves 0 and 1 bring a and its scales, 2 and 3 b and its
  const bool of_a = wave < 2;
  const long pitch = of_a ? p.a_pitch : p.b_pitch;
  const int rows = of_a ? rows_a : rows_b;
  const v4i data = buffer_words(of_a ? p.a + m0 * pitch : p.b + n0 * pitch, (unsigned long long)((rows - 1) * pitch + row_bytes));
  const int s0 = n0 >> p.b_shift, s_rows = ((n0 + rows_b - 1) >> p.b_shift) - s0 + 1;
  const v4i scales =
      of_a ? buffer_words(p.sa + (long)m0 * p.sa_row, (unsigned long long)(((rows_a - 1) * p.sa_row + (count - 1) * p.sa_block + 1) * 4))
           : buffer_words(p.sb + (long)s0 * p.sb_row, (unsigned long long)(((s_rows - 1) * p.sb_row + (count - 1) * p.sb_block + 1) * 4));
  uint32_t off[8];
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    const int row = (wave & 1) * 64 + c * 8 + lane / 8;
    off[c] = (uint32_t)(min(row, rows - 1) * pitch) + 16 * ((lane & 7) ^ swizzle(row));
  }
  const int s_row = min((wave & 1) * 64 + lane, rows - 1);
  const uint32_t s_off = of_a ? (uint32_t)(s_row * p.sa_row * 4) : (uint32_t)((((n0 + s_row) >> p.b_shift) - s0) * p.sb_row * 4);
  const uint32_t s_step = (uint32_t)((of_a ? p.sa_block : p.sb_block) * 4);
  const uint32_t base = lds_address(lds), to = base + (of_a ? 0 : kB) + (wave & 1) * 8192, s_to = base + kScales + wave * 256;
  auto issue = [&](int kb, int slot) {
#pragma unroll
    for (int c = 0; c < 8; ++c) lds_dma16(data, off[c], (uint32_t)kb * 128u, to + slot * kStage + c * 1024);
    lds_dma4(scales, s_off, (uint32_t)kb * s_step, s_to + slot * kStage);
  };

  const int wm = wave & 1, wn = wave >> 1, row_in = lane & 31, half = lane >> 5;
  v16f acc[2][2];
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[x][j][r] = 0.f;

  issue(0, 0);
  for (int i = 0; i < count; ++i) {
    const uint8_t* st = lds + (i & 1) * kStage;
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (i + 1 < count) issue(i + 1, (i + 1) & 1);
    const int left = p.k - i * 128;
    if (left < 128) {  // zeros behind K
      for (int u = threadIdx.x; u < 256 * 8; u += 256) {
        const int row = u >> 3, unit = (u & 7) ^ swizzle(row), keep = left - unit * 16;
        if (keep >= 16) continue;
        uint32_t* w = reinterpret_cast<uint32_t*>(lds + (i & 1) * kStage + u * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int bytes = keep - 4 * e;
          w[e] = bytes <= 0 ? 0u : bytes >= 4 ? w[e] : w[e] & ((1u << (8 * bytes)) - 1u);
        }
      }
      __syncthreads();
    }
    // a lane's 64 values of its row: units 4 * half .. 4 * half + 3
    auto unit = [&](int row, int u) {
      return *reinterpret_cast<const v4i*>(st + row * 128 + 16 * ((4 * half + u) ^ swizzle(row)));
    };
    v8h wb[2][8];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const v4i w = unit(128 + wn * 64 + j * 32 + row_in, u);
        wb[j][2 * u] = widen<KIND_B>(w[0], w[1]), wb[j][2 * u + 1] = widen<KIND_B>(w[2], w[3]);
      }
    const float sb_all = BROW ? 0.f : *reinterpret_cast<const float*>(st + kScales + 512 + wn * 256);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      v16f t[2];
#pragma unroll
      for (int r = 0; r < 16; ++r) t[0][r] = t[1][r] = 0.f;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const v4i w = unit(wm * 64 + x * 32 + row_in, u);
        const v8h lo = widen<KIND_A>(w[0], w[1]), hi = widen<KIND_A>(w[2], w[3]);
#pragma unroll
        for (int j = 0; j < 2; ++j) t[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(wb[j][2 * u], lo, t[j], 0, 0, 0);
#pragma unroll
        for (int j = 0; j < 2; ++j) t[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(wb[j][2 * u + 1], hi, t[j], 0, 0, 0);
      }
      const float sa = *reinterpret_cast<const float*>(st + kScales + (wm * 64 + x * 32 + row_in) * 4);
      const float s = BROW ? sa : sa * sb_all;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          v4f sv;
          if constexpr (BROW) sv = *reinterpret_cast<const v4f*>(st + kScales + 512 + (wn * 64 + j * 32 + q * 8 + half * 4) * 4);
#pragma unroll
          for (int r = 0; r < 4; ++r)
            acc[x][j][q * 4 + r] = __builtin_fmaf(t[j][q * 4 + r], BROW ? s * sv[r] : s, acc[x][j][q * 4 + r]);
        }
    }
  }
  // Through LDS, so that a store is four runs of 256 bytes and not 32 of 32 (5489 x
  // 13153 x 300: 126 us, 138 without): unit u of row r of a wave's 64 x 64 lies at
  // r * 256 + 16 * (u ^ (r % 16)).
  __syncthreads();
  uint8_t* own = lds + wave * 16384;
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const v16f& v = acc[x][j];
        *reinterpret_cast<v4f*>(own + (x * 32 + row_in) * 256 + 16 * ((j * 8 + q * 2 + half) ^ (row_in & 15))) =
            v4f{v[q * 4], v[q * 4 + 1], v[q * 4 + 2], v[q * 4 + 3]};
      }
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int r = 0; r < 64; r += 4) {
    const int row = r + lane / 16, unit = lane & 15, m = m0 + wm * 64 + row;
    const v4f v = *reinterpret_cast<const v4f*>(own + row * 256 + 16 * (unit ^ (row & 15)));
    if (m < p.m) store_four(p, m, n0 + wn * 64 + unit * 4, v);
  }
}

template <int KIND_A, int KIND_B>
hipError_t launch(const Fp8Product& p, hipStream_t s) {
  const dim3 grid(p.tiles_m * p.tiles_n);
  if (p.b_shift == 0) hipLaunchKernelGGL((fp8_wide_kernel<KIND_A, KIND_B, true>), grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((fp8_wide_kernel<KIND_A, KIND_B, false>), grid, dim3(256), 0, s, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_fp8_wide(Fp8Product& p, bool e5_a, bool e5_b, hipStream_t s) {
  p.tiles_m = (p.m + 127) / 128, p.tiles_n = (p.n + 127) / 128;
  if (e5_a) return e5_b ? launch<1, 1>(p, s) : launch<1, 0>(p, s);
  return e5_b ? launch<0, 1>(p, s) : launch<0, 0>(p, s);
}

}  // namespace shk
