// 8-bit floating-point products with few rows of a (a decode step's tokens): b is
// streamed from memory once.
//
// A workgroup holds 16 * NT columns of the result (rows of b) and all rows of a.
// Its eight waves take K's blocks in turn, so that together they read runs of 1
// KiB of each row of b, and nothing is shared while they do: a wave loads both
// operands' fragments straight into registers, one block ahead, multiplies a block
// for each 16 x 16 results, and folds it into its own f32 sums.  Behind the loop the
// eight sums are added in LDS, in order of the waves.
// Results of all types go through the f16 matrix unit, whose sums are f32 ones
// (k_fp8.hip says what the 8-bit one keeps): widening the codes hides behind b but
// for 1 to 3%, 16 x 11008 x 4096 in 11.1 us where the 8-bit unit takes 10.9, 32 x
// 4096 x 4096 in 9.8 and 9.6, 64 x 4096 x 1024 in 6.0 and 5.8.
// K is not cut over workgroups: 16 rows of b keep a CU's share of the memory rate
// busy, and a sum over workgroups would be another launch.
// Bound by that share: b at 4 TB/s.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "shk_fp8product.h"
#include "shk_fp8wide.h"

namespace shk {
namespace {

constexpr int kWaves = 8;

// Units `group` and `group + 4` of a block of a row.
__device__ __forceinline__ v8i load_block(const uint8_t* at) {
  return __builtin_shufflevector(__builtin_bit_cast(v4i, *reinterpret_cast<const any_u4*>(at)),
                                 __builtin_bit_cast(v4i, *reinterpret_cast<const any_u4*>(at + 64)), 0, 1, 2, 3, 4, 5, 6, 7);
}

// The same where `left` bytes of the row are left from `at` on; zeros behind them.
__device__ __forceinline__ v8i load_end(const uint8_t* at, int left) {
  v8i v{0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int h = 0; h < 2; ++h, left -= 64, at += 64) {
    if (left >= 16) {
      const u4 u = *reinterpret_cast<const any_u4*>(at);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * h + e] = (int)u[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll 1
        for (int byte = 0; byte < min(4, left - 4 * e); ++byte) v[4 * h + e] |= (int)at[4 * e + byte] << (8 * byte);
    }
  }
  return v;
}

template <int MT, int NT, int KIND_A, int KIND_B, bool BROW>
__global__ __launch_bounds__(64 * kWaves) void fp8_few_kernel(const Fp8Product p) {
  __shared__ v4f sums[kWaves][MT * NT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row_in = lane & 15, group = lane >> 4, n0 = blockIdx.x * 16 * NT;
  const int whole = p.k >> 7, left = (p.k & 127) - 16 * group;  // left: of the last block, from this lane's bytes on
  const uint8_t *a[MT], *b[NT];
  const float* sa[MT];
#pragma unroll
  for (int x = 0; x < MT; ++x) {
    const long m = min(x * 16 + row_in, p.m - 1);
    a[x] = p.a + m * p.a_pitch + 16 * group, sa[x] = p.sa + m * p.sa_row;
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) b[j] = p.b + (long)min(n0 + j * 16 + row_in, p.n - 1) * p.b_pitch + 16 * group;

  struct Block {
    v8i a[MT], b[NT];
    float sa[MT];
    float sb[NT][BROW ? 4 : 1];
  };
  auto load_scales = [&](int kb, Block& f) {
#pragma unroll
    for (int x = 0; x < MT; ++x) f.sa[x] = sa[x][kb * p.sa_block];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int r = 0; r < (BROW ? 4 : 1); ++r) {
        const int n = BROW ? min(n0 + j * 16 + group * 4 + r, p.n - 1) : min(n0 + j * 16, p.n - 1) >> 7;
        f.sb[j][r] = p.sb[n * p.sb_row + kb * p.sb_block];
      }
  };
  auto load = [&](int kb, Block& f) {
#pragma unroll
    for (int j = 0; j < NT; ++j) f.b[j] = load_block(b[j] + kb * 128);
#pragma unroll
    for (int x = 0; x < MT; ++x) f.a[x] = load_block(a[x] + kb * 128);
    load_scales(kb, f);
  };
  v4f acc[MT][NT];
#pragma unroll
  for (int x = 0; x < MT; ++x)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[x][j] = v4f{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](const Block& f) {
#pragma unroll
    for (int x = 0; x < MT; ++x)
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const v4f t = product128<KIND_A, KIND_B, true>(f.b[j], f.a[x]);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          acc[x][j][r] = __builtin_fmaf(t[r], f.sa[x] * f.sb[j][BROW ? r : 0], acc[x][j][r]);
      }
  };
  Block next;
  if (wave < whole) load(wave, next);
  for (int kb = wave; kb < whole; kb += kWaves) {
    const Block now = next;
    if (kb + kWaves < whole) load(kb + kWaves, next);
    multiply(now);
  }
  if ((p.k & 127) != 0 && whole % kWaves == wave) {  // K ends in a block
#pragma unroll
    for (int j = 0; j < NT; ++j) next.b[j] = load_end(b[j] + whole * 128, left);
#pragma unroll
    for (int x = 0; x < MT; ++x) next.a[x] = load_end(a[x] + whole * 128, left);
    load_scales(whole, next);
    multiply(next);
  }
#pragma unroll
  for (int x = 0; x < MT; ++x)
#pragma unroll
    for (int j = 0; j < NT; ++j) sums[wave][x * NT + j][lane] = acc[x][j];
  __syncthreads();
#pragma unroll
  for (int t = 0; t < MT * NT; t += kWaves) {
    const int tile = t + wave;
    if (tile >= MT * NT) continue;
    v4f v = sums[0][tile][lane];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += sums[w][tile][lane];
    const int m = tile / NT * 16 + row_in, n = n0 + tile % NT * 16 + group * 4;
    if (m < p.m) store_four(p, m, n, v);
  }
}

template <int MT, int NT, int KIND_A, int KIND_B>
hipError_t launch(const Fp8Product& p, hipStream_t s) {
  const dim3 grid((p.n + 16 * NT - 1) / (16 * NT)), group(64 * kWaves);
  if (p.b_shift == 0) hipLaunchKernelGGL((fp8_few_kernel<MT, NT, KIND_A, KIND_B, true>), grid, group, 0, s, p);
  else hipLaunchKernelGGL((fp8_few_kernel<MT, NT, KIND_A, KIND_B, false>), grid, group, 0, s, p);
  return hipGetLastError();
}

template <int MT, int NT>
hipError_t launch_columns(const Fp8Product& p, bool e5_a, bool e5_b, hipStream_t s) {
  if (e5_a) return e5_b ? launch<MT, NT, 1, 1>(p, s) : launch<MT, NT, 1, 0>(p, s);
  return e5_b ? launch<MT, NT, 0, 1>(p, s) : launch<MT, NT, 0, 0>(p, s);
}

// As many columns a workgroup as leave each CU one, four times 16 at most: what a
// CU can have on its way is limited (41 GB/s each, measured), and every workgroup
// reads all of a.  16 x 11008 x 4096: 11.7 us with 48 columns (230 workgroups),
// 16 with 16 or 32.
template <int MT>
hipError_t launch_rows(const Fp8Product& p, bool e5_a, bool e5_b, hipStream_t s) {
  if (p.n <= 4096) return launch_columns<MT, 1>(p, e5_a, e5_b, s);
  if (p.n <= 8192) return launch_columns<MT, 2>(p, e5_a, e5_b, s);
  if (p.n <= 12288) return launch_columns<MT, 3>(p, e5_a, e5_b, s);
  return launch_columns<MT, 4>(p, e5_a, e5_b, s);
}

}  // namespace

hipError_t launch_fp8_few(Fp8Product& p, bool e5_a, bool e5_b, hipStream_t s) {
  return p.m <= 16 ? launch_rows<1>(p, e5_a, e5_b, s) : p.m <= 32 ? launch_rows<2>(p, e5_a, e5_b, s)
                                                                 : launch_columns<4, 1>(p, e5_a, e5_b, s);
}

}  // namespace shk
