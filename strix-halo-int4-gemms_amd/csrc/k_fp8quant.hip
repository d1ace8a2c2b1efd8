// Values to 8-bit floating point with a scale for each block of 128:
//   s = fl32(max|x| / L),  c = fp8(clamp(fl32(x / s), -L, L)),
// L = 448 (e4m3) or 57344 (e5m2).  One pass over memory: a block's values stay
// in registers between the maximum and the codes.
//
// fp8_rows: blocks of one row by 128 columns; 16 lanes hold one, 8 values each (of
// ROWS rows).
// fp8_tile: a workgroup holds 128 rows by 128 columns, a thread 8 rows by 8
// columns; for blocks of 128 x 128, and for the operand x^T, whose blocks of one
// row are x's columns.  Transposed codes pass through LDS in units of 8 bytes
// (8 rows of one column), unit u of column c at c * 128 + 8 * (u ^ (c / 8)): both
// sides are spread over the banks (18% of the LDS's cycles are conflicts, and it is
// busy 11% of the time).
// Bound by memory.  11008 x 4096 bf16 (135 MB): rows 27 us, 5 TB/s; tiles 26 to 29,
// transposed too.  16-bit values wait in registers as they are: as f32 they take
// twice as many, a third of the tiles waits for the others, and it was 35 to 38.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "shk_common.h"
#include "shk_fp8.h"
#include "shk_lanes.h"
#include "shk_loads.h"

namespace shk {
namespace {

struct Convert {
  const uint8_t* x;
  long rows, cols, stride;  // elements
  uint8_t* codes;
  long pitch;
  float* scales;
  long s_row, s_block;
};

template <int TYPE>
constexpr int kSize = TYPE == SHK_SRC_F32 ? 4 : 2;

// Eight values as they are in memory.
template <int TYPE>
struct Eight {
  u4 u[kSize<TYPE> / 2];
  __device__ __forceinline__ float operator[](int e) const {
    if constexpr (TYPE == SHK_SRC_F32) return __uint_as_float(u[e / 4][e % 4]);
    const uint16_t h = (uint16_t)(u[0][e / 2] >> (16 * (e % 2)));
    return TYPE == SHK_SRC_BF16 ? bf16_bits_to_f32(h) : (float)__builtin_bit_cast(_Float16, h);
  }
};

// x[at .. at + 8), zeros behind the `count` of them that lie inside.  Whole ones
// come in vectors, of any alignment.
template <int TYPE>
__device__ __forceinline__ Eight<TYPE> load8(const uint8_t* x, long at, long count) {
  Eight<TYPE> v;
  if (count >= 8) {
    const any_u4* src = reinterpret_cast<const any_u4*>(x + at * kSize<TYPE>);
#pragma unroll
    for (int i = 0; i < kSize<TYPE> / 2; ++i) v.u[i] = src[i];
    return v;
  }
#pragma unroll
  for (int i = 0; i < kSize<TYPE> / 2; ++i) v.u[i] = u4{0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < count) {
      if constexpr (TYPE == SHK_SRC_F32) v.u[e / 4][e % 4] = reinterpret_cast<const uint32_t*>(x)[at + e];
      else v.u[0][e / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(x)[at + e] << (16 * (e % 2));
    }
  return v;
}

// Magnitudes compare as integers: a NaN is larger than an infinity, and stays.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

template <int KIND>
constexpr float kLargest = KIND == SHK_FP8_E4M3 ? 448.f : 57344.f;

template <int KIND>
__device__ __forceinline__ float scale_of(uint32_t most) { return __uint_as_float(most) / kLargest<KIND>; }

// fl32(x / s) by a reciprocal, its product and one exact remainder (Markstein's
// theorem) where no step leaves the normal range, else by division; what
// underflows on the way rounds to a code of 0 either way.
template <int KIND>
__device__ __forceinline__ void codes8(const float (&v)[8], float s, float inv, bool plain, uint32_t (&w)[2]) {
  const bool usable = s > 0.f && s < __builtin_inff();
  float q[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float r;
    if (plain) {
      const float q0 = v[e] * inv;
      r = __builtin_fmaf(__builtin_fmaf(-q0, s, v[e]), inv, q0);
    } else {
      r = v[e] / s;
    }
    q[e] = usable ? __builtin_fminf(__builtin_fmaxf(r, -kLargest<KIND>), kLargest<KIND>) : 0.f;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    int u = 0;
    if constexpr (KIND == SHK_FP8_E4M3) {
      u = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * h], q[4 * h + 1], u, false);
      u = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * h + 2], q[4 * h + 3], u, true);
    } else {
      u = __builtin_amdgcn_cvt_pk_bf8_f32(q[4 * h], q[4 * h + 1], u, false);
      u = __builtin_amdgcn_cvt_pk_bf8_f32(q[4 * h + 2], q[4 * h + 3], u, true);
    }
    w[h] = (uint32_t)u;
  }
}

__device__ __forceinline__ bool normal_scale(float s) { return s > 0x1p-60f && s < 0x1p60f; }

// The first `count` of 8 bytes.
__device__ __forceinline__ void store8(uint8_t* to, const uint32_t (&w)[2], long count) {
  if (count >= 8) {
    *reinterpret_cast<any_u2*>(to) = u2{w[0], w[1]};
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < count) to[e] = (uint8_t)(w[e / 4] >> (8 * (e % 4)));
}

template <int TYPE, int KIND, int ROWS>
__global__ __launch_bounds__(256) void fp8_rows(const Convert p) {
  const long blocks = (p.cols + 127) / 128;
  const long unit = (long)blockIdx.x * 16 + threadIdx.x / 16;
  const int part = threadIdx.x % 16;
  const long group = unit / blocks, block = unit - group * blocks, row = group * ROWS;
  if (row >= p.rows) return;  // all 16 lanes of a block
  const long at = block * 128 + part * 8;
  Eight<TYPE> x[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) x[i] = load8<TYPE>(p.x, (row + i) * p.stride + at, row + i < p.rows ? p.cols - at : 0);
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const float v[8] = {x[i][0], x[i][1], x[i][2], x[i][3], x[i][4], x[i][5], x[i][6], x[i][7]};
    uint32_t most = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) most = max(most, magnitude(v[e]));
#pragma unroll
    for (int d = 1; d < 16; d *= 2) most = max(most, across(most, d));
    const float s = scale_of<KIND>(most);
    uint32_t w[2];
    codes8<KIND>(v, s, 1.f / s, normal_scale(s), w);
    if (row + i >= p.rows) break;
    if (at < p.cols) store8(p.codes + (row + i) * p.pitch + at, w, p.cols - at);
    if (part == 0) p.scales[(row + i) * p.s_row + block * p.s_block] = s;
  }
}

// Transposed codes of column c of a tile, 16 rows of it, from LDS.
__device__ __forceinline__ void store_turned(const Convert& p, const uint8_t* lds, int c, int piece, long c0, long r0) {
  const int g = c / 8;
  uint4 w = *reinterpret_cast<const uint4*>(lds + c * 128 + 16 * (piece ^ (g >> 1)));
  if (g & 1) w = make_uint4(w.z, w.w, w.x, w.y);
  const long out = c0 + c, at = r0 + piece * 16, count = p.rows - at;
  if (out >= p.cols || count <= 0) return;
  uint8_t* to = p.codes + out * p.pitch + at;
  if (count >= 16) {
    *reinterpret_cast<any_u4*>(to) = u4{w.x, w.y, w.z, w.w};
    return;
  }
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int e = 0; e < 16; ++e)
    if (e < count) to[e] = (uint8_t)(u[e / 4] >> (8 * (e % 4)));
}

template <int TYPE, int KIND, bool TURN, bool WHOLE>  // WHOLE: one scale for the tile
__global__ __launch_bounds__(256) void fp8_tile(const Convert p) {
  __shared__ __align__(16) uint8_t lds[TURN ? 128 * 128 : 16];
  __shared__ uint32_t tops[4][128];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int cg = threadIdx.x % 16, rg = threadIdx.x / 16;
  const long c0 = (long)blockIdx.x * 128, r0 = (long)blockIdx.y * 128;
  Eight<TYPE> v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const long row = r0 + rg * 8 + i, at = c0 + cg * 8;
    v[i] = load8<TYPE>(p.x, row * p.stride + at, row < p.rows ? p.cols - at : 0);
  }
  uint32_t top[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    top[e] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top[e] = max(top[e], magnitude(v[i][e]));
    top[e] = max(top[e], (uint32_t)__shfl_xor((int)top[e], 16, 64));
    top[e] = max(top[e], (uint32_t)__shfl_xor((int)top[e], 32, 64));
  }
  // values of 16 bits stay as they came, not as twice the registers of f32
  if constexpr (TYPE != SHK_SRC_F32)
#pragma unroll
    for (int i = 0; i < 8; ++i) asm volatile("" : "+v"(v[i].u[0]));
  if constexpr (WHOLE) {
#pragma unroll
    for (int e = 1; e < 8; ++e) top[0] = max(top[0], top[e]);
#pragma unroll
    for (int d = 1; d < 16; d *= 2) top[0] = max(top[0], across(top[0], d));
    if (lane == 0) tops[wave][0] = top[0];
  } else if (lane < 16) {
#pragma unroll
    for (int e = 0; e < 8; ++e) tops[wave][cg * 8 + e] = top[e];
  }
  __syncthreads();
  float s[8], inv[8];
  bool plain = true;
#pragma unroll
  for (int e = 0; e < (WHOLE ? 1 : 8); ++e) {
    uint32_t t = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) t = max(t, tops[w][WHOLE ? 0 : cg * 8 + e]);
    s[e] = scale_of<KIND>(t);
    inv[e] = 1.f / s[e];
    plain &= normal_scale(s[e]);
  }
  if constexpr (WHOLE) {
    if (threadIdx.x == 0)
      p.scales[TURN ? blockIdx.x * p.s_row + blockIdx.y * p.s_block : blockIdx.y * p.s_row + blockIdx.x * p.s_block] = s[0];
  } else if (rg == 0) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c0 + cg * 8 + e < p.cols) p.scales[(c0 + cg * 8 + e) * p.s_row + blockIdx.y * p.s_block] = s[e];
  }
  if constexpr (!TURN) {
    static_assert(TURN || WHOLE, "blocks of one row are fp8_rows'");
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const long row = r0 + rg * 8 + i, at = c0 + cg * 8;
      const float line[8] = {v[i][0], v[i][1], v[i][2], v[i][3], v[i][4], v[i][5], v[i][6], v[i][7]};
      uint32_t w[2];
      codes8<KIND>(line, s[0], inv[0], plain, w);
      if (row < p.rows && at < p.cols) store8(p.codes + row * p.pitch + at, w, p.cols - at);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float column[8] = {v[0][e], v[1][e], v[2][e], v[3][e], v[4][e], v[5][e], v[6][e], v[7][e]};
      uint32_t w[2];
      const float se = s[WHOLE ? 0 : e];
      codes8<KIND>(column, se, inv[WHOLE ? 0 : e], WHOLE ? plain : normal_scale(se), w);
      *reinterpret_cast<uint2*>(lds + (cg * 8 + e) * 128 + 8 * (rg ^ cg)) = make_uint2(w[0], w[1]);
    }
    __syncthreads();
#pragma unroll
    for (int pass = 0; pass < 4; ++pass) store_turned(p, lds, pass * 32 + threadIdx.x / 8, threadIdx.x % 8, c0, r0);
  }
}

// The same with 16 waves, a thread 8 rows by 2 columns, for few tiles: a CU then has
// one or two, whose loads and conversions are what takes the time.
template <int TYPE, int KIND, bool TURN, bool WHOLE>
__global__ __launch_bounds__(1024) void fp8_tile_thin(const Convert p) {
  __shared__ __align__(16) uint8_t lds[TURN ? 128 * 128 : 16];
  __shared__ __align__(16) uint32_t tops[16][WHOLE ? 4 : 128];
  const int lane = threadIdx.x & 63, rg = threadIdx.x >> 6, col = 2 * lane;
  const long c0 = (long)blockIdx.x * 128, r0 = (long)blockIdx.y * 128, count = p.cols - c0 - col;
  float v[2][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const long row = r0 + rg * 8 + i;
    const uint8_t* at = p.x + (row * p.stride + c0 + col) * kSize<TYPE>;
    uint32_t u[2] = {0, 0};
    if (row < p.rows && count > 0) {
      if constexpr (TYPE == SHK_SRC_F32) {
        if (count > 1) {
          const u2 w = *reinterpret_cast<const any_u2*>(at);
          u[0] = w[0], u[1] = w[1];
        } else {
          u[0] = *reinterpret_cast<const uint32_t*>(at);
        }
      } else {
        const uint32_t w = count > 1 ? *reinterpret_cast<const any_u32*>(at) : *reinterpret_cast<const uint16_t*>(at);
        u[0] = w & 0xFFFFu, u[1] = w >> 16;
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e)
      v[e][i] = TYPE == SHK_SRC_F32    ? __uint_as_float(u[e])
                : TYPE == SHK_SRC_BF16 ? bf16_bits_to_f32((uint16_t)u[e])
                                       : (float)__builtin_bit_cast(_Float16, (uint16_t)u[e]);
  }
  uint32_t top[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e) top[e] = max(top[e], magnitude(v[e][i]));
  if constexpr (WHOLE) {
    top[0] = max(top[0], top[1]);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) top[0] = max(top[0], across(top[0], d));
    if (lane == 0) tops[rg][0] = top[0];
  } else {
    *reinterpret_cast<uint2*>(&tops[rg][col]) = make_uint2(top[0], top[1]);
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    if constexpr (WHOLE) {
      top[0] = max(top[0], tops[w][0]);
    } else {
      const uint2 t = *reinterpret_cast<const uint2*>(&tops[w][col]);
      top[0] = max(top[0], t.x), top[1] = max(top[1], t.y);
    }
  }
  uint32_t w[2][2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const float s = scale_of<KIND>(top[WHOLE ? 0 : e]);
    codes8<KIND>(v[e], s, 1.f / s, normal_scale(s), w[e]);
    if constexpr (WHOLE) {
      if (threadIdx.x == 0 && e == 0)
        p.scales[TURN ? blockIdx.x * p.s_row + blockIdx.y * p.s_block : blockIdx.y * p.s_row + blockIdx.x * p.s_block] = s;
    } else {
      if (rg == 0 && count > e) p.scales[(c0 + col + e) * p.s_row + blockIdx.y * p.s_block] = s;
    }
  }
  if constexpr (!TURN) {
    static_assert(TURN || WHOLE, "blocks of one row are fp8_rows'");
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const long row = r0 + rg * 8 + i;
      uint8_t* to = p.codes + row * p.pitch + c0 + col;
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (row < p.rows && count > e) to[e] = (uint8_t)(w[e][i / 4] >> (8 * (i % 4)));
    }
  } else {
#pragma unroll
    for (int e = 0; e < 2; ++e)
      *reinterpret_cast<uint2*>(lds + (col + e) * 128 + 8 * (rg ^ (col / 8))) = make_uint2(w[e][0], w[e][1]);
    __syncthreads();
    const int c = threadIdx.x / 8, piece = threadIdx.x % 8;
    store_turned(p, lds, c, piece, c0, r0);
  }
}

template <int TYPE, int KIND>
hipError_t launch(const Convert& p, bool turn, bool whole, hipStream_t s) {
  if (!turn && !whole) {
    // two rows a lane of 16-bit values where there are blocks for several rounds of
    // the chip: 8192 x 4096 bf16 21.4 us and 24.7 with one, 4096 x 4096 12.9 and
    // 13.2, but 1024 x 4096 6.1 and 5.5; f32 gains nothing (29.5 and 29.3)
    const long blocks = (p.cols + 127) / 128;
    const bool two = TYPE != SHK_SRC_F32 && p.rows * blocks >= 1 << 17;
    const long units = (two ? (p.rows + 1) / 2 : p.rows) * blocks;
    const dim3 grid((unsigned)((units + 15) / 16));
    if (two) hipLaunchKernelGGL((fp8_rows<TYPE, KIND, TYPE == SHK_SRC_F32 ? 1 : 2>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((fp8_rows<TYPE, KIND, 1>), grid, dim3(256), 0, s, p);
  } else {
    const dim3 grid((unsigned)((p.cols + 127) / 128), (unsigned)((p.rows + 127) / 128));
    // few tiles: 300 x 600 transposed 6.8 us and 9.6 by whole vectors, 1000 x 1040 7.0
    // and 9.2, 2048 x 4096 10.1 and 11.1, but 4096 x 4096 17.0 and 15.7; with one scale
    // a tile 1000 x 1040 6.1 and 7.9, but 2048 x 2048 7.5 and 7.0
    if ((long)grid.x * grid.y <= (turn && !whole ? 512 : 128)) {
      if (!turn) hipLaunchKernelGGL((fp8_tile_thin<TYPE, KIND, false, true>), grid, dim3(1024), 0, s, p);
      else if (whole) hipLaunchKernelGGL((fp8_tile_thin<TYPE, KIND, true, true>), grid, dim3(1024), 0, s, p);
      else hipLaunchKernelGGL((fp8_tile_thin<TYPE, KIND, true, false>), grid, dim3(1024), 0, s, p);
    } else if (!turn) hipLaunchKernelGGL((fp8_tile<TYPE, KIND, false, true>), grid, dim3(256), 0, s, p);
    else if (whole) hipLaunchKernelGGL((fp8_tile<TYPE, KIND, true, true>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((fp8_tile<TYPE, KIND, true, false>), grid, dim3(256), 0, s, p);
  }
  return hipGetLastError();
}

template <int TYPE>
hipError_t launch_kind(const Convert& p, bool e5, bool turn, bool whole, hipStream_t s) {
  return e5 ? launch<TYPE, SHK_FP8_E5M2>(p, turn, whole, s) : launch<TYPE, SHK_FP8_E4M3>(p, turn, whole, s);
}

}  // namespace

hipError_t launch_fp8_quantize(const shk_fp8_quantize& a, hipStream_t s) {
  if (a.rows * a.cols == 0) return hipSuccess;
  const Convert p{static_cast<const uint8_t*>(a.x), a.rows, a.cols, a.x_stride, static_cast<uint8_t*>(a.codes),
                  a.code_pitch, a.scales, a.scale_row_stride, a.scale_block_stride};
  const bool e5 = a.kind == SHK_FP8_E5M2, turn = a.transpose != 0, whole = a.block_rows == 128;
  if (a.type == SHK_SRC_F32) return launch_kind<SHK_SRC_F32>(p, e5, turn, whole, s);
  if (a.type == SHK_SRC_F16) return launch_kind<SHK_SRC_F16>(p, e5, turn, whole, s);
  return launch_kind<SHK_SRC_BF16>(p, e5, turn, whole, s);
}

}  // namespace shk
