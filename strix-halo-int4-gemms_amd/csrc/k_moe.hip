// The gated mixture-of-experts layer for a few tokens, on packed int4 weights
// and activations that are not quantized:
//
//   h[p] = (x[t] U_e) * silu(x[t] G_e)       for each pair p = (t, j), e = ids[t, j]
//   y[t] = sum_j share[t, j] * (h[t, j] D_e)
//
// Few tokens reach an expert, so the layer is the time to stream the weights
// of the experts that are hit: each is read once, and each pass over it
// serves all its rows.  Two products share one body (moe_product): a
// workgroup takes 64 columns (of up and of gate, or of down) of one expert,
// its eight waves a slice of K each, joined through LDS.
//
// Products are v_mfma_f32_16x16x32_bf16 with the weights in the rows and the
// tokens in the columns.  A code v enters as v + 24, which one shift and one
// and-or make of two nibbles: with n = v + 8 (the sign bit flipped), bf16's
// 0x4180 | n << 3 is 16 + n exactly.  The offset comes out as 24 times the
// sum of the token's activations, which a product with a matrix of ones gives
// in the same order and rounding; an offset of 24 against codes of up to 8
// costs about two bits of the f32 sum, against 1.25 operations a code for an
// exact one.  Activations of more bits than bf16 (f16 x, and h, which stays
// in f32 between the products) enter as two bf16 terms, high and low: 16
// bits, so no rounding between x and y is coarser than 2^-17.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <cstring>

#include "shk_common.h"
#include "shk_moe.h"

namespace shk {
namespace {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 8;
constexpr int kCols = 64;          // columns of a workgroup (of up and of gate)
constexpr int kMostPairs = 1024;   // (token, expert) pairs of a call
constexpr int kMostExperts = 1024;

struct MoeArgs {
  const void* x;
  long x_stride;
  const uint8_t* w;        // codes of this product
  const uint16_t* scale;
  const void* ids;
  const float* share;
  float* h;                // [pairs][inner]
  float* part;             // [pairs][hidden]
  void* out;
  int k, k_packed, cols;   // this product's K, its bytes, and columns (of one half)
  int group, groups;       // scale group (0: per channel) and groups of K
  int tokens, top, experts, hidden, inner;
  int type, id8;
};

__device__ __forceinline__ int id_of(const MoeArgs& a, int p) {
  const long id = a.id8 ? (long)static_cast<const int64_t*>(a.ids)[p] : (long)static_cast<const int32_t*>(a.ids)[p];
  return id >= 0 && id < a.experts ? (int)id : -1;
}

// Eight activations from element k of a row, as bf16 terms in the order
// 0 4 1 5 2 6 3 7 of the codes (expand).  Those at or past `left` are zero.
template <int TYPE>
constexpr int kTerms = TYPE == SHK_SRC_BF16 ? 1 : 2;

template <int TYPE>
__device__ __forceinline__ void load_x(const void* row, long k, int left, b8 (&t)[kTerms<TYPE>]) {
  if constexpr (TYPE == SHK_SRC_BF16) {
    uint32_t u[4] = {0, 0, 0, 0};
    const uint16_t* p = static_cast<const uint16_t*>(row) + k;
    if (left >= 8) {
      __builtin_memcpy(u, p, 16);
    } else {
      for (int i = 0; i < left; ++i) u[i / 2] |= (uint32_t)p[i] << (16 * (i % 2));
    }
    const uint32_t o[4] = {perm_b32(u[2], u[0], 0x05040100u), perm_b32(u[2], u[0], 0x07060302u),
                           perm_b32(u[3], u[1], 0x05040100u), perm_b32(u[3], u[1], 0x07060302u)};
    __builtin_memcpy(&t[0], o, 16);
  } else {
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if constexpr (TYPE == SHK_SRC_F32) {
      const float* p = static_cast<const float*>(row) + k;
      if (left >= 8) {
        __builtin_memcpy(v, p, 32);
      } else {
        for (int i = 0; i < left; ++i) v[i] = p[i];
      }
    } else {
      const _Float16* p = static_cast<const _Float16*>(row) + k;
      if (left >= 8) {
        _Float16 f[8];
        __builtin_memcpy(f, p, 16);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)f[i];
      } else {
        for (int i = 0; i < left; ++i) v[i] = (float)p[i];
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float f = v[i / 2 + 4 * (i % 2)];
      const __bf16 hi = (__bf16)f;
      t[0][i] = hi;
      t[1][i] = (__bf16)(f - (float)hi);
    }
  }
}

// The eight codes of a dword, each plus 24, in the order 0 4 1 5 2 6 3 7.
__device__ __forceinline__ b8 expand(uint32_t w) {
  w ^= 0x88888888u;
  const uint32_t o[4] = {((w << 3) & 0x00780078u) | 0x41804180u, ((w >> 1) & 0x00780078u) | 0x41804180u,
                         ((w >> 5) & 0x00780078u) | 0x41804180u, ((w >> 9) & 0x00780078u) | 0x41804180u};
  return __builtin_bit_cast(b8, *reinterpret_cast<const uint4*>(o));
}

__device__ __forceinline__ f4 mfma_bf16(b8 a, b8 b, f4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// The codes of 32 K values for the 64 columns from n0, as the operand rows of
// four products: lane (g, c) holds K k0 + 8 g .. + 7 of the columns 4 c + j.
// GUARD: the step or the columns end in this tile; bytes outside the matrix
// are not read (their products meet activations of zero, or are not stored).
template <int LAYOUT, bool GUARD>
__device__ __forceinline__ void load_w(const uint8_t* w, const MoeArgs& a, int total, int k0, int n0, int n_end,
                                       uint32_t (&o)[4]) {
  const int lane = threadIdx.x & 63, g = lane / 16, c = lane % 16;
  const int kp = k0 / 2 + 4 * g;  // first byte along K
  if constexpr (LAYOUT == SHK_LAYOUT_NT) {  // [n][k_packed]: a row's four bytes
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = GUARD ? min(n0 + 4 * c + j, n_end - 1) : n0 + 4 * c + j;
      const uint8_t* p = w + (long)n * a.k_packed + kp;
      if (!GUARD || kp + 4 <= a.k_packed) {
        __builtin_memcpy(&o[j], p, 4);
      } else {
        o[j] = 0;
        for (int i = 0; i < a.k_packed - kp; ++i) o[j] |= (uint32_t)p[i] << (8 * i);
      }
    }
  } else {  // [k_packed][n]: four rows of four columns, transposed
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = GUARD ? min(kp + i, a.k_packed - 1) : kp + i, n = n0 + 4 * c;
      const uint8_t* p = w + (long)row * total + n;
      if (!GUARD || n + 4 <= n_end) {
        __builtin_memcpy(&r[i], p, 4);
      } else {
        r[i] = 0;
        for (int j = 0; j < n_end - n; ++j) r[i] |= (uint32_t)p[j] << (8 * j);
      }
    }
    transpose4x4(r[0], r[1], r[2], r[3], o[0], o[1], o[2], o[3]);
  }
}

// One product of the layer.  HALVES 2: up and gate, h = up * silu(gate) to
// a.h; HALVES 1: down, to a.part.  RT: row tiles of 16 tokens a pass.
template <int LAYOUT, int HALVES, int RT, int TYPE>
__global__ __launch_bounds__(64 * kWaves, 2) void moe_product(const MoeArgs a) {
  constexpr int kTiles = 4 * HALVES, kPitch = kCols * HALVES + 4;
  __shared__ float red[kWaves][16 * kPitch];
  __shared__ uint16_t list[kMostPairs];
  __shared__ int count[kMostExperts];
  const int lane = threadIdx.x & 63, g = lane / 16, c = lane % 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int pairs = a.tokens * a.top;

  // the blockIdx.y-th expert that is hit, and its pairs in order
  for (int e = threadIdx.x; e < a.experts; e += 64 * kWaves) count[e] = 0;
  __syncthreads();
  for (int p = threadIdx.x; p < pairs; p += 64 * kWaves) {
    const int e = id_of(a, p);
    if (e >= 0) atomicAdd(&count[e], 1);
  }
  __syncthreads();
  int expert = -1, rank = blockIdx.y;
  for (int e0 = 0; e0 < a.experts; e0 += 64) {
    unsigned long hit = __ballot(e0 + lane < a.experts && count[e0 + lane] > 0);
    const int here = __popcll(hit);
    if (rank < here) {
      for (int i = 0; i < rank; ++i) hit &= hit - 1;
      expert = e0 + __builtin_ctzll(hit);
      break;
    }
    rank -= here;
  }
  expert = __builtin_amdgcn_readfirstlane(expert);
  if (expert < 0) return;  // the same for all threads
  const int rows = count[expert];
  if (wave == 0) {
    int at = 0;
    for (int p0 = 0; p0 < pairs; p0 += 64) {
      const bool mine = p0 + lane < pairs && id_of(a, p0 + lane) == expert;
      const unsigned long all = __ballot(mine);
      if (mine) list[at + __popcll(all & ((1ul << lane) - 1))] = (uint16_t)(p0 + lane);
      at += __popcll(all);
    }
  }
  __syncthreads();

  const int n0 = blockIdx.x * kCols, total = a.cols * HALVES;
  const uint8_t* w = a.w + (long)expert * total * a.k_packed;
  const uint16_t* scale = a.scale + (long)expert * (a.group ? a.groups : 1) * total;
  const bool edge = n0 + kCols > a.cols;

  // this wave's K: whole scale groups, in steps of 32
  const int unit = a.group > 32 ? a.group : 32;
  const int units = (a.k + unit - 1) / unit, each = (units + kWaves - 1) / kWaves;
  const int k_first = wave * each * unit, k_last = min(a.k, (wave + 1) * each * unit);

  const __bf16 one = (__bf16)1.0f;
  const b8 ones = {one, one, one, one, one, one, one, one};

  for (int row0 = 0; row0 < rows; row0 += 16 * RT) {
    const void* src[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int r = row0 + 16 * t + c;
      src[t] = nullptr;
      if (r < rows) {
        const int p = list[r];
        if constexpr (HALVES == 2)
          src[t] = static_cast<const uint8_t*>(a.x) + (long)(p / a.top) * a.x_stride * (TYPE == SHK_SRC_F32 ? 4 : 2);
        else
          src[t] = a.h + (long)p * a.inner;
      }
    }
    f4 acc[RT][kTiles], sum[RT], all[RT][kTiles];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      sum[t] = f4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < kTiles; ++j) acc[t][j] = all[t][j] = f4{0, 0, 0, 0};
    }
    for (int k0 = k_first; k0 < k_last; k0 += 32) {
      b8 x[RT][kTerms<TYPE>];
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const int left = src[t] == nullptr ? 0 : a.k - (k0 + 8 * g);
        load_x<TYPE>(src[t], k0 + 8 * g, left, x[t]);
      }
#pragma unroll
      for (int half = 0; half < HALVES; ++half) {
        uint32_t codes[4];
        const int from = n0 + half * a.cols, end = (half + 1) * a.cols;
        if (edge || k0 + 32 > a.k) load_w<LAYOUT, true>(w, a, total, k0, from, end, codes);
        else load_w<LAYOUT, false>(w, a, total, k0, from, end, codes);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const b8 v = expand(codes[j]);
#pragma unroll
          for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int i = 0; i < kTerms<TYPE>; ++i) acc[t][4 * half + j] = mfma_bf16(v, x[t][i], acc[t][4 * half + j]);
        }
      }
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int i = 0; i < kTerms<TYPE>; ++i) sum[t] = mfma_bf16(ones, x[t][i], sum[t]);
      if (a.group && (k0 + 32 >= k_last || (k0 + 32) % a.group == 0)) {
        // the group ends: its sums, without the offset, times its scales
        const uint16_t* s = scale + (long)(k0 / a.group) * total;
#pragma unroll
        for (int half = 0; half < HALVES; ++half)
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int n = n0 + 16 * g + 4 * r + j;
              const float f = load_bf16(s + half * a.cols + min(n, a.cols - 1));
#pragma unroll
              for (int t = 0; t < RT; ++t)
                all[t][4 * half + j][r] += f * (acc[t][4 * half + j][r] - 24.0f * sum[t][r]);
            }
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          sum[t] = f4{0, 0, 0, 0};
#pragma unroll
          for (int j = 0; j < kTiles; ++j) acc[t][j] = f4{0, 0, 0, 0};
        }
      }
    }
    // the waves' sums; lane (g, c) holds token c, columns 16 g + 4 r + j
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      __syncthreads();
#pragma unroll
      for (int half = 0; half < HALVES; ++half)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          f4 v;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            v[j] = a.group ? all[t][4 * half + j][r] : acc[t][4 * half + j][r] - 24.0f * sum[t][r];
          *reinterpret_cast<f4*>(&red[wave][c * kPitch + half * kCols + 16 * g + 4 * r]) = v;
        }
      __syncthreads();
      const int here = min(rows - row0 - 16 * t, 16);
      for (int i = threadIdx.x; i < here * kCols; i += 64 * kWaves) {
        const int r = i / kCols, n = i % kCols;
        if (n0 + n >= a.cols) continue;
        float v[HALVES];
#pragma unroll
        for (int half = 0; half < HALVES; ++half) {
          v[half] = 0.0f;
#pragma unroll
          for (int q = 0; q < kWaves; ++q) v[half] += red[q][r * kPitch + half * kCols + n];
          if (!a.group) v[half] *= load_bf16(scale + half * a.cols + n0 + n);
        }
        const long p = list[row0 + 16 * t + r];
        if constexpr (HALVES == 2) a.h[p * a.inner + n0 + n] = v[0] * (v[1] / (1.0f + __expf(-v[1])));
        else a.part[p * a.hidden + n0 + n] = v[0];
      }
    }
  }
}

// y[t] = sum_j share[t, j] * part[t, j], in the order of j.
__global__ __launch_bounds__(256) void moe_join(const MoeArgs a) {
  const long at = (long)blockIdx.x * 256 + threadIdx.x;
  if (at >= (long)a.tokens * a.hidden) return;
  const int t = (int)(at / a.hidden), n = (int)(at - (long)t * a.hidden);
  float y = 0.0f;
  for (int j = 0; j < a.top; ++j) {
    const int p = t * a.top + j;
    if (id_of(a, p) >= 0) y += a.share[p] * a.part[(long)p * a.hidden + n];
  }
  if (a.type == SHK_SRC_BF16) static_cast<uint16_t*>(a.out)[at] = (uint16_t)f32_to_bf16_rne(y);
  else static_cast<_Float16*>(a.out)[at] = (_Float16)y;
}

template <int LAYOUT, int HALVES, int TYPE>
void launch_product(const MoeArgs& a, dim3 grid, hipStream_t s) {
  if (a.tokens <= 16) hipLaunchKernelGGL((moe_product<LAYOUT, HALVES, 1, TYPE>), grid, dim3(64 * kWaves), 0, s, a);
  else hipLaunchKernelGGL((moe_product<LAYOUT, HALVES, 2, TYPE>), grid, dim3(64 * kWaves), 0, s, a);
}

hipError_t launch_join(const MoeArgs& a, hipStream_t s) {
  const long values = (long)a.tokens * a.hidden;
  hipLaunchKernelGGL(moe_join, dim3((unsigned)((values + 255) / 256)), dim3(256), 0, s, a);
  return hipGetLastError();
}

template <int LAYOUT>
hipError_t launch_layout(const shk_moe& x, MoeArgs a, hipStream_t s) {
  const unsigned hit = (unsigned)std::min(x.tokens * x.top, x.experts);
  a.w = static_cast<const uint8_t*>(x.up_gate);
  a.scale = static_cast<const uint16_t*>(x.up_gate_scale);
  a.k = a.hidden, a.k_packed = (a.hidden + 1) / 2, a.cols = a.inner;
  a.groups = a.group ? (a.k + a.group - 1) / a.group : 1;
  dim3 grid((unsigned)((a.cols + kCols - 1) / kCols), hit);
  hipError_t err = hipSuccess;
  if (hit == 0) return launch_join(a, s);
  if (x.type == SHK_SRC_BF16) launch_product<LAYOUT, 2, SHK_SRC_BF16>(a, grid, s);
  else launch_product<LAYOUT, 2, SHK_SRC_F16>(a, grid, s);
  err = hipGetLastError();
  if (err != hipSuccess) return err;
  a.w = static_cast<const uint8_t*>(x.down);
  a.scale = static_cast<const uint16_t*>(x.down_scale);
  a.k = a.inner, a.k_packed = (a.inner + 1) / 2, a.cols = a.hidden;
  a.groups = a.group ? (a.k + a.group - 1) / a.group : 1;
  grid.x = (unsigned)((a.cols + kCols - 1) / kCols);
  launch_product<LAYOUT, 1, SHK_SRC_F32>(a, grid, s);
  err = hipGetLastError();
  return err != hipSuccess ? err : launch_join(a, s);
}

}  // namespace

int64_t moe_workspace(const shk_moe& a) { return a.tokens * a.top * (a.inner + a.hidden) * 4; }

hipError_t launch_moe(const shk_moe& x, hipStream_t s) {
  MoeArgs a{};
  a.x = x.x, a.x_stride = x.x_stride;
  a.ids = x.ids, a.id8 = x.id_bytes == 8;
  a.share = x.share;
  a.h = static_cast<float*>(x.workspace);
  a.part = a.h + x.tokens * x.top * x.inner;
  a.out = x.out;
  a.group = (int)x.group;
  a.tokens = (int)x.tokens, a.top = (int)x.top, a.experts = (int)x.experts;
  a.hidden = (int)x.hidden, a.inner = (int)x.inner;
  a.type = (int)x.type;
  return x.layout == SHK_LAYOUT_NT ? launch_layout<SHK_LAYOUT_NT>(x, a, s) : launch_layout<SHK_LAYOUT_NN>(x, a, s);
}

}  // namespace shk
