// Query and key heads: the norm of a head, its rotation by position, and, where
// there is a cache, the quantized keys and values, in one pass over memory.
//
// A row is a head of a token; its lanes (head_dim / 8, rounded up to a power of
// two) hold 8 values each.  The value that a lane's value turns with is read
// beside it (from L1: the same row), so that only the sum of squares crosses
// lanes.  A workgroup takes whole rounds of rows, first all its loads; while they
// are on their way its threads compute the angles of the tokens that it meets
// into LDS.  An angle is positions * turns in 64 bits, less its nearest quarter:
// what is left is at most an eighth of a turn, exact in f32 to 2^-24 of itself.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "shk_common.h"
#include "shk_kvrows.h"
#include "shk_step.h"

namespace shk {
namespace {

struct Rotate {
  const uint8_t* x[3];  // queries, keys, values
  long token_stride[3], head_stride[3];
  uint8_t* out[2];
  long out_token_stride[2], out_head_stride[2];
  const void* weight[2];
  const void* positions;
  const double* turns;
  float amplitude, eps;
  unsigned rows, per_token;  // per_token: heads + kv_heads, and kv_heads more with a cache
  unsigned heads, kv_heads;
  int dim, half, rotated;
  int position8, weight_type;
  // the cache
  uint8_t* codes[2];
  uint16_t* scales[2];
  const void* slots;
  long slots_total;
  int slot8, page_shift, bits;
};

__device__ __forceinline__ float weight_of(const Rotate& p, int which, int i) {
  if (p.weight_type == SHK_SRC_F32) return static_cast<const float*>(p.weight[which])[i];
  const uint16_t h = static_cast<const uint16_t*>(p.weight[which])[i];
  return p.weight_type == SHK_SRC_BF16 ? bf16_bits_to_f32(h) : half_bits(h);
}

template <int TYPE>
__device__ __forceinline__ float element(const uint8_t* x, long i) {
  if constexpr (TYPE == SHK_SRC_F32) return reinterpret_cast<const float*>(x)[i];
  const uint16_t h = reinterpret_cast<const uint16_t*>(x)[i];
  return TYPE == SHK_SRC_BF16 ? bf16_bits_to_f32(h) : half_bits(h);
}

// Cosine and sine of `turn` turns: the nearest quarter apart, and the series of
// both up to an eighth of a turn (the first terms left out are below 2^-28).
__device__ __forceinline__ float2 turned(double turn) {
  turn -= __builtin_rint(turn);
  const double quarter = __builtin_rint(4.0 * turn);
  const float x = (float)((turn - 0.25 * quarter) * 6.283185307179586476925);
  const float z = x * x;
  float s = __builtin_fmaf(z, 1.f / 362880.f, -1.f / 5040.f);
  s = __builtin_fmaf(z, s, 1.f / 120.f);
  s = __builtin_fmaf(z, s, -1.f / 6.f);
  s = __builtin_fmaf(z * s, x, x);
  float c = __builtin_fmaf(z, -1.f / 3628800.f, 1.f / 40320.f);
  c = __builtin_fmaf(z, c, -1.f / 720.f);
  c = __builtin_fmaf(z, c, 1.f / 24.f);
  c = __builtin_fmaf(z, c, -0.5f);
  c = __builtin_fmaf(z, c, 1.f);
  const int q = (int)quarter & 3;
  const float a = (q & 1) ? s : c, b = (q & 1) ? c : s;
  return make_float2(q == 1 || q == 2 ? -a : a, q >= 2 ? -b : b);
}

// One value rounded to its type.
template <int TYPE>
__device__ __forceinline__ float rounded(float v) {
  if constexpr (TYPE == SHK_SRC_F32) return v;
  else if constexpr (TYPE == SHK_SRC_BF16) return bf16_bits_to_f32((uint16_t)f32_to_bf16_rne(v));
  else return (float)(_Float16)v;
}

// VEC: every row starts on 16 bytes and is whole 8s, and so is `half` if pairs
// lie apart.
template <int TYPE, int LANES, bool VEC, bool APART, int ROUNDS>
__global__ __launch_bounds__(256) void rotate_kernel(const Rotate p) {
  constexpr int PER = 256 / LANES;  // rows of a round
  extern __shared__ float2 angles[];
  const int part = threadIdx.x % LANES, first_value = part * 8;
  const unsigned start = blockIdx.x * (PER * ROUNDS), mine = start + threadIdx.x / LANES;
  const bool inside = first_value < p.dim;
  const int count = min(8, p.dim - first_value);
  float v[ROUNDS][8], w[ROUNDS][8];
  unsigned token[ROUNDS], head[ROUNDS];
  int kind[ROUNDS];
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i) {
    const unsigned row = mine + i * PER;
    token[i] = row / p.per_token;
    const unsigned h = row - token[i] * p.per_token;
    kind[i] = row >= p.rows || !inside ? -1 : h < p.heads ? 0 : h < p.heads + p.kv_heads ? 1 : 2;
    head[i] = kind[i] == 0 ? h : kind[i] == 1 ? h - p.heads : h - p.heads - p.kv_heads;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[i][e] = w[i][e] = 0.f;
    if (kind[i] < 0) continue;
    const uint8_t* x = p.x[kind[i]] + ((long)token[i] * p.token_stride[kind[i]] + (long)head[i] * p.head_stride[kind[i]]) *
                                          kSize<TYPE>;
    if constexpr (VEC) {
      load8<TYPE, true>(x + first_value * kSize<TYPE>, v[i]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < count) v[i][e] = element<TYPE>(x, first_value + e);
    }
    if (APART && kind[i] < 2 && first_value < p.rotated) {
      if constexpr (VEC) {
        load8<TYPE, true>(x + (first_value < p.half ? first_value + p.half : first_value - p.half) * kSize<TYPE>, w[i]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int at = first_value + e;
          if (at < p.rotated) w[i][e] = element<TYPE>(x, at < p.half ? at + p.half : at - p.half);
        }
      }
    }
  }
  const unsigned last = min(start + PER * ROUNDS, p.rows) - 1, token0 = start / p.per_token;
  const unsigned tokens = last / p.per_token - token0 + 1;
  for (unsigned i = threadIdx.x; i < tokens * p.half; i += 256) {
    const unsigned t = i / p.half;
    const long at = token0 + t;
    const double position = p.position8 ? (double)static_cast<const int64_t*>(p.positions)[at]
                                        : (double)static_cast<const int32_t*>(p.positions)[at];
    float2 cs = turned(position * p.turns[i - t * p.half]);
    cs.x *= p.amplitude, cs.y *= p.amplitude;
    angles[i] = cs;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i) {
    const bool turns = kind[i] == 0 || kind[i] == 1;
    const int which = kind[i] == 1;
    if (p.weight[0] != nullptr) {  // of both or of none
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = __builtin_fmaf(v[i][e], v[i][e], sum);
#pragma unroll
      for (int d = 1; d < LANES; d *= 2) sum += __shfl_xor(sum, d, 64);
      const float scale = 1.f / __builtin_sqrtf(sum / (float)p.dim + p.eps);
      if (turns) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int at = first_value + e;
          if (VEC || e < count) v[i][e] = v[i][e] * scale * weight_of(p, which, at);
          if (APART && at < p.rotated)
            w[i][e] = w[i][e] * scale * weight_of(p, which, at < p.half ? at + p.half : at - p.half);
        }
      }
    }
    if (turns) {
      const float2* cs = angles + (token[i] - token0) * p.half;
      if constexpr (APART) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int at = first_value + e;
          if (at >= p.rotated) continue;
          const bool low = at < p.half;
          const float2 c = cs[low ? at : at - p.half];
          v[i][e] = __builtin_fmaf(v[i][e], c.x, (low ? -w[i][e] : w[i][e]) * c.y);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const int at = first_value + e;
          if (at >= p.rotated) continue;
          const float2 c = cs[at / 2];
          const float a = v[i][e], b = v[i][e + 1];
          v[i][e] = __builtin_fmaf(a, c.x, -b * c.y);
          v[i][e + 1] = __builtin_fmaf(b, c.x, a * c.y);
        }
      }
    }
    if (kind[i] >= 1 && p.bits != 0) {
      // as kv_write_kernel does: a NaN is larger than an infinity, and both stay
      uint32_t most = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[i][e] = rounded<TYPE>(v[i][e]);
        most = max(most, __float_as_uint(v[i][e]) & 0x7FFFFFFFu);
      }
#pragma unroll
      for (int d = 1; d < LANES; d *= 2) most = max(most, (uint32_t)__shfl_xor((int)most, d, 64));
      const long slot = p.slot8 ? static_cast<const int64_t*>(p.slots)[token[i]]
                                : static_cast<const int32_t*>(p.slots)[token[i]];
      if (slot < 0 || slot >= p.slots_total) continue;
      const uint32_t sb = f32_to_bf16_rne(__uint_as_float(most) / (p.bits == 4 ? 7.0f : 127.0f));
      const long at = cache_row(slot, head[i], p.kv_heads, p.page_shift);
      uint8_t* dst = p.codes[kind[i] - 1] + at * (p.dim * p.bits / 8) + part * p.bits;
      int c[8];
      if (p.bits == 4) {
        codes8<4>(v[i], __uint_as_float(sb << 16), c);
        store_codes<4>(dst, c);
      } else {
        codes8<8>(v[i], __uint_as_float(sb << 16), c);
        store_codes<8>(dst, c);
      }
      if (part == 0) p.scales[kind[i] - 1][at] = (uint16_t)sb;
    } else if (kind[i] >= 0) {
      uint8_t* out = p.out[which] + ((long)token[i] * p.out_token_stride[which] + (long)head[i] * p.out_head_stride[which] +
                                     first_value) * kSize<TYPE>;
      uint32_t u[TYPE == SHK_SRC_F32 ? 8 : 4];
      if constexpr (TYPE == SHK_SRC_F32) {
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = __float_as_uint(v[i][e]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (TYPE == SHK_SRC_BF16)
            u[e] = f32_to_bf16_rne(v[i][2 * e]) | (f32_to_bf16_rne(v[i][2 * e + 1]) << 16);
          else
            u[e] = __builtin_bit_cast(uint16_t, (_Float16)v[i][2 * e]) |
                   ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[i][2 * e + 1]) << 16);
        }
      }
      if constexpr (VEC) {
#pragma unroll
        for (int e = 0; e < (TYPE == SHK_SRC_F32 ? 2 : 1); ++e)
          reinterpret_cast<uint4*>(out)[e] = make_uint4(u[4 * e], u[4 * e + 1], u[4 * e + 2], u[4 * e + 3]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (e >= count) continue;
          if constexpr (TYPE == SHK_SRC_F32) reinterpret_cast<uint32_t*>(out)[e] = u[e];
          else reinterpret_cast<uint16_t*>(out)[e] = (uint16_t)(u[e / 2] >> (16 * (e % 2)));
        }
      }
    }
  }
}

template <int TYPE, int LANES, bool VEC, bool APART, int ROUNDS>
hipError_t launch(const Rotate& p, hipStream_t s) {
  constexpr unsigned PER = 256 / LANES * ROUNDS;
  // tokens that a workgroup can meet
  const unsigned tokens = (PER + p.per_token - 2) / p.per_token + 1;
  hipLaunchKernelGGL((rotate_kernel<TYPE, LANES, VEC, APART, ROUNDS>), dim3((p.rows + PER - 1) / PER), dim3(256),
                     tokens * p.half * sizeof(float2), s, p);
  return hipGetLastError();
}

template <int TYPE, int LANES, bool VEC>
hipError_t launch_pairs(const Rotate& p, bool apart, hipStream_t s) {
  // one round while that leaves CUs idle, else four, whose loads go out together
  const bool few = !VEC || p.rows <= 256u * (256 / LANES) * 4;
  if constexpr (VEC) {
    if (!few) return apart ? launch<TYPE, LANES, VEC, true, 4>(p, s) : launch<TYPE, LANES, VEC, false, 4>(p, s);
  }
  return apart ? launch<TYPE, LANES, VEC, true, 1>(p, s) : launch<TYPE, LANES, VEC, false, 1>(p, s);
}

template <int TYPE, int LANES>
hipError_t launch_vec(const Rotate& p, bool vec, bool apart, hipStream_t s) {
  return vec ? launch_pairs<TYPE, LANES, true>(p, apart, s) : launch_pairs<TYPE, LANES, false>(p, apart, s);
}

template <int TYPE>
hipError_t launch_type(const Rotate& p, bool vec, bool apart, hipStream_t s) {
  if (p.dim <= 64) return launch_vec<TYPE, 8>(p, vec, apart, s);
  if (p.dim <= 128) return launch_vec<TYPE, 16>(p, vec, apart, s);
  return launch_vec<TYPE, 32>(p, vec, apart, s);
}

}  // namespace

hipError_t launch_rotate(const shk_kv_cache* c, const shk_rotate& a, hipStream_t s) {
  Rotate p{};
  const long size = a.type == SHK_SRC_F32 ? 4 : 2;
  p.x[0] = static_cast<const uint8_t*>(a.q), p.x[1] = static_cast<const uint8_t*>(a.k);
  p.x[2] = static_cast<const uint8_t*>(a.values);
  p.token_stride[0] = a.q_token_stride, p.token_stride[1] = a.k_token_stride, p.token_stride[2] = a.value_token_stride;
  p.head_stride[0] = a.q_head_stride, p.head_stride[1] = a.k_head_stride, p.head_stride[2] = a.value_head_stride;
  p.out[0] = static_cast<uint8_t*>(a.q_out), p.out[1] = static_cast<uint8_t*>(a.k_out);
  p.out_token_stride[0] = a.q_out_token_stride, p.out_token_stride[1] = a.k_out_token_stride;
  p.out_head_stride[0] = a.q_out_head_stride, p.out_head_stride[1] = a.k_out_head_stride;
  p.weight[0] = a.q_weight, p.weight[1] = a.k_weight;
  p.weight_type = (int)a.weight_type;
  p.positions = a.positions, p.position8 = a.position_bytes == 8;
  p.turns = a.turns, p.amplitude = (float)a.amplitude, p.eps = (float)a.eps;
  p.heads = (unsigned)a.heads, p.kv_heads = (unsigned)a.kv_heads;
  p.per_token = p.heads + p.kv_heads * (c != nullptr ? 2 : 1);
  p.rows = (unsigned)a.tokens * p.per_token;
  p.dim = (int)a.head_dim, p.rotated = (int)a.rotated, p.half = p.rotated / 2;
  uintptr_t all = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) |
                  reinterpret_cast<uintptr_t>(a.q_out) | reinterpret_cast<uintptr_t>(a.k_out) |
                  (uintptr_t)(size * (a.q_token_stride | a.q_head_stride | a.k_token_stride | a.k_head_stride |
                                      a.q_out_token_stride | a.q_out_head_stride | a.head_dim));
  if (c != nullptr) {
    p.codes[0] = static_cast<uint8_t*>(c->key_codes), p.codes[1] = static_cast<uint8_t*>(c->value_codes);
    p.scales[0] = static_cast<uint16_t*>(c->key_scales), p.scales[1] = static_cast<uint16_t*>(c->value_scales);
    p.slots = a.slots, p.slot8 = a.slot_bytes == 8;
    p.slots_total = c->pages * c->page_size;
    p.page_shift = __builtin_ctzl((unsigned long)c->page_size);
    p.bits = (int)c->bits;
    all |= reinterpret_cast<uintptr_t>(a.values) | (uintptr_t)(size * (a.value_token_stride | a.value_head_stride));
  } else {
    all |= (uintptr_t)(size * (a.k_out_token_stride | a.k_out_head_stride));
  }
  const bool apart = a.interleaved == 0;
  const bool vec = (all & 15) == 0 && a.head_dim % 8 == 0 && (!apart || p.half % 8 == 0);
  if (a.type == SHK_SRC_F32) return launch_type<SHK_SRC_F32>(p, vec, apart, s);
  if (a.type == SHK_SRC_F16) return launch_type<SHK_SRC_F16>(p, vec, apart, s);
  return launch_type<SHK_SRC_BF16>(p, vec, apart, s);
}

}  // namespace shk
