// Query and key heads: the norm of a head, its rotation by position, and, where
// there is a cache, the quantized keys and values, in one pass over memory.
//
// A row is a head of a token; its lanes (head_dim / 8, rounded up to a power of
// two) hold 8 values each.  The value that a lane's value turns with is read
// beside it (from L1: the same row), so that only the sum of squares crosses
// lanes.  A workgroup takes whole rounds of rows, first all its loads; while they
// are on their way its threads compute the angles of the tokens that it meets
// into LDS.  An angle is positions * turns in 64 bits, less its nearest quarter:
// what is left is at most an eighth of a turn, held in f32 to 2^-24 of itself beside
// the 2^-53 of the whole angle that the product loses, and as much that `turns` did
// (together less, up to 2^27 radians).
//
// Bound by memory, and by latency for a few tokens.  8191 tokens of 40 heads of 128
// (168 MB): 35 us, 4.8 TB/s.  The vector unit is near: 44 us before addresses took
// products of 32 bits and sums over lanes moves, 38 without stores past the caches.
// 24 tokens, with norm and cache, 4.7 us.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "shk_common.h"
#include "shk_kvrows.h"
#include "shk_lanes.h"
#include "shk_loads.h"
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
  unsigned inverse[2];       // floor(2^64 / per_token) + 1, low half first
  float per_dim, per_half;   // 1 / dim, 1 / half
  unsigned token_bytes[3], head_bytes[3], out_token_bytes[2], out_head_bytes[2];  // the strides, where these hold them
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

// The angles of the tokens that a workgroup meets, cosines and sines apart, and
// both norms' weights, in LDS.
struct Shared {
  float* cosines;  // [tokens][half]
  float* sines;
  float* weights;  // [2][dim]
};

__device__ __forceinline__ Shared shared_parts(float* lds, const Rotate& p, unsigned tokens) {
  return Shared{lds, lds + tokens * p.half, lds + 2 * tokens * p.half};
}

// What a thread brings to them: asked for before the rows, since loads return in
// order, and worked out while the rows are on their way.  `angle` and `weight`:
// those that it begins with, of every 256.
struct Asked {
  double position, turns;
  float weight;
  int angles, angle, weights;  // numbers of angles and weights, and the first angle
};

__device__ __forceinline__ double position_of(const Rotate& p, long token) {
  return p.position8 ? (double)static_cast<const int64_t*>(p.positions)[token]
                     : (double)static_cast<const int32_t*>(p.positions)[token];
}

// i / half: i is below 2^15, and i + 1/2 is nowhere near a multiple of half.
__device__ __forceinline__ int quotient(const Rotate& p, int i) { return (int)(((float)i + 0.5f) * p.per_half); }

__device__ __forceinline__ Asked ask_shared(const Rotate& p, unsigned token0, unsigned tokens) {
  Asked r{0.0, 0.0, 0.f, (int)tokens * p.half, (int)threadIdx.x, p.weight[0] != nullptr ? 2 * p.dim : 0};
  if (r.angle < r.angles) {
    const int t = quotient(p, r.angle);
    r.position = position_of(p, (long)token0 + t);
    r.turns = p.turns[r.angle - t * p.half];
  }
  if ((int)threadIdx.x < r.weights) {
    const bool key = (int)threadIdx.x >= p.dim;
    r.weight = weight_of(p, key, (int)threadIdx.x - (key ? p.dim : 0));
  }
  return r;
}

__device__ __forceinline__ void fill_shared(const Shared& s, const Rotate& p, unsigned token0, const Asked& r) {
  for (int i = r.angle; i < r.angles; i += 256) {
    double angle = r.position * r.turns;
    if (i != r.angle) {
      const int t = quotient(p, i);
      angle = position_of(p, (long)token0 + t) * p.turns[i - t * p.half];
    }
    const float2 cs = turned(angle);
    s.cosines[i] = cs.x * p.amplitude, s.sines[i] = cs.y * p.amplitude;
  }
  for (int i = threadIdx.x; i < r.weights; i += 256)
    s.weights[i] = i < 256 ? r.weight : weight_of(p, i >= p.dim, i >= p.dim ? i - p.dim : i);
}

// row / per_token, the upper half of row * inverse: exact for every 32-bit row.
__device__ __forceinline__ unsigned token_of(const Rotate& p, unsigned row) {
  return (unsigned)(((unsigned long long)row * p.inverse[1] + __umulhi(row, p.inverse[0])) >> 32);
}

// Sum of squares of a row.
template <int LANES>
__device__ __forceinline__ float squares_of(const float (&v)[8]) {
  float sum = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) sum = __builtin_fmaf(v[e], v[e], sum);
#pragma unroll
  for (int d = 1; d < LANES; d *= 2) sum += __uint_as_float(across(__float_as_uint(sum), d));
  return sum;
}

// 1 / sqrt(mean + eps), to 2^-23.  The root's instruction takes no subnormal numbers,
// and squares of magnitudes below 2^-63 or above 2^63 leave the range: a head whose
// mean is near either end takes its values (v, and w, its partners) times a power of
// two, which the result undoes.  All lanes of a row have its sum.
template <int LANES>
__device__ __forceinline__ float norm_of(const Rotate& p, bool head, float (&v)[8], float (&w)[8]) {
  const float sum = squares_of<LANES>(v);
  float mean = __builtin_fmaf(sum, p.per_dim, p.eps);
  if (__builtin_expect(!(mean > 0x1p-100f && sum < 0x1p120f), 0)) {
    const float by = !head ? 1.f : sum < 1.f ? 0x1p100f : 0x1p-70f;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= by, w[e] *= by;
    mean = __builtin_fmaf(squares_of<LANES>(v), p.per_dim, p.eps * by * by);
  }
  return __builtin_amdgcn_rsqf(mean);
}

// A row of one round: which head of which token.
struct Place {
  unsigned token, head;
  int kind;  // 0 query, 1 key, 2 value, -1 none
};

__device__ __forceinline__ Place place_of(const Rotate& p, unsigned row, bool inside) {
  Place r;
  r.token = token_of(p, row);
  const unsigned h = row - r.token * p.per_token;
  r.kind = row >= p.rows || !inside ? -1 : h < p.heads ? 0 : h < p.heads + p.kv_heads ? 1 : 2;
  r.head = r.kind == 0 ? h : r.kind == 1 ? h - p.heads : h - p.heads - p.kv_heads;
  return r;
}

// One of three arguments: a choice, where an index would be a load.
template <class T>
__device__ __forceinline__ T pick(int kind, T query, T key, T value) {
  return kind == 0 ? query : kind == 1 ? key : value;
}

// The quantized row of a key or value, as kv_write_kernel makes it: a NaN is
// larger than an infinity, and both stay.
template <int TYPE, int LANES>
__device__ __forceinline__ void into_cache(const Rotate& p, const Place& r, int part, float (&v)[8]) {
  uint32_t most = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    v[e] = rounded<TYPE>(v[e]);
    most = max(most, __float_as_uint(v[e]) & 0x7FFFFFFFu);
  }
#pragma unroll
  for (int d = 1; d < LANES; d *= 2) most = max(most, across(most, d));
  const long slot = p.slot8 ? static_cast<const int64_t*>(p.slots)[r.token] : static_cast<const int32_t*>(p.slots)[r.token];
  if (slot < 0 || slot >= p.slots_total) return;
  const uint32_t sb = f32_to_bf16_rne(__uint_as_float(most) / (p.bits == 4 ? 7.0f : 127.0f));
  const long at = cache_row(slot, r.head, p.kv_heads, p.page_shift);
  uint8_t* dst = p.codes[r.kind - 1] + at * (p.dim * p.bits / 8) + part * p.bits;
  int c[8];
  if (p.bits == 4) {
    codes8<4>(v, __uint_as_float(sb << 16), c);
    store_codes<4>(dst, c);
  } else {
    codes8<8>(v, __uint_as_float(sb << 16), c);
    store_codes<8>(dst, c);
  }
  if (part == 0) p.scales[r.kind - 1][at] = (uint16_t)sb;
}

template <int TYPE>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  // v_cvt_pk_bf16_f32 leaves a quiet NaN one, and arithmetic makes no other
  if constexpr (TYPE == SHK_SRC_BF16) return pack_bf16x2_nonan(a, b);
  return __builtin_bit_cast(uint16_t, (_Float16)a) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)b) << 16);
}

// Eight floats of LDS, on 16 bytes.
__device__ __forceinline__ void read8(const float* from, float (&v)[8]) {
  const float4 a = reinterpret_cast<const float4*>(from)[0], b = reinterpret_cast<const float4*>(from)[1];
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}

// PAST: past the caches, for more than they hold until it is read again.
template <bool PAST>
__device__ __forceinline__ void store16(uint8_t* to, u4 v) {
  if constexpr (PAST) __builtin_nontemporal_store(v, reinterpret_cast<u4*>(to));
  else *reinterpret_cast<u4*>(to) = v;
}

// Rows on 16 bytes, strides of 32 bits, whose values, turning ones and (APART) half of them are whole
// 8s: a lane turns with all its values or none, and its partners are one load.
template <int TYPE, int LANES, bool APART, int ROUNDS>
__global__ __launch_bounds__(256) void rotate_kernel(const Rotate p) {
  constexpr int PER = 256 / LANES;  // rows of a round
  extern __shared__ __align__(16) float lds[];
  const int part = threadIdx.x % LANES, first = part * 8;
  const unsigned start = blockIdx.x * (PER * ROUNDS), mine = start + threadIdx.x / LANES;
  const bool inside = first < p.dim, turning = first < p.rotated, low = first < p.half;
  const int partner = APART ? (low ? first + p.half : first - p.half) : 0;
  const unsigned last = min(start + PER * ROUNDS, p.rows) - 1, token0 = token_of(p, start);
  const unsigned tokens = token_of(p, last) - token0 + 1;
  const Asked asked = ask_shared(p, token0, tokens);
  Place place[ROUNDS];
  float v[ROUNDS][8], w[APART ? ROUNDS : 1][8];
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i) {
    place[i] = place_of(p, mine + i * PER, inside);
    const Place& r = place[i];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[i][e] = w[APART ? i : 0][e] = 0.f;
    if (r.kind < 0) continue;
    const uint8_t* x = pick(r.kind, p.x[0], p.x[1], p.x[2]) +
                       (unsigned long long)r.token * pick(r.kind, p.token_bytes[0], p.token_bytes[1], p.token_bytes[2]) +
                       (unsigned long long)r.head * pick(r.kind, p.head_bytes[0], p.head_bytes[1], p.head_bytes[2]);
    load8<TYPE, true>(x + first * kSize<TYPE>, v[i]);
    if constexpr (APART)
      if (r.kind < 2 && turning) load8<TYPE, true>(x + partner * kSize<TYPE>, w[i]);
  }
  const Shared s = shared_parts(lds, p, tokens);
  fill_shared(s, p, token0, asked);
  __syncthreads();
  const bool norm = p.weight[0] != nullptr;
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i) {
    const Place& r = place[i];
    const bool head = r.kind == 0 || r.kind == 1;
    float scale = 1.f;
    if (norm) {
      scale = norm_of<LANES>(p, head, v[i], w[APART ? i : 0]);
      if (head) {
        float weight[8];
        read8(s.weights + (r.kind == 1 ? p.dim : 0) + first, weight);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] *= scale * weight[e];
      }
    }
    if (head && turning) {
      float c[8], n[8];
      const float* angles = s.cosines + (r.token - token0) * p.half;
      const long sines = s.sines - s.cosines;
      if constexpr (APART) {
        const float* at = angles + (low ? first : partner);
        read8(at, c);
        read8(at + sines, n);
        float weight[8];
        if (norm) {
          read8(s.weights + (r.kind == 1 ? p.dim : 0) + partner, weight);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) weight[e] = 1.f;
        }
        const float turn = low ? -scale : scale;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = __builtin_fmaf(w[i][e] * (turn * weight[e]), n[e], v[i][e] * c[e]);
      } else {
        const float4 cc = *reinterpret_cast<const float4*>(angles + first / 2);
        const float4 nn = *reinterpret_cast<const float4*>(angles + sines + first / 2);
        c[0] = cc.x, c[1] = cc.y, c[2] = cc.z, c[3] = cc.w;
        n[0] = nn.x, n[1] = nn.y, n[2] = nn.z, n[3] = nn.w;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float a = v[i][2 * e], b = v[i][2 * e + 1];
          v[i][2 * e] = __builtin_fmaf(-b, n[e], a * c[e]);
          v[i][2 * e + 1] = __builtin_fmaf(a, n[e], b * c[e]);
        }
      }
    }
    if (r.kind >= 1 && p.bits != 0) {
      into_cache<TYPE, LANES>(p, r, part, v[i]);
    } else if (r.kind >= 0) {
      uint8_t* out = (r.kind == 0 ? p.out[0] : p.out[1]) +
                     (unsigned long long)r.token * (r.kind == 0 ? p.out_token_bytes[0] : p.out_token_bytes[1]) +
                     (unsigned long long)r.head * (r.kind == 0 ? p.out_head_bytes[0] : p.out_head_bytes[1]) + first * kSize<TYPE>;
      if constexpr (TYPE == SHK_SRC_F32) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
          store16<(ROUNDS > 1)>(out + 16 * e, u4{__float_as_uint(v[i][4 * e]), __float_as_uint(v[i][4 * e + 1]),
                                                 __float_as_uint(v[i][4 * e + 2]), __float_as_uint(v[i][4 * e + 3])});
      } else {
        store16<(ROUNDS > 1)>(out, u4{pack2<TYPE>(v[i][0], v[i][1]), pack2<TYPE>(v[i][2], v[i][3]),
                                      pack2<TYPE>(v[i][4], v[i][5]), pack2<TYPE>(v[i][6], v[i][7])});
      }
    }
  }
}

// Any strides, sizes and alignment: value by value (4000 tokens of 40 heads of 80, 40
// of them turning: 54 us for 51 MB).
template <int TYPE, int LANES, bool APART>
__global__ __launch_bounds__(256) void rotate_any_kernel(const Rotate p) {
  constexpr int PER = 256 / LANES;
  extern __shared__ __align__(16) float lds[];
  const int part = threadIdx.x % LANES, first = part * 8, count = min(8, p.dim - first);
  const unsigned start = blockIdx.x * PER;
  const Place r = place_of(p, start + threadIdx.x / LANES, count > 0);
  const bool head = r.kind == 0 || r.kind == 1, norm = p.weight[0] != nullptr;
  float v[8] = {}, w[8] = {};
  if (r.kind >= 0) {
    const uint8_t* x = p.x[r.kind] + ((long)r.token * p.token_stride[r.kind] + (long)r.head * p.head_stride[r.kind]) *
                                         kSize<TYPE>;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int at = first + e;
      if (e < count) v[e] = element<TYPE>(x, at);
      if (APART && head && at < p.rotated) w[e] = element<TYPE>(x, at < p.half ? at + p.half : at - p.half);
    }
  }
  const unsigned last = min(start + PER, p.rows) - 1, token0 = token_of(p, start);
  const unsigned tokens = token_of(p, last) - token0 + 1;
  const Shared s = shared_parts(lds, p, tokens);
  fill_shared(s, p, token0, ask_shared(p, token0, tokens));
  __syncthreads();
  float scale = 1.f;
  if (norm) scale = norm_of<LANES>(p, head, v, w);
  if (head) {
    const float* weight = s.weights + (r.kind == 1 ? p.dim : 0);
    const unsigned angles = (r.token - token0) * p.half;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (norm && e < count) v[e] *= scale * weight[first + e];
#pragma unroll
    for (int e = 0; e < 8; e += APART ? 1 : 2) {
      const int at = first + e;
      if (at >= p.rotated) continue;
      if constexpr (APART) {
        const bool low = at < p.half;
        const int pair = low ? at : at - p.half;
        const float turn = (low ? -scale : scale) * (norm ? weight[low ? at + p.half : pair] : 1.f);
        v[e] = __builtin_fmaf(w[e] * turn, s.sines[angles + pair], v[e] * s.cosines[angles + pair]);
      } else {
        const float c = s.cosines[angles + at / 2], n = s.sines[angles + at / 2], a = v[e], b = v[e + 1];
        v[e] = __builtin_fmaf(-b, n, a * c);
        v[e + 1] = __builtin_fmaf(a, n, b * c);
      }
    }
  }
  if (r.kind >= 1 && p.bits != 0) {
    into_cache<TYPE, LANES>(p, r, part, v);
  } else if (r.kind >= 0) {
    uint8_t* out = p.out[r.kind] + ((long)r.token * p.out_token_stride[r.kind] +
                                    (long)r.head * p.out_head_stride[r.kind] + first) * kSize<TYPE>;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (e >= count) continue;
      if constexpr (TYPE == SHK_SRC_F32) reinterpret_cast<float*>(out)[e] = v[e];
      else reinterpret_cast<uint16_t*>(out)[e] = (uint16_t)pack2<TYPE>(v[e], 0.f);
    }
  }
}

// LDS of a workgroup of `rows` rows: angles of the tokens that it can meet, weights.
unsigned shared_bytes(const Rotate& p, unsigned rows) {
  const unsigned tokens = (rows + p.per_token - 2) / p.per_token + 1;
  return (2 * tokens * p.half + (p.weight[0] != nullptr ? 2 * p.dim : 0)) * sizeof(float);
}

template <int TYPE, int LANES, bool APART, int ROUNDS>
hipError_t launch(const Rotate& p, hipStream_t s) {
  constexpr unsigned PER = 256 / LANES * ROUNDS;
  hipLaunchKernelGGL((rotate_kernel<TYPE, LANES, APART, ROUNDS>), dim3((p.rows + PER - 1) / PER), dim3(256),
                     shared_bytes(p, PER), s, p);
  return hipGetLastError();
}

template <int TYPE, int LANES, bool APART>
hipError_t launch_pairs(const Rotate& p, bool vec, hipStream_t s) {
  constexpr unsigned PER = 256 / LANES;
  if (!vec) {
    hipLaunchKernelGGL((rotate_any_kernel<TYPE, LANES, APART>), dim3((p.rows + PER - 1) / PER), dim3(256),
                       shared_bytes(p, PER), s, p);
    return hipGetLastError();
  }
  // one round while that leaves CUs idle, else two, whose loads go out together
  // (8191 tokens of 40 heads of 128: 35 us with two, 39 with four, whose registers
  // halve the waves, 43 with one; two without stores past the caches 38)
  return p.rows <= 256 * PER * 4 ? launch<TYPE, LANES, APART, 1>(p, s) : launch<TYPE, LANES, APART, 2>(p, s);
}

template <int TYPE, int LANES>
hipError_t launch_vec(const Rotate& p, bool vec, bool apart, hipStream_t s) {
  return apart ? launch_pairs<TYPE, LANES, true>(p, vec, s) : launch_pairs<TYPE, LANES, false>(p, vec, s);
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
  const unsigned long long inverse = ~0ULL / p.per_token + 1;  // per_token is 2 or more, 2^64 - 1 divides alike
  p.inverse[0] = (unsigned)inverse, p.inverse[1] = (unsigned)(inverse >> 32);
  p.per_dim = 1.f / (float)a.head_dim;
  p.per_half = a.rotated > 0 ? 2.f / (float)a.rotated : 0.f;
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
  unsigned long long widest = 0;  // a negative stride is wide, too
  for (int i = 0; i < 3; ++i) {
    widest |= (unsigned long long)p.token_stride[i] * size | (unsigned long long)p.head_stride[i] * size;
    p.token_bytes[i] = (unsigned)(p.token_stride[i] * size), p.head_bytes[i] = (unsigned)(p.head_stride[i] * size);
  }
  for (int i = 0; i < 2; ++i) {
    widest |= (unsigned long long)p.out_token_stride[i] * size | (unsigned long long)p.out_head_stride[i] * size;
    p.out_token_bytes[i] = (unsigned)(p.out_token_stride[i] * size);
    p.out_head_bytes[i] = (unsigned)(p.out_head_stride[i] * size);
  }
  const bool apart = a.interleaved == 0;
  const bool vec = (all & 15) == 0 && widest >> 32 == 0 && a.head_dim % 8 == 0 && a.rotated % (apart ? 16 : 8) == 0;
  if (a.type == SHK_SRC_F32) return launch_type<SHK_SRC_F32>(p, vec, apart, s);
  if (a.type == SHK_SRC_F16) return launch_type<SHK_SRC_F16>(p, vec, apart, s);
  return launch_type<SHK_SRC_BF16>(p, vec, apart, s);
}

}  // namespace shk
