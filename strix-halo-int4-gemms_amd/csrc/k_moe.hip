// The gated mixture-of-experts layer for a few tokens, on packed int4 weights
// and activations that are not quantized:
//
//   h[p] = (x[t] U_e) * silu(x[t] G_e)       for each pair p = (t, j), e = ids[t, j]
//   y[t] = sum_j share[t, j] * (h[t, j] D_e)
//
// Few tokens reach an expert, so the layer is the time to stream the weights
// of the experts that are hit.  Two products share one body (moe_product): a
// workgroup takes 16 pairs of one expert and 128 columns (64 of up and of
// gate, or 128 of down), its waves a slice of K each, joined through LDS.  An
// expert with more than 16 pairs has a workgroup for each 16 of them, side by
// side: all but the first find the codes in the caches.  (Two tiles of 16 in
// one workgroup take twice the registers for the sums and leave fewer
// workgroups: 253 us instead of 240 for 122 pairs of 16 experts of 4096 x
// 11008, 90 instead of 53 for 306 pairs of 16 experts of 320 x 4320.)
//
// Measured: 61 tokens over 16 experts (14 are hit) of 4096 x 11008, 949 MB of
// codes: up and gate 151 us, down 85, 4.0 TB/s together; the same loads without
// the products take 110 and 60.  16 tokens over 64 experts (41 hit) of 2048 x
// 1408 in groups of 128: 35 and 26 us for 183 MB, where a wave has eight pieces
// and its start (the pairs of its expert) and end (the sums of the waves) are
// half of it.  One token through two experts: 10 us each, with 48 and 32
// workgroups on 256 CUs: ids, codes and the waves' join behind each other.
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
#include <type_traits>

#include "shk_common.h"
#include "shk_loads.h"
#include "shk_moe.h"

#ifndef SHK_LAYOUT
#error "SHK_LAYOUT must be defined: the weights' layout, 0 NN or 1 NT"
#endif

namespace shk {
namespace {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));

typedef __attribute__((address_space(1))) const uint16_t* global_halves;

constexpr int kHalf = kMoeColumns / 2;  // columns of half a workgroup's tile
constexpr int kPitch = 2 * kHalf + 4;  // floats of an LDS row of sums: rows start on different banks
constexpr int kSuper = kMoePiece;        // K values a wave loads at a time, four products deep
constexpr int kLargeGroups = 1;    // scale groups of at least a piece
constexpr int kSmallGroups = 2;    // of 32 or 64
constexpr int kMostPairs = 1024;   // (token, expert) pairs of a call
constexpr int kMostExperts = 1024;

constexpr int kRows = 16;          // pairs of a workgroup, the columns of a product

struct MoeArgs {
  const void* x;
  long x_stride;
  const uint8_t* w;        // codes of this product
  const uint16_t* scale;
  const void* ids;
  const float* share;
  uint16_t* h;             // [pairs][high, low][inner_pad]: bf16 terms, eights in the order of expand
  float* part;             // [pairs][hidden]
  int* arrived;            // a counter for each tile of the down product
  void* out;
  int k, k_packed, cols;   // this product's K, its bytes, and columns (of up alone)
  int group, groups;       // scale group (0: per channel) and groups of K
  int tokens, top, experts, hidden, inner, inner_pad, tiles;
  int type, id8;
  int joined;              // the down product adds up the pairs itself
};

__device__ __forceinline__ int id_of(const MoeArgs& a, int p) {
  const long id = a.id8 ? (long)static_cast<const int64_t*>(a.ids)[p] : (long)static_cast<const int32_t*>(a.ids)[p];
  return id >= 0 && id < a.experts ? (int)id : -1;
}

__device__ __forceinline__ f4 mfma_bf16(b8 a, b8 b, f4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// The eight codes of a dword, each plus 24, in the order 0 4 1 5 2 6 3 7.
__device__ __forceinline__ b8 expand(uint32_t w) {
  // 0x41C0: 16, with the nibble's sign bit flipped on the way
  return __builtin_bit_cast(b8, u4{((w << 3) & 0x00780078u) ^ 0x41C041C0u, ((w >> 1) & 0x00780078u) ^ 0x41C041C0u,
                                   ((w >> 5) & 0x00780078u) ^ 0x41C041C0u, ((w >> 9) & 0x00780078u) ^ 0x41C041C0u});
}

// Where a product's codes come from: the expert's matrix, and the end of all
// experts' (nothing is read past it).
struct Codes {
  const uint8_t *w, *end;
  int total, k_packed;  // columns of a row (NN) and bytes of one (NT)
};

// 16 dwords of a lane: the codes of 128 K values from k0 for 64 columns from
// n0, as they are stored.  What lies outside the expert's matrix meets
// activations of zero or is not stored, so it may be anything.
template <int LAYOUT>
__device__ __forceinline__ void load_half(const Codes& s, int k0, int n0, uint32_t (&o)[16]) {
  const int lane = threadIdx.x & 63, g = lane / 16, c = lane % 16;
  if constexpr (LAYOUT == SHK_LAYOUT_NT) {  // [n][k_packed]: 16 bytes of the rows 4 c + j
    const uint32_t mine = (uint32_t)(4 * c * s.k_packed + 16 * g);
    const uint8_t* p = s.w + (long)n0 * s.k_packed + k0 / 2;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const u4 v = load_at<any_u4>(p + (long)j * s.k_packed, mine);
      o[4 * j] = v[0], o[4 * j + 1] = v[1], o[4 * j + 2] = v[2], o[4 * j + 3] = v[3];
    }
  } else {  // [k_packed][n]: four columns of the rows 16 q + 4 g + i
    const uint32_t mine = (uint32_t)(4 * g * s.total + 4 * c);
    const uint8_t* p = s.w + (long)(k0 / 2) * s.total + n0;
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] = load_at<any_u32>(p + (long)(16 * (i / 4) + i % 4) * s.total, mine);
  }
}

// The codes of 128 K values for the 128 columns of a tile, in two halves of
// 64 columns from n0 and n1.  WIDE: the halves are one stretch of columns,
// and a lane's are 8 c + 4 half + j (otherwise 4 c + j of each half).
template <int LAYOUT, bool WIDE>
__device__ __forceinline__ void load_w(const Codes& s, int k0, int n0, int n1, uint32_t (&o)[2][16]) {
  if constexpr (WIDE) {  // [k_packed][n]: eight columns of a row
    const int lane = threadIdx.x & 63, g = lane / 16, c = lane % 16;
    const uint32_t mine = (uint32_t)(4 * g * s.total + 8 * c);
    const uint8_t* p = s.w + (long)(k0 / 2) * s.total + n0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const u2 v = load_at<any_u2>(p + (long)(16 * (i / 4) + i % 4) * s.total, mine);
      o[0][i] = v[0], o[1][i] = v[1];
    }
  } else {
    load_half<LAYOUT>(s, k0, n0, o[0]);
    load_half<LAYOUT>(s, k0, n1, o[1]);
  }
}

// The same where part of it lies past the end of all codes (at most the last
// expert's last pieces), by way of 16 dwords of LDS a lane: few registers, and
// eight loads at a time.
template <int LAYOUT, bool WIDE>
__device__ __forceinline__ void load_w_end(const Codes& s, int k0, int n0, uint32_t* lds, uint32_t (&o)[16]) {
  const int lane = threadIdx.x & 63, g = lane / 16, c = lane % 16;
#pragma unroll 1
  for (int i0 = 0; i0 < 16; i0 += 8) {
    uint32_t v[8];
    long over[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = i0 + u;
      const uint8_t* p = LAYOUT == SHK_LAYOUT_NT
                             ? s.w + (long)(n0 + 4 * c + i / 4) * s.k_packed + k0 / 2 + 16 * g + 4 * (i % 4)
                             : s.w + (long)(k0 / 2 + 16 * (i / 4) + 4 * g + i % 4) * s.total + n0 + (WIDE ? 8 : 4) * c;
      // the last dword there is, shifted to where it would be
      over[u] = p - (s.end - 4);
      v[u] = *(__attribute__((address_space(1))) const any_u32*)(s.end - 4 + min(over[u], 0l));
    }
#pragma unroll
    for (int u = 0; u < 8; ++u)
      lds[(i0 + u) * 64 + lane] = over[u] <= 0 ? v[u] : (over[u] < 4 ? v[u] >> (8 * over[u]) : 0u);
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) o[i] = lds[i * 64 + lane];
}

// Whether load_w of this piece stays inside all experts' codes.
template <int LAYOUT>
__device__ __forceinline__ bool inside(const Codes& s, int k0, int n0) {
  const long last = LAYOUT == SHK_LAYOUT_NT ? (long)(n0 + kHalf - 1) * s.k_packed + k0 / 2 + kSuper / 2
                                            : (long)(k0 / 2 + kSuper / 2 - 1) * s.total + n0 + kHalf;
  return s.w + last <= s.end;
}

// The operand dwords of product step q (32 K values) for the columns 4 c + j
// of a half: eight codes of the K values k0 + 32 q + 8 g.
template <int LAYOUT>
__device__ __forceinline__ void arrange(uint32_t (&w)[16]) {
  if constexpr (LAYOUT == SHK_LAYOUT_NT) {
    // lane group g holds 16 bytes of its own K values: the four groups
    // exchange dwords, so that dword q is the group's share of step q
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t* r = w + 4 * j;
      auto a = __builtin_amdgcn_permlane32_swap(r[0], r[2], false, false);
      auto b = __builtin_amdgcn_permlane32_swap(r[1], r[3], false, false);
      auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
      auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
      r[0] = c[0], r[1] = c[1], r[2] = d[0], r[3] = d[1];
    }
  }
}
template <int LAYOUT>
__device__ __forceinline__ void step_codes(const uint32_t (&w)[16], int q, uint32_t (&o)[4]) {
  if constexpr (LAYOUT == SHK_LAYOUT_NT) {
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = w[4 * j + q];
  } else {
    transpose4x4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3], o[0], o[1], o[2], o[3]);
  }
}

// Activations of the K values k0 + 32 q + 8 g. FIRST: a row of x, in its own
// type; otherwise the two terms of a row of h, which is padded and in order.
template <bool FIRST, int TYPE>
constexpr int kLoads = FIRST ? 1 : 2;   // 16-byte loads a step
template <bool FIRST, int TYPE>
constexpr int kTerms = FIRST && TYPE == SHK_SRC_BF16 ? 1 : 2;

template <bool FIRST, int TYPE>
__device__ __forceinline__ void load_x(const MoeArgs& a, global_halves row, int k, u4 (&o)[kLoads<FIRST, TYPE>]) {
  if constexpr (FIRST) {
    o[0] = *(__attribute__((address_space(1))) const any_u4*)(row + k);
  } else {
    o[0] = *(__attribute__((address_space(1))) const u4*)(row + k);
    o[1] = *(__attribute__((address_space(1))) const u4*)(row + a.inner_pad + k);
  }
}

// Eight 16-bit values without the first n (none for n <= 0), zeros behind.
__device__ __forceinline__ u4 drop(u4 v, int n) {
  n = max(n, 0);
  if (n & 1) v = u4{perm_b32(v[1], v[0], 0x05040302u), perm_b32(v[2], v[1], 0x05040302u),
                    perm_b32(v[3], v[2], 0x05040302u), v[3] >> 16};
  if (n & 2) v = u4{v[1], v[2], v[3], 0};
  if (n & 4) v = u4{v[2], v[3], 0, 0};
  return n < 8 ? v : u4{0, 0, 0, 0};
}

// As bf16 terms in the order 0 4 1 5 2 6 3 7.
template <bool FIRST, int TYPE>
__device__ __forceinline__ void terms(const u4 (&u)[kLoads<FIRST, TYPE>], b8 (&t)[kTerms<FIRST, TYPE>]) {
  if constexpr (!FIRST) {
    t[0] = __builtin_bit_cast(b8, u[0]);
    t[1] = __builtin_bit_cast(b8, u[1]);
  } else {
    const u4 o = {perm_b32(u[0][2], u[0][0], 0x05040100u), perm_b32(u[0][2], u[0][0], 0x07060302u),
                  perm_b32(u[0][3], u[0][1], 0x05040100u), perm_b32(u[0][3], u[0][1], 0x07060302u)};
    if constexpr (TYPE == SHK_SRC_BF16) {
      t[0] = __builtin_bit_cast(b8, o);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float f = (float)__builtin_bit_cast(_Float16, (uint16_t)(o[i / 2] >> (16 * (i % 2))));
        t[0][i] = (__bf16)f;
        t[1][i] = (__bf16)(f - (float)t[0][i]);
      }
    }
  }
}

// Where the columns of lane group g's sums r start, in the 128 of a tile.
template <bool WIDE>
__device__ __forceinline__ int column(int half, int g, int r) {
  return WIDE ? 32 * g + 8 * r + 4 * half : kHalf * half + 16 * g + 4 * r;
}

// A workgroup's tile for the first `rows` pairs of the list, at most 16.
template <int LAYOUT, bool FIRST, int TYPE, int GROUPED, int kWaves>
__device__ __forceinline__ void moe_rows(const MoeArgs& a, const Codes& s, const uint16_t* scale, const uint16_t* list,
                                         int rows, int n0, int k_first, int k_last, int k_step, float* red,
                                         uint32_t* lds_scale) {
  constexpr int kT = kTerms<FIRST, TYPE>, kL = kLoads<FIRST, TYPE>;
  const int lane = threadIdx.x & 63, g = lane / 16, c = lane % 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int n1 = n0 + (FIRST ? a.cols : kHalf);  // the second half's first column
  const __bf16 one = (__bf16)1.0f;
  const b8 ones = {one, one, one, one, one, one, one, one};

  // columns of a product without a row repeat the last one; they are not stored
  const int pair = list[min(c, rows - 1)];
  const global_halves src = FIRST ? (global_halves)a.x + (pair / a.top) * a.x_stride
                                  : (global_halves)a.h + (long)pair * 2 * a.inner_pad;
  f4 acc[8], sum[2], all[GROUPED ? 8 : 1];
  sum[0] = sum[1] = f4{0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    acc[j] = f4{0, 0, 0, 0};
    if constexpr (GROUPED) all[j] = f4{0, 0, 0, 0};
  }
  uint32_t* lds = reinterpret_cast<uint32_t*>(red) + 1024 * wave;
  constexpr bool kWide = !FIRST && LAYOUT == SHK_LAYOUT_NN;
  struct Block {  // 128 K values: the codes of both halves, the activations, and the scales of up to four groups
    uint32_t w[2][16];
    u4 x[4][kL];
    uint32_t sc[GROUPED == kSmallGroups ? 4 : 1];  // of two columns: the half lane / 32, columns 2 (lane % 32)
  };
  // Pieces from before `whole` lie inside the codes, the activations and the
  // scales.
  const int sc_n = (lane < 32 ? n0 : n1) + 2 * (lane % 32);
  auto fits = [&](int k0) {
    const int last = GROUPED ? min((k0 + kSuper - 1) / a.group, a.groups - 1) : 0;
    const bool scales = !GROUPED || scale + (long)last * s.total + n1 + kHalf <=
                                        a.scale + (long)a.experts * a.groups * s.total;
    return scales && inside<LAYOUT>(s, k0, n0) && inside<LAYOUT>(s, k0, n1);
  };
  int whole = FIRST ? min(k_last, a.k - kSuper + 1) : k_last;
  while (whole > k_first && !fits(whole - 1)) whole -= kSuper;
  const int last = k_first + (max(whole - k_first, 1) - 1) / k_step * k_step;  // the last of them
  auto load_scales = [&](int k0, auto end, Block& b) {
    if constexpr (GROUPED) {
#pragma unroll
      for (int i = 0; i < (GROUPED == kSmallGroups ? 4 : 1); ++i)
        if (i < 2 || a.group == 32) {
          const uint16_t* p = scale + (long)min(k0 / a.group + i, a.groups - 1) * s.total;
          if constexpr (decltype(end)::value)
            b.sc[i] = p[min(sc_n, s.total - 1)] | ((uint32_t)p[min(sc_n + 1, s.total - 1)] << 16);
          else
            b.sc[i] = load_at<any_u32>(p, 2u * (uint32_t)sc_n);
        }
    }
  };
  auto load_rows = [&](int k0, u4 (&x)[4][kL]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) load_x<FIRST, TYPE>(a, src, k0 + 32 * q + 8 * g, x[q]);
  };
  auto load_end = [&](int k0, Block& b) {
    load_scales(k0, std::true_type{}, b);
    if (inside<LAYOUT>(s, k0, n0) && inside<LAYOUT>(s, k0, n1)) {
      load_w<LAYOUT, kWide>(s, k0, n0, n1, b.w);
    } else {
      load_w_end<LAYOUT, kWide>(s, k0, n0, lds, b.w[0]);
      load_w_end<LAYOUT, kWide>(s, k0, kWide ? n0 + 4 : n1, lds, b.w[1]);
    }
    if constexpr (FIRST) {  // zeros past the end of x
      if (a.k >= 8) {
        // the last eight values there are, shifted to where they would be
#pragma unroll
        for (int q = 0; q < 4; ++q) load_x<FIRST, TYPE>(a, src, min(k0 + 32 * q + 8 * g, a.k - 8), b.x[q]);
#pragma unroll
        for (int q = 0; q < 4; ++q) b.x[q][0] = drop(b.x[q][0], k0 + 32 * q + 8 * g - (a.k - 8));
      } else {
        uint16_t* h = reinterpret_cast<uint16_t*>(lds) + 8 * lane;
#pragma unroll 1
        for (int i = 0; i < 32; ++i) {
          const int k = k0 + 32 * (i / 8) + 8 * g + i % 8;
          h[512 * (i / 8) + i % 8] = k < a.k ? src[k] : (uint16_t)0;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) b.x[q][0] = *reinterpret_cast<const u4*>(h + 512 * q);
      }
    } else {
      load_rows(k0, b.x);
    }
  };
  auto share_scales = [&](const Block& b) {  // to where the other lanes read them
    if constexpr (GROUPED) {
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int i = 0; i < (GROUPED == kSmallGroups ? 4 : 1); ++i) lds_scale[64 * i + lane] = b.sc[i];
      __builtin_amdgcn_wave_barrier();
    }
  };
  // A half's sums of a group that ends, without the offset, times its scales.
  auto scale_half = [&](auto half, int group) {
    constexpr int kAt = decltype(half)::value;
    constexpr int kSum = GROUPED == kSmallGroups ? kAt : 0;
    const uint16_t* sc = reinterpret_cast<const uint16_t*>(lds_scale) + 128 * group;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const u2 v = *reinterpret_cast<const u2*>(sc + column<kWide>(kAt, g, r));
      const float f[4] = {bf16_bits_to_f32((uint16_t)v[0]), __uint_as_float(v[0] & 0xFFFF0000u),
                          bf16_bits_to_f32((uint16_t)v[1]), __uint_as_float(v[1] & 0xFFFF0000u)};
      for (int j = 0; j < 4; ++j) {
        all[4 * kAt + j][r] += f[j] * (acc[4 * kAt + j][r] - 24.0f * sum[kSum][r]);
        acc[4 * kAt + j][r] = 0.0f;
      }
    }
  };
  auto multiply = [&](auto half, Block& b) {
    __builtin_amdgcn_sched_barrier(0);  // what has been asked for ahead stays ahead
    constexpr int kAt = decltype(half)::value;
    constexpr int kSum = GROUPED == kSmallGroups ? kAt : 0;
    uint32_t(&w)[16] = b.w[kAt];
    arrange<LAYOUT>(w);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      b8 xt[kT];
      terms<FIRST, TYPE>(b.x[q], xt);
#pragma unroll
      for (int i = 0; i < kT; ++i)
        if (kSum == kAt) sum[kSum] = mfma_bf16(ones, xt[i], sum[kSum]);
      uint32_t o[4];
      step_codes<LAYOUT>(w, q, o);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const b8 v = expand(o[j]);
#pragma unroll
        for (int i = 0; i < kT; ++i) acc[4 * kAt + j] = mfma_bf16(v, xt[i], acc[4 * kAt + j]);
      }
      if constexpr (GROUPED == kSmallGroups) {
        if (q % 2 == 1 || a.group == 32) {
          scale_half(half, 32 * q / a.group);
          sum[kAt] = f4{0, 0, 0, 0};
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto finish = [&](int k0) {  // a group of 128 or more ends with this piece
    if constexpr (GROUPED == kLargeGroups) {
      if (k0 + kSuper >= k_last || (k0 + kSuper) % a.group == 0) {
        scale_half(std::integral_constant<int, 0>{}, 0);
        scale_half(std::integral_constant<int, 1>{}, 0);
        sum[0] = f4{0, 0, 0, 0};
      }
    }
  };
  constexpr std::integral_constant<int, 0> h0{};
  constexpr std::integral_constant<int, 1> h1{};
  // What is loaded ahead is loaded whether it comes or not (the last piece
  // again): a load that may not happen would have to be waited for as if it
  // were the latest.
  int k0 = k_first;
  if (k0 < whole) {
    if constexpr (kWide || LAYOUT == SHK_LAYOUT_NT) {
      // the next 128 K values are on their way while these are multiplied
      auto load = [&](int k, Block& b) {
        load_scales(k, std::false_type{}, b);
        load_w<LAYOUT, kWide>(s, k, n0, n1, b.w);
        load_rows(k, b.x);
      };
      auto use = [&](Block& b) {
        share_scales(b);
        multiply(h0, b);
        multiply(h1, b);
        finish(k0);
        return (k0 += k_step) < whole;
      };
      Block b0, b1;
      load(k0, b0);
      while (true) {
        load(min(k0 + k_step, last), b1);
        if (!use(b0)) break;
        load(min(k0 + k_step, last), b0);
        if (!use(b1)) break;
      }
    } else {
      // Each half's codes are on their way while the other half is
      // multiplied: two sets of 32 loads would pass the 63 that can be counted.
      Block b;
      load_rows(k0, b.x);
      load_half<LAYOUT>(s, k0, n0, b.w[0]);
      load_half<LAYOUT>(s, k0, n1, b.w[1]);
      for (; k0 < whole; k0 += k_step) {
        const int next = min(k0 + k_step, last);
        load_scales(k0, std::false_type{}, b);
        share_scales(b);
        multiply(h0, b);
        u4 x[4][kL];
        load_rows(next, x);
        load_half<LAYOUT>(s, next, n0, b.w[0]);
        multiply(h1, b);
        finish(k0);
        load_half<LAYOUT>(s, next, n1, b.w[1]);
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int i = 0; i < kL; ++i) b.x[q][i] = x[q][i];
      }
    }
  }
  for (; k0 < k_last; k0 += k_step) {
    Block b;
    load_end(k0, b);
    share_scales(b);
    multiply(h0, b);
    multiply(h1, b);
    finish(k0);
  }
  // The waves' sums: lane (g, c) holds token c, columns column(half, g, r)
  // + j.  The second half of the waves hand theirs to the first half.
  f4 v[8];  // [half][r] over j
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (GROUPED) v[4 * half + r][j] = all[4 * half + j][r];
        else v[4 * half + r][j] = acc[4 * half + j][r] - 24.0f * sum[0][r];
      }
  float* mine = &red[(wave % (kWaves / 2)) * 16 * kPitch + c * kPitch];
  __syncthreads();
  if (wave >= kWaves / 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i) *reinterpret_cast<f4*>(mine + column<kWide>(i / 4, g, i % 4)) = v[i];
  }
  __syncthreads();
  if (wave < kWaves / 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f4* at = reinterpret_cast<f4*>(mine + column<kWide>(i / 4, g, i % 4));
      *at += v[i];
    }
  }
  __syncthreads();
  if constexpr (FIRST) {
    for (int i = threadIdx.x; i < rows * kHalf; i += 64 * kWaves) {
      const int r = i / kHalf, n = i % kHalf, col = n0 + n;
      if (col >= a.inner_pad) continue;
      float h = 0.0f;  // up to inner_pad
      if (col < a.cols) {
        float up = 0.0f, gate = 0.0f;
#pragma unroll
        for (int q = 0; q < kWaves / 2; ++q) {
          up += red[q * 16 * kPitch + r * kPitch + n];
          gate += red[q * 16 * kPitch + r * kPitch + kHalf + n];
        }
        if constexpr (!GROUPED) up *= load_bf16(scale + col), gate *= load_bf16(scale + a.cols + col);
        h = up * (gate / (1.0f + __expf(-gate)));
      }
      // place 2 i + u of an eight holds its element i + 4 u
      const int at = (col & ~7) | (2 * (col & 3) + ((col >> 2) & 1));
      const uint32_t hi = f32_to_bf16_rne(h);
      uint16_t* dst = a.h + (long)list[r] * 2 * a.inner_pad + at;
      dst[0] = (uint16_t)hi;
      dst[a.inner_pad] = (uint16_t)f32_to_bf16_rne(h - bf16_bits_to_f32((uint16_t)hi));
    }
  } else {
    for (int i = threadIdx.x; i < rows * 2 * kHalf; i += 64 * kWaves) {
      const int r = i / (2 * kHalf), n = i % (2 * kHalf), col = n0 + n;
      if (col >= a.cols) continue;
      float v2 = 0.0f;
#pragma unroll
      for (int q = 0; q < kWaves / 2; ++q) v2 += red[q * 16 * kPitch + r * kPitch + n];
      if constexpr (!GROUPED) v2 *= load_bf16(scale + col);
      __hip_atomic_store(a.part + (long)list[r] * a.hidden + col, v2, __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
    }
  }
}

// y[t, n] = sum_j share[t, j] * part[t, j][n], in the order of j.
__device__ __forceinline__ void join_value(const MoeArgs& a, int t, int n) {
  float y = 0.0f;
  for (int j = 0; j < a.top; ++j) {
    const int p = t * a.top + j;
    if (id_of(a, p) >= 0)
      y += a.share[p] * __hip_atomic_load(a.part + (long)p * a.hidden + n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  const long at = (long)t * a.hidden + n;
  if (a.type == SHK_SRC_BF16) static_cast<uint16_t*>(a.out)[at] = (uint16_t)f32_to_bf16_rne(y);
  else static_cast<_Float16*>(a.out)[at] = (_Float16)y;
}

// The 128 columns from n0, by one workgroup.
template <int kWaves>
__device__ __forceinline__ void join_tile(const MoeArgs& a, int n0) {
  for (int i = threadIdx.x; i < a.tokens * 2 * kHalf; i += 64 * kWaves)
    if (n0 + i % (2 * kHalf) < a.hidden) join_value(a, i / (2 * kHalf), n0 + i % (2 * kHalf));
}

__global__ __launch_bounds__(256) void moe_join(const MoeArgs a) {
  const long at = (long)blockIdx.x * 256 + threadIdx.x;
  if (at < (long)a.tokens * a.hidden) join_value(a, (int)(at / a.hidden), (int)(at % a.hidden));
}

// One product of the layer.  FIRST: up and gate, h = up * silu(gate) to a.h,
// the halves of the tile being the same 64 columns of each; otherwise down,
// 128 columns, to a.part.
template <int LAYOUT, bool FIRST, int TYPE, int GROUPED, int kWaves>
__global__ __launch_bounds__(64 * kWaves, 2) void moe_product(const MoeArgs a) {
  constexpr int kStep = FIRST ? kHalf : 2 * kHalf;  // columns from one workgroup to the next
  // the waves' sums, and before them 1024 dwords a wave for what ends in a piece
  __shared__ __align__(16) float red[kWaves / 2 * 16 * kPitch];
  static_assert(sizeof(red) >= kWaves * 4096, "room for the pieces that end");
  __shared__ uint32_t lds_scale[GROUPED ? kWaves * 256 : 1];  // a wave's four groups of 128 scales
  __shared__ uint16_t list[kRows];
  __shared__ int16_t id[kMostPairs];
  __shared__ int count[kMostExperts];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int pairs = a.tokens * a.top;

  // Workgroups go round the 8 XCDs in turn.  Where a row's piece is half a
  // cache line (64 columns of NN), neighbouring tiles go to one XCD, which then
  // fetches the line once: 205 -> 158 us for 14 experts of 2048 x 22016 bytes.
  // Elsewhere that only narrows an XCD's addresses.
  constexpr bool kNeighbours = FIRST && LAYOUT == SHK_LAYOUT_NN;
  const int tile = kNeighbours ? (blockIdx.x % 8) * (gridDim.x / 8) + blockIdx.x / 8 : blockIdx.x;
  if (FIRST && blockIdx.y == 0)  // the down product counts from zero
    for (int i = blockIdx.x * 64 * kWaves + threadIdx.x; i < a.tiles; i += gridDim.x * 64 * kWaves) a.arrived[i] = 0;
  if (tile * kStep >= (FIRST ? a.inner_pad : a.cols)) return;

  // The pairs of each expert that is hit are dealt out in order, kRows at a
  // time: this workgroup's are the blockIdx.y-th.  `row0` counts the expert's
  // pairs before them, `shares` all such parts.
  int expert = -1, rank = blockIdx.y, row0 = 0, rows = 0, shares = 0;
  if (pairs <= 64) {
    // experts in the order of their first pairs, all in a wave's registers
    const int mine = lane < pairs ? id_of(a, lane) : -1;
    unsigned long open = __ballot(mine >= 0), same = 0;
    while (open != 0) {
      const int e = __shfl(mine, __builtin_ctzll(open), 64);
      const unsigned long all = __ballot(mine == e);
      const int before = rank - shares, here = (__popcll(all) + kRows - 1) / kRows;
      if (before >= 0 && before < here) expert = e, same = all, row0 = kRows * before;
      shares += here;
      open &= ~all;
    }
    rows = __popcll(same) - row0;
    const int at = __popcll(same & ((1ul << lane) - 1)) - row0;
    if (wave == 0 && expert >= 0 && mine == expert && at >= 0 && at < kRows) list[at] = (uint16_t)lane;
  } else {
    // counted in LDS
    for (int e = threadIdx.x; e < a.experts; e += 64 * kWaves) count[e] = 0;
    __syncthreads();
    for (int p = threadIdx.x; p < pairs; p += 64 * kWaves) {
      const int e = id_of(a, p);
      id[p] = (int16_t)e;
      if (e >= 0) atomicAdd(&count[e], 1);
    }
    __syncthreads();
    for (int e0 = 0; e0 < a.experts; e0 += 64) {
      const int n = e0 + lane < a.experts ? count[e0 + lane] : 0, here = (n + kRows - 1) / kRows;
      int upto = here;  // with the lanes before
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const int v = __shfl_up(upto, d, 64);
        upto += lane >= d ? v : 0;
      }
      const int before = rank - shares - (upto - here);
      const unsigned long at = __ballot(before >= 0 && before < here);
      if (at != 0) {
        const int l = __builtin_ctzll(at);
        expert = e0 + l, row0 = kRows * __shfl(before, l, 64), rows = __shfl(n, l, 64) - row0;
      }
      shares += __shfl(upto, 63, 64);
    }
    if (wave == 0 && expert >= 0) {
      int at = -row0;
      for (int p0 = 0; p0 < pairs && at < kRows; p0 += 64) {
        const bool mine = p0 + lane < pairs && id[p0 + lane] == expert;
        const unsigned long all = __ballot(mine);
        const int to = at + __popcll(all & ((1ul << lane) - 1));
        if (mine && to >= 0 && to < kRows) list[to] = (uint16_t)(p0 + lane);
        at += __popcll(all);
      }
    }
  }
  expert = __builtin_amdgcn_readfirstlane(expert);
  rows = __builtin_amdgcn_readfirstlane(min(rows, kRows));
  shares = __builtin_amdgcn_readfirstlane(shares);
  if constexpr (!FIRST)
    if (a.joined && shares == 0 && blockIdx.y == 0) join_tile<kWaves>(a, tile * kStep);  // no token asks for any expert
  if (expert < 0) return;  // the same for all threads
  __syncthreads();

  constexpr int kColumns = FIRST ? 2 : 1;
  const Codes s{a.w + (long)expert * kColumns * a.cols * a.k_packed,
                a.w + (long)a.experts * kColumns * a.cols * a.k_packed, kColumns * a.cols, a.k_packed};
  const int n0 = tile * kStep;
  const uint16_t* scale = a.scale + (long)expert * (GROUPED ? a.groups : 1) * s.total;

  // This wave's K: whole pieces and whole scale groups.  A piece is half a
  // cache line of NT's rows: there the waves take pieces in turn, so that both
  // halves are asked for at about the same time.
  const bool turns = LAYOUT == SHK_LAYOUT_NT && a.group <= kSuper;
  const int unit = GROUPED ? max(a.group, kSuper) : kSuper;
  const int units = (a.k + unit - 1) / unit, each = (units + kWaves - 1) / kWaves;
  const int k_first = turns ? wave * kSuper : min(a.k, wave * each * unit);
  const int k_last = turns ? a.k : min(a.k, (wave + 1) * each * unit), k_step = turns ? kWaves * kSuper : kSuper;

  moe_rows<LAYOUT, FIRST, TYPE, GROUPED, kWaves>(a, s, scale, list, rows, n0, k_first, k_last, k_step, red,
                                                 lds_scale + 256 * wave);
  if (!FIRST && a.joined) {
    // The last workgroup of a tile adds up its pairs, in a fixed order.  This
    // rests on gfx942's memory model as LLVM's AMDGPU guide states it, which
    // gfx950 shares: a device-scope store (sc1) has reached the level that all
    // XCDs see once vmcnt counts it off, and a device-scope load (sc1) takes
    // nothing older from its own caches.  Every wave waits for its stores
    // before the barrier, so they are there before thread 0 counts the
    // workgroup, and the last one's loads come after its count.  A release and
    // acquire count would also write back and invalidate the caches
    // (buffer_wbl2, buffer_inv), for ordinary stores and loads, of which none
    // is shared here: 16 pairs of 64 experts of 4096 x 1408 53.6 us instead of
    // 47.5.
    __shared__ int last;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0)
      last = __hip_atomic_fetch_add(a.arrived + tile, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == shares - 1;
    __syncthreads();
    if (last) join_tile<kWaves>(a, tile * kStep);
  }
}

template <int LAYOUT, bool FIRST, int TYPE, int GROUPED>
void launch_waves(const MoeArgs& a, dim3 grid, hipStream_t s) {
  // A workgroup's waves share K.  Few workgroups (at most one on each of the
  // 256 CUs): eight, the shortest way through.  Many: every wave's start and
  // end count, and two waves halve them, until K is so long that workgroups
  // become uneven.  Without scale groups to add up in between, up and gate
  // come to that sooner.  Four waves in between and for a long K.
  // The layer of 16 tokens, 6 of 64 experts, us with two / four waves for
  // up and gate (inner 2560 up to hidden 2048, 1408 from 2816):
  //   hidden             512    1088   1536   2048    2816    3584     4096
  //   NN, bf16         43/45   71/73  78/78  92/93   74/70   97/91  105/98
  //   NN, f16          44/47   74/75  81/80  96/94   79/72  103/93
  //   NT, bf16         48/53   82/84  86/86  98/96   80/76  103/97
  //   NT, f16          52/53   88/86  93/89  106/100 77/78  100/100
  //   NN, groups of 128 (inner 1408)  53/58          73/79   98/101
  //   NT, groups of 128 (inner 1408)  57/61  64/67   80/82  103/103 113/110
  // and for down (hidden 2816):
  //   inner              704    1408   2816
  //   NN               60/63   74/79  125/130
  //   NT, groups of 128 61/66  80/83  139/142
  // With two / four / eight for one of the products, up and gate then down:
  //   16 tokens, 6 of 64 experts of 2048 x 1408, NT, groups of 128
  //                                   64 / 68 / 81       64 / 66 / 75
  //   61 tokens, 2 of 16 experts of 4096 x 11008, NN
  //                                   241 / 234 / 274    250 / 234 / 240
  //   16 tokens, 2 of 16 experts of 2048 x 1408 (408 and 272 workgroups), NN
  //                                   33 / 29 / 32       32 / 29 / 30
  constexpr int kTwoBelow = FIRST && !GROUPED ? 1536 : 4096;
  if (grid.x * grid.y <= 256)
    hipLaunchKernelGGL((moe_product<LAYOUT, FIRST, TYPE, GROUPED, 8>), grid, dim3(512), 0, s, a);
  else if (a.k < kTwoBelow && grid.x * grid.y > 1024)
    hipLaunchKernelGGL((moe_product<LAYOUT, FIRST, TYPE, GROUPED, 2>), grid, dim3(128), 0, s, a);
  else
    hipLaunchKernelGGL((moe_product<LAYOUT, FIRST, TYPE, GROUPED, 4>), grid, dim3(256), 0, s, a);
}

template <int LAYOUT, bool FIRST, int TYPE>
hipError_t launch_product(const MoeArgs& a, unsigned columns, unsigned hit, hipStream_t s) {
  constexpr unsigned kStep = FIRST ? kHalf : 2 * kHalf;
  const dim3 grid(((columns + kStep - 1) / kStep + 7) / 8 * 8, hit);
  if (a.group >= kSuper) launch_waves<LAYOUT, FIRST, TYPE, kLargeGroups>(a, grid, s);
  else if (a.group) launch_waves<LAYOUT, FIRST, TYPE, kSmallGroups>(a, grid, s);
  else launch_waves<LAYOUT, FIRST, TYPE, 0>(a, grid, s);
  return hipGetLastError();
}

hipError_t launch_layer(const shk_moe& x, MoeArgs a, hipStream_t s) {
  constexpr int LAYOUT = SHK_LAYOUT;
  // with no pairs the down product still writes the zeros
  const long pairs = x.tokens * x.top, most = std::min(pairs, (long)x.experts);
  const unsigned hit = (unsigned)std::max(1L, most + (pairs - most) / 16);
  a.w = static_cast<const uint8_t*>(x.up_gate);
  a.scale = static_cast<const uint16_t*>(x.up_gate_scale);
  a.k = a.hidden, a.k_packed = (a.hidden + 1) / 2, a.cols = a.inner;
  a.groups = a.group ? (a.k + a.group - 1) / a.group : 1;
  // the columns up to inner_pad are written too, as zeros
  hipError_t err = x.type == SHK_SRC_BF16 ? launch_product<LAYOUT, true, SHK_SRC_BF16>(a, (unsigned)a.inner_pad, hit, s)
                                          : launch_product<LAYOUT, true, SHK_SRC_F16>(a, (unsigned)a.inner_pad, hit, s);
  if (err != hipSuccess) return err;
  a.w = static_cast<const uint8_t*>(x.down);
  a.scale = static_cast<const uint16_t*>(x.down_scale);
  a.k = a.inner, a.k_packed = (a.inner + 1) / 2, a.cols = a.hidden;
  a.groups = a.group ? (a.k + a.group - 1) / a.group : 1;
  err = launch_product<LAYOUT, false, SHK_SRC_BF16>(a, (unsigned)a.cols, hit, s);
  if (err != hipSuccess || a.joined) return err;
  const long values = (long)a.tokens * a.hidden;
  hipLaunchKernelGGL(moe_join, dim3((unsigned)((values + 255) / 256)), dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace

#if SHK_LAYOUT == 0  // SHK_LAYOUT_NN
hipError_t launch_moe_nn(const shk_moe& x, hipStream_t s) {
#else
hipError_t launch_moe_nt(const shk_moe& x, hipStream_t s) {
#endif
  MoeArgs a{};
  a.x = x.x, a.x_stride = x.x_stride;
  a.ids = x.ids, a.id8 = x.id_bytes == 8;
  a.share = x.share;
  a.h = static_cast<uint16_t*>(x.workspace);
  a.part = static_cast<float*>(x.workspace) + x.tokens * x.top * moe_inner_pad(x);
  a.arrived = reinterpret_cast<int*>(a.part + x.tokens * x.top * x.hidden);
  a.tiles = (int)moe_down_tiles(x);
  a.out = x.out;
  a.group = (int)x.group;
  a.tokens = (int)x.tokens, a.top = (int)x.top, a.experts = (int)x.experts;
  a.hidden = (int)x.hidden, a.inner = (int)x.inner, a.inner_pad = (int)moe_inner_pad(x);
  a.type = (int)x.type;
  // One workgroup a tile adds few pairs sooner than another launch starts; with
  // many it would keep all others waiting (96 pairs: 29 us of the down product
  // became 50, where the launch is 4).
  a.joined = x.tokens * x.top <= 16;
  return launch_layer(x, a, s);
}

}  // namespace shk
