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
#include <type_traits>

#include "shk_common.h"
#include "shk_moe.h"

namespace shk {
namespace {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 8;
constexpr int kHalf = 64;          // columns of half a workgroup's tile
constexpr int kSuper = 128;        // K values a wave loads at a time, four products deep
constexpr int kMostPairs = 1024;   // (token, expert) pairs of a call
constexpr int kMostExperts = 1024;

struct MoeArgs {
  const void* x;
  long x_stride;
  const uint8_t* w;        // codes of this product
  const uint16_t* scale;
  const void* ids;
  const float* share;
  uint16_t* h;             // [pairs][high, low][inner_pad]: bf16 terms, eights in the order of expand
  float* part;             // [pairs][hidden]
  void* out;
  int k, k_packed, cols;   // this product's K, its bytes, and columns (of up alone)
  int group, groups;       // scale group (0: per channel) and groups of K
  int tokens, top, experts, hidden, inner, inner_pad;
  int type, id8;
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
  w ^= 0x88888888u;
  return __builtin_bit_cast(b8, u4{((w << 3) & 0x00780078u) | 0x41804180u, ((w >> 1) & 0x00780078u) | 0x41804180u,
                                   ((w >> 5) & 0x00780078u) | 0x41804180u, ((w >> 9) & 0x00780078u) | 0x41804180u});
}

// Where a product's codes come from: the expert's matrix, and the end of all
// experts' (nothing is read past it).
struct Codes {
  const uint8_t *w, *end;
  int total, k_packed;  // columns of a row (NN) and bytes of one (NT)
};

// A uniform address, kept in scalar registers: the compiler would otherwise
// keep one 64-bit vector address for every load of a piece.
__device__ __forceinline__ const uint8_t* scalar(const uint8_t* p) {
  asm("" : "+s"(p));
  return p;
}

// 16 dwords of a lane: the codes of 128 K values from k0 for 64 columns from
// n0, as they are stored.  What lies outside the expert's matrix meets
// activations of zero or is not stored, so it may be anything.
template <int LAYOUT>
__device__ __forceinline__ void load_w(const Codes& s, int k0, int n0, uint32_t (&o)[16]) {
  const int lane = threadIdx.x & 63, g = lane / 16, c = lane % 16;
  if constexpr (LAYOUT == SHK_LAYOUT_NT) {  // [n][k_packed]: 16 bytes of the rows 4 c + j
    const uint32_t mine = (uint32_t)(4 * c * s.k_packed + 16 * g);
    const uint8_t* p = s.w + (long)n0 * s.k_packed + k0 / 2;
#pragma unroll
    for (int j = 0; j < 4; ++j) __builtin_memcpy(&o[4 * j], scalar(p + (long)j * s.k_packed) + mine, 16);
  } else {  // [k_packed][n]: four columns of the rows 16 q + 4 g + i
    const uint32_t mine = (uint32_t)(4 * g * s.total + 4 * c);
    const uint8_t* p = s.w + (long)(k0 / 2) * s.total + n0;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      __builtin_memcpy(&o[i], scalar(p + (long)(16 * (i / 4) + i % 4) * s.total) + mine, 4);
  }
}

// The same where part of it lies past the end of all codes, by way of 16
// dwords of LDS a lane (few registers; at most the last expert's last pieces).
template <int LAYOUT>
__device__ __forceinline__ void load_w_end(const Codes& s, int k0, int n0, uint32_t* lds, uint32_t (&o)[16]) {
  const int lane = threadIdx.x & 63, g = lane / 16, c = lane % 16;
#pragma unroll 1
  for (int i = 0; i < 16; ++i) {
    const uint8_t* p = LAYOUT == SHK_LAYOUT_NT
                           ? s.w + (long)(n0 + 4 * c + i / 4) * s.k_packed + k0 / 2 + 16 * g + 4 * (i % 4)
                           : s.w + (long)(k0 / 2 + 16 * (i / 4) + 4 * g + i % 4) * s.total + n0 + 4 * c;
    // the last dword there is, shifted to where it would be
    const long over = p - (s.end - 4);
    uint32_t v;
    __builtin_memcpy(&v, over > 0 ? s.end - 4 : p, 4);
    lds[i * 64 + lane] = over <= 0 ? v : (over < 4 ? v >> (8 * over) : 0u);
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
__device__ __forceinline__ void load_x(const MoeArgs& a, const uint16_t* row, int k, u4 (&o)[kLoads<FIRST, TYPE>]) {
  if constexpr (FIRST) {
    __builtin_memcpy(&o[0], row + k, 16);
  } else {
    o[0] = *reinterpret_cast<const u4*>(row + k);
    o[1] = *reinterpret_cast<const u4*>(row + a.inner_pad + k);
  }
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

// One product of the layer.  FIRST: up and gate, h = up * silu(gate) to a.h,
// the halves of the tile being the same 64 columns of each; otherwise down,
// 128 columns, to a.part.  RT: row tiles of 16 tokens a pass.
template <int LAYOUT, bool FIRST, int RT, int TYPE, bool GROUPED>
__global__ __launch_bounds__(64 * kWaves, 2) void moe_product(const MoeArgs a) {
  constexpr int kPitch = 2 * kHalf + 4;
  constexpr int kStep = FIRST ? kHalf : 2 * kHalf;  // columns from one workgroup to the next
  constexpr int kT = kTerms<FIRST, TYPE>, kL = kLoads<FIRST, TYPE>;
  // the waves' sums, and before them 1024 dwords a wave for what ends in a piece
  __shared__ __align__(16) float red[kWaves / 2][16 * kPitch];
  static_assert(sizeof(red) >= kWaves * 4096, "room for the pieces that end");
  __shared__ uint16_t list[kMostPairs];
  __shared__ int count[kMostExperts];
  const int lane = threadIdx.x & 63, g = lane / 16, c = lane % 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int pairs = a.tokens * a.top;

  // the blockIdx.y-th expert that is hit, and its pairs in order
  int expert = -1, rank = blockIdx.y, rows = 0;
  if (pairs <= 64) {
    // experts in the order of their first pairs, all in a wave's registers
    const int id = lane < pairs ? id_of(a, lane) : -1;
    unsigned long open = __ballot(id >= 0), same = 0;
    for (; open != 0; --rank) {
      const int e = __shfl(id, __builtin_ctzll(open), 64);
      same = __ballot(id == e);
      if (rank == 0) {
        expert = e;
        break;
      }
      open &= ~same;
    }
    if (expert < 0) return;  // the same for all threads
    rows = __popcll(same);
    if (wave == 0 && id == expert) list[__popcll(same & ((1ul << lane) - 1))] = (uint16_t)lane;
  } else {
    // experts in ascending order, counted in LDS
    for (int e = threadIdx.x; e < a.experts; e += 64 * kWaves) count[e] = 0;
    __syncthreads();
    for (int p = threadIdx.x; p < pairs; p += 64 * kWaves) {
      const int e = id_of(a, p);
      if (e >= 0) atomicAdd(&count[e], 1);
    }
    __syncthreads();
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
    if (expert < 0) return;
    rows = count[expert];
    if (wave == 0) {
      int at = 0;
      for (int p0 = 0; p0 < pairs; p0 += 64) {
        const bool mine = p0 + lane < pairs && id_of(a, p0 + lane) == expert;
        const unsigned long all = __ballot(mine);
        if (mine) list[at + __popcll(all & ((1ul << lane) - 1))] = (uint16_t)(p0 + lane);
        at += __popcll(all);
      }
    }
  }
  expert = __builtin_amdgcn_readfirstlane(expert);
  rows = __builtin_amdgcn_readfirstlane(rows);
  __syncthreads();

  constexpr int kColumns = FIRST ? 2 : 1;
  const Codes s{a.w + (long)expert * kColumns * a.cols * a.k_packed,
                a.w + (long)a.experts * kColumns * a.cols * a.k_packed, kColumns * a.cols, a.k_packed};
  const int n0 = blockIdx.x * kStep, n1 = n0 + (FIRST ? a.cols : kHalf);  // the halves' first columns
  const uint16_t* scale = a.scale + (long)expert * (GROUPED ? a.groups : 1) * s.total;

  // this wave's K: whole scale groups, in steps of 32
  const int unit = GROUPED ? a.group : 32;
  const int units = (a.k + unit - 1) / unit, each = (units + kWaves - 1) / kWaves;
  const int k_first = min(a.k, wave * each * unit), k_last = min(a.k, (wave + 1) * each * unit);

  const __bf16 one = (__bf16)1.0f;
  const b8 ones = {one, one, one, one, one, one, one, one};

  for (int row0 = 0; row0 < rows; row0 += 16 * RT) {
    if (row0 > 0) __syncthreads();  // red has been read
    // columns of a product without a row repeat the last one; they are not stored
    const uint16_t* src[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int p = list[min(row0 + 16 * t + c, rows - 1)];
      src[t] = FIRST ? static_cast<const uint16_t*>(a.x) + (p / a.top) * a.x_stride : a.h + (long)p * 2 * a.inner_pad;
    }
    f4 acc[RT][8], sum[RT][2], all[RT][GROUPED ? 8 : 1];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      sum[t][0] = sum[t][1] = f4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        acc[t][j] = f4{0, 0, 0, 0};
        if constexpr (GROUPED) all[t][j] = f4{0, 0, 0, 0};
      }
    }
    uint32_t* lds = reinterpret_cast<uint32_t*>(&red[0][0]) + 1024 * wave;
    u4 x[RT][4][kL];
    uint32_t w0[16], w1[16];
    auto codes = [&](int k0, int n, uint32_t (&w)[16]) {
      if (inside<LAYOUT>(s, k0, n)) load_w<LAYOUT>(s, k0, n, w);
      else load_w_end<LAYOUT>(s, k0, n, lds, w);
    };
    auto activations = [&](int k0, u4 (&o)[RT][4][kL]) {
      if (FIRST && k0 + kSuper > a.k) {  // x ends in this piece: zeros past it, by way of LDS
        uint16_t* h = reinterpret_cast<uint16_t*>(lds) + 8 * lane;
#pragma unroll
        for (int t = 0; t < RT; ++t) {
#pragma unroll 1
          for (int i = 0; i < 32; ++i) {
            const int k = k0 + 32 * (i / 8) + 8 * g + i % 8;
            h[512 * (i / 8) + i % 8] = k < a.k ? src[t][k] : (uint16_t)0;
          }
#pragma unroll
          for (int q = 0; q < 4; ++q) o[t][q][0] = *reinterpret_cast<const u4*>(h + 512 * q);
        }
        return;
      }
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int q = 0; q < 4; ++q) load_x<FIRST, TYPE>(a, src[t], k0 + 32 * q + 8 * g, o[t][q]);
    };
    auto multiply = [&](int k0, auto half, uint32_t (&w)[16]) {
      constexpr int kAt = decltype(half)::value;
      arrange<LAYOUT>(w);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int k = k0 + 32 * q;
        if (k < k_last) {
          b8 xt[RT][kT];
#pragma unroll
          for (int t = 0; t < RT; ++t) {
            terms<FIRST, TYPE>(x[t][q], xt[t]);
#pragma unroll
            for (int i = 0; i < kT; ++i) sum[t][kAt] = mfma_bf16(ones, xt[t][i], sum[t][kAt]);
          }
          uint32_t o[4];
          step_codes<LAYOUT>(w, q, o);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const b8 v = expand(o[j]);
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
              for (int i = 0; i < kT; ++i) acc[t][4 * kAt + j] = mfma_bf16(v, xt[t][i], acc[t][4 * kAt + j]);
          }
          if constexpr (GROUPED) {
            if (k + 32 >= k_last || (k + 32) % a.group == 0) {
              // the group ends: its sums, without the offset, times its scales
              const uint16_t* sc = scale + (long)(k / a.group) * s.total;
              const int n = (kAt ? n1 : n0) + 16 * g;
              uint16_t f[16];
              if ((kAt ? n1 : n0) + kHalf <= s.total) {
                __builtin_memcpy(f, sc + n, 32);
              } else {
                uint16_t* h = reinterpret_cast<uint16_t*>(lds) + 16 * lane;
#pragma unroll 1
                for (int i = 0; i < 16; ++i) h[i] = sc[min(n + i, s.total - 1)];
                __builtin_memcpy(f, h, 32);
              }
#pragma unroll
              for (int t = 0; t < RT; ++t) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
#pragma unroll
                  for (int r = 0; r < 4; ++r)
                    all[t][4 * kAt + j][r] +=
                        bf16_bits_to_f32(f[4 * r + j]) * (acc[t][4 * kAt + j][r] - 24.0f * sum[t][kAt][r]);
                  acc[t][4 * kAt + j] = f4{0, 0, 0, 0};
                }
                sum[t][kAt] = f4{0, 0, 0, 0};
              }
            }
          }
        }
      }
    };
    // Each half's codes are on their way while the other half is multiplied;
    // so are the next activations where two sets of them fit the registers.
    constexpr bool kAhead = RT * kL == 1;
    if (k_first < k_last) {
      if constexpr (kAhead) activations(k_first, x);
      codes(k_first, n0, w0);
    }
    for (int k0 = k_first; k0 < k_last; k0 += kSuper) {
      const bool more = k0 + kSuper < k_last;
      if constexpr (!kAhead) activations(k0, x);
      codes(k0, n1, w1);
      multiply(k0, std::integral_constant<int, 0>{}, w0);
      if (more) codes(k0 + kSuper, n0, w0);
      if constexpr (kAhead) {
        u4 xn[RT][4][kL];
        if (more) activations(k0 + kSuper, xn);
        multiply(k0, std::integral_constant<int, 1>{}, w1);
        if (more) {
#pragma unroll
          for (int q = 0; q < 4; ++q) x[0][q][0] = xn[0][q][0];
        }
      } else {
        multiply(k0, std::integral_constant<int, 1>{}, w1);
      }
    }
    // The waves' sums: lane (g, c) holds token c, columns 16 g + 4 r + j of
    // each half.  Waves 4 to 7 hand theirs to waves 0 to 3 first.
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      f4 v[8];  // [half][r] over j
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (GROUPED) v[4 * half + r][j] = all[t][4 * half + j][r];
            else v[4 * half + r][j] = acc[t][4 * half + j][r] - 24.0f * sum[t][half][r];
          }
      float* mine = &red[wave % (kWaves / 2)][c * kPitch + 16 * g];
      __syncthreads();
      if (wave >= kWaves / 2) {
#pragma unroll
        for (int i = 0; i < 8; ++i) *reinterpret_cast<f4*>(mine + (i / 4) * kHalf + 4 * (i % 4)) = v[i];
      }
      __syncthreads();
      if (wave < kWaves / 2) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          f4* at = reinterpret_cast<f4*>(mine + (i / 4) * kHalf + 4 * (i % 4));
          *at += v[i];
        }
      }
      __syncthreads();
      const int here = min(rows - row0 - 16 * t, 16);
      if constexpr (FIRST) {
        for (int i = threadIdx.x; i < here * kHalf; i += 64 * kWaves) {
          const int r = i / kHalf, n = i % kHalf, col = n0 + n;
          if (col >= a.inner_pad) continue;
          float h = 0.0f;  // up to inner_pad
          if (col < a.cols) {
            float up = 0.0f, gate = 0.0f;
#pragma unroll
            for (int q = 0; q < kWaves / 2; ++q) up += red[q][r * kPitch + n], gate += red[q][r * kPitch + kHalf + n];
            if constexpr (!GROUPED) up *= load_bf16(scale + col), gate *= load_bf16(scale + a.cols + col);
            h = up * (gate / (1.0f + __expf(-gate)));
          }
          // place 2 i + u of an eight holds its element i + 4 u
          const int at = (col & ~7) | (2 * (col & 3) + ((col >> 2) & 1));
          const uint32_t hi = f32_to_bf16_rne(h);
          uint16_t* dst = a.h + (long)list[row0 + 16 * t + r] * 2 * a.inner_pad + at;
          dst[0] = (uint16_t)hi;
          dst[a.inner_pad] = (uint16_t)f32_to_bf16_rne(h - bf16_bits_to_f32((uint16_t)hi));
        }
      } else {
        for (int i = threadIdx.x; i < here * 2 * kHalf; i += 64 * kWaves) {
          const int r = i / (2 * kHalf), n = i % (2 * kHalf), col = n0 + n;
          if (col >= a.cols) continue;
          float v2 = 0.0f;
#pragma unroll
          for (int q = 0; q < kWaves / 2; ++q) v2 += red[q][r * kPitch + n];
          if constexpr (!GROUPED) v2 *= load_bf16(scale + col);
          a.part[(long)list[row0 + 16 * t + r] * a.hidden + col] = v2;
        }
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

template <int LAYOUT, bool FIRST, int TYPE, bool GROUPED>
void launch_rt(const MoeArgs& a, dim3 grid, hipStream_t s) {
  constexpr dim3 block(64 * kWaves);
  if (a.tokens <= 16) hipLaunchKernelGGL((moe_product<LAYOUT, FIRST, 1, TYPE, GROUPED>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((moe_product<LAYOUT, FIRST, 2, TYPE, GROUPED>), grid, block, 0, s, a);
}

template <int LAYOUT, bool FIRST, int TYPE>
hipError_t launch_product(const MoeArgs& a, unsigned columns, unsigned hit, hipStream_t s) {
  const dim3 grid((columns + (FIRST ? kHalf : 2 * kHalf) - 1) / (FIRST ? kHalf : 2 * kHalf), hit);
  if (a.group) launch_rt<LAYOUT, FIRST, TYPE, true>(a, grid, s);
  else launch_rt<LAYOUT, FIRST, TYPE, false>(a, grid, s);
  return hipGetLastError();
}

hipError_t launch_join(const MoeArgs& a, hipStream_t s) {
  const long values = (long)a.tokens * a.hidden;
  hipLaunchKernelGGL(moe_join, dim3((unsigned)((values + 255) / 256)), dim3(256), 0, s, a);
  return hipGetLastError();
}

template <int LAYOUT>
hipError_t launch_layout(const shk_moe& x, MoeArgs a, hipStream_t s) {
  const unsigned hit = (unsigned)std::min(x.tokens * x.top, x.experts);
  if (hit == 0) return launch_join(a, s);
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
  return err != hipSuccess ? err : launch_join(a, s);
}

}  // namespace

// h's rows are whole pieces of 128 K values, the rest zero.
static long inner_pad(const shk_moe& a) { return (a.inner + kSuper - 1) / kSuper * kSuper; }

int64_t moe_workspace(const shk_moe& a) { return a.tokens * a.top * (inner_pad(a) + a.hidden) * 4; }

hipError_t launch_moe(const shk_moe& x, hipStream_t s) {
  MoeArgs a{};
  a.x = x.x, a.x_stride = x.x_stride;
  a.ids = x.ids, a.id8 = x.id_bytes == 8;
  a.share = x.share;
  a.h = static_cast<uint16_t*>(x.workspace);
  a.part = static_cast<float*>(x.workspace) + x.tokens * x.top * inner_pad(x);
  a.out = x.out;
  a.group = (int)x.group;
  a.tokens = (int)x.tokens, a.top = (int)x.top, a.experts = (int)x.experts;
  a.hidden = (int)x.hidden, a.inner = (int)x.inner, a.inner_pad = (int)inner_pad(x);
  a.type = (int)x.type;
  return x.layout == SHK_LAYOUT_NT ? launch_layout<SHK_LAYOUT_NT>(x, a, s) : launch_layout<SHK_LAYOUT_NN>(x, a, s);
}

}  // namespace shk
