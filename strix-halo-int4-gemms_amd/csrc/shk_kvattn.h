// Attention of a few query rows over a piece of the quantized cache: what the
// streaming kernel and the shared-prefix kernel have in common (k_kvattn.hip).
//
// Tokens are taken 64 at a time, in four blocks i of 16:
//
//   S^T = K q^T   v_mfma_f32_16x16x32_f16, tokens in the rows, query rows in
//                 the columns: lane (g = lane / 16, c = lane % 16) gets the
//                 tokens 16 i + 4 g + r, r = 0..3, of query row c.
//   O^T = V^T P^T the same instruction with head_dim in the rows; its second
//                 operand wants query row c and 8 tokens of lane group g,
//                 which is what the lane holds after the softmax when the 32
//                 tokens of a product are taken in the order (i, g, r).  P
//                 never leaves its lane.
//
// K and V stay as they are stored until they reach a product.  The codes are
// small integers, so f16 holds them exactly; a token's scale multiplies its
// score (K) or its probability (V) instead of head_dim values.  q enters as
// q * 2^-e with its row's largest magnitude in [1, 2): bf16 and f16 values
// then keep all their bits in f16 down to 2^-14 of the largest one.
//
// A row's probabilities are taken relative to
//   m = max(score) + exponent(max |v_scale|) - 13,
// in powers of two and over what the row has met so far, not to the largest
// score: 2^(score - m) * v_scale is then at most 2^15, so f16 does not
// overflow and keeps all its bits down to 2^-27 of the largest probability
// times the largest scale.  The two need not be one token's: where they are
// not, the error is small beside the largest |v|, not beside the output.  An
// exponent below -80 counts as -80, so that the sum cannot overflow either.
// Probabilities below 2^-126 of a reference are lost: a row's sum keeps its
// bits for scales up to 2^100, and 12 of them for the largest there are.  For
// f16 outputs the term is split into two f16 terms, because one rounding to 11
// bits would be as large as the output's own.  Maxima, sums and outputs are f32.
#pragma once

#include "shk_common.h"
#include "shk_kvcache.h"
#include "shk_loads.h"

namespace shk {

constexpr int kKvTile = 64;
constexpr float kLog2e = 1.4426950408889634f;

// Two codes that sit in the low bytes / nibbles of a dword's halves, as f16:
// 0x6400 | n is 1024 + n exactly, n the code with its sign bit flipped (code + 8
// or + 128), which the exclusive or does on the way.
__device__ __forceinline__ h2 nib_lo(uint32_t w) {
  return __builtin_bit_cast(h2, (w & 0x000F000Fu) ^ 0x64086408u) - (h2)(_Float16)1032.0f;
}
__device__ __forceinline__ h2 nib_hi(uint32_t w) {  // bits 4..7: 1024 + 16 n, over 16
  return __builtin_elementwise_fma(__builtin_bit_cast(h2, (w & 0x00F000F0u) ^ 0x64806480u), (h2)(_Float16)0.0625f,
                                   (h2)(_Float16)-72.0f);
}
__device__ __forceinline__ h2 byte_pair(uint32_t w) {  // w = byte | byte << 16
  return __builtin_bit_cast(h2, w ^ 0x64806480u) - (h2)(_Float16)1152.0f;
}

__device__ __forceinline__ h8 join(h2 a, h2 b, h2 c, h2 d) {
  return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// 8 codes of one row as a product's operand.  int4 codes 0..7 of a dword come
// in the order 0 4 1 5 2 6 3 7 (kv_order), which q's operand repeats.
__device__ __forceinline__ h8 row_codes4(uint32_t w) {
  const uint32_t u = w >> 8;
  return join(nib_lo(w), nib_hi(w), nib_lo(u), nib_hi(u));
}
__device__ __forceinline__ h8 row_codes8(uint32_t lo, uint32_t hi) {
  return join(byte_pair(perm_b32(0, lo, 0x0C010C00u)), byte_pair(perm_b32(0, lo, 0x0C030C02u)),
              byte_pair(perm_b32(0, hi, 0x0C010C00u)), byte_pair(perm_b32(0, hi, 0x0C030C02u)));
}
template <int BITS>
__device__ __forceinline__ constexpr int kv_order(int i) {
  return BITS == 4 ? (i / 2) + 4 * (i % 2) : i;
}

__device__ __forceinline__ f4 mfma_f16(h8 a, h8 b, f4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Combines the four lane groups (lanes c, c + 16, c + 32, c + 48).  A register
// swapped with itself gives the even rows of 16 lanes twice and the odd ones
// twice (then the halves), at the speed of a VALU operation: a shuffle by way of
// LDS is waited for three times a step.
template <typename F>
__device__ __forceinline__ uint32_t groups(uint32_t v, F f) {
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = f(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return f(b[0], b[1]);
}
__device__ __forceinline__ uint32_t groups_most(uint32_t v) {
  return groups(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}
__device__ __forceinline__ float groups_max(float v) {
  return __uint_as_float(groups(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(__builtin_fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}
__device__ __forceinline__ float groups_sum(float v) {
  return __uint_as_float(groups(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}

// max(a, |b|), a NaN where b is one: two of them are one instruction.
__device__ __forceinline__ float larger(float a, float b) {
  return __builtin_elementwise_maximum(a, __builtin_fabsf(b));
}

// 2^(x / 2).  References may lie up to 207 apart, which 2^x does not hold; a
// sum that is large by as much is weighted with this twice.
__device__ __forceinline__ float half_weight(float x) { return __builtin_amdgcn_exp2f(0.5f * x); }

struct KvView {  // one key head of the cache
  const uint8_t *kc, *vc;
  const uint16_t *ks, *vs;
  int pages, page_shift, heads, head;

  // The page of a block of 16 tokens, asked for a step before it is needed.
  __device__ __forceinline__ int page_of(const int32_t* table, int blk) const { return table[blk >> (page_shift - 4)]; }
  // The block's first row; a page outside the cache reads as the first one
  // and is remembered.
  __device__ __forceinline__ long row_of(int page, int blk, bool& bad) const {
    page = __builtin_amdgcn_readfirstlane(page);
    if ((unsigned)page >= (unsigned)pages) page = 0, bad = true;
    return ((long)(page * heads + head) << page_shift) + ((blk << 4) & ((1 << page_shift) - 1));
  }
};

// A lane's share of a block of 16 tokens: 1/4 of the K row of token c, 1/16
// of the V rows of the tokens 4 g + r.
template <int BITS, int D>
struct KvBlock {
  static constexpr int kRow = D * BITS / 8;              // bytes of a cached row
  static constexpr int kK = kRow / 16;                   // dwords
  static constexpr int kV = kRow >= 64 ? kRow / 64 : 1;  // dwords (2 bytes of one at 32)
  uint32_t k[kK], v[4][kV];

  __device__ __forceinline__ void load_k(const KvView& kv, long row0) {
    const int lane = threadIdx.x & 63, g = lane / 16, c = lane % 16;
    const uint8_t* ks = kv.kc + row0 * kRow;
    const uint32_t my_k = (uint32_t)(c * kRow + g * (kRow / 4));
    if constexpr (kK == 2) {
      const u2 w = load_at<u2>(ks, my_k);
      k[0] = w[0], k[1] = w[1];
    } else {
#pragma unroll
      for (int j = 0; j < kK; j += 4) {
        const u4 w = load_at<u4>(ks, my_k, 4 * j);
        k[j] = w[0], k[j + 1] = w[1], k[j + 2] = w[2], k[j + 3] = w[3];
      }
    }
  }
  __device__ __forceinline__ void load_v(const KvView& kv, long row0) {
    const int lane = threadIdx.x & 63, g = lane / 16, c = lane % 16;
    const uint8_t* vs = kv.vc + row0 * kRow;
    const uint32_t my_v = (uint32_t)(4 * g * kRow + c * (kRow / 16));
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if constexpr (kRow == 32) {
        v[r][0] = load_at<uint16_t>(vs, my_v, r * kRow);
      } else if constexpr (kV == 1) {
        v[r][0] = load_at<uint32_t>(vs, my_v, r * kRow);
      } else if constexpr (kV == 2) {
        const u2 w = load_at<u2>(vs, my_v, r * kRow);
        v[r][0] = w[0], v[r][1] = w[1];
      } else {
        const u4 w = load_at<u4>(vs, my_v, r * kRow);
        v[r][0] = w[0], v[r][1] = w[1], v[r][2] = w[2], v[r][3] = w[3];
      }
    }
  }

  __device__ __forceinline__ h8 k_operand(int step) const {
    if constexpr (BITS == 4) return row_codes4(k[step]);
    else return row_codes8(k[2 * step], k[2 * step + 1]);
  }
  // V of the tokens 4 g + 2 x and + 1, for head_dim (D / 16) c + 4 w + j: four
  // values of j at a time.
  __device__ __forceinline__ void v_pairs(int w, int x, h2 (&f)[4]) const {
    if constexpr (BITS == 4) {
      const uint32_t y = perm_b32(v[2 * x + 1][w / 2], v[2 * x][w / 2], w % 2 ? 0x07060302u : 0x05040100u);
      f[0] = nib_lo(y), f[1] = nib_hi(y), f[2] = nib_lo(y >> 8), f[3] = nib_hi(y >> 8);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        f[j] = byte_pair(perm_b32(v[2 * x + 1][w], v[2 * x][w], 0x0C000C00u | (uint32_t)((4 + j) << 16) | (uint32_t)j));
    }
  }
};

// bf16 scales of the tokens 4 g + r of a block.
__device__ __forceinline__ u2 load_scales(const uint16_t* s, long row0) {
  return load_at<u2>(s + row0, 8 * ((threadIdx.x & 63) / 16));
}
__device__ __forceinline__ f4 widen_scales(u2 w) {
  return f4{bf16_bits_to_f32((uint16_t)w[0]), __uint_as_float(w[0] & 0xFFFF0000u), bf16_bits_to_f32((uint16_t)w[1]),
            __uint_as_float(w[1] & 0xFFFF0000u)};
}

// A wave's query rows (16 * RT, row c of tile t in lane c of every group) and
// their running softmax.
template <int BITS, int D, int RT, int TYPE>
struct KvRows {
  static constexpr int kSteps = D / 32, kOut = D / 16;
  static constexpr bool kSplitP = TYPE == SHK_SRC_F16;

  h8 q[RT][kSteps];
  float qs[RT];  // 2^e of the row, times |softmax scale| and log2(e)
  f4 o[RT][kOut];
  float m[RT], l[RT];  // reference and sum (the lane's tokens only)
  uint32_t big[RT];    // bits of the largest |v scale| that the row has seen

  // q[c][g * (D / 4) + 8 s + kv_order(i)] for step s; null rows are zero.
  __device__ __forceinline__ void begin(const void* const (&row)[RT], float scale) {
    const int g = (threadIdx.x & 63) / 16;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      float v[kSteps][8];
      uint32_t most = 0;
      const uint4* src = static_cast<const uint4*>(row[t]) + g * (D / 32);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (row[t] != nullptr) w = src[s];
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint16_t hb = (uint16_t)(i % 2 ? u[i / 2] >> 16 : u[i / 2]);
          v[s][i] = TYPE == SHK_SRC_BF16 ? bf16_bits_to_f32(hb) : (float)__builtin_bit_cast(_Float16, hb);
          most = max(most, __float_as_uint(v[s][i]) & 0x7FFFFFFFu);
        }
      }
      most = groups_most(most);
      // the largest magnitude's exponent, within what both 2^e and 2^-e hold
      const int e = min(max((int)(most >> 23), 1), 253);
      const float inv = __builtin_copysignf(__uint_as_float((uint32_t)(254 - e) << 23), scale);
      // Never 0, which would make NaN of a masked -inf: a scale of 0, or one
      // that a row of zeros leaves no bits of, is as flat at the smallest f32.
      qs[t] = __builtin_fmaxf(__uint_as_float((uint32_t)e << 23) * (__builtin_fabsf(scale) * kLog2e), 0x1p-149f);
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) q[t][s][i] = (_Float16)(v[s][kv_order<BITS>(i)] * inv);
      m[t] = -__builtin_inff();
      l[t] = 0.0f;
      big[t] = 0;
#pragma unroll
      for (int j = 0; j < kOut; ++j) o[t][j] = f4{0, 0, 0, 0};
    }
  }

  // Scores (before the row's factor) of 16 * NB tokens and their scales to the
  // second product's operands; o shrinks where a row's reference grew.  It
  // grows only past twice its value, which the 13 leaves room for: the shrink
  // runs in few steps instead of nearly all.
  // limit[t]: the row's tokens end there, counted from the step's first;
  // `ends`: some row's do (uniform).  What a row does not see may hold
  // anything, NaN too: it stays out of the row's scores, largest scale and
  // products.
  template <int NB>
  __device__ __forceinline__ void soften(f4 (&s)[RT][NB], const f4 (&ks)[NB], f4 (&vs)[NB], bool ends,
                                         const int (&limit)[RT], h8 (&p)[RT][NB / 2], h8 (&pl)[RT][NB / 2]) {
    const int g = (threadIdx.x & 63) / 16;
    auto unseen = [&](int t, int i, int r) { return 16 * i + 4 * g + r >= limit[t]; };
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int i = 0; i < NB; ++i) s[t][i] *= ks[i];
    if (ends) {
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float v = unseen(t, i, r) ? 0.0f : vs[i][r];
            if (unseen(t, i, r)) s[t][i][r] = -__builtin_inff();
            if constexpr (RT == 1) vs[i][r] = v;
            most = larger(most, v);
          }
        big[t] = max(big[t], groups_most(__float_as_uint(most)));
      }
    } else {
      float most = 0.0f;
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) most = larger(most, vs[i][r]);
      const uint32_t bits = groups_most(__float_as_uint(most));
#pragma unroll
      for (int t = 0; t < RT; ++t) big[t] = max(big[t], bits);
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      // an infinite or NaN scale needs no room: its outputs are not finite
      // whatever the reference, and the row's sum keeps its bits
      const int e = big[t] < 0x7F800000u ? max((int)(big[t] >> 23), 47) : 47;
      const float up = (float)(e - 127 - 13);
      float top = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = __builtin_fmaxf(top, s[t][i][r]);
      top = groups_max(top) * qs[t] + up;
      top = top > m[t] + 1.0f ? top : m[t];
      const float base = top == -__builtin_inff() ? 0.0f : top;
      const float half = half_weight(m[t] - base);
      m[t] = top;
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float pv = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i][r], qs[t], -base));
          sum += pv;
          float w = pv * vs[i][r];
          // w as rounded to f32 for both terms: otherwise one use of hi is made
          // by v_fma_mixlo_f16, which rounds the product once, and where w lies
          // between two f16 values the terms are of different ones
          if constexpr (kSplitP) asm("" : "+v"(w));
          const _Float16 hi = (_Float16)w;
          p[t][i / 2][4 * (i % 2) + r] = hi;
          if constexpr (kSplitP) pl[t][i / 2][4 * (i % 2) + r] = (_Float16)(w - (float)hi);
        }
      if (RT > 1 && ends) {  // a scale that one tile sees and another does not
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (unseen(t, i, r)) {  // 0 times a scale that may be NaN
              p[t][i / 2][4 * (i % 2) + r] = (_Float16)0.0f;
              if constexpr (kSplitP) pl[t][i / 2][4 * (i % 2) + r] = (_Float16)0.0f;
            }
      }
      l[t] = l[t] * half * half + sum;
      if (__any(half != 1.0f)) {
#pragma unroll
        for (int j = 0; j < kOut; ++j) o[t][j] *= half * half;
      }
    }
  }

  // o^T += V^T P^T for 32 tokens and 16 values of head_dim.
  template <int NH>
  __device__ __forceinline__ void add(int j, const h8& v, const h8 (&p)[RT][NH], const h8 (&pl)[RT][NH], int h) {
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      o[t][j] = mfma_f16(v, p[t][h], o[t][j]);
      if constexpr (kSplitP) o[t][j] = mfma_f16(v, pl[t][h], o[t][j]);
    }
  }
};

}  // namespace shk
