// Attention of a few query rows over a piece of the quantized cache: the
// streaming tile that the decode kernel runs (k_kvattn.hip).
//
// One workgroup of four waves serves one key head and up to 16 * RT query
// rows (the queries of a sequence that read this key head, or, for a shared
// prefix, those of all sequences).  A wave takes 64 tokens at a time, 16 by
// 16 in four blocks i, and keeps everything in registers:
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
// Probabilities enter as p * (v_scale / 2^ref) * 2^13, ref the exponent of
// the largest v_scale that the wave has met: at most 2^15, so f16 does not
// overflow, and normal down to 2^-28 of the largest; for f16 outputs they are split into two f16 terms, because
// one rounding to 11 bits would be as large as the output's own.
// Sums, maxima and outputs are f32.
#pragma once

#include "shk_common.h"
#include "shk_kvcache.h"

namespace shk {

constexpr int kKvTile = 64;  // tokens of a wave's step
constexpr float kLog2e = 1.4426950408889634f;

// Two codes that sit in the low bytes / nibbles of a dword's halves, as f16.
// 0x6400 | n is 1024 + n, exactly; int4 codes come offset by 8 (their sign
// bits flipped), int8 codes by 128.
__device__ __forceinline__ h2 nib_lo(uint32_t w) {
  return __builtin_bit_cast(h2, (w & 0x000F000Fu) | 0x64006400u) - (h2)(_Float16)1032.0f;
}
__device__ __forceinline__ h2 nib_hi(uint32_t w) {  // bits 4..7: 1024 + 16 n, over 16
  return __builtin_elementwise_fma(__builtin_bit_cast(h2, (w & 0x00F000F0u) | 0x64006400u), (h2)(_Float16)0.0625f,
                                   (h2)(_Float16)-72.0f);
}
__device__ __forceinline__ h2 byte_pair(uint32_t w) {  // w = u0 | u1 << 16, u = code + 128
  return __builtin_bit_cast(h2, w | 0x64006400u) - (h2)(_Float16)1152.0f;
}

__device__ __forceinline__ h8 join(h2 a, h2 b, h2 c, h2 d) {
  return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// 8 codes of one row as a product's operand.  int4 codes 0..7 of a dword come
// in the order 0 4 1 5 2 6 3 7 (kv_order), which q's operand repeats.
__device__ __forceinline__ h8 codes4(uint32_t w) {
  w ^= 0x88888888u;
  const uint32_t u = w >> 8;
  return join(nib_lo(w), nib_hi(w), nib_lo(u), nib_hi(u));
}
__device__ __forceinline__ h8 codes8(uint32_t lo, uint32_t hi) {
  lo ^= 0x80808080u, hi ^= 0x80808080u;
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

// Largest / sum over the four lane groups (lanes c, c + 16, c + 32, c + 48).
__device__ __forceinline__ float groups_max(float v) {
  v = __builtin_fmaxf(v, __shfl_xor(v, 16, 64));
  return __builtin_fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float groups_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

struct KvView {  // one key head of the cache
  const uint8_t *kc, *vc;
  const uint16_t *ks, *vs;
  int pages, page_shift, heads, head;
};

struct KvRow {     // what a lane's query row needs
  const void* q;   // null: no such row
  int limit;       // tokens it sees of this piece
};

template <int BITS, int D, int RT, int TYPE>
struct KvTile {
  static constexpr int kRow = D * BITS / 8;       // bytes of a cached row
  static constexpr int kK = kRow / 16;            // dwords of a lane's share of a K row
  static constexpr int kV = kRow >= 64 ? kRow / 64 : 1;  // dwords of a lane's share of a V row (2 bytes of one at 32)
  static constexpr int kSteps = D / 32, kOut = D / 16;
  static constexpr bool kSplitP = TYPE == SHK_SRC_F16;

  h8 q[RT][kSteps];
  float qs[RT];  // 2^e of the row, times softmax scale and log2(e)
  f4 o[RT][kOut];
  float m[RT], l[RT];
  int ref;       // biased exponent that v scales are taken relative to
  bool bad;      // a page outside the cache

  // q[c][g * (D / 4) + 8 s + kv_order(i)] for step s.
  __device__ __forceinline__ void begin(const KvRow (&row)[RT], float scale) {
    const int g = (threadIdx.x & 63) / 16;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      float v[kSteps][8];
      uint32_t most = 0;
      const uint4* src = static_cast<const uint4*>(row[t].q) + g * (D / 32);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (row[t].q != nullptr) w = src[s];
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint16_t hb = (uint16_t)(i % 2 ? u[i / 2] >> 16 : u[i / 2]);
          v[s][i] = TYPE == SHK_SRC_BF16 ? bf16_bits_to_f32(hb) : (float)__builtin_bit_cast(_Float16, hb);
          most = max(most, __float_as_uint(v[s][i]) & 0x7FFFFFFFu);
        }
      }
      most = max(most, (uint32_t)__shfl_xor((int)most, 16, 64));
      most = max(most, (uint32_t)__shfl_xor((int)most, 32, 64));
      // the largest magnitude's exponent, within what both 2^e and 2^-e hold
      const int e = min(max((int)(most >> 23), 1), 253);
      const float inv = __uint_as_float((uint32_t)(254 - e) << 23);
      qs[t] = __uint_as_float((uint32_t)e << 23) * (scale * kLog2e);
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) q[t][s][i] = (_Float16)(v[s][kv_order<BITS>(i)] * inv);
      m[t] = -__builtin_inff();
      l[t] = 0.0f;
#pragma unroll
      for (int j = 0; j < kOut; ++j) o[t][j] = f4{0, 0, 0, 0};
    }
    ref = 1;
    bad = false;
  }

  // Tokens [t0, t0 + 64) of a sequence of n (t0 < n, a multiple of 64).
  __device__ __forceinline__ void step(const KvView& kv, const int32_t* table, int t0, int n, const int (&limit)[RT],
                                       int least_limit) {
    const int lane = threadIdx.x & 63, g = lane / 16, c = lane % 16;
    const int last = (n - 1) >> 4;  // the last block that holds a token; later ones repeat it, masked
    uint32_t kw[4][kK], vw[16][kV];
    uint2 ksw[4], vsw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int blk = min((t0 >> 4) + i, last);
      int page = table[blk >> (kv.page_shift - 4)];
      if ((unsigned)page >= (unsigned)kv.pages) page = 0, bad = true;
      const int in_page = (blk << 4) & ((1 << kv.page_shift) - 1);
      const long row0 = (((long)page * kv.heads + kv.head) << kv.page_shift) + in_page;
      const uint32_t* ksrc = reinterpret_cast<const uint32_t*>(kv.kc + (row0 + c) * kRow) + g * kK;
      if constexpr (kK == 2) {
        const uint2 w = *reinterpret_cast<const uint2*>(ksrc);
        kw[i][0] = w.x, kw[i][1] = w.y;
      } else {
#pragma unroll
        for (int j = 0; j < kK; j += 4) {
          const uint4 w = *reinterpret_cast<const uint4*>(ksrc + j);
          kw[i][j] = w.x, kw[i][j + 1] = w.y, kw[i][j + 2] = w.z, kw[i][j + 3] = w.w;
        }
      }
      ksw[i] = *reinterpret_cast<const uint2*>(kv.ks + row0 + 4 * g);
      vsw[i] = *reinterpret_cast<const uint2*>(kv.vs + row0 + 4 * g);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint8_t* vsrc = kv.vc + (row0 + 4 * g + r) * kRow + c * (kRow / 16);
        uint32_t* dst = vw[4 * i + r];
        if constexpr (kRow == 32) {
          dst[0] = *reinterpret_cast<const uint16_t*>(vsrc);
        } else if constexpr (kV == 1) {
          dst[0] = *reinterpret_cast<const uint32_t*>(vsrc);
        } else if constexpr (kV == 2) {
          const uint2 w = *reinterpret_cast<const uint2*>(vsrc);
          dst[0] = w.x, dst[1] = w.y;
        } else {
          const uint4 w = *reinterpret_cast<const uint4*>(vsrc);
          dst[0] = w.x, dst[1] = w.y, dst[2] = w.z, dst[3] = w.w;
        }
      }
    }
    float s[RT][4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f4 acc[RT];
#pragma unroll
      for (int t = 0; t < RT; ++t) acc[t] = f4{0, 0, 0, 0};
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
        h8 k;
        if constexpr (BITS == 4) k = codes4(kw[i][st]);
        else k = shk::codes8(kw[i][2 * st], kw[i][2 * st + 1]);
#pragma unroll
        for (int t = 0; t < RT; ++t) acc[t] = mfma_f16(k, q[t][st], acc[t]);
      }
      const float ks[4] = {bf16_bits_to_f32((uint16_t)ksw[i].x), __uint_as_float(ksw[i].x & 0xFFFF0000u),
                           bf16_bits_to_f32((uint16_t)ksw[i].y), __uint_as_float(ksw[i].y & 0xFFFF0000u)};
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[t][i][r] = acc[t][r] * (ks[r] * qs[t]);
    }
    float vs[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      vs[i][0] = bf16_bits_to_f32((uint16_t)vsw[i].x), vs[i][1] = __uint_as_float(vsw[i].x & 0xFFFF0000u);
      vs[i][2] = bf16_bits_to_f32((uint16_t)vsw[i].y), vs[i][3] = __uint_as_float(vsw[i].y & 0xFFFF0000u);
    }
    if (t0 + kKvTile > least_limit) {  // some row ends in this step
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int at = t0 + 16 * i + 4 * g + r;
#pragma unroll
          for (int t = 0; t < RT; ++t)
            if (at >= limit[t]) s[t][i][r] = -__builtin_inff();
          if (at >= n) vs[i][r] = 0.0f;  // never written: may hold anything
        }
    }
    // exponent of the largest v scale so far
    uint32_t big = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) big = max(big, __float_as_uint(vs[i][r]));
    big = max(big, (uint32_t)__shfl_xor((int)big, 16, 64));
    big = max(big, (uint32_t)__shfl_xor((int)big, 32, 64));
    const int e = max(ref, min((int)((big >> 23) & 0xFF), 253));
    const float inv = __uint_as_float((uint32_t)(254 - e) << 23) * 8192.0f;
    const float shrink = e == ref ? 1.0f : (e - ref < 127 ? __uint_as_float((uint32_t)(127 - (e - ref)) << 23) : 0.0f);
    ref = e;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) vs[i][r] *= inv;
    h8 p[RT][2], pl[RT][2];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      float top = m[t];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = __builtin_fmaxf(top, s[t][i][r]);
      top = groups_max(top);
      const float base = top == -__builtin_inff() ? 0.0f : top;
      const float alpha = __builtin_amdgcn_exp2f(m[t] - base);
      m[t] = top;
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float pv = __builtin_amdgcn_exp2f(s[t][i][r] - base);
          sum += pv;
          const float w = pv * vs[i][r];
          const _Float16 hi = (_Float16)w;
          p[t][i / 2][4 * (i % 2) + r] = hi;
          if constexpr (kSplitP) pl[t][i / 2][4 * (i % 2) + r] = (_Float16)(w - (float)hi);
        }
      l[t] = l[t] * alpha + sum;
      const float a = alpha * shrink;
      if (__any(a != 1.0f)) {
#pragma unroll
        for (int j = 0; j < kOut; ++j) o[t][j] *= a;
      }
    }
    // O^T += V^T P^T, 32 tokens (blocks 2 h and 2 h + 1) at a time
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if constexpr (BITS == 4) {
#pragma unroll
        for (int w = 0; w < (kOut + 3) / 4; ++w) {  // four head_dim values a piece
          h2 f[4][4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const uint32_t a = vw[8 * h + 2 * x][w / 2], b = vw[8 * h + 2 * x + 1][w / 2];
            const uint32_t y = perm_b32(b, a, w % 2 ? 0x07060302u : 0x05040100u) ^ 0x88888888u;
            f[0][x] = nib_lo(y), f[1][x] = nib_hi(y), f[2][x] = nib_lo(y >> 8), f[3][x] = nib_hi(y >> 8);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) pv_step(4 * w + j, join(f[j][0], f[j][1], f[j][2], f[j][3]), p, pl, h);
        }
      } else {
#pragma unroll
        for (int j = 0; j < kOut; ++j) {
          h2 f[4];
          const uint32_t sel = 0x0C000C00u | (uint32_t)((4 + j % 4) << 16) | (uint32_t)(j % 4);
#pragma unroll
          for (int x = 0; x < 4; ++x)
            f[x] = byte_pair(perm_b32(vw[8 * h + 2 * x + 1][j / 4], vw[8 * h + 2 * x][j / 4], sel) ^ 0x00800080u);
          pv_step(j, join(f[0], f[1], f[2], f[3]), p, pl, h);
        }
      }
    }
  }

  __device__ __forceinline__ void pv_step(int j, const h8& v, const h8 (&p)[RT][2], const h8 (&pl)[RT][2], int h) {
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      o[t][j] = mfma_f16(v, p[t][h], o[t][j]);
      if constexpr (kSplitP) o[t][j] = mfma_f16(v, pl[t][h], o[t][j]);
    }
  }
};

}  // namespace shk
