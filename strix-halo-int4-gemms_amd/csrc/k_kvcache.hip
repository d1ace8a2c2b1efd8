// Keys and values into the quantized cache (kv_write) and out of it (kv_read).
//
// One row (token, head) is head_dim values x, stored as codes c and one scale:
//   s = bf16(fl32(max|x| / Q)),  c = clamp(rint(fl32(x / s)), -Q, Q),
// Q = 7 or 127.  Both kernels are one pass over memory: each value and each
// code is touched once, by the lane that owns 8 consecutive values of a row
// (16 bytes of a 2-byte type in, 4 or 8 bytes of codes out); head_dim / 8
// lanes share a row and exchange its maximum.  Keys and values go side by side,
// so a lane has two rows on their way (write) or four (read).
//
// Bound by memory.  Measured with 8 heads of 128, bf16: 8191 tokens to int8,
// 50.7 MB, 14.0 us (3.6 TB/s; about 4 us of it are the launch's start and end,
// which is all that a few tokens take); 65536 tokens from int4, 338 MB of which
// 268 are stores, 79 us (4.3 TB/s, where a copy of 2 GiB runs at 4.9).  What is
// read out goes past the caches, values (114 -> 88 us) and codes (88 -> 77);
// what is written does not (f32 values read past them: 295 -> 333 us).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>

#include "shk_common.h"
#include "shk_kvcache.h"
#include "shk_kvrows.h"

namespace shk {
namespace {

struct Rows {
  const uint8_t* x[2];   // keys, values
  uint8_t* codes[2];
  uint16_t* scales[2];
  long token_stride[2], head_stride[2];
  const void* slots;
  long slots_total;      // pages * page_size
  unsigned rows;         // tokens * kv_heads
  unsigned heads;
  int slot8, page_shift;
};

// Rows of a lane, each of keys and of values.
constexpr int kWriteRows = 1, kReadRows = 2;

// The slot of a token, -1 outside the cache.
__device__ __forceinline__ long slot_of(const Rows& p, long t) {
  const long slot = p.slot8 ? static_cast<const int64_t*>(p.slots)[t] : static_cast<const int32_t*>(p.slots)[t];
  return slot >= 0 && slot < p.slots_total ? slot : -1;
}

template <int TYPE, int BITS, int D, bool VEC>
__global__ __launch_bounds__(256) void kv_write_kernel(const Rows p) {
  constexpr int LANES = D / 8;  // of a row
  const int part = threadIdx.x % LANES;
  const unsigned first = blockIdx.x * (256 / LANES * kWriteRows) + threadIdx.x / LANES;
  long slot[kWriteRows];
  unsigned head[kWriteRows];
  float v[kWriteRows][2][8] = {};
#pragma unroll
  for (int i = 0; i < kWriteRows; ++i) {
    const unsigned row = first + i * (256 / LANES), t = row / p.heads;
    head[i] = row - t * p.heads;
    slot[i] = row < p.rows ? slot_of(p, t) : -1;
#pragma unroll
    for (int which = 0; which < 2; ++which)
      if (slot[i] >= 0)
        load8<TYPE, VEC>(p.x[which] + ((long)t * p.token_stride[which] + head[i] * p.head_stride[which] + part * 8) *
                                          kSize<TYPE>, v[i][which]);
  }
#pragma unroll
  for (int i = 0; i < kWriteRows; ++i)
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      // magnitudes as integers: a NaN is larger than an infinity, and both stay
      uint32_t most = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(v[i][which][e]) & 0x7FFFFFFFu);
#pragma unroll
      for (int d = 1; d < LANES; d *= 2) most = max(most, (uint32_t)__shfl_xor((int)most, d, 64));
      if (slot[i] < 0) continue;
      const uint32_t sb = f32_to_bf16_rne(__uint_as_float(most) / (BITS == 4 ? 7.0f : 127.0f));
      int c[8];
      codes8<BITS>(v[i][which], __uint_as_float(sb << 16), c);
      const long out = cache_row(slot[i], head[i], p.heads, p.page_shift);
      uint8_t* dst = p.codes[which] + out * (D * BITS / 8) + part * BITS;
      store_codes<BITS>(dst, c);
      if (part == 0) p.scales[which][out] = (uint16_t)sb;
    }
}

// Streamed past the caches.
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void stream16(void* p, v4u v) { __builtin_nontemporal_store(v, static_cast<v4u*>(p)); }

// Eight values at element address p.  FINITE: none is a NaN.
template <int TYPE, bool VEC, bool FINITE>
__device__ __forceinline__ void store8(uint8_t* p, const float (&v)[8]) {
  uint32_t o[TYPE == SHK_SRC_F32 ? 8 : 4];
  if constexpr (TYPE == SHK_SRC_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (TYPE == SHK_SRC_F16)
        o[i] = __builtin_bit_cast(uint16_t, (_Float16)v[2 * i]) |
               ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * i + 1]) << 16);
      else if constexpr (FINITE) o[i] = pack_bf16x2_nonan(v[2 * i], v[2 * i + 1]);
      else o[i] = f32_to_bf16_rne(v[2 * i]) | (f32_to_bf16_rne(v[2 * i + 1]) << 16);
    }
  }
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < (TYPE == SHK_SRC_F32 ? 2 : 1); ++i)
      stream16(p + 16 * i, v4u{o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]});
  } else {
    __builtin_memcpy(__builtin_assume_aligned(p, 2), o, sizeof(o));
  }
}

template <int TYPE, int BITS, int D, bool VEC>
__global__ __launch_bounds__(256) void kv_read_kernel(const Rows p) {
  constexpr int LANES = D / 8;
  const int part = threadIdx.x % LANES;
  const unsigned first = blockIdx.x * (256 / LANES * kReadRows) + threadIdx.x / LANES;
  unsigned t[kReadRows], head[kReadRows];
  long slot[kReadRows];
  uint2 w[kReadRows][2] = {};
  float scale[kReadRows][2];
#pragma unroll
  for (int i = 0; i < kReadRows; ++i) {
    const unsigned row = first + i * (256 / LANES);
    t[i] = row / p.heads;
    head[i] = row - t[i] * p.heads;
    slot[i] = row < p.rows ? slot_of(p, t[i]) : -1;
    const long at = slot[i] >= 0 ? cache_row(slot[i], head[i], p.heads, p.page_shift) : 0;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      scale[i][which] = __builtin_nanf("");
      if (slot[i] < 0) continue;
      const uint8_t* src = p.codes[which] + at * (D * BITS / 8) + part * BITS;
      if constexpr (BITS == 4) {
        w[i][which].x = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(src));
      } else {
        const v2u u = __builtin_nontemporal_load(reinterpret_cast<const v2u*>(src));
        w[i][which] = make_uint2(u[0], u[1]);
      }
      scale[i][which] = bf16_bits_to_f32(p.scales[which][at]);
    }
  }
#pragma unroll
  for (int i = 0; i < kReadRows; ++i) {
    if (first + i * (256 / LANES) >= p.rows) continue;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint2 u = w[i][which];
        const int code = BITS == 4 ? (int32_t)(u.x << (28 - 4 * e)) >> 28
                                   : (int8_t)((e < 4 ? u.x : u.y) >> (8 * (e % 4)));
        v[e] = (float)code * scale[i][which];
      }
      uint8_t* dst = const_cast<uint8_t*>(p.x[which]) +
                     ((long)t[i] * p.token_stride[which] + head[i] * p.head_stride[which] + part * 8) * kSize<TYPE>;
      // an infinite scale makes NaN of a zero code
      if (__builtin_fabsf(scale[i][which]) < __builtin_inff()) store8<TYPE, VEC, true>(dst, v);
      else store8<TYPE, VEC, false>(dst, v);
    }
  }
}

long rows_of_workgroup(bool write, long d) { return 256 / (d / 8) * (write ? kWriteRows : kReadRows); }

template <int TYPE, int BITS, int D, bool VEC>
hipError_t launch(bool write, const Rows& p, hipStream_t s) {
  const long kPer = rows_of_workgroup(write, D);
  const dim3 grid((unsigned)((p.rows + kPer - 1) / kPer));
  if (write) hipLaunchKernelGGL((kv_write_kernel<TYPE, BITS, D, VEC>), grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((kv_read_kernel<TYPE, BITS, D, VEC>), grid, dim3(256), 0, s, p);
  return hipGetLastError();
}

template <int TYPE, int BITS, int D>
hipError_t launch_d(bool write, bool vec, const Rows& p, hipStream_t s) {
  return vec ? launch<TYPE, BITS, D, true>(write, p, s) : launch<TYPE, BITS, D, false>(write, p, s);
}

template <int TYPE, int BITS>
hipError_t launch_b(bool write, bool vec, long d, const Rows& p, hipStream_t s) {
  if (d == 64) return launch_d<TYPE, BITS, 64>(write, vec, p, s);
  if (d == 128) return launch_d<TYPE, BITS, 128>(write, vec, p, s);
  return launch_d<TYPE, BITS, 256>(write, vec, p, s);
}

template <int TYPE>
hipError_t launch_t(bool write, bool vec, const shk_kv_cache& c, const Rows& p, hipStream_t s) {
  return c.bits == 4 ? launch_b<TYPE, 4>(write, vec, c.head_dim, p, s)
                     : launch_b<TYPE, 8>(write, vec, c.head_dim, p, s);
}

hipError_t rows_launch(bool write, const shk_kv_cache& c, const shk_kv_rows& r, hipStream_t s) {
  Rows p{};
  p.x[0] = static_cast<const uint8_t*>(r.keys), p.x[1] = static_cast<const uint8_t*>(r.values);
  p.codes[0] = static_cast<uint8_t*>(c.key_codes), p.codes[1] = static_cast<uint8_t*>(c.value_codes);
  p.scales[0] = static_cast<uint16_t*>(c.key_scales), p.scales[1] = static_cast<uint16_t*>(c.value_scales);
  p.token_stride[0] = r.key_token_stride, p.token_stride[1] = r.value_token_stride;
  p.head_stride[0] = r.key_head_stride, p.head_stride[1] = r.value_head_stride;
  p.slots = r.slots;
  p.slots_total = c.pages * c.page_size;
  p.rows = (unsigned)(r.tokens * c.kv_heads);
  p.slot8 = r.slot_bytes == 8;
  p.heads = (unsigned)c.kv_heads;
  p.page_shift = __builtin_ctzl((unsigned long)c.page_size);
  if (p.rows == 0) return hipSuccess;
  // 16-byte accesses where every row starts on 16 bytes
  const long size = r.type == SHK_SRC_F32 ? 4 : 2;
  const bool vec = ((reinterpret_cast<uintptr_t>(r.keys) | reinterpret_cast<uintptr_t>(r.values) |
                     (uintptr_t)(size * (r.key_token_stride | r.key_head_stride | r.value_token_stride |
                                         r.value_head_stride))) & 15) == 0;
  if (r.type == SHK_SRC_F32) return launch_t<SHK_SRC_F32>(write, vec, c, p, s);
  if (r.type == SHK_SRC_F16) return launch_t<SHK_SRC_F16>(write, vec, c, p, s);
  return launch_t<SHK_SRC_BF16>(write, vec, c, p, s);
}

}  // namespace

int64_t kv_rows_most(bool write, const shk_kv_cache& c) {
  // rows are counted in 32 bits
  return std::min(kMostWorkgroups * rows_of_workgroup(write, c.head_dim), (int64_t)INT_MAX) / c.kv_heads;
}

hipError_t launch_kv_write(const shk_kv_cache& c, const shk_kv_rows& r, hipStream_t s) {
  return rows_launch(true, c, r, s);
}
hipError_t launch_kv_read(const shk_kv_cache& c, const shk_kv_rows& r, hipStream_t s) {
  return rows_launch(false, c, r, s);
}

}  // namespace shk
