// Attention of each sequence's newest tokens over the quantized cache
// (shk_kvattn.h has the mathematics of a tile).
//
// A workgroup is one piece of one sequence (or of the shared prefix) for one
// key head and up to 16 * RT of its query rows; its four waves take every
// fourth 64 tokens and are joined through LDS.  Pieces of a sequence are
// joined by kv_join_kernel from their f32 outputs, maxima and sums.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "shk_kvattn.h"

namespace shk {
namespace {

struct AttnArgs {
  const uint16_t* q;
  long q_batch, q_query, q_head;  // strides in elements
  const uint8_t *kc, *vc;
  const uint16_t *ks, *vs;
  const int32_t *table, *lengths, *prefix_pages;
  long table_stride;
  uint16_t* out;
  float* lse;
  float* part_o;   // [pieces][rows][D]
  float2* part_ml; // [pieces][rows]: maximum (in powers of two) and sum
  float scale;
  int type;
  int batch, queries, heads, kv_heads, ratio;
  int pages, page_shift, table_tokens, prefix;
  int own_splits, prefix_splits;  // pieces of a sequence and of the prefix
  int own_tiles, prefix_tiles;    // 16 * RT row tiles of a key head
};

template <int D>
__device__ __forceinline__ void store_row(const AttnArgs& a, long row, int d, f4 v) {
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    b[i] = a.type == SHK_SRC_BF16 ? f32_to_bf16_rne(v[i]) : __builtin_bit_cast(uint16_t, (_Float16)v[i]);
  *reinterpret_cast<uint2*>(a.out + row * D + d) = make_uint2(b[0] | (b[1] << 16), b[2] | (b[3] << 16));
}

__device__ __forceinline__ float natural_lse(float m, float l) {
  return m == -__builtin_inff() && !(l != l) ? -__builtin_inff() : (m + __log2f(l)) * 0.6931471805599453f;
}

template <int BITS, int D, int RT, int TYPE>
__global__ __launch_bounds__(256, D == 256 || RT == 2 ? 2 : 3) void kv_attention_kernel(const AttnArgs a) {
  using Tile = KvTile<BITS, D, RT, TYPE>;
  constexpr int kPitch = D + 4;  // floats of an LDS row: the 16 rows start on different banks
  __shared__ float red_o[4][16 * kPitch];
  __shared__ float red_m[4][16], red_l[4][16];
  const int lane = threadIdx.x & 63, g = lane / 16, c = lane % 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);

  // which piece: those of the sequences first, then those of the prefix
  int unit = blockIdx.x;
  const int own_units = a.batch * a.kv_heads * a.own_tiles * a.own_splits;
  const bool shared = unit >= own_units;
  if (shared) unit -= own_units;
  const int splits = shared ? a.prefix_splits : a.own_splits, tiles = shared ? a.prefix_tiles : a.own_tiles;
  const int split = unit % splits;
  unit /= splits;
  const int tile = unit % tiles;
  unit /= tiles;
  const int head = unit % a.kv_heads;
  const int b0 = unit / a.kv_heads;  // 0 for the prefix
  const int n = shared ? a.prefix : min(max(a.lengths[b0], 0), a.table_tokens);
  const int piece = shared ? a.own_splits + split : split;
  const int rows_here = a.queries * a.ratio * (shared ? a.batch : 1);

  KvRow row[RT];
  long out_row[RT];
  int limit[RT], least = n;
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = (tile * RT + t) * 16 + c;
    row[t].q = nullptr;
    out_row[t] = -1;
    limit[t] = n;
    if (r < rows_here) {
      const int per = a.queries * a.ratio;
      const int b = shared ? r / per : b0, in = shared ? r % per : r;
      const int query = in / a.ratio, h = head * a.ratio + in % a.ratio;
      row[t].q = a.q + b * a.q_batch + query * a.q_query + h * a.q_head;
      out_row[t] = ((long)b * a.queries + query) * a.heads + h;
      if (!shared) limit[t] = max(n - a.queries + query + 1, 0);
    }
    least = min(least, limit[t]);
  }
#pragma unroll
  for (int d = 1; d < 16; d *= 2) least = min(least, __shfl_xor(least, d, 64));
  least = __builtin_amdgcn_readfirstlane(least);

  const KvView kv{a.kc, a.vc, a.ks, a.vs, a.pages, a.page_shift, a.kv_heads, head};
  const int32_t* table = shared ? a.prefix_pages : a.table + b0 * a.table_stride;
  const int steps = (n + kKvTile - 1) / kKvTile;
  const int each = (steps + splits - 1) / splits;
  const int first = split * each, end = min(first + each, steps);

  Tile tl;
  tl.begin(row, a.scale);
  for (int i = first + wave; i < end; i += 4) tl.step(kv, table, i * kKvTile, n, limit, least);

  // the waves' outputs, relative to the largest of their maxima
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const float l = groups_sum(tl.l[t]);
    if (t > 0) __syncthreads();
    if (g == 0) red_m[wave][c] = tl.m[t], red_l[wave][c] = tl.bad ? __builtin_nanf("") : l;
    __syncthreads();
    float top = red_m[0][c];
#pragma unroll
    for (int w = 1; w < 4; ++w) top = __builtin_fmaxf(top, red_m[w][c]);
    const float base = top == -__builtin_inff() ? 0.0f : top;
    const float back = __uint_as_float((uint32_t)tl.ref << 23) * 0x1p-13f * __builtin_amdgcn_exp2f(tl.m[t] - base);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < Tile::kOut; j += 4)
        *reinterpret_cast<f4*>(&red_o[wave][c * kPitch + (4 * g + r) * Tile::kOut + j]) =
            f4{tl.o[t][j][r], tl.o[t][j + 1][r], tl.o[t][j + 2][r], tl.o[t][j + 3][r]} * back;
    __syncthreads();
    // 16 threads a row, D / 16 values each
    const int rr = threadIdx.x / 16, part = threadIdx.x % 16;
    float rtop = red_m[0][rr];
#pragma unroll
    for (int w = 1; w < 4; ++w) rtop = __builtin_fmaxf(rtop, red_m[w][rr]);
    const float rbase = rtop == -__builtin_inff() ? 0.0f : rtop;
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) sum += red_l[w][rr] * __builtin_amdgcn_exp2f(red_m[w][rr] - rbase);
    // the row's place in the output, from the lane that holds the row
    const long at = __shfl(out_row[t], rr, 64);
    if (at >= 0) {
      const bool whole = a.own_splits + a.prefix_splits == 1;
      const float f = !whole ? 1.0f : (sum == 0.0f ? 0.0f : 1.0f / sum);
#pragma unroll
      for (int k = 0; k < D / 64; ++k) {
        const int d = (k * 16 + part) * 4;
        f4 v = f4{0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < 4; ++w) v += *reinterpret_cast<const f4*>(&red_o[w][rr * kPitch + d]);
        v *= f;
        if (whole) store_row<D>(a, at, d, v);
        else *reinterpret_cast<f4*>(a.part_o + ((long)piece * a.batch * a.queries * a.heads + at) * D + d) = v;
      }
      if (part == 0) {
        if (!whole) a.part_ml[(long)piece * a.batch * a.queries * a.heads + at] = make_float2(rtop, sum);
        else if (a.lse != nullptr) a.lse[at] = natural_lse(rtop, sum);
      }
    }
  }
}

// Joins the pieces of a row: 32 lanes a row, D / 32 values each.
template <int D>
__global__ __launch_bounds__(256) void kv_join_kernel(const AttnArgs a) {
  const long rows = (long)a.batch * a.queries * a.heads;
  const long row = ((long)blockIdx.x * 256 + threadIdx.x) / 32;
  if (row >= rows) return;
  const int part = threadIdx.x % 32, pieces = a.own_splits + a.prefix_splits;
  float top = -__builtin_inff();
  for (int s = 0; s < pieces; ++s) top = __builtin_fmaxf(top, a.part_ml[s * rows + row].x);
  const float base = top == -__builtin_inff() ? 0.0f : top;
  float sum = 0.0f;
  constexpr int N = D / 32 < 4 ? 1 : D / 128;  // 16-byte pieces of a lane; D = 64: half the lanes
  f4 v[N] = {};
  const bool on = part * 4 < D;
  for (int s = 0; s < pieces; ++s) {
    const float2 ml = a.part_ml[s * rows + row];
    if (ml.x == -__builtin_inff() && ml.y == 0.0f) continue;  // nothing seen
    const float w = __builtin_amdgcn_exp2f(ml.x - base);
    sum += ml.y * w;
    if (on) {
#pragma unroll
      for (int k = 0; k < N; ++k)
        v[k] += *reinterpret_cast<const f4*>(a.part_o + (s * rows + row) * D + (k * 32 + part) * 4) * w;
    }
  }
  const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
  if (on) {
#pragma unroll
    for (int k = 0; k < N; ++k) store_row<D>(a, row, (k * 32 + part) * 4, v[k] * f);
  }
  if (part == 0 && a.lse != nullptr) a.lse[row] = natural_lse(top, sum);
}

long cdiv(long a, long b) { return (a + b - 1) / b; }

// Pieces of the sequences and of the prefix, and the row tiles' height.
struct Plan {
  int rt, own_tiles, prefix_tiles, own_splits, prefix_splits;
};

Plan plan_of(const shk_kv_cache& c, const shk_kv_attention& a) {
  const long rows = a.queries * (a.heads / c.kv_heads);
  Plan p;
  // two row tiles of 256 columns would not fit the registers
  p.rt = c.head_dim == 256 ? 1 : rows > 16 || (a.prefix_length > 0 && rows * a.batch > 16) ? 2 : 1;
  p.own_tiles = (int)cdiv(rows, 16 * p.rt);
  p.prefix_tiles = a.prefix_length > 0 ? (int)cdiv(rows * a.batch, 16 * p.rt) : 0;
  const long want = 768;  // workgroups of a launch: three on each of 256 CUs
  const long own = a.batch * c.kv_heads * p.own_tiles;
  const long tokens = a.table_pages * c.page_size;
  p.own_splits = (int)std::max(1L, std::min({cdiv(want, own), cdiv(tokens, 4 * kKvTile), 64L}));
  p.prefix_splits = 0;
  if (a.prefix_length > 0)
    p.prefix_splits = (int)std::max(1L, std::min({cdiv(want, (long)c.kv_heads * p.prefix_tiles),
                                                  cdiv(a.prefix_length, 4 * kKvTile), 64L}));
  return p;
}

long part_rows(const shk_kv_attention& a, const Plan& p) {
  return p.own_splits + p.prefix_splits > 1 ? (p.own_splits + p.prefix_splits) * a.batch * a.queries * a.heads : 0;
}

template <int BITS, int D, int RT, int TYPE>
hipError_t launch(const AttnArgs& a, hipStream_t s) {
  const long per_head = (long)a.batch * a.own_tiles * a.own_splits + (long)a.prefix_tiles * a.prefix_splits;
  const long units = a.kv_heads * per_head;
  if (units > 0x7FFFFF) return hipErrorInvalidValue;  // a launch holds fewer than 2^32 work-items
  hipLaunchKernelGGL((kv_attention_kernel<BITS, D, RT, TYPE>), dim3((unsigned)units), dim3(256), 0, s, a);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess || a.own_splits + a.prefix_splits == 1) return err;
  const long rows = (long)a.batch * a.queries * a.heads;
  hipLaunchKernelGGL((kv_join_kernel<D>), dim3((unsigned)cdiv(rows, 8)), dim3(256), 0, s, a);
  return hipGetLastError();
}

template <int BITS, int D, int TYPE>
hipError_t launch_rt(int rt, const AttnArgs& a, hipStream_t s) {
  if constexpr (D < 256)
    if (rt == 2) return launch<BITS, D, 2, TYPE>(a, s);
  return launch<BITS, D, 1, TYPE>(a, s);
}

template <int BITS, int TYPE>
hipError_t launch_d(long d, int rt, const AttnArgs& a, hipStream_t s) {
  if (d == 64) return launch_rt<BITS, 64, TYPE>(rt, a, s);
  if (d == 128) return launch_rt<BITS, 128, TYPE>(rt, a, s);
  return launch_rt<BITS, 256, TYPE>(rt, a, s);
}

}  // namespace

int64_t kv_attention_workspace(const shk_kv_cache& c, const shk_kv_attention& a) {
  return part_rows(a, plan_of(c, a)) * (c.head_dim * 4 + 8);
}

hipError_t launch_kv_attention(const shk_kv_cache& c, const shk_kv_attention& x, hipStream_t s) {
  const Plan p = plan_of(c, x);
  AttnArgs a{};
  a.q = static_cast<const uint16_t*>(x.q);
  a.q_batch = x.q_batch_stride, a.q_query = x.q_query_stride, a.q_head = x.q_head_stride;
  a.kc = static_cast<const uint8_t*>(c.key_codes), a.vc = static_cast<const uint8_t*>(c.value_codes);
  a.ks = static_cast<const uint16_t*>(c.key_scales), a.vs = static_cast<const uint16_t*>(c.value_scales);
  a.table = x.page_table, a.lengths = x.lengths, a.prefix_pages = x.prefix_pages;
  a.table_stride = x.table_stride;
  a.out = static_cast<uint16_t*>(x.out);
  a.lse = x.lse;
  a.part_o = static_cast<float*>(x.workspace);
  a.part_ml = reinterpret_cast<float2*>(a.part_o + part_rows(x, p) * c.head_dim);
  a.scale = (float)x.scale;
  a.type = (int)x.type;
  a.batch = (int)x.batch, a.queries = (int)x.queries, a.heads = (int)x.heads, a.kv_heads = (int)c.kv_heads;
  a.ratio = (int)(x.heads / c.kv_heads);
  a.pages = (int)c.pages;
  a.page_shift = __builtin_ctzl((unsigned long)c.page_size);
  a.table_tokens = (int)(x.table_pages * c.page_size);
  a.prefix = (int)x.prefix_length;
  a.own_splits = p.own_splits, a.prefix_splits = p.prefix_splits;
  a.own_tiles = p.own_tiles, a.prefix_tiles = p.prefix_tiles;
  if (c.bits == 4)
    return x.type == SHK_SRC_BF16 ? launch_d<4, SHK_SRC_BF16>(c.head_dim, p.rt, a, s)
                                  : launch_d<4, SHK_SRC_F16>(c.head_dim, p.rt, a, s);
  return x.type == SHK_SRC_BF16 ? launch_d<8, SHK_SRC_BF16>(c.head_dim, p.rt, a, s)
                                : launch_d<8, SHK_SRC_F16>(c.head_dim, p.rt, a, s);
}

}  // namespace shk
