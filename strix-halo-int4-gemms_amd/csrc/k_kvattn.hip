// Attention of each sequence's newest tokens over the quantized cache
// (shk_kvattn.h has the mathematics of a step).
//
// kv_stream_kernel serves a sequence's own tokens (and a shared prefix with up
// to 64 query rows over the batch).  A workgroup is one key head and up to
// 16 * RT query rows; its four waves take every fourth step of 16 * NB tokens,
// each from memory to its own registers, and are joined through LDS.  The tokens of all sequences are
// dealt out evenly: in pieces of 256, a workgroup gets the same number of
// consecutive ones, whichever sequences they belong to.
//
// kv_prefix_kernel serves a shared prefix with many query rows (those of all
// sequences): the four waves have different rows, take the same 64 tokens,
// and each widens a quarter of them into LDS for all.
//
// kv_join_kernel joins the pieces of a row from their f32 outputs, references
// and sums.
//
// What bounds them, measured with 8 key heads of 128, four query heads each:
// * 4 sequences of up to 131072 tokens, int4 (317 MB): stream 70 us, 4.5 TB/s
//   of the 6.2 that a sum over memory reads at.  The vector unit, which widens
//   the codes and does the softmax, is busy half of the time, the matrix unit
//   a tenth.
// * 32 sequences of up to 4096 tokens, int8 (134 MB): stream 35 us, join 6.
//   A wave has four to eight steps, so its start (page numbers, then scales
//   and keys) and its end are a third of it.
// * 1 sequence of 1001 tokens: stream 8 us with 32 workgroups, join 5, two
//   dependent launches; the host needs 13 to prepare them.
// * 8 sequences of up to 6000 tokens with 40 rows of each of 2 key heads of 256,
//   int8 (30 MB): stream 27 us, join 6.  Rows are tiles of 16, so three
//   workgroups each fetch and widen the same tokens (94 MB), and the int8 heads
//   of 256 spill 4 to 8 vector registers (20 to 36 bytes of scratch a lane).
// * 64 sequences after a shared prefix of 65536 tokens, int4 (69 Gflop, 80 MB):
//   115 us, 600 Tflop/s.  Each 64 tokens are widened once for 128 rows, twice
//   for the 256 rows there are, and every wave reads them all from LDS for its
//   32.  Vector unit busy 54%, matrix unit 24, LDS 26: a wave does widening,
//   products and softmax in turn, two waves share a SIMD, and barriers keep
//   them in step.
// All forms of both kernels spill 12 to 98 scalar registers into lanes of
// vector registers, most of them between the steps' addresses and page numbers.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "shk_kvattn.h"

namespace shk {
namespace {

constexpr int kPiece = 4 * kKvTile;  // tokens that a workgroup's waves take at a time

struct AttnArgs {
  const uint16_t* q;
  long q_batch, q_query, q_head;  // strides in elements
  const uint8_t *kc, *vc;
  const uint16_t *ks, *vs;
  const int32_t *table, *lengths, *prefix_pages;
  long table_stride;
  uint16_t* out;
  float* lse;
  // Outputs of pieces and their (reference, sum): own [kv_heads][slots][own
  // rows], then prefix [splits][kv_heads][batch * own rows].
  float* part_o;
  float2* part_ml;
  float scale;
  int type;
  int batch, queries, heads, kv_heads, ratio;
  int pages, page_shift, table_tokens, prefix;
  int own_groups, own_tiles;        // workgroups of a key head and row tile; row tiles of 16 * RT rows
  int prefix_splits, prefix_tiles;  // pieces of the prefix; row tiles of its kernel
  int slots;                        // own_groups + batch
  int direct;                       // one piece a sequence at most and no prefix: out is written at once
};

__device__ __forceinline__ int own_rows(const AttnArgs& a) { return a.queries * a.ratio; }
__device__ __forceinline__ long own_parts(const AttnArgs& a) { return (long)a.kv_heads * a.slots * own_rows(a); }
__device__ __forceinline__ int tokens_of(const AttnArgs& a, int b) { return min(max(a.lengths[b], 0), a.table_tokens); }
// Pieces of a sequence; with `direct`, each is one piece, the empty ones too.
__device__ __forceinline__ int pieces_of(const AttnArgs& a, int tokens) {
  return a.direct ? 1 : (tokens + kPiece - 1) / kPiece;
}

template <int D>
__device__ __forceinline__ void store_row(const AttnArgs& a, long row, int d, f4 v) {
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    b[i] = a.type == SHK_SRC_BF16 ? f32_to_bf16_rne(v[i]) : __builtin_bit_cast(uint16_t, (_Float16)v[i]);
  *reinterpret_cast<uint2*>(a.out + row * D + d) = make_uint2(b[0] | (b[1] << 16), b[2] | (b[3] << 16));
}

// The power of two of l goes off against the one in m first: log2(l) would
// round to that of the value scales, up to 2^-18.
__device__ __forceinline__ float natural_lse(float m, float l) {
  const float whole = m + (float)__builtin_amdgcn_frexp_expf(l);
  const float lse = (whole + __log2f(__builtin_amdgcn_frexp_mantf(l))) * 0.6931471805599453f;
  return m == -__builtin_inff() && !(l != l) ? m : lse;
}

// The first of `total` pieces that workgroup j of `spread` takes, and the
// workgroup that takes a piece.
__device__ __forceinline__ int share(int j, int total, int spread) { return (int)((long)j * total / spread); }
__device__ __forceinline__ int taker(int piece, int total, int spread) {
  return (int)(((long)(piece + 1) * spread - 1) / total);
}

// Pieces of the sequences before b.
__device__ __forceinline__ int pieces_before(const AttnArgs& a, int b) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int b0 = 0; b0 < b; b0 += 64) n += b0 + lane < b ? pieces_of(a, tokens_of(a, b0 + lane)) : 0;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) n += __shfl_xor(n, d, 64);
  return n;
}

// Query row r of a key head's rows, for one sequence or (b0 < 0) all of them.
__device__ __forceinline__ void query_row(const AttnArgs& a, int head, int b0, int r, const void*& src, int& query,
                                          long& out) {
  const int per = own_rows(a);
  const int b = b0 < 0 ? r / per : b0, in = b0 < 0 ? r % per : r;
  query = in / a.ratio;
  const int h = head * a.ratio + in % a.ratio;
  src = a.q + b * a.q_batch + query * a.q_query + h * a.q_head;
  out = ((long)b * a.queries + query) * a.heads + h;
}

// One piece of a row, from 16 threads (part) of D / 16 values each: to the
// output where it is the only one, or to the parts.
template <int D>
__device__ __forceinline__ void store_piece(const AttnArgs& a, bool direct, long out_row, long part_row, int d, f4 v) {
  if (direct) store_row<D>(a, out_row, d, v);
  else *reinterpret_cast<f4*>(a.part_o + part_row * D + d) = v;
}

// The LDS of a workgroup of either kind.
template <int D>
struct StreamShared {
  static constexpr int kPitch = D + 4;  // floats of a row: the 16 rows start on different banks
  float o[4][16 * kPitch];              // the waves' outputs, references and sums
  float m[4][16], l[4][16];
};
template <int D>
struct PrefixShared {
  static constexpr int kBuffers = D == 256 ? 1 : 2;  // 64 KB a workgroup: two on a CU
  // the products' operands as the lanes read them: K by block and step, V by
  // 32 tokens and 16 values of head_dim
  h8 k[kBuffers][4][D / 32][64];
  h8 v[kBuffers][2][D / 16][64];
  float scale[kBuffers][2][kKvTile];
  int bad;
};

template <int BITS, int D, int RT, int TYPE>
__device__ __forceinline__ void stream_pieces(const AttnArgs& a, int unit, StreamShared<D>& lds) {
  using Rows = KvRows<BITS, D, RT, TYPE>;
  // blocks of 16 tokens a wave takes at a time: half of the usual four where
  // two row tiles or 256 columns take the registers (int8 at 256 spills even so)
  constexpr int NB = D * RT >= 256 ? 2 : 4;
  constexpr int kStep = 16 * NB, kPer = kPiece / kStep;
  constexpr int kPitch = StreamShared<D>::kPitch;
  auto &red_o = lds.o;
  auto &red_m = lds.m, &red_l = lds.l;
  const int lane = threadIdx.x & 63, g = lane / 16, c = lane % 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);

  // which pieces: those of the sequences first, then those of the prefix
  const int own_units = a.kv_heads * a.own_tiles * a.own_groups;
  const bool shared = unit >= own_units;
  if (shared) unit -= own_units;
  const int groups = shared ? a.prefix_splits : a.own_groups, tiles = shared ? a.prefix_tiles : a.own_tiles;
  const int head = unit % a.kv_heads;
  unit /= a.kv_heads;
  const int tile = unit % tiles, j = unit / tiles;
  // the pieces of the first 64 sequences, a lane each, and their sums
  const int tokens0 = !shared && lane < a.batch ? tokens_of(a, lane) : 0;
  const int pieces0 = !shared && lane < a.batch ? pieces_of(a, tokens0) : 0;
  int upto0 = pieces0;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int up = __shfl_up(upto0, d, 64);
    if (lane >= d) upto0 += up;
  }
  int total = shared ? pieces_of(a, a.prefix) : __shfl(upto0, 63, 64);
  if (!shared && a.batch > 64) total = pieces_before(a, a.batch);
  total = __builtin_amdgcn_readfirstlane(total);
  const int spread = max(min(groups, total), 1);  // workgroups with a piece
  const int first = j < spread ? share(j, total, spread) : total;
  const int end = j < spread ? share(j + 1, total, spread) : total;
  const int rows_here = own_rows(a) * (shared ? a.batch : 1);
  const KvView kv{a.kc, a.vc, a.ks, a.vs, a.pages, a.page_shift, a.kv_heads, head};

  int b = 0, before = 0;  // the sequence that holds piece `first`, and the pieces before it
  if (!shared && first < end) {
    int upto = upto0, own = pieces0;
    for (int b0 = 0;;) {
      const unsigned long past = __ballot(before + upto > first);
      if (past != 0) {
        const int at = __builtin_ctzll(past);
        b = b0 + at;
        before += __shfl(upto - own, at, 64);
        break;
      }
      before += __shfl(upto, 63, 64);
      b0 += 64;
      own = b0 + lane < a.batch ? pieces_of(a, tokens_of(a, b0 + lane)) : 0;
      upto = own;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const int up = __shfl_up(upto, d, 64);
        if (lane >= d) upto += up;
      }
    }
    b = __builtin_amdgcn_readfirstlane(b);
    before = __builtin_amdgcn_readfirstlane(before);
  }
  // a sequence without tokens has no piece; a prefix split may have none either
  for (int piece = first; piece < end || (shared && piece == first); ++b) {
    const int n = shared ? a.prefix
                         : (b < 64 ? __builtin_amdgcn_readfirstlane(__shfl(tokens0, b, 64)) : tokens_of(a, b));
    const int mine = min(end, before + pieces_of(a, n));  // this sequence's pieces end there
    if (!shared && mine <= piece) {
      before += pieces_of(a, n);
      continue;
    }
    const void* src[RT];
    long out_row[RT];
    int limit[RT], least = n;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int r = (tile * RT + t) * 16 + c;
      src[t] = nullptr;
      out_row[t] = -1;
      limit[t] = n;
      if (r < rows_here) {
        int query;
        query_row(a, head, shared ? -1 : b, r, src[t], query, out_row[t]);
        if (!shared) limit[t] = max(n - a.queries + query + 1, 0);
      }
      least = min(least, limit[t]);
    }
#pragma unroll
    for (int d = 1; d < 16; d *= 2) least = min(least, __shfl_xor(least, d, 64));
    least = __builtin_amdgcn_readfirstlane(least);

    const int32_t* table = shared ? a.prefix_pages : a.table + b * a.table_stride;
    const int last = (n - 1) >> 4;  // the last block that holds a token; later ones repeat it, masked
    bool bad = false;
    Rows rows;
    rows.begin(src, a.scale);
    // A step's V is asked for with the next step's K, so half of the bytes are
    // always on their way.
    const int step0 = kPer * (piece - before) + wave, step_end = min(kPer * (mine - before), (n + kStep - 1) / kStep);
    const int step_last = step0 + (max(step_end - step0, 1) - 1) / 4 * 4;
    struct Keys {
      KvBlock<BITS, D> blk[NB];
      u2 scales[NB];
    };
    long rows_now[NB], rows_next[NB];  // first rows of the blocks
    int page[NB];                    // and pages of those after
    auto pages = [&](int i) {
#pragma unroll
      for (int x = 0; x < NB; ++x) page[x] = kv.page_of(table, min(NB * min(i, step_last) + x, last));
    };
    auto find_rows = [&](int i, long (&r)[NB]) {
#pragma unroll
      for (int x = 0; x < NB; ++x) r[x] = kv.row_of(page[x], min(NB * min(i, step_last) + x, last), bad);
    };
    auto load_keys = [&](const long (&r)[NB], Keys& k) {
#pragma unroll
      for (int x = 0; x < NB; ++x) k.blk[x].load_k(kv, r[x]), k.scales[x] = load_scales(kv.ks, r[x]);
    };
    auto step = [&](int i, Keys& now, Keys& next) {
      u2 vss[NB];
#pragma unroll
      for (int x = 0; x < NB; ++x) now.blk[x].load_v(kv, rows_now[x]), vss[x] = load_scales(kv.vs, rows_now[x]);
      find_rows(i + 4, rows_next);
      load_keys(rows_next, next);
      pages(i + 8);
#pragma unroll
      for (int x = 0; x < NB; ++x) rows_now[x] = rows_next[x];
      __builtin_amdgcn_sched_barrier(0);  // what has been asked for stays ahead
      f4 s[RT][NB], ks[NB], vs[NB];
#pragma unroll
      for (int x = 0; x < NB; ++x) {
#pragma unroll
        for (int t = 0; t < RT; ++t) s[t][x] = f4{0, 0, 0, 0};
#pragma unroll
        for (int st = 0; st < Rows::kSteps; ++st) {
          const h8 k = now.blk[x].k_operand(st);
#pragma unroll
          for (int t = 0; t < RT; ++t) s[t][x] = mfma_f16(k, rows.q[t][st], s[t][x]);
        }
        ks[x] = widen_scales(now.scales[x]);
        vs[x] = widen_scales(vss[x]);
      }
      const int t0 = i * kStep;
      int left[RT];
#pragma unroll
      for (int t = 0; t < RT; ++t) left[t] = limit[t] - t0;
      h8 p[RT][NB / 2], pl[RT][NB / 2];
      rows.template soften<NB>(s, ks, vs, t0 + kStep > least, left, p, pl);
#pragma unroll
      for (int h = 0; h < NB / 2; ++h)
#pragma unroll
        for (int w = 0; w < Rows::kOut / 4; ++w) {
          h2 f[4][4];
#pragma unroll
          for (int x = 0; x < 4; ++x) now.blk[2 * h + x / 2].v_pairs(w, x % 2, f[x]);
#pragma unroll
          for (int jj = 0; jj < 4; ++jj)
            rows.template add<NB / 2>(4 * w + jj, join(f[0][jj], f[1][jj], f[2][jj], f[3][jj]), p, pl, h);
        }
    };
    if (step0 < step_end) {
      Keys now, next;
      pages(step0);
      find_rows(step0, rows_now);
      load_keys(rows_now, now);
      pages(step0 + 4);
#pragma unroll 1
      for (int i = step0; i < step_end; i += 4) {
        step(i, now, next);
#pragma unroll
        for (int x = 0; x < NB; ++x) {
#pragma unroll
          for (int w = 0; w < KvBlock<BITS, D>::kK; ++w) now.blk[x].k[w] = next.blk[x].k[w];
          now.scales[x] = next.scales[x];
        }
      }
    }

    // the waves' outputs, relative to the largest of their references
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const float l = groups_sum(rows.l[t]);
      __syncthreads();
      if (g == 0) red_m[wave][c] = rows.m[t], red_l[wave][c] = bad ? __builtin_nanf("") : l;
      __syncthreads();
      float top = red_m[0][c];
#pragma unroll
      for (int w = 1; w < 4; ++w) top = __builtin_fmaxf(top, red_m[w][c]);
      const float back = __builtin_amdgcn_exp2f(rows.m[t] - (top == -__builtin_inff() ? 0.0f : top));
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int jj = 0; jj < Rows::kOut; jj += 4)
          *reinterpret_cast<f4*>(&red_o[wave][c * kPitch + (4 * g + r) * Rows::kOut + jj]) =
              f4{rows.o[t][jj][r], rows.o[t][jj + 1][r], rows.o[t][jj + 2][r], rows.o[t][jj + 3][r]} * back;
      __syncthreads();
      // 16 threads a row, D / 16 values each
      const int rr = threadIdx.x / 16, part = threadIdx.x % 16;
      float rtop = red_m[0][rr];
#pragma unroll
      for (int w = 1; w < 4; ++w) rtop = __builtin_fmaxf(rtop, red_m[w][rr]);
      const float rbase = rtop == -__builtin_inff() ? 0.0f : rtop;
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float half = half_weight(red_m[w][rr] - rbase);
        sum += red_l[w][rr] * half * half;
      }
      const long at = __shfl(out_row[t], rr, 64);  // from the lane that holds the row
      if (at >= 0) {
        const int row = (tile * RT + t) * 16 + rr;
        const long to = shared ? own_parts(a) + ((long)j * a.kv_heads + head) * rows_here + row
                               : ((long)head * a.slots + j + b) * rows_here + row;
        const float f = !a.direct ? 1.0f : (sum == 0.0f ? 0.0f : 1.0f / sum);
#pragma unroll
        for (int k = 0; k < D / 64; ++k) {
          const int d = (k * 16 + part) * 4;
          f4 v = f4{0, 0, 0, 0};
#pragma unroll
          for (int w = 0; w < 4; ++w) v += *reinterpret_cast<const f4*>(&red_o[w][rr * kPitch + d]);
          store_piece<D>(a, a.direct, at, to, d, v * f);
        }
        if (part == 0) {
          if (!a.direct) a.part_ml[to] = make_float2(rtop, sum);
          else if (a.lse != nullptr) a.lse[at] = natural_lse(rtop, sum);
        }
      }
    }
    piece = max(mine, piece + (shared ? 1 : 0));
    before += pieces_of(a, n);
    if (shared) break;
  }
}

template <int BITS, int D, int RT, int TYPE>
__device__ __forceinline__ void prefix_pieces(const AttnArgs& a, int unit, PrefixShared<D>& lds) {
  using Rows = KvRows<BITS, D, RT, TYPE>;
  using Block = KvBlock<BITS, D>;
  constexpr int kBuffers = PrefixShared<D>::kBuffers;
  constexpr int kSteps = Rows::kSteps, kOut = Rows::kOut;
  auto &lds_k = lds.k;
  auto &lds_v = lds.v;
  auto &lds_s = lds.scale;
  int &lds_bad = lds.bad;
  const int lane = threadIdx.x & 63, g = lane / 16, c = lane % 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int head = unit % a.kv_heads;
  unit /= a.kv_heads;
  const int split = unit % a.prefix_splits, tile = unit / a.prefix_splits;
  const int n = a.prefix, rows_here = own_rows(a) * a.batch;
  const int steps = (n + kKvTile - 1) / kKvTile, each = (steps + a.prefix_splits - 1) / a.prefix_splits;
  const int first = split * each, end = min(first + each, steps);
  const KvView kv{a.kc, a.vc, a.ks, a.vs, a.pages, a.page_shift, a.kv_heads, head};
  const int last = (n - 1) >> 4;

  const void* src[RT];
  int row[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    row[t] = ((tile * 4 + wave) * RT + t) * 16 + c;
    src[t] = nullptr;
    int query;
    long out;
    if (row[t] < rows_here) query_row(a, head, -1, row[t], src[t], query, out);
  }
  Rows rows;
  rows.begin(src, a.scale);
  bool bad = false;
  if (threadIdx.x == 0) lds_bad = 0;

  Block mine;  // this wave's 16 of the 64 tokens
  u2 ksw, vsw;
  int page = first < end ? kv.page_of(a.prefix_pages, min(4 * first + wave, last)) : 0;
  auto load = [&](int step) {
    const long row0 = kv.row_of(page, min(4 * step + wave, last), bad);
    mine.load_k(kv, row0);
    mine.load_v(kv, row0);
    ksw = load_scales(kv.ks, row0);
    vsw = load_scales(kv.vs, row0);
    page = kv.page_of(a.prefix_pages, min(4 * min(step + 1, end - 1) + wave, last));
  };
  if (first < end) load(first);
  for (int step = first, at = 0; step < end; ++step, at = (at + 1) % kBuffers) {
#pragma unroll
    for (int st = 0; st < kSteps; ++st) lds_k[at][wave][st][lane] = mine.k_operand(st);
#pragma unroll
    for (int w = 0; w < kOut / 4; ++w) {
      h2 f[2][4];
      mine.v_pairs(w, 0, f[0]);
      mine.v_pairs(w, 1, f[1]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint2 pair = make_uint2(__builtin_bit_cast(uint32_t, f[0][j]), __builtin_bit_cast(uint32_t, f[1][j]));
        reinterpret_cast<uint2*>(&lds_v[at][wave / 2][4 * w + j][lane])[wave % 2] = pair;
      }
    }
    if (c == 0) {
      *reinterpret_cast<f4*>(&lds_s[at][0][16 * wave + 4 * g]) = widen_scales(ksw);
      *reinterpret_cast<f4*>(&lds_s[at][1][16 * wave + 4 * g]) = widen_scales(vsw);
    }
    load(min(step + 1, end - 1));  // on its way while this one is multiplied; the last one is loaded twice
    __syncthreads();
    f4 ks[4], vs[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      ks[x] = *reinterpret_cast<const f4*>(&lds_s[at][0][16 * x + 4 * g]);
      vs[x] = *reinterpret_cast<const f4*>(&lds_s[at][1][16 * x + 4 * g]);
    }
    f4 s[RT][4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
#pragma unroll
      for (int t = 0; t < RT; ++t) s[t][x] = f4{0, 0, 0, 0};
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
        const h8 k = lds_k[at][x][st][lane];
#pragma unroll
        for (int t = 0; t < RT; ++t) s[t][x] = mfma_f16(k, rows.q[t][st], s[t][x]);
      }
    }
    int left[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) left[t] = n - step * kKvTile;
    h8 p[RT][2], pl[RT][2];
    rows.template soften<4>(s, ks, vs, left[0] < kKvTile, left, p, pl);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < kOut; ++j) rows.template add<2>(j, lds_v[at][h][j][lane], p, pl, h);
    if constexpr (kBuffers == 1) __syncthreads();
  }
  __syncthreads();  // lds_bad has been cleared; a page outside the cache is every row's
  if (bad && lane == 0) lds_bad = 1;
  __syncthreads();
  bad = lds_bad != 0;
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const float l = groups_sum(rows.l[t]);
    if (row[t] >= rows_here) continue;
    const long to = own_parts(a) + ((long)split * a.kv_heads + head) * rows_here + row[t];
    if (g == 0) a.part_ml[to] = make_float2(rows.m[t], bad ? __builtin_nanf("") : l);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < kOut; j += 4)
        *reinterpret_cast<f4*>(a.part_o + to * D + (4 * g + r) * kOut + j) =
            f4{rows.o[t][j][r], rows.o[t][j + 1][r], rows.o[t][j + 2][r], rows.o[t][j + 3][r]};
  }
}

template <int BITS, int D, int RT, int TYPE>
__global__ __launch_bounds__(256, 2) void kv_stream_kernel(const AttnArgs a) {
  __shared__ __align__(16) StreamShared<D> lds;
  stream_pieces<BITS, D, RT, TYPE>(a, blockIdx.x, lds);
}

// The prefix's workgroups and those of the sequences' own tokens in one
// launch: the latter fill the CUs that the former leave.
template <int BITS, int D, int PREFIX_RT, int RT, int TYPE>
__global__ __launch_bounds__(256, 2) void kv_prefix_kernel(const AttnArgs a) {
  __shared__ __align__(16) union {
    PrefixShared<D> prefix;
    StreamShared<D> stream;
  } lds;
  const int units = a.kv_heads * a.prefix_tiles * a.prefix_splits;
  if ((int)blockIdx.x < units) prefix_pieces<BITS, D, PREFIX_RT, TYPE>(a, blockIdx.x, lds.prefix);
  else stream_pieces<BITS, D, RT, TYPE>(a, blockIdx.x - units, lds.stream);
}

// Joins the pieces of a row, a workgroup each: lane p of every wave looks at
// piece p, then wave w adds up the outputs of the pieces w, w + 4, ..., D / 64
// values a lane.
template <int D>
__global__ __launch_bounds__(256) void kv_join_kernel(const AttnArgs a) {
  typedef float fv __attribute__((ext_vector_type(D / 64)));
  __shared__ fv part[4][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const long row = blockIdx.x;
  const int h = (int)(row % a.heads), query = (int)(row / a.heads % a.queries), b = (int)(row / a.heads / a.queries);
  const int head = h / a.ratio, in = query * a.ratio + h % a.ratio, per = own_rows(a);
  // pieces before the sequence, its own, and all
  int before = 0, total = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const int n = b0 + lane < a.batch ? pieces_of(a, tokens_of(a, b0 + lane)) : 0;
    total += n;
    before += b0 + lane < b ? n : 0;
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) total += __shfl_xor(total, d, 64), before += __shfl_xor(before, d, 64);
  const int mine = pieces_of(a, tokens_of(a, b));
  const int spread = max(min(a.own_groups, total), 1);
  const int first = mine == 0 ? 0 : taker(before, total, spread);
  const int own = mine == 0 ? 0 : taker(before + mine - 1, total, spread) - first + 1;
  const int count = own + a.prefix_splits;
  const long own_at = ((long)head * a.slots + first + b) * per + in;
  const long prefix_at = own_parts(a) + (long)head * per * a.batch + (long)b * per + in;
  const long prefix_step = (long)a.kv_heads * per * a.batch;
  auto place = [&](int p) { return p < own ? own_at + (long)p * per : prefix_at + (p - own) * prefix_step; };
  float top = -__builtin_inff();
  for (int p = lane; p < count; p += 64) top = __builtin_fmaxf(top, a.part_ml[place(p)].x);
#pragma unroll
  for (int d = 1; d < 64; d *= 2) top = __builtin_fmaxf(top, __shfl_xor(top, d, 64));
  const float base = top == -__builtin_inff() ? 0.0f : top;
  float sum = 0.0f;
  fv v = {};
  for (int p0 = 0; p0 < count; p0 += 64) {
    float weight = 0.0f;
    if (p0 + lane < count) {
      // A piece of NaN keys has reference -inf, so a weight of 0 does not mean
      // that it says nothing: 0 times its NaN sum and outputs stays NaN.
      const float2 ml = a.part_ml[place(p0 + lane)];
      const float half = half_weight(ml.x - base);
      weight = half * half;
      sum += ml.y * half * half;
    }
    const int here = min(count - p0, 64);
    for (int p = wave; p < here; p += 32) {  // eight loads at a time
      fv o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        o[i] = reinterpret_cast<const fv*>(a.part_o + place(p0 + min(p + 4 * i, here - 1)) * D)[lane];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float w = __shfl(weight, min(p + 4 * i, here - 1), 64);
        if (p + 4 * i < here) v += o[i] * w;
      }
    }
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d, 64);
  part[wave][lane] = v;
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int w = 1; w < 4; ++w) v += part[w][lane];
  v *= sum == 0.0f ? 0.0f : 1.0f / sum;
  uint16_t o[D / 64];
#pragma unroll
  for (int i = 0; i < D / 64; ++i)
    o[i] = a.type == SHK_SRC_BF16 ? (uint16_t)f32_to_bf16_rne(v[i]) : __builtin_bit_cast(uint16_t, (_Float16)v[i]);
  __builtin_memcpy(a.out + row * D + lane * (D / 64), o, sizeof(o));
  if (lane == 0 && a.lse != nullptr) a.lse[row] = natural_lse(top, sum);
}

long cdiv(long a, long b) { return (a + b - 1) / b; }

struct Plan {
  int rt, prefix_rt;                  // row tiles of a wave in the two kernels
  bool prefix_kernel;                 // the prefix has a kernel of its own
  int own_groups, own_tiles, prefix_splits, prefix_tiles;
  bool direct;
};

// For at least one query row.
Plan plan_of(const shk_kv_cache& c, const shk_kv_attention& a) {
  const long rows = a.queries * (a.heads / c.kv_heads), all = rows * a.batch, tokens = a.table_pages * c.page_size;
  const bool wide = c.head_dim == 256;  // two row tiles of 256 columns would not fit the registers
  Plan p{};
  const bool prefix = a.prefix_length > 0;
  // The prefix's own kernel widens a token once for up to 128 rows, the
  // streaming one once for 16 * rt but without barriers.  Us with the one / the
  // other after 2000 and 32768 shared tokens, int4: 64 rows of 128 20 / 17 and
  // 45 / 41, 96 rows 22 / 22 and 50 / 63; of 256 23 / 21 and 56 / 58, 25 / 27 and
  // 74 / 93; 256 rows of 128 after 65536 tokens 121 / 145.
  p.prefix_kernel = prefix && all > 64;
  // Two row tiles read a sequence's tokens once for 32 rows: 24 sequences of up
  // to 8000 tokens with 32 rows 61 us instead of 68.  Where only the batch has
  // more than 16 rows, two tiles for its prefix gain after a long one (64 rows
  // 38 us, with one tile 41) what they lose after a short one (19 and 17).
  p.rt = wide || rows <= 16 ? 1 : 2;
  p.prefix_rt = wide ? 1 : 2;
  p.own_tiles = (int)cdiv(rows, 16 * p.rt);
  p.direct = !prefix && tokens <= kPiece;
  const long want = 512;  // two workgroups on each of the 256 CUs
  p.own_groups = p.direct ? (int)a.batch
                          : (int)std::max(1L, std::min(want / (c.kv_heads * p.own_tiles),
                                                       a.batch * cdiv(tokens, kPiece)));
  if (prefix) {
    p.prefix_tiles = (int)cdiv(all, p.prefix_kernel ? 64 * p.prefix_rt : 16 * p.rt);
    p.prefix_splits = (int)std::max(1L, std::min(cdiv(want, c.kv_heads * p.prefix_tiles),
                                                 cdiv(a.prefix_length, kPiece)));
  }
  return p;
}

long part_rows(const shk_kv_cache& c, const shk_kv_attention& a, const Plan& p) {
  const long rows = a.queries * (a.heads / c.kv_heads);
  return p.direct ? 0 : c.kv_heads * rows * (p.own_groups + a.batch + (long)p.prefix_splits * a.batch);
}

template <int BITS, int D, int RT, int TYPE>
hipError_t launch_rt(const AttnArgs& a, const Plan& p, hipStream_t s) {
  const long own = (long)a.kv_heads * a.own_tiles * a.own_groups;
  const long prefix = (long)a.kv_heads * a.prefix_tiles * a.prefix_splits;
  const dim3 grid((unsigned)(own + prefix)), block(256);
  if (p.prefix_kernel)
    hipLaunchKernelGGL((kv_prefix_kernel<BITS, D, D == 256 ? 1 : 2, RT, TYPE>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((kv_stream_kernel<BITS, D, RT, TYPE>), grid, block, 0, s, a);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess || a.direct) return err;
  const long rows = (long)a.batch * a.queries * a.heads;
  hipLaunchKernelGGL((kv_join_kernel<D>), dim3((unsigned)rows), block, 0, s, a);
  return hipGetLastError();
}

template <int BITS, int D, int TYPE>
hipError_t launch_kernels(const AttnArgs& a, const Plan& p, hipStream_t s) {
  if constexpr (D < 256)
    if (p.rt == 2) return launch_rt<BITS, D, 2, TYPE>(a, p, s);
  return launch_rt<BITS, D, 1, TYPE>(a, p, s);
}

template <int BITS, int TYPE>
hipError_t launch_d(long d, const AttnArgs& a, const Plan& p, hipStream_t s) {
  if (d == 64) return launch_kernels<BITS, 64, TYPE>(a, p, s);
  if (d == 128) return launch_kernels<BITS, 128, TYPE>(a, p, s);
  return launch_kernels<BITS, 256, TYPE>(a, p, s);
}

}  // namespace

int64_t kv_attention_workspace(const shk_kv_cache& c, const shk_kv_attention& a) {
  return part_rows(c, a, plan_of(c, a)) * (c.head_dim * 4 + 8);
}

bool kv_attention_fits(const shk_kv_cache& c, const shk_kv_attention& a) {
  const Plan p = plan_of(c, a);
  const long first = c.kv_heads * ((long)p.own_tiles * p.own_groups + (long)p.prefix_tiles * p.prefix_splits);
  const long join = p.direct ? 0 : a.batch * a.queries * a.heads;  // a workgroup a row
  return std::max(first, join) <= kMostWorkgroups;
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
  a.part_ml = reinterpret_cast<float2*>(a.part_o + part_rows(c, x, p) * c.head_dim);
  a.scale = (float)x.scale;
  a.type = (int)x.type;
  a.batch = (int)x.batch, a.queries = (int)x.queries, a.heads = (int)x.heads, a.kv_heads = (int)c.kv_heads;
  a.ratio = (int)(x.heads / c.kv_heads);
  a.pages = (int)c.pages;
  a.page_shift = __builtin_ctzl((unsigned long)c.page_size);
  a.table_tokens = (int)(x.table_pages * c.page_size);
  a.prefix = (int)x.prefix_length;
  a.own_groups = p.own_groups, a.own_tiles = p.own_tiles;
  a.prefix_splits = p.prefix_splits, a.prefix_tiles = p.prefix_tiles;
  a.slots = p.own_groups + a.batch;
  a.direct = p.direct;
  if (c.bits == 4)
    return x.type == SHK_SRC_BF16 ? launch_d<4, SHK_SRC_BF16>(c.head_dim, a, p, s)
                                  : launch_d<4, SHK_SRC_F16>(c.head_dim, a, p, s);
  return x.type == SHK_SRC_BF16 ? launch_d<8, SHK_SRC_BF16>(c.head_dim, a, p, s)
                                : launch_d<8, SHK_SRC_F16>(c.head_dim, a, p, s);
}

}  // namespace shk
