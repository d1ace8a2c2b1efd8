// Drafted tokens against the target's probabilities: how many are kept, and the
// token that follows them, drawn from what the draft left of the target.
//
// The kept drafts are a handful of gathers, which a wave tests at once; every
// wave does so for itself.  The draw needs the sum of one row's weights before the
// place where the running sum passes its share u of it.  Sums are 64 bits: over a
// vocabulary f32 would move the place by whole tokens, and the order of adding
// would show.
//  * verify_whole, up to 32768 tokens: a workgroup has a sequence's rows in its
//    registers, one launch.  Bound by latency (tokens, gathers, rows, each asked
//    for with what came before), and by what one CU can read.
//  * verify_sums and verify_draw: the vocabulary is cut into pieces over all CUs,
//    added first, then the piece and the token in it are found.  Bound by the one
//    row of each kind that a sequence reads, and by the second launch: 61 x 131072
//    f32 (61 MB) 13 us (4.6 TB/s) and 11.5.
// f32, replayed, whole and in pieces: 1 x 2048 3.7 and 13.5 us, 128 x 16384 9 and
// 24, 1 x 32768 8.5 and 11.2, 128 x 32768 12 and 19.5.
#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>

#include "shk_common.h"
#include "shk_lanes.h"
#include "shk_loads.h"
#include "shk_step.h"

namespace shk {
namespace {

constexpr int kThreads = 256;
constexpr int kPieces = 256;           // at most, of a row
constexpr int kPiece = kThreads * 8;   // values of a step of a workgroup

struct Pieces {
  int count, size;  // size: values of a piece, whole steps
};

struct Sum {
  double left, all;  // of max(target - draft, 0), of target
};

// What verify_sums leaves for verify_draw: kept drafts of each sequence, then the
// sums of its pieces.
__host__ __device__ constexpr long kept_bytes(long batch) { return (batch * 4 + 15) / 16 * 16; }

template <int TYPE>
__device__ __forceinline__ float value_of(const void* x, long i) {
  if constexpr (TYPE == SHK_SRC_F32) return static_cast<const float*>(x)[i];
  const uint16_t h = static_cast<const uint16_t*>(x)[i];
  return TYPE == SHK_SRC_BF16 ? bf16_bits_to_f32(h) : (float)__builtin_bit_cast(_Float16, h);
}

// Values [at, at + 8) of a row, those from `count` on as 0.  Whole ones come in
// vectors, of any alignment.
template <int TYPE>
__device__ __forceinline__ void load8(const void* x, long at, long count, float (&v)[8]) {
  if (count >= 8) {
    constexpr int SIZE = TYPE == SHK_SRC_F32 ? 4 : 2;
    const any_u4* src = reinterpret_cast<const any_u4*>(static_cast<const uint8_t*>(x) + at * SIZE);
    u4 u[SIZE / 2];
#pragma unroll
    for (int i = 0; i < SIZE / 2; ++i) u[i] = src[i];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (TYPE == SHK_SRC_F32) {
        v[e] = __uint_as_float(u[e / 4][e % 4]);
      } else {
        const uint16_t h = (uint16_t)(u[0][e / 2] >> (16 * (e % 2)));
        v[e] = TYPE == SHK_SRC_BF16 ? bf16_bits_to_f32(h) : (float)__builtin_bit_cast(_Float16, h);
      }
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = e < count ? value_of<TYPE>(x, at + e) : 0.f;
}

__device__ __forceinline__ long token_of(const shk_verify& p, long i) {
  return p.token_bytes == 8 ? static_cast<const int64_t*>(p.tokens)[i] : static_cast<const int32_t*>(p.tokens)[i];
}

__device__ __forceinline__ int drafts_of(const shk_verify& p, long b) {
  return p.counts == nullptr ? (int)p.drafts : min(max(p.counts[b], 0), (int)p.drafts);
}

// Drafts of sequence b that are kept; every lane of a wave gets the number.
template <int TYPE>
__device__ __forceinline__ int kept_of(const shk_verify& p, long b) {
  const int lane = threadIdx.x & 63;
  bool keeps = false;
  if (lane < drafts_of(p, b)) {
    const long token = token_of(p, b * p.drafts + lane);
    if (token >= 0 && token < p.vocab) {
      const double have = value_of<TYPE>(p.target, b * p.target_batch_stride + lane * p.target_row_stride + token);
      const double drawn =
          p.draft == nullptr ? 1.0 : value_of<TYPE>(p.draft, b * p.draft_batch_stride + lane * p.draft_row_stride + token);
      keeps = (double)p.uniforms[b * (p.drafts + 1) + lane] * drawn < have;
    }
  }
  const unsigned long long lost = ~__ballot(keeps);
  return lost == 0 ? 64 : __builtin_ctzll(lost);
}

// The row that the next token of sequence b is drawn from.
struct Row {
  long target, draft;  // of their first values; draft < 0: none
  long certain;        // the token that a draft without probabilities was certain of, or -1
};

__device__ __forceinline__ Row row_of(const shk_verify& p, long b, int kept) {
  Row r{b * p.target_batch_stride + kept * p.target_row_stride, -1, -1};
  if (kept < drafts_of(p, b)) {
    if (p.draft != nullptr) r.draft = b * p.draft_batch_stride + kept * p.draft_row_stride;
    else r.certain = token_of(p, b * p.drafts + kept);
  }
  return r;
}

// Target and draft at values [t, t + 8); of a draft without probabilities the
// token that it was certain of takes everything.
template <int TYPE>
__device__ __forceinline__ void values8(const shk_verify& p, const Row& r, long t, float (&have)[8], float (&gone)[8]) {
  const long count = p.vocab - t;
  load8<TYPE>(p.target, r.target + t, count, have);
  if (r.draft >= 0) {
    load8<TYPE>(p.draft, r.draft + t, count, gone);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) gone[e] = t + e == r.certain ? __builtin_inff() : 0.f;
  }
}

// The weights of a value; NaN and negative ones count as 0.
__device__ __forceinline__ Sum weight_of(float have, float gone) {
  const double all = __builtin_fmaxf(have, 0.f);
  return Sum{__builtin_fmax(all - (double)gone, 0.0), all};
}

template <int TYPE>
__device__ __forceinline__ void weights8(const shk_verify& p, const Row& r, long t, Sum (&w)[8]) {
  float have[8], gone[8];
  values8<TYPE>(p, r, t, have, gone);
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = weight_of(have[e], gone[e]);
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void verify_sums(const shk_verify p, const Pieces pieces) {
  __shared__ Sum parts[kThreads / 64];
  const long b = blockIdx.y;
  const int kept = kept_of<TYPE>(p, b);
  const Row r = row_of(p, b, kept);
  const long from = (long)blockIdx.x * pieces.size, to = min(from + pieces.size, (long)p.vocab);
  Sum mine{0.0, 0.0};
  for (long t = from + threadIdx.x * 8; t < to; t += kPiece) {
    Sum w[8];
    weights8<TYPE>(p, r, t, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) mine.left += w[e].left, mine.all += w[e].all;
  }
  mine.left = wave_inclusive(mine.left), mine.all = wave_inclusive(mine.all);
  if ((threadIdx.x & 63) == 63) parts[threadIdx.x >> 6] = mine;
  __syncthreads();
  if (threadIdx.x == 0) {
    Sum s = parts[0];
    for (int w = 1; w < kThreads / 64; ++w) s.left += parts[w].left, s.all += parts[w].all;
    uint8_t* work = static_cast<uint8_t*>(p.workspace);
    reinterpret_cast<Sum*>(work + kept_bytes(p.batch))[b * pieces.count + blockIdx.x] = s;
    if (blockIdx.x == 0) reinterpret_cast<int32_t*>(work)[b] = kept;
  }
}

// Inclusive sums over the workgroup's threads, of both weights.
__device__ __forceinline__ Sum group_inclusive(Sum v, Sum (&parts)[kThreads / 64]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v.left = wave_inclusive(v.left), v.all = wave_inclusive(v.all);
  if (lane == 63) parts[wave] = v;
  __syncthreads();
  Sum before{0.0, 0.0};
  for (int w = 0; w < wave; ++w) before.left += parts[w].left, before.all += parts[w].all;
  return Sum{before.left + v.left, before.all + v.all};
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void verify_draw(const shk_verify p, const Pieces pieces) {
  __shared__ Sum parts[2][kThreads / 64], total;
  __shared__ double before;
  __shared__ int piece, passes, holds, holds_here;
  const long b = blockIdx.x;
  const uint8_t* work = static_cast<const uint8_t*>(p.workspace);
  const int kept = reinterpret_cast<const int32_t*>(work)[b];
  const Row r = row_of(p, b, kept);
  const Sum* sums = reinterpret_cast<const Sum*>(work + kept_bytes(p.batch)) + b * pieces.count;
  const Sum mine = (int)threadIdx.x < pieces.count ? sums[threadIdx.x] : Sum{0.0, 0.0};
  // what is needed at the end, asked for now
  const double uniform = p.uniforms[b * (p.drafts + 1) + p.drafts];
  const long drafted = (int)threadIdx.x < (int)p.drafts ? token_of(p, b * p.drafts + threadIdx.x) : -1;
  const int lost = drafts_of(p, b) - kept, length = p.lengths != nullptr ? p.lengths[b] : 0;
  const Sum upto = group_inclusive(mine, parts[0]);
  if (threadIdx.x == 0) piece = passes = INT_MAX, holds = holds_here = -1;
  if (threadIdx.x == kThreads - 1) total = upto;
  __syncthreads();
  const bool rest = total.left > 0.0;
  const double share = uniform * (rest ? total.left : total.all);
  const double run = rest ? upto.left : upto.all, own = rest ? mine.left : mine.all;
  // the first piece whose running sum passes the share; the last that holds
  // anything where a share of the whole sum, or more, was asked for
  if (own > 0.0) {
    if (run > share) atomicMin(&piece, (int)threadIdx.x);
    atomicMax(&holds, (int)threadIdx.x);
  }
  __syncthreads();
  const int at = piece < kThreads ? piece : holds;
  if ((int)threadIdx.x == at) before = run - own;
  __syncthreads();
  long token = -1;
  if (at >= 0) {
    double carry = before;
    const long from = (long)at * pieces.size, to = min(from + pieces.size, (long)p.vocab);
    for (long base = from; base < to; base += kPiece) {
      const long t = base + threadIdx.x * 8;
      Sum w[8], sum{0.0, 0.0};
      weights8<TYPE>(p, r, t, w);
      double values[8], mass = 0.0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        values[e] = t + e < to ? (rest ? w[e].left : w[e].all) : 0.0;
        mass += values[e];
      }
      sum.left = mass;
      const double through = carry + group_inclusive(sum, parts[1]).left;
      double upto_e = through - mass;
      int first = -1, last = -1;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        upto_e += values[e];
        if (values[e] > 0.0) {
          last = (int)(t - from) + e;
          if (first < 0 && upto_e > share) first = last;
        }
      }
      if (first >= 0) atomicMin(&passes, first);
      if (last >= 0) atomicMax(&holds_here, last);
      if (threadIdx.x == kThreads - 1) before = through;
      __syncthreads();
      if (passes != INT_MAX) break;
      carry = before;
    }
    // rounding can leave the running sum of a piece just below its own sum
    token = from + (passes != INT_MAX ? passes : holds_here);
  }
  const int i = threadIdx.x;  // there are fewer drafts than threads
  if (i <= (int)p.drafts) p.out[b * (p.drafts + 1) + i] = i < kept ? drafted : i == kept ? token : -1;
  if (i == 0) {
    p.kept[b] = kept;
    if (p.lengths != nullptr) p.lengths[b] = length - lost;
  }
}

// A whole sequence in a workgroup: wave w has the values [w, w + 1) * 512 * STEPS,
// a lane 8 of each 512.  The waves' sums say which of them holds the place, and
// that one goes through its values again, which are still in its registers.
template <int TYPE, int WAVES, int STEPS>
__global__ __launch_bounds__(64 * WAVES) void verify_whole(const shk_verify p) {
  __shared__ Sum parts[WAVES];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long b = blockIdx.x;
  const double uniform = p.uniforms[b * (p.drafts + 1) + p.drafts];
  const long drafted = lane < (int)p.drafts ? token_of(p, b * p.drafts + lane) : -1;
  const int length = p.lengths != nullptr ? p.lengths[b] : 0;
  const int kept = kept_of<TYPE>(p, b);
  const Row r = row_of(p, b, kept);
  const long from = (long)wave * 512 * STEPS + lane * 8;
  float have[STEPS][8], gone[STEPS][8];
#pragma unroll
  for (int i = 0; i < STEPS; ++i) values8<TYPE>(p, r, from + i * 512, have[i], gone[i]);
  Sum mine{0.0, 0.0};
#pragma unroll
  for (int i = 0; i < STEPS; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const Sum w = weight_of(have[i][e], gone[i][e]);
      mine.left += w.left, mine.all += w.all;
    }
  // what was read stays, not the weights made of it, which are twice as large
#pragma unroll
  for (int i = 0; i < STEPS; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) asm volatile("" : "+v"(have[i][e]), "+v"(gone[i][e]));
  mine.left = wave_inclusive(mine.left), mine.all = wave_inclusive(mine.all);
  if (lane == 63) parts[wave] = mine;
  __syncthreads();
  Sum total{0.0, 0.0};
#pragma unroll
  for (int i = 0; i < WAVES; ++i) total.left += parts[i].left, total.all += parts[i].all;
  const bool rest = total.left > 0.0;
  const double share = uniform * (rest ? total.left : total.all);
  // the first wave whose running sum passes the share; the last that holds
  // anything where a share of the whole sum, or more, was asked for
  int at = -1;
  bool passed = false;
  double run = 0.0, carry = 0.0;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) {
    const double own = rest ? parts[i].left : parts[i].all;
    if (own > 0.0 && !passed) at = i, carry = run, passed = run + own > share;
    run += own;
  }
  if (wave != max(at, 0)) return;
  long token = -1;
  if (at >= 0) {
    passed = false;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      if (passed) continue;
      double values[8], mass = 0.0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const Sum w = weight_of(have[i][e], gone[i][e]);
        values[e] = rest ? w.left : w.all;
        mass += values[e];
      }
      const double through = carry + wave_inclusive(mass);
      double upto = through - mass;
      int first = -1, last = -1;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        upto += values[e];
        if (values[e] > 0.0) {
          last = e;
          if (first < 0 && upto > share) first = e;
        }
      }
      // rounding can leave the running sum of a wave just below its own sum: the
      // last value that holds anything, then
      const unsigned long long passes = __ballot(first >= 0), holds = __ballot(last >= 0);
      passed = passes != 0;
      if (passed) {
        const int l = __builtin_ctzll(passes);
        token = ((long)at * STEPS + i) * 512 + l * 8 + __builtin_amdgcn_readlane(first, l);
      } else if (holds != 0) {
        const int l = 63 - __builtin_clzll(holds);
        token = ((long)at * STEPS + i) * 512 + l * 8 + __builtin_amdgcn_readlane(last, l);
      }
      carry = __shfl(through, 63, 64);
    }
  }
  if (lane <= (int)p.drafts) p.out[b * (p.drafts + 1) + lane] = lane < kept ? drafted : lane == kept ? token : -1;
  if (lane == 0) {
    p.kept[b] = kept;
    if (p.lengths != nullptr) p.lengths[b] = length - (drafts_of(p, b) - kept);
  }
}

constexpr long kWhole = 16 * 512 * 4;  // values that a workgroup's registers hold

Pieces pieces_of(const shk_verify& a) {
  // one step each, more where a row has more steps than a workgroup threads
  const long steps = (a.vocab + kPiece - 1) / kPiece, each = (steps + kPieces - 1) / kPieces;
  return Pieces{(int)((steps + each - 1) / each), (int)(each * kPiece)};
}

template <int TYPE>
hipError_t launch(const shk_verify& a, hipStream_t s) {
  const dim3 one((unsigned)a.batch);
  if (a.vocab <= 4 * 512) hipLaunchKernelGGL((verify_whole<TYPE, 4, 1>), one, dim3(256), 0, s, a);
  else if (a.vocab <= 16 * 512) hipLaunchKernelGGL((verify_whole<TYPE, 16, 1>), one, dim3(1024), 0, s, a);
  else if (a.vocab <= 16 * 512 * 2) hipLaunchKernelGGL((verify_whole<TYPE, 16, 2>), one, dim3(1024), 0, s, a);
  else if (a.vocab <= kWhole) hipLaunchKernelGGL((verify_whole<TYPE, 16, 4>), one, dim3(1024), 0, s, a);
  if (a.vocab <= kWhole) return hipGetLastError();
  const Pieces pieces = pieces_of(a);
  hipLaunchKernelGGL((verify_sums<TYPE>), dim3(pieces.count, (unsigned)a.batch), dim3(kThreads), 0, s, a, pieces);
  if (hipError_t e = hipGetLastError()) return e;
  hipLaunchKernelGGL((verify_draw<TYPE>), dim3((unsigned)a.batch), dim3(kThreads), 0, s, a, pieces);
  return hipGetLastError();
}

}  // namespace

int64_t verify_workspace(const shk_verify& a) {
  if (a.vocab <= kWhole) return 0;
  return kept_bytes(a.batch) + a.batch * pieces_of(a).count * (int64_t)sizeof(Sum);
}

hipError_t launch_verify(const shk_verify& a, hipStream_t s) {
  if (a.type == SHK_SRC_F32) return launch<SHK_SRC_F32>(a, s);
  if (a.type == SHK_SRC_F16) return launch<SHK_SRC_F16>(a, s);
  return launch<SHK_SRC_BF16>(a, s);
}

}  // namespace shk
