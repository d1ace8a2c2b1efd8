// Drafted tokens against the target's probabilities: how many are kept, and the
// token that follows them, drawn from what the draft left of the target.
//
// The kept drafts are a handful of gathers, which a wave tests at once; every
// workgroup does so for itself.  The draw needs the sum of one row's weights
// before the place where the running sum passes its share u of it: the vocabulary
// is cut into pieces, verify_sums adds each piece, and verify_draw finds the
// piece and then the token in it.  Sums are 64 bits: over a vocabulary f32 would
// move the place by whole tokens, and the order of adding would show.
// Bound by the one row of each kind that a sequence reads, or by two launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "shk_common.h"
#include "shk_step.h"

namespace shk {
namespace {

constexpr int kThreads = 256;
constexpr int kPieces = 256;  // at most, of a row

struct Pieces {
  int count, size;  // size: values of a piece, whole 8s
};

struct Sum {
  double left, all;  // of max(target - draft, 0), of target
};

template <int TYPE>
__device__ __forceinline__ float value_of(const void* x, long i) {
  if constexpr (TYPE == SHK_SRC_F32) return static_cast<const float*>(x)[i];
  const uint16_t h = static_cast<const uint16_t*>(x)[i];
  return TYPE == SHK_SRC_BF16 ? bf16_bits_to_f32(h) : (float)__builtin_bit_cast(_Float16, h);
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

// Weights of value t; NaN and negative ones count as 0.
template <int TYPE>
__device__ __forceinline__ Sum weight_at(const shk_verify& p, const Row& r, long t) {
  Sum w;
  w.all = __builtin_fmax((double)value_of<TYPE>(p.target, r.target + t), 0.0);
  w.left = w.all;
  if (r.draft >= 0) w.left = __builtin_fmax(w.all - (double)value_of<TYPE>(p.draft, r.draft + t), 0.0);
  else if (t == r.certain) w.left = 0.0;
  return w;
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d, 64);
  return v;
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void verify_sums(const shk_verify p, const Pieces pieces) {
  __shared__ double parts[2][kThreads / 64];
  const long b = blockIdx.y;
  const Row r = row_of(p, b, kept_of<TYPE>(p, b));
  const long from = (long)blockIdx.x * pieces.size, to = min(from + pieces.size, (long)p.vocab);
  Sum mine{0.0, 0.0};
  for (long t = from + threadIdx.x; t < to; t += kThreads) {
    const Sum w = weight_at<TYPE>(p, r, t);
    mine.left += w.left, mine.all += w.all;
  }
  mine.left = wave_sum(mine.left), mine.all = wave_sum(mine.all);
  if ((threadIdx.x & 63) == 0) parts[0][threadIdx.x >> 6] = mine.left, parts[1][threadIdx.x >> 6] = mine.all;
  __syncthreads();
  if (threadIdx.x == 0) {
    Sum s{0.0, 0.0};
    for (int w = 0; w < kThreads / 64; ++w) s.left += parts[0][w], s.all += parts[1][w];
    static_cast<Sum*>(p.workspace)[b * pieces.count + blockIdx.x] = s;
  }
}

// Inclusive sum over the workgroup's threads.
__device__ __forceinline__ double group_inclusive(double v, double (&parts)[kThreads / 64]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const double o = __shfl_up(v, d, 64);
    if (lane >= d) v += o;
  }
  __syncthreads();
  if (lane == 63) parts[wave] = v;
  __syncthreads();
  double before = 0.0;
  for (int w = 0; w < wave; ++w) before += parts[w];
  return before + v;
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void verify_draw(const shk_verify p, const Pieces pieces) {
  __shared__ double parts[kThreads / 64], before_piece, total_all;
  __shared__ int piece, passes, holds;
  const long b = blockIdx.x;
  const int kept = kept_of<TYPE>(p, b);
  const Row r = row_of(p, b, kept);
  const Sum* sums = static_cast<const Sum*>(p.workspace) + b * pieces.count;
  const Sum mine = (int)threadIdx.x < pieces.count ? sums[threadIdx.x] : Sum{0.0, 0.0};
  const double left = group_inclusive(mine.left, parts), all = group_inclusive(mine.all, parts);
  if (threadIdx.x == 0) piece = passes = kThreads, holds = -1;
  if (threadIdx.x == kThreads - 1) before_piece = left, total_all = all;
  __syncthreads();
  const bool rest = before_piece > 0.0;
  const double total = rest ? before_piece : total_all, upto = rest ? left : all, own = rest ? mine.left : mine.all;
  const double share = (double)p.uniforms[b * (p.drafts + 1) + p.drafts] * total;
  __syncthreads();
  // the first piece whose running sum passes the share; the last that holds
  // anything where a share of the whole sum, or more, was asked for
  if (own > 0.0) {
    if (upto > share) atomicMin(&piece, (int)threadIdx.x);
    atomicMax(&holds, (int)threadIdx.x);
  }
  __syncthreads();
  const int at = piece < kThreads ? piece : holds;
  if ((int)threadIdx.x == at) before_piece = upto - own;
  __syncthreads();
  long token = -1;
  if (at >= 0) {
    double run = before_piece;
    const long from = (long)at * pieces.size, to = min(from + pieces.size, (long)p.vocab);
    int best = -1, most = -1;  // offsets in the piece
    for (long base = from; base < to && best < 0; base += kThreads) {
      const long t = base + threadIdx.x;
      double w = 0.0;
      if (t < to) {
        const Sum s = weight_at<TYPE>(p, r, t);
        w = rest ? s.left : s.all;
      }
      const double sum = run + group_inclusive(w, parts);
      if (threadIdx.x == 0) passes = kThreads, holds = -1;
      __syncthreads();
      if (w > 0.0) {
        if (sum > share) atomicMin(&passes, (int)threadIdx.x);
        atomicMax(&holds, (int)threadIdx.x);
      }
      if (threadIdx.x == kThreads - 1) before_piece = sum;
      __syncthreads();
      if (passes < kThreads) best = (int)(base - from) + passes;
      if (holds >= 0) most = (int)(base - from) + holds;
      run = before_piece;
      __syncthreads();
    }
    // rounding can leave the running sum of a piece just below its own sum
    token = from + (best >= 0 ? best : most);
  }
  for (int i = threadIdx.x; i <= (int)p.drafts; i += kThreads)
    p.out[b * (p.drafts + 1) + i] = i < kept ? token_of(p, b * p.drafts + i) : i == kept ? token : -1;
  if (threadIdx.x == 0) {
    p.kept[b] = kept;
    if (p.lengths != nullptr) p.lengths[b] -= drafts_of(p, b) - kept;
  }
}

Pieces pieces_of(const shk_verify& a) {
  // enough workgroups for the chip, pieces of at least 2048 values
  const long want = std::min<long>(kPieces, std::max<long>(1, 1024 / std::max<int64_t>(1, a.batch)));
  long size = std::max<long>(2048, ((a.vocab + want - 1) / want + 7) / 8 * 8);
  return Pieces{(int)((a.vocab + size - 1) / size), (int)size};
}

template <int TYPE>
hipError_t launch(const shk_verify& a, hipStream_t s) {
  const Pieces pieces = pieces_of(a);
  hipLaunchKernelGGL((verify_sums<TYPE>), dim3(pieces.count, (unsigned)a.batch), dim3(kThreads), 0, s, a, pieces);
  if (hipError_t e = hipGetLastError()) return e;
  hipLaunchKernelGGL((verify_draw<TYPE>), dim3((unsigned)a.batch), dim3(kThreads), 0, s, a, pieces);
  return hipGetLastError();
}

}  // namespace

int64_t verify_workspace(const shk_verify& a) { return a.batch * pieces_of(a).count * (int64_t)sizeof(Sum); }

hipError_t launch_verify(const shk_verify& a, hipStream_t s) {
  if (a.type == SHK_SRC_F32) return launch<SHK_SRC_F32>(a, s);
  if (a.type == SHK_SRC_F16) return launch<SHK_SRC_F16>(a, s);
  return launch<SHK_SRC_BF16>(a, s);
}

}  // namespace shk
