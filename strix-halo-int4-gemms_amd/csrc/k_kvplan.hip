// Pages of a step: from the lengths of a batch's sequences and their numbers of
// new tokens, which pages each gets, and slot and position of every token.
//
// Three prefix sums over the batch (tokens, pages that come back, pages asked
// for) fit a workgroup's LDS, so every workgroup makes them for itself from a few
// KB in L2 and then numbers its share of the tokens; a token finds its sequence
// by a binary search.  Nobody changes the pool meanwhile: each workgroup takes a
// ticket when it has read what it needs, and the last one writes the new state.
// Bound by latency: one launch, the sums, a search, two dependent reads.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>

#include "shk_step.h"

namespace shk {
namespace {

constexpr int kThreads = 512;
constexpr int kEach = kPlanBatch / kThreads;  // sequences of a thread
constexpr long kManyTokens = 1L << 40;        // more than any capacity, far from overflow

struct Sums {
  int start[kPlanBatch + 1];  // first token of a sequence
  int back[kPlanBatch + 1];   // first page that it gives back
  int ask[kPlanBatch + 1];    // first page that it asks for
};

// The last i of [0, n) with first[i] <= x, n > 0 and first[0] <= x.
__device__ __forceinline__ int find(const int* first, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (first[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ long wave_inclusive(long v, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const long o = __shfl_up(v, d, 64);
    if (lane >= d) v += o;
  }
  return v;
}

struct Sequence {
  int length, owned, fresh;  // before the step; fresh: new tokens, negative if it ended
};

__device__ __forceinline__ Sequence sequence(const shk_kv_plan& p, int b) {
  Sequence s;
  s.length = max(p.lengths[b], 0);
  s.owned = min(max(p.owned[b], 0), (int)p.width);
  s.fresh = p.new_tokens[b];
  return s;
}

// Pages that the sequence would hold; past the table's width it holds none more.
__device__ __forceinline__ long pages_of(const Sequence& s, int shift) {
  return ((long)s.length + s.fresh + (1L << shift) - 1) >> shift;
}

__global__ __launch_bounds__(kThreads) void kv_plan_kernel(const shk_kv_plan p, int shift) {
  extern __shared__ uint8_t lds[];
  Sums& sums = *reinterpret_cast<Sums*>(lds);
  __shared__ long carry[3][kThreads / 64];
  __shared__ int last;
  const int batch = (int)p.batch, width = (int)p.width, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int had = min(max(*p.free_count, 0), (int)p.free_total);

  const int first = threadIdx.x * kEach;
  Sequence mine[kEach];
  long own[3] = {0, 0, 0};
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    mine[i] = Sequence{0, 0, 0};
    if (first + i < batch) mine[i] = sequence(p, first + i);
    if (mine[i].fresh < 0) own[1] += mine[i].owned;
    else own[0] += mine[i].fresh;
  }
  long upto[3];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    upto[k] = wave_inclusive(own[k], lane);
    if (lane == 63) carry[k][wave] = upto[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    upto[k] -= own[k];
    for (int w = 0; w < wave; ++w) upto[k] += carry[k][w];
  }
  // a sequence past the table or the capacity asks for nothing
  long at = upto[0], asks[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    asks[i] = 0;
    if (first + i >= batch || mine[i].fresh < 0) continue;
    at += mine[i].fresh;
    const long pages = pages_of(mine[i], shift);
    if (pages <= width && at <= p.capacity) asks[i] = max(pages - mine[i].owned, 0L);
    own[2] += asks[i];
  }
  upto[2] = wave_inclusive(own[2], lane);
  if (lane == 63) carry[2][wave] = upto[2];
  __syncthreads();
  upto[2] -= own[2];
  for (int w = 0; w < wave; ++w) upto[2] += carry[2][w];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int b = first + i;
    if (b > batch) break;
    sums.start[b] = (int)min(upto[0], (long)INT_MAX);
    sums.back[b] = (int)min(upto[1], (long)INT_MAX);
    sums.ask[b] = (int)min(upto[2], (long)INT_MAX);
    if (mine[i].fresh < 0) upto[1] += mine[i].owned;
    else upto[0] += mine[i].fresh;
    upto[2] += asks[i];
  }
  if (threadIdx.x == kThreads - 1 && batch == kPlanBatch) {
    sums.start[batch] = (int)min(upto[0], (long)INT_MAX);
    sums.back[batch] = (int)min(upto[1], (long)INT_MAX);
    sums.ask[batch] = (int)min(upto[2], (long)INT_MAX);
  }
  __syncthreads();
  const int back = min(sums.back[batch], (int)p.free_total - had);  // what the stack has places for
  const int top = had + back;

  // page j of those that are asked for: from the top of the stack, where the
  // pages that come back are
  auto popped = [&](int j) {
    const int place = top - 1 - j;
    if (place < had) return p.free_pages[place];
    const int s = find(sums.back, batch, place - had);
    return p.page_table[(long)s * width + (place - had - sums.back[s])];
  };
  // whether sequence b got what it asked for (its new tokens have places)
  auto fits = [&](int b, const Sequence& s) {
    return s.fresh >= 0 && pages_of(s, shift) <= width && sums.start[b] + (long)s.fresh <= p.capacity &&
           (sums.ask[b + 1] == sums.ask[b] || sums.ask[b + 1] <= top);
  };

  const int total = sums.start[batch];
  for (long i = blockIdx.x * (long)kThreads + threadIdx.x; i < p.capacity; i += (long)gridDim.x * kThreads) {
    int b = -1, position = 0;
    long slot = -1;
    if (i < total) {
      b = find(sums.start, batch, (int)i);
      const Sequence s = sequence(p, b);
      position = s.length + (int)i - sums.start[b];
      if (fits(b, s)) {
        const int column = position >> shift;
        const int page = column < s.owned ? p.page_table[(long)b * width + column]
                                          : popped(sums.ask[b] + column - s.owned);
        slot = ((long)page << shift) + (position & ((1 << shift) - 1));
      }
    }
    p.slots[i] = slot;
    p.positions[i] = position;
    p.sequences[i] = b;
  }

  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(p.ticket, 1) == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  // asks that fit are the first ones; each finds its sequence and column
  int got = 0;
  {
    int lo = 0, hi = batch;  // the most sequences whose asks all fit
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (sums.ask[mid] <= top) lo = mid;
      else hi = mid - 1;
    }
    got = sums.ask[lo];
  }
  for (int j = threadIdx.x; j < got; j += kThreads) {
    const int b = find(sums.ask, batch, j);
    const Sequence s = sequence(p, b);
    p.page_table[(long)b * width + s.owned + (j - sums.ask[b])] = popped(j);
  }
  for (int r = threadIdx.x; r < back; r += kThreads) {
    const int s = find(sums.back, batch, r);
    p.free_pages[had + r] = p.page_table[(long)s * width + (r - sums.back[s])];
  }
  __syncthreads();  // the pool's old state was read
  for (int b = threadIdx.x; b <= batch; b += kThreads) {
    p.starts[b] = sums.start[b];
    if (b == batch) break;
    const Sequence s = sequence(p, b);
    const bool in = fits(b, s);
    p.taken[b] = in ? s.fresh : 0;
    p.lengths[b] = s.fresh < 0 ? 0 : in ? s.length + s.fresh : s.length;
    p.owned[b] = s.fresh < 0 ? 0 : s.owned + (in ? sums.ask[b + 1] - sums.ask[b] : 0);
  }
  if (threadIdx.x == 0) {
    *p.free_count = top - got;
    *p.ticket = 0;
  }
}

}  // namespace

hipError_t launch_kv_plan(const shk_kv_plan& a, hipStream_t s) {
  // a workgroup for each 2048 tokens, at most one for each CU
  const long groups = std::min(256L, std::max(1L, (long)((a.capacity + 2047) / 2048)));
  hipLaunchKernelGGL(kv_plan_kernel, dim3((unsigned)groups), dim3(kThreads), sizeof(Sums), s, a,
                     __builtin_ctzl((unsigned long)a.page_size));
  return hipGetLastError();
}

}  // namespace shk
