// Pages of a step: from the lengths of a batch's sequences and their numbers of
// new tokens, which pages each gets, and slot and position of every token.
//
// Three prefix sums over the batch (tokens, pages that come back, pages asked
// for) fit a workgroup's LDS with the sequences themselves, so every workgroup
// makes them for itself from a few KB in L2 and then numbers its share of the
// tokens; a token finds its sequence by a binary search.  What is written on the
// way is what nobody reads in this step: fresh columns of the table (by the first
// token of each page, or for a sequence without tokens by a thread of its own) and
// the stack above its old top.  Lengths, owned pages and
// the stack's height change when every workgroup has taken a ticket, by the last.
// Bound by latency: one launch, the sums, a search, two dependent reads.  64
// sequences 5.5 us, 500 with 150000 tokens 9 (12.7 with a fence at the ticket).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>

#include "shk_lanes.h"
#include "shk_step.h"

namespace shk {
namespace {

constexpr int kThreads = 512;

template <int MOST>  // sequences
struct Batch {
  int start[MOST + 1];  // first token of a sequence
  int back[MOST + 1];   // first page that it gives back
  int ask[MOST + 1];    // first page that it asks for
  int length[MOST], owned[MOST];  // before the step, 0 where it ends
  int fresh[MOST];                // new tokens, negative where it ends
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

__device__ __forceinline__ int saturated(long v) { return (int)min(v, (long)INT_MAX); }

template <int MOST>
__global__ __launch_bounds__(kThreads) void kv_plan_kernel(const shk_kv_plan p, int shift) {
  constexpr int EACH = MOST / kThreads;  // sequences of a thread
  __shared__ Batch<MOST> s;
  __shared__ long carry[3][kThreads / 64];
  __shared__ int last;
  const int batch = (int)p.batch, width = (int)p.width, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int had = min(max(*p.free_count, 0), (int)p.free_total);

  const int first = threadIdx.x * EACH;
  int length[EACH], owned[EACH], fresh[EACH];
  long own[3] = {0, 0, 0};
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    length[i] = owned[i] = fresh[i] = 0;
    if (first + i < batch) {
      fresh[i] = p.new_tokens[first + i];
      length[i] = max(p.lengths[first + i], 0);
      owned[i] = min(max(p.owned[first + i], 0), width);
    }
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    if (fresh[i] < 0) own[1] += owned[i];
    else own[0] += fresh[i];
  }
  long upto[3] = {wave_inclusive(own[0]), wave_inclusive(own[1]), 0};
  if (lane == 63) carry[0][wave] = upto[0], carry[1][wave] = upto[1];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    upto[k] -= own[k];
    for (int w = 0; w < wave; ++w) upto[k] += carry[k][w];
  }
  // a sequence past the table or the capacity asks for nothing
  long at = upto[0], asks[EACH];
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    asks[i] = 0;
    if (first + i >= batch || fresh[i] < 0) continue;
    at += fresh[i];
    const long pages = ((long)length[i] + fresh[i] + (1L << shift) - 1) >> shift;
    if (pages <= width && at <= p.capacity) asks[i] = max(pages - owned[i], 0L);
    own[2] += asks[i];
  }
  upto[2] = wave_inclusive(own[2]);
  if (lane == 63) carry[2][wave] = upto[2];
  __syncthreads();
  upto[2] -= own[2];
  for (int w = 0; w < wave; ++w) upto[2] += carry[2][w];
#pragma unroll
  for (int i = 0; i <= EACH; ++i) {
    const int b = first + i;
    if (b > batch || (i == EACH && b != batch)) break;
    s.start[b] = saturated(upto[0]), s.back[b] = saturated(upto[1]), s.ask[b] = saturated(upto[2]);
    if (i == EACH || b == batch) break;
    s.length[b] = length[i], s.owned[b] = owned[i], s.fresh[b] = fresh[i];
    if (fresh[i] < 0) upto[1] += owned[i];
    else upto[0] += fresh[i];
    upto[2] += asks[i];
  }
  __syncthreads();
  const int total = s.start[batch];
  const int back = min(s.back[batch], (int)p.free_total - had);  // what the stack has places for
  const int top = had + back;

  // page r of those that come back
  auto returned = [&](int r) {
    const int b = find(s.back, batch, r);
    return p.page_table[(long)b * width + (r - s.back[b])];
  };
  // page j of those that are asked for: from the top of the stack, where the
  // pages that come back are
  auto popped = [&](int j) {
    const int place = top - 1 - j;
    return place < had ? p.free_pages[place] : returned(place - had);
  };
  // whether the new tokens of a sequence have places; sums of pages that saturated
  // are larger than any stack, and say nothing of what one sequence asks for
  auto fits = [&](int b) {
    const long pages = ((long)s.length[b] + s.fresh[b] + (1L << shift) - 1) >> shift;
    return s.fresh[b] >= 0 && pages <= width && s.start[b] + (long)s.fresh[b] <= p.capacity &&
           (pages <= s.owned[b] || s.ask[b + 1] <= top);
  };

  const long mine = blockIdx.x * (long)kThreads + threadIdx.x, all = (long)gridDim.x * kThreads;
  for (long i = mine; i < p.capacity; i += all) {
    int b = -1, position = 0;
    long slot = -1;
    if (i < total) {
      b = find(s.start, batch, (int)i);
      position = s.length[b] + (int)i - s.start[b];
      if (fits(b)) {
        const int column = position >> shift, held = s.owned[b];
        int* const row = p.page_table + (long)b * width;
        int page;
        if (column < held) {
          page = row[column];
        } else {
          page = popped(s.ask[b] + column - held);
          // the first token of a page enters it; a sequence's first token also
          // pages below it, which a pool that owns what it holds does not lack
          if ((position & ((1 << shift) - 1)) == 0 || i == s.start[b]) row[column] = page;
          if (i == s.start[b])
            for (int c = held; c < column; ++c) row[c] = popped(s.ask[b] + c - held);
        }
        slot = ((long)page << shift) + (position & ((1 << shift) - 1));
      }
    }
    p.slots[i] = slot;
    p.positions[i] = position;
    p.sequences[i] = b;
  }
  // pages of a sequence without new tokens, whose length a caller set past what it
  // owns
  for (long b = mine; b < batch; b += all)
    if (s.fresh[b] == 0 && s.ask[b + 1] > s.ask[b] && fits((int)b))
      for (int j = s.ask[b]; j < s.ask[b + 1]; ++j) p.page_table[b * width + s.owned[b] + j - s.ask[b]] = popped(j);
  for (long r = mine; r < back; r += all) p.free_pages[had + r] = returned((int)r);

  if (gridDim.x > 1) {
    // The ticket says that this workgroup has read what the last one will change: its
    // loads are back.  Nothing that it wrote is read by another, so nothing need be
    // made visible (a fence writes the L2's lines back).
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0)
      last = __hip_atomic_fetch_add(p.ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
    __syncthreads();
    if (!last) return;
  }
  for (int b = threadIdx.x; b <= batch; b += kThreads) {
    p.starts[b] = s.start[b];
    if (b == batch) break;
    const bool in = fits(b);
    p.taken[b] = in ? s.fresh[b] : 0;
    p.lengths[b] = s.fresh[b] < 0 ? 0 : in ? s.length[b] + s.fresh[b] : s.length[b];
    p.owned[b] = s.fresh[b] < 0 ? 0 : s.owned[b] + (in ? s.ask[b + 1] - s.ask[b] : 0);
  }
  if (threadIdx.x == 0) {
    int lo = 0, hi = batch;  // the most sequences whose asks all fit
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (s.ask[mid] <= top) lo = mid;
      else hi = mid - 1;
    }
    *p.free_count = top - s.ask[lo];
    if (gridDim.x > 1) *p.ticket = 0;
  }
}

}  // namespace

hipError_t launch_kv_plan(const shk_kv_plan& a, hipStream_t s) {
  // two tokens a thread, at most a workgroup for each CU
  const long groups = std::min(256L, std::max(1L, (long)((a.capacity + 2 * kThreads - 1) / (2 * kThreads))));
  const int shift = __builtin_ctzl((unsigned long)a.page_size);
  // 512 sequences are one a thread
  if (a.batch <= kThreads)
    hipLaunchKernelGGL((kv_plan_kernel<kThreads>), dim3((unsigned)groups), dim3(kThreads), 0, s, a, shift);
  else
    hipLaunchKernelGGL((kv_plan_kernel<kPlanBatch>), dim3((unsigned)groups), dim3(kThreads), 0, s, a, shift);
  return hipGetLastError();
}

}  // namespace shk
