// 8-bit floating-point products on tiles of 256 x 256: the matrix unit kept fed.
//
// A stage is one block of K (128): 256 rows of each operand, 64 KiB, in one of two
// LDS slots, and their scales, in one of three.  Eight waves hold 128 x 64 of the
// tile each: per stage 32 MFMAs (32 cycles of a SIMD each), whose results are folded
// into the f32 sums with four multiply-adds (16 cycles) while the next ones run: the
// sums have to lie where the vector unit reaches them, and 128 of them with both
// operands' fragments fill a wave's 256 registers.
//
// The order of a stage is fixed step by step (one MFMA, the fold of the one
// before the last, now and then an LDS read two row tiles ahead), with scheduling
// barriers between: left to itself the compiler hoists the reads and spills.
// Three quarters through, when the last fragment of the stage is in registers,
// the waves meet: behind that barrier the next stage is complete (its copy was
// issued a whole stage ago), so its first fragments are read under the last
// MFMAs, and this stage's rows are all in registers: their slot is free.  The copies
// of the stage after next are spread over the following steps; in one burst they
// cost 500 cycles a stage.  Scales of b's rows are read by the folds, behind that
// barrier too, and those of the stage after next are copied before the next one, so
// that a wave may still read the ones while another's copy brings the others: they
// have three slots, and the barrier between a slot's last reads and its next copy is
// the following stage's.
//
// Bound by power, then by the matrix unit: at 8192^3 a stage takes 2600 cycles
// (2048 of MFMAs) at 1.6 GHz; with operands of one value it runs at 2.3 GHz.
// 8192^3 428 to 449 us (2500 TFLOP/s), 573 to 589 where each row of b has its own
// scales; 4096 x 11008 x 4096 160 to 179, 221 with those (three rounds of workgroups
// for 2.7 of work).
// Measured and dropped: fragments of b straight from memory (the 16 rows of a
// load cost the vector memory path 5600 cycles a stage), folds grouped by row.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "shk_fp8product.h"

namespace shk {
namespace {

typedef __attribute__((address_space(3))) const v4i lds_v4i;
typedef __attribute__((address_space(3))) const v4f lds_v4f;
typedef __attribute__((address_space(3))) const float lds_float;

constexpr int kB = 256 * 128;            // where b lies in a stage
constexpr int kStage = 512 * 128;
constexpr int kScales = 2 * kStage;      // behind both slots of rows
constexpr int kScaleSlots = 3, kScaleSlot = 2048;  // 256 of a's, 256 of b's
constexpr int kRead = 23;                // the step behind which a stage's barrier is
constexpr int kCopyScales = 8;           // the step that copies the next stage's scales

// What is behind K in the last stage is whatever follows the rows: zeros instead,
// `left` of 128 values stay.
__device__ __forceinline__ void clear_tail(uint8_t* st, int left) {
  for (int u = threadIdx.x; u < 512 * 8; u += 512) {
    const int row = u >> 3, unit = (u & 7) ^ (row & 7), keep = left - unit * 16;
    if (keep >= 16) continue;
    uint32_t* w = reinterpret_cast<uint32_t*>(st + u * 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int bytes = keep - 4 * e;
      w[e] = bytes <= 0 ? 0u : bytes >= 4 ? w[e] : w[e] & ((1u << (8 * bytes)) - 1u);
    }
  }
}

template <int KIND_A, int KIND_B, bool BROW>
__global__ __launch_bounds__(512) void fp8_big_kernel(const Fp8Product p) {
  __shared__ __align__(16) uint8_t lds[kScales + kScaleSlots * kScaleSlot];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int tm, tn;
  tile_of(p, 4, tm, tn);
  const int m0 = tm * 256, n0 = tn * 256, rows_a = min(256, p.m - m0), rows_b = min(256, p.n - n0);
  // whole blocks; a last one that K ends in comes behind the loop
  const int blocks = (p.k + 127) >> 7, count = p.k >> 7, left = p.k & 127;
  const long row_bytes = (p.k + 15) & ~15;

  // waves 0 to 3 bring a and its scales, 4 to 7 b and its
  const bool of_a = wave < 4;
  const long pitch = of_a ? p.a_pitch : p.b_pitch;
  const int s0 = n0 >> p.b_shift, s_rows = ((n0 + rows_b - 1) >> p.b_shift) - s0 + 1;
  // rows behind the operand's end lie behind the resource's, and come as zeros
  const v4i rows = buffer_words(of_a ? p.a + m0 * pitch : p.b + n0 * pitch,
                                (unsigned long long)(((of_a ? rows_a : rows_b) - 1) * pitch + row_bytes));
  const v4i scales =
      of_a ? buffer_words(p.sa + (long)m0 * p.sa_row, (unsigned long long)(((rows_a - 1) * p.sa_row + (blocks - 1) * p.sa_block + 1) * 4))
           : buffer_words(p.sb + (long)s0 * p.sb_row, (unsigned long long)(((s_rows - 1) * p.sb_row + (blocks - 1) * p.sb_block + 1) * 4));
  const int s_row = (wave & 3) * 64 + lane;
  const uint32_t s_off = of_a ? (uint32_t)(s_row * p.sa_row * 4) : (uint32_t)((((n0 + s_row) >> p.b_shift) - s0) * p.sb_row * 4);
  const uint32_t s_step = (uint32_t)((of_a ? p.sa_block : p.sb_block) * 4);
  // a piece is 8 rows; unit u of row r lies at r * 128 + 16 * (u ^ (r % 8))
  const uint32_t off = (uint32_t)(((wave & 3) * 64 + lane / 8) * pitch) + 16 * ((lane & 7) ^ (lane / 8));
  const uint32_t step8 = (uint32_t)(8 * pitch), base = lds_address(lds);
  const uint32_t to = base + (of_a ? 0 : kB) + (wave & 3) * 8192, s_to = base + kScales + wave * 256;
  auto piece = [&](int kb, int slot, int c) {  // 8 of a wave's rows
    lds_dma16(rows, off, (uint32_t)kb * 128u + c * step8, to + slot * kStage + c * 1024);
  };
  auto piece_scales = [&](int kb, uint32_t at) { lds_dma4(scales, s_off, (uint32_t)kb * s_step, s_to + at); };

  const int wm = wave & 1, wn = wave >> 1, row_in = lane & 15, group = lane >> 4;
  v4f acc[8][4];
#pragma unroll
  for (int x = 0; x < 8; ++x)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[x][j] = v4f{0.f, 0.f, 0.f, 0.f};
  // a lane's fragment: units group and group + 4 of its row; the addresses of the
  // stage that is read are moved in place, so that every offset fits an instruction
  const uint32_t frag = base + row_in * 128 + 16 * (group ^ (row_in & 7));
  uint32_t a_lo = frag + wm * 16384, a_hi = (frag ^ 64) + wm * 16384;
  uint32_t b_lo = frag + kB + wn * 8192, b_hi = (frag ^ 64) + kB + wn * 8192;
  uint32_t sa_at = base + kScales + (wm * 128 + row_in) * 4;
  uint32_t sb_at = base + kScales + 1024 + (wn * 64 + (BROW ? group * 4 : 0)) * 4;
  auto fragment = [&](uint32_t lo, uint32_t hi, int at) {
    return __builtin_shufflevector(*(lds_v4i*)(uintptr_t)(lo + at), *(lds_v4i*)(uintptr_t)(hi + at), 0, 1, 2, 3, 4, 5, 6, 7);
  };
  auto scale = [&](uint32_t at, int off) { return *(lds_float*)(uintptr_t)(at + off); };

#pragma unroll
  for (int c = 0; c < 8; ++c) piece(0, 0, c);
  piece_scales(0, 0);
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  asm volatile("s_barrier" ::: "memory");
#pragma unroll
  for (int c = 0; c < 4; ++c) piece(max(min(1, count - 1), 0), 1, c);
  v8i fb[2][4], fa[2];
  float sa[2] = {scale(sa_at, 0), scale(sa_at, 64)}, sb = BROW ? 0.f : scale(sb_at, 0);
#pragma unroll
  for (int j = 0; j < 4; ++j) fb[0][j] = fragment(b_lo, b_hi, j * 2048);
  fa[0] = fragment(a_lo, a_hi, 0), fa[1] = fragment(a_lo, a_hi, 2048);
  uint32_t s_at = 0;  // the slot of the stage's scales

  auto stage = [&](int i, auto slot_of, v8i (&now)[4], v8i (&next)[4]) {
    constexpr int slot = decltype(slot_of)::value, turn = slot ? -kStage : kStage;
    const int soon = min(i + 1, count - 1), later = min(i + 2, count - 1);
    const uint32_t s_next = s_at == (kScaleSlots - 1) * kScaleSlot ? 0 : s_at + kScaleSlot, s_turn = s_next - s_at;
    v4f t[3], row_scales;
    float s_now = 0.f, s_old = 0.f, sb_next = 0.f;
    v8i f[10] = {fa[0], fa[1]};  // this stage's eight row tiles, the next one's first two
    float q[10] = {sa[0], sa[1]};
#pragma unroll
    for (int step = 0; step < 34; ++step) {
      const int x = step >> 2, j = step & 3;
      if (step < 32) {
        if (j == 0) {
          s_old = s_now;
          s_now = BROW ? q[x] : q[x] * sb;
          if (x < 6) f[x + 2] = fragment(a_lo, a_hi, (x + 2) * 2048), q[x + 2] = scale(sa_at, (x + 2) * 64);
          else f[x + 2] = fragment(a_lo, a_hi, (x - 6) * 2048), q[x + 2] = scale(sa_at, (x - 6) * 64);
          if (!BROW && x == 6) sb_next = scale(sb_at, 0);
        }
        if (x == 6) next[j] = fragment(b_lo, b_hi, j * 2048);
        t[step % 3] = mfma128<KIND_A, KIND_B>(now[j], f[x]);
        if (step >= 24 && step % 2 == 0) piece(later, slot, (step - 24) / 2);
        if (step < 8 && step % 2 == 0) piece(soon, slot ^ 1, 4 + step / 2);
        if (step == kCopyScales) piece_scales(soon, s_next);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (step >= 2) {
        const int fx = (step - 2) >> 2, fj = (step - 2) & 3;
        const float s = fx == x || step >= 32 ? s_now : s_old;
        if constexpr (BROW) row_scales = *(lds_v4f*)(uintptr_t)(sb_at + fj * 64);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          acc[fx][fj][r] = __builtin_fmaf(t[(step - 2) % 3][r], BROW ? s * row_scales[r] : s, acc[fx][fj][r]);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (step == kRead) {
        __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
        asm volatile("s_barrier" ::: "memory");
        a_lo += turn, a_hi += turn, b_lo += turn, b_hi += turn, sa_at += s_turn;
        if constexpr (!BROW) sb_at += s_turn;
        asm volatile("" : "+v"(a_lo), "+v"(a_hi), "+v"(b_lo), "+v"(b_hi), "+v"(sa_at), "+v"(sb_at));
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if constexpr (BROW) {
      sb_at += s_turn;
      asm volatile("" : "+v"(sb_at));
    }
    s_at = s_next;
    fa[0] = f[8], fa[1] = f[9], sa[0] = q[8], sa[1] = q[9], sb = sb_next;
  };
  int i = 0;
  for (; i + 1 < count; i += 2) {
    stage(i, std::integral_constant<int, 0>{}, fb[0], fb[1]);
    stage(i + 1, std::integral_constant<int, 1>{}, fb[1], fb[0]);
  }
  if (i < count) stage(i, std::integral_constant<int, 0>{}, fb[0], fb[1]);

  // the copies behind the last stage, and every wave's reads
  __builtin_amdgcn_s_waitcnt(0x0070);
  asm volatile("s_barrier" ::: "memory");
  if (left != 0) {
#pragma unroll
    for (int c = 0; c < 8; ++c) piece(count, 0, c);
    piece_scales(count, 0);
    __builtin_amdgcn_s_waitcnt(0x0F70);
    asm volatile("s_barrier" ::: "memory");
    clear_tail(lds, left);
    __syncthreads();
    const uint32_t a_row = base + wm * 16384 + row_in * 128, b_row = base + kB + wn * 8192 + row_in * 128;
    const uint32_t lo = 16 * (group ^ (row_in & 7)), sa_row = base + kScales + (wm * 128 + row_in) * 4;
    const uint32_t sb_row = base + kScales + 1024 + (wn * 64 + (BROW ? group * 4 : 0)) * 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const v8i b = fragment(b_row + lo, b_row + (lo ^ 64), j * 2048);
      v4f sv;
      if constexpr (BROW) sv = *(lds_v4f*)(uintptr_t)(sb_row + j * 64);
      else sv[0] = scale(sb_row, 0);
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const v4f t = mfma128<KIND_A, KIND_B>(b, fragment(a_row + lo, a_row + (lo ^ 64), x * 2048));
        const float s = scale(sa_row, x * 64);
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[x][j][r] = __builtin_fmaf(t[r], s * sv[BROW ? r : 0], acc[x][j][r]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __syncthreads();
  }
  // results through LDS for rows of 128 bytes: a wave's 128 x 64, unit u of row r
  // at r * 128 + 16 * (u ^ (r % 8))
  uint8_t* mine = lds + wave * 16384;
  const bool bf16 = p.out_type == SHK_SRC_BF16;
#pragma unroll
  for (int x = 0; x < 8; ++x)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = x * 16 + row_in, u = j * 2 + (group >> 1);
      const v4f v = acc[x][j];
      uint2 w;
      if (bf16) {
        w = make_uint2(pack_bf16x2_nonan(v[0], v[1]), pack_bf16x2_nonan(v[2], v[3]));
      } else {
        w.x = __builtin_bit_cast(uint16_t, (_Float16)v[0]) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[1]) << 16);
        w.y = __builtin_bit_cast(uint16_t, (_Float16)v[2]) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[3]) << 16);
      }
      *reinterpret_cast<uint2*>(mine + r * 128 + 16 * (u ^ (r & 7)) + (group & 1) * 8) = w;
    }
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const int r = k * 8 + lane / 8, u = lane & 7, m = m0 + wm * 128 + r, n = n0 + wn * 64 + u * 8;
    const u4 v = *reinterpret_cast<const u4*>(mine + r * 128 + 16 * (u ^ (r & 7)));
    if (m >= p.m) continue;
    uint16_t* at = static_cast<uint16_t*>(p.out) + (long)m * p.out_stride + n;
    if (n + 8 <= p.n) {
      *reinterpret_cast<any_u4*>(at) = v;  // of any alignment, as store_four's
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (n + e < p.n) at[e] = (uint16_t)(v[e / 2] >> (16 * (e % 2)));
    }
  }
}

template <int KIND_A, int KIND_B>
hipError_t launch(Fp8Product& p, hipStream_t s) {
  const dim3 grid(p.tiles_m * p.tiles_n);
  if (p.b_shift == 0) hipLaunchKernelGGL((fp8_big_kernel<KIND_A, KIND_B, true>), grid, dim3(512), 0, s, p);
  else hipLaunchKernelGGL((fp8_big_kernel<KIND_A, KIND_B, false>), grid, dim3(512), 0, s, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_fp8_big(Fp8Product& p, bool e5_a, bool e5_b, hipStream_t s) {
  p.tiles_m = (p.m + 255) / 256, p.tiles_n = (p.n + 255) / 256;
  if (e5_a) return e5_b ? launch<1, 1>(p, s) : launch<1, 0>(p, s);
  return e5_b ? launch<0, 1>(p, s) : launch<0, 0>(p, s);
}

}  // namespace shk
