// Products of two operands that both lie along the summed dimension, C[m, n] = sum_k A[m, k] B[n, k], on the matrix instructions: 8-bit
// integers (16x16x64, 32-bit integer sums) and float16 / bfloat16 (16x16x32, float32 sums).  Both read 16 bytes a lane and 64 bytes a row and
// step, so the code sees bytes.
//
// A workgroup of four waves, one on each SIMD, owns BM x BN of C.  Steps of 64 bytes of every row of its operands go straight from memory to
// LDS (no registers in between) into a ring of S slots; S - 1 are in flight or waiting.  A wave keeps the operands of the step that it multiplies
// in registers and reads the next step's between the matrix instructions.  16-byte pieces of a row are placed by an exclusive-or with
// the row's number, which spreads the sixteen rows that a read touches over all banks.
//
// Rows start on 16-byte boundaries and hold whole 16-byte pieces (zeros behind the last value).  Rows beyond the operand repeat its last one (their
// results are not stored), pieces beyond the last come back as zeros from the buffer's range check.
#pragma once

#include "wide_common.h"

namespace nf {

typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef __bf16 b8_t __attribute__((ext_vector_type(8)));

struct I8 {};

template <typename EL>
struct Mma;
template <>
struct Mma<I8> {
  typedef i32x4_t acc_t;
  __device__ static __forceinline__ acc_t run(i32x4_t a, i32x4_t b, acc_t c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
};
template <>
struct Mma<F16> {
  typedef f32x4_t acc_t;
  __device__ static __forceinline__ acc_t run(i32x4_t a, i32x4_t b, acc_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
  }
};
template <>
struct Mma<BF16> {
  typedef f32x4_t acc_t;
  __device__ static __forceinline__ acc_t run(i32x4_t a, i32x4_t b, acc_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), c, 0, 0, 0);
  }
};

constexpr int STEP = 64;  // bytes of a row in one step

struct GemmArgs {
  const char *a, *b;
  int64_t lda, ldb;  // bytes between rows
  int m, n, kbytes;
  int tiles_m, tiles_n;
  int splits, split_steps;  // the summed dimension in `splits` runs of `split_steps` steps
};

// The place of a workgroup: neighbours in launch order sit on different XCDs, so each XCD takes a run of the tiles, and walks it in columns
// of GROUP row tiles, which its L2 then shares.
struct Tile {
  int m, n, split;
};
__device__ __forceinline__ Tile tile_of(const GemmArgs& g, int id) {
  const int tiles = g.tiles_m * g.tiles_n, all = tiles * g.splits;
  constexpr int XCDS = 8, GROUP = 4;
  const int each = all / XCDS, more = all % XCDS, xcd = id % XCDS;
  id = xcd * each + (xcd < more ? xcd : more) + id / XCDS;
  Tile t;
  t.split = id / tiles;
  id -= t.split * tiles;
  const int per = GROUP * g.tiles_n, group = id / per, first = group * GROUP;
  const int high = g.tiles_m - first < GROUP ? g.tiles_m - first : GROUP;
  id -= group * per;
  t.m = first + id % high;
  t.n = id / high;
  return t;
}

template <typename EL, int BM, int BN, int WM, int WN, int S>
struct Gemm {
  static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
  static constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  static constexpr int LA = BM / 16 / WAVES, LB = BN / 16 / WAVES;  // 1 KB loads (16 rows) of a wave and step
  static constexpr int SLOT = (BM + BN) * STEP;
  static constexpr int LDS = S * SLOT;
  static_assert(LA * WAVES * 16 == BM && LB * WAVES * 16 == BN, "whole loads");
  typedef typename Mma<EL>::acc_t acc_t;

  // acc[i][j]: rows m = 16 i + lane % 16 and columns n = 16 j + 4 (lane / 16) + 0..3 of the wave's part
  template <typename Acc>
  __device__ static __forceinline__ void run(const GemmArgs& g, const Tile& t, char* lds, Acc (&acc)[FM][FN]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m0 = t.m * BM, n0 = t.n * BN;
    const int first = t.split * g.split_steps;
    const int left = (g.kbytes + STEP - 1) / STEP - first, steps = left < g.split_steps ? left : g.split_steps;
    const int am = g.m - m0 < BM ? g.m - m0 : BM, bn = g.n - n0 < BN ? g.n - n0 : BN;
    const __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc((void*)(g.a + (int64_t)m0 * g.lda), 0, (int)((am - 1) * g.lda + g.kbytes), 0x00020000);
    const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc((void*)(g.b + (int64_t)n0 * g.ldb), 0, (int)((bn - 1) * g.ldb + g.kbytes), 0x00020000);
    // a load's lane: row lane / 4 of its sixteen, piece (lane % 4) of the slot's row
    const int piece = (lane & 3) ^ ((lane >> 4) & 3);
    int ao[LA], bo[LB];
#pragma unroll
    for (int j = 0; j < LA; ++j) {
      const int r = (wave * LA + j) * 16 + (lane >> 2);
      ao[j] = (r < am ? r : am - 1) * (int)g.lda + piece * 16;
    }
#pragma unroll
    for (int j = 0; j < LB; ++j) {
      const int r = (wave * LB + j) * 16 + (lane >> 2);
      bo[j] = (r < bn ? r : bn - 1) * (int)g.ldb + piece * 16;
    }
    const auto issue = [&](int step, int slot) {
      const int k = (first + step) * STEP;
      const bool in = k + piece * 16 < g.kbytes && step < steps;
      char* to = lds + slot * SLOT;
#pragma unroll
      for (int j = 0; j < LA; ++j)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (__attribute__((address_space(3))) void*)(to + (wave * LA + j) * 1024), 16, in ? ao[j] + k : -16, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < LB; ++j)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (__attribute__((address_space(3))) void*)(to + BM * STEP + (wave * LB + j) * 1024), 16, in ? bo[j] + k : -16, 0, 0, 0);
    };
    const int wm = wave / WN, wn = wave % WN;
    const int r = lane & 15, at = r * STEP + (((lane >> 4) ^ (r >> 2)) & 3) * 16;
    const auto a_at = [&](int slot, int i) { return *(const i32x4_t*)(lds + slot * SLOT + (wm * FM + i) * 1024 + at); };
    const auto b_at = [&](int slot, int j) { return *(const i32x4_t*)(lds + slot * SLOT + BM * STEP + (wn * FN + j) * 1024 + at); };
#pragma unroll
    for (int s = 0; s < S - 1; ++s) issue(s, s);
    constexpr int L = LA + LB;
    wait_and_meet<(S - 2) * L>();
    i32x4_t fa[FM], fb[FN], fc[FN];
#pragma unroll
    for (int i = 0; i < FM; ++i) fa[i] = a_at(0, i);
#pragma unroll
    for (int j = 0; j < FN; ++j) fb[j] = b_at(0, j);
    int slot = 0;  // of the step being multiplied
    // one step: its operands are in registers; those of the next take their place as they are used up
    const auto turn = [&](int step, const i32x4_t(&now)[FN], i32x4_t(&then)[FN]) {
      // every wave has its operands of `step` in registers, and step + 1 is in LDS: the slot before `slot` is free
      wait_and_meet<(S - 3) * L>();
      issue(step + S - 1, slot == 0 ? S - 1 : slot - 1);
      slot = slot + 1 == S ? 0 : slot + 1;
#pragma unroll
      for (int i = 0; i < FM; ++i) {
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = Mma<EL>::run(now[j], fa[i], acc[i][j]);
        fa[i] = a_at(slot, i);
#pragma unroll
        for (int j = i * FN / FM; j < (i + 1) * FN / FM; ++j) then[j] = b_at(slot, j);
        __builtin_amdgcn_sched_barrier(0);  // the reads stay here, a step ahead of their use
      }
    };
    for (int step = 0; step < steps; step += 2) {  // an odd number of steps ends with one of zeros
      turn(step, fb, fc);
      turn(step + 1, fc, fb);
    }
    wait_and_meet<0>();  // nothing may still be on its way to LDS when it is used again, or at the workgroup's end
  }

  // all but the last LEFT loads of this wave are in LDS, its reads are done, and so are the other waves'
  template <int LEFT>
  __device__ static __forceinline__ void wait_and_meet() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory");
  }
};

}  // namespace nf
