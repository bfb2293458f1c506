// Products C[m, n] = sum_k A[m, k] B[n, k] on the matrix instructions: 8-bit integers (16x16x64, 32-bit integer sums) and float16 / bfloat16
// (16x16x32, float32 sums).  Both take 16 bytes a lane and 64 bytes of a row and step, so the code sees bytes.  Operands of 16 bits may also lie
// across the summed dimension, A as [k][m] or B as [k][n] ("crosswise"): LDS's transposing read hands them to the instruction.
//
// A workgroup owns BM x BN of C.  Steps of 64 bytes of every row of its operands go straight from memory to
// LDS (no registers in between) into a ring of S slots; S - 1 are in flight or waiting.  A wave keeps the operands of the step that it multiplies
// in registers and reads the next step's between the matrix instructions.  16-byte pieces of a row are placed by an exclusive-or with
// the row's number, which spreads the sixteen rows that a read touches over all banks.
//
// Rows start on 16-byte boundaries and hold whole 16-byte pieces (along the summed dimension: with zeros behind the last value).  Rows of C beyond
// the operand repeat its last one, columns of a crosswise operand beyond it are whatever the buffer holds: neither is stored.  What lies
// beyond the end of the summed dimension comes back as zeros from the buffer's range check.
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
  int m, n, kbytes;  // kbytes: of the summed dimension (crosswise: twice its rows)
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

// The descriptor of `bytes` bytes from p on, and a load of 16 bytes a lane, 1 KB, straight to LDS: lane l's go to `to` + 16 l; a lane whose offset
// leaves the descriptor's range gets zeros.  As assembly without outputs, because the compiler waits for every such load in front of a
// transposing read; what waits is Gemm::wait_and_meet.  (M0 is the compiler's own scratch register, set right before each use.  Loads that the compiler does not count make its own waits longer, never shorter.)
__device__ __forceinline__ i32x4_t buffer_of(const char* p, int bytes) {
  const uint64_t v = (uint64_t)(uintptr_t)p;
  return i32x4_t{__builtin_amdgcn_readfirstlane((int)(uint32_t)v), __builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32) & 0xffff),
                 __builtin_amdgcn_readfirstlane(bytes), 0x00020000};
}
__device__ __forceinline__ void load_to_lds(i32x4_t buffer, int offset, uint32_t to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(offset), "s"(buffer), "s"(to) : "memory");
}

// One operand of a workgroup: R rows of C's side, and the loads that bring a step of it to LDS.
//
// Along the summed dimension a step is R rows of 64 bytes; piece p of row r lies at place p ^ (r / 4).  Crosswise it is 32 rows of 2 R bytes; the
// 32-byte segments, sixteen values that one transposing read takes from each of sixteen rows, are spread over the banks by
// an exclusive-or with the row's bits 0, 1 and 3.
template <bool CROSS, int R, int WAVES>
struct Side {
  static constexpr int LOADS = R / 16 / WAVES;  // of 1 KB, by a wave and step
  static constexpr int BYTES = R * STEP;
  static_assert(LOADS * WAVES * 16 == R, "whole loads");
  const char* base;  // of the workgroup's first row (crosswise: column)
  int64_t ld;
  int count;    // rows there are (crosswise: bytes of a row from the first column on)
  int at[LOADS], row[LOADS];

  __device__ __forceinline__ Side(const char* p, int64_t ld_, int first, int total, int lane, int wave) : ld(ld_) {
    if constexpr (CROSS) {
      base = p + (int64_t)first * 2;
      count = ((total - first) * 2 + 15) / 16 * 16;
      constexpr int PIECES = R / 8;
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        row[j] = (wave * LOADS + j) * (64 / PIECES) + lane / PIECES;
        const int p16 = lane % PIECES, spread = (row[j] & 3) | (row[j] >> 1 & 4), col = (((p16 >> 1) ^ spread) << 1 | (p16 & 1)) * 16;
        at[j] = col < count ? row[j] * (int)ld + col : -16;
      }
    } else {
      base = p + (int64_t)first * ld;
      count = total - first < R ? total - first : R;
      const int piece = (lane & 3) ^ (lane >> 4 & 3);
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        const int r = (wave * LOADS + j) * 16 + (lane >> 2);
        at[j] = (r < count ? r : count - 1) * (int)ld + piece * 16;
        row[j] = piece * 16;
      }
    }
  }
  // step k0 / 64 (k0 in bytes of the summed dimension) into `to`; zeros from `end` on
  __device__ __forceinline__ void load(uint32_t to, int k0, int end, int wave) const {
    if constexpr (CROSS) {
      const int rows = (end - k0) / 2, most = rows < 32 ? rows : 32, have = most > 1 ? most : 1;
      const i32x4_t r = buffer_of(base + (int64_t)(k0 / 2) * ld, (have - 1) * (int)ld + count);
#pragma unroll
      for (int j = 0; j < LOADS; ++j) load_to_lds(r, row[j] < rows ? at[j] : -16, to + (wave * LOADS + j) * 1024);
    } else {
      const i32x4_t r = buffer_of(base, (count - 1) * (int)ld + ((end + 15) & ~15));
      const bool in = k0 + row[0] < end;
#pragma unroll
      for (int j = 0; j < LOADS; ++j) load_to_lds(r, in ? at[j] + k0 : -16, to + (wave * LOADS + j) * 1024);
    }
  }
  // where a lane reads its part of the sixteen rows of C from tile `first` on
  __device__ static __forceinline__ int read_at(int lane, int first) {
    const int i = lane & 15, g = lane >> 4;
    if constexpr (CROSS) {
      const int k = 8 * g + (i >> 2), spread = (k & 3) | (k >> 1 & 4);
      return k * (2 * R) + ((first ^ spread) << 5) + (i & 3) * 8;
    } else {
      return first * 1024 + i * STEP + ((g ^ (i >> 2)) & 3) * 16;
    }
  }
  // tile `first` + i of the step at `from`, where first is a multiple of a power of two above i
  __device__ static __forceinline__ i32x4_t read(const char* from, int at, int i) {
    if constexpr (CROSS) {
      typedef short s4_t __attribute__((ext_vector_type(4)));
      const auto* p = (__attribute__((address_space(3))) s4_t*)(from + (at ^ (i << 5)));
      union {
        s4_t half[2];
        i32x4_t whole;
      } v;
      v.half[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4_t*)p);
      v.half[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4_t*)p + R);  // four rows on
      return v.whole;
    } else {
      return *(const i32x4_t*)(from + at + i * 1024);
    }
  }
};

template <typename EL, int BM, int BN, int WM, int WN, int S, bool AX = false, bool BX = false>
struct Gemm {
  static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
  static constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  static constexpr int SLOT = (BM + BN) * STEP;
  static constexpr int LDS = S * SLOT;
  typedef Side<AX, BM, WAVES> A;
  typedef Side<BX, BN, WAVES> B;
  static_assert(!(AX || BX) || !std::is_same<EL, I8>::value, "the transposing read takes 16-bit values");
  static_assert((FM & (FM - 1)) == 0 && (FN & (FN - 1)) == 0 && BM >= 128 && BN >= 128, "what the spread over the banks assumes");
  typedef typename Mma<EL>::acc_t acc_t;

  // acc[i][j]: rows m = 16 i + lane % 16 and columns n = 16 j + 4 (lane / 16) + 0..3 of the wave's part
  template <typename Acc>
  __device__ static __forceinline__ void run(const GemmArgs& g, const Tile& t, char* lds, Acc (&acc)[FM][FN]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int first = t.split * g.split_steps;
    const int left = (g.kbytes + STEP - 1) / STEP - first, steps = left < g.split_steps ? left : g.split_steps;
    const int end = (first + steps) * STEP < g.kbytes ? (first + steps) * STEP : g.kbytes;
    const A side_a(g.a, g.lda, t.m * BM, g.m, lane, wave);
    const B side_b(g.b, g.ldb, t.n * BN, g.n, lane, wave);
    const uint32_t ring = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds);
    const auto issue = [&](int step, int slot) {
      const uint32_t to = ring + slot * SLOT;
      side_a.load(to, (first + step) * STEP, end, wave);
      side_b.load(to + BM * STEP, (first + step) * STEP, end, wave);
    };
    const int wm = wave / WN, wn = wave % WN;
    const int at_a = A::read_at(lane, wm * FM), at_b = B::read_at(lane, wn * FN);
    const auto a_at = [&](int slot, int i) { return A::read(lds + slot * SLOT, at_a, i); };
    const auto b_at = [&](int slot, int j) { return B::read(lds + slot * SLOT + BM * STEP, at_b, j); };
#pragma unroll
    for (int s = 0; s < S - 1; ++s) issue(s, s);
    constexpr int L = A::LOADS + B::LOADS;
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

// ---- host ---------------------------------------------------------------------------------------
inline int64_t round_up(int64_t v, int64_t unit) { return (v + unit - 1) / unit * unit; }
// whether rows of `bytes` with `ld` bytes between them can be read as they are; 256 of them stay inside 31 bits
inline bool rows_fit(const void* p, int64_t ld, int64_t bytes) { return bytes % 16 == 0 && ld % 16 == 0 && (uintptr_t)p % 16 == 0 && ld < (1 << 22); }

// Tiles of 256 x 256 where there are enough of them for the chip, else of 128 x 128, with the summed dimension in runs of at least
// eight steps so that some 512 workgroups come together.
struct TilePlan {
  int bm, splits, split_steps;
  int64_t slot_bytes;
};
inline TilePlan tile_plan(int64_t m, int64_t n, int64_t kbytes) {
  TilePlan p{};
  const int64_t big = ((m + 255) / 256) * ((n + 255) / 256), small = ((m + 127) / 128) * ((n + 127) / 128);
  p.bm = big >= 192 ? 256 : 128;
  const int64_t tiles = p.bm == 256 ? big : small, steps = (kbytes + STEP - 1) / STEP;
  int64_t splits = p.bm == 256 ? 1 : 512 / tiles;
  if (splits > steps / 8) splits = steps / 8;
  if (splits < 1) splits = 1;
  p.split_steps = (int)((steps + splits - 1) / splits);
  p.splits = (int)((steps + p.split_steps - 1) / p.split_steps);
  if (p.splits > 1) p.slot_bytes = round_up(p.splits * m * round_up(n, 4) * 4, 256);
  return p;
}
// copies rows to 16-byte boundaries, filled up with zeros to whole 16-byte pieces (int8_linear.hip)
int pack_rows(const char* from, int64_t ld, int64_t bytes, char* to, int64_t rows, hipStream_t s);

}  // namespace nf
