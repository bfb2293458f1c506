// Products C[m, n] = sum_k A[m, k] B[n, k] on the matrix instructions: 8-bit integers (16x16x64, 32-bit integer sums) and float16 / bfloat16
// (16x16x32, float32 sums).  Both take 16 bytes a lane and 64 bytes of a row and step, so the code sees bytes.  Operands of 16 bits may also lie
// across the summed dimension, A as [k][m] or B as [k][n] ("crosswise"): LDS's transposing read hands them to the instruction.
//
// A workgroup owns BM x BN of C.  Steps of 128 bytes of every row of its operands (whole cache lines: with 64 bytes the L2 hands out twice
// the bytes, 0.40 us instead of 0.27 for 32 KB on all compute units) go straight from memory to LDS, no registers in between, into a ring of five
// slots, each one operand's step: A, B, A, B, A.  A step is multiplied in two halves; a wave keeps the operands of the half that it multiplies in
// registers and reads the next half's between the matrix instructions.  There is one meeting of the waves in a step, behind its first half: then
// all of the step is in registers, its two slots are free, and the next step has to be there.
//
// On tiles of 256 x 256: bf16 16384 x 4096 x 4096 along the sum 395 us alone, 408 - 425 in a training step (1290 - 1390 TFLOP/s), both operands crosswise 396 - 415;
// int8 16384 x 8192 x 8192 798 - 848 us by the card (2590 - 2760 Tops/s).  The matrix units are busy for 70 % of the clocks (74 % crosswise, int8 69 %), at some 1.9 GHz; what
// bounds the rest is the loads: without them (their data stale) 1730 TFLOP/s.  Measured and not kept: matrix instructions of 32x32, 3 to 10 % slower; 64-byte steps
// with a meeting every second one, 12 %; priorities for the waves that multiply, -4 to +7 %; groups of 2, 8 or 16 row tiles, up to 10 %.
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

constexpr int STEP = 128, HALF = 64;  // bytes of a row in one step, and in one matrix instruction

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
// transposing read; what waits is Gemm::wait_and_meet.  (Loads that the compiler does not count make its own waits longer, never shorter.)
__device__ __forceinline__ i32x4_t buffer_of(const char* p, int bytes) {
  const uint64_t v = (uint64_t)(uintptr_t)p;
  return i32x4_t{__builtin_amdgcn_readfirstlane((int)(uint32_t)v), __builtin_amdgcn_readfirstlane((int)(uint32_t)(v >> 32) & 0xffff),
                 __builtin_amdgcn_readfirstlane(bytes), 0x00020000};
}
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // (M0 is a reserved register: nothing is allocated to it, but the compiler may hold a value of its own there)
__device__ __forceinline__ void load_to_lds(i32x4_t buffer, int offset, uint32_t to) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(offset), "s"(buffer), "s"(to) : "memory", "m0");
}
#pragma clang diagnostic pop

// One operand of a workgroup: R rows of C's side, and the loads that bring a step of it to LDS.
//
// Along the summed dimension a step is R rows of 128 bytes; piece p (16 bytes) of row r lies at place p ^ (r / 2 % 8).  Crosswise it is 64 rows of 2 R bytes;
// the 32-byte segments, sixteen values that one transposing read takes from each of sixteen rows, are spread over the banks by
// an exclusive-or with the row's bits 0, 1 and 3.  No read meets a bank twice that way (a wave's 16-byte reads are served in four parts, the first
// of lanes 0-3, 12-15 and 20-27).
template <bool CROSS, int R, int WAVES>
struct Side {
  static constexpr int LOADS = R / 8 / WAVES;  // of 1 KB, by a wave and step
  static constexpr int BYTES = R * STEP;
  static_assert(LOADS * WAVES * 8 == R, "whole loads");
  const char* base;  // of the workgroup's first row (crosswise: column)
  int64_t ld;
  int count;    // rows there are (crosswise: bytes of a row from the first column on)
  int at[LOADS], row[LOADS];  // a load's offset, and the row of its step (along: the byte of its row) that it starts at

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
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        const int r = (wave * LOADS + j) * 8 + (lane >> 3), piece = (lane & 7) ^ (r >> 1 & 7);
        at[j] = (r < count ? r : count - 1) * (int)ld + piece * 16;
        row[j] = piece * 16;
      }
    }
  }
  // what the loads of one step share: the step at k0 (in bytes of the summed dimension), zeros from `end` on
  struct Step {
    i32x4_t buffer;
    int k0, left;  // left: rows (crosswise), bytes of a row that there are
  };
  __device__ __forceinline__ Step step(int k0, int end) const {
    if constexpr (CROSS) {
      const int rows = (end - k0) / 2, most = rows < 64 ? rows : 64, have = most > 1 ? most : 1;
      return {buffer_of(base + (int64_t)(k0 / 2) * ld, (have - 1) * (int)ld + count), k0, rows};
    } else {
      return {buffer_of(base, (count - 1) * (int)ld + ((end + 15) & ~15)), k0, end - k0};
    }
  }
  // load j of a step into the slot at `to`
  __device__ __forceinline__ void load(const Step& s, int j, uint32_t to, int wave) const {
    load_to_lds(s.buffer, row[j] < s.left ? (CROSS ? at[j] : at[j] + s.k0) : -16, to + (wave * LOADS + j) * 1024);
  }
  // where a lane reads its part of the sixteen rows of C from tile `first` on
  __device__ static __forceinline__ int read_at(int lane, int first) {
    const int i = lane & 15, g = lane >> 4;
    if constexpr (CROSS) {
      const int k = 8 * g + (i >> 2), spread = (k & 3) | (k >> 1 & 4);
      return k * (2 * R) + ((first ^ spread) << 5) + (i & 3) * 8;
    } else {
      return first * (16 * STEP) + i * STEP + (g ^ (i >> 1)) * 16;
    }
  }
  // tile `first` + i of a half of the step at `from`, where first is a multiple of a power of two above i
  __device__ static __forceinline__ i32x4_t read(const char* from, int at, int i, int half) {
    if constexpr (CROSS) {
      typedef short s4_t __attribute__((ext_vector_type(4)));
      const auto* p = (__attribute__((address_space(3))) s4_t*)(from + half * (64 * R) + (at ^ (i << 5)));
      union {
        s4_t part[2];
        i32x4_t whole;
      } v;
      v.part[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4_t*)p);
      v.part[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4_t*)p + R);  // four rows on
      return v.whole;
    } else {
      return *(const i32x4_t*)(from + (at ^ (half * 64)) + i * (16 * STEP));
    }
  }
};

// the sum of a fragment's eight values and s
template <typename EL>
__device__ __forceinline__ float add8(i32x4_t v, float s) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int two = v[i];  // (a bit cast of the vector's element itself takes its first one)
    if constexpr (std::is_same<EL, BF16>::value)
      s = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(nf_bf16x2, two), nf_bf16x2{(__bf16)1.0f, (__bf16)1.0f}, s, false);
    else if constexpr (std::is_same<EL, F16>::value)
      s = __builtin_amdgcn_fdot2(__builtin_bit_cast(nf_f16x2, two), nf_f16x2{(_Float16)1.0f, (_Float16)1.0f}, s, false);
  }
  return s;
}

template <typename EL, int BM, int BN, int WM, int WN, bool AX = false, bool BX = false>
struct Gemm {
  static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
  static constexpr int FM = BM / WM / 16, FN = BN / WN / 16, ROWS_M = BM, WAVES_N = WN;
  static constexpr int WAVES_SIMD = FM * FN > 32 ? 1 : 2;  // a wave of 128 x 128 takes all of a SIMD's registers
  typedef Side<AX, BM, WAVES> A;
  typedef Side<BX, BN, WAVES> B;
  static constexpr int SLOT = A::BYTES > B::BYTES ? A::BYTES : B::BYTES, SLOTS = 5;
  static constexpr int LDS = SLOTS * SLOT;
  static_assert(!(AX || BX) || !std::is_same<EL, I8>::value, "the transposing read takes 16-bit values");
  static_assert((FM & (FM - 1)) == 0 && (FN & (FN - 1)) == 0 && BM >= 128 && BN >= 128, "what the spread over the banks assumes");
  typedef typename Mma<EL>::acc_t acc_t;

  // acc[i][j]: rows m = 16 i + lane % 16 and columns n = 16 j + 4 (lane / 16) + 0..3 of the wave's part
  // SUMS: sums[i] becomes the lane's part of the sum of A's row m (the four lanes with the same lane % 16 hold one each).
  template <bool SUMS = false, typename Acc>
  __device__ static __forceinline__ void run(const GemmArgs& g, const Tile& t, char* lds, Acc (&acc)[FM][FN], float* sums = nullptr) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int first = t.split * g.split_steps;
    const int left = (g.kbytes + STEP - 1) / STEP - first, steps = left < g.split_steps ? left : g.split_steps;
    const int end = (first + steps) * STEP < g.kbytes ? (first + steps) * STEP : g.kbytes;
    const A side_a(g.a, g.lda, t.m * BM, g.m, lane, wave);
    const B side_b(g.b, g.ldb, t.n * BN, g.n, lane, wave);
    const uint32_t ring = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds);
    const int wm = wave / WN, wn = wave % WN;
    const int at_a = A::read_at(lane, wm * FM), at_b = B::read_at(lane, wn * FN);
    const auto after = [](int slot, int n) { return slot + n >= SLOTS ? slot + n - SLOTS : slot + n; };
    const auto load_a = [&](int step, int slot) {
      const typename A::Step s = side_a.step((first + step) * STEP, end);
#pragma unroll
      for (int j = 0; j < A::LOADS; ++j) side_a.load(s, j, ring + slot * SLOT, wave);
    };
    load_a(0, 0);
    {
      const typename B::Step s = side_b.step(first * STEP, end);
#pragma unroll
      for (int j = 0; j < B::LOADS; ++j) side_b.load(s, j, ring + SLOT, wave);
    }
    load_a(1, 2);
    {
      const typename B::Step s = side_b.step((first + 1) * STEP, end);
#pragma unroll
      for (int j = 0; j < B::LOADS; ++j) side_b.load(s, j, ring + 3 * SLOT, wave);
    }
    wait_and_meet<A::LOADS + B::LOADS>();
    i32x4_t fa[FM], fb[FN], fc[FN];
#pragma unroll
    for (int i = 0; i < FM; ++i) fa[i] = A::read(lds, at_a, i, 0);
#pragma unroll
    for (int j = 0; j < FN; ++j) fb[j] = B::read(lds + SLOT, at_b, j, 0);
    // One half of a step: its operands are in registers; those of the next half (from the slots at a and b) take their place as they are used up,
    // and `load` sends the loads that fall into this half, one behind each of its first rows of tiles.  (All of them at once, behind the meeting,
    // queue up in front of the matrix instructions.)  The last row's operand moves aside, so that the last read is a row old when the half ends.
    const auto half = [&](auto sum_c, const i32x4_t(&now)[FN], i32x4_t(&then)[FN], const char* a, const char* b, int h, auto&& load, int loads) {
      const i32x4_t last = fa[FM - 1];
      fa[FM - 1] = A::read(a, at_a, FM - 1, h);
#pragma unroll
      for (int i = 0; i < FM; ++i) {
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = Mma<EL>::run(now[j], i < FM - 1 ? fa[i] : last, acc[i][j]);
        if constexpr (decltype(sum_c)::value != 0) sums[i] = add8<EL>(i < FM - 1 ? fa[i] : last, sums[i]);
        if (i < FM - 1) fa[i] = A::read(a, at_a, i, h);
#pragma unroll
        for (int j = i * FN / (FM - 1); j < (i + 1) * FN / (FM - 1) && j < FN; ++j) then[j] = B::read(b, at_b, j, h);
#pragma unroll
        for (int j = i * PER_ROW; j < (i + 1) * PER_ROW; ++j)
          if (j < loads) load(j);
        __builtin_amdgcn_sched_barrier(0);  // the reads stay here, half a step ahead of their use
      }
    };
    int slot = 0;  // of A's step; B's is the next one
    for (int step = 0; step < steps; ++step) {
      const int a1 = after(slot, 2), b1 = after(slot, 3), b0 = after(slot, 1);
      {
        // A of the step after the next goes where B of the last step was
        const typename A::Step s = side_a.step((first + step + 2) * STEP, end);
        const uint32_t to = ring + after(slot, 4) * SLOT;
        const auto load = [&](int j) { side_a.load(s, j, to, wave); };
        half(Int<SUMS>{}, fb, fc, lds + slot * SLOT, lds + b0 * SLOT, 1, load, A::LOADS);
      }
      wait_and_meet<A::LOADS>();
      {
        // B of it where A of this step was
        const typename B::Step s = side_b.step((first + step + 2) * STEP, end);
        const uint32_t to = ring + slot * SLOT;
        const auto load = [&](int j) { side_b.load(s, j, to, wave); };
        half(Int<SUMS>{}, fc, fb, lds + a1 * SLOT, lds + b1 * SLOT, 0, load, B::LOADS);
      }
      slot = a1;
    }
    wait_and_meet<0>();  // nothing may still be on its way to LDS when it is used again, or at the workgroup's end
  }

  // The sums in rows, behind run(): pass(rows) once or twice, where rows(body) calls body(m, v, ask(m)) for eight neighbouring columns from column() on of each row of
  // the pass.  They go through LDS, so that a row leaves in whole cache lines, and what the caller tells apart (types, activations) it tells apart behind
  // them, not with the accumulators live in every branch.  ask() loads what a row's results go together with, four rows ahead of their use.
  static constexpr int LPR = 2 * FN;  // lanes to a row
  __device__ static __forceinline__ int column(const Tile& t) {
    return t.n * BN + (int)(threadIdx.x >> 6) % WN * (BN / WN) + (int)(threadIdx.x & 63) % LPR * 8;
  }
  template <typename Acc, typename Ask, typename Pass>
  __device__ static __forceinline__ void each8(const Tile& t, char* lds, const Acc (&acc)[FM][FN], Ask&& ask, Pass&& pass) {
    typedef typename std::remove_cv<typename std::remove_reference<decltype(acc[0][0][0])>::type>::type E;
    constexpr int LD = 16 * FN + 4, PASSES = 16 * FM * LD * 4 * WAVES <= LDS ? 1 : 2, ROWS = 16 * FM / PASSES, STRIDE = 64 / LPR;
    static_assert(ROWS * LD * 4 * WAVES <= LDS, "a strip for every wave");
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, m0 = t.m * BM + wave / WN * (BM / WM) + lane / LPR;
    E* strip = (E*)lds + wave * (ROWS * LD);
    constexpr int GROUP = ROWS / STRIDE < 4 ? ROWS / STRIDE : 4;  // rows of a lane and turn of the loop
    decltype(ask(0)) with[GROUP];
    const auto ask_for = [&](int m) {
#pragma unroll
      for (int u = 0; u < GROUP; ++u) with[u] = ask(m + u * STRIDE);
    };
    ask_for(m0);
    const auto run_pass = [&](auto p_c) {
      constexpr int p = decltype(p_c)::value;
#pragma unroll
      for (int i = 0; i < FM / PASSES; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) *(Acc*)(strip + (16 * i + (lane & 15)) * LD + 16 * j + 4 * (lane >> 4)) = acc[p * (FM / PASSES) + i][j];
      pass([&](auto&& body) {
#pragma unroll 1
        for (int r = 0; r < ROWS; r += GROUP * STRIDE) {
          const int m = m0 + p * ROWS + r;
          decltype(ask(0)) now[GROUP];
#pragma unroll
          for (int u = 0; u < GROUP; ++u) now[u] = with[u];
          ask_for(m + GROUP * STRIDE);  // (behind a tile's end: masked as rows that are not there)
#pragma unroll
          for (int u = 0; u < GROUP; ++u) {
            E v[8];
            const E* from = strip + (lane / LPR + r + u * STRIDE) * LD + lane % LPR * 8;
            *(Acc*)v = *(const Acc*)from;
            *(Acc*)(v + 4) = *(const Acc*)(from + 4);
            body(m + u * STRIDE, v, now[u]);
          }
        }
      });
    };
    run_pass(Int<0>{});
    if constexpr (PASSES == 2) run_pass(Int<1>{});
  }

  static constexpr int PER_ROW = (A::LOADS + FM - 1) / FM > (B::LOADS + FM - 1) / FM ? (A::LOADS + FM - 1) / FM : (B::LOADS + FM - 1) / FM;

  // all but the last LEFT loads of this wave are in LDS, all of its reads are done, and so for the other waves
  template <int LEFT>
  __device__ static __forceinline__ void wait_and_meet() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory");
  }
};

// p[n .. n + 7] of a vector of `count` as float32; zeros behind its end
__device__ __forceinline__ void vector8(const void* p, int dt, int n, int count, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = n + i < count ? load_as_f32(p, n + i, dt) : 0.0f;
}

// 16 bytes of a row from any address; bytes beyond the row's end are zeros.  A piece that reaches over the end is read as the row's last 16 bytes
// and shifted (byte by byte that took longer than all the rest of a short product: 19 x 5000 x 4098 18.2 us instead of 13.6).
__device__ __forceinline__ i32x4_t load16(const char* row, int at, int end) {
  uint64_t v[2] = {0, 0};
  if (end >= 16) {
    const int from = at < end - 16 ? at : end - 16, gone = at - from;  // bytes that belong in front
    __builtin_memcpy(v, row + from, 16);
    const int bits = 8 * (gone & 7);
    const uint64_t across = bits == 0 ? 0 : v[1] << (64 - bits);
    const uint64_t lo = v[0] >> bits | across, hi = v[1] >> bits;
    v[0] = gone < 8 ? lo : gone < 16 ? hi : 0;
    v[1] = gone < 8 ? hi : 0;
  } else {
#pragma unroll
    for (int i = 0; i < 15; ++i)
      if (at + i < end) v[i / 8] |= (uint64_t)(uint8_t)row[at + i] << (i % 8 * 8);
  }
  i32x4_t r;
  __builtin_memcpy(&r, v, 16);
  return r;
}

// Rows cut into pieces, J to each of a workgroup's 256 threads: thread t has pieces t, t + 256, ..  One division of 64 bits for all of them, which is
// the same for every thread.
template <int J>
struct Cut {
  static constexpr int PIECES = 256 * J;
  int64_t row0;
  uint32_t rest, each;  // of the workgroup's first piece in its row; pieces of a row
  __device__ __forceinline__ Cut(int64_t block, int each_) : each((uint32_t)each_) {
    row0 = block * PIECES / each_;
    rest = (uint32_t)(block * PIECES - row0 * each_);
  }
  // this thread's j-th piece
  __device__ __forceinline__ int64_t row(int j, int* piece) const {
    const uint32_t at = rest + threadIdx.x + 256 * j, r = at / each;
    *piece = (int)(at - r * each);
    return row0 + r;
  }
};
// One piece a thread where that fills the chip just so (1003 x 777 3.0 us, with four 4.2), four beyond (16384 x 4096 bf16 57 us, with one 61).
inline int cut_pieces(int64_t pieces) { return pieces < (1 << 19) ? 1 : 4; }
inline int64_t cut_blocks(int64_t pieces, int each) { return (pieces + 256 * each - 1) / (256 * each); }

__device__ __forceinline__ int64_t block_number() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }
// rows copied to 16-byte boundaries and filled up with zeros to whole pieces of 16 bytes; a workgroup's part of them
struct Copy {
  const char* from;
  int64_t ld, rows;  // ld: bytes
  char* to;
  int bytes;       // of a row
  int64_t blocks;  // none: nothing to copy
};
template <int J>
__device__ __forceinline__ void copy_rows(int64_t block, const Copy& a) {
  const Cut<J> cut(block, (a.bytes + 15) / 16);
  i32x4_t v[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    int piece;
    const int64_t row = cut.row(j, &piece);
    if (row < a.rows) v[j] = load16(a.from + row * a.ld, piece * 16, a.bytes);
  }
#pragma unroll
  for (int j = 0; j < J; ++j) {
    int piece;
    const int64_t row = cut.row(j, &piece);
    if (row < a.rows) *(i32x4_t*)(a.to + (row * cut.each + piece) * 16) = v[j];
  }
}

// ---- host ---------------------------------------------------------------------------------------
// A grid for `blocks` workgroups, of which one dimension alone could not hold them all: block_number() tells them apart; the last row of the grid may hold more.
inline dim3 grid_of(int64_t blocks) {
  const int64_t most = 1 << 20;
  return blocks <= most ? dim3((unsigned)blocks) : dim3((unsigned)most, (unsigned)((blocks + most - 1) / most));
}
inline int64_t round_up(int64_t v, int64_t unit) { return (v + unit - 1) / unit * unit; }
// whether rows of `bytes` with `ld` bytes between them can be read as they are; 256 of them stay inside 31 bits
inline bool rows_fit(const void* p, int64_t ld, int64_t bytes) { return bytes % 16 == 0 && ld % 16 == 0 && (uintptr_t)p % 16 == 0 && ld < (1 << 22); }

// Tiles of 256 x 256, one to a compute unit, or of 128 x 128, two to one (two take 0.7 of the time of a large one, one alone 0.4), and the summed dimension in
// `splits` runs of steps: what takes the least time for all of them.  us: 1.6 for a step of 256 x 256 on all units, 8 (small tiles 3) for a round's way in and out, and for
// partial sums another launch, written and read at 4.5 TB/s.  What it chooses against the choice by tiles alone, bf16, us: dW of 4426 x 1907 over 29941 rows (five
// runs of large tiles, one of small) 550 / 951, of 1600 x 3264 over 26317 332 / 497; 1180 x 3784 x 7299 76 / 85; without runs 29941 x 1907 x 4426 crosswise 461 / 619;
// never more than the 3 % that runs differ by over 39 such shapes.
struct TilePlan {
  int bm, splits, split_steps;
  int64_t slot_bytes;
};
inline TilePlan tile_plan(int64_t m, int64_t n, int64_t kbytes) {
  constexpr int64_t CUS = 256;
  TilePlan p{};
  const int64_t big = ((m + 255) / 256) * ((n + 255) / 256), small = ((m + 127) / 128) * ((n + 127) / 128);
  const int64_t steps = (kbytes + STEP - 1) / STEP;
  const auto sums = [&](int64_t s) { return s == 1 ? 0.0 : 2.5 + (double)(s * m * n) * 8.0 / 4.5e6; };
  int64_t splits = 1;
  double best = 1e30;
  if (small <= CUS) {
    // few tiles: 0.85 for a step, what memory takes to answer (2^18 rows into 256 x 256 took 142 instead of 62 with 27 runs instead of 128)
    p.bm = 128;
    for (int64_t s = 1; s == 1 || (s * small <= 2 * CUS && s * 2 <= steps); s = s < 8 ? s + 1 : s * 5 / 4) {
      const double cost = 0.85 * (double)((steps + s - 1) / s) + sums(s);
      if (cost < best) best = cost, splits = s;
    }
  } else {
    for (int64_t s = 1; s == 1 || (s <= 8 && s * 8 <= steps); ++s) {
      const int64_t full = s * small / (2 * CUS), last = s * small % (2 * CUS), rounds = (s * big + CUS - 1) / CUS;
      const double each = 1.6 * (double)((steps + s - 1) / s), more = sums(s);
      const double cost_big = (each + 8.0) * (double)rounds + more;
      const double cost_small = (0.7 * each + 3.0) * (double)full + (last == 0 ? 0.0 : (last <= CUS ? 0.4 : 0.7) * each + 3.0) + more;
      if (cost_big < best) best = cost_big, splits = s, p.bm = 256;
      if (cost_small < best) best = cost_small, splits = s, p.bm = 128;
    }
  }
  p.split_steps = (int)((steps + splits - 1) / splits);
  p.splits = (int)((steps + p.split_steps - 1) / p.split_steps);
  if (p.splits > 1) p.slot_bytes = round_up(p.splits * m * round_up(n, 8) * 4, 256);
  return p;
}
// whether one launch holds the plan's workgroups (of two threads for each row of a tile)
inline bool tiles_fit(const TilePlan& p, int64_t m, int64_t n) {
  return (double)((m + p.bm - 1) / p.bm) * (double)((n + p.bm - 1) / p.bm) * p.splits * (2 * p.bm) < 4294967296.0;
}
inline Copy copy_of(const void* from, int64_t ld, int64_t rows, int64_t bytes, char* to, int each) {
  return {(const char*)from, ld, rows, to, (int)bytes, cut_blocks(rows * ((bytes + 15) / 16), each)};
}
// copies of one or two operands' rows in one launch (int8_linear.hip)
struct Pack {
  const void* from;
  int64_t ld, rows, bytes;
  char* to;  // NULL: nothing to copy
};
int pack_rows(const Pack& a, const Pack& b, hipStream_t s);
// nf_quantize_rows on checked arguments; where h is asked for and rows hold at most MOST_BESIDE values, `also` (one piece a thread) is copied in the same launch
// (quantize_rows.hip)
constexpr int64_t MOST_BESIDE = 32768;
int quantize_and_copy(const void* x, int64_t xs, int dtype, int8_t* q, float* scale, void* h, int64_t hs, int act, int64_t rows, int64_t width, const Copy& also,
                      hipStream_t s);

}  // namespace nf
