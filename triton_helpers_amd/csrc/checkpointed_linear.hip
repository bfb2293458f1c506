// A linear layer behind an activation that keeps its input as 8-bit rows for the backward:
//
//   forward   y = act(x) W^T + b;                kept: q, s with x^ = s q (quantize_rows.hip), half of what a 16-bit x takes
//   backward  dx = (dy W) * act'(x^);  dW = dy^T act(x^);  db = sum over rows of dy
//
// Three products of 2 M N K operations on the 16-bit matrix instructions (gemm_tile.h).  The forward's lie along the summed dimension; dx takes W,
// and dW both dy and act(x^), crosswise, as they are in memory.  The gate of dx is applied to the sums in registers.  act(x) and act(x^) are
// written out in 16 bits by streams of their own (a product reads its operand once for each 256 channels of the result).  That rounding (half a step of the
// type for each value) is what the 16-bit matrix instructions take; sums stay in float32 and are rounded once.  Many rows of few channels have kernels of
// their own that read each row once (checkpointed_narrow.hip).
//
// 16384 x 4096 x 4096 bf16 with GELU, forward and backward 1367 - 1445 us by the card; launched alone 8-bit rows and act(x) 60, forward product 400 - 420, sums of dy's columns 42 + 5, act(x^) 50, dx 455 - 470
// (its gate, a GELU's slope of 2^26 values, takes 45 of it), dW 400 - 415.  Three products alone take 1230 at the forward's rate.
#include "checkpointed_narrow.h"
#include "gemm_tile.h"

namespace nf {

enum { OUT_BIAS, OUT_GATE, OUT_PLAIN };

struct Out {
  void* y;
  int64_t ldy;
  const void* bias;
  int bias_dt, act;
  const int8_t* q;  // the gate's rows, without gaps
  const float* s;
  int m, n, y_dt;
  float* sums;  // dW: partial sums of dy's columns [split][m] (of a single run: unused), NULL where they are not wanted
  void* db;     // where they go, in type db_dt
  int db_dt;
};

// the gate of eight columns of a row
struct Gate {
  int q[2];
  float s;
};
template <bool GATE>
__device__ __forceinline__ Gate gate_of(const Out& e, int m, int n) {
  Gate g{};
  if constexpr (GATE) {
    if (e.act != NF_ACT_NONE && m < e.m && n < e.n) {
      const int8_t* q = e.q + (int64_t)m * e.n + n;
      const int left = e.n - n;
      if (left >= 8) {
        __builtin_memcpy(g.q, q, 8);
      } else {
        int8_t c[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = q[i < left ? i : 0];
        __builtin_memcpy(g.q, c, 8);
      }
      g.s = e.s[m];
    }
  }
  return g;
}
// eight columns of a row; b: their biases
template <int MODE, int ACT, typename YT>
__device__ __forceinline__ void put8(const Out& e, int m, int n, const float (&v)[8], const float (&b)[8], const Gate& g) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (MODE == OUT_GATE) r[i] = gated<ACT>(v[i], g.s * (float)(g.q[i / 4] << (24 - i % 4 * 8) >> 24));
    else r[i] = MODE == OUT_BIAS ? v[i] + b[i] : v[i];
  }
  store8<YT>((typename YT::storage*)e.y + (int64_t)m * e.ldy + n, e.n - n, r);
}

// body(activation, type of y) under branches that are the same for every thread
template <int MODE, typename T, typename Body>
__device__ __forceinline__ void with_out(const Out& e, Body&& body) {
  if constexpr (MODE == OUT_GATE) with_act(e.act, [&](auto act_c) { body(act_c, T{}); });
  else if constexpr (MODE == OUT_BIAS) body(Int<NF_ACT_NONE>{}, T{});
  else if (e.y_dt == NF_F32) body(Int<NF_ACT_NONE>{}, F32{});
  else body(Int<NF_ACT_NONE>{}, T{});
}

template <typename T, typename G, int MODE>
__global__ __launch_bounds__(G::THREADS, G::WAVES_SIMD) void keep_tile_k(GemmArgs g, Out e, float* slots) {
  __shared__ __attribute__((aligned(1024))) char lds[G::LDS];
  f32x4_t acc[G::FM][G::FN] = {};
  const Tile t = tile_of(g, blockIdx.x);
  if constexpr (MODE == OUT_PLAIN && G::ROWS_M == 128) {
    // db on the way: the first column of tiles holds each value of dy once; one of the waves that share a row of them adds it up.  (The sums
    // take instructions of every wave: nothing in the small tiles, which wait for memory, but 40 % in the large ones.)
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool summing = e.sums != nullptr && t.n == 0 && wave % G::WAVES_N == 0;
    float sums[G::FM] = {};
    G::template run<true>(g, t, lds, acc, sums);
    if (summing) {
      const int m = t.m * G::ROWS_M + wave / G::WAVES_N * (16 * G::FM) + lane;
#pragma unroll
      for (int i = 0; i < G::FM; ++i) {
        float v = sums[i] + __shfl_xor(sums[i], 16);
        v += __shfl_xor(v, 32);
        if (lane < 16 && m + 16 * i < g.m) {
          if (slots == nullptr) store_any(e.db, m + 16 * i, e.db_dt, v);
          else e.sums[(int64_t)t.split * g.m + m + 16 * i] = v;
        }
      }
    }
  } else {
    G::run(g, t, lds, acc);
  }
  const int n = G::column(t);
  if (slots != nullptr) {  // [split][m][n rounded up to 8]
    const int64_t ld = (g.n + 7) / 8 * 8;
    float* o = slots + (int64_t)t.split * g.m * ld + n;
    G::each8(t, lds, acc, [](int) { return 0; }, [&](auto&& rows) {
      rows([&](int m, const float (&v)[8], int) {
        if (m < g.m && n < g.n) __builtin_memcpy(__builtin_assume_aligned(o + (int64_t)m * ld, 16), v, 32);
      });
    });
    return;
  }
  float b[8] = {};
  if (MODE == OUT_BIAS && e.bias != nullptr) vector8(e.bias, e.bias_dt, n, e.n, b);
  G::each8(t, lds, acc, [&](int m) { return gate_of<MODE == OUT_GATE>(e, m, n); }, [&](auto&& rows) {
    with_out<MODE, T>(e, [&](auto act_c, auto y_c) {
      rows([&](int m, const float (&v)[8], const Gate& gate) {
        if (m < g.m && n < g.n) put8<MODE, decltype(act_c)::value, decltype(y_c)>(e, m, n, v, b, gate);
      });
    });
  });
}

// the sums of the runs; dW's launch has workgroups for db's sums in front
inline int64_t db_blocks(const Out& e) { return e.sums == nullptr ? 0 : (e.m + 255) / 256; }
template <typename T, int MODE>
__global__ __launch_bounds__(256) void keep_sum_k(const float* slots, int splits, Out e, int db_blocks) {
  if (MODE == OUT_PLAIN && (int)blockIdx.x < db_blocks) {
    const int m = blockIdx.x * 256 + threadIdx.x;
    if (m >= e.m) return;
    float v = 0.0f;
#pragma unroll 4
    for (int k = 0; k < splits; ++k) v += e.sums[(int64_t)k * e.m + m];
    store_any(e.db, m, e.db_dt, v);
    return;
  }
  const int64_t parts = (e.n + 7) / 8, ld = parts * 8, each = (int64_t)e.m * ld;
  const int64_t at = (int64_t)(blockIdx.x - db_blocks) * 256 + threadIdx.x;
  if (at >= e.m * parts) return;
  const int m = (int)(at / parts), n = (int)(at % parts) * 8;
  float v[8] = {}, b[8] = {};
#pragma unroll 4
  for (int k = 0; k < splits; ++k) {
    const float* p = slots + k * each + (int64_t)m * ld + n;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += p[i];
  }
  if (MODE == OUT_BIAS && e.bias != nullptr) vector8(e.bias, e.bias_dt, n, e.n, b);
  with_out<MODE, T>(e, [&](auto act_c, auto y_c) {
    constexpr int ACT = decltype(act_c)::value;
    put8<MODE, ACT, decltype(y_c)>(e, m, n, v, b, gate_of<MODE == OUT_GATE>(e, m, n));
  });
}

// What the backward's products read and the caller does not have: copies of dy and W on 16-byte boundaries, and act(s q) in 16 bits, each with rows
// filled up with zeros to whole 16-byte pieces.  Streams, 16 bytes a thread and store; one launch for all of them (of what a small layer's step takes,
// launches are the most).
struct Prepare {
  Copy copy[2];
  const int8_t* q;
  const float* s;
  uint16_t* h;
  int64_t rows, blocks;  // none of either: no act(x^) is wanted
  int width, act;
};
template <typename T, int J>
__global__ __launch_bounds__(256) void prepare_k(Prepare a) {
  int64_t block = block_number();
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    if (block < a.copy[c].blocks) {
      copy_rows<J>(block, a.copy[c]);
      return;
    }
    block -= a.copy[c].blocks;
  }
  if (block >= a.blocks) return;  // (a grid of two dimensions holds some more than there are)
  const Cut<J> cut(block, (a.width + 7) / 8);
  int q[J][2];
  float scale[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    int piece;
    const int64_t row = cut.row(j, &piece);
    const int n = a.width - piece * 8;
    q[j][0] = q[j][1] = 0;
    scale[j] = 0.0f;
    if (row < a.rows) {
      const int8_t* p = a.q + row * a.width + piece * 8;
      if (n >= 8) {
        __builtin_memcpy(q[j], p, 8);
      } else {
#pragma unroll
        for (int i = 0; i < 7; ++i)
          if (i < n) q[j][i / 4] |= (p[i] & 255) << (i % 4 * 8);
      }
      scale[j] = a.s[row];
    }
  }
  with_act(a.act, [&](auto act_c) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      int piece;
      const int64_t row = cut.row(j, &piece);
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = scale[j] * (float)(q[j][i / 4] << (24 - i % 4 * 8) >> 24);
        v[i] = piece * 8 + i < a.width ? act_value<decltype(act_c)::value>(x) : 0.0f;
      }
      if (row < a.rows) store8<T>(a.h + (row * cut.each + piece) * 8, 8, v);
    }
  });
}

// Partial column sums: `across` threads (32 or 64) side by side, eight columns each, the others below; the workgroups of a strip take turns at the rows.  16384 x
// 4096 bf16: 43 us with 64 threads across and 2048 workgroups, 51 with 32, 56 with 1024 workgroups, 50 with 256.
template <typename T>
__global__ __launch_bounds__(256) void column_sums_k(const uint16_t* dy, int64_t ld, int64_t rows, int n, int across, float* slots) {
  __shared__ float part[8 * 256];
  const int t = threadIdx.x & (across - 1), c = (blockIdx.x * across + t) * 8, r = threadIdx.x / across, down = 256 / across;
  float s[8] = {};
  if (c < n) {
#pragma unroll 8
    for (int64_t row = blockIdx.y * down + r; row < rows; row += gridDim.y * down) {
      float v[8];
      load8<T>(dy + row * ld + c, n - c, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] += v[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) part[(r * across + t) * 8 + i] = s[i];
  __syncthreads();
  for (int j = threadIdx.x; j < across * 8; j += 256) {
    const int column = blockIdx.x * across * 8 + j;
    if (column >= n) break;
    float v = part[j];
    for (int i = 1; i < down; ++i) v += part[i * across * 8 + j];
    slots[(int64_t)blockIdx.y * n + column] = v;
  }
}

template <typename T, int MODE, bool AX, bool BX>
int product(GemmArgs g, const TilePlan& p, const Out& e, float* slots, hipStream_t s) {
  g.splits = p.splits;
  g.split_steps = p.split_steps;
  const auto go = [&](auto b_c, auto wm_c, auto wn_c) {
    constexpr int B = decltype(b_c)::value, WM = decltype(wm_c)::value, WN = decltype(wn_c)::value;
    typedef Gemm<T, B, B, WM, WN, AX, BX> G;
    g.tiles_m = (g.m + B - 1) / B;
    g.tiles_n = (g.n + B - 1) / B;
    hipLaunchKernelGGL((keep_tile_k<T, G, MODE>), dim3((unsigned)(g.tiles_m * g.tiles_n * g.splits)), dim3(G::THREADS), 0, s, g, e,
                       p.splits > 1 ? slots : nullptr);
  };
  // (16384 x 4096 x 4096: where both operands lie along the sum four waves of 128 x 128, which read LDS three quarters as often, take 400 us at best, eight of 64 x 128
  // 410, of 128 x 64 2 % more; where one is crosswise eight of 128 x 64 take 440 and 400, of 64 x 128 2 to 5 % more, four 510 and 410)
  if (p.bm == 128) go(Int<128>{}, Int<2>{}, Int<2>{});
  else if constexpr (AX || BX) go(Int<256>{}, Int<2>{}, Int<4>{});
  else go(Int<256>{}, Int<2>{}, Int<2>{});
  const int rc = check_launch("checkpointed_linear");
  if (rc != 0 || p.splits == 1) return rc;
  // (many runs: over several threads)
  if (MODE == OUT_PLAIN && e.n % 8 == 0 && p.splits > 8) {
    const int rc = sum_slots(slots, p.splits, (int64_t)e.m * e.n, e.y, e.y_dt, s);
    return rc != 0 || e.sums == nullptr ? rc : sum_slots(e.sums, p.splits, e.m, e.db, e.db_dt, s);
  }
  const int64_t first = db_blocks(e), blocks = first + (e.m * (int64_t)((e.n + 7) / 8) + 255) / 256;
  hipLaunchKernelGGL((keep_sum_k<T, MODE>), dim3((unsigned)blocks), dim3(256), 0, s, slots, p.splits, e, (int)first);
  return check_launch("checkpointed_linear_sum");
}

// (256 rows of a copied operand stay inside 31 bits, as rows_fit asks of the caller's own)
constexpr int64_t MOST_CHANNELS = 1 << 20;
inline bool sizes_ok(int64_t rows, int64_t n, int64_t k) {
  return rows > 0 && rows <= (1ll << 29) && n >= 1 && n <= MOST_CHANNELS && k >= 1 && k <= MOST_CHANNELS;
}

struct KeepFwd {
  bool narrow;
  int64_t ldh, h_bytes, w_bytes;
  TilePlan tile;
  int64_t total() const { return h_bytes + w_bytes + tile.slot_bytes; }
};
KeepFwd keep_fwd(const void* x, int64_t xs, const void* w, int64_t ws, int64_t rows, int64_t n, int64_t k, int act) {
  KeepFwd p{};
  p.ldh = round_up(k, 8);
  p.narrow = narrow_fits(rows, n, k) && rows_fit(x, xs * 2, k * 2) && rows_fit(w, ws * 2, k * 2);
  if (p.narrow) return p;
  if (act != NF_ACT_NONE || !rows_fit(x, xs * 2, k * 2)) p.h_bytes = round_up(rows * p.ldh * 2, 256);
  if (!rows_fit(w, ws * 2, k * 2)) p.w_bytes = round_up(n * p.ldh * 2, 256);
  p.tile = tile_plan(rows, n, k * 2);
  return p;
}

struct KeepBwd {
  bool narrow;
  int64_t ldk, ldn, dy_bytes, w_bytes, h_bytes, sum_bytes;
  int across, strips, groups;
  bool sums_in_dw;
  TilePlan dx, dw;
  int64_t slots() const { return dx.slot_bytes > dw.slot_bytes ? dx.slot_bytes : dw.slot_bytes; }
  int64_t total() const { return dy_bytes + w_bytes + h_bytes + sum_bytes + slots(); }
};
KeepBwd keep_bwd(const void* dy, int64_t dys, const void* w, int64_t ws, int64_t rows, int64_t n, int64_t k, bool need_dx, bool need_dw, bool need_db) {
  KeepBwd p{};
  p.ldk = round_up(k, 8);
  p.ldn = round_up(n, 8);
  p.narrow = need_dw && narrow_fits(rows, n, k) && rows_fit(dy, dys * 2, n * 2) && (!need_dx || rows_fit(w, ws * 2, k * 2));
  if (p.narrow) {
    p.groups = narrow_groups(rows);
    p.sum_bytes = round_up((int64_t)p.groups * n * 4, 256) + (int64_t)p.groups * n * k * 4;
    return p;
  }
  if ((need_dx || need_dw) && !rows_fit(dy, dys * 2, n * 2)) p.dy_bytes = round_up(rows * p.ldn * 2, 256);
  if (need_dx) {
    if (!rows_fit(w, ws * 2, k * 2)) p.w_bytes = round_up(n * p.ldk * 2, 256);
    p.dx = tile_plan(rows, k, n * 2);
  }
  if (need_dw) {
    p.h_bytes = round_up(rows * p.ldk * 2, 256);
    p.dw = tile_plan(n, k, rows * 2);
  }
  p.sums_in_dw = need_db && need_dw && p.dw.bm == 128;
  if (p.sums_in_dw) {
    if (p.dw.splits > 1) p.sum_bytes = round_up((int64_t)p.dw.splits * n * 4, 256);
  } else if (need_db) {
    p.across = n <= 256 ? 32 : 64;
    p.strips = (int)((n + 8 * p.across - 1) / (8 * p.across));
    const int64_t most = 2048 / p.strips + 1, want = (rows + 63) / 64;
    p.groups = (int)(want < most ? want : most);
    p.sum_bytes = round_up((int64_t)p.groups * n * 4, 256);
  }
  return p;
}

template <typename T>
int fwd(const KeepFwd& p, const void* x, int64_t xs, const void* w, int64_t ws, const void* bias, int bias_dt, void* y, int64_t ys, int8_t* q, float* scale,
        int64_t rows, int64_t n, int64_t k, int act, char* at, void* stream) {
  char *h = at, *packed = at + p.h_bytes;
  float* slots = (float*)(packed + p.w_bytes);
  hipStream_t s = (hipStream_t)stream;
  if (p.narrow) return narrow_fwd({x, w, bias, y, q, scale, xs, ws, ys, rows, (int)n, (int)k, bias_dt, act}, T::code, s);
  const bool beside = p.w_bytes > 0 && p.h_bytes > 0 && k <= MOST_BESIDE && cut_pieces(p.w_bytes / 16) == 1;
  if (q != nullptr || p.h_bytes > 0) {
    const Copy also = beside ? copy_of(w, ws * 2, n, k * 2, packed, 1) : Copy{};
    if (const int rc = quantize_and_copy(x, xs, T::code, q, scale, p.h_bytes > 0 ? h : nullptr, p.ldh, act, rows, k, also, s)) return rc;
  }
  if (p.w_bytes > 0 && !beside)
    if (const int rc = pack_rows({w, ws * 2, n, k * 2, packed}, {}, s)) return rc;
  const GemmArgs g{p.h_bytes > 0 ? h : (const char*)x, p.w_bytes > 0 ? packed : (const char*)w, (p.h_bytes > 0 ? p.ldh : xs) * 2,
                   (p.w_bytes > 0 ? p.ldh : ws) * 2, (int)rows, (int)n, (int)k * 2, 0, 0, 0, 0};
  const Out e{y, ys, bias, bias_dt, NF_ACT_NONE, nullptr, nullptr, (int)rows, (int)n, T::code, nullptr, nullptr, 0};
  return product<T, OUT_BIAS, false, false>(g, p.tile, e, slots, s);
}

template <typename T>
int bwd(const KeepBwd& p, const void* dy, int64_t dys, const int8_t* q, const float* scale, const void* w, int64_t ws, void* dx, void* dw, int dw_dt,
        void* db, int db_dt, int64_t rows, int64_t n, int64_t k, int act, char* at, hipStream_t s) {
  char *packed_dy = at, *packed_w = packed_dy + p.dy_bytes, *h = packed_w + p.w_bytes, *sums = h + p.h_bytes;
  float* slots = (float*)(sums + p.sum_bytes);
  if (p.narrow) {
    float *part_db = (float*)sums, *part_dw = (float*)(sums + round_up((int64_t)p.groups * n * 4, 256));
    if (const int rc = narrow_bwd({dy, w, q, scale, dx, part_dw, db == nullptr ? nullptr : part_db, dys, ws, rows, (int)n, (int)k, act}, T::code, s)) return rc;
    if (db != nullptr)
      if (const int rc = sum_slots(part_db, p.groups, n, db, db_dt, s)) return rc;
    return sum_slots(part_dw, p.groups, n * k, dw, dw_dt, s);
  }
  if (db != nullptr && !p.sums_in_dw) {
    hipLaunchKernelGGL((column_sums_k<T>), dim3(p.strips, p.groups), dim3(256), 0, s, (const uint16_t*)dy, dys, rows, (int)n, p.across, (float*)sums);
    if (const int rc = check_launch("column_sums")) return rc;
    if (const int rc = sum_slots((const float*)sums, p.groups, n, db, db_dt, s)) return rc;
  }
  Prepare make{};
  int64_t blocks = 0;
  const int each = cut_pieces((p.dy_bytes + p.w_bytes + p.h_bytes) / 16);
  const auto copy = [&](int i, const void* from, int64_t ld, int64_t count, int64_t width, char* to) {
    make.copy[i] = copy_of(from, ld * 2, count, width * 2, to, each);
    blocks += make.copy[i].blocks;
  };
  if (p.dy_bytes > 0) copy(0, dy, dys, rows, n, packed_dy);
  if (p.w_bytes > 0) copy(1, w, ws, n, k, packed_w);
  if (dw != nullptr) {
    make.q = q, make.s = scale, make.h = (uint16_t*)h, make.rows = rows, make.width = (int)k, make.act = act;
    blocks += make.blocks = cut_blocks(rows * (p.ldk / 8), each);
  }
  if (blocks > 0) {
    if (each == 1) hipLaunchKernelGGL((prepare_k<T, 1>), grid_of(blocks), dim3(256), 0, s, make);
    else hipLaunchKernelGGL((prepare_k<T, 4>), grid_of(blocks), dim3(256), 0, s, make);
    if (const int rc = check_launch("checkpointed_linear_prepare")) return rc;
  }
  const char* a = p.dy_bytes > 0 ? packed_dy : (const char*)dy;
  const int64_t lda = (p.dy_bytes > 0 ? p.ldn : dys) * 2;
  if (dx != nullptr) {
    const GemmArgs g{a, p.w_bytes > 0 ? packed_w : (const char*)w, lda, (p.w_bytes > 0 ? p.ldk : ws) * 2, (int)rows, (int)k, (int)n * 2, 0, 0, 0, 0};
    const Out e{dx, k, nullptr, NF_F32, act, q, scale, (int)rows, (int)k, T::code, nullptr, nullptr, 0};
    if (const int rc = product<T, OUT_GATE, false, true>(g, p.dx, e, slots, s)) return rc;
  }
  if (dw != nullptr) {
    const GemmArgs g{a, h, lda, p.ldk * 2, (int)n, (int)k, (int)rows * 2, 0, 0, 0, 0};
    const Out e{dw, k, nullptr, NF_F32, NF_ACT_NONE, nullptr, nullptr, (int)n, (int)k, dw_dt, p.sums_in_dw ? (float*)sums : nullptr, db, db_dt};
    return product<T, OUT_PLAIN, true, true>(g, p.dw, e, slots, s);
  }
  return 0;
}

}  // namespace nf

using namespace nf;

extern "C" int64_t nf_linear_keep_fwd_workspace_bytes(const void* x, int64_t x_stride, const void* w, int64_t w_stride, int64_t rows, int64_t n, int64_t k,
                                                      int act) {
  return sizes_ok(rows, n, k) ? keep_fwd(x, x_stride, w, w_stride, rows, n, k, act).total() : 0;
}

extern "C" int nf_linear_keep_fwd(const void* x, int64_t x_stride, int dtype, const void* w, int64_t w_stride, const void* bias, int bias_dtype, void* y,
                                  int64_t y_stride, int8_t* q, float* scale, int64_t rows, int64_t n, int64_t k, int act, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  NF_REQUIRE(dtype == NF_F16 || dtype == NF_BF16, NF_EUNSUPPORTED, "dtype code %d: float16 or bfloat16 rows", dtype);
  NF_REQUIRE(dtype_ok(bias_dtype), NF_EINVAL, "unknown dtype code %d", bias_dtype);
  NF_REQUIRE(act >= NF_ACT_NONE && act <= NF_ACT_GELU, NF_EINVAL, "unknown activation %d", act);
  if (rows == 0) return 0;
  NF_REQUIRE(sizes_ok(rows, n, k), NF_EINVAL, "rows=%lld, n=%lld, k=%lld: rows up to 2^29, channels 1..2^20", (long long)rows, (long long)n, (long long)k);
  NF_REQUIRE(x && w && y && (q == nullptr) == (scale == nullptr), NF_EINVAL, "NULL pointer argument");
  NF_REQUIRE((rows == 1 || (x_stride >= k && y_stride >= n)) && (n == 1 || w_stride >= k), NF_EINVAL, "row stride below the row's length");
  const KeepFwd p = keep_fwd(x, x_stride, w, w_stride, rows, n, k, act);
  NF_REQUIRE(p.narrow || tiles_fit(p.tile, rows, n), NF_EUNSUPPORTED, "rows=%lld, n=%lld: more tiles than a launch holds", (long long)rows, (long long)n);
  NF_REQUIRE(!p.narrow || ((uintptr_t)y % 16 == 0 && y_stride % 8 == 0 && y_stride < (1 << 21) && (uintptr_t)q % 16 == 0 && (uintptr_t)scale % 4 == 0), NF_EALIGN,
             "y, its rows and q want 16-byte boundaries");
  NF_REQUIRE(p.total() == 0 || (workspace != nullptr && workspace_bytes >= p.total() && (uintptr_t)workspace % 16 == 0), NF_EINVAL,
             "this call needs a workspace of %lld bytes on a 16-byte boundary", (long long)p.total());
  return dtype == NF_F16 ? fwd<F16>(p, x, x_stride, w, w_stride, bias, bias_dtype, y, y_stride, q, scale, rows, n, k, act, (char*)workspace, stream)
                         : fwd<BF16>(p, x, x_stride, w, w_stride, bias, bias_dtype, y, y_stride, q, scale, rows, n, k, act, (char*)workspace, stream);
}

extern "C" int64_t nf_linear_keep_bwd_workspace_bytes(const void* dy, int64_t dy_stride, const void* w, int64_t w_stride, int64_t rows, int64_t n, int64_t k,
                                                      int need_dx, int need_dw, int need_db) {
  return sizes_ok(rows, n, k) ? keep_bwd(dy, dy_stride, w, w_stride, rows, n, k, need_dx != 0, need_dw != 0, need_db != 0).total() : 0;
}

extern "C" int nf_linear_keep_bwd(const void* dy, int64_t dy_stride, int dtype, const int8_t* q, const float* scale, const void* w, int64_t w_stride, void* dx,
                                  void* dw, int dw_dtype, void* db, int db_dtype, int64_t rows, int64_t n, int64_t k, int act, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  NF_REQUIRE(dtype == NF_F16 || dtype == NF_BF16, NF_EUNSUPPORTED, "dtype code %d: float16 or bfloat16 rows", dtype);
  NF_REQUIRE((dw_dtype == dtype || dw_dtype == NF_F32) && dtype_ok(db_dtype), NF_EUNSUPPORTED, "the weight's gradient is of the rows' type or float32");
  NF_REQUIRE(act >= NF_ACT_NONE && act <= NF_ACT_GELU, NF_EINVAL, "unknown activation %d", act);
  NF_REQUIRE(sizes_ok(rows, n, k), NF_EINVAL, "rows=%lld, n=%lld, k=%lld: rows 1..2^29, channels 1..2^20", (long long)rows, (long long)n, (long long)k);
  if (dx == nullptr && dw == nullptr && db == nullptr) return 0;
  NF_REQUIRE(dy && (db != nullptr || dw != nullptr || dx != nullptr), NF_EINVAL, "NULL pointer argument");
  NF_REQUIRE(dw == nullptr || (q && scale), NF_EINVAL, "NULL pointer argument");
  NF_REQUIRE(dx == nullptr || (w && (act == NF_ACT_NONE || (q && scale))), NF_EINVAL, "NULL pointer argument");
  NF_REQUIRE((rows == 1 || dy_stride >= n) && (n == 1 || dx == nullptr || w_stride >= k), NF_EINVAL, "row stride below the row's length");
  const KeepBwd p = keep_bwd(dy, dy_stride, w, w_stride, rows, n, k, dx != nullptr, dw != nullptr, db != nullptr);
  NF_REQUIRE((p.dx.bm == 0 || tiles_fit(p.dx, rows, k)) && (p.dw.bm == 0 || tiles_fit(p.dw, n, k)), NF_EUNSUPPORTED,
             "rows=%lld, n=%lld, k=%lld: more tiles than a launch holds", (long long)rows, (long long)n, (long long)k);
  NF_REQUIRE(!p.narrow || ((uintptr_t)dx % 16 == 0 && (uintptr_t)q % 16 == 0 && (uintptr_t)scale % 4 == 0), NF_EALIGN, "dx and q want 16-byte boundaries");
  NF_REQUIRE(p.total() == 0 || (workspace != nullptr && workspace_bytes >= p.total() && (uintptr_t)workspace % 16 == 0), NF_EINVAL,
             "this call needs a workspace of %lld bytes on a 16-byte boundary", (long long)p.total());
  hipStream_t s = (hipStream_t)stream;
  return dtype == NF_F16
             ? bwd<F16>(p, dy, dy_stride, q, scale, w, w_stride, dx, dw, dw_dtype, db, db_dtype, rows, n, k, act, (char*)workspace, s)
             : bwd<BF16>(p, dy, dy_stride, q, scale, w, w_stride, dx, dw, dw_dtype, db, db_dtype, rows, n, k, act, (char*)workspace, s);
}
