// Product of 8-bit rows and 8-bit weight rows with a scale for each row of either, bias and activation behind it:
//
//   y[m, n] = act(s[m] t[n] sum_k q[m, k] w[n, k] + b[n])
//
// The sums are exact: 32-bit integers up to 131071 products of at most 2^14.
//
// Up to 64 rows the time is that of reading the weights once: int8_few_rows_k, no LDS for the operands, the summed dimension split over the waves of
// a workgroup; 1 x 4096 x 16384 13.8 us (67 MB, 4.8 TB/s), 19 x 5000 x 4098 10.4 (1.9 TB/s: loads that start off 16 bytes, and three fifths of the chip).  Beyond, tiles on the 8-bit matrix instructions (gemm_tile.h); where the tiles are too few for the chip, the summed
// dimension is split over workgroups, whose integer sums a second kernel adds up (integers: any order gives the same bits).  16384 x 8192 x 8192 798 - 848 us by
// the card (2590 - 2760 Tops/s), 2048 x 4096 x 4096 35 - 38 (1810 - 1960: one round of small tiles, half of it on the way in and out).
#include "gemm_tile.h"

namespace nf {

struct Epilogue {
  const float *s, *t;
  const void* bias;
  void* y;
  int64_t ldy;
  int bias_dt, y_dt, act, m, n;
};

// What eight columns share: their scales and biases (zeros without any).
struct Columns {
  float t[8], b[8];
  __device__ __forceinline__ Columns(const Epilogue& e, int n) {
    vector8(e.t, NF_F32, n, e.n, t);
    if (e.bias != nullptr) vector8(e.bias, e.bias_dt, n, e.n, b);
    else
#pragma unroll
      for (int i = 0; i < 8; ++i) b[i] = 0.0f;
  }
};
// eight columns of a row, whose scale is s
template <int ACT, typename YT>
__device__ __forceinline__ void put8(const Epilogue& e, int m, int n, const int (&sum)[8], float s, const Columns& c) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = act_value<ACT>(fmaf((float)sum[i], s * c.t[i], c.b[i]));
  store8<YT>((typename YT::storage*)e.y + (int64_t)m * e.ldy + n, e.n - n, v);
}

// body(activation, type of y) under one branch that is the same for every thread
template <typename Body>
__device__ __forceinline__ void with_epilogue(const Epilogue& e, Body&& body) {
  with_act(e.act, [&](auto act_c) {
    if (e.y_dt == NF_F32) body(act_c, F32{});
    else if (e.y_dt == NF_F16) body(act_c, F16{});
    else body(act_c, BF16{});
  });
}

// ---- few rows -----------------------------------------------------------------------------------
struct FewRows {
  const char *q, *w;
  int64_t ldq, ldw;
  int k;
  Epilogue e;
};

// 16 MT rows and 16 NT columns a workgroup.  A wave's unit is 256 bytes of each row, 64 bytes in each of four loads (the four groups of sixteen
// lanes take neighbouring pieces); the units are dealt to the W waves in turn, and their sums meet in LDS.
template <int MT, int NT, int W>
__global__ __launch_bounds__(64 * W) void int8_few_rows_k(FewRows a) {
  __shared__ int part[W][MT * NT][4][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16 * NT;
  const char *wp[NT], *qp[MT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int n = n0 + 16 * j + r;
    wp[j] = a.w + (int64_t)(n < a.e.n ? n : a.e.n - 1) * a.ldw;
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = 16 * i + r;
    qp[i] = a.q + (int64_t)(m < a.e.m ? m : a.e.m - 1) * a.ldq;
  }
  i32x4_t acc[MT][NT] = {};
  struct Unit {
    i32x4_t w[NT][4], q[MT][4];
  };
  const auto load = [&](Unit& f, int u, auto whole_c) {
    const int k = u * 256 + g * 16;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        if constexpr (decltype(whole_c)::value != 0) __builtin_memcpy(&f.w[j][s], wp[j] + k + 64 * s, 16);
        else f.w[j][s] = load16(wp[j], k + 64 * s, a.k);
      }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        if constexpr (decltype(whole_c)::value != 0) __builtin_memcpy(&f.q[i][s], qp[i] + k + 64 * s, 16);
        else f.q[i][s] = load16(qp[i], k + 64 * s, a.k);
      }
  };
  const auto multiply = [&](const Unit& f) {
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = Mma<I8>::run(f.w[j][s], f.q[i][s], acc[i][j]);
  };
  // (the scales and biases of the results that this thread will write are asked for before anything else)
  static_assert(MT * NT * 32 <= 64 * W, "a thread for every eight results");
  const int ej = threadIdx.x % (2 * NT), em = threadIdx.x / (2 * NT), en = n0 + 8 * ej;  // columns 8 j.. of row m
  const bool writes = em < 16 * MT && em < a.e.m && en < a.e.n;
  const Columns columns(a.e, writes ? en : a.e.n);
  const float es = writes ? a.e.s[em] : 0.0f;
  const int units = (a.k + 255) / 256;
  const auto load_any = [&](Unit& f, int u) {
    if ((u + 1) * 256 <= a.k) load(f, u, Int<1>{});
    else load(f, u, Int<0>{});
  };
  int u = wave;
  if constexpr (MT * NT <= 2) {  // two units' loads at once
    for (; u + W < units; u += 2 * W) {
      Unit f, h;
      load(f, u, Int<1>{});
      load_any(h, u + W);
      multiply(f);
      multiply(h);
    }
  }
  for (; u < units; u += W) {
    Unit f;
    load_any(f, u);
    multiply(f);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) part[wave][i * NT + j][c][lane] = acc[i][j][c];
  __syncthreads();
  // a thread adds up eight neighbouring columns of a row: lane and numbers as the matrix instruction left them
  if (!writes) return;
  const int from = (ej & 1) * 32 + (em & 15), tile = (em >> 4) * NT + (ej >> 1);
  int sum[8] = {};
#pragma unroll
  for (int v = 0; v < W; ++v)
#pragma unroll
    for (int c = 0; c < 8; ++c) sum[c] += part[v][tile][c & 3][from + (c >> 2) * 16];
  with_epilogue(a.e, [&](auto act_c, auto y_c) { put8<decltype(act_c)::value, decltype(y_c)>(a.e, em, en, sum, es, columns); });
}

// ---- tiles --------------------------------------------------------------------------------------
template <typename G>
__global__ __launch_bounds__(G::THREADS, G::WAVES_SIMD) void int8_tile_k(GemmArgs g, Epilogue e, int* slots) {
  __shared__ __attribute__((aligned(1024))) char lds[G::LDS];
  i32x4_t acc[G::FM][G::FN] = {};
  const Tile t = tile_of(g, blockIdx.x);
  G::run(g, t, lds, acc);
  const int n = G::column(t);
  if (slots != nullptr) {  // [split][m][n rounded up to 8]
    const int64_t ld = (g.n + 7) / 8 * 8;
    int* o = slots + (int64_t)t.split * g.m * ld + n;
    G::each8(t, lds, acc, [](int) { return 0; }, [&](auto&& rows) {
      rows([&](int m, const int (&v)[8], int) {
        if (m < g.m && n < g.n) __builtin_memcpy(__builtin_assume_aligned(o + (int64_t)m * ld, 16), v, 32);
      });
    });
    return;
  }
  const Columns columns(e, n);
  G::each8(t, lds, acc, [&](int m) { return e.s[m < g.m ? m : g.m - 1]; }, [&](auto&& rows) {
    with_epilogue(e, [&](auto act_c, auto y_c) {
      rows([&](int m, const int (&v)[8], float s) {
        if (m < g.m && n < g.n) put8<decltype(act_c)::value, decltype(y_c)>(e, m, n, v, s, columns);
      });
    });
  });
}

__global__ __launch_bounds__(256) void int8_sum_k(const int* slots, int splits, Epilogue e) {
  const int64_t parts = (e.n + 7) / 8, ld = parts * 8, each = (int64_t)e.m * ld;
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= e.m * parts) return;
  const int m = (int)(at / parts), n = (int)(at % parts) * 8;
  int sum[8] = {};
  for (int k = 0; k < splits; ++k) {
    const int* p = slots + k * each + (int64_t)m * ld + n;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] += p[i];
  }
  const Columns columns(e, n);
  const float s = e.s[m];
  with_epilogue(e, [&](auto act_c, auto y_c) { put8<decltype(act_c)::value, decltype(y_c)>(e, m, n, sum, s, columns); });
}

template <int J>
__global__ __launch_bounds__(256) void pack_rows_k(Copy a, Copy b) {
  const int64_t block = block_number();
  if (block < a.blocks) copy_rows<J>(block, a);
  else if (block - a.blocks < b.blocks) copy_rows<J>(block - a.blocks, b);
}

int pack_rows(const Pack& a, const Pack& b, hipStream_t s) {
  const auto pieces = [](const Pack& p) { return p.to == nullptr ? 0 : p.rows * ((p.bytes + 15) / 16); };
  const int each = cut_pieces(pieces(a) + pieces(b));
  const auto copy = [&](const Pack& p) { return p.to == nullptr ? Copy{} : copy_of(p.from, p.ld, p.rows, p.bytes, p.to, each); };
  const Copy ca = copy(a), cb = copy(b);
  const dim3 grid = grid_of(ca.blocks + cb.blocks);
  if (each == 1) hipLaunchKernelGGL((pack_rows_k<1>), grid, dim3(256), 0, s, ca, cb);
  else hipLaunchKernelGGL((pack_rows_k<4>), grid, dim3(256), 0, s, ca, cb);
  return check_launch("pack_rows");
}

constexpr int FEW_ROWS = 64;

struct Plan {
  bool few;
  TilePlan tile;
  int64_t q_bytes, w_bytes;  // of packed copies
  int64_t total() const { return q_bytes + w_bytes + tile.slot_bytes; }
};

Plan plan(const void* q, int64_t ldq, const void* w, int64_t ldw, int64_t m, int64_t n, int64_t k) {
  Plan p{};
  p.few = m <= FEW_ROWS;
  if (p.few) return p;
  if (!rows_fit(q, ldq, k)) p.q_bytes = round_up(m * round_up(k, 16), 256);
  if (!rows_fit(w, ldw, k)) p.w_bytes = round_up(n * round_up(k, 16), 256);
  p.tile = tile_plan(m, n, k);
  return p;
}

template <int BM, int BN, int WM, int WN>
int tile_launch(GemmArgs g, const Epilogue& e, int* slots, hipStream_t s) {
  typedef Gemm<I8, BM, BN, WM, WN> G;
  g.tiles_m = (g.m + BM - 1) / BM;
  g.tiles_n = (g.n + BN - 1) / BN;
  hipLaunchKernelGGL((int8_tile_k<G>), dim3((unsigned)(g.tiles_m * g.tiles_n * g.splits)), dim3(G::THREADS), 0, s, g, e, slots);
  return check_launch("int8_linear");
}

}  // namespace nf

using namespace nf;

extern "C" int64_t nf_int8_linear_workspace_bytes(const int8_t* q, int64_t q_stride, const int8_t* w, int64_t w_stride, int64_t rows, int64_t n, int64_t k) {
  if (rows <= 0 || n <= 0 || k <= 0 || rows >= (1ll << 31) || n > MOST_WIDTH || k > 131071) return 0;
  return plan(q, q_stride, w, w_stride, rows, n, k).total();
}

extern "C" int nf_int8_linear(const int8_t* q, int64_t q_stride, const float* scale, const int8_t* w, int64_t w_stride, const float* w_scale,
                              const void* bias, int bias_dtype, void* y, int64_t y_stride, int y_dtype, int64_t rows, int64_t n, int64_t k, int act,
                              void* workspace, int64_t workspace_bytes, void* stream) {
  NF_REQUIRE(dtype_ok(y_dtype) && dtype_ok(bias_dtype), NF_EINVAL, "unknown dtype code");
  NF_REQUIRE(act >= NF_ACT_NONE && act <= NF_ACT_GELU, NF_EINVAL, "unknown activation %d", act);
  NF_REQUIRE(rows >= 0 && rows < (1ll << 31), NF_EINVAL, "rows=%lld outside 0..2^31-1", (long long)rows);
  NF_REQUIRE(n >= 1 && n <= MOST_WIDTH, NF_EINVAL, "n=%lld outside 1..2^26", (long long)n);
  NF_REQUIRE(k >= 1, NF_EINVAL, "k=%lld below 1", (long long)k);
  NF_REQUIRE(k <= 131071, NF_EUNSUPPORTED, "k=%lld: more than 131071 products leave a 32-bit integer sum", (long long)k);
  if (rows == 0) return 0;
  NF_REQUIRE(q && scale && w && w_scale && y, NF_EINVAL, "NULL pointer argument");
  NF_REQUIRE((rows == 1 || (q_stride >= k && y_stride >= n)) && (n == 1 || w_stride >= k), NF_EINVAL, "row stride below the row's length");
  const Plan p = plan(q, q_stride, w, w_stride, rows, n, k);
  NF_REQUIRE(p.few || tiles_fit(p.tile, rows, n), NF_EUNSUPPORTED, "rows=%lld, n=%lld: more tiles than a launch holds", (long long)rows, (long long)n);
  NF_REQUIRE(p.total() == 0 || (workspace != nullptr && workspace_bytes >= p.total() && (uintptr_t)workspace % 16 == 0), NF_EINVAL,
             "this call needs a workspace of %lld bytes on a 16-byte boundary", (long long)p.total());
  hipStream_t s = (hipStream_t)stream;
  const Epilogue e{scale, w_scale, bias, y, y_stride, bias_dtype, y_dtype, act, (int)rows, (int)n};
  if (p.few) {
    const FewRows a{(const char*)q, (const char*)w, q_stride, w_stride, (int)k, e};
    const auto go = [&](auto mt, auto nt) {
      constexpr int MT = decltype(mt)::value, NT = decltype(nt)::value;
      hipLaunchKernelGGL((int8_few_rows_k<MT, NT, 8>), dim3((unsigned)((n + 16 * NT - 1) / (16 * NT))), dim3(512), 0, s, a);
    };
    // More columns to a workgroup read the rows less often, but leave compute units idle: the least of what the busiest unit loads.  us with 1, 2, 4 groups
    // of 16 columns: 16 rows x 4096 x 16384 18.9, 17.3, 16.5, x 4096 6.8, 8.1, 12.0; 64 rows 42.8, 31.6, 25.5 and 12.1, 14.2, 21.3;
    // 32 x 5000 x 4098 13.9, 11.0, 16.6.  (Sixteen waves instead of eight: never faster, up to 1.5 times slower.)
    const int mt = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    int nt = 1;
    int64_t least = INT64_MAX;
    for (int t = 1; t <= (rows <= 4 ? 1 : 4); t *= 2) {
      const int64_t blocks = (n + 16 * t - 1) / (16 * t), load = (blocks + 255) / 256 * (t + mt);
      if (load < least) least = load, nt = t;
    }
    const auto by_columns = [&](auto mt_c) {
      if (nt == 1) go(mt_c, Int<1>{});
      else if (nt == 2) go(mt_c, Int<2>{});
      else go(mt_c, Int<4>{});
    };
    if (mt == 1) by_columns(Int<1>{});
    else if (mt == 2) by_columns(Int<2>{});
    else by_columns(Int<4>{});
    return check_launch("int8_linear");
  }
  char* ws = (char*)workspace;
  const char *a = (const char*)q, *b = (const char*)w;
  int64_t lda = q_stride, ldb = w_stride;
  if (p.q_bytes > 0) a = ws, lda = round_up(k, 16);
  if (p.w_bytes > 0) b = ws + p.q_bytes, ldb = round_up(k, 16);
  if (p.q_bytes + p.w_bytes > 0) {
    const Pack of_q{q, q_stride, rows, k, p.q_bytes > 0 ? ws : nullptr}, of_w{w, w_stride, n, k, p.w_bytes > 0 ? ws + p.q_bytes : nullptr};
    if (const int rc = pack_rows(of_q, of_w, s)) return rc;
  }
  const GemmArgs g{a, b, lda, ldb, (int)rows, (int)n, (int)k, 0, 0, p.tile.splits, p.tile.split_steps};
  int* slots = p.tile.splits > 1 ? (int*)(ws + p.q_bytes + p.w_bytes) : nullptr;
  // (four waves of 128 x 128 in 8 bits: 1020 us instead of 820, the compiler moves accumulators about inside the loop)
  const int rc = p.tile.bm == 256 ? tile_launch<256, 256, 4, 2>(g, e, slots, s) : tile_launch<128, 128, 2, 2>(g, e, slots, s);
  if (rc != 0 || slots == nullptr) return rc;
  hipLaunchKernelGGL(int8_sum_k, dim3((unsigned)((rows * ((n + 7) / 8) + 255) / 256)), dim3(256), 0, s, slots, p.tile.splits, e);
  return check_launch("int8_sum");
}
