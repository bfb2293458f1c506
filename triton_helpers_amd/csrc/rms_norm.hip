// Root-mean-square norm of rows, with a residual's addition in front and an 8-bit form behind, forward and backward.
//
//   h = x + r;  rstd = (mean(h^2) + eps)^-1/2;  y = h rstd w;  the new residual is h rounded to the residual's type
//   backward, with n = h rstd and g = dy w:  dh = dh' + rstd (g - n mean(g n)),  dw = sum over rows of dy n      (dh': the residual's own)
//
// A stream over HBM: a row is read once, held in registers as float32 through its sums, and written once.  Up to 2048 values a row belongs to
// one wave (sums by lane exchange, no barrier), beyond that to a workgroup; rows that do not fit the registers (above 32768 values, 16384 in the
// backward) are read twice.
// The norm is taken of the unrounded sum; the backward sees the rounded one that was kept (the new residual, which is there anyway: keeping x and the old
// residual in its place would cost a tensor of memory and a ninth of the traffic, and makes a 16-bit dw, whose own rounding is as large, 1.4 times as exact).
//
// 16384 x 4096 bf16 with a residual: forward 96 us (537 MB, 5.6 TB/s; a large copy reaches 4.9, part of this comes out of the memory-side cache), backward 127
// and the sum of its dw 5 (4.2 TB/s); with autograd 229 a step.  5003 x 777 float32: 10.4, 12.5 and 4.2, and the host's 54 - 57 a step.  1 x 4096: 2.8, 6.2 - 6.4 a call.
#include "wide_common.h"

namespace nf {

struct NormFwd {
  const void *x, *r, *w;
  void *y, *h;       // y: the type of x, or int8
  float *scale, *rstd;
  int64_t xs, rs, rows;
  int width, wt;
  float eps;
};

// T threads hold a row, eight values at a time, NV times
template <typename XT, typename RT, int T, int NV, bool EIGHT>
__global__ __launch_bounds__(T < 256 ? 256 : T) void rms_fwd_k(NormFwd a) {
  __shared__ float sums[16];
  __shared__ uint32_t tops[16];
  const int t = threadIdx.x % T;
  const int64_t row = T < 256 ? (int64_t)blockIdx.x * (256 / T) + threadIdx.x / T : blockIdx.x;
  if (row >= a.rows) return;  // up to T = 64: all threads of a row, which meet no barrier
  const auto* x = (const typename XT::storage*)a.x + row * a.xs;
  const auto* r = a.r == nullptr ? nullptr : (const typename RT::storage*)a.r + row * a.rs;
  float h[NV][8], w[NV][8];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * T + t) * 8, n = a.width - c;
    load8<XT>(x + c, n, h[j]);
  }
  if (r != nullptr) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * T + t) * 8, n = a.width - c;
      float v[8];
      load8<RT>(r + c, n, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[j][i] += v[i];
    }
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * T + t) * 8, n = a.width - c;
    if (a.w != nullptr) load8_any(a.w, c, n, a.wt, w[j]);
  }
  float s = 0.0f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fmaf(h[j][i], h[j][i], s);
  if (a.h != nullptr) {
    auto* o = (typename RT::storage*)a.h + row * a.width;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * T + t) * 8;
      store8<RT>(o + c, a.width - c, h[j]);
    }
  }
  s = row_sum<T>(s, sums);
  const float rstd = 1.0f / sqrtf(s / (float)a.width + a.eps);
  if (a.rstd != nullptr && t == 0) a.rstd[row] = rstd;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) h[j][i] = a.w != nullptr ? h[j][i] * rstd * w[j][i] : h[j][i] * rstd;
  if constexpr (EIGHT) {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t b = (j * T + t) * 8 + i < a.width ? magnitude_bits(h[j][i]) : 0u;
        top = top > b ? top : b;
      }
    const EightBit e = eight_bit(row_max<T>(top, tops));
    if (t == 0) a.scale[row] = e.scale;
    int8_t* o = (int8_t*)a.y + row * a.width;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * T + t) * 8;
      store8_q<false>(o + c, a.width - c, h[j], e);
    }
  } else {
    auto* o = (typename XT::storage*)a.y + row * a.width;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * T + t) * 8;
      store8<XT>(o + c, a.width - c, h[j]);
    }
  }
}

// rows of any width: the values are read again for the norm (and once more for the 8-bit form)
template <typename XT, typename RT, bool EIGHT>
__global__ __launch_bounds__(1024) void rms_fwd_wide_k(NormFwd a) {
  __shared__ float sums[16];
  __shared__ uint32_t tops[16];
  const int64_t row = blockIdx.x;
  const auto* x = (const typename XT::storage*)a.x + row * a.xs;
  const auto* r = a.r == nullptr ? nullptr : (const typename RT::storage*)a.r + row * a.rs;
  const auto sum_at = [&](int c, float(&h)[8]) {
    load8<XT>(x + c, a.width - c, h);
    if (r != nullptr) {
      float v[8];
      load8<RT>(r + c, a.width - c, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] += v[i];
    }
  };
  float s = 0.0f;
  for (int c = threadIdx.x * 8; c < a.width; c += 8192) {
    float h[8];
    sum_at(c, h);
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fmaf(h[i], h[i], s);
    if (a.h != nullptr) store8<RT>((typename RT::storage*)a.h + row * a.width + c, a.width - c, h);
  }
  s = row_sum<1024>(s, sums);
  const float rstd = 1.0f / sqrtf(s / (float)a.width + a.eps);
  if (a.rstd != nullptr && threadIdx.x == 0) a.rstd[row] = rstd;
  const auto normed_at = [&](int c, float(&h)[8]) {
    sum_at(c, h);
    float w[8];
    if (a.w != nullptr) load8_any(a.w, c, a.width - c, a.wt, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = a.w != nullptr ? h[i] * rstd * w[i] : h[i] * rstd;
  };
  EightBit e{};
  if constexpr (EIGHT) {
    uint32_t top = 0;
    for (int c = threadIdx.x * 8; c < a.width; c += 8192) {
      float h[8];
      normed_at(c, h);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t b = c + i < a.width ? magnitude_bits(h[i]) : 0u;
        top = top > b ? top : b;
      }
    }
    e = eight_bit(row_max<1024>(top, tops));
    if (threadIdx.x == 0) a.scale[row] = e.scale;
  }
  for (int c = threadIdx.x * 8; c < a.width; c += 8192) {
    float h[8];
    normed_at(c, h);
    if constexpr (EIGHT) {
      store8_q<false>((int8_t*)a.y + row * a.width + c, a.width - c, h, e);
    } else {
      store8<XT>((typename XT::storage*)a.y + row * a.width + c, a.width - c, h);
    }
  }
}

// ---- backward ---------------------------------------------------------------------------------
struct NormBwd {
  const void *dy, *dh, *h, *w;  // dh: the gradient that reached the new residual (NULL: none)
  const float* rstd;
  void *dx, *dr;                // dr: NULL where the residual's gradient is dx
  float* slots;                 // [groups][width] partial sums of dw, NULL without a weight's gradient
  int64_t dys, dhs, hs, rows;
  int width, wt;
};

// HT: the type of h (the residual's, or that of x without one).  A group of T threads walks rows `group`, `group + groups`, ...
template <typename XT, typename HT, int T, int NV>
__global__ __launch_bounds__(T < 256 ? 256 : T) void rms_bwd_k(NormBwd a) {
  __shared__ float sums[2][16];
  constexpr int PER = T < 256 ? 256 / T : 1;  // groups of a workgroup
  __shared__ float others[PER > 1 ? PER - 1 : 1][PER > 1 ? T * NV * 8 : 1];
  const int t = threadIdx.x % T;
  const int64_t groups = (int64_t)gridDim.x * PER, group = blockIdx.x * PER + threadIdx.x / T;
  float dw[NV][8] = {}, w[NV][8];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * T + t) * 8;
    if (a.w != nullptr) load8_any(a.w, c, a.width - c, a.wt, w[j]);
  }
  int turn = 0;
  for (int64_t row = group; row < a.rows; row += groups, turn ^= 1) {
    const auto* dy = (const typename XT::storage*)a.dy + row * a.dys;
    const auto* hp = (const typename HT::storage*)a.h + row * a.hs;
    const float rstd = a.rstd[row];
    float g[NV][8], n[NV][8];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * T + t) * 8;
      load8<XT>(dy + c, a.width - c, g[j]);
      load8<HT>(hp + c, a.width - c, n[j]);
    }
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        n[j][i] *= rstd;
        dw[j][i] = fmaf(g[j][i], n[j][i], dw[j][i]);
        if (a.w != nullptr) g[j][i] *= w[j][i];
        s = fmaf(g[j][i], n[j][i], s);
      }
    const float mean = row_sum<T>(s, sums[turn]) / (float)a.width;  // the next row's sums go to the other half: one barrier a row
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * T + t) * 8;
      float d[8] = {};
      if (a.dh != nullptr) load8<HT>((const typename HT::storage*)a.dh + row * a.dhs + c, a.width - c, d);
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] = fmaf(rstd, fmaf(-n[j][i], mean, g[j][i]), d[i]);
      if (a.dx != nullptr) store8<XT>((typename XT::storage*)a.dx + row * a.width + c, a.width - c, d);
      if (a.dr != nullptr) store8<HT>((typename HT::storage*)a.dr + row * a.width + c, a.width - c, d);
    }
  }
  if (a.slots == nullptr) return;
  if constexpr (PER > 1) {  // the workgroup's groups leave one slot
    if (threadIdx.x >= T) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) others[threadIdx.x / T - 1][(j * 8 + i) * T + t] = dw[j][i];
    }
    __syncthreads();
    if (threadIdx.x >= T) return;
#pragma unroll
    for (int k = 0; k < PER - 1; ++k)
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) dw[j][i] += others[k][(j * 8 + i) * T + t];
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * T + t) * 8;
    store8<F32>(a.slots + (int64_t)blockIdx.x * a.width + c, a.width - c, dw[j]);
  }
}

template <typename XT, typename HT>
__global__ __launch_bounds__(1024) void rms_bwd_wide_k(NormBwd a) {
  __shared__ float sums[2][16];
  int turn = 0;
  bool first = true;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1, first = false) {
    const auto* dy = (const typename XT::storage*)a.dy + row * a.dys;
    const auto* hp = (const typename HT::storage*)a.h + row * a.hs;
    const float rstd = a.rstd[row];
    const auto at = [&](int c, float(&g)[8], float(&n)[8], float(&w)[8]) {
      load8<XT>(dy + c, a.width - c, g);
      load8<HT>(hp + c, a.width - c, n);
      if (a.w != nullptr) load8_any(a.w, c, a.width - c, a.wt, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        n[i] *= rstd;
        if (a.w == nullptr) w[i] = 1.0f;
      }
    };
    float s = 0.0f;
    for (int c = threadIdx.x * 8; c < a.width; c += 8192) {
      float g[8], n[8], w[8];
      at(c, g, n, w);
      if (a.slots != nullptr) {  // a thread's own values of its group's own slot
        float v[8] = {};
        float* slot = a.slots + (int64_t)blockIdx.x * a.width + c;
        if (!first) load8<F32>(slot, a.width - c, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = fmaf(g[i], n[i], v[i]);
        store8<F32>(slot, a.width - c, v);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) s = fmaf(g[i] * w[i], n[i], s);
    }
    const float mean = row_sum<1024>(s, sums[turn]) / (float)a.width;
    for (int c = threadIdx.x * 8; c < a.width; c += 8192) {
      float g[8], n[8], w[8], d[8] = {};
      at(c, g, n, w);
      if (a.dh != nullptr) load8<HT>((const typename HT::storage*)a.dh + row * a.dhs + c, a.width - c, d);
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] = fmaf(rstd, fmaf(-n[i], mean, g[i] * w[i]), d[i]);
      if (a.dx != nullptr) store8<XT>((typename XT::storage*)a.dx + row * a.width + c, a.width - c, d);
      if (a.dr != nullptr) store8<HT>((typename HT::storage*)a.dr + row * a.width + c, a.width - c, d);
    }
  }
}

// column sums of the groups' partial sums, in a fixed order (the same bits on every run)
__global__ __launch_bounds__(1024) void sum_slots_k(const float* slots, int64_t groups, int width, void* out, int dt) {
  __shared__ float part[32][33];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), g = threadIdx.x >> 5;
  float s = 0.0f;
  if (c < width) {
#pragma unroll 8
    for (int64_t k = g; k < groups; k += 32) s += slots[k * width + c];
  }
  part[g][threadIdx.x & 31] = s;
  __syncthreads();
  if (g == 0 && c < width) {
#pragma unroll
    for (int i = 1; i < 32; ++i) s += part[i][threadIdx.x];
    store_any(out, c, dt, s);
  }
}
int sum_slots(const float* slots, int64_t groups, int64_t width, void* out, int dt, hipStream_t s) {
  hipLaunchKernelGGL(sum_slots_k, dim3((unsigned)((width + 31) / 32)), dim3(1024), 0, s, slots, groups, (int)width, out, dt);
  return check_launch("sum_slots");
}

constexpr int NORM_ONE_PASS = 32768;  // the widest row that a workgroup's registers hold
// Threads that share a row.  (A wave's row needs no barrier; a workgroup's asks for a row with more loads at once.)
inline int norm_threads(int width) { return width <= 2048 ? 64 : width <= 8192 ? 256 : 1024; }
// Groups of a backward: each walks as many rows as the others, and a workgroup of them leaves one row of partial sums of dw.
inline int64_t norm_groups(int64_t rows, int width) {
  const int64_t most = width <= 2048 ? 4096 : width <= 8192 ? 1024 : 256, each = (rows + most - 1) / most;
  return (rows + each - 1) / each;
}

template <typename XT, typename RT>
int fwd_launch_some(const NormFwd& a, bool eight, hipStream_t s) {
  const auto go = [&](auto t_c, auto nv_c, auto e_c) {
    constexpr int T = decltype(t_c)::value, NV = decltype(nv_c)::value;
    constexpr bool E = decltype(e_c)::value != 0;
    const int64_t per = T < 256 ? 256 / T : 1, blocks = (a.rows + per - 1) / per;
    hipLaunchKernelGGL((rms_fwd_k<XT, RT, T, NV, E>), dim3((unsigned)blocks), dim3(T < 256 ? 256 : T), 0, s, a);
  };
  const auto by_width = [&](auto e_c) {
    // a few rows: as many threads to each as its values take, for the time of one row is that of its loads and sums
    if (a.rows <= 512 && a.width > 512 && a.width <= 2048) go(Int<256>{}, Int<1>{}, e_c);
    else if (a.rows <= 256 && a.width > 2048 && a.width <= 8192) go(Int<1024>{}, Int<1>{}, e_c);
    else if (a.width <= 128) go(Int<16>{}, Int<1>{}, e_c);
    else if (a.width <= 256) go(Int<32>{}, Int<1>{}, e_c);
    else if (a.width <= 512) go(Int<64>{}, Int<1>{}, e_c);
    else if (a.width <= 1024) go(Int<64>{}, Int<2>{}, e_c);
    else if (a.width <= 2048) go(Int<64>{}, Int<4>{}, e_c);
    else if (a.width <= 4096) go(Int<256>{}, Int<2>{}, e_c);
    else if (a.width <= 8192) go(Int<256>{}, Int<4>{}, e_c);
    else if (a.width <= NORM_ONE_PASS) go(Int<1024>{}, Int<4>{}, e_c);
    else hipLaunchKernelGGL((rms_fwd_wide_k<XT, RT, decltype(e_c)::value != 0>), dim3((unsigned)a.rows), dim3(1024), 0, s, a);
  };
  if (eight) by_width(Int<1>{});
  else by_width(Int<0>{});
  return check_launch("rms_norm_fwd");
}

template <typename XT, typename RT>
int fwd_launch(const NormFwd& a, bool eight, hipStream_t s) {
  typedef typename XT::storage X;
  typedef typename RT::storage R;
  for (int64_t row = 0; row < a.rows; row += MOST_BLOCKS) {
    NormFwd part = a;
    part.rows = a.rows - row < MOST_BLOCKS ? a.rows - row : MOST_BLOCKS;
    part.x = (const X*)a.x + row * a.xs;
    if (a.r != nullptr) part.r = (const R*)a.r + row * a.rs;
    if (a.h != nullptr) part.h = (R*)a.h + row * a.width;
    part.y = (char*)a.y + row * a.width * (eight ? 1 : (int64_t)sizeof(X));
    if (a.scale != nullptr) part.scale = a.scale + row;
    if (a.rstd != nullptr) part.rstd = a.rstd + row;
    if (const int rc = fwd_launch_some<XT, RT>(part, eight, s)) return rc;
  }
  return 0;
}

template <typename XT, typename HT>
int bwd_launch(const NormBwd& a, int64_t groups, hipStream_t s) {
  const auto go = [&](auto t_c, auto nv_c) {
    constexpr int T = decltype(t_c)::value, NV = decltype(nv_c)::value;
    const int64_t per = T < 256 ? 256 / T : 1;
    hipLaunchKernelGGL((rms_bwd_k<XT, HT, T, NV>), dim3((unsigned)((groups + per - 1) / per)), dim3(T < 256 ? 256 : T), 0, s, a);
  };
  if (a.width <= 512) go(Int<64>{}, Int<1>{});
  else if (a.width <= 1024) go(Int<64>{}, Int<2>{});
  else if (a.width <= 2048) go(Int<64>{}, Int<4>{});
  else if (a.width <= 4096) go(Int<256>{}, Int<2>{});
  else if (a.width <= 8192) go(Int<256>{}, Int<4>{});
  else if (a.width <= NORM_ONE_PASS / 2) go(Int<1024>{}, Int<2>{});  // three rows of values: four vectors each would spill
  else hipLaunchKernelGGL((rms_bwd_wide_k<XT, HT>), dim3((unsigned)groups), dim3(1024), 0, s, a);
  return check_launch("rms_norm_bwd");
}

// the slots that the launch writes: one for each workgroup
inline int64_t slot_rows(int64_t rows, int width) {
  const int64_t g = norm_groups(rows, width);
  return norm_threads(width) == 64 ? (g + 3) / 4 : g;
}

}  // namespace nf

using namespace nf;

extern "C" int nf_rms_norm_fwd(const void* x, int64_t x_stride, int x_dtype, const void* residual, int64_t residual_stride, int residual_dtype,
                               const void* weight, int weight_dtype, void* y, float* scale, void* new_residual, float* rstd, int64_t rows,
                               int64_t width, float eps, void* stream) {
  NF_REQUIRE(dtype_ok(x_dtype) && dtype_ok(residual_dtype) && dtype_ok(weight_dtype), NF_EINVAL, "unknown dtype code");
  NF_REQUIRE(residual_dtype == x_dtype || residual_dtype == NF_F32, NF_EUNSUPPORTED, "the residual is of the rows' type or float32");
  NF_REQUIRE(rows >= 0 && rows < (1ll << 31), NF_EINVAL, "rows=%lld outside 0..2^31-1", (long long)rows);
  NF_REQUIRE(width >= 1 && width <= MOST_WIDTH, NF_EINVAL, "width=%lld outside 1..2^26", (long long)width);
  NF_REQUIRE(eps >= 0.0f, NF_EINVAL, "eps must be >= 0");
  if (rows == 0) return 0;
  NF_REQUIRE(x && y, NF_EINVAL, "NULL pointer argument");
  NF_REQUIRE(rows == 1 || (x_stride >= width && (residual == nullptr || residual_stride >= width)), NF_EINVAL, "row stride below the width");
  NF_REQUIRE(new_residual == nullptr || residual != nullptr, NF_EINVAL, "a new residual without a residual");
  const NormFwd a{x, residual, weight, y, new_residual, scale, rstd, x_stride, residual_stride, rows, (int)width, weight_dtype, eps};
  const bool eight = scale != nullptr;
  hipStream_t s = (hipStream_t)stream;
  if (x_dtype == NF_F32) return fwd_launch<F32, F32>(a, eight, s);
  const bool wide = residual != nullptr && residual_dtype == NF_F32;
  if (x_dtype == NF_F16) return wide ? fwd_launch<F16, F32>(a, eight, s) : fwd_launch<F16, F16>(a, eight, s);
  return wide ? fwd_launch<BF16, F32>(a, eight, s) : fwd_launch<BF16, BF16>(a, eight, s);
}

extern "C" int64_t nf_rms_norm_bwd_workspace_bytes(int64_t rows, int64_t width) {
  if (rows <= 0 || width < 1 || width > MOST_WIDTH) return 0;
  return slot_rows(rows, (int)width) * width * 4;
}

extern "C" int nf_rms_norm_bwd(const void* dy, int64_t dy_stride, int x_dtype, const void* d_residual, int64_t d_residual_stride, const void* h,
                               int64_t h_stride, int h_dtype, const float* rstd, const void* weight, int weight_dtype, void* dx, void* dr, void* dw,
                               int64_t rows, int64_t width, void* workspace, int64_t workspace_bytes, void* stream) {
  NF_REQUIRE(dtype_ok(x_dtype) && dtype_ok(h_dtype) && dtype_ok(weight_dtype), NF_EINVAL, "unknown dtype code");
  NF_REQUIRE(h_dtype == x_dtype || h_dtype == NF_F32, NF_EUNSUPPORTED, "the residual is of the rows' type or float32");
  NF_REQUIRE(rows >= 0 && rows < (1ll << 31), NF_EINVAL, "rows=%lld outside 0..2^31-1", (long long)rows);
  NF_REQUIRE(width >= 1 && width <= MOST_WIDTH, NF_EINVAL, "width=%lld outside 1..2^26", (long long)width);
  NF_REQUIRE(dw == nullptr || weight != nullptr, NF_EINVAL, "a weight's gradient without a weight");
  if (rows == 0) {
    NF_REQUIRE(dw == nullptr, NF_EINVAL, "no rows: the weight's gradient is the caller's to clear");
    return 0;
  }
  NF_REQUIRE(dy && h && rstd, NF_EINVAL, "NULL pointer argument");
  NF_REQUIRE(rows == 1 || (dy_stride >= width && h_stride >= width && (d_residual == nullptr || d_residual_stride >= width)), NF_EINVAL,
             "row stride below the width");
  NF_REQUIRE(dw == nullptr || (workspace != nullptr && workspace_bytes >= nf_rms_norm_bwd_workspace_bytes(rows, width) && (uintptr_t)workspace % 4 == 0),
             NF_EINVAL, "the weight's gradient needs a workspace of %lld bytes", (long long)nf_rms_norm_bwd_workspace_bytes(rows, width));
  const NormBwd a{dy, d_residual, h, weight, rstd, dx, dr, dw == nullptr ? nullptr : (float*)workspace, dy_stride, d_residual_stride, h_stride, rows,
                  (int)width, weight_dtype};
  hipStream_t s = (hipStream_t)stream;
  const int64_t groups = norm_groups(rows, (int)width);
  int rc;
  if (x_dtype == NF_F32) rc = bwd_launch<F32, F32>(a, groups, s);
  else if (x_dtype == NF_F16) rc = h_dtype == NF_F32 ? bwd_launch<F16, F32>(a, groups, s) : bwd_launch<F16, F16>(a, groups, s);
  else rc = h_dtype == NF_F32 ? bwd_launch<BF16, F32>(a, groups, s) : bwd_launch<BF16, BF16>(a, groups, s);
  if (rc != 0 || dw == nullptr) return rc;
  return sum_slots((const float*)workspace, slot_rows(rows, (int)width), width, dw, weight_dtype, s);
}
