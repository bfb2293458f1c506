// Rows as 8-bit integers with one scale each, q = rint(v (127 / a)) and s = a / 127 with a the largest magnitude of the row, and next to them, on
// request, act(v) in the rows' own type with rows padded to whole 16-byte pieces (the operand of the product that the rows go into).
//
// A stream over HBM: a row is read once and held in registers between its maximum and its rounding; rows above 32768 values are read twice.  Short rows
// share a wave (2^18 x 256 57 us instead of 107).  16384 x 4096 bf16 with GELU: 61 us, 335 MB at 5.5 TB/s.
#include "gemm_tile.h"

namespace nf {

struct Quantize {
  const void* x;
  int8_t* q;  // NULL: h alone
  float* scale;
  void* h;  // NULL, or rows of x's type with `hs` values between them; values behind the row's end become zeros
  int64_t xs, hs, rows;
  int width;
  Copy also;  // next to h: rows of another operand, by workgroups behind those of the rows (a launch less for a small layer)
  unsigned row_blocks;
};

template <typename XT, int ACT>
__device__ __forceinline__ void put_act(const Quantize& a, int64_t row, int c, const float (&v)[8]) {
  if (c >= a.hs) return;
  float h[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = c + i < a.width ? act_value<ACT>(v[i]) : 0.0f;
  store8<XT>((typename XT::storage*)a.h + row * a.hs + c, (int)(a.hs - c < 8 ? a.hs - c : 8), h);
}

template <typename XT, int T, int NV, int ACT, bool KEEP>
__global__ __launch_bounds__(T < 256 ? 256 : T) void quantize_k(Quantize a) {
  __shared__ uint32_t tops[16];
  if constexpr (KEEP) {
    if (blockIdx.x >= a.row_blocks) {
      if (threadIdx.x < 256) copy_rows<1>(blockIdx.x - a.row_blocks, a.also);
      return;
    }
  }
  const int t = threadIdx.x % T;
  const int64_t row = T < 256 ? (int64_t)blockIdx.x * (256 / T) + threadIdx.x / T : blockIdx.x;
  if (row >= a.rows) return;  // up to T = 64: all threads of a row, which meet no barrier
  const auto* x = (const typename XT::storage*)a.x + row * a.xs;
  float v[NV][8];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * T + t) * 8;
    load8<XT>(x + c, a.width - c, v[j]);  // zeros behind the end
  }
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t b = magnitude_bits(v[j][i]);
      top = top > b ? top : b;
    }
  if constexpr (KEEP) {
#pragma unroll
    for (int j = 0; j < NV; ++j) put_act<XT, ACT>(a, row, (j * T + t) * 8, v[j]);
    if (a.q == nullptr) return;
  }
  const EightBit e = eight_bit(row_max<T>(top, tops));
  if (t == 0) a.scale[row] = e.scale;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * T + t) * 8;
    store8_q<sizeof(typename XT::storage) == 2>(a.q + row * a.width + c, a.width - c, v[j], e);
  }
}

template <typename XT, int ACT, bool KEEP>
__global__ __launch_bounds__(1024) void quantize_wide_k(Quantize a) {
  __shared__ uint32_t tops[16];
  const int64_t row = blockIdx.x;
  const auto* x = (const typename XT::storage*)a.x + row * a.xs;
  uint32_t top = 0;
  for (int c = threadIdx.x * 8; c < a.width; c += 8192) {
    float v[8];
    load8<XT>(x + c, a.width - c, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t b = magnitude_bits(v[i]);
      top = top > b ? top : b;
    }
    if constexpr (KEEP) put_act<XT, ACT>(a, row, c, v);
  }
  if (KEEP && a.q == nullptr) return;
  const EightBit e = eight_bit(row_max<1024>(top, tops));
  if (threadIdx.x == 0) a.scale[row] = e.scale;
  for (int c = threadIdx.x * 8; c < a.width; c += 8192) {
    float v[8];
    load8<XT>(x + c, a.width - c, v);
    store8_q<sizeof(typename XT::storage) == 2>(a.q + row * a.width + c, a.width - c, v, e);
  }
}

template <typename XT, int ACT, bool KEEP>
int quantize_launch_some(Quantize a, hipStream_t s) {
  const auto go = [&](auto t_c, auto nv_c) {
    constexpr int T = decltype(t_c)::value, NV = decltype(nv_c)::value;
    const int64_t per = T < 256 ? 256 / T : 1;
    a.row_blocks = (unsigned)((a.rows + per - 1) / per);
    hipLaunchKernelGGL((quantize_k<XT, T, NV, ACT, KEEP>), dim3(a.row_blocks + (unsigned)a.also.blocks), dim3(T < 256 ? 256 : T), 0, s, a);
  };
  // a few rows: as many threads to each as its values take
  if (a.rows <= 512 && a.width > 512 && a.width <= 2048) go(Int<256>{}, Int<1>{});
  else if (a.rows <= 256 && a.width > 2048 && a.width <= 8192) go(Int<1024>{}, Int<1>{});
  else if (a.width <= 128) go(Int<16>{}, Int<1>{});
  else if (a.width <= 256) go(Int<32>{}, Int<1>{});
  else if (a.width <= 512) go(Int<64>{}, Int<1>{});
  else if (a.width <= 1024) go(Int<64>{}, Int<2>{});
  else if (a.width <= 2048) go(Int<64>{}, Int<4>{});
  else if (a.width <= 4096) go(Int<256>{}, Int<2>{});
  else if (a.width <= 8192) go(Int<256>{}, Int<4>{});
  else if (a.width <= 32768) go(Int<1024>{}, Int<4>{});
  else hipLaunchKernelGGL((quantize_wide_k<XT, ACT, KEEP>), dim3((unsigned)a.rows), dim3(1024), 0, s, a);
  return check_launch("quantize_rows");
}

template <typename XT, int ACT, bool KEEP>
int quantize_launch(const Quantize& a, hipStream_t s) {
  typedef typename XT::storage X;
  for (int64_t row = 0; row < a.rows; row += MOST_BLOCKS) {
    Quantize part = a;
    part.rows = a.rows - row < MOST_BLOCKS ? a.rows - row : MOST_BLOCKS;
    part.x = (const X*)a.x + row * a.xs;
    if (a.q != nullptr) part.q = a.q + row * a.width, part.scale = a.scale + row;
    if (a.h != nullptr) part.h = (X*)a.h + row * a.hs;
    if (row > 0) part.also.blocks = 0;
    if (const int rc = quantize_launch_some<XT, ACT, KEEP>(part, s)) return rc;
  }
  return 0;
}

template <typename XT>
int quantize_by_act(const Quantize& a, int act, hipStream_t s) {
  if (a.h == nullptr) return quantize_launch<XT, NF_ACT_NONE, false>(a, s);
  switch (act) {
    case NF_ACT_RELU: return quantize_launch<XT, NF_ACT_RELU, true>(a, s);
    case NF_ACT_RELU2: return quantize_launch<XT, NF_ACT_RELU2, true>(a, s);
    case NF_ACT_SILU: return quantize_launch<XT, NF_ACT_SILU, true>(a, s);
    case NF_ACT_GELU: return quantize_launch<XT, NF_ACT_GELU, true>(a, s);
    default: return quantize_launch<XT, NF_ACT_NONE, true>(a, s);
  }
}

int quantize_and_copy(const void* x, int64_t xs, int dtype, int8_t* q, float* scale, void* h, int64_t hs, int act, int64_t rows, int64_t width, const Copy& also,
                      hipStream_t s) {
  const Quantize a{x, q, scale, h, xs, hs, rows, (int)width, also, 0};
  if (dtype == NF_F32) return quantize_by_act<F32>(a, act, s);
  if (dtype == NF_F16) return quantize_by_act<F16>(a, act, s);
  return quantize_by_act<BF16>(a, act, s);
}

}  // namespace nf

using namespace nf;

extern "C" int nf_quantize_rows(const void* x, int64_t x_stride, int x_dtype, int8_t* q, float* scale, void* h, int64_t h_stride, int act, int64_t rows,
                                int64_t width, void* stream) {
  NF_REQUIRE(dtype_ok(x_dtype), NF_EINVAL, "unknown dtype code %d", x_dtype);
  NF_REQUIRE(act >= NF_ACT_NONE && act <= NF_ACT_GELU, NF_EINVAL, "unknown activation %d", act);
  NF_REQUIRE(rows >= 0 && rows < (1ll << 31), NF_EINVAL, "rows=%lld outside 0..2^31-1", (long long)rows);
  NF_REQUIRE(width >= 1 && width <= MOST_WIDTH, NF_EINVAL, "width=%lld outside 1..2^26", (long long)width);
  NF_REQUIRE(h == nullptr || h_stride == width || h_stride == (width + 7) / 8 * 8, NF_EINVAL, "h_stride=%lld: the width, or the next multiple of 8",
             (long long)h_stride);
  if (rows == 0) return 0;
  NF_REQUIRE(x && (q ? scale != nullptr : h != nullptr), NF_EINVAL, "NULL pointer argument");
  NF_REQUIRE(rows == 1 || x_stride >= width, NF_EINVAL, "row stride below the width");
  return quantize_and_copy(x, x_stride, x_dtype, q, scale, h, h_stride, act, rows, width, Copy{}, (hipStream_t)stream);
}
