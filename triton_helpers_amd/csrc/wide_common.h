// What the kernels of the wide layers (norm, 8-bit rows, products) share: eight values of a row at a time, sums over the threads of a row,
// the 8-bit form of a row, and the activations.
#pragma once

#include <type_traits>

#include "mlp_tile.h"
#include "nf_common.h"

namespace nf {

// Eight consecutive values from any address of their type: one or two 16-byte loads (this chip takes them off 16-byte boundaries), or the n
// that are left of a row, and zeros.
template <typename T>
__device__ __forceinline__ void load8(const typename T::storage* p, int n, float (&v)[8]) {
  typename T::storage raw[8];
  if (n >= 8) {
    __builtin_memcpy(raw, p, sizeof raw);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) raw[i] = i < n ? p[i] : typename T::storage(0);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = T::to_f32(raw[i]);
}
template <typename T>
__device__ __forceinline__ void store8(typename T::storage* p, int n, const float (&v)[8]) {
  typename T::storage raw[8];
  if constexpr (std::is_same<T, F32>::value) {
#pragma unroll
    for (int i = 0; i < 8; ++i) raw[i] = v[i];
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = T::pack(v[2 * i], v[2 * i + 1]);
    __builtin_memcpy(raw, w, sizeof raw);
  }
  if (n >= 8) {
    __builtin_memcpy(p, raw, sizeof raw);
  } else {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < n) p[i] = raw[i];
  }
}
// eight values of a type that is known at run time only (a norm's weight; the branch is the same for every thread)
__device__ __forceinline__ void load8_any(const void* p, int64_t at, int n, int dt, float (&v)[8]) {
  if (dt == NF_F32) load8<F32>((const float*)p + at, n, v);
  else if (dt == NF_F16) load8<F16>((const uint16_t*)p + at, n, v);
  else load8<BF16>((const uint16_t*)p + at, n, v);
}
__device__ __forceinline__ void store_any(void* p, int64_t at, int dt, float v) {
  if (dt == NF_F32) ((float*)p)[at] = v;
  else ((uint16_t*)p)[at] = dt == NF_F16 ? F16::from_f32(v) : BF16::from_f32(v);
}

// ---- over the T threads of a row (up to 64: neighbouring lanes of a wave; else the whole workgroup) -----------------
// (lane exchanges inside the vector unit: through LDS each costs some hundred clocks, one behind the other)
template <int CTRL>
__device__ __forceinline__ uint32_t moved(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false);
}
template <int T, typename V, typename Join>
__device__ __forceinline__ V lanes_join(V v, Join&& join) {
  const auto bits = [](V x) { return __builtin_bit_cast(uint32_t, x); };
  const auto value = [](uint32_t x) { return __builtin_bit_cast(V, x); };
  if constexpr (T >= 2) v = join(v, value(moved<0xb1>(bits(v))));    // neighbours in pairs
  if constexpr (T >= 4) v = join(v, value(moved<0x4e>(bits(v))));    // pairs in fours
  if constexpr (T >= 8) v = join(v, value(moved<0x141>(bits(v))));   // mirrored eights
  if constexpr (T >= 16) v = join(v, value(moved<0x140>(bits(v))));  // mirrored sixteens
  if constexpr (T >= 32) {  // odd sixteens against even ones
    const auto w = __builtin_amdgcn_permlane16_swap(bits(v), bits(v), false, false);
    v = join(value(w[0]), value(w[1]));
  }
  if constexpr (T >= 64) {
    const auto w = __builtin_amdgcn_permlane32_swap(bits(v), bits(v), false, false);
    v = join(value(w[0]), value(w[1]));
  }
  return v;
}
template <int T>
__device__ __forceinline__ float lanes_sum(float v) {
  return lanes_join<T>(v, [](float x, float y) { return x + y; });
}
template <int T>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  return lanes_join<T>(v, [](uint32_t x, uint32_t y) { return x > y ? x : y; });
}
// `shared`: T / 64 values of its own for every call between two barriers
template <int T>
__device__ __forceinline__ float row_sum(float v, float* shared) {
  v = lanes_sum<T < 64 ? T : 64>(v);
  if constexpr (T > 64) {
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < T / 64; ++i) v += shared[i];
  }
  return v;
}
template <int T>
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* shared) {
  v = lanes_max<T < 64 ? T : 64>(v);
  if constexpr (T > 64) {
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < T / 64; ++i) v = v > shared[i] ? v : shared[i];
  }
  return v;
}

// Rows go to launches of at most 2^21 workgroups (a grid of 2^32 threads is refused).
constexpr int64_t MOST_BLOCKS = 1 << 21;
constexpr int64_t MOST_WIDTH = 1 << 26;

// ---- the 8-bit form of a row ----------------------------------------------------------------
// q = rint(v * (127 / a)), s = a / 127, a the largest magnitude.  The magnitudes are compared as bit patterns, in which infinities come
// behind every number and NaN behind them: a row that holds either has no 8-bit form, its scale becomes NaN and with it whatever is
// made of the row.  A row of magnitudes below 2^-120, whose 127 / a would leave float32, counts as zeros.
__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
struct EightBit {
  float scale, inverse;
};
__device__ __forceinline__ EightBit eight_bit(uint32_t largest) {
  const float a = __uint_as_float(largest);
  if (largest >= 0x7f800000u) return {__uint_as_float(0x7fc00000u), 0.0f};
  if (a < 7.5231638e-37f) return {0.0f, 0.0f};
  return {a / 127.0f, 127.0f / a};
}
// Eight values of a row as bytes.  What is added puts the product, rounded to a whole number (half to even, as rint does), into the low byte of its bits.  In a row
// without a form (inverse = 0) infinities and NaN become zeros: NaN that came from 16 bits, and those of the chip, have nothing in their low byte.
template <bool FROM16>
__device__ __forceinline__ void quantized8(const float (&v)[8], EightBit e, uint32_t (&q)[2]) {
#pragma clang fp contract(off)
  uint32_t b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float product = v[i] * e.inverse;
    b[i] = __float_as_uint(product + 12582912.0f);
    if (!FROM16 && e.inverse == 0.0f) b[i] = 0;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t lo = __builtin_amdgcn_perm(b[4 * i + 1], b[4 * i], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[4 * i + 3], b[4 * i + 2], 0x0c0c0400u);
    q[i] = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
  }
}
template <bool FROM16>
__device__ __forceinline__ void store8_q(int8_t* p, int n, const float (&v)[8], EightBit e) {
  uint32_t q[2];
  quantized8<FROM16>(v, e, q);
  if (n >= 8) {
    __builtin_memcpy(p, q, 8);
  } else {
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < n) p[i] = (int8_t)(q[i / 4] >> (i % 4 * 8));
  }
}
// ... and back: s q.  (A byte less 128 is exact, so nothing is rounded but the result.  As one multiplication and addition, s byte - 128 s, a row with
// the largest bfloat16 values would have no finite 128 s.)
__device__ __forceinline__ void kept8(const int (&q)[2], float s, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = s * ((float)(uint8_t)(((uint32_t)q[i / 4] ^ 0x80808080u) >> (i % 4 * 8)) - 128.0f);
}
// the largest magnitude of eight 16-bit values, in their type's bits
__device__ __forceinline__ uint16_t largest16(const uint32_t (&v)[4]) {
  typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
  u16x2_t m = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2_t, v[i] & 0x7fff7fffu));
  return m[0] > m[1] ? m[0] : m[1];
}

// ---- activations ------------------------------------------------------------------------------
// As act_fwd / act_grad, which are made for 16-bit results, but for a GELU that is right to 1.5e-7, and a NaN stays one.
// Phi(-|z|) = q e with e = exp(-z^2 / 2) (Abramowitz & Stegun 7.1.26 with the scales of erfc folded into its constants).  The streams that
// apply a GELU to 16-bit rows spend as long on its instructions as on their memory, so each one counts: no compare, no select.
__device__ __forceinline__ float normal_tail(float z, float* e) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.23164189f, fabsf(z), 1.0f));
  *e = __builtin_amdgcn_exp2f(z * (z * -0.72134752f));
  return t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 0.5307027145f, -0.7265760135f), 0.7107068705f), -0.142248368f), 0.127414796f);
}
template <int ACT>
__device__ __forceinline__ float act_value(float z) {
  if constexpr (ACT == NF_ACT_RELU) return z < 0.0f ? 0.0f : z;
  else if constexpr (ACT == NF_ACT_RELU2) return z < 0.0f ? 0.0f : z * z;
  else if constexpr (ACT == NF_ACT_SILU) return z * __builtin_amdgcn_rcpf(1.0f + __expf(-z));
  else if constexpr (ACT == NF_ACT_GELU) {
    float e;
    const float q = normal_tail(z, &e) * e;
    return fmaf(-fminf(fabsf(z), 1e30f), q, fmaxf(z, 0.0f));  // z Phi(z); q of an infinity is zero, of a NaN a NaN
  } else return z;
}
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if constexpr (ACT == NF_ACT_RELU) return z > 0.0f ? 1.0f : z <= 0.0f ? 0.0f : z;
  else if constexpr (ACT == NF_ACT_RELU2) return z <= 0.0f ? 0.0f : 2.0f * z;
  else if constexpr (ACT == NF_ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.0f + __expf(-z));
    return s * (z * (1.0f - s) + 1.0f);
  } else if constexpr (ACT == NF_ACT_GELU) {
    float e;
    const float q = normal_tail(z, &e), half = copysignf(fmaf(-q, e, 0.5f), z);  // Phi(z) - 1/2
    return fmaf(z * 0.3989422804f, e, 0.5f) + half;
  } else return 1.0f;
}
// v * act'(x^); a closed gate lets nothing through, not even an infinity
template <int ACT>
__device__ __forceinline__ float gated(float v, float x) {
  if constexpr (ACT == NF_ACT_NONE) return v;
  else if constexpr (ACT == NF_ACT_RELU || ACT == NF_ACT_RELU2) return x <= 0.0f ? 0.0f : v * act_slope<ACT>(x);
  else return v * act_slope<ACT>(x);
}

template <int V>
using Int = std::integral_constant<int, V>;

// out[c] = sum over `groups` rows of `slots` (rms_norm.hip)
int sum_slots(const float* slots, int64_t groups, int64_t width, void* out, int dt, hipStream_t s);

}  // namespace nf
