// The linear layer with 8-bit checkpoints where rows are many and channels few (both sides at most 256): streams over the rows.
//
//   forward   a row is read once: its largest magnitude, its 8-bit form out, act(x) in 16 bits to LDS, the product with weights that sit in the
//             waves' registers, y out
//   backward  dy and q are read once: act(x^) to LDS, dW's sums (256 x 256 in the eight waves' registers for as long as the workgroup lives), dx with
//             weights that sit in LDS, its gate, dx out; the workgroups' dW and db are added up afterwards, in a fixed order
//
// As separate passes (8-bit rows; act(x^); three products) the same bytes move two and a half times.  2^18 x 256 x 256 with ReLU, forward and backward:
// 199 - 214 us by the card instead of 353, of which the forward 85, the backward 117, the sums of 256 partial dW 12 and db 5 (launched alone some more); the least that has to move, 670 MB, takes 136 at a
// copy's rate.  The waves wait for memory and for each other: more under way (a third tile) costs registers that hold the weights, a tile of 64 rows (111 us the
// forward) and four waves to a SIMD (162, spilled) were slower.
//
// A workgroup of 512 threads takes 32 rows at a time.  Rows in LDS lie as in Side's crosswise form (gemm_tile.h): the 32-byte segments of a row are
// spread by its bits 0, 1 and 3, free of bank conflicts for the transposing reads and for 16-byte reads along the row alike.
#include "checkpointed_narrow.h"
#include "gemm_tile.h"

namespace nf {

constexpr int TILE = 32, THREADS = 512;

// 16 bytes, piece p of a row of 2 C bytes
template <int C>
__device__ __forceinline__ int place(int row, int p) {
  const int spread = (row & 3) | (row >> 1 & 4);
  return row * (2 * C) + (((p >> 1) ^ spread) << 5 | (p & 1) << 4);
}
// the sixteen rows from `row` on, along the row: piece 4 step + lane / 16
template <int C>
__device__ __forceinline__ i32x4_t along(const char* from, int row, int step, int lane) {
  return *(const i32x4_t*)(from + place<C>(row + (lane & 15), 4 * step + (lane >> 4)));
}
template <typename T>
__device__ __forceinline__ void unpack8(i32x4_t v, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = (uint32_t)v[i];
    f[2 * i] = T::to_f32((uint16_t)w);
    f[2 * i + 1] = T::to_f32((uint16_t)(w >> 16));
  }
}
template <typename T>
__device__ __forceinline__ i32x4_t pack8(const float (&f)[8]) {
  i32x4_t v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (int)T::pack(f[2 * i], f[2 * i + 1]);
  return v;
}
__device__ __forceinline__ i32x4_t load_piece(const uint16_t* p, bool there) {
  i32x4_t v = {0, 0, 0, 0};
  if (there) v = *(const i32x4_t*)p;
  return v;
}
// The rows of a tile as a buffer: loads outside of it give zeros and stores do nothing, without a branch (behind branches the compiler cannot count
// what is under way, and waits for all of it).
constexpr int NOWHERE = -16;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const void* p, int64_t row, int64_t rows, int64_t ld, int bytes) {
  const int64_t left = rows - row;
  const int have = left < 0 ? 0 : left < TILE ? (int)left : TILE;
  const int size = have == 0 ? 0 : (have - 1) * (int)ld + bytes;
  return __builtin_amdgcn_make_buffer_rsrc((char*)p + (have == 0 ? 0 : row * ld), 0, size, 0x00020000);
}
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ i32x4_t get16(__amdgpu_buffer_rsrc_t b, int at) { return __builtin_bit_cast(i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(b, at, 0, 0)); }

// ---- forward ------------------------------------------------------------------------------------
template <typename T, int KP, int NP>
__global__ __launch_bounds__(THREADS, 2) void narrow_fwd_k(NarrowFwd a) {
  constexpr int PIECES = KP / 8, ROWS = THREADS / PIECES, EACH = TILE / ROWS;  // threads to a row, rows at once, rows of a thread
  constexpr int NT = NP / 128, STEPS = KP / 32;
  __shared__ __attribute__((aligned(1024))) char lds[2][TILE * KP * 2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane & 15, g = lane >> 4;
  const int p = threadIdx.x % PIECES, r0 = threadIdx.x / PIECES;
  const bool in = p * 8 < a.k;
  // the weights of this wave's columns, and their biases
  i32x4_t w[NT][STEPS];
  float b[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int n = wave * (16 * NT) + 16 * j;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int c = 32 * s + 8 * g;
      w[j][s] = load_piece((const uint16_t*)a.w + (int64_t)(n + i16) * a.ws + c, n + i16 < a.n && c < a.k);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) b[j][i] = a.bias != nullptr && n + 4 * g + i < a.n ? load_as_f32(a.bias, n + 4 * g + i, a.bias_dt) : 0.0f;
  }
  const int64_t tiles = (a.rows + TILE - 1) / TILE;
  const auto ask = [&](int64_t tile, i32x4_t(&x)[EACH]) {
    const auto buffer = rows_of(a.x, tile * TILE, a.rows, a.xs * 2, a.k * 2);
#pragma unroll
    for (int j = 0; j < EACH; ++j) x[j] = get16(buffer, in ? (r0 + j * ROWS) * (int)a.xs * 2 + p * 16 : NOWHERE);
  };
  const auto prepare = [&](int64_t tile, i32x4_t(&x)[EACH], char* to) {
    float v[EACH][8];
#pragma unroll
    for (int j = 0; j < EACH; ++j) unpack8<T>(x[j], v[j]);
    if (a.q != nullptr) {
      const auto to_q = rows_of(a.q, tile * TILE, a.rows, a.k, a.k);
      const auto to_s = rows_of(a.scale, tile * TILE, a.rows, 4, 4);
      uint32_t top[EACH];
#pragma unroll
      for (int j = 0; j < EACH; ++j) top[j] = largest16({(uint32_t)x[j][0], (uint32_t)x[j][1], (uint32_t)x[j][2], (uint32_t)x[j][3]});
#pragma unroll
      for (int j = 0; j < EACH; ++j) top[j] = lanes_max<PIECES>(top[j]);
#pragma unroll
      for (int j = 0; j < EACH; ++j) {
        const int r = r0 + j * ROWS;
        const EightBit e = eight_bit(magnitude_bits(T::to_f32((uint16_t)top[j])));
        uint32_t q[2];
        quantized8<true>(v[j], e, q);
        __builtin_amdgcn_raw_buffer_store_b64(u32x2_t{q[0], q[1]}, to_q, in ? r * a.k + p * 8 : NOWHERE, 0, 0);
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(e.scale), to_s, p == 0 ? r * 4 : NOWHERE, 0, 0);
      }
    }
    if (a.act != NF_ACT_NONE) {
      with_act(a.act, [&](auto act_c) {
#pragma unroll
        for (int j = 0; j < EACH; ++j)
#pragma unroll
          for (int i = 0; i < 8; ++i) v[j][i] = act_value<decltype(act_c)::value>(v[j][i]);
      });
#pragma unroll
      for (int j = 0; j < EACH; ++j) x[j] = pack8<T>(v[j]);
    }
#pragma unroll
    for (int j = 0; j < EACH; ++j) *(i32x4_t*)(to + place<KP>(r0 + j * ROWS, p)) = x[j];
  };
  // between two meetings a wave multiplies one tile and prepares the next, so that one wave's vector arithmetic runs beside another's products;
  // the rows of two more tiles are under way
  const int64_t far = gridDim.x;
  const auto round = [&](int64_t tile, const char* from, char* to, i32x4_t(&x)[EACH]) {
    f32x4_t acc[2][NT] = {};
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const i32x4_t f = along<KP>(from, 16 * i, s, lane);
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = Mma<T>::run(w[j][s], f, acc[i][j]);
      }
    const auto to_y = rows_of(a.y, tile * TILE, a.rows, a.ys * 2, a.n * 2);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int n = wave * (16 * NT) + 16 * j + 4 * g;  // (n: a multiple of 8 channels)
        const u32x2_t o = {T::pack(acc[i][j][0] + b[j][0], acc[i][j][1] + b[j][1]), T::pack(acc[i][j][2] + b[j][2], acc[i][j][3] + b[j][3])};
        __builtin_amdgcn_raw_buffer_store_b64(o, to_y, n < a.n ? (16 * i + i16) * (int)a.ys * 2 + n * 2 : NOWHERE, 0, 0);
      }
    __builtin_amdgcn_sched_barrier(0);  // the wait for the next tile's rows stays behind the products
    prepare(tile + far, x, to);
    ask(tile + 3 * far, x);
    __syncthreads();
  };
  i32x4_t x0[EACH], x1[EACH];
  ask(blockIdx.x, x0);
  ask(blockIdx.x + far, x1);
  prepare(blockIdx.x, x0, lds[0]);
  ask(blockIdx.x + 2 * far, x0);
  __syncthreads();
  for (int64_t tile = blockIdx.x; tile < tiles; tile += 2 * far) {
    round(tile, lds[0], lds[1], x1);
    round(tile + far, lds[1], lds[0], x0);
  }
}

// ---- backward -----------------------------------------------------------------------------------
template <typename T, int KP, int NP>
__global__ __launch_bounds__(THREADS, 2) void narrow_bwd_k(NarrowBwd a) {
  constexpr int PD = NP / 8, RD = THREADS / PD, ED = TILE / RD;  // dy: threads to a row, rows at once, rows of a thread
  constexpr int PQ = KP / 8, RQ = THREADS / PQ, EQ = TILE / RQ;  // q
  constexpr int XT = KP / 128, STEPS = NP / 32;                  // dx: tiles of 16 columns of a wave; steps of the sum
  constexpr int WN = NP / 64, WK = KP / 32;                      // dW: tiles of a wave, four waves along n and two along k
  typedef Side<true, NP, 8> D;
  typedef Side<true, KP, 8> H;
  __shared__ __attribute__((aligned(1024))) char lds[NP * KP * 2 + TILE * NP * 2 + TILE * KP * 2];
  char *wl = lds, *dl = lds + NP * KP * 2, *hl = dl + TILE * NP * 2;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i16 = lane & 15, g = lane >> 4;
  const int pd = threadIdx.x % PD, rd = threadIdx.x / PD, pq = threadIdx.x % PQ, rq = threadIdx.x / PQ;
  const bool want_x = a.dx != nullptr;
  if (want_x) {
    for (int r = rq; r < NP; r += RQ)
      *(i32x4_t*)(wl + place<KP>(r, pq)) = load_piece((const uint16_t*)a.w + (int64_t)r * a.ws + pq * 8, r < a.n && pq * 8 < a.k);
  }
  const int64_t tiles = (a.rows + TILE - 1) / TILE;
  i32x4_t d[ED];
  int q[EQ][2];
  float s[EQ];
  const auto ask = [&](int64_t tile) {
    const auto from_d = rows_of(a.dy, tile * TILE, a.rows, a.dys * 2, a.n * 2), from_q = rows_of(a.q, tile * TILE, a.rows, a.k, a.k),
               from_s = rows_of(a.scale, tile * TILE, a.rows, 4, 4);
#pragma unroll
    for (int j = 0; j < ED; ++j) d[j] = get16(from_d, pd * 8 < a.n ? (rd + j * RD) * (int)a.dys * 2 + pd * 16 : NOWHERE);
#pragma unroll
    for (int j = 0; j < EQ; ++j) {
      const u32x2_t v = __builtin_amdgcn_raw_buffer_load_b64(from_q, pq * 8 < a.k ? (rq + j * RQ) * a.k + pq * 8 : NOWHERE, 0, 0);
      q[j][0] = (int)v[0];
      q[j][1] = (int)v[1];
      s[j] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(from_s, (rq + j * RQ) * 4, 0, 0));
    }
  };
  ask(blockIdx.x);
  f32x4_t aw[WN][WK] = {};
  float sums[8] = {};
  const int wn = wave >> 1, wk = wave & 1;
  const int at_d = D::read_at(lane, wn * WN), at_h = H::read_at(lane, wk * WK), at_w = H::read_at(lane, wave * XT);
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
#pragma unroll
    for (int j = 0; j < ED; ++j) {
      *(i32x4_t*)(dl + place<NP>(rd + j * RD, pd)) = d[j];
      if (a.db != nullptr) {
        float v[8];
        unpack8<T>(d[j], v);
#pragma unroll
        for (int i = 0; i < 8; ++i) sums[i] += v[i];
      }
    }
#pragma unroll
    for (int j = 0; j < EQ; ++j) {
      float v[8];
      kept8(q[j], s[j], v);
      with_act(a.act, [&](auto act_c) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = act_value<decltype(act_c)::value>(v[i]);
      });
      *(i32x4_t*)(hl + place<KP>(rq + j * RQ, pq)) = pack8<T>(v);
    }
    __syncthreads();
    // the gate of this wave's results (the rows were read a round ago), and the next round's rows
    int gq[2][XT];
    float gs[2];
    if (want_x && a.act != NF_ACT_NONE) {
      const auto from_q = rows_of(a.q, tile * TILE, a.rows, a.k, a.k), from_s = rows_of(a.scale, tile * TILE, a.rows, 4, 4);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        gs[i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(from_s, (16 * i + i16) * 4, 0, 0));
#pragma unroll
        for (int j = 0; j < XT; ++j) {
          const int c = wave * (16 * XT) + 16 * j + 4 * g;
          gq[i][j] = (int)__builtin_amdgcn_raw_buffer_load_b32(from_q, c < a.k ? (16 * i + i16) * a.k + c : NOWHERE, 0, 0);
        }
      }
    }
    ask(tile + gridDim.x);
    {
      i32x4_t fd[WN];
#pragma unroll
      for (int i = 0; i < WN; ++i) fd[i] = D::read(dl, at_d, i, 0);
#pragma unroll
      for (int j = 0; j < WK; ++j) {
        const i32x4_t f = H::read(hl, at_h, j, 0);
#pragma unroll
        for (int i = 0; i < WN; ++i) aw[i][j] = Mma<T>::run(f, fd[i], aw[i][j]);
      }
    }
    if (want_x) {
      f32x4_t ax[2][XT] = {};
#pragma unroll
      for (int t = 0; t < STEPS; ++t) {
        i32x4_t f[XT];
#pragma unroll
        for (int j = 0; j < XT; ++j) f[j] = H::read(wl, at_w, j, t);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const i32x4_t r = along<NP>(dl, 16 * i, t, lane);
#pragma unroll
          for (int j = 0; j < XT; ++j) ax[i][j] = Mma<T>::run(f[j], r, ax[i][j]);
        }
      }
      with_act(a.act, [&](auto act_c) {
        constexpr int ACT = decltype(act_c)::value;
        const auto to_x = rows_of(a.dx, tile * TILE, a.rows, (int64_t)a.k * 2, a.k * 2);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int j = 0; j < XT; ++j) {
            const int c = wave * (16 * XT) + 16 * j + 4 * g;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              v[e] = ax[i][j][e];
              if constexpr (ACT != NF_ACT_NONE) v[e] = gated<ACT>(v[e], gs[i] * (float)(gq[i][j] << (24 - e * 8) >> 24));
            }
            __builtin_amdgcn_raw_buffer_store_b64(u32x2_t{T::pack(v[0], v[1]), T::pack(v[2], v[3])}, to_x, c < a.k ? (16 * i + i16) * a.k * 2 + c * 2 : NOWHERE, 0, 0);
          }
        }
      });
    }
    __syncthreads();  // the tiles have been read
  }
  float* dw = a.dw + (int64_t)blockIdx.x * a.n * a.k;
#pragma unroll
  for (int i = 0; i < WN; ++i)
#pragma unroll
    for (int j = 0; j < WK; ++j) {
      const int n = (wn * WN + i) * 16 + i16, c = (wk * WK + j) * 16 + 4 * g;
      if (n < a.n && c < a.k) *(f32x4_t*)(dw + (int64_t)n * a.k + c) = aw[i][j];
    }
  if (a.db != nullptr) {  // RD threads hold parts of the same columns
    float* part = (float*)lds;
#pragma unroll
    for (int i = 0; i < 8; ++i) part[rd * NP + pd * 8 + i] = sums[i];
    __syncthreads();
    const int c = threadIdx.x;
    if (c < a.n) {
      float v = part[c];
      for (int r = 1; r < RD; ++r) v += part[r * NP + c];
      a.db[(int64_t)blockIdx.x * a.n + c] = v;
    }
  }
}

constexpr int NARROW = 256, NARROW_GROUPS = 256;

// From how many rows on these kernels are the quicker ones (forward + backward, us, here / as separate passes, GELU): 64 x 64 2048 rows 20 / 35, 128 x 128
// 23 / 36, 64 x 256 25 / 37; 256 x 256 2048 rows 47 / 43, 8192 56 / 52, 16384 59 / 65, 2^18 231 / 353 (ReLU).
bool narrow_fits(int64_t rows, int64_t n, int64_t k) {
  return n <= NARROW && k <= NARROW && n % 8 == 0 && k % 8 == 0 && rows >= (n > 128 && k > 128 ? 12288 : 2048);
}
int narrow_groups(int64_t rows) {
  const int64_t tiles = (rows + TILE - 1) / TILE;
  return (int)(tiles < NARROW_GROUPS ? tiles : NARROW_GROUPS);
}

template <typename Body>
void by_size(int k, int n, Body&& body) {
  if (k <= 128 && n <= 128) body(Int<128>{}, Int<128>{});
  else if (k <= 128) body(Int<128>{}, Int<256>{});
  else if (n <= 128) body(Int<256>{}, Int<128>{});
  else body(Int<256>{}, Int<256>{});
}

int narrow_fwd(const NarrowFwd& a, int dtype, hipStream_t s) {
  const int64_t tiles = (a.rows + TILE - 1) / TILE;
  by_size(a.k, a.n, [&](auto k_c, auto n_c) {
    constexpr int KP = decltype(k_c)::value, NP = decltype(n_c)::value;
    constexpr int64_t most = KP == 256 && NP == 256 ? 256 : 512;  // one workgroup to a compute unit, of the smaller ones two
    const unsigned blocks = (unsigned)(tiles < most ? tiles : most);
    if (dtype == NF_F16) hipLaunchKernelGGL((narrow_fwd_k<F16, KP, NP>), dim3(blocks), dim3(THREADS), 0, s, a);
    else hipLaunchKernelGGL((narrow_fwd_k<BF16, KP, NP>), dim3(blocks), dim3(THREADS), 0, s, a);
  });
  return check_launch("checkpointed_narrow_fwd");
}

int narrow_bwd(const NarrowBwd& a, int dtype, hipStream_t s) {
  const unsigned blocks = (unsigned)narrow_groups(a.rows);
  by_size(a.k, a.n, [&](auto k_c, auto n_c) {
    constexpr int KP = decltype(k_c)::value, NP = decltype(n_c)::value;
    if (dtype == NF_F16) hipLaunchKernelGGL((narrow_bwd_k<F16, KP, NP>), dim3(blocks), dim3(THREADS), 0, s, a);
    else hipLaunchKernelGGL((narrow_bwd_k<BF16, KP, NP>), dim3(blocks), dim3(THREADS), 0, s, a);
  });
  return check_launch("checkpointed_narrow_bwd");
}

}  // namespace nf
