// smoe_linear.h — what the kernels of linear_act share: arguments, fragments,
// activations and the map from a tile to its expert's rows.
#pragma once

#include "smoe_elt.h"

namespace smoe {

typedef float v4f_t __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf_t __attribute__((ext_vector_type(8)));
typedef _Float16 v8h_t __attribute__((ext_vector_type(8)));

// D[m][n] += sum over 32 k of A[m][k] B[n][k] for 16 x 16 values: lane l gives
// A row l%16 and B row l%16, both at k = 8 (l/16) .. + 7, and holds
// D[4 (l/16) + i][l%16], i = 0..3.
template <class T>
__device__ __forceinline__ v4f_t mfma32(const v4u_t& a, const v4u_t& b, const v4f_t& c) {
  if constexpr (Elt<T>::kDtype == SMOE_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf_t, a), __builtin_bit_cast(v8bf_t, b), c,
                                                   0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h_t, a), __builtin_bit_cast(v8h_t, b), c, 0, 0,
                                                  0);
}

// The logistic function of x in fp32 from the hardware's exp2 and reciprocal
// (1 ulp each): its error, about 2^-22, is far below the half step of the
// 16-bit values it goes into.
__device__ __forceinline__ float sigmoid_fast(float x) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.4426950408889634f));
}

constexpr float kGelu2C = 1.5957691216057308f;  // 2 sqrt(2 / pi)

// act(z) of one value; SwiGLU pairs two values and is not here.
// 0.5 (1 + tanh a) is the logistic function of 2a.
template <int kAct>
__device__ __forceinline__ float act_value(float z) {
  if constexpr (kAct == SMOE_ACT_RELU) return z > 0.0f ? z : (z != z ? z : 0.0f);
  else if constexpr (kAct == SMOE_ACT_SILU) return z * sigmoid_fast(z);
  else if constexpr (kAct == SMOE_ACT_GELU) return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
  else if constexpr (kAct == SMOE_ACT_GELU_TANH)
    return z * sigmoid_fast(kGelu2C * (z + 0.044715f * z * z * z));
  else return z;
}

// The derivative of act at z.
template <int kAct>
__device__ __forceinline__ float act_slope(float z) {
  if constexpr (kAct == SMOE_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
  else if constexpr (kAct == SMOE_ACT_SILU) {
    const float p = sigmoid_fast(z);
    return p * (1.0f + z * (1.0f - p));
  } else if constexpr (kAct == SMOE_ACT_GELU) {
    const float e = __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);  // exp(-z^2 / 2)
    return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) + z * e * 0.39894228040143268f;
  } else if constexpr (kAct == SMOE_ACT_GELU_TANH) {
    const float p = sigmoid_fast(kGelu2C * (z + 0.044715f * z * z * z));
    return p + z * p * (1.0f - p) * kGelu2C * (1.0f + 0.134145f * z * z);
  } else return 1.0f;
}

// Row tiles of kBM rows, expert by expert: `tile` counts them over all experts
// and the grid holds ceil(R / kBM) + E - 1 (the most there can be).  Every
// thread of the workgroup calls this; false: no such tile.  Bounds outside
// [0, R] or out of order are clamped, so that no row outside the buffers and
// no row twice is ever touched.
struct RowTile {
  int e, row0, rows, lo;  // expert, first row, rows of this tile, the expert's first row
};
__device__ __forceinline__ int clamp_row(const int32_t* offsets, int e, int R) {
  const int v = offsets[e];
  return v < 0 ? 0 : v > R ? R : v;
}
template <int kBM>
__device__ __forceinline__ bool find_row_tile(const int32_t* offsets, int E, int R, int tile, RowTile* out) {
  if (!offsets) {
    out->e = 0;
    out->lo = 0;
    out->row0 = tile * kBM;
    out->rows = R - out->row0 < kBM ? R - out->row0 : kBM;
    return out->rows > 0;
  }
  // one wave's scan over 64 experts at a time, every wave for itself
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int e0 = 0; e0 < E; e0 += 64) {
    const int e = e0 + lane;
    int lo = 0, n = 0;
    if (e < E) {
      lo = clamp_row(offsets, e, R);
      n = clamp_row(offsets, e + 1, R) - lo;
      n = n < 0 ? 0 : n;
    }
    const int t = (n + kBM - 1) / kBM;
    int inc = t;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(inc, d, 64);
      if (lane >= d) inc += up;
    }
    const int first = base + inc - t;
    const unsigned long long hit = __ballot(tile >= first && tile < first + t);
    if (hit) {
      const int src = __builtin_ctzll(hit);
      const int at = tile - __builtin_amdgcn_readlane(first, src);
      const int glo = __builtin_amdgcn_readlane(lo, src), gn = __builtin_amdgcn_readlane(n, src);
      out->e = e0 + src;
      out->lo = glo;
      out->row0 = glo + at * kBM;
      out->rows = gn - at * kBM < kBM ? gn - at * kBM : kBM;
      return true;
    }
    base += __builtin_amdgcn_readlane(inc, 63);
  }
  return false;
}

// The same map with the number of tiles known: one pass over the experts by
// every wave for itself, each lane counting a run of neighbouring experts.
struct RowTiles {
  int total;         // row tiles of all experts
  int first, count;  // of this lane's experts: their first tile, how many
  __device__ __forceinline__ RowTiles(const int32_t* offsets, int E, int R, int bm) {
    first = 0;
    if (!offsets) {
      total = count = (R + bm - 1) / bm;
      return;
    }
    const int lane = threadIdx.x & 63, per = (E + 63) / 64;
    int n = 0;
    for (int i = 0; i < per; ++i) {
      const int e = lane * per + i;
      if (e < E) {
        const int r = clamp_row(offsets, e + 1, R) - clamp_row(offsets, e, R);
        n += r > 0 ? (r + bm - 1) / bm : 0;
      }
    }
    int inc = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(inc, d, 64);
      if (lane >= d) inc += up;
    }
    count = n;
    first = inc - n;
    total = __builtin_amdgcn_readlane(inc, 63);
  }
  // Tile `tile` < total; wave-uniform.
  __device__ __forceinline__ bool find(const int32_t* offsets, int E, int R, int bm, int tile, RowTile* out) const {
    if (!offsets) {
      out->e = out->lo = 0;
      out->row0 = tile * bm;
      out->rows = R - tile * bm < bm ? R - tile * bm : bm;
      return out->rows > 0;
    }
    const unsigned long long hit = __ballot(tile >= first && tile < first + count);
    if (!hit) return false;
    const int src = __builtin_ctzll(hit), per = (E + 63) / 64;
    int at = tile - __builtin_amdgcn_readlane(first, src);
    for (int e = src * per; e < E && e < (src + 1) * per; ++e) {
      const int lo = clamp_row(offsets, e, R), n = clamp_row(offsets, e + 1, R) - lo;
      const int t = n > 0 ? (n + bm - 1) / bm : 0;
      if (at < t) {
        out->e = e;
        out->lo = lo;
        out->row0 = lo + at * bm;
        out->rows = n - at * bm < bm ? n - at * bm : bm;
        return true;
      }
      at -= t;
    }
    return false;
  }
};

// The forward's and the gradients' common description of one product.
struct LinArgs {
  const void *a, *b;      // a: rows of the left operand, b: of the right one
  long long lda, ldb;     // elements between rows
  const void* bias;
  const void* residual;
  long long ldr;
  const int32_t* offsets;
  void *out, *z;
  int E, R, N, K;         // N: rows of the weight, K: its row length
  int bias_f32, act, mode;
  float* part;            // partial sums of `splits` shares of the sum, or NULL
  int splits;
};

// smoe_linear_rows.hip: the product for few rows an expert (0 blocks: others).
int linear_rows_blocks(int R, int E);
bool linear_rows_better(int R, int N, int E, int act);
int linear_rows(const LinArgs& a, int dtype, hipStream_t s);

// The tiled kernels (smoe_linear_mm.h).  what: the product, dx or dW.
enum { kFwd = 0, kDgrad = 1, kWgrad = 2 };
// shares that a dense product's sum is cut into, and the bytes of its partial sums
int linear_mm_splits(int R, int N, int K, int act, int what);
size_t linear_mm_part_bytes(int R, int N, int K, int act, int what);
int linear_mm(LinArgs a, int what, int dtype, hipStream_t s);
int linear_mm_any(const LinArgs& a, int what, int dtype, hipStream_t s);

}  // namespace smoe
