// smoe_linear_rows.hip — linear_act for a few rows per expert: single tokens
// and decode batches (gfx950).
//
// The time is the weights' bytes: each is read once, straight into the
// registers of the one wave that multiplies it.  A workgroup of 8 waves owns
// 16 MB rows and 16 NB weight rows; its waves share the sum, 64 terms at a
// time in turn, kU such units in flight a wave: with two workgroups a compute
// unit about 128 KiB of loads are under way there.  The fragments are the
// MFMA's own: lane l takes 16 bytes of weight row l % 16 at 8 (l / 16), two
// of them a 128-byte line.  x is small and comes from L2 the same way.  At the
// end the eight partial tiles meet in LDS, are added in wave order and
// leave through the epilogue.
//
// us and TB/s: K 4096, N 4096, 1 to 16 rows 13 (2.5); 256 rows over 128 experts,
// K 2048, N 1536 141 (5.7, of the weights of the experts that have rows).
//
// For SwiGLU a workgroup's weight rows are half gate rows and half the up
// rows of the same columns.
#include "smoe_linear.h"

namespace smoe {

constexpr int kRowsWaves = 8;

template <class T, int kMB, int kNB, int kU, int kAct>
__global__ __launch_bounds__(512, 2) void linear_rows_kernel(const LinArgs a) {
  constexpr bool kPair = kAct == SMOE_ACT_SWIGLU;
  static_assert(!kPair || kNB % 2 == 0, "gate and up rows");
  constexpr int kM = kMB * 16, kN = kNB * 16, kOut = kPair ? kN / 2 : kN, kPitch = kN + 4;
  __shared__ float part[kRowsWaves][kM][kPitch];
  RowTile t;
  if (!find_row_tile<kM>(a.offsets, a.E, a.R, blockIdx.y, &t)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int cols = kPair ? a.N / 2 : a.N, n0 = blockIdx.x * kOut, K = a.K;
  const int r = lane & 15, c = (lane >> 4) * 8;
  const T* xr[kMB];
  const T* wr[kNB];
#pragma unroll
  for (int i = 0; i < kMB; ++i) {
    const int m = i * 16 + r;
    xr[i] = (const T*)a.a + (long long)(t.row0 + (m < t.rows ? m : t.rows - 1)) * a.lda + c;
  }
#pragma unroll
  for (int j = 0; j < kNB; ++j) {
    int n = n0 + (kPair ? j % (kNB / 2) : j) * 16 + r;
    n = n < cols ? n : cols - 1;
    if (kPair && j >= kNB / 2) n += cols;
    wr[j] = (const T*)a.b + ((size_t)t.e * a.N + n) * K + c;
  }
  v4f_t acc[kMB][kNB];
#pragma unroll
  for (int i = 0; i < kMB; ++i)
#pragma unroll
    for (int j = 0; j < kNB; ++j) acc[i][j] = v4f_t{0.0f, 0.0f, 0.0f, 0.0f};
  const int full = K / 64;
  int u = wave;
  // kU units at a time while there are as many for this wave
  for (; u + (kU - 1) * kRowsWaves < full; u += kU * kRowsWaves) {
    v4u_t fw[kU][2][kNB], fx[kU][2][kMB];
#pragma unroll
    for (int q = 0; q < kU; ++q) {
      const int k = (u + q * kRowsWaves) * 64;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int j = 0; j < kNB; ++j) fw[q][h][j] = load_piece<T, true>(wr[j] + k + h * 32);
#pragma unroll
        for (int i = 0; i < kMB; ++i) fx[q][h][i] = load_piece<T>(xr[i] + k + h * 32);
      }
    }
    __builtin_amdgcn_sched_barrier(0);  // all of them before the first wait
#pragma unroll
    for (int q = 0; q < kU; ++q)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < kMB; ++i)
#pragma unroll
          for (int j = 0; j < kNB; ++j) acc[i][j] = mfma32<T>(fw[q][h][j], fx[q][h][i], acc[i][j]);
  }
  for (; u * 64 < K; u += kRowsWaves) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = u * 64 + h * 32, n = K - k - c;  // terms from this lane's first
      v4u_t fw[kNB], fx[kMB];
#pragma unroll
      for (int j = 0; j < kNB; ++j) fw[j] = load_some<T>(wr[j] + k, n);
#pragma unroll
      for (int i = 0; i < kMB; ++i) fx[i] = load_some<T>(xr[i] + k, n);
#pragma unroll
      for (int i = 0; i < kMB; ++i)
#pragma unroll
        for (int j = 0; j < kNB; ++j) acc[i][j] = mfma32<T>(fw[j], fx[i], acc[i][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < kMB; ++i)
#pragma unroll
    for (int j = 0; j < kNB; ++j)
      *(v4f_t*)&part[wave][i * 16 + r][j * 16 + (lane >> 4) * 4] = acc[i][j];
  __syncthreads();
  auto sum = [&](int m, int n) {
    float s = part[0][m][n];
#pragma unroll
    for (int w = 1; w < kRowsWaves; ++w) s = s + part[w][m][n];
    return s;
  };
  auto bias = [&](int n) {
    const size_t i = (size_t)t.e * a.N + n;
    return a.bias_f32 ? ((const float*)a.bias)[i] : Elt<T>::to_f32(((const T*)a.bias)[i]);
  };
  for (int q = threadIdx.x; q < kM * kOut; q += kRowsWaves * 64) {
    const int m = q / kOut, cn = q % kOut, n = n0 + cn;
    if (m >= t.rows || n >= cols) continue;
    const size_t row = (size_t)t.row0 + m;
    float v = sum(m, cn);
    if (a.bias) v = v + bias(n);
    if (a.z) ((T*)a.z)[row * a.N + n] = Elt<T>::from_f32(v);
    if constexpr (kPair) {
      float w = sum(m, cn + kOut);
      if (a.bias) w = w + bias(cols + n);
      if (a.z) ((T*)a.z)[row * a.N + cols + n] = Elt<T>::from_f32(w);
      v = act_value<SMOE_ACT_SILU>(v) * w;
    } else {
      v = act_value<kAct>(v);
    }
    if (a.residual) v = v + Elt<T>::to_f32(((const T*)a.residual)[(long long)row * a.ldr + n]);
    ((T*)a.out)[row * cols + n] = Elt<T>::from_f32(v);
  }
}

template <class T, int kMB, int kNB, int kU>
static int rows_launch(const LinArgs& a, hipStream_t s) {
  const bool pair = a.act == SMOE_ACT_SWIGLU;
  const int cols = pair ? a.N / 2 : a.N, bn = pair ? kNB * 8 : kNB * 16;
  const dim3 grid((cols + bn - 1) / bn, (a.R + kMB * 16 - 1) / (kMB * 16) + a.E - 1), block(kRowsWaves * 64);
#define SMOE_ROWS(A) linear_rows_kernel<T, kMB, kNB, kU, A><<<grid, block, 0, s>>>(a)
  if constexpr (kNB % 2 == 0) {
    if (pair) {
      SMOE_ROWS(SMOE_ACT_SWIGLU);
      SMOE_RETURN_LAUNCH();
    }
  }
  switch (a.act) {
    case SMOE_ACT_NONE: SMOE_ROWS(SMOE_ACT_NONE); break;
    case SMOE_ACT_RELU: SMOE_ROWS(SMOE_ACT_RELU); break;
    case SMOE_ACT_SILU: SMOE_ROWS(SMOE_ACT_SILU); break;
    case SMOE_ACT_GELU: SMOE_ROWS(SMOE_ACT_GELU); break;
    default: SMOE_ROWS(SMOE_ACT_GELU_TANH); break;
  }
#undef SMOE_ROWS
  SMOE_RETURN_LAUNCH();
}

template <class T>
static int rows_t(const LinArgs& a, int mb, int nb, hipStream_t s) {
  if (mb == 1) return nb == 1 ? rows_launch<T, 1, 1, 4>(a, s) : nb == 2 ? rows_launch<T, 1, 2, 4>(a, s) : rows_launch<T, 1, 4, 2>(a, s);
  return nb == 1 ? rows_launch<T, 2, 1, 4>(a, s) : nb == 2 ? rows_launch<T, 2, 2, 2>(a, s) : rows_launch<T, 2, 4, 1>(a, s);
}

// 16-row blocks a tile for R rows over E experts, or 0: too many rows.  A
// dense product's rows are known; an expert's are on the device, so for
// experts the mean counts and leaves room for loads above it.
int linear_rows_blocks(int R, int E) {
  const int mean = E == 1 ? R : (R + E - 1) / E * 3 / 2;
  return mean <= 16 ? 1 : mean <= 32 ? 2 : 0;
}

// Whether this kernel is the one for sizes that the tiled kernel covers too:
// where that one's tiles of 128 columns would leave compute units idle, or at
// one or two rows.  us here / there: K 4096, N 4096, 16 rows 13 / 49; N 8192 19 /
// 49; N 28672 54 / 53, 32 rows 63 / 54; K 2048, N 1536, 128 experts: 64 rows 75 /
// 77, 256 135 / 141, 1024 171 / 149.
bool linear_rows_better(int R, int N, int E, int act) {
  if (!linear_rows_blocks(R, E)) return false;
  const int cols = act == SMOE_ACT_SWIGLU ? N / 2 : N, bn = act == SMOE_ACT_SWIGLU ? 64 : 128;
  return R <= 2 * E || (long long)(cols + bn - 1) / bn * (R < E ? R : E) < 200;
}

int linear_rows(const LinArgs& a, int dtype, hipStream_t s) {
  const int mb = linear_rows_blocks(a.R, a.E);
  const int cols = a.act == SMOE_ACT_SWIGLU ? a.N / 2 : a.N, per = a.act == SMOE_ACT_SWIGLU ? 8 : 16;
  // wide column tiles read x less often, narrow ones make enough workgroups
  const long long tiles = (long long)((cols + per - 1) / per) * (a.R < a.E ? a.R : a.E);
  const int nb = tiles >= 1536 ? 4 : tiles >= 1024 || a.act == SMOE_ACT_SWIGLU ? 2 : 1;
  return dtype == SMOE_BF16 ? rows_t<bf16_t>(a, mb, nb, s) : rows_t<f16_t>(a, mb, nb, s);
}

}  // namespace smoe
