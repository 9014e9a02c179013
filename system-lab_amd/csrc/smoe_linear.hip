// smoe_linear.hip — matrix products with bias, activation and residual in the
// epilogue, dense or one weight per expert, and their gradients (gfx950).
//
//   out = act(x W^T + b) + residual          x [R, K], W [N, K] or [E, N, K]
//   dz  = dout act'(z),  db = sum of dz over rows
//   dx  = dz W,          dW = dz^T x
//
// Products are bf16 or fp16 MFMA with fp32 accumulators; bias, activation and
// residual are applied to the fp32 sum and rounded once.  dz is kept in the
// operands' 16-bit type: it is the MFMA operand of both gradients.  That
// rounding is of the size of dx's and dW's own and adds to it as squares do.
#include "smoe_linear.h"

namespace smoe {

constexpr int kLinearMaxDim = 1 << 20, kLinearMaxRows = 1 << 29;

// ------------------------------------------- dz and the biases' gradient ---
// Rows in blocks of 64 of one expert; a thread owns 8 columns (SwiGLU: 8 gate
// columns and their 8 up columns), 32 threads side by side and 8 rows at a
// time.  dz (unless NULL) is rounded to T; the column sums are of the fp32
// values, one partial row a block.  Bound by HBM: 65536 x 1536 values of SwiGLU
// 101 us (5.0 TB/s).
constexpr int kDzRows = 64;
struct DzArgs {
  const void *dout, *z;
  void* dz;
  float* part;  // [blocks, N], or NULL
  const int32_t* offsets;
  long long lddout;
  int E, R, N;
};

template <class T, int kAct>
__global__ __launch_bounds__(256) void linear_dz_kernel(const DzArgs a) {
  constexpr bool kPair = kAct == SMOE_ACT_SWIGLU;
  __shared__ float red[kPair ? 2 : 1][8][32][8 + 1];
  RowTile t;
  if (!find_row_tile<kDzRows>(a.offsets, a.E, a.R, blockIdx.x, &t)) return;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int M = kPair ? a.N / 2 : a.N, c = (blockIdx.y * 32 + tx) * 8, n = M - c;
  float s0[8], s1[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) s0[i] = s1[i] = 0.0f;
  if (n > 0) {
    for (int r = ty; r < t.rows; r += 8) {
      const size_t row = (size_t)t.row0 + r;
      float g[8], z[8];
      load_f32<T>((const T*)a.dout + (long long)row * a.lddout + c, n, g);
      if constexpr (kAct != SMOE_ACT_NONE) load_f32<T>((const T*)a.z + row * a.N + c, n, z);
      if constexpr (kPair) {
        float u[8], dg[8], du[8];
        load_f32<T>((const T*)a.z + row * a.N + M + c, n, u);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float p = sigmoid_fast(z[i]);
          dg[i] = g[i] * u[i] * (p * (1.0f + z[i] * (1.0f - p)));
          du[i] = g[i] * (z[i] * p);
          s0[i] = s0[i] + dg[i];
          s1[i] = s1[i] + du[i];
        }
        if (a.dz) {
          store_f32<T>((T*)a.dz + row * a.N + c, n, dg);
          store_f32<T>((T*)a.dz + row * a.N + M + c, n, du);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if constexpr (kAct != SMOE_ACT_NONE) g[i] = g[i] * act_slope<kAct>(z[i]);
          s0[i] = s0[i] + g[i];
        }
        if (a.dz) store_f32<T>((T*)a.dz + row * a.N + c, n, g);
      }
    }
  }
  if (!a.part) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    red[0][ty][tx][i] = s0[i];
    if constexpr (kPair) red[1][ty][tx][i] = s1[i];
  }
  __syncthreads();
  // thread: column threadIdx.x of the block's 256
  const int col = blockIdx.y * 256 + threadIdx.x;
  if (col >= M) return;
#pragma unroll
  for (int h = 0; h < (kPair ? 2 : 1); ++h) {
    float s = 0.0f;
#pragma unroll
    for (int y = 0; y < 8; ++y) s = s + red[h][y][threadIdx.x >> 3][threadIdx.x & 7];
    a.part[(size_t)blockIdx.x * a.N + h * M + col] = s;
  }
}

// db[e] = the sum of expert e's partial rows, in order.
template <class T>
__global__ __launch_bounds__(256) void linear_db_kernel(const float* part, const int32_t* offsets, int blocks, int R,
                                                        int N, int f32, void* db) {
  const int e = blockIdx.y, c = blockIdx.x * 256 + threadIdx.x;
  int first = 0, count = (R + kDzRows - 1) / kDzRows;
  if (offsets) {
    // the blocks of the experts before e, a wave's lanes counting 64 at a time;
    // bounds out of order may count more blocks than there are
    auto blocks_of = [&](int i) {
      const int n = clamp_row(offsets, i + 1, R) - clamp_row(offsets, i, R);
      return n > 0 ? (n + kDzRows - 1) / kDzRows : 0;
    };
    int before = 0;
    for (int i = threadIdx.x & 63; i < e; i += 64) before += blocks_of(i);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) before += __shfl_xor(before, d, 64);
    first = before < blocks ? before : blocks;
    count = blocks_of(e);
    if (count > blocks - first) count = blocks - first;
  }
  if (c >= N) return;
  float s = 0.0f;
  int b = 0;
  const float* p = part + (size_t)first * N + c;
  for (; b + 8 <= count; b += 8) {  // eight rows in flight, added in order
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = p[(size_t)(b + i) * N];
#pragma unroll
    for (int i = 0; i < 8; ++i) s = s + v[i];
  }
  for (; b < count; ++b) s = s + p[(size_t)b * N];
  if (f32) ((float*)db)[(size_t)e * N + c] = s;
  else ((T*)db)[(size_t)e * N + c] = Elt<T>::from_f32(s);
}

// ------------------------------------------------------------ launching ----
static int row_tiles(int R, int E, int bm) { return (R + bm - 1) / bm + E - 1; }

#define SMOE_LIN_ACTS(CALL)                                            \
  do {                                                                 \
    switch (act) {                                                     \
      case SMOE_ACT_NONE: CALL(SMOE_ACT_NONE); break;                  \
      case SMOE_ACT_RELU: CALL(SMOE_ACT_RELU); break;                  \
      case SMOE_ACT_SILU: CALL(SMOE_ACT_SILU); break;                  \
      case SMOE_ACT_GELU: CALL(SMOE_ACT_GELU); break;                  \
      case SMOE_ACT_GELU_TANH: CALL(SMOE_ACT_GELU_TANH); break;        \
      default: CALL(SMOE_ACT_SWIGLU); break;                           \
    }                                                                  \
  } while (0)

static int linear_fwd(const LinArgs& a, int dtype, hipStream_t s) {
  return linear_rows_better(a.R, a.N, a.E, a.act) ? linear_rows(a, dtype, s) : linear_mm(a, kFwd, dtype, s);
}

// Parts of the gradients' workspace, each a multiple of 256 bytes.
static size_t linear_bwd_db_bytes(int R, int N, int E, bool bias) {
  return bias ? ((size_t)row_tiles(R, E, kDzRows) * N * sizeof(float) + 255) / 256 * 256 : 0;
}
static size_t linear_bwd_cut_bytes(int R, int N, int K) {
  const size_t x = linear_mm_part_bytes(R, N, K, 0, kDgrad), w = linear_mm_part_bytes(R, N, K, 0, kWgrad);
  return x > w ? x : w;
}

template <class T>
static int linear_bwd(const smoe_linear_bwd& q, hipStream_t s) {
  const int act = q.act;
  const bool has_act = act != SMOE_ACT_NONE;
  char* ws = (char*)q.ws;
  const size_t dz_bytes = has_act ? ((size_t)q.R * q.N * sizeof(T) + 255) / 256 * 256 : 0;
  float* part = q.dbias ? (float*)(ws + dz_bytes) : nullptr;
  const bool need_dz = has_act && (q.dx || q.dw);
  const int M = act == SMOE_ACT_SWIGLU ? q.N / 2 : q.N;
  if (need_dz || q.dbias) {
    const DzArgs d{q.dout, q.z, need_dz ? ws : nullptr, part, q.offsets, q.lddout, q.E, q.R, q.N};
    const dim3 grid(row_tiles(q.R, q.E, kDzRows), (M + 255) / 256);
#define SMOE_LD(A) linear_dz_kernel<T, A><<<grid, dim3(256), 0, s>>>(d)
    SMOE_LIN_ACTS(SMOE_LD);
#undef SMOE_LD
  }
  if (q.dbias)
    linear_db_kernel<T><<<dim3((q.N + 255) / 256, q.E), dim3(256), 0, s>>>(
        part, q.offsets, row_tiles(q.R, q.E, kDzRows), q.R, q.N, q.bias_f32, q.dbias);
  // both gradients' shares of a cut sum: one after the other in the same place
  float* cut = nullptr;
  if (!q.offsets && linear_bwd_cut_bytes(q.R, q.N, q.K))
    cut = (float*)(ws + dz_bytes + linear_bwd_db_bytes(q.R, q.N, q.E, q.dbias != nullptr));
  const void* dz = has_act ? (const void*)ws : q.dout;
  const long long lddz = has_act ? q.N : q.lddout;
  if (q.dx) {
    const LinArgs a{dz, q.w, lddz, q.K, nullptr, nullptr, 0, q.offsets, q.dx, nullptr, q.E, q.R, q.N, q.K, 0, 0, 0, cut, 1};
    const int st = linear_mm(a, kDgrad, q.dtype, s);
    if (st) return st;
  }
  if (q.dw) {
    const LinArgs a{dz, q.x, lddz, q.ldx, nullptr, nullptr, 0, q.offsets, q.dw, nullptr, q.E, q.R, q.N, q.K, 0, 0,
                    q.dw_mode, cut, 1};
    return linear_mm(a, kWgrad, q.dtype, s);
  }
  SMOE_RETURN_LAUNCH();
}

static int check_linear(int R, int N, int K, int E, int act, int dtype, const int32_t* offsets) {
  if (R <= 0 || N <= 0 || K <= 0) return SMOE_EINVAL_DIM;
  if (E <= 0 || E > SMOE_MAX_EXPERTS) return SMOE_EINVAL_EXPERTS;
  if (act < SMOE_ACT_NONE || act > SMOE_ACT_SWIGLU) return SMOE_EINVAL_MODE;
  if (dtype != SMOE_BF16 && dtype != SMOE_F16) return SMOE_EINVAL_MODE;
  if (act == SMOE_ACT_SWIGLU && N % 2) return SMOE_EINVAL_DIM;
  if (E > 1 && !offsets) return SMOE_EINVAL_NULL;
  if ((uintptr_t)offsets & 3u) return SMOE_EINVAL_PTRALIGN;
  // what a grid's edges hold
  if (N > kLinearMaxDim || K > kLinearMaxDim || R > kLinearMaxRows) return SMOE_EINVAL_DIM;
  return SMOE_OK;
}

}  // namespace smoe

using namespace smoe;

extern "C" size_t smoe_linear_act_workspace_size(int R, int N, int K, int E, int act) {
  if (R <= 0 || N <= 0 || K <= 0 || E != 1 || linear_rows_better(R, N, E, act)) return 0;
  return linear_mm_part_bytes(R, N, K, act, kFwd);
}

extern "C" int smoe_linear_act(const smoe_linear_fwd* q, void* stream) {
  if (!q) return SMOE_EINVAL_NULL;
  const int st = check_linear(q->R, q->N, q->K, q->E, q->act, q->dtype, q->offsets);
  if (st) return st;
  if (q->ldx < 0 || q->ldr < 0) return SMOE_EINVAL_DIM;
  SMOE_CHECK_ELT(q->x, q->dtype);
  SMOE_CHECK_ELT(q->w, q->dtype);
  SMOE_CHECK_ELT(q->out, q->dtype);
  SMOE_CHECK_OPT(q->bias, q->bias_f32 ? SMOE_F32 : q->dtype);
  SMOE_CHECK_OPT(q->residual, q->dtype);
  SMOE_CHECK_OPT(q->z, q->dtype);
  const size_t need = smoe_linear_act_workspace_size(q->R, q->N, q->K, q->E, q->act);
  if (need && (!q->ws || q->ws_bytes < need)) return SMOE_EINVAL_WORKSPACE;
  if ((uintptr_t)q->ws & 15u) return SMOE_EINVAL_PTRALIGN;
  const LinArgs a{q->x, q->w, q->ldx, q->K, q->bias, q->residual, q->ldr, q->offsets, q->out, q->z,
                  q->E, q->R, q->N, q->K, q->bias_f32, q->act, 0, need ? (float*)q->ws : nullptr, 1};
  hipStream_t s = (hipStream_t)stream;
  return linear_fwd(a, q->dtype, s);
}

extern "C" size_t smoe_linear_act_bwd_workspace_size(int R, int N, int K, int E, int act, int with_bias) {
  if (R <= 0 || N <= 0 || K <= 0 || E <= 0) return 0;
  const size_t dz = act != SMOE_ACT_NONE ? ((size_t)R * N * 2 + 255) / 256 * 256 : 0;
  return dz + linear_bwd_db_bytes(R, N, E, with_bias != 0) + (E == 1 ? linear_bwd_cut_bytes(R, N, K) : 0);
}

extern "C" int smoe_linear_act_bwd(const smoe_linear_bwd* q, void* stream) {
  if (!q) return SMOE_EINVAL_NULL;
  const int st = check_linear(q->R, q->N, q->K, q->E, q->act, q->dtype, q->offsets);
  if (st) return st;
  if (q->lddout < 0 || q->ldx < 0) return SMOE_EINVAL_DIM;
  if (q->dw_mode < SMOE_WGRAD_F32 || q->dw_mode > SMOE_WGRAD_BF16_ACC) return SMOE_EINVAL_MODE;
  SMOE_CHECK_ELT(q->dout, q->dtype);
  if (q->act != SMOE_ACT_NONE) SMOE_CHECK_ELT(q->z, q->dtype);
  if (q->dx) SMOE_CHECK_ELT(q->w, q->dtype);
  if (q->dw) SMOE_CHECK_ELT(q->x, q->dtype);
  SMOE_CHECK_OPT(q->dx, q->dtype);
  SMOE_CHECK_OPT(q->dw, q->dw_mode < SMOE_WGRAD_BF16 ? SMOE_F32 : q->dtype);
  SMOE_CHECK_OPT(q->dbias, q->bias_f32 ? SMOE_F32 : q->dtype);
  const size_t need = smoe_linear_act_bwd_workspace_size(q->R, q->N, q->K, q->E, q->act, q->dbias != nullptr);
  if (need && (!q->ws || q->ws_bytes < need)) return SMOE_EINVAL_WORKSPACE;
  if ((uintptr_t)q->ws & 15u) return SMOE_EINVAL_PTRALIGN;
  hipStream_t s = (hipStream_t)stream;
  return q->dtype == SMOE_BF16 ? linear_bwd<bf16_t>(*q, s) : linear_bwd<f16_t>(*q, s);
}
