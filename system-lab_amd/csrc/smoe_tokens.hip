// smoe_tokens.hip — token rows to their experts and back, unquantised (gfx950).
//
//   permute      xp[r] = w x[t]             for every pair (t, k) with row r
//   its gradient dx[t] = sum_k w dxp[r],    dw[t,k] = <x[t], dxp[r]>
//   unpermute    out[t] = sum_k w y[r]
//   its gradient dy[r] = w dout[t],         dw[t,k] = <dout[t], y[r]>
//
// Two kernels: one token row spread to its K expert rows (scatter), and K
// expert rows summed into their token's (gather), each with or without the
// dot products that are the weights' gradient.  Both move bytes and nothing
// else: a token's row and its K expert rows are each touched once, 16 bytes a
// lane, with the K rows' accesses in flight together.  Products, sums and
// dots are in fp32, in k order and a fixed tree, and are rounded once.
//
// A token is served by W waves of one workgroup that share its columns: one
// where there are tokens enough to fill the chip, up to 16 where there are
// few.  Pairs whose map entry lies outside [0, T*K) have no row: nothing is
// read or written for them, they add nothing, and their dw is 0.
#include "smoe_elt.h"

namespace smoe {

struct TokArgs {
  const void* tok;   // the token rows that are read [T, H] (scatter's source, the dots' operand)
  const void* rows;  // the expert rows that are read [T*K, H]
  void* out;         // scatter: expert rows; gather: token rows
  long long ld_tok, ld_rows;
  const int32_t* inv_map;
  const float* w;  // NULL: no weights
  float* dw;
  int T, K, H, waves;
};

template <class T, int kMaxK, bool kScatter, bool kDot>
__global__ __launch_bounds__(1024) void tokens_kernel(const TokArgs a) {
  constexpr int V = Elt<T>::kVec;
  __shared__ float part[kDot ? 16 * kMaxK : 1];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per = (blockDim.x >> 6) / a.waves;  // tokens of this workgroup
  const int sub = wave % a.waves, K = a.K, H = a.H;
  const int t = blockIdx.x * per + wave / a.waves;
  const bool live = t < a.T;
  const unsigned R = (unsigned)(a.T * K);
  int r[kMaxK];
  float wk[kMaxK], dot[kMaxK];
#pragma unroll
  for (int k = 0; k < kMaxK; ++k) {
    r[k] = -1;
    wk[k] = 0.0f;
    dot[k] = 0.0f;
    if (k < K && live) {
      r[k] = a.inv_map[(size_t)t * K + k];
      wk[k] = a.w ? a.w[(size_t)t * K + k] : 1.0f;
      if ((unsigned)r[k] >= R) r[k] = -1;
    }
  }
  const T* tok = (const T*)a.tok + (long long)t * a.ld_tok;
  const T* rows = (const T*)a.rows;
  if (live) {
    for (int c = (sub * 64 + lane) * V; c < H; c += a.waves * 64 * V) {
      const int n = H - c;
      float x[V];
      if constexpr (kScatter || kDot) load_f32<T>(tok + c, n, x);
      if constexpr (kScatter) {
        T* dst = (T*)a.out;
        float y[kDot ? kMaxK : 1][V];
        if constexpr (kDot) {
#pragma unroll
          for (int k = 0; k < kMaxK; ++k)
            if (r[k] >= 0) load_f32<T>(rows + (long long)r[k] * a.ld_rows + c, n, y[k]);
        }
#pragma unroll
        for (int k = 0; k < kMaxK; ++k) {
          if (r[k] >= 0) {
            float o[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
              o[i] = wk[k] * x[i];
              if constexpr (kDot) dot[k] = __builtin_fmaf(x[i], y[k][i], dot[k]);
            }
            store_f32<T>(dst + (size_t)r[k] * H + c, n, o);
          }
        }
      } else {
        float y[kMaxK][V], acc[V];
#pragma unroll
        for (int k = 0; k < kMaxK; ++k)
          if (r[k] >= 0) load_f32<T>(rows + (long long)r[k] * a.ld_rows + c, n, y[k]);
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = 0.0f;
#pragma unroll
        for (int k = 0; k < kMaxK; ++k) {
          if (r[k] >= 0) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
              acc[i] = __builtin_fmaf(wk[k], y[k][i], acc[i]);
              if constexpr (kDot) dot[k] = __builtin_fmaf(x[i], y[k][i], dot[k]);
            }
          }
        }
        store_f32<T>((T*)a.out + (size_t)t * H + c, n, acc);
      }
    }
  }
  if constexpr (kDot) {
#pragma unroll
    for (int k = 0; k < kMaxK; ++k) {
      if (k < K) {
        dot[k] = wave_sum_tree(dot[k]);
        if (lane == 0) part[wave * kMaxK + k] = dot[k];
      }
    }
    __syncthreads();
    if (live && sub == 0 && lane < K) {
      float s = 0.0f;
      for (int v = 0; v < a.waves; ++v) s = s + part[(wave + v) * kMaxK + lane];
      a.dw[(size_t)t * K + lane] = s;
    }
  }
}

// Waves a token: a power of two that makes about 4096 of them (16 a compute
// unit), but no more than the row has pieces for, and at most 16.
static int token_waves(int T, int H, int vec) {
  const int chunks = (H + 64 * vec - 1) / (64 * vec);
  int w = 1;
  while (w < 16 && w < chunks && (long long)T * w < 4096) w *= 2;
  return w;
}

template <class T, bool kScatter, bool kDot>
static int tokens_launch(TokArgs a, hipStream_t s) {
  a.waves = token_waves(a.T, a.H, Elt<T>::kVec);
  const int threads = a.waves <= 4 ? 256 : a.waves * 64;
  const int per = threads / 64 / a.waves;
  const dim3 grid((a.T + per - 1) / per), block(threads);
  if ((long long)grid.x * threads > 0xffffffffLL) return SMOE_EINVAL_DIM;
#define SMOE_TK(MK) tokens_kernel<T, MK, kScatter, kDot><<<grid, block, 0, s>>>(a)
  if (a.K <= 1) SMOE_TK(1);
  else if (a.K <= 2) SMOE_TK(2);
  else if (a.K <= 4) SMOE_TK(4);
  else if (a.K <= 8) SMOE_TK(8);
  else if (a.K <= 16) SMOE_TK(16);
  else SMOE_TK(32);
#undef SMOE_TK
  SMOE_RETURN_LAUNCH();
}

template <bool kScatter, bool kDot>
static int tokens_call(const TokArgs& a, int dtype, void* stream) {
  hipStream_t s = (hipStream_t)stream;
  if (dtype == SMOE_BF16) return tokens_launch<bf16_t, kScatter, kDot>(a, s);
  if (dtype == SMOE_F16) return tokens_launch<f16_t, kScatter, kDot>(a, s);
  return tokens_launch<float, kScatter, kDot>(a, s);
}

static int check_tokens(const int32_t* inv_map, const float* w, int T, int K, int H, int dtype) {
  if (T <= 0 || H <= 0) return SMOE_EINVAL_DIM;
  if (K <= 0 || K > 32) return SMOE_EINVAL_TOPK;
  if ((long long)T * K > 0x7fffffffLL) return SMOE_EINVAL_DIM;
  if (dtype < SMOE_BF16 || dtype > SMOE_F32) return SMOE_EINVAL_MODE;
  if (!inv_map) return SMOE_EINVAL_NULL;
  if (((uintptr_t)inv_map | (uintptr_t)w) & 3u) return SMOE_EINVAL_PTRALIGN;
  return SMOE_OK;
}

}  // namespace smoe

using namespace smoe;

extern "C" int smoe_permute_tokens(const void* x, long long ldx, const int32_t* inv_map, const float* w,
                                   int T, int K, int H, int dtype, void* xp, void* stream) {
  const int st = check_tokens(inv_map, w, T, K, H, dtype);
  if (st) return st;
  if (ldx < 0) return SMOE_EINVAL_DIM;
  SMOE_CHECK_ELT(x, dtype);
  SMOE_CHECK_ELT(xp, dtype);
  return tokens_call<true, false>({x, nullptr, xp, ldx, 0, inv_map, w, nullptr, T, K, H, 1}, dtype, stream);
}

extern "C" int smoe_permute_tokens_bwd(const void* dxp, long long lddxp, const void* x, long long ldx,
                                       const int32_t* inv_map, const float* w, int T, int K, int H,
                                       int dtype, void* dx, float* dw, void* stream) {
  const int st = check_tokens(inv_map, w, T, K, H, dtype);
  if (st) return st;
  if (lddxp < 0 || ldx < 0) return SMOE_EINVAL_DIM;
  SMOE_CHECK_ELT(dxp, dtype);
  SMOE_CHECK_ELT(dx, dtype);
  const TokArgs a{x, dxp, dx, ldx, lddxp, inv_map, w, dw, T, K, H, 1};
  if (!dw) return tokens_call<false, false>(a, dtype, stream);
  SMOE_CHECK_ELT(x, dtype);
  SMOE_CHECK_ELT(dw, SMOE_F32);
  return tokens_call<false, true>(a, dtype, stream);
}

extern "C" int smoe_unpermute_tokens(const void* y, long long ldy, const int32_t* inv_map, const float* w,
                                     int T, int K, int H, int dtype, void* out, void* stream) {
  return smoe_permute_tokens_bwd(y, ldy, nullptr, 0, inv_map, w, T, K, H, dtype, out, nullptr, stream);
}

extern "C" int smoe_unpermute_tokens_bwd(const void* dout, long long lddout, const void* y, long long ldy,
                                         const int32_t* inv_map, const float* w, int T, int K, int H,
                                         int dtype, void* dy, float* dw, void* stream) {
  const int st = check_tokens(inv_map, w, T, K, H, dtype);
  if (st) return st;
  if (lddout < 0 || ldy < 0) return SMOE_EINVAL_DIM;
  SMOE_CHECK_ELT(dout, dtype);
  SMOE_CHECK_ELT(dy, dtype);
  const TokArgs a{dout, y, dy, lddout, ldy, inv_map, w, dw, T, K, H, 1};
  if (!dw) return tokens_call<true, false>(a, dtype, stream);
  SMOE_CHECK_ELT(y, dtype);
  SMOE_CHECK_ELT(dw, SMOE_F32);
  return tokens_call<true, true>(a, dtype, stream);
}
