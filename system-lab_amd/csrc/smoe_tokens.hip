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
// Bound by HBM: 16384 x 7168 bf16 rows to 8 experts each 427 us (2.11 GB, 4.95
// TB/s; a 1 GiB copy reaches 5.03), the gradient of 8192 x 4096 fp32 rows from
// 2 experts each 146 us (4.6 TB/s).
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
      // the expert rows eight at a time: eight loads in flight
      constexpr int kG = kMaxK < 8 ? kMaxK : 8;
      if constexpr (kScatter) {
        T* dst = (T*)a.out;
#pragma unroll
        for (int k0 = 0; k0 < kMaxK; k0 += kG) {
          v4u_t p[kDot ? kG : 1];
          if constexpr (kDot) {
#pragma unroll
            for (int k = 0; k < kG; ++k)
              if (r[k0 + k] >= 0) p[k] = load_some<T>(rows + (long long)r[k0 + k] * a.ld_rows + c, n);
          }
#pragma unroll
          for (int k = 0; k < kG; ++k) {
            if (r[k0 + k] >= 0) {
              float o[V], y[V];
              if constexpr (kDot) Elt<T>::unpack(p[k], y);
#pragma unroll
              for (int i = 0; i < V; ++i) {
                o[i] = wk[k0 + k] * x[i];
                if constexpr (kDot) dot[k0 + k] = __builtin_fmaf(x[i], y[i], dot[k0 + k]);
              }
              store_f32<T>(dst + (size_t)r[k0 + k] * H + c, n, o);
            }
          }
        }
      } else {
        float acc[V];
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = 0.0f;
#pragma unroll
        for (int k0 = 0; k0 < kMaxK; k0 += kG) {
          v4u_t p[kG];
#pragma unroll
          for (int k = 0; k < kG; ++k)
            if (r[k0 + k] >= 0) p[k] = load_some<T>(rows + (long long)r[k0 + k] * a.ld_rows + c, n);
#pragma unroll
          for (int k = 0; k < kG; ++k) {
            if (r[k0 + k] >= 0) {
              float y[V];
              Elt<T>::unpack(p[k], y);
#pragma unroll
              for (int i = 0; i < V; ++i) {
                acc[i] = __builtin_fmaf(wk[k0 + k], y[i], acc[i]);
                if constexpr (kDot) dot[k0 + k] = __builtin_fmaf(x[i], y[i], dot[k0 + k]);
              }
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

// The expert sort and the permute of a small batch in one launch.  Every
// workgroup has all the pairs' expert ids in LDS and finds its tokens' rows
// by counting: the row of pair p is the number of pairs of a lower expert, and
// of the same expert before p.  The last workgroup counts the experts' rows.
// The same bytes as the sort's own launches, which a batch this small would
// spend more time on than on its rows.
constexpr int kSortPairs = 2048;
struct SortArgs {
  const int32_t* ids;
  int32_t *row_map, *inv_map, *counts, *offsets, *status;
  int E;
};
template <class T, int kMaxK>
__global__ __launch_bounds__(1024) void tokens_sort_kernel(const TokArgs a, const SortArgs q) {
  constexpr int V = Elt<T>::kVec;
  __shared__ int ids[kSortPairs];
  __shared__ int hist[SMOE_MAX_EXPERTS], bad;
  const int K = a.K, H = a.H, R = a.T * K, E = q.E;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool counting = blockIdx.x == gridDim.x - 1;
  for (int p = threadIdx.x; p < R; p += blockDim.x) ids[p] = q.ids[p];
  if (counting) {
    for (int e = threadIdx.x; e < E; e += blockDim.x) hist[e] = 0;
    if (threadIdx.x == 0) bad = 0;
  }
  __syncthreads();
  if (counting) {
    for (int p = threadIdx.x; p < R; p += blockDim.x) {
      const unsigned e = (unsigned)ids[p];
      if (e < (unsigned)E) atomicAdd(&hist[e], 1);  // whole numbers: any order
      else atomicAdd(&bad, 1);
    }
    __syncthreads();
    if (wave) return;
    const int each = (E + 63) / 64;  // a lane's run of neighbouring experts
    int n = 0;
    for (int i = 0; i < each; ++i)
      if (lane * each + i < E) n += hist[lane * each + i];
    int inc = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(inc, d, 64);
      if (lane >= d) inc += up;
    }
    int at = inc - n;
    for (int i = 0; i < each; ++i) {
      const int e = lane * each + i;
      if (e < E) {
        q.counts[e] = hist[e];
        q.offsets[e] = at;
        at += hist[e];
        if (e == E - 1) q.offsets[E] = at;
      }
    }
    if (lane == 0) *q.status = bad;
    return;
  }
  const int per = (blockDim.x >> 6) / a.waves, sub = wave % a.waves;
  const int t = blockIdx.x * per + wave / a.waves;
  if (t >= a.T) return;
  int r[kMaxK];
  float wk[kMaxK];
#pragma unroll
  for (int k = 0; k < kMaxK; ++k) {
    r[k] = -1;
    wk[k] = 1.0f;
    if (k < K) {
      const int p = t * K + k, e = ids[p];
      if (a.w) wk[k] = a.w[p];
      if ((unsigned)e < (unsigned)E) {
        int n = 0;
        for (int o = lane; o < R; o += 64) {
          const int f = ids[o];
          n += (f >= 0 && f < e) || (f == e && o < p);
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) n += __shfl_xor(n, d, 64);
        r[k] = __builtin_amdgcn_readfirstlane(n);
      }
      if (sub == 0 && lane == 0) {
        q.inv_map[p] = r[k];
        if (r[k] >= 0) q.row_map[r[k]] = p;
      }
    }
  }
  const T* tok = (const T*)a.tok + (long long)t * a.ld_tok;
  for (int c = (sub * 64 + lane) * V; c < H; c += a.waves * 64 * V) {
    float x[V], o[V];
    load_f32<T>(tok + c, H - c, x);
#pragma unroll
    for (int k = 0; k < kMaxK; ++k) {
      if (r[k] >= 0) {
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = wk[k] * x[i];
        store_f32<T>((T*)a.out + (size_t)r[k] * H + c, H - c, o);
      }
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

template <class T>
static int tokens_sort_launch(TokArgs a, const SortArgs& q, hipStream_t s) {
  a.waves = token_waves(a.T, a.H, Elt<T>::kVec);
  const int threads = a.waves <= 4 ? 256 : a.waves * 64;
  const int per = threads / 64 / a.waves;
  const dim3 grid((a.T + per - 1) / per + 1), block(threads);
#define SMOE_TS(MK) tokens_sort_kernel<T, MK><<<grid, block, 0, s>>>(a, q)
  if (a.K <= 1) SMOE_TS(1);
  else if (a.K <= 2) SMOE_TS(2);
  else if (a.K <= 4) SMOE_TS(4);
  else if (a.K <= 8) SMOE_TS(8);
  else if (a.K <= 16) SMOE_TS(16);
  else SMOE_TS(32);
#undef SMOE_TS
  SMOE_RETURN_LAUNCH();
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

extern "C" int smoe_sort_permute_tokens(const void* x, long long ldx, const int32_t* topk_idx, const float* w,
                                        int T, int K, int E, int H, int dtype, int32_t* row_map,
                                        int32_t* inv_map, int32_t* counts, int32_t* offsets, void* xp, void* ws,
                                        size_t ws_bytes, void* stream) {
  int st = check_tokens(inv_map, w, T, K, H, dtype);
  if (st) return st;
  if (ldx < 0) return SMOE_EINVAL_DIM;
  SMOE_CHECK_ELT(x, dtype);
  SMOE_CHECK_ELT(xp, dtype);
  if ((long long)T * K > kSortPairs) {
    st = smoe_route_sort(topk_idx, T, K, E, row_map, inv_map, counts, offsets, ws, ws_bytes, stream);
    return st ? st : smoe_permute_tokens(x, ldx, inv_map, w, T, K, H, dtype, xp, stream);
  }
  if (E <= 0 || E > SMOE_MAX_EXPERTS) return SMOE_EINVAL_EXPERTS;
  if (K > E) return SMOE_EINVAL_TOPK;
  if (!topk_idx || !row_map || !counts || !offsets) return SMOE_EINVAL_NULL;
  if (((uintptr_t)topk_idx | (uintptr_t)row_map | (uintptr_t)counts | (uintptr_t)offsets) & 3u)
    return SMOE_EINVAL_PTRALIGN;
  if (!ws || ws_bytes < smoe_route_sort_workspace_size(T, K, E)) return SMOE_EINVAL_WORKSPACE;
  if ((uintptr_t)ws & 15u) return SMOE_EINVAL_PTRALIGN;
  const TokArgs a{x, nullptr, xp, ldx, 0, inv_map, w, nullptr, T, K, H, 1};
  const SortArgs q{topk_idx, row_map, inv_map, counts, offsets,
                   (int32_t*)((char*)ws + SMOE_ROUTE_STATUS_OFFSET), E};
  hipStream_t s = (hipStream_t)stream;
  if (dtype == SMOE_BF16) return tokens_sort_launch<bf16_t>(a, q, s);
  if (dtype == SMOE_F16) return tokens_sort_launch<f16_t>(a, q, s);
  return tokens_sort_launch<float>(a, q, s);
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
