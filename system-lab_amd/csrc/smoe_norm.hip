// smoe_norm.hip — the RMS norms before and after a block, with the block's
// gate and the scaled residual, and their gradients (gfx950).
//
//   in    h   = x rstd w,                      rstd = 1 / sqrt(mean(x^2) + eps)
//   out   out = s x + gate (y rstd w),         rstd of y
// and with n = v rstd (v the normed operand), g the incoming gradient times
// the gate, c = g w:
//   dv    = rstd (c - n mean(c n))  [+ s dskip: the residual's own gradient]
//   dw    = sum over rows of g n,   dgate = (dout n w) summed as it was broadcast
//
// Every row is read once: W waves of one workgroup hold it in registers (raw
// 16-byte pieces, NV a lane) between the sum of squares and the scaling, and
// the parameter vectors come from the caches.  The sums over a row are fp32,
// lane by lane and then in a fixed tree.  The sums over rows are fp32 too:
// each workgroup walks its rows with the columns' sums in registers and
// leaves one partial row, and a second launch adds the partial rows in order,
// so a result never depends on which workgroup ran first.
#include "smoe_elt.h"

namespace smoe {

constexpr int kNormMaxH = 65536;
constexpr int kNormMaxWaves = 16;

// Sum over the W waves of a row; every lane gets it.  kSync rows a block.
__device__ __forceinline__ float row_sum(float v, float* red, int waves, int wave) {
  v = wave_sum_tree(v);
  if (waves == 1) return v;
  if ((threadIdx.x & 63) == 0) red[wave] = v;
  __syncthreads();
  const int first = wave / waves * waves;
  float s = 0.0f;
  for (int i = 0; i < waves; ++i) s = s + red[first + i];
  return s;
}

struct NormFwd {
  const void *v, *x, *weight, *gate;
  void* out;
  float* rstd;
  long long ldv, ldx, ldg;
  float scale, eps;
  int T, H, waves, gate_mode, w_f32, gate_f32;
};

template <class T, int kNV, bool kOut>
__global__ __launch_bounds__(1024) void norm_fwd_kernel(const NormFwd a) {
  constexpr int V = Elt<T>::kVec;
  __shared__ float red[kNormMaxWaves];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per = (blockDim.x >> 6) / a.waves, sub = wave % a.waves;
  const int t0 = blockIdx.x * per + wave / a.waves;
  const bool live = t0 < a.T;
  const int t = live ? t0 : a.T - 1;  // idle waves of the last block repeat a row, unstored
  const int c0 = (sub * 64 + lane) * V, step = a.waves * 64 * V, H = a.H;
  const T* v = (const T*)a.v + (long long)t * a.ldv;
  v4u_t p[kNV];
  float tail[V];
#pragma unroll
  for (int j = 0; j < kNV; ++j) {
    const int c = c0 + j * step;
    if (c + V <= H) p[j] = load_piece<T>(v + c);
    else {
      load_f32<T>(v + c, H - c, tail);
      p[j] = Elt<T>::pack(tail);
    }
  }
  float ss = 0.0f;
#pragma unroll
  for (int j = 0; j < kNV; ++j) {
    float f[V];
    Elt<T>::unpack(p[j], f);
#pragma unroll
    for (int i = 0; i < V; ++i) ss = __builtin_fmaf(f[i], f[i], ss);
  }
  ss = row_sum(ss, red, a.waves, wave);
  const float rstd = 1.0f / __builtin_sqrtf(ss / (float)H + a.eps);
  if (!live) return;
  if (sub == 0 && lane == 0) a.rstd[t] = rstd;
  float gt = 1.0f;
  if constexpr (kOut) {
    if (a.gate_mode == SMOE_GATE_TOKEN)
      gt = a.gate_f32 ? ((const float*)a.gate)[(long long)t * a.ldg]
                      : Elt<T>::to_f32(((const T*)a.gate)[(long long)t * a.ldg]);
  }
#pragma unroll
  for (int j = 0; j < kNV; ++j) {
    const int c = c0 + j * step;
    if (c < H) {
      const int n = H - c;
      float f[V], w[V];
      Elt<T>::unpack(p[j], f);
      if (a.weight) load_param<T>(a.weight, a.w_f32, c, n, w);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        f[i] = f[i] * rstd;
        if (a.weight) f[i] = f[i] * w[i];
      }
      if constexpr (kOut) {
        float x[V], g[V];
        load_f32<T>((const T*)a.x + (long long)t * a.ldx + c, n, x);
        if (a.gate_mode == SMOE_GATE_CHANNEL) load_param<T>(a.gate, a.gate_f32, c, n, g);
        else if (a.gate_mode == SMOE_GATE_FULL) load_param<T>(a.gate, a.gate_f32, (long long)t * a.ldg + c, n, g);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          if (a.gate_mode >= SMOE_GATE_CHANNEL && a.gate_mode != SMOE_GATE_TOKEN) f[i] = f[i] * g[i];
          else f[i] = f[i] * gt;
          f[i] = __builtin_fmaf(a.scale, x[i], f[i]);
        }
      }
      store_f32<T>((T*)a.out + (size_t)t * H + c, n, f);
    }
  }
}

struct NormBwd {
  const void *g, *v, *weight, *gate, *dskip;
  const float* rstd;
  void *dv, *dgate;  // dgate: per token or per value here, per channel in the column pass
  float* part;       // [gridDim.x, H] column sums, or NULL
  long long ldg, ldv, ldgate, ldskip;
  float scale;
  int T, H, waves, gate_mode, w_f32, gate_f32;
};

// One row at a time a workgroup, rows blockIdx.x, + gridDim.x, ...
template <class T, int kNV>
__global__ __launch_bounds__(1024) void norm_bwd_kernel(const NormBwd a) {
  constexpr int V = Elt<T>::kVec;
  __shared__ float red[2][2 * kNormMaxWaves];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c0 = threadIdx.x * V, step = a.waves * 64 * V, H = a.H;
  float col[kNV][V];
#pragma unroll
  for (int j = 0; j < kNV; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) col[j][i] = 0.0f;
  int turn = 0;
  for (int t = blockIdx.x; t < a.T; t += gridDim.x, turn ^= 1) {
    const float rstd = a.rstd[t];
    float gt = 1.0f;
    if (a.gate_mode == SMOE_GATE_TOKEN)
      gt = a.gate_f32 ? ((const float*)a.gate)[(long long)t * a.ldgate]
                      : Elt<T>::to_f32(((const T*)a.gate)[(long long)t * a.ldgate]);
    const T* gp = (const T*)a.g + (long long)t * a.ldg;
    const T* vp = (const T*)a.v + (long long)t * a.ldv;
    float cc[kNV][V], nn[kNV][V];
    float dot = 0.0f, dg = 0.0f;
#pragma unroll
    for (int j = 0; j < kNV; ++j) {
      const int c = c0 + j * step, n = H - c;
      if (n > 0) {
        float w[V], gate[V];
        load_f32<T>(gp + c, n, cc[j]);
        load_f32<T>(vp + c, n, nn[j]);
        if (a.weight) load_param<T>(a.weight, a.w_f32, c, n, w);
        if (a.gate_mode == SMOE_GATE_CHANNEL) load_param<T>(a.gate, a.gate_f32, c, n, gate);
        else if (a.gate_mode == SMOE_GATE_FULL) load_param<T>(a.gate, a.gate_f32, (long long)t * a.ldgate + c, n, gate);
        float full[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float g = cc[j][i];
          nn[j][i] = nn[j][i] * rstd;
          const float gn = g * nn[j][i];
          const float gnw = a.weight ? gn * w[i] : gn;
          if (a.gate_mode == SMOE_GATE_TOKEN) dg = dg + gnw;
          if (a.gate_mode == SMOE_GATE_FULL) full[i] = gnw;
          // the column sums are of g n before a gate a channel, which the
          // column pass applies to the finished sum
          if (a.gate_mode == SMOE_GATE_FULL) g = g * gate[i];
          else g = g * gt;
          col[j][i] = __builtin_fmaf(g, nn[j][i], col[j][i]);
          if (a.gate_mode == SMOE_GATE_CHANNEL) g = g * gate[i];
          cc[j][i] = a.weight ? g * w[i] : g;
          dot = __builtin_fmaf(cc[j][i], nn[j][i], dot);
        }
        if (a.gate_mode == SMOE_GATE_FULL) {
          if (a.gate_f32) {
            float* d = (float*)a.dgate + (size_t)t * H + c;
            store_f32<float>(d, n < 4 ? n : 4, full);
            if (V == 8 && n > 4) store_f32<float>(d + 4, n - 4, full + (V == 8 ? 4 : 0));
          } else {
            store_f32<T>((T*)a.dgate + (size_t)t * H + c, n, full);
          }
        }
      }
    }
    // both row sums; a row's use of its half of red ends before the half is
    // written again two rows later, past the next row's barrier
    dot = wave_sum_tree(dot);
    dg = wave_sum_tree(dg);
    if (a.waves > 1) {
      if (lane == 0) {
        red[turn][wave] = dot;
        red[turn][kNormMaxWaves + wave] = dg;
      }
      __syncthreads();
      dot = 0.0f;
      dg = 0.0f;
      for (int i = 0; i < a.waves; ++i) {
        dot = dot + red[turn][i];
        dg = dg + red[turn][kNormMaxWaves + i];
      }
    }
    if (a.gate_mode == SMOE_GATE_TOKEN && threadIdx.x == 0) {
      if (a.gate_f32) ((float*)a.dgate)[t] = dg;
      else ((T*)a.dgate)[t] = Elt<T>::from_f32(dg);
    }
    const float mean = dot / (float)H;
#pragma unroll
    for (int j = 0; j < kNV; ++j) {
      const int c = c0 + j * step, n = H - c;
      if (n > 0) {
        float sk[V];
        if (a.dskip) load_f32<T>((const T*)a.dskip + (long long)t * a.ldskip + c, n, sk);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float d = rstd * __builtin_fmaf(-nn[j][i], mean, cc[j][i]);
          if (a.dskip) d = __builtin_fmaf(a.scale, sk[i], d);
          cc[j][i] = d;
        }
        store_f32<T>((T*)a.dv + (size_t)t * H + c, n, cc[j]);
      }
    }
  }
  if (a.part) {
#pragma unroll
    for (int j = 0; j < kNV; ++j) {
      const int c = c0 + j * step, n = H - c;
      if (n > 0) {
        float* d = a.part + (size_t)blockIdx.x * H + c;
        store_f32<float>(d, n < 4 ? n : 4, col[j]);
        if (V == 8 && n > 4) store_f32<float>(d + 4, n - 4, col[j] + (V == 8 ? 4 : 0));
      }
    }
  }
}

// The partial rows' column sums S: dweight = S (times a gate a channel), and
// that gate's gradient S w.  64 columns a workgroup, 4 waves over the rows.
template <class T>
__global__ __launch_bounds__(256) void norm_cols_kernel(const float* part, int G, int H, const void* weight,
                                                        int w_f32, const void* gate, int gate_f32, void* dweight,
                                                        void* dgate) {
  __shared__ float acc[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane;
  float s = 0.0f;
  if (c < H)
    for (int g = wave; g < G; g += 4) s = s + part[(size_t)g * H + c];
  acc[wave][lane] = s;
  __syncthreads();
  if (wave || c >= H) return;
  s = acc[0][lane] + acc[1][lane] + acc[2][lane] + acc[3][lane];
  auto param = [&](const void* p, int f32) { return f32 ? ((const float*)p)[c] : Elt<T>::to_f32(((const T*)p)[c]); };
  auto put = [&](void* p, int f32, float v) {
    if (f32) ((float*)p)[c] = v;
    else ((T*)p)[c] = Elt<T>::from_f32(v);
  };
  if (dweight) put(dweight, w_f32, gate ? s * param(gate, gate_f32) : s);
  if (dgate) put(dgate, gate_f32, weight ? s * param(weight, w_f32) : s);
}

// Waves a row (a power of two up to 16) so that a lane holds about two
// pieces; kNV, the pieces a lane, then covers the rest.
static int norm_waves(int H, int vec) {
  int w = 1;
  while (w < kNormMaxWaves && 64 * vec * 2 * w < H) w *= 2;
  return w;
}

// Workgroups of the backward pass: enough rows each (8) that the partial
// rows stay a small part of the traffic, and no more groups than keep the
// chip full.
static int norm_bwd_groups(int T) {
  const int g = (T + 7) / 8;
  return g < 1024 ? g : 1024;
}

static int check_norm(int T, int H, int dtype, int gate_mode, int param_f32) {
  if (T <= 0 || H <= 0 || H > kNormMaxH) return SMOE_EINVAL_DIM;
  if (dtype < SMOE_BF16 || dtype > SMOE_F32) return SMOE_EINVAL_MODE;
  if (gate_mode < SMOE_GATE_NONE || gate_mode > SMOE_GATE_FULL) return SMOE_EINVAL_MODE;
  if (param_f32 < 0 || param_f32 > 3) return SMOE_EINVAL_MODE;
  return SMOE_OK;
}

// kNV for a row of H at `waves` waves: the next of 1, 2, 4, 8, 16.
#define SMOE_NORM_NV(need, CALL) \
  do {                           \
    if ((need) <= 1) CALL(1);    \
    else if ((need) <= 2) CALL(2); \
    else if ((need) <= 4) CALL(4); \
    else if ((need) <= 8) CALL(8); \
    else CALL(16);               \
  } while (0)

template <class T, bool kOut>
static int norm_fwd_launch(NormFwd a, hipStream_t s) {
  constexpr int V = Elt<T>::kVec;
  a.waves = norm_waves(a.H, V);
  const int need = (a.H + a.waves * 64 * V - 1) / (a.waves * 64 * V);
  const int threads = a.waves <= 4 ? 256 : a.waves * 64, per = threads / 64 / a.waves;
  const dim3 grid((a.T + per - 1) / per), block(threads);
  if ((long long)grid.x * threads > 0xffffffffLL) return SMOE_EINVAL_DIM;
#define SMOE_NF(NV) norm_fwd_kernel<T, NV, kOut><<<grid, block, 0, s>>>(a)
  SMOE_NORM_NV(need, SMOE_NF);
#undef SMOE_NF
  SMOE_RETURN_LAUNCH();
}

template <bool kOut>
static int norm_fwd_call(const NormFwd& a, int dtype, void* stream) {
  hipStream_t s = (hipStream_t)stream;
  if (dtype == SMOE_BF16) return norm_fwd_launch<bf16_t, kOut>(a, s);
  if (dtype == SMOE_F16) return norm_fwd_launch<f16_t, kOut>(a, s);
  return norm_fwd_launch<float, kOut>(a, s);
}

template <class T>
static int norm_bwd_launch(NormBwd a, void* dweight, void* dgate_ch, hipStream_t s) {
  constexpr int V = Elt<T>::kVec;
  a.waves = norm_waves(a.H, V);
  const int need = (a.H + a.waves * 64 * V - 1) / (a.waves * 64 * V);
  const int G = norm_bwd_groups(a.T);
  const dim3 grid(G), block(a.waves * 64);
#define SMOE_NB(NV) norm_bwd_kernel<T, NV><<<grid, block, 0, s>>>(a)
  SMOE_NORM_NV(need, SMOE_NB);
#undef SMOE_NB
  if (a.part)
    norm_cols_kernel<T><<<dim3((a.H + 63) / 64), dim3(256), 0, s>>>(
        a.part, G, a.H, a.weight, a.w_f32, a.gate_mode == SMOE_GATE_CHANNEL ? a.gate : nullptr, a.gate_f32,
        dweight, dgate_ch);
  SMOE_RETURN_LAUNCH();
}

static int norm_bwd_call(NormBwd a, int dtype, void* dweight, void* dgate, void* ws, size_t ws_bytes,
                         void* stream) {
  const bool cols = dweight || (dgate && a.gate_mode == SMOE_GATE_CHANNEL);
  if (cols) {
    if (!ws || ws_bytes < smoe_block_norm_bwd_workspace_size(a.T, a.H)) return SMOE_EINVAL_WORKSPACE;
    if ((uintptr_t)ws & 15u) return SMOE_EINVAL_PTRALIGN;
    a.part = (float*)ws;
  }
  void* ch = a.gate_mode == SMOE_GATE_CHANNEL ? dgate : nullptr;
  a.dgate = ch ? nullptr : dgate;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == SMOE_BF16) return norm_bwd_launch<bf16_t>(a, dweight, ch, s);
  if (dtype == SMOE_F16) return norm_bwd_launch<f16_t>(a, dweight, ch, s);
  return norm_bwd_launch<float>(a, dweight, ch, s);
}

}  // namespace smoe

using namespace smoe;

extern "C" int smoe_block_norm_in(const void* x, long long ldx, const void* weight, int param_f32, float eps,
                                  int T, int H, int dtype, void* h, float* rstd, void* stream) {
  const int st = check_norm(T, H, dtype, SMOE_GATE_NONE, param_f32);
  if (st) return st;
  if (ldx < 0 || !(eps > 0.0f)) return SMOE_EINVAL_DIM;
  SMOE_CHECK_ELT(x, dtype);
  SMOE_CHECK_OPT(weight, (param_f32 & 1) ? SMOE_F32 : dtype);
  SMOE_CHECK_ELT(h, dtype);
  SMOE_CHECK_ELT(rstd, SMOE_F32);
  return norm_fwd_call<false>({x, nullptr, weight, nullptr, h, rstd, ldx, 0, 0, 0.0f, eps, T, H, 1, SMOE_GATE_NONE,
                               param_f32 & 1, 0}, dtype, stream);
}

extern "C" int smoe_block_norm_out(const void* y, long long ldy, const void* x, long long ldx, const void* weight,
                                   const void* gate, long long ldgate, int gate_mode, int param_f32,
                                   float residual_scale, float eps, int T, int H, int dtype, void* out,
                                   float* rstd, void* stream) {
  const int st = check_norm(T, H, dtype, gate_mode, param_f32);
  if (st) return st;
  if (ldy < 0 || ldx < 0 || ldgate < 0 || !(eps > 0.0f)) return SMOE_EINVAL_DIM;
  SMOE_CHECK_ELT(y, dtype);
  SMOE_CHECK_ELT(x, dtype);
  SMOE_CHECK_OPT(weight, (param_f32 & 1) ? SMOE_F32 : dtype);
  if (gate_mode != SMOE_GATE_NONE) SMOE_CHECK_ELT(gate, (param_f32 & 2) ? SMOE_F32 : dtype);
  SMOE_CHECK_ELT(out, dtype);
  SMOE_CHECK_ELT(rstd, SMOE_F32);
  return norm_fwd_call<true>({y, x, weight, gate, out, rstd, ldy, ldx, ldgate, residual_scale, eps, T, H, 1,
                              gate_mode, param_f32 & 1, param_f32 >> 1}, dtype, stream);
}

extern "C" size_t smoe_block_norm_bwd_workspace_size(int T, int H) {
  if (T <= 0 || H <= 0 || H > kNormMaxH) return 0;
  return (size_t)norm_bwd_groups(T) * H * sizeof(float);
}

extern "C" int smoe_block_norm_in_bwd(const void* dh, long long lddh, const void* x, long long ldx,
                                      const float* rstd, const void* weight, int param_f32, const void* dskip,
                                      long long ldskip, float skip_scale, int T, int H, int dtype, void* dx,
                                      void* dweight, void* ws, size_t ws_bytes, void* stream) {
  const int st = check_norm(T, H, dtype, SMOE_GATE_NONE, param_f32);
  if (st) return st;
  if (lddh < 0 || ldx < 0 || ldskip < 0) return SMOE_EINVAL_DIM;
  SMOE_CHECK_ELT(dh, dtype);
  SMOE_CHECK_ELT(x, dtype);
  SMOE_CHECK_ELT(rstd, SMOE_F32);
  SMOE_CHECK_OPT(weight, (param_f32 & 1) ? SMOE_F32 : dtype);
  SMOE_CHECK_OPT(dweight, (param_f32 & 1) ? SMOE_F32 : dtype);
  SMOE_CHECK_OPT(dskip, dtype);
  SMOE_CHECK_ELT(dx, dtype);
  return norm_bwd_call({dh, x, weight, nullptr, dskip, rstd, dx, nullptr, nullptr, lddh, ldx, 0, ldskip, skip_scale,
                        T, H, 1, SMOE_GATE_NONE, param_f32 & 1, 0}, dtype, dweight, nullptr, ws, ws_bytes, stream);
}

extern "C" int smoe_block_norm_out_bwd(const void* dout, long long lddout, const void* y, long long ldy,
                                       const float* rstd, const void* weight, const void* gate, long long ldgate,
                                       int gate_mode, int param_f32, int T, int H, int dtype, void* dy,
                                       void* dweight, void* dgate, void* ws, size_t ws_bytes, void* stream) {
  const int st = check_norm(T, H, dtype, gate_mode, param_f32);
  if (st) return st;
  if (lddout < 0 || ldy < 0 || ldgate < 0) return SMOE_EINVAL_DIM;
  SMOE_CHECK_ELT(dout, dtype);
  SMOE_CHECK_ELT(y, dtype);
  SMOE_CHECK_ELT(rstd, SMOE_F32);
  SMOE_CHECK_OPT(weight, (param_f32 & 1) ? SMOE_F32 : dtype);
  SMOE_CHECK_OPT(dweight, (param_f32 & 1) ? SMOE_F32 : dtype);
  if (gate_mode != SMOE_GATE_NONE) {
    SMOE_CHECK_ELT(gate, (param_f32 & 2) ? SMOE_F32 : dtype);
    SMOE_CHECK_ELT(dgate, (param_f32 & 2) ? SMOE_F32 : dtype);
  }
  SMOE_CHECK_ELT(dy, dtype);
  return norm_bwd_call({dout, y, weight, gate, nullptr, rstd, dy, nullptr, nullptr, lddout, ldy, ldgate, 0, 0.0f, T, H,
                        1, gate_mode, param_f32 & 1, param_f32 >> 1}, dtype, dweight,
                       gate_mode == SMOE_GATE_NONE ? nullptr : dgate, ws, ws_bytes, stream);
}
