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
// 16-byte pieces, kNV a lane) between the sum of squares and the scaling, and
// the parameter vectors come from the caches.  The sums over a row are fp32,
// lane by lane and then in a fixed tree.  The sums over rows are fp32 too:
// each workgroup walks its rows with the columns' sums in registers and
// leaves one partial row, and a second launch adds the partial rows in order,
// so a result never depends on which workgroup ran first.
//
// Bound by HBM.  bf16, us and TB/s: in 16384 x 7168 83 (5.7), out 141 (5.0);
// gradients of 16384 x 7168 in 205 (4.6, with dskip), out with a gate a channel
// 162 (4.4), a token 137 (5.1), a value 240 (4.9).  fp16's conversions make its
// gradients 1.2 to 1.4 times as long.  Rows above 16 K 16-bit values take 1024
// threads, whose registers do not hold a gradient's values: they spill.
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

// A workgroup takes blockDim / 64 / waves rows at a time, one every so many
// waves: rows blockIdx.x, + gridDim.x, ... of its places.  A lane keeps g weight
// and v in fp32 between the row's sum and the result (unpacked twice, fp16 took
// 1.5 times as long: its conversions are slow).
template <class T, int kNV, int kThreads, int kGate>
__global__ __launch_bounds__(kThreads) void norm_bwd_kernel(const NormBwd a) {
  const int gate_mode = kGate < 0 ? a.gate_mode : kGate;
  constexpr int V = Elt<T>::kVec;
  __shared__ float red[2][kNormMaxWaves];
  extern __shared__ float cols[];  // [H], where the workgroup has several rows
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per = (blockDim.x >> 6) / a.waves, place = wave / a.waves, sub = wave % a.waves;
  const int c0 = (sub * 64 + lane) * V, step = a.waves * 64 * V, H = a.H;
  // a lane's columns are the same in every row: weight, times a gate a channel,
  // stays in registers
  float col[kNV][V], fac[kNV][V];
#pragma unroll
  for (int j = 0; j < kNV; ++j) {
    const int at = c0 + j * step, left = H - at;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      col[j][i] = 0.0f;
      fac[j][i] = 1.0f;
    }
    if (left > 0) {
      if (a.weight) load_param<T>(a.weight, a.w_f32, at, left, fac[j]);
      if (gate_mode == SMOE_GATE_CHANNEL) {
        float gate[V];
        load_param<T>(a.gate, a.gate_f32, at, left, gate);
#pragma unroll
        for (int i = 0; i < V; ++i) fac[j][i] = fac[j][i] * gate[i];
      }
    }
  }
  int turn = 0;
  for (int t0 = blockIdx.x * per; t0 < a.T; t0 += gridDim.x * per, turn ^= 1) {
    const int t = t0 + place;
    const bool live = t < a.T;  // the last rows may leave places empty
    float dot = 0.0f, rstd = 0.0f, gt = 1.0f;
    v4u_t pg[kNV], pv[kNV], ps[kNV];
    float cc[kNV][V], vv[kNV][V];
    auto full_gate = [&](int at, float* gate) {
      load_param<T>(a.gate, a.gate_f32, (long long)t * a.ldgate + at, H - at, gate);
    };
    if (live) {
      const T* gp = (const T*)a.g + (long long)t * a.ldg;
      const T* vp = (const T*)a.v + (long long)t * a.ldv;
#pragma unroll
      for (int j = 0; j < kNV; ++j) {
        const int at = c0 + j * step;
        if (at + V <= H) {
          pg[j] = load_piece<T>(gp + at);
          pv[j] = load_piece<T>(vp + at);
        } else if (at < H) {
          float f[V];
          load_f32<T>(gp + at, H - at, f);
          pg[j] = Elt<T>::pack(f);
          load_f32<T>(vp + at, H - at, f);
          pv[j] = Elt<T>::pack(f);
        }
      }
      if (a.dskip) {
        const T* sp = (const T*)a.dskip + (long long)t * a.ldskip;
#pragma unroll
        for (int j = 0; j < kNV; ++j) {
          const int at = c0 + j * step;
          if (at + V <= H) ps[j] = load_piece<T>(sp + at);
          else if (at < H) {
            float f[V];
            load_f32<T>(sp + at, H - at, f);
            ps[j] = Elt<T>::pack(f);
          }
        }
      }
      rstd = a.rstd[t];
      if (gate_mode == SMOE_GATE_TOKEN)
        gt = a.gate_f32 ? ((const float*)a.gate)[(long long)t * a.ldgate]
                        : Elt<T>::to_f32(((const T*)a.gate)[(long long)t * a.ldgate]);
      const float scale = rstd * gt;
#pragma unroll
      for (int j = 0; j < kNV; ++j) {
        const int at = c0 + j * step, left = H - at;
        if (left > 0) {
          // the row's sum is of g v weight (times a gate a channel or a value);
          // rstd and a gate a token are the row's and come in after it
          float* g = cc[j];
          float* v = vv[j];
          float gate[V], dfull[V];
          Elt<T>::unpack(pg[j], g);
          Elt<T>::unpack(pv[j], v);
          if (gate_mode == SMOE_GATE_FULL) full_gate(at, gate);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            float c = g[i] * fac[j][i], gv = g[i] * v[i];
            if (gate_mode == SMOE_GATE_FULL) {
              dfull[i] = c * v[i] * rstd;
              c = c * gate[i];
              gv = gv * gate[i];
            }
            g[i] = c;
            dot = __builtin_fmaf(c, v[i], dot);
            // a gate a channel is left out of the columns' sums and applied
            // to the finished ones
            col[j][i] = __builtin_fmaf(gv, scale, col[j][i]);
          }
          if (gate_mode == SMOE_GATE_FULL) {
            if (a.gate_f32) {
              float* d = (float*)a.dgate + (size_t)t * H + at;
              store_f32<float>(d, left < 4 ? left : 4, dfull);
              if (V == 8 && left > 4) store_f32<float>(d + 4, left - 4, dfull + (V == 8 ? 4 : 0));
            } else {
              store_f32<T>((T*)a.dgate + (size_t)t * H + at, left, dfull);
            }
          }
        }
      }
    }
    dot = wave_sum_tree(dot);
    if (a.waves > 1) {
      // a row's use of its half of red ends before the half is written again
      // two rows later, past the next row's barrier
      if (lane == 0) red[turn][wave] = dot;
      __syncthreads();
      dot = 0.0f;
      for (int i = 0; i < a.waves; ++i) dot = dot + red[turn][place * a.waves + i];
    }
    if (!live) continue;
    dot = dot * rstd;  // sum of g n weight: a token's dgate
    if (gate_mode == SMOE_GATE_TOKEN && sub == 0 && lane == 0) {
      if (a.gate_f32) ((float*)a.dgate)[t] = dot;
      else ((T*)a.dgate)[t] = Elt<T>::from_f32(dot);
    }
    // rstd (c - n mean(c n)) = (rstd gate) g weight - (rstd^2 mean(c n)) v
    const float up = rstd * gt, down = rstd * (rstd * (gt * dot / (float)H));
#pragma unroll
    for (int j = 0; j < kNV; ++j) {
      const int at = c0 + j * step, left = H - at;
      if (left > 0) {
        float g[V], sk[V];
        if (a.dskip) Elt<T>::unpack(ps[j], sk);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float c = __builtin_fmaf(-down, vv[j][i], up * cc[j][i]);
          if (a.dskip) c = __builtin_fmaf(a.scale, sk[i], c);
          g[i] = c;
        }
        store_f32<T>((T*)a.dv + (size_t)t * H + at, left, g);
      }
    }
  }
  if (!a.part) return;
  // the places' column sums, added in order, are the workgroup's partial row
  for (int p = 0; p < per; ++p) {
    if (p == place) {
#pragma unroll
      for (int j = 0; j < kNV; ++j) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int c = c0 + j * step + i;
          if (c < H) {
            if (p > 0) col[j][i] = cols[c] + col[j][i];
            if (p + 1 < per) cols[c] = col[j][i];
          }
        }
        const int at = c0 + j * step, left = H - at;
        if (p + 1 == per && left > 0) {
          float* d = a.part + (size_t)blockIdx.x * H + at;
          store_f32<float>(d, left < 4 ? left : 4, col[j]);
          if (V == 8 && left > 4) store_f32<float>(d + 4, left - 4, col[j] + (V == 8 ? 4 : 0));
        }
      }
    }
    if (p + 1 < per) __syncthreads();
  }
}

// The partial rows' column sums S: dweight = S (times a gate a channel), and
// that gate's gradient S w.  64 columns a workgroup, 16 waves over the rows.
template <class T>
__global__ __launch_bounds__(1024) void norm_cols_kernel(const float* part, int G, int H, const void* weight,
                                                         int w_f32, const void* gate, int gate_f32, void* dweight,
                                                         void* dgate) {
  __shared__ float acc[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane;
  float s = 0.0f;
  if (c < H) {
    int g = wave;
    for (; g + 7 * 16 < G; g += 8 * 16) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = part[(size_t)(g + i * 16) * H + c];
#pragma unroll
      for (int i = 0; i < 8; ++i) s = s + v[i];
    }
    for (; g < G; g += 16) s = s + part[(size_t)g * H + c];
  }
  acc[wave][lane] = s;
  __syncthreads();
  if (wave || c >= H) return;
  s = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) s = s + acc[i][lane];
  auto param = [&](const void* p, int f32) { return f32 ? ((const float*)p)[c] : Elt<T>::to_f32(((const T*)p)[c]); };
  auto put = [&](void* p, int f32, float v) {
    if (f32) ((float*)p)[c] = v;
    else ((T*)p)[c] = Elt<T>::from_f32(v);
  };
  if (dweight) put(dweight, w_f32, gate ? s * param(gate, gate_f32) : s);
  if (dgate) put(dgate, gate_f32, weight ? s * param(weight, w_f32) : s);
}

// Waves a row (a power of two up to 16) so that a lane holds about `pieces`;
// kNV, the pieces a lane, then covers the rest.
static int norm_waves(int H, int vec, int pieces) {
  int w = 1;
  while (w < kNormMaxWaves && 64 * vec * pieces * w < H) w *= 2;
  return w;
}

// The backward pass: up to four pieces a lane, so that rows up to 2048 16-bit
// values need one wave and no barrier (six or eight pieces were slower, by
// registers; two as well, by barriers); threads of a workgroup, rows it holds
// at a time; and workgroups: two rows a place at least, so that the partial
// rows stay a small part of the traffic, two a compute unit at most.
constexpr int kBwdPieces = 4;
struct NormBwdPlan {
  int waves, threads, per, groups;
};
static NormBwdPlan norm_bwd_plan(int T, int H, int dtype) {
  NormBwdPlan p;
  p.waves = norm_waves(H, dtype == SMOE_F32 ? 4 : 8, kBwdPieces);
  p.threads = p.waves <= 4 ? 256 : p.waves * 64;
  p.per = p.threads / 64 / p.waves;
  const int g = (T + 2 * p.per - 1) / (2 * p.per);
  p.groups = g < 512 ? g : 512;
  return p;
}

static int check_norm(int T, int H, int dtype, int gate_mode, int param_f32) {
  if (T <= 0 || H <= 0 || H > kNormMaxH) return SMOE_EINVAL_DIM;
  if (dtype < SMOE_BF16 || dtype > SMOE_F32) return SMOE_EINVAL_MODE;
  if (gate_mode < SMOE_GATE_NONE || gate_mode > SMOE_GATE_FULL) return SMOE_EINVAL_MODE;
  if (param_f32 < 0 || param_f32 > 3) return SMOE_EINVAL_MODE;
  return SMOE_OK;
}

// kNV for a row of H at `waves` waves: the next of 1, 2, 4, 8, and for fp32,
// whose pieces hold half as many values, 16.
#define SMOE_NORM_NV(need, CALL)                           \
  do {                                                     \
    if ((need) <= 1) CALL(1);                              \
    else if ((need) <= 2) CALL(2);                         \
    else if ((need) <= 4) CALL(4);                         \
    else if (V == 8 || (need) <= 8) CALL(8);               \
    else CALL((V == 4 ? 16 : 8));                          \
  } while (0)

template <class T, bool kOut>
static int norm_fwd_launch(NormFwd a, hipStream_t s) {
  constexpr int V = Elt<T>::kVec;
  a.waves = norm_waves(a.H, V, 2);
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
  const NormBwdPlan p = norm_bwd_plan(a.T, a.H, Elt<T>::kDtype);
  a.waves = p.waves;
  const int need = (a.H + a.waves * 64 * V - 1) / (a.waves * 64 * V), G = p.groups;
  const dim3 grid(G), block(p.threads);
  const size_t lds = a.part && p.per > 1 ? a.H * sizeof(float) : 0;
  if (p.threads <= 256) {
    // the common row lengths: every count of pieces and every gate by itself
#define SMOE_NB(NV, GATE) norm_bwd_kernel<T, NV, 256, GATE><<<grid, block, lds, s>>>(a)
#define SMOE_NBG(NV)                                                   \
  do {                                                                 \
    if (a.gate_mode == SMOE_GATE_NONE) SMOE_NB(NV, SMOE_GATE_NONE);    \
    else if (a.gate_mode == SMOE_GATE_CHANNEL) SMOE_NB(NV, SMOE_GATE_CHANNEL); \
    else if (a.gate_mode == SMOE_GATE_TOKEN) SMOE_NB(NV, SMOE_GATE_TOKEN);     \
    else SMOE_NB(NV, SMOE_GATE_FULL);                                  \
  } while (0)
    if (need <= 1) SMOE_NBG(1);
    else if (need <= 2) SMOE_NBG(2);
    else if (need <= 3) SMOE_NBG(3);
    else SMOE_NBG(4);
  } else if (p.threads <= 512) {
    norm_bwd_kernel<T, 4, 512, -1><<<grid, block, lds, s>>>(a);
  } else {
    if (need <= 4) norm_bwd_kernel<T, 4, 1024, -1><<<grid, block, lds, s>>>(a);
    else if (V == 8 || need <= 8) norm_bwd_kernel<T, 8, 1024, -1><<<grid, block, lds, s>>>(a);
    else norm_bwd_kernel<T, V == 4 ? 16 : 8, 1024, -1><<<grid, block, lds, s>>>(a);
  }
#undef SMOE_NBG
#undef SMOE_NB
  if (a.part)
    norm_cols_kernel<T><<<dim3((a.H + 63) / 64), dim3(1024), 0, s>>>(
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
  // whichever element type needs more
  const int a = norm_bwd_plan(T, H, SMOE_BF16).groups, b = norm_bwd_plan(T, H, SMOE_F32).groups;
  return (size_t)(a > b ? a : b) * H * sizeof(float);
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
