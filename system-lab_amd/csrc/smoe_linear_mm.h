// smoe_linear_mm.h — the tiled MFMA kernels of linear_act and its gradients
// (gfx950).
//
// One kernel, three products (kWhat):
//   kFwd    D[m][n] = sum_k x[m][k] W[n][k]    both summed along their rows
//   kDgrad  D[m][k] = sum_n dz[m][n] W[n][k]   W's rows run across the sum
//   kWgrad  D[n][k] = sum_r dz[r][n] x[r][k]   both operands' rows run across it
//
// A workgroup owns a kBM x kBN tile of one expert at a time, a wave kRB x kCB
// blocks of 16 x 16 of it.  A step is 64 terms of the sum of both operands,
// staged in LDS by direct global->LDS loads (three left stages, two right ones)
// two steps ahead.
//
// "Row" operands (the sum along the row) lie in LDS as 128-byte rows in the
// swizzled order of smoe_mfma.h and are read 16 bytes a lane.  "Turned"
// operands lie as they do in memory, 64 rows of the tile's columns, and are
// read by ds_read_b64_tr_b16, which hands every lane four rows of one column:
// no transposed copy of weights or activations is ever made.  Their 16-byte
// chunks are swizzled by the row so that the 16 lanes of a read touch
// distinct banks.
//
// The right operand goes into the MFMA first, so that a lane holds four
// neighbouring columns of one output row; and the tile's columns are dealt
// to the blocks such that a lane's blocks pair up to runs of 8 columns: it
// stores whole 16-byte pieces, with no staging.  For SwiGLU the blocks alternate
// between gate and up rows of W, and gate and up of a value meet in a lane.
//
// Operands whose rows do not lie in 16-byte pieces at 16-byte addresses (odd
// lengths, odd strides: kAny) take another way into the same LDS places: by
// registers, a step further ahead, as the direct loads need the alignment.
// us at R = K = 4000, N = 4004 against the aligned 4096^3 of the same tiles:
// 236, dx 286, dW 382 against 109, 109, 116.
//
// Bound by the matrix unit at the clock that the chip's power leaves it: 8192^3
// 780 us (1409 TFLOP/s), dx 784, dW 835; 8192 x 4096 x 14336 700 (1374).  With
// experts by their last tiles' empty rows and, in dW, by few steps a tile:
// 65536 rows over 128 experts, 2048 x 1536, 462, dx 454, dW 580.  (Boxes differ by
// 7%; the library's product took 697 to 755 for 8192^3 on them.)
//
// Terms past the end of the sum (K % 64, an expert's last rows) are loaded
// from a 16-byte zero for both operands.  Rows and columns past the tile's end
// repeat the last valid ones and are not stored.
#pragma once

#include "smoe_linear.h"
#include "smoe_mfma.h"

namespace smoe {

__device__ __attribute__((aligned(16))) const uint32_t g_zero16[4] = {0, 0, 0, 0};

constexpr int kStep = 64;  // terms of the sum a step: 128 bytes of a row operand

// A direct load of 16 bytes a lane from the lane's own address.
__device__ __forceinline__ void dma16_at(const void* p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(p) : "memory");
}

typedef short v4s_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s_t* lds_v4s;

template <int kWR_, int kWN_, int kRB_, int kCB_>
struct MmCfg {
  static constexpr int kWR = kWR_, kWN = kWN_, kRB = kRB_, kCB = kCB_;
  static_assert(kCB == 4, "col_of");
  static constexpr int kWaves = kWR * kWN, kThreads = kWaves * 64;
  static constexpr int kBM = kWR * kRB * 16, kBN = kWN * kCB * 16;
  static constexpr int kABytes = kBM * 128, kBBytes = kBN * 128;
  static constexpr int kB0 = 3 * kABytes, kLds = kB0 + 2 * kBBytes;  // three left stages, two right ones
  static constexpr int kASegs = kABytes / 1024 / kWaves, kBSegs = kBBytes / 1024 / kWaves;
  static_assert(kASegs * kWaves * 1024 == kABytes && kBSegs * kWaves * 1024 == kBBytes, "segments");
  static_assert(kLds <= 160 * 1024, "LDS");
};

// Swizzles of turned operands: XORed into the 16-byte chunk index of row k.
// Left: a read takes 4 rows x 32 contiguous bytes, so rows move by 32-byte
// units.  Right: 4 rows x 4 neighbouring chunks, 8 bytes of each, so rows
// move by four chunks: 16 places of the 256-byte bank round.
__device__ __forceinline__ int swz_left(int k) { return ((k & 3) | ((k >> 3) & 1) << 2) << 1; }
__device__ __forceinline__ int swz_right(int k) { return (k & 3) << 2; }

// Column (of a wave's 64) that block j's index r (0..15, four to a lane
// quarter) stands for: a quarter's two neighbouring blocks make 8 columns in a
// run, the four quarters' runs 32, so that one store of 16 bytes a lane
// writes 64 contiguous bytes of 16 rows.
__device__ __forceinline__ int col_of(int j, int r) { return (j >> 1) * 32 + (r >> 2) * 8 + (j & 1) * 4 + (r & 3); }

// One output tile: rows m0 .. + mrows, columns n0 .. + ncols of expert e, the
// sum over len terms from `lo` (kWgrad: the expert's first row; cut sums: the
// share's first step).
struct MmTile {
  int e, m0, mrows, n0, ncols, len;
  long long lo;
};

// The weight gradients' tiles first .. last of an XCD: eighths of the work, not
// of the tiles, as an expert's tiles cost its steps and about kOver more for
// the store.  Every wave for itself; each lane counts neighbouring experts.
__device__ __forceinline__ void share_work(const LinArgs& a, int tiles, int xcd, int* first, int* last) {
  constexpr int kOver = 6;
  auto cost = [&](int e) {
    const int n = a.offsets ? clamp_row(a.offsets, e + 1, a.R) - clamp_row(a.offsets, e, a.R) : a.R;
    return (long long)((n > 0 ? (n + kStep - 1) / kStep : 0) + kOver);
  };
  const int lane = threadIdx.x & 63, each = (a.E + 63) / 64;
  long long mine = 0;
  for (int i = 0; i < each; ++i)
    if (lane * each + i < a.E) mine += cost(lane * each + i) * tiles;
  long long inc = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const long long up = __shfl_up(inc, d, 64);
    if (lane >= d) inc += up;
  }
  const long long total = __shfl(inc, 63, 64);
  // the first tile that starts at or after a point of the work
  auto tile_from = [&](long long at) {
    if (at >= total) return a.E * tiles;
    const int src = __builtin_ctzll(__ballot(at < inc));
    long long left = at - __shfl(inc - mine, src, 64);
    int e = src * each;
    for (; e < a.E; ++e) {
      const long long c = cost(e) * tiles;
      if (left < c) break;
      left -= c;
    }
    const long long c = cost(e);
    return e * tiles + (int)((left + c - 1) / c);
  };
  *first = __builtin_amdgcn_readfirstlane(tile_from(total * xcd / 8));
  *last = __builtin_amdgcn_readfirstlane(tile_from(total * (xcd + 1) / 8));
}

template <class T, class C, int kWhat, int kAct, bool kAny>
__global__ __launch_bounds__(C::kThreads, 2) void linear_mm_kernel(const LinArgs a) {
  constexpr int kBM = C::kBM, kBN = C::kBN, kRB = C::kRB, kCB = C::kCB;
  constexpr int kASegs = C::kASegs, kBSegs = C::kBSegs;
  constexpr bool kPair = kWhat == kFwd && kAct == SMOE_ACT_SWIGLU;
  constexpr bool kTurnA = kWhat == kWgrad, kTurnB = kWhat != kFwd;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[C::kLds];
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wid / C::kWN, wn = wid % C::kWN;

  // ---- this workgroup's tile --------------------------------------------
  // cols: columns of the output; kBNo: of them, this tile's
  const int cols = kWhat == kFwd ? (kPair ? a.N / 2 : a.N) : a.K;
  constexpr int kBNo = kPair ? kBN / 2 : kBN;
  const int NT = (cols + kBNo - 1) / kBNo;
  // Each XCD takes a contiguous share of the tiles, its workgroups in turn.  The
  // order is row tiles in groups of kGM by all column tiles, rows fastest
  // (kWgrad: expert by expert), so that an XCD's 32 compute units share 4 row
  // tiles and 8 column tiles at a time.
  constexpr int kGM = 4;
  const int xcd = blockIdx.x & 7, per = gridDim.x >> 3;
  int first, last;  // this XCD's tiles
  const RowTiles rt(kWhat == kWgrad ? nullptr : a.offsets, a.E, a.R, kBM);
  const int MT = kWhat == kWgrad ? (a.N + kBM - 1) / kBM : rt.total;
  if constexpr (kWhat == kWgrad) {
    share_work(a, MT * NT, xcd, &first, &last);
  } else {
    const int total = MT * NT, chunk = (total + 7) / 8;
    first = xcd * chunk;
    last = first + chunk < total ? first + chunk : total;
  }
  auto locate = [&](int tile, MmTile* t) {
    if (tile >= last) return false;
    t->e = kWhat == kWgrad ? tile / (MT * NT) : 0;
    t->lo = 0;
    const int r = tile - t->e * (MT * NT), grp = r / (kGM * NT), q = r - grp * (kGM * NT);
    const int gm = MT - grp * kGM < kGM ? MT - grp * kGM : kGM;
    const int mt = grp * kGM + q % gm;
    t->n0 = q / gm * kBNo;
    t->ncols = cols - t->n0 < kBNo ? cols - t->n0 : kBNo;
    if constexpr (kWhat == kWgrad) {
      t->m0 = mt * kBM;
      t->mrows = a.N - t->m0;
      int hi = a.R;
      if (a.offsets) {
        t->lo = clamp_row(a.offsets, t->e, a.R);
        hi = clamp_row(a.offsets, t->e + 1, a.R);
      }
      t->len = hi > t->lo ? hi - (int)t->lo : 0;
    } else {
      RowTile w;
      if (!rt.find(a.offsets, a.E, a.R, kBM, mt, &w)) return false;
      t->e = w.e;
      t->m0 = w.row0;
      t->mrows = w.rows;
      t->len = kWhat == kFwd ? a.K : a.N;
    }
    t->mrows = t->mrows < kBM ? t->mrows : kBM;
    return true;
  };

  // ---- loaders ------------------------------------------------------------
  // row pitches in bytes
  typedef typename std::conditional<kAny, size_t, uint32_t>::type pitch_t;
  const pitch_t pa = (pitch_t)a.lda * 2, pb = (pitch_t)a.ldb * 2;
  const size_t sa = kTurnA ? (size_t)kStep * pa : kStep * 2, sb = kTurnB ? (size_t)kStep * pb : kStep * 2;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr_t)smem;
  const uint32_t a_lds = __builtin_amdgcn_readfirstlane(lds0 + wid * kASegs * 1024);
  const uint32_t b_lds = __builtin_amdgcn_readfirstlane(lds0 + C::kB0 + wid * kBSegs * 1024);
  auto row_seg = [&](int seg, int* row, int* chunk) {
    *row = tile_row(seg * 8 + (lane >> 3));
    *chunk = (lane & 7) ^ (*row & 7);
  };
  auto turn_seg = [&](int seg, int width, int* k, int* slot) {
    const int p = seg * 64 + lane;
    *k = p / (width / 8);
    *slot = p % (width / 8);
  };
  // of the current tile: steps, whole steps, the operands' first bytes and, by
  // segment, the lane's byte offset from the step's base
  int steps, full, len;
  const uint8_t *a_base, *b_base;
  // (kAny: oa, ob are the piece's row, or the place of its columns among the
  // tile's, and la, lb how many of its columns exist)
  uint32_t oa[kASegs], ob[kBSegs];
  int la[kASegs], lb[kBSegs];
  auto setup = [&](const MmTile& t) {
    long long skip = 0;
    len = t.len;
    if (a.splits > 1) {  // this workgroup's share of the sum, in whole steps
      const long long all = (len + kStep - 1) / kStep;
      skip = all * blockIdx.y / a.splits;
      const int end = (int)(all * (blockIdx.y + 1) / a.splits) * kStep;
      len = (len < end ? len : end) - (int)skip * kStep;
    }
    steps = (len + kStep - 1) / kStep;
    full = len / kStep;
    const T* A = (const T*)a.a + (kTurnA ? t.lo * a.lda + t.m0 : (long long)t.m0 * a.lda);
    const T* B = (const T*)a.b;
    if constexpr (kWhat == kFwd) B += (size_t)t.e * a.N * a.K;
    else if constexpr (kWhat == kDgrad) B += (size_t)t.e * a.N * a.K + t.n0;
    else B += t.lo * a.ldb + t.n0;
    a_base = uniform_ptr((const uint8_t*)A + skip * sa);
    b_base = uniform_ptr((const uint8_t*)B + skip * sb);
    // opaque: the lane's share of the addresses is formed here, tile by tile,
    // instead of being held over the loop
    int ln = lane;
    asm volatile("" : "+v"(ln));
#pragma unroll
    for (int j = 0; j < kASegs; ++j) {
      const int seg = wid * kASegs + j;
      if constexpr (kTurnA) {
        const int p = seg * 64 + ln, k = p / (kBM / 8), c = (p % (kBM / 8) ^ swz_left(k)) * 8;
        if constexpr (kAny) oa[j] = c, la[j] = t.mrows - c;
        else oa[j] = k * pa + (uint32_t)(c < t.mrows - 8 ? c : t.mrows - 8) * 2;
      } else {
        const int r = tile_row(seg * 8 + (ln >> 3));
        if constexpr (kAny) oa[j] = r < t.mrows ? r : t.mrows - 1;
        else oa[j] = (uint32_t)(r < t.mrows ? r : t.mrows - 1) * pa + ((ln & 7) ^ (r & 7)) * 16;
      }
    }
#pragma unroll
    for (int j = 0; j < kBSegs; ++j) {
      const int seg = wid * kBSegs + j;
      if constexpr (kTurnB) {
        const int p = seg * 64 + ln, k = p / (kBN / 8), c = (p % (kBN / 8) ^ swz_right(k)) * 8;
        if constexpr (kAny) ob[j] = c, lb[j] = t.ncols - c;
        else ob[j] = k * pb + (uint32_t)(c < t.ncols - 8 ? c : t.ncols - 8) * 2;
      } else {
        const int row = tile_row(seg * 8 + (ln >> 3));
        const int w = row / (kCB * 16), b = row % (kCB * 16) / 16, r = row & 15;
        // SwiGLU: gate and up rows of the same 8 columns a quarter, in turn
        int c = kPair ? w * 32 + (r >> 2) * 8 + (b >> 1) * 4 + (r & 3) : w * 64 + col_of(b, r);
        c = t.n0 + (c < t.ncols ? c : t.ncols - 1) + (kPair && (b & 1) ? cols : 0);
        if constexpr (kAny) ob[j] = c;
        else ob[j] = (uint32_t)c * pb + ((ln & 7) ^ (row & 7)) * 16;
      }
    }
  };
  // this wave's pieces (1 KiB) of step s into the stages at sta and stb
  auto send = [&](int s, uint32_t sta, uint32_t stb) __attribute__((always_inline)) {
    const uint8_t *ga = a_base + s * sa, *gb = b_base + s * sb;
    if (s < full) {
#pragma unroll
      for (int j = 0; j < kBSegs; ++j) dma16(gb, ob[j], b_lds + stb + j * 1024);
#pragma unroll
      for (int j = 0; j < kASegs; ++j) dma16(ga, oa[j], a_lds + sta + j * 1024);
    } else {  // the last, partial step: terms past the end read as zeros
      const int left = len - s * kStep;
      int term, x;
#pragma unroll
      for (int j = 0; j < kBSegs; ++j) {
        if constexpr (kTurnB) turn_seg(wid * kBSegs + j, kBN, &term, &x);
        else row_seg(wid * kBSegs + j, &x, &term), term *= 8;
        dma16_at(term < left ? (const void*)(gb + ob[j]) : (const void*)g_zero16, b_lds + stb + j * 1024);
      }
#pragma unroll
      for (int j = 0; j < kASegs; ++j) {
        if constexpr (kTurnA) turn_seg(wid * kASegs + j, kBM, &term, &x);
        else row_seg(wid * kASegs + j, &x, &term), term *= 8;
        dma16_at(term < left ? (const void*)(ga + oa[j]) : (const void*)g_zero16, a_lds + sta + j * 1024);
      }
    }
  };

  // kAny: a step's pieces into registers, those past the operand's end as
  // zeros, and from there to the same places
  v4u_t ra_[kAny ? kASegs : 1], rb_[kAny ? kBSegs : 1];
  auto fetch = [&](int s) {
    const int left = len - s * kStep;
    int term, x;
#pragma unroll
    for (int j = 0; j < kASegs; ++j) {
      const uint8_t* base = a_base + s * sa;
      if constexpr (kTurnA) {
        turn_seg(wid * kASegs + j, kBM, &term, &x);
        ra_[j] = load_some<T>((const T*)(base + (size_t)term * pa) + oa[j], term < left ? la[j] : 0);
      } else {
        row_seg(wid * kASegs + j, &x, &term);
        ra_[j] = load_some<T>((const T*)(base + (size_t)oa[j] * pa) + term * 8, left - term * 8);
      }
    }
#pragma unroll
    for (int j = 0; j < kBSegs; ++j) {
      const uint8_t* base = b_base + s * sb;
      if constexpr (kTurnB) {
        turn_seg(wid * kBSegs + j, kBN, &term, &x);
        rb_[j] = load_some<T>((const T*)(base + (size_t)term * pb) + ob[j], term < left ? lb[j] : 0);
      } else {
        row_seg(wid * kBSegs + j, &x, &term);
        rb_[j] = load_some<T>((const T*)(base + (size_t)ob[j] * pb) + term * 8, left - term * 8);
      }
    }
  };
  auto put = [&](uint32_t sta, uint32_t stb) {
#pragma unroll
    for (int j = 0; j < kBSegs; ++j)
      *(v4u_t*)(smem + C::kB0 + stb + (wid * kBSegs + j) * 1024 + lane * 16) = rb_[j];
#pragma unroll
    for (int j = 0; j < kASegs; ++j) *(v4u_t*)(smem + sta + (wid * kASegs + j) * 1024 + lane * 16) = ra_[j];
  };

  // ---- fragments ----------------------------------------------------------
  // Lane l supplies row l % 16 of a block at the 8 terms 32 kk + 8 (l / 16) ..
  const int g = lane >> 4, jr = (lane & 15) >> 2, q4 = lane & 3;
  const uint32_t ra = swz(wr * kRB * 16 + (lane & 15), g), rb = swz(wn * kCB * 16 + (lane & 15), g);
  // turned: the lane's row of a read is 32 kk + 8 g + 4 h + jr, whose swizzle
  // does not depend on kk and h
  uint32_t ta[kTurnA ? kRB : 1], tb[kTurnB ? kCB / 2 : 1];
  if constexpr (kTurnA) {
#pragma unroll
    for (int i = 0; i < kRB; ++i) {
      const int chunk = (wr * kRB + i) * 2 + (q4 >> 1);
      ta[i] = (8 * g + jr) * (kBM * 2) + (chunk ^ swz_left(8 * g + jr)) * 16 + (q4 & 1) * 8;
    }
  }
  if constexpr (kTurnB) {
#pragma unroll
    for (int j = 0; j < kCB / 2; ++j) {
      const int chunk = wn * 8 + j * 4 + q4;
      tb[j] = (8 * g + jr) * (kBN * 2) + (chunk ^ swz_right(8 * g + jr)) * 16;
    }
  }
  auto tr = [&](uint32_t at) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(smem + at));
  };
  auto pair_of = [](v4s_t lo4, v4s_t hi4) {
    return __builtin_bit_cast(v4u_t, __builtin_shufflevector(lo4, hi4, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  auto frag_a = [&](uint32_t st, int kk, int i) -> v4u_t {
    if constexpr (kTurnA) {
      const uint32_t at = st + ta[i] + kk * 32 * (kBM * 2);
      return pair_of(tr(at), tr(at + 4 * (kBM * 2)));
    } else {
      return *(const v4u_t*)(smem + st + (ra ^ (kk * 64)) + i * 2048);
    }
  };
  auto frag_b = [&](uint32_t st, int kk, int j) -> v4u_t {
    if constexpr (kTurnB) {
      const uint32_t at = st + C::kB0 + tb[j >> 1] + (j & 1) * 8 + kk * 32 * (kBN * 2);
      return pair_of(tr(at), tr(at + 4 * (kBN * 2)));
    } else {
      return *(const v4u_t*)(smem + st + C::kB0 + (rb ^ (kk * 64)) + j * 2048);
    }
  };

  v4f_t acc[kRB][kCB];

  // Each step is two phases of 32 terms; in a phase a wave reads its fragments
  // and then runs its kRB x kCB MFMAs, with a barrier after either part.  Of
  // eight waves the second four are one barrier behind the first: each SIMD
  // has one wave of either half, and while one reads (and sends for the stages
  // two steps on) the other keeps the matrix unit busy.  In barrier
  // intervals, the first half reads phase p in 2p and computes it in 2p + 1,
  // the second half in 2p + 1 and 2p + 2.
  //
  // Step s (phases 2s, 2s + 1): both phases' right fragments are read with
  // the first phase's left ones, so the right stage is free from interval
  // 4s + 2, when the first half's second phase refills it for step s + 2.  The
  // left stages are three: that of step s + 2 was last read in interval 4s - 1.
  // Step s + 2 is first read in interval 4s + 8, so the first half waits for
  // its pieces before the barrier of 4s + 7, the end of a second phase's
  // MFMAs, and the second half before the same barrier, the end of a second
  // phase's reads.  A load has five to four intervals of 512 cycles to land.
  constexpr bool kHalves = C::kWaves == 8;
  const bool second = kHalves && wid >= 4;
  constexpr int kPieces = kASegs + kBSegs;
  v4u_t fb[2][kCB], fa[kRB];
  auto barrier = [] {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // every piece but the last step's has landed (all: that one too)
  auto landed = [&](bool all) {
    asm volatile("" ::: "memory");
    if (kAny) __builtin_amdgcn_s_waitcnt(15 | 3 << 14 | 7 << 4);  // by registers: LDS writes alone
    else if (all) wait_vm_lgkm0<0>();
    else wait_vm_lgkm0<kPieces>();
  };
  auto multiply = [&](int kk) {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int i = 0; i < kRB; ++i)
#pragma unroll
      for (int j = 0; j < kCB; ++j) acc[i][j] = mfma32<T>(fb[kk][j], fa[i], acc[i][j]);
    __builtin_amdgcn_s_setprio(0);
  };
  // the first two steps of a tile, sent while the tile before is stored
  auto start = [&] {
    if constexpr (kAny) {
      if (steps > 0) {
        fetch(0);
        put(0, 0);
      }
      if (steps > 1) {
        fetch(1);
        put(C::kABytes, C::kBBytes);
      }
      if (steps > 2) fetch(2);
    } else {
      if (steps > 0) send(0, 0, 0);
      if (steps > 1) send(1, C::kABytes, C::kBBytes);
    }
  };
  // The steps of a tile.  A wave whose rows all lie past the tile's end (an
  // expert's last tile) keeps sending and meeting the others, and reads and
  // multiplies nothing: 478 -> 462 us for 65536 rows over 128 experts, 2048 x 1536.
  auto run = [&](auto has_rows) __attribute__((always_inline)) {
    constexpr bool kRows = decltype(has_rows)::value;
    uint32_t sta = 0, far = 2 * C::kABytes;  // left stages of this step and of two steps on
    for (int s = 0; s < steps; ++s) {
      const uint32_t stb = (s & 1) * C::kBBytes;
      const bool refill = s + 2 < steps;
      if constexpr (kRows) {
#pragma unroll
        for (int j = 0; j < kCB; ++j) fb[0][j] = frag_b(stb, 0, j);
#pragma unroll
        for (int i = 0; i < kRB; ++i) fa[i] = frag_a(sta, 0, i);
#pragma unroll
        for (int j = 0; j < kCB; ++j) fb[1][j] = frag_b(stb, 1, j);
      }
      __builtin_amdgcn_s_waitcnt(15 | 3 << 14 | 7 << 4);  // lgkmcnt(0) alone
      barrier();
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (kRows) multiply(0);
      __builtin_amdgcn_sched_barrier(0);
      barrier();
      if constexpr (kRows) {
#pragma unroll
        for (int i = 0; i < kRB; ++i) fa[i] = frag_a(sta, 1, i);
      }
      if constexpr (kAny) {
        if (refill) put(far, stb);
        if (s + 3 < steps) fetch(s + 3);
      } else {
        if (refill) send(s + 2, far, stb);
      }
      if (second) landed(!refill);
      else __builtin_amdgcn_s_waitcnt(15 | 3 << 14 | 7 << 4);
      barrier();
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (kRows) multiply(1);
      __builtin_amdgcn_sched_barrier(0);
      if (!second) landed(!refill);
      barrier();
      far = sta;
      sta = sta == 2 * C::kABytes ? 0 : sta + C::kABytes;
    }
  };
  auto sum = [&](int rows) {
#pragma unroll
    for (int i = 0; i < kRB; ++i)
#pragma unroll
      for (int j = 0; j < kCB; ++j) acc[i][j] = v4f_t{0.0f, 0.0f, 0.0f, 0.0f};
    if (steps == 0) return;
    landed(steps == 1);
    barrier();
    if (second) barrier();
    if (wr * kRB * 16 < rows) run(std::true_type{});
    else run(std::false_type{});
    if (kHalves && !second) barrier();
  };

  // ---- epilogue -------------------------------------------------------------
  // A lane holds rows 16 i + lane % 16 of its wave's and kRuns runs of 8
  // columns, 32 columns apart: both runs of a row are stored one after the
  // other, a whole 128-byte line (runs in the outer loop, half lines a pass,
  // took 9 us longer a round of dW tiles' 128 KiB).
  constexpr int kRuns = kPair ? 1 : 2;
  // a cut sum's share as it is; mm_join_kernel does the rest
  auto store_share = [&](const MmTile& t) {
    const size_t width = kPair ? a.N : cols;
    float* part = a.part + (size_t)blockIdx.y * (kWhat == kWgrad ? a.N : a.R) * width;
#pragma unroll
    for (int i = 0; i < kRB; ++i) {
      const int m = wr * kRB * 16 + i * 16 + (lane & 15);
      if (m >= t.mrows) continue;
#pragma unroll
      for (int p = 0; p < kRuns; ++p) {
        const int n = t.n0 + wn * (kPair ? 32 : 64) + g * 8 + p * 32, np = t.n0 + t.ncols - n;
        float* d = part + (size_t)(t.m0 + m) * width + n;
#pragma unroll
        for (int j = 0; j < kCB / kRuns; ++j) {
          const int c = (kPair ? j >> 1 : j) * 4;
          if (c < np)
            store_f32<float>(d + c + (kPair && (j & 1) ? cols : 0), np - c, (const float*)&acc[i][p * 2 + j]);
        }
      }
    }
  };
  auto store_fwd = [&](const MmTile& t) {
    const int n0 = t.n0 + wn * (kPair ? 32 : 64) + g * 8;
    float b0[kRuns][8], b1[8];
#pragma unroll
    for (int p = 0; p < kRuns; ++p) {
      const int n = n0 + p * 32, np = t.n0 + t.ncols - n;
#pragma unroll
      for (int x = 0; x < 8; ++x) b0[p][x] = b1[x] = 0.0f;
      if (a.bias && np > 0) {
        load_param<T>(a.bias, a.bias_f32, (size_t)t.e * a.N + n, np, b0[p]);
        if constexpr (kPair) load_param<T>(a.bias, a.bias_f32, (size_t)t.e * a.N + cols + n, np, b1);
      }
    }
    constexpr int kAhead = 4;  // rows whose residuals are in flight together
    v4u_t res[kAhead][kRuns];
#pragma unroll
    for (int i = 0; i < kRB; ++i) {
      if (a.residual && i % kAhead == 0) {
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
          const int m = wr * kRB * 16 + (i + q) * 16 + (lane & 15);
          const T* r = (const T*)a.residual + (long long)(t.m0 + (m < t.mrows ? m : t.mrows - 1)) * a.ldr + n0;
#pragma unroll
          for (int p = 0; p < kRuns; ++p)
            if (n0 + p * 32 + 8 <= t.n0 + t.ncols) res[q][p] = load_piece<T>(r + p * 32);
        }
      }
      const int m = wr * kRB * 16 + i * 16 + (lane & 15);
      if (m >= t.mrows) continue;
      const size_t row = (size_t)t.m0 + m;
#pragma unroll
      for (int p = 0; p < kRuns; ++p) {
        const int n = n0 + p * 32, np = t.n0 + t.ncols - n;  // columns of the run that exist
        if (np <= 0) break;
        float v[8];
        if constexpr (kPair) {
          float u[8];
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            v[x] = acc[i][x / 4 * 2][x & 3] + b0[p][x];
            u[x] = acc[i][x / 4 * 2 + 1][x & 3] + b1[x];
          }
          if (a.z) {
            store_f32<T>((T*)a.z + row * a.N + n, np, v);
            store_f32<T>((T*)a.z + row * a.N + cols + n, np, u);
          }
#pragma unroll
          for (int x = 0; x < 8; ++x) v[x] = act_value<SMOE_ACT_SILU>(v[x]) * u[x];
        } else {
#pragma unroll
          for (int x = 0; x < 8; ++x) v[x] = acc[i][p * 2 + x / 4][x & 3] + b0[p][x];
          if (a.z) store_f32<T>((T*)a.z + row * a.N + n, np, v);
#pragma unroll
          for (int x = 0; x < 8; ++x) v[x] = act_value<kAct>(v[x]);
        }
        if (a.residual) {
          float r[8];
          if (np >= 8) Elt<T>::unpack(res[i % kAhead][p], r);
          else load_f32<T>((const T*)a.residual + (long long)row * a.ldr + n, np, r);
#pragma unroll
          for (int x = 0; x < 8; ++x) v[x] = v[x] + r[x];
        }
        store_f32<T>((T*)a.out + row * cols + n, np, v);
      }
    }
  };
  auto store_grad = [&](const MmTile& t) {
    if (kWhat == kWgrad && t.len == 0 && (a.mode & 1)) return;  // nothing to add
#pragma unroll
    for (int i = 0; i < kRB; ++i) {
      const int m = wr * kRB * 16 + i * 16 + (lane & 15);
      if (m >= t.mrows) continue;
      const size_t row = (size_t)t.m0 + m;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int n = t.n0 + wn * 64 + g * 8 + p * 32, np = t.n0 + t.ncols - n;
        if (np <= 0) break;
        float v[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) v[x] = acc[i][p * 2 + x / 4][x & 3];
        if constexpr (kWhat == kDgrad) {
          store_f32<T>((T*)a.out + row * cols + n, np, v);
        } else {
          const size_t at = ((size_t)t.e * a.N + row) * cols + n;
          if (a.mode < 2) {
            float* d = (float*)a.out + at;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (np <= 4 * h) break;
              float w[4];
              if (a.mode & 1) {
                load_f32<float>(d + 4 * h, np - 4 * h, w);
#pragma unroll
                for (int x = 0; x < 4; ++x) v[4 * h + x] = w[x] + v[4 * h + x];
              }
              store_f32<float>(d + 4 * h, np - 4 * h, v + 4 * h);
            }
          } else {
            T* d = (T*)a.out + at;
            if (a.mode & 1) {
              float w[8];
              load_f32<T>(d, np, w);
#pragma unroll
              for (int x = 0; x < 8; ++x) v[x] = w[x] + v[x];
            }
            store_f32<T>(d, np, v);
          }
        }
      }
    }
  };

  // A workgroup's tiles one after the other: the next one's first two steps are
  // loaded while this one's results are stored.
  int tile = first + (blockIdx.x >> 3);
  MmTile cur;
  bool have = locate(tile, &cur);
  if (have) {
    setup(cur);
    start();
  }
  while (have) {
    const MmTile done = cur;
    sum(__builtin_amdgcn_readfirstlane(done.mrows));
    tile += per;
    have = locate(tile, &cur);
    if (have) {
      setup(cur);
      start();
    }
    if (a.splits > 1) store_share(done);
    else if constexpr (kWhat == kFwd) store_fwd(done);
    else store_grad(done);
  }
}

// The shares of a cut sum added in order, and the product's epilogue.  Four
// columns a thread.
template <class T, int kWhat, int kAct>
__global__ __launch_bounds__(256) void mm_join_kernel(const LinArgs a) {
  constexpr bool kPair = kWhat == kFwd && kAct == SMOE_ACT_SWIGLU;
  const int rows = kWhat == kWgrad ? a.N : a.R;
  const int width = kWhat == kFwd ? a.N : a.K, cols = kPair ? a.N / 2 : width;
  const int c = (blockIdx.x * 256 + threadIdx.x) * 4, np = cols - c;
  const size_t row = blockIdx.y, size = (size_t)rows * width;
  if (np <= 0) return;
  const float* p = a.part + row * width + c;
  float v[4], u[4], t[4];
  load_f32<float>(p, np, v);
  if constexpr (kPair) load_f32<float>(p + cols, np, u);
  for (int s = 1; s < a.splits; ++s) {
    load_f32<float>(p + s * size, np, t);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = v[i] + t[i];
    if constexpr (kPair) {
      load_f32<float>(p + s * size + cols, np, t);
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = u[i] + t[i];
    }
  }
  auto put = [&](T* d, const float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < np) d[i] = Elt<T>::from_f32(f[i]);
  };
  if constexpr (kWhat == kFwd) {
    auto bias = [&](int n) { return a.bias_f32 ? ((const float*)a.bias)[n] : Elt<T>::to_f32(((const T*)a.bias)[n]); };
    if (a.bias) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i < np) {
          v[i] = v[i] + bias(c + i);
          if constexpr (kPair) u[i] = u[i] + bias(cols + c + i);
        }
      }
    }
    if (a.z) {
      put((T*)a.z + row * width + c, v);
      if constexpr (kPair) put((T*)a.z + row * width + cols + c, u);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kPair) v[i] = act_value<SMOE_ACT_SILU>(v[i]) * u[i];
      else v[i] = act_value<kAct>(v[i]);
      if (a.residual && i < np) v[i] = v[i] + Elt<T>::to_f32(((const T*)a.residual)[(long long)row * a.ldr + c + i]);
    }
    put((T*)a.out + row * cols + c, v);
  } else if constexpr (kWhat == kDgrad) {
    put((T*)a.out + row * width + c, v);
  } else {
    const size_t at = row * width + c;
    if (a.mode < 2) {
      float* d = (float*)a.out + at;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < np) d[i] = (a.mode & 1) ? d[i] + v[i] : v[i];
    } else {
      T* d = (T*)a.out + at;
      if (a.mode & 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < np) v[i] = Elt<T>::to_f32(d[i]) + v[i];
      }
      put(d, v);
    }
  }
}

// ------------------------------------------------------------- launching ---
typedef MmCfg<2, 4, 8, 4> MmBig;    // 256 x 256, 8 waves
typedef MmCfg<2, 2, 4, 4> MmSmall;  // 128 x 128, 4 waves

template <class T, class C, int kWhat, bool kAny>
static int mm_launch(const LinArgs& a, hipStream_t s) {
  const int cols = kWhat == kFwd ? (a.act == SMOE_ACT_SWIGLU ? a.N / 2 : a.N) : a.K;
  const int bn = kWhat == kFwd && a.act == SMOE_ACT_SWIGLU ? C::kBN / 2 : C::kBN;
  const long long nt = (cols + bn - 1) / bn;
  const long long mt = kWhat == kWgrad ? (long long)((a.N + C::kBM - 1) / C::kBM) * a.E
                                       : (a.R + C::kBM - 1) / C::kBM + a.E - 1;
  if (mt * nt > 0x7fffffffLL) return SMOE_EINVAL_DIM;
  // as many workgroups as run at once, each with its share of the tiles
  constexpr long long kRun = C::kLds > 80 * 1024 ? 256 : 512;
  const long long blocks = mt * nt < kRun ? (mt * nt + 7) / 8 * 8 : kRun;
  const dim3 grid((unsigned)blocks, a.splits > 1 ? a.splits : 1), block(C::kThreads);
  const dim3 jgrid((cols + 1023) / 1024, kWhat == kWgrad ? a.N : a.R);
#define SMOE_MM(A)                                                                     \
  do {                                                                                 \
    linear_mm_kernel<T, C, kWhat, A, kAny><<<grid, block, 0, s>>>(a);                        \
    if (a.splits > 1) mm_join_kernel<T, kWhat, A><<<jgrid, dim3(256), 0, s>>>(a);      \
  } while (0)
  if constexpr (kWhat == kFwd) {
    switch (a.act) {
      case SMOE_ACT_NONE: SMOE_MM(SMOE_ACT_NONE); break;
      case SMOE_ACT_RELU: SMOE_MM(SMOE_ACT_RELU); break;
      case SMOE_ACT_SILU: SMOE_MM(SMOE_ACT_SILU); break;
      case SMOE_ACT_GELU: SMOE_MM(SMOE_ACT_GELU); break;
      case SMOE_ACT_GELU_TANH: SMOE_MM(SMOE_ACT_GELU_TANH); break;
      default: SMOE_MM(SMOE_ACT_SWIGLU); break;
    }
  } else {
    SMOE_MM(SMOE_ACT_NONE);
  }
#undef SMOE_MM
  SMOE_RETURN_LAUNCH();
}

template <class T, class C, bool kAny>
static int linear_mm_c(const LinArgs& a, int what, hipStream_t s) {
  if (what == kFwd) return mm_launch<T, C, kFwd, kAny>(a, s);
  if (what == kDgrad) return mm_launch<T, C, kDgrad, kAny>(a, s);
  return mm_launch<T, C, kWgrad, kAny>(a, s);
}

}  // namespace smoe
