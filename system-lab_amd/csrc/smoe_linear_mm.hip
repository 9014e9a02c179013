// smoe_linear_mm.hip — the tiled kernels of linear_act for 16-byte aligned
// operands, and which tile, cut and way of loading a product takes.
#include "smoe_linear_mm.h"

namespace smoe {

// Rows of 16-byte pieces at 16-byte addresses, and 256 of them within the 32
// bits of a lane's offset.
static bool mm_rows_ok(const void* p, long long ld, int len) {
  return ((uintptr_t)p & 15u) == 0 && ld % 8 == 0 && len % 8 == 0 && ld <= (1 << 22);
}

static bool mm_aligned(const LinArgs& a, int what) {
  const int ra = what == kFwd ? a.K : a.N;  // the left operand's row length; the right one's is K
  return mm_rows_ok(a.a, a.lda, ra) && mm_rows_ok(a.b, a.ldb, a.K) &&
         // a weight's rows are addressed from its expert's first row
         (what != kFwd || (long long)a.N * a.K * 2 <= 0xffffffffLL);
}

// Big tiles need rows to fill them and as many tiles as compute units; small
// ones run two workgroups a unit.  us big / small, K 4096, N 4096, no experts:
// R 4096 121 / 154, R 3000 95 / 108, R 2048 83 / 64; K 2048, N 1536, 128 experts:
// R 65536 528 / 613, R 32768 310 / 338, R 16384 249 / 224; dx of the same 483 /
// 655, 296 / 363, 239 / 237.  dW's tiles do not depend on the rows: of 4096 x 4096
// 121 / 146 at R 4096, 59 / 78 at R 2048, of 2048 x 2048 (64 tiles) 175 / 99.
static bool mm_big(const LinArgs& a, int what) {
  const int cols = what == kFwd && a.act == SMOE_ACT_SWIGLU ? a.N / 2 : what == kFwd ? a.N : a.K;
  const int bn = what == kFwd && a.act == SMOE_ACT_SWIGLU ? 128 : 256;
  const long long nt = (cols + bn - 1) / bn;
  if (what == kWgrad) return nt * ((a.N + 255) / 256) * a.E >= 128;
  const int rows = a.R / a.E;  // an expert's mean
  return rows >= 192 && nt * ((rows + 255) / 256) * a.E >= 192;
}

// A dense product of few tiles cuts its sum into shares that fill the chip
// (with experts there are tiles enough, or too few rows to matter).  The model:
// a round of small tiles takes about 0.75 us a step with one workgroup a unit and
// 1.0 with two; the shares' fp32 sums are written and read at 4 TB/s and
// joined in a launch of their own (4 us).
int linear_mm_splits(int R, int N, int K, int act, int what) {
  const bool pair = what == kFwd && act == SMOE_ACT_SWIGLU;
  const long long rows = what == kWgrad ? N : R, width = what == kFwd ? N : K, len = what == kFwd ? K : what == kDgrad ? N : R;
  const int bn = pair ? 64 : 128;
  const long long cols = pair ? N / 2 : width, tiles = (rows + 127) / 128 * ((cols + bn - 1) / bn);
  const double steps = (double)((len + kStep - 1) / kStep);
  if (tiles >= 256 || rows > 65535) return 1;
  int best = 1;
  double least = steps * 0.75;
  for (int s = 2; s <= 16 && s * 4 <= steps; s *= 2) {
    const long long wgs = tiles * s;
    const double round = wgs <= 256 ? 0.75 : 1.0 * (double)((wgs + 511) / 512);
    const double t = round * steps / s + 4.0 + (double)s * rows * width * 8.0 / 4e6;
    if (t < least) {
      least = t;
      best = s;
    }
  }
  return best;
}

size_t linear_mm_part_bytes(int R, int N, int K, int act, int what) {
  const int s = linear_mm_splits(R, N, K, act, what);
  return s > 1 ? (size_t)s * (what == kWgrad ? N : R) * (what == kFwd ? N : K) * sizeof(float) : 0;
}

template <class T>
static int linear_mm_t(const LinArgs& a, int what, hipStream_t s) {
  if (a.splits == 1 && mm_big(a, what)) return linear_mm_c<T, MmBig, false>(a, what, s);
  return linear_mm_c<T, MmSmall, false>(a, what, s);
}

int linear_mm(LinArgs a, int what, int dtype, hipStream_t s) {
  a.splits = a.part && !a.offsets ? linear_mm_splits(a.R, a.N, a.K, a.act, what) : 1;
  if (!mm_aligned(a, what)) return linear_mm_any(a, what, dtype, s);
  return dtype == SMOE_BF16 ? linear_mm_t<bf16_t>(a, what, s) : linear_mm_t<f16_t>(a, what, s);
}

}  // namespace smoe
