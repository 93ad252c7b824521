// The gated half of a feed-forward block: y = act(x G^T + g) * (x U^T + u), both
// products, the activation and their product in one kernel.
//
// Products of float32 on the f16 matrix cores (Ootomo and Yokota, 2022): an operand is
// a pair h + l / 2048 of f16 values under a power of two of its own row (a pixel of x, an
// output channel of G or U), and h h + (h l + l h) / 2048 is taken.  A pair is within 2^-22 of
// its element as long as that is not below 2^-29 of its row's largest, and within 2^-50 of the
// largest below; what is left out, l l, is 2^-22 of the product at most.  Rows that hold a
// nonzero element below kUneven of their largest, infinities or NaN are not multiplied so, but in plain float32, on the
// float32 matrix cores, from x and the weights as they were given: such a row of x (the rows beside it keep their pairs,
// so that no row's bits hang on another's), and all of a panel of 32 output channels that holds such weights.
#include <algorithm>
#include <chrono>
#include <memory>
#include <mutex>
#include <new>

#include "activation.h"

namespace sy {

// Fragments: panels of 32 rows, in steps of 16 elements, hi then lo: a step's part is
// 64 16-byte units, unit 32 h + r the elements 8 h .. 8 h + 7 of row r.
constexpr int kStep = 128;  // units of a step

// Elements of a row below this share of its largest (as a power of two) make it uneven.
constexpr int kUneven = -31;
constexpr int kPlainRow = 1 << 16;  // set in a row's word, whose low bits are its power's exponent field

struct GatedPlan {
  int oc, ic, act;
  int panels, steps;      // of 32 output channels; of 16 input channels, even
  u32x4* w = nullptr;     // [panel][gate, up][step] fragments
  int* w_row = nullptr;   // [panel][gate, up][32] words
  int* w_plain = nullptr; // [panel]: uneven
  float* bias = nullptr;  // [gate, up][panels * 32]
  float* raw = nullptr;   // [gate, up][oc][ic] and 4 floats that quads may reach
};

struct GatedArgs {
  const float* x;
  float* y;
  long long ldx, ldy;
  int rows, ic, oc, act, panels, steps;
  const u32x4* w;
  const int *w_row, *w_plain;
  const float *bias, *raw;
  // x's fragments, by row_blocks of 32.
  const u32x4* xs;
  const int *x_row, *x_plain;
  int xpanels;
  int row_tiles, col_tiles;
};

// Exponent field of the power of two that takes a largest magnitude m into [2^14,
// 2^15); rows below 2^-113 keep the largest power there is.
__device__ __forceinline__ int gated_field(unsigned m) { return min(268 - (int)(m >> 23), 254); }

__device__ __forceinline__ unsigned magnitude(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }

// The part of a row that a thread holds: its largest magnitude, and its smallest but for zeros, less one.
struct Range {
  unsigned top = 0, low = ~0u;
  __device__ void look(float v) {
    const unsigned m = magnitude(v);
    top = max(top, m);
    low = min(low, m - 1);
  }
  // Whether the row, whose largest is `largest`, must be computed plainly for this part's sake.
  __device__ bool uneven(unsigned largest) const {
    const int e = (int)(largest >> 23);
    return e == 255 || low < (unsigned)max(max(e + kUneven, 0) << 23, 1) - 1;
  }
};

// Four elements of a row of `end` from `at`.  The memory takes quads at any multiple of four bytes; one that meets the
// row's end is read from within the row, and put right where it is used: a branch between loads would have
// every load waited for (1200 rows of 255 to 690 channels 12.9 us so, 12.5 without).
typedef f32x4 f32x4_any __attribute__((aligned(4)));
struct Quad {
  int from, shift, left;  // where it is read, how far that is ahead, elements that are there
  __device__ Quad(int at, int end) : from(max(min(at, end - 4), 0)), shift(at - from), left(end - at) {}
  // Of rows of fewer than four elements the quad is read whole, too.
  __device__ f32x4 load(const float* row) const { return *(const f32x4_any*)(row + from); }
  __device__ f32x4 mend(f32x4 t) const {
    if (shift & 1) t = f32x4{t[1], t[2], t[3], t[3]};
    if (shift & 2) t = f32x4{t[2], t[3], t[3], t[3]};
#pragma unroll
    for (int e = 0; e < 4; ++e) t[e] = e < left ? t[e] : 0.f;
    return t;
  }
};

// Largest value over aligned groups of 32 or 64 lanes, in each of them.
template <int LANES>
__device__ __forceinline__ unsigned lanes_max(unsigned m) {
  m = max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0xb1, 0xf, 0xf, true));   // lane ^ 1
  m = max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x4e, 0xf, 0xf, true));   // lane ^ 2
  m = max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x141, 0xf, 0xf, true));  // 7 - lane
  m = max(m, (unsigned)__builtin_amdgcn_mov_dpp((int)m, 0x140, 0xf, 0xf, true));  // 15 - lane
  const auto a = __builtin_amdgcn_permlane16_swap(m, m, false, false);
  m = max(a[0], a[1]);
  if (LANES == 64) {
    const auto b = __builtin_amdgcn_permlane32_swap(m, m, false, false);
    m = max(b[0], b[1]);
  }
  return m;
}

__device__ __forceinline__ void pair8(const f32x4 (&x)[2], float s, u32x4& h, u32x4& l) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = x[i >> 1][2 * i & 3], b = x[i >> 1][(2 * i & 3) + 1];
    const f16x2 hi = __builtin_convertvector((f32x2v{a * s, b * s}), f16x2);
    const f32x2v r = {__builtin_fmaf(a, s, -(float)hi[0]), __builtin_fmaf(b, s, -(float)hi[1])};
    h[i] = __builtin_bit_cast(unsigned, hi);
    l[i] = __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2v{r[0] * 2048.f, r[1] * 2048.f}), f16x2));
  }
}

// Unit of row r in a step of a panel in LDS: a wave that splits a row writes a quad of it to every half step, 512 bytes
// apart, and the rows change places there so that these go to all banks.
__device__ __forceinline__ int place(int step, int half, int r) { return half * 32 + (r ^ ((2 * step + half) & 31)); }

// A panel of 32 rows per workgroup, in lots of kLot elements: a wave takes every eighth row in
// whole lines, a lane four elements; the first kHeld lots stay in registers between the search for
// the rows' largest and the split.  Fragments leave through LDS, in whole lines too.  Rows past the last are
// zeros.  `more`: the panel's flag is that of an earlier call, too.  Memory bounds it: 16384 rows of 1024 elements 28 us,
// 4.8 TB/s.
constexpr int kLot = 256, kLotSteps = kLot / 16, kHeld = 4;
__global__ __launch_bounds__(512) void gated_split_kernel(const float* x, long long ldx, int rows, int ic, int steps,
                                                          u32x4* out, int* words, int* plain, int stride,
                                                          int offset, bool more) {
  __shared__ u32x4 lds[2][kLotSteps * kStep];
  __shared__ int any;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long long row0 = (long long)blockIdx.x * 32, panel = (long long)blockIdx.x * stride + offset;
  const int lots = (steps + kLotSteps - 1) / kLotSteps;
  if (threadIdx.x == 0) any = more ? plain[blockIdx.x] : 0;
  auto load = [&](int lot, f32x4(&v)[4]) __attribute__((always_inline)) {
    const Quad q(lot * kLot + 4 * lane, ic);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = q.load(x + min(row0 + wave + 8 * i, (long long)rows - 1) * ldx);
  };
  Range range[4];
  auto look = [&](int lot, f32x4(&v)[4]) __attribute__((always_inline)) {
    const Quad q(lot * kLot + 4 * lane, ic);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = q.mend(v[i]);
#pragma unroll
      for (int e = 0; e < 4; ++e) range[i].look(v[i][e]);
    }
  };
  f32x4 held[kHeld][4];
#pragma unroll
  for (int l = 0; l < kHeld; ++l)
    if (l < lots) load(l, held[l]);
#pragma unroll
  for (int l = 0; l < kHeld; ++l)
    if (l < lots) look(l, held[l]);
  for (int l = kHeld; l < lots; ++l) {
    f32x4 v[4];
    load(l, v);
    look(l, v);
  }
  __syncthreads();  // `any` stands
  float scale[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned t = lanes_max<64>(range[i].top);
    const bool here = row0 + wave + 8 * i < rows, bad = here && __any(range[i].uneven(t));
    const int field = gated_field(t);
    scale[i] = here ? exp_float(field) : 0.f;
    if (lane == 0) {
      words[panel * 32 + wave + 8 * i] = field | (bad ? kPlainRow : 0);
      if (bad) any = 1;
    }
  }
  u32x4* to = out + panel * steps * kStep;
  auto put = [&](int lot, const f32x4(&v)[4]) __attribute__((always_inline)) {
    u32x4* at_lds = lds[lot & 1];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u32x2 h, l;
      split4(v[i], scale[i], h, l);
      // Elements 4 lane .. + 3: step lane / 4, half (lane / 2) % 2, its first or second four.
      u32x2* at = (u32x2*)(at_lds + (lane >> 2) * kStep + place(lane >> 2, (lane >> 1) & 1, wave + 8 * i)) + (lane & 1);
      at[0] = h;
      at[128] = l;
    }
    __syncthreads();
    const int units = min(kLotSteps, steps - lot * kLotSteps) * kStep;
    for (int u = threadIdx.x; u < units; u += 512) {
      const int step = u / kStep, part = u & 64, half = (u >> 5) & 1;
      to[lot * kLotSteps * kStep + u] = at_lds[step * kStep + part + place(step, half, u & 31)];
    }
  };
#pragma unroll
  for (int l = 0; l < kHeld; ++l)
    if (l < lots) put(l, held[l]);
  for (int l = kHeld; l < lots; ++l) {
    const Quad q(l * kLot + 4 * lane, ic);
    f32x4 v[4];
    load(l, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = q.mend(v[i]);
    put(l, v);
  }
  __syncthreads();
  if (threadIdx.x == 0) plain[blockIdx.x] = any;
}

// Four weights of output channel `col` (gate or up) from input channel k: their own bits, not the pairs'.  Channels
// past the last are the last's.
__device__ __forceinline__ f32x4 gated_weights(const GatedArgs& a, int which, int col, int k) {
  const Quad q(k, a.ic);
  return q.mend(q.load(a.raw + ((long long)which * a.oc + min(col, a.oc - 1)) * a.ic));
}

// 32 x 32 gate and up sums of a wave in plain float32, over steps [k0, k1).  Rows of four elements and more; those past the
// last are the last's.
__device__ __forceinline__ void gated_plain(const GatedArgs& a, long long row0, int panel, int k0, int k1, int lane,
                                            f32x16 (&acc)[2]) {
  const int half = lane >> 5, r32 = lane & 31;
  const float* x = a.x + min(row0 + r32, (long long)a.rows - 1) * a.ldx;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[0][r] = acc[1][r] = 0.f;
  for (int k = 16 * k0; k < 16 * k1; k += 8) {
    const int c = k + 4 * half;
    const Quad q(c, a.ic);
    const f32x4 xv = q.mend(q.load(x));
    const f32x4 g = gated_weights(a, 0, 32 * panel + r32, c), u = gated_weights(a, 1, 32 * panel + r32, c);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      acc[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(xv[e], g[e], acc[0], 0, 0, 0);
      acc[1] = __builtin_amdgcn_mfma_f32_32x32x2f32(xv[e], u[e], acc[1], 0, 0, 0);
    }
  }
}

// A wave's 32 x 32 sums, gate and up, to the output: rows from row0, channel `col` of lane r32.  SOME: only
// the rows whose bit is set in `rows`.
template <bool SOME = false>
__device__ __forceinline__ void gated_out(const GatedArgs& a, int row0, int col, int half, float (&g)[16], float (&u)[16],
                                          unsigned rows = ~0u) {
  const float gb = a.bias[col], ub = a.bias[a.panels * 32 + col];
#pragma unroll
  for (int r = 0; r < 16; ++r) g[r] += gb;
  activate(a.act, g);
  if (col >= a.oc) return;
  float* y = a.y + (row0 + 4 * half) * a.ldy + col;
  if (!SOME && row0 + 32 <= a.rows) {
#pragma unroll
    for (int r = 0; r < 16; ++r) y[(8 * (r >> 2) + (r & 3)) * a.ldy] = g[r] * (u[r] + ub);
    return;
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int row = 8 * (r >> 2) + (r & 3);
    if (row0 + 4 * half + row < a.rows && (!SOME || (rows >> (row + 4 * half) & 1))) y[row * a.ldy] = g[r] * (u[r] + ub);
  }
}

// WM x WN waves, each two panels of rows by 32 output channels (gate and up): x and the weights
// arrive split, in the order of the matrix instruction's lanes.  x goes through LDS, two
// steps at a time, two stages in turn; the weights straight into registers, a stage ahead: with both in LDS
// its ports are busy as long as the matrix cores.  A step's fragments of x are read while the one before it
// is multiplied, over the barrier too: it stands before a stage's last products.  The matrix cores bound it: 16384 rows of
// 1024 to 2816 channels 519 us, 364 TFLOP/s (the cores busy 60 per cent of the time), and with the split
// 350 where the float32 matrix instructions could reach 150.
template <int WM, int WN>
__global__ __launch_bounds__(WM* WN * 64, 2) void gated_kernel(const GatedArgs a) {
  constexpr int TM = 2, NW = WM * WN, PA = TM * WM;
  constexpr int CHUNKS = 4 * PA, IT = CHUNKS / NW;  // of x, 1 KB each
  static_assert(CHUNKS % NW == 0, "whole chunks to a wave");
  __shared__ u32x4 frag[2][CHUNKS][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, r32 = lane & 31, wm = wave / WN, wn = wave % WN;
  // Each XCD takes a contiguous run of tiles, 8 row tiles by 4 column tiles at a time.
  const unsigned G = gridDim.x, L = blockIdx.x, xcd = L & 7, q8 = G >> 3, rem = G & 7;
  const unsigned P = xcd * q8 + (xcd < rem ? xcd : rem) + (L >> 3);
  const unsigned band = 8u * a.col_tiles, first = P / band * 8, high = min(8u, a.row_tiles - first);
  const int rt = first + P % band % high, ct = P % band / high;

  const u32x4* src[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int c = wave + i * NW;
    src[i] = a.xs + (long long)min(rt * PA + (c >> 2), a.xpanels - 1) * a.steps * kStep + (c & 3) * 64 + lane;
  }
  const u32x4* w = a.w + 2LL * min(ct * WN + wn, a.panels - 1) * a.steps * kStep + lane;
  const long long up = (long long)a.steps * kStep;
  f32x16 acc[TM][2], crs[TM][2];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = crs[i][j][r] = 0.f;
  u32x4 reg[IT];
  auto gload = [&](int s) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < IT; ++i) reg[i] = src[i][s * 2 * kStep];
  };
  auto put = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < IT; ++i) frag[buf][wave + i * NW][lane] = reg[i];
  };
  f16x8 av[2][TM][2], bv[2][2][2];
  auto wload = [&](int s, int k) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int p = 0; p < 2; ++p) bv[k][j][p] = __builtin_bit_cast(f16x8, w[j * up + (2 * s + k) * kStep + 64 * p]);
  };
  auto fetch = [&](int buf, int k) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int i = 0; i < TM; ++i)
        av[k][i][p] = __builtin_bit_cast(f16x8, frag[buf][(wm * TM + i) * 4 + 2 * k + p][lane]);
  };
  auto multiply = [&](int k) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        crs[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(av[k][i][1], bv[k][j][0], crs[i][j], 0, 0, 0);
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(av[k][i][0], bv[k][j][0], acc[i][j], 0, 0, 0);
      }
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        crs[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(av[k][i][0], bv[k][j][1], crs[i][j], 0, 0, 0);
  };
  const int stages = a.steps / 2;
  gload(0);
  wload(0, 0);
  wload(0, 1);
  put(0);
  gload(min(1, stages - 1));
  __syncthreads();
  fetch(0, 0);
  for (int s = 0; s < stages; ++s) {
    const int buf = s & 1, next = min(s + 1, stages - 1);
    fetch(buf, 1);
    __builtin_amdgcn_sched_barrier(0);
    multiply(0);
    wload(next, 0);
    put(buf ^ 1);  // the last stage's again, past the end
    gload(min(s + 2, stages - 1));
    __syncthreads();
    fetch(buf ^ 1, 0);
    __builtin_amdgcn_sched_barrier(0);
    multiply(1);
    wload(next, 1);
  }

  const int panel = ct * WN + wn, col = 32 * panel + r32;
  if (panel >= a.panels) return;
  const int gw = a.w_row[panel * 64 + r32] & 0xff, uw = a.w_row[panel * 64 + 32 + r32] & 0xff;
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int xp = (rt * WM + wm) * TM + i;
    if (xp >= a.xpanels) return;
    float g[16], u[16];
    const int* words = a.x_row + xp * 32 + 4 * half;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int f = words[8 * (r >> 2) + (r & 3)] & 0xff;
      g[r] = __builtin_ldexpf(__builtin_fmaf(crs[i][0][r], 1.f / 2048, acc[i][0][r]), 254 - f - gw);
      u[r] = __builtin_ldexpf(__builtin_fmaf(crs[i][1][r], 1.f / 2048, acc[i][1][r]), 254 - f - uw);
    }
    const int w_plain = a.w_plain[panel];
    if (a.x_plain[xp] | w_plain) {
      f32x16 t[2];
      gated_plain(a, (long long)xp * 32, panel, 0, a.steps, lane, t);
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (w_plain || (words[8 * (r >> 2) + (r & 3)] & kPlainRow)) {
          g[r] = t[0][r];
          u[r] = t[1][r];
        }
    }
    gated_out(a, xp * 32, col, half, g, u);
  }
}

// 16 x 16 gate and up sums of a wave in plain float32, over elements k0 .. k0 + 31 of the
// rows from row0 and the channels from col0, added to acc.
__device__ __forceinline__ void gated_plain16(const GatedArgs& a, int row0, int col0, int k0, int lane, f32x4 (&acc)[2]) {
  const int row = row0 + (lane & 15), col = col0 + (lane & 15);
  const float* x = a.x + (long long)min(row, a.rows - 1) * a.ldx;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int c = k0 + 16 * h + 4 * (lane >> 4);
    f32x4 xv;
#pragma unroll
    for (int e = 0; e < 4; ++e) xv[e] = row < a.rows && c + e < a.ic ? x[c + e] : 0.f;
    const f32x4 g = gated_weights(a, 0, col, c), u = gated_weights(a, 1, col, c);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      acc[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(xv[e], g[e], acc[0], 0, 0, 0);
      acc[1] = __builtin_amdgcn_mfma_f32_16x16x4f32(xv[e], u[e], acc[1], 0, 0, 0);
    }
  }
}

// Few rows: 16 of them by 16 output channels to a workgroup, the steps shared out over its eight
// waves, both operands straight from memory into the matrix instruction's registers, kAhead
// pairs of steps at once.  A wave splits x itself while the weights are on their way, under powers of the pairs of steps
// it has in hand, and brings each lot's sums to their true scale; a row that is uneven in a lot is
// plain in all of the wave's, by itself.
// The weights' bytes bound it: a row of 1024 to 2816 channels 6.1 us, 3.8 TB/s and half of it the launch, 32 rows
// 10.5.  TINY: rows of fewer than four elements, which are not read in quads, and plain always: pairs would save nothing.
constexpr int kFewWaves = 8, kAhead = 4;
template <bool TINY>
__global__ __launch_bounds__(kFewWaves * 64, 2) void gated_few_kernel(const GatedArgs a) {
  __shared__ float sums[kFewWaves][2][16][17];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, oct = lane >> 4;  // row or channel; elements 8 oct .. 8 oct + 7 of a pair of steps
  const int tile = blockIdx.x / (2 * a.panels), rest = blockIdx.x - tile * 2 * a.panels, row0 = 16 * tile;
  const int panel = rest >> 1, sub = (rest & 1) * 16, pairs = a.steps / 2;
  const int share = (pairs + kFewWaves - 1) / kFewWaves, p0 = min(wave * share, pairs), p1 = min(p0 + share, pairs);
  // A fragment's unit: step oct / 2, half oct % 2, channel sub + r16.
  const u32x4* w = a.w + (long long)2 * panel * a.steps * kStep + (oct >> 1) * kStep + (oct & 1) * 32 + sub + r16;
  const long long up = (long long)a.steps * kStep;
  const float* xr = a.x + (long long)min(row0 + r16, a.rows - 1) * a.ldx;
  const int w_plain = a.w_plain[panel];
  const int wf[2] = {a.w_row[panel * 64 + sub + r16] & 0xff, a.w_row[panel * 64 + 32 + sub + r16] & 0xff};
  f32x4 total[2] = {};
  unsigned long long odd = 0;  // the lanes that met what makes their row plain
  for (int p = TINY ? p1 : p0; p < p1; p += kAhead) {
    f16x8 wv[kAhead][2][2];
    f32x4 xv[kAhead][2];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) xv[u][h] = Quad(min(p + u, pairs) * 32 + 8 * oct + 4 * h, a.ic).load(xr);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const long long at = (long long)min(p + u, pairs - 1) * 2 * kStep;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int s = 0; s < 2; ++s) wv[u][j][s] = __builtin_bit_cast(f16x8, w[j * up + at + 64 * s]);
    }
    if (p + kAhead > p1 || 32 * (p + kAhead) > a.ic) {  // the row's end, or the wave's
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          xv[u][h] = Quad(p + u < p1 ? (p + u) * 32 + 8 * oct + 4 * h : a.ic, a.ic).mend(xv[u][h]);
    }
    Range range;
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) range.look(xv[u][h][e]);
    unsigned top = range.top;
#pragma unroll
    for (int off = 16; off < 64; off <<= 1) top = max(top, (unsigned)__shfl_xor((int)top, off));
    odd |= __ballot(range.uneven(top));
    const int field = gated_field(top);
    const float scale = exp_float(field);
    f32x4 acc[2] = {}, crs[2] = {};
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      u32x4 h, l;
      pair8(xv[u], scale, h, l);
      const f16x8 xh = __builtin_bit_cast(f16x8, h), xl = __builtin_bit_cast(f16x8, l);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        crs[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xl, wv[u][j][0], crs[j], 0, 0, 0);
        acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xh, wv[u][j][0], acc[j], 0, 0, 0);
        crs[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xh, wv[u][j][1], crs[j], 0, 0, 0);
      }
    }
    // Lane r's field is that of row r; the lane's sums are rows 4 oct .. 4 oct + 3 of channel r16.
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int f = __shfl(field, 4 * oct + r);
#pragma unroll
      for (int j = 0; j < 2; ++j)
        total[j][r] += __builtin_ldexpf(__builtin_fmaf(crs[j][r], 1.f / 2048, acc[j][r]), 254 - f - wf[j]);
    }
  }
  if (TINY || w_plain != 0 || odd != 0) {
    f32x4 plain[2] = {};
    for (int p = p0; p < p1; ++p) gated_plain16(a, row0, 32 * panel + sub, 32 * p, lane, plain);
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (TINY || w_plain != 0 || (odd >> (4 * oct + r) & 0x0001000100010001ull) != 0) {  // by any of the lanes that hold the row
        total[0][r] = plain[0][r];
        total[1][r] = plain[1][r];
      }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) sums[wave][j][4 * oct + r][r16] = total[j][r];
  __syncthreads();
  const int row = threadIdx.x >> 4, col = 32 * panel + sub + r16;
  if (row >= 16 || row0 + row >= a.rows) return;
  float g = 0.f, u = 0.f;
#pragma unroll
  for (int x = 0; x < kFewWaves; ++x) {
    g += sums[x][0][row][r16];
    u += sums[x][1][row][r16];
  }
  if (col >= a.oc) return;
  float v[1] = {g + a.bias[col]};
  activate(a.act, v);
  a.y[(row0 + row) * a.ldy + col] = v[0] * (u + a.bias[a.panels * 32 + col]);
}

// A middling number of tiles: a panel of rows by PAN panels of output channels to a workgroup, each
// panel's steps shared out over 8 / PAN waves.  x goes through LDS in lots of kLot elements, two
// in turn, loaded row by row in whole lines and split by the workgroup itself (a kernel of its own would
// cost more than the products); weights come straight from memory.  Latency bounds it, and the split's vector
// work: 256 rows of 1024 to 688 channels 17.9 us, 40 TFLOP/s, 1200 of 600 to 690 22.6, 88.
template <int PAN>
__global__ __launch_bounds__(512, 2) void gated_mid_kernel(const GatedArgs a) {
  constexpr int KW = 8 / PAN, SH = kLotSteps / KW;  // waves of a panel, their steps of a lot
  constexpr int LOT = kLotSteps * kStep;
  __shared__ u32x4 lds[2][LOT];
  __shared__ float sums[8][2][32][33];
  __shared__ int fields[32];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, r32 = lane & 31, part = wave % KW;
  const int cols = (a.panels + PAN - 1) / PAN, tile = blockIdx.x / cols, first = (blockIdx.x - tile * cols) * PAN;
  const int panel = min(first + wave / KW, a.panels - 1), row0 = tile * 32;
  const u32x4* w = a.w + (long long)2 * panel * a.steps * kStep + lane;
  const long long up = (long long)a.steps * kStep;
  // A wave takes every eighth row, a lane four elements of it.
  auto load = [&](int k0, f32x4(&v)[4]) __attribute__((always_inline)) {
    const Quad q(16 * k0 + 4 * lane, a.ic);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = q.load(a.x + (long long)min(row0 + wave + 8 * i, a.rows - 1) * a.ldx);
  };
  auto mend = [&](int k0, f32x4(&v)[4]) __attribute__((always_inline)) {
    const Quad q(16 * k0 + 4 * lane, a.ic);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = q.mend(v[i]);
  };
  // Weights of steps k and on, four at a time.
  f16x8 wv[4][2][2];
  auto load_w = [&](int k) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int s = 0; s < 2; ++s)
          wv[u][j][s] = __builtin_bit_cast(f16x8, w[j * up + (long long)min(k + u, a.steps - 1) * kStep + 64 * s]);
  };
  // The rows' powers: the first lot stays in registers, the others come four at a time.
  Range range[4];
  auto look = [&](const f32x4(&t)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) range[i].look(t[i][e]);
  };
  f32x4 v[4];
  load(0, v);
  load_w(part * SH);
  for (int k0 = kLotSteps; k0 < a.steps; k0 += 4 * kLotSteps) {
    f32x4 t[4][4];
    auto at = [&](int l) { return min(k0 + l * kLotSteps, (a.steps - 1) / kLotSteps * kLotSteps); };
#pragma unroll
    for (int l = 0; l < 4; ++l) load(at(l), t[l]);
#pragma unroll
    for (int l = 0; l < 4; ++l) {
      mend(at(l), t[l]);
      look(t[l]);
    }
  }
  mend(0, v);
  look(v);
  float scale[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned t = lanes_max<64>(range[i].top);
    const int field = gated_field(t), bad = __any(range[i].uneven(t)) ? kPlainRow : 0;
    scale[i] = exp_float(field);
    if (lane == 0) fields[wave + 8 * i] = field | bad;
  }
  auto put = [&](u32x4* to) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u32x2 h, l;
      split4(v[i], scale[i], h, l);
      // Elements 4 lane .. + 3: step lane / 4, half (lane / 2) % 2, its first or second four.
      u32x2* at = (u32x2*)(to + (lane >> 2) * kStep + place(lane >> 2, (lane >> 1) & 1, wave + 8 * i)) + (lane & 1);
      at[0] = h;
      at[128] = l;
    }
  };
  put(lds[0]);
  f32x16 acc[2], crs[2];
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[j][r] = crs[j][r] = 0.f;
  __syncthreads();
  int now = 0;
  for (int k0 = 0; k0 < a.steps; k0 += kLotSteps, now ^= 1) {
    const bool more = k0 + kLotSteps < a.steps;
    if (more) load(k0 + kLotSteps, v);
#pragma unroll
    for (int u = 0; u < SH; ++u) {
      const int k = part * SH + u;
      if (k0 + k < a.steps) {
        const u32x4* f = lds[now] + k * kStep + place(k, half, r32);
        const f16x8 xh = __builtin_bit_cast(f16x8, f[0]), xl = __builtin_bit_cast(f16x8, f[64]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          crs[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xl, wv[u & 3][j][0], crs[j], 0, 0, 0);
          acc[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xh, wv[u & 3][j][0], acc[j], 0, 0, 0);
          crs[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xh, wv[u & 3][j][1], crs[j], 0, 0, 0);
        }
      }
      if ((u & 3) == 3) load_w(u + 1 < SH ? k0 + k + 1 : k0 + kLotSteps + part * SH);
    }
    if (more) {
      mend(k0 + kLotSteps, v);
      put(lds[now ^ 1]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int row = 8 * (r >> 2) + 4 * half + (r & 3), f = fields[row] & 0xff;
#pragma unroll
    for (int j = 0; j < 2; ++j)
      sums[wave][j][row][r32] = __builtin_ldexpf(__builtin_fmaf(crs[j][r], 1.f / 2048, acc[j][r]),
                                                 254 - f - (a.w_row[panel * 64 + 32 * j + r32] & 0xff));
  }
  // Plain rows' sums take the place of theirs.
  const int w_plain = a.w_plain[panel];
  if (__any(fields[r32] & kPlainRow) || w_plain) {
    const int share = (a.steps + KW - 1) / KW;
    gated_plain(a, row0, panel, min(part * share, a.steps), min((part + 1) * share, a.steps), lane, acc);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = 8 * (r >> 2) + 4 * half + (r & 3);
      if (w_plain || (fields[row] & kPlainRow)) {
        sums[wave][0][row][r32] = acc[0][r];
        sums[wave][1][row][r32] = acc[1][r];
      }
    }
  }
  __syncthreads();
  if (first + wave / KW >= a.panels) return;
  const int col = 32 * panel + r32;
  if (col >= a.oc) return;
  const float gb = a.bias[col], ub = a.bias[a.panels * 32 + col];
  float g[16 / KW], u[16 / KW];
#pragma unroll
  for (int i = 0; i < 16 / KW; ++i) {
    const int row = 2 * (KW * i + part) + half;
    g[i] = gb;
    u[i] = ub;
#pragma unroll
    for (int x = 0; x < KW; ++x) {
      g[i] += sums[wave - part + x][0][row][r32];
      u[i] += sums[wave - part + x][1][row][r32];
    }
  }
  activate(a.act, g);
#pragma unroll
  for (int i = 0; i < 16 / KW; ++i) {
    const int row = row0 + 2 * (KW * i + part) + half;
    if (row < a.rows) a.y[row * a.ldy + col] = g[i] * u[i];
  }
}

// Short rows (up to 256 Q elements, and 128 with LANES 32) and many: 32 PX rows by panels of output channels, one to a wave, to a
// workgroup.  It loads its rows at once, in whole lines, splits them into LDS, where they stay, and
// goes through a column of tiles (every col_tiles-th) with the weights straight from memory and no
// further barrier.  LANES lanes hold a row, Q quads each.  The split's and the outputs' vector work bounds it, and the
// launch: 1200 rows of 255 to 690 channels 10.4 us, 82 TFLOP/s, 60000 of 256 to 384 104 us, 226.
template <int PX, int LANES, int Q>
__global__ __launch_bounds__(256, 2) void gated_short_kernel(const GatedArgs a) {
  constexpr int SIDE = 64 / LANES, LOADS = 8 * PX / SIDE;  // rows side by side in a wave's load; loads of a wave
  extern __shared__ u32x4 xs[];                            // [PX][steps] fragments
  __shared__ __align__(16) int words[32 * PX];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, r32 = lane & 31, l = lane % LANES, side = lane / LANES;
  const int tile = blockIdx.x / a.col_tiles, first = blockIdx.x - tile * a.col_tiles, row0 = tile * 32 * PX;
  const long long up = (long long)a.steps * kStep;
  constexpr int AHEAD = PX == 1 ? 4 : 2;  // steps of weights under way
  f16x8 wv[AHEAD][2][2];
  auto load_w = [&](int panel, int k, int u) __attribute__((always_inline)) {
    const u32x4* w = a.w + (long long)2 * panel * a.steps * kStep + lane + min(k, a.steps - 1) * kStep;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int s = 0; s < 2; ++s) wv[u][j][s] = __builtin_bit_cast(f16x8, w[j * up + 64 * s]);
  };
  {
    const int mine = wave * 8 * PX + side;  // the first of a lane's rows
    f32x4 v[LOADS][Q];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const float* x = a.x + (unsigned long long)(unsigned)min(row0 + mine + i * SIDE, a.rows - 1) * (unsigned)a.ldx;
#pragma unroll
      for (int j = 0; j < Q; ++j) v[i][j] = Quad(4 * (l + LANES * j), a.ic).load(x);
    }
    const int panel = min(first * 4 + wave, a.panels - 1);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) load_w(panel, u, u);
    unsigned top[LOADS], low[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      Range range;
#pragma unroll
      for (int j = 0; j < Q; ++j) {
        v[i][j] = Quad(4 * (l + LANES * j), a.ic).mend(v[i][j]);
#pragma unroll
        for (int e = 0; e < 4; ++e) range.look(v[i][j][e]);
      }
      low[i] = range.low;
      top[i] = lanes_max<LANES>(range.top);
    }
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      Range range;
      range.low = low[i];
      const unsigned long long bad = __ballot(range.uneven(top[i])) >> (side * LANES & 63);
      low[i] = (LANES == 64 ? bad : (unsigned)bad) != 0 ? kPlainRow : 0;
    }
    if (l == 0)
#pragma unroll
      for (int i = 0; i < LOADS; ++i) words[mine + i * SIDE] = gated_field(top[i]) | low[i];
#pragma unroll
    for (int j = 0; j < Q; ++j) {
      const int step = (l + LANES * j) >> 2;
      if (step < a.steps)
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
          const int r = mine + i * SIDE;
          u32x2 h, lo;
          split4(v[i][j], exp_float(gated_field(top[i])), h, lo);
          u32x2* at = (u32x2*)(xs + ((r >> 5) * a.steps + step) * kStep + place(step, (l >> 1) & 1, r & 31)) + (l & 1);
          at[0] = h;
          at[128] = lo;
        }
    }
  }
  __syncthreads();
  bool plain[PX], again = false;
#pragma unroll
  for (int i = 0; i < PX; ++i) plain[i] = __any(words[32 * i + r32] & kPlainRow);
  for (int ct = first; 4 * ct < a.panels; ct += a.col_tiles) {
    const int panel = min(4 * ct + wave, a.panels - 1), next = min(4 * (ct + a.col_tiles) + wave, a.panels - 1);
    f32x16 acc[PX][2], crs[PX][2];
#pragma unroll
    for (int i = 0; i < PX; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = crs[i][j][r] = 0.f;
    for (int k0 = 0; k0 < a.steps; k0 += AHEAD)
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const int k = k0 + u;
        if (k < a.steps) {
          f16x8 av[PX][2];
#pragma unroll
          for (int i = 0; i < PX; ++i)
#pragma unroll
            for (int p = 0; p < 2; ++p)
              av[i][p] = __builtin_bit_cast(f16x8, xs[(i * a.steps + k) * kStep + 64 * p + place(k, half, r32)]);
#pragma unroll
          for (int i = 0; i < PX; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              crs[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(av[i][1], wv[u][j][0], crs[i][j], 0, 0, 0);
              acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(av[i][0], wv[u][j][0], acc[i][j], 0, 0, 0);
            }
#pragma unroll
          for (int i = 0; i < PX; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
              crs[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(av[i][0], wv[u][j][1], crs[i][j], 0, 0, 0);
        }
        load_w(panel, k + AHEAD, u);
      }
    if (4 * ct + wave >= a.panels) break;
    const int col = 32 * panel + r32;
    const int gw = a.w_row[panel * 64 + r32] & 0xff, uw = a.w_row[panel * 64 + 32 + r32] & 0xff;
    const bool w_plain = a.w_plain[panel];
#pragma unroll
    for (int i = 0; i < PX; ++i) {
      float g[16], u[16];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int4 f = *(const int4*)&words[32 * i + 8 * q + 4 * half];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * q + e, to = 254 - ((&f.x)[e] & 0xff);
          g[r] = __builtin_ldexpf(__builtin_fmaf(crs[i][0][r], 1.f / 2048, acc[i][0][r]), to - gw);
          u[r] = __builtin_ldexpf(__builtin_fmaf(crs[i][1][r], 1.f / 2048, acc[i][1][r]), to - uw);
        }
      }
      if (i == PX - 1)
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) load_w(next, u, u);
      again |= plain[i] || w_plain;
      if (w_plain) continue;
      gated_out(a, row0 + 32 * i, col, half, g, u);
    }
  }
  if (!again) return;
  // Panels that were left out and plain rows, whose outputs were not theirs yet, in plain float32 (inside the loop
  // above they would cost it its registers).  A lane writes what it wrote there.
  for (int ct = first; 4 * ct + wave < a.panels; ct += a.col_tiles) {
    const int panel = 4 * ct + wave, col = 32 * panel + r32;
    const bool w_plain = a.w_plain[panel];
#pragma unroll 1
    for (int i = 0; i < PX; ++i) {
      // (Bits of lanes past 32 repeat the others'.)
      const unsigned rows = w_plain ? ~0u : (unsigned)__ballot(words[32 * i + r32] & kPlainRow);
      if (rows == 0) continue;
      f32x16 t[2];
      gated_plain(a, row0 + 32 * i, panel, 0, a.steps, lane, t);
      float g[16], u[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        g[r] = t[0][r];
        u[r] = t[1][r];
      }
      gated_out<true>(a, row0 + 32 * i, col, half, g, u, rows);
    }
  }
}

static int gated_pack(sy_ctx* ctx, const float* gate, const float* up, const float* gate_bias, const float* up_bias,
                      GatedPlan* p) {
  const size_t values = (size_t)p->oc * p->ic, cols = (size_t)p->panels * 32;
  std::vector<float> bias;
  try {
    bias.assign(2 * cols, 0.f);
  } catch (const std::bad_alloc&) {
    SY_CHECK(false, SY_ENOMEM, "no memory for a gated layer's biases");
  }
  if (gate_bias) std::copy(gate_bias, gate_bias + p->oc, bias.begin());
  if (up_bias) std::copy(up_bias, up_bias + p->oc, bias.begin() + cols);
  SY_HIP(hipMalloc((void**)&p->w, cols * 2 * p->steps * 16 * 4));
  SY_HIP(hipMalloc((void**)&p->w_row, cols * 2 * sizeof(int)));
  SY_HIP(hipMalloc((void**)&p->w_plain, p->panels * sizeof(int)));
  SY_HIP(hipMalloc((void**)&p->bias, 2 * cols * sizeof(float)));
  SY_HIP(hipMalloc((void**)&p->raw, (2 * values + 4) * sizeof(float)));  // rows are read by quads
  SY_TRY(sy_memcpy(ctx, p->raw, gate, values * sizeof(float), 0));
  SY_TRY(sy_memcpy(ctx, p->raw + values, up, values * sizeof(float), 0));
  SY_TRY(sy_memcpy(ctx, p->bias, bias.data(), 2 * cols * sizeof(float), 0));
  for (int m = 0; m < 2; ++m)
    hipLaunchKernelGGL(gated_split_kernel, dim3(p->panels), dim3(512), 0, ctx->stream, p->raw + m * values,
                       (long long)p->ic, p->oc, p->ic, p->steps, p->w, p->w_row, p->w_plain, 2, m, m == 1);
  return check_launch("gated_split");
}

int op_gated_create(sy_ctx* ctx, const float* gate, const float* up, const float* gate_bias, const float* up_bias,
                    int oc, int ic, int act, uint64_t* gated) {
  SY_CHECK(gate && up && gated, SY_EINVAL, "null argument");
  SY_CHECK(oc > 0 && ic > 0, SY_EINVAL, "gated projections of %d to %d channels", ic, oc);
  SY_CHECK(act >= SY_ACT_NONE && act <= SY_ACT_SIGMOID, SY_EINVAL, "unknown activation %d", act);
  SY_CHECK((long long)oc * ic < (1LL << 31) && oc < (1 << 24) && ic < (1 << 24), SY_EUNSUPPORTED,
           "gated projections of %d to %d channels", ic, oc);
  SY_CHECK(ctx, SY_EINVAL, "null context");
  SY_CHECK(!ctx->capturing, SY_ESTATE, "weight upload during graph capture");
  // Allocations would end another context's capture.
  std::unique_lock<std::shared_timed_mutex> lock(capture_lock(), std::defer_lock);
  SY_CHECK(lock.try_lock_for(std::chrono::seconds(60)), SY_ESTATE,
           "weight upload waited 60 s for graph captures on other contexts to end");
  std::unique_ptr<GatedPlan> p(new (std::nothrow) GatedPlan);
  SY_CHECK(p, SY_ENOMEM, "no memory for a gated layer");
  p->oc = oc;
  p->ic = ic;
  p->act = act;
  p->panels = (oc + 31) / 32;
  p->steps = (ic + 31) / 32 * 2;
  DeviceScope device(ctx);
  int rc = gated_pack(ctx, gate, up, gate_bias, up_bias, p.get());
  void* held[] = {p->w, p->w_row, p->w_plain, p->bias, p->raw};
  if (rc == SY_OK) {
    try {
      ctx->owned.reserve(ctx->owned.size() + 5);
      ctx->gateds.push_back(std::move(p));
    } catch (const std::bad_alloc&) {
      set_error("no memory for a gated layer");
      rc = SY_ENOMEM;
    }
  }
  if (rc != SY_OK) {
    (void)hipStreamSynchronize(ctx->stream);
    for (void* h : held)
      if (h) (void)hipFree(h);
    return rc;
  }
  for (void* h : held)
    if (h) ctx->owned.push_back(h);
  *gated = ctx->gateds.size();
  return SY_OK;
}

int op_gated_run(sy_ctx* ctx, uint64_t gated, const sy_tensor* x, const sy_tensor* y) {
  SY_CHECK(gated > 0 && gated <= ctx->gateds.size(), SY_EINVAL, "unknown gated handle %llu", (unsigned long long)gated);
  const GatedPlan& p = *ctx->gateds[gated - 1];
  SY_TRY(check_view(x, "gated input"));
  SY_TRY(check_view(y, "gated output"));
  SY_CHECK(x->c == p.ic && y->c == p.oc, SY_EINVAL, "gated projections of %d to %d channels: views have %d and %d", p.ic,
           p.oc, x->c, y->c);
  SY_CHECK(y->n == x->n && y->h == x->h && y->w == x->w, SY_EINVAL, "gated output shape mismatch");
  SY_CHECK((((uintptr_t)x->data | (uintptr_t)y->data) & 3) == 0, SY_EINVAL, "gated views must be 4-byte aligned");
  SY_CHECK(!views_overlap(x, y), SY_EINVAL, "gated output overlaps its input");
  const long long rows = pixels(*x);
  SY_CHECK((long long)x->n * x->h < (1LL << 30) && rows < (1LL << 30), SY_EUNSUPPORTED, "gated projections of 2^30 pixels and more");
  GatedArgs a{};
  a.x = x->data;
  a.y = y->data;
  a.ldx = x->ldc;
  a.ldy = y->ldc;
  a.rows = (int)rows;
  a.ic = p.ic;
  a.oc = p.oc;
  a.act = p.act;
  a.panels = p.panels;
  a.steps = p.steps;
  a.w = p.w;
  a.w_row = p.w_row;
  a.w_plain = p.w_plain;
  a.bias = p.bias;
  a.raw = p.raw;
  a.xpanels = (a.rows + 31) / 32;
  DeviceScope device(ctx);
  const double flops = 4.0 * rows * p.ic * p.oc, bytes = 4.0 * ((double)rows * (p.ic + p.oc) + 2.0 * p.ic * p.oc);
  // 32 rows of 1024 to 2816 channels 10.5 us here, 17.6 as a middling number of tiles; 64 of 256 to 688 (176 workgroups)
  // 6.4, 7.5 as short rows; 256 of 128 to 256 (256) 5.1 and 5.7, 400 of 128 to 256 (400) 6.3 and 6.2, 33 of 2048 to 4096 (768) 40
  // and 33 as a middling number.
  if (a.rows <= 32 || a.ic < 4 || 2LL * p.panels * ((a.rows + 15) / 16) <= 256) {
    ProfScope prof(ctx, "gated_few", flops, bytes);
    const long long grid = 2LL * p.panels * ((a.rows + 15) / 16);
    SY_CHECK(grid * kFewWaves * 64 < (1LL << 32), SY_EUNSUPPORTED, "gated grid too large");
    hipLaunchKernelGGL(a.ic < 4 ? gated_few_kernel<true> : gated_few_kernel<false>, dim3((unsigned)grid), dim3(kFewWaves * 64), 0, ctx->stream, a);
    return check_launch("gated_few");
  }
  if (a.ic <= 512) {
    // Short rows: three column tiles (of 128 channels) or four at most, or 900 tiles; else the products are so
    // many that splitting x beforehand pays (20000 rows of 256 to 512 channels 58 us here, 53 so, to 256 33.7 and 38; 4000
    // of 512 to 512 (500 tiles) 24.3 and 26.9, 2048 to 2048 (1024) 41.8 and 37.3).  Longer rows than 512: 64 KB and more of
    // LDS, where fewer waves would hide less.
    // Where 64 rows to a workgroup make 512 of them, that, and every column tile in turn: 60000 rows of 256 to 384 channels
    // 104 us, 122 with 32 rows, 123 split beforehand; 9471 of 90 to 360 15.5 to 24, 17.9, 19.7.  With 32 rows, every
    // column tile in turn where there are 400 workgroups: 14161 of 137 to 377 26.4 us, a tile to each 30.4; 9471 of 90 to
    // 360 21.6 and 17.9.
    const int cols = (a.panels + 3) / 4, wide = (a.rows + 63) / 64;
    auto go = [&](auto kernel, int tiles, int px) {
      ProfScope prof(ctx, "gated_short", flops, bytes);
      hipLaunchKernelGGL(kernel, dim3((unsigned)(tiles * a.col_tiles)), dim3(256), (size_t)px * a.steps * kStep * 16,
                         ctx->stream, a);
      return check_launch("gated_short");
    };
    if (a.ic <= 256 && wide >= 512 && cols <= 4) {
      SY_CHECK(wide * 256LL < (1LL << 32), SY_EUNSUPPORTED, "gated grid too large");
      a.col_tiles = 1;
      return a.steps <= 8 ? go(gated_short_kernel<2, 32, 1>, wide, 2) : go(gated_short_kernel<2, 64, 1>, wide, 2);
    }
    if ((cols <= 3 && a.ic <= 256) || (long long)a.xpanels * cols <= 900) {
      a.col_tiles = a.xpanels >= 400 ? 1 : cols;
      if (a.ic > 256) return go(gated_short_kernel<1, 64, 2>, a.xpanels, 1);
      return a.steps <= 8 ? go(gated_short_kernel<1, 32, 1>, a.xpanels, 1) : go(gated_short_kernel<1, 64, 1>, a.xpanels, 1);
    }
  }
  // One workgroup to a CU: 1200 rows of 600 to 690 channels (228 of them) 22.6 us here, 27.4 split beforehand; to 1365
  // (418) 44.1 and 28.8.  Two panels to a workgroup where those find room, too: 400 rows of 600 to 600 14.2 us, four 20.8.
  const long long mids = a.xpanels * ((p.panels + 3LL) / 4), wide = a.xpanels * ((p.panels + 1LL) / 2);
  if (mids <= 256) {
    ProfScope prof(ctx, "gated_mid", flops, bytes);
    if (wide <= 256)
      hipLaunchKernelGGL(gated_mid_kernel<2>, dim3((unsigned)wide), dim3(512), 0, ctx->stream, a);
    else
      hipLaunchKernelGGL(gated_mid_kernel<4>, dim3((unsigned)mids), dim3(512), 0, ctx->stream, a);
    return check_launch("gated_mid");
  }
  size_t at = 0;
  auto take = [&](size_t size) {
    const size_t from = at;
    at += (size + 255) & ~size_t(255);
    return from;
  };
  const size_t xs_at = take((size_t)a.xpanels * p.steps * kStep * 16), row_at = take((size_t)a.xpanels * 32 * sizeof(int)),
               plain_at = take((size_t)a.xpanels * sizeof(int));
  SY_TRY(ensure_scratch(ctx, at));
  u32x4* xs = (u32x4*)(ctx->scratch + xs_at);
  int *x_row = (int*)(ctx->scratch + row_at), *x_plain = (int*)(ctx->scratch + plain_at);
  a.xs = xs;
  a.x_row = x_row;
  a.x_plain = x_plain;
  {
    ProfScope prof(ctx, "gated_split", 0, 8.0 * rows * p.ic);
    hipLaunchKernelGGL(gated_split_kernel, dim3(a.xpanels), dim3(512), 0, ctx->stream, a.x, a.ldx, a.rows, a.ic, a.steps,
                       xs, x_row, x_plain, 1, 0, false);
    SY_TRY(check_launch("gated_split"));
  }
  ProfScope prof(ctx, "gated", flops, bytes);
  auto tiles = [&](int rows, int cols) {
    a.row_tiles = (a.xpanels + rows - 1) / rows;
    a.col_tiles = (a.panels + cols - 1) / cols;
    return (long long)a.row_tiles * a.col_tiles;
  };
  auto launch = [&](auto kernel, int rows, int cols, int waves) {
    const long long grid = tiles(rows, cols);
    SY_CHECK(grid * waves * 64 < (1LL << 32), SY_EUNSUPPORTED, "gated grid too large");
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(waves * 64), 0, ctx->stream, a);
    return check_launch("gated");
  };
  // Two panels of output channels to a workgroup where there are no more: 60000 rows of 512 to 64 channels 83 us, 99 where
  // half the waves have none.
  if (a.panels <= 2) return launch(gated_kernel<1, 2>, 2, 2, 2);
  return launch(gated_kernel<1, 4>, 2, 4, 4);
}

}  // namespace sy

extern "C" {

int sy_gated_create(sy_ctx* ctx, const float* gate, const float* up, const float* gate_bias, const float* up_bias,
                    int oc, int ic, int act, uint64_t* gated) {
  return sy::op_gated_create(ctx, gate, up, gate_bias, up_bias, oc, ic, act, gated);
}

int sy_gated_run(sy_ctx* ctx, uint64_t gated, const sy_tensor* x, const sy_tensor* y) {
  SY_CHECK(ctx, SY_EINVAL, "null context");
  return sy::op_gated_run(ctx, gated, x, y);
}

}  // extern "C"
