// The gated half of a feed-forward block: y = act(x G^T + g) * (x U^T + u), both
// products, the activation and their product in one kernel.
//
// Products of float32 on the f16 matrix cores (Ootomo and Yokota, 2022): an operand is
// a pair h + l / 2048 of f16 values under a power of two of its own row (a pixel of x, an
// output channel of G or U), and h h + (h l + l h) / 2048 is taken.  A pair is within 2^-22 of
// its element as long as that is not below 2^-29 of its row's largest, and within 2^-50 of the
// largest below; what is left out, l l, is 2^-22 of the product at most.  Rows that hold a
// nonzero element below kUneven of their largest, infinities or NaN are not multiplied so: the tiles
// that meet them are computed in plain float32, on the float32 matrix cores.
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
  float* raw = nullptr;   // [gate, up][oc][ic], where a panel is uneven
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
  bool quads;  // x can be read 16 bytes at a time
};

// Exponent field of the power of two that takes a largest magnitude m into [2^14,
// 2^15); rows below 2^-113 keep the largest power there is.
__device__ __forceinline__ int gated_field(unsigned m) { return min(268 - (int)(m >> 23), 254); }

__device__ __forceinline__ unsigned magnitude(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }

// Whether a row with the largest magnitude m must be computed plainly, from its smallest nonzero one.
__device__ __forceinline__ bool uneven(unsigned largest, unsigned smallest) {
  const int e = (int)(largest >> 23);
  return e == 255 || (smallest != 0x7fffffffu && (int)(smallest >> 23) < e + kUneven && smallest != 0);
}

// Eight elements of a row of `end` from `at`, zeros from `end` on.
__device__ __forceinline__ void load8(const float* row, int at, int end, bool quads, float (&v)[8]) {
  if (quads) {  // end is a multiple of 4
    const f32x4 a = *(const f32x4*)(row + min(at, end - 4)), b = *(const f32x4*)(row + min(at + 4, end - 4));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = a[e];
      v[4 + e] = b[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = row[min(at + e, end - 1)];
  }
  if (at + 8 > end)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = at + e < end ? v[e] : 0.f;
}

__device__ __forceinline__ void pair8(const float (&x)[8], float s, u32x4& h, u32x4& l) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = x[2 * i], b = x[2 * i + 1];
    const f16x2 hi = __builtin_convertvector((f32x2v{a * s, b * s}), f16x2);
    const f32x2v r = {__builtin_fmaf(a, s, -(float)hi[0]), __builtin_fmaf(b, s, -(float)hi[1])};
    h[i] = __builtin_bit_cast(unsigned, hi);
    l[i] = __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2v{r[0] * 2048.f, r[1] * 2048.f}), f16x2));
  }
}

// A panel of 32 rows per workgroup, 16 lanes to a row: its largest element, then its
// pairs; the first kHeld octets of a lane stay in registers between.  Rows past the last are zeros.
// `more`: the panel's flag is that of an earlier call, too.
constexpr int kHeld = 2;
__global__ __launch_bounds__(512) void gated_split_kernel(const float* x, long long ldx, int rows, int ic, int steps,
                                                          bool quads, u32x4* out, int* words, int* plain, int stride,
                                                          int offset, bool more) {
  __shared__ int any;
  const int r = threadIdx.x >> 4, q = threadIdx.x & 15;
  const long long row = (long long)blockIdx.x * 32 + r;
  const long long panel = (long long)blockIdx.x * stride + offset;
  const float* xr = x + min(row, (long long)rows - 1) * ldx;
  if (threadIdx.x == 0) any = more ? plain[blockIdx.x] : 0;
  __syncthreads();
  unsigned top = 0, low = 0x7fffffffu;
  float held[kHeld][8];
  auto look = [&](const float(&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const unsigned m = magnitude(v[e]);
      top = max(top, m);
      low = min(low, m ? m : 0x7fffffffu);
    }
  };
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (q + 16 * i < 2 * steps) load8(xr, 8 * (q + 16 * i), ic, quads, held[i]);
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (q + 16 * i < 2 * steps) look(held[i]);
  for (int o = q + 16 * kHeld; o < 2 * steps; o += 16) {
    float v[8];
    load8(xr, 8 * o, ic, quads, v);
    look(v);
  }
#pragma unroll
  for (int off = 1; off < 16; off <<= 1) {
    top = max(top, (unsigned)__shfl_xor((int)top, off));
    low = min(low, (unsigned)__shfl_xor((int)low, off));
  }
  if (row >= rows) top = 0, low = 0x7fffffffu;
  const bool bad = uneven(top, low);
  const int field = bad && top >> 23 == 255 ? 127 : gated_field(top);
  if (q == 0) {
    words[panel * 32 + r] = field | (bad ? kPlainRow : 0);
    if (bad) any = 1;
  }
  const float s = row < rows ? exp_float(field) : 0.f;
  u32x4* to = out + panel * steps * kStep;
  auto put = [&](int o, const float(&v)[8]) {
    u32x4 h, l;
    pair8(v, s, h, l);
    to[(o >> 1) * kStep + (o & 1) * 32 + r] = h;
    to[(o >> 1) * kStep + 64 + (o & 1) * 32 + r] = l;
  };
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (q + 16 * i < 2 * steps) put(q + 16 * i, held[i]);
  for (int o = q + 16 * kHeld; o < 2 * steps; o += 16) {
    float v[8];
    load8(xr, 8 * o, ic, quads, v);
    put(o, v);
  }
  __syncthreads();
  if (threadIdx.x == 0) plain[blockIdx.x] = any;
}

// Four weights of output channel `col` (gate or up) from input channel k.
__device__ __forceinline__ f32x4 gated_weights(const GatedArgs& a, int which, int col, int k) {
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (a.raw) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (col < a.oc && k + e < a.ic) v[e] = a.raw[((long long)which * a.oc + col) * a.ic + k + e];
    return v;
  }
  typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
  const long long panel = 2LL * (col >> 5) + which;
  const _Float16* w = (const _Float16*)(a.w + (panel * a.steps + (k >> 4)) * kStep + ((k >> 3) & 1) * 32 + (col & 31)) + (k & 7);
  const f16x4 hi = *(const f16x4*)w, lo = *(const f16x4*)(w + 512);
  const float s = exp_float(254 - (a.w_row[panel * 32 + (col & 31)] & 0xff));
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf((float)lo[e], 1.f / 2048, (float)hi[e]) * s;
  return v;
}

// 32 x 32 gate and up sums of a wave in plain float32, over steps [k0, k1).
__device__ __forceinline__ void gated_plain(const GatedArgs& a, long long row0, int panel, int k0, int k1, int lane,
                                            f32x16 (&acc)[2]) {
  const int half = lane >> 5, r32 = lane & 31;
  const long long row = row0 + r32;
  const float* x = a.x + min(row, (long long)a.rows - 1) * a.ldx;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[0][r] = acc[1][r] = 0.f;
  for (int k = 16 * k0; k < 16 * k1; k += 8) {
    const int c = k + 4 * half;
    f32x4 xv;
#pragma unroll
    for (int e = 0; e < 4; ++e) xv[e] = row < a.rows && c + e < a.ic ? x[c + e] : 0.f;
    const f32x4 g = gated_weights(a, 0, 32 * panel + r32, c), u = gated_weights(a, 1, 32 * panel + r32, c);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      acc[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(xv[e], g[e], acc[0], 0, 0, 0);
      acc[1] = __builtin_amdgcn_mfma_f32_32x32x2f32(xv[e], u[e], acc[1], 0, 0, 0);
    }
  }
}

// WM x WN waves, each 64 rows by 32 output channels (gate and up): x and the weights
// arrive split, in the order of the matrix instruction's lanes; two steps at a time
// go through LDS, two stages in turn with one barrier between.
template <int WM, int WN>
__global__ __launch_bounds__(WM* WN * 64, 2) void gated_kernel(const GatedArgs a) {
  constexpr int NW = WM * WN, PA = 2 * WM, PB = 2 * WN;  // panels of x and of the weights
  constexpr int CHUNKS = 4 * (PA + PB), IT = CHUNKS / NW;   // 1 KB each
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
    const int c = wave + i * NW, p = c >> 2;
    const u32x4* base = p < PA ? a.xs + (long long)min(rt * PA + p, a.xpanels - 1) * a.steps * kStep
                               : a.w + (long long)min(ct * PB + p - PA, 2 * a.panels - 1) * a.steps * kStep;
    src[i] = base + (c & 3) * 64 + lane;
  }
  f32x16 acc[2][2], crs[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
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
  const int stages = a.steps / 2;
  gload(0);
  put(0);
  __syncthreads();
  for (int s = 0; s < stages; ++s) {
    if (s + 1 < stages) gload(s + 1);
    const u32x4(*f)[64] = frag[s & 1];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      f16x8 av[2][2], bv[2][2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          av[i][p] = __builtin_bit_cast(f16x8, f[(wm * 2 + i) * 4 + 2 * k + p][lane]);
          bv[i][p] = __builtin_bit_cast(f16x8, f[(PA + wn * 2 + i) * 4 + 2 * k + p][lane]);
        }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          crs[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(av[i][1], bv[j][0], crs[i][j], 0, 0, 0);
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(av[i][0], bv[j][0], acc[i][j], 0, 0, 0);
        }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          crs[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(av[i][0], bv[j][1], crs[i][j], 0, 0, 0);
    }
    if (s + 1 < stages) put((s + 1) & 1);
    __syncthreads();
  }

  const int panel = ct * WN + wn, col = 32 * panel + r32;
  if (panel >= a.panels) return;
  const bool live = col < a.oc;
  const float gb = a.bias[col], ub = a.bias[a.panels * 32 + col];
  const int gw = a.w_row[panel * 64 + r32] & 0xff, uw = a.w_row[panel * 64 + 32 + r32] & 0xff;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int xp = (rt * WM + wm) * 2 + i;
    if (xp >= a.xpanels) return;
    f32x16 g, u;
    if (a.x_plain[xp] | a.w_plain[panel]) {
      f32x16 t[2];
      gated_plain(a, (long long)xp * 32, panel, 0, a.steps, lane, t);
      g = t[0];
      u = t[1];
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int f = a.x_row[xp * 32 + 8 * (r >> 2) + 4 * half + (r & 3)] & 0xff;
        g[r] = __builtin_ldexpf(__builtin_fmaf(crs[i][0][r], 1.f / 2048, acc[i][0][r]), 254 - f - gw);
        u[r] = __builtin_ldexpf(__builtin_fmaf(crs[i][1][r], 1.f / 2048, acc[i][1][r]), 254 - f - uw);
      }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = xp * 32 + 8 * (r >> 2) + 4 * half + (r & 3);
      if (live && row < a.rows) a.y[row * a.ldy + col] = activate(a.act, g[r] + gb) * (u[r] + ub);
    }
  }
}

// Few tiles: TM panels of rows and 32 output channels to a workgroup, the steps shared
// out over its NK waves, both operands straight from memory into the matrix
// instruction's registers, kAhead steps of them under way.  A wave splits its own share of x,
// under powers of that share's rows, and is plain by itself.
constexpr int kAhead = 4;
template <int TM, int NK>
__global__ __launch_bounds__(NK * 64) void gated_few_kernel(const GatedArgs a) {
  __shared__ float sums[NK][2][TM * 32][33];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, r32 = lane & 31;
  const int tile = blockIdx.x / a.panels, panel = blockIdx.x - tile * a.panels, row0 = tile * TM * 32;
  const int share = (a.steps + NK - 1) / NK, k0 = min(wave * share, a.steps), k1 = min(k0 + share, a.steps);
  const u32x4* w = a.w + (long long)2 * panel * a.steps * kStep + lane;
  const long long up = (long long)a.steps * kStep;
  const int w_plain = a.w_plain[panel];
  const float* xr[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) xr[i] = a.x + (long long)min(row0 + 32 * i + r32, a.rows - 1) * a.ldx;
  f16x8 wv[kAhead][2][2];
  float xv[kAhead][TM][8];
  auto load_w = [&](int k) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int p = 0; p < 2; ++p)
          wv[u][j][p] = __builtin_bit_cast(f16x8, w[j * up + (long long)min(k + u, a.steps - 1) * kStep + 64 * p]);
  };
  auto load_x = [&](int k) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
#pragma unroll
      for (int i = 0; i < TM; ++i) load8(xr[i], min(k + u, a.steps) * 16 + 8 * half, a.ic, a.quads, xv[u][i]);
  };
  f32x16 acc[TM][2], crs[TM][2];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = crs[i][j][r] = 0.f;
  unsigned top[TM] = {}, low[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) low[i] = 0x7fffffffu;
  if (k0 < k1) {
    load_w(k0);
    // The share's largest and smallest elements, from behind, so that its first steps stay in registers.
    for (int k = k0 + (k1 - k0 - 1) / kAhead * kAhead; k >= k0; k -= kAhead) {
      load_x(k);
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const unsigned m = k + u < k1 ? magnitude(xv[u][i][e]) : 0;
            top[i] = max(top[i], m);
            low[i] = min(low[i], m ? m : 0x7fffffffu);
          }
    }
  }
  bool plain = w_plain != 0;
  int field[TM];
  float scale[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    top[i] = max(top[i], (unsigned)__shfl_xor((int)top[i], 32));
    low[i] = min(low[i], (unsigned)__shfl_xor((int)low[i], 32));
    plain |= uneven(top[i], low[i]);
    field[i] = gated_field(top[i]);
    scale[i] = exp_float(field[i]);
  }
  if (__any(plain)) {
#pragma unroll
    for (int i = 0; i < TM; ++i) gated_plain(a, row0 + 32 * i, panel, k0, k1, lane, acc[i]);
  } else {
    for (int k = k0; k < k1; k += kAhead) {
      f16x8 xp[kAhead][TM][2], wp[kAhead][2][2];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          u32x4 h, l;
          pair8(xv[u][i], k + u < k1 ? scale[i] : 0.f, h, l);
          xp[u][i][0] = __builtin_bit_cast(f16x8, h);
          xp[u][i][1] = __builtin_bit_cast(f16x8, l);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int p = 0; p < 2; ++p) wp[u][j][p] = wv[u][j][p];
      }
      if (k + kAhead < k1) {
        load_w(k + kAhead);
        load_x(k + kAhead);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            crs[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xp[u][i][1], wp[u][j][0], crs[i][j], 0, 0, 0);
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xp[u][i][0], wp[u][j][0], acc[i][j], 0, 0, 0);
            crs[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xp[u][i][0], wp[u][j][1], crs[i][j], 0, 0, 0);
          }
    }
    // Lane r's field is that of row r.
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int f = __shfl(field[i], 8 * (r >> 2) + 4 * half + (r & 3));
#pragma unroll
        for (int j = 0; j < 2; ++j)
          acc[i][j][r] = __builtin_ldexpf(__builtin_fmaf(crs[i][j][r], 1.f / 2048, acc[i][j][r]),
                                          254 - f - (a.w_row[panel * 64 + 32 * j + r32] & 0xff));
      }
  }
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) sums[wave][j][32 * i + 8 * (r >> 2) + 4 * half + (r & 3)][r32] = acc[i][j][r];
  __syncthreads();
  const int rows = min(TM * 32, a.rows - row0), col = 32 * panel + r32;
  const float gb = a.bias[col], ub = a.bias[a.panels * 32 + col];
  for (int row = threadIdx.x >> 5; row < rows; row += NK * 2) {
    float g = 0.f, u = 0.f;
#pragma unroll
    for (int x = 0; x < NK; ++x) {
      g += sums[x][0][row][r32];
      u += sums[x][1][row][r32];
    }
    if (col < a.oc) a.y[(row0 + row) * a.ldy + col] = activate(a.act, g + gb) * (u + ub);
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
  SY_HIP(hipMalloc((void**)&p->raw, 2 * values * sizeof(float)));
  SY_TRY(sy_memcpy(ctx, p->raw, gate, values * sizeof(float), 0));
  SY_TRY(sy_memcpy(ctx, p->raw + values, up, values * sizeof(float), 0));
  SY_TRY(sy_memcpy(ctx, p->bias, bias.data(), 2 * cols * sizeof(float), 0));
  for (int m = 0; m < 2; ++m)
    hipLaunchKernelGGL(gated_split_kernel, dim3(p->panels), dim3(512), 0, ctx->stream, p->raw + m * values,
                       (long long)p->ic, p->oc, p->ic, p->steps, p->ic % 4 == 0, p->w, p->w_row, p->w_plain, 2, m, m == 1);
  SY_TRY(check_launch("gated_split"));
  std::vector<int> plain;
  try {
    plain.resize(p->panels);
  } catch (const std::bad_alloc&) {
    SY_CHECK(false, SY_ENOMEM, "no memory for a gated layer");
  }
  SY_TRY(sy_memcpy(ctx, plain.data(), p->w_plain, p->panels * sizeof(int), 1));
  if (std::find(plain.begin(), plain.end(), 1) == plain.end()) {
    SY_HIP(hipFree(p->raw));
    p->raw = nullptr;
  }
  return SY_OK;
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
  // The last quad of a row must not pass the buffer's end.
  a.quads = ((uintptr_t)x->data & 15) == 0 && x->ldc % 4 == 0 && p.ic % 4 == 0;
  a.xpanels = (a.rows + 31) / 32;
  DeviceScope device(ctx);
  const double flops = 4.0 * rows * p.ic * p.oc, bytes = 4.0 * ((double)rows * (p.ic + p.oc) + 2.0 * p.ic * p.oc);
  static const int kFew = getenv("FEW") ? atoi(getenv("FEW")) : 0;
  if (a.rows <= 32 || kFew) {
    ProfScope prof(ctx, "gated_few", flops, bytes);
    const int tm = kFew ? kFew / 10 : 1, nk = kFew ? kFew % 10 : 8;
    const dim3 grid((unsigned)(p.panels * ((a.xpanels + tm - 1) / tm)));
    if (tm == 1 && nk == 8) hipLaunchKernelGGL((gated_few_kernel<1, 8>), grid, dim3(nk * 64), 0, ctx->stream, a);
    if (tm == 1 && nk == 4) hipLaunchKernelGGL((gated_few_kernel<1, 4>), grid, dim3(nk * 64), 0, ctx->stream, a);
    if (tm == 2 && nk == 4) hipLaunchKernelGGL((gated_few_kernel<2, 4>), grid, dim3(nk * 64), 0, ctx->stream, a);
    if (tm == 2 && nk == 8) hipLaunchKernelGGL((gated_few_kernel<2, 8>), grid, dim3(nk * 64), 0, ctx->stream, a);
    return check_launch("gated_few");
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
                       a.quads, xs, x_row, x_plain, 1, 0, false);
    SY_TRY(check_launch("gated_split"));
  }
  ProfScope prof(ctx, "gated", flops, bytes);
  auto tiles = [&](int wm, int wn) {
    a.row_tiles = (a.xpanels + 2 * wm - 1) / (2 * wm);
    a.col_tiles = (a.panels + wn - 1) / wn;
    return (long long)a.row_tiles * a.col_tiles;
  };
  auto launch = [&](auto kernel, int wm, int wn) {
    const long long grid = tiles(wm, wn);
    SY_CHECK(grid * wm * wn * 64 < (1LL << 32), SY_EUNSUPPORTED, "gated grid too large");
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(wm * wn * 64), 0, ctx->stream, a);
    return check_launch("gated");
  };
  if (tiles(4, 2) >= 512) return launch(gated_kernel<4, 2>, 4, 2);
  return launch(gated_kernel<2, 1>, 2, 1);
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
