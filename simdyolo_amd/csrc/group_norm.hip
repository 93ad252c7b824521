// Group normalisation (Wu and He, 2018) of NHWC views with an activation:
// y = act((x - mean) / sqrt(var + eps) gamma + beta), mean and variance over an
// image's pixels and a group's channels.
//
// Sums are those of d = x - p and d^2 in 64 bits, p the first element of the group:
// exact but for 2^-53 of each term, so neither a mean far from zero nor a long sum
// costs precision, and one pass over the data gives both.  64-bit additions run at half
// the rate of 32-bit ones, far above what memory feeds them with.  No atomics: results do not
// depend on the order in which workgroups end.
#include <algorithm>
#include <cmath>

#include "activation.h"

namespace sy {

struct NormArgs {
  const float* x;
  float* y;
  const float *gamma, *beta;
  long long ldx, ldy;
  int n, t, c, groups, each;  // each: channels of a group
  int act;
  double eps, share;          // share: 1 / elements of a group
  // Runs of groups (columns of a workgroup) and pieces of the pixels.
  int run, runs, cols, rows;  // groups of a run, runs; columns (of VEC channels), pixels side by side
  int blocks;                 // a run is a group's share of columns: so many to a group (1: whole groups)
  int piece, pieces;
  int lanes;                  // rows_kernel: lanes of a group
  double2* sums;              // [n][groups][blocks][pieces]
  float* pivot;               // [n][groups]
};

template <int VEC>
struct Vec;
template <>
struct Vec<4> {
  typedef f32x4 type __attribute__((aligned(4)));  // the memory takes quads at any multiple of four bytes
};
template <>
struct Vec<1> {
  typedef float __attribute__((ext_vector_type(1))) type;
};

struct Moments {
  double s, q;
  __device__ void add(float x, double p) {
    const double d = (double)x - p;
    s += d;
    q = __builtin_fma(d, d, q);
  }
};

// Mean (in two floats) and 1 / sqrt(var + eps): the hardware's estimate (2^-23 and
// better) and one step of Newton's, where a library's division and root would
// cost more than the rest of a token's work.  Both under a power of two, `pre`, which x is multiplied with as the mean
// is taken off: 1 but where the spread is past 2^100, so that differences or the factor leave float32, or (without
// eps) below 2^-100, so that the factor or the mean's second part does.
struct Scale {
  float hi, lo, r, pre;
};
__device__ __forceinline__ Scale scale_of(const NormArgs& a, const Moments& m, double p) {
  const double d = m.s * a.share;
  double mean = p + d, var = __builtin_fma(m.q, a.share, -d * d);
  var = (var < 0 ? 0 : var) + a.eps;  // NaN stays
  double e = __builtin_amdgcn_rsq(var);
  e *= __builtin_fma(-0.5 * var * e, e, 1.5);
  Scale s;
  s.pre = var > 0x1p200 ? 0x1p-60f : var < 0x1p-200 ? 0x1p60f : 1.f;
  mean *= (double)s.pre;
  s.hi = (float)mean;
  s.lo = __builtin_fabsf(s.hi) < INFINITY ? (float)(mean - (double)s.hi) : 0.f;
  s.r = (float)(var > 0x1p200 ? e * 0x1p60 : var < 0x1p-200 ? e * 0x1p-60 : e);
  return s;
}

// Before the activation.
__device__ __forceinline__ float normal(float x, const Scale& s, float g, float b) {
  return __builtin_fmaf(__builtin_fmaf(x, s.pre, -s.hi) - s.lo, s.r * g, b);
}

template <int VEC>
__device__ __forceinline__ void put(float* to, const float* from) {
  typedef typename Vec<VEC>::type vec;
  vec t;
#pragma unroll
  for (int e = 0; e < VEC; ++e) t[e] = from[e];
  *(vec*)to = t;
}

// v plus that of the lane that DPP control ctrl reads.
template <int ctrl>
__device__ __forceinline__ double plus_dpp(double v) {
  const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
  const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)b, ctrl, 0xf, 0xf, false);
  const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), ctrl, 0xf, 0xf, false);
  return v + __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}

// Sum over aligned groups of `lanes` (a power of two), in each of them.
__device__ __forceinline__ double plus_lanes(double v, int lanes) {
  if (lanes > 1) v = plus_dpp<0xb1>(v);   // lane ^ 1
  if (lanes > 2) v = plus_dpp<0x4e>(v);   // lane ^ 2
  if (lanes > 4) v = plus_dpp<0x141>(v);  // 7 - lane
  if (lanes > 8) v = plus_dpp<0x140>(v);  // 15 - lane
  if (lanes > 16) v += __shfl_xor(v, 16);
  if (lanes > 32) v += __shfl_xor(v, 32);
  return v;
}

// A group of an image by `lanes` neighbouring lanes, its elements in their
// registers: small images, single tokens.  Memory bounds it: 8400 tokens of 256 channels, one group
// each, 8.3 us, 2.1 TB/s, half of that the launch.
template <int VEC, int V>
__global__ __launch_bounds__(256) void norm_rows_kernel(const NormArgs a) {
  typedef typename Vec<VEC>::type vec;
  const int lanes = a.lanes, lane = threadIdx.x & (lanes - 1);
  const long long all = (long long)a.n * a.groups;
  long long item = (long long)blockIdx.x * (256 / lanes) + threadIdx.x / lanes;
  const bool live = item < all;
  item = live ? item : all - 1;
  const long long img = item / a.groups;
  const int g = (int)(item - img * a.groups), units = a.each / VEC, total = a.t * units;
  const float* x = a.x + img * a.t * a.ldx + g * a.each;
  float* y = a.y + img * a.t * a.ldy + g * a.each;
  vec v[V];
  int px[V], ch[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int u = min(lane + i * lanes, total - 1);
    px[i] = u / units;
    ch[i] = (u - px[i] * units) * VEC;
    v[i] = *(const vec*)(x + px[i] * a.ldx + ch[i]);
  }
  vec ga[V], be[V];
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int c = g * a.each + ch[i] + e;
      ga[i][e] = a.gamma ? a.gamma[c] : 1.f;
      be[i][e] = a.beta ? a.beta[c] : 0.f;
    }
  const double p = (double)x[0];
  Moments m{0, 0};
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (lane + i * lanes < total)
#pragma unroll
      for (int e = 0; e < VEC; ++e) m.add(v[i][e], p);
  m.s = plus_lanes(m.s, lanes);
  m.q = plus_lanes(m.q, lanes);
  const Scale s = scale_of(a, m, p);
  float o[V * VEC];
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[i * VEC + e] = normal(v[i][e], s, ga[i][e], be[i][e]);
  activate(a.act, o);
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (live && lane + i * lanes < total) put<VEC>(y + px[i] * a.ldy + ch[i], &o[i * VEC]);
}

// The moments of the run's groups from every thread's own, E of them, each of one group: a
// wave adds up a group's, in one order.  cols_each and used: of a group and of all, side by side.
template <int E>
__device__ __forceinline__ void meet(const NormArgs& a, const Moments (&m)[E], double2* red, int cols_each, int used,
                                     int groups, Moments* out) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
#pragma unroll
  for (int e = 0; e < E; ++e) red[threadIdx.x * E + e] = make_double2(m[e].s, m[e].q);
  __syncthreads();
  const int per = a.rows * cols_each;
  for (int g = wave; g < groups; g += waves) {
    Moments s{0, 0};
    for (int i = lane; i < per; i += 64) {
      const int r = i / cols_each, at = r * used + g * cols_each + i - r * cols_each;
      s.s += red[at].x;
      s.q += red[at].y;
    }
    s.s = plus_lanes(s.s, 64);
    s.q = plus_lanes(s.q, 64);
    if (lane == 0) out[g] = s;
  }
  __syncthreads();
}

constexpr int kMaxRun = 256;  // groups of a run at most: one to a column of 256 threads and more

// A group of one image per workgroup, its elements in registers: a thread stays with
// its column (VEC channels) and goes down the pixels.  Neighbouring groups, which share
// lines of memory where they have few channels, are neighbours on one XCD.  Latency bounds it, of
// the launch and one trip to memory: a 20x20 map of 256 channels, 32 groups 3.9 us.
constexpr int kGroupVec = 4;  // vectors that a thread holds
template <int VEC>
__global__ __launch_bounds__(1024) void norm_group_kernel(const NormArgs a) {
  constexpr int V = kGroupVec;
  typedef typename Vec<VEC>::type vec;
  __shared__ double2 red[16];
  const unsigned item = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  if (item >= (unsigned)a.n * a.groups) return;
  const int img = item / a.groups, g = item - img * a.groups;
  const int row = threadIdx.x / a.cols, col = threadIdx.x - row * a.cols, c = g * a.each + col * VEC;
  const bool live = row < a.rows;
  const float* x = a.x + (long long)img * a.t * a.ldx;
  float* y = a.y + (long long)img * a.t * a.ldy;
  vec v[V];
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = *(const vec*)(x + min(row + i * a.rows, a.t - 1) * a.ldx + c);
  const double p = (double)x[g * a.each];
  float ga[VEC], be[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    ga[e] = a.gamma ? a.gamma[c + e] : 1.f;
    be[e] = a.beta ? a.beta[c + e] : 0.f;
  }
  Moments m{0, 0};
  if (live)
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (row + i * a.rows < a.t)
#pragma unroll
        for (int e = 0; e < VEC; ++e) m.add(v[i][e], p);
  m.s = plus_lanes(m.s, 64);
  m.q = plus_lanes(m.q, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = make_double2(m.s, m.q);
  __syncthreads();
  m = {red[0].x, red[0].y};
  for (unsigned w = 1; w < blockDim.x >> 6; ++w) {
    m.s += red[w].x;
    m.q += red[w].y;
  }
  if (!live) return;
  const Scale s = scale_of(a, m, p);
  float o[V * VEC];
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[i * VEC + e] = normal(v[i][e], s, ga[e], be[e]);
  activate(a.act, o);
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (row + i * a.rows < a.t) put<VEC>(y + (row + i * a.rows) * a.ldy + c, &o[i * VEC]);
}

constexpr int kDeep = 4;  // pixels of a thread under way

// Larger images: the moments of a piece of the pixels and a run of groups, then
// every piece normalised by the moments of all.  MIX: a column's four channels may be of
// several groups, and have moments each.  Two launches, since a piece waits for all others' moments; x is
// read twice, the second time from the last-level cache where it fits (256 MB), and y goes past the caches
// so that it does.  Memory bounds both: eight 160x160 maps of 256 channels, 32 groups 103 us, 4.1 TB/s of
// what has to be moved (6.1 with the second reading), 38 of them for the sums at 5.5 TB/s.  Five 45x75 maps
// of 108 channels, 12 groups 11.6 us: launches and one trip to memory each.
template <int VEC, bool MIX>
__global__ __launch_bounds__(256) void norm_sums_kernel(const NormArgs a) {
  typedef typename Vec<VEC>::type vec;
  constexpr int E = MIX ? VEC : 1, W = MIX ? 1 : VEC;  // moments of a thread; channels of one
  __shared__ double2 red[256 * E];
  __shared__ Moments total[kMaxRun];
  const int piece = blockIdx.x % a.pieces, rest = blockIdx.x / a.pieces, img = rest / a.runs, run = rest - img * a.runs;
  const int g0 = run / a.blocks * a.run, first = run % a.blocks * a.cols;  // group, its column
  const int groups = min(a.run, a.groups - g0);
  const int cols_each = min(a.each / W - first, a.cols * E), cols = groups * cols_each / E;
  const int row = threadIdx.x / a.cols, col = threadIdx.x - row * a.cols, col1 = min(col, cols - 1);
  const bool live = row < a.rows && col < cols;
  const int c = g0 * a.each + (first + col1) * VEC;
  const float* x = a.x + (long long)img * a.t * a.ldx;
  const int from = piece * a.piece, to = min(from + a.piece, a.t);
  double p[E];
  Moments m[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    p[e] = (double)x[(g0 + (col1 * E + e) / cols_each) * a.each];
    m[e] = {0, 0};
  }
  if (live) {
    for (int i = from + row; i < to; i += kDeep * a.rows) {
      vec v[kDeep];
#pragma unroll
      for (int k = 0; k < kDeep; ++k) v[k] = *(const vec*)(x + min(i + k * a.rows, to - 1) * a.ldx + c);
#pragma unroll
      for (int k = 0; k < kDeep; ++k)
        if (i + k * a.rows < to)
#pragma unroll
          for (int e = 0; e < VEC; ++e) m[e % E].add(v[k][e], p[e % E]);
    }
  }
  meet<E>(a, m, red, cols_each, a.cols * E, groups, total);
  if (piece == 0 && run % a.blocks == 0)
    for (int i = threadIdx.x; i < groups; i += 256)
      a.pivot[(long long)img * a.groups + g0 + i] = x[(g0 + i) * a.each];
  for (int i = threadIdx.x; i < groups; i += 256)
    a.sums[(((long long)img * a.groups + g0 + i) * a.blocks + run % a.blocks) * a.pieces + piece] =
        make_double2(total[i].s, total[i].q);
}

template <int VEC, bool MIX>
__global__ __launch_bounds__(256) void norm_apply_kernel(const NormArgs a) {
  typedef typename Vec<VEC>::type vec;
  constexpr int E = MIX ? VEC : 1, W = MIX ? 1 : VEC;
  __shared__ Scale scale[kMaxRun];
  const int piece = blockIdx.x % a.pieces, rest = blockIdx.x / a.pieces, img = rest / a.runs, run = rest - img * a.runs;
  const int g0 = run / a.blocks * a.run, first = run % a.blocks * a.cols, lane = threadIdx.x & 63;
  const int groups = min(a.run, a.groups - g0);
  const int cols_each = min(a.each / W - first, a.cols * E), cols = groups * cols_each / E;
  const float* x = a.x + (long long)img * a.t * a.ldx;
  float* y = a.y + (long long)img * a.t * a.ldy;
  const int row = threadIdx.x / a.cols, col = min((int)threadIdx.x - row * a.cols, cols - 1);
  const int c = g0 * a.each + (first + col) * VEC;
  const int from = piece * a.piece, to = min(from + a.piece, a.t);
  // The first pixels and the weights are under way while the moments meet.
  int i = from + row;
  vec v[kDeep];
#pragma unroll
  for (int k = 0; k < kDeep; ++k) v[k] = *(const vec*)(x + min(i + k * a.rows, to - 1) * a.ldx + c);
  float ga[VEC], be[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    ga[e] = a.gamma ? a.gamma[c + e] : 1.f;
    be[e] = a.beta ? a.beta[c + e] : 0.f;
  }
  for (int g = threadIdx.x >> 6; g < groups; g += 4) {
    const int parts = a.blocks * a.pieces;
    const double2* sums = a.sums + ((long long)img * a.groups + g0 + g) * parts;
    Moments m{0, 0};
    for (int p = lane; p < parts; p += 64) {
      m.s += sums[p].x;
      m.q += sums[p].y;
    }
    m.s = plus_lanes(m.s, 64);
    m.q = plus_lanes(m.q, 64);
    if (lane == 0) scale[g] = scale_of(a, m, (double)a.pivot[((long long)img * a.groups + g0 + g)]);
  }
  __syncthreads();
  if (row >= a.rows || (int)threadIdx.x - row * a.cols >= cols) return;
  Scale s[E];
#pragma unroll
  for (int e = 0; e < E; ++e) s[e] = scale[(col * E + e) / cols_each];
  while (i < to) {
    float o[kDeep * VEC];
#pragma unroll
    for (int k = 0; k < kDeep; ++k)
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[k * VEC + e] = normal(v[k][e], s[e % E], ga[e], be[e]);
    const int at = i;
    i += kDeep * a.rows;
    if (i < to)
#pragma unroll
      for (int k = 0; k < kDeep; ++k) v[k] = *(const vec*)(x + min(i + k * a.rows, to - 1) * a.ldx + c);
    activate(a.act, o);
#pragma unroll
    for (int k = 0; k < kDeep; ++k)
      if (at + k * a.rows < to) {
        vec t;
#pragma unroll
        for (int e = 0; e < VEC; ++e) t[e] = o[k * VEC + e];
        __builtin_nontemporal_store(t, (vec*)(y + (at + k * a.rows) * a.ldy + c));
      }
  }
}

// Elements of a group that 64 lanes hold: kRowsVec vectors each.
constexpr int kRowsVec = 4;

int op_group_norm(sy_ctx* ctx, const sy_tensor* x, int groups, const float* gamma, const float* beta, float eps,
                  int act, const sy_tensor* y) {
  SY_TRY(check_view(x, "group norm input"));
  SY_TRY(check_view(y, "group norm output"));
  SY_CHECK(y->n == x->n && y->c == x->c && y->h == x->h && y->w == x->w, SY_EINVAL,
           "group norm output shape mismatch");
  SY_CHECK(groups > 0 && x->c % groups == 0, SY_EINVAL, "%d channels in %d groups", x->c, groups);
  SY_CHECK(act >= SY_ACT_NONE && act <= SY_ACT_SIGMOID, SY_EINVAL, "unknown activation %d", act);
  SY_CHECK(std::isfinite(eps) && eps >= 0, SY_EINVAL, "group norm eps must be 0 or more and finite");
  SY_CHECK((long long)x->h * x->w < (1LL << 30), SY_EUNSUPPORTED, "group norm over 2^30 pixels and more");
  SY_CHECK((((uintptr_t)x->data | (uintptr_t)y->data | (uintptr_t)gamma | (uintptr_t)beta) & 3) == 0, SY_EINVAL,
           "group norm operands must be 4-byte aligned");
  const bool same = x->data == y->data && x->ldc == y->ldc;
  SY_CHECK(same || !views_overlap(x, y), SY_EINVAL, "group norm output overlaps its input other than in place");
  for (const float* p : {gamma, beta})
    if (p) {
      const sy_tensor t{(float*)p, 1, x->c, 1, 1, x->c, SY_LAYOUT_NHWC};
      SY_CHECK(!views_overlap(&t, y), SY_EINVAL, "group norm output overlaps its weights");
    }
  SY_CHECK(ctx, SY_EINVAL, "null context");
  NormArgs a{};
  a.x = x->data;
  a.y = y->data;
  a.gamma = gamma;
  a.beta = beta;
  a.ldx = x->ldc;
  a.ldy = y->ldc;
  a.n = x->n;
  a.t = x->h * x->w;
  a.c = x->c;
  a.groups = groups;
  a.each = x->c / groups;
  a.act = act;
  a.eps = eps;
  a.share = 1.0 / ((double)a.t * a.each);
  const bool quads = a.each % 4 == 0;
  const int vec = quads ? 4 : 1;
  const long long units = (long long)a.t * (a.each / vec);  // of a group
  const double bytes = 8.0 * a.n * (double)a.t * a.c, flops = 8.0 * a.n * (double)a.t * a.c;
  DeviceScope device(ctx);
  ProfScope prof(ctx, "group_norm", flops, bytes);
  if (units <= 64 * kRowsVec) {
    a.lanes = 1;
    while (a.lanes < 64 && a.lanes < units) a.lanes *= 2;
    const long long grid = ((long long)a.n * groups * a.lanes + 255) / 256;
    SY_CHECK(grid * 256 < (1LL << 32), SY_EUNSUPPORTED, "group norm over %d images of %d groups", a.n, groups);
    const int v = (int)((units + a.lanes - 1) / a.lanes);
    auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(256), 0, ctx->stream, a); };
    if (quads)
      v <= 1 ? launch(norm_rows_kernel<4, 1>) : launch(norm_rows_kernel<4, kRowsVec>);
    else
      launch(norm_rows_kernel<1, kRowsVec>);
    return check_launch("group_norm");
  }
  const int each = a.each / vec;
  if (each <= 1024 && (a.t + 1024 / each - 1) / (1024 / each) <= kGroupVec) {
    int threads = 256;
    while (each > threads || (a.t + threads / each - 1) / (threads / each) > kGroupVec) threads *= 2;
    a.cols = each;
    a.rows = threads / each;
    const long long grid = ((long long)a.n * groups + 7) / 8 * 8;
    SY_CHECK(grid * threads < (1LL << 32), SY_EUNSUPPORTED, "group norm over %d images of %d groups", a.n, groups);
    hipLaunchKernelGGL(quads ? norm_group_kernel<4> : norm_group_kernel<1>, dim3((unsigned)grid), dim3(threads), 0,
                       ctx->stream, a);
    return check_launch("group_norm");
  }
  // A run of groups: 128 bytes of a pixel and more.  Where groups are not of whole quads but a pixel is, runs of two or
  // four groups are, too; their columns have four moments each, which pays for large maps: eight 160x160 maps of 60
  // channels, 4 groups 45.5 us, 66.5 channel by channel, of 180, 12 groups 112 and 128, sixteen 45x75 of 108, 12 groups
  // 21.8 and 25.3, but five of those 13.2 and 11.9.
  const int whole = a.each % 2 ? 4 : 2;
  const bool mix = !quads && a.c % 4 == 0 && whole * a.each <= 1024 && (double)a.n * a.t * a.c >= 4e6;
  if (mix) {
    a.run = std::min(groups, (32 / a.each + whole - 1) / whole * whole + (a.each > 32 ? whole : 0));
    a.cols = a.run * a.each / 4;
    a.blocks = 1;
  } else {
    a.run = std::min({groups, std::max(1, 256 / each), std::max(1, (32 / vec + each - 1) / each)});
    a.cols = std::min(a.run * each, 256);
    a.blocks = (each + 255) / 256;
  }
  a.rows = 256 / a.cols;
  a.runs = a.blocks > 1 ? groups * a.blocks : (groups + a.run - 1) / a.run;
  // Pieces: 8 pixels of a thread and more in up to 8192 workgroups, 4 where those would be fewer than 1024: one 80x80 map
  // of 64 channels 9.2 us with 4, 11.9 with 8, 16.7 with 16 (its few waves work through them one by one); eight 160x160
  // maps of 256 channels 108 with 4 and 104 with 8.
  const long long runs = (long long)a.n * a.runs;
  const int least = a.t * runs >= 1024LL * 4 * a.rows ? 8 : 4;
  a.piece = (int)std::max<long long>(least * a.rows, (a.t * runs + 8191) / 8192);
  a.pieces = (a.t + a.piece - 1) / a.piece;
  const long long grid = runs * a.pieces;
  SY_CHECK(grid * 256 < (1LL << 32), SY_EUNSUPPORTED, "group norm over %d images of %d groups", a.n, groups);
  const size_t sums = sizeof(double2) * (size_t)a.n * groups * a.blocks * a.pieces;
  SY_TRY(ensure_scratch(ctx, sums + sizeof(float) * (size_t)a.n * groups));
  a.sums = (double2*)ctx->scratch;
  a.pivot = (float*)(ctx->scratch + sums);
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(256), 0, ctx->stream, a); };
  launch(quads ? norm_sums_kernel<4, false> : mix ? norm_sums_kernel<4, true> : norm_sums_kernel<1, false>);
  launch(quads ? norm_apply_kernel<4, false> : mix ? norm_apply_kernel<4, true> : norm_apply_kernel<1, false>);
  return check_launch("group_norm");
}

}  // namespace sy

extern "C" int sy_group_norm(sy_ctx* ctx, const sy_tensor* x, int groups, const float* gamma, const float* beta,
                             float eps, int act, const sy_tensor* y) {
  return sy::op_group_norm(ctx, x, groups, gamma, beta, eps, act, y);
}
