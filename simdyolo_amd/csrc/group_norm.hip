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
  double eps;
  // Runs of groups (columns of a workgroup) and pieces of the pixels.
  int run, runs, cols, rows;  // groups of a run, runs; columns (of VEC channels), pixels side by side
  int blocks;                 // a run is a group's share of columns: so many to a group (1: whole groups)
  int piece, pieces;
  int lanes;                  // rows_kernel: lanes of a group
  double2* sums;              // [n][groups][blocks][pieces]
};

template <int VEC>
struct Vec;
template <>
struct Vec<4> {
  typedef f32x4 type;
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

// Mean (in two floats) and 1 / sqrt(var + eps).
struct Scale {
  float hi, lo, r;
};
__device__ __forceinline__ Scale scale_of(const NormArgs& a, const Moments& m, double p, double count) {
  const double d = m.s / count, mean = p + d;
  double var = m.q / count - d * d;
  var = var < 0 ? 0 : var;  // NaN stays
  Scale s;
  s.hi = (float)mean;
  s.lo = __builtin_fabsf(s.hi) < INFINITY ? (float)(mean - (double)s.hi) : 0.f;
  s.r = (float)(1.0 / sqrt(var + a.eps));
  return s;
}

__device__ __forceinline__ float normal(const NormArgs& a, float x, const Scale& s, float g, float b) {
  return activate(a.act, __builtin_fmaf((x - s.hi) - s.lo, s.r * g, b));
}

__device__ __forceinline__ double shuffle_xor(double v, int lane) { return __shfl_xor(v, lane); }

// A group of an image by `lanes` neighbouring lanes, its elements in their
// registers: small images, single tokens.
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
  const double p = (double)x[0];
  Moments m{0, 0};
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (lane + i * lanes < total)
#pragma unroll
      for (int e = 0; e < VEC; ++e) m.add(v[i][e], p);
  for (int off = 1; off < lanes; off <<= 1) {
    m.s += shuffle_xor(m.s, off);
    m.q += shuffle_xor(m.q, off);
  }
  const Scale s = scale_of(a, m, p, (double)a.t * a.each);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (!live || lane + i * lanes >= total) continue;
    vec o;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int c = g * a.each + ch[i] + e;
      o[e] = normal(a, v[i][e], s, a.gamma ? a.gamma[c] : 1.f, a.beta ? a.beta[c] : 0.f);
    }
    *(vec*)(y + px[i] * a.ldy + ch[i]) = o;
  }
}

// The moments of the run's groups from every thread's own (VEC channels of one
// group): a wave adds up a group's threads, in one order.
__device__ __forceinline__ void meet(const NormArgs& a, const Moments& m, double2* red, int cols_each, int used,
                                     int groups, Moments* out) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  red[threadIdx.x] = make_double2(m.s, m.q);
  __syncthreads();
  const int per = a.rows * cols_each;
  for (int g = wave; g < groups; g += waves) {
    Moments s{0, 0};
    for (int i = lane; i < per; i += 64) {
      const int r = i / cols_each, at = r * used + g * cols_each + i - r * cols_each;
      s.s += red[at].x;
      s.q += red[at].y;
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      s.s += shuffle_xor(s.s, off);
      s.q += shuffle_xor(s.q, off);
    }
    if (lane == 0) out[g] = s;
  }
  __syncthreads();
}

constexpr int kMaxRun = 256;  // groups of a run at most: one to a column of 256 threads and more

// A run of groups of one image per workgroup, its elements in registers: a thread
// stays with its column (VEC channels) and goes down the pixels.
template <int VEC, int V>
__global__ __launch_bounds__(1024) void norm_run_kernel(const NormArgs a) {
  typedef typename Vec<VEC>::type vec;
  __shared__ double2 red[1024];
  __shared__ Moments total[kMaxRun];
  __shared__ Scale scale[kMaxRun];
  const int img = blockIdx.x / a.runs, g0 = (blockIdx.x - img * a.runs) * a.run;
  const int groups = min(a.run, a.groups - g0), cols_each = a.each / VEC, cols = groups * cols_each;
  const int row = threadIdx.x / a.cols, col = threadIdx.x - row * a.cols;
  const bool live = row < a.rows && col < cols;
  const int g = min(col / cols_each, groups - 1), c = g0 * a.each + min(col, cols - 1) * VEC;
  const float* x = a.x + (long long)img * a.t * a.ldx;
  float* y = a.y + (long long)img * a.t * a.ldy;
  vec v[V];
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = *(const vec*)(x + min(row + i * a.rows, a.t - 1) * a.ldx + c);
  const double p = (double)x[(g0 + g) * a.each];
  Moments m{0, 0};
  if (live)
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (row + i * a.rows < a.t)
#pragma unroll
        for (int e = 0; e < VEC; ++e) m.add(v[i][e], p);
  meet(a, m, red, cols_each, a.cols, groups, total);
  if (live && row == 0 && col % cols_each == 0) scale[g] = scale_of(a, total[g], p, (double)a.t * a.each);
  __syncthreads();
  if (!live) return;
  const Scale s = scale[g];
  float ga[VEC], be[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    ga[e] = a.gamma ? a.gamma[c + e] : 1.f;
    be[e] = a.beta ? a.beta[c + e] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (row + i * a.rows >= a.t) break;
    vec o;
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[e] = normal(a, v[i][e], s, ga[e], be[e]);
    *(vec*)(y + (row + i * a.rows) * a.ldy + c) = o;
  }
}

// Larger images: the moments of a piece of the pixels and a run of groups, then
// every piece normalised by the moments of all.
template <int VEC>
__global__ __launch_bounds__(256) void norm_sums_kernel(const NormArgs a) {
  typedef typename Vec<VEC>::type vec;
  __shared__ double2 red[256];
  __shared__ Moments total[kMaxRun];
  const int piece = blockIdx.x % a.pieces, rest = blockIdx.x / a.pieces, img = rest / a.runs, run = rest - img * a.runs;
  const int g0 = run / a.blocks * a.run, first = run % a.blocks * a.cols;  // group, its column
  const int groups = min(a.run, a.groups - g0);
  const int cols_each = min(a.each / VEC - first, a.cols), cols = groups * cols_each;
  const int row = threadIdx.x / a.cols, col = threadIdx.x - row * a.cols;
  const bool live = row < a.rows && col < cols;
  const int g = min(col / cols_each, groups - 1), c = g0 * a.each + (first + min(col, cols - 1)) * VEC;
  const float* x = a.x + (long long)img * a.t * a.ldx;
  const int from = piece * a.piece, to = min(from + a.piece, a.t);
  const double p = (double)x[(g0 + g) * a.each];
  Moments m{0, 0};
  if (live) {
    int i = from + row;
    for (; i + 3 * a.rows < to; i += 4 * a.rows) {
      vec v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = *(const vec*)(x + (i + k * a.rows) * a.ldx + c);
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e) m.add(v[k][e], p);
    }
    for (; i < to; i += a.rows) {
      const vec v = *(const vec*)(x + i * a.ldx + c);
#pragma unroll
      for (int e = 0; e < VEC; ++e) m.add(v[e], p);
    }
  }
  meet(a, m, red, cols_each, a.cols, groups, total);
  for (int i = threadIdx.x; i < groups; i += 256)
    a.sums[(((long long)img * a.groups + g0 + i) * a.blocks + run % a.blocks) * a.pieces + piece] =
        make_double2(total[i].s, total[i].q);
}

template <int VEC>
__global__ __launch_bounds__(256) void norm_apply_kernel(const NormArgs a) {
  typedef typename Vec<VEC>::type vec;
  __shared__ Scale scale[kMaxRun];
  const int piece = blockIdx.x % a.pieces, rest = blockIdx.x / a.pieces, img = rest / a.runs, run = rest - img * a.runs;
  const int g0 = run / a.blocks * a.run, first = run % a.blocks * a.cols, lane = threadIdx.x & 63;
  const int groups = min(a.run, a.groups - g0);
  const int cols_each = min(a.each / VEC - first, a.cols), cols = groups * cols_each;
  const float* x = a.x + (long long)img * a.t * a.ldx;
  float* y = a.y + (long long)img * a.t * a.ldy;
  for (int g = threadIdx.x >> 6; g < groups; g += 4) {
    const int parts = a.blocks * a.pieces;
    const double2* sums = a.sums + ((long long)img * a.groups + g0 + g) * parts;
    Moments m{0, 0};
    for (int i = lane; i < parts; i += 64) {
      m.s += sums[i].x;
      m.q += sums[i].y;
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      m.s += shuffle_xor(m.s, off);
      m.q += shuffle_xor(m.q, off);
    }
    if (lane == 0) scale[g] = scale_of(a, m, (double)x[(g0 + g) * a.each], (double)a.t * a.each);
  }
  __syncthreads();
  const int row = threadIdx.x / a.cols, col = threadIdx.x - row * a.cols;
  if (row >= a.rows || col >= cols) return;
  const int c = g0 * a.each + (first + col) * VEC;
  const Scale s = scale[col / cols_each];
  float ga[VEC], be[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    ga[e] = a.gamma ? a.gamma[c + e] : 1.f;
    be[e] = a.beta ? a.beta[c + e] : 0.f;
  }
  const int from = piece * a.piece, to = min(from + a.piece, a.t);
  auto put = [&](int i, const vec& v) {
    vec o;
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[e] = normal(a, v[e], s, ga[e], be[e]);
    __builtin_nontemporal_store(o, (vec*)(y + i * a.ldy + c));
  };
  int i = from + row;
  for (; i + 3 * a.rows < to; i += 4 * a.rows) {
    vec v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = *(const vec*)(x + (i + k * a.rows) * a.ldx + c);
#pragma unroll
    for (int k = 0; k < 4; ++k) put(i + k * a.rows, v[k]);
  }
  for (; i < to; i += a.rows) put(i, *(const vec*)(x + i * a.ldx + c));
}

// Elements of a group that 64 lanes hold: kRowsVec vectors each.
constexpr int kRowsVec = 16;

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
  const bool quads = a.each % 4 == 0 && a.ldx % 4 == 0 && a.ldy % 4 == 0 &&
                     (((uintptr_t)x->data | (uintptr_t)y->data) & 15) == 0;
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
      v <= 1 ? launch(norm_rows_kernel<4, 1>) : v <= 4 ? launch(norm_rows_kernel<4, 4>) : launch(norm_rows_kernel<4, kRowsVec>);
    else
      v <= 4 ? launch(norm_rows_kernel<1, 4>) : launch(norm_rows_kernel<1, kRowsVec>);
    return check_launch("group_norm");
  }
  // A run of groups: 128 bytes of a pixel and more.
  const int each = a.each / vec;
  auto columns = [&](int threads) {
    a.run = std::min({groups, std::max(1, threads / each), std::max(1, (32 / vec + each - 1) / each)});
    a.cols = std::min(a.run * each, threads);
    a.rows = threads / a.cols;
    a.blocks = (each + threads - 1) / threads;
    a.runs = a.blocks > 1 ? groups * a.blocks : (groups + a.run - 1) / a.run;
    return (a.t + a.rows - 1) / a.rows;  // pixels of a thread
  };
  const int most = quads ? 16 : 64;  // vectors that a thread holds
  if (each <= 1024 && columns(1024) <= most) {
    int threads = 256;
    while (threads < 1024 && (each > threads || columns(threads) > (a.n * (long long)a.runs < 512 ? most / 4 : most)))
      threads *= 2;
    const int v = columns(threads);
    const long long grid = (long long)a.n * a.runs;
    SY_CHECK(grid * threads < (1LL << 32), SY_EUNSUPPORTED, "group norm over %d images of %d groups", a.n, groups);
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(threads), 0, ctx->stream, a);
    };
    if (quads)
      v <= 4 ? launch(norm_run_kernel<4, 4>) : launch(norm_run_kernel<4, 16>);
    else
      v <= 16 ? launch(norm_run_kernel<1, 16>) : launch(norm_run_kernel<1, 64>);
    return check_launch("group_norm");
  }
  (void)columns(256);
  // Pieces: a few workgroups to a CU, but 16 pixels of a thread and more.
  const long long runs = (long long)a.n * a.runs;
  a.piece = (int)std::max<long long>(16 * a.rows, (a.t * runs + 2047) / 2048);
  a.pieces = (a.t + a.piece - 1) / a.piece;
  const long long grid = runs * a.pieces;
  SY_CHECK(grid * 256 < (1LL << 32), SY_EUNSUPPORTED, "group norm over %d images of %d groups", a.n, groups);
  SY_TRY(ensure_scratch(ctx, sizeof(double2) * (size_t)a.n * groups * a.blocks * a.pieces));
  a.sums = (double2*)ctx->scratch;
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(256), 0, ctx->stream, a); };
  launch(quads ? norm_sums_kernel<4> : norm_sums_kernel<1>);
  launch(quads ? norm_apply_kernel<4> : norm_apply_kernel<1>);
  return check_launch("group_norm");
}

}  // namespace sy

extern "C" int sy_group_norm(sy_ctx* ctx, const sy_tensor* x, int groups, const float* gamma, const float* beta,
                             float eps, int act, const sy_tensor* y) {
  return sy::op_group_norm(ctx, x, groups, gamma, beta, eps, act, y);
}
