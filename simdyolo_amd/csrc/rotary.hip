// Rotary positions (Su et al., 2021): channels of every query and key head in pairs (a, b), each turned
// by the token's position times the pair's frequency, y = (a c - b s, b c + a s).
#include <cmath>
#include <new>

#include "sy_internal.h"

namespace sy {

typedef float f32x4 __attribute__((ext_vector_type(4)));

struct RotaryPart {
  const float* x;
  float* y;
  long long ldx, ldy;
  int heads, xs, ys;
  int same;  // in place: channels that are not rotated stay
};

struct RotaryArgs {
  RotaryPart part[2];
  const int* positions;
  long long tokens;  // of all images
  int parts, per, width, tile;  // tokens of an image and of its rows; of a workgroup
  int head_dim, dim, axes, half;
  float amplitude;
  double turns[kRotaryMaxDim / 2];
};

// Cosine and sine of t turns.  The quarter turns come off in 64 bits, so that the rest, at most 1/8 turn, carries 24 bits
// as long as t, a product of 64 bits, does: up to 2^25 turns (positions up to 2^27 at frequency 1).  At positions of 2^31
// the product is within 2^-23 of a turn.
__device__ __forceinline__ float2 turn(double t) {
  t -= rint(t);
  const double quarters = rint(t * 4.0);
  const float r = (float)(t * 4.0 - quarters);
  float s, c;
  sincospif(0.5f * r, &s, &c);
  const int q = (int)quarters & 3;
  const float x = q & 1 ? s : c, y = q & 1 ? c : s;
  return make_float2(q == 1 || q == 2 ? -x : x, q & 2 ? -y : y);
}

enum { kHalves4 = 0, kInterleaved = 1, kHalves1 = 2 };

// `tile` tokens per workgroup: their cosines and sines into LDS once, then every head of queries and keys.  Bound by
// memory: 32,768 tokens of 40 heads of 128 channels (1.34 GB) in 264 us, 5.1 TB/s, the rate of a large copy; q and k of
// eight 80x80 maps out of their qkv tensor (105 MB) 18 - 21 us.  A second sine for every head would cost as much as the
// memory; 64-bit arithmetic is one product and two roundings for each pair and token.
// Interleaved pairs are two to a 16-byte unit.  With the halves of an axis apart, a unit is four channels
// of either half, or one where a half is not a multiple of four.
template <int LAYOUT>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs a) {
  extern __shared__ float2 table[];  // [tile][dim / 2]
  const long long first = (long long)blockIdx.x * a.tile;
  const int count = (int)min((long long)a.tile, a.tokens - first), pairs = a.dim / 2;
  for (int i = threadIdx.x; i < count * pairs; i += 256) {
    const int t = i / pairs, p = i - t * pairs, axis = p / a.half;
    const long long token = first + t;
    int at;
    if (a.positions) {
      at = a.positions[token * a.axes + axis];
    } else {
      const int pixel = (int)(token % a.per);
      at = a.axes == 1 ? pixel : axis == 0 ? pixel / a.width : pixel % a.width;
    }
    const float2 cs = turn(at * a.turns[p - axis * a.half]);
    table[i] = make_float2(cs.x * a.amplitude, cs.y * a.amplitude);
  }
  __syncthreads();
  const int rotated = LAYOUT == kHalves4 ? a.dim / 8 : LAYOUT == kInterleaved ? (a.dim + 3) / 4 : pairs;
  const int whole = LAYOUT == kHalves4       ? rotated + (a.head_dim - a.dim) / 4
                    : LAYOUT == kInterleaved ? a.head_dim / 4
                                             : rotated + a.head_dim - a.dim;
  for (int part = 0; part < a.parts; ++part) {
    const RotaryPart& p = a.part[part];
    const int units = p.same ? rotated : whole, row = p.heads * units;
    for (int i = threadIdx.x; i < count * row; i += 256) {
      const int t = i / row, rest = i - t * row, head = rest / units, u = rest - head * units;
      const float* x = p.x + (first + t) * p.ldx + head * p.xs;
      float* y = p.y + (first + t) * p.ldy + head * p.ys;
      const float2* cs = table + t * pairs;
      if (LAYOUT == kInterleaved) {
        const f32x4 v = *(const f32x4*)(x + 4 * u);
        f32x4 o = v;
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (2 * u + e < pairs) {
            const float2 w = cs[2 * u + e];
            o[2 * e] = v[2 * e] * w.x - v[2 * e + 1] * w.y;
            o[2 * e + 1] = v[2 * e + 1] * w.x + v[2 * e] * w.y;
          }
        *(f32x4*)(y + 4 * u) = o;
      } else if (LAYOUT == kHalves4) {
        if (u >= rotated) {
          const int c = a.dim + 4 * (u - rotated);
          *(f32x4*)(y + c) = *(const f32x4*)(x + c);
          continue;
        }
        const int axis = 4 * u / a.half, c = 4 * u + axis * a.half;
        const f32x4 v0 = *(const f32x4*)(x + c), v1 = *(const f32x4*)(x + c + a.half);
        f32x4 o0, o1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 w = cs[4 * u + e];
          o0[e] = v0[e] * w.x - v1[e] * w.y;
          o1[e] = v1[e] * w.x + v0[e] * w.y;
        }
        *(f32x4*)(y + c) = o0;
        *(f32x4*)(y + c + a.half) = o1;
      } else {
        if (u >= rotated) {
          const int c = a.dim + u - rotated;
          y[c] = x[c];
          continue;
        }
        const int axis = u / a.half, c = u + axis * a.half;
        const float v0 = x[c], v1 = x[c + a.half];
        const float2 w = cs[u];
        y[c] = v0 * w.x - v1 * w.y;
        y[c + a.half] = v1 * w.x + v0 * w.y;
      }
    }
  }
}

// Whether heads of `dim` channels in two views may share memory: views_overlap, but for heads of one
// buffer that lie between each other (q and k of a qkv tensor).
static bool heads_overlap(const sy_tensor* a, int as, int ah, const sy_tensor* b, int bs, int bh, int dim) {
  if (!views_overlap(a, b)) return false;
  if (a->ldc != b->ldc || as != bs || a->n != b->n || a->h != b->h || a->w != b->w) return true;
  long long d = ((long long)(uintptr_t)b->data - (long long)(uintptr_t)a->data) / (long long)sizeof(float);
  int last = bh;
  if (d < 0) {
    d = -d;
    last = ah;
  }
  return !(d >= dim && d + dim <= as && (long long)(last - 1) * as + d + dim <= a->ldc);
}

int op_rotary_create(sy_ctx* ctx, const sy_rotary_config* c, uint64_t* rotary) {
  SY_CHECK(c && rotary, SY_EINVAL, "null argument");
  SY_CHECK(c->axes == 1 || c->axes == 2, SY_EINVAL, "rotary positions have 1 or 2 axes, not %d", c->axes);
  SY_CHECK(c->head_dim > 0 && c->dim > 0 && c->dim <= c->head_dim, SY_EINVAL, "rotary dim %d of head dim %d", c->dim,
           c->head_dim);
  SY_CHECK(c->dim % (2 * c->axes) == 0, SY_EINVAL, "rotary dim %d is not a multiple of twice its %d axes", c->dim,
           c->axes);
  SY_CHECK(c->head_dim % 4 == 0 && c->head_dim <= kRotaryMaxDim, SY_EUNSUPPORTED,
           "rotary needs a head dim that is a multiple of 4 up to %d", kRotaryMaxDim);
  SY_CHECK(c->interleaved == 0 || c->interleaved == 1, SY_EINVAL, "rotary interleaved is 0 or 1");
  SY_CHECK(std::isfinite(c->base) && c->base > 0, SY_EINVAL, "rotary base must be positive and finite");
  SY_CHECK(c->scaling >= SY_ROTARY_PLAIN && c->scaling <= SY_ROTARY_PARTS, SY_EINVAL, "unknown rotary scaling %d",
           c->scaling);
  const int part = c->dim / c->axes;
  if (c->scaling != SY_ROTARY_PLAIN)
    SY_CHECK(std::isfinite(c->factor) && c->factor >= 1, SY_EINVAL, "rotary scaling factor must be 1 or more");
  if (c->scaling == SY_ROTARY_BASE)
    SY_CHECK(part > 2, SY_EINVAL, "rotary base scaling needs more than one pair per axis");
  if (c->scaling == SY_ROTARY_PARTS)
    SY_CHECK(c->original > 0 && std::isfinite(c->low) && std::isfinite(c->high) && c->low >= 0 && c->high > c->low,
             SY_EINVAL, "rotary scaling by parts needs original > 0 and 0 <= low < high");
  SY_CHECK(ctx, SY_EINVAL, "null context");
  std::unique_ptr<RotaryPlan> p(new (std::nothrow) RotaryPlan);
  SY_CHECK(p, SY_ENOMEM, "no memory for a rotary plan");
  p->cfg = *c;
  p->half = part / 2;
  p->amplitude = 1.f;
  const double pi2 = 6.283185307179586476925, factor = c->factor;
  double base = c->base;
  if (c->scaling == SY_ROTARY_BASE) base *= std::pow(factor, part / (part - 2.0));
  if (c->scaling == SY_ROTARY_PARTS) p->amplitude = (float)(0.1 * std::log(factor) + 1.0);
  for (int i = 0; i < p->half; ++i) {
    double f = std::pow(base, -2.0 * i / part);
    if (c->scaling == SY_ROTARY_LINEAR) f /= factor;
    if (c->scaling == SY_ROTARY_PARTS) {
      const double turns = c->original * f / pi2;
      const double keep = std::fmin(1.0, std::fmax(0.0, (turns - c->low) / ((double)c->high - c->low)));
      f *= keep + (1.0 - keep) / factor;
    }
    p->turns[i] = f / pi2;
  }
  try {
    ctx->rotaries.push_back(std::move(p));
  } catch (const std::bad_alloc&) {
    SY_CHECK(false, SY_ENOMEM, "no memory for a rotary plan");
  }
  *rotary = ctx->rotaries.size();
  return SY_OK;
}

int op_rotary_run(sy_ctx* ctx, uint64_t rotary, const sy_rotary_heads* parts, int n_parts, const int32_t* positions) {
  SY_CHECK(rotary > 0 && rotary <= ctx->rotaries.size(), SY_EINVAL, "unknown rotary handle %llu",
           (unsigned long long)rotary);
  SY_CHECK(parts && (n_parts == 1 || n_parts == 2), SY_EINVAL, "rotary takes one or two sets of heads");
  const RotaryPlan& p = *ctx->rotaries[rotary - 1];
  RotaryArgs a{};
  double values = 0;
  for (int i = 0; i < n_parts; ++i) {
    const sy_rotary_heads& h = parts[i];
    SY_TRY(check_view(&h.x, "rotary input"));
    SY_TRY(check_view(&h.y, "rotary output"));
    SY_CHECK(h.heads > 0, SY_EINVAL, "rotary needs a head");
    SY_CHECK((long long)h.heads * p.cfg.head_dim < (1LL << 27), SY_EUNSUPPORTED, "rotary over %d heads", h.heads);
    const int xs = h.x_stride ? h.x_stride : p.cfg.head_dim, ys = h.y_stride ? h.y_stride : p.cfg.head_dim;
    for (const auto& v : {std::make_pair(&h.x, xs), std::make_pair(&h.y, ys)}) {
      SY_CHECK(v.second >= p.cfg.head_dim && v.second % 4 == 0, SY_EINVAL, "rotary head stride %d", v.second);
      SY_CHECK((long long)(h.heads - 1) * v.second + p.cfg.head_dim <= v.first->c, SY_EINVAL,
               "rotary view has %d channels for %d heads of %d, %d apart", v.first->c, h.heads, p.cfg.head_dim,
               v.second);
      SY_CHECK(((uintptr_t)v.first->data & 15) == 0 && v.first->ldc % 4 == 0, SY_EINVAL,
               "rotary views must be 16-byte aligned with ldc %% 4 == 0");
    }
    SY_CHECK(h.x.n == parts[0].x.n && h.x.h == parts[0].x.h && h.x.w == parts[0].x.w && h.y.n == h.x.n &&
                 h.y.h == h.x.h && h.y.w == h.x.w,
             SY_EINVAL, "rotary views differ in n, h or w");
    const bool same = h.x.data == h.y.data && h.x.ldc == h.y.ldc && xs == ys;
    SY_CHECK(same || !heads_overlap(&h.x, xs, h.heads, &h.y, ys, h.heads, p.cfg.head_dim), SY_EINVAL,
             "rotary output overlaps its input other than in place");
    a.part[i] = {h.x.data, h.y.data, h.x.ldc, h.y.ldc, h.heads, xs, ys, same};
    values += (double)h.heads * (same ? p.cfg.dim : p.cfg.head_dim);
  }
  if (n_parts == 2) {
    const sy_rotary_heads *u = &parts[0], *v = &parts[1];
    const int d = p.cfg.head_dim;
    SY_CHECK(!heads_overlap(&u->y, a.part[0].ys, u->heads, &v->x, a.part[1].xs, v->heads, d) &&
                 !heads_overlap(&u->x, a.part[0].xs, u->heads, &v->y, a.part[1].ys, v->heads, d) &&
                 !heads_overlap(&u->y, a.part[0].ys, u->heads, &v->y, a.part[1].ys, v->heads, d),
             SY_EINVAL, "rotary output overlaps another set of heads");
  }
  const sy_tensor& x = parts[0].x;
  const long long per = (long long)x.h * x.w;
  SY_CHECK(per < (1LL << 31), SY_EUNSUPPORTED, "rotary over 2^31 tokens and more");
  a.positions = positions;
  a.tokens = x.n * per;
  a.parts = n_parts;
  a.per = (int)per;
  a.width = x.w;
  a.head_dim = p.cfg.head_dim;
  a.dim = p.cfg.dim;
  a.axes = p.cfg.axes;
  a.half = p.half;
  a.amplitude = p.amplitude;
  for (int i = 0; i < p.half; ++i) a.turns[i] = p.turns[i];
  a.tile = 8;  // tokens: fewer where the chip would not be full (one token for each of 32 sequences: 5.0 us)
  while (a.tile > 1 && a.tokens / a.tile < 2048) a.tile /= 2;
  const long long grid = (a.tokens + a.tile - 1) / a.tile;
  SY_CHECK(grid * 256 < (1LL << 32), SY_EUNSUPPORTED, "rotary grid too large");
  DeviceScope device(ctx);
  const size_t lds = sizeof(float2) * a.tile * (a.dim / 2);
  ProfScope prof(ctx, "rotary", 3.0 * a.tokens * values * a.dim / a.head_dim, 8.0 * a.tokens * values);
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(256), lds, ctx->stream, a);
  };
  if (p.cfg.interleaved)
    launch(rotary_kernel<kInterleaved>);
  else if (p.half % 4 == 0)
    launch(rotary_kernel<kHalves4>);
  else
    launch(rotary_kernel<kHalves1>);
  return check_launch("rotary");
}

}  // namespace sy

extern "C" {

int sy_rotary_create(sy_ctx* ctx, const sy_rotary_config* cfg, uint64_t* rotary) {
  return sy::op_rotary_create(ctx, cfg, rotary);
}

int sy_rotary_run(sy_ctx* ctx, uint64_t rotary, const sy_rotary_heads* parts, int n_parts, const int32_t* positions) {
  SY_CHECK(ctx, SY_EINVAL, "null context");
  return sy::op_rotary_run(ctx, rotary, parts, n_parts, positions);
}

}  // extern "C"
