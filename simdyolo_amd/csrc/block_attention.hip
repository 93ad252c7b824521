// Attention over the key blocks chosen for each query.
#include <cfloat>
#include <cmath>

#include "sy_internal.h"

namespace sy {

struct BlockArgs {
  const float *q, *k, *v;
  float* o;
  const int *blocks, *starts, *lengths;
  long long ldq, ldk, ldv, ldo;
  BlockShape s;
};

// Keys of image b that query i sees: those before this position.
__device__ __forceinline__ int visible(const BlockArgs& a, int b, int i) {
  int end = a.lengths ? min(max(a.lengths[b], 0), a.s.tk) : a.s.tk;
  if (a.s.causal) {
    const long long at = (long long)(a.starts ? a.starts[b] : 0) + i;
    end = (int)min((long long)end, max(at + 1, 0LL));
  }
  return end;
}

// One wave per query and head, in plain float32; a lane scores one key of 64 and holds two channels.
__global__ __launch_bounds__(64) void block_attention_kernel(const BlockArgs a) {
  const BlockShape& s = a.s;
  const int lane = threadIdx.x;
  const long long row = blockIdx.x;
  const int h = (int)(row % s.heads), i = (int)(row / s.heads % s.tq), b = (int)(row / s.heads / s.tq);
  const int g = h / s.group, end = visible(a, b, i);
  const float* q = a.q + ((long long)b * s.tq + i) * a.ldq + (long long)h * s.qs;
  const float* kb = a.k + (long long)b * s.tk * a.ldk + (long long)g * s.ks;
  const float* vb = a.v + (long long)b * s.tk * a.ldv + (long long)g * s.vs;
  const int* list = a.blocks + (((long long)b * s.tq + i) * s.kv + g) * s.selected;
  float mx = -INFINITY, sum = 0.f, acc[2] = {0.f, 0.f};
  bool any = false;
  for (int n = 0; n < s.selected; ++n) {
    const int j = list[n];
    if (j < 0 || j >= s.blocks) continue;
    const int y0 = j / s.bx * s.bh, x0 = j % s.bx * s.bw;
    const int cols = min(s.bw, s.kw - x0), keys = min(s.bh, s.kh - y0) * cols;
    for (int t0 = 0; t0 < keys; t0 += 64) {
      const int t = t0 + lane, at = (y0 + t / cols) * s.kw + x0 + t % cols;
      const bool on = t < keys && at < end;
      float x = 0.f;
      if (on)
        for (int c = 0; c < s.kd; ++c) x = __builtin_fmaf(q[c], kb[at * a.ldk + c], x);
      x = on ? x * s.scale : -INFINITY;
      if (!__any(on)) continue;
      any = true;
      float top = x;
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
      top = fmaxf(top, mx);
      if (top == -INFINITY && !__any(x != x)) continue;  // weighs nothing beside a finite score
      const float e = on ? expf(x - top) : 0.f;
      float es = e;
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) es += __shfl_xor(es, off);
      const float f = mx == -INFINITY ? 0.f : expf(mx - top);
      mx = top;
      sum = sum * f + es;
      acc[0] *= f;
      acc[1] *= f;
      for (int u = 0; u < min(64, keys - t0); ++u) {
        const float w = __shfl(e, u);
        const int from = __shfl(at, u);
        if (!__shfl((int)on, u)) continue;
#pragma unroll
        for (int d = 0; d < 2; ++d)
          if (lane + 64 * d < s.hd) acc[d] = __builtin_fmaf(w, vb[from * a.ldv + lane + 64 * d], acc[d]);
      }
    }
  }
  float* o = a.o + ((long long)b * s.tq + i) * a.ldo + (long long)h * s.hd;
#pragma unroll
  for (int d = 0; d < 2; ++d)
    if (lane + 64 * d < s.hd) o[lane + 64 * d] = any ? acc[d] / sum : 0.f;
}

int op_block_attention(sy_ctx* ctx, const sy_block_config* cfg, const sy_tensor* q, const sy_tensor* k,
                       const sy_tensor* v, const int32_t* blocks, const int32_t* starts, const int32_t* lengths,
                       const sy_tensor* o) {
  BlockArgs a{};
  BlockShape& s = a.s;
  SY_TRY(block_shape(cfg, &s));
  SY_TRY(block_heads(q, s.heads, s.kd, s.qs, "block queries"));
  SY_TRY(block_heads(k, s.kv, s.kd, s.ks, "block keys"));
  SY_TRY(block_heads(v, s.kv, s.hd, s.vs, "block values"));
  SY_TRY(block_heads(o, s.heads, s.hd, s.hd, "block attention output"));
  SY_CHECK(blocks, SY_EINVAL, "null blocks");
  SY_CHECK(o->c == s.heads * s.hd && o->n == q->n && o->h == q->h && o->w == q->w, SY_EINVAL,
           "block attention output shape mismatch");
  SY_CHECK(k->n == q->n && v->n == q->n && v->h == k->h && v->w == k->w, SY_EINVAL,
           "block queries, keys and values differ in n, h or w");
  SY_CHECK((k->h == 1 && s.bh == 1) || (!lengths && !s.causal), SY_EINVAL,
           "lengths and causal need keys and blocks one pixel high");
  SY_CHECK(!views_overlap(o, q) && !views_overlap(o, k) && !views_overlap(o, v), SY_EINVAL,
           "block attention output overlaps an input");
  SY_CHECK(ctx, SY_EINVAL, "null context");
  s.n = q->n;
  s.tq = q->h * q->w;
  s.tk = k->h * k->w;
  s.kh = k->h;
  s.kw = k->w;
  s.by = (k->h + s.bh - 1) / s.bh;
  s.bx = (k->w + s.bw - 1) / s.bw;
  s.blocks = s.by * s.bx;
  a.q = q->data;
  a.k = k->data;
  a.v = v->data;
  a.o = o->data;
  a.blocks = blocks;
  a.starts = starts;
  a.lengths = lengths;
  a.ldq = q->ldc;
  a.ldk = k->ldc;
  a.ldv = v->ldc;
  a.ldo = o->ldc;
  const long long rows = (long long)s.n * s.tq * s.heads;
  SY_CHECK(rows * 64 < (1LL << 32), SY_EUNSUPPORTED, "block attention grid too large");
  DeviceScope device(ctx);
  const double keys = std::min((double)s.selected * s.bh * s.bw, (double)s.tk);
  ProfScope prof(ctx, "block_attention", 2.0 * rows * keys * (s.kd + s.hd),
                 4.0 * s.n * ((double)s.tq * s.heads * (s.kd + s.hd) + (double)s.tk * s.kv * (s.kd + s.hd)));
  hipLaunchKernelGGL(block_attention_kernel, dim3((unsigned)rows), dim3(64), 0, ctx->stream, a);
  return check_launch("block_attention");
}

}  // namespace sy

extern "C" int sy_block_attention(sy_ctx* ctx, const sy_block_config* cfg, const sy_tensor* q, const sy_tensor* k,
                                  const sy_tensor* v, const int32_t* blocks, const int32_t* starts,
                                  const int32_t* lengths, const sy_tensor* o) {
  return sy::op_block_attention(ctx, cfg, q, k, v, blocks, starts, lengths, o);
}
