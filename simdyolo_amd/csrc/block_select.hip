// Which key blocks each query attends to: mean keys of the blocks, and for every query the blocks whose
// mean has the largest product with it.
//
// The choice is made on scores in 64 bits: a product of floats is exact there and 128 of them sum within
// 2^-46, so it does not hang on the order of a sum as it would in 32 bits.
#include <cfloat>
#include <cmath>

#include "sy_internal.h"

namespace sy {

typedef float f32x4 __attribute__((ext_vector_type(4)));

// The config alone; the views' part is filled in by the callers.
int block_shape(const sy_block_config* c, BlockShape* s) {
  SY_CHECK(c, SY_EINVAL, "null block config");
  SY_CHECK(c->heads > 0 && c->kv_heads > 0 && c->heads % c->kv_heads == 0, SY_EINVAL,
           "%d heads do not share %d key heads", c->heads, c->kv_heads);
  SY_CHECK(c->key_dim > 0 && c->head_dim > 0, SY_EINVAL, "block attention dims %d, %d", c->key_dim, c->head_dim);
  SY_CHECK(c->key_dim % 4 == 0 && c->head_dim % 4 == 0 && c->key_dim <= 128 && c->head_dim <= 128, SY_EUNSUPPORTED,
           "block attention needs key/head dims that are multiples of 4 up to 128");
  SY_CHECK(c->block_h > 0 && c->block_w > 0, SY_EINVAL, "block of %dx%d keys", c->block_h, c->block_w);
  SY_CHECK((long long)c->block_h * c->block_w <= 1024, SY_EUNSUPPORTED, "blocks hold up to 1024 keys, not %dx%d",
           c->block_h, c->block_w);
  SY_CHECK(c->selected > 0, SY_EINVAL, "%d selected blocks", c->selected);
  SY_CHECK(c->selected <= 64, SY_EUNSUPPORTED, "up to 64 selected blocks, not %d", c->selected);
  SY_CHECK(c->causal == 0 || c->causal == 1, SY_EINVAL, "causal is 0 or 1");
  SY_CHECK(!c->causal || c->block_h == 1, SY_EINVAL, "causal blocks are one pixel high");
  SY_CHECK(std::isfinite(c->scale) && c->scale > 0, SY_EINVAL, "scale must be positive and finite");
  s->heads = c->heads;
  s->kv = c->kv_heads;
  s->group = c->heads / c->kv_heads;
  s->kd = c->key_dim;
  s->hd = c->head_dim;
  s->qs = c->q_stride ? c->q_stride : c->key_dim;
  s->ks = c->k_stride ? c->k_stride : c->key_dim;
  s->vs = c->v_stride ? c->v_stride : c->head_dim;
  s->bh = c->block_h;
  s->bw = c->block_w;
  s->selected = c->selected;
  s->causal = c->causal;
  s->scale = c->scale;
  return SY_OK;
}

// A view that holds `heads` heads of `dim` channels, `stride` apart, read 16 bytes at a time.
int block_heads(const sy_tensor* t, int heads, int dim, int stride, const char* what) {
  SY_TRY(check_view(t, what));
  SY_CHECK(stride >= dim && stride % 4 == 0, SY_EINVAL, "%s: head stride %d", what, stride);
  SY_CHECK((long long)(heads - 1) * stride + dim <= t->c, SY_EINVAL, "%s: %d channels for %d heads of %d, %d apart",
           what, t->c, heads, dim, stride);
  SY_CHECK(((uintptr_t)t->data & 15) == 0 && t->ldc % 4 == 0, SY_EINVAL,
           "%s must be 16-byte aligned with ldc %% 4 == 0", what);
  SY_CHECK((long long)t->h * t->w < (1LL << 30), SY_EUNSUPPORTED, "%s: 2^30 tokens and more", what);
  return SY_OK;
}

// --------------------------------------------------------------------- means

struct MeansArgs {
  const float* k;
  float* m;
  const int *starts, *lengths;
  long long ldk, ldm;
  int tk, kh, kw, bh, bw, bx, blocks, ks, kd, units, lanes, tokens, slots;
};

// One workgroup per block (with `tokens`: per block that may hold some) and image.  A lane sums four
// channels over every (256 / lanes)-th key; the partial sums meet in LDS in one order.
__global__ __launch_bounds__(256) void means_kernel(const MeansArgs a) {
  __shared__ double part[256][4];
  const int b = blockIdx.x / a.slots, slot = blockIdx.x % a.slots;
  const int length = a.lengths ? min(max(a.lengths[b], 0), a.tk) : a.tk;
  int j = slot;
  if (a.tokens) {
    const long long from = a.starts ? a.starts[b] : 0, to = from + a.tokens - 1;
    if (to < 0) return;
    const long long first = max(from, 0LL) / a.bw;
    if (first + slot > to / a.bw || first + slot >= a.blocks) return;
    j = (int)first + slot;
  }
  const int y0 = j / a.bx * a.bh, x0 = j % a.bx * a.bw;
  const int rows = min(a.bh, a.kh - y0), cols = min(a.bw, a.kw - x0);
  const int keys = rows == 1 ? max(min(cols, length - (y0 * a.kw + x0)), 0) : rows * cols;
  const int lane = threadIdx.x % a.lanes, group = threadIdx.x / a.lanes, groups = 256 / a.lanes;
  const double inv = keys ? 1.0 / keys : 0.0;
  for (int u0 = 0; u0 < a.units; u0 += a.lanes) {
    const int u = u0 + lane, head = 4 * u / a.kd;
    double s[4] = {0, 0, 0, 0};
    if (u < a.units) {
      const float* kb = a.k + (long long)b * a.tk * a.ldk + head * a.ks + (4 * u - head * a.kd);
      for (int t = group; t < keys; t += groups) {
        const long long row = (long long)(y0 + t / cols) * a.kw + x0 + t % cols;
        const f32x4 v = *(const f32x4*)(kb + row * a.ldk);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += v[e];
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) part[threadIdx.x][e] = s[e];
    __syncthreads();
    if (group == 0 && u < a.units) {
      for (int g = 1; g < groups; ++g)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += part[g * a.lanes + lane][e];
      f32x4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = (float)(s[e] * inv);
      *(f32x4*)(a.m + ((long long)b * a.blocks + j) * a.ldm + 4 * u) = o;
    }
    __syncthreads();
  }
}

static int means_view(const BlockShape& s, const sy_tensor* m) {
  SY_TRY(check_view(m, "block means"));
  SY_CHECK(m->c == s.kv * s.kd, SY_EINVAL, "block means have %d channels, expected kv_heads * key_dim = %d", m->c,
           s.kv * s.kd);
  SY_CHECK(((uintptr_t)m->data & 15) == 0 && m->ldc % 4 == 0, SY_EINVAL,
           "block means must be 16-byte aligned with ldc %% 4 == 0");
  SY_CHECK((long long)m->h * m->w < (1LL << 24), SY_EUNSUPPORTED, "2^24 blocks and more");
  return SY_OK;
}

int op_block_means(sy_ctx* ctx, const sy_block_config* cfg, const sy_tensor* k, const int32_t* starts, int tokens,
                   const int32_t* lengths, const sy_tensor* m) {
  BlockShape s{};
  SY_TRY(block_shape(cfg, &s));
  SY_TRY(block_heads(k, s.kv, s.kd, s.ks, "block keys"));
  SY_TRY(means_view(s, m));
  const long long by = (k->h + (long long)s.bh - 1) / s.bh, bx = (k->w + (long long)s.bw - 1) / s.bw;
  SY_CHECK(m->n == k->n && m->h == by && m->w == bx, SY_EINVAL, "block means are %dx%dx%d, expected %dx%lldx%lld",
           m->n, m->h, m->w, k->n, by, bx);
  SY_CHECK(tokens >= 0, SY_EINVAL, "%d tokens", tokens);
  SY_CHECK((k->h == 1 && s.bh == 1) || (!lengths && !tokens && !s.causal), SY_EINVAL,
           "lengths, tokens and causal need keys and blocks one pixel high");
  SY_CHECK(!views_overlap(k, m), SY_EINVAL, "block means overlap the keys");
  SY_CHECK(ctx, SY_EINVAL, "null context");
  MeansArgs a{};
  a.k = k->data;
  a.m = m->data;
  a.starts = starts;
  a.lengths = lengths;
  a.ldk = k->ldc;
  a.ldm = m->ldc;
  a.tk = k->h * k->w;
  a.kh = k->h;
  a.kw = k->w;
  a.bh = s.bh;
  a.bw = s.bw;
  a.bx = (int)bx;
  a.blocks = (int)(by * bx);
  a.ks = s.ks;
  a.kd = s.kd;
  a.units = s.kv * s.kd / 4;
  a.lanes = 1;
  while (a.lanes < a.units && a.lanes < 256) a.lanes *= 2;
  a.tokens = tokens;
  a.slots = tokens ? (int)std::min<long long>(a.blocks, (tokens - 1LL) / s.bw + 2) : a.blocks;
  const long long grid = (long long)k->n * a.slots;
  SY_CHECK(grid * 256 < (1LL << 32), SY_EUNSUPPORTED, "block means grid too large");
  DeviceScope device(ctx);
  const double read = tokens ? (double)a.slots * s.bw : (double)a.tk;
  ProfScope prof(ctx, "block_means", (double)k->n * read * s.kv * s.kd,
                 4.0 * k->n * s.kv * s.kd * (std::min(read, (double)a.tk) + a.slots));
  hipLaunchKernelGGL(means_kernel, dim3((unsigned)grid), dim3(256), 0, ctx->stream, a);
  return check_launch("block_means");
}

// ----------------------------------------------------------------- selection

struct SelectArgs {
  const float *q, *m;
  const int *starts, *lengths;
  int* out;
  long long ldq, ldm, rows;
  int tq, blocks, bw, kv, group, kd, qs, selected, causal;
};

// 64-bit scores in an order of integers: NaN below every number, zeros alike.
__device__ __forceinline__ long long score_key(double s) {
  if (s != s) return LLONG_MIN + 1;
  const long long b = __builtin_bit_cast(long long, s + 0.0);
  return b < 0 ? LLONG_MIN + 2 + ~b : b;
}

constexpr int kSelectChunk = 1024;
constexpr long long kHidden = LLONG_MIN;

// One wave per query and key head.
__global__ __launch_bounds__(64) void select_kernel(const SelectArgs a) {
  __shared__ double qsum[128];
  __shared__ long long key[kSelectChunk + 64];
  __shared__ int id[64], best_id[64];
  __shared__ long long best_key[64];
  const int lane = threadIdx.x;
  const long long row = blockIdx.x;
  const int g = (int)(row % a.kv), i = (int)(row / a.kv % a.tq);
  const long long b = row / a.kv / a.tq;
  const float* q = a.q + (b * a.tq + i) * a.ldq + (long long)g * a.group * a.qs;
  for (int c = lane; c < a.kd; c += 64) {
    double s = 0;
    for (int h = 0; h < a.group; ++h) s += q[(long long)h * a.qs + c];
    qsum[c] = s;
  }
  long long seen = a.blocks, forced = -1;  // blocks seen; one that is always taken
  if (a.lengths) seen = min(seen, ((long long)max(a.lengths[b], 0) + a.bw - 1) / a.bw);
  if (a.causal) {
    const long long at = (long long)(a.starts ? a.starts[b] : 0) + i;
    seen = at < 0 ? 0 : min(seen, at / a.bw + 1);
    if (at >= 0 && at / a.bw < seen) forced = at / a.bw;
  }
  int kept = 0;
  __syncthreads();
  for (long long j0 = 0; j0 < seen; j0 += kSelectChunk) {
    const int count = (int)min((long long)kSelectChunk, seen - j0);
    for (int t = lane; t < count; t += 64) {
      const float* m = a.m + (b * a.blocks + j0 + t) * a.ldm + g * a.kd;
      double s = 0;
      for (int c = 0; c < a.kd; ++c) s = __builtin_fma(qsum[c], (double)m[c], s);
      key[kept + t] = j0 + t == forced ? LLONG_MAX : score_key(s);
    }
    if (lane < kept) {
      key[lane] = best_key[lane];
      id[lane] = best_id[lane];
    }
    __syncthreads();
    // Candidates in ascending order of blocks: the first largest is the one wanted.
    const int all = kept + count, want = min(a.selected, all);
    for (int n = 0; n < want; ++n) {
      long long top = kHidden;
      int at = 0x7fffffff;
      for (int t = lane; t < all; t += 64)
        if (key[t] > top) {
          top = key[t];
          at = t;
        }
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) {
        const long long ok = __shfl_xor(top, off);
        const int oa = __shfl_xor(at, off);
        if (ok > top || (ok == top && oa < at)) {
          top = ok;
          at = oa;
        }
      }
      __syncthreads();
      if (lane == 0) {
        best_key[n] = top;
        best_id[n] = at < kept ? id[at] : (int)(j0 + at - kept);
        key[at] = kHidden;
      }
      __syncthreads();
    }
    kept = want;
    // Ascending again.
    const int mine = lane < kept ? best_id[lane] : 0x7fffffff;
    const long long mykey = lane < kept ? best_key[lane] : 0;
    int place = 0;
    for (int t = 0; t < kept; ++t) place += best_id[t] < mine;
    __syncthreads();
    if (lane < kept) {
      best_id[place] = mine;
      best_key[place] = mykey;
    }
    __syncthreads();
  }
  if (lane < a.selected) a.out[row * a.selected + lane] = lane < kept ? best_id[lane] : -1;
}

int op_block_select(sy_ctx* ctx, const sy_block_config* cfg, const sy_tensor* q, const sy_tensor* m,
                    const int32_t* starts, const int32_t* lengths, int32_t* blocks) {
  BlockShape s{};
  SY_TRY(block_shape(cfg, &s));
  SY_TRY(block_heads(q, s.heads, s.kd, s.qs, "block queries"));
  SY_TRY(means_view(s, m));
  SY_CHECK(blocks, SY_EINVAL, "null blocks");
  SY_CHECK(m->n == q->n, SY_EINVAL, "%d images of queries, %d of block means", q->n, m->n);
  SY_CHECK((m->h == 1 && s.bh == 1) || (!lengths && !s.causal), SY_EINVAL,
           "lengths and causal need keys and blocks one pixel high");
  SY_CHECK(ctx, SY_EINVAL, "null context");
  SelectArgs a{};
  a.q = q->data;
  a.m = m->data;
  a.starts = starts;
  a.lengths = lengths;
  a.out = blocks;
  a.ldq = q->ldc;
  a.ldm = m->ldc;
  a.tq = q->h * q->w;
  a.blocks = m->h * m->w;
  a.bw = s.bw;
  a.kv = s.kv;
  a.group = s.group;
  a.kd = s.kd;
  a.qs = s.qs;
  a.selected = s.selected;
  a.causal = s.causal;
  a.rows = (long long)q->n * a.tq * s.kv;
  SY_CHECK(a.rows * 64 < (1LL << 32), SY_EUNSUPPORTED, "block select grid too large");
  DeviceScope device(ctx);
  ProfScope prof(ctx, "block_select", 2.0 * a.rows * a.blocks * s.kd,
                 4.0 * q->n * ((double)a.tq * (s.heads * s.kd + s.kv * s.selected) + (double)a.blocks * s.kv * s.kd));
  hipLaunchKernelGGL(select_kernel, dim3((unsigned)a.rows), dim3(64), 0, ctx->stream, a);
  return check_launch("block_select");
}

}  // namespace sy

extern "C" {

int sy_block_means(sy_ctx* ctx, const sy_block_config* cfg, const sy_tensor* k, const int32_t* starts, int tokens,
                   const int32_t* lengths, const sy_tensor* means) {
  return sy::op_block_means(ctx, cfg, k, starts, tokens, lengths, means);
}

int sy_block_select(sy_ctx* ctx, const sy_block_config* cfg, const sy_tensor* q, const sy_tensor* means,
                    const int32_t* starts, const int32_t* lengths, int32_t* blocks) {
  return sy::op_block_select(ctx, cfg, q, means, starts, lengths, blocks);
}

}  // extern "C"
