// Which key blocks each query attends to: mean keys of the blocks, and for every query the blocks whose
// mean has the largest product with it.
//
// The choice is made on scores in 64 bits: products of floats are exact there (those of a sum of several heads round
// once) and 128 of them sum within 2^-45 of their magnitudes, whatever the order, which differs between the kernels
// below.  In 32 bits a choice would hang on it far more often.
#include <cfloat>
#include <climits>
#include <cmath>

#include "split.h"
#include "sy_internal.h"

namespace sy {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

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
  int tk, kh, kw, bh, bw, bx, blocks, ks, kd, units, lanes, pieces, tokens, slots;
};

// One workgroup per image, block (with `tokens`: that may hold some) and 128 channels.  A lane sums four channels over
// every (256 / lanes)-th key, eight keys under way at a time; the partial sums meet in LDS in one order.  Bound by
// memory: four 160x160 maps of 128 channels (52 MB) in 11 us, 4.8 TB/s; one token's block of 16 caches 4 us, the latency of
// a launch and its loads.
__global__ __launch_bounds__(256) void means_kernel(const MeansArgs a) {
  __shared__ double part[256][4];
  const int piece = blockIdx.x % a.pieces, bs = blockIdx.x / a.pieces, b = bs / a.slots, slot = bs % a.slots;
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
  const int u = piece * a.lanes + lane, head = 4 * u / a.kd;
  double s[4] = {0, 0, 0, 0};
  if (u < a.units) {
    const float* kb = a.k + ((long long)b * a.tk + (long long)y0 * a.kw + x0) * a.ldk + head * a.ks + (4 * u - head * a.kd);
    int y = 0, x = group;
    for (int t = group; t < keys; t += 8 * groups) {
      f32x4 v[8];
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        for (; x >= cols; x -= cols) ++y;
        const bool on = t + n * groups < keys;
        v[n] = *(const f32x4*)(kb + (on ? ((long long)y * a.kw + x) * a.ldk : 0));
        if (!on) v[n] = f32x4{0.f, 0.f, 0.f, 0.f};
        x += groups;
      }
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += v[n][e];
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
  while (a.lanes < a.units && a.lanes < 32) a.lanes *= 2;
  a.pieces = (a.units + a.lanes - 1) / a.lanes;
  a.tokens = tokens;
  a.slots = tokens ? (int)std::min<long long>(a.blocks, (tokens - 1LL) / s.bw + 2) : a.blocks;
  const long long grid = (long long)k->n * a.slots * a.pieces;
  SY_CHECK(grid * 256 < (1LL << 32), SY_EUNSUPPORTED, "block means grid too large");
  DeviceScope device(ctx);
  const double read = tokens ? (double)a.slots * s.bw : (double)a.tk;
  ProfScope prof(ctx, "block_means", (double)k->n * read * s.kv * s.kd,
                 4.0 * k->n * s.kv * s.kd * (std::min(read, (double)a.tk) + a.slots));
  hipLaunchKernelGGL(means_kernel, dim3((unsigned)grid), dim3(256), 0, ctx->stream, a);
  return check_launch("block_means");
}

// ----------------------------------------------------------------- selection
//
// Many queries: scores in float32 from the matrix cores with a bound e on their error.  The largest ones of each query are
// kept, so that the `selected`-th, t, is known; no block further than 2 e below t is chosen, whatever the rounding, and
// every block further than 2 e above it is.  Up to 16 of 4,096 blocks are kept with their numbers; of more, the scores are
// formed again and compared with t - 2 e.  Where more than `selected` lie there, some queries in a hundred, those within
// 2 e of t are scored again in 64 bits.  Queries of zeros (padding), and all where the means are zeros, need no scores.
// Few queries: scores in 64 bits, then a ranking.

struct SelectArgs {
  const float *q, *m;
  const int *starts, *lengths;
  int* out;
  long long ldq, ldm, rows;
  int tq, blocks, bw, kv, group, kd, qs, selected, causal;
  // many queries: the means' parts, made by `chunks` workgroups for each key head, and their norms
  u32x4* parts;
  float* norm;
  int tiles, chunks;
  int tag_bits;      // of a block's number in its scores
  float tag_error;   // twice what they cost, of a score
  // few queries: scores, and how many of them a workgroup takes
  long long* keys;
  int queries;
};

// 64-bit scores in an order of integers: NaN below every number, zeros alike.
__device__ __forceinline__ long long score_key(double s) {
  if (s != s) return LLONG_MIN + 1;
  const long long b = __builtin_bit_cast(long long, s + 0.0);
  return b < 0 ? LLONG_MIN + 2 + ~b : b;
}
constexpr long long kHidden = LLONG_MIN;

// Blocks that query i of image b sees, and the one that is always taken (-1: none).
__device__ __forceinline__ int seen_blocks(const SelectArgs& a, int b, int i, int* forced) {
  long long seen = a.blocks;
  *forced = -1;
  if (a.lengths) seen = min(seen, ((long long)max(a.lengths[b], 0) + a.bw - 1) / a.bw);
  if (a.causal) {
    const long long at = (long long)(a.starts ? a.starts[b] : 0) + i;
    if (at < 0) return 0;
    const long long own = at / a.bw;
    if (own < seen) *forced = (int)own;
    seen = min(seen, own + 1);
  }
  return (int)seen;
}

// Ranking by one wave: of the keys key(j), j < count, the `selected` largest, ties by the lower j.  Lane n ends with the
// n-th; the number of them is returned.  Every lane keeps four new keys and one of the best so far in order;
// the largest head of all is taken `selected` times.
template <class F>
__device__ __forceinline__ int rank_wave(int count, int selected, int lane, F key, long long* best_key, int* best_id) {
  int kept = 0;
  long long bk = kHidden;
  int bi = 0x7fffffff;
  for (int j0 = 0; j0 < count; j0 += 256) {
    long long k[5];
    int id[5];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = j0 + 64 * u + lane;
      k[u] = j < count ? key(j) : kHidden;
      id[u] = j;
    }
    if (kept == selected) {
      const long long least = __shfl(bk, selected - 1);
      if (!__any(max(max(k[0], k[1]), max(k[2], k[3])) > least)) continue;
    }
    k[4] = lane < kept ? bk : kHidden;
    id[4] = lane < kept ? bi : 0x7fffffff;
#pragma unroll
    for (int pass = 0; pass < 4; ++pass)
#pragma unroll
      for (int u = 4; u > pass; --u) {
        const bool up = k[u] > k[u - 1] || (k[u] == k[u - 1] && id[u] < id[u - 1]);
        const long long tk = up ? k[u] : k[u - 1];
        const int ti = up ? id[u] : id[u - 1];
        k[u] = up ? k[u - 1] : k[u];
        id[u] = up ? id[u - 1] : id[u];
        k[u - 1] = tk;
        id[u - 1] = ti;
      }
    int n = 0;
    for (; n < selected; ++n) {
      // The high halves first; where they agree, the low ones (in the order of signed numbers), then the lower block.
      const int hi = (int)(k[0] >> 32), top = wave_max_i32(hi);
      unsigned long long heads = __ballot(hi == top);
      if (heads & (heads - 1)) {
        const int low = hi == top ? (int)((unsigned)k[0] ^ 0x80000000u) : INT_MIN, top_low = wave_max_i32(low);
        heads &= __ballot(low == top_low);
        if (heads & (heads - 1)) {
          const int mine = heads >> lane & 1 ? -id[0] : INT_MIN, first = wave_max_i32(mine);
          heads = __ballot(mine == first);
        }
      }
      const int winner = __builtin_ctzll(heads);
      const long long best = (long long)top << 32 | (unsigned)__builtin_amdgcn_readlane((int)k[0], winner);
      if (best == kHidden) break;
      const int won = __builtin_amdgcn_readlane(id[0], winner);
      if (lane == n) {
        bk = best;
        bi = won;
      }
      if (lane == winner) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          k[u] = k[u + 1];
          id[u] = id[u + 1];
        }
        k[4] = kHidden;
        id[4] = 0x7fffffff;
      }
    }
    kept = n;
  }
  *best_key = bk;
  *best_id = lane < kept ? bi : 0x7fffffff;
  return kept;
}

// Writes a wave's ranking in ascending order of blocks, then -1.
__device__ __forceinline__ void write_row(int* out, int selected, int kept, int lane, int id) {
  int place = 0;
  for (int n = 0; n < kept; ++n) place += __builtin_amdgcn_readlane(id, n) < id;
  if (lane < selected) out[lane < kept ? place : lane] = lane < kept ? id : -1;
}

// The sum of the query heads that share a key head, in 64 bits: channel c.
__device__ __forceinline__ double query_sum(const SelectArgs& a, const float* q, int c) {
  double s = 0;
#pragma unroll 4
  for (int h = 0; h < a.group; ++h) s += q[(long long)h * a.qs + c];
  return s;
}

// The sum of query i's heads of group g, in 64 bits, two channels to a lane.
__device__ __forceinline__ void query_sums(const SelectArgs& a, int b, int i, int g, int lane, double (&s)[2]) {
  const float* q = a.q + ((long long)b * a.tq + i) * a.ldq + (long long)g * a.group * a.qs + min(2 * lane, a.kd - 2);
  s[0] = s[1] = 0;
#pragma unroll 8
  for (int h = 0; h < a.group; ++h) {
    const f32x2v v = *(const f32x2v*)(q + (long long)h * a.qs);
    s[0] += v[0];
    s[1] += v[1];
  }
}

__device__ __forceinline__ long long exact_key(const SelectArgs& a, int b, int g, int j, const double* qsum) {
  const float* m = a.m + ((long long)b * a.blocks + j) * a.ldm + g * a.kd;
  double s = 0;
#pragma unroll 4
  for (int c = 0; c < a.kd; c += 4) {
    const f32x4 v = *(const f32x4*)(m + c);
#pragma unroll
    for (int e = 0; e < 4; ++e) s = __builtin_fma(qsum[c + e], (double)v[e], s);
  }
  return score_key(s);
}

// The last query that a wave has ranked so, and its choice.
struct Ranked {
  double q[2];
  int seen = -1, forced, kept, id;
};

// One query in 64 bits by one wave: a lane scores a block of 64.  Where many blocks are alike (a constant area of a map),
// so are the queries there, one after the other: the choice of the one before is theirs.
__device__ __forceinline__ void select_exact(const SelectArgs& a, int b, int i, int g, int lane, double* qsum, Ranked& last) {
  double q[2];
  query_sums(a, b, i, g, lane, q);
  int forced;
  const int seen = seen_blocks(a, b, i, &forced);
  // (A NaN differs from itself: such a query is ranked.)
  if (seen != last.seen || forced != last.forced || !__all(q[0] == last.q[0] && q[1] == last.q[1])) {
    if (2 * lane < a.kd) {
      qsum[2 * lane] = q[0];
      qsum[2 * lane + 1] = q[1];
    }
    __builtin_amdgcn_wave_barrier();
    long long bk;
    last.kept = rank_wave(seen, a.selected, lane,
                          [&](int j) { return j == forced ? (long long)LLONG_MAX : exact_key(a, b, g, j, qsum); }, &bk, &last.id);
    __builtin_amdgcn_wave_barrier();
    last.q[0] = q[0];
    last.q[1] = q[1];
    last.seen = seen;
    last.forced = forced;
  }
  write_row(a.out + (((long long)b * a.tq + i) * a.kv + g) * a.selected, a.selected, last.kept, lane, last.id);
}

// The same among `count` candidates (up to 64, more than wanted), of which those marked kDoubtful are scored: sixteen
// lanes to one, KS channels to a lane, four at a time.
constexpr int kDoubtful = 1 << 30;
template <int KS>
__device__ __forceinline__ void select_among(const SelectArgs& a, int b, int i, int g, int lane, const int* pool, int count) {
  const int entry = lane < count ? pool[lane] : 0, id = lane < count ? entry & ~kDoubtful : INT_MAX;
  const unsigned long long doubtful = __ballot(entry & kDoubtful);
  const int c = KS * (lane & 15);
  f32x2v m[KS / 2];
  double qsum[KS];
  long long key = kHidden;
  for (unsigned long long todo = doubtful; todo;) {
    int at[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      at[u] = todo ? __builtin_ctzll(todo) : -1;
      todo &= todo - 1;
    }
    const int mine = lane < 32 ? (lane < 16 ? at[0] : at[1]) : (lane < 48 ? at[2] : at[3]);
    const float* from = a.m + ((long long)b * a.blocks + __shfl(id, max(mine, at[0]))) * a.ldm + g * a.kd;
#pragma unroll
    for (int x = 0; x < KS / 2; ++x) m[x] = *(const f32x2v*)(from + min(c + 2 * x, a.kd - 2));
    if (at[0] == __builtin_ctzll(doubtful)) {  // the first time
      const float* q = a.q + ((long long)b * a.tq + i) * a.ldq + (long long)g * a.group * a.qs;
#pragma unroll
      for (int x = 0; x < KS; ++x) qsum[x] = 0;
#pragma unroll 4
      for (int h = 0; h < a.group; ++h)
#pragma unroll
        for (int x = 0; x < KS / 2; ++x) {
          const f32x2v v = *(const f32x2v*)(q + (long long)h * a.qs + min(c + 2 * x, a.kd - 2));
          qsum[2 * x] += v[0];
          qsum[2 * x + 1] += v[1];
        }
    }
    double s = 0;
#pragma unroll
    for (int x = 0; x < KS / 2; ++x)
      if (c + 2 * x < a.kd) s = __builtin_fma(qsum[2 * x + 1], (double)m[x][1], __builtin_fma(qsum[2 * x], (double)m[x][0], s));
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) s += __shfl_xor(s, off);
    const long long k = score_key(s);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const long long of = __shfl(k, 16 * u);
      if (lane == at[u]) key = of;
    }
  }
  int before = count - __builtin_popcountll(doubtful);
  for (unsigned long long todo = doubtful; todo; todo &= todo - 1) {
    const int n = __builtin_ctzll(todo);
    const long long k = __shfl(key, n);
    before += k > key || (k == key && __shfl(id, n) < id);
  }
  const unsigned long long chosen = __ballot(lane < count && (!(doubtful >> lane & 1) || before < a.selected));
  int place = 0;
  for (unsigned long long todo = chosen; todo; todo &= todo - 1)
    place += __builtin_amdgcn_readlane(id, __builtin_ctzll(todo)) < id;
  if ((chosen >> lane & 1) && place < a.selected) a.out[(((long long)b * a.tq + i) * a.kv + g) * a.selected + place] = id;
}

// Eight floats as two bf16 parts, v = p[0] + p[1] up to 2^-18 of v.
__device__ __forceinline__ void halves8(const float (&x)[8], bf16x8 (&p)[2]) {
  u32x4 w[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f32x2v v = {x[2 * i], x[2 * i + 1]};
    const unsigned hi = __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2));
    v[0] -= __builtin_bit_cast(float, hi << 16);
    v[1] -= __builtin_bit_cast(float, hi & 0xffff0000u);
    w[0][i] = hi;
    w[1][i] = __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2));
  }
  p[0] = __builtin_bit_cast(bf16x8, w[0]);
  p[1] = __builtin_bit_cast(bf16x8, w[1]);
}

// A sum of squares, not 0 unless all of what was squared is (bits: or'ed over it).
__device__ __forceinline__ float norm_of(float squares, unsigned bits) {
  return (bits & 0x7fffffffu) && squares == 0.f ? FLT_MIN : squares;
}

constexpr int kPools = 8;      // doubtful queries of a wave whose candidates are kept (second pass)
constexpr int kPartTiles = 8;  // 32-block tiles of a workgroup below

// The means of one key head as the A operands of the matrix instructions (32 blocks x 16 channels, two parts
// each), and their norms, squared.  Means that no query sees (a cache's, behind the last token) are taken as 0,
// so that what stands there does not widen the bound or send every query through 64 bits.
template <int KS>
__global__ __launch_bounds__(256) void means_parts_kernel(const SelectArgs a) {
  const int plane = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks, b = plane / a.kv, g = plane % a.kv;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  int forced;
  const int seen = seen_blocks(a, b, a.tq - 1, &forced);
  for (int t = wave; t < kPartTiles; t += 4) {
    const int tile = chunk * kPartTiles + t, j = tile * 32 + (lane & 31);
    if (tile >= a.tiles) break;
    const float* m = a.m + ((long long)b * a.blocks + min(j, a.blocks - 1)) * a.ldm + g * a.kd;
    float norm = 0.f;
    unsigned bits = 0;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      float f[8];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int c = 16 * ks + 8 * half + 4 * u;
        const f32x4 v = c < a.kd && j < seen ? *(const f32x4*)(m + c) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f[4 * u + e] = v[e];
          norm = __builtin_fmaf(v[e], v[e], norm);
        }
        bits |= magnitude_bits(v);
      }
      bf16x8 p[2];
      halves8(f, p);
      u32x4* to = a.parts + (((long long)plane * a.tiles + tile) * KS + ks) * 2 * 64 + lane;
      to[0] = __builtin_bit_cast(u32x4, p[0]);
      to[64] = __builtin_bit_cast(u32x4, p[1]);
    }
    norm = norm_of(norm, bits);
    norm += __shfl_xor(norm, 32);
    if (half == 0 && j < a.blocks) a.norm[(long long)plane * a.blocks + j] = norm;
  }
}

// 32 queries of one key head per wave, four waves to a workgroup that share nothing.
//
// S^T = M Q^T: a lane holds a query's scores of the blocks 8 (r / 4) + 4 half + r % 4 of a tile.  The SMAX + 1 largest
// so far stay sorted in registers: a new score moves through them by one median of three each.  (Fewer wanted:
// the list starts with infinities.)  The two halves' lists meet at the end.
//
// Tags: the lowest tag_bits of a score are the tile and r, so that the lists name their blocks.  That moves a score by up to
// u = 2^(tag_bits - 23) of itself: 2 u |t| more between two of them at the border, taken with 2.125 u for the scores near t
// that are a little larger than it.  (Otherwise: a second pass over all scores.)
//
// Error of a score: a part is off by 2^-8 of what it stands for, so two of them by 2^-16, twice (operands), and the
// product of the second parts is left out, 2^-16 again: 3 x 2^-16 of sum |q||m|.  Sums of at most 24 matrix
// instructions with 16 products each, and q rounded from 64 bits, stay below 2^-18.  sum |q||m| <= |q||m| in norms,
// which sums in float32 and two roots change by less than 2^-16 of themselves: e = 3.5 x 2^-16 |q| max|m|.  Norms
// outside 2^-40 .. 2^40 could lose parts to underflow: all blocks of those queries are scored in 64 bits.
//
// Bound by vector work, which keeps the SIMDs busy nine tenths of the time: 3,600 operations per wave (32 queries, 400 blocks
// of 32 channels, 8 wanted), of them 1,900 medians; the matrix cores work a sixth of it.  Four maps of 25,600 queries, 4
// heads: 106 to 121 us with the means' parts; with a second pass over the scores 140; 64 queries to a wave, which halves
// the reads of the means, 154; where every query is in doubt between more blocks than the lists hold, and ranked in
// 64 bits, 2,450 (one mean 1,000 times as long as the others, which widens the bound for all, or means all alike but
// queries that are not; one mean 10 / 100 times as long 130 / 302).  Two causal rows of 16,001 tokens, 16 / 4 heads of
// 128 channels, 16 of 251 blocks: 90 us, of them 50 the queries' way from memory; with all candidates of doubtful queries
// scored again 117, their heads read in 32-byte pieces besides 126.
// kTwice: a second pass over the scores; kTags: their blocks' numbers in them; kRaw: that, on the means as they are.
enum { kTwice, kTags, kRaw };
template <int KS, int SMAX, int MODE>
__global__ __launch_bounds__(256, SMAX > 16 ? 1 : KS == 2 ? 4 : KS == 4 ? 3 : 1) void select_tile_kernel(const SelectArgs a) {
  __shared__ double qsum[4][128];
  constexpr bool TAGS = MODE != kTwice;
  constexpr int kRow = 2 * SMAX + 3;  // candidates of a query (odd: its lanes' banks differ)
  constexpr int KB = KS < 4 ? KS : 4, kStage = 32 * (16 * KB + 4);
  __shared__ __align__(16) float stage[4][kStage];  // query sums; candidates
  static_assert(kStage >= (TAGS ? 32 * kRow : kPools * 64), "candidates of a wave");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, r32 = lane & 31;
  int* pool = (int*)stage[wave];
  const int groups = (a.tq + 127) / 128;
  const int plane = blockIdx.x / groups, b = plane / a.kv, g = plane - b * a.kv;
  const int i0 = (blockIdx.x - plane * groups) * 128 + wave * 32;
  if (i0 >= a.tq) return;

  bf16x8 q[KS][2];
  int forced;
  const int i = i0 + r32;
  const int seen = seen_blocks(a, b, min(i, a.tq - 1), &forced);
  const int last = __builtin_amdgcn_readfirstlane((wave_max_i32(seen) + 31) / 32);
  // The largest norm of the means whose scores count: not of the block that holds the last token, whose mean, of few keys,
  // may be many times as long as the others (NaN above all).
  const int scored = wave_max_i32(forced >= 0 ? forced : seen);
  int top = 0;
  for (int j = lane; MODE != kRaw && j < scored + lane; j += 512) {
    int v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = ((const int*)a.norm)[(long long)plane * a.blocks + min(j + 64 * u, scored - 1)];
#pragma unroll
    for (int u = 0; u < 8; ++u) top = max(top, v[u] & 0x7fffffff);
  }
  float qn = 0.f;
  unsigned q_bits = 0;
  {
    // Up to 64 channels of a head at a time, in whole lines: a lane sums four channels of every STEP-th row over the heads,
    // and the sums change their layout in LDS.
    constexpr int kLanes = 4 * KB, kStep = 64 / kLanes, kSteps = 32 / kStep;
    float* sums = stage[wave];
    const int sub = lane % kLanes, first = lane / kLanes;
    const float* p = a.q + (long long)b * a.tq * a.ldq + (long long)g * a.group * a.qs;
#pragma unroll
    for (int k0 = 0; k0 < KS; k0 += KB) {
      const int c = 16 * k0 + 4 * sub;
      const float* from[kSteps];
      double s[kSteps][4];
#pragma unroll
      for (int t = 0; t < kSteps; ++t) {
        from[t] = p + (long long)min(i0 + t * kStep + first, a.tq - 1) * a.ldq + min(c, a.kd - 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[t][e] = 0.0;
      }
      for (int h = 0; h < a.group; ++h) {
        f32x4 v[kSteps];
#pragma unroll
        for (int t = 0; t < kSteps; ++t) v[t] = *(const f32x4*)(from[t] + (long long)h * a.qs);
#pragma unroll
        for (int t = 0; t < kSteps; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[t][e] += v[t][e];
      }
#pragma unroll
      for (int t = 0; t < kSteps; ++t) {
        f32x4 f;
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = c < a.kd ? (float)s[t][e] : 0.f;
        *(f32x4*)&sums[(t * kStep + first) * (16 * KB + 4) + 4 * sub] = f;
      }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int ks = 0; ks < KB; ++ks) {
        float f[8];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const f32x4 v = *(const f32x4*)&sums[r32 * (16 * KB + 4) + 16 * ks + 8 * half + 4 * u];
#pragma unroll
          for (int e = 0; e < 4; ++e) f[4 * u + e] = v[e];
          q_bits |= magnitude_bits(v);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) qn = __builtin_fmaf(f[e], f[e], qn);
        halves8(f, q[k0 + ks]);
      }
      __builtin_amdgcn_wave_barrier();
    }
    qn = norm_of(qn, q_bits);
    qn += __shfl_xor(qn, 32);
  }
  const u32x4* parts = a.parts + (long long)plane * a.tiles * KS * 2 * 64 + lane;

  // Scores of tile n, whose parts are under way, with what is not seen at -inf and what is forced at +inf (with tags, which
  // have no room beside an infinity, it is left out).
  const unsigned keep = ~0u << a.tag_bits;
  u32x4 m[KS][2];
  const float* means = a.m + (long long)b * a.blocks * a.ldm + g * a.kd;
  auto load = [&](int n) __attribute__((always_inline)) {
    if (MODE == kRaw) {
      const float* from = means + min(32 * n + r32, a.blocks - 1) * a.ldm;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int u = 0; u < 2; ++u) m[ks][u] = *(const u32x4*)(from + min(16 * ks + 8 * half + 4 * u, a.kd - 4));
      return;
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int p = 0; p < 2; ++p) m[ks][p] = parts[((long long)n * KS + ks) * 128 + 64 * p];
  };
  auto scores = [&](int n) __attribute__((always_inline)) {
    f32x16 sc;
#pragma unroll
    for (int r = 0; r < 16; ++r) sc[r] = 0.f;
    float norm = 0.f;
    unsigned bits = 0;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      bf16x8 p[2] = {__builtin_bit_cast(bf16x8, m[ks][0]), __builtin_bit_cast(bf16x8, m[ks][1])};
      if (MODE == kRaw) {
        float f[8];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const f32x4 v = __builtin_bit_cast(f32x4, m[ks][u]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            f[4 * u + e] = 16 * ks + 8 * half + 4 * u < a.kd ? v[e] : 0.f;
            norm = __builtin_fmaf(f[4 * u + e], f[4 * u + e], norm);
            bits |= __builtin_bit_cast(unsigned, f[4 * u + e]);
          }
        }
        halves8(f, p);
      }
      sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(p[1], q[ks][0], sc, 0, 0, 0);
      sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(p[0], q[ks][1], sc, 0, 0, 0);
      sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(p[0], q[ks][0], sc, 0, 0, 0);
    }
    load(min(n + 1, last - 1));
    if (MODE == kRaw) {
      norm = norm_of(norm, bits);
      norm += __shfl_xor(norm, 32);
      if (32 * n + r32 < scored) top = max(top, __builtin_bit_cast(int, norm) & 0x7fffffff);
    }
    if (TAGS)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float x = sc[r];
        sc[r] = __builtin_bit_cast(float, (__builtin_bit_cast(unsigned, x) & keep) | (unsigned)(16 * n + r));
      }
    const int room = seen - 32 * n - 4 * half, own = forced - 32 * n - 4 * half;
    if (__any(room < 32 || (own >= 0 && own < 32)))
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int at = 8 * (r >> 2) + (r & 3);
        sc[r] = at >= room ? -INFINITY : at == own ? (TAGS ? -INFINITY : INFINITY) : sc[r];
      }
    return sc;
  };

  const int wanted = a.selected - (TAGS && forced >= 0);
  float list[SMAX + 1];
#pragma unroll
  for (int n = 0; n <= SMAX; ++n) list[n] = n < SMAX - wanted && half == 0 ? INFINITY : -INFINITY;
  if (last > 0) load(0);
  for (int n = 0; n < last; ++n) {
    const f32x16 sc = scores(n);
    float top = sc[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, sc[r]);
    if (!__any(top > list[SMAX])) continue;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
#pragma unroll
      for (int u = SMAX; u > 0; --u) list[u] = __builtin_amdgcn_fmed3f(list[u - 1], list[u], sc[r]);
      list[0] = fmaxf(list[0], sc[r]);
    }
  }

  // The n-th largest of two sorted lists is the least of the maxima of one's u-th and the other's (n - 1 - u)-th.
  float nth = INFINITY, after = INFINITY, other[SMAX + 1];
#pragma unroll
  for (int n = 0; n <= SMAX; ++n) other[n] = __shfl_xor(list[n], 32);
#pragma unroll
  for (int n = 0; n < SMAX; ++n) nth = fminf(nth, fmaxf(list[n], other[SMAX - 1 - n]));
#pragma unroll
  for (int n = 0; n <= SMAX; ++n) after = fminf(after, fmaxf(list[n], other[SMAX - n]));
  const float kn = scored ? __builtin_bit_cast(float, wave_max_i32(top)) : 1.f;
  // A query of zeros (padding), or means of zeros, has scores that are all 0 if the others are finite: the lowest blocks.
  const bool zero = (qn == 0.f && kn < INFINITY) || (kn == 0.f && qn < INFINITY);
  // Whether all blocks of this lane's query are scored in 64 bits.
  bool exact = !zero && !(qn >= 0x1p-80f && qn <= 0x1p80f && kn >= 0x1p-80f && kn <= 0x1p80f);
  const float slack = 7.f / 65536 * (__builtin_sqrtf(qn) * __builtin_sqrtf(kn));  // 2 e
  // Scores from here up are candidates.
  const float from = __builtin_fabsf(nth) == INFINITY ? nth : nth - (TAGS ? slack + a.tag_error * __builtin_fabsf(nth) : slack);
  const float sure = nth + (nth - from);  // scores above are chosen, whatever their errors (NaN: there is no doubt)
  const bool doubt = !exact && !zero && i < a.tq && seen > a.selected && !(after < from);
  const bool mine = half == 0 && i < a.tq;
  int* out = a.out + (((long long)b * a.tq + i) * a.kv + g) * a.selected;
  if (zero && mine) {  // (the block that is always taken is the last one seen)
    const int count = min(seen, a.selected);
    for (int n = 0; n < a.selected; ++n) out[n] = n >= count ? -1 : n == count - 1 && forced >= 0 ? forced : n;
  }

  if constexpr (TAGS) {
    // Candidates of both halves side by side, the lower half's first, then the block that is always taken.
    exact |= doubt && (list[SMAX] >= from || other[SMAX] >= from);  // maybe more than the lists hold
    const int mark = doubt ? kDoubtful : 0;
    int own = 0;
#pragma unroll
    for (int n = 0; n <= SMAX; ++n) own += list[n] >= from && __builtin_fabsf(list[n]) < INFINITY;
    const int others = __shfl_xor(own, 32), count = own + others + (forced >= 0);
    int* row = pool + r32 * kRow;
    int to = half ? others : 0;
#pragma unroll
    for (int n = 0; n <= SMAX; ++n)
      if (list[n] >= from && __builtin_fabsf(list[n]) < INFINITY) {
        const int tag = __builtin_bit_cast(unsigned, list[n]) & ~keep;
        row[to++] = ((tag >> 4) * 32 + (tag & 12) * 2 + 4 * half + (tag & 3)) | (list[n] > sure ? 0 : mark);
      }
    if (half && forced >= 0) row[count - 1] = forced;
    __builtin_amdgcn_wave_barrier();
    if (i < a.tq && !exact && !doubt && !zero) {
      int id[SMAX];
#pragma unroll
      for (int n = 0; n < SMAX; ++n) id[n] = n < count ? row[n] : INT_MAX;
#pragma unroll
      for (int e = 0; e < SMAX; e += 2) {  // every second one for each half
        const int one = half ? id[e + 1] : id[e];
        int place = 0;
#pragma unroll
        for (int n = 0; n < SMAX; ++n) place += id[n] < one;
        if (e + half < a.selected) out[e + half < count ? place : e + half] = e + half < count ? one : -1;
      }
    }
    __builtin_amdgcn_wave_barrier();
    for (unsigned long long todo = __ballot(mine && doubt && !exact); todo; todo &= todo - 1) {
      const int x = __builtin_ctzll(todo);
      select_among<KS>(a, b, i0 + x, g, lane, pool + x * kRow, __builtin_amdgcn_readlane(count, x));
    }
    Ranked ranked;
    for (unsigned long long todo = __ballot(mine && exact); todo; todo &= todo - 1)
      select_exact(a, b, i0 + __builtin_ctzll(todo), g, lane, qsum[wave], ranked);
    return;
  }

  const unsigned doubts = (unsigned)__ballot(doubt);  // of the lower half; the upper one agrees
  int slot = doubt ? __builtin_popcount(doubts & ((1u << r32) - 1)) : -1;  // of a doubtful query's candidates
  if (slot >= kPools) {
    slot = -1;
    exact = true;
  }

  int count = 0;
  if (last > 0) load(0);
  for (int n = 0; n < last; ++n) {
    const f32x16 sc = scores(n);
    unsigned w = 0, near = 0;
#pragma unroll
    for (int r = 15; r >= 0; --r) w = w + w + (sc[r] >= from);
    if (!__any(w != 0)) continue;
    // Four blocks of this half, four of the other, and so on.
    auto both = [&](unsigned w) {
      w = (w | w << 8) & 0x00ff00ffu;
      w = (w | w << 4) & 0x0f0f0f0fu;
      const unsigned o = (unsigned)__shfl_xor((int)w, 32);
      return half ? o | w << 4 : w | o << 4;
    };
    w = both(w);
    if (doubts) {
#pragma unroll
      for (int r = 15; r >= 0; --r) near = near + near + !(sc[r] > sure);
      near = both(near);
    }
    const int room = seen - 32 * n;
    if (room < 32) w &= room > 0 ? (1u << room) - 1 : 0u;
    while (__any(w != 0)) {
      if (w) {
        const int j = 32 * n + __builtin_ctz(w);
        const int mark = near & (w & -w) ? kDoubtful : 0;
        w &= w - 1;
        if (mine && !exact && !zero) {
          if (slot >= 0) {
            if (count < 64) pool[slot * 64 + count] = j | mark;
          } else if (count < a.selected) {
            out[count] = j;
          }
        }
        ++count;
      }
    }
  }
  __builtin_amdgcn_wave_barrier();
  if (slot >= 0 && count > 64) exact = true;
  if (mine && !exact && !zero && slot < 0)
    for (int n = count; n < a.selected; ++n) out[n] = -1;
  for (unsigned long long todo = __ballot(mine && !exact && slot >= 0); todo; todo &= todo - 1) {
    const int x = __builtin_ctzll(todo);
    select_among<KS>(a, b, i0 + x, g, lane, pool + __builtin_amdgcn_readlane(slot, x) * 64,
                     __builtin_amdgcn_readlane(count, x));
  }
  Ranked ranked;
  for (unsigned long long todo = __ballot(mine && exact); todo; todo &= todo - 1)
    select_exact(a, b, i0 + __builtin_ctzll(todo), g, lane, qsum[wave], ranked);
}

constexpr int kScoreQueries = 8;
constexpr int kCandidates = 256;  // of a ranking

// Scores of 64 blocks and up to eight queries in 64 bits, four lanes to a block.  For one token against caches the time is
// that of the means' way from memory (34 MB in 7 us).
template <int KS>
__global__ __launch_bounds__(256) void score_kernel(const SelectArgs a) {
  __shared__ double qsum[kScoreQueries][128];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, quarter = 4 * (lane & 3);
  const int chunks = (a.blocks + 63) / 64, chunk = blockIdx.x % chunks, rest = blockIdx.x / chunks;
  const int batches = (a.tq + a.queries - 1) / a.queries, plane = rest / batches, b = plane / a.kv, g = plane - b * a.kv;
  const int i0 = (rest - plane * batches) * a.queries, count = min(a.queries, a.tq - i0);
  const int j = chunk * 64 + wave * 16 + (lane >> 2);
  f32x4 k[KS];
  const float* m = a.m + ((long long)b * a.blocks + min(j, a.blocks - 1)) * a.ldm + g * a.kd + quarter;
#pragma unroll
  for (int n = 0; n < KS; ++n) k[n] = 16 * n + quarter < a.kd ? *(const f32x4*)(m + 16 * n) : f32x4{0.f, 0.f, 0.f, 0.f};
  for (int x = threadIdx.x; x < count * 128; x += 256) {
    const int i = x >> 7, c = x & 127;
    const float* q = a.q + ((long long)b * a.tq + i0 + i) * a.ldq + (long long)g * a.group * a.qs;
    qsum[i][c] = c < a.kd ? query_sum(a, q, c) : 0.0;
  }
  __syncthreads();
  for (int i = 0; i < count; ++i) {
    int forced;
    const int seen = seen_blocks(a, b, i0 + i, &forced);
    double s = 0;
#pragma unroll
    for (int n = 0; n < KS; ++n)
      if (16 * n + quarter < a.kd)
#pragma unroll
        for (int e = 0; e < 4; ++e) s = __builtin_fma(qsum[i][16 * n + quarter + e], (double)k[n][e], s);
    s += __shfl_xor(s, 1);
    s += __shfl_xor(s, 2);
    if ((lane & 3) == 0 && j < a.blocks)
      a.keys[((long long)plane * a.tq + i0 + i) * a.blocks + j] =
          j >= seen ? kHidden : j == forced ? LLONG_MAX : score_key(s);
  }
}

// One query per workgroup.  The n-th largest of the threads' own largest scores (their upper bits) is no more than the n-th
// largest of all: the blocks from there up, a few more than wanted, are ranked by counting those before each.  Where they
// do not fit (many blocks alike), one wave ranks all.  Bound by its steps one after another: 7.5 us for 16 of 1,024 blocks,
// however many queries there are up to the number of CUs; taking the largest of all heads of four waves' lists 11.
__global__ __launch_bounds__(256) void rank_kernel(const SelectArgs a) {
  __shared__ __align__(16) int top[256];
  __shared__ int bound, count, chosen[64];
  __shared__ long long key[kCandidates];
  __shared__ int id[kCandidates];
  const int tid = threadIdx.x, lane = tid & 63;
  const long long* keys = a.keys + (long long)blockIdx.x * a.blocks;
  const int row = blockIdx.x % a.tq, plane = blockIdx.x / a.tq;  // keys are [plane][query]
  int* out = a.out + (((long long)(plane / a.kv) * a.tq + row) * a.kv + plane % a.kv) * a.selected;
  long long k[4];  // of the first 1024 blocks, the others are read twice
  int most = INT_MIN;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    k[u] = tid + 256 * u < a.blocks ? keys[tid + 256 * u] : kHidden;
    most = max(most, (int)(k[u] >> 32));
  }
#pragma unroll 4
  for (int j = tid + 1024; j < a.blocks; j += 256) most = max(most, (int)(keys[j] >> 32));
  most = (most & ~255) | (255 - tid);  // each its own
  top[tid] = most;
  if (tid == 0) count = 0;
  if (tid < 64) chosen[tid] = INT_MAX;
  __syncthreads();
  int before = 0;
#pragma unroll 8
  for (int n = 0; n < 64; ++n) {
    const i32x4 t = *(const i32x4*)&top[4 * n];
#pragma unroll
    for (int e = 0; e < 4; ++e) before += t[e] > most;
  }
  if (before == a.selected - 1) bound = most & ~255;
  __syncthreads();
  const int least = bound;
  auto offer = [&](int j, long long x) {
    if (x == kHidden || (int)(x >> 32) < least) return;
    const int at = atomicAdd(&count, 1);
    if (at < kCandidates) {
      key[at] = x;
      id[at] = j;
    }
  };
#pragma unroll
  for (int u = 0; u < 4; ++u) offer(tid + 256 * u, k[u]);
  for (int j = tid + 1024; j < a.blocks; j += 256) offer(j, keys[j]);
  __syncthreads();
  const int found = count;
  if (found > kCandidates) {
    if (tid >= 64) return;
    long long bk;
    int bi;
    const int kept = rank_wave(a.blocks, a.selected, lane, [&](int j) { return keys[j]; }, &bk, &bi);
    write_row(out, a.selected, kept, lane, bi);
    return;
  }
  if (tid < found) {
    const long long mine = key[tid];
    const int j = id[tid];
    int rank = 0;
#pragma unroll 4
    for (int n = 0; n < found; ++n) rank += key[n] > mine || (key[n] == mine && id[n] < j);
    if (rank < a.selected) chosen[rank] = j;
  }
  __syncthreads();
  if (tid < 64) {
    const int mine = chosen[lane];
    int place = 0;
#pragma unroll 8
    for (int n = 0; n < a.selected; ++n) place += chosen[n] < mine;
    if (lane < a.selected) out[mine != INT_MAX ? place : lane] = mine != INT_MAX ? mine : -1;
  }
}

// The matrix cores from here on, and where there are few blocks (both take 10 us then).  Below, a wave's walk through all
// blocks takes longer than all scores in 64 bits: 512 blocks of 128 channels, 16 of them, 4 key heads and 1 / 128 / 512 queries
// 34 / 41 / 43 us against 11 / 18 / 39; 128 blocks of 64 channels, 32 key heads, 8 / 32 / 64 queries 15 / 15 / 17 against
// 10 / 15 / 20.
constexpr int kManyRows = 2048, kFewBlocks = 64;
// Numbers of up to 11 bits (128 tiles, 4,096 blocks) in the scores of lists of up to 16: 8 / 16 of 400 blocks of 32 channels 112 /
// 150 us, with a second pass 149 / 190; of 128 channels 111 and 180.  More blocks would cost the scores too many bits.
constexpr int kTagBits = 11;
// Means split by every wave for itself, up to so many tiles x steps of all waves (beyond, the waves' 40 operations each take
// longer than the launch that would do it once): a 20x20 map 7.0 us against 9.9, a 48x48 one of four images and 4 heads 11.3
// against 13.8, 160x160 of 32 channels 30.4 against 30.7 (at 41,600), eight 88x88 of 64 53 against 47 (at 125,000).
constexpr long long kRawSteps = 1 << 15;

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
  SY_CHECK((long long)q->n * s.kv < (1 << 24), SY_EUNSUPPORTED, "block select over %d x %d key heads", q->n, s.kv);
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
  DeviceScope device(ctx);
  const int planes = q->n * s.kv, steps = s.kd <= 32 ? 2 : s.kd <= 64 ? 4 : 8;
  const double flops = 2.0 * a.rows * a.blocks * s.kd;
  const double bytes =
      4.0 * q->n * ((double)a.tq * (s.heads * s.kd + s.kv * s.selected) + (double)a.blocks * s.kv * s.kd);
  if (a.rows < kManyRows && a.blocks > kFewBlocks) {
    const long long chunks = (long long)planes * ((a.blocks + 63) / 64);
    a.queries = (int)std::min<long long>(kScoreQueries, std::max(1LL, chunks * a.tq / 2048));  // eight workgroups to a CU
    const long long grid = chunks * ((a.tq + a.queries - 1) / a.queries);
    SY_CHECK(grid * 256 < (1LL << 32) && a.rows * 256 < (1LL << 32), SY_EUNSUPPORTED, "block select grid too large");
    SY_TRY(ensure_scratch(ctx, sizeof(long long) * a.rows * a.blocks));
    a.keys = (long long*)ctx->scratch;
    {
      ProfScope prof(ctx, "block_score", flops, bytes);
      const dim3 g((unsigned)grid);
      if (steps <= 4)
        hipLaunchKernelGGL(score_kernel<4>, g, dim3(256), 0, ctx->stream, a);
      else
        hipLaunchKernelGGL(score_kernel<8>, g, dim3(256), 0, ctx->stream, a);
      SY_TRY(check_launch("block_score"));
    }
    ProfScope prof(ctx, "block_rank", 0, 8.0 * a.rows * a.blocks);
    hipLaunchKernelGGL(rank_kernel, dim3((unsigned)a.rows), dim3(256), 0, ctx->stream, a);
    return check_launch("block_rank");
  }
  a.tiles = (a.blocks + 31) / 32;
  a.chunks = (a.tiles + kPartTiles - 1) / kPartTiles;
  const size_t parts = sizeof(u32x4) * 128 * (size_t)planes * a.tiles * steps;
  const long long groups = (a.tq + 127) / 128;
  SY_CHECK((long long)planes * groups * 256 < (1LL << 32) && (long long)planes * a.chunks * 256 < (1LL << 32),
           SY_EUNSUPPORTED, "block select grid too large");
  int bits = 4;
  while (1LL << (bits - 4) < a.tiles) ++bits;
  a.tag_bits = bits;
  a.tag_error = 2.125f * std::ldexp(1.f, bits - 23);
  const bool raw = s.selected <= 16 && bits <= kTagBits && 4LL * planes * groups * a.tiles * steps <= kRawSteps;
  if (!raw) {
    SY_TRY(ensure_scratch(ctx, parts + sizeof(float) * planes * (size_t)a.blocks));
    a.parts = (u32x4*)ctx->scratch;
    a.norm = (float*)(ctx->scratch + parts);
    ProfScope prof(ctx, "block_parts", 0, 8.0 * planes * (double)a.blocks * s.kd);
    const dim3 g((unsigned)(planes * a.chunks));
    if (steps == 2)
      hipLaunchKernelGGL(means_parts_kernel<2>, g, dim3(256), 0, ctx->stream, a);
    else if (steps == 4)
      hipLaunchKernelGGL(means_parts_kernel<4>, g, dim3(256), 0, ctx->stream, a);
    else
      hipLaunchKernelGGL(means_parts_kernel<8>, g, dim3(256), 0, ctx->stream, a);
    SY_TRY(check_launch("block_parts"));
  }
  ProfScope prof(ctx, "block_select", flops, bytes);
  const dim3 g((unsigned)(planes * groups));
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, g, dim3(256), 0, ctx->stream, a); };
  auto pick = [&](auto raw8, auto raw16, auto tags8, auto tags16, auto twice8, auto twice16, auto twice32, auto twice64) {
    if (raw)
      launch(s.selected <= 8 ? raw8 : raw16);
    else if (bits <= kTagBits && s.selected <= 16)
      launch(s.selected <= 8 ? tags8 : tags16);
    else
      launch(s.selected <= 8 ? twice8 : s.selected <= 16 ? twice16 : s.selected <= 32 ? twice32 : twice64);
  };
  if (steps == 2)
    pick(select_tile_kernel<2, 8, kRaw>, select_tile_kernel<2, 16, kRaw>, select_tile_kernel<2, 8, kTags>,
         select_tile_kernel<2, 16, kTags>, select_tile_kernel<2, 8, kTwice>, select_tile_kernel<2, 16, kTwice>,
         select_tile_kernel<2, 32, kTwice>, select_tile_kernel<2, 64, kTwice>);
  else if (steps == 4)
    pick(select_tile_kernel<4, 8, kRaw>, select_tile_kernel<4, 16, kRaw>, select_tile_kernel<4, 8, kTags>,
         select_tile_kernel<4, 16, kTags>, select_tile_kernel<4, 8, kTwice>, select_tile_kernel<4, 16, kTwice>,
         select_tile_kernel<4, 32, kTwice>, select_tile_kernel<4, 64, kTwice>);
  else
    pick(select_tile_kernel<8, 8, kRaw>, select_tile_kernel<8, 16, kRaw>, select_tile_kernel<8, 8, kTags>,
         select_tile_kernel<8, 16, kTags>, select_tile_kernel<8, 8, kTwice>, select_tile_kernel<8, 16, kTwice>,
         select_tile_kernel<8, 32, kTwice>, select_tile_kernel<8, 64, kTwice>);
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
