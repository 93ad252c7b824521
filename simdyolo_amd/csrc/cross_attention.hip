// Attention to states of another length: o = softmax(scale q k^T) v over the
// visible states of each image.
#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>

#include "parts.h"

namespace sy {

constexpr int kCrossKeys = 32;  // states of a tile

// What a piece of the states leaves for a row beside its weighted values: the
// maximum as an exponent of 2, and the sum of weights (0 without a visible state).
struct CrossStat {
  float top, sum;
};

struct CrossArgs {
  const float *q, *k, *v;
  float* o;
  const int* lengths;
  const uint8_t* mask;
  long long mask_image, mask_head, mask_query;
  long long ldq, ldo;
  int ldk, ldv;
  int tq, tk, heads, kv, group, kd, hd, qs, ks, vs;
  float scale, c;       // c: scale log2(e)
  int rows, tiles;      // rows (query, head of the group) of an image and key head, their tiles
  int splits, piece;    // pieces of the states, a multiple of kCrossKeys each
  unsigned items;
  CrossStat* stat;      // [image, key head][piece][row], where there are several
  float* part;          // weighted values
};

__device__ __forceinline__ int cross_end(const CrossArgs& a, int b) {
  return a.lengths ? min(max(a.lengths[b], 0), a.tk) : a.tk;
}

__device__ __forceinline__ const uint8_t* cross_mask(const CrossArgs& a, int b, int head, int i) {
  return a.mask ? a.mask + b * a.mask_image + head * a.mask_head + i * a.mask_query : nullptr;
}

// Work item of a workgroup: each of the 8 XCDs takes workgroups in turn, and with
// them one eighth of the items in a row, which read the same states.
__device__ __forceinline__ unsigned cross_item() { return (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3); }

// One row's output in plain float32 by one wave: lane `lane`'s channels lane and
// lane + 64.  States that are not visible are not touched; weights are normalised before they
// meet the values, so that no finite average overflows.
__device__ __forceinline__ void cross_row(const CrossArgs& a, int b, int i, int head, int lane, float (&z)[2]) {
  const float* q = a.q + ((long long)b * a.tq + i) * a.ldq + (long long)head * a.qs;
  const float* k = a.k + (long long)b * a.tk * a.ldk + (long long)(head / a.group) * a.ks;
  const float* v = a.v + (long long)b * a.tk * a.ldv + (long long)(head / a.group) * a.vs;
  const uint8_t* mask = cross_mask(a, b, head, i);
  const int end = cross_end(a, b);
  auto sees = [&](int j) { return j < end && (!mask || mask[j] != 0); };
  auto score = [&](int j) {
    if (!sees(j)) return -INFINITY;
    const float* kr = k + (long long)j * a.ldk;
    float s = 0.f;
    for (int c = 0; c < a.kd; ++c) s = __builtin_fmaf(q[c] * a.scale, kr[c], s);
    return s;
  };
  float top = -INFINITY, sum = 0.f;
  for (int j = lane; j < end; j += 64) top = fmaxf(top, score(j));
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
  for (int j = lane; j < end; j += 64)
    if (sees(j)) sum += expf(score(j) - top);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
  z[0] = z[1] = 0.f;
  for (int j0 = 0; j0 < end; j0 += 64) {
    const int j = j0 + lane;
    const bool seen = sees(j);
    const float e = seen ? expf(score(j) - top) / sum : 0.f;
    for (unsigned long long todo = __ballot(seen); todo; todo &= todo - 1) {
      const int t = __builtin_ctzll(todo);
      const float et = __shfl(e, t);
      const float* vr = v + (long long)(j0 + t) * a.ldv;
#pragma unroll
      for (int x = 0; x < 2; ++x)
        if (lane + 64 * x < a.hd) z[x] = __builtin_fmaf(et, vr[lane + 64 * x], z[x]);
    }
  }
}

// Products of part pairs, the smallest first.
constexpr int kPairA[6] = {2, 1, 0, 1, 0, 0}, kPairB[6] = {0, 1, 2, 0, 1, 0};

// 32 rows (a query and a head of the group that shares the key head) to a wave, NW
// waves to a workgroup, over one piece of the states, 32 at a time.
//
// Both products take float32 operands as three bf16 parts each (attention.hip), six part
// products of nine: no operand's precision depends on another's size.  The workgroup splits
// a tile's keys and values once, into LDS, in the order in which the matrix
// instruction's lanes take them, two tiles in turn: while one is multiplied the next one's
// loads are under way, with one barrier between.
//
// S^T = K Q^T: a lane holds one row's scores (states 8 (r / 4) + 4 half + r % 4), so
// that maximum and sum are in-lane but for one exchange at the end, and the weights are already
// the B operand of O^T = V^T P^T under the state order 8 (e / 4) + 4 half + e % 4 of a
// 16-state step, in which V is laid out.  A row's output factor is its lane's.
//
// The running maximum (Milakov and Gimelshein, 2018) is that of s c, rounded once; weights are
// 2^(s c - m) with one rounding of the exponent.  It moves, and the sums with it, only
// where a score passes it by kSlack: weights reach 2^kSlack until then, which costs
// bf16 parts nothing.
constexpr float kSlack = 8.f;
template <int KS, int DT, int NW>
__global__ __launch_bounds__(NW * 64, NW == 1 ? 1 : 2) void cross_kernel(const CrossArgs a) {
  constexpr int NT = NW * 64;
  constexpr int KU = KS * 64, VU = 2 * DT * 64;  // 8-element units of a tile's keys and values
  constexpr int KI = (KU + NT - 1) / NT, VI = (VU + NT - 1) / NT;
  __shared__ u32x4 frag[2 * (KU + VU) * 3];
  const unsigned item = cross_item();
  if (item >= a.items) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, r32 = lane & 31;
  const int tile = item % a.tiles, rest = item / a.tiles, split = rest % a.splits, plane = rest / a.splits;
  const int b = plane / a.kv, g = plane - b * a.kv;
  const int from = split * a.piece, to = min(from + a.piece, cross_end(a, b));
  const int row = (tile * NW + wave) * 32 + r32, row1 = min(row, a.rows - 1);
  const int qi = row1 / a.group, head = g * a.group + row1 - qi * a.group;
  const float* kb = a.k + (long long)b * a.tk * a.ldk + (long long)g * a.ks;
  const float* vb = a.v + (long long)b * a.tk * a.ldv + (long long)g * a.vs;
  const uint8_t* mask = cross_mask(a, b, head, qi);

  // A tile's units on their way: keys two by two quads, values eight states of a channel.
  f32x4 kr[KI][2];
  float vr[VI][8];
  auto load = [&](int j0) __attribute__((always_inline)) {
    const float* kt = kb + (long long)j0 * a.ldk;
    const float* vt = vb + (long long)j0 * a.ldv;
    const int last = to - 1 - j0;  // states from here on are read from the last visible one
#pragma unroll
    for (int i = 0; i < KI; ++i) {
      const int u = tid + i * NT, oct = u % (2 * KS), r = min(u / (2 * KS), last);
      if (KU % NT != 0 && u >= KU) break;
#pragma unroll
      for (int e = 0; e < 2; ++e) kr[i][e] = *(const f32x4*)(kt + (unsigned)(r * a.ldk + min(8 * oct + 4 * e, a.kd - 4)));
    }
#pragma unroll
    for (int i = 0; i < VI; ++i) {
      const int u = tid + i * NT, f = u >> 6, d = f % DT, st = f / DT;
      if (VU % NT != 0 && u >= VU) break;
      const int c = min(32 * d + r32, a.hd - 1);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        vr[i][e] = vt[(unsigned)(min(16 * st + 8 * (e >> 2) + 4 * half + (e & 3), last) * a.ldv + c)];
    }
  };
  auto stage = [&](u32x4* to_lds) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < KI; ++i) {
      const int u = tid + i * NT, oct = u % (2 * KS), r = u / (2 * KS);
      if (KU % NT != 0 && u >= KU) break;
      bf16x8 p[3];
      parts8(kr[i][0], kr[i][1], p);
      // Lanes of one key write 16 bytes each, 1.5 KB apart: its place within the fragment goes round with them.
      u32x4* at = to_lds + (oct >> 1) * 192 + (oct & 1) * 32 + (r ^ oct);
#pragma unroll
      for (int s = 0; s < 3; ++s) at[s * 64] = __builtin_bit_cast(u32x4, p[s]);
    }
#pragma unroll
    for (int i = 0; i < VI; ++i) {
      const int u = tid + i * NT;
      if (VU % NT != 0 && u >= VU) break;
      bf16x8 p[3];
      parts8(f32x4{vr[i][0], vr[i][1], vr[i][2], vr[i][3]}, f32x4{vr[i][4], vr[i][5], vr[i][6], vr[i][7]}, p);
      u32x4* at = to_lds + KU * 3 + (u >> 6) * 192 + lane;
#pragma unroll
      for (int s = 0; s < 3; ++s) at[s * 64] = __builtin_bit_cast(u32x4, p[s]);
    }
  };

  f32x16 acc[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;
  float mrun = -INFINITY, lrun = 0.f;
  unsigned any = 0;  // the row has a visible state

  if (from < to) {
    load(from);
    bf16x8 q[KS][3];
    {
      const float* qr = a.q + ((long long)b * a.tq + qi) * a.ldq + (long long)head * a.qs;
      const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int c = 16 * ks + 8 * half;
        parts8(c < a.kd ? *(const f32x4*)(qr + c) : zero, c + 4 < a.kd ? *(const f32x4*)(qr + c + 4) : zero, q[ks]);
      }
    }
    stage(frag);
    __syncthreads();
    int now = 0;
    for (int j0 = from; j0 < to; j0 += kCrossKeys, now ^= 1) {
      const bool more = j0 + kCrossKeys < to;
      if (more) load(j0 + kCrossKeys);
      const u32x4* f = frag + now * (KU + VU) * 3;
      unsigned seen[4] = {~0u, ~0u, ~0u, ~0u};
      if (mask) {
        if (j0 + kCrossKeys <= to) {
#pragma unroll
          for (int x = 0; x < 4; ++x) __builtin_memcpy(&seen[x], mask + j0 + 8 * x + 4 * half, 4);
        } else {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            seen[x] = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int j = j0 + 8 * x + 4 * half + e;
              if (j < to) seen[x] |= (unsigned)mask[j] << 8 * e;
            }
          }
        }
      }
      const unsigned some = seen[0] | seen[1] | seen[2] | seen[3];
      any |= some;
      if (__any(some != 0)) {
        f32x16 s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          bf16x8 kp[3];
#pragma unroll
          for (int p = 0; p < 3; ++p)
            kp[p] = __builtin_bit_cast(bf16x8, f[(ks * 3 + p) * 64 + half * 32 + (r32 ^ (2 * ks + half))]);
#pragma unroll
          for (int x = 0; x < 6; ++x)
            s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kp[kPairA[x]], q[ks][kPairB[x]], s, 0, 0, 0);
        }
        if (mask) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (!(seen[r >> 2] >> 8 * (r & 3) & 0xff)) s[r] = -INFINITY;
        }
        if (j0 + kCrossKeys > to) {
          asm volatile("");  // a branch, not 16 selects in every tile
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (j0 + 8 * (r >> 2) + 4 * half + (r & 3) >= to) s[r] = -INFINITY;
        }
        float mx = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
        mx = fmaxf(mx, __shfl_xor(mx, 32)) * a.c;
        if (__any(mx - mrun > kSlack)) {
          mx = fmaxf(mx, mrun);
          const float w = __builtin_amdgcn_exp2f(mrun - (mx == -INFINITY ? 0.f : mx));
          mrun = mx;
          lrun *= w;
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[d][r] *= w;
        }
        const float m = mrun == -INFINITY ? 0.f : mrun;  // no weight yet: all are 0
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.c, -m));
          sum += s[r];
        }
        lrun += sum;
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          bf16x8 p[3];
          parts8(f32x4{s[8 * st], s[8 * st + 1], s[8 * st + 2], s[8 * st + 3]},
                 f32x4{s[8 * st + 4], s[8 * st + 5], s[8 * st + 6], s[8 * st + 7]}, p);
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            bf16x8 vp[3];
#pragma unroll
            for (int x = 0; x < 3; ++x)
              vp[x] = __builtin_bit_cast(bf16x8, f[KU * 3 + ((st * DT + d) * 3 + x) * 64 + lane]);
#pragma unroll
            for (int x = 0; x < 6; ++x)
              acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vp[kPairA[x]], p[kPairB[x]], acc[d], 0, 0, 0);
          }
        }
      }
      if (more) stage(frag + (now ^ 1) * (KU + VU) * 3);
      __syncthreads();
    }
  }

  float l = lrun + __shfl_xor(lrun, 32);
  any |= __shfl_xor((int)any, 32);
  if (any && mrun == -INFINITY && from < to) l = NAN;  // visible, but no finite score: again, in plain float32
  const bool live = row < a.rows;
  if (a.splits > 1) {
    const long long at = ((long long)plane * a.splits + split) * a.rows + row1;
    if (live && half == 0) a.stat[at] = {mrun, l};
    if (live && l != 0.f)
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int c = 32 * d + 8 * x + 4 * half;
          if (c < a.hd)
            *(f32x4*)(a.part + at * a.hd + c) = f32x4{acc[d][4 * x], acc[d][4 * x + 1], acc[d][4 * x + 2], acc[d][4 * x + 3]};
        }
    return;
  }
  float* o = a.o + ((long long)b * a.tq + qi) * a.ldo + (long long)head * a.hd;
  bool again = false;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int c = 32 * d + 8 * x + 4 * half;
      f32x4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        y[e] = l == 0.f ? 0.f : acc[d][4 * x + e] / l;
        again |= live && c < a.hd && !(__builtin_fabsf(y[e]) <= FLT_MAX);
      }
      if (live && c < a.hd) *(f32x4*)(o + c) = y;
    }
  unsigned long long todo = __ballot(again);
  for (todo = (todo | todo >> 32) & 0xffffffffu; todo; todo &= todo - 1) {
    const int t = __builtin_ctzll(todo), ri = __shfl(qi, t), rh = __shfl(head, t);
    float z[2];
    cross_row(a, b, ri, rh, lane, z);
    float* ro = a.o + ((long long)b * a.tq + ri) * a.ldo + (long long)rh * a.hd;
#pragma unroll
    for (int x = 0; x < 2; ++x)
      if (lane + 64 * x < a.hd) ro[lane + 64 * x] = z[x];
  }
}

// Joins the pieces of a row: L lanes to a row, four channels to a lane.
template <int L>
__global__ __launch_bounds__(256) void cross_join_kernel(const CrossArgs a, long long rows) {
  const int lane = threadIdx.x & 63, c = 4 * (threadIdx.x % L);
  const long long at = (long long)blockIdx.x * (256 / L) + threadIdx.x / L;
  const bool live = at < rows;
  const long long plane = min(at, rows - 1) / a.rows;
  const int row = (int)(min(at, rows - 1) - plane * a.rows);
  const int b = (int)(plane / a.kv), g = (int)(plane - (long long)b * a.kv), qi = row / a.group;
  const int head = g * a.group + row - qi * a.group;
  const CrossStat* stat = a.stat + plane * a.splits * a.rows + row;
  const float* part = a.part + (plane * a.splits * a.rows + row) * a.hd + min(c, a.hd - 4);
  float top = -INFINITY;
  for (int x = 0; x < a.splits; ++x) top = fmaxf(top, stat[(long long)x * a.rows].top);
  float sum = 0.f;
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
  for (int x = 0; x < a.splits; ++x) {
    const CrossStat s = stat[(long long)x * a.rows];
    if (s.sum == 0.f) continue;
    const float w = __builtin_amdgcn_exp2f(s.top - top);
    const f32x4 p = *(const f32x4*)(part + (long long)x * a.rows * a.hd);
    sum = __builtin_fmaf(s.sum, w, sum);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = __builtin_fmaf(p[e], w, y[e]);
  }
  bool again = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    y[e] = sum == 0.f ? 0.f : y[e] / sum;
    again |= live && c < a.hd && !(__builtin_fabsf(y[e]) <= FLT_MAX);
  }
  if (live && c < a.hd) *(f32x4*)(a.o + ((long long)b * a.tq + qi) * a.ldo + (long long)head * a.hd + c) = y;
  for (unsigned long long todo = __ballot(again); todo;) {
    const int t = __builtin_ctzll(todo) & ~(L - 1);
    const int rb = __shfl(b, t), ri = __shfl(qi, t), rh = __shfl(head, t);
    float z[2];
    cross_row(a, rb, ri, rh, lane, z);
    float* o = a.o + ((long long)rb * a.tq + ri) * a.ldo + (long long)rh * a.hd;
#pragma unroll
    for (int x = 0; x < 2; ++x)
      if (lane + 64 * x < a.hd) o[lane + 64 * x] = z[x];
    todo &= ~(((1ull << L) - 1) << t);
  }
}

typedef void (*CrossKernel)(const CrossArgs);
template <int NW>
static CrossKernel pick_cross(int kd, int hd) {
  auto by_hd = [&](CrossKernel d1, CrossKernel d2, CrossKernel d4) { return hd <= 32 ? d1 : hd <= 64 ? d2 : d4; };
  if (kd <= 32) return by_hd(cross_kernel<2, 1, NW>, cross_kernel<2, 2, NW>, cross_kernel<2, 4, NW>);
  if (kd <= 64) return by_hd(cross_kernel<4, 1, NW>, cross_kernel<4, 2, NW>, cross_kernel<4, 4, NW>);
  return by_hd(cross_kernel<8, 1, NW>, cross_kernel<8, 2, NW>, cross_kernel<8, 4, NW>);
}

int op_cross_attention(sy_ctx* ctx, const sy_cross_config* c, const sy_tensor* q, const sy_tensor* k,
                       const sy_tensor* v, const int32_t* lengths, const sy_key_mask* mask, const sy_tensor* o) {
  SY_CHECK(c, SY_EINVAL, "null cross attention config");
  SY_CHECK(c->heads > 0 && c->kv_heads > 0 && c->heads % c->kv_heads == 0, SY_EINVAL, "%d heads for %d key heads",
           c->heads, c->kv_heads);
  SY_CHECK(c->key_dim > 0 && c->head_dim > 0, SY_EINVAL, "cross attention head dims %d and %d", c->key_dim, c->head_dim);
  SY_CHECK(c->key_dim % 4 == 0 && c->head_dim % 4 == 0 && c->key_dim <= 128 && c->head_dim <= 128, SY_EUNSUPPORTED,
           "cross attention needs head dims that are multiples of 4 up to 128");
  SY_CHECK(std::isfinite(c->scale) && c->scale > 0, SY_EINVAL, "cross attention scale must be positive and finite");
  SY_CHECK((long long)c->heads * 128 < (1LL << 31), SY_EUNSUPPORTED, "cross attention over %d heads", c->heads);
  CrossArgs a{};
  a.heads = c->heads;
  a.kv = c->kv_heads;
  a.group = c->heads / c->kv_heads;
  a.kd = c->key_dim;
  a.hd = c->head_dim;
  a.qs = c->q_stride ? c->q_stride : a.kd;
  a.ks = c->k_stride ? c->k_stride : a.kd;
  a.vs = c->v_stride ? c->v_stride : a.hd;
  SY_TRY(block_heads(q, a.heads, a.kd, a.qs, "cross attention queries"));
  SY_TRY(block_heads(k, a.kv, a.kd, a.ks, "cross attention keys"));
  SY_TRY(block_heads(v, a.kv, a.hd, a.vs, "cross attention values"));
  SY_TRY(block_heads(o, a.heads, a.hd, a.hd, "cross attention output"));
  SY_CHECK(o->c == a.heads * a.hd && o->n == q->n && o->h == q->h && o->w == q->w, SY_EINVAL,
           "cross attention output shape mismatch");
  SY_CHECK(k->n == q->n && v->n == q->n && v->h == k->h && v->w == k->w, SY_EINVAL,
           "cross attention queries, keys and values differ in n, h or w");
  SY_CHECK(!views_overlap(o, q) && !views_overlap(o, k) && !views_overlap(o, v), SY_EINVAL,
           "cross attention output overlaps an input");
  SY_CHECK(k->ldc < (1 << 24) && v->ldc < (1 << 24), SY_EUNSUPPORTED, "cross attention states of 2^24 channels and more");
  if (mask) {
    SY_CHECK(mask->data, SY_EINVAL, "null mask data");
    SY_CHECK(mask->image >= 0 && mask->head >= 0 && mask->query >= 0, SY_EINVAL, "negative mask stride");
  }
  SY_CHECK((long long)q->n * a.kv < (1 << 24) && (long long)q->h * q->w * a.group < (1LL << 31) - 1024, SY_EUNSUPPORTED,
           "cross attention over %d x %dx%d queries", q->n, q->h, q->w);
  SY_CHECK(ctx, SY_EINVAL, "null context");
  a.q = q->data;
  a.k = k->data;
  a.v = v->data;
  a.o = o->data;
  a.lengths = lengths;
  if (mask) {
    a.mask = mask->data;
    a.mask_image = mask->image;
    a.mask_head = mask->head;
    a.mask_query = mask->query;
  }
  a.ldq = q->ldc;
  a.ldk = k->ldc;
  a.ldv = v->ldc;
  a.ldo = o->ldc;
  a.tq = q->h * q->w;
  a.tk = k->h * k->w;
  a.scale = c->scale;
  a.c = c->scale * 1.4426950408889634f;
  a.rows = a.tq * a.group;
  const long long planes = (long long)q->n * a.kv;
  static const int kNw = getenv("NW") ? atoi(getenv("NW")) : 0;
  const int nw = a.rows <= 64 ? 1 : kNw ? kNw : a.rows <= 128 ? 4 : 8;
  a.tiles = (a.rows + 32 * nw - 1) / (32 * nw);
  const long long whole = planes * a.tiles;
  // Pieces: where the rows alone leave CUs without work, of four tiles and more.
  const long long want = (nw == 1 ? 2048 : nw == 4 ? 768 : 384) / whole;
  a.splits = (int)std::max<long long>(1, std::min<long long>(want, a.tk / (4 * kCrossKeys)));
  a.piece = ((a.tk + a.splits - 1) / a.splits + kCrossKeys - 1) / kCrossKeys * kCrossKeys;
  a.splits = (a.tk + a.piece - 1) / a.piece;
  const long long items = whole * a.splits, grid = (items + 7) / 8 * 8;
  SY_CHECK(grid * nw * 64 < (1LL << 32), SY_EUNSUPPORTED, "cross attention over %lld rows", planes * a.rows);
  a.items = (unsigned)items;
  DeviceScope device(ctx);
  if (a.splits > 1) {
    const size_t rows = (size_t)planes * a.splits * a.rows;
    const size_t stat_at = (sizeof(float) * rows * a.hd + 255) & ~size_t(255);
    SY_TRY(ensure_scratch(ctx, stat_at + sizeof(CrossStat) * rows));
    a.part = (float*)ctx->scratch;
    a.stat = (CrossStat*)(ctx->scratch + stat_at);
  }
  {
    const double scores = (double)q->n * a.heads * a.tq * a.tk;
    ProfScope prof(ctx, "cross_attention", 2 * scores * (a.kd + a.hd),
                   4.0 * q->n * ((double)a.tq * a.heads + (double)a.tk * a.kv) * (a.kd + a.hd));
    CrossKernel kernel = nw == 1 ? pick_cross<1>(a.kd, a.hd) : nw == 4 ? pick_cross<4>(a.kd, a.hd) : pick_cross<8>(a.kd, a.hd);
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(nw * 64), 0, ctx->stream, a);
    SY_TRY(check_launch("cross_attention"));
  }
  if (a.splits > 1) {
    const long long rows = planes * a.rows;
    ProfScope prof(ctx, "cross_join", 0, 4.0 * rows * a.hd * (a.splits + 1));
    if (a.hd <= 64)
      hipLaunchKernelGGL(cross_join_kernel<16>, dim3((unsigned)((rows + 15) / 16)), dim3(256), 0, ctx->stream, a, rows);
    else
      hipLaunchKernelGGL(cross_join_kernel<32>, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, ctx->stream, a, rows);
    SY_TRY(check_launch("cross_join"));
  }
  return SY_OK;
}

}  // namespace sy

extern "C" int sy_cross_attention(sy_ctx* ctx, const sy_cross_config* cfg, const sy_tensor* q, const sy_tensor* k,
                                  const sy_tensor* v, const int32_t* lengths, const sy_key_mask* mask,
                                  const sy_tensor* o) {
  return sy::op_cross_attention(ctx, cfg, q, k, v, lengths, mask, o);
}
