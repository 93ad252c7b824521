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
  int run;              // row tiles of a workgroup that goes through many
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

// A query's channels 16 ks + 8 half .. + 7 of a head, zeros past the last.
template <int KS>
__device__ __forceinline__ void cross_query(const CrossArgs& a, int b, int i, int head, f32x4 (&raw)[KS][2]) {
  const float* q = a.q + ((long long)b * a.tq + i) * a.ldq + (long long)head * a.qs;
  const int half = (threadIdx.x & 63) >> 5;
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int c = 16 * ks + 8 * half + 4 * e;
      raw[ks][e] = c < a.kd ? *(const f32x4*)(q + c) : zero;
    }
}

// What a wave keeps of its 32 rows: the weighted values (channel 32 d + lane % 32 of rows 8 (r / 4)
// + 4 half + r % 4), and of row lane % 32 the maximum, the lane's share of the sum, and whether a
// state was visible.
template <int DT>
struct CrossRows {
  f32x16 acc[DT];
  float top, sum;
  unsigned any;
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[d][r] = 0.f;
    top = -INFINITY;
    sum = 0.f;
    any = 0;
  }
};

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
// bf16 parts nothing.  The largest score's own weight is 2^(s c - m), up to half a step of m beside 1: a factor
// of all weights that the sum takes out again while |m| is below kFar, where it lies between 2^-8 and 2^8.  Farther out
// it could leave no weight at all (or s c is not finite): a row whose maximum ends there is formed again in plain float32,
// which subtracts before it multiplies.  A sum of 0 therefore means that no state was visible.
//
// The six products bound it where head dims are large, and the vector work beside them, which hardly overlaps
// with them: 4096 queries to 8400 states of two images, 16 heads of 128 channels 2.6 ms, 217 TFLOP/s (the
// matrix cores busy 59 per cent of the time, the vector units 27); 300 queries to 8400 masked states of eight
// images, 8 heads of 32 channels 173 us, 119 TFLOP/s (28 and 48: 16 scores of a lane cost 340 vector instructions,
// weights, their parts and the mask, against 24 matrix instructions).
constexpr float kSlack = 8.f, kFar = 0x1p28f;

// Whether weights relative to this maximum, of a row that sees a state, say nothing.
__device__ __forceinline__ bool cross_far(float top) { return !(__builtin_fabsf(top) < kFar); }

// A row's mask bytes of the tile at j0, the lane's states four by four; 0 past `to`.
__device__ __forceinline__ void cross_seen(const uint8_t* mask, int j0, int to, unsigned (&seen)[4]) {
  const int half = (threadIdx.x & 63) >> 5;
  if (j0 + kCrossKeys <= to) {
#pragma unroll
    for (int x = 0; x < 4; ++x) __builtin_memcpy(&seen[x], mask + j0 + 8 * x + 4 * half, 4);
    return;
  }
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

// One tile: states j0 .. j0 + 31 up to `to`.  key(ks, p) and value(i, p) give their parts, then() follows the last
// of the keys.  seen: the tile's mask bytes, where there are any.
template <int KS, int DT, class Key, class Value, class Then>
__device__ __forceinline__ void cross_tile(const CrossArgs& a, Key key, Value value, Then then, int j0, int to,
                                           const unsigned (&seen)[4], const bf16x8 (&q)[KS][3], CrossRows<DT>& w) {
  const int half = (threadIdx.x & 63) >> 5;
  if (a.mask) {
    const unsigned some = seen[0] | seen[1] | seen[2] | seen[3];
    w.any |= some;
    if (!__any(some != 0)) return then();
  } else {
    w.any = 1;
  }
  // Fragments are read a step ahead of the products that take them.
  f32x16 s;
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] = 0.f;
  bf16x8 kp[2][3];
  key(0, kp[0]);
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    if (ks + 1 < KS) key(ks + 1, kp[(ks + 1) & 1]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int x = 0; x < 6; ++x)
      s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kp[ks & 1][kPairA[x]], q[ks][kPairB[x]], s, 0, 0, 0);
  }
  then();
  bf16x8 vp[2][3];
  value(0, vp[0]);
  if (a.mask) {
    // The top bit of every byte that is not 0, spread over a word, picks the score.
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const unsigned t = ((seen[x] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | seen[x];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned keep = (unsigned)((int)(t << (24 - 8 * e)) >> 31);
        const float score = s[4 * x + e];
        const unsigned bits = (keep & __builtin_bit_cast(unsigned, score)) | (~keep & 0xff800000u);
        s[4 * x + e] = __builtin_bit_cast(float, bits);
      }
    }
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
  {
    const unsigned bits = __builtin_bit_cast(unsigned, mx);
    const auto both = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);  // the row's other half, without LDS
    const unsigned low = both[0], high = both[1];
    mx = fmaxf(__builtin_bit_cast(float, low), __builtin_bit_cast(float, high)) * a.c;
  }
  const bool move = mx - w.top > kSlack;  // row by row, so that no row's bits hang on another's scores
  if (__any(move)) {
    const float x = move ? __builtin_amdgcn_exp2f(w.top - mx) : 1.f;
    const bool before = __any(w.top != -INFINITY);
    w.top = move ? mx : w.top;
    w.sum *= x;
    if (before)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float xr = __shfl(x, 8 * (r >> 2) + 4 * half + (r & 3));
#pragma unroll
        for (int d = 0; d < DT; ++d) w.acc[d][r] *= xr;
      }
  }
  const float m = w.top == -INFINITY ? 0.f : w.top;  // no weight yet: all are 0
  float sum = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.c, -m));
    sum += s[r];
  }
  w.sum += sum;
#pragma unroll
  for (int st = 0; st < 2; ++st) {
    bf16x8 p[3];
    parts8(f32x4{s[8 * st], s[8 * st + 1], s[8 * st + 2], s[8 * st + 3]},
           f32x4{s[8 * st + 4], s[8 * st + 5], s[8 * st + 6], s[8 * st + 7]}, p);
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      const int i = st * DT + d;
      if (i + 1 < 2 * DT) value(i + 1, vp[(i + 1) & 1]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int x = 0; x < 6; ++x)
        w.acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(p[kPairA[x]], vp[i & 1][kPairB[x]], w.acc[d], 0, 0, 0);
    }
  }
}

// A tile whose parts are in LDS, at f.
template <int KS, int DT>
__device__ __forceinline__ void cross_tile(const CrossArgs& a, const u32x4* f, int j0, int to, const unsigned (&seen)[4],
                                           const bf16x8 (&q)[KS][3], CrossRows<DT>& w) {
  const int lane = threadIdx.x & 63, half = lane >> 5, r32 = lane & 31;
  const u32x4* v = f + KS * 192 + lane;
  auto key = [&](int ks, bf16x8(&k)[3]) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < 3; ++x)
      k[x] = __builtin_bit_cast(bf16x8, f[(ks * 3 + x) * 64 + half * 32 + (r32 ^ (2 * ks + half))]);
  };
  auto value = [&](int i, bf16x8(&p)[3]) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < 3; ++x) p[x] = __builtin_bit_cast(bf16x8, v[(i * 3 + x) * 64]);
  };
  cross_tile<KS, DT>(a, key, value, [] {}, j0, to, seen, q, w);
}

// The outputs of 32 rows from row0, or what a piece leaves for them, in whole lines of
// memory.  states: the piece has any.
template <int DT>
__device__ __forceinline__ void cross_finish(const CrossArgs& a, const CrossRows<DT>& w, int plane, int split, int row0,
                                             bool states) {
  const int lane = threadIdx.x & 63, half = lane >> 5, r32 = lane & 31;
  const int b = plane / a.kv, g = plane - b * a.kv, row1 = min(row0 + r32, a.rows - 1);
  float l = w.sum + __shfl_xor(w.sum, 32);
  const unsigned any = w.any | (unsigned)__shfl_xor((int)w.any, 32);
  if (any && states && cross_far(w.top)) l = NAN;  // visible, but no finite score or a far one: again, in plain float32
  // Where row 0 of the tile goes, and how far row1 is from it.
  float* out;
  long long step, mine;  // floats from row to row; to row1, where they differ
  if (a.splits > 1) {
    const long long at = ((long long)plane * a.splits + split) * a.rows + row0;
    if (half == 0 && row0 + r32 < a.rows) a.stat[at + r32] = {w.top, l};
    out = a.part + at * a.hd;
    step = a.hd;
    mine = 0;
  } else {
    const int qi = row1 / a.group;
    out = a.o + (long long)b * a.tq * a.ldo + (long long)g * a.group * a.hd;
    step = a.ldo;
    mine = qi * a.ldo + (long long)(row1 - qi * a.group) * a.hd;
    if (a.group == 1) out += row0 * a.ldo;
  }
  const float factor = a.splits > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;  // 0: there is nothing to weigh
  float f[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) f[r] = __shfl(factor, 8 * (r >> 2) + 4 * half + (r & 3));
  float odd = 0.f;  // not 0 where a value is not finite
  if ((a.splits > 1 || a.group == 1) && row0 + 32 <= a.rows) {
    float* at = out + 4 * half * step + r32;
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      if (32 * d + r32 >= a.hd) break;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float y = w.acc[d][r] * f[r];
        odd = __builtin_fmaf(y, 0.f, odd);
        __builtin_nontemporal_store(y, at + (8 * (r >> 2) + (r & 3)) * step + 32 * d);
      }
    }
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int at = 8 * (r >> 2) + (r & 3), row = at + 4 * half;
      const long long off =
          a.splits > 1 || a.group == 1
              ? row * step
              : (long long)(unsigned)__shfl((int)mine, row) | (long long)__shfl((int)(mine >> 32), row) << 32;
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const float y = w.acc[d][r] * f[r];
        if (32 * d + r32 < a.hd && row0 + row < a.rows) {
          odd = __builtin_fmaf(y, 0.f, odd);
          __builtin_nontemporal_store(y, out + off + 32 * d + r32);
        }
      }
    }
  }
  if (a.splits > 1 || !__any(odd != 0.f)) return;
  unsigned again = 0;  // rows with such a value
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int at = 8 * (r >> 2) + (r & 3);
    bool bad = false;
#pragma unroll
    for (int d = 0; d < DT; ++d) bad |= !(__builtin_fabsf(w.acc[d][r] * f[r]) <= FLT_MAX);
    const unsigned long long who = __ballot(bad);
    again |= ((unsigned)who != 0 ? 1u : 0u) << at | ((who >> 32) != 0 ? 1u : 0u) << (at + 4);
  }
  for (; again; again &= again - 1) {
    const int t = __builtin_ctz(again);
    if (row0 + t >= a.rows) return;
    const int ri = (row0 + t) / a.group, rh = g * a.group + row0 + t - ri * a.group;
    float* ro = a.o + ((long long)b * a.tq + ri) * a.ldo + (long long)rh * a.hd;
    float z[2];
    cross_row(a, b, ri, rh, lane, z);
#pragma unroll
    for (int x = 0; x < 2; ++x)
      if (lane + 64 * x < a.hd) ro[lane + 64 * x] = z[x];
  }
}

// States on their way to LDS: NT threads take 8-element units of SUB tiles, keys as two
// quads of a row, values as eight states of a channel, split them and put them down in the
// order in which the matrix instruction's lanes take them.
template <int KS, int DT, int NT, int SUB>
struct CrossStage {
  static constexpr int TILE = (KS + 2 * DT) * 192;  // 16-byte units of a tile
  static constexpr int KU = SUB * KS * 64, VU = SUB * 2 * DT * 64;
  static constexpr int KI = (KU + NT - 1) / NT, VI = (VU + NT - 1) / NT;
  f32x4 kr[KI][2];
  float vr[VI][8];
  // Where the keys do not keep every thread busy the values begin with those that are left.
  static __device__ __forceinline__ int value_tid() {
    return KU % NT ? (int)(threadIdx.x + NT - KU % NT) % NT : (int)threadIdx.x;
  }
  // The tiles at j0 of a head's keys and values; past `to` the last state is read again.
  __device__ __forceinline__ void load(const CrossArgs& a, const float* kb, const float* vb, int j0, int to) {
    const int half = (threadIdx.x & 63) >> 5, r32 = threadIdx.x & 31;
    const float* kt = kb + (long long)j0 * a.ldk;
    const float* vt = vb + (long long)j0 * a.ldv;
    const int last = to - 1 - j0;
#pragma unroll
    for (int i = 0; i < KI; ++i) {
      const int u = threadIdx.x + i * NT, oct = u % (2 * KS), r = min(u / (2 * KS), last);
      if (KU % NT != 0 && u >= KU) break;
#pragma unroll
      for (int e = 0; e < 2; ++e)
        kr[i][e] = *(const f32x4*)(kt + (unsigned)(r * a.ldk + min(8 * oct + 4 * e, a.kd - 4)));
    }
#pragma unroll
    for (int i = 0; i < VI; ++i) {
      const int u = value_tid() + i * NT, f = u >> 6, d = f % DT, st = f / DT;
      if (VU % NT != 0 && u >= VU) break;
      const int c = min(32 * d + r32, a.hd - 1);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        vr[i][e] = vt[(unsigned)(min(16 * st + 8 * (e >> 2) + 4 * half + (e & 3), last) * a.ldv + c)];
    }
  }
  __device__ __forceinline__ void put(u32x4* lds) const {
#pragma unroll
    for (int i = 0; i < KI; ++i) {
      const int u = threadIdx.x + i * NT, oct = u % (2 * KS), r = u / (2 * KS);
      if (KU % NT != 0 && u >= KU) break;
      bf16x8 p[3];
      parts8(kr[i][0], kr[i][1], p);
      // Lanes of one key write 16 bytes each, 1.5 KB apart: its place within the fragment goes round with them.
      u32x4* at = lds + (r >> 5) * TILE + (oct >> 1) * 192 + (oct & 1) * 32 + ((r & 31) ^ oct);
#pragma unroll
      for (int s = 0; s < 3; ++s) at[s * 64] = __builtin_bit_cast(u32x4, p[s]);
    }
#pragma unroll
    for (int i = 0; i < VI; ++i) {
      const int u = value_tid() + i * NT, f = u >> 6, sub = f / (2 * DT);
      if (VU % NT != 0 && u >= VU) break;
      bf16x8 p[3];
      parts8(f32x4{vr[i][0], vr[i][1], vr[i][2], vr[i][3]}, f32x4{vr[i][4], vr[i][5], vr[i][6], vr[i][7]}, p);
      u32x4* at = lds + sub * TILE + KS * 192 + (f - sub * 2 * DT) * 192 + (u & 63);
#pragma unroll
      for (int s = 0; s < 3; ++s) at[s * 64] = __builtin_bit_cast(u32x4, p[s]);
    }
  }
};

template <int KS, int DT, int NW>
__global__ __launch_bounds__(NW * 64, 2) void cross_kernel(const CrossArgs a) {
  typedef CrossStage<KS, DT, NW * 64, 1> Stage;
  __shared__ u32x4 frag[2][Stage::TILE];
  const unsigned item = cross_item();
  if (item >= a.items) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tile = item % a.tiles, rest = item / a.tiles, split = rest % a.splits, plane = rest / a.splits;
  const int b = plane / a.kv, g = plane - b * a.kv;
  const int from = split * a.piece, to = min(from + a.piece, cross_end(a, b));
  const int row = (tile * NW + wave) * 32 + (threadIdx.x & 31), row1 = min(row, a.rows - 1);
  const int qi = row1 / a.group, head = g * a.group + row1 - qi * a.group;
  const float* kb = a.k + (long long)b * a.tk * a.ldk + (long long)g * a.ks;
  const float* vb = a.v + (long long)b * a.tk * a.ldv + (long long)g * a.vs;
  const uint8_t* mask = cross_mask(a, b, head, qi);
  const bool some = (tile * NW + wave) * 32 < a.rows;  // the wave has rows
  CrossRows<DT> rows;
  rows.clear();
  if (from < to) {
    Stage stage;
    stage.load(a, kb, vb, from, to);
    bf16x8 q[KS][3];
    {
      f32x4 raw[KS][2];
      cross_query<KS>(a, b, qi, head, raw);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) parts8(raw[ks][0], raw[ks][1], q[ks]);
    }
    stage.put(frag[0]);
    // Mask bytes are loaded ahead, too, where there are registers for them.
    constexpr bool AHEAD = KS + 2 * DT < 16;
    unsigned next[4];
    if (AHEAD && mask) cross_seen(mask, from, to, next);
    __syncthreads();
    int now = 0;
    for (int j0 = from; j0 < to; j0 += kCrossKeys, now ^= 1) {
      const bool more = j0 + kCrossKeys < to;
      if (!AHEAD && mask) cross_seen(mask, j0, to, next);
      unsigned seen[4] = {next[0], next[1], next[2], next[3]};
      if (more) {
        if (AHEAD && mask) cross_seen(mask, j0 + kCrossKeys, to, next);
        stage.load(a, kb, vb, j0 + kCrossKeys, to);
      }
      if (some) cross_tile<KS, DT>(a, frag[now], j0, to, seen, q, rows);
      if (more) stage.put(frag[now ^ 1]);
      __syncthreads();
    }
  }
  cross_finish<DT>(a, rows, plane, split, (tile * NW + wave) * 32, from < to);
}

// Few states: a workgroup splits all of them once and goes through many rows, its
// waves on their own, the next rows' queries under way.  25600 queries to 77 states of four images, 8 heads of 64
// channels 132 us, 3.2 TB/s (outputs go past the caches, in whole lines): without any state it is 92, memory; the products and
// weights do not run under that (matrix cores busy 26 per cent of the time, vector units 32).
constexpr int kShortLds = 150 * 1024, kShortWaves = 4;
constexpr int short_bytes(int ks, int dt) { return (ks + 2 * dt) * 192 * 16; }  // of a tile
template <int KS, int DT>
__global__ __launch_bounds__(kShortWaves * 64, KS >= 5 ? 1 : 2) void cross_short_kernel(const CrossArgs a) {
  constexpr int NW = kShortWaves;
  typedef CrossStage<KS, DT, NW * 64, 1> Stage;
  extern __shared__ u32x4 frag[];
  // Images' lengths differ: every XCD takes workgroups of all of them.
  const int planes = a.items / a.tiles;  // tiles: runs of row tiles here
  if (blockIdx.x >= a.items) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r32 = threadIdx.x & 31;
  const int run = blockIdx.x / planes, plane = blockIdx.x - run * planes;
  const int b = plane / a.kv, g = plane - b * a.kv, to = cross_end(a, b);
  const float* kb = a.k + (long long)b * a.tk * a.ldk + (long long)g * a.ks;
  const float* vb = a.v + (long long)b * a.tk * a.ldv + (long long)g * a.vs;
  const int first = run * a.run, last = min(first + a.run, (a.rows + 31) / 32);
  auto place = [&](int tile, int& qi, int& head) {
    const int row = min(tile * 32 + r32, a.rows - 1);
    qi = row / a.group;
    head = g * a.group + row - qi * a.group;
  };
  int qi, head;
  f32x4 raw[KS][2];
  place(min(first + wave, last - 1), qi, head);
  {
    Stage stage;
    if (to > 0) stage.load(a, kb, vb, 0, to);
    cross_query<KS>(a, b, qi, head, raw);
    for (int j0 = 0; j0 < to; j0 += kCrossKeys) {
      stage.put(frag + j0 / kCrossKeys * Stage::TILE);
      if (j0 + kCrossKeys < to) stage.load(a, kb, vb, j0 + kCrossKeys, to);
    }
  }
  __syncthreads();
  bf16x8 q[KS][3];
  auto split = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) parts8(raw[ks][0], raw[ks][1], q[ks]);
  };
  split();
  for (int tile = first + wave; tile < last; tile += NW) {
    const uint8_t* mask = cross_mask(a, b, head, qi);
    if (tile + NW < last) {
      place(tile + NW, qi, head);
      cross_query<KS>(a, b, qi, head, raw);
    }
    CrossRows<DT> rows;
    rows.clear();
    for (int j0 = 0; j0 < to; j0 += kCrossKeys) {
      unsigned seen[4];
      if (mask) cross_seen(mask, j0, to, seen);
      cross_tile<KS, DT>(a, frag + j0 / kCrossKeys * Stage::TILE, j0, to, seen, q, rows);
    }
    split();  // before the stores: waiting for loads behind them would wait for them, too
    cross_finish<DT>(a, rows, plane, 0, tile * 32, to > 0);
  }
}

// Little work: 32 rows to a workgroup, and every fourth of their tiles to each of its waves, which take the states
// straight into the order of the matrix instruction's lanes and split them for themselves: no barrier, and
// no tile waits for another's loads.  What the waves hold meets in LDS at the end.  Latency bounds it: 400 queries to 77
// states, 8 heads of 32 channels 5.8 us, 4 of them the launch.
constexpr int kLoneWaves = 4;
template <int KS, int DT>
__global__ __launch_bounds__(kLoneWaves * 64, KS + 2 * DT <= 8 && KS < 6 ? 2 : 1) void cross_lone_kernel(const CrossArgs a) {
  constexpr int NW = kLoneWaves;
  __shared__ f32x4 others[NW - 1][DT * 4][64];
  __shared__ float tops[NW][32], sums[NW][32];
  __shared__ unsigned seens[NW][32];
  const unsigned item = cross_item();
  if (item >= a.items) return;
  const int lane = threadIdx.x & 63, half = lane >> 5, r32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tile = item % a.tiles, plane = item / a.tiles;
  const int b = plane / a.kv, g = plane - b * a.kv, to = cross_end(a, b);
  const int row1 = min(tile * 32 + r32, a.rows - 1), qi = row1 / a.group, head = g * a.group + row1 - qi * a.group;
  const float* kb = a.k + (long long)b * a.tk * a.ldk + (long long)g * a.ks;
  const float* vb = a.v + (long long)b * a.tk * a.ldv + (long long)g * a.vs;
  const uint8_t* mask = cross_mask(a, b, head, qi);
  f32x4 kr[KS][2];
  float vr[2 * DT][8];
  auto load_k = [&](int j0) __attribute__((always_inline)) {
    const float* k = kb + (long long)min(j0 + r32, to - 1) * a.ldk;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int e = 0; e < 2; ++e) kr[ks][e] = *(const f32x4*)(k + min(16 * ks + 8 * half + 4 * e, a.kd - 4));
  };
  auto load_v = [&](int j0) __attribute__((always_inline)) {
    const float* v = vb + (long long)j0 * a.ldv;
    const int last = to - 1 - j0;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float* at = v + (unsigned)(min(8 * (e >> 2) + 4 * half + (e & 3), last) * a.ldv);
#pragma unroll
      for (int d = 0; d < DT; ++d) vr[(e >> 3) * DT + d][e & 7] = at[min(32 * d + r32, a.hd - 1)];
    }
  };
  CrossRows<DT> rows;
  rows.clear();
  int j0 = wave * kCrossKeys;
  if (j0 < to) {
    bf16x8 q[KS][3];
    f32x4 raw[KS][2];
    cross_query<KS>(a, b, qi, head, raw);
    load_k(j0);
    load_v(j0);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) parts8(raw[ks][0], raw[ks][1], q[ks]);
    do {
      const int next = j0 + NW * kCrossKeys;
      unsigned seen[4];
      if (mask) cross_seen(mask, j0, to, seen);
      cross_tile<KS, DT>(
          a,
          [&](int ks, bf16x8(&p)[3]) __attribute__((always_inline)) { parts8(kr[ks][0], kr[ks][1], p); },
          [&](int i, bf16x8(&p)[3]) __attribute__((always_inline)) {
            parts8(f32x4{vr[i][0], vr[i][1], vr[i][2], vr[i][3]}, f32x4{vr[i][4], vr[i][5], vr[i][6], vr[i][7]}, p);
          },
          [&]() __attribute__((always_inline)) {
            if (next < to) load_k(next);
          },
          j0, to, seen, q, rows);
      if (next < to) load_v(next);
      j0 = next;
    } while (j0 < to);
  }
  // The waves' maxima, then their sums on the common one.
  const unsigned any = rows.any | (unsigned)__shfl_xor((int)rows.any, 32);
  const float sum = rows.sum + __shfl_xor(rows.sum, 32);
  if (half == 0) {
    tops[wave][r32] = rows.top;
    sums[wave][r32] = sum;
    seens[wave][r32] = any;
  }
  __syncthreads();
  float top = tops[0][r32], l = 0.f;
  unsigned all = 0;
#pragma unroll
  for (int w = 1; w < NW; ++w) top = fmaxf(top, tops[w][r32]);
  // A NaN keeps its place in the sum: its factor is 0, 1 or NaN.
  auto share = [&](float t) { return t == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(t - top); };
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    l = __builtin_fmaf(sums[w][r32], share(tops[w][r32]), l);
    all |= seens[w][r32];
  }
  const float x = share(rows.top);
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const float xr = __shfl(x, 8 * (r >> 2) + 4 * half + (r & 3));
#pragma unroll
    for (int d = 0; d < DT; ++d) rows.acc[d][r] *= xr;
  }
  if (wave > 0) {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        others[wave - 1][4 * d + i][lane] =
            f32x4{rows.acc[d][4 * i], rows.acc[d][4 * i + 1], rows.acc[d][4 * i + 2], rows.acc[d][4 * i + 3]};
  }
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int w = 0; w < NW - 1; ++w) {
        const f32x4 t = others[w][4 * d + i][lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) rows.acc[d][4 * i + e] += t[e];
      }
  rows.top = top;
  rows.sum = half == 0 ? l : 0.f;
  rows.any = all;
  cross_finish<DT>(a, rows, plane, 0, tile * 32, to > 0);
}

// v summed over aligned groups of 16 lanes, in each of them.
__device__ __forceinline__ float plus16(float v) {
#define SY_PLUS(ctrl) v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl, 0xf, 0xf, false))
  SY_PLUS(0xb1);   // lane ^ 1
  SY_PLUS(0x4e);   // lane ^ 2
  SY_PLUS(0x141);  // 7 - lane
  SY_PLUS(0x140);  // 15 - lane
#undef SY_PLUS
  return v;
}

// Few rows (a token's query): up to G rows of an image and key head, in plain float32.
// 16 lanes take a state, 4 C channels each, and go through every 16th state of
// the piece with a maximum and sums of their own; the workgroup's 16 meet at the end.  Memory bounds it, the states being
// read once: a token of 32 images to up to 1500 states, 8 heads of 64 channels 28 us, 4.4 TB/s.
template <int C, int G>
__global__ __launch_bounds__(256) void cross_few_kernel(const CrossArgs a) {
  constexpr int U = G * C >= 8 ? 4 : 8;  // states under way
  __shared__ f32x4 O[4][G][16 * C];
  __shared__ CrossStat S[4][G];
  const unsigned item = cross_item();
  if (item >= a.items) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = tid & 15;
  const int split = item % a.splits, plane = item / a.splits, b = plane / a.kv, g = plane - b * a.kv;
  const int from = split * a.piece, to = min(from + a.piece, cross_end(a, b));
  const float* kb = a.k + (long long)b * a.tk * a.ldk + (long long)g * a.ks;
  const float* vb = a.v + (long long)b * a.tk * a.ldv + (long long)g * a.vs;
  int kc[C], vc[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    kc[c] = min(64 * c + 4 * l16, a.kd - 4);
    vc[c] = min(64 * c + 4 * l16, a.hd - 4);
  }
  f32x4 q[G][C], acc[G][C];
  float top[G], sum[G];
  const uint8_t* mask[G];
#pragma unroll
  for (int r = 0; r < G; ++r) {
    const int row = min(r, a.rows - 1), qi = row / a.group, head = g * a.group + row - qi * a.group;
    const float* qr = a.q + ((long long)b * a.tq + qi) * a.ldq + (long long)head * a.qs;
    mask[r] = cross_mask(a, b, head, qi);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      q[r][c] = 64 * c + 4 * l16 < a.kd ? *(const f32x4*)(qr + kc[c]) : f32x4{0.f, 0.f, 0.f, 0.f};
      acc[r][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    top[r] = -INFINITY;
    sum[r] = 0.f;
  }
  unsigned any = 0;
  for (int j0 = from + (tid >> 4); j0 < to; j0 += 16 * U) {
    f32x4 k[U][C], v[U][C];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const long long j = min(j0 + 16 * u, to - 1);
        k[u][c] = *(const f32x4*)(kb + j * a.ldk + kc[c]);
        v[u][c] = *(const f32x4*)(vb + j * a.ldv + vc[c]);
      }
    uint8_t seen[G][U];
    if (a.mask)
#pragma unroll
      for (int r = 0; r < G; ++r)
#pragma unroll
        for (int u = 0; u < U; ++u) seen[r][u] = mask[r][min(j0 + 16 * u, to - 1)];
#pragma unroll
    for (int r = 0; r < G; ++r) {
      float s[U], mx = -INFINITY;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float t = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) t = __builtin_fmaf(q[r][c][e], k[u][c][e], t);
        t = plus16(t);
        const bool sees = j0 + 16 * u < to && (!a.mask || seen[r][u] != 0);
        any |= (unsigned)sees << r;
        s[u] = sees ? t : -INFINITY;
        mx = fmaxf(mx, s[u]);
      }
      mx *= a.c;
      if (mx > top[r]) {
        const float x = __builtin_amdgcn_exp2f(top[r] - mx);
        top[r] = mx;
        sum[r] *= x;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[r][c][e] *= x;
      }
      const float m = top[r] == -INFINITY ? 0.f : top[r];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u], a.c, -m));
        sum[r] += p;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[r][c][e] = __builtin_fmaf(p, v[u][c][e], acc[r][c][e]);
      }
    }
  }
  // The wave's four, then the workgroup's waves.
#pragma unroll
  for (int r = 0; r < G; ++r) {
    float t = fmaxf(top[r], __shfl_xor(top[r], 16));
    t = fmaxf(t, __shfl_xor(t, 32));
    const float x = top[r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top[r] - t);
    // A NaN keeps its place in the sum: x is 1 then or NaN itself.
    sum[r] *= x;
    sum[r] += __shfl_xor(sum[r], 16);
    sum[r] += __shfl_xor(sum[r], 32);
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        acc[r][c][e] *= x;
        acc[r][c][e] += __shfl_xor(acc[r][c][e], 16);
        acc[r][c][e] += __shfl_xor(acc[r][c][e], 32);
      }
      if (lane < 16) O[wave][r][16 * c + l16] = acc[r][c];
    }
    const bool seen = __any(any >> r & 1);
    if (lane == 0) S[wave][r] = {t, seen && t == -INFINITY ? NAN : sum[r]};
  }
  __syncthreads();
  for (int r = wave; r < min(G, a.rows); r += 4) {
    const int qi = r / a.group, head = g * a.group + r - qi * a.group;
    float t = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) t = fmaxf(t, S[w][r].top);
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (S[w][r].sum == 0.f) continue;
      const float x = __builtin_amdgcn_exp2f(S[w][r].top - t);
      l = __builtin_fmaf(S[w][r].sum, x, l);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = __builtin_fmaf(O[w][r][min(lane, 16 * C - 1)][e], x, y[e]);
    }
    if (t != -INFINITY && cross_far(t)) l = NAN;  // -inf: nothing visible, or NaN already
    const bool live = lane < 16 * C && 4 * lane < a.hd;
    if (a.splits > 1) {
      const long long at = ((long long)plane * a.splits + split) * a.rows + r;
      if (lane == 0) a.stat[at] = {t, l};
      if (live) *(f32x4*)(a.part + at * a.hd + 4 * lane) = y;
      continue;
    }
    float* o = a.o + ((long long)b * a.tq + qi) * a.ldo + (long long)head * a.hd;
    bool again = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      y[e] = l == 0.f ? 0.f : y[e] / l;
      again |= live && !(__builtin_fabsf(y[e]) <= FLT_MAX);
    }
    if (live) *(f32x4*)(o + 4 * lane) = y;
    if (__any(again)) {
      float z[2];
      cross_row(a, b, qi, head, lane, z);
#pragma unroll
      for (int x = 0; x < 2; ++x)
        if (lane + 64 * x < a.hd) o[lane + 64 * x] = z[x];
    }
  }
}

// Joins the pieces of a row (about 4 us, most of it the launch), W lanes to a row: L of them take four channels each of
// every (W / L)-th piece.
template <int L, int W>
__global__ __launch_bounds__(256) void cross_join_kernel(const CrossArgs a, long long rows) {
  constexpr int SG = W / L;
  const int lane = threadIdx.x & 63, l = lane & (W - 1), c = 4 * (l % L), sg = l / L;
  const long long at = (long long)blockIdx.x * (256 / W) + threadIdx.x / W;
  const bool here = at < rows;
  const long long at1 = here ? at : rows - 1, plane = at1 / a.rows;
  const int row = (int)(at1 - plane * a.rows);
  const int b = (int)(plane / a.kv), g = (int)(plane - (long long)b * a.kv), qi = row / a.group;
  const int head = g * a.group + row - qi * a.group;
  const CrossStat* stat = a.stat + plane * a.splits * a.rows + row;
  const float* part = a.part + (plane * a.splits * a.rows + row) * a.hd + min(c, a.hd - 4);
  float top = -INFINITY;
  for (int x = l; x < a.splits; x += W) top = fmaxf(top, stat[(long long)x * a.rows].top);
#pragma unroll
  for (int off = W / 2; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
  float sum = 0.f;
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int x = sg; x < a.splits; x += SG) {
    const CrossStat s = stat[(long long)x * a.rows];
    const f32x4 p = *(const f32x4*)(part + (long long)x * a.rows * a.hd);
    const bool none = s.sum == 0.f;  // nothing was left there then
    const float w = __builtin_amdgcn_exp2f(s.top - top);
    sum = none ? sum : __builtin_fmaf(s.sum, w, sum);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = none ? y[e] : __builtin_fmaf(p[e], w, y[e]);
  }
#pragma unroll
  for (int off = L; off < W; off <<= 1) {
    sum += __shfl_xor(sum, off);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] += __shfl_xor(y[e], off);
  }
  if (top != -INFINITY && cross_far(top)) sum = NAN;  // a piece whose weights came to 0 may hold it
  const bool live = here && l < L && c < a.hd;
  bool again = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    y[e] = sum == 0.f ? 0.f : y[e] / sum;
    again |= live && !(__builtin_fabsf(y[e]) <= FLT_MAX);
  }
  if (live) *(f32x4*)(a.o + ((long long)b * a.tq + qi) * a.ldo + (long long)head * a.hd + c) = y;
  for (unsigned long long todo = __ballot(again); todo;) {
    const int t = __builtin_ctzll(todo) & ~(W - 1);
    const int rb = __shfl(b, t), ri = __shfl(qi, t), rh = __shfl(head, t);
    float* o = a.o + ((long long)rb * a.tq + ri) * a.ldo + (long long)rh * a.hd;
    float z[2];
    cross_row(a, rb, ri, rh, lane, z);
#pragma unroll
    for (int x = 0; x < 2; ++x)
      if (lane + 64 * x < a.hd) o[lane + 64 * x] = z[x];
    todo &= W == 64 ? 0 : ~(((1ull << (W & 63)) - 1) << t);
  }
}

typedef void (*CrossKernel)(const CrossArgs);
#define SY_CROSS_DT(kernel, KS, ...)                       \
  (dt == 1   ? kernel<KS, 1 __VA_ARGS__>                  \
   : dt == 2 ? kernel<KS, 2 __VA_ARGS__>                  \
   : dt == 3 ? kernel<KS, 3 __VA_ARGS__>                  \
             : kernel<KS, 4 __VA_ARGS__>)
#define SY_CROSS_PICK(kernel, ...)                         \
  (ks == 2   ? SY_CROSS_DT(kernel, 2, __VA_ARGS__)        \
   : ks == 3 ? SY_CROSS_DT(kernel, 3, __VA_ARGS__)        \
   : ks == 4 ? SY_CROSS_DT(kernel, 4, __VA_ARGS__)        \
   : ks == 5 ? SY_CROSS_DT(kernel, 5, __VA_ARGS__)        \
   : ks == 6 ? SY_CROSS_DT(kernel, 6, __VA_ARGS__)        \
             : SY_CROSS_DT(kernel, 8, __VA_ARGS__))
#define SY_COMMA ,
template <int NW>
static CrossKernel pick_cross(int ks, int dt) {
  return SY_CROSS_PICK(cross_kernel, SY_COMMA NW);
}
static CrossKernel pick_short(int ks, int dt) { return SY_CROSS_PICK(cross_short_kernel); }
static CrossKernel pick_lone(int ks, int dt) { return SY_CROSS_PICK(cross_lone_kernel); }
#undef SY_COMMA
#undef SY_CROSS_PICK
#undef SY_CROSS_DT
static CrossKernel pick_few(int kd, int hd, int rows) {
  if (std::max(kd, hd) <= 64)
    return rows == 1 ? cross_few_kernel<1, 1> : rows == 2 ? cross_few_kernel<1, 2> : cross_few_kernel<1, 4>;
  return rows == 1 ? cross_few_kernel<2, 1> : rows == 2 ? cross_few_kernel<2, 2> : cross_few_kernel<2, 4>;
}

// Waves of a workgroup and pieces of the states: the least estimated time, in cycles.  A wave's
// tile takes 192 (ks + 2 dt) of the matrix cores, about 850 of other vector work and its share of
// splitting the states (200 (ks + 2 dt)); the waves of a SIMD overlap by a quarter; loads and barrier take 2,500 (of
// eight waves 3,200) anyway.  Whether each wave takes tiles for itself instead (cross_lone_kernel), with no overlap:
// 400 rows of 8 heads of 32 to 77 states 6.2 us so, 7.6 not, 450 rows of 12 key heads to 171 10.7 and 15.8, 536 rows of 12 to
// 213 9.8 and 15.3, but 800 rows of one to 2000 35 and 16.
static void cross_plan(CrossArgs& a, int ks, int dt, long long planes, long long row_tiles, int* nw, bool* lone) {
  const int cus = 256, s = ks + 2 * dt;
  const long long key_tiles = (a.tk + kCrossKeys - 1) / kCrossKeys;
  double best = INFINITY;
  for (int w : {4, 8}) {
    // Workgroups to a CU, as their registers allow.
    const int there = w == 8 || s >= 14 ? 1 : s <= 6 && ks == 2 ? 3 : 2;
    const long long whole = planes * ((row_tiles + w - 1) / w);
    for (long long x = 1; x <= std::max<long long>(1, std::min<long long>(64, key_tiles / 2)); ++x) {
      const long long rounds = (whole * x + cus * there - 1) / (cus * there);
      const long long together = std::min<long long>(there, (whole * x + cus - 1) / cus);
      const double tile =
          std::max(w == 8 ? 3200.0 : 2500.0, 0.75 * together * w / 4 * (192.0 * s + 850 + 200.0 * s / w));
      const double join = x > 1 ? 10000 + 0.5 * planes * a.rows * x / 256 : 0;
      const double time = rounds * ((key_tiles + x - 1) / x + 3) * tile + join;
      if (time < best) {
        best = time;
        *nw = w;
        a.tiles = (int)((row_tiles + w - 1) / w);
        a.splits = (int)x;
      }
    }
  }
  const long long rounds = (planes * row_tiles + cus - 1) / cus;
  // (Beside it a join costs 3,500: 300 rows of two key heads to 900 states 14.7 us so, 11.9 in pieces; of eight to 600 11.3
  // and 13.7.)
  if (a.splits > 1) best -= 6500;
  *lone = rounds * ((key_tiles + kLoneWaves - 1) / kLoneWaves * (392.0 * s + 850) + 800.0 * s - 1400) < best;
  if (*lone) {
    *nw = kLoneWaves;
    a.tiles = (int)row_tiles;
    a.splits = 1;
  }
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
  // Whether `bytes` bytes at p share memory with o (or lie between its pixels).
  auto meets = [&](const void* p, long double bytes) {
    const long double from = (long double)(uintptr_t)p, at = (long double)(uintptr_t)o->data;
    const long double size = 4.0L * (((long double)pixels(*o) - 1) * o->ldc + o->c);
    return from < at + size && at < from + bytes;
  };
  if (mask) {
    SY_CHECK(mask->data, SY_EINVAL, "null mask data");
    SY_CHECK(mask->image >= 0 && mask->head >= 0 && mask->query >= 0, SY_EINVAL, "negative mask stride");
    SY_CHECK(!meets(mask->data, (long double)mask->image * (q->n - 1) + (long double)mask->head * (a.heads - 1) +
                                    (long double)mask->query * ((double)q->h * q->w - 1) + (double)k->h * k->w),
             SY_EINVAL, "cross attention output overlaps the mask");
  }
  SY_CHECK(!lengths || !meets(lengths, 4.0L * q->n), SY_EINVAL, "cross attention output overlaps the lengths");
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
  // Steps of 16 channels, tiles of 32.
  const int ks = a.kd <= 32 ? 2 : a.kd <= 96 ? (a.kd + 15) / 16 : 8, dt = (a.hd + 31) / 32;
  int nw = 0;  // waves of a workgroup; 0: few rows, or few states
  bool lone = false;  // each with tiles of its own
  const long long row_tiles = (a.rows + 31) / 32;
  // 64 heads on 8 key heads of 16 images' 4000 states, a row tile of 8 rows each: 68 us on the matrix cores, 105 in
  // plain float32; 32 heads, 4 rows each, of 8 images 103 and 55.
  const bool few = a.rows <= 4;
  const bool brief = !few && (a.tk + kCrossKeys - 1) / kCrossKeys * short_bytes(ks, dt) <= kShortLds && row_tiles * planes >= 2048;
  a.splits = 1;
  if (few) {
    a.tiles = 1;
    a.splits = (int)std::max<long long>(1, a.tk <= 384 ? 1 : std::min<long long>(256 / planes, a.tk / 64));
  } else if (brief) {
    a.run = (int)std::max<long long>(8, (row_tiles * planes + 511) / 512);
    a.run = (a.run + kShortWaves - 1) / kShortWaves * kShortWaves;
    a.tiles = (int)((row_tiles + a.run - 1) / a.run);
  } else {
    cross_plan(a, ks, dt, planes, row_tiles, &nw, &lone);
  }
  a.piece = ((a.tk + a.splits - 1) / a.splits + kCrossKeys - 1) / kCrossKeys * kCrossKeys;
  a.splits = (a.tk + a.piece - 1) / a.piece;
  const long long items = planes * a.tiles * a.splits, grid = (items + 7) / 8 * 8;
  const int threads = few ? 256 : brief ? kShortWaves * 64 : nw * 64;
  SY_CHECK(grid * threads < (1LL << 32), SY_EUNSUPPORTED, "cross attention over %lld rows", planes * a.rows);
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
    CrossKernel kernel = few     ? pick_few(a.kd, a.hd, a.rows)
                         : brief ? pick_short(ks, dt)
                         : lone ? pick_lone(ks, dt)
                         : nw == 4 ? pick_cross<4>(ks, dt)
                                   : pick_cross<8>(ks, dt);
    const size_t lds = brief ? (size_t)(a.tk + kCrossKeys - 1) / kCrossKeys * short_bytes(ks, dt) : 0;
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(threads), lds, ctx->stream, a);
    SY_TRY(check_launch("cross_attention"));
  }
  if (a.splits > 1) {
    const long long rows = planes * a.rows;
    ProfScope prof(ctx, "cross_join", 0, 4.0 * rows * a.hd * (a.splits + 1));
    // A wave to a row from 8 pieces on: 2,400 rows of 32 pieces 3.9 us against 10 of 16 lanes to a row.
    auto join = a.splits < 8 ? (a.hd <= 32   ? cross_join_kernel<8, 8>
                                : a.hd <= 64 ? cross_join_kernel<16, 16>
                                             : cross_join_kernel<32, 32>)
                             : (a.hd <= 32   ? cross_join_kernel<8, 64>
                                : a.hd <= 64 ? cross_join_kernel<16, 64>
                                             : cross_join_kernel<32, 64>);
    const int each = a.splits >= 8 ? 4 : a.hd <= 32 ? 32 : a.hd <= 64 ? 16 : 8;  // rows of a workgroup
    hipLaunchKernelGGL(join, dim3((unsigned)((rows + each - 1) / each)), dim3(256), 0, ctx->stream, a, rows);
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
