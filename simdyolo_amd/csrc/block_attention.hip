// Attention over the key blocks chosen for each query.
//
// A query's blocks are its own choice, so neighbouring queries share few of them, and a matrix
// instruction wants 32 queries on the same keys.  The work is therefore done block by block: the
// (query, slot) pairs are sorted by the block they name, a workgroup takes up to 128 rows (a query times a
// head of the group that shares the key head) of one block's list, and leaves for each its maximum score,
// sum of weights and weighted sum of values (split over the long axis as in flash-decoding, Dao et al., 2023).
// A last kernel joins a query's slots.  With few queries (a token against a cache) the pairs are taken as
// they stand.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "split.h"
#include "sy_internal.h"

namespace sy {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kKeys = 64;    // keys of a tile; longer blocks are so many tiles ("parts" of the block)
constexpr int kRows = 128;   // rows of a tile: 32 for each of four waves
constexpr int kMaxBlocks = 12288;  // of a sorted list: counters in LDS

struct BlockArgs {
  const float *q, *k, *v;
  float* o;
  const int *blocks, *starts, *lengths;
  long long ldq, ldk, ldv, ldo;
  BlockShape s;
  int parts;         // tiles of a block along its keys
  // Segments: `span` queries of one image and key head each, `segs` of them to a plane.
  int span, segs, first;  // first: of the launch
  int sorted;        // 0: tiles are the (query, slot) pairs themselves
  int row_tiles;     // of a pair, where not sorted
  // Sorted lists of each segment.
  int chunks, tile_cap;  // chunks of the counting sort; tiles at most
  int *counts, *list, *tile_count;
  int4* tiles;
  // Results of the launch's segments, row by row.
  float2* stat;      // maximum (in powers of two) and sum
  float* part;       // weighted values
};

constexpr int kChunk = 1024;  // queries that a workgroup of the sort counts

// Keys of image b that query i sees: those before this position.
__device__ __forceinline__ int visible(const BlockArgs& a, int b, int i) {
  int end = a.lengths ? min(max(a.lengths[b], 0), a.s.tk) : a.s.tk;
  if (a.s.causal) {
    const long long at = (long long)(a.starts ? a.starts[b] : 0) + i;
    end = (int)min((long long)end, max(at + 1, 0LL));
  }
  return end;
}

// Whether block j exists and has a key before `end` (windows of maps: any).
__device__ __forceinline__ bool block_seen(const BlockArgs& a, int j, int end) {
  return j >= 0 && j < a.s.blocks && (a.s.kh > 1 ? end > 0 : (long long)j * a.s.bw < end);
}

__device__ __forceinline__ const int* list_of(const BlockArgs& a, int b, int i, int g) {
  return a.blocks + (((long long)b * a.s.tq + i) * a.s.kv + g) * a.s.selected;
}

// --------------------------------------------------------------- sorted lists

// Counts, per segment and chunk of queries, how often each block is named.
__global__ __launch_bounds__(256) void block_count_kernel(const BlockArgs a) {
  extern __shared__ int hist[];
  const BlockShape& s = a.s;
  const int seg = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
  const int plane = seg / a.segs, b = plane / s.kv, g = plane % s.kv;
  const int i0 = seg % a.segs * a.span, i1 = min(i0 + a.span, s.tq);
  const int from = i0 + chunk * kChunk, to = min(from + kChunk, i1);
  for (int j = threadIdx.x; j < s.blocks; j += 256) hist[j] = 0;
  __syncthreads();
  const int pairs = max(to - from, 0) * s.selected;
  for (int t = threadIdx.x; t < pairs; t += 256) {
    const int d = t / s.selected, i = from + d;
    const int j = list_of(a, b, i, g)[t - d * s.selected];
    if (block_seen(a, j, visible(a, b, i))) atomicAdd(&hist[j], 1);
  }
  __syncthreads();
  int* out = a.counts + ((long long)seg * a.chunks + chunk) * s.blocks;
  for (int j = threadIdx.x; j < s.blocks; j += 256) out[j] = hist[j];
}

// Exclusive sum over the workgroup's 1024 threads; *total: of all.
__device__ __forceinline__ int2 scan1024(int2 v, int2* lds, int2* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int2 x = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int ax = __shfl_up(x.x, off), ay = __shfl_up(x.y, off);
    if (lane >= off) {
      x.x += ax;
      x.y += ay;
    }
  }
  if (lane == 63) lds[wave] = x;
  __syncthreads();
  int2 before = make_int2(0, 0), all = make_int2(0, 0);
  for (int w = 0; w < 16; ++w) {
    const int2 t = lds[w];
    if (w < wave) before = make_int2(before.x + t.x, before.y + t.y);
    all = make_int2(all.x + t.x, all.y + t.y);
  }
  __syncthreads();
  *total = all;
  return make_int2(before.x + x.x - v.x, before.y + x.y - v.y);
}

// Per segment: where each chunk's pairs of each block start in the list, and the tiles.
__global__ __launch_bounds__(1024) void block_scan_kernel(const BlockArgs a) {
  __shared__ int2 lds[16];
  __shared__ int4 work[1024];
  const BlockShape& s = a.s;
  const int seg = blockIdx.x;
  int* counts = a.counts + (long long)seg * a.chunks * s.blocks;
  int4* tiles = a.tiles + (long long)seg * a.tile_cap;
  int2 base = make_int2(0, 0);
  for (int j0 = 0; j0 < s.blocks; j0 += 1024) {
    const int j = j0 + threadIdx.x;
    int n = 0;
    if (j < s.blocks)
      for (int c = 0; c < a.chunks; ++c) n += counts[(long long)c * s.blocks + j];
    const int t = (int)(((long long)n * s.group + kRows - 1) / kRows);
    int2 total;
    const int2 at = scan1024(make_int2(n, t * a.parts), lds, &total);
    if (j < s.blocks) {
      int place = base.x + at.x;
      for (int c = 0; c < a.chunks; ++c) {
        int* p = counts + (long long)c * s.blocks + j;
        const int m = *p;
        *p = place;
        place += m;
      }
    }
    // The tiles of this thread's block, written by all threads of a wave in turn.
    work[threadIdx.x] = make_int4(base.x + at.x, n, base.y + at.y, t);
    __syncthreads();
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int u = wave; u < min(1024, s.blocks - j0); u += 16) {
      const int4 w = work[u];
      for (int x = lane; x < w.w * a.parts; x += 64)
        tiles[w.z + x] = make_int4(j0 + u, x % a.parts | (x / a.parts) << 8, w.x, w.y);
    }
    __syncthreads();
    base = make_int2(base.x + total.x, base.y + total.y);
  }
  if (threadIdx.x == 0) a.tile_count[seg] = base.y;
}

// Puts the pairs in the order of their blocks (within a block in no certain order: a row's result does not
// depend on its neighbours in a tile).
__global__ __launch_bounds__(256) void block_scatter_kernel(const BlockArgs a) {
  extern __shared__ int hist[];
  const BlockShape& s = a.s;
  const int seg = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
  const int plane = seg / a.segs, b = plane / s.kv, g = plane % s.kv;
  const int i0 = seg % a.segs * a.span, i1 = min(i0 + a.span, s.tq);
  const int from = i0 + chunk * kChunk, to = min(from + kChunk, i1);
  const int* place = a.counts + ((long long)seg * a.chunks + chunk) * s.blocks;
  for (int j = threadIdx.x; j < s.blocks; j += 256) hist[j] = place[j];
  __syncthreads();
  int* list = a.list + (long long)seg * a.span * s.selected;
  const int pairs = max(to - from, 0) * s.selected;
  for (int t = threadIdx.x; t < pairs; t += 256) {
    const int d = t / s.selected, i = from + d;
    const int j = list_of(a, b, i, g)[t - d * s.selected];
    if (block_seen(a, j, visible(a, b, i))) list[atomicAdd(&hist[j], 1)] = (i - i0) * s.selected + t - d * s.selected;
  }
}

// ---------------------------------------------------------------------- tiles

// Eight floats as three bf16 parts each, v = p[0] + p[1] + p[2] exactly.
__device__ __forceinline__ void parts8(const float (&x)[8], bf16x8 (&p)[3]) {
  u32x4 w[3];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f32x2v v = {x[2 * i], x[2 * i + 1]};
#pragma unroll
    for (int s = 0; s < 3; ++s) {
      const unsigned b = __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2));
      w[s][i] = b;
      if (s < 2) {
        v[0] -= __builtin_bit_cast(float, b << 16);
        v[1] -= __builtin_bit_cast(float, b & 0xffff0000u);
      }
    }
  }
#pragma unroll
  for (int s = 0; s < 3; ++s) p[s] = __builtin_bit_cast(bf16x8, w[s]);
}

// main + rest += a b: the leading parts' product in main, the five next ones in rest.
__device__ __forceinline__ void mfma_parts(const bf16x8 (&a)[3], const bf16x8 (&b)[3], f32x16& main, f32x16& rest) {
  rest = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[2], b[0], rest, 0, 0, 0);
  main = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[0], main, 0, 0, 0);
  rest = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[1], b[1], rest, 0, 0, 0);
  rest = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[2], rest, 0, 0, 0);
  rest = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[1], b[0], rest, 0, 0, 0);
  rest = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[0], b[1], rest, 0, 0, 0);
}

// One tile: up to 64 keys of a block, up to 128 rows.
//
// Keys, then values, stand in LDS as three bf16 parts (Henry, Tang and Heinecke, 2019: a float's 24 bits over
// its whole exponent range, six of the nine part products taken), in the order in which the matrix
// instruction's lanes take them, so that a fragment is one 16-byte read without bank conflicts.  The values' loads are
// under way while the keys are multiplied, and take the keys' place afterwards.
//
// S^T = K Q^T: a lane holds one row's scores (keys 8 (r / 4) + 4 half + r % 4), so maximum and sum are in-lane
// but for one exchange, and the weights are already the A operand of O = P V under the key order
// 8 (e / 4) + 4 half + e % 4 of a 16-key step, in which V is laid out.  O comes out with channels across
// lanes: rows are stored in whole lines.
//
// The maximum m is the largest score times c = scale log2(e), rounded once; weights are 2^(s c - m) with one
// rounding of the exponent, and m is kept as it is, so that slots join exactly.
template <int KS, int DT>
__global__ __launch_bounds__(256, KS * DT >= 16 ? 2 : 3) void block_tile_kernel(const BlockArgs a) {
  constexpr int KF = 2 * KS * 3, VF = 4 * DT * 3;         // fragments of 64 lanes x 16 bytes
  constexpr int KI = (kKeys * KS * 2 + 255) / 256;        // 8-channel pieces of keys per thread
  constexpr int VI = (8 * 32 * DT + 255) / 256;           // 8-key pieces of values per thread
  __shared__ u32x4 frag[(KF > VF ? KF : VF) * 64];
  __shared__ int token[kKeys];
  __shared__ int place[kRows];
  const BlockShape& s = a.s;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, r32 = lane & 31;

  // The tile: block, part of it, rows.
  int seg, j, part, row0, rows, from = 0, pair = 0;
  if (a.sorted) {
    seg = blockIdx.x / a.tile_cap;
    const int t = blockIdx.x - seg * a.tile_cap;
    seg += a.first;
    if (t >= a.tile_count[seg]) return;
    const int4 rec = a.tiles[(long long)seg * a.tile_cap + t];
    j = rec.x;
    part = rec.y & 255;
    row0 = (rec.y >> 8) * kRows;
    from = rec.z;
    rows = rec.w * s.group;
  } else {
    int t = blockIdx.x;
    part = t % a.parts;
    t /= a.parts;
    row0 = t % a.row_tiles * kRows;
    t /= a.row_tiles;
    pair = t % (a.span * s.selected);
    seg = a.first + t / (a.span * s.selected);
    rows = s.group;
  }
  const int plane = seg / a.segs, b = plane / s.kv, g = plane - b * s.kv;
  const int i0 = seg % a.segs * a.span;
  if (!a.sorted) {
    const int i = i0 + pair / s.selected;
    if (i >= s.tq) return;
    j = list_of(a, b, i, g)[pair % s.selected];
    if (!block_seen(a, j, visible(a, b, i))) return;
  }
  const int y0 = j / s.bx * s.bh, x0 = j % s.bx * s.bw;
  const int cols = min(s.bw, s.kw - x0), size = min(s.bh, s.kh - y0) * cols;
  const int origin = y0 * s.kw + x0;
  // Keys of this part that exist: in the window and, in a sequence, before its end.
  int keys = size;
  if (a.lengths) keys = min(keys, min(max(a.lengths[b], 0), s.tk) - origin);
  keys = min(max(keys - part * kKeys, 0), kKeys);
  if (tid < kKeys) {
    const int t = tid < keys ? part * kKeys + tid : 0;
    token[tid] = origin + t / cols * s.kw + t % cols;
  }

  // The lane's row.
  const int row = row0 + wave * 32 + r32;
  const bool mine = row < rows, busy = row0 + wave * 32 < rows;
  int i = 0, h = 0, limit = 0, at = -1;
  {
    const int rr = min(row, rows - 1), e = rr / s.group;
    h = rr - e * s.group;
    const int id = a.sorted ? a.list[(long long)seg * a.span * s.selected + from + e] : pair;
    const int d = id / s.selected;
    i = i0 + d;
    at = (((seg - a.first) * a.span + d) * s.selected + id - d * s.selected) * a.parts + part;
    limit = keys;
    if (s.causal) limit = min(limit, visible(a, b, i) - origin - part * kKeys);
    if (half == 0) place[wave * 32 + r32] = mine ? at * s.group + h : -1;
  }
  __syncthreads();

  // Loads: queries, keys, values.
  const float* kb = a.k + (long long)b * s.tk * a.ldk + (long long)g * s.ks;
  const float* vb = a.v + (long long)b * s.tk * a.ldv + (long long)g * s.vs;
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  f32x4 kr[KI][2];
  float vr[VI][8];
#pragma unroll
  for (int n = 0; n < KI; ++n) {
    const int x = tid + 256 * n, key = x / (2 * KS), c = 8 * (x - key * 2 * KS);
    const float* p = kb + token[key & (kKeys - 1)] * a.ldk + c;
    kr[n][0] = c < s.kd ? *(const f32x4*)p : zero;
    kr[n][1] = c + 4 < s.kd ? *(const f32x4*)(p + 4) : zero;
  }
  f32x4 qr[KS][2];
  {
    const float* p = a.q + ((long long)b * s.tq + i) * a.ldq + ((long long)g * s.group + h) * s.qs + 8 * half;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int u = 0; u < 2; ++u) qr[ks][u] = 16 * ks + 8 * half + 4 * u < s.kd ? *(const f32x4*)(p + 16 * ks + 4 * u) : zero;
  }
#pragma unroll
  for (int n = 0; n < VI; ++n) {
    const int x = tid + 256 * n, c = x % (32 * DT), piece = x / (32 * DT);  // piece: 2 st + half
    const int first = 16 * (piece >> 1) + 4 * (piece & 1);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int key = first + 8 * (e >> 2) + (e & 3);
      const float v = vb[token[key] * a.ldv + min(c, s.hd - 1)];
      vr[n][e] = key < keys ? v : 0.f;
    }
  }

  // Keys into LDS: piece c of key t is lanes t % 32 + 32 (c % 2) of step c / 2.
#pragma unroll
  for (int n = 0; n < KI; ++n) {
    const int x = tid + 256 * n, key = x / (2 * KS), c = x - key * 2 * KS;
    if (KI * 256 == kKeys * KS * 2 || key < kKeys) {
      bf16x8 p[3];
      const float f[8] = {kr[n][0][0], kr[n][0][1], kr[n][0][2], kr[n][0][3], kr[n][1][0], kr[n][1][1], kr[n][1][2], kr[n][1][3]};
      parts8(f, p);
#pragma unroll
      for (int m = 0; m < 3; ++m)
        frag[(((key >> 5) * KS + (c >> 1)) * 3 + m) * 64 + (c & 1) * 32 + (key & 31)] = __builtin_bit_cast(u32x4, p[m]);
    }
  }
  __syncthreads();

  float w[32];
  float mx = -INFINITY, sum = 0.f;
  if (busy) {
    f32x16 sc[2], rest[2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[t][r] = rest[t][r] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      bf16x8 q[3];
      const float f[8] = {qr[ks][0][0], qr[ks][0][1], qr[ks][0][2], qr[ks][0][3], qr[ks][1][0], qr[ks][1][1], qr[ks][1][2], qr[ks][1][3]};
      parts8(f, q);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        bf16x8 k[3];
#pragma unroll
        for (int m = 0; m < 3; ++m) k[m] = __builtin_bit_cast(bf16x8, frag[((t * KS + ks) * 3 + m) * 64 + lane]);
        mfma_parts(k, q, sc[t], rest[t]);
      }
    }
    const float c = s.scale * 1.4426950408889634f;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float x = sc[t][r] + rest[t][r];
        w[16 * t + r] = 32 * t + 8 * (r >> 2) + 4 * half + (r & 3) < limit ? x : -INFINITY;
        mx = fmaxf(mx, w[16 * t + r]);
      }
    mx = fmaxf(mx, __shfl_xor(mx, 32)) * c;
    const float base = mx == -INFINITY ? 0.f : mx;  // no key, or none that weighs
#pragma unroll
    for (int r = 0; r < 32; ++r) {
      w[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(w[r], c, -base));
      sum += w[r];
    }
    sum += __shfl_xor(sum, 32);
  }
  __syncthreads();

#pragma unroll
  for (int n = 0; n < VI; ++n) {
    const int x = tid + 256 * n, c = x % (32 * DT), piece = x / (32 * DT);
    bf16x8 p[3];
    parts8(vr[n], p);
#pragma unroll
    for (int m = 0; m < 3; ++m)
      frag[(((piece >> 1) * DT + (c >> 5)) * 3 + m) * 64 + (piece & 1) * 32 + (c & 31)] = __builtin_bit_cast(u32x4, p[m]);
  }
  __syncthreads();
  if (!busy) return;

  bf16x8 wp[4][3];
#pragma unroll
  for (int st = 0; st < 4; ++st) {
    const float f[8] = {w[8 * st], w[8 * st + 1], w[8 * st + 2], w[8 * st + 3], w[8 * st + 4], w[8 * st + 5], w[8 * st + 6], w[8 * st + 7]};
    parts8(f, wp[st]);
  }
  if (half == 0 && mine) a.stat[place[wave * 32 + r32]] = make_float2(mx, sum);
#pragma unroll
  for (int d = 0; d < DT; ++d) {
    if (32 * d >= s.hd) break;
    f32x16 acc, rest;
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] = rest[r] = 0.f;
#pragma unroll
    for (int st = 0; st < 4; ++st) {
      bf16x8 v[3];
#pragma unroll
      for (int m = 0; m < 3; ++m) v[m] = __builtin_bit_cast(bf16x8, frag[((st * DT + d) * 3 + m) * 64 + lane]);
      mfma_parts(wp[st], v, acc, rest);
    }
    const int c = 32 * d + r32;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int to = place[wave * 32 + 8 * (r >> 2) + 4 * half + (r & 3)];
      if (to >= 0 && c < s.hd) a.part[(long long)to * s.hd + c] = acc[r] + rest[r];
    }
  }
}

// ----------------------------------------------------------------------- join

// One row in plain float32 by one wave, weights normalised before they meet the values so that no finite average
// overflows.  A lane scores one key of 64 and holds channels lane and lane + 64.
__device__ __attribute__((noinline)) void block_row(const BlockArgs& a, int b, int i, int h, int lane, float (&y)[2]) {
  const BlockShape& s = a.s;
  const int g = h / s.group, end = visible(a, b, i);
  const float* q = a.q + ((long long)b * s.tq + i) * a.ldq + (long long)h * s.qs;
  const float* kb = a.k + (long long)b * s.tk * a.ldk + (long long)g * s.ks;
  const float* vb = a.v + (long long)b * s.tk * a.ldv + (long long)g * s.vs;
  const int* list = list_of(a, b, i, g);
  float mx = -INFINITY, sum = 0.f, acc[2] = {0.f, 0.f};
  for (int pass = 0; pass < 3; ++pass) {  // maximum, sum, values
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
        if (pass == 0) {
          mx = fmaxf(mx, x);
          continue;
        }
        const float e = on ? expf(x - mx) : 0.f;
        if (pass == 1) {
          sum += e;
          continue;
        }
        const float p = e / sum;
        for (int u = 0; u < min(64, keys - t0); ++u) {
          const float w = __shfl(p, u);
          const int from = __shfl(at, u);
          if (!__shfl((int)on, u)) continue;
#pragma unroll
          for (int d = 0; d < 2; ++d)
            if (lane + 64 * d < s.hd) acc[d] = __builtin_fmaf(w, vb[from * a.ldv + lane + 64 * d], acc[d]);
        }
      }
    }
    if (pass < 2)
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) {
        mx = fmaxf(mx, __shfl_xor(mx, off));
        if (pass == 1) sum += __shfl_xor(sum, off);
      }
  }
  y[0] = acc[0];
  y[1] = acc[1];
}

// Joins the slots of each row: lanes of 4 channels, L of them to a row.  A row that comes out infinite or NaN
// (operands that are, sums that overflow, parts of hidden keys that are not finite) is computed again in plain
// float32.
template <int L>
__global__ __launch_bounds__(256) void block_join_kernel(const BlockArgs a, long long rows) {
  const BlockShape& s = a.s;
  const int lane = threadIdx.x & 63;
  const long long row = (long long)blockIdx.x * (256 / L) + threadIdx.x / L;  // (segment, query, head of the group)
  const int c = 4 * (threadIdx.x % L);
  const int h = (int)(row % s.group), d = (int)(row / s.group % a.span), ls = (int)(row / s.group / a.span);
  const int seg = a.first + ls, plane = seg / a.segs, b = plane / s.kv, g = plane - b * s.kv;
  const int i = seg % a.segs * a.span + d;
  const bool live = row < rows && i < s.tq;
  bool again = false, any = false;
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
  if (live) {
    const int* list = list_of(a, b, i, g);
    const int end = visible(a, b, i);
    const long long slot0 = ((long long)ls * a.span + d) * s.selected;
    float mx = -INFINITY, sum = 0.f;
    for (int n = 0; n < s.selected; ++n) {
      if (!block_seen(a, list[n], end)) continue;
      any = true;
      for (int p = 0; p < a.parts; ++p) mx = fmaxf(mx, a.stat[((slot0 + n) * a.parts + p) * s.group + h].x);
    }
    for (int n = 0; n < s.selected; ++n) {
      if (!block_seen(a, list[n], end)) continue;
      for (int p = 0; p < a.parts; ++p) {
        const long long r = ((slot0 + n) * a.parts + p) * s.group + h;
        const float2 st = a.stat[r];
        const float f = st.x == -INFINITY && !(st.y != st.y) ? 0.f : __builtin_amdgcn_exp2f(st.x - mx);
        sum = __builtin_fmaf(st.y, f, sum);
        if (c < s.hd) {
          const f32x4 v = *(const f32x4*)(a.part + r * s.hd + c);
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = __builtin_fmaf(v[e], f, y[e]);
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      y[e] = any ? y[e] / sum : 0.f;
      again |= c < s.hd && !(__builtin_fabsf(y[e]) <= FLT_MAX);
    }
    if (c < s.hd) *(f32x4*)(a.o + ((long long)b * s.tq + i) * a.ldo + (long long)(g * s.group + h) * s.hd + c) = y;
  }
  for (unsigned long long todo = __ballot(again); todo;) {
    const int from = __builtin_ctzll(todo) & ~(L - 1);
    const int rb = __shfl(b, from), ri = __shfl(i, from), rh = __shfl(g * s.group + h, from);
    float z[2];
    block_row(a, rb, ri, rh, lane, z);
    float* o = a.o + ((long long)rb * s.tq + ri) * a.ldo + (long long)rh * s.hd;
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (lane + 64 * e < s.hd) o[lane + 64 * e] = z[e];
    todo &= ~((L == 64 ? ~0ull : (1ull << L) - 1) << from);
  }
}

// Bytes of results that one launch leaves and the next one joins.
constexpr double kPartials = 96e6;

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
  a.parts = (int)(((long long)s.bh * s.bw + kKeys - 1) / kKeys);
  const int planes = s.n * s.kv;
  SY_CHECK((long long)s.n * s.kv < (1 << 24) && (long long)s.tq * s.selected < (1LL << 31), SY_EUNSUPPORTED,
           "block attention over %d x %d queries", s.n, s.tq);
  // Segments: as many queries as keep the results of one in kPartials bytes.
  const double per_query = 4.0 * s.selected * a.parts * s.group * (s.hd + 2);
  a.span = (int)std::min<double>(s.tq, std::max(1.0, std::floor(kPartials / per_query)));
  a.segs = (s.tq + a.span - 1) / a.span;
  const long long segments = (long long)planes * a.segs;
  const int together = (int)std::min<double>((double)segments, std::max(1.0, std::floor(kPartials / (per_query * a.span))));
  a.row_tiles = (s.group + kRows - 1) / kRows;
  a.sorted = s.blocks <= kMaxBlocks && (long long)s.tq * s.selected > 64;
  a.chunks = (a.span + kChunk - 1) / kChunk;
  a.tile_cap = (int)std::min<long long>(
      a.parts * (std::min<long long>(s.blocks, (long long)a.span * s.selected) + (long long)a.span * s.selected * s.group / kRows + 1),
      0x7fffffff);
  const long long result_rows = (long long)together * a.span * s.selected * a.parts * s.group;
  SY_CHECK(result_rows < (1LL << 31), SY_EUNSUPPORTED, "block attention over %d heads to a key head", s.group);
  // Scratch: results, then lists.
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t from = at;
    at += (bytes + 255) & ~size_t(255);
    return from;
  };
  const size_t part_at = take(sizeof(float) * result_rows * s.hd), stat_at = take(sizeof(float2) * result_rows);
  const size_t count_at = a.sorted ? take(sizeof(int) * segments * a.chunks * s.blocks) : 0;
  const size_t list_at = a.sorted ? take(sizeof(int) * segments * a.span * s.selected) : 0;
  const size_t tile_at = a.sorted ? take(sizeof(int4) * segments * a.tile_cap) : 0;
  const size_t number_at = a.sorted ? take(sizeof(int) * segments) : 0;
  DeviceScope device(ctx);
  SY_TRY(ensure_scratch(ctx, at));
  a.part = (float*)(ctx->scratch + part_at);
  a.stat = (float2*)(ctx->scratch + stat_at);
  a.counts = (int*)(ctx->scratch + count_at);
  a.list = (int*)(ctx->scratch + list_at);
  a.tiles = (int4*)(ctx->scratch + tile_at);
  a.tile_count = (int*)(ctx->scratch + number_at);
  const double keys = std::min((double)s.selected * s.bh * s.bw, (double)s.tk);
  if (a.sorted) {
    ProfScope prof(ctx, "block_sort", 0, 8.0 * s.n * (double)s.tq * s.kv * s.selected);
    const size_t lds = sizeof(int) * s.blocks;
    const dim3 grid((unsigned)(segments * a.chunks));
    hipLaunchKernelGGL(block_count_kernel, grid, dim3(256), lds, ctx->stream, a);
    hipLaunchKernelGGL(block_scan_kernel, dim3((unsigned)segments), dim3(1024), 0, ctx->stream, a);
    hipLaunchKernelGGL(block_scatter_kernel, grid, dim3(256), lds, ctx->stream, a);
    SY_TRY(check_launch("block_sort"));
  }
  for (long long first = 0; first < segments; first += together) {
    const int now = (int)std::min<long long>(together, segments - first);
    const double share = (double)now / segments;
    a.first = (int)first;
    {
      ProfScope prof(ctx, "block_attention", share * 2.0 * s.n * s.tq * s.heads * keys * (s.kd + s.hd),
                     share * 4.0 * s.n * ((double)s.tq * s.heads * (s.kd + s.hd) + (double)s.tk * s.kv * (s.kd + s.hd)));
      const long long grid = (long long)now * (a.sorted ? a.tile_cap : (long long)a.span * s.selected * a.row_tiles * a.parts);
      SY_CHECK(grid * 256 < (1LL << 32), SY_EUNSUPPORTED, "block attention grid too large");
      auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(256), 0, ctx->stream, a); };
      auto pick = [&](auto two, auto four) { s.hd <= 64 ? launch(two) : launch(four); };
      if (s.kd <= 32)
        pick(block_tile_kernel<2, 2>, block_tile_kernel<2, 4>);
      else if (s.kd <= 64)
        pick(block_tile_kernel<4, 2>, block_tile_kernel<4, 4>);
      else
        pick(block_tile_kernel<8, 2>, block_tile_kernel<8, 4>);
      SY_TRY(check_launch("block_attention"));
    }
    {
      const long long rows = (long long)now * a.span * s.group;
      ProfScope prof(ctx, "block_join", 0, 4.0 * rows * s.hd * (s.selected * a.parts + 1));
      if (s.hd <= 64)
        hipLaunchKernelGGL(block_join_kernel<16>, dim3((unsigned)((rows + 15) / 16)), dim3(256), 0, ctx->stream, a, rows);
      else
        hipLaunchKernelGGL(block_join_kernel<32>, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, ctx->stream, a, rows);
      SY_TRY(check_launch("block_join"));
    }
  }
  return SY_OK;
}

}  // namespace sy

extern "C" int sy_block_attention(sy_ctx* ctx, const sy_block_config* cfg, const sy_tensor* q, const sy_tensor* k,
                                  const sy_tensor* v, const int32_t* blocks, const int32_t* starts,
                                  const int32_t* lengths, const sy_tensor* o) {
  return sy::op_block_attention(ctx, cfg, q, k, v, blocks, starts, lengths, o);
}
