// Attention over the key blocks chosen for each query.
//
// A query's blocks are its own choice, so neighbouring queries share few of them, and a matrix
// instruction wants 32 queries on the same keys.  The work is therefore done block by block: the
// (query, slot) pairs are sorted by the block they name, a workgroup takes up to 512 rows (a query times a
// head of the group that shares the key head) of one block's list, and leaves for each its maximum score,
// sum of weights and weighted sum of values, split over the long axis as flash-decoding does (Dao, Haziza, Massa and
// Sizov, 2023).  A last kernel joins a query's slots.  With few queries (a token against a cache) the pairs are
// taken as they stand.
//
// Measured, us (sort + tiles + join, under a tracer): two 160x160 maps, 4 heads of 32 / 64 channels, 8 of 400 blocks of 64
// keys 22 + 121 + 89; 8,192 causal tokens, 16 heads and 4 key heads of 128, 16 of 128 blocks 17 + 389 + 193; plain
// float32, a wave to a query, 14,900 and 61,700.  The results are written and read once, 0.43 and 1.0 GB: the join is bound
// by them, and the tiles of 64 channels (3.5 TB/s); those of 128 by two waves per SIMD that share it between vector work (50%
// of the time) and matrix products (30%).
#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>

#include "split.h"
#include "sy_internal.h"

namespace sy {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kFlat = 8;
// Largest factor of a score, and least value, that f16 pairs hold (their powers of two apart).
constexpr float kWide = 0x1p-8f, kFine = 0x1p-14f;
constexpr int kKeys = 64;    // keys of a tile; longer blocks are so many tiles ("parts" of the block)
constexpr int kTileRows = 512;  // rows of a tile at most
constexpr int kScan = 2048;  // pairs of an image and key head that a tile's workgroup goes through itself
// Blocks of a sorted list: counters in LDS.  More go pair by pair, however many queries there are (4,096 of 4 heads of 64, 16
// of 12,288 blocks of 16 keys 287 us, of 12,289 509).
constexpr int kMaxBlocks = 12288;

// What a tile leaves for a row beside its weighted values: the maximum (as a power of two), the sum of weights, and the
// power of two that the values want.
struct Stat {
  float top, sum;
  int scale;
};
constexpr int kNoPower = -4096;  // below every power of a product

struct BlockArgs {
  const float *q, *k, *v;
  float* o;
  const int *blocks, *starts, *lengths;
  long long ldq, ldk, ldv, ldo;
  BlockShape s;
  int parts;         // tiles of a block along its keys
  // Segments: `span` queries of one image and key head each, `segs` of them to a plane.
  int span, segs, first;  // first: of the launch
  int now;           // segments of the launch
  // Sorted lists of each segment of the launch.
  int rows;          // of a tile
  unsigned trash;    // a row of results that nobody reads
  int chunk, chunks, tile_cap;  // queries of a workgroup of the sort, such workgroups; tiles at most
  int *counts, *list, *tile_count;
  int* pos;          // place of each pair in its list
  int4* tiles;
  // Results of the launch's segments, row by row.
  Stat* stat;
  float* part;       // weighted values
};

constexpr int kSortThreads = 512;

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

// The pairs of one chunk of a launch's segment, four at a time in every thread: f(pair, block) for those whose block
// is seen.
template <class F>
__device__ __forceinline__ void for_pairs(const BlockArgs& a, int of_launch, int chunk, F f) {
  const BlockShape& s = a.s;
  const int seg = a.first + of_launch, plane = seg / a.segs, b = plane / s.kv, g = plane - b * s.kv;
  const int i0 = seg % a.segs * a.span, i1 = min(i0 + a.span, s.tq);
  const int from = i0 + chunk * a.chunk, to = min(from + a.chunk, i1);
  const int pairs = max(to - from, 0) * s.selected, skip = (from - i0) * s.selected;
  const int* lists = list_of(a, b, from, g);
  const int length = a.lengths ? min(max(a.lengths[b], 0), s.tk) : s.tk;
  const long long start = a.starts ? a.starts[b] : 0;
  for (int t0 = threadIdx.x; t0 < pairs; t0 += 4 * kSortThreads) {
    int j[4], d[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int t = min(t0 + u * kSortThreads, pairs - 1);
      d[u] = t / s.selected;
      j[u] = lists[(long long)d[u] * s.kv * s.selected + t - d[u] * s.selected];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int t = t0 + u * kSortThreads;
      int end = length;
      if (s.causal) end = (int)min((long long)end, max(start + from + d[u] + 1, 0LL));
      if (t < pairs && block_seen(a, j[u], end)) f(skip + t, j[u]);
    }
  }
}

// Counts, per segment and chunk of queries, how often each block is named.
__global__ __launch_bounds__(kSortThreads) void block_count_kernel(const BlockArgs a) {
  extern __shared__ int hist[];
  const int seg = blockIdx.x / a.chunks, chunk = blockIdx.x - seg * a.chunks;
  for (int j = threadIdx.x; j < a.s.blocks; j += kSortThreads) hist[j] = 0;
  __syncthreads();
  for_pairs(a, seg, chunk, [&](int, int j) { atomicAdd(&hist[j], 1); });
  __syncthreads();
  int* out = a.counts + ((long long)seg * a.chunks + chunk) * a.s.blocks;
  for (int j = threadIdx.x; j < a.s.blocks; j += kSortThreads) out[j] = hist[j];
}

__device__ __forceinline__ int3 operator+(int3 a, int3 b) { return make_int3(a.x + b.x, a.y + b.y, a.z + b.z); }

// Exclusive sum over the workgroup's threads; *total: of all.
__device__ __forceinline__ int3 scan_threads(int3 v, int3* lds, int3* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int3 x = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int3 o = make_int3(__shfl_up(x.x, off), __shfl_up(x.y, off), __shfl_up(x.z, off));
    if (lane >= off) x = x + o;
  }
  if (lane == 63) lds[wave] = x;
  __syncthreads();
  int3 before = make_int3(0, 0, 0), all = before;
#pragma unroll
  for (int w = 0; w < kSortThreads / 64; ++w) {
    if (w < wave) before = before + lds[w];
    all = all + lds[w];
  }
  __syncthreads();
  *total = all;
  return make_int3(before.x + x.x - v.x, before.y + x.y - v.y, before.z + x.z - v.z);
}

// Rows of each tile of a block's list of `all`: equal shares, in 32s.
__device__ __forceinline__ int tile_share(const BlockArgs& a, int all) {
  const int tiles = (all + a.rows - 1) / a.rows;
  return ((all + tiles - 1) / max(tiles, 1) + 31) & ~31;
}

// Puts the pairs in the order of their blocks (within a block by chunk, within a chunk in no certain order: a row's
// result does not depend on its neighbours in a tile).  Every chunk's workgroup sums the counts of its segment for itself and
// writes the tiles that begin among its own pairs, so that tiles stand in the order of their first queries: those
// under way together read the same queries (8,192 causal tokens, whose queries are 17 MB to a key head, block by block).
// With one chunk it does the counting, too.
__global__ __launch_bounds__(kSortThreads) void block_scatter_kernel(const BlockArgs a) {
  extern __shared__ int hist[];
  __shared__ int3 lds[kSortThreads / 64];
  const BlockShape& s = a.s;
  const int seg = blockIdx.x / a.chunks, chunk = blockIdx.x - seg * a.chunks, lane = threadIdx.x & 63;
  const int* counts = a.counts + (long long)seg * a.chunks * s.blocks;
  int4* tiles = a.tiles + (long long)seg * a.tile_cap;
  if (a.chunks == 1) {
    for (int j = threadIdx.x; j < s.blocks; j += kSortThreads) hist[j] = 0;
    __syncthreads();
    for_pairs(a, seg, chunk, [&](int, int j) { atomicAdd(&hist[j], 1); });
    __syncthreads();
  }
  // Block j's pairs, those of earlier chunks, and its tiles that begin before this chunk's pairs and behind them.
  struct Count {
    int n, before, from, to;
  };
  auto count = [&](int j) {
    Count c{0, 0, 0, 0};
    int own = 0;
    if (j < s.blocks) {
      if (a.chunks == 1)
        c.n = own = hist[j];
      else
#pragma unroll 8
        for (int x = 0; x < a.chunks; ++x) {
          const int m = counts[(long long)x * s.blocks + j];
          c.n += m;
          if (x < chunk) c.before += m;
          if (x == chunk) own = m;
        }
    }
    if (c.n) {
      const int share = tile_share(a, c.n * s.group);
      c.from = (c.before * s.group + share - 1) / share;
      c.to = ((c.before + own) * s.group + share - 1) / share;
    }
    return c;
  };
  int3 base = make_int3(0, 0, 0), total;  // pairs, this chunk's tiles, earlier chunks' tiles
  if (a.chunks > 1 && s.blocks > kSortThreads) {
    for (int j = threadIdx.x; j < s.blocks; j += kSortThreads) base.z += count(j).from * a.parts;
    (void)scan_threads(base, lds, &total);
    base = make_int3(0, total.z, 0);
  }
  for (int j0 = 0; j0 < s.blocks; j0 += kSortThreads) {
    const int j = j0 + threadIdx.x;
    const Count c = count(j);
    const int items = (c.to - c.from) * a.parts;
    const int3 at = scan_threads(make_int3(c.n, items, s.blocks > kSortThreads ? 0 : c.from * a.parts), lds, &total);
    if (j < s.blocks) hist[j] = base.x + at.x + c.before;
    const int list_at = base.x + at.x, tile_at = base.y + total.z + at.y;
    auto put = [&](int j, int x, int from, int first, int n, int to) {
      tiles[to + x] = make_int4(j, x % a.parts | (from + x / a.parts) << 8, first, n);
    };
    constexpr int kAlone = 16;  // items that a thread writes; a wave together, beyond
    if (items <= kAlone)
      for (int x = 0; x < items; ++x) put(j, x, c.from, list_at, c.n, tile_at);
    for (unsigned long long todo = __ballot(items > kAlone); todo; todo &= todo - 1) {
      const int l = __builtin_ctzll(todo), many = __shfl(items, l), from = __shfl(c.from, l), first = __shfl(list_at, l),
                n = __shfl(c.n, l), to = __shfl(tile_at, l);
      for (int x = lane; x < many; x += 64) put(j - lane + l, x, from, first, n, to);
    }
    base = make_int3(base.x + total.x, base.y + total.z + total.y, 0);
  }
  if (chunk == a.chunks - 1 && threadIdx.x == 0) a.tile_count[seg] = base.y;
  __syncthreads();
  int* list = a.list + (long long)seg * a.span * s.selected;
  int* pos = a.pos + (long long)seg * a.span * s.selected;
  for_pairs(a, seg, chunk, [&](int pair, int j) {
    const int at = atomicAdd(&hist[j], 1);
    list[at] = pair;
    pos[pair] = at;
  });
}

// ---------------------------------------------------------------------- tiles

// Exponent field of the power of two that takes a largest magnitude m into [2^14, 2^15): a row in that range splits
// into pairs of f16, h + l / 2048, within 2^-22 of each element, or 2^-36 (2^-50 of m) where that is more.  Rows below
// 2^-113 keep the largest scale there is, and with it every bit of a float.
__device__ __forceinline__ int pair_field(float m) { return min(268 - (int)(__builtin_bit_cast(unsigned, m) >> 23), 254); }

__device__ __forceinline__ void pairs8(const float (&x)[8], float s, f16x8& h, f16x8& l) {
  u32x4 hw, lw;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = x[2 * i], b = x[2 * i + 1];
    const f16x2 hi = __builtin_convertvector((f32x2v{a * s, b * s}), f16x2);
    const f32x2v r = {__builtin_fmaf(a, s, -(float)hi[0]), __builtin_fmaf(b, s, -(float)hi[1])};
    hw[i] = __builtin_bit_cast(unsigned, hi);
    lw[i] = __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2v{r[0] * 2048.f, r[1] * 2048.f}), f16x2));
  }
  h = __builtin_bit_cast(f16x8, hw);
  l = __builtin_bit_cast(f16x8, lw);
}

// Largest magnitude of eight; a NaN counts as the larger.
__device__ __forceinline__ float max8(const float (&x)[8]) {
  unsigned m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, __builtin_bit_cast(unsigned, x[e]) & 0x7fffffffu);
  return __builtin_bit_cast(float, m);
}

// Largest (non-negative, as bits) of W neighbouring lanes, in each of them.
template <int W>
__device__ __forceinline__ float max_lanes(float f) {
  int m = __builtin_bit_cast(int, f);
  m = max(m, __builtin_amdgcn_update_dpp(0, m, 0xb1, 0xf, 0xf, false));               // lane ^ 1
  m = max(m, __builtin_amdgcn_update_dpp(0, m, 0x4e, 0xf, 0xf, false));               // lane ^ 2
  if (W > 4) m = max(m, __builtin_amdgcn_update_dpp(0, m, 0x141, 0xf, 0xf, false));  // 7 - lane
  if (W > 8) m = max(m, __builtin_amdgcn_update_dpp(0, m, 0x140, 0xf, 0xf, false));  // 15 - lane
  return __builtin_bit_cast(float, m);
}

// Work item of a workgroup: each of the 8 XCDs takes workgroups in turn, and with them one eighth of the items in a
// row, so that tiles of one block and the queries of one head meet in one L2.
__device__ __forceinline__ unsigned item_of(unsigned block, unsigned grid) { return (block & 7) * (grid >> 3) + (block >> 3); }

// One tile: up to 64 keys of a block and a.rows rows of its list, 32 at a time for each of four waves.
//
// Products of float32 on the f16 matrix cores: an operand is a pair h + l / 2048 of f16 values under a power of two of
// its own row (a query, a key, the values of a key, the weights of a query), and h h + (h l + l h) / 2048 is taken:
// 3 x 2^-22 of each product at most, whatever the other rows hold, as long as elements are not below 2^-29 of their
// row's largest.  The powers of queries and keys come back onto the scores; those of the values meet the weights
// before these are split, so that a key's weight counts as much as what it brings; the last one, of the weights' row, is
// left to the join.  Where the largest elements of all keys (of all values) of a tile are within 2^kFlat of each other
// they share one power, which needs none per score (per weight); 2^-29 becomes 2^-21 of a smaller row's then.
//
// Elements below that keep an absolute precision, 2^-36 under their power: for a score 1.5 x 2^-20 under both powers from
// each channel and so, as long as its factor is at most kWide, less than 2^-20 of its exponent.  Rows past that
// (|q||k| scale of 2^20 and more) leave NaN for their sum: the join computes them in plain float32.  A tile that has values
// so far below the others of their key gives every channel a power of its own, too, which comes off the results (2^-90
// and less: plain float32).
//
// Keys and values stand in LDS as pairs, in the order in which the matrix instruction's lanes take them, so that a
// fragment is one 16-byte read without bank conflicts.  Once they stand there the waves run on their own: no
// barrier, the next rows' queries under way while the weights meet the values.
//
// S^T = K Q^T: a lane holds one row's scores (keys 8 (r / 4) + 4 half + r % 4), so maximum and sum are in-lane
// but for one exchange, and the weights are already the A operand of O = P V under the key order
// 8 (e / 4) + 4 half + e % 4 of a 16-key step, in which V is laid out.  O comes out with channels across
// lanes: rows are stored in whole lines.
//
// The maximum m is the largest score times c = scale log2(e), rounded once; weights are 2^(s c - m) with one
// rounding of the exponent, and m is kept as it is, so that slots join exactly.
template <int KS, int DT, bool WHOLE>
__global__ __launch_bounds__(256, KS * DT >= 16 ? 2 : KS * DT == 4 ? 4 : 3) void block_tile_kernel(const BlockArgs a) {
  constexpr int KF = 2 * KS * 2, VF = 4 * DT * 2;  // fragments of 64 lanes x 16 bytes
  constexpr int KI = kKeys * KS * 2 / 256;         // 8-channel pieces of keys per thread
  constexpr int VI = 8 * 32 * DT / 256;            // 8-key pieces of values per thread
  __shared__ u32x4 frag[(KF + VF) * 64];
  __shared__ unsigned v_at[kKeys];                 // floats from the block's first key
  __shared__ float k_top[kKeys], v_top[kKeys];     // largest magnitude of a key, of its values
  __shared__ __align__(16) int k_power[kKeys], v_power[kKeys];
  __shared__ unsigned place[4][32];
  __shared__ int pair_at[kTileRows];
  __shared__ int uneven, c_power[32 * DT];         // whether channels have powers of their own; these, 14 above
  const BlockShape& s = a.s;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, r32 = lane & 31;

  const unsigned item = item_of(blockIdx.x, gridDim.x);
  const int ls = item / a.tile_cap, seg = a.first + ls;
  const int t = item - ls * a.tile_cap;
  if (ls >= a.now) return;
  const int plane = seg / a.segs, b = plane / s.kv, g = plane - b * s.kv, i0 = (seg - plane * a.segs) * a.span;
  const bool scan = !a.list;
  int4 rec;  // block, part of it and number of the tile, first entry of its list, length of the list
  unsigned long long named[kScan / 256];
  int before = 0;
  if (scan) {
    // A small call without lists: those of all queries are gone through here for the ones that name the block.
    const int j = t / a.parts % s.blocks;
    int n = 0;
#pragma unroll
    for (int u = 0; u < kScan / 256; ++u) {
      const int pair = wave * (kScan / 4) + 64 * u + lane, d = min(pair, s.tq * s.selected - 1) / s.selected;
      const int is = list_of(a, b, d, g)[min(pair, s.tq * s.selected - 1) - d * s.selected];
      named[u] = __ballot(pair < s.tq * s.selected && is == j && block_seen(a, j, visible(a, b, d)));
      n += __builtin_popcountll(named[u]);
    }
    if (lane == 0) place[0][wave] = n;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int m = place[0][w];
      before += w < wave ? m : 0;
      all += m;
    }
    __syncthreads();
    rec = make_int4(j, t % a.parts | t / (a.parts * s.blocks) << 8, 0, all);
    if (all == 0) return;
  } else {
    rec = a.tiles[(long long)ls * a.tile_cap + t];  // under way with the count
    if (t >= a.tile_count[ls]) return;
  }
  // Its share of the block's rows: as many as the other tiles', in 32s.
  const int all = rec.w * s.group, share = tile_share(a, all);
  const int j = rec.x, part = rec.y & 255, row0 = (rec.y >> 8) * share;
  const int rows = min(all - row0, share);
  if (rows <= 0) return;
  const int* list = scan ? nullptr : a.list + (long long)ls * a.span * s.selected + rec.z;
  const int y0 = j / s.bx * s.bh, x0 = j % s.bx * s.bw;
  const int cols = min(s.bw, s.kw - x0), size = min(s.bh, s.kh - y0) * cols;
  const int origin = y0 * s.kw + x0;
  // Keys of this part that exist: in the window and, in a sequence, before its end.  Nor does any row see those behind the
  // last query's: a cache may hold anything there (NaN in the block of the last of 8,100 tokens: 624 us, not 4,575).
  const long long start = a.starts ? a.starts[b] : 0;
  int length = a.lengths ? min(max(a.lengths[b], 0), s.tk) : s.tk;
  if (s.causal) length = (int)min((long long)length, max(start + s.tq, 0LL));
  int keys = a.lengths || s.causal ? min(size, length - origin) : size;
  keys = min(max(keys - part * kKeys, 0), kKeys);

  // The lane's row in the wave's turn r: its query, the keys it sees, where its results go.  Channels past key_dim read
  // the last ones again, which the keys' zeros cancel.
  const float* qb = a.q + ((long long)b * s.tq + i0) * a.ldq + (long long)g * s.group * s.qs;
  const int e0 = row0 / s.group, h0 = row0 - e0 * s.group;
  f32x4 qr[KS][2];
  int limit;
  unsigned to;  // row of the results
  auto result_row = [&](int x) __attribute__((always_inline)) {
    const int e = x / s.group;
    const unsigned slot = (unsigned)(ls * a.span * s.selected + (scan ? pair_at[e] : rec.z + e0 + e)) * a.parts + part;
    return slot * s.group + (x - e * s.group);
  };
  auto load_q = [&](int r) __attribute__((always_inline)) {
    const int x = h0 + min(r + r32, rows - 1), e = x / s.group, h = x - e * s.group;
    const int pair = pair_at[e], d = pair / s.selected;
    limit = keys;
    if (s.causal) {
      const long long end = min((long long)length, max(start + i0 + d + 1, 0LL));
      limit = min(keys, (int)end - origin - part * kKeys);
    }
    to = r + r32 < rows ? result_row(x) : a.trash;
    const float* p = qb + (long long)d * a.ldq + h * s.qs;
    constexpr bool kOften = KS * DT < 16;  // whether offsets kept for the loop would be spilled
    if (kOften && s.kd == 16 * KS) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int u = 0; u < 2; ++u) qr[ks][u] = *(const f32x4*)(p + 8 * half + 16 * ks + 4 * u);
      return;
    }
    int at = 8 * half;
    if (kOften) asm("" : "+v"(at));  // made here
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int u = 0; u < 2; ++u) qr[ks][u] = *(const f32x4*)(p + min(at + 16 * ks + 4 * u, s.kd - 4));
  };
  // The key's place in floats from the block's first one; a quotient of numbers below 2^11, exact in float32.
  const float per_row = 1.f / cols;
  auto key_at = [&](int key, long long ld) __attribute__((always_inline)) {
    const int u = key < keys ? part * kKeys + key : 0, y = (int)((u + 0.5f) * per_row);
    return (unsigned)(y * s.kw + u - y * cols) * (unsigned)ld;
  };
  static_assert(kTileRows <= 512, "two pairs to a thread");
  const int entries = (h0 + rows + s.group - 1) / s.group;
  int first_pair[2];
#pragma unroll
  for (int n = 0; n < 2; ++n) first_pair[n] = scan ? 0 : list[e0 + min(tid + 256 * n, entries - 1)];
  if (scan)
#pragma unroll
    for (int u = 0; u < kScan / 256; ++u) {
      const int at = before + __builtin_popcountll(named[u] & ((1ull << lane) - 1)) - e0;
      if ((named[u] >> lane & 1) && at >= 0 && at < entries) pair_at[at] = wave * (kScan / 4) + 64 * u + lane;
      before += __builtin_popcountll(named[u]);
    }

  int r = wave * 32, k_most, v_most;
  bool k_flat, v_flat;
  {
    const float* kb = a.k + ((long long)b * s.tk + origin) * a.ldk + (long long)g * s.ks;
    const float* vb = a.v + ((long long)b * s.tk + origin) * a.ldv + (long long)g * s.vs;
    float kr[KI][8], vm[VI][8], vr[VI][8];
    auto load8 = [&](const float* p, int c, int dim, float (&to8)[8]) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const f32x4 f = *(const f32x4*)(p + min(c + 4 * u, dim - 4));
#pragma unroll
        for (int e = 0; e < 4; ++e) to8[4 * u + e] = c + 4 * u < dim ? f[e] : 0.f;
      }
    };
#pragma unroll
    for (int n = 0; n < KI; ++n) {
      const int x = tid + 256 * n, key = x / (2 * KS);
      load8(kb + key_at(key, a.ldk), 8 * (x - key * 2 * KS), s.kd, kr[n]);
    }
    // The values twice: a key's channels across neighbouring lanes, for their largest, and eight keys of a channel.
#pragma unroll
    for (int n = 0; n < VI; ++n) {
      const int x = tid + 256 * n, key = x / (4 * DT);
      load8(vb + key_at(key, a.ldv), 8 * (x - key * 4 * DT), s.hd, vm[n]);
    }
#pragma unroll
    for (int n = 0; n < 2; ++n)
      if (!scan && tid + 256 * n < kTileRows) pair_at[tid + 256 * n] = first_pair[n];
    if (tid < kKeys) v_at[tid] = key_at(tid, a.ldv);
    if (tid == 0) uneven = 0;
    if (tid < 32 * DT) c_power[tid] = kNoPower;
    __syncthreads();
    load_q(r);
#pragma unroll
    for (int n = 0; n < VI; ++n) {
      const int x = tid + 256 * n, c = min(x % (32 * DT), s.hd - 1), piece = x / (32 * DT);  // piece: 2 step + half
      const int first = 16 * (piece >> 1) + 4 * (piece & 1);
#pragma unroll
      for (int e = 0; e < 8; ++e) vr[n][e] = vb[v_at[first + 8 * (e >> 2) + (e & 3)] + c];
    }
    // Keys that do not exist weigh nothing, whatever stands there.
#pragma unroll
    for (int n = 0; n < KI; ++n) {
      const int x = tid + 256 * n, key = x / (2 * KS);
      const float top = max_lanes<2 * KS>(max8(kr[n]));
      if (x - key * 2 * KS == 0) k_top[key] = key < keys ? top : 0.f;
    }
#pragma unroll
    for (int n = 0; n < VI; ++n) {
      const int x = tid + 256 * n, key = x / (4 * DT);
      const float top = max_lanes<4 * DT>(max8(vm[n]));
      if (x - key * 4 * DT == 0) v_top[key] = key < keys ? top : 0.f;
    }
    __syncthreads();
    // One power for the whole tile where its rows are of one size.
    const float kt = k_top[lane], vt = v_top[lane];
    const int kp = 127 - pair_field(kt), vp = 127 - pair_field(vt);
    k_most = wave_max_i32(kp);
    v_most = wave_max_i32(vp);
    k_flat = !__any(kt != 0.f && kp < k_most - kFlat);
    v_flat = !__any(vt != 0.f && vp < v_most - kFlat);
    if (wave == 0) {
      k_power[lane] = kp;
      v_power[lane] = vp;
    }
    // Piece c of key t: lanes t % 32 + 32 (c % 2) of step c / 2, turned by c so that a thread group's writes meet
    // different banks.
#pragma unroll
    for (int n = 0; n < KI; ++n) {
      const int x = tid + 256 * n, key = x / (2 * KS), c = x - key * 2 * KS;
      f16x8 p[2];
      pairs8(kr[n], exp_float(k_flat ? 127 - k_most : pair_field(k_top[key])), p[0], p[1]);
#pragma unroll
      for (int m = 0; m < 2; ++m)
        frag[(((key >> 5) * KS + (c >> 1)) * 2 + m) * 64 + (c & 1) * 32 + ((key + c) & 31)] = __builtin_bit_cast(u32x4, p[m]);
    }
#pragma unroll
    for (int n = 0; n < VI; ++n) {
      const int x = tid + 256 * n, c = x % (32 * DT), piece = x / (32 * DT);
      const int first = 16 * (piece >> 1) + 4 * (piece & 1);
      float scale = exp_float(127 - v_most);
      if (!v_flat) {  // a power for each of the eight: scaled before the split
#pragma unroll
        for (int e = 0; e < 8; ++e) vr[n][e] *= exp_float(pair_field(v_top[first + 8 * (e >> 2) + (e & 3)]));
        scale = 1.f;
      }
      if (keys < kKeys)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (first + 8 * (e >> 2) + (e & 3) >= keys) vr[n][e] = 0.f;
      // Any value below what pairs hold (of values of one size 1 in 10^9)?  Zeros are none.
      float least = __builtin_fabsf(vr[n][0]);
#pragma unroll
      for (int e = 1; e < 8; ++e) least = fminf(least, __builtin_fabsf(vr[n][e]));
      if (least * scale < kFine)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (vr[n][e] != 0.f && __builtin_fabsf(vr[n][e]) * scale < kFine) uneven = 1;
      f16x8 p[2];
      pairs8(vr[n], scale, p[0], p[1]);
#pragma unroll
      for (int m = 0; m < 2; ++m)
        frag[KF * 64 + (((piece >> 1) * DT + (c >> 5)) * 2 + m) * 64 + (piece & 1) * 32 + (c & 31)] =
            __builtin_bit_cast(u32x4, p[m]);
    }
    __syncthreads();
    if (uneven) {
      const int power = v_flat ? -v_most : 0;
#pragma unroll
      for (int n = 0; n < VI; ++n) {
        const float top = max8(vr[n]);
        if (top > 0.f && top <= FLT_MAX) atomicMax(&c_power[(tid + 256 * n) % (32 * DT)], __builtin_amdgcn_frexp_expf(top) - 1 + power);
      }
      __syncthreads();
#pragma unroll
      for (int n = 0; n < VI; ++n) {
        const int x = tid + 256 * n, ch = x % (32 * DT), piece = x / (32 * DT), own = c_power[ch];
        if (own < 14 - 90 && own != kNoPower) uneven = 2;
#pragma unroll
        for (int e = 0; e < 8; ++e) vr[n][e] = __builtin_ldexpf(vr[n][e], power + 14 - max(own, 14 - 90));
        f16x8 p[2];
        pairs8(vr[n], 1.f, p[0], p[1]);
#pragma unroll
        for (int m = 0; m < 2; ++m)
          frag[KF * 64 + (((piece >> 1) * DT + (ch >> 5)) * 2 + m) * 64 + (piece & 1) * 32 + (ch & 31)] =
              __builtin_bit_cast(u32x4, p[m]);
      }
      __syncthreads();
    }
  }

  auto k_at = [&](int t, int ks, int m) __attribute__((always_inline)) {
    return __builtin_bit_cast(f16x8, frag[((t * KS + ks) * 2 + m) * 64 + half * 32 + ((r32 + 2 * ks + half) & 31)]);
  };
  auto v_at_lane = [&](int st, int d, int m) __attribute__((always_inline)) {
    return __builtin_bit_cast(f16x8, frag[KF * 64 + ((st * DT + d) * 2 + m) * 64 + lane]);
  };

  // (Results pass the caches by, written here and read by the join, and so do the join's outputs: a whole call 258 us on two
  // 160x160 maps, 294 with all of them cached, 615 and 676 on 8,192 causal tokens, whose queries and keys they would
  // push out.)
  // The queries are here before the loop: in it they are waited for with the stores behind them still under way.
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  const float cs = s.scale * 1.4426950408889634f;
  for (; r < rows; r += 128) {
    f32x16 sc[2], rest[2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int x = 0; x < 16; ++x) sc[t][x] = rest[t][x] = 0.f;
    float qm = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qm = fmaxf(qm, fmaxf(max4(qr[ks][0]), max4(qr[ks][1])));
    const int q_field = pair_field(fmaxf(qm, __shfl_xor(qm, 32)));
    const float q_scale = exp_float(q_field);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      f16x8 q[2];
      const float f[8] = {qr[ks][0][0], qr[ks][0][1], qr[ks][0][2], qr[ks][0][3],
                          qr[ks][1][0], qr[ks][1][1], qr[ks][1][2], qr[ks][1][3]};
      pairs8(f, q_scale, q[0], q[1]);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const f16x8 k0 = k_at(t, ks, 0), k1 = k_at(t, ks, 1);
        rest[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k1, q[0], rest[t], 0, 0, 0);
        sc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k0, q[0], sc[t], 0, 0, 0);
        rest[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k0, q[1], rest[t], 0, 0, 0);
      }
    }
    const int seen = limit, q_power = 127 - q_field;
    const unsigned mine = to;
    place[wave][r32] = mine * (unsigned)(4 * s.hd);
    load_q(min(r + 128, rows - 1));  // the last turn: something, to keep the count of loads
    // Key 4 n + e of those that a lane holds is 8 n + 4 half + e.
    float w[32], c = cs;
    int k_top_power = k_most;
    const bool partly = __any(seen < keys);
#pragma unroll
    for (int x = 0; x < 32; ++x) w[x] = __builtin_fmaf(rest[x >> 4][x & 15], 1.f / 2048, sc[x >> 4][x & 15]);
    if (k_flat) {
      c = fmaxf(__builtin_ldexpf(cs, k_most + q_power), FLT_MIN);  // not 0, which would make hidden keys' scores NaN
    } else {
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const i32x4 power = *(const i32x4*)&k_power[8 * n + 4 * half];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[4 * n + e] = __builtin_ldexpf(w[4 * n + e], power[e] + q_power);
      }
      if (partly) {  // hidden keys have no say
        k_top_power = kNoPower;
        for (int t = half; t < seen; t += 2) k_top_power = max(k_top_power, k_power[t]);
        k_top_power = max(k_top_power, __shfl_xor(k_top_power, 32));
      }
    }
    const bool wide = !(__builtin_ldexpf(cs, k_top_power + q_power) <= kWide);
    // Keys that do not exist, and in a causal tile those that some rows do not see.
    if (keys < kKeys && !partly) {
      int end = keys;
      // With large heads compared here: 32 masks kept for the loop would be spilled (8,192 causal tokens 615 us, 604 so).
      if (KS * DT >= 16) asm("" : "+v"(end));
#pragma unroll
      for (int x = 0; x < 32; ++x)
        if (8 * (x >> 2) + 4 * half + (x & 3) >= end) w[x] = -INFINITY;
    }
    if (partly)
#pragma unroll
      for (int x = 0; x < 32; ++x)
        if (8 * (x >> 2) + 4 * half + (x & 3) >= seen) w[x] = -INFINITY;
    float mx = -INFINITY, sum = 0.f;
#pragma unroll
    for (int x = 0; x < 32; ++x) mx = fmaxf(mx, w[x]);
    mx = fmaxf(mx, __shfl_xor(mx, 32)) * c;
    const float base = mx == -INFINITY ? 0.f : mx;  // no key, or none that weighs
#pragma unroll
    for (int x = 0; x < 32; ++x) {
      w[x] = __builtin_amdgcn_exp2f(__builtin_fmaf(w[x], c, -base));
      sum += w[x];
    }
    sum += __shfl_xor(sum, 32);
    // Where values differ in size: weights times their powers, under the power of the largest such product (below 1 then; a
    // key without weight has no say in it, whatever its values).  One power for all: weights are at most 1.
    int most = v_most, w_field = 127 + 14;
    if (!v_flat) {
      w_field = 127 + 15;
      most = 2 * kNoPower;
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const i32x4 power = *(const i32x4*)&v_power[8 * n + 4 * half];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int bits = __builtin_bit_cast(int, w[4 * n + e]);  // not negative; its exponent, or far below for 0
          most = max(most, power[e] + (bits >> 23) + ((bits - 1) >> 31 & kNoPower));
        }
      }
      most = max(most, __shfl_xor(most, 32)) - 126;
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const i32x4 power = *(const i32x4*)&v_power[8 * n + 4 * half];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[4 * n + e] = __builtin_ldexpf(w[4 * n + e], power[e] - most);
      }
    }
    const float w_scale = exp_float(w_field);
    a.stat[half ? a.trash : mine] = Stat{mx, wide ? NAN : sum, most + 127 - w_field};
    f16x8 wp[4][2];
#pragma unroll
    for (int st = 0; st < 4; ++st) {
      const float f[8] = {w[8 * st],     w[8 * st + 1], w[8 * st + 2], w[8 * st + 3],
                          w[8 * st + 4], w[8 * st + 5], w[8 * st + 6], w[8 * st + 7]};
      pairs8(f, w_scale, wp[st][0], wp[st][1]);
    }
    __builtin_amdgcn_wave_barrier();
    unsigned row_at[16];  // bytes
#pragma unroll
    for (int x = 0; x < 16; ++x) row_at[x] = place[wave][8 * (x >> 2) + 4 * half + (x & 3)] + 4 * r32;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      if (!WHOLE && 32 * d >= s.hd) break;
      // The small products of every step first, then the leading ones on top.
      f32x16 acc;
#pragma unroll
      for (int x = 0; x < 16; ++x) acc[x] = 0.f;
      f16x8 lead[4];
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        lead[st] = v_at_lane(st, d, 0);
        const f16x8 v1 = v_at_lane(st, d, 1);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(wp[st][1], lead[st], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(wp[st][0], v1, acc, 0, 0, 0);
      }
#pragma unroll
      for (int x = 0; x < 16; ++x) acc[x] *= 1.f / 2048;
#pragma unroll
      for (int st = 0; st < 4; ++st) acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(wp[st][0], lead[st], acc, 0, 0, 0);
      char* base = (char*)(a.part + 32 * d);
      if (WHOLE || 32 * d + r32 < s.hd)
#pragma unroll
        for (int x = 0; x < 16; ++x) __builtin_nontemporal_store(acc[x], (float*)(base + row_at[x]));
    }
  }
  if (!uneven) return;
  // The channels' own powers come off afterwards, so that the loop does not know of them.  (All channels of one size, and one
  // 1e-12 of the others: two 160x160 maps 232 and 395 us.)
  __threadfence_block();  // results of the wave's other lanes
  const int quads = s.hd / 4;
  for (r = wave * 32; r < rows; r += 128) {
    const int count = min(32, rows - r) * quads;
    for (int n0 = lane; n0 < count; n0 += 4 * 64) {
      f32x4* of[4];
      f32x4 y[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int n = min(n0 + 64 * u, count - 1), x = n / quads;
        const unsigned row = result_row(h0 + r + x);
        of[u] = (f32x4*)(a.part + (size_t)row * s.hd) + (n - x * quads);
        y[u] = *of[u];
        if (uneven == 2 && n == x * quads) a.stat[row].sum = NAN;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int c = min(n0 + 64 * u, count - 1) % quads * 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[u][e] = __builtin_ldexpf(y[u][e], max(c_power[c + e] - 14, -90));
        if (n0 + 64 * u < count) *of[u] = y[u];
      }
    }
  }
}

// ------------------------------------------------------------------ few queries

constexpr int kFewRows = 4;

// One (query, slot) pair and part of its block per workgroup, in plain float32: the keys are read once, for the few
// heads that share them, and the time is their way from memory.  Four lanes score a key (16 keys to a wave), then
// a lane takes two channels over the same 16 keys; the four waves' results meet in LDS.  One token against 16 caches, 16
// blocks of 64 keys for 4 heads of 128 channels (67 MB): 18 us, 3.7 TB/s; as a tile on the matrix cores 33 us.
template <int KS>
__global__ __launch_bounds__(256) void block_few_kernel(const BlockArgs a) {
  __shared__ float weight[kFewRows][kKeys], q[kFewRows][128], out[4][kFewRows][128];
  const BlockShape& s = a.s;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int x = blockIdx.x;
  const int part = x % a.parts;
  x /= a.parts;
  const int pair = x % (a.span * s.selected), ls = x / (a.span * s.selected);
  const int seg = a.first + ls, plane = seg / a.segs, b = plane / s.kv, g = plane - b * s.kv;
  const int i = seg % a.segs * a.span + pair / s.selected;
  if (i >= s.tq) return;
  const int end = visible(a, b, i), j = list_of(a, b, i, g)[pair % s.selected];
  if (!block_seen(a, j, end)) return;
  const int y0 = j / s.bx * s.bh, x0 = j % s.bx * s.bw;
  const int cols = min(s.bw, s.kw - x0), size = min(s.bh, s.kh - y0) * cols;
  const int origin = y0 * s.kw + x0;
  const int keys = min(max(min(size, s.kh > 1 ? size : end - origin) - part * kKeys, 0), kKeys);
  const long long slot = ((long long)(ls * a.span * s.selected) + pair) * a.parts + part;
  auto token = [&](int t) {
    const int u = t < keys ? part * kKeys + t : 0, y = u / cols;
    return (long long)b * s.tk + origin + y * s.kw + u - y * cols;
  };
  // A quarter key's channels 16 n + 4 (lane % 4) .. + 3; two channels of the wave's 16 keys.
  const int key = wave * 16 + (lane >> 2), quarter = 4 * (lane & 3);
  f32x4 k[KS];
  f32x2v v[16];
  {
    const float* p = a.k + token(key) * a.ldk + (long long)g * s.ks + quarter;
#pragma unroll
    for (int n = 0; n < KS; ++n) k[n] = 16 * n + quarter < s.kd ? *(const f32x4*)(p + 16 * n) : f32x4{0.f, 0.f, 0.f, 0.f};
    const float* vb = a.v + (long long)g * s.vs + min(2 * lane, s.hd - 2);
#pragma unroll
    for (int t = 0; t < 16; ++t) v[t] = *(const f32x2v*)(vb + token(wave * 16 + t) * a.ldv);
  }
  const float c = s.scale * 1.4426950408889634f;
  for (int h0 = 0; h0 < s.group; h0 += kFewRows) {
    const int heads = min(kFewRows, s.group - h0);
    __syncthreads();
    for (int u = tid; u < kFewRows * 128; u += 256) {
      const int h = u >> 7, ch = u & 127;
      q[h][ch] = h < heads && ch < s.kd
                     ? a.q[((long long)b * s.tq + i) * a.ldq + (long long)(g * s.group + h0 + h) * s.qs + ch]
                     : 0.f;
    }
    __syncthreads();
    float sc[kFewRows];
#pragma unroll
    for (int h = 0; h < kFewRows; ++h) sc[h] = 0.f;
#pragma unroll
    for (int n = 0; n < KS; ++n)
#pragma unroll
      for (int h = 0; h < kFewRows; ++h) {
        const f32x4 f = *(const f32x4*)&q[h][16 * n + quarter];
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[h] = __builtin_fmaf(k[n][e], f[e], sc[h]);
      }
#pragma unroll
    for (int h = 0; h < kFewRows; ++h) {
      sc[h] += __shfl_xor(sc[h], 1);
      sc[h] += __shfl_xor(sc[h], 2);
    }
    if ((lane & 3) == 0)
#pragma unroll
      for (int h = 0; h < kFewRows; ++h) weight[h][key] = key < keys ? sc[h] : -INFINITY;
    __syncthreads();
    float mx[kFewRows], sum[kFewRows], w[kFewRows];
#pragma unroll
    for (int h = 0; h < kFewRows; ++h) {
      const float x = weight[h][lane];
      float m = x;
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
      mx[h] = m * c;
      w[h] = __builtin_amdgcn_exp2f(__builtin_fmaf(x, c, mx[h] == -INFINITY ? 0.f : -mx[h]));
      sum[h] = w[h];
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) sum[h] += __shfl_xor(sum[h], off);
    }
    f32x2v acc[kFewRows];
#pragma unroll
    for (int h = 0; h < kFewRows; ++h) acc[h] = f32x2v{0.f, 0.f};
#pragma unroll
    for (int t = 0; t < 16; ++t) {
      if (wave * 16 + t >= keys) break;
#pragma unroll
      for (int h = 0; h < kFewRows; ++h) {
        const float p = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w[h]), wave * 16 + t));
        acc[h][0] = __builtin_fmaf(p, v[t][0], acc[h][0]);
        acc[h][1] = __builtin_fmaf(p, v[t][1], acc[h][1]);
      }
    }
#pragma unroll
    for (int h = 0; h < kFewRows; ++h) *(f32x2v*)&out[wave][h][2 * lane] = acc[h];
    __syncthreads();
    for (int u = tid; u < heads * s.hd; u += 256) {
      const int h = u / s.hd, ch = u - h * s.hd;
      a.part[(slot * s.group + h0 + h) * s.hd + ch] = (out[0][h][ch] + out[1][h][ch]) + (out[2][h][ch] + out[3][h][ch]);
    }
    if (tid == 0)
#pragma unroll
      for (int h = 0; h < kFewRows; ++h)
        if (h < heads) a.stat[slot * s.group + h0 + h] = Stat{mx[h], sum[h], 0};
  }
}

// ----------------------------------------------------------------------- join

// One row in plain float32 by one wave, weights normalised before they meet the values so that no finite average
// overflows.  A lane scores one key of 64 and holds channels lane and lane + 64.
__device__ __forceinline__ void block_row(const BlockArgs& a, int b, int i, int h, int lane, float (&y)[2]) {
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

// Joins the slots of each row: L lanes of 4 channels to a row, at 5.4 TB/s.  The lanes first take a slot each (which block it
// names, its statistics), then all of them go through the slots' values, whose loads depend on nothing.  A row
// that comes out infinite or NaN (operands that are, sums that overflow, hidden keys of a tile that are not
// finite, rows too uneven for f16 pairs) is computed again in plain float32.
template <int L>
__global__ __launch_bounds__(256) void block_join_kernel(const BlockArgs a, long long rows) {
  const BlockShape& s = a.s;
  const int lane = threadIdx.x & 63, sub = lane & (L - 1), c = 4 * sub;
  const long long row = (long long)blockIdx.x * (256 / L) + threadIdx.x / L;  // (segment, query, head of the group)
  const int h = (int)(row % s.group);
  const long long query = row / s.group;
  const int d = (int)(query % a.span), ls = (int)(query / a.span);
  const int seg = a.first + ls, plane = seg / a.segs, b = plane / s.kv, g = plane - b * s.kv;
  const int i = seg % a.segs * a.span + d;
  const bool live = row < rows && i < s.tq;
  const int* list = list_of(a, live ? b : 0, live ? i : 0, live ? g : 0);
  const int end = live ? visible(a, b, i) : 0, slots = s.selected * a.parts;
  const long long home = live ? (long long)ls * a.span * s.selected : 0, first = live ? (long long)d * s.selected : 0;
  const float* part = a.part + min(c, s.hd - 4);
  float top = -INFINITY, sum = 0.f;
  int power = INT_MIN;  // of y
  bool any = false;
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
  for (int n0 = 0; n0 < slots; n0 += L) {
    const int n = n0 + sub;
    const bool on = n < slots && block_seen(a, list[min(n, slots - 1) / a.parts], end);
    any |= on;
    Stat st = {-INFINITY, 0.f, 0};
    int at = 0;
    if (on) {
      const int p = n / a.parts;
      const long long pair = a.pos ? a.pos[home + first + p] : first + p;
      at = (int)(((home + pair) * a.parts + (n - p * a.parts)) * s.group + h);
      st = a.stat[at];
    }
    float mx = st.top;
#pragma unroll
    for (int off = 1; off < L; off <<= 1) mx = fmaxf(mx, __shfl_xor(mx, off));
    mx = fmaxf(mx, top);
    // A slot's weight is 2^(its maximum - mx) as mantissa and exponent, which joins the power that its values want: the largest
    // of these powers takes the sum, so a slot without weight leaves the others' bits alone, whatever its values.
    const bool weighs = st.top != -INFINITY, had = top != -INFINITY;
    const float x = weighs ? st.top - mx : 0.f, low = fmaxf(floorf(x), kNoPower), f = weighs ? __builtin_amdgcn_exp2f(x) : 0.f;
    const float ox = had ? top - mx : 0.f, olow = fmaxf(floorf(ox), kNoPower);
    sum = __builtin_fmaf(sum, had ? __builtin_amdgcn_exp2f(ox) : 0.f, st.sum * f);
    top = mx;
    const int at_power = st.scale + (int)low, old_power = power + (int)olow;
    int most = max(weighs ? at_power : INT_MIN, had ? old_power : INT_MIN);
#pragma unroll
    for (int off = 1; off < L; off <<= 1) most = max(most, __shfl_xor(most, off));
    const float old = had ? __builtin_ldexpf(__builtin_amdgcn_exp2f(ox - floorf(ox)), old_power - most) : 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] *= old;
    power = most;
    // Negative: there is nothing to read.  A slot without weight is read all the same: a NaN in it is the row's.
    const float fv = !on ? -1.f : weighs ? __builtin_ldexpf(__builtin_amdgcn_exp2f(x - floorf(x)), at_power - most) : 0.f;
    const int count = min(L, slots - n0);
    for (int u0 = 0; u0 < count; u0 += 8) {
      f32x4 v[8];
      float w[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        w[u] = __shfl(fv, (lane & ~(L - 1)) + min(u0 + u, L - 1));
        const int row = __shfl(at, (lane & ~(L - 1)) + min(u0 + u, L - 1));
        v[u] = __builtin_nontemporal_load((const f32x4*)(part + (long long)row * s.hd));
      }
#pragma unroll
      for (int u = 0; u < 8; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (u0 + u < count) y[e] = w[u] < 0.f ? y[e] : __builtin_fmaf(v[u][e], w[u], y[e]);
    }
  }
#pragma unroll
  for (int off = 1; off < L; off <<= 1) {
    sum += __shfl_xor(sum, off);
    any = any | (bool)__shfl_xor((int)any, off);
  }
  bool again = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    y[e] = any ? __builtin_ldexpf(y[e] / sum, power) : 0.f;
    again |= live && c < s.hd && !(__builtin_fabsf(y[e]) <= FLT_MAX);
  }
  if (live && c < s.hd)
    __builtin_nontemporal_store(y, (f32x4*)(a.o + ((long long)b * s.tq + i) * a.ldo + (long long)(g * s.group + h) * s.hd + c));
  for (unsigned long long todo = __ballot(again); todo;) {
    const int from = __builtin_ctzll(todo) & ~(L - 1);
    const int rb = __shfl(b, from), ri = __shfl(i, from), rh = __shfl(g * s.group + h, from);
    float z[2];
    block_row(a, rb, ri, rh, lane, z);
    float* o = a.o + ((long long)rb * s.tq + ri) * a.ldo + (long long)rh * s.hd;
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (lane + 64 * e < s.hd) o[lane + 64 * e] = z[e];
    todo &= ~(((1ull << L) - 1) << from);
  }
}

// Tiles find their rows themselves, without the sort, where there are up to so many (every block of each image and key head
// may be named by all pairs) and lists of up to kScan: attention on one 20x20 map, 2 / 4 heads of 32 / 64 channels, 4 of 25
// blocks 15.5 / 15.3 us against 19 / 19.5; with 1,300 tiles of 64 / 64 channels 26 against 23.
constexpr int kScanTiles = 512;

// Bytes of results that one launch leaves and the next one joins.  Fewer would stay in the 256 MiB cache in front of
// memory, but cost more in half-filled launches: 8,192 causal tokens of 16 heads (1.0 GB) 978 us in pieces of 256 MB, 681 of
// 400 MB, 615 in one; two 160x160 maps (0.43 GB) 302, 286 and 258.
constexpr double kPartials = 1200e6;

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
  SY_CHECK((long long)q->n * s.kv < (1 << 24) && (long long)q->h * q->w * s.selected < (1LL << 31), SY_EUNSUPPORTED,
           "block attention over %d x %dx%d queries", q->n, q->h, q->w);
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
  // Segments: as many queries as keep the results of one in kPartials bytes
  // (and, pair by pair, its workgroups in 2^23), and as many segments to a launch.
  const double per_query = std::max((sizeof(float) * s.hd + sizeof(Stat)) * (double)s.selected * a.parts * s.group / kPartials,
                                    (double)s.selected * a.parts / (1 << 23));  // share of a launch
  a.span = (int)std::min<double>(s.tq, std::max(1.0, std::floor(1.0 / per_query)));
  a.segs = (s.tq + a.span - 1) / a.span;
  const long long segments = (long long)planes * a.segs;
  const int together = (int)std::min<double>((double)segments, std::max(1.0, std::floor(1.0 / (per_query * a.span))));
  // Pair by pair where sorting would not save many tiles: a tile of either kind takes about 10 ns (of 128 channels a
  // sorted one 30), the sort and its longer tiles 10 us.  64 queries of 4 heads, 16 of 512 blocks each: 48 us pair by
  // pair, 81 sorted; 256 queries 153 and 89; one 20x20 map (2 heads, 4 of 25 blocks) 32 and 21.
  const double singles = (double)planes * s.tq * s.selected * a.parts;
  const double shared = (double)planes * a.parts * std::min((double)s.blocks, (double)s.tq * s.selected);
  const bool sorted = s.blocks <= kMaxBlocks && singles > 1.5 * shared + 1024;
  // Rows of a tile at most: many, so that the keys are laid out seldom, but a round of tiles on the whole chip (three
  // workgroups to a CU).
  a.rows = kTileRows;
  while (a.rows > 128 && (double)together * a.span * s.selected * a.parts * s.group < 768.0 * a.rows) a.rows /= 2;
  // 2048 pairs to a workgroup of the sort, but at most 32 of them to a segment (each reads all their counts).
  a.chunk = std::max(std::max(1, 2048 / s.selected), (a.span + 31) / 32);
  a.chunks = (a.span + a.chunk - 1) / a.chunk;
  const long long pairs = (long long)a.span * s.selected;
  auto scan_tiles = [&](long long rows) {
    return planes * (long long)a.parts * s.blocks * ((pairs * s.group + rows - 1) / rows);
  };
  const bool scan = sorted && a.segs == 1 && pairs <= kScan && scan_tiles(kTileRows) <= kScanTiles;
  while (scan && scan_tiles(a.rows) > kScanTiles) a.rows *= 2;
  const long long tile_cap =
      scan ? scan_tiles(a.rows) / planes : a.parts * (std::min<long long>(s.blocks, pairs) + pairs * s.group / a.rows + 1);
  const long long result_rows = together * pairs * a.parts * s.group;
  SY_CHECK((result_rows + 1) * s.hd < (1LL << 30) - 128 && tile_cap * together < (1LL << 24), SY_EUNSUPPORTED,
           "block attention over %d heads to a key head", s.group);
  SY_CHECK(!sorted || (long long)together * a.chunks * kSortThreads < (1LL << 32), SY_EUNSUPPORTED,
           "block attention over %d lists", together);
  SY_CHECK(((s.bh - 1.0) * s.kw + s.bw) * std::max(k->ldc, v->ldc) < 4294967296.0, SY_EUNSUPPORTED,
           "block windows that span 2^32 floats and more");
  a.tile_cap = (int)tile_cap;
  a.trash = (unsigned)result_rows;
  // Scratch, of one launch: results, then lists.
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t from = at;
    at += (bytes + 255) & ~size_t(255);
    return from;
  };
  const size_t part_at = take(sizeof(float) * ((result_rows + 1) * s.hd + 128)),
               stat_at = take(sizeof(Stat) * (result_rows + 1));
  const size_t count_at = sorted && !scan ? take(sizeof(int) * together * a.chunks * s.blocks) : 0;
  const size_t list_at = sorted && !scan ? take(sizeof(int) * together * pairs) : 0;
  const size_t pos_at = sorted && !scan ? take(sizeof(int) * together * pairs) : 0;
  const size_t tile_at = sorted && !scan ? take(sizeof(int4) * together * tile_cap) : 0;
  const size_t number_at = sorted && !scan ? take(sizeof(int) * together) : 0;
  DeviceScope device(ctx);
  SY_TRY(ensure_scratch(ctx, at));
  a.part = (float*)(ctx->scratch + part_at);
  a.stat = (Stat*)(ctx->scratch + stat_at);
  a.counts = (int*)(ctx->scratch + count_at);
  a.list = sorted && !scan ? (int*)(ctx->scratch + list_at) : nullptr;
  a.pos = sorted && !scan ? (int*)(ctx->scratch + pos_at) : nullptr;
  a.tiles = (int4*)(ctx->scratch + tile_at);
  a.tile_count = (int*)(ctx->scratch + number_at);
  const double keys = std::min((double)s.selected * s.bh * s.bw, (double)s.tk);
  for (long long first = 0; first < segments; first += together) {
    const int now = (int)std::min<long long>(together, segments - first);
    const double share = (double)now / segments;
    a.first = (int)first;
    a.now = now;
    if (sorted && !scan) {
      ProfScope prof(ctx, "block_sort", 0, share * 8.0 * s.n * (double)s.tq * s.kv * s.selected);
      const size_t lds = sizeof(int) * s.blocks;
      const dim3 grid((unsigned)(now * a.chunks)), threads(kSortThreads);
      if (a.chunks > 1) hipLaunchKernelGGL(block_count_kernel, grid, threads, lds, ctx->stream, a);
      hipLaunchKernelGGL(block_scatter_kernel, grid, threads, lds, ctx->stream, a);
      SY_TRY(check_launch("block_sort"));
    }
    {
      ProfScope prof(ctx, sorted ? "block_attention" : "block_few", share * 2.0 * s.n * s.tq * s.heads * keys * (s.kd + s.hd),
                     share * 4.0 * s.n * ((double)s.tq * s.heads * (s.kd + s.hd) + (double)s.tk * s.kv * (s.kd + s.hd)));
      if (sorted) {
        const unsigned grid = (unsigned)((now * tile_cap + 7) / 8 * 8);
        auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, ctx->stream, a); };
        auto pick = [&](auto whole2, auto part2, auto whole4, auto part4) {
          if (s.hd <= 64)
            launch(s.hd == 64 ? whole2 : part2);
          else
            launch(s.hd == 128 ? whole4 : part4);
        };
        if (s.kd <= 32)
          pick(block_tile_kernel<2, 2, true>, block_tile_kernel<2, 2, false>, block_tile_kernel<2, 4, true>,
               block_tile_kernel<2, 4, false>);
        else if (s.kd <= 64)
          pick(block_tile_kernel<4, 2, true>, block_tile_kernel<4, 2, false>, block_tile_kernel<4, 4, true>,
               block_tile_kernel<4, 4, false>);
        else
          pick(block_tile_kernel<8, 2, true>, block_tile_kernel<8, 2, false>, block_tile_kernel<8, 4, true>,
               block_tile_kernel<8, 4, false>);
      } else {
        const dim3 grid((unsigned)(now * pairs * a.parts));
        if (s.kd <= 64)
          hipLaunchKernelGGL(block_few_kernel<4>, grid, dim3(256), 0, ctx->stream, a);
        else
          hipLaunchKernelGGL(block_few_kernel<8>, grid, dim3(256), 0, ctx->stream, a);
      }
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
