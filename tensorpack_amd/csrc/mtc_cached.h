// Attention of the newest tokens over a paged cache: how the work is dealt out, joined and launched. The kernels are
// templates over a Store, which knows how the cache holds K and V:
//   Call                         CachedCall, or one that adds to it
//   E                            the 16-bit type of q, o and the tiles
//   kKeys                        split keys: keys of a unit, a wave's step (at least kLeastKeys)
//   kCodes                       whether the cache is MTC_CACHE_CODES8
//   kStart, kStartAlone          units that stand for an item's start, in runs of blocks and of single waves (up to most_start(kCodes))
//   kCostRows, kCostKeys         of a unit of split rows, of split keys, for dealing blocks to prefixes and own parts
//   kShort                       up to as many units per item on average, runs of single waves
//   kKeysBytes<DP>               LDS that keys<DP, ...> uses
//   keys<DP, MODE, PREFIX>(...)  one item's keys [from, to) into a partial result, few rows
//   rows<DP, PREFIX>(...)        the same, up to 128 rows
//   join_again(...)              whether the row was computed anew, because of what it does not see
#pragma once

#include <algorithm>
#include <cmath>

#include "mtc_codes.h"
#include "mtc_host.h"
#include "mtc_rowtile.h"
#include "mtc_serve.h"

namespace mtc {
namespace attn {

// ---------------------------------------------------------------------------
// the newest tokens over a paged cache
// ---------------------------------------------------------------------------
// Work. An item is one K/V head and one tile of query rows over the keys of one entry: of a sequence's
// own part (rows: its tokens x the heads of the K/V head) or of a group's prefix (rows: those of all members).
// Items are cut into units of keys, with a few more at their start that stand for the time an item takes whatever its
// length; the units of all items, in order, are dealt out to the blocks in equal runs, so short and long sequences
// fill the chip alike and nothing on the host depends on lengths. A run crosses items; each crossing gives one partial
// result (maximum, sum, weighted values). Its slot is run + item: both only grow along the runs and every crossing
// raises one of them, so no two share a slot.
//
// Three ways through an item's keys, for 16, 32 and 128 rows:
//   split keys   16 or 32 rows (the first two), units of kKeys keys (32 of 16-bit numbers, 64 of codes): for few rows the
//                keys' bytes are all that counts, and every wave keeps loads of its own in flight. A run belongs to a block, whose waves take every fourth unit and are joined
//                at the end, or, where items are short, to a single wave (64 sequences of 100 keys, 8 K/V heads: an item
//                takes a block or a wave about 5 us of waiting whatever its length)
//   split rows   up to 128 rows, units of 64 keys, a run per block: as in k_prompt, 32 rows per wave, and the waves share
//                each tile of keys in LDS
constexpr int kCachedWaves = 4;
constexpr int kCachedThreads = 64 * kCachedWaves;
constexpr int kCachedBlocks = 512;         // two per CU
constexpr int kXcds = 8;
constexpr int kLeastKeys = 32;             // of any Store
constexpr int most_start(bool codes) { return codes ? 5 : 4; }
constexpr int kJoinHead = 8;               // words
constexpr int kManyRows = 128;             // split rows: rows of a tile
// Measured over the 16-bit cache with 64 sequences on one prefix of 8192, 16 x 6 drafts on prefixes of 1536, 32 sequences of 0 to
// 16384 and 64 of 1 to 512 (14/2 heads of 64, 32/8 of 128): starts of 1/2, 2/3, 2/5 and 3/3 units are within 6 %
// of each other but for 1/2 (32 ragged: 48 us against 43); a prefix's unit at 0.9, 1.5 and 2.8 times a unit of keys
// gives the first case 47, 37 and 34 us, at 5 times 38.
constexpr int kStartRows = 2;              // split rows: units that stand for an item's start
constexpr int kLeastRows = 2;                    // split rows: units of a run (drafts 14.9 us; 4: 17.4, 8: 21)
enum { kNone = 0, kOneTile = 1, kTwoTiles = 2, kRows = 3 };      // 16 rows, 32 rows, split rows
__host__ __device__ constexpr int mode_rows(int mode) { return mode == kRows ? kManyRows : 16 * mode; }
template <class Store>
__host__ __device__ constexpr int mode_start(int mode, bool alone) {
  static_assert(std::max({Store::kStart, Store::kStartAlone, kStartRows}) <= most_start(Store::kCodes), "plan_cached counts with it");
  return mode == kRows ? kStartRows : alone ? Store::kStartAlone : Store::kStart;
}
template <class Store>
__host__ __device__ constexpr int mode_unit(int mode) { return mode == kRows ? kPromptKeys : Store::kKeys; }

struct Pass {                              // the own parts, or the prefixes
  float* part;                             // [slot][stride][dim]
  float* ml;                               // [slot][stride][2]: maximum (times c), sum
  int32_t stride, slots;
};
// Units dealt out to runs: the first `rest` of them get each + 1, the others each.
struct Deal {
  int32_t each, rest;
  __device__ __forceinline__ int start(int run) const { return run * each + min(run, rest); }
  __device__ __forceinline__ int run_of(int unit) const {        // only where units were dealt: each + 1 > 0
    const int big = rest * (each + 1);
    return unit < big ? unit / (each + 1) : rest + (unit - big) / max(each, 1);
  }
};
struct JoinPart {                          // what k_join needs of an entry
  int32_t units_before, items_before, units, tiles;
};
struct JoinEntry {                         // of a sequence: its own part, its group's prefix (units 0: none)
  JoinPart own, pre;
  int32_t first, reserved;                 // first sequence of the group
};
struct CachedCall {
  const uint16_t* pool;
  int64_t page_elems;                      // elements of a page, all layers
  int64_t k_off, v_off;                    // of the layer's K and V within a page
  int32_t kv_heads, dim, page_log, n_pages, max_pages, max_seqs;
  const int32_t *table, *lens;
  mtc_heads q, o;
  const int32_t *seqs, *q_lens, *groups, *prefix_lens;
  int32_t n_seqs, tokens, heads, n_groups;
  float c;
  Pass own, pre;
  int32_t* join;                           // Deal of the own parts, of the prefixes, their starts (kJoinHead words); then the entries
};

struct Seq {
  int row, len, q_len;                     // table row (0 if out of range: it then holds nothing), tokens, queries
};
__device__ __forceinline__ Seq cached_seq(const CachedCall& a, int b) {
  Seq s;
  s.row = a.seqs ? a.seqs[b] : b;
  s.q_len = a.q_lens ? min(max(a.q_lens[b], 0), a.tokens) : a.tokens;
  const bool good = (uint32_t)s.row < (uint32_t)a.max_seqs;
  if (!good) s.row = 0;
  s.len = good ? min(max(a.lens[s.row], 0), a.max_pages << a.page_log) : 0;
  return s;
}
__device__ __forceinline__ int row_sees(int len, int q_len, int t) { return t < q_len ? max(len - q_len + t + 1, 0) : 0; }
__device__ __forceinline__ int group_start(const CachedCall& a, int g) { return min(max(a.groups[g], 0), a.n_seqs); }
__device__ __forceinline__ int prefix_tokens(const CachedCall& a, int g) {
  return min(max(a.prefix_lens[g], 0) >> a.page_log, a.max_pages) << a.page_log;
}
// The group g with start(g) <= b < start(g + 1), -1: none.
template <class Start>
__device__ __forceinline__ int group_of(int n_groups, int b, Start start) {
  int lo = 0, hi = n_groups;
  if (hi == 0 || start(0) > b || start(hi) <= b) return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start(mid) <= b) lo = mid; else hi = mid;
  }
  return lo;
}

// What the lists say of the sequences and groups: read once into LDS where they fit (two rounds of loads for
// the whole call instead of a chain of them per lookup), else looked up in memory each time.
constexpr int kBook = 512;
struct Book {
  int2* seq;                               // row | q_len << 16, len
  int* group;                              // starts
  int* prefix;                             // tokens
  bool kept;
  __device__ __forceinline__ Seq get(const CachedCall& a, int b) const {
    if (!kept) return cached_seq(a, b);
    const int2 x = seq[b];
    return Seq{x.x & 0xFFFF, x.y, x.x >> 16};
  }
  __device__ __forceinline__ int start(const CachedCall& a, int g) const { return kept ? group[g] : group_start(a, g); }
  __device__ __forceinline__ int tokens(const CachedCall& a, int g) const { return kept ? prefix[g] : prefix_tokens(a, g); }
};
__device__ void fill_book(const CachedCall& a, const Book& k) {
  if (!k.kept) return;
  for (int i = threadIdx.x; i < a.n_seqs; i += kCachedThreads) {
    const Seq s = cached_seq(a, i);
    k.seq[i] = make_int2(s.row | s.q_len << 16, s.len);
  }
  for (int i = threadIdx.x; i <= a.n_groups && a.n_groups; i += kCachedThreads) {
    k.group[i] = group_start(a, i);
    if (i < a.n_groups) k.prefix[i] = prefix_tokens(a, i);
  }
  __syncthreads();
}

struct Entry {
  int rows, tiles, items;                  // query rows, row tiles, items (tiles of every K/V head)
  int units;                               // of keys, of each item; 0: none
  int from, to;                            // keys
  int first, group;                        // batch entry that the keys belong to; own part: its group
  Seq seq;                                 // of `first`
  __device__ __forceinline__ int with(int start) const { return units ? units + start : 0; }
};
template <class Store, bool PREFIX, int MODE>
__device__ __forceinline__ Entry cached_entry(const CachedCall& a, const Book& book, int e) {
  Entry r;
  const int per = a.tokens * (a.heads / a.kv_heads);
  r.from = 0;
  if constexpr (PREFIX) {
    r.first = book.start(a, e);
    r.rows = max(book.start(a, e + 1) - r.first, 0) * per;
    r.group = e;
    r.seq = book.get(a, min(r.first, a.n_seqs - 1));
    r.to = r.rows ? min(book.tokens(a, e), r.seq.len) : 0;
  } else {
    r.first = e;
    r.rows = per;
    r.seq = book.get(a, e);
    r.group = group_of(a.n_groups, e, [&](int g) { return book.start(a, g); });
    if (r.group >= 0) r.from = book.tokens(a, r.group);
    r.to = r.seq.len;
  }
  r.tiles = (r.rows + mode_rows(MODE) - 1) / mode_rows(MODE);
  r.items = a.kv_heads * r.tiles;
  r.units = r.to > r.from ? (r.to - r.from + mode_unit<Store>(MODE) - 1) / mode_unit<Store>(MODE) : 0;
  return r;
}

// Running sums over the entries: every thread of the block has the sums before its run of entries [e0, e1).
struct Scan {
  int e0, e1, units, own, items;           // own: units of the run
  int total, all_items;
  int held, own_held, all_held;            // items that have keys
  // Units of keys become units with `start` more for each item.
  __device__ __forceinline__ void add_starts(int start) {
    units += start * held;
    own += start * own_held;
    total += start * all_held;
  }
};
template <class Store, bool PREFIX, int MODE>
__device__ Scan cached_scan(const CachedCall& a, const Book& book, int (&shared)[3][kCachedWaves]) {
  const int n = PREFIX ? a.n_groups : a.n_seqs, per = (n + kCachedThreads - 1) / kCachedThreads;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Scan r;
  r.e0 = min((int)threadIdx.x * per, n);
  r.e1 = min(r.e0 + per, n);
  int u = 0, it = 0, held = 0;
  for (int e = r.e0; e < r.e1; ++e) {
    const Entry x = cached_entry<Store, PREFIX, MODE>(a, book, e);
    u += x.items * x.units;
    it += x.items;
    held += x.units ? x.items : 0;
  }
  const int su = wave_scan(u), si = wave_scan(it), sh = wave_scan(held);
  if (lane == 63) {
    shared[0][wave] = su;
    shared[1][wave] = si;
    shared[2][wave] = sh;
  }
  __syncthreads();
  r.own = u;
  r.own_held = held;
  r.units = su - u;
  r.items = si - it;
  r.held = sh - held;
  r.total = r.all_items = r.all_held = 0;
#pragma unroll
  for (int w = 0; w < kCachedWaves; ++w) {
    if (w < wave) {
      r.units += shared[0][w];
      r.items += shared[1][w];
      r.held += shared[2][w];
    }
    r.total += shared[0][w];
    r.all_items += shared[1][w];
    r.all_held += shared[2][w];
  }
  return r;
}

// Page ids of 64 consecutive table entries, one per lane.
struct PageWindow {
  const int32_t* row;
  int at, ids, max_pages;
  __device__ __forceinline__ void load(int page) {
    at = page;
    const int i = page + (threadIdx.x & 63);
    ids = i < max_pages ? row[i] : -1;
  }
  __device__ __forceinline__ int operator()(int page) const { return __builtin_amdgcn_readlane(ids, min(page - at, 63)); }
};

// Query row rr of an item: its place in q, and the keys it sees.
template <bool PREFIX>
__device__ __forceinline__ const uint16_t* cached_query(const CachedCall& a, const Book& book, const Entry& x, int kvh, int rr, int& seen) {
  const int G = a.heads / a.kv_heads, per = a.tokens * G;
  const bool good = rr < x.rows;
  const int b = PREFIX && good ? x.first + rr / per : min(x.first, a.n_seqs - 1), t = good ? rr % per / G : 0, h = kvh * G + rr % G;
  if constexpr (PREFIX) {
    const Seq s = book.get(a, b);
    seen = good ? row_sees(s.len, s.q_len, t) : 0;
  } else {
    seen = good ? row_sees(x.seq.len, x.seq.q_len, t) : 0;
  }
  return reinterpret_cast<const uint16_t*>(a.q.data) + ((int64_t)b * a.tokens + t) * a.q.row_stride + (int64_t)h * a.q.head_stride;
}

// A wave's part of an item: rows rt * 16 + n of up to 16 MT, element i of o[rt][d] dim 16 d + 4 w + i. By the wave alone, or joined with
// the block's other waves.
template <int DP, int MT>
__device__ __forceinline__ void store_keys(const Pass& ps, char* lds, int slot, bool alone, int rows, int D, f32x4 (&o)[MT][DP / 16],
                                           float (&top)[MT], float (&sum)[MT]) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, w = lane >> 4;
#pragma unroll
  for (int rt = 0; rt < MT; ++rt) sum[rt] = half_sum(sum[rt] + __shfl_xor(sum[rt], 16));
  const bool store = slot >= 0 && slot < ps.slots;
  if (alone) {
#pragma unroll
    for (int rt = 0; rt < MT; ++rt) {
      const int r = rt * 16 + n;
      if (!store || r >= rows) continue;
      const int64_t at = (int64_t)slot * ps.stride + r;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d)
        if (d * 16 + 4 * w < D) *reinterpret_cast<f32x4*>(ps.part + at * D + d * 16 + 4 * w) = o[rt][d];
      if (w == 0) *reinterpret_cast<float2*>(ps.ml + at * 2) = make_float2(top[rt], sum[rt]);
    }
    return;
  }
  // join the four waves
  constexpr int kPad = DP + 4;
  float* const buf = reinterpret_cast<float*>(lds);                 // [wave][16][kPad]
  float* const ml = buf + kCachedWaves * 16 * kPad;                 // [wave][16 MT][2]
  __syncthreads();                                                  // every wave is done with its tiles
#pragma unroll
  for (int rt = 0; rt < MT; ++rt)
    if (w == 0) {
      ml[(wave * 16 * MT + rt * 16 + n) * 2] = top[rt];
      ml[(wave * 16 * MT + rt * 16 + n) * 2 + 1] = sum[rt];
    }
  __syncthreads();
#pragma unroll
  for (int rt = 0; rt < MT; ++rt) {
    const int r = rt * 16 + n;
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int v = 0; v < kCachedWaves; ++v) m = fmaxf(m, ml[(v * 16 * MT + r) * 2]);
    const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int v = 0; v < kCachedWaves; ++v) l += ml[(v * 16 * MT + r) * 2 + 1] * exp2_fast(ml[(v * 16 * MT + r) * 2] - base);
    const float f = exp2_fast(top[rt] - base);
#pragma unroll
    for (int d = 0; d < DP / 16; ++d)
      *reinterpret_cast<f32x4*>(buf + (wave * 16 + n) * kPad + d * 16 + 4 * w) = o[rt][d] * f;
    if (store && wave == 0 && w == 0 && r < rows) {
      float* at = ps.ml + ((int64_t)slot * ps.stride + r) * 2;
      at[0] = m;
      at[1] = l;
    }
    __syncthreads();
    for (int i = tid; i < 16 * (DP / 4); i += kCachedThreads) {
      const int rr = i / (DP / 4), d = i % (DP / 4) * 4;
      f32x4 y = f32x4{};
#pragma unroll
      for (int v = 0; v < kCachedWaves; ++v) y += *reinterpret_cast<const f32x4*>(buf + (v * 16 + rr) * kPad + d);
      if (store && rt * 16 + rr < rows && d < D)
        *reinterpret_cast<f32x4*>(ps.part + ((int64_t)slot * ps.stride + rt * 16 + rr) * D + d) = y;
    }
    __syncthreads();
  }
}

// The partial result of row r of an item, out of a row tile (sum: of both lane halves).
template <bool BF, int DP>
__device__ __forceinline__ void store_rows(const Pass& ps, int slot, int r, int D, const RowTile<BF, DP>& rt, float sum) {
  const int half = (threadIdx.x >> 5) & 1;
  float* po = ps.part + ((int64_t)slot * ps.stride + r) * D;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int dim = d * 32 + 2 * e + 4 * half;
      if (dim < D) *reinterpret_cast<f32x4*>(po + dim) = f32x4{rt.o[d][e], rt.o[d][e + 1], rt.o[d][e + 2], rt.o[d][e + 3]};
    }
  if (half == 0) {
    float* pm = ps.ml + ((int64_t)slot * ps.stride + r) * 2;
    pm[0] = rt.top;
    pm[1] = sum;
  }
}

// How the units of a pass are dealt out.
struct Plan {
  Deal deal;
  int runs;
  bool alone;                              // runs of single waves, not of blocks
  int start;                               // units of an item's start
};
template <class Store>
__device__ __forceinline__ bool short_items(const Scan& sc, int mode) {
  const int start = mode_start<Store>(mode, false);
  return mode != kRows && sc.total + start * sc.all_held <= (Store::kShort + start) * sc.all_items;
}
template <class Store>
__device__ __forceinline__ Plan deal_out(Scan& sc, int blocks, int mode) {
  Plan p;
  p.alone = short_items<Store>(sc, mode);
  p.start = mode_start<Store>(mode, p.alone);
  sc.add_starts(p.start);
  const int units = sc.total;
  const int least = mode == kRows ? kLeastRows : 1;
  p.runs = min(p.alone ? blocks * kCachedWaves : blocks, (units + least - 1) / least);
  p.deal.each = units / max(p.runs, 1);
  p.deal.rest = units % max(p.runs, 1);
  return p;
}

// The runs of block `me` of `blocks`.
template <class Store, int DP, int MODE, bool PREFIX>
__device__ void cached_run(const typename Store::Call& a, const Book& book, char* lds, const Scan& sc, const Plan& plan, int me, int blocks) {
  __shared__ int found[kCachedWaves][3];
  const int n = PREFIX ? a.n_groups : a.n_seqs;
  const int wave = plan.alone ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  if (me >= plan.runs) return;                                       // its other waves' runs come after
  if (threadIdx.x < 3 * kCachedWaves) (&found[0][0])[threadIdx.x] = 0;
  __syncthreads();
  for (int k = 0; k < (plan.alone ? kCachedWaves : 1); ++k) {
    const int run = me + k * blocks, u = plan.deal.start(run);
    if (run >= plan.runs || u < sc.units || u >= sc.units + sc.own) continue;   // one thread: its run of entries holds u
    int before = sc.units, items = sc.items;
    for (int e = sc.e0; e < sc.e1; ++e) {
      const Entry x = cached_entry<Store, PREFIX, MODE>(a, book, e);
      const int all = x.items * x.with(plan.start);
      if (u < before + all) {
        found[k][0] = e;
        found[k][1] = u - before;
        found[k][2] = items;
        break;
      }
      before += all;
      items += x.items;
    }
  }
  __syncthreads();
  const int run = me + wave * blocks;
  if (run >= plan.runs) return;
  // (groups that are not in order can overflow the sums: what follows stays within the entries all the same)
  int e = min(max(__builtin_amdgcn_readfirstlane(found[wave][0]), 0), n - 1), items = __builtin_amdgcn_readfirstlane(found[wave][2]);
  const int in = max(__builtin_amdgcn_readfirstlane(found[wave][1]), 0);
  int left = plan.deal.each + (run < plan.deal.rest);
  Entry x = cached_entry<Store, PREFIX, MODE>(a, book, e);
  if (x.units == 0 || x.items == 0) return;
  int item = min(in / x.with(plan.start), x.items - 1), unit = in % x.with(plan.start);
  while (true) {
    const int units = min(left, x.with(plan.start) - unit);
    const int from = x.from + max(unit - plan.start, 0) * mode_unit<Store>(MODE);
    const int to = min(x.from + (unit + units - plan.start) * mode_unit<Store>(MODE), x.to);
    if (to > from) {
      if constexpr (MODE == kRows) Store::template rows<DP, PREFIX>(a, book, lds, x, item, from, to, run + items + item);
      else Store::template keys<DP, MODE, PREFIX>(a, book, lds, x, item, from, to, run + items + item, plan.alone);
    }
    left -= units;
    if (left <= 0) break;
    unit = 0;
    if (++item == x.items) {
      item = 0;
      do {                                               // left > 0: a further entry has units
        items += x.items;
        if (++e >= n) return;
        x = cached_entry<Store, PREFIX, MODE>(a, book, e);
      } while (x.items == 0 || x.units == 0);
    }
  }
}

// Run of the at-th of `each` blocks of an XCD: XCD after XCD in consecutive runs, as many on each.
__device__ __forceinline__ int spread(int xcd, int at, int each, int runs) {
  const int per = (min(runs, each * kXcds) + kXcds - 1) / kXcds;
  return at < per ? xcd * per + at : runs;
}

// 512 blocks whatever the call. Every block reads the lists and sums the units by itself (3.5 us until its first keys'
// copies start, 4.5 with groups), which is less than a planning launch would take.
// Bound by memory for few rows: 32 sequences of 8192, 32/8 heads of 128: 1.07 GB in 190 to 194 us, 5.6 TB/s (a 1 GiB copy: 5.2);
// 32 ragged up to 16384: 252 MB in 41 us. 64 sequences on one prefix of 8192: 35 us, where the prefix's 2048 units of
// 128 rows take 9.6 us of the whole chip and 26 MB of own keys 4.6; what is left is the start, the partial results (64 KB a
// run) and blocks that share a CU. Smallest calls: 6 us.
template <class Store, int DP, int OWN, int PRE>
__global__ __launch_bounds__(kCachedThreads, 2) void k_cached(const typename Store::Call a) {
  constexpr int kStage = Store::template kKeysBytes<DP>, kTiles = 4 * kPromptKeys * DP * 2;
  constexpr int kBytes = (OWN == kRows || PRE == kRows) && kTiles > kStage ? kTiles : kStage;
  __shared__ __attribute__((aligned(1024))) char lds[kBytes];
  __shared__ int shared[2][3][kCachedWaves];
  static_assert(kCachedWaves * (16 * (DP + 4) + 32 * 2) * 4 <= kStage, "the join fits the tiles' space");
  __shared__ int2 book_seq[kBook];
  __shared__ int book_group[PRE == kNone ? 1 : kBook + 1], book_prefix[PRE == kNone ? 1 : kBook];
  const Book book{book_seq, book_group, book_prefix, a.n_seqs <= kBook};
  fill_book(a, book);
  Scan own = cached_scan<Store, false, OWN>(a, book, shared[0]);
  Scan pre;
  pre.total = pre.all_items = pre.all_held = 0;
  if constexpr (PRE != kNone) pre = cached_scan<Store, true, PRE>(a, book, shared[1]);

  // blocks for the prefixes: their share of the cost
  int n_pre = 0;
  if constexpr (PRE != kNone) {
    auto cost = [](const Scan& sc, int mode) {
      return (sc.total + mode_start<Store>(mode, short_items<Store>(sc, mode)) * sc.all_held) * (mode == kRows ? Store::kCostRows : Store::kCostKeys);
    };
    const float wp = cost(pre, PRE), wo = cost(own, OWN);
    if (pre.total) n_pre = own.total ? min(max((int)(kCachedBlocks / kXcds * wp / (wp + wo) + 0.5f), 1), kCachedBlocks / kXcds - 1) * kXcds : kCachedBlocks;
  }
  const Plan own_plan = deal_out<Store>(own, kCachedBlocks - n_pre, OWN);
  Plan pre_plan = own_plan;
  if constexpr (PRE != kNone) pre_plan = deal_out<Store>(pre, n_pre, PRE);
  if (blockIdx.x == kCachedBlocks - 1) {                 // for k_join
    if (threadIdx.x == 0) {
      reinterpret_cast<Deal*>(a.join)[0] = own_plan.deal;
      reinterpret_cast<Deal*>(a.join)[1] = pre_plan.deal;
      a.join[4] = own_plan.start;
      a.join[5] = pre_plan.start;
    }
    JoinEntry* je = reinterpret_cast<JoinEntry*>(a.join + kJoinHead);
    JoinPart* jg = reinterpret_cast<JoinPart*>(je + a.n_seqs);      // the groups' parts, until the sequences have them
    int u, it;
    if constexpr (PRE != kNone) {
      u = pre.units;
      it = pre.items;
      for (int e = pre.e0; e < pre.e1; ++e) {
        const Entry x = cached_entry<Store, true, PRE>(a, book, e);
        jg[e] = JoinPart{u, it, x.with(pre_plan.start), x.tiles};
        u += x.items * x.with(pre_plan.start);
        it += x.items;
      }
      __syncthreads();
    }
    u = own.units;
    it = own.items;
    for (int e = own.e0; e < own.e1; ++e) {
      const Entry x = cached_entry<Store, false, OWN>(a, book, e);
      je[e].own = JoinPart{u, it, x.with(own_plan.start), x.tiles};
      je[e].pre = PRE != kNone && x.group >= 0 ? jg[x.group] : JoinPart{0, 0, 0, 0};
      je[e].first = PRE != kNone && x.group >= 0 ? book.start(a, x.group) : 0;
      u += x.items * x.with(own_plan.start);
      it += x.items;
    }
  }
  // consecutive runs on one XCD: row tiles that read the same keys then share its L2
  const int xcd = blockIdx.x % kXcds, at = blockIdx.x / kXcds, pre_each = n_pre / kXcds, own_each = kCachedBlocks / kXcds - pre_each;
  if constexpr (PRE != kNone) {
    if (at < pre_each) {
      cached_run<Store, DP, PRE, true>(a, book, lds, pre, pre_plan, spread(xcd, at, pre_each, pre_plan.runs), n_pre);
      return;
    }
  }
  cached_run<Store, DP, OWN, false>(a, book, lds, own, own_plan, spread(xcd, at - pre_each, own_each, own_plan.runs), kCachedBlocks - n_pre);
}

// One wave per (sequence, token, head): the partial results of its row, the prefix's and the own part's. A lane holds
// four dims: a quarter (DP 64) or half of the wave reads one slot's row, so one load covers several slots, and eight
// loads are in flight (one dim a lane and four loads: 9 to 15 us for 32 ragged sequences, now 4.8).
template <class Store, int DP>
__global__ __launch_bounds__(kCachedThreads) void k_join(const typename Store::Call a, int own_rows, int pre_rows) {
  constexpr int kLanes = DP / 4, kPer = 64 / kLanes, kBatch = 8;      // lanes and slots per load, loads in flight
  const int b = blockIdx.x, lane = threadIdx.x & 63;
  const int G = a.heads / a.kv_heads, D = a.dim;
  const int row = blockIdx.y * kCachedWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);   // t * heads + h
  if (row >= a.tokens * a.heads) return;
  const int t = row / a.heads, h = row % a.heads, kvh = h / G;
  const Deal* deals = reinterpret_cast<const Deal*>(a.join);
  const JoinEntry je = reinterpret_cast<const JoinEntry*>(a.join + kJoinHead)[b];
  const int own_start = a.join[4], pre_start = a.join[5];
  const int sub = lane / kLanes, dim = lane % kLanes * 4;
  float m = -INFINITY, l = 0.0f;
  f32x4 y = f32x4{};
  auto add = [&](const Pass& ps, const JoinPart& x, int tile_rows, int start, int rr, const Deal& deal) {
    if (x.units <= start) return;
    const int item = kvh * x.tiles + rr / tile_rows, r = rr % tile_rows;
    const int u0 = x.units_before + item * x.units;
    const int i0 = deal.run_of(u0 + start), i1 = deal.run_of(u0 + x.units - 1), s0 = i0 + x.items_before + item;
    const int n = s0 < 0 ? 0 : min(i1 - i0 + 1, ps.slots - s0);
    const float* pm = ps.ml + ((int64_t)s0 * ps.stride + r) * 2;
    const float* po = ps.part + ((int64_t)s0 * ps.stride + r) * D + dim;
    const int64_t step = (int64_t)ps.stride * D;
    for (int c0 = 0; c0 < n; c0 += 64) {                 // one slot per lane: maximum, weight, sum
      float2 ml = make_float2(-INFINITY, 0.0f);
      if (c0 + lane < n) ml = *reinterpret_cast<const float2*>(pm + (int64_t)(c0 + lane) * ps.stride * 2);
      const float top = fmaxf(m, wave_max(ml.x)), base = top == -INFINITY ? 0.0f : top;
      const float f = exp2_fast(m - base), w = exp2_fast(ml.x - base);
      l = l * f + wave_sum(ml.y * w);
      y *= f;
      m = top;
      const int k = min(64, n - c0);
      for (int i = 0; i < k; i += kPer * kBatch) {
        f32x4 z[kBatch];
#pragma unroll
        for (int v = 0; v < kBatch; ++v) {
          const int at = i + v * kPer + sub;
          z[v] = at < k && dim < D ? *reinterpret_cast<const f32x4*>(po + (c0 + at) * step) : f32x4{};
        }
#pragma unroll
        for (int v = 0; v < kBatch; ++v) y += z[v] * __shfl(w, min(i + v * kPer + sub, 63));
      }
    }
  };
  add(a.pre, je.pre, max(pre_rows, 1), pre_start, ((b - je.first) * a.tokens + t) * G + h % G, deals[1]);
  add(a.own, je.own, own_rows, own_start, t * G + h % G, deals[0]);
#pragma unroll
  for (int d = kLanes; d < 64; d <<= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] += __shfl_xor(y[i], d);
  const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
  y *= inv;
  uint16_t* out = reinterpret_cast<uint16_t*>(a.o.data) + ((int64_t)b * a.tokens + t) * a.o.row_stride + (int64_t)h * a.o.head_stride;
  if (Store::join_again(a, b, t, h, kvh, y, out)) return;
  if (sub == 0 && dim < D) *reinterpret_cast<u32x2*>(out + dim) = u32x2{Store::E::pack(y[0], y[1]), Store::E::pack(y[2], y[3])};
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
inline int check_attention(int dtype, int heads, int kv_heads, int dim, float scale) {
  if (dtype != MTC_DTYPE_BF16 && dtype != MTC_DTYPE_F16) return host::fail(MTC_E_DTYPE, "attention takes bf16 or f16, got dtype %d", dtype);
  if (heads < 1 || kv_heads < 1 || heads % kv_heads)
    return host::fail(MTC_E_SHAPE, "%d query heads over %d K/V heads", heads, kv_heads);
  if (dim < 8 || dim > MTC_ATTN_MAX_DIM || dim % 8)
    return host::fail(MTC_E_SHAPE, "head size %d: a multiple of 8 from 8 to %d", dim, MTC_ATTN_MAX_DIM);
  if (!(scale > 0.0f) || !std::isfinite(scale)) return host::fail(MTC_E_SHAPE, "scale must be positive and finite");
  return MTC_OK;
}

// How an item's rows are taken: the least of 16, 32 and 128 rows that holds them.
inline int mode_for(int64_t rows) { return rows <= 16 ? kOneTile : rows <= 32 ? kTwoTiles : kRows; }

struct CachedPlan {
  int own_mode, pre_mode;
  int own_stride, pre_stride;        // rows of a slot
  int64_t own_slots, pre_slots;
  size_t own_bytes, pre_bytes, join_bytes;
  size_t bytes() const { return own_bytes + pre_bytes + join_bytes; }
};

inline size_t round_up(size_t x, size_t to) { return (x + to - 1) / to * to; }

inline int plan_cached(const mtc_cache_desc* c, const mtc_cached_args* a, CachedPlan* p) {
  if (!a) return host::fail(MTC_E_NULL, "args is NULL");
  if (int rc = mtc_check_cache_desc(c)) return rc;
  if (a->abi_version != MTC_ABI_VERSION) return host::fail(MTC_E_VERSION, "args of ABI %u, library %d", a->abi_version, MTC_ABI_VERSION);
  if (int rc = check_attention(codes::base_type(*c), a->heads, c->kv_heads, c->dim, a->scale)) return rc;
  if (a->reserved != 0) return host::fail(MTC_E_SHAPE, "reserved must be 0");
  if (a->layer < 0 || a->layer >= c->n_layers) return host::fail(MTC_E_SHAPE, "layer %d of %d", a->layer, c->n_layers);
  if (a->n_seqs < 0 || a->n_seqs > MTC_CACHED_MAX_SEQS) return host::fail(MTC_E_SHAPE, "%d sequences, at most %d", a->n_seqs, MTC_CACHED_MAX_SEQS);
  if (!a->seqs && a->n_seqs > c->max_seqs) return host::fail(MTC_E_SHAPE, "%d sequences, the cache holds %d", a->n_seqs, c->max_seqs);
  if (a->tokens < 1 || a->tokens > MTC_CACHED_MAX_TOKENS)
    return host::fail(MTC_E_SHAPE, "%d tokens per sequence: 1 to %d", a->tokens, MTC_CACHED_MAX_TOKENS);
  if (a->n_groups < 0 || a->n_groups > a->n_seqs) return host::fail(MTC_E_SHAPE, "%d groups of %d sequences", a->n_groups, a->n_seqs);
  if ((int64_t)a->tokens * a->heads > 0xFFFF || (int64_t)a->tokens * a->heads * a->n_seqs > 0x3FFFFFF)   // 2^32 threads a launch
    return host::fail(MTC_E_SHAPE, "%d sequences of %d tokens of %d heads: too many query rows", a->n_seqs, a->tokens, a->heads);
  const int64_t per = (int64_t)a->tokens * (a->heads / c->kv_heads), all = per * a->n_seqs;
  p->own_mode = mode_for(per);
  // groups are on the device: the rows of an average one decide
  p->pre_mode = a->n_groups ? mode_for(std::max<int64_t>(all / a->n_groups, 17)) : kNone;
  auto runs = [](int mode) { return kCachedBlocks * (mode == kRows ? 1 : kCachedWaves); };
  auto tiles = [](int64_t rows, int mode) { return (rows + mode_rows(mode) - 1) / mode_rows(mode); };
  auto stride = [](int64_t rows, int mode) { return (int)std::min<int64_t>((rows + 15) / 16 * 16, mode_rows(mode)); };
  p->own_stride = stride(per, p->own_mode);
  p->own_slots = runs(p->own_mode) + (int64_t)a->n_seqs * c->kv_heads * tiles(per, p->own_mode);
  p->pre_stride = p->pre_mode ? stride(all, p->pre_mode) : 0;
  p->pre_slots = p->pre_mode ? runs(p->pre_mode) + (int64_t)c->kv_heads * (tiles(all, p->pre_mode) + a->n_groups) : 0;
  // the kernels count units in 32 bits
  const int64_t units = (int64_t)c->max_pages * c->page_size / kLeastKeys + 1 + most_start(codes::is_codes(*c));
  if (units * (p->own_slots + p->pre_slots) > 0x7FFFFFFF)
    return host::fail(MTC_E_SHAPE, "%d sequences of up to %d pages of %d tokens, %d row tiles: too much for one call", a->n_seqs, c->max_pages,
                c->page_size, (int)tiles(per, p->own_mode));
  p->own_bytes = round_up((size_t)p->own_slots * p->own_stride * (c->dim + 2) * 4, 256);
  p->pre_bytes = round_up((size_t)p->pre_slots * p->pre_stride * (c->dim + 2) * 4, 256);
  p->join_bytes = round_up(4 * kJoinHead + sizeof(JoinEntry) * (size_t)a->n_seqs + sizeof(JoinPart) * (size_t)a->n_groups, 256);
  return MTC_OK;
}

template <class Store, int DP, int OWN>
void launch_cached(const typename Store::Call& a, int pre, hipStream_t st) {
  if (pre == kNone) k_cached<Store, DP, OWN, kNone><<<kCachedBlocks, kCachedThreads, 0, st>>>(a);
  else if (pre == kTwoTiles) k_cached<Store, DP, OWN, kTwoTiles><<<kCachedBlocks, kCachedThreads, 0, st>>>(a);
  else k_cached<Store, DP, OWN, kRows><<<kCachedBlocks, kCachedThreads, 0, st>>>(a);
}
template <class Store, int DP>
void launch_cached(const typename Store::Call& a, int own, int pre, hipStream_t st) {
  if (own == kOneTile) launch_cached<Store, DP, kOneTile>(a, pre, st);
  else if (own == kTwoTiles) launch_cached<Store, DP, kTwoTiles>(a, pre, st);
  else launch_cached<Store, DP, kRows>(a, pre, st);
}

template <class Store>
int run_cached(const typename Store::Call& a, const CachedPlan& p, hipStream_t st) {
  if (a.dim <= 64) launch_cached<Store, 64>(a, p.own_mode, p.pre_mode, st);
  else launch_cached<Store, 128>(a, p.own_mode, p.pre_mode, st);
  if (int rc = host::check_launch("k_cached")) return rc;
  const dim3 grid(a.n_seqs, (a.tokens * a.heads + kCachedWaves - 1) / kCachedWaves);
  if (a.dim <= 64) k_join<Store, 64><<<grid, kCachedThreads, 0, st>>>(a, mode_rows(p.own_mode), mode_rows(p.pre_mode));
  else k_join<Store, 128><<<grid, kCachedThreads, 0, st>>>(a, mode_rows(p.own_mode), mode_rows(p.pre_mode));
  return host::check_launch("k_join");
}

}  // namespace attn
}  // namespace mtc
