// gfx950 attention kernels and their C-ABI (include/mtc_serve.h).
//
//   k_prompt  : whole prompts, packed sequences, causal or not
//   k_cached  : the newest tokens of each sequence over a paged cache (mtc_cached.h), here of 16-bit numbers; work split evenly over the blocks
//   k_join    : joins k_cached's partial results per row
//
// Both multiply keys by queries with the keys as rows: S^T = K Q^T puts one query into each lane's
// column, so a softmax row lives in one lane (plus its partners in the other lane groups), and the
// same registers, rounded to 16 bits, are the right operand of O^T = V^T P^T without a shuffle: the
// matrix instruction's reduction index may be numbered freely as long as both operands agree, and
// V^T is read from LDS in that numbering by the transposing read.

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>

#include "mtc_attn8.h"
#include "mtc_cached.h"
#include "mtc_host.h"
#include "mtc_serve.h"

#define MTC_API extern "C" __attribute__((visibility("default")))

using mtc::host::check_launch;
using mtc::host::fail;
using mtc::host::ok;
using namespace mtc::attn;

namespace {

// ---------------------------------------------------------------------------
// whole prompts
// ---------------------------------------------------------------------------
constexpr int kPromptWaves = 4;                   // 32 query rows each
constexpr int kPromptRows = 32 * kPromptWaves;

struct PromptTile {
  int tile;          // query tile of its sequence, -1: none
  int q0, n, k0, m;  // the sequence's rows of q and k
};

__device__ __forceinline__ void prompt_range(const int32_t* cu, int b, int rows, int& at, int& n) {
  at = min(max(cu[b], 0), rows);
  n = min(max(cu[b + 1], at), rows) - at;
}

// The rank-th query tile of the call, the tiles with the largest place in their sequence first (with a
// causal mask these see most keys; started last they would run alone at the end). Every lane gets it. The ranges of the first
// 64 sequences stay in the lanes, one each: one round of loads for calls of up to 64.
__device__ PromptTile prompt_tile(const mtc_prompt_args& a, int rank) {
  const int lane = threadIdx.x & 63;
  auto tiles = [](int n) { return (n + kPromptRows - 1) / kPromptRows; };
  auto range = [&](int b, int& q0, int& n) { prompt_range(a.cu_q, b, a.q_rows, q0, n); };
  int q0 = 0, n0 = 0, k0 = 0, m0 = 0;               // of sequence `lane`
  if (lane < a.n_seqs) {
    range(lane, q0, n0);
    prompt_range(a.cu_k, lane, a.k_rows, k0, m0);
  }
  const int t0 = tiles(n0);
  auto count = [&](int level) {                     // tiles at `level` or above
    int s = max(0, t0 - level);
    for (int b = lane + 64; b < a.n_seqs; b += 64) {
      int at, n;
      range(b, at, n);
      s += max(0, tiles(n) - level);
    }
    return __builtin_amdgcn_readlane(wave_scan(s), 63);
  };
  PromptTile r;
  r.tile = -1;
  r.q0 = r.n = r.k0 = r.m = 0;
  int seq = 0;
  if (a.n_seqs == 1) {
    const int t = __builtin_amdgcn_readfirstlane(t0);
    if (rank >= t) return r;
    r.tile = t - 1 - rank;
  } else {
    if (rank >= count(0)) return r;
    int lo = 0, hi = (a.q_rows + kPromptRows - 1) / kPromptRows;     // count(lo) > rank >= count(hi)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (count(mid) > rank) lo = mid; else hi = mid;
    }
    int left = rank - count(hi);                    // the left-th sequence with more than lo tiles
    for (int b0 = 0; b0 < a.n_seqs; b0 += 64) {
      int t = t0;
      if (b0) {
        int at, n = 0;
        if (b0 + lane < a.n_seqs) range(b0 + lane, at, n);
        t = tiles(n);
      }
      const uint64_t mask = __ballot(t > lo);
      const int c = __popcll(mask);
      if (left < c) {
        const uint64_t hit = __ballot(t > lo && __popcll(mask & ((1ull << lane) - 1)) == left);
        seq = b0 + __ffsll((unsigned long long)hit) - 1;
        break;
      }
      left -= c;
    }
    r.tile = lo;
  }
  seq = __builtin_amdgcn_readfirstlane(seq);
  if (seq < 64) {
    r.q0 = __builtin_amdgcn_readlane(q0, seq);
    r.n = __builtin_amdgcn_readlane(n0, seq);
    r.k0 = __builtin_amdgcn_readlane(k0, seq);
    r.m = __builtin_amdgcn_readlane(m0, seq);
  } else {
    range(seq, r.q0, r.n);
    prompt_range(a.cu_k, seq, a.k_rows, r.k0, r.m);
  }
  return r;
}

// One block per tile of 128 queries and head: softmax in one pass over the keys (running maximum m and sum l; o and l are
// scaled by 2^(m - m') when m moves to m'), 64 keys a step, K and V copied to LDS a step ahead of their use. 128 queries in
// four waves let two blocks share a CU, whose barriers then do not stop each other: four waves of 32 queries read 16
// KiB of each tile per 32 matrix instructions, which LDS supplies while they run.
// Bound by the matrix and vector units: of a wave's 3100 cycles a step with 128 dims (two waves a SIMD), 975 are matrix
// instructions, 815 vector issue, 760 waits for LDS and barriers. 1 x 16384, 32/8 heads of 128, causal: 1951 to 2012 us,
// 1.09 to 1.13 PFLOP/s, the clock at 1.75 GHz under the load (an 8192^3 library product: 1.22 PFLOP/s). Calls of few blocks wait for
// the longest (512 new queries on 4608 keys: 72 steps of 1.6 us, 117 to 124 us). Not kept: two waves per 32 queries with half the
// keys each (129 us), two sets of four waves on alternate tiles (130 us).
//
// PARTS: for calls of few tiles (a short chunk of new tokens on many older ones), `parts.n` blocks share a tile, each with a run
// of its steps, and k_prompt_join joins their partial results (5 to 7 us). A call, unsplit and split: 117 queries on 5175 keys,
// 14/2 heads of 40: 83.6 -> 18.6 us; 100 on 2000, 32/8 of 128: 62.1 -> 25.2; 400 on 16000, 8/1 of 128: 454 -> 51.0; 1 on 600,
// 32/8 of 128: 22.6 -> 12.1; 300 on 600, 14/2 of 64, the least gain: 14.1 -> 13.3.
struct PromptParts {
  float* o;                // [part][row of q][head][dim]
  float* ml;               // [part][row of q][head][2]: maximum (times c), sum (0: no keys, o is not written)
  int32_t n;
};
template <bool BF, int DP, bool PARTS>
__global__ __launch_bounds__(64 * kPromptWaves, 2) void k_prompt(const mtc_prompt_args a, const PromptParts parts) {
  using E = Elem<BF>;
  constexpr int kRow = DP * 2;                             // bytes of an LDS row
  constexpr int kTile = kPromptKeys * kRow;
  constexpr int kCopies = kTile / 1024 / kPromptWaves;     // 1 KiB copies per wave and tile
  constexpr int kCopyRows = 1024 / kRow;
  __shared__ __attribute__((aligned(1024))) char lds[4 * kTile];   // K, V; two buffers each

  const int H = a.heads, KV = a.kv_heads, D = a.dim;
  // heads of one K/V head apart by KV places: blocks that share keys share an XCD (and its L2) when the
  // count of K/V heads is a multiple or a divisor of 8
  const int j = blockIdx.x % H;
  const int kvh = j % KV, head = kvh * (H / KV) + j / KV;
  const int rank_part = blockIdx.x / H, part = PARTS ? rank_part % parts.n : 0;
  PromptTile pt = prompt_tile(a, PARTS ? rank_part / parts.n : rank_part);
  pt.tile = __builtin_amdgcn_readfirstlane(pt.tile);      // the same in every lane: scalars from here on
  pt.q0 = __builtin_amdgcn_readfirstlane(pt.q0);
  pt.n = __builtin_amdgcn_readfirstlane(pt.n);
  pt.k0 = __builtin_amdgcn_readfirstlane(pt.k0);
  pt.m = __builtin_amdgcn_readfirstlane(pt.m);
  if (pt.tile < 0) return;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, col = lane & 31;
  const int row = pt.tile * kPromptRows + wave * 32 + col;         // this lane's query
  const int shift = pt.m - pt.n + 1;
  auto sees = [&](int r) { return a.causal ? min(max(r + shift, 0), pt.m) : pt.m; };
  const int seen = row < pt.n ? sees(row) : 0;
  const int last_row = min(pt.tile * kPromptRows + kPromptRows, pt.n) - 1;
  const int wave_last = min(pt.tile * kPromptRows + wave * 32 + 31, pt.n - 1);
  const int wave_first = pt.tile * kPromptRows + wave * 32;
  const int wave_keys = wave_first < pt.n ? sees(wave_last) : 0;   // keys that any row of the wave sees
  const int all_keys = wave_first + 31 < pt.n ? sees(wave_first) : 0;   // keys that all its rows see
  const int all_steps = (sees(last_row) + kPromptKeys - 1) / kPromptKeys;
  const int step0 = PARTS ? all_steps * part / parts.n : 0;          // this block's tiles of keys: step0 ..
  const int steps = (PARTS ? all_steps * (part + 1) / parts.n : all_steps) - step0;

  const uint16_t* qp = reinterpret_cast<const uint16_t*>(a.q.data) + (int64_t)(pt.q0 + row) * a.q.row_stride +
                       (int64_t)head * a.q.head_stride;
  RowTile<BF, DP> rt;
  rt.start(qp, row < pt.n, D, lds);

  const uint32_t k_bytes = (uint32_t)(a.k.row_stride * 2), v_bytes = (uint32_t)(a.v.row_stride * 2);
  const uint64_t k_base = (uint64_t)(uintptr_t)a.k.data + 2 * ((int64_t)pt.k0 * a.k.row_stride + (int64_t)kvh * a.k.head_stride);
  const uint64_t v_base = (uint64_t)(uintptr_t)a.v.data + 2 * ((int64_t)pt.k0 * a.v.row_stride + (int64_t)kvh * a.v.head_stride);
  uint32_t k_off[kCopies], v_off[kCopies];
#pragma unroll
  for (int i = 0; i < kCopies; ++i) {
    const uint32_t r = (wave * kCopies + i) * kCopyRows + lane / (kRow / 16), place = lane % (kRow / 16);
    const uint32_t kc = place ^ k_key<DP>(r), vc = place ^ v_key<DP>(r);
    k_off[i] = (int)kc * 8 < D ? r * k_bytes + kc * 16 : kOutOfRange;
    v_off[i] = (int)vc * 8 < D ? r * v_bytes + vc * 16 : kOutOfRange;
  }
  const uint32_t lds0 = lds_addr(lds);
  auto copy = [&](uint64_t base, uint32_t bytes, const uint32_t* off, int t, uint32_t place) {
    const int at = (step0 + t) * kPromptKeys;
    const uint32_t rows = (uint32_t)min(kPromptKeys, pt.m - at);
    const u32x4 r = buffer_rsrc(base + (uint64_t)at * bytes, (rows - 1) * bytes + D * 2);
    const uint32_t dst = lds0 + place * kTile + wave * kCopies * 1024;
#pragma unroll
    for (int i = 0; i < kCopies; ++i) copy16(r, off[i], __builtin_amdgcn_readfirstlane(dst + i * 1024));
  };
  // places: keys of even and odd tiles, values of even and odd tiles
  auto copy_keys = [&](int t) { copy(k_base, k_bytes, k_off, t, t & 1); };
  auto copy_values = [&](int t) { copy(v_base, v_bytes, v_off, t, 2 + (t & 1)); };

  const float c = a.scale * kLog2e;
  rt.run(
      steps, min(max((wave_keys + kPromptKeys - 1) / kPromptKeys - step0, 0), steps), min(max(all_keys / kPromptKeys - step0, 0), steps), c,
      [&]() {
        copy_keys(0);
        copy_values(0);
        if (steps > 1) copy_keys(1);
        if (steps > 1) wait_copies<2 * kCopies>(); else wait_copies<kCopies>();
        lds_barrier();
      },
      [&](int t) {
        wait_copies<0>();
        lds_barrier();                               // and nobody reads tile t's keys or tile t - 1's values any more
        if (t + 1 < steps) copy_values(t + 1);
        if (t + 2 < steps) copy_keys(t + 2);
      },
      [&](int t) { return seen - (step0 + t) * kPromptKeys; });

  const float sum = half_sum(rt.sum);
  if constexpr (PARTS) {
    if (row >= pt.n) return;
    const int64_t at = ((int64_t)part * a.q_rows + pt.q0 + row) * H + head;
    if (half == 0) *reinterpret_cast<float2*>(parts.ml + at * 2) = make_float2(rt.top, sum);
    if (sum == 0.0f) return;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int dim = d * 32 + 2 * e + 4 * half;
        if (dim < D) *reinterpret_cast<f32x4*>(parts.o + at * D + dim) = f32x4{rt.o[d][e], rt.o[d][e + 1], rt.o[d][e + 2], rt.o[d][e + 3]};
      }
    return;
  }
  const float inv = sum > 0.0f ? 1.0f / sum : sum == 0.0f ? 0.0f : sum;
  bool fine = true;
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      rt.o[d][e] *= inv;
      fine = fine && finite(rt.o[d][e]);
    }
  // rows to compute again: their q is still needed, and o may be q
  uint64_t again = __ballot(row < pt.n && !fine);
  again = (again | (again >> 32)) & 0xFFFFFFFFull;
  const int read = min((wave_keys + kPromptKeys - 1) / kPromptKeys * kPromptKeys, pt.m);    // keys that the wave multiplied
  for (uint64_t ask = again; ask; ask &= ask - 1) {
    const int i = __ffsll((unsigned long long)ask) - 1;
    bool clean = true;                             // nothing unseen can have got in: the row's own keys made it so
    for (int key = sees(wave_first + i); key < read; ++key) {
      const uint16_t* v = reinterpret_cast<const uint16_t*>((uintptr_t)v_base) + (int64_t)key * a.v.row_stride;
      clean = clean && !(lane < D && !finite16<BF>(v[lane])) && !(lane + 64 < D && !finite16<BF>(v[lane + 64]));
    }
    if (!__ballot(!clean)) again &= ~(1ull << i);
  }
  uint16_t* op = reinterpret_cast<uint16_t*>(a.o.data) + (int64_t)(pt.q0 + row) * a.o.row_stride +
                 (int64_t)head * a.o.head_stride;
  const bool store = row < pt.n && !(again >> col & 1);
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int e = 0; e < 16; e += 8) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = E::pack(rt.o[d][e + 2 * i], rt.o[d][e + 2 * i + 1]);
      // the halves hold dims 4 half + 0..3 of 8-dim groups e/4 and e/4 + 1: after the swap each has one group whole
      const auto x = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false), y = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
      const int at = d * 32 + 2 * e + 8 * half;
      if (store && at < D) *reinterpret_cast<u32x4*>(op + at) = u32x4{x[0], y[0], x[1], y[1]};
    }
  for (; again; again &= again - 1) {
    const int r = wave_first + __ffsll((unsigned long long)again) - 1;
    float o0, o1;
    plain_row<BF>(reinterpret_cast<const uint16_t*>(a.q.data) + (int64_t)(pt.q0 + r) * a.q.row_stride + (int64_t)head * a.q.head_stride,
                  D, sees(r), c,
                  [&](int key, const uint16_t*& k, const uint16_t*& v) {
                    k = reinterpret_cast<const uint16_t*>((uintptr_t)k_base) + (int64_t)key * a.k.row_stride;
                    v = reinterpret_cast<const uint16_t*>((uintptr_t)v_base) + (int64_t)key * a.v.row_stride;
                  },
                  o0, o1);
    uint16_t* out = reinterpret_cast<uint16_t*>(a.o.data) + (int64_t)(pt.q0 + r) * a.o.row_stride + (int64_t)head * a.o.head_stride;
    if (lane < D) out[lane] = E::round(o0);
    if (lane + 64 < D) out[lane + 64] = E::round(o1);
  }
}

// Joins the parts of a call: a row is DP / 4 lanes, four dims each, so a wave joins two or four rows at once, with four parts'
// loads under way. A lane also holds its part's maximum and sum (kMostParts <= DP / 4).
constexpr int kMostParts = 16;
template <int DP>
constexpr int kJoinRows = kPromptWaves * 256 / DP;              // of a block
template <bool BF, int DP>
__global__ __launch_bounds__(64 * kPromptWaves) void k_prompt_join(const mtc_prompt_args a, const PromptParts parts) {
  constexpr int kLanes = DP / 4, kChunks = kPromptRows / kJoinRows<DP>;
  const int H = a.heads, D = a.dim, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int head = blockIdx.x % H, kvh = head / (H / a.kv_heads);
  PromptTile pt = prompt_tile(a, blockIdx.x / H / kChunks);
  pt.tile = __builtin_amdgcn_readfirstlane(pt.tile);
  pt.q0 = __builtin_amdgcn_readfirstlane(pt.q0);
  pt.n = __builtin_amdgcn_readfirstlane(pt.n);
  pt.k0 = __builtin_amdgcn_readfirstlane(pt.k0);
  pt.m = __builtin_amdgcn_readfirstlane(pt.m);
  if (pt.tile < 0) return;
  const int row0 = pt.tile * kPromptRows + blockIdx.x / H % kChunks * kJoinRows<DP> + wave * (64 / kLanes);
  if (row0 >= pt.n) return;
  const int in = lane % kLanes, row = row0 + lane / kLanes;
  const int64_t at = (int64_t)(pt.q0 + min(row, pt.n - 1)) * H + head;
  const int64_t step = (int64_t)a.q_rows * H;                  // from a part to the next
  float2 ml = make_float2(-INFINITY, 0.0f);
  if (in < parts.n) ml = *reinterpret_cast<const float2*>(parts.ml + (at + in * step) * 2);
  const bool has = ml.y != 0.0f;                               // a NaN too
  float top = has ? ml.x : -INFINITY;
#pragma unroll
  for (int x = 1; x < kMostParts; x *= 2) top = fmaxf(top, __shfl_xor(top, x));
  top = __shfl(top, lane - in);
  const float w = has ? exp2_fast(ml.x - (top == -INFINITY ? 0.0f : top)) : 0.0f;
  float l = has ? ml.y * w : 0.0f;
#pragma unroll
  for (int x = 1; x < kMostParts; x *= 2) l += __shfl_xor(l, x);
  l = __shfl(l, lane - in);
  const uint64_t with = __ballot(has);
  float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  const bool mine = 4 * in < D;
  for (int p = 0; p < parts.n; p += 4) {
    f32x4 z[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {                              // a part without keys wrote nothing: not looked at
      z[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (mine && (with >> (lane - in + p + j) & 1))
        z[j] = *reinterpret_cast<const f32x4*>(parts.o + (at + (p + j) * step) * D + 4 * in);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float wp = __shfl(w, lane - in + p + j);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = __builtin_fmaf(z[j][e], wp, y[e]);
    }
  }
  const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] *= inv;
  uint16_t* op = reinterpret_cast<uint16_t*>(a.o.data) + (int64_t)pt.q0 * a.o.row_stride + (int64_t)head * a.o.head_stride;
  // as in k_prompt: not of the row's own making if a key that it does not see, in the tiles taken for its wave, holds one
  const uint64_t bad = __ballot(row < pt.n && !(finite(y[0]) && finite(y[1]) && finite(y[2]) && finite(y[3])));
  uint32_t again = 0;                              // bit i: row row0 + i is computed again (before it is stored: o may be q)
  const float c = a.scale * kLog2e;
  const int64_t hk = (int64_t)kvh * a.k.head_stride, hv = (int64_t)kvh * a.v.head_stride;
  const uint16_t* kb = reinterpret_cast<const uint16_t*>(a.k.data) + (int64_t)pt.k0 * a.k.row_stride + hk;
  const uint16_t* vb = reinterpret_cast<const uint16_t*>(a.v.data) + (int64_t)pt.k0 * a.v.row_stride + hv;
  for (int i = 0; bad && i < 64 / kLanes; ++i) {
    if (!(bad >> (i * kLanes) & ((1ull << kLanes) - 1))) continue;
    const int r = row0 + i, seen = a.causal ? min(max(r + pt.m - pt.n + 1, 0), pt.m) : pt.m;
    bool clean = true;
    for (int key = seen; key < min(seen + kPromptKeys + 32, pt.m); ++key) {      // the wave's last row saw up to 31 more
      const uint16_t* v = vb + (int64_t)key * a.v.row_stride;
      clean = clean && !(lane < D && !finite16<BF>(v[lane])) && !(lane + 64 < D && !finite16<BF>(v[lane + 64]));
    }
    if (!__ballot(!clean)) continue;
    again |= 1u << i;
    float o0, o1;
    plain_row<BF>(reinterpret_cast<const uint16_t*>(a.q.data) + (int64_t)(pt.q0 + r) * a.q.row_stride + (int64_t)head * a.q.head_stride,
                  D, seen, c,
                  [&](int key, const uint16_t*& k, const uint16_t*& v) {
                    k = kb + (int64_t)key * a.k.row_stride;
                    v = vb + (int64_t)key * a.v.row_stride;
                  },
                  o0, o1);
    uint16_t* out = op + (int64_t)r * a.o.row_stride;
    if (lane < D) out[lane] = Elem<BF>::round(o0);
    if (lane + 64 < D) out[lane + 64] = Elem<BF>::round(o1);
  }
  if (mine && row < pt.n && !(again >> (lane / kLanes) & 1)) {
    u32x2 packed = {Elem<BF>::pack(y[0], y[1]), Elem<BF>::pack(y[2], y[3])};
    *reinterpret_cast<u32x2*>(op + (int64_t)row * a.o.row_stride + 4 * in) = packed;
  }
}

constexpr int kWaveKeys = 32;                     // split keys: per wave and step

// Buffer over up to 16 rows (of one page) of K or V from token p on, cut at token `to`; no rows if the page id is bad.
__device__ __forceinline__ u32x4 page_rows(const CachedCall& a, int id, int64_t off, int p, int to) {
  const int rows = min(to - p, 16);
  const bool good = rows > 0 && (uint32_t)id < (uint32_t)a.n_pages;
  const int64_t at = (int64_t)(good ? id : 0) * a.page_elems + off + (int64_t)(p & ((1 << a.page_log) - 1)) * a.dim;
  return buffer_rsrc((uint64_t)(uintptr_t)(a.pool + at), good ? (uint32_t)(rows * a.dim * 2) : 0u);
}

// One item's keys [from, to) (from a multiple of 16) into a partial result, by the block (the keys split over its waves)
// or by this wave alone.
template <bool BF, int DP, int MT, bool PREFIX>
__device__ void split_keys(const CachedCall& a, const Book& book, char* lds, const Entry& x, int item, int from, int to, int slot, bool alone) {
  using E = Elem<BF>;
  constexpr int kRow = DP * 2;
  constexpr int kHalf = 16 * kRow;                       // 16 keys, always of one page
  constexpr int kHalfCopies = kHalf / 1024, kCopyRows = 1024 / kRow;
  constexpr int kTileCopies = 2 * kHalfCopies;
  constexpr int kSteps = DP / 32;
  const int stride = alone ? kWaveKeys : kCachedWaves * kWaveKeys;
  const Pass& ps = PREFIX ? a.pre : a.own;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, w = lane >> 4;
  const int D = a.dim;
  const int kvh = item / x.tiles, row0 = (item % x.tiles) * 16 * MT;
  const int rows = min(x.rows - row0, 16 * MT);

  PageWindow pages{a.table + (int64_t)x.seq.row * a.max_pages, 0, -1, a.max_pages};
  int pos = alone ? from : from + kWaveKeys * wave;
  if (pos < to) pages.load(pos >> a.page_log);

  // this lane's query rows: 16 rt + n
  u32x4 qf[MT][kSteps];
  int seen[MT], all = 0x7FFFFFFF;                        // keys that a row sees, that all rows see
#pragma unroll
  for (int rt = 0; rt < MT; ++rt) {
    const int rr = row0 + rt * 16 + n;
    const uint16_t* qp = cached_query<PREFIX>(a, book, x, kvh, rr, seen[rt]);
    if (rr < x.rows) all = min(all, seen[rt]);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int d = 32 * s + 8 * w;
      qf[rt][s] = rr < x.rows && d < D ? *reinterpret_cast<const u32x4*>(qp + d) : u32x4{0, 0, 0, 0};
    }
  }
#pragma unroll
  for (int d = 8; d; d >>= 1) all = min(all, __shfl_xor(all, d));
  all = __builtin_amdgcn_readfirstlane(all);

  uint32_t k_lane[kHalfCopies], v_lane[kHalfCopies];     // byte offsets within 16 rows
#pragma unroll
  for (int i = 0; i < kHalfCopies; ++i) {
    const uint32_t r = i * kCopyRows + lane / (kRow / 16), place = lane % (kRow / 16);
    const uint32_t kc = place ^ k_key<DP>(r), vc = place ^ v_key<DP>(r);
    k_lane[i] = (int)kc * 8 < D ? r * D * 2 + kc * 16 : kOutOfRange;
    v_lane[i] = (int)vc * 8 < D ? r * D * 2 + vc * 16 : kOutOfRange;
  }
  char* const kt = lds + wave * 4 * kHalf;
  char* const vt = kt + 2 * kHalf;
  const uint32_t k_lds = __builtin_amdgcn_readfirstlane(lds_addr(kt)), v_lds = k_lds + 2 * kHalf;
  const int64_t head_off = ((int64_t)kvh << a.page_log) * D;
  auto copy_keys = [&](int at, int64_t off, uint32_t dst, const uint32_t* lanes) {
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int p = at + 16 * hf;
      const u32x4 r = page_rows(a, pages(p >> a.page_log), off + head_off, p, to);
#pragma unroll
      for (int i = 0; i < kHalfCopies; ++i)
        copy16(r, lanes[i], __builtin_amdgcn_readfirstlane(dst + hf * kHalf + i * 1024));
    }
  };

  f32x4 o[MT][DP / 16];
  float top[MT], sum[MT];
#pragma unroll
  for (int rt = 0; rt < MT; ++rt) {
    top[rt] = -INFINITY;
    sum[rt] = 0.0f;
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) o[rt][d] = f32x4{};
  }
  if (pos < to) {
    copy_keys(pos, a.k_off, k_lds, k_lane);
    copy_keys(pos, a.v_off, v_lds, v_lane);
  }
  while (pos < to) {
    const int next = pos + stride;
    const bool more = next < to;
    wait_copies<kTileCopies>();                          // K is there
    f32x4 s[MT][2];
#pragma unroll
    for (int rt = 0; rt < MT; ++rt) s[rt][0] = s[rt][1] = f32x4{};
#pragma unroll
    for (int st = 0; st < kSteps; ++st)
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const u32x4 kf = read_k<DP>(kt, g * 16 + n, 4 * st + w);
#pragma unroll
        for (int rt = 0; rt < MT; ++rt) s[rt][g] = E::mfma16(kf, qf[rt][st], s[rt][g]);
      }
    wait_lds();
    if (more) {
      if (((next + kWaveKeys - 1) >> a.page_log) - pages.at > 63) pages.load(next >> a.page_log);
      copy_keys(next, a.k_off, k_lds, k_lane);
    }
    // element i of s[rt][g]: key pos + 16 g + 4 w + i, query row 16 rt + n
    u32x4 p[MT];
#pragma unroll
    for (int rt = 0; rt < MT; ++rt) {
      const int end = min(seen[rt], to);
      if (pos + kWaveKeys > min(all, to)) {
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (pos + 16 * g + 4 * w + i >= end) s[rt][g][i] = -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[rt][g][i]);
      mx = half_max(fmaxf(mx, __shfl_xor(mx, 16))) * a.c - E::raise(0.0f);
      const float was = top[rt];
      top[rt] = fmaxf(was, mx);
      const float base = top[rt] == -INFINITY ? 0.0f : top[rt];
      const float fade = exp2_fast(was - base);
      sum[rt] *= fade;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) o[rt][d] *= fade;
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          const float y0 = exp2_fast(__builtin_fmaf(s[rt][g][i], a.c, -base));
          const float y1 = exp2_fast(__builtin_fmaf(s[rt][g][i + 1], a.c, -base));
          const uint32_t y = E::pack(y0, y1);            // weights of 16 bits: the matrix core's operand
          sum[rt] = E::add2(y, sum[rt]);                 // and what is summed, so that the quotient's parts agree
          p[rt][2 * g + (i >> 1)] = y;
        }
    }
    if (more) wait_copies<kTileCopies>();                // V is there
    else wait_copies<0>();
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) {
      const u32x2 lo = read_v<DP>(vt, 4 * w, d * 16, n), hi = read_v<DP>(vt, 16 + 4 * w, d * 16, n);
#pragma unroll
      for (int rt = 0; rt < MT; ++rt) o[rt][d] = E::mfma16(u32x4{lo[0], lo[1], hi[0], hi[1]}, p[rt], o[rt][d]);
    }
    wait_lds();
    if (more) copy_keys(next, a.v_off, v_lds, v_lane);
    pos = next;
  }

  store_keys<DP, MT>(ps, lds, slot, alone, rows, D, o, top, sum);
}

// The same with the rows split over the waves, 32 each, and tiles of 64 keys shared by the block.
template <bool BF, int DP, bool PREFIX>
__device__ void split_rows(const CachedCall& a, const Book& book, char* lds, const Entry& x, int item, int from, int to, int slot) {
  constexpr int kRow = DP * 2;
  constexpr int kTile = kPromptKeys * kRow;
  constexpr int kCopies = 16 * kRow / 1024, kCopyRows = 1024 / kRow;      // a wave copies 16 of the 64 keys
  const Pass& ps = PREFIX ? a.pre : a.own;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, col = lane & 31;
  const int D = a.dim;
  const int kvh = item / x.tiles, row0 = (item % x.tiles) * kManyRows + wave * 32;
  const bool busy = row0 < x.rows;                       // the wave has rows

  PageWindow pages{a.table + (int64_t)x.seq.row * a.max_pages, 0, -1, a.max_pages};
  pages.load(from >> a.page_log);
  RowTile<BF, DP> rt;
  int seen;
  const uint16_t* qp = cached_query<PREFIX>(a, book, x, kvh, row0 + col, seen);
  rt.start(qp, row0 + col < x.rows, D, lds);
  seen = min(seen, to);
  int all = row0 + col < x.rows ? seen : 0x7FFFFFFF;
#pragma unroll
  for (int d = 16; d; d >>= 1) all = min(all, __shfl_xor(all, d));
  all = min(__builtin_amdgcn_readfirstlane(all), to);
  all = max(all, from);

  uint32_t k_lane[kCopies], v_lane[kCopies];
#pragma unroll
  for (int i = 0; i < kCopies; ++i) {
    const uint32_t r = i * kCopyRows + lane / (kRow / 16), place = lane % (kRow / 16);
    const uint32_t kc = place ^ k_key<DP>(r), vc = place ^ v_key<DP>(r);      // 16 rows on, the keys are the same
    k_lane[i] = (int)kc * 8 < D ? r * D * 2 + kc * 16 : kOutOfRange;
    v_lane[i] = (int)vc * 8 < D ? r * D * 2 + vc * 16 : kOutOfRange;
  }
  const int64_t head_off = ((int64_t)kvh << a.page_log) * D;
  const uint32_t lds0 = lds_addr(lds) + wave * 16 * kRow;
  auto copy = [&](int64_t off, const uint32_t* lanes, int t, uint32_t place) {
    const int p = from + t * kPromptKeys + wave * 16;
    const u32x4 r = page_rows(a, pages(p >> a.page_log), off + head_off, p, to);
    const uint32_t dst = lds0 + place * kTile;
#pragma unroll
    for (int i = 0; i < kCopies; ++i) copy16(r, lanes[i], __builtin_amdgcn_readfirstlane(dst + i * 1024));
  };
  auto copy_keys = [&](int t) { copy(a.k_off, k_lane, t, t & 1); };
  auto copy_values = [&](int t) { copy(a.v_off, v_lane, t, 2 + (t & 1)); };
  const int steps = (to - from + kPromptKeys - 1) / kPromptKeys;
  rt.run(
      steps, busy ? steps : 0, (all - from) / kPromptKeys, a.c,
      [&]() {
        copy_keys(0);
        copy_values(0);
        if (steps > 1) copy_keys(1);
        if (steps > 1) wait_copies<2 * kCopies>(); else wait_copies<kCopies>();
        lds_barrier();
      },
      [&](int t) {
        wait_copies<0>();
        lds_barrier();
        const int next = from + (t + 1) * kPromptKeys;
        if (((next + 2 * kPromptKeys - 1) >> a.page_log) - pages.at > 63) pages.load(next >> a.page_log);
        if (t + 1 < steps) copy_values(t + 1);
        if (t + 2 < steps) copy_keys(t + 2);
      },
      [&](int t) { return seen - from - t * kPromptKeys; });
  lds_barrier();                                         // the next item may fill the tiles
  const int r = wave * 32 + col;
  const float sum = half_sum(rt.sum);
  if (slot >= 0 && slot < ps.slots && row0 + col < x.rows) store_rows<BF, DP>(ps, slot, r, D, rt, sum);
}

template <bool BF>
struct Store16 {
  static constexpr bool kCodes = false;
  static constexpr int kKeys = kWaveKeys, kStart = 4, kStartAlone = 4, kShort = 8;
  static constexpr float kCostRows = 2.2f, kCostKeys = 0.8f;
  typedef CachedCall Call;
  using E = Elem<BF>;
  template <int DP>
  static constexpr int kKeysBytes = kCachedWaves * 2 * kWaveKeys * DP * 2;      // one tile of keys, one of values a wave
  template <int DP, int MODE, bool PREFIX>
  static __device__ __forceinline__ void keys(const Call& a, const Book& book, char* lds, const Entry& x, int item, int from, int to, int slot,
                                              bool alone) {
    split_keys<BF, DP, MODE, PREFIX>(a, book, lds, x, item, from, to, slot, alone);
  }
  template <int DP, bool PREFIX>
  static __device__ __forceinline__ void rows(const Call& a, const Book& book, char* lds, const Entry& x, int item, int from, int to, int slot) {
    split_rows<BF, DP, PREFIX>(a, book, lds, x, item, from, to, slot);
  }
  // Rows that came out not finite, if keys were read that they do not see.
  static __device__ __forceinline__ bool join_again(const Call& a, int b, int t, int h, int kvh, const f32x4& y, uint16_t* out) {
    const int D = a.dim, lane = threadIdx.x & 63;
    bool again = __ballot(!(finite(y[0]) && finite(y[1]) && finite(y[2]) && finite(y[3])));
    Seq s{0, 0, 0};
    int seen = 0;
    if (again) {                                           // only if keys were read that the row does not see
      s = cached_seq(a, b);
      seen = row_sees(s.len, s.q_len, t);
      const int g = group_of(a.n_groups, b, [&](int i) { return group_start(a, i); });
      again = seen < s.len || (g >= 0 && seen < prefix_tokens(a, g));
    }
    if (again) {
      const int32_t* table = a.table + (int64_t)s.row * a.max_pages;
      float y0, y1;
      plain_row<BF>(reinterpret_cast<const uint16_t*>(a.q.data) + ((int64_t)b * a.tokens + t) * a.q.row_stride + (int64_t)h * a.q.head_stride,
                    D, seen, a.c,
                    [&](int key, const uint16_t*& k, const uint16_t*& v) {
                      const int id = min(max(table[key >> a.page_log], 0), a.n_pages - 1);
                      const uint16_t* p = a.pool + (int64_t)id * a.page_elems +
                                          (((int64_t)kvh << a.page_log) + (key & ((1 << a.page_log) - 1))) * D;
                      k = p + a.k_off;
                      v = p + a.v_off;
                    },
                    y0, y1);
      if (lane < D) out[lane] = Elem<BF>::round(y0);
      if (lane + 64 < D) out[lane + 64] = Elem<BF>::round(y1);
      return true;
    }
    return false;
  }
};

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
int check_heads(const char* what, const mtc_heads& x, bool empty) {
  if (!x.data && !empty) return fail(MTC_E_NULL, "%s is NULL", what);
  if ((uintptr_t)x.data % 16) return fail(MTC_E_SHAPE, "%s must be 16-byte aligned", what);
  if (x.row_stride < 0 || x.head_stride < 0 || x.row_stride % 8 || x.head_stride % 8)
    return fail(MTC_E_SHAPE, "%s: strides %lld, %lld must be non-negative multiples of 8 elements", what,
                (long long)x.row_stride, (long long)x.head_stride);
  // offsets within a tile of 64 rows stay below 2^31 bytes
  if (x.row_stride >= (1ll << 24)) return fail(MTC_E_SHAPE, "%s: row stride %lld is too large", what, (long long)x.row_stride);
  return MTC_OK;
}

// At most so many query tiles (the sequences' lengths are on the device): n rows are (n - 1) / kPromptRows + 1 tiles.
int64_t prompt_tiles(const mtc_prompt_args& a) {
  const int seqs = std::min(a.n_seqs, a.q_rows);
  return (int64_t)(a.q_rows - seqs) / kPromptRows + seqs;
}

// Blocks that share a tile's keys, from the sizes that the host knows (as if one sequence had all the keys): as many as fill the
// chip's 512 places, with two steps or more each, where the steps that a part saves (1.6 us each at 128 dims, 0.8 at 64) are
// worth its partial results (0.7 us a MB, out and back): steps t / n + n MB 0.7 is least at n = sqrt(steps t / (0.7 MB)).
// Below eight steps the join's launch costs more than it saves (1 query on 300 keys: 8.9 -> 9.6 us, 4 x 64: 5.4 -> 8.8).
int prompt_parts(const mtc_prompt_args& a) {
  const int64_t blocks = prompt_tiles(a) * a.heads, steps = a.k_rows / kPromptKeys;
  if (steps < 8 || blocks > 256) return 1;
  const double mb = 1e-6 * a.q_rows * a.heads * (a.dim + 2) * 4;
  const int64_t worth = (int64_t)std::min(std::sqrt((double)steps * (a.dim <= 64 ? 0.8 : 1.6) / (0.7 * mb)), (double)kMostParts);
  return (int)std::max<int64_t>(std::min(std::min(512 / blocks, steps / 2), worth), 1);
}
size_t prompt_workspace(const mtc_prompt_args& a) {
  const int n = prompt_parts(a);
  return n < 2 ? 0 : (size_t)n * a.q_rows * a.heads * (a.dim + 2) * 4 + 16;
}

template <bool BF, int DP>
int launch_prompt(const mtc_prompt_args& a, void* workspace, hipStream_t st) {
  const unsigned blocks = (unsigned)(prompt_tiles(a) * a.heads);
  PromptParts parts{nullptr, nullptr, prompt_parts(a)};
  if (parts.n < 2) {
    k_prompt<BF, DP, false><<<blocks, 64 * kPromptWaves, 0, st>>>(a, parts);
    return check_launch("k_prompt");
  }
  parts.ml = (float*)workspace;                    // an even count of floats: the rows of o stay 16-byte aligned below
  parts.o = parts.ml + (((size_t)parts.n * a.q_rows * a.heads * 2 + 3) & ~(size_t)3);
  k_prompt<BF, DP, true><<<blocks * parts.n, 64 * kPromptWaves, 0, st>>>(a, parts);
  if (int rc = check_launch("k_prompt")) return rc;
  k_prompt_join<BF, DP><<<blocks * (kPromptRows / kJoinRows<DP>), 64 * kPromptWaves, 0, st>>>(a, parts);
  return check_launch("k_prompt_join");
}
template <bool BF>
int launch_prompt(const mtc_prompt_args& a, void* workspace, hipStream_t st) {
  return a.dim <= 64 ? launch_prompt<BF, 64>(a, workspace, st) : launch_prompt<BF, 128>(a, workspace, st);
}

int check_prompt(const mtc_prompt_args* a) {
  if (!a) return fail(MTC_E_NULL, "args is NULL");
  if (a->abi_version != MTC_ABI_VERSION) return fail(MTC_E_VERSION, "args of ABI %u, library %d", a->abi_version, MTC_ABI_VERSION);
  if (int rc = check_attention(a->dtype, a->heads, a->kv_heads, a->dim, a->scale)) return rc;
  if (a->n_seqs < 0 || a->q_rows < 0 || a->k_rows < 0) return fail(MTC_E_SHAPE, "negative sizes");
  if (prompt_tiles(*a) * a->heads > 0xFFFFFF) return fail(MTC_E_SHAPE, "too many query tiles");     // 2^32 threads a launch
  return MTC_OK;
}

}  // namespace

MTC_API size_t mtc_prompt_attention_workspace_bytes(const mtc_prompt_args* a) {
  if (check_prompt(a) != MTC_OK || a->n_seqs == 0 || a->q_rows == 0) return 0;
  return prompt_workspace(*a);
}

MTC_API int mtc_prompt_attention(const mtc_prompt_args* a, void* workspace, size_t workspace_bytes, void* hip_stream) {
  if (int rc = check_prompt(a)) return rc;
  if (a->n_seqs == 0 || a->q_rows == 0) return ok();
  if (!a->cu_q || !a->cu_k) return fail(MTC_E_NULL, "cu_q or cu_k is NULL");
  if (int rc = check_heads("q", a->q, false)) return rc;
  if (int rc = check_heads("k", a->k, a->k_rows == 0)) return rc;
  if (int rc = check_heads("v", a->v, a->k_rows == 0)) return rc;
  if (int rc = check_heads("o", a->o, false)) return rc;
  // a tile's rows past the sequence's end must lie past its buffer's end: rows may not overlap
  if ((a->k.row_stride < a->dim || a->v.row_stride < a->dim) && a->k_rows > 1)
    return fail(MTC_E_SHAPE, "rows of k and v overlap: strides %lld, %lld", (long long)a->k.row_stride, (long long)a->v.row_stride);
  if (const size_t need = prompt_workspace(*a)) {
    if (!workspace || workspace_bytes < need)
      return fail(MTC_E_WORKSPACE, "workspace of %zu bytes, needs %zu", workspace ? workspace_bytes : (size_t)0, need);
    if ((uintptr_t)workspace % 256) return fail(MTC_E_WORKSPACE, "workspace must be 256-byte aligned");
  }
  hipStream_t st = (hipStream_t)hip_stream;
  return a->dtype == MTC_DTYPE_BF16 ? launch_prompt<true>(*a, workspace, st) : launch_prompt<false>(*a, workspace, st);
}

MTC_API size_t mtc_cached_attention_workspace_bytes(const mtc_cache_desc* c, const mtc_cached_args* a) {
  CachedPlan p;
  if (plan_cached(c, a, &p) != MTC_OK) return 0;
  return p.bytes();
}

MTC_API int mtc_cached_attention(const mtc_cache_desc* c, const mtc_cached_args* a, void* workspace, size_t workspace_bytes,
                                 void* hip_stream) {
  CachedPlan p;
  if (int rc = plan_cached(c, a, &p)) return rc;
  if (a->n_seqs == 0) return ok();
  if (int rc = check_heads("q", a->q, false)) return rc;
  if (int rc = check_heads("o", a->o, false)) return rc;
  if (a->n_groups && (!a->groups || !a->prefix_lens)) return fail(MTC_E_NULL, "groups or prefix_lens is NULL");
  if (!workspace || workspace_bytes < p.bytes())
    return fail(MTC_E_WORKSPACE, "workspace of %zu bytes, needs %zu", workspace ? workspace_bytes : (size_t)0, p.bytes());
  if ((uintptr_t)workspace % 256) return fail(MTC_E_WORKSPACE, "workspace must be 256-byte aligned");
  CodesCall k{};
  const bool bf = mtc::codes::base_type(*c) == MTC_DTYPE_BF16;
  const int64_t head = (int64_t)c->page_size * c->dim;
  k.pool = (const uint16_t*)c->pool;
  k.page_elems = 2 * head * c->kv_heads * c->n_layers;
  k.k_off = 2 * head * c->kv_heads * a->layer;
  k.v_off = k.k_off + head * c->kv_heads;
  k.codes = (const char*)c->pool;
  k.page_bytes = mtc::codes::page_bytes(*c);
  k.room = mtc::codes::row_bytes(c->dim);
  k.k_codes = 2ll * a->layer * c->kv_heads * c->page_size * k.room;
  k.v_codes = k.k_codes + (int64_t)c->kv_heads * c->page_size * k.room;
  k.k_scales = mtc::codes::code_bytes(*c) + 4ll * a->layer * c->kv_heads * (c->page_size / mtc::codes::kBlock);
  k.v_scales = k.k_scales + 2ll * c->kv_heads * (c->page_size / mtc::codes::kBlock);
  k.kv_heads = c->kv_heads;
  k.dim = c->dim;
  k.page_log = __builtin_ctz((unsigned)c->page_size);
  k.n_pages = c->n_pages;
  k.max_pages = c->max_pages;
  k.max_seqs = c->max_seqs;
  k.table = c->table;
  k.lens = c->lens;
  k.q = a->q;
  k.o = a->o;
  k.seqs = a->seqs;
  k.q_lens = a->q_lens;
  k.groups = a->groups;
  k.prefix_lens = a->prefix_lens;
  k.n_seqs = a->n_seqs;
  k.tokens = a->tokens;
  k.heads = a->heads;
  k.n_groups = a->n_groups;
  k.c = a->scale * kLog2e;
  auto pass = [&](char* at, int64_t slots, int stride) {
    float* part = (float*)at;
    return Pass{part, part + slots * stride * c->dim, stride, (int32_t)slots};
  };
  k.own = pass((char*)workspace, p.own_slots, p.own_stride);
  k.pre = pass((char*)workspace + p.own_bytes, p.pre_slots, p.pre_stride);
  k.join = (int32_t*)((char*)workspace + p.own_bytes + p.pre_bytes);
  hipStream_t st = (hipStream_t)hip_stream;
  if (mtc::codes::is_codes(*c)) return run_codes(k, bf, p, st);
  return bf ? run_cached<Store16<true>>(k, p, st) : run_cached<Store16<false>>(k, p, st);
}
