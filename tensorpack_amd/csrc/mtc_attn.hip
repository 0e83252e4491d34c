// gfx950 attention kernels and their C-ABI (include/mtc_serve.h).
//
//   k_prompt  : whole prompts, packed sequences, causal or not
//   k_cached  : the newest tokens of each sequence over a paged cache; work split evenly over the blocks
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

#include "mtc_attn.h"
#include "mtc_host.h"
#include "mtc_serve.h"

#define MTC_API extern "C" __attribute__((visibility("default")))

using mtc::host::check_launch;
using mtc::host::fail;
using mtc::host::ok;
using namespace mtc::attn;

namespace {

// Inclusive sum over the wave's lanes (row shifts, then the rows' totals).
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);      // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);     // row_bcast:15 into rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);     // row_bcast:31 into rows 2 and 3
  return x;
}

// ---------------------------------------------------------------------------
// whole prompts
// ---------------------------------------------------------------------------
constexpr int kPromptWaves = 4;                   // 32 query rows each
constexpr int kPromptRows = 32 * kPromptWaves;
constexpr int kPromptKeys = 64;                   // keys per step

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

// 32 query rows of one wave (one per lane of either half) through tiles of 64 keys: S^T in two 32 x 32 blocks, O^T in
// DP / 32. Element e of a block lies at row 8*(e/4) + 4*half + e%4 (key or dim), column `col` (query).
//
// The scores of the next tile are computed beside the weights of this one: the matrix core multiplies while the vector
// unit takes exponentials, within one wave. Tiles go in pairs, so that the places in LDS are constants and the scores'
// registers change roles instead of being copied.
template <bool BF, int DP>
struct RowTile {
  using E = Elem<BF>;
  static constexpr int kSteps = DP / 16, kRow = DP * 2, kTile = kPromptKeys * kRow;
  // The maximum may lag: weights up to 2^kLag keep their relative precision in 16 bits, and the common factor drops out
  // of the quotient. After the first tiles it seldom moves, which saves the pass over o.
  // (f16, which raises its weights by 15 - lag: 512 on 4608 117 us with lags of 0, 2 and 4 at 126, 122 and 120.)
  static constexpr float kLag = 8.0f, kRaise = E::raise(kLag);
  u32x4 qf[kSteps];
  f32x16 o[DP / 32];
  float top, sum;                    // running maximum (times c; up to kLag behind), this lane's share of the sum
  float mx;                          // of the scores whose weights come next, times c
  uint32_t k_at[kSteps], v_at[DP / 32];   // this lane's places in tiles of even turn: keys at lds, values two tiles on

  __device__ __forceinline__ void start(const uint16_t* qp, bool good, int D, const char* lds) {
    const uint32_t lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31, i16 = lane & 15, base = lds_addr(lds);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int d = 16 * i + 8 * half;
      qf[i] = good && d < D ? *reinterpret_cast<const u32x4*>(qp + d) : u32x4{0, 0, 0, 0};
      k_at[i] = base + col * kRow + (((2 * i + half) ^ k_key<DP>(col)) << 4);          // 32 rows on, the key is the same
    }
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) {
      o[d] = f32x16{};
      v_at[d] = base + 2 * kTile + v_place<DP>(4 * half, d * 32 + 16 * ((lane >> 4) & 1), i16);   // 8 rows on, too
    }
    top = -INFINITY;
    sum = 0.0f;
  }

  // Scores of the keys in the place `at` bytes on
  __device__ __forceinline__ void multiply(uint32_t at, f32x16 (&r)[2]) const {
    r[0] = r[1] = f32x16{};
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
      for (int g = 0; g < 2; ++g) r[g] = E::mfma32(lds_read16(k_at[i] + (at + g * 32 * kRow)), qf[i], r[g]);
  }
  // left (MASKED): keys of the tile that this lane's row sees
  template <bool MASKED>
  __device__ __forceinline__ void maximum(f32x16 (&s)[2], float c, int left) {
    if constexpr (MASKED) {
      left -= 4 * ((threadIdx.x >> 5) & 1);
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (g * 32 + 8 * (e >> 2) + (e & 3) >= left) s[g][e] = -INFINITY;
    }
    mx = -INFINITY;
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[g][e]);
    mx = half_max(mx) * c - kRaise;
  }

  // Weights of s times the values `v` bytes on; NEXT: n becomes the scores of the keys `k` bytes on (MASKED, left: as above)
  template <bool NEXT, bool MASKED>
  __device__ __forceinline__ void step(f32x16 (&s)[2], f32x16 (&n)[2], uint32_t v, uint32_t k, float c, int left) {
    if (__ballot(mx > top + kLag)) {
      const float was = top;
      top = fmaxf(top, mx);
      const float fade = top == -INFINITY ? 1.0f : exp2_fast(was - top);
      sum *= fade;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) o[d] *= fade;
    }
    const float base = top == -INFINITY ? 0.0f : top;
    if constexpr (NEXT) multiply(k, n);
    u32x4 p[4];
    float add[2] = {0.0f, 0.0f};
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const float x = exp2_fast(__builtin_fmaf(s[g][e], c, -base));
        const float y = exp2_fast(__builtin_fmaf(s[g][e + 1], c, -base));
        const uint32_t w = E::pack(x, y);          // weights of 16 bits: the matrix core's operand
        add[(e >> 1) & 1] = E::add2(w, add[(e >> 1) & 1]);     // and what is summed, so that the quotient's parts agree
        p[g * 2 + (e >> 3)][(e & 7) >> 1] = w;
      }
    sum += add[0] + add[1];
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) {
        const u32x2 lo = lds_read_transposed(v_at[d] + (v + ks * 16 * kRow));
        const u32x2 hi = lds_read_transposed(v_at[d] + (v + (ks * 16 + 8) * kRow));
        o[d] = E::mfma32(u32x4{lo[0], lo[1], hi[0], hi[1]}, p[ks], o[d]);
      }
    if constexpr (NEXT) {
      maximum<MASKED>(n, c, left);
    }
    if constexpr (NEXT && DP == 128) {
      // Order: LDS reads four ahead of the multiplications that take them, the weights spread over the first half of those
      // (1 x 16384, 32/8 x 128: 1981 -> 1937 us; with 64 dims it costs a wave per SIMD: 39 -> 45 us for 24 ragged 14/2)
      constexpr int kQK = 2 * kSteps, kPV = 4 * (DP / 32), kValu = 6, kExp = (32 + kQK - 1) / kQK;
      __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
      for (int i = 0; i < kQK - 4; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, kValu, 0);
        __builtin_amdgcn_sched_group_barrier(0x400, kExp, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, kValu, 0);
        __builtin_amdgcn_sched_group_barrier(0x400, kExp, 0);
      }
#pragma unroll
      for (int i = 0; i < kPV - 4; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
      }
    }
  }

  // All tiles: `mine` of them have keys for this wave, of which all rows see the first `full` whole. first_keys() makes tile
  // 0's keys readable, turn(t) tile t's values and tile t + 1's keys, and starts the copies of what comes after; left(t):
  // keys of tile t that this lane's row sees.
  template <class First, class Turn, class Left>
  __device__ __forceinline__ void run(int tiles, int mine, int full, float c, First first_keys, Turn turn, Left left) {
    if (tiles <= 0) return;
    f32x16 a[2], b[2];
    int t = 0;
    first_keys();
    if (mine > 0) {
      multiply(0, a);
      maximum<true>(a, c, left(0));
      for (; t + 2 < full; t += 2) {
        turn(t);
        step<true, false>(a, b, 0, kTile, c, 0);
        turn(t + 1);
        step<true, false>(b, a, kTile, 0, c, 0);
      }
      for (; t + 1 < mine; ++t) {
        turn(t);
        step<true, true>(a, b, (t & 1) * kTile, ((t + 1) & 1) * kTile, c, left(t + 1));
        a[0] = b[0];
        a[1] = b[1];
      }
      turn(t);
      step<false, false>(a, b, (t & 1) * kTile, 0, c, 0);
      ++t;
    }
    for (; t < tiles; ++t) turn(t);                  // copies for the other waves
  }
};

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
// Three ways through an item's keys:
//   split keys   16 or 32 rows, units of 32 keys: for few rows the keys' bytes are all that counts, and every wave keeps
//                loads of its own in flight. A run belongs to a block, whose waves take every fourth unit and are joined
//                at the end, or, where items are short, to a single wave (64 sequences of 100 keys, 8 K/V heads: an item
//                takes a block or a wave about 5 us of waiting whatever its length)
//   split rows   up to 128 rows, units of 64 keys, a run per block: as in k_prompt, 32 rows per wave, and the waves share
//                each tile of keys in LDS
constexpr int kCachedWaves = 4;
constexpr int kCachedThreads = 64 * kCachedWaves;
constexpr int kCachedBlocks = 512;         // two per CU
constexpr int kXcds = 8;
constexpr int kWaveKeys = 32;              // split keys: per wave and step
constexpr int kManyRows = 128;             // split rows: rows of a tile
// Measured on the device with 64 sequences on one prefix of 8192, 16 x 6 drafts on prefixes of 1536, 32 sequences of 0 to
// 16384 and 64 of 1 to 512 (14/2 heads of 64, 32/8 of 128): starts of 1/2, 2/3, 2/5 and 3/3 units are within 6 %
// of each other but for 1/2 (32 ragged: 48 us against 43); a prefix's unit at 0.9, 1.5 and 2.8 times a unit of keys
// gives the first case 47, 37 and 34 us, at 5 times 38.
constexpr int kStartRows = 2, kStartKeys = 4;    // units that stand for an item's start
constexpr int kShortItem = 8;                    // split keys: up to as many units per item on average, runs of single waves
constexpr int kLeastRows = 2;                    // split rows: units of a run (drafts 14.9 us; 4: 17.4, 8: 21)
constexpr float kCostRows = 2.2f, kCostKeys = 0.8f;      // of a unit, for dealing blocks to prefixes and own parts
enum { kNone = 0, kOneTile = 1, kTwoTiles = 2, kRows = 3 };      // 16 rows, 32 rows, split rows
__host__ __device__ constexpr int mode_rows(int mode) { return mode == kRows ? kManyRows : 16 * mode; }
__host__ __device__ constexpr int mode_start(int mode) { return mode == kRows ? kStartRows : kStartKeys; }
__host__ __device__ constexpr int mode_unit(int mode) { return mode == kRows ? kPromptKeys : kWaveKeys; }

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
  int32_t* join;                           // Deal of the own parts, of the prefixes; then the entries
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
  int units;                               // of each item, its start among them; 0: no keys
  int from, to;                            // keys
  int first, group;                        // batch entry that the keys belong to; own part: its group
  Seq seq;                                 // of `first`
};
template <bool PREFIX, int MODE>
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
  r.units = r.to > r.from ? (r.to - r.from + mode_unit(MODE) - 1) / mode_unit(MODE) + mode_start(MODE) : 0;
  return r;
}

// Running sums over the entries: every thread of the block has the sums before its run of entries [e0, e1).
struct Scan {
  int e0, e1, units, own, items;
  int total, all_items;
};
template <bool PREFIX, int MODE>
__device__ Scan cached_scan(const CachedCall& a, const Book& book, int (&shared)[2][kCachedWaves]) {
  const int n = PREFIX ? a.n_groups : a.n_seqs, per = (n + kCachedThreads - 1) / kCachedThreads;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Scan r;
  r.e0 = min((int)threadIdx.x * per, n);
  r.e1 = min(r.e0 + per, n);
  int u = 0, it = 0;
  for (int e = r.e0; e < r.e1; ++e) {
    const Entry x = cached_entry<PREFIX, MODE>(a, book, e);
    u += x.items * x.units;
    it += x.items;
  }
  const int su = wave_scan(u), si = wave_scan(it);
  if (lane == 63) {
    shared[0][wave] = su;
    shared[1][wave] = si;
  }
  __syncthreads();
  r.own = u;
  r.units = su - u;
  r.items = si - it;
  r.total = r.all_items = 0;
#pragma unroll
  for (int w = 0; w < kCachedWaves; ++w) {
    if (w < wave) {
      r.units += shared[0][w];
      r.items += shared[1][w];
    }
    r.total += shared[0][w];
    r.all_items += shared[1][w];
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

// Buffer over up to 16 rows (of one page) of K or V from token p on, cut at token `to`; no rows if the page id is bad.
__device__ __forceinline__ u32x4 page_rows(const CachedCall& a, int id, int64_t off, int p, int to) {
  const int rows = min(to - p, 16);
  const bool good = rows > 0 && (uint32_t)id < (uint32_t)a.n_pages;
  const int64_t at = (int64_t)(good ? id : 0) * a.page_elems + off + (int64_t)(p & ((1 << a.page_log) - 1)) * a.dim;
  return buffer_rsrc((uint64_t)(uintptr_t)(a.pool + at), good ? (uint32_t)(rows * a.dim * 2) : 0u);
}

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

  // element i of o[rt][d] is dim 16 d + 4 w + i of row 16 rt + n
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
  rt.sum = half_sum(rt.sum);
  if (slot >= 0 && slot < ps.slots && row0 + col < x.rows) {
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
      pm[1] = rt.sum;
    }
  }
}

// How the units of a pass are dealt out.
struct Plan {
  Deal deal;
  int runs;
  bool alone;                              // runs of single waves, not of blocks
};
__device__ __forceinline__ Plan deal_out(int units, int items, int blocks, int mode) {
  Plan p;
  p.alone = mode != kRows && units <= (kShortItem + mode_start(mode)) * items;
  const int least = mode == kRows ? kLeastRows : 1;
  p.runs = min(p.alone ? blocks * kCachedWaves : blocks, (units + least - 1) / least);
  p.deal.each = units / max(p.runs, 1);
  p.deal.rest = units % max(p.runs, 1);
  return p;
}

// The runs of block `me` of `blocks`.
template <bool BF, int DP, int MODE, bool PREFIX>
__device__ void cached_run(const CachedCall& a, const Book& book, char* lds, const Scan& sc, const Plan& plan, int me, int blocks) {
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
      const Entry x = cached_entry<PREFIX, MODE>(a, book, e);
      if (u < before + x.items * x.units) {
        found[k][0] = e;
        found[k][1] = u - before;
        found[k][2] = items;
        break;
      }
      before += x.items * x.units;
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
  Entry x = cached_entry<PREFIX, MODE>(a, book, e);
  if (x.units == 0 || x.items == 0) return;
  int item = min(in / x.units, x.items - 1), unit = in % x.units;
  while (true) {
    const int units = min(left, x.units - unit);
    const int from = x.from + max(unit - mode_start(MODE), 0) * mode_unit(MODE);
    const int to = min(x.from + (unit + units - mode_start(MODE)) * mode_unit(MODE), x.to);
    if (to > from) {
      if constexpr (MODE == kRows) split_rows<BF, DP, PREFIX>(a, book, lds, x, item, from, to, run + items + item);
      else split_keys<BF, DP, MODE, PREFIX>(a, book, lds, x, item, from, to, run + items + item, plan.alone);
    }
    left -= units;
    if (left <= 0) break;
    unit = 0;
    if (++item == x.items) {
      item = 0;
      do {                                               // left > 0: a further entry has units
        items += x.items;
        if (++e >= n) return;
        x = cached_entry<PREFIX, MODE>(a, book, e);
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
template <bool BF, int DP, int OWN, int PRE>
__global__ __launch_bounds__(kCachedThreads, 2) void k_cached(const CachedCall a) {
  constexpr int kStage = kCachedWaves * 2 * kWaveKeys * DP * 2;     // = 2 buffers of K and V tiles of 64 keys for split rows, halved
  constexpr int kBytes = OWN == kRows || PRE == kRows ? 4 * kPromptKeys * DP * 2 : kStage;
  __shared__ __attribute__((aligned(1024))) char lds[kBytes];
  __shared__ int shared[2][2][kCachedWaves];
  static_assert(kCachedWaves * (16 * (DP + 4) + 32 * 2) * 4 <= kStage, "the join fits the tiles' space");
  __shared__ int2 book_seq[kBook];
  __shared__ int book_group[PRE == kNone ? 1 : kBook + 1], book_prefix[PRE == kNone ? 1 : kBook];
  const Book book{book_seq, book_group, book_prefix, a.n_seqs <= kBook};
  fill_book(a, book);
  const Scan own = cached_scan<false, OWN>(a, book, shared[0]);
  Scan pre;
  pre.total = pre.all_items = 0;
  if constexpr (PRE != kNone) pre = cached_scan<true, PRE>(a, book, shared[1]);

  // blocks for the prefixes: their share of the cost
  int n_pre = 0;
  if constexpr (PRE != kNone) {
    auto cost = [](const Scan& sc, int mode) {
      return sc.total * (mode == kRows ? kCostRows : kCostKeys);
    };
    const float wp = cost(pre, PRE), wo = cost(own, OWN);
    if (pre.total) n_pre = own.total ? min(max((int)(kCachedBlocks / kXcds * wp / (wp + wo) + 0.5f), 1), kCachedBlocks / kXcds - 1) * kXcds : kCachedBlocks;
  }
  const Plan own_plan = deal_out(own.total, own.all_items, kCachedBlocks - n_pre, OWN);
  Plan pre_plan = own_plan;
  if constexpr (PRE != kNone) pre_plan = deal_out(pre.total, pre.all_items, n_pre, PRE);
  if (blockIdx.x == kCachedBlocks - 1) {                 // for k_join
    if (threadIdx.x == 0) {
      reinterpret_cast<Deal*>(a.join)[0] = own_plan.deal;
      reinterpret_cast<Deal*>(a.join)[1] = pre_plan.deal;
    }
    JoinEntry* je = reinterpret_cast<JoinEntry*>(a.join + 4);
    JoinPart* jg = reinterpret_cast<JoinPart*>(je + a.n_seqs);      // the groups' parts, until the sequences have them
    int u, it;
    if constexpr (PRE != kNone) {
      u = pre.units;
      it = pre.items;
      for (int e = pre.e0; e < pre.e1; ++e) {
        const Entry x = cached_entry<true, PRE>(a, book, e);
        jg[e] = JoinPart{u, it, x.units, x.tiles};
        u += x.items * x.units;
        it += x.items;
      }
      __syncthreads();
    }
    u = own.units;
    it = own.items;
    for (int e = own.e0; e < own.e1; ++e) {
      const Entry x = cached_entry<false, OWN>(a, book, e);
      je[e].own = JoinPart{u, it, x.units, x.tiles};
      je[e].pre = PRE != kNone && x.group >= 0 ? jg[x.group] : JoinPart{0, 0, 0, 0};
      je[e].first = PRE != kNone && x.group >= 0 ? book.start(a, x.group) : 0;
      u += x.items * x.units;
      it += x.items;
    }
  }
  // consecutive runs on one XCD: row tiles that read the same keys then share its L2
  const int xcd = blockIdx.x % kXcds, at = blockIdx.x / kXcds, pre_each = n_pre / kXcds, own_each = kCachedBlocks / kXcds - pre_each;
  if constexpr (PRE != kNone) {
    if (at < pre_each) {
      cached_run<BF, DP, PRE, true>(a, book, lds, pre, pre_plan, spread(xcd, at, pre_each, pre_plan.runs), n_pre);
      return;
    }
  }
  cached_run<BF, DP, OWN, false>(a, book, lds, own, own_plan, spread(xcd, at - pre_each, own_each, own_plan.runs), kCachedBlocks - n_pre);
}

// One wave per (sequence, token, head): the partial results of its row, the prefix's and the own part's. A lane holds
// four dims: a quarter (DP 64) or half of the wave reads one slot's row, so one load covers several slots, and eight
// loads are in flight (one dim a lane and four loads: 9 to 15 us for 32 ragged sequences, now 4.8).
template <bool BF, int DP>
__global__ __launch_bounds__(kCachedThreads) void k_join(const CachedCall a, int own_rows, int own_start, int pre_rows, int pre_start) {
  constexpr int kLanes = DP / 4, kPer = 64 / kLanes, kBatch = 8;      // lanes and slots per load, loads in flight
  const int b = blockIdx.x, lane = threadIdx.x & 63;
  const int G = a.heads / a.kv_heads, D = a.dim;
  const int row = blockIdx.y * kCachedWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);   // t * heads + h
  if (row >= a.tokens * a.heads) return;
  const int t = row / a.heads, h = row % a.heads, kvh = h / G;
  const Deal* deals = reinterpret_cast<const Deal*>(a.join);
  const JoinEntry je = reinterpret_cast<const JoinEntry*>(a.join + 4)[b];
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
    return;
  }
  if (sub == 0 && dim < D) *reinterpret_cast<u32x2*>(out + dim) = u32x2{Elem<BF>::pack(y[0], y[1]), Elem<BF>::pack(y[2], y[3])};
}

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

int check_attention(int dtype, int heads, int kv_heads, int dim, float scale) {
  if (dtype != MTC_DTYPE_BF16 && dtype != MTC_DTYPE_F16) return fail(MTC_E_DTYPE, "attention takes bf16 or f16, got dtype %d", dtype);
  if (heads < 1 || kv_heads < 1 || heads % kv_heads)
    return fail(MTC_E_SHAPE, "%d query heads over %d K/V heads", heads, kv_heads);
  if (dim < 8 || dim > MTC_ATTN_MAX_DIM || dim % 8)
    return fail(MTC_E_SHAPE, "head size %d: a multiple of 8 from 8 to %d", dim, MTC_ATTN_MAX_DIM);
  if (!(scale > 0.0f) || !std::isfinite(scale)) return fail(MTC_E_SHAPE, "scale must be positive and finite");
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

// How an item's rows are taken: the least of 16, 32 and 128 rows that holds them.
int mode_for(int64_t rows) { return rows <= 16 ? kOneTile : rows <= 32 ? kTwoTiles : kRows; }

struct CachedPlan {
  int own_mode, pre_mode;
  int own_stride, pre_stride;        // rows of a slot
  int64_t own_slots, pre_slots;
  size_t own_bytes, pre_bytes, join_bytes;
  size_t bytes() const { return own_bytes + pre_bytes + join_bytes; }
};

size_t round_up(size_t x, size_t to) { return (x + to - 1) / to * to; }

int plan_cached(const mtc_cache_desc* c, const mtc_cached_args* a, CachedPlan* p) {
  if (!a) return fail(MTC_E_NULL, "args is NULL");
  if (int rc = mtc_check_cache_desc(c)) return rc;
  if (a->abi_version != MTC_ABI_VERSION) return fail(MTC_E_VERSION, "args of ABI %u, library %d", a->abi_version, MTC_ABI_VERSION);
  if (int rc = check_attention(c->dtype, a->heads, c->kv_heads, c->dim, a->scale)) return rc;
  if (a->reserved != 0) return fail(MTC_E_SHAPE, "reserved must be 0");
  if (a->layer < 0 || a->layer >= c->n_layers) return fail(MTC_E_SHAPE, "layer %d of %d", a->layer, c->n_layers);
  if (a->n_seqs < 0 || a->n_seqs > MTC_CACHED_MAX_SEQS) return fail(MTC_E_SHAPE, "%d sequences, at most %d", a->n_seqs, MTC_CACHED_MAX_SEQS);
  if (!a->seqs && a->n_seqs > c->max_seqs) return fail(MTC_E_SHAPE, "%d sequences, the cache holds %d", a->n_seqs, c->max_seqs);
  if (a->tokens < 1 || a->tokens > MTC_CACHED_MAX_TOKENS)
    return fail(MTC_E_SHAPE, "%d tokens per sequence: 1 to %d", a->tokens, MTC_CACHED_MAX_TOKENS);
  if (a->n_groups < 0 || a->n_groups > a->n_seqs) return fail(MTC_E_SHAPE, "%d groups of %d sequences", a->n_groups, a->n_seqs);
  if ((int64_t)a->tokens * a->heads > 0xFFFF || (int64_t)a->tokens * a->heads * a->n_seqs > 0x3FFFFFF)   // 2^32 threads a launch
    return fail(MTC_E_SHAPE, "%d sequences of %d tokens of %d heads: too many query rows", a->n_seqs, a->tokens, a->heads);
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
  const int64_t units = (int64_t)c->max_pages * c->page_size / kWaveKeys + 1 + std::max(mode_start(kOneTile), mode_start(kRows));
  if (units * (p->own_slots + p->pre_slots) > 0x7FFFFFFF)
    return fail(MTC_E_SHAPE, "%d sequences of up to %d pages of %d tokens, %d row tiles: too much for one call", a->n_seqs, c->max_pages,
                c->page_size, (int)tiles(per, p->own_mode));
  p->own_bytes = round_up((size_t)p->own_slots * p->own_stride * (c->dim + 2) * 4, 256);
  p->pre_bytes = round_up((size_t)p->pre_slots * p->pre_stride * (c->dim + 2) * 4, 256);
  p->join_bytes = round_up(16 + sizeof(JoinEntry) * (size_t)a->n_seqs + sizeof(JoinPart) * (size_t)a->n_groups, 256);
  return MTC_OK;
}

template <bool BF, int DP, int OWN>
void launch_cached(const CachedCall& a, int pre, hipStream_t st) {
  if (pre == kNone) k_cached<BF, DP, OWN, kNone><<<kCachedBlocks, kCachedThreads, 0, st>>>(a);
  else if (pre == kTwoTiles) k_cached<BF, DP, OWN, kTwoTiles><<<kCachedBlocks, kCachedThreads, 0, st>>>(a);
  else k_cached<BF, DP, OWN, kRows><<<kCachedBlocks, kCachedThreads, 0, st>>>(a);
}
template <bool BF, int DP>
void launch_cached(const CachedCall& a, int own, int pre, hipStream_t st) {
  if (own == kOneTile) launch_cached<BF, DP, kOneTile>(a, pre, st);
  else if (own == kTwoTiles) launch_cached<BF, DP, kTwoTiles>(a, pre, st);
  else launch_cached<BF, DP, kRows>(a, pre, st);
}

template <bool BF>
int run_cached(const CachedCall& a, const CachedPlan& p, hipStream_t st) {
  if (a.dim <= 64) launch_cached<BF, 64>(a, p.own_mode, p.pre_mode, st);
  else launch_cached<BF, 128>(a, p.own_mode, p.pre_mode, st);
  if (int rc = check_launch("k_cached")) return rc;
  const dim3 grid(a.n_seqs, (a.tokens * a.heads + kCachedWaves - 1) / kCachedWaves);
  if (a.dim <= 64) k_join<BF, 64><<<grid, kCachedThreads, 0, st>>>(a, mode_rows(p.own_mode), mode_start(p.own_mode), mode_rows(p.pre_mode), mode_start(p.pre_mode));
  else k_join<BF, 128><<<grid, kCachedThreads, 0, st>>>(a, mode_rows(p.own_mode), mode_start(p.own_mode), mode_rows(p.pre_mode), mode_start(p.pre_mode));
  return check_launch("k_join");
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
  CachedCall k;
  const int64_t head = (int64_t)c->page_size * c->dim;
  k.pool = (const uint16_t*)c->pool;
  k.page_elems = 2 * head * c->kv_heads * c->n_layers;
  k.k_off = 2 * head * c->kv_heads * a->layer;
  k.v_off = k.k_off + head * c->kv_heads;
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
  return c->dtype == MTC_DTYPE_BF16 ? run_cached<true>(k, p, (hipStream_t)hip_stream) : run_cached<false>(k, p, (hipStream_t)hip_stream);
}
