// gfx950 kernels of attention over the 8-bit cache (include/mtc_serve.h): k_cached and k_join of mtc_cached.h over codes.
//
// Codes become numbers of the cache's 16-bit type on their way into LDS: code 2^e is one exactly, so nothing is rounded there, and
// from the tiles on the kernels are those of the 16-bit cache. The bytes that a call reads are half, which is what bounds
// few rows; the conversion costs 2.75 vector instructions per code (bytes to fp32, one fused multiply-add, pairs packed).
// Memory cannot hold an infinity or a NaN here (scales are bounded as they are read, codes are integers), so a key that a row does
// not see has no part in it by its weight of 0 alone, and no row is computed again.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mtc_attn8.h"

using mtc::host::check_launch;

namespace mtc {
namespace attn {
namespace {

// 16 codes as two pieces of 8 numbers: (u - 128) s = u s - 128 s of u = code + 128, exact in fp32.
template <bool BF>
__device__ __forceinline__ void expand(u32x4 z, float s, u32x4& lo, u32x4& hi) {
  using E = Elem<BF>;
  const float minus = -128.0f * s;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = z[i] ^ 0x80808080u;
    const float a = __builtin_fmaf((float)(w & 0xFF), s, minus), b = __builtin_fmaf((float)(w >> 8 & 0xFF), s, minus);
    const float c = __builtin_fmaf((float)(w >> 16 & 0xFF), s, minus), d = __builtin_fmaf((float)(w >> 24), s, minus);
    u32x4& to = i < 2 ? lo : hi;
    to[2 * (i & 1)] = E::pack(a, b);
    to[2 * (i & 1) + 1] = E::pack(c, d);
  }
}

// 16 rows (one block of codes: of one page and scale) on their way from memory to a tile: a wave holds them in its lanes.
template <bool BF, int DP>
struct Codes16 {
  static constexpr int kLanes = DP / 16, kRows = 64 / kLanes, kLoads = 16 / kRows;      // lanes of a row, rows of a load
  u32x4 z[kLoads];
  uint16_t scale;

  // Rows from token p on; none if the page id is bad or p is not below `to`. (Rows past `to` in the block hold something; the weights are 0 there.)
  __device__ __forceinline__ void load(const CodesCall& a, int id, int64_t codes_off, int64_t scales_off, int p, int to) {
    const int lane = threadIdx.x & 63, piece = lane % kLanes * 16, in = p & ((1 << a.page_log) - 1);
    const bool good = p < to && (uint32_t)id < (uint32_t)a.n_pages;
    scale = 0;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) z[i] = u32x4{0, 0, 0, 0};
    if (!good) return;
    const char* const page = a.codes + (int64_t)id * a.page_bytes;
    if (piece < a.room)
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        z[i] = *reinterpret_cast<const u32x4*>(page + codes_off + (int64_t)(in + i * kRows + lane / kLanes) * a.room + piece);
    scale = *reinterpret_cast<const uint16_t*>(page + scales_off + in / codes::kBlock * 2);
  }
  // Into rows 0 .. 15 of a tile whose rows have the key `key`.
  template <class Key>
  __device__ __forceinline__ void put(char* tile, Key key) const {
    const int lane = threadIdx.x & 63, piece = lane % kLanes * 2;
    const float s = codes::scale_of<BF>(scale);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const uint32_t row = i * kRows + lane / kLanes;
      u32x4 lo, hi;
      expand<BF>(z[i], s, lo, hi);
      *reinterpret_cast<u32x4*>(tile + row * (DP * 2) + ((piece ^ key(row)) << 4)) = lo;
      *reinterpret_cast<u32x4*>(tile + row * (DP * 2) + (((piece + 1) ^ key(row)) << 4)) = hi;
    }
  }
};

// Orders this wave's LDS accesses before and after it (LDS serves a wave in order).
__device__ __forceinline__ void own_lds() { asm volatile("" ::: "memory"); }

// One item's keys [from, to) (from a multiple of 16) into a partial result, by the block (the keys split over its waves)
// or by this wave alone. Each wave has a tile of 32 keys and one of values of its own; the next ones are in flight in its registers.
template <bool BF, int DP, int MT, bool PREFIX>
__device__ void split_keys(const CodesCall& a, const Book& book, char* lds, const Entry& x, int item, int from, int to, int slot, bool alone) {
  using E = Elem<BF>;
  constexpr int kHalf = 16 * DP * 2;
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

  const int64_t head = ((int64_t)kvh << a.page_log), head_codes = head * a.room, head_scales = head / codes::kBlock * 2;
  Codes16<BF, DP> kc[2], vc[2];
  auto load = [&](Codes16<BF, DP>(&to_regs)[2], int at, int64_t codes_off, int64_t scales_off) {
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int p = at + 16 * hf;
      to_regs[hf].load(a, pages(p >> a.page_log), codes_off + head_codes, scales_off + head_scales, p, to);
    }
  };
  if (pos < to) {
    load(kc, pos, a.k_codes, a.k_scales);
    load(vc, pos, a.v_codes, a.v_scales);
  }

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

  char* const kt = lds + wave * 4 * kHalf;
  char* const vt = kt + 2 * kHalf;
  f32x4 o[MT][DP / 16];
  float top[MT], sum[MT];
#pragma unroll
  for (int rt = 0; rt < MT; ++rt) {
    top[rt] = -INFINITY;
    sum[rt] = 0.0f;
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) o[rt][d] = f32x4{};
  }
  while (pos < to) {
    const int next = pos + stride;
    const bool more = next < to;
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) kc[hf].put(kt + hf * kHalf, k_key<DP>);
    own_lds();
    if (more) {
      if (((next + kWaveKeys - 1) >> a.page_log) - pages.at > 63) pages.load(next >> a.page_log);
      load(kc, next, a.k_codes, a.k_scales);
    }
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
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) vc[hf].put(vt + hf * kHalf, v_key<DP>);
    own_lds();
    if (more) load(vc, next, a.v_codes, a.v_scales);
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) {
      const u32x2 lo = read_v<DP>(vt, 4 * w, d * 16, n), hi = read_v<DP>(vt, 16 + 4 * w, d * 16, n);
#pragma unroll
      for (int rt = 0; rt < MT; ++rt) o[rt][d] = E::mfma16(u32x4{lo[0], lo[1], hi[0], hi[1]}, p[rt], o[rt][d]);
    }
    own_lds();
    pos = next;
  }
  store_keys<DP, MT>(ps, lds, slot, alone, rows, D, o, top, sum);
}

// The same with the rows split over the waves, 32 each, and tiles of 64 keys shared by the block: each wave brings 16 keys.
template <bool BF, int DP, bool PREFIX>
__device__ void split_rows(const CodesCall& a, const Book& book, char* lds, const Entry& x, int item, int from, int to, int slot) {
  constexpr int kRow = DP * 2;
  constexpr int kTile = kPromptKeys * kRow;
  const Pass& ps = PREFIX ? a.pre : a.own;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31;
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

  const int64_t head = ((int64_t)kvh << a.page_log), head_codes = head * a.room, head_scales = head / codes::kBlock * 2;
  Codes16<BF, DP> kc, vc;
  char* const mine = lds + wave * 16 * kRow;
  auto load_keys = [&](int t) {
    const int p = from + t * kPromptKeys + wave * 16;
    kc.load(a, pages(p >> a.page_log), a.k_codes + head_codes, a.k_scales + head_scales, p, to);
  };
  auto load_values = [&](int t) {
    const int p = from + t * kPromptKeys + wave * 16;
    vc.load(a, pages(p >> a.page_log), a.v_codes + head_codes, a.v_scales + head_scales, p, to);
  };
  auto put_keys = [&](int t) { kc.put(mine + (t & 1) * kTile, k_key<DP>); };
  auto put_values = [&](int t) { vc.put(mine + (2 + (t & 1)) * kTile, v_key<DP>); };
  const int steps = (to - from + kPromptKeys - 1) / kPromptKeys;
  rt.run(
      steps, busy ? steps : 0, (all - from) / kPromptKeys, a.c,
      [&]() {
        load_keys(0);
        load_values(0);
        put_keys(0);
        if (steps > 1) load_keys(1);
        put_values(0);
        if (steps > 1) load_values(1);
        if (steps > 1) put_keys(1);
        if (steps > 2) load_keys(2);
        lds_barrier();
      },
      // tile t's values and tile t + 1's keys were put before the barrier; the next ones are put, those after them start
      [&](int t) {
        lds_barrier();
        const int next = from + (t + 2) * kPromptKeys;
        if (t + 1 < steps) put_values(t + 1);
        if (t + 2 < steps) put_keys(t + 2);
        if (t + 2 < steps) {
          if (((next + 2 * kPromptKeys - 1) >> a.page_log) - pages.at > 63) pages.load(next >> a.page_log);
          load_values(t + 2);
        }
        if (t + 3 < steps) load_keys(t + 3);
      },
      [&](int t) { return seen - from - t * kPromptKeys; });
  lds_barrier();                                         // the next item may fill the tiles
  const int r = wave * 32 + col;
  const float sum = half_sum(rt.sum);
  if (slot >= 0 && slot < ps.slots && row0 + col < x.rows) store_rows<BF, DP>(ps, slot, r, D, rt, sum);
}

template <bool BF>
struct StoreCodes {
  typedef CodesCall Call;
  using E = Elem<BF>;
  template <int DP, int MODE, bool PREFIX>
  static __device__ __forceinline__ void keys(const Call& a, const Book& book, char* lds, const Entry& x, int item, int from, int to, int slot,
                                              bool alone) {
    split_keys<BF, DP, MODE, PREFIX>(a, book, lds, x, item, from, to, slot, alone);
  }
  template <int DP, bool PREFIX>
  static __device__ __forceinline__ void rows(const Call& a, const Book& book, char* lds, const Entry& x, int item, int from, int to, int slot) {
    split_rows<BF, DP, PREFIX>(a, book, lds, x, item, from, to, slot);
  }
  static __device__ __forceinline__ bool join_again(const Call&, int, int, int, int, const f32x4&, uint16_t*) { return false; }
};

}  // namespace

int run_codes(const CodesCall& a, bool bf, const CachedPlan& p, hipStream_t st) {
  return bf ? run_cached<StoreCodes<true>>(a, p, st) : run_cached<StoreCodes<false>>(a, p, st);
}

}  // namespace attn
}  // namespace mtc
