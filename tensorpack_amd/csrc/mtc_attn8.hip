// gfx950 kernels of attention over the 8-bit cache (include/mtc_serve.h): k_cached and k_join of mtc_cached.h over codes.
//
// The bytes that a call reads are half of a 16-bit cache's, which is what bounds few rows; what the kernels add is the way from
// codes to the matrix core's 16-bit operands, and it differs:
//   few rows   codes lie in LDS as they are; each wave makes f16 whole numbers of them, 1.25 vector instructions a code, and scales are
//              folded into scores and weights
//   many rows  each code is read by four waves, so a wave makes numbers of the cache's type of its quarter (code 2^e is one exactly,
//              nothing is rounded; 2.75 instructions a code: bytes to fp32, a fused multiply-add, pairs packed) and puts those into the
//              tile; from there on the kernel is that of the 16-bit cache
// Weights are rounded to 16 bits once, as the matrix core's operands have to be, and summed as rounded: to f16's 11 bits by few rows over
// either cache, to the cache's type by many, bf16's 8 bits among them (as over the 16-bit cache). Relative error against 64 bits, rounding
// of the result included: 64 sequences on one prefix (bf16, many rows) 2.1e-3, fp32 weights 1.7e-3; 16 x 6 drafts (f16) 2.4e-4 and 2.1e-4; bf16, few
// rows 1.5e-3 both.
// Memory cannot hold an infinity or a NaN here (scales are bounded as they are read, K's and V's alike, codes are integers), so a key that a
// row does not see has no part in it by its weight of 0 alone, and no row is computed again.
//
// 32 sequences of 8192, 32/8 heads of 128, 537 MB: 109 us a pass, 4.9 TB/s (a 1 GiB copy: 5.14; the 16-bit cache: 193). 32 ragged ones up to
// 16384, 92 MB: 27.6 us, with the join 31 a pass; its start is much of it (the lists, the table, the first keys: one of 200 keys takes 8 us), and
// items that change within a block's run. As 16-bit numbers in LDS, 32 keys a step, it took 29.6 us and 32 of 8192 114.
// 64 sequences on a prefix of 8192: 36 us, of which some 21 are start, fill and the partial results of 64 KB a run; a step of 64 keys
// takes 3.1 us with two blocks a CU, half of it conversions. Runs of 4 or 8 units at least (fewer partial results): 43.4 and 48.5 us a
// pass against 43.8; the first two tiles' copies issued together: 43.5 and 43.5.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mtc_attn8.h"

using mtc::host::check_launch;

namespace mtc {
namespace attn {
namespace {

// ---------------------------------------------------------------------------
// few rows: codes in LDS
// ---------------------------------------------------------------------------
// Subtiles of 32 keys (or their values) as memory has them, a row of DP bytes cut into 16-byte pieces; piece c of row r lies at place
// c ^ codes_key(r). Both readings take the same piece of rows that differ: keys 16 consecutive rows at a time, values the rows
// 4 w .. 4 w + 3 and 16 + 4 w .. of two w.
template <int DP>
__device__ __forceinline__ uint32_t codes_key(uint32_t row) {
  return DP == 128 ? (row >> 1 & 7u) ^ (row >> 4 & 1u) << 2 : (row >> 2 & 3u) ^ (row >> 4 & 1u) << 1;
}

// Codes as f16 numbers of the same value. A byte u under 0x64 is 1024 + u; u = code + 128.
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& a, uint32_t& b) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  w ^= 0x80808080u;
  const h2 minus = {(_Float16)-1152.0f, (_Float16)-1152.0f};
  a = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) + minus);
  b = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) + minus);
}

// Transposed read of bytes: of the 16 lanes of a group, lane i fetches 8 bytes (half i & 1 of a 16-byte piece of row i / 2 of 8) and
// gets column i of these rows.
__device__ __forceinline__ u32x2 read_transposed8(uint32_t at) {
  typedef int i32x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2*)(uintptr_t)at));
}

// Global -> LDS copy of 4 bytes per lane, to lds + 4 lane. (The wait state after m0 is written stands here, as in copy16.)
__device__ __forceinline__ void copy4(uint64_t from, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 3\n\tglobal_load_lds_dword %0, off" : : "v"(from), "s"(lds) : "memory", "m0");
}
// Waits until at most `base` copies and those of `further` whole tiles (EACH copies) are in flight.
template <int BASE, int EACH, int MOST>
__device__ __forceinline__ void wait_tiles(int further) {
  if constexpr (MOST == 0) {
    wait_copies<BASE>();
  } else {
    if (further >= MOST) wait_copies<BASE + MOST * EACH>();
    else wait_tiles<BASE, EACH, MOST - 1>(further);
  }
}

__device__ const uint32_t no_scale = 0;    // of keys on no page: the least there is, so that their zeros never are the largest values

// The nearest number of 11 bits. (NaN stays NaN: matrix instructions and exponentials give no payload that could carry over.)
__device__ __forceinline__ float round11(float x) {
  return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, x) + 0x1000u) & ~0x1FFFu);
}

constexpr int kWaveKeys = 64;              // split keys: per wave and step
constexpr int kSubs = kWaveKeys / 32;      // matrix steps of 32 keys (the depth of a product with the values)
constexpr int kBlocks = kWaveKeys / codes::kBlock;
template <int DP>
struct KeyTiles {
  static constexpr int kTile = kWaveKeys * DP, kDeep = 128 / DP;                 // bytes of a tile, tiles ahead
  static constexpr int kScales = 256;                                            // LDS of a tile's scales (2 kBlocks words are used)
  static constexpr int kBytes = kDeep * (2 * kTile + kScales);                   // of a wave
};

// One item's keys [from, to) (from a multiple of 16) into a partial result, by the block (the keys split over its waves)
// or by this wave alone.
//
// Codes reach LDS as they are (direct copies, kDeep tiles of 64 keys ahead) and become f16 between LDS and the matrix core, 1.25
// vector instructions each, for either type of cache. bf16 q are scaled by a power of two, the row's largest to 2^15 or more, so that an
// element loses at most 2^-40 of the largest (a score 2^-40 max |q| sum |k|: less than its fp32 sum does, unless K is 0 where q is
// large). Scales are folded in where there is one number per key instead of per element: a key's into its score, a value's into
// its weight. With s = score (log2), m its running maximum and e = log2 of the value's scale:
//   l = sum 2^(s - m),   o = sum 2^(s + e - t) code,   t the running maximum of s + e;   result 2^(t - m) o / l
// so that weights keep f16's precision whatever the scales are. m and t are rounded up to whole numbers: a key's weights in l and o
// then differ by a power of two, and one rounding, to f16's 11 bits (half a step: 2^-11), serves both, so that a constant V comes out as
// itself. (f16 has a weight's rounded bits from 2^-14 on; below that it loses less than 2^-24 of one, where the row's largest is 2^6 or
// more.) Bounds, any q, and one rounding cost 2 % (32 ragged sequences: 30.3 -> 30.9 us a pass; heads of 64: 26.7 -> 27.7).
template <bool BF, int DP, int MT, bool PREFIX>
__device__ void split_keys(const CodesCall& a, const Book& book, char* lds, const Entry& x, int item, int from, int to, int slot, bool alone) {
  using H = Elem<false>;
  using Tiles = KeyTiles<DP>;
  constexpr int kTile = Tiles::kTile, kDeep = Tiles::kDeep, kSub = 32 * DP, kHalf = 16 * DP;      // bytes of 64, 32, 16 keys
  constexpr int kHalfCopies = kHalf / 1024, kCopyRows = 1024 / DP, kCopies = kBlocks * kHalfCopies;      // of 16 keys, of a tile
  constexpr int kKeyCopies = kCopies + 1, kBoth = kKeyCopies + kCopies;          // keys with scales; with their values
  constexpr int kSteps = DP / 32;
  constexpr float kLag = 8.0f;                           // bits that weights may grow before o is scaled down
  const int stride = alone ? kWaveKeys : kCachedWaves * kWaveKeys;
  const Pass& ps = PREFIX ? a.pre : a.own;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, w = lane >> 4;
  const int D = a.dim;
  const int kvh = item / x.tiles, row0 = (item % x.tiles) * 16 * MT;
  const int rows = min(x.rows - row0, 16 * MT);

  PageWindow pages{a.table + (int64_t)x.seq.row * a.max_pages, 0, -1, a.max_pages};
  const int first = alone ? from : from + kWaveKeys * wave;
  const int tiles = first < to ? (to - first + stride - 1) / stride : 0;
  if (tiles) pages.load(first >> a.page_log);

  uint32_t from_lane[2][kHalfCopies];                    // byte offsets within 16 rows
#pragma unroll
  for (int hf = 0; hf < 2; ++hf)
#pragma unroll
    for (int i = 0; i < kHalfCopies; ++i) {
      const uint32_t r = i * kCopyRows + lane / (DP / 16), c = lane % (DP / 16) ^ codes_key<DP>(16 * hf + r);
      from_lane[hf][i] = (int)c * 16 < a.room ? r * a.room + c * 16 : kOutOfRange;
    }
  char* const mine = lds + wave * Tiles::kBytes;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(mine));
  const int64_t head = ((int64_t)kvh << a.page_log), head_codes = head * a.room, head_scales = head / codes::kBlock * 2;
  const int mask = (1 << a.page_log) - 1;
  auto copy_codes = [&](int p0, int64_t off, uint32_t dst) {
#pragma unroll
    for (int hf = 0; hf < kBlocks; ++hf) {
      const int p = p0 + 16 * hf, id = pages(p >> a.page_log), count = min(to - p, 16);
      const bool good = count > 0 && (uint32_t)id < (uint32_t)a.n_pages;
      const char* at = a.codes + (int64_t)(good ? id : 0) * a.page_bytes + off + head_codes + (int64_t)(p & mask) * a.room;
      const u32x4 r = buffer_rsrc((uint64_t)(uintptr_t)at, good ? (uint32_t)(count * a.room) : 0u);
#pragma unroll
      for (int i = 0; i < kHalfCopies; ++i) copy16(r, from_lane[hf & 1][i], __builtin_amdgcn_readfirstlane(dst + hf * kHalf + i * 1024));
    }
  };
  // a word that holds the scale (every lane copies one, so that copies can be counted): lanes 0 .. kBlocks - 1 of the keys' blocks, the next ones of the values'
  auto scale_at = [&](int p, int is_v) { return (is_v ? a.v_scales : a.k_scales) + head_scales + (int64_t)((p & mask) / codes::kBlock * 2); };
  auto copy_scales = [&](int p0, uint32_t dst) {
    const int p = p0 + 16 * (lane % kBlocks), id = __shfl(pages.ids, min((p >> a.page_log) - pages.at, 63));
    const char* at = a.codes + (int64_t)id * a.page_bytes + (scale_at(p, lane / kBlocks & 1) & ~3ll);
    copy4((uint64_t)(uintptr_t)((uint32_t)id < (uint32_t)a.n_pages ? at : (const char*)&no_scale), __builtin_amdgcn_readfirstlane(dst));
  };
  auto place = [&](int t) { return (uint32_t)(t % kDeep); };
  auto copy_keys = [&](int t) {
    const int p = first + t * stride;
    if (((p + kWaveKeys - 1) >> a.page_log) - pages.at > 63) pages.load(p >> a.page_log);
    copy_scales(p, lds0 + kDeep * 2 * kTile + place(t) * Tiles::kScales);
    copy_codes(p, a.k_codes, lds0 + place(t) * 2 * kTile);
  };
  auto copy_values = [&](int t) { copy_codes(first + t * stride, a.v_codes, lds0 + place(t) * 2 * kTile + kTile); };
  // this lane's query rows 16 rt + n: piece 4 j + w of 16 dims is multiplied in steps 2 j and 2 j + 1
  u32x4 qf[MT][kSteps];
  int seen[MT], all = 0x7FFFFFFF;                        // keys that a row sees, that all rows see
#pragma unroll
  for (int rt = 0; rt < MT; ++rt) {
    const int rr = row0 + rt * 16 + n;
    const uint16_t* qp = cached_query<PREFIX>(a, book, x, kvh, rr, seen[rt]);
    if (rr < x.rows) all = min(all, seen[rt]);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int d = 16 * (4 * (s >> 1) + w) + 8 * (s & 1);
      qf[rt][s] = rr < x.rows && d < D ? *reinterpret_cast<const u32x4*>(qp + d) : u32x4{0, 0, 0, 0};
    }
  }
  // they are here before the copies start (waits for loads count those too)
#pragma unroll
  for (int rt = 0; rt < MT; ++rt)
#pragma unroll
    for (int s = 0; s < kSteps; ++s) asm volatile("" : "+v"(qf[rt][s]));

#pragma unroll
  for (int t = 0; t < kDeep; ++t)
    if (t < tiles) {
      copy_keys(t);
      copy_values(t);
    }

  // A score in log2 is a product of q and codes, times scale, times 2^(rest + the exponent of K's scale): of the powers of two, -115 to 112 of q's
  // scaling and -100 to 100, neither factor leaves fp32's range, nor becomes 0.
  // (read by itself: else the compiler keeps it and its neighbours among the arguments in LDS, 4 KB a block, 31 -> 42 us for f16)
  const float c = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, a.c)));
  float scale[MT];
  int rest[MT];
#pragma unroll
  for (int rt = 0; rt < MT; ++rt) {
    scale[rt] = c;
    rest[rt] = 0;
    if constexpr (BF) {
      uint32_t most = 0;                                 // the row's largest magnitude
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) most = max(max(most, qf[rt][s][i] << 16 & 0x7FFF0000u), qf[rt][s][i] & 0x7FFF0000u);
      most = max(most, (uint32_t)__shfl_xor((int)most, 16));
      most = max(most, (uint32_t)__shfl_xor((int)most, 32));
      const int raised = min(max((int)(most >> 23) - 127, -100), 127) - 15;      // q is scaled by 2^-raised: a normal number, its inverse too
      const float by = codes::power(-raised);
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t u = qf[rt][s][i];
          qf[rt][s][i] = H::pack(Elem<true>::widen((uint16_t)u) * by, Elem<true>::widen((uint16_t)(u >> 16)) * by);
        }
      const int now = min(max(raised, -90), 90);
      scale[rt] = fminf(scale[rt] * codes::power(now), 3.40282347e+38f);
      rest[rt] = raised - now;
    }
  }
#pragma unroll
  for (int d = 8; d; d >>= 1) all = min(all, __shfl_xor(all, d));
  all = __builtin_amdgcn_readfirstlane(all);

  const uint32_t v_row = (n < 8 ? 0u : 16u) + 4 * w + (n >> 1 & 3u);      // that this lane fetches for the transposed read
  const uint32_t v_at = lds0 + kTile + v_row * DP + 8 * (n & 1);
  const uint32_t v_key = codes_key<DP>(v_row);

  f32x4 o[MT][DP / 16];
  float top[MT], most[MT], sum[MT];                      // m, t and this lane's share of l
#pragma unroll
  for (int rt = 0; rt < MT; ++rt) {
    top[rt] = most[rt] = -INFINITY;
    sum[rt] = 0.0f;
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) o[rt][d] = f32x4{};
  }
  for (int t = 0; t < tiles; ++t) {
    const int pos = first + t * stride;
    const uint32_t buf = place(t) * 2 * kTile;
    wait_tiles<kCopies, kBoth, kDeep - 1>(tiles - 1 - t);          // keys and scales are there
    f32x4 s[MT][kBlocks];
#pragma unroll
    for (int rt = 0; rt < MT; ++rt)
#pragma unroll
      for (int g = 0; g < kBlocks; ++g) s[rt][g] = f32x4{};
#pragma unroll
    for (int j = 0; j < kSteps / 2; ++j)
#pragma unroll
      for (int g = 0; g < kBlocks; ++g) {
        const uint32_t r = (g & 1) * 16 + n;             // in its 32 keys
        const u32x4 k = *reinterpret_cast<const u32x4*>(mine + buf + (g >> 1) * kSub + r * DP + ((4 * j + w) ^ codes_key<DP>(r)) * 16);
        u32x4 lo, hi;
        uint32_t u, v;
        widen4(k[0], u, v);
        lo[0] = u; lo[1] = v;
        widen4(k[1], u, v);
        lo[2] = u; lo[3] = v;
        widen4(k[2], u, v);
        hi[0] = u; hi[1] = v;
        widen4(k[3], u, v);
        hi[2] = u; hi[3] = v;
#pragma unroll
        for (int rt = 0; rt < MT; ++rt) {
          s[rt][g] = H::mfma16(lo, qf[rt][2 * j], s[rt][g]);
          s[rt][g] = H::mfma16(hi, qf[rt][2 * j + 1], s[rt][g]);
        }
      }
    int ks[kBlocks];                                     // log2 of the keys' scales, of the values', of the tile's blocks
    float ve[kBlocks];
    const char* const sc = mine + kDeep * 2 * kTile + place(t) * Tiles::kScales;
#pragma unroll
    for (int g = 0; g < kBlocks; ++g) {
      const int p = pos + 16 * g;
      ks[g] = codes::exponent_of<BF>(*reinterpret_cast<const uint16_t*>(sc + 4 * g + (scale_at(p, 0) & 2)));
      ve[g] = (float)codes::exponent_of<BF>(*reinterpret_cast<const uint16_t*>(sc + 4 * (kBlocks + g) + (scale_at(p, 1) & 2)));
    }
    wait_lds();
    if (t + kDeep < tiles) copy_keys(t + kDeep);
    // element i of s[rt][g]: key pos + 16 g + 4 w + i, query row 16 rt + n
    u32x4 p[MT][kSubs];
#pragma unroll
    for (int rt = 0; rt < MT; ++rt) {
      const int end = min(seen[rt], to);
#pragma unroll
      for (int g = 0; g < kBlocks; ++g) s[rt][g] *= scale[rt];
      if (pos + kWaveKeys > min(all, to)) {
#pragma unroll
        for (int g = 0; g < kBlocks; ++g)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (pos + 16 * g + 4 * w + i >= end) s[rt][g][i] = -INFINITY;
      }
      float m1 = -INFINITY, t1 = -INFINITY, by[kBlocks];
#pragma unroll
      for (int g = 0; g < kBlocks; ++g) {
        const float mx = fmaxf(fmaxf(s[rt][g][0], s[rt][g][1]), fmaxf(s[rt][g][2], s[rt][g][3]));
        by[g] = codes::power(rest[rt] + ks[g]);
        m1 = fmaxf(m1, mx * by[g]);
        t1 = fmaxf(t1, __builtin_fmaf(mx, by[g], ve[g]));
      }
      m1 = half_max(fmaxf(m1, __shfl_xor(m1, 16)));
      t1 = half_max(fmaxf(t1, __shfl_xor(t1, 16)));
      const float was = top[rt];
      top[rt] = fmaxf(was, __builtin_ceilf(m1));
      const float base = top[rt] == -INFINITY ? 0.0f : top[rt];
      sum[rt] *= exp2_fast(was - base);
      if (__ballot(t1 > most[rt] + 15.0f)) {             // weights stay below 2^15 in f16
        const float before = most[rt];
        most[rt] = fmaxf(before, __builtin_ceilf(t1) - (15.0f - kLag));
        const float fade = most[rt] == -INFINITY ? 1.0f : exp2_fast(before - most[rt]);
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) o[rt][d] *= fade;
      }
      const float shift = base - (most[rt] == -INFINITY ? 0.0f : most[rt]);
      float add[2] = {0.0f, 0.0f};
#pragma unroll
      for (int g = 0; g < kBlocks; ++g) {
        const float f = codes::power((int)fminf(fmaxf(ve[g] + shift, -126.0f), 126.0f));
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          const float y0 = round11(exp2_fast(__builtin_fmaf(s[rt][g][i], by[g], -base)));
          const float y1 = round11(exp2_fast(__builtin_fmaf(s[rt][g][i + 1], by[g], -base)));
          add[i >> 1] += y0 + y1;
          p[rt][g >> 1][2 * (g & 1) + (i >> 1)] = H::pack(y0 * f, y1 * f);
        }
      }
      sum[rt] += add[0] + add[1];
    }
    // values are there
    if (t + kDeep < tiles) wait_copies<kKeyCopies + (kDeep - 1) * kBoth>();
    else wait_tiles<0, kBoth, kDeep - 1>(tiles - 1 - t);
#pragma unroll
    for (int h = 0; h < kSubs; ++h)
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) {
        const u32x2 c = read_transposed8(v_at + buf + h * kSub + ((d ^ v_key) << 4));
        uint32_t v0, v1, v2, v3;
        widen4(c[0], v0, v1);
        widen4(c[1], v2, v3);
#pragma unroll
        for (int rt = 0; rt < MT; ++rt) o[rt][d] = H::mfma16(u32x4{v0, v1, v2, v3}, p[rt][h], o[rt][d]);
      }
    wait_lds();
    if (t + kDeep < tiles) copy_values(t + kDeep);
  }
#pragma unroll
  for (int rt = 0; rt < MT; ++rt) {
    const float f = most[rt] == -INFINITY ? 1.0f : exp2_fast(most[rt] - top[rt]);
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) o[rt][d] *= f;
  }
  store_keys<DP, MT>(ps, lds, slot, alone, rows, D, o, top, sum);
}

// ---------------------------------------------------------------------------
// many rows: numbers in LDS
// ---------------------------------------------------------------------------
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

// 16 rows (one block: of one page and scale), a wave's share of a tile. The codes are copied into the place of the numbers; each lane
// then takes back the 16 bytes that it brought, and the wave writes its rows of numbers over them.
template <bool BF, int DP>
struct Rows16 {
  static constexpr int kLanes = DP / 16, kCopyRows = 64 / kLanes, kCopies = 16 / kCopyRows;      // lanes of a row, rows of a copy
  uint16_t scale;

  // Rows from token p on into `place`; zeros past token `to`, or if the page id is bad.
  __device__ __forceinline__ void copy(const CodesCall& a, int id, int64_t codes_off, int64_t scales_off, int p, int to, uint32_t place) {
    const uint32_t lane = threadIdx.x & 63, piece = lane % kLanes * 16;
    const int in = p & ((1 << a.page_log) - 1), count = min(to - p, 16);
    const bool good = count > 0 && (uint32_t)id < (uint32_t)a.n_pages;
    const char* const page = a.codes + (int64_t)(good ? id : 0) * a.page_bytes;
    scale = *reinterpret_cast<const uint16_t*>(page + scales_off + in / codes::kBlock * 2);
    const u32x4 r = buffer_rsrc((uint64_t)(uintptr_t)(page + codes_off + (int64_t)in * a.room), good ? (uint32_t)(count * a.room) : 0u);
#pragma unroll
    for (int i = 0; i < kCopies; ++i)
      copy16(r, (int)piece < a.room ? (i * kCopyRows + lane / kLanes) * a.room + piece : kOutOfRange,
             __builtin_amdgcn_readfirstlane(place + i * 1024));
  }
  // When the copies have landed. Rows of a tile whose rows have the key `key`.
  template <class Key>
  __device__ __forceinline__ void widen(char* place, Key key) const {
    const uint32_t lane = threadIdx.x & 63, piece = lane % kLanes * 2;
    const float s = codes::scale_of<BF>(scale);
    u32x4 z[kCopies];
#pragma unroll
    for (int i = 0; i < kCopies; ++i) z[i] = *reinterpret_cast<const u32x4*>(place + i * 1024 + lane * 16);
    asm volatile("" ::: "memory");                         // (LDS serves a wave in order)
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const uint32_t row = i * kCopyRows + lane / kLanes;
      u32x4 lo, hi;
      expand<BF>(z[i], s, lo, hi);
      *reinterpret_cast<u32x4*>(place + row * (DP * 2) + ((piece ^ key(row)) << 4)) = lo;
      *reinterpret_cast<u32x4*>(place + row * (DP * 2) + (((piece + 1) ^ key(row)) << 4)) = hi;
    }
  }
};

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
  Rows16<BF, DP> kc, vc;
  char* const mine = lds + wave * 16 * kRow;
  const uint32_t lds0 = lds_addr(mine);
  auto copy_keys = [&](int t) {
    const int p = from + t * kPromptKeys + wave * 16;
    kc.copy(a, pages(p >> a.page_log), a.k_codes + head_codes, a.k_scales + head_scales, p, to, lds0 + (t & 1) * kTile);
  };
  auto copy_values = [&](int t) {
    const int p = from + t * kPromptKeys + wave * 16;
    vc.copy(a, pages(p >> a.page_log), a.v_codes + head_codes, a.v_scales + head_scales, p, to, lds0 + (2 + (t & 1)) * kTile);
  };
  auto widen_keys = [&](int t) { kc.widen(mine + (t & 1) * kTile, k_key<DP>); };
  auto widen_values = [&](int t) { vc.widen(mine + (2 + (t & 1)) * kTile, v_key<DP>); };
  const int steps = (to - from + kPromptKeys - 1) / kPromptKeys;
  rt.run(
      steps, busy ? steps : 0, (all - from) / kPromptKeys, a.c,
      [&]() {
        copy_keys(0);
        wait_copies<0>();
        widen_keys(0);
        copy_values(0);
        if (steps > 1) copy_keys(1);
        lds_barrier();
      },
      [&](int t) {
        wait_copies<0>();
        widen_values(t);
        if (t + 1 < steps) widen_keys(t + 1);
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
struct StoreCodes {
  // Starts measured on 32 and 96 ragged sequences up to 16384 and 4000 (blocks: 2, 3, 4, 5, 6, 8 units give 36, 32.6, 30.3, 30.7, 30.6, 30.6
  // and 92, 82, 72.7, 68.9, 69.2, 71.2 us), on 64 up to 512 (waves: 1, 2, 4 units give 16.8, 17.2, 19.9) and on 8 up to 2048 (items of up to 4,
  // 6, 8 units taken by waves: 16.5, 15.0, 14.3). A unit of keys at 0.8, 1.6, 2.5 beside one of rows at 2.2: 64 on a prefix of 8192 43.2, 47.8, 45.5.
  static constexpr bool kCodes = true;
  static constexpr int kKeys = kWaveKeys, kStart = 5, kStartAlone = 1, kShort = 8;
  static constexpr float kCostRows = 2.2f, kCostKeys = 0.8f;
  typedef CodesCall Call;
  using E = Elem<BF>;
  template <int DP>
  static constexpr int kKeysBytes = kCachedWaves * KeyTiles<DP>::kBytes;
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
