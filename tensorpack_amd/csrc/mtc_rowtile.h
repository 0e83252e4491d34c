// 32 query rows of one wave through tiles of 64 keys in LDS: the inner loop of the attention kernels with many rows.
#pragma once

#include "mtc_attn.h"

namespace mtc {
namespace attn {

constexpr int kPromptKeys = 64;                   // keys per step

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

}  // namespace attn
}  // namespace mtc
