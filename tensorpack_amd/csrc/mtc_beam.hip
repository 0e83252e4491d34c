// gfx950 kernels of a beam search step (include/mtc_serve.h).
//
// k_beam reads the logits once: a wave holds its chunk of a row in registers, takes its maximum and sum of exponentials and its n
// best values. k_beam_join puts a row's sums together and picks the n best of all rows' candidates. A chunk's n best are enough,
// since within a row the order of scores is the order of the logits.

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "mtc_host.h"
#include "mtc_values.h"

#define MTC_API extern "C" __attribute__((visibility("default")))

using mtc::host::check_launch;
using mtc::host::fail;
using mtc::host::ok;
using namespace mtc::attn;

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kList = 256;                 // candidates that a wave's list holds
constexpr int kJoinList = 2048;            // and the join's

struct Candidate {
  float x;
  int32_t v;
};
struct Stat {
  float top, sum;                          // of exp(x - top)
};
// Workspace: Stat [row][chunk], then Candidate [row][chunk][n]
struct Parts {
  Stat* stat;
  Candidate* best;
  int32_t chunks;
};

// A value that n or a few more of the lanes' values reach, -inf if fewer than n are above that: the n-th largest, but for its distance to
// the largest, of which 5 bits behind the leading one are found, bit by bit by counting lanes. (Taking the largest away n times costs 150
// cycles each; the least maximum of n groups of lanes is as quick as this, but n ln n values reach it, twice as many in the worst of a hundred
// chunks, which the others wait for: a row of 32000 and 16 picks takes 19 us by that, 10 by this.)
__device__ __forceinline__ float reached(float x, int n) {
  const float top = wave_top(x);
  if (top == -INFINITY) return top;
  const uint32_t far = __builtin_bit_cast(uint32_t, top - x);                // not negative
  uint32_t t = 0;
#pragma unroll
  for (int bit = 30; bit >= 18; --bit) {
    const uint32_t to = t | ((1u << bit) - 1);
    t |= __popcll(__ballot(far <= to)) < n ? 1u << bit : 0u;
  }
  if (t >= 0x7F800000u) return -INFINITY;
  return -wave_top(far <= (t | ((1u << 18) - 1)) ? -x : -INFINITY);
}
constexpr float kLeast = -3.402823466e38f;  // of what is above -inf
constexpr int kTwo = 24;                   // picks beyond which a bound is made of lanes' second values
// As above, from each lane's largest value and another: more than kTwo picks are bounded by the others of half as many lanes, where the lanes'
// maxima alone give little (64 picks: the least of all; 64 beams of 32000 and 64 picks 1170 us without, 43 with; 32 of 8 beams 19.4 and 16.9; 17
// of 8 beams 11.2 and 15.6).
__device__ __forceinline__ float reached(float x, float second, int n) {
  return n > kTwo ? reached(second, (n + 1) / 2) : reached(x, n);
}

// Chunks of 512 ROUNDS logits, 8 ROUNDS a lane. What can be among the n best is not below a value that n of the lanes' maxima reach:
// a few values, which each lane marks by a bit, reads again (from a cache) and ranks in LDS by counting. (Many equal values overflow the
// list: then the best are taken one after another.)
// 256 rows of 128003 bf16, a fifth of them ended, 52 MB: 22.4 us, of which the loads and the maxima take 13 (memory alone 10): all waves'
// loads arrive at much the same time, so little of the selection lies under them. Blocks that load their next chunk ahead were slower (34 to
// 42 us), as were waves that load two chunks and then select from each (of 2048 23.4, of 4096 27.4); sums kept round by round no faster (24). Four rows of 32000 fp32: 4.4 us.
template <int DT, int ROUNDS>
__global__ __launch_bounds__(kThreads) void k_beam(const mtc_beam_args a, const Parts parts) {
  using V = Value<DT>;
  typedef typename V::type T;
  constexpr int kEach = 8 * ROUNDS;
  __shared__ Candidate lists[kWaves][kList];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = blockIdx.y, chunk = blockIdx.x * kWaves + wave;
  if (chunk >= parts.chunks || (a.done && a.done[row])) return;
  const T* p = reinterpret_cast<const T*>(a.logits) + (row / a.beams) * a.stride[0] + (row % a.beams) * a.stride[1];
  const int from = chunk * 64 * kEach + lane * 8;          // element e: from + e / 8 * 512 + e % 8
  float x[kEach];
  const int end = a.vocab - chunk * 64 * kEach;             // of the row, in the chunk
  Loose<T, 8> y[ROUNDS];                                   // all loads before the first is looked at
  if (end >= 64 * kEach) {
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) y[r] = *reinterpret_cast<const Loose<T, 8>*>(p + from + r * 512);
#pragma unroll
    for (int e = 0; e < kEach; ++e) x[e] = V::get(y[e / 8].x[e % 8]);
  } else {
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      if ((r + 1) * 512 <= end) {
        y[r] = *reinterpret_cast<const Loose<T, 8>*>(p + from + r * 512);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[r].x[j] = r * 512 < end ? p[min(from + r * 512 + j, a.vocab - 1)] : T(0);
      }
    }
#pragma unroll
    for (int e = 0; e < kEach; ++e) x[e] = from + e / 8 * 512 + e % 8 < a.vocab ? V::get(y[e / 8].x[e % 8]) : -INFINITY;
  }
  float half[2] = {-INFINITY, -INFINITY};
#pragma unroll
  for (int e = 0; e < kEach; ++e) half[e / 4 % 2] = fmaxf(half[e / 4 % 2], x[e]);
  const float mine = fmaxf(half[0], half[1]);
  const float top = wave_top(mine), base = top == -INFINITY ? 0.0f : top;
  // A term goes through ROUNDS sums, then 3 and 6, not 64: at most 17 * 2^-24 of the log's error. (The exponentials add 3 * 2^-24, and 2.3 * 2^-24 times a
  // term's distance from the maximum, as far as such terms make up the sum: 24 * 2^-24 for 2^20 terms.)
  float sums[8] = {};
#pragma unroll
  for (int e = 0; e < kEach; ++e) sums[e % 8] += exp2_fast((x[e] - base) * kLog2e);
#pragma unroll
  for (int d = 4; d; d >>= 1)
#pragma unroll
    for (int e = 0; e < d; ++e) sums[e] += sums[e + d];
  const float sum = wave_sum(sums[0]);
  const int64_t part = (int64_t)row * parts.chunks + chunk;
  if (lane == 0) parts.stat[part] = Stat{top, sum};
  Candidate* const out = parts.best + part * a.n;

  const float least = fmaxf(reached(mine, fminf(half[0], half[1]), a.n), kLeast);
  uint32_t low = 0, high = 0;
#pragma unroll
  for (int e = 0; e < kEach; ++e) (e < 32 ? low : high) |= x[e] >= least ? 1u << (e % 32) : 0u;
  uint64_t left = (uint64_t)high << 32 | low;
  int count = 0;
  Candidate* const list = lists[wave];
  while (const uint64_t all = __ballot(left != 0)) {
    const int at = count + __popcll(all & ((1ull << lane) - 1));
    if (left && at < kList) {
      const int e = __builtin_ctzll(left);
      list[at].v = from + e / 8 * 512 + e % 8;
    }
    left &= left - 1;
    count += __popcll(all);
  }
  auto own_lds = []() {                                    // LDS serves a wave in order
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
  };
  own_lds();
  if (count <= kList) {
    for (int i = lane; i < count; i += 64) list[i].x = V::get(p[list[i].v]);
    own_lds();
    for (int i = lane; i < count; i += 64) {
      const Candidate me = list[i];
      int rank = 0;
#pragma unroll 8
      for (int j = 0; j < count; ++j) {
        const Candidate it = list[j];
        rank += (int)(it.x > me.x) | ((int)(it.x == me.x) & (int)(it.v < me.v));        // without branches
      }
      if (rank < a.n) out[rank] = me;
    }
    if (lane >= count && lane < a.n) out[lane] = Candidate{-INFINITY, -1};
    return;
  }
  Candidate last{INFINITY, -1};                            // (a value of +inf is no candidate: its row has none)
  for (int k = 0; k < a.n; ++k) {
    Candidate best{-INFINITY, 0x7FFFFFFF};
#pragma unroll
    for (int e = 0; e < kEach; ++e) {                      // places ascend in e
      const int v = from + e / 8 * 512 + e % 8;
      const bool take = ((x[e] < last.x) | ((x[e] == last.x) & (v > last.v))) & (x[e] > best.x);
      best.x = take ? x[e] : best.x;
      best.v = take ? v : best.v;
    }
    const float t = wave_top(best.x);
    int v = best.x == t ? best.v : 0x7FFFFFFF;
#pragma unroll
    for (int d = 32; d; d >>= 1) v = min(v, __shfl_xor(v, d));
    last = Candidate{t, t == -INFINITY ? -1 : v};
    if (lane == 0) out[k] = last;
  }
}

// One block per prompt. Scores are fp64 here: log sums and the beams' scores can be far larger than the differences between the
// logits that decide.
struct Pick {
  double score;
  uint64_t place;                          // w << 32 | v
};
__device__ __forceinline__ bool before(const Pick& a, const Pick& b) {      // without branches
  return (a.score > b.score) | ((a.score == b.score) & (a.place < b.place));
}
__device__ __forceinline__ uint64_t place_of(int w, int v) { return (uint64_t)w << 32 | (uint32_t)v; }
// A thread per chunk of a beam (or several), whose candidates fall: the first ones give a bound, and few chunks have more than one
// above it. Bound by its chain (loads, log sums, bound, ranks): 4 beams of 63 chunks 4.6 us, 32 prompts of 8 beams of 32 chunks 5.9 us.
constexpr int kJoinThreads = 512, kJoinWaves = kJoinThreads / 64;
constexpr int kAhead = 4;                  // candidates of a chunk that are loaded before the bound is known
__global__ __launch_bounds__(kJoinThreads) void k_beam_join(const mtc_beam_args a, const Parts parts) {
  __shared__ double offset[MTC_BEAM_MAX];
  __shared__ int ended[MTC_BEAM_MAX];
  __shared__ Pick list[kJoinList];
  __shared__ float firsts[kJoinThreads], seconds[kJoinThreads];
  __shared__ int count;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int items = a.beams * parts.chunks;
  const Candidate* const best = parts.best + (int64_t)b * items * a.n;
  // everything is loaded in one round (of beams that have ended, whatever is there: it is not used)
  Candidate ahead[kAhead];                                 // of item `tid`
#pragma unroll
  for (int k = 0; k < kAhead; ++k) ahead[k] = tid < items && k < a.n ? best[(int64_t)tid * a.n + k] : Candidate{-INFINITY, -1};
  if (tid == 0) count = 0;
  for (int w = wave; w < a.beams; w += kJoinWaves) {
    const int row = b * a.beams + w;
    const Stat* s = parts.stat + (int64_t)row * parts.chunks;
    Stat x = lane < parts.chunks ? s[lane] : Stat{-INFINITY, 0.0f};
    const double score = a.scores[row];
    const bool over = a.done && a.done[row];
    for (int c = lane + 64; c < parts.chunks; c += 64) {
      const Stat y = s[c];
      const float t = fmaxf(x.top, y.top), u = t == -INFINITY ? 0.0f : t;
      x = Stat{t, x.sum * expf(x.top - u) + y.sum * expf(y.top - u)};
    }
    const float top = wave_top(x.top), base = top == -INFINITY ? 0.0f : top;
    const double sum = wave_sum((double)(x.sum * expf(x.top - base)));
    if (lane == 0) {
      offset[w] = over ? score : score - ((double)top + log(sum));
      ended[w] = over;
    }
  }
  __syncthreads();
  const int my_w = min(tid / parts.chunks, a.beams - 1);
  const bool mine_over = tid < a.beams && ended[tid];      // beam `tid` stands as a candidate
  auto score = [&](int w, float x) { return offset[w] + (double)x; };
  const bool go_on = tid < items && !ended[my_w];
  // The block's bound: a lane of each wave makes one of 64 groups, of which every wave finds the same bound.
  float mine = -INFINITY, second = -INFINITY;
  auto hold = [&](float x) {
    x = fmaxf(x, -INFINITY);                               // NaN, of a row that has no candidates
    second = fmaxf(second, fminf(mine, x));
    mine = fmaxf(mine, x);
  };
  if (mine_over) hold((float)offset[tid]);
  if (go_on) {
    hold((float)score(my_w, ahead[0].x));
    hold((float)score(my_w, ahead[1].x));
  }
  for (int i = tid + kJoinThreads; i < items; i += kJoinThreads) {
    const int w = i / parts.chunks;
    if (!ended[w]) hold((float)score(w, best[(int64_t)i * a.n].x));
  }
  firsts[tid] = mine;
  seconds[tid] = second;
  __syncthreads();
#pragma unroll
  for (int w = 1; w < kJoinWaves; ++w) {
    const int at = (tid + 64 * w) % kJoinThreads;
    hold(firsts[at]);
    hold(seconds[at]);
  }
  const float from = fmaxf(reached(mine, second, a.n), kLeast);
  auto above = [&](int w, float x) { return (float)score(w, x) >= from; };
  auto offer = [&](int at, const Pick& p) {
    if (at < kJoinList) list[at] = p;
  };
  auto rest = [&](int i, int w, int k) {                   // of item i, from candidate k on, to the first below the bound
    for (; k < a.n; ++k) {
      const Candidate c = best[(int64_t)i * a.n + k];
      if (!above(w, c.x)) break;
      offer(atomicAdd(&count, 1), Pick{score(w, c.x), place_of(w, c.v)});
    }
  };
  if (mine_over && (float)offset[tid] >= from) offer(atomicAdd(&count, 1), Pick{offset[tid], place_of(tid, 0)});
  if (go_on) {
    int some = 0;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) some += above(my_w, ahead[k].x);
    if (some) {
      const int at = atomicAdd(&count, some);
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (k < some) offer(at + k, Pick{score(my_w, ahead[k].x), place_of(my_w, ahead[k].v)});
      if (some == kAhead) rest(tid, my_w, kAhead);
    }
  }
  for (int i = tid + kJoinThreads; i < items; i += kJoinThreads) {
    const int w = i / parts.chunks;
    if (!ended[w]) rest(i, w, 0);
  }
  __syncthreads();
  const int found = count;
  auto put = [&](int k, const Pick& p) {
    const int w = (int)(p.place >> 32), row = b * a.beams + w;
    const int64_t at = (int64_t)b * a.n + k;
    a.out_scores[at] = (float)p.score;
    a.tokens[at] = ended[w] ? a.pad : (int32_t)p.place;
    a.parents[at] = row;
  };
  auto none = [&](int k) {
    const int64_t at = (int64_t)b * a.n + k;
    a.out_scores[at] = -INFINITY;
    a.tokens[at] = -1;
    a.parents[at] = b * a.beams + min(k, a.beams - 1);
  };
  if (found <= kJoinList) {
    for (int i = tid; i < found; i += kJoinThreads) {
      const Pick me = list[i];
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < found; ++j) rank += before(list[j], me);
      if (rank < a.n) put(rank, me);
    }
    if (tid >= found && tid < a.n) none(tid);
    return;
  }
  // more equal scores than the list holds: one pick after another
  bool first = true;
  Pick last{INFINITY, 0};
  for (int k = 0; k < a.n; ++k) {
    Pick p{-INFINITY, ~0ull};
    auto take = [&](const Pick& q) {
      if ((q.score > -INFINITY) & (first | before(last, q)) & before(q, p)) p = q;
    };
    if (mine_over) take(Pick{offset[tid], place_of(tid, 0)});
    for (int i = tid; i < items; i += kJoinThreads) {
      const int w = i / parts.chunks;
      if (ended[w]) continue;
      for (int j = 0; j < a.n; ++j) {
        const Candidate c = best[(int64_t)i * a.n + j];
        const Pick q{score(w, c.x), place_of(w, c.v)};
        if (q.score < p.score) break;                      // nor is any after it better
        take(q);
      }
    }
    __syncthreads();                                       // the list's last readers
    list[tid] = p;
    __syncthreads();
    for (int s = kJoinThreads / 2; s; s >>= 1) {
      if (tid < s && before(list[tid + s], list[tid])) list[tid] = list[tid + s];
      __syncthreads();
    }
    last = list[0];
    first = false;
    if (tid == 0) {
      if (last.score > -INFINITY) put(k, last); else none(k);
    }
  }
}

// Chunks of 512 logits, which spread few rows over the chip, or of 4096, which leave the join fewer candidates and fill the chip with many rows.
// Measured, us a call, chunks of 4096 and of 512: 1 x 4 beams of 32000 10.3, 8.9; 16 x 4 10.8, 10.0; 32 x 4 11.0, 11.9; 64 x 4 13.3, 15.9; 1 x 4 of 128003
// 10.5, 10.5; 1 x 8 11.4, 13.1; 1 x 16 14.4, 21.4; 32 x 8 27.6, 43.1; short rows: 256 x 8 of 8192 18.8, 25.0; 256 x 4 of 5003 13.9, 13.9; 1024 x 4 of
// 1500 24.9, 19.0.
constexpr int kManyRounds = 8;
int beam_rounds(const mtc_beam_args& a) {
  const int64_t prompt = (int64_t)a.beams * a.vocab;
  return a.vocab >= 8192 && (prompt >= (512 << 10) || a.n_prompts * prompt >= (3 << 20)) ? kManyRounds : 1;
}
int beam_chunks(const mtc_beam_args& a) {
  const int size = 512 * beam_rounds(a);
  return (a.vocab + size - 1) / size;
}
size_t stat_bytes(const mtc_beam_args& a) {
  return ((size_t)a.n_prompts * a.beams * beam_chunks(a) * sizeof(Stat) + 255) & ~(size_t)255;
}
size_t beam_workspace(const mtc_beam_args& a) {
  return stat_bytes(a) + (size_t)a.n_prompts * a.beams * beam_chunks(a) * a.n * sizeof(Candidate);
}

int check_beam(const mtc_beam_args* a) {
  if (!a) return fail(MTC_E_NULL, "args is NULL");
  if (a->abi_version != MTC_ABI_VERSION) return fail(MTC_E_VERSION, "args of ABI %u, library %d", a->abi_version, MTC_ABI_VERSION);
  if (a->dtype != MTC_DTYPE_F32 && a->dtype != MTC_DTYPE_BF16 && a->dtype != MTC_DTYPE_F16)
    return fail(MTC_E_DTYPE, "logits of dtype %d", a->dtype);
  if (a->beams < 1 || a->beams > MTC_BEAM_MAX || a->n < 1 || a->n > MTC_BEAM_MAX)
    return fail(MTC_E_SHAPE, "%d beams, %d picks: 1 to %d", a->beams, a->n, MTC_BEAM_MAX);
  if (a->vocab < 1 || a->vocab > 0x3FFFFFFF) return fail(MTC_E_SHAPE, "vocabulary of %d", a->vocab);
  if (a->n_prompts < 0 || (int64_t)a->n_prompts * a->beams > 65535)
    return fail(MTC_E_SHAPE, "%d prompts of %d beams: up to 65535 rows", a->n_prompts, a->beams);
  if (a->reserved != 0) return fail(MTC_E_SHAPE, "reserved must be 0");
  if (a->n_prompts && (int64_t)a->n_prompts * a->beams * beam_chunks(*a) > 0xFFFFFF)       // 2^32 threads a launch
    return fail(MTC_E_SHAPE, "%d rows of a vocabulary of %d: too many", a->n_prompts * a->beams, a->vocab);
  return MTC_OK;
}

template <int DT>
int run_beam(const mtc_beam_args& a, const Parts& parts, hipStream_t st) {
  const dim3 grid((parts.chunks + kWaves - 1) / kWaves, a.n_prompts * a.beams);
  if (beam_rounds(a) == kManyRounds) k_beam<DT, kManyRounds><<<grid, kThreads, 0, st>>>(a, parts);
  else k_beam<DT, 1><<<grid, kThreads, 0, st>>>(a, parts);
  if (int rc = check_launch("k_beam")) return rc;
  k_beam_join<<<a.n_prompts, kJoinThreads, 0, st>>>(a, parts);
  return check_launch("k_beam_join");
}

}  // namespace

MTC_API size_t mtc_beam_workspace_bytes(const mtc_beam_args* a) {
  if (check_beam(a) != MTC_OK || a->n_prompts == 0) return 0;
  return beam_workspace(*a);
}

MTC_API int mtc_beam_select(const mtc_beam_args* a, void* workspace, size_t workspace_bytes, void* hip_stream) {
  if (int rc = check_beam(a)) return rc;
  if (a->n_prompts == 0) return ok();
  if (!a->logits || !a->scores || !a->out_scores || !a->tokens || !a->parents)
    return fail(MTC_E_NULL, "logits, scores, out_scores, tokens or parents is NULL");
  const size_t need = beam_workspace(*a);
  if (!workspace || workspace_bytes < need)
    return fail(MTC_E_WORKSPACE, "workspace of %zu bytes, needs %zu", workspace ? workspace_bytes : (size_t)0, need);
  if ((uintptr_t)workspace % 256) return fail(MTC_E_WORKSPACE, "workspace must be 256-byte aligned");
  const Parts parts{(Stat*)workspace, (Candidate*)((char*)workspace + stat_bytes(*a)), beam_chunks(*a)};
  hipStream_t st = (hipStream_t)hip_stream;
  if (a->dtype == MTC_DTYPE_F32) return run_beam<MTC_DTYPE_F32>(*a, parts, st);
  if (a->dtype == MTC_DTYPE_BF16) return run_beam<MTC_DTYPE_BF16>(*a, parts, st);
  return run_beam<MTC_DTYPE_F16>(*a, parts, st);
}
