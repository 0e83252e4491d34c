// gfx950 kernels of a beam search step (include/mtc_serve.h).
//
// k_beam reads the logits once: a wave holds its chunk of a row in registers, takes its maximum and sum of exponentials and its n
// best values. k_beam_join puts a row's sums together and picks the n best of all rows' candidates. A chunk's n best are enough,
// since within a row the order of scores is the order of the logits.

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

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
constexpr int kJoinList = 1024;            // and the join's

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

// Maximum over the wave, in every lane (row shifts, then the rows' maxima).
__device__ __forceinline__ float wave_top(float x) {
  auto step = [](float y, auto ctrl, auto rows) {
    const int u = __builtin_bit_cast(int, y);
    return fmaxf(y, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(u, u, decltype(ctrl)::value, decltype(rows)::value, 0xF, false)));
  };
  x = step(x, std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xF>{});
  x = step(x, std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xF>{});
  x = step(x, std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xF>{});
  x = step(x, std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xF>{});
  x = step(x, std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xA>{});
  x = step(x, std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xC>{});
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}
// The n-th largest of the lanes' values, -inf if fewer are above that.
__device__ __forceinline__ float nth_top(float x, int n) {
  float t = -INFINITY;
  for (int i = 0; i < n; ++i) {
    t = wave_top(x);
    if (t == -INFINITY) break;
    const uint64_t at = __ballot(x == t);
    if ((int)(threadIdx.x & 63) == __ffsll((unsigned long long)at) - 1) x = -INFINITY;
  }
  return t;
}

// Chunks of 512 ROUNDS logits, 8 ROUNDS a lane. What can be among the n best is not below the n-th largest of the lanes' maxima:
// mostly n or a few more values, which are ranked in LDS by counting. (Many equal values overflow the list: then the best are
// taken one after another.)
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
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int at = from + r * 512;
    if (at + 8 <= a.vocab) {
      const Loose<T, 8> y = *reinterpret_cast<const Loose<T, 8>*>(p + at);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[8 * r + j] = V::get(y.x[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[8 * r + j] = at + j < a.vocab ? V::get(p[at + j]) : -INFINITY;
    }
  }
  float mine = -INFINITY;
#pragma unroll
  for (int e = 0; e < kEach; ++e) mine = fmaxf(mine, x[e]);
  const float top = wave_top(mine), base = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f;
#pragma unroll
  for (int e = 0; e < kEach; ++e) sum += exp2_fast((x[e] - base) * kLog2e);
  sum = wave_sum(sum);
  const int64_t part = (int64_t)row * parts.chunks + chunk;
  if (lane == 0) parts.stat[part] = Stat{top, sum};
  Candidate* const out = parts.best + part * a.n;

  const float least = nth_top(mine, a.n);
  int count = 0;
  Candidate* const list = lists[wave];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const bool take = x[e] >= least && x[e] > -INFINITY;
    const uint64_t all = __ballot(take);
    if (!all) continue;
    const int at = count + __popcll(all & ((1ull << lane) - 1));
    if (take && at < kList) list[at] = Candidate{x[e], from + e / 8 * 512 + e % 8};
    count += __popcll(all);
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  if (count <= kList) {
    for (int i = lane; i < count; i += 64) {
      const Candidate me = list[i];
      int rank = 0;
      for (int j = 0; j < count; ++j) {
        const Candidate it = list[j];
        rank += it.x > me.x || (it.x == me.x && it.v < me.v);
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
      const bool after = x[e] < last.x || (x[e] == last.x && v > last.v);
      if (after && x[e] > best.x) best = Candidate{x[e], v};
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
  int32_t w, v;
};
__device__ __forceinline__ bool before(const Pick& a, const Pick& b) {
  return a.score > b.score || (a.score == b.score && (a.w < b.w || (a.w == b.w && a.v < b.v)));
}
__global__ __launch_bounds__(kThreads) void k_beam_join(const mtc_beam_args a, const Parts parts) {
  __shared__ double offset[MTC_BEAM_MAX];
  __shared__ Pick list[kJoinList];
  __shared__ float least[kWaves];
  __shared__ int count;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (tid == 0) count = 0;
  for (int w = wave; w < a.beams; w += kWaves) {
    const int row = b * a.beams + w;
    double o = a.scores[row];
    if (!(a.done && a.done[row])) {
      const Stat* s = parts.stat + (int64_t)row * parts.chunks;
      float top = -INFINITY;
      for (int c = lane; c < parts.chunks; c += 64) top = fmaxf(top, s[c].top);
      top = wave_top(top);
      double sum = 0.0;
      for (int c = lane; c < parts.chunks; c += 64)
        if (!(s[c].top == -INFINITY && s[c].sum == 0.0f)) sum += (double)s[c].sum * exp((double)s[c].top - (double)top);
      sum = wave_sum(sum);
      o -= (double)top + log(sum);
    }
    if (lane == 0) offset[w] = o;
  }
  __syncthreads();
  const int64_t each = (int64_t)parts.chunks * a.n, total = each * a.beams;
  const Candidate* best = parts.best + (int64_t)b * total;
  // candidate i: of the chunks, then one per beam that has ended
  auto pick = [&](int64_t i) {
    if (i >= total) {
      const int w = (int)(i - total);
      return Pick{a.done && a.done[b * a.beams + w] ? offset[w] : -INFINITY, w, 0};
    }
    const int w = (int)(i / each);
    if (a.done && a.done[b * a.beams + w]) return Pick{-INFINITY, w, 0};
    const Candidate c = best[i];
    return Pick{offset[w] + (double)c.x, w, c.v};
  };
  float mine = -INFINITY;
  for (int64_t i = tid; i < total + a.beams; i += kThreads) mine = fmaxf(mine, (float)pick(i).score);
  const float nth = nth_top(mine, a.n);
  if (lane == 0) least[wave] = nth;
  __syncthreads();
  float from = least[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) from = fmaxf(from, least[w]);
  for (int64_t i = tid; i < total + a.beams; i += kThreads) {
    const Pick p = pick(i);
    if ((float)p.score >= from && p.score > -INFINITY) {
      const int at = atomicAdd(&count, 1);
      if (at < kJoinList) list[at] = p;
    }
  }
  __syncthreads();
  const int found = count;
  auto put = [&](int k, const Pick& p) {
    const int row = b * a.beams + p.w;
    const int64_t at = (int64_t)b * a.n + k;
    a.out_scores[at] = (float)p.score;
    a.tokens[at] = a.done && a.done[row] ? a.pad : p.v;
    a.parents[at] = row;
  };
  auto none = [&](int k) {
    const int64_t at = (int64_t)b * a.n + k;
    a.out_scores[at] = -INFINITY;
    a.tokens[at] = -1;
    a.parents[at] = b * a.beams + min(k, a.beams - 1);
  };
  if (found <= kJoinList) {
    for (int i = tid; i < found; i += kThreads) {
      const Pick me = list[i];
      int rank = 0;
      for (int j = 0; j < found; ++j) rank += before(list[j], me);
      if (rank < a.n) put(rank, me);
    }
    if (tid >= found && tid < a.n) none(tid);
    return;
  }
  // more equal scores than the list holds: one pick after another
  Pick last{INFINITY, -1, -1};
  for (int k = 0; k < a.n; ++k) {
    Pick p{-INFINITY, 0x7FFFFFFF, 0};
    for (int64_t i = tid; i < total + a.beams; i += kThreads) {
      const Pick q = pick(i);
      if (q.score > -INFINITY && before(last, q) && before(q, p)) p = q;
    }
    __syncthreads();                                       // the list's last readers
    list[tid] = p;
    __syncthreads();
    for (int s = kThreads / 2; s; s >>= 1) {
      if (tid < s && before(list[tid + s], list[tid])) list[tid] = list[tid + s];
      __syncthreads();
    }
    last = list[0];
    if (tid == 0) {
      if (last.score > -INFINITY) put(k, last); else none(k);
    }
  }
}

// Chunks of 4096 logits once these fill the chip (two waves a SIMD), else of 512.
int beam_rounds(const mtc_beam_args& a) { return (int64_t)a.n_prompts * a.beams * a.vocab >= (8 << 20) ? 8 : 1; }
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
  if (beam_rounds(a) == 8) k_beam<DT, 8><<<grid, kThreads, 0, st>>>(a, parts);
  else k_beam<DT, 1><<<grid, kThreads, 0, st>>>(a, parts);
  if (int rc = check_launch("k_beam")) return rc;
  k_beam_join<<<a.n_prompts, kThreads, 0, st>>>(a, parts);
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
