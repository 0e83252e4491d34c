// gfx950 kernels of the paged cache's bookkeeping and of draft verification, with their C-ABI
// (include/mtc_serve.h).
//
// Bookkeeping runs on the device in a few small launches, so a serving loop need not wait for the GPU to
// know which page is free, and can be captured into a graph. The free set is refs == 0 and the lowest free ids are
// given out first: results then depend on no order of blocks (counts change by integer atomics), and no
// list of free pages has to be kept. state[1] is a page below which none is free, so the search for
// free pages seldom reads more than it gives out.
//
// All of it is bound by the length of its chains of dependent loads (list -> length -> table -> count), about 0.7 us each,
// not by bytes: 64 forks 4.8 us, 64 sequences freed 4.9, 64 extended 8.4. Copies of pages run at memory speed: 455
// pages of 192 KiB moved (compaction of a pool of 4096), 179 MB read and written in 28.6 us.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "mtc_attn.h"
#include "mtc_codes.h"
#include "mtc_host.h"
#include "mtc_serve.h"
#include "mtc_values.h"

#define MTC_API extern "C" __attribute__((visibility("default")))

using mtc::host::check_launch;
using mtc::host::fail;
using mtc::host::ok;
using namespace mtc::attn;
namespace codes = mtc::codes;

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kStatus = 0, kFirstFree = 1, kPairs = 2, kDone = 3;      // words of state

// scratch: pairs of pages to copy (src, dst), a page map or list of free ids, one offset per sequence of a call
__host__ __device__ inline int32_t* scratch_src(const mtc_cache_desc& c) { return c.scratch; }
__host__ __device__ inline int32_t* scratch_dst(const mtc_cache_desc& c) { return c.scratch + c.n_pages; }
__host__ __device__ inline int32_t* scratch_ids(const mtc_cache_desc& c) { return c.scratch + 2 * (int64_t)c.n_pages; }
__host__ __device__ inline int32_t* scratch_start(const mtc_cache_desc& c) { return c.scratch + 3 * (int64_t)c.n_pages; }

__device__ __forceinline__ int pages_of(const mtc_cache_desc& c, int tokens) {
  return (tokens + c.page_size - 1) / c.page_size;
}
// Tokens of sequence s, as far as its table row can hold them: lens may hold anything.
__device__ __forceinline__ int held(const mtc_cache_desc& c, int s) {
  return min(max(c.lens[s], 0), c.max_pages * c.page_size);
}

// Exclusive sum over the block's threads (two counts at once where they are packed); the total in `total`.
__device__ uint64_t block_scan(uint64_t x, uint64_t& total) {
  __shared__ uint64_t part[kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t s = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t y = __shfl_up(s, d);
    if (lane >= d) s += y;
  }
  __syncthreads();
  if (lane == 63) part[wave] = s;
  __syncthreads();
  uint64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) before += part[w];
    total += part[w];
  }
  return before + s - x;
}

// Block-wide OR of error bits.
__device__ int block_or(int x) {
  __shared__ int all;
  __syncthreads();
  if (threadIdx.x == 0) all = 0;
  __syncthreads();
  if (x) atomicOr(&all, x);
  __syncthreads();
  return all;
}

// Sequence numbers seen in a list: one bit each.
constexpr int kMarkWords = MTC_CACHE_MAX_SLOTS / 32;
__device__ __forceinline__ void clear_marks(uint32_t* marks) {
  for (int i = threadIdx.x; i < kMarkWords; i += blockDim.x) marks[i] = 0;
}
__device__ __forceinline__ bool mark(uint32_t* marks, int s) {         // true: it was marked already
  return (atomicOr(&marks[s >> 5], 1u << (s & 31)) >> (s & 31)) & 1;
}

// One block. A thread plans sequence i of each round of 1024; lists of up to 1024 (any but the largest batches) take
// one round, whose plan stays in registers. Loads come in three dependent steps (list, lengths, last page and its count).
struct Extend {
  int s, len, count, old, need;            // need: new pages, the copy of a shared last page (old >= 0) first
};
__global__ __launch_bounds__(kThreads) void k_extend(const mtc_cache_desc c, const int32_t* seqs, const int32_t* counts, int n) {
  __shared__ uint32_t marks[kMarkWords];
  __shared__ int freed;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int32_t* const start = scratch_start(c);
  int32_t* const ids = scratch_ids(c);
  clear_marks(marks);
  if (tid == 0) freed = c.n_pages;
  __syncthreads();

  int bad = 0;
  auto plan = [&](int i, bool check) {
    Extend x{0, 0, 0, -1, 0};
    if (i >= n) return x;
    x.s = seqs[i];
    x.count = counts[i];
    if ((uint32_t)x.s >= (uint32_t)c.max_seqs || (check && mark(marks, x.s))) {
      bad |= MTC_CACHE_BAD_SEQ;
      return x;
    }
    x.len = c.lens[x.s];
    if (x.count < 0 || x.len < 0) bad |= MTC_CACHE_BAD_LENGTH;
    else if ((int64_t)x.len + x.count > (int64_t)c.max_pages * c.page_size) bad |= MTC_CACHE_TABLE_FULL;
    if (bad) return x;
    if (x.len % c.page_size && x.count > 0) {
      const int p = c.table[(int64_t)x.s * c.max_pages + x.len / c.page_size];
      if ((uint32_t)p < (uint32_t)c.n_pages && c.refs[p] > 1) x.old = p;
    }
    x.need = pages_of(c, x.len + x.count) - pages_of(c, x.len) + (x.old >= 0);
    return x;
  };
  constexpr uint64_t kLow = (1ull << 44) - 1;              // 1024 x 2^26 pages stay below 2^44
  int64_t need = 0, copies = 0;
  Extend mine{};
  int64_t my_copy = 0;
  for (int i0 = 0; i0 < n; i0 += kThreads) {
    mine = plan(i0 + tid, true);
    uint64_t total;
    const uint64_t at = block_scan((uint64_t)(mine.old >= 0) << 44 | (uint64_t)mine.need, total);
    if (i0 + tid < n) start[i0 + tid] = (int)min(need + (int64_t)(at & kLow), (int64_t)c.n_pages);
    my_copy = copies + (int64_t)(at >> 44);
    need += (int64_t)(total & kLow);
    copies += (int64_t)(total >> 44);
  }
  bad = block_or(bad);
  if (!bad && need > c.n_pages) bad = MTC_CACHE_NO_PAGES;
  // the lowest free ids, in order
  int64_t found = 0;
  int next_free = c.state[kFirstFree];
  if (!bad && need) {
    const int from = max(next_free, 0);
    for (int64_t p0 = from; p0 < c.n_pages && found < need; p0 += kThreads) {
      const int64_t p = p0 + tid;
      const bool is = p < c.n_pages && c.refs[p] == 0;
      uint64_t total;
      const int64_t at = found + (int64_t)block_scan(is, total);
      if (is && at < need) ids[at] = (int)p;
      found += (int64_t)total;
    }
    if (found < need) bad = MTC_CACHE_NO_PAGES;
  }
  __syncthreads();                                         // ids and start are written
  if (bad) {
    if (tid == 0) {
      c.state[kStatus] |= bad;
      c.state[kPairs] = 0;
    }
    return;
  }
  if (need) next_free = ids[need - 1] + 1;
  // pairs of pages to copy, in the list's order
  int64_t before = 0;
  for (int i0 = 0; i0 < n; i0 += kThreads) {
    if (n > kThreads) {
      mine = plan(i0 + tid, false);
      uint64_t total;
      my_copy = before + (int64_t)block_scan(mine.old >= 0, total);
      before += (int64_t)total;
    }
    if (mine.old >= 0) {
      scratch_src(c)[my_copy] = mine.old;
      scratch_dst(c)[my_copy] = ids[start[i0 + tid]];
    }
  }
  // new pages: by the sequence's thread where there are a few, by a wave where there are many
  auto take = [&](const Extend& x, int first, int k0, int step) {
    const int have = pages_of(c, x.len), more = x.need - (x.old >= 0);
    for (int k = k0; k < more; k += step) {
      const int p = ids[first + (x.old >= 0) + k];
      c.table[(int64_t)x.s * c.max_pages + have + k] = p;
      c.refs[p] = 1;
    }
  };
  constexpr int kFew = 4;
  for (int i0 = 0; i0 < n; i0 += kThreads) {
    if (n > kThreads) mine = plan(i0 + tid, false);
    const int first = i0 + tid < n ? start[i0 + tid] : 0;
    if (mine.need <= kFew) take(mine, first, 0, 1);
    for (uint64_t many = __ballot(mine.need > kFew); many; many &= many - 1) {
      const int l = __ffsll((unsigned long long)many) - 1;
      const Extend x{__shfl(mine.s, l), __shfl(mine.len, l), 0, __shfl(mine.old, l), __shfl(mine.need, l)};
      take(x, __shfl(first, l), lane, 64);
    }
  }
  __syncthreads();                                         // every last page has been judged by its count
  for (int i = tid; i < (int)copies; i += kThreads) {
    const int old = scratch_src(c)[i];
    if (atomicSub(&c.refs[old], 1) == 1) atomicMin(&freed, old);
    c.refs[scratch_dst(c)[i]] = 1;
  }
  for (int i = tid; i < n; i += kThreads) {
    const int s = seqs[i], len = c.lens[s], count = counts[i];
    if (len % c.page_size && count > 0) {
      // copied, if its new ids are one more than its new pages: the first of them takes the last page's place
      const int have = pages_of(c, len), end = i + 1 < n ? start[i + 1] : (int)need;
      if (end - start[i] > pages_of(c, len + count) - have) c.table[(int64_t)s * c.max_pages + have - 1] = ids[start[i]];
    }
    c.lens[s] = len + count;
  }
  __syncthreads();
  if (tid == 0) {
    c.state[kPairs] = (int)copies;
    c.state[kFirstFree] = min(next_free, freed);
  }
}

// Whole pages: unit = 16 KiB of one page (or what is left of it). Pairs of ids out of range are left out.
constexpr int kCopyThreads = 256;
__device__ void copy_pages(char* pool, const char* from, int64_t page_bytes, int n_pages, int from_pages, const int32_t* src,
                           const int32_t* dst, int n, int block, int blocks) {
  constexpr int kUnitBytes = kCopyThreads * 16 * 4;
  const int64_t per = (page_bytes + kUnitBytes - 1) / kUnitBytes;
  for (int64_t u = block; u < per * n; u += blocks) {
    const int i = (int)(u / per);
    const int a = src[i], b = dst[i];
    if ((uint32_t)a >= (uint32_t)from_pages || (uint32_t)b >= (uint32_t)n_pages) continue;
    const int64_t at = (u % per) * kUnitBytes + threadIdx.x * 16;
    const char* s = from + (int64_t)a * page_bytes;
    char* d = pool + (int64_t)b * page_bytes;
    u32x4 x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (at + k * kCopyThreads * 16 < page_bytes) x[k] = *reinterpret_cast<const u32x4*>(s + at + k * kCopyThreads * 16);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (at + k * kCopyThreads * 16 < page_bytes) *reinterpret_cast<u32x4*>(d + at + k * kCopyThreads * 16) = x[k];
  }
}
__global__ __launch_bounds__(kCopyThreads) void k_copy_pages(char* pool, const char* from, int64_t page_bytes, int n_pages,
                                                             int from_pages, const int32_t* src, const int32_t* dst,
                                                             const int32_t* count, int n) {
  copy_pages(pool, from, page_bytes, n_pages, from_pages, src, dst, count ? *count : n, blockIdx.x, gridDim.x);
}

// Every block checks the whole list, then does its share; lens change only in the block that comes here last, when every
// block has read them. (The count orders those reads before its writes; nothing written by one block is read by another,
// so no fence, whose write-back of the caches costs more than the kernel.) One block alone needs no count.
__device__ bool last_block(int32_t* done) {
  __shared__ int last;
  __syncthreads();
  if (gridDim.x == 1) return true;
  if (threadIdx.x == 0) {
    last = __hip_atomic_fetch_add(done, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
    if (last) __hip_atomic_store(done, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  return last;
}

__global__ __launch_bounds__(kThreads) void k_truncate(const mtc_cache_desc c, const int32_t* seqs, const int32_t* new_lens, int n) {
  __shared__ uint32_t marks[kMarkWords];
  clear_marks(marks);
  __syncthreads();
  int bad = 0;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int s = seqs[i];
    if ((uint32_t)s >= (uint32_t)c.max_seqs || mark(marks, s)) bad |= MTC_CACHE_BAD_SEQ;
    else if (new_lens && (new_lens[i] < 0 || new_lens[i] > held(c, s))) bad |= MTC_CACHE_BAD_LENGTH;
  }
  bad = block_or(bad);
  if (!bad) {
    const int lane = threadIdx.x & 63;
    for (int i = blockIdx.x * kWaves + (threadIdx.x >> 6); i < n; i += gridDim.x * kWaves) {
      const int s = seqs[i], keep = pages_of(c, new_lens ? new_lens[i] : 0), have = pages_of(c, held(c, s));
      int32_t* const row = c.table + (int64_t)s * c.max_pages;
      int lowest = c.n_pages;
      for (int k = keep + lane; k < have; k += 64) {
        const int p = row[k];
        row[k] = -1;
        if ((uint32_t)p < (uint32_t)c.n_pages && atomicSub(&c.refs[p], 1) == 1) lowest = min(lowest, p);
      }
#pragma unroll
      for (int d = 32; d; d >>= 1) lowest = min(lowest, __shfl_xor(lowest, d));
      if (lane == 0 && lowest < c.n_pages) atomicMin(&c.state[kFirstFree], lowest);
    }
  }
  if (!last_block(&c.state[kDone])) return;
  if (!bad)
    for (int i = threadIdx.x; i < n; i += kThreads) c.lens[seqs[i]] = new_lens ? new_lens[i] : 0;
  if (threadIdx.x == 0 && bad) c.state[kStatus] |= bad;
}

__global__ __launch_bounds__(kThreads) void k_fork(const mtc_cache_desc c, const int32_t* src, const int32_t* dst, int n) {
  __shared__ uint32_t targets[kMarkWords];
  clear_marks(targets);
  __syncthreads();
  int bad = 0;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int s = src[i], d = dst[i];
    if ((uint32_t)s >= (uint32_t)c.max_seqs || (uint32_t)d >= (uint32_t)c.max_seqs || mark(targets, d)) bad |= MTC_CACHE_BAD_SEQ;
    else if (c.lens[d] != 0) bad |= MTC_CACHE_NOT_EMPTY;
  }
  bad = block_or(bad);
  if (!bad) {
    int both = 0;
    for (int i = threadIdx.x; i < n; i += kThreads)
      if ((targets[src[i] >> 5] >> (src[i] & 31)) & 1) both = MTC_CACHE_NOT_EMPTY;
    bad = block_or(both);
  }
  if (!bad) {
    const int lane = threadIdx.x & 63;
    for (int i = blockIdx.x * kWaves + (threadIdx.x >> 6); i < n; i += gridDim.x * kWaves) {
      const int have = pages_of(c, held(c, src[i]));
      const int32_t* const from = c.table + (int64_t)src[i] * c.max_pages;
      int32_t* const to = c.table + (int64_t)dst[i] * c.max_pages;
      for (int k = lane; k < have; k += 64) {
        const int p = from[k];
        to[k] = p;
        if ((uint32_t)p < (uint32_t)c.n_pages) atomicAdd(&c.refs[p], 1);
      }
    }
  }
  if (!last_block(&c.state[kDone])) return;
  if (!bad)
    for (int i = threadIdx.x; i < n; i += kThreads) c.lens[dst[i]] = held(c, src[i]);
  if (threadIdx.x == 0 && bad) c.state[kStatus] |= bad;
}

// A block takes a few columns of the table at a time, of all the call's rows: what they held is read before anything is written,
// so that any sequence may take any other's place. Takers are counted before leavers, so that a page that stays held never counts 0.
// Bound by its chain of loads and atomics (list, lengths, table, counts): 4 beams of 8 pages 4.8 us, 256 of up to 58 7.7 us.
constexpr int kReorderIds = MTC_CACHED_MAX_SEQS;
constexpr int kReorderBlocks = 256;
__host__ __device__ inline int reorder_columns(int n) { return min(32, max(1, kThreads / n)); }      // an entry a thread, if they fit
__global__ __launch_bounds__(kThreads) void k_reorder(const mtc_cache_desc c, const int32_t* seqs, const int32_t* parents, int n) {
  __shared__ uint32_t marks[kMarkWords];
  __shared__ int32_t ids[kReorderIds];
  __shared__ int32_t kept_seq[kThreads], kept_from[kThreads], kept_pages[kThreads];      // of the first rows
  __shared__ int longest;
  clear_marks(marks);
  if (threadIdx.x == 0) longest = 0;
  __syncthreads();
  const int columns = reorder_columns(n);
  int bad = 0, most = 0;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int s = seqs[i], from = parents[i];
    int pages = 0;
    if ((uint32_t)s >= (uint32_t)c.max_seqs || mark(marks, s) || (uint32_t)from >= (uint32_t)n) bad = MTC_CACHE_BAD_SEQ;
    else pages = pages_of(c, held(c, s));
    most = max(most, pages);
    if (i < kThreads) {
      kept_seq[i] = s;
      kept_from[i] = from;
      kept_pages[i] = pages;
    }
  }
  most = (int)wave_umax((uint32_t)most);
  if ((threadIdx.x & 63) == 0 && most) atomicMax(&longest, most);
  bad = __syncthreads_or(bad) ? MTC_CACHE_BAD_SEQ : 0;
  most = longest;
  auto seq = [&](int i) { return i < kThreads ? kept_seq[i] : seqs[i]; };
  auto from = [&](int i) { return i < kThreads ? kept_from[i] : parents[i]; };
  for (int first = blockIdx.x * columns; !bad && first < most; first += gridDim.x * columns) {
    __syncthreads();                                       // the last readers of ids
    for (int x = threadIdx.x; x < n * columns; x += kThreads) {
      const int i = x / columns, s = seq(i), k = first + x % columns;
      ids[x] = k < (i < kThreads ? kept_pages[i] : pages_of(c, held(c, s))) ? c.table[(int64_t)s * c.max_pages + k] : -1;
    }
    __syncthreads();
    for (int x = threadIdx.x; x < n * columns; x += kThreads) {
      const int i = x / columns, k = x % columns, p = ids[from(i) * columns + k];
      if (p == ids[x]) continue;
      if ((uint32_t)p < (uint32_t)c.n_pages) atomicAdd(&c.refs[p], 1);
      c.table[(int64_t)seq(i) * c.max_pages + first + k] = p;         // first + k < max_pages: one of the two rows holds it
    }
    __syncthreads();
    int lowest = c.n_pages;
    for (int x = threadIdx.x; x < n * columns; x += kThreads) {
      const int p = ids[x];
      if (p == ids[from(x / columns) * columns + x % columns] || (uint32_t)p >= (uint32_t)c.n_pages) continue;
      if (atomicSub(&c.refs[p], 1) == 1) lowest = min(lowest, p);
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) lowest = min(lowest, __shfl_xor(lowest, d));
    if ((threadIdx.x & 63) == 0 && lowest < c.n_pages) atomicMin(&c.state[kFirstFree], lowest);
  }
  if (!last_block(&c.state[kDone])) return;
  if (!bad) {
    for (int i = threadIdx.x; i < n; i += kThreads) ids[i] = held(c, seq(from(i)));
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) c.lens[seq(i)] = ids[i];
  }
  if (threadIdx.x == 0 && bad) c.state[kStatus] |= bad;
}

// One block; a thread takes four consecutive pages of each round of 4096. A page is held or free (a count below 0 is free),
// so that there are as many free pages below `live` as held ones from there on.
__global__ __launch_bounds__(kThreads) void k_compact_plan(const mtc_cache_desc c) {
  constexpr int kEach = 4;
  const int tid = threadIdx.x;
  auto counts = [&](int64_t p, int (&r)[kEach]) {
#pragma unroll
    for (int k = 0; k < kEach; ++k) r[k] = p + k < c.n_pages ? max(c.refs[p + k], 0) : -1;
  };
  int used = 0, r[kEach];                                // the counts of round 0 stay here where it is the only one
  counts(c.n_pages, r);                                  // threads past the last page: no pages
  for (int64_t p = (int64_t)tid * kEach; p < c.n_pages; p += kThreads * kEach) {
    counts(p, r);
#pragma unroll
    for (int k = 0; k < kEach; ++k) used += r[k] > 0;
  }
  uint64_t total;
  block_scan(used, total);
  const int64_t live = (int64_t)total;
  int64_t movers = 0, holes = 0;
  for (int64_t p0 = 0; p0 < c.n_pages; p0 += kThreads * kEach) {
    const int64_t p = p0 + (int64_t)tid * kEach;
    if (p0 || c.n_pages > kThreads * kEach) counts(p, r);
    uint64_t n = 0;
#pragma unroll
    for (int k = 0; k < kEach; ++k) n += p + k >= live ? (uint64_t)(r[k] > 0) << 32 : (uint64_t)(r[k] == 0);
    const uint64_t at = block_scan(n, total);
    int64_t m = movers + (int64_t)(at >> 32), h = holes + (int64_t)(at & 0xFFFFFFFFu);
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      if (p + k >= live && r[k] > 0) scratch_src(c)[m++] = (int)(p + k);
      if (p + k < live && r[k] == 0) scratch_dst(c)[h++] = (int)(p + k);
    }
    movers += (int64_t)(total >> 32);
    holes += (int64_t)(total & 0xFFFFFFFFu);
  }
  __syncthreads();
  for (int64_t i = tid; i < movers; i += kThreads) {
    const int a = scratch_src(c)[i], b = scratch_dst(c)[i];
    scratch_ids(c)[a] = b;                                 // where page a went; read for ids from `live` on only
    c.refs[b] = c.refs[a];
    c.refs[a] = 0;
  }
  if (tid == 0) {
    c.state[kPairs] = (int)movers;
    c.state[kFirstFree] = (int)live;
  }
}

// The first blocks rename the moved pages in the table, the others copy them.
__global__ __launch_bounds__(kCopyThreads) void k_compact(const mtc_cache_desc c, int64_t page_bytes, int table_blocks) {
  if ((int)blockIdx.x >= table_blocks) {
    copy_pages((char*)c.pool, (const char*)c.pool, page_bytes, c.n_pages, c.n_pages, scratch_src(c), scratch_dst(c), c.state[kPairs],
               blockIdx.x - table_blocks, gridDim.x - table_blocks);
    return;
  }
  const int live = c.state[kFirstFree], lane = threadIdx.x & 63;
  for (int s = blockIdx.x * 4 + (threadIdx.x >> 6); s < c.max_seqs; s += table_blocks * 4) {
    const int have = pages_of(c, held(c, s));
    int32_t* const row = c.table + (int64_t)s * c.max_pages;
    for (int k = lane; k < have; k += 64) {
      const int p = row[k];
      if (p >= live && p < c.n_pages) row[k] = scratch_ids(c)[p];
    }
  }
}

// One thread per 8 elements of K or V: each finds its row's sequence by bisection (64 rows: 4.4 us, the chain of loads).
template <bool BF, bool F32>
__global__ __launch_bounds__(256) void k_append(const mtc_cache_desc c, int layer, const mtc_heads k, const mtc_heads v, int rows,
                                                const int32_t* seqs, const int32_t* cu, int n) {
  const int pieces = c.dim / 8;
  const int64_t per_row = 2ll * c.kv_heads * pieces;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= per_row * rows) return;
  const int r = (int)(i / per_row), in = (int)(i % per_row);
  const int piece = in % pieces, h = in / pieces % c.kv_heads, is_v = in / pieces / c.kv_heads;
  if (cu[0] > r || cu[n] <= r) return;
  int lo = 0, hi = n;                                     // cu[lo] <= r < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= r) lo = mid; else hi = mid;
  }
  const int s = seqs[lo];
  if ((uint32_t)s >= (uint32_t)c.max_seqs) return;
  const int pos = held(c, s) - (cu[lo + 1] - r);
  if (pos < 0 || pos >= c.max_pages * c.page_size) return;
  const int page = c.table[(int64_t)s * c.max_pages + pos / c.page_size];
  if ((uint32_t)page >= (uint32_t)c.n_pages) return;
  const mtc_heads& x = is_v ? v : k;
  const int64_t from = (int64_t)r * x.row_stride + (int64_t)h * x.head_stride + piece * 8;
  u32x4 y;
  if constexpr (F32) {
    const f32x4* p = reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(x.data) + from);
    const f32x4 a = p[0], b = p[1];
    using E = Elem<BF>;
    y = u32x4{E::pack(a[0], a[1]), E::pack(a[2], a[3]), E::pack(b[0], b[1]), E::pack(b[2], b[3])};
  } else {
    y = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(x.data) + from);
  }
  const int64_t to = ((((int64_t)page * c.n_layers + layer) * 2 + is_v) * c.kv_heads + h) * c.page_size + pos % c.page_size;
  *reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(c.pool) + to * c.dim + piece * 8) = y;
}

// ---------------------------------------------------------------------------
// the 8-bit cache
// ---------------------------------------------------------------------------
// Byte offsets, within a page, of the codes of token 0 and of the scales of block 0 of (layer, K or V, head).
__device__ __forceinline__ int64_t codes_at(const mtc_cache_desc& c, int layer, int is_v, int h) {
  return (((int64_t)layer * 2 + is_v) * c.kv_heads + h) * c.page_size * codes::row_bytes(c.dim);
}
__device__ __forceinline__ int64_t scales_at(const mtc_cache_desc& c, int layer, int is_v, int h) {
  return codes::code_bytes(c) + (((int64_t)layer * 2 + is_v) * c.kv_heads + h) * (c.page_size / codes::kBlock) * 2;
}

// 16 elements of a row from `d` on, as they lie in memory (those past dim are 0), and in fp32.
template <int SRC>
struct Row16 {
  u32x4 raw[SRC == MTC_DTYPE_F32 ? 4 : 2];
  __device__ __forceinline__ void load(const mtc_heads& x, int64_t row, int h, int d, int dim) {
    const int64_t at = row * x.row_stride + (int64_t)h * x.head_stride + d;
    constexpr int kEach = SRC == MTC_DTYPE_F32 ? 4 : 8;    // elements of 16 bytes
    const char* const p = (const char*)x.data + at * (16 / kEach);
#pragma unroll
    for (int i = 0; i < 16 / kEach; ++i)
      raw[i] = d + i * kEach < dim ? *reinterpret_cast<const u32x4*>(p + i * 16) : u32x4{0, 0, 0, 0};
  }
  __device__ __forceinline__ float operator[](int j) const {
    if constexpr (SRC == MTC_DTYPE_F32) {
      const uint32_t u = raw[j >> 2][j & 3];
      return __builtin_bit_cast(float, u);
    } else {
      return Elem<SRC == MTC_DTYPE_BF16>::widen((uint16_t)(raw[j >> 3][j >> 1 & 3] >> (16 * (j & 1))));
    }
  }
  // fp32 bits of the largest magnitude (as whole numbers these are in the order of the magnitudes, NaN last).
  __device__ __forceinline__ uint32_t top() const {
    if constexpr (SRC == MTC_DTYPE_F32) {
      uint32_t t = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) t = max(t, raw[i >> 2][i & 3] & 0x7FFFFFFFu);
      return t;
    } else {
      typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
      u16x2 t = {0, 0};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t u = raw[i >> 2][i & 3] & 0x7FFF7FFFu;
        t = __builtin_elementwise_max(t, __builtin_bit_cast(u16x2, u));
      }
      const uint16_t m = t[0] > t[1] ? t[0] : t[1];
      return __builtin_bit_cast(uint32_t, Elem<SRC == MTC_DTYPE_BF16>::widen(m));
    }
  }
};
// Four codes of values from `from` on, times a power of two, rounded to nearest even. Added to 1.5 2^23, a number up to 2^22 in
// magnitude is rounded to a whole one whose lowest byte is the code: one fused multiply-add (the product is exact).
template <class Y>
__device__ __forceinline__ uint32_t pack_codes(const Y& y, int from, float by) {
  uint32_t u[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) u[j] = __builtin_bit_cast(uint32_t, __builtin_fmaf(y[from + j], by, 12582912.0f));
  const uint32_t lo = __builtin_amdgcn_perm(u[1], u[0], 0x0C0C0400u), hi = __builtin_amdgcn_perm(u[3], u[2], 0x0C0C0400u);
  return lo | hi << 16;
}
// The same for any values: cut at 127, NaN to 0.
template <class Y>
__device__ __forceinline__ uint32_t pack_any(const Y& y, int from, float by) {
  uint32_t r = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float v = y[from + j] * by;
    const int q = v == v ? (int)__builtin_rintf(fminf(fmaxf(v, -127.0f), 127.0f)) : 0;
    r |= (uint32_t)(q & 0xFF) << (8 * j);
  }
  return r;
}

__device__ __forceinline__ int cut(const int32_t* cu, int i, int rows) { return min(max(cu[i], 0), rows); }

// A wave per block of 16 tokens that gets new ones, K or V, and head: the whole block is in its lanes (16 bytes each, twice at
// most), so its largest value, and the older codes' rounding to a larger scale, need one exchange and no second pass.
// Which block: sequence i's blocks have the numbers from cu[i] / 16 + 2 i on. It has at most rows / 16 + 2, so that
// numbers of two never meet, and a bisection of cu finds the sequence. The new rows, and the block's old codes and scale, are on
// their way while the list and the page's holders are checked.
// 16384 tokens of 8 heads of 128 (67 MB bf16 in, 34 MB out) 20.8 us, 4.8 TB/s; one token of 64 sequences 6.6 us, the chain of loads.
template <bool BF, int SRC>
__global__ __launch_bounds__(256) void k_append8(const mtc_cache_desc c, int layer, const mtc_heads k, const mtc_heads v, int rows,
                                                 const int32_t* seqs, const int32_t* cu, int n) {
  using namespace codes;
  const int u = blockIdx.x, lane = threadIdx.x & 63;
  auto start = [&](int i) { return cut(cu, i, rows) / kBlock + 2 * i; };
  int lo = 0, hi = n;                                      // start(lo) <= u < start(hi)
  if (start(0) > u || start(n) <= u) return;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start(mid) <= u) lo = mid; else hi = mid;
  }
  const int r0 = cut(cu, lo, rows), count = cut(cu, lo + 1, rows) - r0, s = seqs[lo];
  if (count <= 0 || (uint32_t)s >= (uint32_t)c.max_seqs) return;
  const int len = held(c, s), p0 = max(len - count, 0), skip = max(count - len, 0);     // rows before token 0
  const int block = p0 / kBlock + (u - start(lo));
  if (block * kBlock >= len) return;
  const int at = block * kBlock, room = row_bytes(c.dim), pieces = room / 16;
  const int page = c.table[(int64_t)s * c.max_pages + at / c.page_size];
  if ((uint32_t)page >= (uint32_t)c.n_pages) return;
  char* const base = (char*)c.pool + (int64_t)page * page_bytes(c);
  const int in = at % c.page_size;
  const bool older = at < p0;
  int token[2];                                            // of this lane's two pieces; len: none
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int chunk = lane + 64 * x;
    token[x] = chunk < room ? at + chunk / pieces : len;
  }
  auto codes_of = [&](int item) { return reinterpret_cast<u32x4*>(base + codes_at(c, layer, item & 1, item >> 1) + (int64_t)in * room); };
  auto scale_at = [&](int item) { return reinterpret_cast<uint16_t*>(base + scales_at(c, layer, item & 1, item >> 1)) + in / kBlock; };
  Row16<SRC> y[2];                                         // a new token's elements, or an older one's codes (in raw[0])
  uint16_t old_scale = 0;
  auto load = [&](int item) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int chunk = lane + 64 * x;
      if (token[x] >= len) continue;
      if (token[x] >= p0) y[x].load(item & 1 ? v : k, r0 + skip + token[x] - p0, item >> 1, chunk % pieces * 16, c.dim);
      else y[x].raw[0] = codes_of(item)[chunk];
    }
    if (older) old_scale = *scale_at(item);
  };
  const int first = blockIdx.y * 4 + (threadIdx.x >> 6), step = gridDim.y * 4;
  if (first < 2 * c.kv_heads) load(first);
  int twice = 0;
  for (int j = threadIdx.x; j < n; j += 256) twice |= j != lo && seqs[j] == s && cut(cu, j + 1, rows) > cut(cu, j, rows);
  twice = __syncthreads_or(twice);
  const bool shared = c.refs[page] > 1;
  if (twice || shared) {
    if (threadIdx.x == 0) atomicOr(&c.state[kStatus], (twice ? MTC_CACHE_BAD_SEQ : 0) | (shared ? MTC_CACHE_SHARED_PAGE : 0));
    return;
  }
  for (int item = first; item < 2 * c.kv_heads; item += step) {
    u32x4* const to = codes_of(item);
    const int was = older ? exponent_of<BF>(old_scale) : Range<BF>::lo;
    uint32_t bits = 0;                                     // of the largest magnitude; not less than infinity's: one is not finite
#pragma unroll
    for (int x = 0; x < 2; ++x)
      if (token[x] >= p0 && token[x] < len) bits = max(bits, y[x].top());
    bits = wave_umax(bits);
    float top = __builtin_bit_cast(float, bits);
    const bool wild = bits >= 0x7F800000u;
    if (wild) {                                            // the largest finite one
      top = 0.0f;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (token[x] < p0 || token[x] >= len) continue;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float a = fabsf(y[x][j]);
          top = fmaxf(top, a < INFINITY ? a : 0.0f);
        }
      }
      top = wave_max(top);
    }
    const int e = max(was, exponent_for<BF>(top));
    if (lane == 0) *scale_at(item) = (uint16_t)((e + 127) << 7);
    const float by = power(-e);
    const bool cut_off = wild || top > 127.0f * power(Range<BF>::hi);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      if (token[x] >= len) continue;
      u32x4 z;
      if (token[x] >= p0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) z[i] = cut_off ? pack_any(y[x], 4 * i, by) : pack_codes(y[x], 4 * i, by);
      } else if (e > was) {
        const float less = e - was > 40 ? 0.0f : power(was - e);           // codes below 2^7: nothing of them is left
        z = y[x].raw[0];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t w = z[i];
          const float o[4] = {(float)(int8_t)w, (float)(int8_t)(w >> 8), (float)(int8_t)(w >> 16), (float)(int8_t)(w >> 24)};
          z[i] = pack_codes(o, 0, less);
        }
      } else {
        continue;
      }
      to[lane + 64 * x] = z;
    }
    if (item + step < 2 * c.kv_heads) load(item + step);
  }
}

// One thread per 16 codes: each finds its row's sequence by bisection (counted by the block in one round of loads instead: 25 us for
// the first of these). 16384 tokens of 8 heads of 128 (34 MB in, 67 MB bf16 out) 22 us, 4.6 TB/s; 32 tokens of 64 sequences 5.9 us.
template <bool BF, int DST>
__global__ __launch_bounds__(256) void k_read8(const mtc_cache_desc c, int layer, const mtc_heads k, const mtc_heads v, int rows,
                                               const int32_t* seqs, const int32_t* cu, int n) {
  using namespace codes;
  const int room = row_bytes(c.dim), pieces = room / 16;
  const int64_t per_row = 2ll * c.kv_heads * pieces;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= per_row * rows) return;
  const int r = (int)(i / per_row), in = (int)(i % per_row);
  const int piece = in % pieces, h = in / pieces % c.kv_heads, is_v = in / pieces / c.kv_heads;
  if (cut(cu, 0, rows) > r || cut(cu, n, rows) <= r) return;
  int lo = 0, hi = n;                                      // cu[lo] <= r < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cut(cu, mid, rows) <= r) lo = mid; else hi = mid;
  }
  const int s = seqs[lo];
  u32x4 z{};
  float scale = 0.0f;
  if ((uint32_t)s < (uint32_t)c.max_seqs) {
    const int pos = held(c, s) - (cut(cu, lo + 1, rows) - r);
    if (pos >= 0 && pos < c.max_pages * c.page_size) {
      const int page = c.table[(int64_t)s * c.max_pages + pos / c.page_size];
      if ((uint32_t)page < (uint32_t)c.n_pages) {
        const char* const base = (const char*)c.pool + (int64_t)page * page_bytes(c);
        const int p = pos % c.page_size;
        z = *reinterpret_cast<const u32x4*>(base + codes_at(c, layer, is_v, h) + (int64_t)p * room + piece * 16);
        scale = scale_of<BF>(reinterpret_cast<const uint16_t*>(base + scales_at(c, layer, is_v, h))[p / kBlock]);
      }
    }
  }
  const mtc_heads& x = is_v ? v : k;
  const int64_t to = (int64_t)r * x.row_stride + (int64_t)h * x.head_stride + piece * 16;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    if (piece * 16 + half * 8 >= c.dim) break;
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t w = z[2 * half + (j >> 2)];
      y[j] = (float)(int8_t)(w >> (8 * (j & 3))) * scale;
    }
    if constexpr (DST == MTC_DTYPE_F32) {
      f32x4* p = reinterpret_cast<f32x4*>(reinterpret_cast<float*>(x.data) + to + half * 8);
      p[0] = f32x4{y[0], y[1], y[2], y[3]};
      p[1] = f32x4{y[4], y[5], y[6], y[7]};
    } else {
      using E = Elem<BF>;
      *reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(x.data) + to + half * 8) =
          u32x4{E::pack(y[0], y[1]), E::pack(y[2], y[3]), E::pack(y[4], y[5]), E::pack(y[6], y[7])};
    }
  }
}

// ---------------------------------------------------------------------------
// verification of drafted tokens
// ---------------------------------------------------------------------------
constexpr int kVerifyThreads = 256;
constexpr int kMaxDrafted = 64;

struct Best {
  float rest, all;                 // largest score over w = max(p - q, 0) (or p where nothing was rejected), and over p
  int32_t rest_i, all_i;           // its first index, -1: none
};
struct Found {                     // of one block
  Best best;
  int32_t accepted, reserved[3];
};
constexpr float kNoScore = -1.0f;  // below every score of a w > 0
// Without branches: of 16 elements a thread, each would be taken by some lane.
__device__ __forceinline__ void better(float& a, int32_t& ai, float b, int32_t bi) {
  const bool take = b > a || (b == a && (uint32_t)bi < (uint32_t)ai);
  a = take ? b : a;
  ai = take ? bi : ai;
}

template <int DT>
struct Prob;
template <>
struct Prob<MTC_DTYPE_F32> {
  typedef float type;
  static __device__ __forceinline__ float get(float x) { return x; }
};
template <>
struct Prob<MTC_DTYPE_BF16> {
  typedef uint16_t type;
  static __device__ __forceinline__ float get(uint16_t x) { return Elem<true>::widen(x); }
};
template <>
struct Prob<MTC_DTYPE_F16> {
  typedef uint16_t type;
  static __device__ __forceinline__ float get(uint16_t x) { return Elem<false>::widen(x); }
};

// 8 elements from an address of the element's alignment only.
template <class T>
struct __attribute__((packed, aligned(sizeof(T)))) Eight {
  T x[8];
};

__device__ __forceinline__ int64_t draft_at(const mtc_verify_args& a, int b, int j) {
  const int64_t i = (int64_t)b * a.drafts_stride + j;
  return a.index_bytes == 8 ? reinterpret_cast<const int64_t*>(a.drafts)[i] : reinterpret_cast<const int32_t*>(a.drafts)[i];
}

// Accepted drafts of sequence b (every lane of the wave gets it); k: its drafts.
template <int DT>
__device__ int accepted(const mtc_verify_args& a, int b, int& k) {
  typedef typename Prob<DT>::type T;
  const int j = threadIdx.x & 63;
  const int64_t x = j < a.n_drafted ? draft_at(a, b, j) : -1;
  const float u = j < a.n_drafted ? a.u[(int64_t)b * a.u_stride + j] : 0.0f;
  k = a.n_drafts ? min(max(a.n_drafts[b], 0), a.n_drafted) : a.n_drafted;
  float p = 0.0f, q = 0.0f;        // outside the vocabulary: never accepted
  if (x >= 0 && x < a.vocab) {
    p = Prob<DT>::get(reinterpret_cast<const T*>(a.p)[(int64_t)b * a.p_stride[0] + (int64_t)j * a.p_stride[1] + x]);
    q = Prob<DT>::get(reinterpret_cast<const T*>(a.q)[(int64_t)b * a.q_stride[0] + (int64_t)j * a.q_stride[1] + x]);
  }
  const bool good = j >= k || u * q < p;           // past the last draft: k ends the run below
  const uint64_t wrong = __ballot(!good);
  return wrong ? __ffsll((unsigned long long)wrong) - 1 : k;
}

// One block per sequence and span of the vocabulary, one pass: the scores of both candidates for w (what is left of p,
// and p itself, should nothing be left) are kept, so no second look at the row is needed. Bound by memory and the chain
// before it: 64 x 7 drafts, 128003 bf16 probabilities, 54 MB in 15 us (the chain and launch: about 5). The noise does not depend on how many drafts were accepted, so its
// loads are in flight while that chain of dependent loads (drafts, their probabilities) is followed.
template <int DT, int ROUNDS>
__global__ __launch_bounds__(kVerifyThreads) void k_verify(const mtc_verify_args a, Found* found) {
  typedef typename Prob<DT>::type T;
  using P = Prob<DT>;
  constexpr int kSpan = kVerifyThreads * 8;
  const int b = blockIdx.y, tid = threadIdx.x;
  const float* e = a.noise + (int64_t)b * a.noise_stride;
  const int from = blockIdx.x * (ROUNDS * kSpan) + tid * 8;
  Eight<float> ev[ROUNDS];
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r)
    if (from + r * kSpan + 8 <= a.vocab) ev[r] = *reinterpret_cast<const Eight<float>*>(e + from + r * kSpan);
  int k;
  const int n = accepted<DT>(a, b, k);
  const bool minus = n < k;
  const T* p = reinterpret_cast<const T*>(a.p) + (int64_t)b * a.p_stride[0] + (int64_t)n * a.p_stride[1];
  const T* q = minus ? reinterpret_cast<const T*>(a.q) + (int64_t)b * a.q_stride[0] + (int64_t)n * a.q_stride[1] : p;
  Best best{kNoScore, kNoScore, -1, -1};
  auto one = [&](int i, float w, float d, float z) {       // i ascends in a thread: the first of equals stays
    const float all = w > 0.0f ? w * z : kNoScore, rest = d > 0.0f ? d * z : kNoScore;
    const bool x = all > best.all, y = rest > best.rest;
    best.all = x ? all : best.all;
    best.all_i = x ? i : best.all_i;
    best.rest = y ? rest : best.rest;
    best.rest_i = y ? i : best.rest_i;
  };
  Eight<T> pv[ROUNDS], qv[ROUNDS];
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int i = from + r * kSpan;
    if (i + 8 <= a.vocab) {
      pv[r] = *reinterpret_cast<const Eight<T>*>(p + i);
      if (minus) qv[r] = *reinterpret_cast<const Eight<T>*>(q + i);
    }
  }
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int i = from + r * kSpan;
    if (i + 8 <= a.vocab) {
#pragma unroll
      for (int j = 0; j < 8; ++j) one(i + j, P::get(pv[r].x[j]), minus ? P::get(pv[r].x[j]) - P::get(qv[r].x[j]) : 0.0f, ev[r].x[j]);
    } else {
      for (int j = i; j < a.vocab; ++j) one(j, P::get(p[j]), minus ? P::get(p[j]) - P::get(q[j]) : 0.0f, e[j]);
    }
  }
  auto fold = [&]() {
#pragma unroll
    for (int d = 32; d; d >>= 1) {
      better(best.rest, best.rest_i, __shfl_xor(best.rest, d), __shfl_xor(best.rest_i, d));
      better(best.all, best.all_i, __shfl_xor(best.all, d), __shfl_xor(best.all_i, d));
    }
  };
  fold();
  __shared__ Best waves[kVerifyThreads / 64];
  if ((tid & 63) == 0) waves[tid >> 6] = best;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kVerifyThreads / 64; ++w) {
      better(best.rest, best.rest_i, waves[w].rest, waves[w].rest_i);
      better(best.all, best.all_i, waves[w].all, waves[w].all_i);
    }
    found[(int64_t)b * gridDim.x + blockIdx.x] = Found{best, n, {0, 0, 0}};
  }
}

__global__ __launch_bounds__(64) void k_verify_join(const mtc_verify_args a, const Found* found, int splits) {
  const int b = blockIdx.x, lane = threadIdx.x;
  const int n = found[(int64_t)b * splits].accepted;
  Best r{kNoScore, kNoScore, -1, -1};
  for (int i = lane; i < splits; i += 64) {
    const Best x = found[(int64_t)b * splits + i].best;
    better(r.rest, r.rest_i, x.rest, x.rest_i);
    better(r.all, r.all_i, x.all, x.all_i);
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    better(r.rest, r.rest_i, __shfl_xor(r.rest, d), __shfl_xor(r.rest_i, d));
    better(r.all, r.all_i, __shfl_xor(r.all, d), __shfl_xor(r.all_i, d));
  }
  const int next = r.rest_i >= 0 ? r.rest_i : r.all_i;
  for (int j = lane; j <= a.n_drafted; j += 64) {
    const int64_t t = j < n ? draft_at(a, b, j) : j == n ? next : -1;
    const int64_t at = (int64_t)b * (a.n_drafted + 1) + j;
    if (a.index_bytes == 8) reinterpret_cast<int64_t*>(a.tokens)[at] = t;
    else reinterpret_cast<int32_t*>(a.tokens)[at] = (int32_t)t;
  }
  if (lane == 0) a.accepted[b] = n;
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
int64_t page_bytes(const mtc_cache_desc* c) {
  return codes::is_codes(*c) ? codes::page_bytes(*c) : 2ll * c->n_layers * 2 * c->kv_heads * c->page_size * c->dim;
}

// Blocks that keep every CU's loads in flight, or one per unit of the most pages that may move.
unsigned copy_grid(const mtc_cache_desc* c, int64_t pages) {
  const int64_t units = (page_bytes(c) + kCopyThreads * 64 - 1) / (kCopyThreads * 64) * pages;
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>(units, 4096));
}

int check_list(const mtc_cache_desc* c, const int32_t* a, const char* what, int n) {
  if (int rc = mtc_check_cache_desc(c)) return rc;
  if (n < 0 || n > MTC_CACHED_MAX_SEQS) return fail(MTC_E_SHAPE, "%d sequences: 0 to %d", n, MTC_CACHED_MAX_SEQS);
  if (n && !a) return fail(MTC_E_NULL, "%s is NULL", what);
  return MTC_OK;
}

// The checks of append and read.
int check_rows(const mtc_cache_desc* c, int layer, const mtc_heads* k, const mtc_heads* v, int dtype, int rows, const int32_t* seqs,
               const int32_t* cu, int n) {
  if (int rc = check_list(c, seqs, "seqs", n)) return rc;
  if (layer < 0 || layer >= c->n_layers) return fail(MTC_E_SHAPE, "layer %d of %d", layer, c->n_layers);
  if (dtype != MTC_DTYPE_F32 && dtype != codes::base_type(*c)) return fail(MTC_E_DTYPE, "k and v of dtype %d, a cache of %d", dtype, c->dtype);
  if (rows < 0) return fail(MTC_E_SHAPE, "%d rows", rows);
  if (n == 0 || rows == 0) return MTC_OK;
  if (!cu || !k || !v || !k->data || !v->data) return fail(MTC_E_NULL, "k, v or cu is NULL");
  const int align = dtype == MTC_DTYPE_F32 ? 4 : 8;
  for (const mtc_heads* x : {k, v})
    if ((uintptr_t)x->data % 16 || x->row_stride % align || x->head_stride % align)
      return fail(MTC_E_SHAPE, "k and v: 16-byte aligned, strides multiples of 16 bytes");
  return MTC_OK;
}

unsigned list_grid(int n) { return (unsigned)std::min((n + kWaves - 1) / kWaves, 256); }

// Two rounds of a block's loads per block once that still gives every CU several blocks, else one.
int verify_rounds(const mtc_verify_args* a) { return (int64_t)a->n_seqs * a->vocab >= (4 << 20) ? 2 : 1; }
int verify_splits(const mtc_verify_args* a) {
  const int span = kVerifyThreads * 8 * verify_rounds(a);
  return (a->vocab + span - 1) / span;
}

int check_verify(const mtc_verify_args* a) {
  if (!a) return fail(MTC_E_NULL, "args is NULL");
  if (a->abi_version != MTC_ABI_VERSION) return fail(MTC_E_VERSION, "args of ABI %u, library %d", a->abi_version, MTC_ABI_VERSION);
  if (a->dtype != MTC_DTYPE_F32 && a->dtype != MTC_DTYPE_BF16 && a->dtype != MTC_DTYPE_F16)
    return fail(MTC_E_DTYPE, "probabilities of dtype %d", a->dtype);
  if (a->index_bytes != 4 && a->index_bytes != 8) return fail(MTC_E_DTYPE, "tokens of %d bytes: 4 or 8", a->index_bytes);
  if (a->n_seqs < 0 || a->n_seqs > 65535) return fail(MTC_E_SHAPE, "%d sequences: 0 to 65535", a->n_seqs);
  if (a->n_drafted < 0 || a->n_drafted > kMaxDrafted) return fail(MTC_E_SHAPE, "%d drafts: 0 to %d", a->n_drafted, kMaxDrafted);
  if (a->vocab < 1 || a->vocab > 0x3FFFFFFF) return fail(MTC_E_SHAPE, "vocabulary of %d", a->vocab);
  if ((int64_t)verify_splits(a) * a->n_seqs > 0xFFFFFF)                                    // 2^32 threads a launch
    return fail(MTC_E_SHAPE, "%d sequences of a vocabulary of %d: too many", a->n_seqs, a->vocab);
  return MTC_OK;
}

template <int DT>
int run_verify(const mtc_verify_args& a, Found* found, hipStream_t st) {
  const int splits = verify_splits(&a);
  const dim3 grid(splits, a.n_seqs);
  if (verify_rounds(&a) == 2) k_verify<DT, 2><<<grid, kVerifyThreads, 0, st>>>(a, found);
  else k_verify<DT, 1><<<grid, kVerifyThreads, 0, st>>>(a, found);
  if (int rc = check_launch("k_verify")) return rc;
  k_verify_join<<<a.n_seqs, 64, 0, st>>>(a, found, splits);
  return check_launch("k_verify_join");
}

}  // namespace

MTC_API int mtc_check_cache_desc(const mtc_cache_desc* c) {
  if (!c) return fail(MTC_E_NULL, "cache descriptor is NULL");
  if (c->abi_version != MTC_ABI_VERSION) return fail(MTC_E_VERSION, "cache descriptor of ABI %u, library %d", c->abi_version, MTC_ABI_VERSION);
  const int type = codes::base_type(*c);
  if (type != MTC_DTYPE_BF16 && type != MTC_DTYPE_F16) return fail(MTC_E_DTYPE, "a cache holds bf16 or f16, or codes of them, got dtype %d", c->dtype);
  if (c->n_pages < 1 || c->n_layers < 1 || c->kv_heads < 1 || c->max_seqs < 1 || c->max_pages < 1 || c->reserved != 0)
    return fail(MTC_E_DESC, "cache of %d pages, %d layers, %d heads, %d sequences of %d pages", c->n_pages, c->n_layers, c->kv_heads,
                c->max_seqs, c->max_pages);
  if (c->dim < 8 || c->dim > MTC_ATTN_MAX_DIM || c->dim % 8)
    return fail(MTC_E_DESC, "head size %d: a multiple of 8 from 8 to %d", c->dim, MTC_ATTN_MAX_DIM);
  if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
    return fail(MTC_E_DESC, "page size %d: a power of two from 16 to 256", c->page_size);
  if (c->max_seqs > MTC_CACHE_MAX_SLOTS) return fail(MTC_E_DESC, "%d sequences, at most %d", c->max_seqs, MTC_CACHE_MAX_SLOTS);
  if (c->n_pages > 0x1FFFFFFF || (int64_t)c->max_pages * c->page_size > 0x3FFFFFFF)
    return fail(MTC_E_DESC, "%d pages, %d of %d tokens per sequence: too many", c->n_pages, c->max_pages, c->page_size);
  if (2ll * c->kv_heads * c->page_size * c->dim * 2 * c->n_layers > (1ll << 40)) return fail(MTC_E_DESC, "pages are too large");
  if (!c->pool || !c->table || !c->lens || !c->refs || !c->state || !c->scratch) return fail(MTC_E_NULL, "a cache array is NULL");
  if ((uintptr_t)c->pool % 16) return fail(MTC_E_DESC, "the pool must be 16-byte aligned");
  return ok();
}

MTC_API size_t mtc_cache_scratch_ints(int n_pages, int max_seqs) {
  if (n_pages < 1 || max_seqs < 1) return 0;
  return 3 * (size_t)n_pages + std::min(max_seqs, MTC_CACHED_MAX_SEQS);
}

MTC_API int mtc_cache_extend(const mtc_cache_desc* c, const int32_t* seqs, const int32_t* counts, int n, void* hip_stream) {
  if (int rc = check_list(c, seqs, "seqs", n)) return rc;
  if (n == 0) return ok();
  if (!counts) return fail(MTC_E_NULL, "counts is NULL");
  if (n > c->max_seqs) return fail(MTC_E_SHAPE, "%d sequences, the cache holds %d", n, c->max_seqs);
  hipStream_t st = (hipStream_t)hip_stream;
  k_extend<<<1, kThreads, 0, st>>>(*c, seqs, counts, n);
  if (int rc = check_launch("k_extend")) return rc;
  k_copy_pages<<<copy_grid(c, n), kCopyThreads, 0, st>>>((char*)c->pool, (const char*)c->pool, page_bytes(c), c->n_pages, c->n_pages,
                                                         scratch_src(*c), scratch_dst(*c), c->state + kPairs, 0);
  return check_launch("k_copy_pages");
}

MTC_API int mtc_cache_fork(const mtc_cache_desc* c, const int32_t* src, const int32_t* dst, int n, void* hip_stream) {
  if (int rc = check_list(c, src, "src", n)) return rc;
  if (n == 0) return ok();
  if (!dst) return fail(MTC_E_NULL, "dst is NULL");
  k_fork<<<list_grid(n), kThreads, 0, (hipStream_t)hip_stream>>>(*c, src, dst, n);
  return check_launch("k_fork");
}

MTC_API int mtc_cache_reorder(const mtc_cache_desc* c, const int32_t* seqs, const int32_t* parents, int n, void* hip_stream) {
  if (int rc = check_list(c, seqs, "seqs", n)) return rc;
  if (n == 0) return ok();
  if (!parents) return fail(MTC_E_NULL, "parents is NULL");
  const int columns = reorder_columns(n);
  k_reorder<<<std::min((c->max_pages + columns - 1) / columns, kReorderBlocks), kThreads, 0, (hipStream_t)hip_stream>>>(*c, seqs, parents, n);
  return check_launch("k_reorder");
}

MTC_API int mtc_cache_truncate(const mtc_cache_desc* c, const int32_t* seqs, const int32_t* new_lens, int n, void* hip_stream) {
  if (int rc = check_list(c, seqs, "seqs", n)) return rc;
  if (n == 0) return ok();
  k_truncate<<<list_grid(n), kThreads, 0, (hipStream_t)hip_stream>>>(*c, seqs, new_lens, n);
  return check_launch("k_truncate");
}

MTC_API int mtc_cache_compact(const mtc_cache_desc* c, void* hip_stream) {
  if (int rc = mtc_check_cache_desc(c)) return rc;
  hipStream_t st = (hipStream_t)hip_stream;
  k_compact_plan<<<1, kThreads, 0, st>>>(*c);
  if (int rc = check_launch("k_compact_plan")) return rc;
  const int table_blocks = std::min((c->max_seqs + 3) / 4, 256);
  k_compact<<<table_blocks + copy_grid(c, c->n_pages / 2 + 1), kCopyThreads, 0, st>>>(*c, page_bytes(c), table_blocks);
  return check_launch("k_compact");
}

MTC_API int mtc_cache_copy_pages(const mtc_cache_desc* c, const void* from_pool, int from_pages, const int32_t* src,
                                 const int32_t* dst, int n, void* hip_stream) {
  if (int rc = mtc_check_cache_desc(c)) return rc;
  if (n < 0) return fail(MTC_E_SHAPE, "%d pages", n);
  if (n == 0) return ok();
  if (!from_pool || !src || !dst) return fail(MTC_E_NULL, "from_pool, src or dst is NULL");
  if (from_pages < 1 || (uintptr_t)from_pool % 16) return fail(MTC_E_SHAPE, "from_pool: %d pages, 16-byte aligned", from_pages);
  k_copy_pages<<<copy_grid(c, n), kCopyThreads, 0, (hipStream_t)hip_stream>>>((char*)c->pool, (const char*)from_pool, page_bytes(c),
                                                                              c->n_pages, from_pages, src, dst, nullptr, n);
  return check_launch("k_copy_pages");
}

MTC_API int mtc_cache_append(const mtc_cache_desc* c, int layer, const mtc_heads* k, const mtc_heads* v, int src_dtype, int rows,
                             const int32_t* seqs, const int32_t* cu, int n, void* hip_stream) {
  if (int rc = check_rows(c, layer, k, v, src_dtype, rows, seqs, cu, n)) return rc;
  if (n == 0 || rows == 0) return ok();
  hipStream_t st = (hipStream_t)hip_stream;
  const bool bf = codes::base_type(*c) == MTC_DTYPE_BF16, f32 = src_dtype == MTC_DTYPE_F32;
  if (codes::is_codes(*c)) {
    const int64_t units = (int64_t)rows / codes::kBlock + 2 * n;
    // one item a wave, but where the blocks fill the chip already: each reads the list of sequences. Measured with a read of the newest
    // tokens, one and several items a wave: 8 heads of 128, 64 sequences of 1 token 9.5, 12.1 us; 64 of 100 17.8, 18.2; 512 of 1 23.4, 20.8; 1
    // of 16384 24.5, 22.9; 64 of 512 55.4, 51.3
    const int items = (2 * c->kv_heads + 3) / 4;
    if (units > 0xFFFFFF / items || items > 0xFFFF) return fail(MTC_E_SHAPE, "%d rows of %d heads: too many", rows, c->kv_heads);
    const dim3 g((unsigned)units, units < 1024 ? items : 1);
    if (bf && f32) k_append8<true, MTC_DTYPE_F32><<<g, 256, 0, st>>>(*c, layer, *k, *v, rows, seqs, cu, n);
    else if (bf) k_append8<true, MTC_DTYPE_BF16><<<g, 256, 0, st>>>(*c, layer, *k, *v, rows, seqs, cu, n);
    else if (f32) k_append8<false, MTC_DTYPE_F32><<<g, 256, 0, st>>>(*c, layer, *k, *v, rows, seqs, cu, n);
    else k_append8<false, MTC_DTYPE_F16><<<g, 256, 0, st>>>(*c, layer, *k, *v, rows, seqs, cu, n);
    return check_launch("k_append8");
  }
  const int64_t blocks = ((int64_t)rows * 2 * c->kv_heads * (c->dim / 8) + 255) / 256;
  if (blocks > 0xFFFFFF) return fail(MTC_E_SHAPE, "%d rows: too many", rows);
  const dim3 g((unsigned)blocks);
  if (bf && f32) k_append<true, true><<<g, 256, 0, st>>>(*c, layer, *k, *v, rows, seqs, cu, n);
  else if (bf) k_append<true, false><<<g, 256, 0, st>>>(*c, layer, *k, *v, rows, seqs, cu, n);
  else if (f32) k_append<false, true><<<g, 256, 0, st>>>(*c, layer, *k, *v, rows, seqs, cu, n);
  else k_append<false, false><<<g, 256, 0, st>>>(*c, layer, *k, *v, rows, seqs, cu, n);
  return check_launch("k_append");
}

MTC_API int mtc_cache_read(const mtc_cache_desc* c, int layer, const mtc_heads* k, const mtc_heads* v, int dst_dtype, int rows,
                           const int32_t* seqs, const int32_t* cu, int n, void* hip_stream) {
  if (int rc = check_rows(c, layer, k, v, dst_dtype, rows, seqs, cu, n)) return rc;
  if (!codes::is_codes(*c)) return fail(MTC_E_DTYPE, "a cache of dtype %d holds no codes", c->dtype);
  if (n == 0 || rows == 0) return ok();
  hipStream_t st = (hipStream_t)hip_stream;
  const bool bf = codes::base_type(*c) == MTC_DTYPE_BF16, f32 = dst_dtype == MTC_DTYPE_F32;
  const int64_t blocks = ((int64_t)rows * 2 * c->kv_heads * (codes::row_bytes(c->dim) / 16) + 255) / 256;
  if (blocks > 0xFFFFFF) return fail(MTC_E_SHAPE, "%d rows: too many", rows);
  const dim3 g((unsigned)blocks);
  if (bf && f32) k_read8<true, MTC_DTYPE_F32><<<g, 256, 0, st>>>(*c, layer, *k, *v, rows, seqs, cu, n);
  else if (bf) k_read8<true, MTC_DTYPE_BF16><<<g, 256, 0, st>>>(*c, layer, *k, *v, rows, seqs, cu, n);
  else if (f32) k_read8<false, MTC_DTYPE_F32><<<g, 256, 0, st>>>(*c, layer, *k, *v, rows, seqs, cu, n);
  else k_read8<false, MTC_DTYPE_F16><<<g, 256, 0, st>>>(*c, layer, *k, *v, rows, seqs, cu, n);
  return check_launch("k_read8");
}

MTC_API size_t mtc_verify_workspace_bytes(const mtc_verify_args* a) {
  if (check_verify(a) != MTC_OK) return 0;
  return (size_t)a->n_seqs * verify_splits(a) * sizeof(Found);
}

MTC_API int mtc_verify_drafts(const mtc_verify_args* a, void* workspace, size_t workspace_bytes, void* hip_stream) {
  if (int rc = check_verify(a)) return rc;
  if (a->n_seqs == 0) return ok();
  if (!a->p || !a->noise || !a->tokens || !a->accepted) return fail(MTC_E_NULL, "p, noise, tokens or accepted is NULL");
  if (a->n_drafted && (!a->q || !a->u || !a->drafts)) return fail(MTC_E_NULL, "q, u or drafts is NULL");
  const size_t need = (size_t)a->n_seqs * verify_splits(a) * sizeof(Found);
  if (!workspace || workspace_bytes < need)
    return fail(MTC_E_WORKSPACE, "workspace of %zu bytes, needs %zu", workspace ? workspace_bytes : (size_t)0, need);
  if ((uintptr_t)workspace % 256) return fail(MTC_E_WORKSPACE, "workspace must be 256-byte aligned");
  Found* found = (Found*)workspace;
  hipStream_t st = (hipStream_t)hip_stream;
  if (a->dtype == MTC_DTYPE_F32) return run_verify<MTC_DTYPE_F32>(*a, found, st);
  if (a->dtype == MTC_DTYPE_BF16) return run_verify<MTC_DTYPE_BF16>(*a, found, st);
  return run_verify<MTC_DTYPE_F16>(*a, found, st);
}
