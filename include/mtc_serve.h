/*
 * C-ABI of libmtc_hip.so, serving operators: attention over whole prompts, a paged K/V cache with
 * the attention that reads it, and the verification of drafted tokens. No counterpart in the
 * reference, whose layers end at the linear product.
 *
 * The conventions of mtc_hip.h hold: plain C types, caller-owned device buffers, no allocation,
 * asynchronous launches on the given HIP stream (NULL = default stream), 0 or a negative MTC_E*
 * code, mtc_last_error(). Sizes and strides are checked on the host. Values that live on the
 * device (offsets, lengths, page ids, sequence numbers) are bounded by the kernels: none of them
 * leads to an access outside the buffers that the call names.
 */
#ifndef MTC_SERVE_H
#define MTC_SERVE_H

#include "mtc_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { MTC_DTYPE_F16 = 2 };            /* beside MTC_DTYPE_F32 and MTC_DTYPE_BF16 */

#define MTC_ATTN_MAX_DIM 128           /* head size: a multiple of 8 up to this */
#define MTC_ROTARY_MAX_DIM 1024        /* head size of mtc_rotary */
#define MTC_CACHED_MAX_TOKENS 16       /* queries per sequence of mtc_cached_attention */
#define MTC_CACHED_MAX_SEQS 8192       /* sequences of one cached or bookkeeping call */
#define MTC_CACHE_MAX_SLOTS 65536      /* sequences that one cache can hold (max_seqs) */

/* A strided (rows, heads, dim) view; element strides, unit stride along dim. The base is 16-byte
 * aligned and both strides are multiples of 8 elements. */
typedef struct mtc_heads {
  void* data;
  int64_t row_stride;
  int64_t head_stride;
} mtc_heads;

/*
 * Attention over whole prompts. Sequence b owns rows cu_q[b] .. cu_q[b+1] of q and o and rows
 * cu_k[b] .. cu_k[b+1] of k and v (n_seqs + 1 offsets each, from 0, not falling; offsets past q_rows
 * / k_rows are cut there). Query head h reads K/V head h / (heads / kv_heads).
 *   o[t, h] = sum_j softmax_j(scale * q[t, h] . k[j]) v[j]
 * over all keys of its sequence, or with `causal` over keys j <= t + (keys - queries), the queries
 * being the last tokens. A row that sees no key is 0. Keys that a row does not see have no part in it,
 * whatever they hold (infinities and NaN included). dtype: bf16 or f16 for q, k, v and o; products
 * on the matrix cores, sums and softmax in fp32. Rows of o outside every sequence are not written. o may be q itself
 * (the same address and strides); it shares no other memory with q, k or v.
 * Workspace: mtc_prompt_attention_workspace_bytes (0 but for calls of few rows on many keys, whose keys are split over
 * blocks), 256-byte aligned, no initialisation.
 */
typedef struct mtc_prompt_args {
  uint32_t abi_version;
  int32_t dtype;
  int32_t n_seqs;
  int32_t heads;
  int32_t kv_heads;
  int32_t dim;
  int32_t q_rows;
  int32_t k_rows;
  int32_t causal;
  float scale;
  mtc_heads q;
  mtc_heads k;
  mtc_heads v;
  mtc_heads o;
  const int32_t* cu_q;
  const int32_t* cu_k;
} mtc_prompt_args;

size_t mtc_prompt_attention_workspace_bytes(const mtc_prompt_args* a);
int mtc_prompt_attention(const mtc_prompt_args* a, void* workspace, size_t workspace_bytes, void* hip_stream);

/*
 * The paged cache. The pool holds n_pages pages, each contiguous:
 *   page = [n_layers][2 (K, V)][kv_heads][page_size][dim] of dtype
 * so one copy moves a page of every layer. Sequence s (0 <= s < max_seqs) holds lens[s] tokens;
 * token i lies in page table[s * max_pages + i / page_size] at place i % page_size. Entries past the
 * last page are -1. refs[p] counts the sequences that hold page p (0: free). state[0] collects
 * MTC_CACHE_* bits, state[1] is a page id below which no page is free; the other words are scratch.
 * scratch: mtc_cache_scratch_ints() words, no initialisation. page_size: a power of two, 16 to 256.
 *
 * Bookkeeping calls take device lists of distinct sequence numbers. A call whose list names a sequence
 * out of range or twice, that runs out of pages or of table entries, or whose lengths do not fit, changes
 * nothing and sets its bit in state[0] (no host synchronisation; the caller reads it when it likes).
 * A length outside 0 .. max_pages * page_size counts as the nearest of the two; extend refuses it.
 * Results do not depend on the order in which blocks run.
 *
 * 8-bit caches: dtype MTC_DTYPE_BF16 or MTC_DTYPE_F16 with MTC_CACHE_CODES8. A page is
 *   [n_layers][2 (K, V)][kv_heads][page_size][dim rounded up to a multiple of 16] int8 codes, then
 *   [n_layers][2][kv_heads][page_size / MTC_CODES8_BLOCK] bf16 scales, rounded up to a multiple of 16 bytes;
 * a value is code * scale, of a code from -127 to 127 and a scale for each MTC_CODES8_BLOCK tokens of one head, a power of two from 2^-100 to 2^100 (bf16)
 * or 2^-24 to 2^9 (f16): every value is a number of the dtype. Bookkeeping calls and mtc_cached_attention take both kinds.
 */
enum {
  MTC_CACHE_BAD_SEQ = 1,      /* sequence number out of range or twice in a list */
  MTC_CACHE_NO_PAGES = 2,     /* not enough free pages */
  MTC_CACHE_TABLE_FULL = 4,   /* a sequence would need more than max_pages entries */
  MTC_CACHE_BAD_LENGTH = 8,   /* negative count or present length, or a length above the present one */
  MTC_CACHE_NOT_EMPTY = 16,   /* fork into a sequence that holds tokens, or that is a source of the call */
  MTC_CACHE_SHARED_PAGE = 32  /* append to an 8-bit cache into a page that several sequences hold */
};
enum { MTC_CACHE_CODES8 = 16 };        /* flag of mtc_cache_desc.dtype */
#define MTC_CODES8_BLOCK 16            /* tokens of a scale */

typedef struct mtc_cache_desc {
  uint32_t abi_version;
  int32_t dtype;
  int32_t n_pages;
  int32_t n_layers;
  int32_t kv_heads;
  int32_t dim;
  int32_t page_size;
  int32_t max_seqs;
  int32_t max_pages;
  int32_t reserved;           /* 0 */
  void* pool;                 /* 16-byte aligned */
  int32_t* table;
  int32_t* lens;
  int32_t* refs;
  int32_t* state;             /* 4 words */
  int32_t* scratch;
} mtc_cache_desc;

int mtc_check_cache_desc(const mtc_cache_desc* c);
size_t mtc_cache_scratch_ints(int n_pages, int max_seqs);

/* Room for counts[i] more tokens of sequence seqs[i], i < n: lens grow; new pages are the lowest free ids,
 * in the list's order. A partly filled last page that another sequence holds too (before the call) is copied
 * to a new page first (the first of that sequence's). The tokens' K and V are written by mtc_cache_append. */
int mtc_cache_extend(const mtc_cache_desc* c, const int32_t* seqs, const int32_t* counts, int n, void* hip_stream);

/* dst[i] becomes a second holder of every page of src[i] (src may repeat; dst are empty). No data moves. */
int mtc_cache_fork(const mtc_cache_desc* c, const int32_t* src, const int32_t* dst, int n, void* hip_stream);

/* Sequence seqs[i] keeps its first new_lens[i] tokens (NULL: none); pages that nobody holds become free. */
int mtc_cache_truncate(const mtc_cache_desc* c, const int32_t* seqs, const int32_t* new_lens, int n,
                       void* hip_stream);

/* Pages in use take the ids 0 .. used-1: the pages beyond move, in order, into the free ids below, in order. */
int mtc_cache_compact(const mtc_cache_desc* c, void* hip_stream);

/* Page dst[i] of this pool = page src[i] of from_pool (a pool of the same geometry with from_pages pages; may be
 * this one). dst are distinct and none is a src of the same pool. Ids out of range copy nothing.
 * No bookkeeping changes. */
int mtc_cache_copy_pages(const mtc_cache_desc* c, const void* from_pool, int from_pages, const int32_t* src,
                         const int32_t* dst, int n, void* hip_stream);

/* Writes K and V of the newest tokens: rows cu[i] .. cu[i+1] of k and v (offsets from 0, cut at `rows`) become the
 * last cu[i+1] - cu[i] tokens of sequence seqs[i] in `layer`, rounded to the pool's dtype (src_dtype: fp32 or the
 * pool's). Rows that would fall before token 0 or on no page are not written. */
int mtc_cache_append(const mtc_cache_desc* c, int layer, const mtc_heads* k, const mtc_heads* v, int src_dtype,
                     int rows, const int32_t* seqs, const int32_t* cu, int n, void* hip_stream);
/* Into an 8-bit cache: a block's exponent e is the least with max |x| <= 127 2^e over its new tokens (finite ones), not less than
 * that of the older tokens it holds; new codes are x 2^-e, rounded to nearest even and cut to -127 .. 127 (NaN: 0), codes of the older
 * tokens code 2^(old e - e), rounded. A block's tokens come from one sequence of a call: nothing is written into a page that several
 * sequences hold (MTC_CACHE_SHARED_PAGE), nor for a sequence that the list names twice (MTC_CACHE_BAD_SEQ). */

/* Reads an 8-bit cache back: rows cu[i] .. cu[i+1] of k and v (offsets from 0, cut at `rows`; as many heads and dims as the cache)
 * become the last cu[i+1] - cu[i] tokens of sequence seqs[i] in `layer`. dst_dtype: the cache's (exact) or fp32. Rows before
 * token 0 or on no page become 0, those of no sequence stay as they are. Strides are multiples of 16 bytes. */
int mtc_cache_read(const mtc_cache_desc* c, int layer, const mtc_heads* k, const mtc_heads* v, int dst_dtype, int rows,
                   const int32_t* seqs, const int32_t* cu, int n, void* hip_stream);

/* Sequence seqs[i] becomes a holder of what seqs[parents[i]] held before the call, i < n, all at once: pages that nobody
 * holds any more become free. parents may repeat; one out of 0 .. n-1 is MTC_CACHE_BAD_SEQ. No data moves. */
int mtc_cache_reorder(const mtc_cache_desc* c, const int32_t* seqs, const int32_t* parents, int n, void* hip_stream);

/*
 * Attention of the newest `tokens` tokens (1 .. MTC_CACHED_MAX_TOKENS) of n_seqs sequences over the
 * cache, their own K and V included (append first). q and o: rows b * tokens + t. q_lens[b]
 * (NULL: tokens) rows of sequence b count: row t < q_lens[b] sees the first
 * lens[s] - q_lens[b] + t + 1 tokens of s = seqs[b] (NULL: b); a row that sees none, or t >= q_lens[b], is 0.
 * o may be q itself (the same address and strides); it shares no other memory with q or the cache.
 *
 * Shared prefixes: groups (n_groups + 1 offsets into the batch, from 0 to n_seqs, not falling) and
 * prefix_lens (n_groups): the sequences groups[g] .. groups[g+1] hold the same pages for their first
 * prefix_lens[g] tokens (as after a fork). These tokens are read from the group's first sequence
 * and multiplied with the rows of all its members at once; prefix_lens are rounded down to whole pages.
 * n_groups = 0: every sequence by itself.
 *
 * Workspace: mtc_cached_attention_workspace_bytes, 256-byte aligned, no initialisation.
 */
typedef struct mtc_cached_args {
  uint32_t abi_version;
  int32_t layer;
  int32_t n_seqs;
  int32_t tokens;
  int32_t heads;
  int32_t n_groups;
  float scale;
  int32_t reserved;           /* 0 */
  mtc_heads q;
  mtc_heads o;
  const int32_t* seqs;
  const int32_t* q_lens;
  const int32_t* groups;
  const int32_t* prefix_lens;
} mtc_cached_args;

size_t mtc_cached_attention_workspace_bytes(const mtc_cache_desc* c, const mtc_cached_args* a);
int mtc_cached_attention(const mtc_cache_desc* c, const mtc_cached_args* a, void* workspace, size_t workspace_bytes,
                         void* hip_stream);

/*
 * Verification of drafted tokens by rejection sampling with given random numbers. For sequence b with
 * k = n_drafts[b] (NULL: n_drafted; cut to 0 .. n_drafted) drafts x_0 .. x_{k-1} drawn from q:
 * draft j is accepted while u[b, j] * q[b, j, x_j] < p[b, j, x_j] (fp32 product); with n accepted, the next token
 * is the first index of the largest w_i * noise[b, i] over w_i > 0, where w = p[b, n] if n = k, else
 * max(p[b, n] - q[b, n], 0), or p[b, n] where that is 0 everywhere (-1 if no w_i > 0). With noise_i = 1 / Exp(1)
 * the next token has the probabilities w / sum(w). Differences and products are fp32.
 *   p (n_seqs, n_drafted + 1, vocab), q (n_seqs, n_drafted, vocab), dtype fp32, bf16 or f16, element
 *   strides of the first two axes; u (n_seqs, n_drafted) and noise (n_seqs, vocab) fp32; drafts and tokens
 *   int32 or int64 (index_bytes 4 or 8); tokens (n_seqs, n_drafted + 1): the accepted drafts, the next
 *   token, then -1; accepted (n_seqs) int32. A draft outside the vocabulary is rejected.
 * Workspace: mtc_verify_workspace_bytes, 256-byte aligned, no initialisation.
 */
typedef struct mtc_verify_args {
  uint32_t abi_version;
  int32_t dtype;
  int32_t index_bytes;
  int32_t n_seqs;
  int32_t n_drafted;
  int32_t vocab;
  const void* p;
  int64_t p_stride[2];
  const void* q;
  int64_t q_stride[2];
  const float* u;
  int64_t u_stride;
  const float* noise;
  int64_t noise_stride;
  const void* drafts;
  int64_t drafts_stride;
  const int32_t* n_drafts;
  void* tokens;               /* contiguous */
  int32_t* accepted;
} mtc_verify_args;

size_t mtc_verify_workspace_bytes(const mtc_verify_args* a);
int mtc_verify_drafts(const mtc_verify_args* a, void* workspace, size_t workspace_bytes, void* hip_stream);

/*
 * Rotary positions. Pair i < rotated / 2 of row r turns by t = positions[r] f_i radians:
 *   (x, y) -> amplitude (x cos t - y sin t, x sin t + y cos t)
 * of dims (i, i + rotated / 2), or (2 i, 2 i + 1) if interleaved; dims from `rotated` on are copied. turns[i] =
 * round(2^64 f_i / 2 pi) modulo 2^64: the product with a position, modulo 2^64, is the exact fraction of a turn.
 *   q (rows, heads, dim) -> oq, k (rows, kv_heads, dim) -> ok: dtype fp32, bf16 or f16; heads or kv_heads may be 0. dim: a multiple of 8 up to
 *   MTC_ROTARY_MAX_DIM. Strides are multiples of 16 bytes. oq may be q itself (the same address and strides), ok k; they
 *   share no other memory with q or k.
 */
typedef struct mtc_rotary_args {
  uint32_t abi_version;
  int32_t dtype;
  int32_t rows;
  int32_t heads;
  int32_t kv_heads;
  int32_t dim;
  int32_t rotated;
  int32_t interleaved;
  float amplitude;
  int32_t reserved;           /* 0 */
  mtc_heads q;
  mtc_heads k;
  mtc_heads oq;
  mtc_heads ok;
  const int32_t* positions;
  const uint64_t* turns;
} mtc_rotary_args;

int mtc_rotary(const mtc_rotary_args* a, void* hip_stream);

/*
 * One step of beam search: of every prompt's beams x vocabulary continuations the n with the highest score
 *   scores[b, w] + logits[b, w, v] - log sum_u exp logits[b, w, u]
 * in falling order, equal ones in the order of w * vocab + v. A beam with done[b, w] (NULL: none) is not continued: it stands
 * as one candidate of its present score, with the token `pad` (in the order: v = 0); its logits are not read. Candidates of score -inf or NaN are none
 * (a logit of -inf is a token that may not come; a NaN or +inf among a beam's logits leaves that beam without candidates). Logarithms and
 * exponentials are fp32 or better, sums of scores fp64.
 *   logits (n_prompts, beams, vocab) fp32, bf16 or f16, element strides of the first two axes; scores (n_prompts, beams)
 *   fp32 and done bytes, contiguous; outputs (n_prompts, n): scores fp32, tokens, parents (b * beams + w). Where there are fewer candidates
 *   than n: -inf, -1 and the row b * beams + min(place, beams - 1).
 * Workspace: mtc_beam_workspace_bytes, 256-byte aligned, no initialisation.
 */
#define MTC_BEAM_MAX 64                /* beams of a prompt, and n */
typedef struct mtc_beam_args {
  uint32_t abi_version;
  int32_t dtype;
  int32_t n_prompts;
  int32_t beams;
  int32_t vocab;
  int32_t n;
  int32_t pad;
  int32_t reserved;           /* 0 */
  const void* logits;
  int64_t stride[2];
  const float* scores;
  const uint8_t* done;
  float* out_scores;
  int32_t* tokens;
  int32_t* parents;
} mtc_beam_args;

size_t mtc_beam_workspace_bytes(const mtc_beam_args* a);
int mtc_beam_select(const mtc_beam_args* a, void* workspace, size_t workspace_bytes, void* hip_stream);

#ifdef __cplusplus
}
#endif

#endif /* MTC_SERVE_H */
