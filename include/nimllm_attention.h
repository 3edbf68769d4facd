/*
 * nimllm_attention.h -- C ABI of the MI355X (gfx950) rotary positions, paged
 * key/value cache and attention.
 *
 * What stands between two of nimllm_lmhead.h's projections when several
 * contexts decode together: the counterpart, for device memory and a cache in
 * pages, of rope and attnTask over the dense fp32 cache of nimllm's forward
 * pass (src/nimllm/model.nim:300-302, :362-393, :446).  One step of a layer is
 *
 *   nls_lm_head       x -> q, k, v              (three projections)
 *   nls_cache_append  q, k rotated; k, v to their pages
 *   nls_paged_attention
 *   nls_lm_head       attention -> x            (the output projection)
 *
 * with nls_cache_reserve once per step before it, for the step's tokens.
 *
 * Contexts occupy the `slots` rows of a page table.  Position p of slot s is
 * token p % page_size of page table[s][p / page_size].  Lengths, table and
 * reference counts live on the device and every call is ordered on `stream`
 * (a hipStream_t, NULL = default stream): nothing here synchronises, allocates
 * or keeps anything between calls, so a step can be captured and replayed.
 * The device has to be current whose memory the pointers name.  Calls that
 * change one cache's tables, and calls that read it, are ordered by the
 * caller (one stream, or events); a workspace belongs to one call at a time.
 *
 * Status codes are nimllm_sampler.h's NLS_* values.  Element types are the
 * GGML codes of nimllm_lmhead.h: NLS_GGML_F32 (0), NLS_GGML_F16 (1) and
 * NLS_GGML_BF16 (30).
 */
#ifndef NIMLLM_ATTENTION_H
#define NIMLLM_ATTENTION_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Rows of heads, [tokens, heads, head_dim]: strides in elements, the elements
 * of one head side by side. */
typedef struct nls_heads {
  void* d;
  int64_t token_stride;
  int64_t head_stride;
} nls_heads;

/* ---- rotary positions ---- */

enum { NLS_ROPE_NONE = 0, NLS_ROPE_LINEAR = 1, NLS_ROPE_YARN = 2 };

/* How far each pair turns per position: base^(-2j/dim), then
 *   linear  divided by `factor`
 *   yarn    divided by `factor` where a pair turns less than beta_slow times
 *           over original_context positions, as it is where it turns more than
 *           beta_fast times, blended in between; the amplitude is
 *           attn_factor * (0.1 ln(factor) + 1), attn_factor otherwise
 * and divided by freq_factors[j] (host, dim / 2 entries, none 0, or NULL), the
 * rope_freqs tensor of a GGUF file. */
typedef struct nls_rope_scaling {
  int32_t kind;
  double base;
  double factor;
  double original_context;
  double beta_fast;
  double beta_slow;
  double attn_factor;
  const double* freq_factors;
} nls_rope_scaling;

/* Host only: the dim / 2 angles per position and the amplitude. */
int32_t nls_rope_frequencies(const nls_rope_scaling* scaling, int32_t dim, double* freqs, double* amplitude);

/* The first `dim` elements of each head are turned, in pairs (2j, 2j + 1) when
 * `interleaved`, else (j, j + dim / 2); the others pass.  d_freqs: dim / 2
 * float64 on the device. */
typedef struct nls_rope_plan {
  const double* d_freqs;
  int32_t dim;
  int32_t interleaved;
  float amplitude;
} nls_rope_plan;

/*
 * y[t, h, :] = x[t, h, :] turned by positions[t] * freqs (`inverse`: by minus
 * that, with the same amplitude, which takes a gradient of y to one of x).
 * Angles and their reduction are float64, sines, cosines and products fp32,
 * rounded once to `type`.  y may be x.  d_positions: int32 [tokens], any value.
 */
int32_t nls_rope(const nls_rope_plan* plan, int32_t type, const nls_heads* x, const nls_heads* y, int32_t tokens,
                 int32_t heads, int32_t head_dim, const int32_t* d_positions, int32_t inverse, void* stream);

/* ---- the cache ---- */

/* One layer's keys and values: the key of page p, head h, token t starts at
 * d_kv + p * page_stride + h * head_stride + t * token_stride (elements), the
 * value value_offset elements behind it.  All four strides are multiples of 8
 * (page_stride and token_stride below 2^30), d_kv is 16-byte aligned, head_dim a
 * multiple of 8 up to 256, page_size a power of two up to 4096.  A table entry outside [0, pages) is no page: what
 * it would hold is neither read nor written, and attention sees no key there. */
typedef struct nls_paged_kv {
  void* d_kv;
  int32_t type;
  int32_t pages;
  int32_t page_size;
  int32_t kv_heads;
  int32_t head_dim;
  int64_t page_stride;
  int64_t value_offset;
  int64_t head_stride;
  int64_t token_stride;
  const int32_t* d_table; /* [slots, max_pages], rows table_stride apart */
  int64_t table_stride;
  int32_t slots;
  int32_t max_pages;
  const int32_t* d_lens; /* [slots]: tokens of each context, this call's among them */
} nls_paged_kv;

/* The new tokens of a call: sequence i's are rows [d_starts[i], d_starts[i+1])
 * of q, k, v and the outputs, and they are the last ones of slot d_slots[i]
 * (slot i when d_slots is NULL).  `tokens` rows are there in all; rows before
 * d_starts[0] and behind d_starts[seqs] belong to no sequence, and none of the
 * outputs' is written.  d_starts never falls.  A sequence of a slot outside
 * [0, slots) has no keys, and its tokens are not appended.  Fewer than 2^24
 * tokens, and fewer than 2^30 rows of heads. */
typedef struct nls_chunks {
  int32_t seqs;
  int32_t tokens;
  const int32_t* d_starts; /* [seqs + 1] */
  const int32_t* d_slots;  /* [seqs] or NULL */
} nls_chunks;

/*
 * The new tokens into the cache: q_out = q turned (q may be NULL, with heads
 * 0; q_out may be q), k turned and v as it is to the pages of their positions,
 * converted to the cache's type.  plan may be NULL (nothing is turned).
 * `type` is that of q, k and v.  Two tokens never share a place, unless a slot
 * is named twice or a page is held twice: then either's row may stay.
 */
int32_t nls_cache_append(const nls_paged_kv* kv, const nls_chunks* chunks, const nls_rope_plan* plan, int32_t type,
                         const nls_heads* q, const nls_heads* q_out, int32_t heads, const nls_heads* k,
                         const nls_heads* v, void* stream);

/*
 * out[t, h] = sum_j softmax_j(scale * q[t, h] . k_j) v_j over the keys j of
 * t's slot, of head h / (heads / kv_heads), with
 *   j <= p                   p: t's position, lens - (its place from the end)
 *   j >  p - window          when window > 0
 *   j >= d_first[slot]       when d_first is not NULL
 * lse[t, h] = ln sum_j exp(scale * q . k_j) where d_lse (fp32, [tokens, heads]
 * contiguous) is not NULL.  A row without a key, or whose every score is
 * -infinity, has out = 0 and lse = -infinity.  What a key that a row does not
 * see holds, infinities and NaN among it, does not reach that row; an infinite
 * value that it does see makes it infinite or NaN.  (An infinite key that it
 * sees makes its score infinite, or NaN where fp32 queries meet 16-bit keys.)
 * scale: finite, up to 2.3e38 either way (log2 e times it is finite too).
 * type (q and out): F32 with any cache type, F16 or BF16 with the same one.
 * Scores, statistics and sums are fp32.  fp32 queries and weights meet 16-bit
 * keys and values as sums of 16-bit parts: three of bf16, which are exact, or two
 * of fp16, 22 bits (or 2^-38 of the row's largest element).  16-bit queries'
 * weights are rounded to the cache's type in sequences of more than 16 rows
 * (tokens times heads per kv head), and to 16 bits or more in others, so a token
 * may come out a rounding apart in another batch.  Weighted values are summed
 * before they are divided: in an fp32 or bf16 cache, values beyond 2^88 may
 * overflow in long sums.
 * max_new and max_len say what the caller expects of the longest chunk and
 * context (0: not known).  They choose how the work is split; results hold
 * whatever the true values are.
 * d_work: nls_paged_attention_workspace() bytes, 256-byte aligned.
 */
size_t nls_paged_attention_workspace(const nls_paged_kv* kv, const nls_chunks* chunks, int32_t heads, int32_t max_new,
                                     int64_t max_len, int32_t window);
int32_t nls_paged_attention(const nls_paged_kv* kv, const nls_chunks* chunks, int32_t type, const nls_heads* q,
                            const nls_heads* out, int32_t heads, float scale, int32_t window, const int32_t* d_first,
                            float* d_lse, int32_t max_new, int64_t max_len, void* d_work, size_t work_bytes,
                            void* stream);

/* ---- pages ---- */

/* The contents of all layers: page p of layer l is page_bytes bytes at
 * d_kv + l * layer_stride + p * page_stride (bytes).  All are multiples of 16,
 * d_kv is 16-byte aligned. */
typedef struct nls_page_pool {
  void* d_kv;
  int32_t layers;
  int64_t page_bytes;
  int64_t layer_stride;
  int64_t page_stride;
} nls_page_pool;

/* Who holds what: refs[p] counts the table entries that name page p (0: free).
 * Slot s holds ceil(lens[s] / page_size) pages; its further entries are -1. */
typedef struct nls_page_tables {
  int32_t* d_table;
  int64_t table_stride;
  int32_t slots; /* at most 65536 */
  int32_t max_pages;
  int32_t* d_lens;
  int32_t* d_refs;
  int32_t pages; /* at most 524288 */
  int32_t page_size;
} nls_page_tables;

/* What reserve, fork and release write to *d_status: all of the call was done,
 * or none of it for the reason given. */
enum {
  NLS_PAGES_DONE = 0,
  NLS_PAGES_NONE_LEFT = 1, /* fewer free pages than the call takes */
  NLS_PAGES_ROW_FULL = 2,  /* a context would outgrow max_pages */
  NLS_PAGES_BAD_ENTRY = 3  /* a slot out of range or named where it may not be, or a negative count */
};

/* Device workspace of the calls below, 256-byte aligned: one size for all of
 * them, so that one buffer serves each in turn (compact's three words per page
 * are the most of it; release checks it as the others do and uses none). */
size_t nls_cache_workspace(const nls_page_tables* tables, int32_t count);

/* Slot s grows by counts[s] (int32 [slots]) tokens: pages for them, the lowest
 * free ones in the order of the slots, and lens[s] += counts[s]. */
int32_t nls_cache_reserve(const nls_page_tables* tables, const int32_t* d_counts, int32_t* d_status, void* d_work,
                          size_t work_bytes, void* stream);

/* For each i < count, the empty slot dst[i] becomes a copy of slot src[i]: its
 * full pages are shared, its last partial one is copied to the lowest free
 * page (in the order of i).  Each dst once; no slot in both lists. */
int32_t nls_cache_fork(const nls_page_pool* pool, const nls_page_tables* tables, const int32_t* d_src,
                       const int32_t* d_dst, int32_t count, int32_t* d_status, void* d_work, size_t work_bytes,
                       void* stream);

/* The listed slots let go of their pages and are empty; one named twice is
 * released once. */
int32_t nls_cache_release(const nls_page_tables* tables, const int32_t* d_slots, int32_t count, int32_t* d_status,
                          void* d_work, size_t work_bytes, void* stream);

/* Moves pages so that the held ones are 0 .. *d_live - 1: the held pages from
 * there on, in ascending order, to the free ones below it, in ascending
 * order.  lens may be NULL in the tables. */
int32_t nls_cache_compact(const nls_page_pool* pool, const nls_page_tables* tables, int32_t* d_live, void* d_work,
                          size_t work_bytes, void* stream);

/* Page src[i] to page dst[i] in every layer, i < count; pairs with a page
 * outside [0, pages) are passed over.  A page that is a destination is in the
 * lists once. */
int32_t nls_cache_copy_pages(const nls_page_pool* pool, int32_t pages, const int32_t* d_src, const int32_t* d_dst,
                             int32_t count, void* stream);

#ifdef __cplusplus
}
#endif

#endif
