// nls_attend_api.cpp -- host side of the C ABI in include/nimllm_attention.h:
// the arguments' checks and the launches.  Every check comes before any device
// work, and no call keeps anything.
#include <hip/hip_runtime.h>

#include <cmath>

#include "../../include/nimllm_attention.h"
#include "../../include/nimllm_sampler.h"
#include "nls_internal.h"
#include "nls_paged.h"

using namespace nls;

namespace {

int bad(const char* what) { return api_error(NLS_ERR_INVALID_ARGUMENT, what); }
int done(hipError_t e, const char* what) { return e == hipSuccess ? NLS_OK : api_hip_error(e, what); }

bool elem_type(int t) { return t == kF32 || t == kF16 || t == kBF16; }
int elem_bytes(int t) { return t == kF32 ? 4 : 2; }
bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
hipStream_t stream_of(void* s) { return reinterpret_cast<hipStream_t>(s); }

constexpr int kMaxTokens = (1 << 24) - 1;  // a workgroup of 256 each: fewer than 2^32 threads

// A strided view [tokens, heads, dim] whose elements side by side do not
// overlap between heads or tokens when it is written.
const char* check_heads(const nls_heads* x, int type, int heads, int tokens, int dim, bool written) {
  if (!x || !x->d) return "NULL rows of heads";
  if (!aligned(x->d, elem_bytes(type))) return "rows of heads: misaligned pointer";
  const int64_t big = int64_t{1} << 40;
  if (x->token_stride < 0 || x->head_stride < 0 || x->token_stride > big || x->head_stride > big)
    return "rows of heads: a stride is negative or too large";
  if (written) {
    const bool tokens_outer = x->token_stride >= x->head_stride;
    const int64_t in = tokens_outer ? x->head_stride : x->token_stride, out = tokens_outer ? x->token_stride : x->head_stride;
    const int64_t n_in = tokens_outer ? heads : tokens, n_out = tokens_outer ? tokens : heads;
    if ((n_in > 1 && in < dim) || (n_out > 1 && out < (n_in - 1) * in + dim))
      return "rows of heads: an output's strides overlap";
  }
  return nullptr;
}
bool wide_ok(const nls_heads* x, int type, int n) {
  return !x || !x->d || (aligned(x->d, 16) && x->token_stride % n == 0 && x->head_stride % n == 0 &&
                         (n * elem_bytes(type)) % 16 == 0);
}
HeadsView view(const nls_heads* x) { return x ? HeadsView{x->d, x->token_stride, x->head_stride} : HeadsView{}; }

const char* check_plan(const nls_rope_plan* p, int dim) {
  if (p->dim < 0 || p->dim > dim || (p->dim & 1)) return "rope plan: dim is odd or beyond the head";
  if (p->dim > 0 && (!p->d_freqs || !aligned(p->d_freqs, 8))) return "rope plan: NULL or misaligned frequencies";
  return nullptr;
}

const char* check_kv(const nls_paged_kv* kv) {
  if (!kv) return "NULL cache";
  if (!elem_type(kv->type)) return "cache: element type is not F32, F16 or BF16";
  if (kv->pages < 1 || kv->slots < 1 || kv->max_pages < 1 || kv->kv_heads < 1) return "cache: a size is below 1";
  if (kv->page_size < 1 || kv->page_size > kMaxPageSize || (kv->page_size & (kv->page_size - 1)))
    return "cache: page_size is not a power of two up to 4096";
  if (kv->head_dim < 8 || kv->head_dim > kMaxHeadDim || kv->head_dim % 8)
    return "cache: head_dim is not a multiple of 8 up to 256";
  if (!kv->d_kv || !aligned(kv->d_kv, 16)) return "cache: NULL or misaligned d_kv";
  if (!kv->d_table || !kv->d_lens || !aligned(kv->d_table, 4) || !aligned(kv->d_lens, 4))
    return "cache: NULL or misaligned table or lens";
  const int64_t big = int64_t{1} << 40;
  const int64_t st[4] = {kv->page_stride, kv->value_offset, kv->head_stride, kv->token_stride};
  for (int64_t x : st)
    if (x < 0 || x > big || x % 8) return "cache: a stride is negative, too large or no multiple of 8";
  if (kv->page_stride >= int64_t{1} << 30 || kv->token_stride >= int64_t{1} << 30)
    return "cache: page_stride or token_stride is 2^30 elements or more";
  if (kv->value_offset < kv->head_dim || (kv->pages > 1 && kv->page_stride < kv->head_dim) ||
      (kv->kv_heads > 1 && kv->head_stride < kv->head_dim) || (kv->page_size > 1 && kv->token_stride < kv->head_dim))
    return "cache: strides overlap";
  if (kv->table_stride < 0 || kv->table_stride > big || (kv->slots > 1 && kv->table_stride < kv->max_pages))
    return "cache: table_stride is shorter than max_pages";
  return nullptr;
}

const char* check_chunks(const nls_chunks* c) {
  if (!c) return "NULL chunks";
  if (c->seqs < 0 || c->tokens < 0) return "chunks: a negative size";
  if (c->tokens > kMaxTokens) return "chunks: 2^24 tokens or more";
  if (c->seqs > 0 && c->tokens > 0 && (!c->d_starts || !aligned(c->d_starts, 4) || !aligned(c->d_slots, 4)))
    return "chunks: NULL or misaligned starts or slots";
  return nullptr;
}

PagedArgs paged(const nls_paged_kv* kv, const nls_chunks* c) {
  PagedArgs a{};
  a.kv = kv->d_kv;
  a.pages = kv->pages;
  a.page_shift = __builtin_ctz((unsigned)kv->page_size);
  a.kv_heads = kv->kv_heads;
  a.dim = kv->head_dim;
  a.page_stride = kv->page_stride;
  a.value_offset = kv->value_offset;
  a.head_stride = kv->head_stride;
  a.token_stride = kv->token_stride;
  a.table = kv->d_table;
  a.table_stride = kv->table_stride;
  a.slots = kv->slots;
  a.max_pages = kv->max_pages;
  a.lens = kv->d_lens;
  a.seqs = c->seqs;
  a.tokens = c->tokens;
  a.starts = c->d_starts;
  a.slot_of = c->d_slots;
  return a;
}

// The sizes alone, which the workspace goes by too.
const char* check_sizes(const nls_paged_kv* kv, const nls_chunks* c, int heads, int max_new, int64_t max_len,
                        int window) {
  if (!kv || !c) return "NULL cache or chunks";
  if (kv->kv_heads < 1 || kv->head_dim < 8 || kv->head_dim > kMaxHeadDim || kv->head_dim % 8 || kv->max_pages < 1 ||
      kv->page_size < 1 || kv->page_size > kMaxPageSize || (kv->page_size & (kv->page_size - 1)))
    return "cache: a size out of range";
  if (c->seqs < 0 || c->tokens < 0) return "chunks: a negative size";
  if (heads < 1 || heads % kv->kv_heads) return "heads is no multiple of the cache's";
  // (a launch has fewer than 2^32 threads: one workgroup per sequence, kv head
  // and 16 heads of its group, 16 rows each where parts are joined)
  if (heads > 65535 || (int64_t)c->tokens * heads > 0x3fffffff ||
      (int64_t)c->seqs * kv->kv_heads * ((heads / kv->kv_heads + 15) / 16) >= int64_t{1} << 20)
    return "too many rows of heads (2^30), or sequences times heads (2^20)";
  if (max_new < 0 || max_len < 0 || window < 0) return "a negative size";
  return nullptr;
}

AttendArgs attend_args(const nls_paged_kv* kv, const nls_chunks* c, int heads, int window) {
  AttendArgs a{};
  a.p = paged(kv, c);
  a.heads = heads;
  a.group = heads / kv->kv_heads;
  a.window = window;
  return a;
}

size_t align256(size_t n) { return (n + 255) & ~size_t{255}; }

const char* check_tables(const nls_page_tables* t, bool lens) {
  if (!t) return "NULL tables";
  if (t->slots < 1 || t->max_pages < 1 || t->pages < 1) return "tables: a size is below 1";
  if (t->pages > kMaxPages || t->slots > kMaxSlots) return "tables: more than 524288 pages or 65536 slots";
  if (t->page_size < 1 || t->page_size > kMaxPageSize || (t->page_size & (t->page_size - 1)))
    return "tables: page_size is not a power of two up to 4096";
  if (t->table_stride < 0 || (t->slots > 1 && t->table_stride < t->max_pages) || t->table_stride > (int64_t{1} << 31) ||
      (int64_t)t->slots * t->max_pages > 0x7fffffff)
    return "tables: table_stride is shorter than max_pages, or 2^31 entries";
  if (!t->d_table || !t->d_refs || (lens && !t->d_lens) || !aligned(t->d_table, 4) || !aligned(t->d_refs, 4) ||
      !aligned(t->d_lens, 4))
    return "tables: NULL or misaligned table, lens or refs";
  return nullptr;
}
TableArgs tables(const nls_page_tables* t) {
  return {t->d_table, t->table_stride, t->slots, t->max_pages, t->d_lens, t->d_refs, t->pages,
          __builtin_ctz((unsigned)t->page_size)};
}
const char* check_pool(const nls_page_pool* p, int pages) {
  if (!p) return "NULL pool";
  if (p->layers < 1 || p->page_bytes < 16) return "pool: a size is below its least";
  const int64_t big = int64_t{1} << 42;
  if (p->page_bytes % 16 || p->layer_stride % 16 || p->page_stride % 16 || p->page_bytes > (int64_t{1} << 32) ||
      p->layer_stride < 0 || p->layer_stride > big || p->page_stride < 0 || p->page_stride > big)
    return "pool: a stride or page_bytes is negative, too large or no multiple of 16";
  if ((pages > 1 && p->page_stride < p->page_bytes) || (p->layers > 1 && p->layer_stride < p->page_bytes))
    return "pool: strides overlap";
  if (!p->d_kv || !aligned(p->d_kv, 16)) return "pool: NULL or misaligned d_kv";
  return nullptr;
}
PoolArgs pool(const nls_page_pool* p) {
  return {static_cast<char*>(p->d_kv), p->layers, p->page_bytes, p->layer_stride, p->page_stride};
}

// int32 words of the page calls' work area (nls_pages.hip says what they hold)
size_t page_words(const nls_page_tables* t, int count) {
  const size_t reserve = (size_t)t->slots, fork = 1 + 2 * (size_t)count, compact = 1 + 3 * (size_t)t->pages;
  const size_t n = reserve > fork ? reserve : fork;
  return n > compact ? n : compact;
}
const char* check_work(const nls_page_tables* t, int count, const void* work, size_t bytes) {
  return !work || !aligned(work, 256) || bytes < align256(4 * page_words(t, count))
             ? "workspace: NULL, misaligned or too small"
             : nullptr;
}

}  // namespace

#define NLS_CHECK(call)                        \
  do {                                         \
    if (const char* why_ = (call)) return bad(why_); \
  } while (0)

extern "C" {

int32_t nls_rope_frequencies(const nls_rope_scaling* s, int32_t dim, double* freqs, double* amplitude) {
  if (!s || !amplitude || dim < 0 || (dim & 1) || (dim > 0 && !freqs)) return bad("rope: NULL or an odd dim");
  if (s->kind != NLS_ROPE_NONE && s->kind != NLS_ROPE_LINEAR && s->kind != NLS_ROPE_YARN)
    return bad("rope: no such scaling");
  if (!(s->base > 0) || !std::isfinite(s->base) || !std::isfinite(s->attn_factor)) return bad("rope: base or attn_factor");
  if (s->kind != NLS_ROPE_NONE && (!(s->factor > 0) || !std::isfinite(s->factor))) return bad("rope: factor");
  for (int j = 0; s->freq_factors && j < dim / 2; ++j)
    if (!(std::fabs(s->freq_factors[j]) > 0)) return bad("rope: a frequency factor is 0 or NaN");
  double lo = 0, hi = 0;
  if (s->kind == NLS_ROPE_YARN) {
    if (!(s->original_context > 0) || !(s->beta_fast > 0) || !(s->beta_slow > 0) || !(s->base > 1) ||
        !std::isfinite(s->original_context) || !std::isfinite(s->beta_fast) || !std::isfinite(s->beta_slow))
      return bad("rope: yarn's context, betas or base");
    // the pair that turns b times over the original context
    auto pair = [&](double b) {
      return dim * std::log(s->original_context / (b * 2.0 * M_PI)) / (2.0 * std::log(s->base));
    };
    lo = std::fmax(std::floor(pair(s->beta_fast)), 0.0);
    hi = std::fmin(std::ceil(pair(s->beta_slow)), dim - 1.0);
  }
  for (int j = 0; j < dim / 2; ++j) {
    double f = std::pow(s->base, -2.0 * j / dim);
    if (s->kind == NLS_ROPE_LINEAR) f /= s->factor;
    if (s->kind == NLS_ROPE_YARN) {
      const double ramp = std::fmin(std::fmax((j - lo) / std::fmax(hi - lo, 0.001), 0.0), 1.0);
      f = f / s->factor * ramp + f * (1.0 - ramp);
    }
    freqs[j] = s->freq_factors ? f / s->freq_factors[j] : f;
  }
  *amplitude = s->attn_factor * (s->kind == NLS_ROPE_YARN ? 0.1 * std::log(s->factor) + 1.0 : 1.0);
  return NLS_OK;
}

int32_t nls_rope(const nls_rope_plan* plan, int32_t type, const nls_heads* x, const nls_heads* y, int32_t tokens,
                 int32_t heads, int32_t head_dim, const int32_t* d_positions, int32_t inverse, void* stream) {
  if (!plan) return bad("NULL plan");
  if (!elem_type(type)) return bad("rope: element type is not F32, F16 or BF16");
  if (tokens < 0 || tokens > kMaxTokens || heads < 0 || head_dim < 1 || head_dim > kMaxHeadDim)
    return bad("rope: a size out of range");
  NLS_CHECK(check_plan(plan, head_dim));
  if (tokens == 0 || heads == 0) return NLS_OK;
  NLS_CHECK(check_heads(x, type, heads, tokens, head_dim, false));
  NLS_CHECK(check_heads(y, type, heads, tokens, head_dim, true));
  if (x->d == y->d && (x->token_stride != y->token_stride || x->head_stride != y->head_stride))
    return bad("rope: in place with other strides");
  if (!d_positions || !aligned(d_positions, 4)) return bad("rope: NULL or misaligned positions");
  if ((int64_t)heads * head_dim > 0x3fffffff) return bad("rope: too many heads");
  TurnArgs t{};
  t.x = view(x);
  t.y = view(y);
  t.heads = heads;
  t.dim = head_dim;
  t.freqs = plan->d_freqs;
  t.rot = plan->dim;
  t.interleaved = plan->interleaved != 0;
  t.amplitude = plan->amplitude;
  t.sign = inverse ? -1.f : 1.f;
  t.tokens = tokens;
  t.positions = d_positions;
  const int n = type == kF32 ? 4 : 8;
  const bool wide = wide_ok(x, type, n) && wide_ok(y, type, n) && t.rot % (2 * n) == 0 && head_dim % n == 0;
  return done(launch_rope(t, type, wide, stream_of(stream)), "nls_rope");
}

int32_t nls_cache_append(const nls_paged_kv* kv, const nls_chunks* chunks, const nls_rope_plan* plan, int32_t type,
                         const nls_heads* q, const nls_heads* q_out, int32_t heads, const nls_heads* k,
                         const nls_heads* v, void* stream) {
  NLS_CHECK(check_kv(kv));
  NLS_CHECK(check_chunks(chunks));
  if (!elem_type(type) || (type != kF32 && type != kv->type))
    return bad("append: q, k and v are F32, or of the cache's type");
  if (heads < 0 || (int64_t)heads * kv->head_dim > 0x1fffffff || (int64_t)kv->kv_heads * kv->head_dim > 0x1fffffff)
    return bad("append: heads out of range");
  if (plan) NLS_CHECK(check_plan(plan, kv->head_dim));
  if (chunks->tokens == 0 || chunks->seqs == 0) return NLS_OK;
  if (heads > 0) {
    NLS_CHECK(check_heads(q, type, heads, chunks->tokens, kv->head_dim, false));
    NLS_CHECK(check_heads(q_out, type, heads, chunks->tokens, kv->head_dim, true));
    if (q->d == q_out->d && (q->token_stride != q_out->token_stride || q->head_stride != q_out->head_stride))
      return bad("append: in place with other strides");
  }
  NLS_CHECK(check_heads(k, type, kv->kv_heads, chunks->tokens, kv->head_dim, false));
  NLS_CHECK(check_heads(v, type, kv->kv_heads, chunks->tokens, kv->head_dim, false));
  TurnArgs t{};
  if (heads > 0) {
    t.x = view(q);
    t.y = view(q_out);
  }
  t.heads = heads;
  t.dim = kv->head_dim;
  if (plan && plan->dim > 0) {
    t.freqs = plan->d_freqs;
    t.rot = plan->dim;
    t.interleaved = plan->interleaved != 0;
    t.amplitude = plan->amplitude;
    t.sign = 1.f;
  }
  t.tokens = chunks->tokens;
  t.k = view(k);
  t.v = view(v);
  const bool wide = (heads == 0 || (wide_ok(q, type, 8) && wide_ok(q_out, type, 8))) && wide_ok(k, type, 8) &&
                    wide_ok(v, type, 8) && t.rot % 16 == 0;
  return done(launch_append(t, paged(kv, chunks), type, kv->type, wide, stream_of(stream)), "nls_cache_append");
}

size_t nls_paged_attention_workspace(const nls_paged_kv* kv, const nls_chunks* chunks, int32_t heads, int32_t max_new,
                                     int64_t max_len, int32_t window) {
  if (check_sizes(kv, chunks, heads, max_new, max_len, window)) return 0;
  return align256(attend_workspace(attend_args(kv, chunks, heads, window), max_new, max_len));
}

int32_t nls_paged_attention(const nls_paged_kv* kv, const nls_chunks* chunks, int32_t type, const nls_heads* q,
                            const nls_heads* out, int32_t heads, float scale, int32_t window, const int32_t* d_first,
                            float* d_lse, int32_t max_new, int64_t max_len, void* d_work, size_t work_bytes,
                            void* stream) {
  NLS_CHECK(check_kv(kv));
  NLS_CHECK(check_chunks(chunks));
  NLS_CHECK(check_sizes(kv, chunks, heads, max_new, max_len, window));
  if (!elem_type(type) || (type != kF32 && type != kv->type))
    return bad("attention: q and out are F32, or of the cache's type");
  // (the kernels take exponents of base 2: an infinite factor times a score of 0 is NaN)
  if (!std::isfinite(scale * 1.4426950408889634f)) return bad("attention: scale, or scale times log2 e, is not finite");
  if (chunks->tokens == 0 || chunks->seqs == 0) return NLS_OK;
  NLS_CHECK(check_heads(q, type, heads, chunks->tokens, kv->head_dim, false));
  NLS_CHECK(check_heads(out, type, heads, chunks->tokens, kv->head_dim, true));
  if (!aligned(d_first, 4) || !aligned(d_lse, 4)) return bad("attention: misaligned first or lse");
  AttendArgs a = attend_args(kv, chunks, heads, window);
  a.q = view(q);
  a.out = view(out);
  a.scale = scale;
  a.first = d_first;
  a.lse = d_lse;
  const size_t need = align256(attend_workspace(a, max_new, max_len));
  if (need > 0 && (!d_work || work_bytes < need || !aligned(d_work, 256)))
    return bad("attention: workspace NULL, misaligned or too small");
  return done(launch_attend(a, type, kv->type, max_new, max_len, d_work, stream_of(stream)), "nls_paged_attention");
}

size_t nls_cache_workspace(const nls_page_tables* t, int32_t count) {
  if (!t || count < 0 || t->slots < 1 || t->pages < 1 || t->pages > kMaxPages) return 0;
  return align256(4 * page_words(t, count));
}

int32_t nls_cache_reserve(const nls_page_tables* t, const int32_t* d_counts, int32_t* d_status, void* d_work,
                          size_t work_bytes, void* stream) {
  NLS_CHECK(check_tables(t, true));
  NLS_CHECK(check_work(t, 0, d_work, work_bytes));
  if (!d_counts || !d_status || !aligned(d_counts, 4) || !aligned(d_status, 4)) return bad("reserve: NULL or misaligned");
  return done(launch_reserve(tables(t), d_counts, d_status, static_cast<int32_t*>(d_work), stream_of(stream)),
              "nls_cache_reserve");
}

int32_t nls_cache_fork(const nls_page_pool* p, const nls_page_tables* t, const int32_t* d_src, const int32_t* d_dst,
                       int32_t count, int32_t* d_status, void* d_work, size_t work_bytes, void* stream) {
  NLS_CHECK(check_tables(t, true));
  NLS_CHECK(check_pool(p, t->pages));
  if (count < 0 || count > t->slots) return bad("fork: count is negative or beyond the slots");
  NLS_CHECK(check_work(t, count, d_work, work_bytes));
  if (!d_status || !aligned(d_status, 4) || (count > 0 && (!d_src || !d_dst)) || !aligned(d_src, 4) || !aligned(d_dst, 4))
    return bad("fork: NULL or misaligned");
  return done(launch_fork(pool(p), tables(t), d_src, d_dst, count, d_status, static_cast<int32_t*>(d_work),
                          stream_of(stream)),
              "nls_cache_fork");
}

int32_t nls_cache_release(const nls_page_tables* t, const int32_t* d_slots, int32_t count, int32_t* d_status,
                          void* d_work, size_t work_bytes, void* stream) {
  NLS_CHECK(check_tables(t, true));
  if (count < 0) return bad("release: count is negative");
  NLS_CHECK(check_work(t, 0, d_work, work_bytes));
  if (!d_status || !aligned(d_status, 4) || (count > 0 && !d_slots) || !aligned(d_slots, 4))
    return bad("release: NULL or misaligned");
  return done(launch_release(tables(t), d_slots, count, d_status, stream_of(stream)),
              "nls_cache_release");
}

int32_t nls_cache_compact(const nls_page_pool* p, const nls_page_tables* t, int32_t* d_live, void* d_work,
                          size_t work_bytes, void* stream) {
  NLS_CHECK(check_tables(t, false));
  NLS_CHECK(check_pool(p, t->pages));
  NLS_CHECK(check_work(t, 0, d_work, work_bytes));
  if (!d_live || !aligned(d_live, 4)) return bad("compact: NULL or misaligned");
  return done(launch_compact(pool(p), tables(t), d_live, static_cast<int32_t*>(d_work), stream_of(stream)),
              "nls_cache_compact");
}

int32_t nls_cache_copy_pages(const nls_page_pool* p, int32_t pages, const int32_t* d_src, const int32_t* d_dst,
                             int32_t count, void* stream) {
  if (pages < 1 || count < 0) return bad("copy: a size out of range");
  NLS_CHECK(check_pool(p, pages));
  if (count == 0) return NLS_OK;
  if (!d_src || !d_dst || !aligned(d_src, 4) || !aligned(d_dst, 4)) return bad("copy: NULL or misaligned");
  return done(launch_copy_pages(pool(p), pages, d_src, d_dst, count, stream_of(stream)), "nls_cache_copy_pages");
}

}  // extern "C"
