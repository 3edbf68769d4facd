// nls_pages.hip -- pages of the cache: taken, shared, released, moved together.
//
// What decides which page goes where runs in one workgroup: the reference
// counts become a bitmap in LDS (a wave's ballot is 64 pages), the words'
// counts are summed once, and every page's rank among the free (or held) ones
// follows without another pass.  Reading 100 000 counts takes one workgroup a
// few microseconds; contents move in a launch of their own over the whole GPU,
// bound by their bytes: 2036 pages of 128 KB in each of 16 layers, 4.3 GB read
// and 4.3 written, 1.66 ms, 5.1 TB/s.  Nothing depends on the order in which workgroups
// run.
//
// Work area (int32): [0] pairs to move, then the pairs; reserve's ranks.
#include "nls_paged.h"

namespace nls {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;
constexpr int kCopyThreads = 256;
typedef uint32_t Vec16 __attribute__((ext_vector_type(4)));
constexpr int kCopyBytes = 16 * 4 * kCopyThreads;  // of one page, per step of a workgroup

// Exclusive prefix sum of one value per thread; *total is the sum.
__device__ int block_scan(int x, int* sh, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int s = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(s, d);
    if (lane >= d) s += y;
  }
  __syncthreads();  // sh may hold an earlier scan's sums
  if (lane == 63) sh[wave] = s;
  __syncthreads();
  int base = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < kPlanWaves; ++w) {
    if (w < wave) base += sh[w];
    sum += sh[w];
  }
  *total = sum;
  return base + s - x;
}

// ranks[w]: how many bits of bits[0 .. w) are set.  Returns how many are in all.
__device__ int rank_bitmap(int words, const uint64_t* bits, int* ranks, int* sh) {
  const int per = (words + kPlanThreads - 1) / kPlanThreads, w0 = threadIdx.x * per;
  int n = 0;
  for (int i = 0; i < per; ++i)
    if (w0 + i < words) n += __popcll(bits[w0 + i]);
  int total;
  int r = block_scan(n, sh, &total);
  for (int i = 0; i < per; ++i)
    if (w0 + i < words) {
      ranks[w0 + i] = r;
      r += __popcll(bits[w0 + i]);
    }
  __syncthreads();
  return total;
}

// bits[w]: the free pages among 64 w .. 64 w + 63; ranks[w]: how many are free
// below them.  Returns the number of free pages.
__device__ int free_bitmap(const int32_t* refs, int pages, uint64_t* bits, int* ranks, int* sh) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, words = (pages + 63) >> 6;
  for (int w = wave; w < words; w += kPlanWaves) {
    const int p = w * 64 + lane;
    const uint64_t b = __ballot(p < pages && refs[p < pages ? p : 0] == 0);
    if (lane == 0) bits[w] = b;
  }
  __syncthreads();
  return rank_bitmap(words, bits, ranks, sh);
}

// The r-th free page, r below their number: the last word with no more than r
// free pages before it, then the bit.  Each thread finds its own, so that no list
// goes through memory.
__device__ int free_page(const uint64_t* bits, const int* ranks, int pages, int r) {
  int lo = 0, hi = ((pages + 63) >> 6) - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (ranks[mid] <= r)
      lo = mid;
    else
      hi = mid - 1;
  }
  // (words without a free page have the rank of the next: the search ends behind them)
  uint64_t b = bits[lo];
  int n = r - ranks[lo], at = 0;
#pragma unroll
  for (int w = 32; w; w >>= 1) {
    const int below = __popcll(b & ((uint64_t{1} << w) - 1));
    if (n >= below) {
      n -= below;
      b >>= w;
      at += w;
    }
  }
  return lo * 64 + at;
}

struct PlanLds {
  uint64_t* bits;
  int* ranks;
};
__device__ PlanLds plan_lds(int pages) {
  extern __shared__ uint64_t plan_words[];
  const int words = (pages + 63) >> 6;
  return {plan_words, reinterpret_cast<int*>(plan_words + words)};
}
size_t plan_lds_bytes(int pages) { return (size_t)((pages + 63) >> 6) * 12; }

// Slots by kPlanThreads: what each takes and the rank of its first page among
// the free ones (first in `work` where there are more slots than threads).
__global__ __launch_bounds__(kPlanThreads) void reserve_kernel(TableArgs t, const int32_t* counts, int32_t* status,
                                                               int32_t* work) {
  __shared__ int sh[kPlanWaves];
  __shared__ int s_len[kPlanThreads], s_take[kPlanThreads], s_base[kPlanThreads];
  const PlanLds lds = plan_lds(t.pages);
  const int ps = 1 << t.page_shift;
  int total = 0, full = 0, bad = 0;
  for (int s0 = 0; s0 < t.slots; s0 += kPlanThreads) {
    const int s = s0 + threadIdx.x;
    int need = 0, len = 0, n = 0;
    if (s < t.slots) {
      len = t.lens[s];
      n = counts[s];
      const int64_t have = ((int64_t)len + ps - 1) >> t.page_shift, want = ((int64_t)len + n + ps - 1) >> t.page_shift;
      if (n < 0 || len < 0)
        bad = 1;
      else if (want > t.max_pages || (int64_t)len + n > 0x7fffffff)
        full = 1;
      else
        need = (int)(want - have);
    }
    int sum;
    const int b = total + block_scan(need, sh, &sum);
    s_len[threadIdx.x] = len;
    s_take[threadIdx.x] = n;
    s_base[threadIdx.x] = b;
    if (s < t.slots) work[s] = b;
    // (slots x max_pages is below 2^31, checked on the host)
    total += sum;
  }
  const int free_pages = free_bitmap(t.refs, t.pages, lds.bits, lds.ranks, sh);
  bad = __syncthreads_or(bad);
  full = __syncthreads_or(full);
  const int st = bad ? 3 : full ? 2 : free_pages < total ? 1 : 0;
  if (threadIdx.x == 0) *status = st;
  if (st) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int s0 = 0; s0 < t.slots; s0 += kPlanThreads) {
    if (t.slots > kPlanThreads) {  // more than LDS holds: again, a block at a time
      __syncthreads();
      const int s = s0 + threadIdx.x;
      if (s < t.slots) {
        s_len[threadIdx.x] = t.lens[s];
        s_take[threadIdx.x] = counts[s];
        s_base[threadIdx.x] = work[s];
      }
      __syncthreads();
    }
    const int here = t.slots - s0 < kPlanThreads ? t.slots - s0 : kPlanThreads;
    for (int i = wave; i < here; i += kPlanWaves) {
      const int len = s_len[i], n = s_take[i], s = s0 + i;
      if (n == 0) continue;
      const int have = (int)(((int64_t)len + ps - 1) >> t.page_shift);
      const int want = (int)(((int64_t)len + n + ps - 1) >> t.page_shift);
      for (int j = lane; j < want - have; j += 64) {
        const int page = free_page(lds.bits, lds.ranks, t.pages, s_base[i] + j);
        t.table[s * t.table_stride + have + j] = page;
        t.refs[page] = 1;
      }
      if (lane == 0) t.lens[s] = len + n;
    }
  }
}

// Forks by kPlanThreads.  work: [0] pairs to copy, [1 ..] sources, then
// destinations.
__global__ __launch_bounds__(kPlanThreads) void fork_kernel(TableArgs t, const int32_t* src, const int32_t* dst,
                                                            int count, int32_t* status, int32_t* work) {
  __shared__ int sh[kPlanWaves];
  __shared__ uint32_t mark[kMaxSlots / 32];  // the slots that are destinations
  __shared__ int s_src[kPlanThreads], s_dst[kPlanThreads], s_len[kPlanThreads], s_rank[kPlanThreads];
  const PlanLds lds = plan_lds(t.pages);
  int32_t* from = work + 1;
  int32_t* to = from + count;
  const int mask = (1 << t.page_shift) - 1;
  for (int i = threadIdx.x; i < (t.slots + 31) / 32; i += kPlanThreads) mark[i] = 0;
  __syncthreads();
  int bad = 0, full = 0, total = 0;
  for (int i = threadIdx.x; i < count; i += kPlanThreads) {
    const int d = dst[i];
    if ((uint32_t)d >= (uint32_t)t.slots || (uint32_t)src[i] >= (uint32_t)t.slots)
      bad = 1;
    else if (atomicOr(&mark[d >> 5], 1u << (d & 31)) >> (d & 31) & 1)
      bad = 1;  // named twice
  }
  const int free_pages = free_bitmap(t.refs, t.pages, lds.bits, lds.ranks, sh);  // (its barriers end the marking)
  for (int i0 = 0; i0 < count; i0 += kPlanThreads) {
    const int i = i0 + threadIdx.x;
    int s = 0, d = 0, len = 0;
    if (i < count) {
      s = src[i];
      d = dst[i];
      if ((uint32_t)d < (uint32_t)t.slots && (uint32_t)s < (uint32_t)t.slots) {
        len = t.lens[s];
        if (t.lens[d] != 0 || len < 0 || (mark[s >> 5] >> (s & 31) & 1)) bad = 1;
        if (((int64_t)len + mask) >> t.page_shift > t.max_pages) full = 1;
      }
    }
    int sum;
    const int part = (len & mask) != 0, r = total + block_scan(part, sh, &sum);
    s_src[threadIdx.x] = s;
    s_dst[threadIdx.x] = d;
    s_len[threadIdx.x] = len;
    s_rank[threadIdx.x] = r;
    total += sum;
  }
  bad = __syncthreads_or(bad);
  full = __syncthreads_or(full);
  const int st = bad ? 3 : full ? 2 : free_pages < total ? 1 : 0;
  if (threadIdx.x == 0) {
    *status = st;
    work[0] = st ? 0 : total;
  }
  if (st) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int before = 0;
  for (int i0 = 0; i0 < count; i0 += kPlanThreads) {
    if (count > kPlanThreads) {  // more than LDS holds: again, a block at a time
      const int i = i0 + threadIdx.x;
      const int len = i < count ? t.lens[src[i]] : 0;
      int sum;
      const int r = before + block_scan((len & mask) != 0, sh, &sum);
      s_src[threadIdx.x] = i < count ? src[i] : 0;
      s_dst[threadIdx.x] = i < count ? dst[i] : 0;
      s_len[threadIdx.x] = len;
      s_rank[threadIdx.x] = r;
      before += sum;
      __syncthreads();
    }
    const int here = count - i0 < kPlanThreads ? count - i0 : kPlanThreads;
    for (int i = wave; i < here; i += kPlanWaves) {
      const int len = s_len[i], whole = len >> t.page_shift;
      const int32_t* a = t.table + s_src[i] * t.table_stride;
      int32_t* b = t.table + s_dst[i] * t.table_stride;
      const bool part = (len & mask) != 0;
      for (int j = lane; j < whole + part; j += 64) {
        const int page = a[j];
        if (j < whole) {
          b[j] = page;
          if ((uint32_t)page < (uint32_t)t.pages) atomicAdd(&t.refs[page], 1);
        } else {
          const int r = s_rank[i], mine = free_page(lds.bits, lds.ranks, t.pages, r);
          from[r] = page;
          to[r] = mine;
          b[j] = mine;
          t.refs[mine] = 1;
        }
      }
      if (lane == 0) t.lens[s_dst[i]] = len;
    }
    if (count > kPlanThreads) __syncthreads();  // the next block's numbers take the same LDS
  }
}

__global__ __launch_bounds__(kPlanThreads) void release_kernel(TableArgs t, const int32_t* slots, int count,
                                                               int32_t* status) {
  __shared__ int s_slot[kPlanThreads], s_len[kPlanThreads];
  int bad = 0;
  for (int i = threadIdx.x; i < count; i += kPlanThreads) bad |= (uint32_t)slots[i] >= (uint32_t)t.slots;
  bad = __syncthreads_or(bad);
  if (threadIdx.x == 0) *status = bad ? 3 : 0;
  if (bad) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int i0 = 0; i0 < count; i0 += kPlanThreads) {
    const int i = i0 + threadIdx.x;
    if (i < count) {
      s_slot[threadIdx.x] = slots[i];
      s_len[threadIdx.x] = atomicExch(&t.lens[slots[i]], 0);  // a slot named twice has its length once
    }
    __syncthreads();
    const int here = count - i0 < kPlanThreads ? count - i0 : kPlanThreads;
    for (int e = wave; e < here; e += kPlanWaves) {
      const int len = s_len[e];
      int32_t* row = t.table + s_slot[e] * t.table_stride;
      int64_t n = ((int64_t)(len < 0 ? 0 : len) + (1 << t.page_shift) - 1) >> t.page_shift;
      if (n > t.max_pages) n = t.max_pages;
      for (int j = lane; j < n; j += 64) {
        const int page = row[j];
        row[j] = -1;
        if ((uint32_t)page < (uint32_t)t.pages) atomicSub(&t.refs[page], 1);
      }
    }
    __syncthreads();  // the next block's numbers take the same LDS
  }
}

// work: [0] pairs, [1 ..] sources, then destinations, then each page's place
__global__ __launch_bounds__(kPlanThreads) void compact_kernel(TableArgs t, int32_t* live_out, int32_t* work) {
  __shared__ int sh[kPlanWaves];
  const PlanLds lds = plan_lds(t.pages);
  int32_t* from = work + 1;
  int32_t* to = from + t.pages;
  int32_t* place = to + t.pages;
  const int free_pages = free_bitmap(t.refs, t.pages, lds.bits, lds.ranks, sh);
  const int live = t.pages - free_pages;
  // free pages below `live`: as many as held ones from there on
  const int edge = live >> 6;
  int moves = 0;
  if (live < t.pages) moves = lds.ranks[edge] + __popcll(lds.bits[edge] & ((uint64_t{1} << (live & 63)) - 1));
  const int held_below = live - moves;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, words = (t.pages + 63) >> 6;
  for (int w = wave; w < words; w += kPlanWaves) {
    const int p = w * 64 + lane;
    if (p >= t.pages) continue;
    const uint64_t b = lds.bits[w];
    const int r = lds.ranks[w] + __popcll(b & ((uint64_t{1} << lane) - 1));
    const bool is_free = (b >> lane) & 1;
    if (is_free && p < live) to[r] = p;
    if (!is_free && p >= live) from[(p - r) - held_below] = p;
    place[p] = p;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < moves; i += kPlanThreads) {
    const int a = from[i], b = to[i];
    place[a] = b;
    t.refs[b] = t.refs[a];
    t.refs[a] = 0;
  }
  if (threadIdx.x == 0) {
    work[0] = moves;
    *live_out = live;
  }
}

// One page of one layer after another: pair (i, layer), whose bytes several
// workgroups share when they are many.  Stores are non-temporal: with ordinary
// ones the launch's end waits for the copies to leave L2 (48 forks, reserve
// and release, 50 MB copied: 58.5 us, with them 44.8; non-temporal loads too
// 46.7).  Four loads of a thread go out together: two or eight cost more where
// many pages move (2036 pages in 16 layers: 1.68 ms, 1.75 and 2.62).
__device__ void copy_pairs(const PoolArgs& p, int pages, const int32_t* src, const int32_t* dst, int pairs, int block,
                           int blocks) {
  const int parts = (int)((p.page_bytes + kCopyBytes - 1) / kCopyBytes);
  const int64_t items = (int64_t)pairs * p.layers * parts;
  for (int64_t it = block; it < items; it += blocks) {
    const int part = (int)(it % parts);
    const int64_t rest = it / parts;
    const int layer = (int)(rest % p.layers), i = (int)(rest / p.layers);
    const int a = src[i], b = dst[i];
    if ((uint32_t)a >= (uint32_t)pages || (uint32_t)b >= (uint32_t)pages) continue;
    const char* from = p.kv + layer * p.layer_stride + a * p.page_stride;
    char* to = p.kv + layer * p.layer_stride + b * p.page_stride;
    const int64_t o = (int64_t)part * kCopyBytes + threadIdx.x * 16;
    Vec16 x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (o + k * 16 * kCopyThreads < p.page_bytes)
        x[k] = *reinterpret_cast<const Vec16*>(from + o + k * 16 * kCopyThreads);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (o + k * 16 * kCopyThreads < p.page_bytes)
        __builtin_nontemporal_store(x[k], reinterpret_cast<Vec16*>(to + o + k * 16 * kCopyThreads));
  }
}

__global__ __launch_bounds__(kCopyThreads) void copy_kernel(PoolArgs p, int pages, const int32_t* src,
                                                            const int32_t* dst, const int32_t* n, int count) {
  copy_pairs(p, pages, src, dst, n ? *n : count, blockIdx.x, gridDim.x);
}

// Compaction's second launch: the table's entries, then the pages' contents.
__global__ __launch_bounds__(kCopyThreads) void move_kernel(PoolArgs p, TableArgs t, const int32_t* work,
                                                            int table_blocks) {
  if ((int)blockIdx.x < table_blocks) {
    const int32_t* place = work + 1 + 2 * (int64_t)t.pages;
    const int64_t n = (int64_t)t.slots * t.max_pages;
    for (int64_t i = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x; i < n; i += (int64_t)table_blocks * kCopyThreads) {
      int32_t* e = t.table + i / t.max_pages * t.table_stride + i % t.max_pages;
      const int page = *e;
      if ((uint32_t)page < (uint32_t)t.pages && place[page] != page) *e = place[page];
    }
    return;
  }
  copy_pairs(p, t.pages, work + 1, work + 1 + t.pages, work[0], blockIdx.x - table_blocks, gridDim.x - table_blocks);
}

// Where reorder's work area has what: [0] the status, [1] pairs to copy, then
// their sources and destinations, each slot's old length, the page its partial
// last one is copied to (-1: none), its first child, how many entries let go of a
// page (of those whose count is above 1), and the old table.
struct ReorderWork {
  int32_t *head, *from, *to, *len, *fresh, *first, *gone, *rows;
  __device__ __host__ ReorderWork(int32_t* w, int slots, int pages)
      : head(w), from(w + 2), to(from + slots), len(to + slots), fresh(len + slots), first(fresh + slots),
        gone(first + slots), rows(gone + pages) {}
};
// Pages of a context (whose length may be all that an int holds).
__device__ __forceinline__ int pages_of(int len, int shift) { return (int)(((uint32_t)len + ((1u << shift) - 1)) >> shift); }
// (written by this workgroup before a barrier, with atomics among it)
__device__ __forceinline__ int settled(const int32_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// What goes where.  A page is free for a copy when nobody held it, or only
// slots whose contexts end here: it is marked by those, and the mark is taken off
// by every row as it will be.  Where its count is above the entries that let go of it
// someone else holds it, outside of these rows: those of a count above 1 are counted,
// if any is marked still (which LDS tells for up to 65536 pages: 2 us of 78 less).  The first workgroup: what bounds it are the two passes
// over the table: a wave takes eight rows at a time, with the slots' numbers in LDS
// (512 slots of 73 entries: 47 us when entries are dealt out to threads by a
// division each, 33 by rows, 30 since the other workgroups keep the table).
constexpr int kSlotsHeld = 2048, kWordsHeld = 1024;
__global__ __launch_bounds__(kPlanThreads) void reorder_kernel(TableArgs t, const int32_t* src, int32_t* status,
                                                               int32_t* work) {
  __shared__ int sh[kPlanWaves];
  __shared__ int s_src[kSlotsHeld], s_len[kSlotsHeld], s_first[kSlotsHeld];
  __shared__ uint64_t s_many[kWordsHeld];  // pages of counts above 1
  const PlanLds lds = plan_lds(t.pages);
  const ReorderWork w(work, t.slots, t.pages);
  if (blockIdx.x > 0) {  // the table as it was, by the other workgroups
    const uint32_t n = (uint32_t)t.slots * (uint32_t)t.max_pages, per = t.max_pages;  // (below 2^31)
    for (uint32_t e = (blockIdx.x - 1) * kPlanThreads + threadIdx.x; e < n; e += (gridDim.x - 1) * kPlanThreads)
      w.rows[e] = t.table[(int64_t)(e / per) * t.table_stride + e % per];
    return;
  }
  const int mask = (1 << t.page_shift) - 1;
  const bool held = t.slots <= kSlotsHeld;
  int bad = 0;
  for (int s = threadIdx.x; s < t.slots; s += kPlanThreads) {
    const int len = t.lens[s], p = src[s];
    if (p < -1 || p >= t.slots || len < 0 || ((int64_t)len + mask) >> t.page_shift > t.max_pages) bad = 1;
    w.len[s] = len;
    if (held) {
      s_src[s] = p;
      s_len[s] = len;
      s_first[s] = t.slots;
    } else {
      __hip_atomic_store(&w.first[s], t.slots, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  bad = __syncthreads_or(bad);
  if (bad) {
    if (threadIdx.x == 0) *status = w.head[0] = 3;
    return;
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, words = (t.pages + 63) >> 6;
  // f(word, this lane's page, its count) for all words of the bitmap
  auto over_counts = [&](auto f) {
    constexpr int kWords = 8;
    for (int i0 = wave * kWords; i0 < words; i0 += kPlanWaves * kWords) {
      int refs[kWords];
#pragma unroll
      for (int u = 0; u < kWords; ++u) {
        const int p = (i0 + u) * 64 + lane;
        refs[u] = p < t.pages ? t.refs[p] : 1;
      }
#pragma unroll
      for (int u = 0; u < kWords; ++u)
        if (i0 + u < words) f(i0 + u, (i0 + u) * 64 + lane, refs[u]);
    }
  };
  over_counts([&](int word, int, int refs) {
    const uint64_t b = __ballot(refs == 0), many = __ballot(refs > 1);
    if (lane == 0) lds.bits[word] = b;
    if (lane == 0 && word < kWordsHeld) s_many[word] = many;
  });
  // the partial page of a parent stays with itself, else with its first child
  for (int s = threadIdx.x; s < t.slots; s += kPlanThreads) {
    const int p = held ? s_src[s] : src[s];
    if (p >= 0) atomicMin(held ? &s_first[p] : &w.first[p], p == s ? -1 : s);
  }
  __syncthreads();
  auto src_of = [&](int s) { return held ? s_src[s] : src[s]; };
  auto len_of = [&](int s) { return held ? s_len[s] : w.len[s]; };
  auto first_of = [&](int s) { return held ? s_first[s] : settled(&w.first[s]); };
  uint32_t* marks = reinterpret_cast<uint32_t*>(lds.bits);
  // f(page) for the entries of the rows that end here: eight rows at a time to a
  // wave, 128 entries of each
  constexpr int kRows = 8, kCols = 2;
  auto over_ending = [&](auto f) {
    for (int s0 = wave * kRows; s0 < t.slots; s0 += kPlanWaves * kRows) {
      int used[kRows], most = 0;
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        const int s = s0 + u;
        used[u] = s < t.slots && src_of(s) != s ? pages_of(len_of(s), t.page_shift) : 0;
        most = used[u] > most ? used[u] : most;
      }
      for (int j0 = lane; j0 < most; j0 += 64 * kCols) {
        int page[kRows][kCols];
#pragma unroll
        for (int u = 0; u < kRows; ++u)
#pragma unroll
          for (int c = 0; c < kCols; ++c) {
            const int j = j0 + 64 * c;
            page[u][c] = j < used[u] ? t.table[(s0 + u) * t.table_stride + j] : -1;
          }
#pragma unroll
        for (int u = 0; u < kRows; ++u)
#pragma unroll
          for (int c = 0; c < kCols; ++c)
            if ((uint32_t)page[u][c] < (uint32_t)t.pages) f(page[u][c]);
      }
    }
  };
  over_ending([&](int p) { atomicOr(&marks[p >> 5], 1u << (p & 31)); });
  __syncthreads();
  for (int s0 = wave * kRows; s0 < t.slots; s0 += kPlanWaves * kRows) {
    int from[kRows], keep[kRows], most = 0;
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const int s = s0 + u;
      from[u] = s < t.slots ? src_of(s) : -1;
      keep[u] = 0;
      if (from[u] >= 0) {
        // (a parent's pages once, by the child that keeps them all)
        if (from[u] == s || first_of(from[u]) == s) keep[u] = pages_of(len_of(from[u]), t.page_shift);
      }
      most = keep[u] > most ? keep[u] : most;
    }
    for (int j0 = lane; j0 < most; j0 += 64 * kCols) {
      int page[kRows][kCols];
#pragma unroll
      for (int u = 0; u < kRows; ++u)
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          const int j = j0 + 64 * c;
          page[u][c] = j < keep[u] ? t.table[from[u] * t.table_stride + j] : -1;
        }
#pragma unroll
      for (int u = 0; u < kRows; ++u)
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          const int p = page[u][c];
          if ((uint32_t)p < (uint32_t)t.pages) atomicAnd(&marks[p >> 5], ~(1u << (p & 31)));
        }
    }
  }
  __syncthreads();
  int several = words > kWordsHeld;
  if (!several)
    for (int i = threadIdx.x; i < words; i += kPlanThreads) several |= (lds.bits[i] & s_many[i]) != 0;
  if (__syncthreads_or(several)) {
    over_counts([&](int word, int p, int refs) {
      if (refs > 1 && (lds.bits[word] >> lane) & 1)
        __hip_atomic_store(&w.gone[p], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    });
    __syncthreads();
    over_ending([&](int p) {
      if (((marks[p >> 5] >> (p & 31)) & 1) && t.refs[p] > 1) atomicAdd(&w.gone[p], 1);
    });
    __syncthreads();
    over_counts([&](int word, int p, int refs) {
      const bool mine = refs > 1 && (lds.bits[word] >> lane) & 1;
      const uint64_t stays = __ballot(mine && settled(&w.gone[mine ? p : 0]) < refs);
      if (lane == 0) lds.bits[word] &= ~stays;
    });
    __syncthreads();
  }
  const int free_pages = rank_bitmap(words, lds.bits, lds.ranks, sh);
  int total = 0;
  for (int s0 = 0; s0 < t.slots; s0 += kPlanThreads) {
    const int s = s0 + threadIdx.x;
    int copies = 0, p = -1, len = 0;
    if (s < t.slots && (p = src_of(s)) >= 0) {
      len = len_of(p);
      copies = (len & mask) != 0 && p != s && first_of(p) != s;
    }
    int sum;
    const int r = total + block_scan(copies, sh, &sum);
    if (s < t.slots) {
      int mine = -1;
      if (copies && r < free_pages) {
        mine = free_page(lds.bits, lds.ranks, t.pages, r);
        w.from[r] = t.table[(int64_t)p * t.table_stride + (len >> t.page_shift)];
        w.to[r] = mine;
      }
      w.fresh[s] = mine;
    }
    total += sum;
  }
  if (threadIdx.x == 0) {
    const int st = free_pages < total ? 1 : 0;
    *status = w.head[0] = st;
    w.head[1] = st ? 0 : total;
  }
}

// The tables as planned, and the copies.
__global__ __launch_bounds__(kCopyThreads) void reorder_apply_kernel(PoolArgs p, TableArgs t, const int32_t* src,
                                                                     int32_t* work, int table_blocks) {
  const ReorderWork w(work, t.slots, t.pages);
  if (w.head[0]) return;
  if ((int)blockIdx.x >= table_blocks) {
    copy_pairs(p, t.pages, w.from, w.to, w.head[1], blockIdx.x - table_blocks, gridDim.x - table_blocks);
    return;
  }
  const uint32_t n = (uint32_t)t.slots * (uint32_t)t.max_pages, per = t.max_pages;  // (below 2^31)
  for (uint32_t e = blockIdx.x * kCopyThreads + threadIdx.x; e < n; e += table_blocks * kCopyThreads) {
    const int s = (int)(e / per), j = (int)(e % per), from = src[s];
    if (from == s) continue;
    const int had = pages_of(w.len[s], t.page_shift), len = from < 0 ? 0 : w.len[from];
    const int whole = len >> t.page_shift, has = pages_of(len, t.page_shift);
    if (j == 0) t.lens[s] = len;
    if (j >= had && j >= has) continue;
    const int was = j < had ? w.rows[e] : -1;
    int page = -1;
    if (j < has) page = j < whole || w.fresh[s] < 0 ? w.rows[(int64_t)from * t.max_pages + j] : w.fresh[s];
    if (page == was) continue;
    t.table[(int64_t)s * t.table_stride + j] = page;
    if ((uint32_t)was < (uint32_t)t.pages) atomicSub(&t.refs[was], 1);
    if ((uint32_t)page < (uint32_t)t.pages) atomicAdd(&t.refs[page], 1);
  }
}

hipError_t allow_lds(const void* f, int pages) {
  const size_t n = plan_lds_bytes(pages);
  return n > 32000 ? hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)n) : hipSuccess;
}

// Workgroups that copy `items` pieces of kCopyBytes: all at once up to what
// fills the GPU, then one after another.
int copy_blocks(int64_t items) { return (int)(items < 1 ? 1 : items > 2048 ? 2048 : items); }
int64_t copy_items(const PoolArgs& p, int64_t pairs) {
  return pairs * p.layers * ((p.page_bytes + kCopyBytes - 1) / kCopyBytes);
}

}  // namespace

hipError_t launch_reserve(const TableArgs& t, const int32_t* counts, int32_t* status, int32_t* work, hipStream_t s) {
  const hipError_t e = allow_lds(reinterpret_cast<const void*>(reserve_kernel), t.pages);
  if (e != hipSuccess) return e;
  reserve_kernel<<<1, kPlanThreads, plan_lds_bytes(t.pages), s>>>(t, counts, status, work);
  return hipGetLastError();
}

hipError_t launch_fork(const PoolArgs& p, const TableArgs& t, const int32_t* src, const int32_t* dst, int count,
                       int32_t* status, int32_t* work, hipStream_t s) {
  hipError_t e = allow_lds(reinterpret_cast<const void*>(fork_kernel), t.pages);
  if (e != hipSuccess) return e;
  fork_kernel<<<1, kPlanThreads, plan_lds_bytes(t.pages), s>>>(t, src, dst, count, status, work);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  copy_kernel<<<copy_blocks(copy_items(p, count)), kCopyThreads, 0, s>>>(p, t.pages, work + 1, work + 1 + count, work,
                                                                         0);
  return hipGetLastError();
}

hipError_t launch_release(const TableArgs& t, const int32_t* slots, int count, int32_t* status, hipStream_t s) {
  release_kernel<<<1, kPlanThreads, 0, s>>>(t, slots, count, status);
  return hipGetLastError();
}

hipError_t launch_compact(const PoolArgs& p, const TableArgs& t, int32_t* live, int32_t* work, hipStream_t s) {
  hipError_t e = allow_lds(reinterpret_cast<const void*>(compact_kernel), t.pages);
  if (e != hipSuccess) return e;
  compact_kernel<<<1, kPlanThreads, plan_lds_bytes(t.pages), s>>>(t, live, work);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  const int64_t entries = (int64_t)t.slots * t.max_pages;
  const int tb = (int)(entries < 1 ? 0 : entries > 64 * kCopyThreads * 8 ? 64 : (entries + kCopyThreads * 8 - 1) / (kCopyThreads * 8));
  // (at most half of the pages move)
  move_kernel<<<tb + copy_blocks(copy_items(p, (t.pages + 1) / 2)), kCopyThreads, 0, s>>>(p, t, work, tb);
  return hipGetLastError();
}

hipError_t launch_reorder(const PoolArgs& p, const TableArgs& t, const int32_t* src, int32_t* status, int32_t* work,
                          hipStream_t s) {
  hipError_t e = allow_lds(reinterpret_cast<const void*>(reorder_kernel), t.pages);
  if (e != hipSuccess) return e;
  const int64_t entries = (int64_t)t.slots * t.max_pages;
  const int copying = (int)(entries > 64 * kPlanThreads ? 64 : (entries + kPlanThreads - 1) / kPlanThreads);
  reorder_kernel<<<1 + copying, kPlanThreads, plan_lds_bytes(t.pages), s>>>(t, src, status, work);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  const int tb = (int)(entries > 256 * kCopyThreads ? 256 : (entries + kCopyThreads - 1) / kCopyThreads);
  reorder_apply_kernel<<<tb + copy_blocks(copy_items(p, t.slots)), kCopyThreads, 0, s>>>(p, t, src, work, tb);
  return hipGetLastError();
}

hipError_t launch_copy_pages(const PoolArgs& p, int pages, const int32_t* src, const int32_t* dst, int count,
                             hipStream_t s) {
  copy_kernel<<<copy_blocks(copy_items(p, count)), kCopyThreads, 0, s>>>(p, pages, src, dst, nullptr, count);
  return hipGetLastError();
}

}  // namespace nls
