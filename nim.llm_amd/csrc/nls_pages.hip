// nls_pages.hip -- pages of the cache: taken, shared, released, moved together.
//
// What decides which page goes where runs in one workgroup: the reference
// counts become a bitmap in LDS (a wave's ballot is 64 pages), the words'
// counts are summed once, and every page's rank among the free (or held) ones
// follows without another pass.  Reading 100 000 counts takes one workgroup a
// few microseconds; contents move in a launch of their own over the whole GPU,
// bound by their bytes: 2036 pages of 128 KB in each of 16 layers, 4.3 GB read
// and 4.3 written, 1.69 ms, 5.1 TB/s.  Nothing depends on the order in which workgroups
// run.
//
// Work area (int32): [0] pairs to move, then the ranks' pages or the pairs.
#include "nls_paged.h"

namespace nls {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;
constexpr int kCopyThreads = 256;
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

// out[r] = the r-th free page, r < count
__device__ void list_free(const uint64_t* bits, const int* ranks, int pages, int count, int32_t* out) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, words = (pages + 63) >> 6;
  for (int w = wave; w < words; w += kPlanWaves) {
    const uint64_t b = bits[w];
    const int r = ranks[w] + __popcll(b & ((uint64_t{1} << lane) - 1));
    if (((b >> lane) & 1) && r < count) out[r] = w * 64 + lane;
  }
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

// need[s]: the pages that slot s takes, base[s]: the rank of its first one
__global__ __launch_bounds__(kPlanThreads) void reserve_kernel(TableArgs t, const int32_t* counts, int32_t* status,
                                                               int32_t* work) {
  __shared__ int sh[kPlanWaves];
  const PlanLds lds = plan_lds(t.pages);
  int32_t* base = work;
  int32_t* ids = work + t.slots;
  const int64_t ps = int64_t{1} << t.page_shift;
  int total = 0, full = 0, bad = 0;
  for (int s0 = 0; s0 < t.slots; s0 += kPlanThreads) {
    const int s = s0 + threadIdx.x;
    int need = 0;
    if (s < t.slots) {
      const int64_t len = t.lens[s], n = counts[s];
      const int64_t have = (len + ps - 1) >> t.page_shift, want = (len + n + ps - 1) >> t.page_shift;
      if (n < 0 || len < 0)
        bad = 1;
      else if (want > t.max_pages || len + n > 0x7fffffff)
        full = 1;
      else
        need = (int)(want - have);
    }
    int sum;
    const int b = block_scan(need, sh, &sum);
    if (s < t.slots) base[s] = total + b;
    // (slots x max_pages is below 2^31, checked on the host)
    total += sum;
  }
  bad = __syncthreads_or(bad);
  full = __syncthreads_or(full);
  const int free_pages = free_bitmap(t.refs, t.pages, lds.bits, lds.ranks, sh);
  const int st = bad ? 3 : full ? 2 : free_pages < total ? 1 : 0;
  if (threadIdx.x == 0) *status = st;
  if (st) return;
  list_free(lds.bits, lds.ranks, t.pages, total, ids);
  __syncthreads();  // ids and base, written by other threads of this workgroup
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int s = wave; s < t.slots; s += kPlanWaves) {
    const int64_t len = t.lens[s], n = counts[s];
    if (n == 0) continue;
    const int have = (int)((len + ps - 1) >> t.page_shift), want = (int)((len + n + ps - 1) >> t.page_shift);
    for (int j = lane; j < want - have; j += 64) {
      const int page = ids[base[s] + j];
      t.table[s * t.table_stride + have + j] = page;
      t.refs[page] = 1;
    }
    if (lane == 0) t.lens[s] = (int)(len + n);
  }
}

// work: [0] pairs, [1 ..] sources, then destinations; then marks of the slots
__global__ __launch_bounds__(kPlanThreads) void fork_kernel(TableArgs t, const int32_t* src, const int32_t* dst,
                                                            int count, int32_t* status, int32_t* work) {
  __shared__ int sh[kPlanWaves];
  const PlanLds lds = plan_lds(t.pages);
  int32_t* from = work + 1;
  int32_t* to = from + count;
  int32_t* rank = to + count;
  int32_t* mark = rank + count;
  const int mask = (1 << t.page_shift) - 1;
  for (int s = threadIdx.x; s < t.slots; s += kPlanThreads) mark[s] = 0;
  __syncthreads();
  int bad = 0, full = 0;
  for (int i = threadIdx.x; i < count; i += kPlanThreads) {
    const int d = dst[i], s = src[i];
    if ((uint32_t)d >= (uint32_t)t.slots || (uint32_t)s >= (uint32_t)t.slots) {
      bad = 1;
      continue;
    }
    if (t.lens[d] != 0 || t.lens[s] < 0) bad = 1;
    if (((int64_t)t.lens[s] + mask) >> t.page_shift > t.max_pages) full = 1;
    if (atomicAdd(&mark[d], 1)) bad = 1;
  }
  bad = __syncthreads_or(bad);
  if (!bad)
    for (int i = threadIdx.x; i < count; i += kPlanThreads)
      // (an atomic reads where the atomics above wrote)
      if (atomicAdd(&mark[src[i]], 0)) bad = 1;
  bad = __syncthreads_or(bad);
  full = __syncthreads_or(full);
  int total = 0;
  if (!bad)
    for (int i0 = 0; i0 < count; i0 += kPlanThreads) {
      const int i = i0 + threadIdx.x;
      const int part = i < count && (t.lens[src[i]] & mask) != 0;
      int sum;
      const int b = block_scan(part, sh, &sum);
      if (i < count) rank[i] = part ? total + b : -1;
      total += sum;
    }
  const int free_pages = free_bitmap(t.refs, t.pages, lds.bits, lds.ranks, sh);
  const int st = bad ? 3 : full ? 2 : free_pages < total ? 1 : 0;
  if (threadIdx.x == 0) {
    *status = st;
    work[0] = st ? 0 : total;
  }
  if (st) return;
  list_free(lds.bits, lds.ranks, t.pages, total, to);
  __syncthreads();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int i = wave; i < count; i += kPlanWaves) {
    const int len = t.lens[src[i]], whole = len >> t.page_shift;
    const int32_t* a = t.table + src[i] * t.table_stride;
    int32_t* b = t.table + dst[i] * t.table_stride;
    for (int j = lane; j < whole; j += 64) {
      const int page = a[j];
      b[j] = page;
      if ((uint32_t)page < (uint32_t)t.pages) atomicAdd(&t.refs[page], 1);
    }
    if (lane == 0) {
      const int r = rank[i];
      if (r >= 0) {
        from[r] = a[whole];
        b[whole] = to[r];
        t.refs[to[r]] = 1;
      }
      t.lens[dst[i]] = len;
    }
  }
}

__global__ __launch_bounds__(kPlanThreads) void release_kernel(TableArgs t, const int32_t* slots, int count,
                                                               int32_t* status, int32_t* work) {
  int bad = 0;
  for (int i = threadIdx.x; i < count; i += kPlanThreads) bad |= (uint32_t)slots[i] >= (uint32_t)t.slots;
  bad = __syncthreads_or(bad);
  if (threadIdx.x == 0) *status = bad ? 3 : 0;
  if (bad) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int i = wave; i < count; i += kPlanWaves) {
    const int s = slots[i];
    int len = 0;
    if (lane == 0) len = atomicExch(&t.lens[s], 0);  // a slot named twice is one wave's
    len = __shfl(len, 0);
    int64_t n = ((int64_t)(len < 0 ? 0 : len) + (1 << t.page_shift) - 1) >> t.page_shift;
    if (n > t.max_pages) n = t.max_pages;
    for (int j = lane; j < n; j += 64) {
      const int page = t.table[s * t.table_stride + j];
      t.table[s * t.table_stride + j] = -1;
      if ((uint32_t)page < (uint32_t)t.pages) atomicSub(&t.refs[page], 1);
    }
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
// workgroups share when they are many.
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
    uint4 x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (o + k * 16 * kCopyThreads < p.page_bytes)
        x[k] = *reinterpret_cast<const uint4*>(from + o + k * 16 * kCopyThreads);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (o + k * 16 * kCopyThreads < p.page_bytes)
        *reinterpret_cast<uint4*>(to + o + k * 16 * kCopyThreads) = x[k];
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

hipError_t allow_lds(const void* f, int pages) {
  const size_t n = plan_lds_bytes(pages);
  return n > 60000 ? hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)n) : hipSuccess;
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

hipError_t launch_release(const TableArgs& t, const int32_t* slots, int count, int32_t* status, int32_t* work,
                          hipStream_t s) {
  release_kernel<<<1, kPlanThreads, 0, s>>>(t, slots, count, status, work);
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

hipError_t launch_copy_pages(const PoolArgs& p, int pages, const int32_t* src, const int32_t* dst, int count,
                             hipStream_t s) {
  copy_kernel<<<copy_blocks(copy_items(p, count)), kCopyThreads, 0, s>>>(p, pages, src, dst, nullptr, count);
  return hipGetLastError();
}

}  // namespace nls
