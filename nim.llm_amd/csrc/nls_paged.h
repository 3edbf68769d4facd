// nls_paged.h -- what the kernels over the paged cache share: their arguments
// and the arithmetic of sequences, positions, pages and tiles.  The inline
// functions are plain C++ where hipcc is not the compiler, so that a program on
// the CPU can check them.
#pragma once
#include <stdint.h>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#define NLS_HD __host__ __device__ __forceinline__
#else
#define NLS_HD inline
#endif

namespace nls {

constexpr int kMaxHeadDim = 256;
constexpr int kMaxPageSize = 4096;
constexpr int kMaxLen = 0x7fffff00;  // tokens of a context: a step behind the last one is an int too
constexpr int kMaxPages = 1 << 19;  // one bit and half a bit of LDS each in the page kernels

enum ElemType { kF32 = 0, kF16 = 1, kBF16 = 30 };

// A layer of the cache and the batch of chunks (nls_paged_kv, nls_chunks).
struct PagedArgs {
  void* kv;
  int pages, page_shift, kv_heads, dim;
  int64_t page_stride, value_offset, head_stride, token_stride;
  const int32_t* table;
  int64_t table_stride;
  int slots, max_pages;
  const int32_t* lens;
  int seqs, tokens;
  const int32_t* starts;
  const int32_t* slot_of;
};

// A sequence of the batch: its rows of q and its slot's length, cut to what
// the arrays hold, whatever the device's numbers say.
struct Chunk {
  int slot;      // -1: no such slot
  int begin, n;  // rows of q
  int64_t len;   // tokens of the slot, the n new ones among them
};

NLS_HD Chunk chunk_of(const PagedArgs& a, int seq) {
  Chunk c;
  int b = a.starts[seq], e = a.starts[seq + 1];
  b = b < 0 ? 0 : b > a.tokens ? a.tokens : b;
  e = e < b ? b : e > a.tokens ? a.tokens : e;
  c.begin = b;
  c.n = e - b;
  c.slot = a.slot_of ? a.slot_of[seq] : seq;
  if (c.slot < 0 || c.slot >= a.slots) c.slot = -1;
  int64_t most = (int64_t)a.max_pages << a.page_shift;
  if (most > kMaxLen) most = kMaxLen;
  int64_t len = c.slot < 0 ? 0 : a.lens[c.slot];
  c.len = len < 0 ? 0 : len > most ? most : len;
  return c;
}

// The position of the sequence's i-th new token; negative where the slot is
// shorter than its new tokens say.  It goes by the slot's own length, so that
// a length beyond the table does not move the tokens that fit.
NLS_HD int64_t position_of(const PagedArgs& a, const Chunk& c, int i) {
  return c.slot < 0 ? -1 : (int64_t)a.lens[c.slot] - c.n + i;
}

// The page of a position of a slot, or -1 where there is none.
NLS_HD int page_of(const PagedArgs& a, int slot, int64_t pos) {
  if (slot < 0 || pos < 0 || (pos >> a.page_shift) >= a.max_pages) return -1;
  const int p = a.table[(int64_t)slot * a.table_stride + (pos >> a.page_shift)];
  return (uint32_t)p < (uint32_t)a.pages ? p : -1;
}

NLS_HD int64_t token_offset(const PagedArgs& a, int page, int64_t pos) {
  return (int64_t)page * a.page_stride + (pos & (((int64_t)1 << a.page_shift) - 1)) * a.token_stride;
}

// Tiles of `rows` (token, head of the group) rows: sequence s owns the tiles
// from tile_base(s) on.  tile_base rises by at least one tile per sequence and
// by at least as many as the sequence's rows fill, so no sums over the
// sequences before it are needed; some of the tiles are empty.
NLS_HD int64_t tile_base(int start, int group, int rows, int seq) {
  return (int64_t)(start < 0 ? 0 : start) * group / rows + seq;
}
NLS_HD int64_t tile_count(int tokens, int group, int rows, int seqs) {
  return (int64_t)tokens * group / rows + seqs;
}

constexpr int kMaxSlots = 1 << 16;  // of a page table: one bit of LDS each

// ---- rotary positions and the cache's writes (nls_rope.hip)

struct HeadsView {
  void* d;
  int64_t token_stride, head_stride;
};

struct TurnArgs {
  HeadsView x, y;  // q and its result (or rope's x and y); heads 0: none
  int heads, dim;
  const double* freqs;  // NULL: nothing is turned
  int rot, interleaved;
  float amplitude, sign;
  int tokens;
  const int32_t* positions;  // rope; the cache's positions otherwise
  HeadsView k, v;            // cache_append
};

#ifdef __HIPCC__
// wide: 8 elements at a time (rope's fp32: 4), where pointers, strides and the
// turned part allow it; else one
hipError_t launch_rope(const TurnArgs& t, int type, bool wide, hipStream_t s);
hipError_t launch_append(const TurnArgs& t, const PagedArgs& a, int type, int cache_type, bool wide, hipStream_t s);

// ---- pages (nls_pages.hip)

struct PoolArgs {
  char* kv;
  int layers;
  int64_t page_bytes, layer_stride, page_stride;
};
struct TableArgs {
  int32_t* table;
  int64_t table_stride;
  int slots, max_pages;
  int32_t* lens;
  int32_t* refs;
  int pages, page_shift;
};
hipError_t launch_reserve(const TableArgs& t, const int32_t* counts, int32_t* status, int32_t* work, hipStream_t s);
hipError_t launch_fork(const PoolArgs& p, const TableArgs& t, const int32_t* src, const int32_t* dst, int count,
                       int32_t* status, int32_t* work, hipStream_t s);
hipError_t launch_release(const TableArgs& t, const int32_t* slots, int count, int32_t* status, hipStream_t s);
hipError_t launch_compact(const PoolArgs& p, const TableArgs& t, int32_t* live, int32_t* work, hipStream_t s);
hipError_t launch_reorder(const PoolArgs& p, const TableArgs& t, const int32_t* src, int32_t* status, int32_t* work,
                          hipStream_t s);
hipError_t launch_copy_pages(const PoolArgs& p, int pages, const int32_t* src, const int32_t* dst, int count,
                             hipStream_t s);

// ---- attention (nls_attend.hip)

struct AttendArgs {
  PagedArgs p;
  int cache_type;
  HeadsView q, out;
  int heads, group;
  float scale;
  int window;
  const int32_t* first;
  float* lse;  // or NULL
};
hipError_t launch_attend(const AttendArgs& a, int type, int cache_type, int max_new, int64_t max_len, void* work,
                         hipStream_t s);
size_t attend_workspace(const AttendArgs& a, int max_new, int64_t max_len);
#endif

}  // namespace nls
