// nls_quant.h -- pages whose keys and values are blocks of 32 elements of a
// head: an fp16 factor d and a whole number c each, value d c.
//
//   Q8_0  c in -127 .. 127, held as c + 128 in a byte
//   Q4_0  c in -8 .. 7, held as c + 8 in half a byte
//
// (d is not negative; of a file's Q4_0 it may be, so that the largest element is
// always -8 d.  Here a block whose largest element is positive has that at 7 d: the
// mean square error of normal elements is 1.27 times theirs there and 1.14 over all.
// Attention counts on that sign: it compares factors as bits.)
//
// A page holds, for each kv head, its keys and then its values: the codes of
// page_size rows, then the factors, block by block, page_size of each (so that
// the factors of neighbouring tokens come in one load).  Within a row of codes
// the elements lie as the matrix cores take them, so that a lane's operands are
// one piece of the row:
//   keys    lane quarter g of a product over block x takes elements
//           32 x + 8 g + 0 .. 7; its units of all blocks are side by side
//   values  lane i takes element 32 x + i and 32 x + 16 + i of every block x:
//           those of four blocks are side by side, then of two, then of one
// The inline functions are plain C++ where hipcc is not the compiler.
#pragma once
#include <stddef.h>

#include "nls_paged.h"

namespace nls {

enum QuantType { kQ4_0 = 2, kQ8_0 = 8 };
constexpr int kMinQuantPage = 16;  // tokens

NLS_HD bool quant_type(int t) { return t == kQ4_0 || t == kQ8_0; }

struct QuantShape {
  int bits, groups;  // groups: blocks of a row
  int row;           // bytes of a row's codes
  int codes, half;   // of a page's codes of one head's keys (or values); with their factors
};
NLS_HD QuantShape quant_shape(int type, int dim, int page_size) {
  QuantShape s;
  s.bits = type == kQ8_0 ? 8 : 4;
  s.groups = dim / 32;
  s.row = dim * s.bits / 8;
  s.codes = page_size * s.row;
  s.half = s.codes + page_size * s.groups * 2;
  return s;
}
// k: 0 keys, 1 values
NLS_HD int64_t quant_base(const QuantShape& s, int head, int k) { return (int64_t)(head * 2 + k) * s.half; }
NLS_HD int64_t quant_page_bytes(const QuantShape& s, int kv_heads) { return (int64_t)kv_heads * 2 * s.half; }

// The planes of a row of values: n of them, the first groups / 4 four blocks wide.
struct Plane {
  int first, wide;  // blocks
};
NLS_HD int plane_count(int groups) { return groups / 4 + ((groups >> 1) & 1) + (groups & 1); }
NLS_HD Plane plane_of(int groups, int n) {
  Plane p;
  const int fours = groups / 4;
  if (n < fours) {
    p.first = n * 4;
    p.wide = 4;
  } else if (n == fours && (groups & 2)) {
    p.first = fours * 4;
    p.wide = 2;
  } else {
    p.first = groups - 1;
    p.wide = 1;
  }
  return p;
}
// Where lane i's piece of a plane begins in a row, and where the codes of key
// unit (block x, quarter g) do.
NLS_HD int value_at(const QuantShape& s, const Plane& p, int i) { return (p.first * 16 + i * p.wide) * s.bits / 4; }
NLS_HD int key_at(const QuantShape& s, int x, int g) { return (g * s.groups + x) * s.bits; }
// The place of a key unit's element e among the half bytes of its word: elements
// 2 n and 2 n + 1 are 16 bits apart.
NLS_HD int nibble_of(int e) { return e / 2 + 4 * (e & 1); }

#ifdef __HIPCC__
// Tokens of a workgroup: one where there are few, so that they run side by side;
// else enough that their look-ups, a chain of four loads, are one wait among many.
constexpr int kTokensMost = 8;
inline int tokens_of_group(int tokens) { return tokens < 2048 ? 1 : kTokensMost; }

struct TokenPlace {
  int seq;      // -1: the row is of no sequence
  int page;     // -1: none
  int64_t pos;  // in its slot
};
// Where tokens first .. first + n - 1 belong, by the first wave; a barrier is the
// caller's.
__device__ __forceinline__ void find_places(const PagedArgs& a, int first, int n, TokenPlace* places) {
  if (threadIdx.x >= 64) return;
  const int lane = threadIdx.x;
  // the starts not behind the first token, 64 at a time; then each lane goes on
  // from there for its own
  int seq = -1;
  for (int s0 = 0; s0 < a.seqs + 1; s0 += 64) {
    const int s = s0 + lane;
    const int m = __popcll(__ballot(s <= a.seqs && a.starts[s <= a.seqs ? s : a.seqs] <= first));
    seq += m;
    if (m < 64) break;
  }
  if (lane >= n) return;
  const int token = first + lane;
  while (seq < a.seqs && a.starts[seq + 1] <= token) ++seq;
  TokenPlace p{-1, -1, 0};
  if (seq >= 0 && seq < a.seqs) {
    const Chunk c = chunk_of(a, seq);
    p.seq = seq;
    p.pos = position_of(a, c, token - c.begin);
    p.page = page_of(a, c.slot, p.pos);
  }
  places[lane] = p;
}

// f(Width<blocks>) for a plane's width.
template <int W>
struct Width {
  __device__ constexpr operator int() const { return W; }
};
template <typename F>
__device__ __forceinline__ void by_width(int wide, F&& f) {
  if (wide == 4)
    f(Width<4>{});
  else if (wide == 2)
    f(Width<2>{});
  else
    f(Width<1>{});
}

// cache_append and cache_read over such pages (nls_rope.hip, nls_quant.hip)
hipError_t launch_append_quant(const TurnArgs& t, const PagedArgs& a, int type, int cache_type, bool wide, hipStream_t s);
struct ReadArgs {
  PagedArgs p;
  HeadsView k, v;
};
hipError_t launch_read(const ReadArgs& a, int type, int cache_type, bool wide, hipStream_t s);
#endif

}  // namespace nls
