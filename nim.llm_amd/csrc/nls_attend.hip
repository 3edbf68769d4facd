// nls_attend.hip -- attention of chunks of new tokens over the paged cache.
//
//   s_j = scale q . k_j,  m = max s_j,  o = sum exp(s_j - m) v_j / sum exp(s_j - m)
//
// in one pass over the keys with a running maximum: when it rises by t, what
// was summed so far shrinks by exp(-t).  Exponents are base 2, of
// (scale log2 e) q . k.
//
// Rows of one kv head's group share its keys, so a tile of rows is (token,
// head of the group) pairs and the products run on the matrix cores.  All
// products are taken transposed, S^T = K Q^T and O^T = V^T P^T: then a lane
// holds one row's scores (its column of S^T), its statistics are one register,
// and the weights are in place as the right operand of the second product.
// That product's depth is the keys in any order, so a lane's scores serve as
// they lie: with g = lane / 16, it holds keys 4 g .. 4 g + 3 of each 16.
//
// fp32 queries over a 16-bit cache: keys and values are what the cache holds,
// exactly; queries and weights are split into 2 (fp16) or 3 (bf16) parts of
// that type, each with a product of its own, so that nothing is rounded to 16
// bits.  An fp32 cache goes through the fp32 products (16 x 16 x 4).
#include "nls_attend.h"

namespace nls {
namespace {

// ---------------------------------------------------------------- few rows

// Rows of a sequence that fit one tile of 16 (single tokens, groups of up to 16
// heads; short chunks of small groups): bound by the bytes of K and V.  A
// workgroup takes one (sequence, kv head) and one part of its keys, its waves
// every fourth step of 32 (fp32: 16) keys, straight from global memory into
// the operands: K rows by 16-byte pieces; V rows likewise, 16 lanes to a row,
// and turned in registers, since lane i of O^T's tile e may stand for element
// E i + e of the head as well as any other.  No LDS before the waves are
// joined, so that a CU's waves keep as many bytes in flight as registers hold.
// kv heads are side by side in the grid: workgroups of one head alone meet the
// same few channels (64 contexts of up to 16384 keys in bf16, heads of 128: 556
// us, against 468).  That case now takes 442 us, 6.2 TB/s; one token over 131071
// keys, fp32 over fp16, 80 us, 6.8 TB/s (a plain read: 7.1).  Eight waves to a
// workgroup are slower (526 us, and 98 for the one token).
constexpr int kFewWaves = 4;
constexpr int kFewThreads = 64 * kFewWaves;

template <typename T, typename TC, int D>
struct Few {
  static constexpr int kParts = parts_of<T, TC>();
  // weights: 16-bit queries' too are two parts, since products cost nothing here
  static constexpr int kWeightParts = sizeof(T) == 2 ? 2 : kParts;
  static constexpr int KT = Elem<TC>::kKeys, NSUB = KT / 16;
  static constexpr int KC = sizeof(TC) == 2 ? D / 32 : D / 16;   // K pieces of 16 bytes per lane and 16 keys
  static constexpr int KD = sizeof(TC) == 2 ? 8 : 4;             // elements of such a piece
  static constexpr int E = sizeof(TC) == 2 && D >= 128 ? 8 : 4;  // elements of a lane's piece of a V row
  static constexpr int U = D / (16 * E);
  static constexpr int kTiles = D / 16;  // tiles of O^T: (u, e)
};

// A lane's piece of a V row, as words; operand(): tile e's, for the keys of the
// pieces v[0 ..], U pieces apart.
template <typename TC, int E>
struct VPiece {
  static constexpr int kWords = E * (int)sizeof(TC) / 4;
  uint32_t w[kWords];
};
template <typename TC>
constexpr uint32_t exponent_bits() {
  return __is_same(TC, _Float16) ? 0x7c00u : __is_same(TC, __bf16) ? 0x7f80u : 0x7f800000u;
}
template <typename TC>
constexpr uint32_t one_bits() {
  return __is_same(TC, _Float16) ? 0x3c00u : __is_same(TC, __bf16) ? 0x3f80u : 0x3f800000u;
}
// the sign bit's place of each element of a word that is an infinity or NaN:
// an exponent of ones and one more carries there
template <typename TC>
__device__ __forceinline__ uint32_t odd_elements(uint32_t w) {
  constexpr uint32_t rep = sizeof(TC) == 4 ? 1u : 0x10001u, top = sizeof(TC) == 4 ? 0x80000000u : 0x8000u;
  constexpr uint32_t e = exponent_bits<TC>();
  return ((w & e * rep) + (top - e) * rep) & top * rep;
}
template <typename TC, typename V, int E, int U>
__device__ __forceinline__ V operand(const VPiece<TC, E> (*v)[U], int u, int e) {
  u4 x;
  if constexpr (sizeof(TC) == 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = v[j][u].w[e];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      x[j] = __builtin_amdgcn_perm(v[2 * j + 1][u].w[e / 2], v[2 * j][u].w[e / 2], e & 1 ? 0x07060302u : 0x05040100u);
  }
  return __builtin_bit_cast(V, x);
}

// kPad: heads narrower than D
template <typename T, typename TC, int D, bool kPad>
__global__ __launch_bounds__(kFewThreads, D == 256 ? 1 : 2) void few_kernel(AttendArgs a, Parts parts, int tiles, bool chunk_runs) {
  using F = Few<T, TC, D>;
  using vec = typename Elem<TC>::vec;
  constexpr int NP = F::kParts, NW = F::kWeightParts, KT = F::KT, NSUB = F::NSUB;
  extern __shared__ float few_lds[];  // [wave][16][D + 4] sums
  __shared__ float sh_m[kFewWaves][16], sh_l[kFewWaves][16];

  const int kvh = blockIdx.x % a.p.kv_heads, task = blockIdx.x / a.p.kv_heads, part = blockIdx.z;
  const int seq = task / tiles, tile = task - seq * tiles;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
  const Chunk c = chunk_of(a.p, seq);
  const int rows = c.n * a.group;
  // More rows are the chunk kernel's; where the caller's word was that there are
  // none, they are done here, one tile after another and unsplit.
  const bool over = rows > 16 && c.n != 1;
  if (over && (chunk_runs || part > 0)) return;
  const Sees sees = sees_of(a, c);
  for (int r0 = tile * 16; r0 < rows; r0 += tiles * 16) {
    const int rn = rows - r0 < 16 ? rows - r0 : 16;
    const int t0 = r0 / a.group, t1 = (r0 + rn - 1) / a.group;
    const Span span = span_of(sees, t0, t1, parts.keys, over ? 1 : parts.most);
    if (part >= span.parts) return;
    const int k0 = span.begin(part, parts.keys), k1 = span.end(part, parts.keys);

    // this lane's row: column i of the transposed tiles
    const bool row_ok = i < rn;
    const int row = r0 + (row_ok ? i : 0);
    const int64_t at_pos = sees.p0 + row / a.group;
    const int pos = as_int(at_pos), low = as_int(sees.low(at_pos));
    // a step whose keys lie within these is seen whole by every row
    const int all_lo = as_int(sees.low(sees.p0 + t1)), all_hi = as_int(sees.p0 + t0);
    const int dim = a.p.dim;

    vec q[F::KC][NP];
    float qs = 1.f;  // queries over fp16: the row divided by a power of two
    {
      const T* src = static_cast<const T*>(a.q.d) + (int64_t)(c.begin + row / a.group) * a.q.token_stride +
                     (int64_t)(kvh * a.group + row % a.group) * a.q.head_stride;
      float x[F::KC][F::KD], top = 0.f;
#pragma unroll
      for (int k = 0; k < F::KC; ++k)
#pragma unroll
        for (int j = 0; j < F::KD; ++j) {
          const int d = k * 4 * F::KD + g * F::KD + j;
          x[k][j] = row_ok && d < dim ? (float)src[d] : 0.f;
          top = fmaxf(top, fabsf(x[k][j]));
        }
      if constexpr (sizeof(T) == 4 && __is_same(TC, _Float16)) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        // the largest element into [2^13, 2^14): its lower part keeps 11 bits too
        const int e = top > 0.f && top < __builtin_inff() ? ilogbf(top) - 13 : 0;
        qs = ldexpf(1.f, e);
#pragma unroll
        for (int k = 0; k < F::KC; ++k)
#pragma unroll
          for (int j = 0; j < F::KD; ++j) x[k][j] = ldexpf(x[k][j], -e);
      }
#pragma unroll
      for (int k = 0; k < F::KC; ++k)
#pragma unroll
        for (int j = 0; j < F::KD; ++j) split<NP>(x[k][j], q[k], j);
    }
    const float sc = a.scale * kLog2e * qs;

    const TC* base = static_cast<const TC*>(a.p.kv) + (int64_t)kvh * a.p.head_stride;
    const int mask = (1 << a.p.page_shift) - 1;
    f4 o[F::kTiles];
#pragma unroll
    for (int t = 0; t < F::kTiles; ++t) o[t] = f4{0, 0, 0, 0};
    float m = minus_inf(), l = 0.f;

    // page[s]: that of key 16 s + i of a step, -1 where there is none (what is
    // read there is page 0, and counts for nothing)
    struct Pages {
      int at[NSUB];
    };
    const int32_t* table = a.p.table + (int64_t)c.slot * a.p.table_stride;  // (no keys without a slot)
    const uint32_t page_bytes = (uint32_t)a.p.page_stride * (uint32_t)sizeof(TC);
    const uint32_t token_bytes = (uint32_t)a.p.token_stride * (uint32_t)sizeof(TC);
    auto row_at = [&](const char* from, int page, uint32_t key) {
      return reinterpret_cast<const TC*>(from + (uint64_t)(uint32_t)(page < 0 ? 0 : page) * page_bytes +
                                         (uint64_t)(key & (uint32_t)mask) * token_bytes);
    };
    // (the entries as they are: what is done with them waits for the loads)
    auto entries_at = [&](int kb) {
      Pages p;
#pragma unroll
      for (int s = 0; s < NSUB; ++s) {
        const int key = kb + s * 16 + i;
        p.at[s] = table[(key < k1 ? key : k1 - 1) >> a.p.page_shift];
      }
      return p;
    };
    auto pages_of = [&](int kb, const Pages& e) {
      Pages p;
#pragma unroll
      for (int s = 0; s < NSUB; ++s)
        p.at[s] = kb + s * 16 + i < k1 && (uint32_t)e.at[s] < (uint32_t)a.p.pages ? e.at[s] : -1;
      return p;
    };
    vec k[NSUB][F::KC];
    using VP = VPiece<TC, F::E>;
    VP v[NSUB * 4][F::U];
    const char* base_k = reinterpret_cast<const char*>(base + g * F::KD);
    const char* base_v = reinterpret_cast<const char*>(base + a.p.value_offset + i * F::E);
    auto fetch_k = [&](int kb, const Pages& pg) {
#pragma unroll
      for (int s = 0; s < NSUB; ++s) {
        const TC* row_k = row_at(base_k, pg.at[s], (uint32_t)kb + s * 16 + i);
#pragma unroll
        for (int x = 0; x < F::KC; ++x) {
          const int d = x * 4 * F::KD;
          k[s][x] = *reinterpret_cast<const vec*>(row_k + (!kPad || d + g * F::KD < dim ? d : -g * F::KD));
        }
      }
    };
    auto fetch_v = [&](int kb, const Pages& pg) {
#pragma unroll
      for (int s = 0; s < NSUB; ++s) {
        const TC* row_v = nullptr;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          // keys 4 g .. 4 g + 3 share a page of at least 4 tokens
          if (r == 0 || a.p.page_shift < 2) {
            row_v = row_at(base_v, __shfl(pg.at[s], g * 4 + r), (uint32_t)kb + s * 16 + g * 4 + r);
          } else {
            row_v += a.p.token_stride;
          }
#pragma unroll
          for (int u = 0; u < F::U; ++u) {
            const int d = u * 16 * F::E;
            typedef uint32_t words __attribute__((ext_vector_type(VP::kWords)));
            // (past the caches: 102 -> 92 us for one token over 131071 keys; K's
          // 64-byte pieces of a row meet in the cache and are not)
          const words x = __builtin_nontemporal_load(reinterpret_cast<const words*>(row_v + (!kPad || d + i * F::E < dim ? d : -i * F::E)));
#pragma unroll
            for (int y = 0; y < VP::kWords; ++y) v[s * 4 + r][u].w[y] = x[y];
          }
        }
      }
    };

    // K of a step is requested while the step before it is in its weights, V while
    // it is in its scores, the page table two steps ahead.
    constexpr int kStep = kFewWaves * KT;
    int kb = k0 + wave * KT;
    Pages page, page1, entry1;
    if (kb < k1) {
      page = pages_of(kb, entries_at(kb));
      entry1 = entries_at(kb + kStep);
      fetch_k(kb, page);
      fetch_v(kb, page);
    }
    for (; kb < k1; kb += kStep) {
      const bool more = kb + kStep < k1;
      bool whole = kb >= all_lo && kb + KT - 1 <= all_hi;
#pragma unroll
      for (int s = 0; s < NSUB; ++s) whole = whole && __ballot(page.at[s] >= 0) == ~uint64_t{0};
      float w[NSUB * 4];
#pragma unroll
      for (int s = 0; s < NSUB; ++s) {
        f4 acc{0, 0, 0, 0};
#pragma unroll
        for (int x = 0; x < F::KC; ++x) {
          vec kk = k[s][x];
          if constexpr (kPad)
            if (x * 4 * F::KD + g * F::KD >= dim) kk = vec{};
#pragma unroll
          for (int n = NP - 1; n >= 0; --n) acc = mma16(kk, q[x][n], acc);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) w[s * 4 + r] = acc[r] * sc;
      }
      if (more) {
        page1 = pages_of(kb + kStep, entry1);
        entry1 = entries_at(kb + 2 * kStep);
        fetch_k(kb + kStep, page1);
      }
      uint32_t vis = 0xffffffffu;
      if (!whole) {
        const int from = low - kb, to = pos - kb;  // of this row's keys, within the step
#pragma unroll
        for (int j = 0; j < NSUB * 4; ++j) {
          const int n = (j >> 2) * 16 + g * 4 + (j & 3);
          const bool there = __shfl(page.at[j >> 2], g * 4 + (j & 3)) >= 0;
          if (!there || n < from || n > to) {
            vis &= ~(1u << j);
            w[j] = minus_inf();
          }
          if (!there)
#pragma unroll
            for (int u = 0; u < F::U; ++u) v[j][u] = VP{};
        }
      }
      float top = w[0];
#pragma unroll
      for (int j = 1; j < NSUB * 4; ++j) top = fmaxf(top, w[j]);
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      if (__ballot(top > m)) {
        top = ceilf(fmaxf(top, m));  // whole: what it is taken from is exact
        const float shrink = exp2_(m - (top == minus_inf() ? 0.f : top));
        m = top;
        l *= shrink;
#pragma unroll
        for (int t = 0; t < F::kTiles; ++t) o[t] *= shrink;
      }
      const float back = Elem<TC>::kShift - (m == minus_inf() ? 0.f : m);
      constexpr int kDepth = sizeof(vec) / sizeof(TC);
      vec p[NW];
#pragma unroll
      for (int j = 0; j < kDepth; ++j) {
        const float x = exp2_(w[j] + back);
        l += x;
        split<NW>(x, p, j);
      }
      // Values that are not finite meet weights of 0 in the rows that do not see
      // their keys, which would be NaN there: where rows see different keys they
      // count as 0, and the rows that see them turn to NaN.
      if (!whole) {
        uint32_t odd = 0;
#pragma unroll
        for (int j = 0; j < kDepth; ++j)
#pragma unroll
          for (int u = 0; u < F::U; ++u)
#pragma unroll
            for (int y = 0; y < VP::kWords; ++y) odd |= odd_elements<TC>(v[j][u].w[y]);
        if (__ballot(odd != 0)) {
          vec seen;
#pragma unroll
          for (int j = 0; j < kDepth; ++j) seen[j] = (vis >> j) & 1 ? 1.f : 0.f;
#pragma unroll
          for (int u = 0; u < F::U; ++u) {
            VP is[kDepth][1];
#pragma unroll
            for (int j = 0; j < kDepth; ++j)
#pragma unroll
              for (int y = 0; y < VP::kWords; ++y) {
                const uint32_t bad = odd_elements<TC>(here(v[j][u].w[y])) >> (sizeof(TC) == 4 ? 31 : 15);
                is[j][0].w[y] = bad * one_bits<TC>();
                v[j][u].w[y] &= ~(bad * (sizeof(TC) == 4 ? 0xffffffffu : 0xffffu));
              }
#pragma unroll
            for (int e = 0; e < F::E; ++e) {
              const f4 count = mma16(operand<TC, vec, F::E, 1>(is, 0, e), seen, f4{0, 0, 0, 0});
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (count[r] > 0.f) o[u * F::E + e][r] = __builtin_nanf("");
            }
          }
        }
      }
#pragma unroll
      for (int u = 0; u < F::U; ++u)
#pragma unroll
        for (int e = 0; e < F::E; ++e) {
          const vec x = operand<TC, vec, F::E, F::U>(v, u, e);
#pragma unroll
          for (int n = NW - 1; n >= 0; --n) o[u * F::E + e] = mma16(x, p[n], o[u * F::E + e]);
        }
      if (more) {
        fetch_v(kb + kStep, page1);
        page = page1;
      }
    }

    // the waves' sums, relative to the largest of their maxima
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g == 0) {
      sh_m[wave][i] = m;
      sh_l[wave][i] = l;
    }
    __syncthreads();
    float top = sh_m[0][i];
#pragma unroll
    for (int x = 1; x < kFewWaves; ++x) top = fmaxf(top, sh_m[x][i]);
    const float from = top == minus_inf() ? 0.f : top;
    const float f = exp2_(m - from);
    float* mine = few_lds + (wave * 16 + i) * (D + 4);
#pragma unroll
    for (int u = 0; u < F::U; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < F::E; e += 4) {
          f4 x;
#pragma unroll
          for (int y = 0; y < 4; ++y) x[y] = o[u * F::E + e + y][r] * f;
          *reinterpret_cast<f4*>(mine + u * 16 * F::E + (g * 4 + r) * F::E + e) = x;
        }
    __syncthreads();
    for (int idx = threadIdx.x; idx < 16 * (D / 4); idx += kFewThreads) {
      const int r = idx / (D / 4), d = idx % (D / 4) * 4;
      if (r >= rn) break;
      float rt = sh_m[0][r], sum = 0.f;
#pragma unroll
      for (int x = 1; x < kFewWaves; ++x) rt = fmaxf(rt, sh_m[x][r]);
      const float rf = rt == minus_inf() ? 0.f : rt;
      f4 s{0, 0, 0, 0};
#pragma unroll
      for (int x = 0; x < kFewWaves; ++x) {
        s += *reinterpret_cast<const f4*>(few_lds + (x * 16 + r) * (D + 4) + d);
        sum += sh_l[x][r] * exp2_(sh_m[x][r] - rf);
      }
      if (span.parts > 1) {
        const int64_t at = part * parts.rows + ((int64_t)task * a.p.kv_heads + kvh) * 16 + r;
        *reinterpret_cast<f4*>(parts.o + at * D + d) = s;
        if (d == 0) parts.ml[at] = f4{rt, sum, sum, 0.f};
        continue;
      }
      const int rr = r0 + r, token = c.begin + rr / a.group, head = kvh * a.group + rr % a.group;
      T* out = static_cast<T*>(a.out.d) + (int64_t)token * a.out.token_stride + (int64_t)head * a.out.head_stride;
#pragma unroll
      for (int y = 0; y < 4; ++y)
        if (d + y < dim) out[d + y] = (T)(sum == 0.f ? 0.f : s[y] / sum);
      if (a.lse && d == 0)
        a.lse[(int64_t)token * a.heads + head] =
            sum == 0.f ? minus_inf() : (rf + (__builtin_amdgcn_logf(sum) - Elem<TC>::kShift)) * kLn2;
    }
    if (!over) return;
    __syncthreads();  // the next tile's sums take the same LDS
  }
}

// ---------------------------------------------------------------- joining parts

// One row's parts: weights from their maxima, then the weighted sum, D / 4 lanes
// across the row and the parts side by side.  kWaves waves take a row: four
// where rows are few and their parts many, else one.
constexpr int kJoinThreads = 256;

// The first few_rows rows are (sequence, one of its first `per` tokens, head),
// of few_kernel; the others all of the call's, of chunk_kernel.
template <typename T, int D, int kWaves>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(AttendArgs a, Parts few, Parts chunk, int64_t few_rows,
                                                            int per, int tiles, bool alone, float few_shift,
                                                            float chunk_shift) {
  constexpr int kAcross = D / 4, kSide = 64 * kWaves / kAcross;
  constexpr int kRows = kJoinThreads / (64 * kWaves);  // of a workgroup
  __shared__ f4 sums[kRows][kSide][kAcross];
  __shared__ f4 ls[kRows][kSide];
  const int lane = threadIdx.x & 63, sub = threadIdx.x / (64 * kWaves), in = threadIdx.x % (64 * kWaves);
  const int64_t index = (int64_t)blockIdx.x * kRows + sub;
  const bool is_few = index < few_rows;
  const int64_t rest = is_few ? index : index - few_rows;
  const int head = (int)(rest % a.heads), kvh = head / a.group, size = is_few ? 16 : kChunkTile;
  const Parts parts = is_few ? few : chunk;
  const float shift = is_few ? few_shift : chunk_shift;
  int token = (int)(rest / a.heads), seq = -1, parts_n = 0;
  int64_t at = 0;
  if (is_few) {
    seq = token / per;
  } else if (token < a.p.tokens) {
    for (int s0 = 0; s0 < a.p.seqs + 1; s0 += 64) {
      const int s = s0 + lane;
      const int n = __popcll(__ballot(s <= a.p.seqs && a.p.starts[s <= a.p.seqs ? s : a.p.seqs] <= token));
      seq += n;
      if (n < 64) break;
    }
  }
  if (seq >= 0 && seq < a.p.seqs) {
    const Chunk c = chunk_of(a.p, seq);
    const int rows = c.n * a.group;
    if (is_few) token = c.begin + token % per;
    const int rr = (token - c.begin) * a.group + head % a.group, r0 = rr / size * size;
    if (token < c.begin + c.n && (alone || (rows > 16 && c.n != 1) != is_few)) {
      const int rn = rows - r0 < size ? rows - r0 : size;
      at = is_few ? (((int64_t)seq * tiles + rr / size) * a.p.kv_heads + kvh) * size + rr % size : rest;
      parts_n = span_of(sees_of(a, c), r0 / a.group, (r0 + rn - 1) / a.group, parts.keys, parts.most).parts;
    }
  }
  if (parts_n <= 1) parts_n = 0;  // (written by the kernel before)
  const int x = in % kAcross, side = in / kAcross;
  f4 s{0, 0, 0, 0};
  float m = minus_inf(), l = 0.f, lr = 0.f;
  constexpr int kBatch = kWaves == 4 ? 8 : 4;  // parts whose loads are in flight together
  for (int p0 = side; p0 < parts_n; p0 += kBatch * kSide) {
    f4 ml[kBatch], o[kBatch];
#pragma unroll
    for (int y = 0; y < kBatch; ++y) {
      const int p = p0 + y * kSide < parts_n ? p0 + y * kSide : p0;
      ml[y] = parts.ml[p * parts.rows + at];
      o[y] = *reinterpret_cast<const f4*>(parts.o + (p * parts.rows + at) * D + x * 4);
    }
    float top = m;
#pragma unroll
    for (int y = 0; y < kBatch; ++y) top = fmaxf(top, ml[y][0]);
    const float from = top == minus_inf() ? 0.f : top, f = exp2_(m - from);
    s *= f;
    l *= f;
    lr *= f;
    m = top;
#pragma unroll
    for (int y = 0; y < kBatch; ++y) {
      if (p0 + y * kSide >= parts_n) break;
      const float w = exp2_(ml[y][0] - from);
      s += o[y] * w;
      l += ml[y][1] * w;
      lr += ml[y][2] * w;
    }
  }
  sums[sub][side][x] = s;
  if (x == 0) ls[sub][side] = f4{m, l, lr, 0.f};
  __syncthreads();
  if (side || parts_n == 0) return;
#pragma unroll
  for (int y = 1; y < kSide; ++y) m = fmaxf(m, ls[sub][y][0]);
  const float from = m == minus_inf() ? 0.f : m;
  float sum = 0.f, sumr = 0.f;
  s = f4{0, 0, 0, 0};
#pragma unroll
  for (int y = 0; y < kSide; ++y) {
    const f4 ml = ls[sub][y];
    const float w = exp2_(ml[0] - from);
    s += sums[sub][y][x] * w;
    sum += ml[1] * w;
    sumr += ml[2] * w;
  }
  T* out = static_cast<T*>(a.out.d) + (int64_t)token * a.out.token_stride + (int64_t)head * a.out.head_stride;
#pragma unroll
  for (int y = 0; y < 4; ++y)
    if (x * 4 + y < a.p.dim) out[x * 4 + y] = (T)(sumr == 0.f ? 0.f : s[y] / sumr);
  if (a.lse && x == 0)
    a.lse[(int64_t)token * a.heads + head] =
        sum == 0.f ? minus_inf() : (from + (__builtin_amdgcn_logf(sum) - shift)) * kLn2;
}

int width_of(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

// Parts of the keys, so that `tasks` workgroups become about `want`, of no fewer
// than `least` keys each and, so that long and short contexts of a batch take
// their turns, no more than `top`; but not beyond 8192 workgroups, whose sums
// wait in the workspace.
Parts parts_of_keys(int64_t most, int64_t tasks, int64_t want, int64_t least, int64_t top) {
  Parts p{};
  const int64_t n = (want + tasks - 1) / tasks, cap = n > 8192 / tasks ? n : 8192 / tasks;
  int64_t keys = (most + n - 1) / n;
  if (keys > top) keys = top;
  if (keys < least) keys = least;
  if (keys < (most + cap - 1) / cap) keys = (most + cap - 1) / cap;
  p.keys = (int)((keys + 127) / 128 * 128);
  const int64_t m = (most + p.keys - 1) / p.keys;
  p.most = (int)(m < 1 ? 1 : m);
  return p;
}

// How the call is dealt out, by its sizes and the caller's hints alone.
AttendPlan plan_of(const AttendArgs& a, int max_new, int64_t max_len) {
  AttendPlan p{};
  if (a.p.seqs < 1 || a.p.tokens < 1) return p;
  const int D = width_of(a.p.dim);
  int64_t most = (int64_t)a.p.max_pages << a.p.page_shift;
  if (most > kMaxLen) most = kMaxLen;  // (a longer table's rest is never used)
  if (max_len > 0 && max_len < most) most = max_len;
  int64_t longest = max_new > 0 && max_new < a.p.tokens ? max_new : a.p.tokens;
  if (a.window > 0 && most > (int64_t)a.window + longest) most = (int64_t)a.window + longest;
  const size_t per_row = D * sizeof(float) + sizeof(f4);
  p.chunk = longest > 1 && longest * a.group > 16;
  // One sequence that may be a chunk is taken for one: its rows are few only
  // where the others belong to no sequence.
  p.few = !(p.chunk && a.p.seqs == 1);
  if (p.few) {
    p.few_tiles = (a.group + 15) / 16;
    const int64_t tasks = (int64_t)a.p.seqs * p.few_tiles * a.p.kv_heads;
    // Parts of at least 256 keys, and as many as give every CU two workgroups (one
    // token over 131071 keys: 101 us so, 119 with three, 138 with parts of 512);
    // up to 768 keys are not split: the second launch costs the host the 5 us that
    // it saves the GPU (517 keys: 14.6 us whole, 12.5 in three parts; 24 contexts
    // of 517: 12.9 whole, 19.2 split).
    p.few_parts = parts_of_keys(most, tasks, 512, most <= 768 ? 768 : 256, 2048);
    p.few_parts.rows = tasks * 16;
    p.few_bytes = p.few_parts.most > 1 ? p.few_parts.most * p.few_parts.rows * per_row : 0;
  }
  if (p.chunk) {
    p.chunk_tiles = tile_count(a.p.tokens, a.group, kChunkTile, a.p.seqs);
    // Two workgroups per CU, of the tiles that have rows when they are all of one
    // sequence (509 tokens of 28 heads beside 16 that decode: 167 us when the
    // empty tiles of those count too, 145 us so); parts of at least 512 keys.
    const int64_t wgs = ((int64_t)a.p.tokens * a.group + kChunkTile - 1) / kChunkTile * a.p.kv_heads;
    p.chunk_parts = parts_of_keys(most, wgs, 512, 512, most);
    p.chunk_parts.rows = (int64_t)a.p.tokens * a.heads;
    p.chunk_bytes = p.chunk_parts.most > 1 ? p.chunk_parts.most * p.chunk_parts.rows * per_row : 0;
  }
  return p;
}

Parts placed(Parts p, void* work, int D) {
  p.o = static_cast<float*>(work);
  p.ml = reinterpret_cast<f4*>(p.o + p.most * p.rows * D);
  return p;
}

template <typename T, typename TC, int D, bool kPad>
hipError_t attend_width(const AttendArgs& a, const AttendPlan& p, int type, int cache_type, char* work, hipStream_t s) {
  const Parts few = placed(p.few_parts, work, D);
  const Parts chunk = placed(p.chunk_parts, work + (p.few_bytes + 255) / 256 * 256, D);
  constexpr size_t lds = (size_t)kFewWaves * 16 * (D + 4) * sizeof(float);
  hipError_t e;
  if (p.few) {
    if (lds > 60000) {
      e = hipFuncSetAttribute(reinterpret_cast<const void*>(few_kernel<T, TC, D, kPad>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
      if (e != hipSuccess) return e;
    }
    few_kernel<T, TC, D, kPad><<<dim3(a.p.kv_heads * a.p.seqs * p.few_tiles, 1, few.most), kFewThreads, lds, s>>>(
        a, few, p.few_tiles, p.chunk);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  if (p.chunk && (e = launch_chunk(a, type, cache_type, chunk, p.chunk_tiles, !p.few, s)) != hipSuccess) return e;
  const int per = a.group >= 16 ? 1 : 16 / a.group;  // tokens that few_kernel takes of a sequence
  const int64_t few_rows = few.most > 1 ? (int64_t)a.p.seqs * per * a.heads : 0;
  const int64_t rows = few_rows + (chunk.most > 1 ? (int64_t)a.p.tokens * a.heads : 0);
  if (rows == 0) return hipSuccess;
  if (rows < 1024)
    join_kernel<T, D, 4><<<(unsigned)rows, kJoinThreads, 0, s>>>(a, few, chunk, few_rows, per, p.few_tiles, !p.few,
                                                                Elem<TC>::kShift, chunk_shift<TC>());
  else
    join_kernel<T, D, 1><<<(unsigned)((rows + 3) / 4), kJoinThreads, 0, s>>>(a, few, chunk, few_rows, per, p.few_tiles, !p.few,
                                                                          Elem<TC>::kShift, chunk_shift<TC>());
  return hipGetLastError();
}

template <typename T, typename TC>
hipError_t attend_types(const AttendArgs& a, const AttendPlan& p, int type, int cache_type, char* work, hipStream_t s) {
  const int dim = a.p.dim;
  if (dim == 64) return attend_width<T, TC, 64, false>(a, p, type, cache_type, work, s);
  if (dim < 64) return attend_width<T, TC, 64, true>(a, p, type, cache_type, work, s);
  if (dim == 128) return attend_width<T, TC, 128, false>(a, p, type, cache_type, work, s);
  if (dim < 128) return attend_width<T, TC, 128, true>(a, p, type, cache_type, work, s);
  if (dim == 256) return attend_width<T, TC, 256, false>(a, p, type, cache_type, work, s);
  return attend_width<T, TC, 256, true>(a, p, type, cache_type, work, s);
}

}  // namespace

size_t attend_workspace(const AttendArgs& a, int max_new, int64_t max_len) {
  const AttendPlan p = plan_of(a, max_new, max_len);
  return (p.few_bytes + 255) / 256 * 256 + p.chunk_bytes;
}

hipError_t launch_attend(const AttendArgs& a, int type, int cache_type, int max_new, int64_t max_len, void* work,
                         hipStream_t s) {
  const AttendPlan p = plan_of(a, max_new, max_len);
  char* w = static_cast<char*>(work);
  if (type == kF32) {
    if (cache_type == kF32) return attend_types<float, float>(a, p, type, cache_type, w, s);
    if (cache_type == kF16) return attend_types<float, _Float16>(a, p, type, cache_type, w, s);
    return attend_types<float, __bf16>(a, p, type, cache_type, w, s);
  }
  if (type == kF16) return attend_types<_Float16, _Float16>(a, p, type, cache_type, w, s);
  return attend_types<__bf16, __bf16>(a, p, type, cache_type, w, s);
}

}  // namespace nls
