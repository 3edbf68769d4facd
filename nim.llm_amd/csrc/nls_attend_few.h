// nls_attend_few.h -- attention of sequences of few rows: the work of one
// workgroup, for a launch of their own or beside chunks.
#pragma once
#include "nls_attend.h"

namespace nls {

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
constexpr size_t few_lds_bytes(int D) { return (size_t)kFewWaves * 16 * (D + 4) * sizeof(float); }

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

// Workgroup group_at of one part's.  kPad: heads narrower than D
template <typename T, typename TC, int D, bool kPad>
__device__ __forceinline__ void few_rows(const AttendArgs& a, const Parts& parts, int tiles, bool chunk_runs, int group_at,
                                         int part) {
  using F = Few<T, TC, D>;
  using vec = typename Elem<TC>::vec;
  constexpr int NP = F::kParts, NW = F::kWeightParts, KT = F::KT, NSUB = F::NSUB;
  extern __shared__ float few_lds[];  // [wave][16][D + 4] sums
  __shared__ float sh_m[kFewWaves][16], sh_l[kFewWaves][16];

  const int kvh = group_at % a.p.kv_heads, task = group_at / a.p.kv_heads;
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
        const int e = query_exponent(top);
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
    const float sc = a.scale * kLog2e;  // (behind qs: times it, it may leave fp32's range where the score does not)

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
            // (past the caches: one token over 131071 keys 104 -> 89 us, 48 contexts
            // of 4000 147 -> 133; shared pages lose less: 48 forks of 4000 67.6 us
            // either way, of 16000 235 -> 246, groups of 32 heads 34.5 -> 35.2 (8 of
            // 16000) and 89.2 -> 89.8 (64 of 4000).  K's 64-byte pieces of a row meet
            // in the cache and are not)
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
        for (int r = 0; r < 4; ++r) w[s * 4 + r] = acc[r] * qs * sc;
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
      // (the shift behind the difference, which is exact: it would be rounded within
      // a maximum of 2^24 or more, and weights of 2^16 are beyond fp16)
      const float from = m == minus_inf() ? 0.f : m;
      constexpr int kDepth = sizeof(vec) / sizeof(TC);
      vec p[NW];
#pragma unroll
      for (int j = 0; j < kDepth; ++j) {
        const float y = w[j] - from, x = exp2_(Elem<TC>::kShift == 0.f ? y : y + Elem<TC>::kShift);
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

}  // namespace nls
