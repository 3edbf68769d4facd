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
constexpr int kFewWaves = 4;
constexpr int kFewThreads = 64 * kFewWaves;

template <typename T, typename TC, int D>
struct Few {
  static constexpr int kParts = parts_of<T, TC>();
  static constexpr int KT = Elem<TC>::kKeys, NSUB = KT / 16;
  static constexpr int KC = sizeof(TC) == 2 ? D / 32 : D / 16;   // K pieces of 16 bytes per lane and 16 keys
  static constexpr int KD = sizeof(TC) == 2 ? 8 : 4;             // elements of such a piece
  static constexpr int E = sizeof(TC) == 2 && D >= 128 ? 8 : 4;  // elements of a lane's piece of a V row
  static constexpr int U = D / (16 * E);
  static constexpr int kTiles = D / 16;  // tiles of O^T: (u, e)
};

template <typename TC, int E>
struct VPiece {
  TC v[E];
};

template <typename T, typename TC, int D>
__global__ __launch_bounds__(kFewThreads) void few_kernel(AttendArgs a, Parts parts, int tiles, bool chunk_runs) {
  using F = Few<T, TC, D>;
  using vec = typename Elem<TC>::vec;
  constexpr int NP = F::kParts, KT = F::KT, NSUB = F::NSUB;
  extern __shared__ float few_lds[];  // [wave][16][D + 4] sums; before that, a step's weights
  __shared__ float sh_m[kFewWaves][16], sh_l[kFewWaves][16];

  const int task = blockIdx.x, kvh = blockIdx.y, part = blockIdx.z;
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
  const int64_t k0 = span.lo + part * parts.keys, k1 = part + 1 == span.parts ? span.hi : k0 + parts.keys;

  // this lane's row: column i of the transposed tiles
  const bool row_ok = i < rn;
  const int row = r0 + (row_ok ? i : 0);
  const int64_t pos = sees.p0 + row / a.group, low = sees.low(pos);
  // a step whose keys lie within these is seen whole by every row
  const int64_t all_lo = sees.low(sees.p0 + t1), all_hi = sees.p0 + t0;
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
  const int64_t mask = (int64_t{1} << a.p.page_shift) - 1;
  f4 o[F::kTiles];
#pragma unroll
  for (int t = 0; t < F::kTiles; ++t) o[t] = f4{0, 0, 0, 0};
  float m = minus_inf(), l = 0.f;

  int page[NSUB];
  auto pages_at = [&](int64_t kb) {
#pragma unroll
    for (int s = 0; s < NSUB; ++s) {
      const int64_t key = kb + s * 16 + i;
      page[s] = key < k1 ? page_of(a.p, c.slot, key) : -1;
    }
  };
  int64_t kb = k0 + wave * KT;
  if (kb < k1) pages_at(kb);
  for (; kb < k1; kb += kFewWaves * KT) {
    vec k[NSUB][F::KC];
    VPiece<TC, F::E> v[NSUB * 4][F::U];
    bool whole = kb >= all_lo && kb + KT - 1 <= all_hi;
    bool vok[NSUB * 4];
#pragma unroll
    for (int s = 0; s < NSUB; ++s) {
      whole = whole && __ballot(page[s] >= 0) == ~uint64_t{0};
      // (a place that is no key reads page 0, and what it reads counts for nothing)
      const TC* row_k = base + (int64_t)(page[s] < 0 ? 0 : page[s]) * a.p.page_stride + ((kb + s * 16 + i) & mask) * a.p.token_stride;
#pragma unroll
      for (int x = 0; x < F::KC; ++x) {
        const int d = x * 4 * F::KD + g * F::KD;
        k[s][x] = *reinterpret_cast<const vec*>(row_k + (d < dim ? d : 0));
      }
    }
#pragma unroll
    for (int s = 0; s < NSUB; ++s)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int p = __shfl(page[s], g * 4 + r);
        vok[s * 4 + r] = p >= 0;
        const TC* row_v = base + a.p.value_offset + (int64_t)(p < 0 ? 0 : p) * a.p.page_stride +
                          ((kb + s * 16 + g * 4 + r) & mask) * a.p.token_stride;
#pragma unroll
        for (int u = 0; u < F::U; ++u) {
          const int d = u * 16 * F::E + i * F::E;
          __builtin_memcpy(&v[s * 4 + r][u], __builtin_assume_aligned(row_v + (d < dim ? d : 0), sizeof(TC) * F::E),
                           sizeof(TC) * F::E);
        }
      }
    const int64_t next = kb + kFewWaves * KT;
    bool vis[NSUB * 4];
    float s_[NSUB * 4];
    if (dim < D) {
#pragma unroll
      for (int s = 0; s < NSUB; ++s)
#pragma unroll
        for (int x = 0; x < F::KC; ++x)
          if (x * 4 * F::KD + g * F::KD >= dim) k[s][x] = vec{};
    }
#pragma unroll
    for (int s = 0; s < NSUB; ++s) {
      f4 acc{0, 0, 0, 0};
#pragma unroll
      for (int n = NP - 1; n >= 0; --n)
#pragma unroll
        for (int x = 0; x < F::KC; ++x) acc = mma16(k[s][x], q[x][n], acc);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int64_t key = kb + s * 16 + g * 4 + r;
        vis[s * 4 + r] = whole || (vok[s * 4 + r] && key >= low && key <= pos);
        s_[s * 4 + r] = acc[r];
      }
    }
    if (next < k1) pages_at(next);
    float top = minus_inf();
#pragma unroll
    for (int j = 0; j < NSUB * 4; ++j) top = vis[j] ? fmaxf(top, s_[j] * sc) : top;
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    top = fmaxf(top, m);
    const float from = top == minus_inf() ? 0.f : top;
    const float shrink = exp2_(m - from);
    m = top;
    float w[NSUB * 4], sum = 0.f;
#pragma unroll
    for (int j = 0; j < NSUB * 4; ++j) {
      w[j] = vis[j] ? exp2_(__builtin_fmaf(s_[j], sc, Elem<TC>::kShift - from)) : 0.f;
      sum += w[j];
    }
    l = l * shrink + sum;
#pragma unroll
    for (int t = 0; t < F::kTiles; ++t) o[t] *= shrink;

    // A value that is not finite meets weights of 0 in the rows that do not see
    // it: such steps, where rows see different keys, go key by key.
    bool plain = true;
    if (!whole) {
      bool odd = false;
#pragma unroll
      for (int j = 0; j < NSUB * 4; ++j)
#pragma unroll
        for (int u = 0; u < F::U; ++u) {
          if (!vok[j]) v[j][u] = VPiece<TC, F::E>{};
#pragma unroll
          for (int e = 0; e < F::E; ++e) odd |= !(fabsf((float)v[j][u].v[e]) < __builtin_inff());
        }
      plain = __ballot(odd) == 0;
    }
    if (plain) {
      if constexpr (sizeof(TC) == 2) {
        vec p[NP];
#pragma unroll
        for (int j = 0; j < 8; ++j) split<NP>(w[j], p, j);
#pragma unroll
        for (int u = 0; u < F::U; ++u)
#pragma unroll
          for (int e = 0; e < F::E; ++e) {
            vec x;
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = v[j][u].v[e];
#pragma unroll
            for (int n = NP - 1; n >= 0; --n) o[u * F::E + e] = mma16(x, p[n], o[u * F::E + e]);
          }
      } else {
#pragma unroll
        for (int u = 0; u < F::U; ++u)
#pragma unroll
          for (int e = 0; e < F::E; ++e) {
            f4 x, p;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              x[j] = v[j][u].v[e];
              p[j] = w[j];
            }
            o[u * F::E + e] = mma16(x, p, o[u * F::E + e]);
          }
      }
    } else {
      float* pw = few_lds + wave * 16 * (KT + 1);
#pragma unroll
      for (int j = 0; j < NSUB * 4; ++j) pw[i * (KT + 1) + (j >> 2) * 16 + g * 4 + (j & 3)] = vis[j] ? w[j] : -1.f;
      __builtin_amdgcn_wave_barrier();
      for (int n = 0; n < KT; ++n) {
        const float x = pw[i * (KT + 1) + n];
        const int64_t key = kb + n;
        const int p = key < k1 ? page_of(a.p, c.slot, key) : -1;
        if (p < 0 || x == -1.f) continue;
        const TC* row_v = base + a.p.value_offset + (int64_t)p * a.p.page_stride + (key & mask) * a.p.token_stride;
#pragma unroll
        for (int u = 0; u < F::U; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int e = 0; e < F::E; ++e) {
              const int d = u * 16 * F::E + (g * 4 + r) * F::E + e;
              if (d < dim) o[u * F::E + e][r] += x * (float)row_v[d];
            }
      }
      __builtin_amdgcn_wave_barrier();
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
      if (d == 0) parts.ml[at] = make_float2(rt, sum);
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

// One row's parts: weights from their maxima, then the weighted sum; a
// workgroup takes a row, D / 4 lanes across it and the parts side by side.
constexpr int kJoinThreads = 256;

template <typename T, int D>
__global__ __launch_bounds__(kJoinThreads) void few_join_kernel(AttendArgs a, Parts parts, int tiles, float shift) {
  constexpr int kAcross = D / 4, kSide = kJoinThreads / kAcross;
  __shared__ f4 sums[kSide][kAcross];
  __shared__ float ls[kSide];
  const int task = blockIdx.x / 16, r = blockIdx.x % 16, kvh = blockIdx.y;
  const int seq = task / tiles, tile = task - seq * tiles;
  const Chunk c = chunk_of(a.p, seq);
  const int rows = c.n * a.group;
  if ((rows > 16 && c.n != 1) || tile * 16 + r >= rows) return;
  const int r0 = tile * 16, rn = rows - r0 < 16 ? rows - r0 : 16;
  const Span span = span_of(sees_of(a, c), r0 / a.group, (r0 + rn - 1) / a.group, parts.keys, parts.most);
  if (span.parts <= 1) return;
  const int64_t at = ((int64_t)task * a.p.kv_heads + kvh) * 16 + r;
  float top = minus_inf();
  for (int p = threadIdx.x & 63; p < span.parts; p += 64) top = fmaxf(top, parts.ml[p * parts.rows + at].x);
#pragma unroll
  for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  const float from = top == minus_inf() ? 0.f : top;
  const int x = threadIdx.x % kAcross, side = threadIdx.x / kAcross;
  f4 s{0, 0, 0, 0};
  float l = 0.f;
#pragma unroll 4
  for (int p = side; p < span.parts; p += kSide) {
    const float2 ml = parts.ml[p * parts.rows + at];
    const float w = exp2_(ml.x - from);
    s += *reinterpret_cast<const f4*>(parts.o + (p * parts.rows + at) * D + x * 4) * w;
    l += ml.y * w;
  }
  sums[side][x] = s;
  if (x == 0) ls[side] = l;
  __syncthreads();
  if (side) return;
  float sum = ls[0];
#pragma unroll
  for (int y = 1; y < kSide; ++y) {
    s += sums[y][x];
    sum += ls[y];
  }
  const int rr = r0 + r, token = c.begin + rr / a.group, head = kvh * a.group + rr % a.group;
  T* out = static_cast<T*>(a.out.d) + (int64_t)token * a.out.token_stride + (int64_t)head * a.out.head_stride;
#pragma unroll
  for (int y = 0; y < 4; ++y)
    if (x * 4 + y < a.p.dim) out[x * 4 + y] = (T)(sum == 0.f ? 0.f : s[y] / sum);
  if (a.lse && x == 0)
    a.lse[(int64_t)token * a.heads + head] =
        sum == 0.f ? minus_inf() : (from + (__builtin_amdgcn_logf(sum) - shift)) * kLn2;
}

// ---------------------------------------------------------------- the others

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
  return x;
}

template <typename T, typename TC>
__global__ __launch_bounds__(64) void attend_kernel(AttendArgs a) {
  const int token = blockIdx.x, head = blockIdx.y, lane = threadIdx.x;
  int seq = -1;
  for (int s0 = 0; s0 < a.p.seqs + 1; s0 += 64) {
    const int s = s0 + lane;
    const int n = __popcll(__ballot(s <= a.p.seqs && a.p.starts[s <= a.p.seqs ? s : a.p.seqs] <= token));
    seq += n;
    if (n < 64) break;
  }
  if (seq < 0 || seq >= a.p.seqs) return;
  const Chunk c = chunk_of(a.p, seq);
  if (c.n * a.group <= 16 || c.n == 1) return;
  const int64_t pos = position_of(a.p, c, token - c.begin);
  int64_t lo = a.first && c.slot >= 0 ? a.first[c.slot] : 0, hi = pos + 1 < c.len ? pos + 1 : c.len;
  if (lo < 0) lo = 0;
  if (a.window > 0 && pos + 1 - a.window > lo) lo = pos + 1 - a.window;
  const T* q = static_cast<const T*>(a.q.d) + token * a.q.token_stride + head * a.q.head_stride;
  float x[4], o[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = lane + 64 * i < a.p.dim ? (float)q[lane + 64 * i] : 0.f;
  float m = -__builtin_inff(), l = 0;
  for (int64_t j = lo; j < hi; ++j) {
    const int page = page_of(a.p, c.slot, j);
    if (page < 0) continue;
    const TC* k = static_cast<const TC*>(a.p.kv) + token_offset(a.p, page, j) + head / a.group * a.p.head_stride;
    const TC* v = k + a.p.value_offset;
    float s = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (lane + 64 * i < a.p.dim) s += x[i] * (float)k[lane + 64 * i];
    s = wave_sum(s) * a.scale;
    if (s == -__builtin_inff()) continue;
    const float top = fmaxf(m, s), f = expf(m - top), w = expf(s - top);
    l = l * f + w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (lane + 64 * i < a.p.dim) o[i] = o[i] * f + w * (float)v[lane + 64 * i];
    m = top;
  }
  T* out = static_cast<T*>(a.out.d) + token * a.out.token_stride + head * a.out.head_stride;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 64 * i < a.p.dim) out[lane + 64 * i] = (T)(l != 0 ? o[i] / l : 0.f);
  if (a.lse && lane == 0) a.lse[(int64_t)token * a.heads + head] = l != 0 ? m + logf(l) : -__builtin_inff();
}

int width_of(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

// How the call is dealt out, by its sizes and the caller's hints alone.
AttendPlan plan_of(const AttendArgs& a, int max_new, int64_t max_len) {
  AttendPlan p{};
  if (a.p.seqs < 1 || a.p.tokens < 1) return p;
  const int D = width_of(a.p.dim);
  int64_t most = (int64_t)a.p.max_pages << a.p.page_shift;
  if (max_len > 0 && max_len < most) most = max_len;
  int64_t longest = max_new > 0 && max_new < a.p.tokens ? max_new : a.p.tokens;
  if (a.window > 0 && most > (int64_t)a.window + longest) most = (int64_t)a.window + longest;
  p.few = true;
  p.few_tiles = (a.group + 15) / 16;
  const int64_t tasks = (int64_t)a.p.seqs * p.few_tiles * a.p.kv_heads;
  // Parts of at least 256 keys, and as many as give every CU three workgroups.
  const int64_t want = (768 + tasks - 1) / tasks;
  int64_t keys = (most + want - 1) / want;
  if (keys > 2048) keys = 2048;
  if (keys < 256) keys = 256;
  p.few_keys = (keys + 127) / 128 * 128;
  int64_t n = (most + p.few_keys - 1) / p.few_keys;
  p.few_most = (int)(n < 1 ? 1 : n > 4096 ? 4096 : n);
  p.few_rows = tasks * 16;
  p.few_bytes = p.few_most > 1 ? (size_t)p.few_most * p.few_rows * (D * sizeof(float) + sizeof(float2)) : 0;
  p.chunk = longest > 1 && longest * a.group > 16;
  return p;
}

template <typename T, typename TC, int D>
hipError_t few_of(const AttendArgs& a, const AttendPlan& p, void* work, hipStream_t s) {
  Parts parts{};
  parts.rows = p.few_rows;
  parts.keys = p.few_keys;
  parts.most = p.few_most;
  parts.o = static_cast<float*>(work);
  parts.ml = reinterpret_cast<float2*>(parts.o + (int64_t)p.few_most * p.few_rows * D);
  constexpr size_t lds = (size_t)kFewWaves * 16 * (D + 4) * sizeof(float);
  if (lds > 60000) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(few_kernel<T, TC, D>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
  }
  few_kernel<T, TC, D><<<dim3(a.p.seqs * p.few_tiles, a.p.kv_heads, p.few_most), kFewThreads, lds, s>>>(a, parts, p.few_tiles, p.chunk);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.few_most <= 1) return e;
  few_join_kernel<T, D><<<dim3(a.p.seqs * p.few_tiles * 16, a.p.kv_heads), kJoinThreads, 0, s>>>(a, parts, p.few_tiles,
                                                                                        Elem<TC>::kShift);
  return hipGetLastError();
}

template <typename T, typename TC>
hipError_t attend_of(const AttendArgs& a, const AttendPlan& p, void* work, hipStream_t s) {
  hipError_t e = hipSuccess;
  if (p.few) {
    switch (width_of(a.p.dim)) {
      case 64: e = few_of<T, TC, 64>(a, p, work, s); break;
      case 128: e = few_of<T, TC, 128>(a, p, work, s); break;
      default: e = few_of<T, TC, 256>(a, p, work, s); break;
    }
  }
  if (e == hipSuccess && p.chunk) {
    attend_kernel<T, TC><<<dim3(a.p.tokens, a.heads), 64, 0, s>>>(a);
    e = hipGetLastError();
  }
  return e;
}

}  // namespace

size_t attend_workspace(const AttendArgs& a, int max_new, int64_t max_len) {
  const AttendPlan p = plan_of(a, max_new, max_len);
  return p.few_bytes;
}

hipError_t launch_attend(const AttendArgs& a, int type, int cache_type, int max_new, int64_t max_len, void* work,
                         hipStream_t s) {
  const AttendPlan p = plan_of(a, max_new, max_len);
  if (type == kF32) {
    if (cache_type == kF32) return attend_of<float, float>(a, p, work, s);
    if (cache_type == kF16) return attend_of<float, _Float16>(a, p, work, s);
    return attend_of<float, __bf16>(a, p, work, s);
  }
  if (type == kF16) return attend_of<_Float16, _Float16>(a, p, work, s);
  return attend_of<__bf16, __bf16>(a, p, work, s);
}

}  // namespace nls
