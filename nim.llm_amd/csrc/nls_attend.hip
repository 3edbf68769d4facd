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
  // weights: 16-bit queries' too are two parts, since products cost nothing here
  static constexpr int kWeightParts = sizeof(T) == 2 ? 2 : kParts;
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
  constexpr int NP = F::kParts, NW = F::kWeightParts, KT = F::KT, NSUB = F::NSUB;
  extern __shared__ float few_lds[];  // [wave][16][D + 4] sums
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
    top = ceilf(fmaxf(top, m));  // whole: what it is taken from is exact
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

    if (!whole) {
#pragma unroll
      for (int j = 0; j < NSUB * 4; ++j)
#pragma unroll
        for (int u = 0; u < F::U; ++u)
          if (!vok[j]) v[j][u] = VPiece<TC, F::E>{};
    }
    constexpr int kDepth = sizeof(vec) / sizeof(TC);
    vec p[NW], seen;
#pragma unroll
    for (int j = 0; j < kDepth; ++j) {
      split<NW>(w[j], p, j);
      seen[j] = vis[j] ? 1.f : 0.f;
    }
#pragma unroll
    for (int u = 0; u < F::U; ++u)
#pragma unroll
      for (int e = 0; e < F::E; ++e) {
        vec x;
#pragma unroll
        for (int j = 0; j < kDepth; ++j) x[j] = v[j][u].v[e];
        f4& sum_of = o[u * F::E + e];
        if (!whole) only_seen(x, seen, sum_of, [](vec y, vec z, f4 c) { return mma16(y, z, c); });
#pragma unroll
        for (int n = NW - 1; n >= 0; --n) sum_of = mma16(x, p[n], sum_of);
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

// One row's parts: weights from their maxima, then the weighted sum; a
// workgroup takes a row, D / 4 lanes across it and the parts side by side.
constexpr int kJoinThreads = 256;

// `tiles`: few_kernel's tiles per sequence; 0: the rows are chunk_kernel's.
template <typename T, int D>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(AttendArgs a, Parts parts, int tiles, float shift) {
  constexpr int kAcross = D / 4, kSide = kJoinThreads / kAcross;
  __shared__ f4 sums[kSide][kAcross];
  __shared__ float ls[kSide], lrs[kSide];
  const int size = tiles ? 16 : kChunkTile;
  const int task = blockIdx.x / size, r = blockIdx.x % size, kvh = blockIdx.y;
  int seq = -1, r0;
  if (tiles) {
    seq = task / tiles;
    r0 = (task - seq * tiles) * 16;
  } else {
    const int lane = threadIdx.x & 63;
    for (int s0 = 0; s0 < a.p.seqs; s0 += 64) {
      const int s = s0 + lane;
      const int n = __popcll(__ballot(s < a.p.seqs && tile_base(a.p.starts[s < a.p.seqs ? s : 0], a.group, kChunkTile, s) <= task));
      seq += n;
      if (n < 64) break;
    }
    if (seq < 0) return;
  }
  const Chunk c = chunk_of(a.p, seq);
  const int rows = c.n * a.group;
  if ((rows <= 16 || c.n == 1) != (tiles > 0)) return;
  if (!tiles) {
    const int64_t x = (task - tile_base(c.begin, a.group, kChunkTile, seq)) * kChunkTile;
    if (x < 0 || x >= rows) return;
    r0 = (int)x;
  }
  if (r0 + r >= rows) return;
  const int rn = rows - r0 < size ? rows - r0 : size;
  const Span span = span_of(sees_of(a, c), r0 / a.group, (r0 + rn - 1) / a.group, parts.keys, parts.most);
  if (span.parts <= 1) return;
  const int64_t at = ((int64_t)task * a.p.kv_heads + kvh) * size + r;
  float top = minus_inf();
  for (int p = threadIdx.x & 63; p < span.parts; p += 64) top = fmaxf(top, parts.ml[p * parts.rows + at][0]);
#pragma unroll
  for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
  const float from = top == minus_inf() ? 0.f : top;
  const int x = threadIdx.x % kAcross, side = threadIdx.x / kAcross;
  f4 s{0, 0, 0, 0};
  float l = 0.f, lr = 0.f;
#pragma unroll 4
  for (int p = side; p < span.parts; p += kSide) {
    const f4 ml = parts.ml[p * parts.rows + at];
    const float w = exp2_(ml[0] - from);
    s += *reinterpret_cast<const f4*>(parts.o + (p * parts.rows + at) * D + x * 4) * w;
    l += ml[1] * w;
    lr += ml[2] * w;
  }
  sums[side][x] = s;
  if (x == 0) {
    ls[side] = l;
    lrs[side] = lr;
  }
  __syncthreads();
  if (side) return;
  float sum = ls[0], sumr = lrs[0];
#pragma unroll
  for (int y = 1; y < kSide; ++y) {
    s += sums[y][x];
    sum += ls[y];
    sumr += lrs[y];
  }
  const int rr = r0 + r, token = c.begin + rr / a.group, head = kvh * a.group + rr % a.group;
  T* out = static_cast<T*>(a.out.d) + (int64_t)token * a.out.token_stride + (int64_t)head * a.out.head_stride;
#pragma unroll
  for (int y = 0; y < 4; ++y)
    if (x * 4 + y < a.p.dim) out[x * 4 + y] = (T)(sumr == 0.f ? 0.f : s[y] / sumr);
  if (a.lse && x == 0)
    a.lse[(int64_t)token * a.heads + head] =
        sum == 0.f ? minus_inf() : (from + (__builtin_amdgcn_logf(sum) - shift)) * kLn2;
}

int width_of(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

// Parts of the keys, so that `tasks` workgroups become about `want`, but of no
// fewer than `least` keys each and no more than `top`.
Parts parts_of_keys(int64_t most, int64_t tasks, int64_t want, int64_t least, int64_t top) {
  Parts p{};
  const int64_t n = (want + tasks - 1) / tasks;
  int64_t keys = (most + n - 1) / n;
  if (keys > top) keys = top;
  if (keys < least) keys = least;
  p.keys = (keys + 127) / 128 * 128;
  const int64_t m = (most + p.keys - 1) / p.keys;
  p.most = (int)(m < 1 ? 1 : m > 4096 ? 4096 : m);
  return p;
}

// How the call is dealt out, by its sizes and the caller's hints alone.
AttendPlan plan_of(const AttendArgs& a, int max_new, int64_t max_len) {
  AttendPlan p{};
  if (a.p.seqs < 1 || a.p.tokens < 1) return p;
  const int D = width_of(a.p.dim);
  int64_t most = (int64_t)a.p.max_pages << a.p.page_shift;
  if (max_len > 0 && max_len < most) most = max_len;
  int64_t longest = max_new > 0 && max_new < a.p.tokens ? max_new : a.p.tokens;
  if (a.window > 0 && most > (int64_t)a.window + longest) most = (int64_t)a.window + longest;
  const size_t per_row = D * sizeof(float) + sizeof(f4);
  p.few = true;
  p.few_tiles = (a.group + 15) / 16;
  const int64_t tasks = (int64_t)a.p.seqs * p.few_tiles * a.p.kv_heads;
  // Parts of at least 256 keys, and as many as give every CU three workgroups.
  p.few_parts = parts_of_keys(most, tasks, 768, 256, 2048);
  p.few_parts.rows = tasks * 16;
  p.few_bytes = p.few_parts.most > 1 ? p.few_parts.most * p.few_parts.rows * per_row : 0;
  p.chunk = longest > 1 && longest * a.group > 16;
  if (p.chunk) {
    p.chunk_tiles = tile_count(a.p.tokens, a.group, kChunkTile, a.p.seqs);
    const int64_t wgs = p.chunk_tiles * a.p.kv_heads;
    p.chunk_parts = parts_of_keys(most, wgs, 512, 512, most);
    p.chunk_parts.rows = wgs * kChunkTile;
    p.chunk_bytes = p.chunk_parts.most > 1 ? p.chunk_parts.most * p.chunk_parts.rows * per_row : 0;
  }
  return p;
}

Parts placed(Parts p, void* work, int D) {
  p.o = static_cast<float*>(work);
  p.ml = reinterpret_cast<f4*>(p.o + p.most * p.rows * D);
  return p;
}

template <typename T, typename TC, int D>
hipError_t attend_width(const AttendArgs& a, const AttendPlan& p, int type, int cache_type, char* work, hipStream_t s) {
  hipError_t e = hipSuccess;
  if (p.few) {
    const Parts parts = placed(p.few_parts, work, D);
    constexpr size_t lds = (size_t)kFewWaves * 16 * (D + 4) * sizeof(float);
    if (lds > 60000) {
      e = hipFuncSetAttribute(reinterpret_cast<const void*>(few_kernel<T, TC, D>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
      if (e != hipSuccess) return e;
    }
    few_kernel<T, TC, D><<<dim3(a.p.seqs * p.few_tiles, a.p.kv_heads, parts.most), kFewThreads, lds, s>>>(
        a, parts, p.few_tiles, p.chunk);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    if (parts.most > 1) {
      join_kernel<T, D><<<dim3(a.p.seqs * p.few_tiles * 16, a.p.kv_heads), kJoinThreads, 0, s>>>(
          a, parts, p.few_tiles, Elem<TC>::kShift);
      if ((e = hipGetLastError()) != hipSuccess) return e;
    }
  }
  if (p.chunk) {
    const Parts parts = placed(p.chunk_parts, work + (p.few_bytes + 255) / 256 * 256, D);
    if ((e = launch_chunk(a, type, cache_type, parts, p.chunk_tiles, s)) != hipSuccess) return e;
    if (parts.most > 1) {
      join_kernel<T, D><<<dim3((unsigned)(p.chunk_tiles * kChunkTile), a.p.kv_heads), kJoinThreads, 0, s>>>(
          a, parts, 0, chunk_shift<TC>());
      e = hipGetLastError();
    }
  }
  return e;
}

template <typename T, typename TC>
hipError_t attend_types(const AttendArgs& a, const AttendPlan& p, int type, int cache_type, char* work, hipStream_t s) {
  switch (width_of(a.p.dim)) {
    case 64: return attend_width<T, TC, 64>(a, p, type, cache_type, work, s);
    case 128: return attend_width<T, TC, 128>(a, p, type, cache_type, work, s);
    default: return attend_width<T, TC, 256>(a, p, type, cache_type, work, s);
  }
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
