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
#include "nls_attend_few.h"
#include "nls_attend_quant.h"

namespace nls {
namespace {

template <typename T, typename TC, int D, bool kPad>
__global__ __launch_bounds__(kFewThreads, D == 256 ? 1 : 2) void few_kernel(AttendArgs a, Parts parts, int tiles, bool chunk_runs) {
  few_rows<T, TC, D, kPad>(a, parts, tiles, chunk_runs, blockIdx.x, blockIdx.z);
}

// ---------------------------------------------------------------- joining parts

// One row's parts: weights from their maxima, then the weighted sum, D / 4 lanes
// across the row and the parts side by side.  kWaves waves take a row: four
// where rows are few and their parts many, else one.
constexpr int kJoinThreads = 256;

// The first few_rows rows are (sequence, one of its first `per` tokens, head),
// of few_rows; the others all of the call's, of chunk_rows.
template <typename T, int D, int kWaves>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(AttendArgs a, Parts few, Parts chunk, int64_t few_rows,
                                                            int per, int tiles, bool alone, int chunk_tile,
                                                            float few_shift, float chunk_shift) {
  constexpr int kAcross = D / 4, kSide = 64 * kWaves / kAcross;
  constexpr int kRows = kJoinThreads / (64 * kWaves);  // of a workgroup
  __shared__ f4 sums[kRows][kSide][kAcross];
  __shared__ f4 ls[kRows][kSide];
  const int lane = threadIdx.x & 63, sub = threadIdx.x / (64 * kWaves), in = threadIdx.x % (64 * kWaves);
  const int64_t index = (int64_t)blockIdx.x * kRows + sub;
  const bool is_few = index < few_rows;
  const int64_t rest = is_few ? index : index - few_rows;
  const int head = (int)(rest % a.heads), kvh = head / a.group, size = is_few ? 16 : chunk_tile;
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

// Parts of the keys, `n` for each of `tasks` workgroups, of no fewer than `least`
// keys each and, so that long and short contexts of a batch take their turns, no
// more than `top`; but not beyond 8192 workgroups, whose sums wait in the
// workspace.
Parts parts_of_keys(int64_t most, int64_t tasks, int64_t n, int64_t least, int64_t top) {
  Parts p{};
  const int64_t cap = top < most && n < 8192 / tasks ? 8192 / tasks : n;
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
AttendPlan plan_of(const AttendArgs& a, int type, int max_new, int64_t max_len) {
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
    // Parts of at least 256 keys (one token over 8000 fp32 keys, heads of 64: 17.7
    // us, with parts of 512 20.8), and as many as give every CU two workgroups (one
    // token over 131071 keys: 94.1 us so, 96.8 with three); up to 768 keys are not
    // split: the second launch costs the host more than it saves the GPU (517 keys:
    // 13.2 us a call whole, 17.2 in three parts, 12.8 and 12.3 in a graph; 24
    // contexts of 517: 17.4 and 18.4, 17.8 and 18.8 in a graph).  Blocks are fewer
    // bytes a key: their parts end at 4096 (64 contexts of up to 16384, Q4_0: 203 us;
    // at 2048 220, at 8192 223).
    p.few_parts = parts_of_keys(most, tasks, (512 + tasks - 1) / tasks, most <= 768 ? 768 : 256, quant_type(a.cache_type) ? 4096 : 2048);
    p.few_parts.rows = tasks * 16;
    p.few_bytes = p.few_parts.most > 1 ? p.few_parts.most * p.few_parts.rows * per_row : 0;
  }
  if (p.chunk) {
    const bool quant = quant_type(a.cache_type);
    const int tile = !quant ? kChunkTile : type == kBF16 ? quant_tile<__bf16>(a.p.dim / 32) : quant_tile<float>(a.p.dim / 32);
    p.chunk_tiles = tile_count(a.p.tokens, a.group, tile, a.p.seqs);
    // Two workgroups per CU (heads of up to 64: three), of the tiles that have rows
    // when they are all of one sequence (509 tokens of 28 heads beside 16 that
    // decode: 141 us when the empty tiles of those count too, 126 us so); parts of
    // at least 512 keys.  No more than that, so that few rows find room, and none
    // waits for a second turn where that many run at once (fp32 queries over a
    // 16-bit cache, and 16-bit ones in heads of 72 to 128), unless a quarter of the
    // places stayed empty (that batch, few rows in the same launch: 135 us when
    // rounded up, 126 so; 512 tokens beside 32 over 8000 keys, bf16: 249 and 210;
    // 1600 tokens over 16000: 582 and 516).  One number for all types: registers let
    // four run at once of 16-bit queries in heads of up to 64, two and one (heads of
    // 72 to 128) over an fp32 cache, one of wider heads (300 tokens over 4000 fp32
    // keys, heads of 128: 227 us when rounded up, 262 so).  Over blocks one workgroup
    // runs where it has eight waves or heads are beyond 128.
    const int64_t wgs = ((int64_t)a.p.tokens * a.group + tile - 1) / tile * a.p.kv_heads;
    const int64_t places = tile > kChunkTile || (quant && D == 256) ? 256 : D == 64 ? 768 : 512, down = places / wgs > 1 ? places / wgs : 1;
    // (tiles of no rows are launched too: sequences beyond number do not multiply)
    const int64_t n = down * wgs * 4 >= places * 3 ? down : down + 1, room = 16384 / (p.chunk_tiles * a.p.kv_heads);
    p.chunk_parts = parts_of_keys(most, wgs, n < room ? n : room > 1 ? room : 1, 512, most);
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

// The rows whose keys were split.
template <typename T, int D>
hipError_t join(const AttendArgs& a, const AttendPlan& p, const Parts& few, const Parts& chunk, int chunk_tile,
                float few_shift, float chunk_shift, hipStream_t s) {
  const int per = a.group >= 16 ? 1 : 16 / a.group;  // tokens that few_rows takes of a sequence
  const int64_t few_rows = few.most > 1 ? (int64_t)a.p.seqs * per * a.heads : 0;
  const int64_t rows = few_rows + (chunk.most > 1 ? (int64_t)a.p.tokens * a.heads : 0);
  if (rows == 0) return hipSuccess;
  if (rows < 1024)
    join_kernel<T, D, 4><<<(unsigned)rows, kJoinThreads, 0, s>>>(a, few, chunk, few_rows, per, p.few_tiles, !p.few,
                                                                chunk_tile, few_shift, chunk_shift);
  else
    join_kernel<T, D, 1><<<(unsigned)((rows + 3) / 4), kJoinThreads, 0, s>>>(a, few, chunk, few_rows, per, p.few_tiles, !p.few,
                                                                          chunk_tile, few_shift, chunk_shift);
  return hipGetLastError();
}

template <typename T, typename TC, int D, bool kPad>
hipError_t attend_width(const AttendArgs& a, const AttendPlan& p, int type, int cache_type, char* work, hipStream_t s) {
  const Parts few = placed(p.few_parts, work, D);
  const Parts chunk = placed(p.chunk_parts, work + (p.few_bytes + 255) / 256 * 256, D);
  constexpr size_t lds = few_lds_bytes(D);
  hipError_t e;
  if (p.few && !(p.chunk && together<TC, D>())) {
    if (lds > 60000) {
      e = hipFuncSetAttribute(reinterpret_cast<const void*>(few_kernel<T, TC, D, kPad>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
      if (e != hipSuccess) return e;
    }
    few_kernel<T, TC, D, kPad><<<dim3(a.p.kv_heads * a.p.seqs * p.few_tiles, 1, few.most), kFewThreads, lds, s>>>(
        a, few, p.few_tiles, p.chunk);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  if (p.chunk &&
      (e = launch_chunk(a, type, cache_type, chunk, p.chunk_tiles, p.few ? &few : nullptr, p.few_tiles, s)) != hipSuccess)
    return e;
  return join<T, D>(a, p, few, chunk, kChunkTile, Elem<TC>::kShift, chunk_shift<TC>(), s);
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

// Pages of blocks.
template <typename T, int D>
hipError_t attend_quant_width(const AttendArgs& a, const AttendPlan& p, int type, int cache_type, char* work,
                              hipStream_t s) {
  const Parts few = placed(p.few_parts, work, D);
  const Parts chunk = placed(p.chunk_parts, work + (p.few_bytes + 255) / 256 * 256, D);
  hipError_t e;
  if (p.few && (e = launch_few_quant(a, type, cache_type, few, p.few_tiles, p.chunk, s)) != hipSuccess) return e;
  if (p.chunk && (e = launch_chunk_quant(a, type, cache_type, chunk, p.chunk_tiles, !p.few, s)) != hipSuccess) return e;
  return join<T, D>(a, p, few, chunk, quant_tile<T>(a.p.dim / 32), kQuantShift, chunk_shift<_Float16>(), s);
}

template <typename T>
hipError_t attend_quant(const AttendArgs& a, const AttendPlan& p, int type, int cache_type, char* work, hipStream_t s) {
  if (a.p.dim <= 64) return attend_quant_width<T, 64>(a, p, type, cache_type, work, s);
  if (a.p.dim <= 128) return attend_quant_width<T, 128>(a, p, type, cache_type, work, s);
  return attend_quant_width<T, 256>(a, p, type, cache_type, work, s);
}

}  // namespace

size_t attend_workspace(const AttendArgs& a, int max_new, int64_t max_len) {
  // (whatever type the queries will be: chunks over blocks are dealt out by it)
  size_t most = 0;
  for (int type : {kF32, kBF16}) {
    const AttendPlan p = plan_of(a, type, max_new, max_len);
    const size_t n = (p.few_bytes + 255) / 256 * 256 + p.chunk_bytes;
    most = n > most ? n : most;
  }
  return most;
}

hipError_t launch_attend(const AttendArgs& a, int type, int cache_type, int max_new, int64_t max_len, void* work,
                         hipStream_t s) {
  const AttendPlan p = plan_of(a, type, max_new, max_len);
  char* w = static_cast<char*>(work);
  if (quant_type(cache_type)) {
    if (a.p.seqs < 1 || a.p.tokens < 1) return hipSuccess;
    if (type == kF32) return attend_quant<float>(a, p, type, cache_type, w, s);
    if (type == kF16) return attend_quant<_Float16>(a, p, type, cache_type, w, s);
    return attend_quant<__bf16>(a, p, type, cache_type, w, s);
  }
  if (type == kF32) {
    if (cache_type == kF32) return attend_types<float, float>(a, p, type, cache_type, w, s);
    if (cache_type == kF16) return attend_types<float, _Float16>(a, p, type, cache_type, w, s);
    return attend_types<float, __bf16>(a, p, type, cache_type, w, s);
  }
  if (type == kF16) return attend_types<_Float16, _Float16>(a, p, type, cache_type, w, s);
  return attend_types<__bf16, __bf16>(a, p, type, cache_type, w, s);
}

}  // namespace nls
