// nls_attend_chunk.hip -- attention of chunks: sequences of more than 16 rows
// (token, head of the group) per kv head.
//
// Bound by the products: 4 D per visible (row, key) on the matrix cores, times
// the parts that fp32 queries and weights are split into.  A workgroup takes 128
// rows of one (sequence, kv head), 32 per wave, and walks the keys in tiles, two
// of which have room in LDS: while all four waves use the current one, K of the
// next is on its way into registers; then it goes to LDS, and V after it, whose
// wait the CU's other waves fill.  As for few rows, S^T = K Q^T and O^T = V^T P^T,
// here with 32 x 32 products: a lane holds one row's scores of keys
// 8 b + 4 h + 0 .. 3 (h = lane / 32), which are its weights' places in the second
// product.
//
// LDS holds K and V rows as they are in memory, their 16-byte pieces permuted
// within a row so that 16 lanes which read 16 rows (K), or 32 which read 4 rows
// (V), meet all banks.  16-bit V is read with the transposing load: 4 keys of
// one element per lane.
//
// The running maximum follows the scores only when it is passed by 2^8: until
// then weights grow up to 2^8 times the largest one seen, which fp32 sums and
// either 16-bit type hold without loss, and the sums need no rescaling.  It is
// a whole number, so that what it is taken from and given back to is exact.
//
// 2048 tokens over 16384 keys, 32 heads of 128, fp32 over fp16: 930 to
// 960 us, 1073 to 1110 TFLOP/s of products, which is what a large fp16 matrix
// product reaches on this card.  Two prompts of 4001, heads of 64, bf16: 160 us, 630 TFLOP/s: 16
// exponentials and about 90 other vector instructions stand beside each 8
// products.  (There, both halves of a tile in turn under each other's
// exponentials take 191 registers, and 206 us.)
//
// Registers that do not suffice, in bytes of scratch per lane: fp32 over bf16 in
// heads of 72 to 128 40, 16-bit queries in heads of up to 64 28 (for the fourth
// wave), and heads beyond 128, one wave per SIMD, 332 (fp32 over bf16), 276 (over
// fp32) and 108 (over fp16).
#include "nls_attend_few.h"

namespace nls {
namespace {

constexpr int kChunkWaves = 4;
constexpr int kChunkThreads = 64 * kChunkWaves;
static_assert(kChunkTile == 32 * kChunkWaves, "32 rows per wave");

__device__ __forceinline__ f16x mma32(h8 a, h8 b, f16x c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f16x mma32(b8 a, b8 b, f16x c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f16x mma32(f4 a, f4 b, f16x c) {
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

template <typename T, typename TC, int D>
struct Tile {
  static constexpr bool kWide = sizeof(TC) == 4;               // an fp32 cache
  static constexpr int NP = parts_of<T, TC>();
  static constexpr int KT = kWide || D == 256 ? 32 : 64;       // keys per tile
  static constexpr int KD = 16 / (int)sizeof(TC);              // elements of a 16-byte piece
  static constexpr int kPieces = D / KD;                       // of a row
  static constexpr int KC = kPieces / 2;                       // steps of the first product
  static constexpr int kTiles = D / 32;                        // of O^T
  static constexpr int kBytes = KT * D * (int)sizeof(TC);      // of K, or V
  static constexpr int kStage = kBytes / 16 / kChunkThreads;   // pieces of K (or V) per thread
  static constexpr int kRowsPerStep = kChunkThreads / kPieces; // rows that the workgroup fetches at a time
  static constexpr float kShift = chunk_shift<TC>();
  // the head's element of row x of O^T's tile t; kRun tiles hold neighbours
  static constexpr int kRun = kWide ? (D == 64 ? 2 : 4) : 1;
  static constexpr int kStore = kRun == 1 ? 4 : kRun;  // neighbouring elements that a lane stores
  static __device__ __forceinline__ constexpr int element(int t, int x) {
    return kWide ? t / kRun * 32 * kRun + x * kRun + t % kRun : t * 32 + x;
  }
  // where piece c of row r lies within the row
  static __device__ __forceinline__ int k_piece(int r, int c) {
    return kPieces >= 16 ? c ^ (r & 15) : c ^ ((r >> 1) & 7);
  }
  static __device__ __forceinline__ int v_piece(int r, int c) {
    if (kWide) return c;
    return kPieces >= 16 ? c ^ ((r & 3) << 2) : c ^ (((r >> 1) & 1) << 2);
  }
};

// The neighbouring elements of this lane's row among tiles t .. t + kRun - 1
// and rows y .. of them: four (16-bit caches: rows y .. y + 3 of one tile).
template <typename L, typename F>
__device__ __forceinline__ void put_run(const f16x* o, int t, int y, int h, float f, F&& to) {
  float x[4];
  const int d = L::element(t, 8 * (y >> 2) + 4 * h + (y & 3));
  if constexpr (L::kRun == 1) {
#pragma unroll
    for (int z = 0; z < 4; ++z) x[z] = o[t][y + z] * f;
    to(d, x);
  } else {
#pragma unroll
    for (int z = 0; z < L::kRun; ++z) x[z] = o[t + z][y] * f;
    to(d, x);
  }
}

typedef short s4x __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4x* lds_s4x;

// Waves per SIMD that registers are kept for.  Narrow heads of 16-bit queries
// have so many instructions beside their products that four waves hide each
// other's best (two prompts of 4001: 171 us with three, 166 with four).
template <typename T, typename TC, int D>
constexpr int chunk_waves() {
  return sizeof(TC) == 4 || D == 256 ? 1 : D == 64 && sizeof(T) == 2 ? 4 : 2;
}

template <typename T, typename TC, int D>
__device__ __forceinline__ void chunk_rows(const AttendArgs& a, const Parts& parts, bool alone, int group_at,
                                           int groups, int part) {
  using L = Tile<T, TC, D>;
  using vec = typename Elem<TC>::vec;
  constexpr int NP = L::NP, KT = L::KT, NS = KT / 32;
  extern __shared__ __align__(16) char chunk_lds[];  // [2][K, V]
  __shared__ uint8_t noted[2][KT][L::kPieces];       // bit j: element j of a piece of V was not finite
  __shared__ int has_noted[2][kChunkWaves];
  __shared__ float max_times[NP == 2 ? kChunkTile : 1];

  const int kvh = group_at % a.p.kv_heads, tile = (groups - 1 - group_at) / a.p.kv_heads;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 31, h = lane >> 5;

  // the sequence whose tiles begin at or before this one
  int seq = -1;
  for (int s0 = 0; s0 < a.p.seqs; s0 += 64) {
    const int s = s0 + lane;
    const int n = __popcll(__ballot(s < a.p.seqs && tile_base(a.p.starts[s < a.p.seqs ? s : 0], a.group, kChunkTile, s) <= tile));
    seq += n;
    if (n < 64) break;
  }
  if (seq < 0) return;
  const Chunk c = chunk_of(a.p, seq);
  const int rows = c.n * a.group;
  if (!alone && (rows <= 16 || c.n == 1)) return;  // few_rows'
  const int64_t r0l = (tile - tile_base(c.begin, a.group, kChunkTile, seq)) * kChunkTile;
  if (r0l < 0 || r0l >= rows) return;
  const int r0 = (int)r0l, rn = rows - r0 < kChunkTile ? rows - r0 : kChunkTile;
  const Sees sees = sees_of(a, c);
  const int t0 = r0 / a.group, t1 = (r0 + rn - 1) / a.group;
  const Span span = span_of(sees, t0, t1, parts.keys, parts.most);
  if (part >= span.parts) return;
  const int k0 = span.begin(part, parts.keys), k1 = span.end(part, parts.keys);

  const int w0 = wave * 32;
  const bool busy = w0 < rn, row_ok = w0 + i < rn;
  const int row = r0 + (row_ok ? w0 + i : 0);
  const int64_t at = sees.p0 + row / a.group;
  const int pos = as_int(at), low = as_int(sees.low(at));
  // keys between these are seen by every row of this wave
  const int last = r0 + (w0 + 31 < rn ? w0 + 31 : rn - 1);
  const int all_lo = as_int(sees.low(sees.p0 + last / a.group)), all_hi = as_int(sees.p0 + (r0 + w0) / a.group);
  const int any_lo = as_int(sees.low(sees.p0 + (r0 + w0) / a.group)), any_hi = as_int(sees.p0 + last / a.group);  // and by some row
  const int tile_lo = as_int(sees.low(sees.p0 + t1)), tile_hi = as_int(sees.p0 + t0);  // and by all of the workgroup's
  const int dim = a.p.dim;

  // the scale's sign goes to the queries: a largest score is a largest product
  const float flip = a.scale < 0.f ? -1.f : a.scale > 0.f ? 1.f : 0.f;
  const float scale2 = a.scale == 0.f ? 1.f : fabsf(a.scale) * kLog2e;
  vec q[L::KC][NP];
  float qs = 1.f;
  {
    const T* src = static_cast<const T*>(a.q.d) + (int64_t)(c.begin + row / a.group) * a.q.token_stride +
                   (int64_t)(kvh * a.group + row % a.group) * a.q.head_stride;
    int e = 0;
    if constexpr (NP == 2) {
      float top = 0.f;
      for (int d = h * L::KD; d < dim; d += 2 * L::KD)
        for (int j = 0; j < L::KD; ++j) top = row_ok ? fmaxf(top, fabsf((float)src[d + j])) : 0.f;
      top = fmaxf(top, __shfl_xor(top, 32));
      // The scale times the power stays a normal number: masked scores would be
      // -infinity times 0.  (Scores are below 2^-80 then, whatever the queries lose.)
      const int least = -126 - ilogbf(scale2);
      e = query_exponent(top);
      e = e < least ? least : e;
      qs = ldexpf(1.f, e);
    }
#pragma unroll
    for (int k = 0; k < L::KC; ++k)
#pragma unroll
      for (int j = 0; j < L::KD; ++j) {
        const int d = (k * 2 + h) * L::KD + j;
        float x = row_ok && d < dim ? (float)src[d] * flip : 0.f;
        if constexpr (NP == 2) x = ldexpf(x, -e);
        split<NP>(x, q[k], j);
      }
  }
  float sc = scale2 * qs;
  if constexpr (NP == 2) {
    // Nor does it pass fp32's range, where scores are 0, infinite or 2^70 apart:
    // the weights are the same, and the maximum gets back what was left out.
    float rest = 1.f;
    if (sc > 0x1p127f) {
      sc = 0x1p127f;
      rest = scale2 * 0x1p-127f * qs;
    }
    if (h == 0) max_times[w0 + i] = rest;  // (read by this wave alone)
  }

  const int piece = threadIdx.x % L::kPieces, srow = threadIdx.x / L::kPieces;
  const bool piece_ok = piece * L::KD < dim;
  // this thread's piece of a row
  const char* base = reinterpret_cast<const char*>(static_cast<const TC*>(a.p.kv) + (int64_t)kvh * a.p.head_stride) +
                     (piece_ok ? piece * 16 : 0);
  const uint32_t page_bytes = (uint32_t)a.p.page_stride * (uint32_t)sizeof(TC);
  const uint32_t token_bytes = (uint32_t)a.p.token_stride * (uint32_t)sizeof(TC);
  const int64_t to_value = a.p.value_offset * (int64_t)sizeof(TC);
  const uint32_t mask = (1u << a.p.page_shift) - 1;
  const int32_t* table = a.p.table + (int64_t)c.slot * a.p.table_stride;  // (no keys without a slot)

  // A lane's key of a tile: its entry of the table, as it is (what is done with
  // it waits for the load), and its page, -1 where there is none.
  auto entry_at = [&](int kb) -> int {
    const int key = kb + (lane & (KT - 1));
    return table[(key < k1 ? key : k1 - 1) >> a.p.page_shift];
  };
  auto page_of_entry = [&](int kb, int entry) -> int {
    return kb + (lane & (KT - 1)) < k1 && (uint32_t)entry < (uint32_t)a.p.pages ? entry : -1;
  };
  u4 stage[L::kStage];  // K of the next tile, then its V
  uint64_t row_of[L::kStage];  // from `base` on
  auto fetch_k = [&](int kb, int page) {
    // (a place that is no key reads page 0; it is not put)
    const uint64_t off = (uint64_t)(uint32_t)(page < 0 ? 0 : page) * page_bytes +
                         (uint64_t)(((uint32_t)kb + (lane & (KT - 1))) & mask) * token_bytes;
    const int lo = (int)(uint32_t)off, hi = (int)(off >> 32);
#pragma unroll
    for (int n = 0; n < L::kStage; ++n) {
      const int r = n * L::kRowsPerStep + srow;
      row_of[n] = (uint64_t)(uint32_t)__shfl(lo, r) | (uint64_t)(uint32_t)__shfl(hi, r) << 32;
      stage[n] = *reinterpret_cast<const u4*>(base + row_of[n]);
    }
  };
  auto fetch_v = [&]() {
#pragma unroll
    for (int n = 0; n < L::kStage; ++n) stage[n] = *reinterpret_cast<const u4*>(base + (row_of[n] + to_value));
  };
  // there: which keys of the tile there are
  auto ok_at = [&](int n, uint64_t there) { return piece_ok && ((there >> (n * L::kRowsPerStep + srow)) & 1); };
  auto put_k = [&](char* to, uint64_t there) {
    if (there != ~uint64_t{0} || dim < D) {
#pragma unroll
      for (int n = 0; n < L::kStage; ++n)
        if (!ok_at(n, there)) stage[n] = u4{0, 0, 0, 0};
    }
#pragma unroll
    for (int n = 0; n < L::kStage; ++n) {
      const int r = n * L::kRowsPerStep + srow;
      *reinterpret_cast<u4*>(to + (r * L::kPieces + L::k_piece(r, piece)) * 16) = stage[n];
    }
  };
  // Values that are not finite meet weights of 0 in the rows that do not see
  // their keys, which would be NaN there.  Where rows see different keys such a
  // value is put as 0, and noted: the rows that see its key turn to NaN after
  // the products.  (This wave's rows may see the whole tile all the same.)
  auto mixed = [&](int kb) { return kb < tile_lo || kb + KT - 1 > tile_hi; };
  auto put_v = [&](char* to, uint64_t there, int kb, int buf) {
    bool any = false;
    if (there != ~uint64_t{0} || dim < D) {
#pragma unroll
      for (int n = 0; n < L::kStage; ++n)
        if (!ok_at(n, there)) stage[n] = u4{0, 0, 0, 0};
    }
    if (mixed(kb)) {
#pragma unroll
      for (int n = 0; n < L::kStage; ++n) {
        TC e[L::KD];
        __builtin_memcpy(e, &stage[n], 16);
        uint32_t bits = 0;
#pragma unroll
        for (int j = 0; j < L::KD; ++j)
          if (!(fabsf((float)e[j]) < __builtin_inff())) {
            bits |= 1u << j;
            e[j] = 0.f;
          }
        __builtin_memcpy(&stage[n], e, 16);
        noted[buf][n * L::kRowsPerStep + srow][piece] = (uint8_t)bits;
        any |= bits != 0;
      }
    }
#pragma unroll
    for (int n = 0; n < L::kStage; ++n) {
      const int r = n * L::kRowsPerStep + srow;
      *reinterpret_cast<u4*>(to + (r * L::kPieces + L::v_piece(r, piece)) * 16) = stage[n];
    }
    const bool wave_any = __ballot(any) != 0;
    if (lane == 0) has_noted[buf][wave] = wave_any;
  };

  f16x o[L::kTiles];
#pragma unroll
  for (int t = 0; t < L::kTiles; ++t) o[t] = f16x{};
  float m = minus_inf(), l = 0.f, lr = 0.f;  // (lr: of the rounded weights)
  float back = __builtin_inff();             // kShift - m: what turns a score into its weight's exponent
  constexpr float kSlack = __is_same(TC, _Float16) ? 32768.f : 256.f;  // 2^8, kShift included

  // 32 keys from kb + sub * 32 on; whole: every row sees all of them
  auto step = [&](bool whole, int sub, const char* lk, const char* lv, int kb, uint64_t there) {
    const char* row_k = lk + (sub * 32 + i) * L::kPieces * 16;
    f16x s{};
    // Products go before another wave's exponentials (2048 tokens over 16384 keys:
    // 1039 -> 1010 us; two prompts of 4001, heads of 64: 166 -> 160 us; the first
    // product's alone: 952 and 166).
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int k = 0; k < L::KC; ++k) {
      const vec x = *reinterpret_cast<const vec*>(row_k + L::k_piece(i, k * 2 + h) * 16);
#pragma unroll
      for (int n = NP - 1; n >= 0; --n) s = mma32(x, q[k][n], s);
    }
    __builtin_amdgcn_s_setprio(0);
    if (!whole) {
      const int lo = low - kb - sub * 32, hi = pos - kb - sub * 32;  // of the 32 keys
      const int from = lo < 0 ? 0 : lo > 32 ? 32 : lo, to = hi < 0 ? 0 : hi > 31 ? 32 : hi + 1;
      // bit n: this row sees key n
      const uint32_t seen = (uint32_t)(there >> (sub * 32)) & (uint32_t)((uint64_t{1} << to) - 1) &
                            ~(uint32_t)((uint64_t{1} << from) - 1);
      const uint32_t mine = seen >> (4 * h);  // (shifted once: 16 bits by number, not 16 registers)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (!((mine >> (8 * (r >> 2) + (r & 3))) & 1)) s[r] = minus_inf();
    }
    // Weights from the maximum so far; when they add up to more than 2^8 of the
    // largest (or to NaN), the maximum is brought up to date first.
    float w[16], sum = 0.f;
    auto weigh = [&](float times, float from) {
      sum = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        w[r] = exp2_(__builtin_fmaf(s[r], times, from));
        sum += w[r];
      }
    };
    weigh(sc, back);
    if (__ballot(!(sum < kSlack))) {
      float top = s[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
      top *= sc;
      top = fmaxf(top, __shfl_xor(top, 32));
      const float to = ceilf(fmaxf(top, m)), from = to == minus_inf() ? 0.f : to;
      const float shrink = exp2_(m - from);
      m = to;
      back = L::kShift - from;
      l *= shrink;
      lr *= shrink;
#pragma unroll
      for (int t = 0; t < L::kTiles; ++t) o[t] *= shrink;
      // So large a product is off by whole numbers when rounded, as `top` was and
      // the fused one is not: all are rounded, so that none passes the largest.
      float times = sc;
      if (__ballot(fabsf(from) > 1048576.f)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] *= sc;
        times = 1.f;
      }
      weigh(times, back);
      if (to == minus_inf()) back = __builtin_inff();  // no key yet: the next one sets it
    }
    l += sum;
    __builtin_amdgcn_s_setprio(1);
    if constexpr (!L::kWide) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {  // 16 keys
        vec p[NP];
#pragma unroll
        for (int j = 0; j < 8; ++j) split<NP>(w[b * 8 + j], p, j);
        if constexpr (rounds_weights<T, TC>()) lr = plus_all(p[0], lr);
#pragma unroll
        for (int t = 0; t < L::kTiles; ++t) {
          // a lane reads 4 elements of one of 4 keys, and gets 4 keys of one element
          const int r = 4 * h + ((lane >> 2) & 3), e = t * 32 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
          const char* at = lv + (sub * 32 + b * 16) * L::kPieces * 16 + (e & 7) * 2;
          const s4x lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lds_s4x)(at + (r * L::kPieces + L::v_piece(r, e >> 3)) * 16));
          const s4x hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lds_s4x)(at + ((r + 8) * L::kPieces + L::v_piece(r + 8, e >> 3)) * 16));
          const vec x = __builtin_bit_cast(vec, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
          for (int n = NP - 1; n >= 0; --n) o[t] = mma32(x, p[n], o[t]);
        }
      }
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r) {  // 2 keys, one to each half of the wave
        const char* at = lv + (sub * 32 + 8 * (r >> 2) + 4 * h + (r & 3)) * L::kPieces * 16;
#pragma unroll
        for (int t = 0; t < L::kTiles; t += L::kRun) {
          float x[L::kRun];
          __builtin_memcpy(x, __builtin_assume_aligned(at + L::element(t, i) * 4, 4 * L::kRun), 4 * L::kRun);
#pragma unroll
          for (int z = 0; z < L::kRun; ++z)
            o[t + z] = __builtin_amdgcn_mfma_f32_32x32x2f32(x[z], w[r], o[t + z], 0, 0, 0);
        }
      }
    }
    __builtin_amdgcn_s_setprio(0);
  };

  uint64_t there = 0, there1 = 0;  // (KT 32: each half is the tile)
  int entry1 = 0;                  // of the next tile
  if (k0 < k1) {
    const int page = page_of_entry(k0, entry_at(k0));
    entry1 = entry_at(k0 + KT);
    there = __ballot(page >= 0);
    fetch_k(k0, page);
    put_k(chunk_lds, there);
    fetch_v();
    put_v(chunk_lds + L::kBytes, there, k0, 0);
  }
  int buf = 0;
  for (int kb = k0; kb < k1; kb += KT, buf ^= 1) {
    const bool more = kb + KT < k1;
    const char* lk = chunk_lds + buf * 2 * L::kBytes;
    const char* lv = lk + L::kBytes;
    char* next = chunk_lds + (buf ^ 1) * 2 * L::kBytes;
    if (more) {
      const int page = page_of_entry(kb + KT, entry1);
      there1 = __ballot(page >= 0);
      entry1 = entry_at(kb + 2 * KT);
      fetch_k(kb + KT, page);
    }
    __syncthreads();
    const bool used = busy && kb <= any_hi && kb + KT > any_lo;
    const bool whole = kb >= all_lo && kb + KT - 1 <= all_hi && there == ~uint64_t{0};
#pragma unroll
    for (int sub = 0; sub < NS; ++sub)
      if (used) step(whole, sub, lk, lv, kb, there);
    // (behind the steps, not between them: 945 -> 932 us for 2048 tokens over
    // 16384 keys)
    if (more) {
      put_k(next, there1);
      fetch_v();
      put_v(next + L::kBytes, there1, kb + KT, buf ^ 1);
    }
    if (used && mixed(kb) && (has_noted[buf][0] | has_noted[buf][1] | has_noted[buf][2] | has_noted[buf][3])) {
#pragma unroll 1
      for (int n = 0; n < KT; ++n) {
        const int key = kb + n;
        const bool sees_it = ((there >> n) & 1) && key >= low && key <= pos;
        const uint8_t* note = &noted[buf][n][0];
#pragma unroll
        for (int t = 0; t < L::kTiles; ++t)
#pragma unroll
          for (int y = 0; y < 16; ++y) {
            const int d = L::element(t, 8 * (y >> 2) + 4 * here(h) + (y & 3));
            if (sees_it && ((note[d / L::KD] >> (d % L::KD)) & 1)) o[t][y] = __builtin_nanf("");
          }
      }
    }
    there = there1;
  }

  if (!row_ok) return;
  l += __shfl_xor(l, 32);
  if constexpr (rounds_weights<T, TC>())
    lr += __shfl_xor(lr, 32);
  else
    lr = l;
  if constexpr (NP == 2) m *= max_times[w0 + i];
  const float from = m == minus_inf() ? 0.f : m;
  const int token = c.begin + row / a.group, head = kvh * a.group + row % a.group;
  if (span.parts > 1) {
    const int64_t at = part * parts.rows + (int64_t)token * a.heads + head;
#pragma unroll
    for (int t = 0; t < L::kTiles; t += L::kRun)
#pragma unroll
      for (int y = 0; y < 16; y += L::kRun == 1 ? 4 : 1)
        put_run<L>(o, t, y, h, 1.f, [&](int d, const float* x) {
          __builtin_memcpy(__builtin_assume_aligned(parts.o + at * D + d, 4 * L::kStore), x, 4 * L::kStore);
        });
    if (h == 0) parts.ml[at] = f4{m, l, lr, 0.f};
    return;
  }
  T* out = static_cast<T*>(a.out.d) + (int64_t)token * a.out.token_stride + (int64_t)head * a.out.head_stride;
  const float f = lr == 0.f ? 0.f : 1.f / lr;
  const bool wide_out = ((reinterpret_cast<uintptr_t>(a.out.d) / sizeof(T) | (uint64_t)a.out.token_stride |
                          (uint64_t)a.out.head_stride) & (L::kStore - 1)) == 0;
#pragma unroll
  for (int t = 0; t < L::kTiles; t += L::kRun)
#pragma unroll
    for (int y = 0; y < 16; y += L::kRun == 1 ? 4 : 1)
      put_run<L>(o, t, y, h, f, [&](int d, const float* x) {
        if (d >= dim) return;
        typedef T run __attribute__((ext_vector_type(L::kStore)));
        run r;
#pragma unroll
        for (int z = 0; z < L::kStore; ++z) r[z] = (T)x[z];
        if (wide_out) {
          __builtin_memcpy(__builtin_assume_aligned(out + d, sizeof r), &r, sizeof r);
        } else {
#pragma unroll
          for (int z = 0; z < L::kStore; ++z) out[d + z] = r[z];
        }
      });
  if (a.lse && h == 0)
    a.lse[(int64_t)token * a.heads + head] =
        l == 0.f ? minus_inf() : (from + (__builtin_amdgcn_logf(l) - L::kShift)) * kLn2;
}

// alone: sequences of few rows are its too
template <typename T, typename TC, int D>
__global__ __launch_bounds__(kChunkThreads, (chunk_waves<T, TC, D>())) void chunk_kernel(AttendArgs a, Parts parts,
                                                                                        bool alone) {
  chunk_rows<T, TC, D>(a, parts, alone, blockIdx.x, gridDim.x, blockIdx.z);
}

// Chunks, and the sequences of few rows behind them in the grid: those fill the
// GPU while the chunks' last workgroups end, and read while others multiply.
template <typename T, typename TC, int D, bool kPad>
__global__ __launch_bounds__(kChunkThreads, (chunk_waves<T, TC, D>())) void both_kernel(AttendArgs a, Parts chunk,
                                                                                       Parts few, int few_tiles,
                                                                                       int chunk_groups, int few_groups) {
  static_assert(kChunkThreads == kFewThreads, "one workgroup for both");
  const int b = blockIdx.x, n = chunk_groups * chunk.most;
  if (b < n)
    chunk_rows<T, TC, D>(a, chunk, false, b % chunk_groups, chunk_groups, b / chunk_groups);
  else
    few_rows<T, TC, D, kPad>(a, few, few_tiles, true, (b - n) % few_groups, (b - n) / few_groups);
}

hipError_t allow_lds(const void* f, size_t lds) {
  return lds > 60000 ? hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) : hipSuccess;
}

template <typename T, typename TC, int D, bool kPad>
hipError_t both_of(const AttendArgs& a, const Parts& parts, int64_t tiles, const Parts& few, int few_tiles,
                   hipStream_t s) {
  constexpr size_t chunk_lds = 4 * Tile<T, TC, D>::kBytes, lds = chunk_lds > few_lds_bytes(D) ? chunk_lds : few_lds_bytes(D);
  const hipError_t e = allow_lds(reinterpret_cast<const void*>(both_kernel<T, TC, D, kPad>), lds);
  if (e != hipSuccess) return e;
  const int chunk_groups = (int)(tiles * a.p.kv_heads), few_groups = a.p.seqs * few_tiles * a.p.kv_heads;
  const int64_t all = (int64_t)chunk_groups * parts.most + (int64_t)few_groups * few.most;
  both_kernel<T, TC, D, kPad><<<(unsigned)all, kChunkThreads, lds, s>>>(a, parts, few, few_tiles, chunk_groups, few_groups);
  return hipGetLastError();
}

template <typename T, typename TC, int D>
hipError_t chunk_of_width(const AttendArgs& a, const Parts& parts, int64_t tiles, const Parts* few, int few_tiles,
                          hipStream_t s) {
  if constexpr (together<TC, D>())
    if (few)
      return a.p.dim == D ? both_of<T, TC, D, false>(a, parts, tiles, *few, few_tiles, s)
                          : both_of<T, TC, D, true>(a, parts, tiles, *few, few_tiles, s);
  constexpr size_t lds = 4 * Tile<T, TC, D>::kBytes;
  const hipError_t e = allow_lds(reinterpret_cast<const void*>(chunk_kernel<T, TC, D>), lds);
  if (e != hipSuccess) return e;
  chunk_kernel<T, TC, D><<<dim3((unsigned)(tiles * a.p.kv_heads), 1, parts.most), kChunkThreads, lds, s>>>(a, parts, !few);
  return hipGetLastError();
}

template <typename T, typename TC>
hipError_t chunk_of_types(const AttendArgs& a, const Parts& parts, int64_t tiles, const Parts* few, int few_tiles,
                          hipStream_t s) {
  if (a.p.dim <= 64) return chunk_of_width<T, TC, 64>(a, parts, tiles, few, few_tiles, s);
  if (a.p.dim <= 128) return chunk_of_width<T, TC, 128>(a, parts, tiles, few, few_tiles, s);
  return chunk_of_width<T, TC, 256>(a, parts, tiles, few, few_tiles, s);
}

}  // namespace

hipError_t launch_chunk(const AttendArgs& a, int type, int cache_type, const Parts& parts, int64_t tiles,
                        const Parts* few, int few_tiles, hipStream_t s) {
  if (type == kF32) {
    if (cache_type == kF32) return chunk_of_types<float, float>(a, parts, tiles, few, few_tiles, s);
    if (cache_type == kF16) return chunk_of_types<float, _Float16>(a, parts, tiles, few, few_tiles, s);
    return chunk_of_types<float, __bf16>(a, parts, tiles, few, few_tiles, s);
  }
  if (type == kF16) return chunk_of_types<_Float16, _Float16>(a, parts, tiles, few, few_tiles, s);
  return chunk_of_types<__bf16, __bf16>(a, parts, tiles, few, few_tiles, s);
}

}  // namespace nls
