// nls_attend_quant_chunk.hip -- attention of chunks over pages of blocks:
// sequences of more than 16 rows (token, head of the group) per kv head.
//
// As for chunks over wide caches (nls_attend_chunk.hip), a wave takes 32 rows of
// one (sequence, kv head), S^T = K Q^T and O^T = V^T P^T are 32 x 32 products,
// tiles of keys are in LDS two at a time, and the maximum follows the scores only
// when it is passed by 2^8.  What differs:
//
//   K   LDS holds the codes as fp16, which is exact.  Two products over a block
//       are its depth; their sums are multiplied by the block's factor in fp32
//       as they are added up, 16 per lane and block.
//   V   LDS holds d c: for bf16 queries rounded to fp16, as their weights are
//       (2^-11 at most, an eighth of the output's own half step), for fp32 and
//       fp16 queries as two fp16 parts, which are exact (both c and d are whole
//       multiples of fp16's least step), their weights two parts as well, and
//       three products: hi hi, hi lo, lo hi.  (fp16 queries with one of each: 924 us
//       for 1246, and the error half as large again as the output's rounding.)
//
// What bounds it: for fp32 queries the matrix cores, with the turning of codes into
// operands on the vector units between their runs; for 16-bit ones, of half as many
// products or fewer, that turning and the exponentials as much.  2048 tokens over
// 16384 keys, 32 heads on 8 of 128, Q4_0: fp32 1320 us, 390 TFLOP/s of the mathematics
// in two and a half times as many products (two and three for one and one); fp16
// (one and three) 1125; bf16 (one and one) 805, 640 TFLOP/s (a bf16 cache, which has
// nothing to turn: 572); 4001 tokens of 32 heads of 64, Q8_0, bf16: 156 us.  Heads
// beyond 128 have one wave a SIMD and tiles of 32 keys: 512 tokens over 8192, bf16,
// heads of 128 148 us, of 160 345.
//
// Values below fp16's normal numbers (2^-14) leave the products' sums fewer bits: they
// are taken to within some 2^-38 (measured: 2^-41), whatever their size.
//
// Factors outside of the second product as well would be 16 products, splits and
// conversions per lane, block and part, more than the third matrix product costs.
#include "nls_attend_quant.h"

namespace nls {
namespace {

__device__ __forceinline__ f16x mma32(h8 a, h8 b, f16x c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

typedef short s4x __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4x* lds_s4x;

template <typename T, int kBits, int GT>
struct QTile {
  static constexpr int D = 32 * GT;
  static constexpr int NP = quant_parts<T>(), NW = weight_parts<T>();
  static constexpr int kRows = quant_tile<T>(GT), kWaves = kRows / 32, kThreads = 64 * kWaves;
  static constexpr int KT = GT == 8 ? 32 : 64;                  // keys per tile
  static constexpr int kRuns = KT / 16;                 // of keys within a page
  static constexpr int kPieces = D / 8;                 // 16-byte pieces of a row
  static constexpr int kBytes = KT * D * 2;             // of one of the three below
  static constexpr int kFactors = GT * KT * 2;
  static constexpr int kStage = kBytes * (1 + NW) + kFactors;  // K, V (and its rest), K's factors
  static constexpr int kUnits = KT * 4 * GT / kThreads;        // key units of a thread
  static constexpr int kWide = GT < 4 ? GT : 4;                // blocks of a plane
  static constexpr int kLanes = KT * 16 * (GT / kWide) / kThreads;  // value pieces of a thread, side by side
  static constexpr int kKeyWords = kUnits * kBits / 4, kValueBytes = kLanes * kWide * kBits / 4;
  static constexpr int kValueWords = (kValueBytes + 3) / 4;
  static_assert(kUnits <= GT && kUnits >= 1 && kLanes >= 2, "a thread's units are of one quarter, its pieces of one plane");
  static __device__ __forceinline__ int k_piece(int r, int c) {
    return kPieces >= 16 ? c ^ (r & 15) : c ^ ((r >> 1) & 7);
  }
  static __device__ __forceinline__ int v_piece(int r, int c) {
    return kPieces >= 16 ? c ^ ((r & 3) << 2) : c ^ (((r >> 1) & 1) << 2);
  }
};

// Heads of NG blocks, in tiles of GT.  Where NG is less a thread's values come in
// pieces of the planes that there are, and become a whole plane's order on their way
// to LDS (512 tokens over 8192, heads of 96 and 192, bf16 over Q4_0: 136 and 383 us;
// with a load for each lane and block, and products over the blocks that are not
// there, 185 and 619).
template <typename T, int kBits, int GT, int NG>
__device__ __forceinline__ void chunk_quant_rows(const AttendArgs& a, const Parts& parts, bool alone, int group_at,
                                                 int groups_n, int part) {
  using L = QTile<T, kBits, GT>;
  constexpr bool kPad = NG < GT;
  constexpr int NP = L::NP, NW = L::NW, KT = L::KT, NS = KT / 32, D = L::D;
  constexpr bool kScaled = !__is_same(T, _Float16);  // rows are divided by a power of two
  constexpr float kShift = chunk_shift<_Float16>();
  extern __shared__ __align__(16) char chunk_lds[];  // [2][K, V, V's rest, K's factors]
  __shared__ uint8_t noted[2][KT];                   // bit x: block x of a value was not finite
  __shared__ int has_noted[2][L::kWaves];
  __shared__ float max_times[kScaled ? L::kRows : 1];

  const int kvh = group_at % a.p.kv_heads, tile = (groups_n - 1 - group_at) / a.p.kv_heads;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 31, h = lane >> 5;

  // the sequence whose tiles begin at or before this one
  int seq = -1;
  for (int s0 = 0; s0 < a.p.seqs; s0 += 64) {
    const int s = s0 + lane;
    const int n = __popcll(__ballot(s < a.p.seqs && tile_base(a.p.starts[s < a.p.seqs ? s : 0], a.group, L::kRows, s) <= tile));
    seq += n;
    if (n < 64) break;
  }
  if (seq < 0) return;
  const Chunk c = chunk_of(a.p, seq);
  const int rows = c.n * a.group;
  if (!alone && (rows <= 16 || c.n == 1)) return;  // few_quant_rows'
  const int64_t r0l = (tile - tile_base(c.begin, a.group, L::kRows, seq)) * L::kRows;
  if (r0l < 0 || r0l >= rows) return;
  const int r0 = (int)r0l, rn = rows - r0 < L::kRows ? rows - r0 : L::kRows;
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
  constexpr int dim = 32 * NG, row_bytes = 4 * NG * kBits;

  // the scale's sign goes to the queries: a largest score is a largest product
  const float flip = a.scale < 0.f ? -1.f : a.scale > 0.f ? 1.f : 0.f;
  const float scale2 = a.scale == 0.f ? 1.f : fabsf(a.scale) * kLog2e;
  h8 q[2 * NG][NP];
  float qs = 1.f;
  {
    const T* src = static_cast<const T*>(a.q.d) + (int64_t)(c.begin + row / a.group) * a.q.token_stride +
                   (int64_t)(kvh * a.group + row % a.group) * a.q.head_stride;
    int e = 0;
    if constexpr (kScaled) {
      float top = 0.f;
      for (int d = h * 8; d < dim; d += 16)
        for (int j = 0; j < 8; ++j) top = row_ok ? fmaxf(top, fabsf((float)src[d + j])) : 0.f;
      top = fmaxf(top, __shfl_xor(top, 32));
      // (the scale times the power stays a normal number: masked scores would be
      // -infinity times 0)
      const int least = -126 - ilogbf(scale2);
      e = query_exponent(top);
      e = e < least ? least : e;
      qs = ldexpf(1.f, e);
    }
#pragma unroll
    for (int k = 0; k < 2 * NG; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int d = (k * 2 + h) * 8 + j;
        float x = row_ok && d < dim ? (float)src[d] * flip : 0.f;
        if constexpr (kScaled) x = ldexpf(x, -e);
        split<NP>(x, q[k], j);
      }
  }
  float sc = scale2 * qs;
  if constexpr (kScaled) {
    // Nor does it pass fp32's range: the maximum gets back what was left out.
    float rest = 1.f;
    if (sc > 0x1p127f) {
      sc = 0x1p127f;
      rest = scale2 * 0x1p-127f * qs;
    }
    if (h == 0) max_times[w0 + i] = rest;  // (read by this wave alone)
  }

  // This thread's part of a tile.  A wave's rows are of one run of 16 keys.
  const int size = 1 << a.p.page_shift;
  const QuantShape shape = quant_shape(kBits == 8 ? kQ8_0 : kQ4_0, dim, size);
  const int unit = threadIdx.x * L::kUnits, k_row = unit / (4 * GT), k_g = unit % (4 * GT) / GT, k_x = unit % GT;
  constexpr int kPlanes = GT / L::kWide;
  const int piece = threadIdx.x * L::kLanes, v_row = piece / (16 * kPlanes), v_plane = piece / 16 % kPlanes, v_i = piece % 16;
  const int run = __builtin_amdgcn_readfirstlane(k_row / 16);  // (v_row's too)
  const int f_x = threadIdx.x / (KT / 8), f_key = threadIdx.x % (KT / 8) * 8;  // K's factors: the first GT KT / 8 threads
  const bool f_mine = f_x < NG;
  const char* base = static_cast<const char*>(a.p.kv) + quant_base(shape, kvh, 0);
  const int32_t* table = a.p.table + (int64_t)c.slot * a.p.table_stride;  // (no keys without a slot)
  // The table's entries of a tile: its runs', and once more this wave's run's and
  // that of this lane's factors.
  struct Entries {
    int at[L::kRuns], run, factors;
  };
  auto entry_of = [&](int key) { return table[(key < k1 ? key : k1 - 1) >> a.p.page_shift]; };
  auto entries_at = [&](int kb) {
    Entries e;
#pragma unroll
    for (int r = 0; r < L::kRuns; ++r) e.at[r] = entry_of(kb + r * 16);
    e.run = entry_of(kb + run * 16);
    e.factors = f_mine ? entry_of(kb + f_key) : 0;
    return e;
  };
  // (from kb on; -1: none, and what is read there is page 0)
  auto page_of_entry = [&](int key, int page) { return key < k1 && (uint32_t)page < (uint32_t)a.p.pages ? page : -1; };
  auto pages_at = [&](int kb, const Entries& e) {
    Entries p;
#pragma unroll
    for (int r = 0; r < L::kRuns; ++r) p.at[r] = page_of_entry(kb + r * 16, __builtin_amdgcn_readfirstlane(e.at[r]));
    p.run = page_of_entry(kb + run * 16, __builtin_amdgcn_readfirstlane(e.run));
    p.factors = page_of_entry(kb + (f_key & ~15), e.factors);
    return p;
  };
  // bit n: key n of the tile is there
  auto there_at = [&](int kb, const Entries& p) {
    uint64_t t = 0;
#pragma unroll
    for (int r = 0; r < L::kRuns; ++r) t |= p.at[r] >= 0 ? uint64_t{0xffff} << (16 * r) : 0;
    if (kb + KT > k1) t &= (uint64_t{1} << (k1 - kb)) - 1;  // (k1 - kb is 1 .. 63 then)
    return t;
  };
  constexpr uint64_t kAll = KT == 64 ? ~uint64_t{0} : 0xffffffffu;

  uint32_t kc[L::kKeyWords], vc[L::kValueWords];
  u4 kf;             // factors of 8 keys
  _Float16 vd[L::kWide];
  // (kPad) the pieces of a row's planes, which vc is made of when they are there
  uint32_t v4[L::kLanes * kBits / 4], v2[L::kLanes * kBits / 8], v1[(L::kLanes * kBits + 15) / 16];
  auto join_planes = [&]() {
    constexpr int kBytes = kBits / 4;  // of a lane and block
    auto bytes_of = [](const uint32_t* from, int n) { return from[n * kBytes / 4] >> (8 * (n * kBytes % 4)) & ((1u << 8 * kBytes) - 1); };
#pragma unroll
    for (int w = 0; w < L::kValueWords; ++w) {
      uint32_t r = 0;
#pragma unroll
      for (int n = 4 / kBytes * w; n < 4 / kBytes * (w + 1); ++n) {
        const int z = n / L::kWide, b = n % L::kWide;
        if ((NG & 2) && b < 2) r |= bytes_of(v2, z * 2 + b) << (8 * (n * kBytes % 4));
        if ((NG & 1) && b == (NG & 2)) r |= bytes_of(v1, z) << (8 * (n * kBytes % 4));
      }
      vc[w] = NG > 4 && v_plane == 0 ? v4[w] : r;
    }
  };
  auto home_of = [&](int page) { return base + (int64_t)(page < 0 ? 0 : page) * a.p.page_stride; };
  auto fetch = [&](int kb, const Entries& p) {
    const char* home = home_of(p.run);
    const int place = ((uint32_t)kb + run * 16) & (size - 1);  // of the run
    const char* keys = home + (place + (k_row & 15)) * row_bytes + (k_g * NG + (kPad ? 0 : k_x)) * kBits;
    const char* values = home + shape.half + (place + (v_row & 15)) * row_bytes;
    const char* factors = home + shape.half + shape.codes + (place + (v_row & 15)) * 2;
    if constexpr (!kPad) {
      __builtin_memcpy(kc, __builtin_assume_aligned(keys, L::kUnits * kBits < 16 ? L::kUnits * kBits : 16), L::kUnits * kBits);
      const char* from = values + (v_plane * 16 * L::kWide + v_i * L::kWide) * (kBits / 4);
      __builtin_memcpy(vc, __builtin_assume_aligned(from, L::kValueBytes < 16 ? L::kValueBytes : 16), L::kValueBytes);
#pragma unroll
      for (int b = 0; b < L::kWide; ++b)
        vd[b] = *reinterpret_cast<const _Float16*>(factors + (v_plane * L::kWide + b) * size * 2);
    } else {
      // (in the place of blocks that are not there the last one, which nothing reads)
#pragma unroll
      for (int u = 0; u < L::kUnits; ++u)
        __builtin_memcpy(kc + u * kBits / 4, __builtin_assume_aligned(keys + min(k_x + u, NG - 1) * kBits, kBits), kBits);
      // pieces of the planes of four blocks, of two, of one
      constexpr int kFours = NG / 4;
      if constexpr (kFours != 0)
        __builtin_memcpy(v4, __builtin_assume_aligned(values + v_i * kBits, L::kLanes * kBits < 16 ? L::kLanes * kBits : 16), L::kLanes * kBits);
      if constexpr ((NG & 2) != 0)
        __builtin_memcpy(v2, __builtin_assume_aligned(values + kFours * 16 * kBits + v_i * kBits / 2, L::kLanes * kBits / 2),
                         L::kLanes * kBits / 2);
      if constexpr ((NG & 1) != 0)
        __builtin_memcpy(v1, __builtin_assume_aligned(values + (NG - 1) * 4 * kBits + v_i * kBits / 4, L::kLanes * kBits / 4),
                         L::kLanes * kBits / 4);
#pragma unroll
      for (int b = 0; b < L::kWide; ++b)
        vd[b] = *reinterpret_cast<const _Float16*>(factors + min(v_plane * L::kWide + b, NG - 1) * size * 2);
    }
    if (f_mine) {
      const char* there = home_of(p.factors);
      kf = *reinterpret_cast<const u4*>(there + shape.codes + (f_x * size + (((uint32_t)kb + f_key) & (size - 1))) * 2);
    }
  };
  // Values that are not finite meet weights of 0 in the rows that do not see
  // their keys, which would be NaN there.  Where rows see different keys such a
  // block is put as 0, and noted: the rows that see its key turn to NaN after
  // the products.  (This wave's rows may see the whole tile all the same.)
  auto mixed = [&](int kb) { return kb < tile_lo || kb + KT - 1 > tile_hi; };
  auto put = [&](char* to, uint64_t there, int kb, int buf) {
#pragma unroll
    for (int u = 0; u < L::kUnits; ++u) {
      const u4 codes = __builtin_bit_cast(u4, key_codes<kBits>(kc + u * kBits / 4));
      *reinterpret_cast<u4*>(to + (k_row * L::kPieces + L::k_piece(k_row, (k_x + u) * 4 + k_g)) * 16) = codes;
    }
    if (f_x < GT) {
      u4 f = f_mine ? kf : u4{0, 0, 0, 0};
      if (there != kAll) {
        const uint32_t ok = (uint32_t)(there >> f_key);
#pragma unroll
        for (int n = 0; n < 4; ++n)
          f[n] &= ((ok >> (2 * n)) & 1 ? 0xffffu : 0u) | ((ok >> (2 * n + 1)) & 1 ? 0xffff0000u : 0u);
      }
      *reinterpret_cast<u4*>(to + L::kBytes * (1 + NW) + (f_x * KT + f_key) * 2) = f;
    }
    if (there != kAll && !((there >> v_row) & 1)) {
#pragma unroll
      for (int b = 0; b < L::kWide; ++b) vd[b] = (_Float16)0.f;
    }
    bool any = false;
    if (mixed(kb)) {
      uint32_t bits = 0;
#pragma unroll
      for (int b = 0; b < L::kWide; ++b)
        if (!(__builtin_fabsf((float)vd[b]) < __builtin_inff())) {
          bits |= 1u << (v_plane * L::kWide + b);
          vd[b] = (_Float16)0.f;
        }
      // (a row's threads are neighbours within a wave)
#pragma unroll
      for (int d = 1; d < 16 * kPlanes / L::kLanes; d <<= 1) bits |= __shfl_xor(bits, d);
      if (v_i == 0 && v_plane == 0) noted[buf][v_row] = (uint8_t)bits;
      any = bits != 0;
    }
    if constexpr (kPad) join_planes();
    // pairs of lanes z, z + 1: elements 32 x + 16 half + v_i + z
    char* hi = to + L::kBytes;
#pragma unroll
    for (int b = 0; b < L::kWide; ++b)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t w[L::kLanes / 2], rest[L::kLanes / 2];
#pragma unroll
        for (int z = 0; z < L::kLanes; z += 2) {
          const int n = kBits == 8 ? (z * L::kWide + b) * 2 + half : z * L::kWide + b;
          const int m = n + L::kWide * kBits / 4;  // the next lane's byte
          const uint32_t pair = __builtin_amdgcn_perm(vc[m / 4], vc[n / 4], 0x0c000c00u | (4 + m % 4) << 16 | n % 4);
          const uint32_t codes = kBits == 8 ? less(pair | 0x64006400u, 1152.f) : half ? high_nibbles(pair) : low_nibbles(pair);
          const h2 d{vd[b], vd[b]}, v = halves(codes) * d;
          w[z / 2] = __builtin_bit_cast(uint32_t, v);
          if constexpr (NW == 2)
            rest[z / 2] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(halves(codes), d, -v));
        }
        const int e = (v_plane * L::kWide + b) * 32 + half * 16 + v_i;
        char* at = hi + (v_row * L::kPieces + L::v_piece(v_row, e >> 3)) * 16 + (e & 7) * 2;
        __builtin_memcpy(__builtin_assume_aligned(at, 2 * L::kLanes), w, 2 * L::kLanes);
        if constexpr (NW == 2)
          __builtin_memcpy(__builtin_assume_aligned(at + L::kBytes, 2 * L::kLanes), rest, 2 * L::kLanes);
      }
    const bool wave_any = __ballot(any) != 0;
    if (lane == 0) has_noted[buf][wave] = wave_any;
  };

  f16x o[NG];
#pragma unroll
  for (int t = 0; t < NG; ++t) o[t] = f16x{};
  float m = minus_inf(), l = 0.f, lr = 0.f;  // (lr: of the rounded weights)
  float back = __builtin_inff();             // kShift - m: what turns a score into its weight's exponent
  constexpr float kSlack = 32768.f;          // 2^8, kShift included

  // 32 keys from kb + sub * 32 on; whole: every row sees all of them
  auto step = [&](bool whole, int sub, const char* lk, int kb, uint64_t there) {
    const char* row_k = lk + (sub * 32 + i) * L::kPieces * 16;
    const char* factors = lk + L::kBytes * (1 + NW) + (sub * 32 + 4 * h) * 2;
    const char* lv = lk + L::kBytes;
    f16x s;
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int x = 0; x < NG; ++x) {
      f16x acc{};
#pragma unroll
      for (int k = 2 * x; k < 2 * x + 2; ++k) {
        const h8 codes = *reinterpret_cast<const h8*>(row_k + L::k_piece(i, k * 2 + h) * 16);
#pragma unroll
        for (int n = NP - 1; n >= 0; --n) acc = mma32(codes, q[k][n], acc);
      }
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const u2 f = *reinterpret_cast<const u2*>(factors + (x * KT + 8 * b) * 2);
        const h2 f0 = halves(f[0]), f1 = halves(f[1]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float d = (float)(r < 2 ? f0[r & 1] : f1[r & 1]);
          s[4 * b + r] = x == 0 ? d * acc[4 * b + r] : __builtin_fmaf(d, acc[4 * b + r], s[4 * b + r]);
        }
      }
    }
    __builtin_amdgcn_s_setprio(0);
    if (!whole) {
      const int lo = low - kb - sub * 32, hi = pos - kb - sub * 32;  // of the 32 keys
      const int from = lo < 0 ? 0 : lo > 32 ? 32 : lo, to = hi < 0 ? 0 : hi > 31 ? 32 : hi + 1;
      // bit n: this row sees key n
      const uint32_t seen = (uint32_t)(there >> (sub * 32)) & (uint32_t)((uint64_t{1} << to) - 1) &
                            ~(uint32_t)((uint64_t{1} << from) - 1);
      const uint32_t mine = seen >> (4 * h);
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
      back = kShift - from;
      l *= shrink;
      lr *= shrink;
#pragma unroll
      for (int t = 0; t < NG; ++t) o[t] *= shrink;
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
#pragma unroll
    for (int b = 0; b < 2; ++b) {  // 16 keys
      h8 p[NW];
#pragma unroll
      for (int j = 0; j < 8; ++j) split<NW>(w[b * 8 + j], p, j);
      if constexpr (NW == 1) lr = plus_all(p[0], lr);
#pragma unroll
      for (int t = 0; t < NG; ++t) {
        // a lane reads 4 elements of one of 4 keys, and gets 4 keys of one element
        const int r = 4 * h + ((lane >> 2) & 3), e = t * 32 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
        const char* at = lv + (sub * 32 + b * 16) * L::kPieces * 16 + (e & 7) * 2;
        const int at_lo = (r * L::kPieces + L::v_piece(r, e >> 3)) * 16;
        const int at_hi = ((r + 8) * L::kPieces + L::v_piece(r + 8, e >> 3)) * 16;
        auto operand = [&](const char* from) {
          const s4x lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4x)(from + at_lo));
          const s4x hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4x)(from + at_hi));
          return __builtin_bit_cast(h8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        };
        const h8 v = operand(at);
        if constexpr (NW == 2) {
          o[t] = mma32(operand(at + L::kBytes), p[0], o[t]);
          o[t] = mma32(v, p[1], o[t]);
        }
        o[t] = mma32(v, p[0], o[t]);
      }
    }
    __builtin_amdgcn_s_setprio(0);
  };

  uint64_t there = 0, there1 = 0;
  Entries entry1;  // of the next tile
  if (k0 < k1) {
    const Entries p = pages_at(k0, entries_at(k0));
    entry1 = entries_at(k0 + KT);
    there = there_at(k0, p);
    fetch(k0, p);
    put(chunk_lds, there, k0, 0);
  }
  int buf = 0;
  for (int kb = k0; kb < k1; kb += KT, buf ^= 1) {
    const bool more = kb + KT < k1;
    const char* lk = chunk_lds + buf * L::kStage;
    if (more) {
      const Entries p = pages_at(kb + KT, entry1);
      there1 = there_at(kb + KT, p);
      entry1 = entries_at(kb + 2 * KT);
      fetch(kb + KT, p);
    }
    __syncthreads();
    const bool used = busy && kb <= any_hi && kb + KT > any_lo;
    const bool whole = kb >= all_lo && kb + KT - 1 <= all_hi && there == kAll;
#pragma unroll
    for (int sub = 0; sub < NS; ++sub)
      if (used) step(whole, sub, lk, kb, there);
    if (more) put(chunk_lds + (buf ^ 1) * L::kStage, there1, kb + KT, buf ^ 1);
    if (used && mixed(kb) && __ballot(lane < L::kWaves && has_noted[buf][lane % L::kWaves])) {
#pragma unroll 1
      for (int n = 0; n < KT; ++n) {
        const int key = kb + n;
        const bool sees_it = ((there >> n) & 1) && key >= low && key <= pos;
        const uint32_t note = noted[buf][n];
#pragma unroll
        for (int t = 0; t < NG; ++t)
          if (sees_it && ((note >> t) & 1))
#pragma unroll
            for (int y = 0; y < 16; ++y) o[t][y] = __builtin_nanf("");
      }
    }
    there = there1;
  }

  if (!row_ok) return;
  l += __shfl_xor(l, 32);
  if constexpr (NW == 1)
    lr += __shfl_xor(lr, 32);
  else
    lr = l;
  if constexpr (kScaled) m *= max_times[w0 + i];
  const float from = m == minus_inf() ? 0.f : m;
  const int token = c.begin + row / a.group, head = kvh * a.group + row % a.group;
  if (span.parts > 1) {
    const int64_t to = part * parts.rows + (int64_t)token * a.heads + head;
#pragma unroll
    for (int t = 0; t < NG; ++t)
#pragma unroll
      for (int y = 0; y < 16; y += 4)
        *reinterpret_cast<f4*>(parts.o + to * D + t * 32 + 2 * y + 4 * h) = f4{o[t][y], o[t][y + 1], o[t][y + 2], o[t][y + 3]};
    if (h == 0) parts.ml[to] = f4{m, l, lr, 0.f};
    return;
  }
  T* out = static_cast<T*>(a.out.d) + (int64_t)token * a.out.token_stride + (int64_t)head * a.out.head_stride;
  const float f = lr == 0.f ? 0.f : 1.f / lr;
  const bool wide_out = ((reinterpret_cast<uintptr_t>(a.out.d) / sizeof(T) | (uint64_t)a.out.token_stride |
                          (uint64_t)a.out.head_stride) & 3) == 0;
#pragma unroll
  for (int t = 0; t < NG; ++t) {
#pragma unroll
    for (int y = 0; y < 16; y += 4) {
      typedef T run_of __attribute__((ext_vector_type(4)));
      run_of r;
#pragma unroll
      for (int z = 0; z < 4; ++z) r[z] = (T)(o[t][y + z] * f);
      T* at = out + t * 32 + 2 * y + 4 * h;
      if (wide_out) {
        __builtin_memcpy(__builtin_assume_aligned(at, sizeof r), &r, sizeof r);
      } else {
#pragma unroll
        for (int z = 0; z < 4; ++z) at[z] = r[z];
      }
    }
  }
  if (a.lse && h == 0)
    a.lse[(int64_t)token * a.heads + head] = l == 0.f ? minus_inf() : (from + (__builtin_amdgcn_logf(l) - kShift)) * kLn2;
}

// alone: sequences of few rows are its too.  Registers for three workgroups of
// 16-bit queries in heads of up to 64 (more of the waiting hidden), one of heads
// beyond 128, whose sums alone are 128 registers.
template <typename T, int kBits, int GT, int NG>
__global__ __launch_bounds__((QTile<T, kBits, GT>::kThreads), GT == 8 ? 1 : GT == 2 && sizeof(T) == 2 ? 3 : 2)
void chunk_quant_kernel(AttendArgs a, Parts parts, bool alone) {
  chunk_quant_rows<T, kBits, GT, NG>(a, parts, alone, blockIdx.x, gridDim.x, blockIdx.z);
}

template <typename T, int kBits, int GT, int NG>
hipError_t chunk_of(const AttendArgs& a, const Parts& parts, int64_t tiles, bool alone, hipStream_t s) {
  constexpr size_t lds = 2 * QTile<T, kBits, GT>::kStage;
  if (lds > 60000) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(chunk_quant_kernel<T, kBits, GT, NG>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
  }
  chunk_quant_kernel<T, kBits, GT, NG>
      <<<dim3((unsigned)(tiles * a.p.kv_heads), 1, parts.most), QTile<T, kBits, GT>::kThreads, lds, s>>>(a, parts, alone);
  return hipGetLastError();
}

template <typename T, int kBits>
hipError_t chunk_width(const AttendArgs& a, const Parts& parts, int64_t tiles, bool alone, hipStream_t s) {
  switch (a.p.dim / 32) {
    case 1: return chunk_of<T, kBits, 2, 1>(a, parts, tiles, alone, s);
    case 2: return chunk_of<T, kBits, 2, 2>(a, parts, tiles, alone, s);
    case 3: return chunk_of<T, kBits, 4, 3>(a, parts, tiles, alone, s);
    case 4: return chunk_of<T, kBits, 4, 4>(a, parts, tiles, alone, s);
    case 5: return chunk_of<T, kBits, 8, 5>(a, parts, tiles, alone, s);
    case 6: return chunk_of<T, kBits, 8, 6>(a, parts, tiles, alone, s);
    case 7: return chunk_of<T, kBits, 8, 7>(a, parts, tiles, alone, s);
    default: return chunk_of<T, kBits, 8, 8>(a, parts, tiles, alone, s);
  }
}

template <typename T>
hipError_t chunk_type(const AttendArgs& a, int cache_type, const Parts& parts, int64_t tiles, bool alone, hipStream_t s) {
  return cache_type == kQ8_0 ? chunk_width<T, 8>(a, parts, tiles, alone, s) : chunk_width<T, 4>(a, parts, tiles, alone, s);
}

}  // namespace

hipError_t launch_chunk_quant(const AttendArgs& a, int type, int cache_type, const Parts& parts, int64_t tiles,
                              bool alone, hipStream_t s) {
  switch (type) {
    case kF32: return chunk_type<float>(a, cache_type, parts, tiles, alone, s);
    case kF16: return chunk_type<_Float16>(a, cache_type, parts, tiles, alone, s);
    default: return chunk_type<__bf16>(a, cache_type, parts, tiles, alone, s);
  }
}

}  // namespace nls
