// nls_attend_quant.h -- attention of sequences of few rows over pages of
// blocks: the work of one workgroup.
//
// With K = d c and V = d c in blocks of 32 elements (nls_quant.h), the codes are
// what meets the queries and the weights on the matrix cores, and the factors
// stay outside of the products:
//   s_j  = scale sum_x d_jx (sum_{e in x} c_je q_e)
//   o_e  = sum_j (p_j d_jx) c_je        for e in block x
// Codes are whole numbers, exact in fp16, so nothing of the cache is rounded;
// a block is the depth of one 16 x 16 x 32 product.
//
// What bounds it: one pass over the blocks, at what this pattern of loads reaches
// (6.2 TB/s with nothing done to what arrives), for 8 bits: 64 contexts of 8192,
// heads of 128, bf16 6.0 TB/s.  For 4 bits the steps between a load and its use
// take as long as the bytes: 4.6 TB/s there, 3.6 with fp32 queries; 64 contexts of
// up to 16384 190 us, one of 131071 (fp32) 49.
// Measured and left: three waves a SIMD, which do not fit and spill; steps of 64
// keys, the same; two steps' loads in flight, no faster; codes as they are in the
// mantissa of a denormal number, which saves the subtraction and no time.  Loads in
// a branch are waited for at its end: the loop's body is compiled with and without
// the next step's (202 -> 191 us).
#pragma once
#include "nls_attend.h"
#include "nls_quant.h"

namespace nls {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));

// Codes as fp16 pairs.  A number c below 2^10 put into the mantissa of 1024 is
// 1024 + c (four bits further up, into that of 64: 64 + c); what is taken off
// is exact.
__device__ __forceinline__ uint32_t less(uint32_t x, float by) {
  const h2 r = __builtin_bit_cast(h2, x) - h2{(_Float16)by, (_Float16)by};
  return __builtin_bit_cast(uint32_t, r);
}
// (a number that the compiler does not know is one register and one instruction
// with the mask; a constant would be an instruction of its own)
template <uint32_t kWord>
__device__ __forceinline__ uint32_t word() {
  uint32_t x;
  asm("v_mov_b32 %0, %1" : "=v"(x) : "i"(kWord));
  return x;
}
__device__ __forceinline__ uint32_t low_nibbles(uint32_t x) { return less((x & 0x000f000fu) | word<0x64006400u>(), 1032.f); }
__device__ __forceinline__ uint32_t high_nibbles(uint32_t x) { return less((x & 0x00f000f0u) | word<0x54005400u>(), 72.f); }

// (a value, not an element of a vector: of that __builtin_bit_cast takes the
// vector's first)
__device__ __forceinline__ h2 halves(uint32_t x) { return __builtin_bit_cast(h2, x); }

// Eight numbers as two halves each.  The first is what both come from: let alone,
// the compiler rounds a product to fp16 from its factors for one and from fp32
// for the other, and in one of some thousands the two do not belong together.
__device__ __forceinline__ void in_two(const float* x, h8* p) {
  u4 hi, lo;
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    uint32_t r = __builtin_bit_cast(uint32_t, h2{(_Float16)x[2 * n], (_Float16)x[2 * n + 1]});
    asm("" : "+v"(r));
    const h2 h = halves(r);
    const h2 rest{(_Float16)__builtin_fmaf((float)h[0], -1.f, x[2 * n]), (_Float16)__builtin_fmaf((float)h[1], -1.f, x[2 * n + 1])};
    hi[n] = r;
    lo[n] = __builtin_bit_cast(uint32_t, rest);
  }
  p[0] = __builtin_bit_cast(h8, hi);
  p[1] = __builtin_bit_cast(h8, lo);
}

// A key unit's 8 elements.
template <int kBits>
__device__ __forceinline__ h8 key_codes(const uint32_t* c) {
  u4 r;
  if constexpr (kBits == 8) {
#pragma unroll
    for (int n = 0; n < 4; ++n)
      r[n] = less(__builtin_amdgcn_perm(0x64646464u, c[n / 2], n & 1 ? 0x04030402u : 0x04010400u), 1152.f);
  } else {
    r[0] = low_nibbles(c[0]);
    r[1] = high_nibbles(c[0]);
    r[2] = low_nibbles(c[0] >> 8);
    r[3] = high_nibbles(c[0] >> 8);
  }
  return __builtin_bit_cast(h8, r);
}
// One element of block x of two tokens' value pieces: element 32 x + 16 h + i of
// lane i.
template <int kBits>
__device__ __forceinline__ uint32_t value_codes(const uint32_t* a, const uint32_t* b, int x, int h) {
  const int n = kBits == 8 ? 2 * x + h : x;  // the byte
  const uint32_t pair = __builtin_amdgcn_perm(b[n / 4], a[n / 4], 0x0c000c00u | (4 + n % 4) << 16 | n % 4);
  if constexpr (kBits == 8) return less(pair | 0x64006400u, 1152.f);
  return h ? high_nibbles(pair) : low_nibbles(pair);
}

// fp32 queries are two fp16 parts, 22 bits; one holds fp16 and bf16 queries whole.
template <typename T>
constexpr int quant_parts() {
  return sizeof(T) == 4 ? 2 : 1;
}
// Weights times factors, likewise; for bf16 queries they are rounded to fp16, once (an
// eighth of the output's own rounding.  Two parts: 64 contexts of up to 16384 257 us
// for 204, 32 of 8192, heads of 128 91 for 71.  Weights rounded first, a packed product
// for two keys then: 192 and 69 for 199 and 72, and twice the error; and small products
// were lost in fp16's denormal numbers unless the factors were scaled, 195 and 71).
template <typename T>
constexpr int weight_parts() {
  return __is_same(T, __bf16) ? 1 : 2;
}
// What is read once: bytes that leave the caches to others (kAlign: 4 or more).
// (Pages that contexts share are read once for each: 8 x 8 contexts of 8000, 7888 of
// them shared by eight, bf16 over Q4_0 heads of 128 121 us, 132 unshared; a bf16
// cache, whose keys stay in the caches, 181 and 337.)
template <int kBytes, int kAlign>
__device__ __forceinline__ void past_caches(uint32_t* to, const char* from) {
  constexpr int kPiece = kBytes >= 16 ? 16 : kBytes >= 8 ? 8 : 4;
  typedef uint32_t words __attribute__((ext_vector_type(kPiece / 4), aligned(kAlign < kPiece ? kAlign : kPiece)));
  const words x = __builtin_nontemporal_load(reinterpret_cast<const words*>(from));
  __builtin_memcpy(to, &x, kPiece);
  if constexpr (kBytes > kPiece) past_caches<kBytes - kPiece, kAlign>(to + kPiece / 4, from + kPiece);
}

// A truth value as a type.
template <bool B>
struct Is {
  __device__ constexpr operator bool() const { return B; }
};

constexpr float kQuantShift = 14.f;  // log2 of the largest weight times factor

// Heads of NG blocks, at most GT (2, 4 or 8: what the factors are dealt out by).
// Each number of blocks has its own loads, plane by plane: 32 contexts of 8192, bf16
// over Q4_0, heads of 96 62 us and of 192 101 (a byte at a time, for any number
// below GT, 182 and 518; of the 418 off 192, 34 are its second wave a SIMD).
template <typename T, int kBits, int GT, int NG>
__device__ __forceinline__ void few_quant_rows(const AttendArgs& a, const Parts& parts, int tiles, bool chunk_runs,
                                               int group_at, int part) {
  constexpr int NP = quant_parts<T>(), NW = weight_parts<T>(), D = 32 * GT, kWaves = 4, kThreads = 256;
  constexpr int NR = 2, KT = 16 * NR;   // runs of 16 keys in a step of a wave, and its keys
  constexpr int KW = kBits / 4;                       // words of a key unit
  constexpr bool kPad = NG < GT;
  constexpr int VW = (GT * kBits / 4 + 3) / 4;        // words of a lane's piece of a value row
  constexpr bool kApart = kBits == 4 && (NG & 3) == 3;  // a last byte that joins its word when it is used
  extern __shared__ float quant_lds[];                // [wave][16][D + 4] sums
  __shared__ float sh_m[kWaves][16], sh_l[kWaves][16];
  __shared__ __align__(16) uint32_t sh_f[kWaves][KT * GT];  // a step's factors, of keys, then of values: [2 GT][KT]

  const int kvh = group_at % a.p.kv_heads, task = group_at / a.p.kv_heads;
  const int seq = task / tiles, tile = task - seq * tiles;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
  const Chunk c = chunk_of(a.p, seq);
  const int rows = c.n * a.group;
  const bool over = rows > 16 && c.n != 1;
  if (over && (chunk_runs || part > 0)) return;
  const Sees sees = sees_of(a, c);
  constexpr int groups = NG, dim = 32 * NG, row_bytes = 4 * NG * kBits;
  const int size = 1 << a.p.page_shift;
  const QuantShape shape = quant_shape(kBits == 8 ? kQ8_0 : kQ4_0, dim, size);
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
    const int all_lo = as_int(sees.low(sees.p0 + t1)), all_hi = as_int(sees.p0 + t0);

    h8 q[GT][NP];
    float sc, rest = 1.f;  // of a row's products, the power of two that the row was divided by among it
    {
      const T* src = static_cast<const T*>(a.q.d) + (int64_t)(c.begin + row / a.group) * a.q.token_stride +
                     (int64_t)(kvh * a.group + row % a.group) * a.q.head_stride;
      float x[GT][8], top = 0.f;
      const bool wide = ((reinterpret_cast<uintptr_t>(a.q.d) / sizeof(T) | (uint64_t)a.q.token_stride | (uint64_t)a.q.head_stride) &
                         (16 / sizeof(T) - 1)) == 0;
#pragma unroll
      for (int b = 0; b < GT; ++b) {
        T y[8];
        if (!kPad || b < groups) {
          if (wide) {
            __builtin_memcpy(y, __builtin_assume_aligned(src + b * 32 + g * 8, 16), sizeof y);
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = src[b * 32 + g * 8 + j];
          }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[b][j] = row_ok && (!kPad || b < groups) ? (float)y[j] : 0.f;
          top = fmaxf(top, fabsf(x[b][j]));
        }
      }
      // the scale's sign goes to the queries: a largest score is a largest product
      const float flip = a.scale < 0.f ? -1.f : a.scale > 0.f ? 1.f : 0.f;
      const float scale2 = a.scale == 0.f ? 1.f : fabsf(a.scale) * kLog2e;
      int e = 0;
      if constexpr (!__is_same(T, _Float16)) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        // (the scale times the power stays a normal number: masked scores would be
        // -infinity times 0)
        const int least = -126 - ilogbf(scale2);
        e = query_exponent(top);
        e = e < least ? least : e;
      }
      sc = scale2 * ldexpf(1.f, e);
      // Nor does it pass fp32's range: the maximum gets back what was left out.
      if (sc > 0x1p127f) {
        sc = 0x1p127f;
        rest = scale2 * 0x1p-127f * ldexpf(1.f, e);
      }
#pragma unroll
      for (int b = 0; b < GT; ++b)
#pragma unroll
        for (int j = 0; j < 8; ++j) split<NP>(ldexpf(x[b][j] * flip, -e), q[b], j);
    }

    f4 o[2 * GT];
#pragma unroll
    for (int t = 0; t < 2 * GT; ++t) o[t] = f4{0, 0, 0, 0};
    // The weights are taken from m + up: 2^up is above any value's factor so far,
    // so that a weight times a factor is at most 1.  most: that bound as fp16's bits.
    float m = minus_inf(), l = 0.f, up = -24.f, back = kQuantShift - up;
    uint32_t most = 0u;

    // A step's keys are runs of 16, each within a page (-1: none; what is read
    // there is page 0, and counts for nothing).
    struct Pages {
      int at[NR];
    };
    const int32_t* table = a.p.table + (int64_t)c.slot * a.p.table_stride;  // (no keys without a slot)
    const char* base = static_cast<const char*>(a.p.kv) + quant_base(shape, kvh, 0);
    auto entries_at = [&](int kb) {
      Pages e;
#pragma unroll
      for (int s = 0; s < NR; ++s) {
        const int key = kb + s * 16;
        e.at[s] = table[(key < k1 ? key : k1 - 1) >> a.p.page_shift];
      }
      return e;
    };
    auto pages_of = [&](int kb, const Pages& e) {
      Pages p;
#pragma unroll
      for (int s = 0; s < NR; ++s) {
        const int page = __builtin_amdgcn_readfirstlane(e.at[s]);
        p.at[s] = kb + s * 16 < k1 && (uint32_t)page < (uint32_t)a.p.pages ? page : -1;
      }
      return p;
    };
    auto home = [&](int page) { return base + (int64_t)(page < 0 ? 0 : page) * a.p.page_stride; };

    uint32_t kc[NR][GT][KW], vc[4 * NR][VW + kApart];
    // A lane's factors: KT GT / 32 tokens' of one block, keys' for the first 32
    // lanes and values' for the others; 16 lanes of the operands want each, out of
    // LDS.
    constexpr int FT = KT * GT / 32, FW = FT / 2, kAcross = 32 / GT;
    static_assert(FT <= 16, "within a run");
    uint32_t fc[FW];
    const int f_x = lane / kAcross % GT, f_token = lane % kAcross * FT;
    const bool f_there = !kPad || f_x < groups;
    uint32_t* factors = sh_f[wave];
    // Row 4 g + r of a run's scores is key 4 r + g, so that one load of values is of
    // four neighbouring rows.  (One address for the wave and 32 bits for the lane,
    // which are computed where they are used: registers are what waves are short of.)
    auto lane_k = [&]() {
      const int n = here(lane) & 15;
      return (uint32_t)((n % 4 * 4 + n / 4) * row_bytes + (here(lane) >> 4) * groups * kBits);
    };
    auto lane_v = [&](int wide) { return (uint32_t)((here(lane) >> 4) * row_bytes + (here(lane) & 15) * (wide * kBits / 4)); };
    auto lane_f = [&]() {
      const int n = here(lane), x = n / kAcross % GT, token = n % kAcross * FT;
      return (uint32_t)((n < 32 ? 0 : shape.half) + shape.codes + ((!kPad || x < groups ? x : 0) * size + (token & 15)) * 2);
    };
    auto fetch_k = [&](int kb, const Pages& p) {
      const uint32_t at_k = lane_k();
#pragma unroll
      for (int s = 0; s < NR; ++s) {
        const int place = (kb + s * 16) & (size - 1);
        const char* codes = home(p.at[s]) + place * row_bytes;
        past_caches<NG * kBits, (NG * kBits) & -(NG * kBits)>(&kc[s][0][0], codes + at_k);
      }
    };
    // the run of this lane's factors
    auto run_page = [&](const Pages& p) {
      int page = p.at[0];
#pragma unroll
      for (int s = 1; s < NR; ++s) page = f_token >= 16 * s ? p.at[s] : page;
      return page;
    };
    auto fetch_f = [&](int kb, const Pages& p) {
      const char* from = home(run_page(p)) + ((kb + (f_token & ~15)) & (size - 1)) * 2;
      __builtin_memcpy(fc, __builtin_assume_aligned(from + lane_f(), 2 * FT < 16 ? 2 * FT : 16), 2 * FT);
    };
    auto fetch_v = [&](int kb, const Pages& p) {
      const uint32_t at_4 = lane_v(4), at_2 = lane_v(2), at_1 = lane_v(1);
#pragma unroll
      for (int s = 0; s < NR; ++s) {
        const int place = (kb + s * 16) & (size - 1);
        const char* codes = home(p.at[s]) + shape.half + place * row_bytes;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          uint32_t* to = vc[s * 4 + r];
          const char* from = codes + r * 4 * row_bytes;
          // planes of four blocks, of two, of one; block x's codes are bytes of to in its order
          constexpr int kFours = NG / 4, kLast = NG - 1;
#pragma unroll
          for (int n = 0; n < kFours; ++n) past_caches<kBits, kBits>(to + n * kBits / 4, from + n * 16 * kBits + at_4);
          if constexpr ((NG & 2) != 0) {
            const char* at = from + kFours * 16 * kBits + at_2;
            if constexpr (kBits == 8)
              past_caches<4, 4>(to + kFours * 2, at);
            else
              to[kFours] = *reinterpret_cast<const uint16_t*>(at);
          }
          if constexpr ((NG & 1) != 0) {
            const char* at = from + kLast * 4 * kBits + at_1;
            if constexpr (kBits == 8)
              to[kLast / 2] = *reinterpret_cast<const uint16_t*>(at);
            else
              to[kApart ? VW : kLast / 4] = *reinterpret_cast<const uint8_t*>(at);
          }
        }
      }
    };
    // the largest factor of the lanes, the power of two above it (of denormal ones too),
    // and the largest one below that
    auto wave_top = [&](uint32_t d) {
#pragma unroll
      for (int x = 1; x < 64; x <<= 1) {
        const uint32_t other = __shfl_xor(d, x);
        d = other > d ? other : d;
      }
      return d;
    };
    auto above = [](uint32_t d) { return d < 0x400u ? 8 - __builtin_clz(d) : (int)(d >> 10) - 14; };
    auto below = [](int e) { return e < -14 ? (1u << (e + 24)) - 1 : (uint32_t)(e + 14) << 10 | 0x3ffu; };
    // a lane's 4 tokens' factors of a plane of sh_f (token 4 r + g of a run is at 4 g + r)
    auto factors_of = [&](int plane, int s) { return *reinterpret_cast<const u2*>(factors + plane * (KT / 2) + s * 8 + g * 2); };

    constexpr int kStep = kWaves * KT;
    int kb = k0 + wave * KT;
    Pages now, entry;
    if (kb < k1) {
      now = pages_of(kb, entries_at(kb));
      entry = entries_at(kb + kStep);
      fetch_f(kb, now);
      fetch_k(kb, now);
      fetch_v(kb, now);
    }
    // (`more`, whether a step follows, is known when this is compiled: behind a
    // branch the compiler does not know how many loads are on their way, and waits
    // for the next step's with this one's.)
    auto work = [&](auto more, const int kb) {
      bool all = kb + KT <= k1;
#pragma unroll
      for (int s = 0; s < NR; ++s) all = all && now.at[s] >= 0;
      const bool whole = kb >= all_lo && kb + KT - 1 <= all_hi && all;
      // The factors, those of tokens that are not there as 0 (the memory there may
      // hold anything).
      if (!f_there || (!all && run_page(now) < 0)) {
#pragma unroll
        for (int n = 0; n < FW; ++n) fc[n] = 0;
      } else if (!all) {
        const int left = k1 - kb - f_token;  // of this lane's tokens
#pragma unroll
        for (int n = 0; n < FW; ++n) fc[n] &= (2 * n < left ? 0xffffu : 0u) | (2 * n + 1 < left ? 0xffff0000u : 0u);
      }
      // (bits of numbers that are not negative, in order.  One that is not finite has no
      // say, and hides none: it wraps to below the others, which are taken down again.)
      typedef uint16_t us2 __attribute__((ext_vector_type(2)));
      us2 dm{0, 0};
#pragma unroll
      for (int n = 0; n < FW; ++n)
        dm = __builtin_elementwise_max(dm, __builtin_bit_cast(us2, halves(fc[n])) + us2{0x8400, 0x8400});
      dm = __builtin_elementwise_sub_sat(dm, us2{0x8400, 0x8400});
      uint32_t dtop = dm[0] > dm[1] ? dm[0] : dm[1];
      dtop = lane < 32 ? 0 : dtop;
      {
        uint16_t* to = reinterpret_cast<uint16_t*>(factors) + (lane < 32 ? 0 : GT * KT) + f_x * KT + (f_token & ~15);
#pragma unroll
        for (int n = 0; n < FT; ++n) {
          const int token = (f_token & 15) + n;
          to[token % 4 * 4 + token / 4] = (uint16_t)(fc[n / 2] >> (16 * (n & 1)));
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();

      float w[4 * NR];
#pragma unroll
      for (int s = 0; s < NR; ++s) {
        f4 sum{0, 0, 0, 0};
#pragma unroll
        for (int x = 0; x < GT; ++x) {
          if (kPad && x >= groups) break;
          const h8 codes = key_codes<kBits>(kc[s][x]);
          f4 acc{0, 0, 0, 0};
#pragma unroll
          for (int n = NP - 1; n >= 0; --n) acc = mma16(codes, q[x][n], acc);
          const u2 d = factors_of(x, s);
          const h2 d01 = halves(d[0]), d23 = halves(d[1]);
          sum[0] = __builtin_fmaf((float)d01[0], acc[0], sum[0]);
          sum[1] = __builtin_fmaf((float)d01[1], acc[1], sum[1]);
          sum[2] = __builtin_fmaf((float)d23[0], acc[2], sum[2]);
          sum[3] = __builtin_fmaf((float)d23[1], acc[3], sum[3]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) w[s * 4 + r] = sum[r];
      }
      const Pages then = now;
      if constexpr (more) {
        now = pages_of(kb + kStep, entry);
        entry = entries_at(kb + 2 * kStep);
        fetch_f(kb + kStep, now);
        fetch_k(kb + kStep, now);
      }
      uint32_t vis = 0xffff;  // bit j: this row sees key j of this lane
      if (!whole) {
        const int from = low - kb, to = (pos < k1 ? pos : k1 - 1) - kb;
#pragma unroll
        for (int j = 0; j < 4 * NR; ++j) {
          const int n = (j >> 2) * 16 + (j & 3) * 4 + g;
          if (then.at[j >> 2] < 0 || n < from || n > to) {
            w[j] = minus_inf();
            vis &= ~(1u << j);
          }
        }
      }
      float top = w[0];
#pragma unroll
      for (int j = 1; j < 4 * NR; ++j) top = fmaxf(top, w[j]);
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      top *= sc;
      if (__ballot(top > m || dtop > most)) {
        float shrink = up;
        if (__ballot(dtop > most)) {
          const uint32_t d = wave_top(dtop);
          if (d > most) {
            const int e = above(d);
            up = (float)e;
            most = below(e);
          }
        }
        top = ceilf(fmaxf(top, m));  // whole: what it is taken from is exact
        shrink = m == minus_inf() ? 0.f : exp2_((m - top) + (shrink - up));
        m = top;
        // (taken to be 0 where there is no score yet)
        back = kQuantShift - up - (m == minus_inf() ? 0.f : m);
        l *= shrink;
#pragma unroll
        for (int t = 0; t < 2 * GT; ++t) o[t] *= shrink;
      }
      // A weight's exponent, the score less the maximum, is one fused product.  A
      // maximum beyond 2^20 leaves no room for the shift beside it, and so large a
      // product is off by whole numbers when rounded, as the maximum was: all are.
      float p[4 * NR];
      if (__ballot(fabsf(back) > 1048576.f)) {
        const float from = m == minus_inf() ? 0.f : m;
#pragma unroll
        for (int j = 0; j < 4 * NR; ++j) p[j] = w[j] * sc - from + (kQuantShift - up);
      } else {
#pragma unroll
        for (int j = 0; j < 4 * NR; ++j) p[j] = __builtin_fmaf(w[j], sc, back);
      }
#pragma unroll
      for (int j = 0; j < 4 * NR; ++j) {
        p[j] = exp2_(p[j]);
        l += p[j];
      }
      auto values = [&](auto seen) {
#pragma unroll
        for (int b = 0; b < NR; b += 2)  // 32 keys: the depth of one product
#pragma unroll
          for (int x = 0; x < GT; ++x) {
            if (kPad && x >= groups) break;
            u4 d;  // of this lane's 8 keys
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              const u2 r = factors_of(GT + x, b + s);
              d[2 * s] = r[0];
              d[2 * s + 1] = r[1];
            }
            // (what this row does not see may be NaN, which its weight of 0 would not
            // keep out)
            if constexpr (!seen)
#pragma unroll
              for (int n = 0; n < 4; ++n)
                d[n] &= ((vis >> (4 * b + 2 * n)) & 1 ? 0xffffu : 0u) | ((vis >> (4 * b + 2 * n + 1)) & 1 ? 0xffff0000u : 0u);
            float pw[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) pw[j] = __builtin_fmaf(p[4 * b + j], (float)halves(d[j / 2])[j & 1], 0.f);
            h8 pd[NW];
            if constexpr (NW == 1) {
#pragma unroll
              for (int j = 0; j < 8; ++j) pd[0][j] = (_Float16)pw[j];  // (one instruction with the product)
            } else {
              in_two(pw, pd);
            }
            h8 codes[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              u4 r;
#pragma unroll
              for (int n = 0; n < 4; ++n) r[n] = value_codes<kBits>(vc[4 * b + 2 * n], vc[4 * b + 2 * n + 1], x, h);
              codes[h] = __builtin_bit_cast(h8, r);
            }
            // (one product does not wait for the other)
#pragma unroll
            for (int n = NW - 1; n >= 0; --n)
#pragma unroll
              for (int h = 0; h < 2; ++h) o[2 * x + h] = mma16(codes[h], pd[n], o[2 * x + h]);
          }
      };
      if constexpr (kApart)
#pragma unroll
        for (int n = 0; n < 4 * NR; ++n) vc[n][VW - 1] |= vc[n][VW] << 16;
      if (whole)
        values(Is<true>{});
      else
        values(Is<false>{});
      if constexpr (more) fetch_v(kb + kStep, now);
    };
    for (; kb + kStep < k1; kb += kStep) work(Is<true>{}, kb);
    if (kb < k1) work(Is<false>{}, kb);

    // the waves' sums, relative to the largest of their maxima alone
    m *= rest;
    const float full = exp2_(up);
    l *= full;
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g == 0) {
      sh_m[wave][i] = m;
      sh_l[wave][i] = l;
    }
    __syncthreads();
    float top = sh_m[0][i];
#pragma unroll
    for (int x = 1; x < kWaves; ++x) top = fmaxf(top, sh_m[x][i]);
    const float f = exp2_(m - (top == minus_inf() ? 0.f : top)) * full;
    float* mine = quant_lds + (wave * 16 + i) * (D + 4);
#pragma unroll
    for (int t = 0; t < 2 * GT; ++t) *reinterpret_cast<f4*>(mine + t * 16 + g * 4) = o[t] * f;
    __syncthreads();
    for (int idx = threadIdx.x; idx < 16 * (D / 4); idx += kThreads) {
      const int r = idx / (D / 4), d = idx % (D / 4) * 4;
      if (r >= rn) break;
      float rt = sh_m[0][r], sum = 0.f;
#pragma unroll
      for (int x = 1; x < kWaves; ++x) rt = fmaxf(rt, sh_m[x][r]);
      const float rf = rt == minus_inf() ? 0.f : rt;
      f4 s{0, 0, 0, 0};
#pragma unroll
      for (int x = 0; x < kWaves; ++x) {
        s += *reinterpret_cast<const f4*>(quant_lds + (x * 16 + r) * (D + 4) + d);
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
            sum == 0.f ? minus_inf() : (rf + (__builtin_amdgcn_logf(sum) - kQuantShift)) * kLn2;
    }
    if (!over) return;
    __syncthreads();  // the next tile's sums take the same LDS
  }
}

// Rows of a workgroup of the chunk kernel, 32 to a wave.  Turning codes into
// operands is work that the waves share: in heads of 96 and 128 whose values are
// two parts eight waves take it (2048 tokens over 16384 keys, Q4_0: fp32 queries
// 1530 us with four, 1424 so; fp16 1721 and 1246); elsewhere four are as fast (bf16,
// heads of 128: 814 and 816) or faster (heads of 64, bf16: 157 and 186).
template <typename T>
constexpr int quant_tile(int groups) {
  return weight_parts<T>() == 2 && (groups == 3 || groups == 4) ? 256 : 128;
}

// Launched by launch_attend (nls_attend.hip), which joins the parts.
hipError_t launch_few_quant(const AttendArgs& a, int type, int cache_type, const Parts& parts, int few_tiles,
                            bool chunk_runs, hipStream_t s);
hipError_t launch_chunk_quant(const AttendArgs& a, int type, int cache_type, const Parts& parts, int64_t tiles,
                              bool alone, hipStream_t s);

}  // namespace nls
