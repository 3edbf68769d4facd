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
__device__ __forceinline__ uint32_t low_nibbles(uint32_t x) { return less((x & 0x000f000fu) | 0x64006400u, 1032.f); }
__device__ __forceinline__ uint32_t high_nibbles(uint32_t x) { return less((x & 0x00f000f0u) | 0x54005400u, 72.f); }

// (a value, not an element of a vector: of that __builtin_bit_cast takes the
// vector's first)
__device__ __forceinline__ h2 halves(uint32_t x) { return __builtin_bit_cast(h2, x); }

// A product as the fp32 number that it is: where it is split, the compiler else
// rounds it to fp16 from its factors for one part and from fp32 for the other,
// and in one of some thousands the two do not belong together.
__device__ __forceinline__ float settled(float x) {
  asm("" : "+v"(x));
  return x;
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

// fp32 queries and weights times factors: two fp16 parts, 22 bits.  16-bit ones:
// one, which holds fp16 and bf16 queries whole and 11 bits of a weight.
template <typename T>
constexpr int quant_parts() {
  return sizeof(T) == 4 ? 2 : 1;
}
constexpr float kQuantShift = 14.f;  // log2 of the largest weight times factor

// kPad: heads of fewer than GT blocks
template <typename T, int kBits, int GT, bool kPad>
__device__ __forceinline__ void few_quant_rows(const AttendArgs& a, const Parts& parts, int tiles, bool chunk_runs,
                                               int group_at, int part) {
  constexpr int NP = quant_parts<T>(), D = 32 * GT, kWaves = 4, kThreads = 256;
  constexpr int KW = kBits / 4;                       // words of a key unit
  constexpr int VW = (GT * kBits / 4 + 3) / 4;        // words of a lane's piece of a value row
  extern __shared__ float quant_lds[];                // [wave][16][D + 4] sums
  __shared__ float sh_m[kWaves][16], sh_l[kWaves][16];

  const int kvh = group_at % a.p.kv_heads, task = group_at / a.p.kv_heads;
  const int seq = task / tiles, tile = task - seq * tiles;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
  const Chunk c = chunk_of(a.p, seq);
  const int rows = c.n * a.group;
  const bool over = rows > 16 && c.n != 1;
  if (over && (chunk_runs || part > 0)) return;
  const Sees sees = sees_of(a, c);
  const int dim = a.p.dim, groups = kPad ? dim / 32 : GT;
  const int size = 1 << a.p.page_shift;
  const QuantShape shape = quant_shape(kBits == 8 ? kQ8_0 : kQ4_0, kPad ? dim : D, size);
  const int row_bytes = kPad ? shape.row : D * kBits / 8;
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
    float qs = 1.f;  // the row divided by a power of two
    {
      const T* src = static_cast<const T*>(a.q.d) + (int64_t)(c.begin + row / a.group) * a.q.token_stride +
                     (int64_t)(kvh * a.group + row % a.group) * a.q.head_stride;
      float x[GT][8], top = 0.f;
#pragma unroll
      for (int b = 0; b < GT; ++b)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int d = b * 32 + g * 8 + j;
          x[b][j] = row_ok && d < dim ? (float)src[d] : 0.f;
          top = fmaxf(top, fabsf(x[b][j]));
        }
      int e = 0;
      if constexpr (!__is_same(T, _Float16)) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        e = query_exponent(top);
        qs = ldexpf(1.f, e);
      }
#pragma unroll
      for (int b = 0; b < GT; ++b)
#pragma unroll
        for (int j = 0; j < 8; ++j) split<NP>(ldexpf(x[b][j], -e), q[b], j);
    }
    const float sc = a.scale * kLog2e;

    f4 o[2 * GT];
#pragma unroll
    for (int t = 0; t < 2 * GT; ++t) o[t] = f4{0, 0, 0, 0};
    // The weights are taken from m + up: `up` is a power of two no less than any
    // value's factor so far, so that a weight times a factor is at most 1.
    float m = minus_inf(), l = 0.f, most = 0.f;  // (most = 2^up, or 0)
    float up = -24.f;                            // (fp16's least number is 2^-24)

    // A step's 32 keys are two runs of 16, each within a page: its first byte of
    // this head, in the same registers for the wave.
    struct Step {
      const char* at[2];
      bool there[2];
    };
    const int32_t* table = a.p.table + (int64_t)c.slot * a.p.table_stride;  // (no keys without a slot)
    const char* base = static_cast<const char*>(a.p.kv) + quant_base(shape, kvh, 0);
    struct Entries {
      int at[2];
    };
    auto entries_at = [&](int kb) {
      Entries e;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int key = kb + s * 16;
        e.at[s] = table[(key < k1 ? key : k1 - 1) >> a.p.page_shift];
      }
      return e;
    };
    auto step_of = [&](int kb, const Entries& e) {
      Step p;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int page = __builtin_amdgcn_readfirstlane(e.at[s]);
        p.there[s] = kb + s * 16 < k1 && (uint32_t)page < (uint32_t)a.p.pages;
        p.at[s] = base + (int64_t)(p.there[s] ? page : 0) * a.p.page_stride;
      }
      return p;
    };
    uint32_t kc[2][GT][KW], vc[8][VW];
    u2 kd[2][GT], vd[2][GT];  // factors of 4 keys
    auto fetch_k = [&](int kb, const Step& p) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int place = (kb + s * 16) & (size - 1);
        const char* codes = p.at[s] + (place + i) * row_bytes + g * groups * kBits;
        const char* factors = p.at[s] + shape.codes + (place + g * 4) * 2;
        if constexpr (!kPad) {
          __builtin_memcpy(kc[s], __builtin_assume_aligned(codes, GT * kBits < 16 ? GT * kBits : 16), GT * kBits);
        } else {
#pragma unroll
          for (int x = 0; x < GT; ++x)
            if (x < groups) __builtin_memcpy(kc[s][x], __builtin_assume_aligned(codes + x * kBits, kBits), kBits);
        }
#pragma unroll
        for (int x = 0; x < GT; ++x)
          if (!kPad || x < groups) kd[s][x] = *reinterpret_cast<const u2*>(factors + x * size * 2);
      }
    };
    auto fetch_v = [&](int kb, const Step& p) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int place = (kb + s * 16) & (size - 1);
        const char* codes = p.at[s] + shape.half + (place + g * 4) * row_bytes;
        const char* factors = p.at[s] + shape.half + shape.codes + (place + g * 4) * 2;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          uint32_t* to = vc[s * 4 + r];
          const char* from = codes + r * row_bytes;
          if constexpr (!kPad) {
            constexpr int kWide = GT < 4 ? GT : 4, kBytes = kWide * kBits / 4;  // of a plane
            if constexpr (kBytes == 2) {
              to[0] = *reinterpret_cast<const uint16_t*>(from + i * 2);
            } else {
#pragma unroll
              for (int n = 0; n < GT / kWide; ++n)
                __builtin_memcpy(to + n * kBytes / 4, __builtin_assume_aligned(from + n * 16 * kBytes + i * kBytes, kBytes),
                                 kBytes);
            }
          } else {
#pragma unroll
            for (int w = 0; w < VW; ++w) to[w] = 0;
#pragma unroll
            for (int x = 0; x < GT; ++x) {
              if (x >= groups) break;
              const int fours = groups & ~3, first = x < fours ? x & ~3 : x < fours + (groups & 2) ? fours : x;
              const int wide = x < fours ? 4 : x < fours + (groups & 2) ? 2 : 1;
              const char* at = from + (first * 16 + i * wide + x - first) * (kBits / 4);
              if constexpr (kBits == 8)
                to[x / 2] |= (uint32_t)*reinterpret_cast<const uint16_t*>(at) << (16 * (x & 1));
              else
                to[x / 4] |= (uint32_t)*reinterpret_cast<const uint8_t*>(at) << (8 * (x & 3));
            }
          }
        }
#pragma unroll
        for (int x = 0; x < GT; ++x)
          if (!kPad || x < groups) vd[s][x] = *reinterpret_cast<const u2*>(factors + x * size * 2);
      }
    };

    constexpr int kStep = kWaves * 32;
    int kb = k0 + wave * 32;
    Step step, step1;
    Entries entry1;
    if (kb < k1) {
      step = step_of(kb, entries_at(kb));
      entry1 = entries_at(kb + kStep);
      fetch_k(kb, step);
      fetch_v(kb, step);
    }
    for (; kb < k1; kb += kStep) {
      const bool more = kb + kStep < k1;
      const bool whole = kb >= all_lo && kb + 31 <= all_hi && kb + 32 <= k1 && step.there[0] && step.there[1];
      float w[8];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        f4 sum{0, 0, 0, 0};
#pragma unroll
        for (int x = 0; x < GT; ++x) {
          if (kPad && x >= groups) break;
          const h8 codes = key_codes<kBits>(kc[s][x]);
          f4 acc{0, 0, 0, 0};
#pragma unroll
          for (int n = NP - 1; n >= 0; --n) acc = mma16(codes, q[x][n], acc);
          const h2 d01 = halves(kd[s][x][0]), d23 = halves(kd[s][x][1]);
          sum[0] = __builtin_fmaf((float)d01[0], acc[0], sum[0]);
          sum[1] = __builtin_fmaf((float)d01[1], acc[1], sum[1]);
          sum[2] = __builtin_fmaf((float)d23[0], acc[2], sum[2]);
          sum[3] = __builtin_fmaf((float)d23[1], acc[3], sum[3]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) w[s * 4 + r] = sum[r] * qs * sc;
      }
      if (more) {
        step1 = step_of(kb + kStep, entry1);
        entry1 = entries_at(kb + 2 * kStep);
        fetch_k(kb + kStep, step1);
      }
      if (!whole) {
        // What this row does not see weighs nothing, and its values' factors,
        // which may be anything there, count as 0 in this lane's products.
        const int from = low - kb, to = (pos < k1 ? pos : k1 - 1) - kb;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int n = (j >> 2) * 16 + g * 4 + (j & 3);
          if (!step.there[j >> 2] || n < from || n > to) {
            w[j] = minus_inf();
#pragma unroll
            for (int x = 0; x < GT; ++x) vd[j >> 2][x][(j & 3) / 2] &= j & 1 ? 0x0000ffffu : 0xffff0000u;
          }
        }
      }
      // the factors' bound
      h2 dm{0, 0};
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int x = 0; x < GT; ++x)
          if (!kPad || x < groups)
#pragma unroll
            for (int y = 0; y < 2; ++y) dm = __builtin_elementwise_max(dm, halves(vd[s][x][y]));
      const float dtop = fmaxf((float)dm[0], (float)dm[1]);
      float top = w[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) top = fmaxf(top, w[j]);
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      if (__ballot(top > m || dtop > most)) {
        float shrink = up;
        if (__ballot(dtop > most)) {
          float d = dtop;
#pragma unroll
          for (int x = 1; x < 64; x <<= 1) d = fmaxf(d, __shfl_xor(d, x));
          up = (float)(ilogbf(d) + 1);
          most = ldexpf(1.f, (int)up);
        }
        top = ceilf(fmaxf(top, m));  // whole: what it is taken from is exact
        shrink = m == minus_inf() ? 0.f : exp2_((m - top) + (shrink - up));
        m = top;
        l *= shrink;
#pragma unroll
        for (int t = 0; t < 2 * GT; ++t) o[t] *= shrink;
      }
      const float from = m == minus_inf() ? 0.f : m, shift = kQuantShift - up;
      float p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        p[j] = exp2_(w[j] - from + shift);
        l += p[j];
      }
#pragma unroll
      for (int x = 0; x < GT; ++x) {
        if (kPad && x >= groups) break;
        h8 pd[NP];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const h2 d = halves(vd[j >> 2][x][(j & 3) / 2]);
          split<NP>(settled(p[j] * (float)d[j & 1]), pd, j);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          u4 codes;
#pragma unroll
          for (int n = 0; n < 4; ++n) codes[n] = value_codes<kBits>(vc[2 * n], vc[2 * n + 1], x, h);
#pragma unroll
          for (int n = NP - 1; n >= 0; --n)
            o[2 * x + h] = mma16(__builtin_bit_cast(h8, codes), pd[n], o[2 * x + h]);
        }
      }
      if (more) {
        fetch_v(kb + kStep, step1);
        step = step1;
      }
    }

    // the waves' sums, relative to the largest of their maxima alone
    const float back = exp2_(up);
    l *= back;
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
    const float f = exp2_(m - (top == minus_inf() ? 0.f : top)) * back;
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

// Launched by launch_attend (nls_attend.hip), which joins the parts.
hipError_t launch_few_quant(const AttendArgs& a, int type, int cache_type, const Parts& parts, int few_tiles,
                            bool chunk_runs, hipStream_t s);
hipError_t launch_chunk_quant(const AttendArgs& a, int type, int cache_type, const Parts& parts, int64_t tiles,
                              bool alone, hipStream_t s);

}  // namespace nls
