// nls_attend_quant.hip -- attention of few rows over pages of blocks, in
// launches of its own.
#include "nls_attend_quant.h"

namespace nls {
namespace {

constexpr int kThreads = 256;

// Waves per SIMD that registers are kept for.  Heads beyond 128 want more than two
// waves have; over 4 bits two are faster all the same (32 contexts of 8192, bf16,
// heads of 160, 192, 224 and 256: 89, 100, 114 and 137 us with two, 126, 134, 148 and
// 161 with one; fp32 of 160 and 192 120 and 137, 167 and 185), but for fp32 queries
// in heads of 224 and 256 (214 either way); over 8 bits one is (192: 179, with two
// 198; fp32 191 and 239).  Three for heads of 96 gain nothing (62 us, 63.5 so).
template <typename T, int kBits, int GT, int NG>
constexpr int few_quant_waves() {
  return GT == 8 ? (kBits == 4 && (sizeof(T) == 2 || NG <= 6) ? 2 : 1) : GT == 4 || (sizeof(T) == 4 && kBits == 8) ? 2 : 3;
}

template <typename T, int kBits, int GT, int NG>
__global__ __launch_bounds__(kThreads, (few_quant_waves<T, kBits, GT, NG>())) void few_quant_kernel(AttendArgs a, Parts parts,
                                                                                               int tiles, bool chunk_runs) {
  few_quant_rows<T, kBits, GT, NG>(a, parts, tiles, chunk_runs, blockIdx.x, blockIdx.z);
}

template <typename T, int kBits, int GT, int NG>
hipError_t few_of(const AttendArgs& a, const Parts& parts, int tiles, bool chunk_runs, hipStream_t s) {
  constexpr size_t lds = (size_t)4 * 16 * (32 * GT + 4) * sizeof(float);
  if (lds > 60000) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(few_quant_kernel<T, kBits, GT, NG>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
  }
  few_quant_kernel<T, kBits, GT, NG>
      <<<dim3(a.p.kv_heads * a.p.seqs * tiles, 1, parts.most), kThreads, lds, s>>>(a, parts, tiles, chunk_runs);
  return hipGetLastError();
}

template <typename T, int kBits>
hipError_t few_width(const AttendArgs& a, const Parts& parts, int tiles, bool chunk_runs, hipStream_t s) {
  switch (a.p.dim / 32) {
    case 1: return few_of<T, kBits, 2, 1>(a, parts, tiles, chunk_runs, s);
    case 2: return few_of<T, kBits, 2, 2>(a, parts, tiles, chunk_runs, s);
    case 3: return few_of<T, kBits, 4, 3>(a, parts, tiles, chunk_runs, s);
    case 4: return few_of<T, kBits, 4, 4>(a, parts, tiles, chunk_runs, s);
    case 5: return few_of<T, kBits, 8, 5>(a, parts, tiles, chunk_runs, s);
    case 6: return few_of<T, kBits, 8, 6>(a, parts, tiles, chunk_runs, s);
    case 7: return few_of<T, kBits, 8, 7>(a, parts, tiles, chunk_runs, s);
    default: return few_of<T, kBits, 8, 8>(a, parts, tiles, chunk_runs, s);
  }
}

template <typename T>
hipError_t few_type(const AttendArgs& a, int cache_type, const Parts& parts, int tiles, bool chunk_runs, hipStream_t s) {
  return cache_type == kQ8_0 ? few_width<T, 8>(a, parts, tiles, chunk_runs, s)
                             : few_width<T, 4>(a, parts, tiles, chunk_runs, s);
}

}  // namespace

hipError_t launch_few_quant(const AttendArgs& a, int type, int cache_type, const Parts& parts, int few_tiles,
                            bool chunk_runs, hipStream_t s) {
  switch (type) {
    case kF32: return few_type<float>(a, cache_type, parts, few_tiles, chunk_runs, s);
    case kF16: return few_type<_Float16>(a, cache_type, parts, few_tiles, chunk_runs, s);
    default: return few_type<__bf16>(a, cache_type, parts, few_tiles, chunk_runs, s);
  }
}

}  // namespace nls
