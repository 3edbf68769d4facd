// Prints where the elements of a row of blocks lie (nls_quant.h), one line each:
// type dim k element byte shift, for a program that knows it otherwise; and
// checks that lanes' pieces fill each row once.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../nim.llm_amd/csrc/nls_quant.h"

using namespace nls;

static void need(bool ok, const char* what) {
  if (!ok) {
    std::printf("wrong: %s\n", what);
    std::exit(1);
  }
}

int main() {
  for (int type : {kQ8_0, kQ4_0})
    for (int dim = 32; dim <= 256; dim += 32)
      for (int size = kMinQuantPage; size <= kMaxPageSize; size *= 4) {
        const QuantShape s = quant_shape(type, dim, size);
        need(s.groups == dim / 32 && s.row == dim * s.bits / 8 && s.codes == s.row * size, "sizes");
        need(s.half == s.codes + s.groups * size * 2 && s.half % 16 == 0 && s.codes % 16 == 0, "pieces of 16 bytes");
        for (int heads : {1, 3, 8}) {
          need(quant_page_bytes(s, heads) == (int64_t)heads * 2 * s.half, "page");
          need(quant_base(s, heads - 1, 1) + s.half == quant_page_bytes(s, heads), "last half");
        }
        if (size != kMinQuantPage) continue;
        std::vector<int> keys(s.row * 2, 0), values(s.row * 2, 0);  // half bytes
        auto take = [&](std::vector<int>& v, int e, int k, int byte, int shift) {
          need(byte >= 0 && byte < s.row, "within the row");
          for (int n = 0; n < s.bits / 4; ++n) need(++v[byte * 2 + shift / 4 + n] == 1, "once");
          std::printf("%d %d %d %d %d %d\n", type, dim, k, e, byte, shift);
        };
        for (int x = 0; x < s.groups; ++x)
          for (int g = 0; g < 4; ++g)
            for (int e = 0; e < 8; ++e) {
              const int at = key_at(s, x, g), n = nibble_of(e);
              take(keys, 32 * x + 8 * g + e, 0, s.bits == 8 ? at + e : at + n / 2, s.bits == 8 ? 0 : 4 * (n % 2));
            }
        int blocks = 0;
        for (int n = 0; n < plane_count(s.groups); ++n) {
          const Plane p = plane_of(s.groups, n);
          need(p.first == blocks, "planes in order");
          blocks += p.wide;
          for (int i = 0; i < 16; ++i)
            for (int x = 0; x < p.wide; ++x)
              for (int h = 0; h < 2; ++h) {
                const int at = value_at(s, p, i) + x * s.bits / 4;
                take(values, 32 * (p.first + x) + 16 * h + i, 1, s.bits == 8 ? at + h : at, s.bits == 8 ? 0 : 4 * h);
              }
        }
        need(blocks == s.groups, "every block");
        for (int n = 0; n < s.row * 2; ++n) need(keys[n] == 1 && values[n] == 1, "every place");
      }
  std::printf("ok\n");
}
