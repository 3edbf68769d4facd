// The index arithmetic of the paged cache (nls_paged.h), checked on the CPU
// against the plain statement of it, bad lengths, starts, slots and pages among
// the inputs.  Prints "ok" and the number of cases.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "../nim.llm_amd/csrc/nls_paged.h"

using namespace nls;

#define CHECK(c)                                          \
  do {                                                    \
    if (!(c)) {                                           \
      std::printf("line %d: %s\n", __LINE__, #c);         \
      std::exit(1);                                       \
    }                                                     \
  } while (0)

int main() {
  std::mt19937 rng(7);
  auto pick = [&](int lo, int hi) { return (int)(lo + (int64_t)(rng() % (uint32_t)(hi - lo + 1))); };
  long cases = 0;
  for (int round = 0; round < 4000; ++round) {
    PagedArgs a{};
    a.pages = pick(1, 50);
    a.page_shift = pick(0, 6);
    a.slots = pick(1, 6);
    a.max_pages = pick(1, 9);
    a.table_stride = a.max_pages + pick(0, 3);
    a.page_stride = 4096;
    a.token_stride = 64;
    a.seqs = pick(1, 6);
    a.tokens = pick(0, 80);
    std::vector<int32_t> table((size_t)a.slots * a.table_stride), lens(a.slots), starts(a.seqs + 1), slots(a.seqs);
    for (auto& t : table) t = pick(0, 9) ? pick(0, a.pages - 1) : pick(0, 1) ? -pick(1, 9) : a.pages + pick(0, 9);
    for (auto& n : lens) n = pick(0, 9) ? pick(0, a.max_pages << a.page_shift) : pick(-5, 2000);
    int at = pick(0, 3);
    for (auto& s : starts) {
      s = at;
      at += pick(0, 20);
    }
    const bool wild = pick(0, 9) == 0;  // starts that fall or are negative: cut to the rows there are
    if (wild) starts[pick(0, a.seqs)] = pick(-100, 300);
    for (auto& s : slots) s = pick(0, 9) ? pick(0, a.slots - 1) : pick(-3, a.slots + 3);
    a.table = table.data();
    a.lens = lens.data();
    a.starts = starts.data();
    a.slot_of = slots.data();
    for (int i = 0; i < a.seqs; ++i) {
      const Chunk c = chunk_of(a, i);
      CHECK(c.begin >= 0 && c.n >= 0 && c.begin + c.n <= a.tokens);
      CHECK(c.len >= 0 && c.len <= ((int64_t)a.max_pages << a.page_shift));
      CHECK(c.slot == (slots[i] >= 0 && slots[i] < a.slots ? slots[i] : -1));
      if (c.slot < 0) CHECK(c.len == 0 && position_of(a, c, 0) == -1);
      for (int64_t pos = -3; pos < ((int64_t)a.max_pages << a.page_shift) + 3; ++pos) {
        const int p = page_of(a, c.slot, pos);
        int want = -1;
        if (c.slot >= 0 && pos >= 0 && pos / (1 << a.page_shift) < a.max_pages) {
          want = table[c.slot * a.table_stride + pos / (1 << a.page_shift)];
          if (want < 0 || want >= a.pages) want = -1;
        }
        CHECK(p == want);
        if (p >= 0) CHECK(token_offset(a, p, pos) == (int64_t)p * 4096 + pos % (1 << a.page_shift) * 64);
        ++cases;
      }
    }
    if (wild) continue;
    // tiles: every sequence's rows lie in its own tiles, and all tiles exist
    for (int group : {1, 3, 4, 7, 16}) {
      for (int rows : {16, 32, 64, 128}) {
        const int total = starts[a.seqs];
        for (int i = 0; i < a.seqs; ++i) {
          const int n = starts[i + 1] - starts[i];
          const int64_t own = ((int64_t)n * group + rows - 1) / rows, base = tile_base(starts[i], group, rows, i);
          const int64_t next = i + 1 < a.seqs ? tile_base(starts[i + 1], group, rows, i + 1)
                                              : tile_count(total, group, rows, a.seqs);
          CHECK(base + own <= next && next > base);
          ++cases;
        }
      }
    }
  }
  std::printf("ok %ld\n", cases);
  return 0;
}
