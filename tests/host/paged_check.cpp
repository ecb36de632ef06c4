// Walks the paged cache's index arithmetic (csrc/sbq_index.h) on the host: the
// rows of the pool that positions lead to, and how the attention cuts random
// sequences into workgroups' parts.  Prints "ok" or the first failure.
#include <stdint.h>
#include <stdio.h>

#include <random>
#include <vector>

#include "sbq_index.h"

using namespace sbq;

static int fail(const char* what, long a = 0, long b = 0, long c = 0) {
  printf("%s %ld %ld %ld\n", what, a, b, c);
  return 1;
}

int main() {
  std::mt19937_64 rng(7);
  auto below = [&](int64_t n) { return (int64_t)(rng() % (uint64_t)n); };

  // rows: inside the pool for its pages, none for anything else, and no two alike
  for (int round = 0; round < 200; ++round) {
    const int log = 4 + (int)below(7), Hk = 1 + (int)below(9);
    const int64_t pages = 1 + below(6), rows = pages * Hk << log;
    std::vector<char> hit(rows);
    for (int32_t id = 0; id < pages; ++id)
      for (int h = 0; h < Hk; ++h)
        for (int64_t pos = 0; pos < 1 << log; ++pos) {
          const int64_t at = paged_row_of(id, pages, pos + (below(1000) << log), h, Hk, log);
          if (at < 0 || at >= rows || hit[at]++) return fail("row", id, h, pos);
        }
    for (int32_t id : {-1, -5, INT32_MIN, INT32_MAX, (int32_t)pages, (int32_t)pages + 1})
      if (paged_row_of(id, pages, below(1 << log), 0, Hk, log) != -1) return fail("bad page", id, pages);
  }
  // (the largest pool)
  if (paged_row_of((1 << 30) - 1, 1 << 30, 1023, 65535, 65536, 10) != ((((int64_t)1 << 30) - 1) * 65536 + 65535) * 1024 + 1023)
    return fail("largest");

  // parts: every block of every sequence in one piece, places apart, and the ones the joining looks at
  for (int round = 0; round < 3000; ++round) {
    const int n = 1 + (int)below(round % 3 ? 20 : 512), slots = 1 + (int)below(round % 2 ? 1024 : 40);
    const float per_slot = 1.0f / (float)slots;
    std::vector<int> blocks(n), before(n), own(n);
    int64_t total = 0;
    const int64_t top = (int64_t)1 << below(round % 5 ? 12 : 20);
    for (int b = 0; b < n; ++b) {
      blocks[b] = (int)below(below(4) ? top + 1 : 3);
      before[b] = (int)total;
      total += own[b] = paged_own(blocks[b]);
      if (paged_own(blocks[b]) < blocks[b] || paged_own(blocks[b]) % kPagedWaves) return fail("own", blocks[b]);
    }
    int each = paged_each((int)total, slots, per_slot);
    if (each < kPagedWaves || (int64_t)each * slots < total) return fail("each", each, slots, total);
    if (each > kPagedWaves && (int64_t)(each - 1) * slots >= total) return fail("each too large", each, slots, total);
    bool padded = false;
    if (n <= slots && round % 4) {  // each sequence from a part of its own on, where the slots suffice
      const int e = (each + 3) / 4 * 4 + 4 * (int)below(3);
      int64_t all = 0;
      for (int b = 0; b < n; ++b) {
        const int p = paged_padded(own[b], e);
        if (p < own[b] || p >= own[b] + e || p % e) return fail("padded", own[b], e, p);
        all += p;
      }
      if (all <= (int64_t)slots * e) {
        padded = true, each = e, total = 0;
        for (int b = 0; b < n; ++b) {
          before[b] = (int)total;
          total += own[b] = paged_padded(own[b], e);
        }
      }
    }
    std::vector<char> used(slots + n), taken(slots);
    for (int b = 0; b < n; ++b) {
      int first, covered = 0;
      const int count = paged_places(b, each, before[b], blocks[b], first);
      if (count < 1 || first < 0 || first + count > slots + n) return fail("places", b, first, count);
      const int s_from = before[b] / each, s_to = (before[b] + own[b] - 1) / each;
      if (s_to >= slots) return fail("slot", s_to, slots);
      for (int s = 0; s < slots; ++s) {
        if (s < s_from - 2 || s > s_to + 2) continue;
        int n0, n1;
        paged_piece(s, each, before[b], blocks[b], n0, n1);
        if (n0 >= n1) continue;
        if (n0 != covered || n1 > (blocks[b] > 1 ? blocks[b] : 1)) return fail("piece", b, n0, n1);
        covered = n1;
        if (taken[s]++ && padded) return fail("two sequences in a part", b, s);
        const int place = s + b;
        if (place < first || place >= first + count || used[place]++) return fail("place", b, s, place);
      }
      if (covered != (blocks[b] > 1 ? blocks[b] : 1)) return fail("covered", b, covered, blocks[b]);
      for (int k = 0; k < count; ++k)
        if (!used[first + k]) return fail("empty place", b, first, k);
    }
  }
  // (the largest totals)
  for (int total : {1 << 30, (1 << 30) - 3, 1, 4, 5})
    for (int slots : {1, 3, 64, 1023, 1024}) {
      const int each = paged_each(total, slots, 1.0f / (float)slots);
      if ((int64_t)each * slots < total || (each > kPagedWaves && (int64_t)(each - 1) * slots >= total)) return fail("each", total, slots, each);
    }
  printf("ok\n");
  return 0;
}
