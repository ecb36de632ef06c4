// Walks the places of the paged attention's partial results (csrc/sbq_index.h) on
// the host, for random sequences cut into slots' parts: every piece of a shared
// sequence at a place of its own, inside the two a slot that the workspace holds,
// and the joining's walk over a sequence's slots meets each of them once.  Prints
// "ok" or the first failure.
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
  std::mt19937_64 rng(11);
  auto below = [&](int64_t n) { return (int64_t)(rng() % (uint64_t)n); };
  int shared = 0;
  for (int round = 0; round < 6000; ++round) {
    const int n = 1 + (int)below(round % 3 ? 20 : 512), slots = 1 + (int)below(round % 2 ? 1024 : 12);
    std::vector<int> blocks(n), before(n), own(n);
    int64_t total = 0;
    const int64_t top = (int64_t)1 << below(round % 5 ? 12 : 20);
    for (int b = 0; b < n; ++b) {
      blocks[b] = (int)below(below(4) ? top + 1 : 3);
      before[b] = (int)total;
      total += own[b] = paged_own(blocks[b]);
    }
    int each = paged_each((int)total, slots, 1.0f / (float)slots);
    if (round % 4 == 0) {  // each sequence from a part of its own on, where the slots suffice
      int64_t all = 0;
      const int e = (each + 3) / 4 * 4;
      for (int b = 0; b < n; ++b) all += paged_padded(own[b], e);
      if (all <= (int64_t)slots * e) {
        each = e, total = 0;
        for (int b = 0; b < n; ++b) {
          before[b] = (int)total;
          total += own[b] = paged_padded(own[b], e);
        }
      }
    }
    std::vector<int> owner(2 * slots, -1);
    for (int b = 0; b < n; ++b) {
      int first;
      const int count = paged_places(b, each, before[b], blocks[b], first);
      const int slot0 = first - b;
      if (count == 1) continue;  // written by its one workgroup
      ++shared;
      int pieces = 0;
      for (int s = slot0 - 1; s <= slot0 + count; ++s) {
        if (s < 0 || s >= slots) {
          if (s >= slot0 && s < slot0 + count) return fail("slot", b, s, slots);
          continue;
        }
        int n0, n1;
        paged_piece(s, each, before[b], blocks[b], n0, n1);
        if (n0 >= n1) {
          if (s >= slot0 && s < slot0 + count) return fail("no piece", b, s);
          continue;
        }
        if (s < slot0 || s >= slot0 + count) return fail("piece outside", b, s);
        if ((n0 == 0) != (s == slot0)) return fail("first piece", b, s, n0);
        const int place = paged_part_place(s, slot0);
        if (place < 0 || place >= 2 * slots) return fail("place", b, s, place);
        if (owner[place] != -1) return fail("two pieces at a place", b, s, place);
        owner[place] = b;
        ++pieces;
      }
      if (pieces != count) return fail("pieces", b, pieces, count);
      for (int k = 0; k < count; ++k)
        if (owner[paged_part_place(slot0 + k, slot0)] != b) return fail("joined", b, k);
    }
  }
  if (shared < 1000) return fail("too few shared sequences", shared);
  printf("ok\n");
  return 0;
}
