// Host-side check of the bounded cache's selection (compiled with g++ by
// tests/test_select_bounds.py; no GPU), through the functions the kernel uses
// (csrc/sbq_index.h): how many keys it sets apart in its kCand words.
//
//   select_check N RECENT [unmasked]
//
// N slots, RECENT of which are among the newest positions, lowest slots first;
// the wanted first digit is theirs.  It is counted kChunk slots at a time,
// slots past the end among the newest, as the launch before the selection
// counts it; the keys are then set apart by every thread.  "unmasked" sets the
// slots past the end apart too.  Prints the two numbers and fails where the
// second passes kCand.
#include <cstdio>
#include <cstdlib>

#include "sbq_index.h"

using namespace sbq;

int main(int argc, char** argv) {
  const long long n = std::atoll(argv[1]), recent = std::atoll(argv[2]);
  const bool masked = argc < 4;
  const int per = 1 << keys_log(n);
  const long long segs = (n + (long long)per * kSelThreads - 1) / ((long long)per * kSelThreads);
  auto newest = [&](long long s) { return s < recent || s >= n; };
  long long counted = 0, apart = 0;
  for (long long s = 0; s < (n + kChunk - 1) / kChunk * kChunk; ++s) counted += newest(s);
  if (segs == 1 && counted <= kCand)
    for (int t = 0; t < kSelThreads; ++t) {
      const long long s0 = (long long)t * per;
      uint32_t mine = 0;
      for (int i = 0; i < per; ++i) mine |= (uint32_t)newest(s0 + i) << i;
      if (masked) mine &= slot_mask(n, s0);
      apart += __builtin_popcount(mine);
    }
  std::printf("%lld %lld\n", counted, apart);
  return apart > kCand;
}
