// sbq_index.h - index arithmetic of the kernels that a host-side bounds check
// also compiles (plain C++: no HIP types or builtins here).  Each function maps
// a work item to the element or byte range it reads or writes; the kernels use
// these functions, and tests/bounds_check.cpp walks every work item of a
// launch through them with g++ and checks the ranges against the buffers.
#pragma once
#include <stdint.h>

#if defined(__HIPCC__)
#define SBQ_HD __host__ __device__ __forceinline__
#else
#define SBQ_HD inline
#endif

namespace sbq {

// Activation quantizer, vector path (K % 16 == 0, Kp = ceil(K / 64) * 64):
// 16-element chunk c of x [M, K] (row stride ldx), cpr = Kp / 16 chunks per
// row.  Returns the element offset of the first of the 16 values loaded.
// Chunks in the padding columns K..Kp-1 load the row's last chunk (their
// values are never used), so no load leaves the row.
SBQ_HD int64_t act_chunk_src(int64_t c, int cpr, int K, int64_t ldx) {
  const int64_t m = c / cpr;
  const int k0 = (int)(c - m * cpr) * 16;
  return m * ldx + (k0 < K - 16 ? k0 : K - 16);
}

// Greedy-token key of output value v at column n (fused argmax of the decode
// GEMV).  The unsigned 64-bit order of keys is torch.argmax's order of
// (value, index): NaN above every number, -0 equal to +0, and among equal
// values the smaller index.  Key 0 is below every key (no candidate).
SBQ_HD unsigned long long argmax_key(float v, int n) {
  uint32_t u = __builtin_bit_cast(uint32_t, v);
  if (v != v) {
    u = 0xffffffffu;
  } else if (v == 0.0f) {
    u = 0x80000000u;  // -0 and +0 alike
  } else {
    u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  }
  return ((unsigned long long)u << 32) | (unsigned long long)(0xffffffffu - (uint32_t)n);
}

// Workgroups b < nblk with b % slots == slot (the fused argmax's members of
// one slot), and the number of slots that have any.
SBQ_HD unsigned argmax_slot_members(unsigned nblk, unsigned slot, unsigned slots) {
  return slot < nblk ? (nblk - slot + slots - 1) / slots : 0u;
}
SBQ_HD unsigned argmax_slots_used(unsigned nblk, unsigned slots) { return nblk < slots ? nblk : slots; }

// Outputs stored as parts: the columns of y [M, N] belong to consecutive parts
// (widths multiples of 4), and part p is a dense [M, width] matrix that starts
// at element M * pstart, pstart the part's first column with every earlier
// width rounded up to 64 columns (so parts start 64 elements apart at least,
// aligned for vector stores).  The table holds two words per 4 columns: the
// part's width, and start / 4 | ((pstart - start) / 4) << kPartPadShift.
// Element offset of column n = of the part holding it: part_base + m * width + n.
constexpr int kPartPadShift = 20;
SBQ_HD int64_t part_base(uint32_t word, int64_t M) {
  const int64_t start = (int64_t)(word & ((1u << kPartPadShift) - 1u)) * 4;
  const int64_t pstart = start + (int64_t)(word >> kPartPadShift) * 4;
  return M * pstart - start;
}

// The bounded cache's selection (sbq_evict.hip) by one workgroup: a thread holds
// 1 << keys_log(n) slots side by side, of segments of as many per thread; slots
// past the last one are keys too, larger than any other.  Keys that share the
// wanted first digit are set apart in kCand words where no more are counted, in
// numbers that a launch before the selection may have taken kChunk slots at a
// time, so that the two see different numbers of slots past the last one: only
// those of slot_mask are set apart.
constexpr int kSelThreads = 1024, kSegKeys = 32, kCand = 2048;
constexpr int kChunk = 4 * kSelThreads;  // slots that one workgroup of a launch before the selection looks at
SBQ_HD constexpr int keys_log(int64_t n) {
  int log = 2;
  while (1 << log < kSegKeys && ((int64_t)kSelThreads << log) < n) ++log;
  return log;
}
// Which of a thread's slots, s0 and up to 31 after it, there are (n in all); one bit each.
SBQ_HD uint32_t slot_mask(int64_t n, int64_t s0) {
  return n - s0 >= 32 ? ~0u : n <= s0 ? 0u : (1u << (n - s0)) - 1u;
}

// The paged cache (sbq_paged.h): the row of position pos and head h in the pool,
// pages of 1 << page_log positions of every one of Hk heads; -1 for an id that
// is no page of the pool.
SBQ_HD int64_t paged_row_of(int32_t id, int64_t pages, int64_t pos, int h, int Hk, int page_log) {
  if (id < 0 || id >= pages) return -1;
  return (((int64_t)id * Hk + h) << page_log) + (pos & ((1 << page_log) - 1));
}

// How its attention cuts a launch's sequences into parts, one for each of `slots`
// workgroups of kPagedWaves waves: a sequence counts its blocks in whole rounds of the
// waves, one round at least (a sequence that sees nothing writes its zeros); a
// part is `each` of all those; slot s's piece of sequence b are blocks n0..n1-1 of it.
constexpr int kPagedWaves = 4;
SBQ_HD int paged_own(int blocks) {
  const int n = (blocks + kPagedWaves - 1) / kPagedWaves * kPagedWaves;
  return n < kPagedWaves ? kPagedWaves : n;
}
SBQ_HD int paged_each(int total, int slots, float per_slot) {  // per_slot: 1 / slots
  int n = (int)((float)total * per_slot);
  while (n > 0 && (int64_t)(n - 1) * slots >= total) --n;
  while ((int64_t)n * slots < total) ++n;
  return n < kPagedWaves ? kPagedWaves : n;
}
// A sequence's blocks in whole parts: then no part holds two sequences, if the slots suffice.
SBQ_HD int paged_padded(int own, int each) { return (int)(((unsigned)own + (unsigned)each - 1u) / (unsigned)each) * each; }
SBQ_HD void paged_piece(int slot, int each, int before, int blocks, int& n0, int& n1) {  // (none: n0 >= n1)
  const int64_t x0 = (int64_t)slot * each;
  const int own = blocks > 1 ? blocks : 1;
  n0 = x0 > before ? (int)(x0 - before) : 0;
  n1 = x0 + each - before < own ? (int)(x0 + each - before) : own;
}
SBQ_HD int paged_places(int b, int each, int before, int blocks, int& first) {  // slots with a piece of it, from first - b on
  const unsigned s0 = (unsigned)before / (unsigned)each, s1 = (unsigned)(before + (blocks > 1 ? blocks : 1) - 1) / (unsigned)each;
  first = (int)s0 + b;
  return (int)(s1 - s0) + 1;
}

// Where a slot leaves the partial result of a sequence in several parts, whose first one
// is slot `first`'s: two places a slot, for the sequence that its part goes on with and
// the one that its part ends with and the next goes on with.
SBQ_HD int paged_part_place(int slot, int first) { return 2 * slot + (slot == first); }

// Column index of a key from argmax_key.
SBQ_HD int argmax_key_index(unsigned long long key) { return (int)(0xffffffffu - (uint32_t)key); }

}  // namespace sbq
