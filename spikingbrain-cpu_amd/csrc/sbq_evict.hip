// sbq_evict.hip - a bounded cache of keys and values that gives up the slots
// which received the least attention.
//
// Slots are ordered by one 32-bit key: free ones 0, then the running sum of
// attention weight as an ordered integer, the `recent` newest positions
// highest; equal keys by slot.  One workgroup finds the m-th smallest key
// digit by digit (11, 11 and 10 bits, a histogram each) and lists the slots on
// one side of it in slot order.  The keys stay in LDS (up to 32768 slots; more
// are read again for every pass), each thread's own ones side by side, so that
// one scan over the threads gives every place in the list; the few keys that
// share the first digit are set apart for the other two passes.  A single new
// token needs no more than the smallest key and its slot.
//
// What bounds it is the latency of the steps of one workgroup, so from 8192
// slots on a launch before it spreads the reading: for an append every
// workgroup leaves the T first of its 4096 slots (which hold the T first of
// all), for a take the 4-byte keys and their first digits' counts.  One token
// into 4096 slots of 8 x 128: 3.9 us; 12 into 32768: 11 us, 4.8 for the choice
// among theirs and 3 for the rows; 4096 of 32768 slots taken: 4, 23 and 7 us.
// Integer counts only, so the result does not depend on timing.
#include "sbq_common.h"
#include "sbq_index.h"
#include "sbq_launch.h"

namespace sbq {

namespace {

constexpr int kSelWaves = kSelThreads / 64, kBins = 2048;

// The order in which slots are given up.
__device__ __forceinline__ uint32_t evict_key(int64_t pos, float weight, int64_t keep_from) {
  if (pos < 0) return 0u;                // free
  if (pos >= keep_from) return ~0u;      // one of the newest
  if (weight != weight) return 0xff900000u;
  const uint32_t b = __float_as_uint(weight + 0.0f);  // (-0 is 0)
  return b >> 31 ? ~b : b | 0x80000000u;  // 0x007fffff (-inf) .. 0xff800000 (+inf)
}

// Exclusive prefix sums of kSelThreads values in thread order; `total` too.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* lds, uint32_t* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  uint32_t sum = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t t = __shfl_up(sum, o, 64);
    if (lane >= o) sum += t;
  }
  __syncthreads();  // (lds is free)
  if (lane == 63) lds[w] = sum;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int k = 0; k < kSelWaves; ++k) {
    const uint32_t t = lds[k];
    before += k < w ? t : 0u;
    all += t;
  }
  *total = all;
  return before + sum - v;
}

struct Select {
  const int64_t* slot_pos;
  const float* weight;
  int n;
  int64_t keep_from;
  const uint32_t* ready;  // not null: the keys themselves
  const uint32_t* first;  // not null: their first digits' counts, kBins for each kChunk slots
};

// A thread's `per` (4, 8, 16 or 32) keys of a segment of per * 1024 slots lie
// side by side in LDS, their 16-byte pieces permuted by the thread (else the
// threads' reads would all meet in the same banks).
// Place of key i of thread t, `per` = 1 << log.
__device__ __forceinline__ int key_at(int t, int i, int log) {
  return (t << log) + ((((i >> 2) ^ t) & ((1 << log) / 4 - 1)) << 2 | (i & 3));
}
__device__ __forceinline__ u32x4 own_keys(const uint32_t* keys, int log, int i) {
  return *(const u32x4*)(keys + key_at(threadIdx.x, i, log));
}

__device__ __forceinline__ void count_digit(uint32_t* hist, uint32_t digit) {
  // (a wave whose keys share the digit, as equal weights do, counts once)
  const uint32_t first = __builtin_amdgcn_readfirstlane(digit);
  const unsigned long long on = __ballot(true);
  if (__ballot(digit == first) == on) {
    if ((threadIdx.x & 63) == (unsigned)__ffsll(on) - 1) atomicAdd(&hist[first], (uint32_t)__popcll(on));
  } else {
    atomicAdd(&hist[digit], 1u);
  }
}

// Keys of segment `seg` into LDS, their first digits counted where hist is
// given.  Slots past the end get the largest key: with m <= n they come after
// every slot that is wanted.
// All loads of a step are issued before the first is looked at, with no branch
// between them.
template <bool READY, int U>
__device__ __forceinline__ void load_keys(const Select& q, int64_t seg, int log, uint32_t* keys, uint32_t* hist) {
  const int per = 1 << log;
  const int64_t s0 = seg * per * kSelThreads;
#pragma unroll 1
  for (int i = 0; i < per; i += U) {
    int64_t pos[U];
    float w[U];
    uint32_t key[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int64_t s = s0 + (i + j) * kSelThreads + threadIdx.x, at = s < q.n ? s : q.n - 1;
      if constexpr (READY) {
        key[j] = q.ready[at];
      } else {
        pos[j] = q.slot_pos[at];
        w[j] = q.weight[at];
      }
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int s = (i + j) * kSelThreads + threadIdx.x;
      if constexpr (!READY) key[j] = evict_key(pos[j], w[j], q.keep_from);
      const uint32_t k = s0 + s >= q.n ? ~0u : key[j];
      keys[key_at(s >> log, s & (per - 1), log)] = k;
      if (hist) count_digit(hist, k >> 21);
    }
  }
}

__device__ __forceinline__ void load_keys(const Select& q, int64_t seg, int log, uint32_t* keys, uint32_t* hist) {
  if (q.ready)
    log >= 3 ? load_keys<true, 8>(q, seg, log, keys, hist) : load_keys<true, 4>(q, seg, log, keys, hist);
  else
    log >= 3 ? load_keys<false, 8>(q, seg, log, keys, hist) : load_keys<false, 4>(q, seg, log, keys, hist);
}

// The slots with the m smallest keys (side 0) or the used ones among the
// others (side 1), listed in slot order; returns how many (0 <= m <= n).
__device__ __forceinline__ int select_slots(const Select& q, int m, int side, int32_t* list) {
  extern __shared__ __align__(16) uint32_t keys[];
  __shared__ uint32_t hist[kBins], cand[kCand], scan[kSelWaves], found[3], ncand;
  const int log = keys_log(q.n), per = 1 << log;
  const int segs = (int)(((int64_t)q.n + per * kSelThreads - 1) >> (log + 10));
  // (the counts are under way while the keys are read)
  const int chunks = (int)(((int64_t)q.n + kChunk - 1) / kChunk);
  u32x2 first[8];
  if (m > 0 && q.first) {
#pragma unroll
    for (int c = 0; c < 8; ++c)
      first[c] = *(const u32x2*)(q.first + (int64_t)min(c, chunks - 1) * kBins + 2 * threadIdx.x);
  }
  for (int i = threadIdx.x; i < kBins; i += kSelThreads) hist[i] = 0;
  if (threadIdx.x == 0) ncand = 0;
  __syncthreads();
  for (int seg = 0; seg < segs; ++seg) {
    if (segs > 1 && (m == 0 || q.first)) break;  // (read where they are wanted, counted already)
    load_keys(q, seg, log, keys, m > 0 && !q.first ? hist : nullptr);
    if (segs > 1) __syncthreads();
  }
  if (m > 0 && q.first) {
    u32x2 sum = (u32x2)(0u);
#pragma unroll
    for (int c = 0; c < 8; ++c) sum += c < chunks ? first[c] : (u32x2)(0u);
#pragma unroll 4
    for (int c = 8; c < chunks; ++c) sum += *(const u32x2*)(q.first + (int64_t)c * kBins + 2 * threadIdx.x);
    hist[2 * threadIdx.x] = sum.x;
    hist[2 * threadIdx.x + 1] = sum.y;
  }
  __syncthreads();

  // the m-th smallest key `kth`, of which `ties` (lowest slots first) belong to the m
  uint32_t kth = 0, ties = m;
  if (m > 0) {
    bool few = false;  // the keys that share the first digit are in `cand`
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
      const uint32_t above = pass == 0 ? 0u : ~0u << (shift + bits);
      if (pass > 0) {
        for (int i = threadIdx.x; i < kBins; i += kSelThreads) hist[i] = 0;
        __syncthreads();
        if (few) {
          for (unsigned i = threadIdx.x; i < ncand; i += kSelThreads) {
            const uint32_t k = cand[i];
            if (((k ^ kth) & above) == 0) count_digit(hist, k >> shift & ((1u << bits) - 1));
          }
        } else {
#pragma unroll 1
          for (int seg = 0; seg < segs; ++seg) {
            if (segs > 1) {
              load_keys(q, seg, log, keys, nullptr);
              __syncthreads();
            }
#pragma unroll 1
            for (int i = 0; i < per; i += 4) {
              const u32x4 k4 = own_keys(keys, log, i);
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (((k4[j] ^ kth) & above) == 0) count_digit(hist, k4[j] >> shift & ((1u << bits) - 1));
            }
            if (segs > 1) __syncthreads();
          }
        }
        __syncthreads();
      }
      const uint32_t a = hist[2 * threadIdx.x], b = hist[2 * threadIdx.x + 1];
      uint32_t total;
      const uint32_t before = block_scan(a + b, scan, &total);
      if (before < ties && ties <= before + a) found[0] = 2 * threadIdx.x, found[1] = before, found[2] = a;
      if (before + a < ties && ties <= before + a + b)
        found[0] = 2 * threadIdx.x + 1, found[1] = before + a, found[2] = b;
      __syncthreads();
      kth |= found[0] << shift;
      ties -= found[1];
      if (pass == 0 && segs == 1 && found[2] <= kCand) {
        few = true;
        uint32_t mine = 0;  // one bit per own key
#pragma unroll 1
        for (int i = 0; i < per; i += 4) {
          const u32x4 k4 = own_keys(keys, log, i);
#pragma unroll
          for (int j = 0; j < 4; ++j) mine |= (uint32_t)(k4[j] >> 21 == found[0]) << (i + j);
        }
        mine &= slot_mask(q.n, (int64_t)threadIdx.x * per);  // (those past the end are not all in found[2])
        uint32_t at = mine ? atomicAdd(&ncand, (uint32_t)__popc(mine)) : 0u;
        for (; mine; mine &= mine - 1) cand[at++] = keys[key_at(threadIdx.x, __ffs(mine) - 1, log)];
      }
      __syncthreads();
    }
  }

  // Of the keys equal to kth the first `ties` are among the m; free slots
  // (key 0) are never among the used ones.  Before a thread's own slots lie
  // `out` keys strictly on the wanted side and `eq` equal ones.
  uint32_t out = 0, eq = 0;
  auto listed = [&](uint32_t strictly, uint32_t equal) {  // entries that so many keys make
    const uint32_t low = min(equal, ties);
    return strictly + (side == 0 ? low : kth == 0 ? 0u : equal - low);
  };
#pragma unroll 1
  for (int seg = 0; seg < segs; ++seg) {
    if (segs > 1) {
      load_keys(q, seg, log, keys, nullptr);
      __syncthreads();
    }
    const int64_t s0 = ((int64_t)seg * kSelThreads + threadIdx.x) * per;
    uint32_t strict = 0, same = 0;  // one bit per own key
#pragma unroll 1
    for (int i = 0; i < per; i += 4) {
      const u32x4 k4 = own_keys(keys, log, i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        strict |= (uint32_t)(side == 0 ? k4[j] < kth : k4[j] > kth) << (i + j);
        same |= (uint32_t)(k4[j] == kth) << (i + j);
      }
    }
    const uint32_t in = slot_mask(q.n, s0);
    strict &= in;
    same &= in;
    uint32_t all_out, all_eq;
    const uint32_t out0 = out + block_scan(__popc(strict), scan, &all_out);
    const uint32_t eq0 = eq + block_scan(__popc(same), scan, &all_eq);
    const uint32_t low0 = min(eq0, ties);
    const uint32_t mine = min(eq0 + (uint32_t)__popc(same), ties) - low0;  // own equal ones among the m
    // The segment's entries gather in LDS (its keys are done with) and leave from there in whole lines:
    // a thread's own run stored from here took 64 lines a wave.
    const uint32_t base = listed(out, eq);
    uint32_t place = out0 + (side == 0 ? low0 : kth == 0 ? 0u : eq0 - low0) - base;
    uint32_t skip = mine, todo = strict | same;
    while (todo) {
      const uint32_t bit = todo & (0u - todo);
      todo ^= bit;
      bool take = strict & bit;
      if (!take) {
        take = side == 0 ? skip > 0 : skip == 0 && kth != 0;
        skip -= skip > 0;
      }
      if (take) keys[place++] = (uint32_t)(s0 + __ffs(bit) - 1);
    }
    out += all_out;
    eq += all_eq;
    __syncthreads();
    const uint32_t n = listed(out, eq) - base;
    for (uint32_t i = threadIdx.x; i < n; i += kSelThreads) list[base + i] = (int32_t)keys[i];
    if (segs > 1) __syncthreads();
  }
  return (int)listed(out, eq);
}

// The m first of up to kRank ready keys, listed in order: each thread counts
// the keys before its own, then the chosen ones before it (64 candidates: some
// 1 us where the digits' passes over as few take 12).
constexpr int kRank = 256;
__device__ __forceinline__ void rank_slots(const uint32_t* ready, int n, int m, int32_t* list) {
  __shared__ __align__(16) uint32_t key[kRank];
  __shared__ unsigned long long chosen[kRank / 64];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  uint32_t k = ~0u;
  if (t < kRank) key[t] = k = t < n ? ready[t] : ~0u;
  __syncthreads();
  int before = 0;
  if (t < kRank) {
    for (int i = 0; i < n; i += 4) {
      const u32x4 k4 = *(const u32x4*)(key + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) before += k4[j] < k || (k4[j] == k && i + j < t);
    }
    const unsigned long long on = __ballot(t < n && before < m);
    if (lane == 0) chosen[w] = on;
  }
  __syncthreads();
  if (t < n && before < m) {
    int place = __popcll(chosen[w] & ((1ull << lane) - 1));
    for (int i = 0; i < w; ++i) place += __popcll(chosen[i]);
    list[place] = t;
  }
}

// The slot of the smallest key (the lowest of equal ones).
__device__ __forceinline__ int first_slot(const Select& q) {
  __shared__ unsigned long long best[kSelWaves];
  unsigned long long v = ~0ull;
#pragma unroll 1
  for (int64_t s0 = threadIdx.x; s0 < q.n; s0 += 4 * kSelThreads) {
    int64_t pos[4];
    float w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t s = s0 + j * kSelThreads, at = s < q.n ? s : s0;
      pos[j] = q.slot_pos[at];
      w[j] = q.weight[at];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t s = s0 + j * kSelThreads;
      const unsigned long long k = (unsigned long long)evict_key(pos[j], w[j], q.keep_from) << 32 | (uint32_t)s;
      if (s < q.n && k < v) v = k;
    }
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned long long t = __shfl_xor(v, o, 64);
    v = t < v ? t : v;
  }
  if ((threadIdx.x & 63) == 0) best[threadIdx.x >> 6] = v;
  __syncthreads();
  v = best[0];
#pragma unroll
  for (int k = 1; k < kSelWaves; ++k) v = best[k] < v ? best[k] : v;
  return (int)(uint32_t)v;
}

// n elements of a row from type ST to type DT; equal types copy bits.
template <int ST, int DT>
__device__ __forceinline__ void copy_elem(void* to, int64_t ti, const void* from, int64_t fi) {
  typedef typename XElem<ST>::T S;
  typedef typename XElem<DT>::T D;
  if constexpr (ST == DT)
    ((D*)to)[ti] = ((const S*)from)[fi];
  else
    ((D*)to)[ti] = (D)(float)((const S*)from)[fi];
}

struct Rows {  // keys and values [n][heads][dim], strides in elements
  void *k, *v;
  int64_t ss, sh;
};

// Elements [e0, e1) step `step` of token row `from` of src to slot `to` of
// dst, keys and values; an element e is (head e / D, column e % D).
template <int ST, int DT>
__device__ __forceinline__ void copy_row(const Rows& src, int64_t from, const Rows& dst, int64_t to, int D, int e0, int e1,
                                         int step) {
  for (int e = e0; e < e1; e += step) {
    const int64_t h = e / D, d = e % D;
    const int64_t fi = from * src.ss + h * src.sh + d, ti = to * dst.ss + h * dst.sh + d;
    copy_elem<ST, DT>(dst.k, ti, src.k, fi);
    copy_elem<ST, DT>(dst.v, ti, src.v, fi);
  }
}

// 16 bytes at a time (equal types, aligned rows): `per` pieces a head, the
// keys' before the values' over the threads.
__device__ __forceinline__ void copy_row16(const Rows& src, int64_t from, const Rows& dst, int64_t to, int per, int es,
                                           int heads) {
  const int half = heads * per;
  for (int e = threadIdx.x; e < 2 * half; e += blockDim.x) {
    const bool val = e >= half;
    const int u = val ? e - half : e;
    const int64_t h = u / per, d = u % per * (16 / es);
    const int64_t fi = (from * src.ss + h * src.sh + d) * es, ti = (to * dst.ss + h * dst.sh + d) * es;
    *(u32x4*)((uint8_t*)(val ? dst.v : dst.k) + ti) = *(const u32x4*)((const uint8_t*)(val ? src.v : src.k) + fi);
  }
}

struct AppendArgs {
  int64_t* slot_pos;
  float* weight;
  int64_t* end;
  const int64_t* start;
  Rows cache, fresh;
  int32_t* list;
  uint32_t* cand_key;  // with several workgroups: the T first of each one's slots
  int32_t* cand_slot;
  int n, T, Hk, D;
  int64_t recent;
  bool rows_too;
};

// A single token, then several.
template <int ST, int DT>
__global__ __launch_bounds__(kSelThreads) void kv_append_one_kernel(AppendArgs a) {
  const int64_t start = *a.start;
  const Select q{a.slot_pos, a.weight, a.n, start + 1 - a.recent, nullptr, nullptr};
  const int s = first_slot(q);  // (every thread has read its slots and *start)
  if (threadIdx.x == 0) {
    a.slot_pos[s] = start;
    a.weight[s] = 0.0f;
    *a.end = start + 1;
  }
  copy_row<ST, DT>(a.fresh, 0, a.cache, s, a.D, threadIdx.x, a.Hk * a.D, kSelThreads);
}

// The T first of every kChunk slots, in slot order, with their keys.
constexpr int kSpreadFrom = 2 * kChunk, kSpreadTokens = kChunk / 8;
__global__ __launch_bounds__(kSelThreads) void kv_first_kernel(AppendArgs a) {
  const int s0 = blockIdx.x * kChunk, n = min(kChunk, a.n - s0), m = min(a.T, n);
  const Select q{a.slot_pos + s0, a.weight + s0, n, *a.start + a.T - a.recent, nullptr, nullptr};
  int32_t* const list = a.cand_slot + (int64_t)blockIdx.x * a.T;
  select_slots(q, m, 0, list);
  __syncthreads();  // the list is written
  for (int i = threadIdx.x; i < m; i += kSelThreads) {
    const int s = list[i];
    a.cand_key[(int64_t)blockIdx.x * a.T + i] = evict_key(q.slot_pos[s], q.weight[s], q.keep_from);
    list[i] = s0 + s;
  }
}

template <int ST, int DT>
__global__ __launch_bounds__(kSelThreads) void kv_append_kernel(AppendArgs a) {
  const int64_t start = *a.start;
  const int chunks = (a.n + kChunk - 1) / kChunk;
  Select q{a.slot_pos, a.weight, a.n, start + a.T - a.recent, a.cand_key, nullptr};
  // (only the last workgroup may have had fewer than T slots, so the candidates are dense and in slot order)
  if (a.cand_key) q.n = (chunks - 1) * a.T + min(a.T, a.n - (chunks - 1) * kChunk);
  if (a.cand_key && q.n <= kRank)
    rank_slots(a.cand_key, q.n, a.T, a.list);
  else
    select_slots(q, a.T, 0, a.list);
  __syncthreads();  // the list is written
  for (int i = threadIdx.x; i < a.T; i += kSelThreads) {
    int s = a.list[i];
    if (a.cand_key) a.list[i] = s = a.cand_slot[s];
    a.slot_pos[s] = start + i;
    a.weight[s] = 0.0f;
  }
  if (threadIdx.x == 0) *a.end = start + a.T;
  if (a.rows_too) {
    __syncthreads();  // the list is in slots
    const int row = a.Hk * a.D;
#pragma unroll 4
    for (int e = threadIdx.x; e < a.T * row; e += kSelThreads) {
      const int i = e / row;
      copy_row<ST, DT>(a.fresh, i, a.cache, a.list[i], a.D, e - i * row, e - i * row + 1, 1);
    }
  }
}

template <int ST, int DT>
__global__ __launch_bounds__(256) void kv_rows_kernel(AppendArgs a, int first) {
  const int i = first + (int)blockIdx.x;
  copy_row<ST, DT>(a.fresh, i, a.cache, a.list[i], a.D, threadIdx.x, a.Hk * a.D, 256);
}

struct TakeArgs {
  const int64_t *slot_pos, *end;
  const float* weight;
  int64_t *to_pos, *to_end;
  float* to_weight;
  Rows src, dst;
  int32_t* list;   // [capacity], then the count
  uint32_t *keys, *first;  // [n] and [chunks][kBins] where a launch before the selection computes them
  int n, capacity, Hk, D, es;
  int64_t recent;
  bool vec;
};

// The keys, and how often each first digit occurs in every kChunk slots: few
// bins (the exponents of like weights) take most of the counts, whose atomics
// wait for each other, so they are spread over workgroups and four copies.
__global__ __launch_bounds__(kSelThreads) void kv_keys_kernel(TakeArgs a) {
  __shared__ uint32_t hist[kBins * 4];
  for (int i = threadIdx.x; i < kBins * 4; i += kSelThreads) hist[i] = 0;
  const int64_t s0 = (int64_t)blockIdx.x * kChunk + threadIdx.x, keep_from = *a.end - a.recent;
  int64_t pos[4];
  float w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t s = s0 + j * kSelThreads, at = s < a.n ? s : a.n - 1;
    pos[j] = a.slot_pos[at];
    w[j] = a.weight[at];
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t s = s0 + j * kSelThreads;
    const uint32_t k = s < a.n ? evict_key(pos[j], w[j], keep_from) : ~0u;  // (as the selection counts the missing ones)
    if (s < a.n) a.keys[s] = k;
    atomicAdd(&hist[(k >> 21) * 4 + (threadIdx.x & 3)], 1u);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += kSelThreads) {
    const u32x4 h = *(const u32x4*)(hist + 4 * i);
    a.first[(int64_t)blockIdx.x * kBins + i] = h.x + h.y + h.z + h.w;
  }
}

__global__ __launch_bounds__(kSelThreads) void kv_take_kernel(TakeArgs a) {
  const int64_t end = *a.end;
  const Select q{a.slot_pos, a.weight, a.n, end - a.recent, a.keys, a.first};
  const int kept = select_slots(q, a.n > a.capacity ? a.n - a.capacity : 0, 1, a.list);
  if (threadIdx.x == 0) {
    a.list[a.capacity] = kept;
    *a.to_end = end;
  }
}

__global__ __launch_bounds__(256) void kv_take_rows_kernel(TakeArgs a, int first) {
  const int i = first + (int)blockIdx.x;
  if (i >= a.list[a.capacity]) {
    if (threadIdx.x == 0) {
      a.to_pos[i] = -1;
      a.to_weight[i] = 0.0f;
    }
    return;
  }
  const int s = a.list[i];
  if (threadIdx.x == 0) {
    a.to_pos[i] = a.slot_pos[s];
    a.to_weight[i] = a.weight[s];
  }
  if (a.vec) {
    copy_row16(a.src, s, a.dst, i, a.D * a.es / 16, a.es, a.Hk);
  } else if (a.es == 4) {
    copy_row<XT_F32, XT_F32>(a.src, s, a.dst, i, a.D, threadIdx.x, a.Hk * a.D, 256);
  } else {
    copy_row<XT_F16, XT_F16>(a.src, s, a.dst, i, a.D, threadIdx.x, a.Hk * a.D, 256);
  }
}

constexpr int64_t kRowsStep = kLaunchThreads / 256;  // rows per launch
constexpr int kInlineElems = 1 << 12;  // key elements that the selecting workgroup still writes itself

template <int ST, int DT>
int append_types(const AppendArgs& a, hipStream_t st) {
  if (a.T == 1) {
    kv_append_one_kernel<ST, DT><<<1, kSelThreads, 0, st>>>(a);
    return check_launch();
  }
  int rc = 0;
  int64_t n = a.n;
  if (a.cand_key) {
    const int chunks = (a.n + kChunk - 1) / kChunk;
    kv_first_kernel<<<chunks, kSelThreads, (size_t)(kSelThreads * 4) << keys_log(kChunk), st>>>(a);
    if ((rc = check_launch())) return rc;
    n = (int64_t)chunks * a.T;
  }
  kv_append_kernel<ST, DT><<<1, kSelThreads, (size_t)(kSelThreads * 4) << keys_log(n), st>>>(a);
  rc = check_launch();
  if (a.rows_too) return rc;
  for (int64_t i = 0; i < a.T && !rc; i += kRowsStep) {
    kv_rows_kernel<ST, DT><<<(unsigned)(a.T - i < kRowsStep ? a.T - i : kRowsStep), 256, 0, st>>>(a, (int)i);
    rc = check_launch();
  }
  return rc;
}

template <int ST>
int append_from(const AppendArgs& a, int ct, hipStream_t st) {
  return ct == XT_F32 ? append_types<ST, XT_F32>(a, st) : ct == XT_F16 ? append_types<ST, XT_F16>(a, st)
                                                                        : append_types<ST, XT_BF16>(a, st);
}

}  // namespace

// The list (one count more), then the candidates of an append or the counts and keys of a take.
int64_t list_words(int64_t count) { return (count + 1 + 3) / 4 * 4; }
int64_t kv_workspace_bytes(int64_t slots, int64_t count) {
  if (slots < kSpreadFrom) return 4 * (count + 1);
  return 4 * (list_words(count) + slots + (slots + kChunk - 1) / kChunk * kBins);
}
static_assert(kSpreadTokens * 8 <= kChunk && 2 * kSpreadTokens * 8 <= 3 * kSpreadFrom, "candidates fit 4 bytes a slot");

int launch_kv_append(const KvAppend& c, hipStream_t st) {
  AppendArgs a{c.slot_pos, c.weight, c.end, c.start, Rows{c.k, c.v, c.k_ss, c.k_sh},
               Rows{const_cast<void*>(c.kn), const_cast<void*>(c.vn), c.n_ss, c.n_sh}, (int32_t*)c.ws, nullptr, nullptr,
               (int)c.slots, (int)c.T, (int)c.Hk, (int)c.D, c.recent, c.T * c.Hk * c.D <= kInlineElems};
  if (c.slots >= kSpreadFrom && c.T > 1 && c.T <= kSpreadTokens) {  // candidates: at most n bytes, and one chunk's
    a.cand_slot = a.list + c.T;
    a.cand_key = (uint32_t*)(a.cand_slot + (c.slots + kChunk - 1) / kChunk * c.T);
  }
  return c.nt == XT_F32 ? append_from<XT_F32>(a, c.ct, st) : c.nt == XT_F16 ? append_from<XT_F16>(a, c.ct, st)
                                                                             : append_from<XT_BF16>(a, c.ct, st);
}

int launch_kv_take(const KvTake& c, hipStream_t st) {
  const int es = c.ct == XT_F32 ? 4 : 2;
  auto ok = [&](const void* p, int64_t ss, int64_t sh) { return (uintptr_t)p % 16 == 0 && ss * es % 16 == 0 && sh * es % 16 == 0; };
  const bool vec = c.D * es % 16 == 0 && ok(c.k, c.k_ss, c.k_sh) && ok(c.v, c.k_ss, c.k_sh) && ok(c.to_k, c.t_ss, c.t_sh) &&
                   ok(c.to_v, c.t_ss, c.t_sh);
  uint32_t* const more = (uint32_t*)c.ws + list_words(c.capacity);
  const bool spread = c.slots >= kSpreadFrom;
  TakeArgs a{c.slot_pos, c.end, c.weight, c.to_pos, c.to_end, c.to_weight,
             Rows{const_cast<void*>(c.k), const_cast<void*>(c.v), c.k_ss, c.k_sh}, Rows{c.to_k, c.to_v, c.t_ss, c.t_sh},
             (int32_t*)c.ws, spread ? more + (c.slots + kChunk - 1) / kChunk * kBins : nullptr, spread ? more : nullptr,
             (int)c.slots, (int)c.capacity, (int)c.Hk, (int)c.D, es, c.recent, vec};
  if (a.keys) {
    kv_keys_kernel<<<(a.n + kChunk - 1) / kChunk, kSelThreads, 0, st>>>(a);
    const int rc = check_launch();
    if (rc) return rc;
  }
  kv_take_kernel<<<1, kSelThreads, (size_t)(kSelThreads * 4) << keys_log(a.n), st>>>(a);
  int rc = check_launch();
  for (int64_t i = 0; i < a.capacity && !rc; i += kRowsStep) {
    kv_take_rows_kernel<<<(unsigned)(a.capacity - i < kRowsStep ? a.capacity - i : kRowsStep), 256, 0, st>>>(a, (int)i);
    rc = check_launch();
  }
  return rc;
}

}  // namespace sbq
