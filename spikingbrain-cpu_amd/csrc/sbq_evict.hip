// sbq_evict.hip - a bounded cache of keys and values that gives up the slots
// which received the least attention.
//
// Slots are ordered by one 32-bit key: free ones 0, then the running sum of
// attention weight as an ordered integer, the `recent` newest positions
// highest; equal keys by slot.  One workgroup finds the m-th smallest key
// digit by digit (11, 11 and 10 bits, a histogram each; only keys that share
// the digits so far count) and lists the slots on one side of it in slot
// order.  The keys stay in LDS (up to 32768 slots; more are read again for
// every pass), each thread's own ones side by side, so that one scan over the
// threads gives every place in the list.  A single new token needs no more
// than the smallest key and its slot.  What bounds it is that workgroup's
// reading of 12 bytes per slot and the latency of its steps; a first level
// over several workgroups would cost another launch, which is more than the
// reading up to some 32768 slots.  Integer counts only, so the result does
// not depend on timing.
#include "sbq_common.h"
#include "sbq_launch.h"

namespace sbq {

namespace {

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64, kBins = 2048;

// The order in which slots are given up.
__device__ __forceinline__ uint32_t evict_key(int64_t pos, float weight, int64_t keep_from) {
  if (pos < 0) return 0u;                // free
  if (pos >= keep_from) return ~0u;      // one of the newest
  if (weight != weight) return 0xff900000u;
  const uint32_t b = __float_as_uint(weight);
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
};

// A thread's keys of a segment of per * 1024 slots lie side by side in LDS,
// 4 words of padding after every 32 (a thread's 16-byte reads would all meet
// in the same banks).
constexpr int kSegKeys = 32;  // per thread at most
__device__ __forceinline__ int key_at(int s) { return s + (s >> 5) * 4; }
constexpr int key_words(int per) { return per * kSelThreads / 32 * 36; }
int keys_per_thread(int64_t n) {
  const int64_t k = (n + kSelThreads - 1) / kSelThreads;
  return k > kSegKeys ? kSegKeys : (int)((k + 3) / 4 * 4);
}

// Keys of segment `seg` into LDS (slots past the end: key 0, never looked at).
__device__ __forceinline__ void load_keys(const Select& q, int64_t seg, int per, uint32_t* keys) {
  const int64_t s0 = seg * per * kSelThreads;
#pragma unroll 1
  for (int i = 0; i < per; i += 4) {
    int64_t pos[4];
    float w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t s = s0 + (i + j) * kSelThreads + threadIdx.x, at = s < q.n ? s : q.n - 1;
      pos[j] = q.slot_pos[at];
      w[j] = q.weight[at];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) keys[key_at((i + j) * kSelThreads + threadIdx.x)] = evict_key(pos[j], w[j], q.keep_from);
  }
}

// The slots with the m smallest keys (side 0) or the used ones among the
// others (side 1), listed in slot order; returns how many (0 <= m <= n).
__device__ __forceinline__ int select_slots(const Select& q, int m, int side, int32_t* list) {
  extern __shared__ __align__(16) uint32_t keys[];
  __shared__ uint32_t hist[kBins], scan[kSelWaves], found[2];
  const int lane = threadIdx.x & 63;
  const int64_t want = ((int64_t)q.n + kSelThreads - 1) / kSelThreads;
  const int per = want > kSegKeys ? kSegKeys : (int)((want + 3) / 4 * 4);
  const int64_t segs = (want + per - 1) / per;
  load_keys(q, 0, per, keys);

  // the m-th smallest key `kth`, of which `ties` (lowest slots first) belong to the m
  uint32_t kth = 0, ties = m;
  if (m > 0) {
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
      const uint32_t above = pass == 0 ? 0u : ~0u << (shift + bits);
      for (int i = threadIdx.x; i < kBins; i += kSelThreads) hist[i] = 0;
#pragma unroll 1
      for (int64_t seg = 0; seg < segs; ++seg) {
        if (segs > 1) {
          __syncthreads();  // (everyone is done with the keys before)
          load_keys(q, seg, per, keys);
        }
        __syncthreads();
        const int64_t s0 = (seg * kSelThreads + threadIdx.x) * per;
#pragma unroll 1
        for (int i = 0; i < per; i += 4) {
          const u32x4 k4 = *(const u32x4*)(keys + key_at(threadIdx.x * per + i));
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const bool on = s0 + i + j < q.n && ((k4[j] ^ kth) & above) == 0;
            const unsigned long long who = __ballot(on);
            if (!who) continue;
            const uint32_t digit = k4[j] >> shift & ((1u << bits) - 1);
            // (a wave whose keys share the digit, as equal weights do, counts once)
            const uint32_t first = __builtin_amdgcn_readlane(digit, __ffsll(who) - 1);
            if (__ballot(on && digit == first) == who) {
              if (lane == __ffsll(who) - 1) atomicAdd(&hist[first], (uint32_t)__popcll(who));
            } else if (on) {
              atomicAdd(&hist[digit], 1u);
            }
          }
        }
      }
      __syncthreads();
      const uint32_t a = hist[2 * threadIdx.x], b = hist[2 * threadIdx.x + 1];
      uint32_t total;
      const uint32_t before = block_scan(a + b, scan, &total);
      if (before < ties && ties <= before + a) found[0] = 2 * threadIdx.x, found[1] = before;
      if (before + a < ties && ties <= before + a + b) found[0] = 2 * threadIdx.x + 1, found[1] = before + a;
      __syncthreads();
      kth |= found[0] << shift;
      ties -= found[1];
    }
  }

  // Of the keys equal to kth the first `ties` are among the m; free slots
  // (key 0) are never among the used ones.  Before a thread's own slots lie
  // `out` listed ones off kth and `eq` equal ones.
  uint32_t out = 0, eq = 0;
#pragma unroll 1
  for (int64_t seg = 0; seg < segs; ++seg) {
    __syncthreads();
    if (segs > 1) {
      load_keys(q, seg, per, keys);
      __syncthreads();
    }
    const int64_t s0 = (seg * kSelThreads + threadIdx.x) * per;
    uint32_t my_out = 0, my_eq = 0;
#pragma unroll 1
    for (int i = 0; i < per; i += 4) {
      const u32x4 k4 = *(const u32x4*)(keys + key_at(threadIdx.x * per + i));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool in = s0 + i + j < q.n;
        my_out += in && (side == 0 ? k4[j] < kth : k4[j] > kth);
        my_eq += in && k4[j] == kth;
      }
    }
    uint32_t all_out, all_eq;
    const uint32_t out0 = out + block_scan(my_out, scan, &all_out), eq0 = eq + block_scan(my_eq, scan, &all_eq);
    uint32_t o = out0, e = eq0;
    if (my_out + my_eq > 0) {
#pragma unroll 1
      for (int i = 0; i < per; ++i) {
        const uint32_t k = keys[key_at(threadIdx.x * per + i)];
        if (s0 + i >= q.n) break;
        const uint32_t low_eq = min(e, ties), high_eq = kth == 0 ? 0u : e - low_eq;  // equal ones before, on each side
        const bool low = k < kth || (k == kth && e < ties), high = k > kth || (k == kth && e >= ties && kth != 0);
        if (side == 0 ? low : high) list[o + (side == 0 ? low_eq : high_eq)] = (int32_t)(s0 + i);
        o += side == 0 ? k < kth : k > kth;
        e += k == kth;
      }
    }
    out += all_out;
    eq += all_eq;
  }
  const uint32_t low_eq = min(eq, ties);
  return (int)(out + (side == 0 ? low_eq : kth == 0 ? 0u : eq - low_eq));
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

// 16 bytes at a time (equal types, aligned rows): e counts 16-byte pieces.
__device__ __forceinline__ void copy_row16(const Rows& src, int64_t from, const Rows& dst, int64_t to, int per, int es,
                                           int e0, int e1, int step) {
  for (int e = e0; e < e1; e += step) {
    const int64_t h = e / per, d = e % per * (16 / es);
    const int64_t fi = (from * src.ss + h * src.sh + d) * es, ti = (to * dst.ss + h * dst.sh + d) * es;
    *(u32x4*)((uint8_t*)dst.k + ti) = *(const u32x4*)((const uint8_t*)src.k + fi);
    *(u32x4*)((uint8_t*)dst.v + ti) = *(const u32x4*)((const uint8_t*)src.v + fi);
  }
}

struct AppendArgs {
  int64_t* slot_pos;
  float* weight;
  int64_t* end;
  const int64_t* start;
  Rows cache, fresh;
  int32_t* list;
  int n, T, Hk, D;
  int64_t recent;
  bool rows_too;
};

// A single token, then several.
template <int ST, int DT>
__global__ __launch_bounds__(kSelThreads) void kv_append_one_kernel(AppendArgs a) {
  const int64_t start = *a.start;
  const Select q{a.slot_pos, a.weight, a.n, start + 1 - a.recent};
  const int s = first_slot(q);  // (every thread has read its slots and *start)
  if (threadIdx.x == 0) {
    a.slot_pos[s] = start;
    a.weight[s] = 0.0f;
    *a.end = start + 1;
  }
  copy_row<ST, DT>(a.fresh, 0, a.cache, s, a.D, threadIdx.x, a.Hk * a.D, kSelThreads);
}

template <int ST, int DT>
__global__ __launch_bounds__(kSelThreads) void kv_append_kernel(AppendArgs a) {
  const int64_t start = *a.start;
  const Select q{a.slot_pos, a.weight, a.n, start + a.T - a.recent};
  select_slots(q, a.T, 0, a.list);
  __syncthreads();  // the list is written
  for (int i = threadIdx.x; i < a.T; i += kSelThreads) {
    const int s = a.list[i];
    a.slot_pos[s] = start + i;
    a.weight[s] = 0.0f;
  }
  if (threadIdx.x == 0) *a.end = start + a.T;
  if (a.rows_too) {
    const int row = a.Hk * a.D;
    for (int i = 0; i < a.T; ++i)
      copy_row<ST, DT>(a.fresh, i, a.cache, a.list[i], a.D, threadIdx.x, row, kSelThreads);
  }
}

template <int ST, int DT>
__global__ __launch_bounds__(256) void kv_rows_kernel(AppendArgs a) {
  copy_row<ST, DT>(a.fresh, blockIdx.x, a.cache, a.list[blockIdx.x], a.D, threadIdx.x, a.Hk * a.D, 256);
}

struct TakeArgs {
  const int64_t *slot_pos, *end;
  const float* weight;
  int64_t *to_pos, *to_end;
  float* to_weight;
  Rows src, dst;
  int32_t* list;  // [capacity], then the count
  int n, capacity, Hk, D, es;
  int64_t recent;
  bool vec;
};

__global__ __launch_bounds__(kSelThreads) void kv_take_kernel(TakeArgs a) {
  const int64_t end = *a.end;
  const Select q{a.slot_pos, a.weight, a.n, end - a.recent};
  const int kept = select_slots(q, a.n > a.capacity ? a.n - a.capacity : 0, 1, a.list);
  if (threadIdx.x == 0) {
    a.list[a.capacity] = kept;
    *a.to_end = end;
  }
}

__global__ __launch_bounds__(256) void kv_take_rows_kernel(TakeArgs a) {
  const int i = blockIdx.x;
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
    const int per = a.D * a.es / 16;
    copy_row16(a.src, s, a.dst, i, per, a.es, threadIdx.x, a.Hk * per, 256);
  } else if (a.es == 4) {
    copy_row<XT_F32, XT_F32>(a.src, s, a.dst, i, a.D, threadIdx.x, a.Hk * a.D, 256);
  } else {
    copy_row<XT_F16, XT_F16>(a.src, s, a.dst, i, a.D, threadIdx.x, a.Hk * a.D, 256);
  }
}

constexpr int kInlineElems = 1 << 15;  // key elements that the selecting workgroup still writes itself

template <int ST, int DT>
int append_types(const AppendArgs& a, hipStream_t st) {
  if (a.T == 1) {
    kv_append_one_kernel<ST, DT><<<1, kSelThreads, 0, st>>>(a);
    return check_launch();
  }
  kv_append_kernel<ST, DT><<<1, kSelThreads, key_words(keys_per_thread(a.n)) * 4, st>>>(a);
  int rc = check_launch();
  if (rc || a.rows_too) return rc;
  kv_rows_kernel<ST, DT><<<a.T, 256, 0, st>>>(a);
  return check_launch();
}

template <int ST>
int append_from(const AppendArgs& a, int ct, hipStream_t st) {
  return ct == XT_F32 ? append_types<ST, XT_F32>(a, st) : ct == XT_F16 ? append_types<ST, XT_F16>(a, st)
                                                                        : append_types<ST, XT_BF16>(a, st);
}

}  // namespace

int launch_kv_append(const KvAppend& c, hipStream_t st) {
  AppendArgs a{c.slot_pos, c.weight, c.end, c.start, Rows{c.k, c.v, c.k_ss, c.k_sh},
               Rows{const_cast<void*>(c.kn), const_cast<void*>(c.vn), c.n_ss, c.n_sh}, (int32_t*)c.ws, (int)c.slots, (int)c.T,
               (int)c.Hk, (int)c.D, c.recent, c.T * c.Hk * c.D <= kInlineElems};
  return c.nt == XT_F32 ? append_from<XT_F32>(a, c.ct, st) : c.nt == XT_F16 ? append_from<XT_F16>(a, c.ct, st)
                                                                             : append_from<XT_BF16>(a, c.ct, st);
}

int launch_kv_take(const KvTake& c, hipStream_t st) {
  const int es = c.ct == XT_F32 ? 4 : 2;
  auto ok = [&](const void* p, int64_t ss, int64_t sh) { return (uintptr_t)p % 16 == 0 && ss * es % 16 == 0 && sh * es % 16 == 0; };
  const bool vec = c.D * es % 16 == 0 && ok(c.k, c.k_ss, c.k_sh) && ok(c.v, c.k_ss, c.k_sh) && ok(c.to_k, c.t_ss, c.t_sh) &&
                   ok(c.to_v, c.t_ss, c.t_sh);
  TakeArgs a{c.slot_pos, c.end, c.weight, c.to_pos, c.to_end, c.to_weight,
             Rows{const_cast<void*>(c.k), const_cast<void*>(c.v), c.k_ss, c.k_sh}, Rows{c.to_k, c.to_v, c.t_ss, c.t_sh},
             (int32_t*)c.ws, (int)c.slots, (int)c.capacity, (int)c.Hk, (int)c.D, es, c.recent, vec};
  kv_take_kernel<<<1, kSelThreads, key_words(keys_per_thread(a.n)) * 4, st>>>(a);
  const int rc = check_launch();
  if (rc) return rc;
  kv_take_rows_kernel<<<a.capacity, 256, 0, st>>>(a);
  return check_launch();
}

}  // namespace sbq
