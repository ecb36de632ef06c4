// sbq_evict.hip - a bounded cache of keys and values that gives up the slots
// which received the least attention.
//
// Slots are ordered by one 32-bit key: free ones 0, then the running sum of
// attention weight as an ordered integer, the `recent` newest positions
// highest; equal keys by slot.  One workgroup finds the m-th smallest key
// digit by digit (11, 11 and 10 bits, a histogram in LDS each; only keys that
// share the digits so far count) and then lists the slots on one side of it in
// slot order.  What bounds it is that workgroup's reading of 12 bytes per
// slot and its steps' latency: a second level over several workgroups would
// cost another launch, more than the reading up to some 32768 slots, which
// the 1024 threads hold in registers.  Integer counts only, so the result
// does not depend on timing.
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

// Keys of the threads' slots in segment `seg`: slot = seg * NK * 1024 + i *
// 1024 + thread; slots past the end get no key (bit i of `in` clear).
template <int NK>
__device__ __forceinline__ uint32_t load_keys(const Select& q, int64_t seg, uint32_t (&key)[NK]) {
  uint32_t in = 0;
#pragma unroll
  for (int i = 0; i < NK; ++i) {
    const int64_t s = (seg * NK + i) * kSelThreads + threadIdx.x;
    key[i] = 0;
    if (s < q.n) {
      key[i] = evict_key(q.slot_pos[s], q.weight[s], q.keep_from);
      in |= 1u << i;
    }
  }
  return in;
}

// The slots with the m smallest keys (side 0) or the used ones among the
// others (side 1), listed in slot order; returns how many (0 <= m <= n).
template <int NK>
__device__ __forceinline__ int select_slots(const Select& q, int m, int side, int32_t* list) {
  __shared__ uint32_t hist[kBins], scan[kSelWaves], found[2];
  __shared__ uint32_t counts[2][NK * kSelWaves];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t segs = ((int64_t)q.n + NK * kSelThreads - 1) / (NK * kSelThreads);
  uint32_t key[NK], in = load_keys<NK>(q, 0, key);

  // the m-th smallest key `kth`, of which `ties` (lowest slots first) belong to the m
  uint32_t kth = 0, ties = m;
  if (m > 0) {
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
      const uint32_t above = pass == 0 ? 0u : ~0u << (shift + bits);
      for (int i = threadIdx.x; i < kBins; i += kSelThreads) hist[i] = 0;
      __syncthreads();
#pragma unroll 1
      for (int64_t seg = 0; seg < segs; ++seg) {
        if (segs > 1) in = load_keys<NK>(q, seg, key);
#pragma unroll
        for (int i = 0; i < NK; ++i) {
          const bool on = (in >> i & 1) && ((key[i] ^ kth) & above) == 0;
          const unsigned long long who = __ballot(on);
          if (!who) continue;
          const uint32_t digit = key[i] >> shift & ((1u << bits) - 1);
          // (a wave whose keys share the digit, as equal weights do, counts once)
          const uint32_t first = __builtin_amdgcn_readlane(digit, __ffsll(who) - 1);
          if (__ballot(on && digit == first) == who) {
            if (lane == __ffsll(who) - 1) atomicAdd(&hist[first], (uint32_t)__popcll(who));
          } else if (on) {
            atomicAdd(&hist[digit], 1u);
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
      __syncthreads();
    }
  }

  uint32_t seen = 0, listed = 0;  // keys equal to kth, slots listed before this segment
#pragma unroll 1
  for (int64_t seg = 0; seg < segs; ++seg) {
    if (segs > 1) in = load_keys<NK>(q, seg, key);
    unsigned long long eq[NK];
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      eq[i] = __ballot((in >> i & 1) && key[i] == kth);
      if (lane == 0) counts[0][i * kSelWaves + w] = __popcll(eq[i]);
    }
    __syncthreads();
    constexpr int NC = NK * kSelWaves;  // <= kSelThreads
    uint32_t total, mine = threadIdx.x < NC ? counts[0][threadIdx.x] : 0u;
    uint32_t before = block_scan(mine, scan, &total);
    if (threadIdx.x < NC) counts[0][threadIdx.x] = seen + before;
    seen += total;
    __syncthreads();
    unsigned long long take[NK];
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const uint32_t rank = counts[0][i * kSelWaves + w] + __popcll(eq[i] & ((1ull << lane) - 1));
      const bool low = m > 0 && (key[i] < kth || (key[i] == kth && rank < ties));
      take[i] = __ballot((in >> i & 1) && (side == 0 ? low : !low && key[i] != 0));
      if (lane == 0) counts[1][i * kSelWaves + w] = __popcll(take[i]);
    }
    __syncthreads();
    mine = threadIdx.x < NC ? counts[1][threadIdx.x] : 0u;
    before = block_scan(mine, scan, &total);
    if (threadIdx.x < NC) counts[1][threadIdx.x] = listed + before;
    listed += total;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NK; ++i)
      if (take[i] >> lane & 1)
        list[counts[1][i * kSelWaves + w] + __popcll(take[i] & ((1ull << lane) - 1))] =
            (int32_t)((seg * NK + i) * kSelThreads + threadIdx.x);
    __syncthreads();  // (the list is written, counts are free)
  }
  return (int)listed;
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

template <int NK, int ST, int DT>
__global__ __launch_bounds__(kSelThreads) void kv_append_kernel(AppendArgs a) {
  const int64_t start = *a.start;
  const Select q{a.slot_pos, a.weight, a.n, start + a.T - a.recent};
  select_slots<NK>(q, a.T, 0, a.list);
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

template <int NK>
__global__ __launch_bounds__(kSelThreads) void kv_take_kernel(TakeArgs a) {
  const int64_t end = *a.end;
  const Select q{a.slot_pos, a.weight, a.n, end - a.recent};
  const int kept = select_slots<NK>(q, a.n > a.capacity ? a.n - a.capacity : 0, 1, a.list);
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
  if (a.n <= 4 * kSelThreads)
    kv_append_kernel<4, ST, DT><<<1, kSelThreads, 0, st>>>(a);
  else if (a.n <= 16 * kSelThreads)
    kv_append_kernel<16, ST, DT><<<1, kSelThreads, 0, st>>>(a);
  else
    kv_append_kernel<32, ST, DT><<<1, kSelThreads, 0, st>>>(a);
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
  if (a.n <= 4 * kSelThreads)
    kv_take_kernel<4><<<1, kSelThreads, 0, st>>>(a);
  else if (a.n <= 16 * kSelThreads)
    kv_take_kernel<16><<<1, kSelThreads, 0, st>>>(a);
  else
    kv_take_kernel<32><<<1, kSelThreads, 0, st>>>(a);
  const int rc = check_launch();
  if (rc) return rc;
  kv_take_rows_kernel<<<a.capacity, 256, 0, st>>>(a);
  return check_launch();
}

}  // namespace sbq
