// sbq_verify.hip - drafted tokens against the target's probabilities.
//
// Draft t is kept iff u[t] q_t(x_t) < p_t(x_t), up to the first that is not.
// The token after the kept ones is drawn from max(p - q, 0) of the refused
// draft's row, or after the last draft from p's next row, as the first index
// (vocabulary order) whose prefix of mass exceeds u[T] * mass.  Together the
// tokens are distributed as p alone would draw them.
//
// Products and sums are in 64 bits: an fp32 prefix over 151936 tokens is off
// by more than many a token's probability.  One row of p and one of q are all
// that a sequence needs, so a first launch finds the row and sums it in
// segments of kVerSeg tokens, each workgroup deciding by itself which drafts
// are kept; a second launch looks the segment up and goes through it once
// more.  A row of up to kVerWhole tokens is one workgroup's, in one launch (1 and 64
// sequences of 1000 tokens 4.4 and 4.7 us, of 16384 7.0 and 8.0, 300 of 16384 16.5; in
// two launches 9.1, 10.1, 9.7, 10.5, 16.7; up to 4096 tokens 256 threads, 1024 are 1 us
// slower there).  Few sequences are bound by the two launches and three dependent
// loads (token, probability, row; 9.3 us), many by the rows' bytes (64 x 151936 fp32 18.4
// us, 4.2 TB/s).
#include <algorithm>

#include "sbq_common.h"
#include "sbq_launch.h"

namespace sbq {

namespace {

constexpr int kVerThreads = 256, kVerPart = 4 * kVerThreads, kVerSeg = 4 * kVerPart;
constexpr int kVerWholeThreads = 1024, kVerWhole = 16 * kVerWholeThreads;  // a row's tokens that one workgroup takes whole

__device__ __forceinline__ double shfl_xor_f64(double v, int o) { return __shfl_xor(v, o, 64); }

// Two sums over the workgroup at once.
__device__ __forceinline__ double2 block_sum(double2 v, double2* lds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v.x += shfl_xor_f64(v.x, o), v.y += shfl_xor_f64(v.y, o);
  __syncthreads();  // (lds is free)
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  double2 sum = make_double2(0.0, 0.0);
  for (int k = 0; k < (int)blockDim.x >> 6; ++k) sum.x += lds[k].x, sum.y += lds[k].y;
  return sum;
}

// N sums of the threads before this one, in thread order; `total` of all.
template <int N>
struct Sums {
  double v[N];
};
template <int N>
__device__ __forceinline__ Sums<N> block_before(Sums<N> x, Sums<N>* lds, Sums<N>* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  Sums<N> sum = x, before, base;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const double t = __shfl_up(sum.v[i], o, 64);
      if (lane >= o) sum.v[i] += t;
    }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    before.v[i] = __shfl_up(sum.v[i], 1, 64);
    if (lane == 0) before.v[i] = 0.0;
    base.v[i] = total->v[i] = 0.0;
  }
  __syncthreads();  // (lds is free)
  if (lane == 63) lds[w] = sum;
  __syncthreads();
  for (int k = 0; k < (int)blockDim.x >> 6; ++k) {
    const Sums<N> s = lds[k];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      base.v[i] = k == w ? total->v[i] : base.v[i];
      total->v[i] += s.v[i];
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) before.v[i] += base.v[i];
  return before;
}

template <int XT>
__device__ __forceinline__ double prob(const void* p, int64_t i) {
  return (double)(float)((const typename XElem<XT>::T*)p)[i];
}

// The four probabilities of a row from token i on (those past the last one 0).
template <int XT, bool VEC>
__device__ __forceinline__ void row4(const void* row, int64_t i, int64_t V, float (&x)[4]) {
  typedef typename XElem<XT>::T T;
  typedef T V4 __attribute__((ext_vector_type(4)));
  if (VEC) {
    V4 v = {(T)0.0f, (T)0.0f, (T)0.0f, (T)0.0f};
    if (i < V) v = *(const V4*)((const T*)row + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = (float)v[j];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = i + j < V ? (float)((const T*)row)[i + j] : 0.0f;
  }
}

// A token's mass after a refusal: p - q, none where that is negative (NaN stays).
__device__ __forceinline__ double rest(float p, float q) {
  const double d = (double)p - (double)q;
  return d < 0.0 ? 0.0 : d;
}

// How many drafts of sequence b are kept (every wave by itself), of `n`.
template <int XT>
__device__ __forceinline__ int kept_of(const VerifyArgs& a, int64_t b, int n) {
  const int lane = threadIdx.x & 63;
  for (int t0 = 0; t0 < n; t0 += 64) {
    const int t = t0 + lane;
    bool ok = true;
    if (t < n) {
      const int64_t x = a.tokens[b * a.T + t];
      ok = x >= 0 && x < a.V;
      if (ok) {
        typedef typename XElem<XT>::T E;
        const double px = prob<XT>((const E*)a.p + b * a.p_sb + t * a.p_st, x);
        const double qx = a.q ? prob<XT>((const E*)a.q + b * a.q_sb + t * a.q_st, x) : 1.0;
        ok = (double)a.u[b * (a.T + 1) + t] * qx < px;
      }
    }
    const uint64_t no = ~__ballot(ok);
    if (no) return t0 + __builtin_ctzll(no);
  }
  return n;
}

// What row kept_of() leads to: of p, of q (null: none), and the token whose
// one-hot q is subtracted (-1: none).
struct VerRow {
  const void *p, *q;
  int64_t hot;
};
template <int XT>
__device__ __forceinline__ VerRow row_of(const VerifyArgs& a, int64_t b, int n, int kept) {
  typedef typename XElem<XT>::T E;
  VerRow r{(const E*)a.p + b * a.p_sb + kept * a.p_st, nullptr, -1};
  if (kept < n) {
    if (a.q)
      r.q = (const E*)a.q + b * a.q_sb + kept * a.q_st;
    else
      r.hot = a.tokens[b * a.T + kept];
  }
  return r;
}

template <int XT, bool VEC>
__device__ __forceinline__ void masses(const VerRow& r, int64_t i, int64_t V, double (&left)[4], double (&all)[4]) {
  float p[4], q[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  row4<XT, VEC>(r.p, i, V, p);
  if (r.q) row4<XT, VEC>(r.q, i, V, q);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    all[j] = (double)p[j];
    left[j] = i + j == r.hot ? rest(p[j], 1.0f) : rest(p[j], q[j]);
  }
}

__device__ __forceinline__ int count_of(const VerifyArgs& a, int64_t b) {
  if (!a.counts) return (int)a.T;
  const int64_t n = a.counts[b];
  return (int)(n < 0 ? 0 : n > a.T ? a.T : n);
}

// The token: threads hold neighbouring masses m, their sums and the sums `at` of
// those before them.  The first thread whose prefix passes `want` scans its own;
// sums in another order can end a rounding below it: then the last one with mass.
template <int N>
__device__ __forceinline__ void choose(const double (&m)[N], double sum, double at, double want, int64_t i0, int64_t* token) {
  __shared__ int found, last;
  const int lane = threadIdx.x & 63;
  if (threadIdx.x == 0) found = INT32_MAX, last = -1;
  __syncthreads();
  const uint64_t past = __ballot(at + sum > want && sum > 0.0), some = __ballot(sum > 0.0);
  if (lane == 0) {
    if (past) atomicMin(&found, (int)threadIdx.x + __builtin_ctzll(past));
    if (some) atomicMax(&last, (int)threadIdx.x + 63 - __builtin_clzll(some));
  }
  __syncthreads();
  if ((int)threadIdx.x == (found != INT32_MAX ? found : last)) {
    int64_t t = -1;
    bool done = want != want;  // (a uniform that is not a number: no token)
#pragma unroll
    for (int j = 0; j < N; ++j) {
      at += m[j];
      if (m[j] > 0.0 && !done) {
        t = i0 + j;
        done = at > want;
      }
    }
    *token = t;
  }
}

template <int XT, bool VEC>
__global__ __launch_bounds__(kVerThreads) void verify_sum_kernel(VerifyArgs a) {
  __shared__ double2 lds[4];
  const int64_t b = a.first + blockIdx.x / a.segs;
  const int seg = blockIdx.x % a.segs, n = count_of(a, b), kept = kept_of<XT>(a, b, n);
  const VerRow r = row_of<XT>(a, b, n, kept);
  double left = 0.0, all = 0.0;
#pragma unroll
  for (int k = 0; k < kVerSeg / kVerPart; ++k) {
    double l[4], w[4];
    masses<XT, VEC>(r, (int64_t)seg * kVerSeg + k * kVerPart + threadIdx.x * 4, a.V, l, w);
    left += (l[0] + l[1]) + (l[2] + l[3]);
    all += (w[0] + w[1]) + (w[2] + w[3]);
  }
  const double2 sums = block_sum(make_double2(left, all), lds);
  if (threadIdx.x == 0) {
    a.part[b * a.segs + seg] = sums;
    if (seg == 0) a.kept[b] = kept;
  }
}

template <int XT, bool VEC>
__global__ __launch_bounds__(kVerThreads) void verify_pick_kernel(VerifyArgs a) {
  __shared__ Sums<2> lds[4];
  __shared__ Sums<1> lds_seg[4];
  __shared__ double seg_before;
  __shared__ int hit;
  const int64_t b = a.first + blockIdx.x;
  const int n = count_of(a, b), kept = (int)a.kept[b], each = (a.segs + kVerThreads - 1) / kVerThreads;
  const double2* const part = a.part + b * a.segs;
  const double u = (double)a.u[b * (a.T + 1) + a.T];
  const int s0 = threadIdx.x * each;
  Sums<2> mine = {{0.0, 0.0}}, totals;
  for (int s = s0; s < min(s0 + each, a.segs); ++s) mine.v[0] += part[s].x, mine.v[1] += part[s].y;
  if (threadIdx.x == 0) hit = -1;
  const Sums<2> before = block_before(mine, lds, &totals);
  const double total_left = totals.v[0], total_all = totals.v[1], before_left = before.v[0], before_all = before.v[1];
  // (without a refusal the two are equal; nothing left after one: p itself)
  const bool use = total_left > 0.0 || total_left != total_left;
  const double total = use ? total_left : total_all, want = u * total;
  if (!(total > 0.0 && total < __builtin_inf())) {  // (NaN too)
    if (threadIdx.x == 0) a.token[b] = -1;
    return;
  }
  // the segment: the last with mass whose prefix is not beyond `want` (threads'
  // prefixes are sums in different orders, so no segment's end is compared)
  double at = use ? before_left : before_all;
  int last = -1;
  for (int s = s0; s < min(s0 + each, a.segs); ++s) {
    const double mass = use ? part[s].x : part[s].y;
    if (at <= want && mass > 0.0) last = s;
    at += mass;
  }
  const uint64_t any = __ballot(last >= 0);
  if (any && (threadIdx.x & 63) == 63 - __builtin_clzll(any)) atomicMax(&hit, last);
  __syncthreads();
  const int seg = hit;
  if (seg < 0) {  // (a uniform that is not a number)
    if (threadIdx.x == 0) a.token[b] = -1;
    return;
  }
  at = use ? before_left : before_all;
  for (int s = s0; s < min(s0 + each, a.segs); ++s) {
    if (s == seg) seg_before = at;
    at += use ? part[s].x : part[s].y;
  }
  __syncthreads();
  // a thread's share of it: neighbours, so that one scan over the threads gives every prefix
  const VerRow r = row_of<XT>(a, b, n, kept);
  constexpr int kEach = kVerSeg / kVerThreads;
  const int64_t i0 = (int64_t)seg * kVerSeg + threadIdx.x * kEach;
  double m[kEach], sum = 0.0;
  Sums<1> total_seg;
#pragma unroll
  for (int k = 0; k < kEach; k += 4) {
    double l[4], w[4];
    masses<XT, VEC>(r, i0 + k, a.V, l, w);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m[k + j] = use ? l[j] : w[j];
      sum += m[k + j];
    }
  }
  at = seg_before + block_before(Sums<1>{{sum}}, lds_seg, &total_seg).v[0];
  choose<kEach>(m, sum, at, want, i0, a.token + b);
}

// Whole rows of up to kVerWhole tokens: a workgroup a sequence, every thread's
// share in registers from the sums to the choice.
template <int XT, bool VEC>
__global__ __launch_bounds__(kVerWholeThreads) void verify_whole_kernel(VerifyArgs a) {
  __shared__ Sums<1> lds[kVerWholeThreads / 64];
  constexpr int kEach = kVerWhole / kVerWholeThreads;
  const int64_t b = a.first + blockIdx.x;
  const double u = (double)a.u[b * (a.T + 1) + a.T];
  const int n = count_of(a, b), kept = kept_of<XT>(a, b, n);
  const VerRow r = row_of<XT>(a, b, n, kept);
  const int each = ((int)(a.V + blockDim.x - 1) / (int)blockDim.x + 3) & ~3;
  const int64_t i0 = (int64_t)threadIdx.x * each;
  double left[kEach], all[kEach], sum_left = 0.0, sum_all = 0.0;
  Sums<1> sums;
#pragma unroll
  for (int k = 0; k < kEach; k += 4) {
    double l[4] = {}, w[4] = {};
    if (k < each) masses<XT, VEC>(r, i0 + k, a.V, l, w);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      left[k + j] = l[j], all[k + j] = w[j];
      sum_left += l[j], sum_all += w[j];
    }
  }
  if (threadIdx.x == 0) a.kept[b] = kept;
  double at = block_before(Sums<1>{{sum_left}}, lds, &sums).v[0], total = sums.v[0];
  // (without a refusal the two are equal; nothing left after one: p itself)
  const bool use = total > 0.0 || total != total;
  if (!use) {
    at = block_before(Sums<1>{{sum_all}}, lds, &sums).v[0], total = sums.v[0];
#pragma unroll
    for (int k = 0; k < kEach; ++k) left[k] = all[k];
    sum_left = sum_all;
  }
  if (!(total > 0.0 && total < __builtin_inf())) {  // (NaN too)
    if (threadIdx.x == 0) a.token[b] = -1;
    return;
  }
  choose<kEach>(left, sum_left, at, u * total, i0, a.token + b);
}

template <int XT, bool VEC>
int launch_verify_xt(VerifyArgs a, hipStream_t st) {
  const int64_t most = std::max<int64_t>(1, kLaunchThreads / kVerThreads / a.segs);  // sequences of a launch
  const int64_t B = a.B;
  if (a.V <= kVerWhole) {
    a.first = 0;
    const unsigned threads = a.V <= 4096 ? 256 : kVerWholeThreads;
    verify_whole_kernel<XT, VEC><<<(unsigned)B, threads, 0, st>>>(a);
    return check_launch();
  }
  for (a.first = 0; a.first < B; a.first += most) {
    a.B = std::min(most, B - a.first);
    verify_sum_kernel<XT, VEC><<<(unsigned)(a.B * a.segs), kVerThreads, 0, st>>>(a);
    if (const int rc = check_launch()) return rc;
    verify_pick_kernel<XT, VEC><<<(unsigned)a.B, kVerThreads, 0, st>>>(a);
    if (const int rc = check_launch()) return rc;
  }
  return 0;
}

}  // namespace

int64_t verify_workspace_bytes(int64_t B, int64_t V) { return V <= kVerWhole ? 0 : B * ((V + kVerSeg - 1) / kVerSeg) * 16; }

int launch_verify(const VerifyArgs& c, int xt, hipStream_t st) {
  VerifyArgs a = c;
  a.segs = (int)((a.V + kVerSeg - 1) / kVerSeg);
  const int64_t n = xt == XT_F32 ? 16 : 8;
  const bool vec = a.V % 4 == 0 && (uintptr_t)a.p % n == 0 && a.p_sb % 4 == 0 && a.p_st % 4 == 0 &&
                   (!a.q || ((uintptr_t)a.q % n == 0 && a.q_sb % 4 == 0 && a.q_st % 4 == 0));
  switch (xt) {
    case XT_F32: return vec ? launch_verify_xt<XT_F32, true>(a, st) : launch_verify_xt<XT_F32, false>(a, st);
    case XT_F16: return vec ? launch_verify_xt<XT_F16, true>(a, st) : launch_verify_xt<XT_F16, false>(a, st);
    default: return vec ? launch_verify_xt<XT_BF16, true>(a, st) : launch_verify_xt<XT_BF16, false>(a, st);
  }
}

}  // namespace sbq
