// sbq_rope.hip - norms of queries and keys for each head, and the rotation to
// their positions, in one pass.
//
//   y = x / sqrt(mean(x^2) + eps) * w            (where there are weights)
//   (y_a, y_b) <- (y_a cos - y_b sin, y_b cos + y_a sin), angle = pos * f[i],
//
// a pair i being the columns (i, i + F) or (2i, 2i + 1).  Every vector is read
// and written once, which is what bounds a long prompt (8192 tokens of 40 x 128 bf16
// 33 us, 5.1 TB/s; of 126 columns, whose halves begin at no vector's alignment, 37);
// a step's few rows are bound by the latency of one load after the launch (4.1 us).
// Other widths of what is not rotated (128 columns, 126 of them rotated: 77 us) leave
// half of the lanes without a piece.  A lane holds four pairs
// (or eight columns that are not rotated), so that a vector of 128 columns lies
// in 16 lanes, four vectors in a wave, and the rotation crosses no lanes.
//
// The angle's product is exact and reduced in 64 bits: at position 131072 an
// fp32 product is off by up to 2^-8 of a radian.  The cosines of a workgroup's
// tokens are computed once, a pair a thread, and kept in LDS for all heads.
#include <algorithm>

#include "sbq_common.h"
#include "sbq_launch.h"

namespace sbq {

namespace {

// Threads, and at most so many tokens a workgroup (from 1024 workgroups on; at 2, 4, 8,
// 16 tokens each 8192 tokens of 40 x 128 bf16 columns take 32.0, 31.8, 31.0, 30.8 us,
// 16000 of 5 x 128 23.4, 16.0, 14.3, 14.1).
constexpr int kRopeThreads = 256, kRopeTokens = 8;

// cos and sin of pos * f.  The product as a sum of two doubles, its distance
// from the nearest quarter turn (pi / 2 in two doubles; from 2^51 on the count of
// quarters is one off at times, which a second look at the rest mends: 520 u of
// error at 2^53 else, 1.1 with it), then the Taylor series over [-pi/4, pi/4] (next
// terms 2e-9 and 1e-10 of the result's scale).
__device__ __forceinline__ float2 turn(int64_t pos, float f) {
  const double a = (double)pos, b = (double)f;
  const double hi = a * b, lo = __builtin_fma(a, b, -hi);
  const double n = __builtin_rint(hi * 0.63661977236758134308);
  double r = __builtin_fma(-n, 1.57079632679489655800, hi);
  r = __builtin_fma(-n, 6.12323399573676603587e-17, r) + lo;
  const double more = __builtin_rint(r * 0.63661977236758134308);
  r = __builtin_fma(-more, 6.12323399573676603587e-17, __builtin_fma(-more, 1.57079632679489655800, r));
  const float x = (float)r, z = x * x;
  float s = __builtin_fmaf(z, 2.7557319e-6f, -1.98412698e-4f);
  s = __builtin_fmaf(z, s, 8.3333333e-3f);
  s = __builtin_fmaf(z, s, -0.166666667f);
  s = __builtin_fmaf(z * x, s, x);
  float c = __builtin_fmaf(z, -2.75573192e-7f, 2.48015873e-5f);
  c = __builtin_fmaf(z, c, -1.38888889e-3f);
  c = __builtin_fmaf(z, c, 4.16666667e-2f);
  c = __builtin_fmaf(z, c, -0.5f);
  c = __builtin_fmaf(z, c, 1.0f);
  const int quarter = ((int)(int64_t)n + (int)more) & 3;  // (of an n past 2^63 nothing is left anyway)
  const float cs = quarter & 1 ? s : c, sn = quarter & 1 ? c : s;
  return make_float2(quarter == 1 || quarter == 2 ? -cs : cs, quarter >= 2 ? -sn : sn);
}

__device__ __forceinline__ void rotate(float a, float b, float2 t, float& ya, float& yb) {
  ya = __builtin_fmaf(a, t.x, -(b * t.y));
  yb = __builtin_fmaf(b, t.x, a * t.y);
}

// N consecutive elements as they lie in memory, n of them there (floats where they
// are used, after whatever their loads are to overlap).  VEC: all or none are there,
// aligned; else whole pieces go by unaligned loads and stores, others by elements.
template <int XT, int N, bool VEC>
struct Piece {
  typedef typename XElem<XT>::T T;
  typedef T V __attribute__((ext_vector_type(N)));
  typedef V Loose __attribute__((aligned(sizeof(T))));
  V x;
  __device__ __forceinline__ void load(const T* p, int n) {
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = (T)0.0f;
    if constexpr (VEC) {
      if (n > 0) x = *(const V*)p;
    } else if (n == N) {
      x = *(const Loose*)p;
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j < n) x[j] = p[j];
    }
  }
  __device__ __forceinline__ void floats(float (&to)[N]) const {
#pragma unroll
    for (int j = 0; j < N; ++j) to[j] = (float)x[j];
  }
  static __device__ __forceinline__ void store(T* p, int n, const float (&y)[N]) {
    V v;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = (T)fp32_rounded(y[j]);
    if constexpr (VEC) {
      if (n > 0) *(V*)p = v;
    } else if (n == N) {
      *(Loose*)p = v;
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j < n) p[j] = v[j];
    }
  }
};

template <int WT, int N>
__device__ __forceinline__ void weights_at(const void* w, int from, float (&to)[N]) {
  Piece<WT, N, false> p;
  p.load((const typename XElem<WT>::T*)w + from, N);
  p.floats(to);
}

// N columns in each of a lane's two pieces.
template <int XT, int N, bool VEC, bool INTER>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(RopeArgs a) {
  typedef typename XElem<XT>::T T;
  extern __shared__ __align__(16) float2 cs[];  // [tokens][items * N]
  const int lane = threadIdx.x & (a.lanes - 1), group = threadIdx.x / a.lanes, groups = kRopeThreads / a.lanes;
  const int64_t token0 = (int64_t)(blockIdx.x / a.parts) * a.tokens;
  const int part = blockIdx.x % a.parts, n_tok = (int)min((int64_t)a.tokens, a.T - token0);
  const int pair_items = (a.pairs + N - 1) / N;

  // The lane's two pieces: from column pa and pb on, na and nb columns of them
  // there.  Where the last lane's would go past the end (not VEC), they begin as much
  // earlier instead, over columns of the lane before, which come out the same twice
  // and are left out of the sum (sa and sb of them).
  int pa, pb, na, nb, pair0 = 0, sa = 0, sb = 0;
  const bool rotated = lane < pair_items;
  if (rotated && !INTER) {
    pa = N * lane;
    if (!VEC && a.pairs >= N && pa + N > a.pairs) sa = sb = pa + N - a.pairs, pa -= sa;
    pair0 = pa, pb = a.pairs + pa;
    na = nb = a.pairs - pa;
  } else {
    const int from = rotated ? 0 : 2 * a.pairs, to = rotated ? 2 * a.pairs : a.D;
    pa = from + 2 * N * (rotated ? lane : lane - pair_items);
    if (!VEC && to - from >= 2 * N && pa < to && pa + 2 * N > to) sa = pa + 2 * N - to, pa -= sa, sb = sa - N;
    pair0 = pa / 2, pb = pa + N;
    na = to - pa, nb = to - pb;
  }
  na = na < 0 ? 0 : na > N ? N : na, nb = nb < 0 ? 0 : nb > N ? N : nb;

  // its vectors: head h of token tok, a step's heads further each time
  const int step = groups * a.parts;
  int tok = 0, h = part * groups + group;
  while (h >= a.rows) h -= a.rows, ++tok;  // a.rows: vectors of a token
  Piece<XT, N, VEC> ra, rb;
  auto fetch = [&]() {
    if (tok >= n_tok) return;
    const bool key = h >= a.heads;
    const T* const p = (const T*)(key ? a.k : a.q) + (token0 + tok) * (key ? a.k_st : a.q_st) +
                       (int64_t)(key ? h - a.heads : h) * (key ? a.k_sh : a.q_sh);
    ra.load(p + pa, na);
    rb.load(p + pb, nb);
  };
  fetch();  // (the first vectors' loads go ahead of the angles)

  for (int i = threadIdx.x; i < n_tok * a.pairs; i += kRopeThreads) {
    const int t_in = i / a.pairs, f = i - t_in * a.pairs;
    const int64_t t = a.first + token0 + t_in;
    cs[t_in * pair_items * N + f] = turn(a.per == 1 ? a.positions[t] : a.positions[t / a.per] + t % a.per, a.inv_freq[f]);
  }
  // the weights of its columns
  float wq[2][N], wk[2][N];
  auto weights = [&](const void* w, float (&to)[2][N]) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int from = k ? pb : pa, n = k ? nb : na;
#pragma unroll
      for (int j = 0; j < N; ++j) to[k][j] = 0.0f;
      if (!w || n <= 0) continue;
      if (VEC || n == N) {  // (of any alignment)
        a.wt == XT_F32   ? weights_at<XT_F32, N>(w, from, to[k])
        : a.wt == XT_F16 ? weights_at<XT_F16, N>(w, from, to[k])
                         : weights_at<XT_BF16, N>(w, from, to[k]);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (j < n) to[k][j] = load_elem(w, a.wt, from + j);
      }
    }
  };
  weights(a.q_weight, wq);
  if (a.kv_heads > 0) weights(a.k_weight, wk);
  __syncthreads();

  const float mean = 1.0f / (float)a.D;
  while (tok < n_tok) {
    const bool key = h >= a.heads;
    const int t_in = tok;
    T* const to = (T*)(key ? a.k_out : a.q_out) + (token0 + t_in) * (key ? a.ko_st : a.qo_st) +
                  (int64_t)(key ? h - a.heads : h) * (key ? a.ko_sh : a.qo_sh);
    float xa[N], xb[N];
    ra.floats(xa);
    rb.floats(xb);
    if (key ? a.k_weight != nullptr : a.q_weight != nullptr) {
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float ca = VEC || j >= sa ? xa[j] : 0.0f, cb = VEC || j >= sb ? xb[j] : 0.0f;
        sum = __builtin_fmaf(ca, ca, __builtin_fmaf(cb, cb, sum));
      }
      for (int o = 1; o < a.lanes; o <<= 1) sum += __shfl_xor(sum, o, 64);
      const float r = 1.0f / __builtin_sqrtf(__builtin_fmaf(sum, mean, a.eps));
#pragma unroll
      for (int j = 0; j < N; ++j) {
        xa[j] = xa[j] * r * (key ? wk[0][j] : wq[0][j]);
        xb[j] = xb[j] * r * (key ? wk[1][j] : wq[1][j]);
      }
    }
    float ya[N], yb[N];
#pragma unroll
    for (int j = 0; j < N; ++j) ya[j] = xa[j], yb[j] = xb[j];
    if (rotated) {
      const float2* const t = cs + t_in * pair_items * N + pair0;
      if constexpr (INTER) {
#pragma unroll
        for (int j = 0; j < N / 2; ++j) {  // (entries past the last pair meet columns past it)
          rotate(xa[2 * j], xa[2 * j + 1], t[j], ya[2 * j], ya[2 * j + 1]);
          rotate(xb[2 * j], xb[2 * j + 1], t[j + N / 2], yb[2 * j], yb[2 * j + 1]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) rotate(xa[j], xb[j], t[j], ya[j], yb[j]);
      }
    }
    Piece<XT, N, VEC>::store(to + pa, na, ya);
    Piece<XT, N, VEC>::store(to + pb, nb, yb);
    h += step;
    while (h >= a.rows) h -= a.rows, ++tok;
    fetch();
  }
}

template <int XT, int N, bool VEC>
int launch_xt(const RopeArgs& a, bool inter, unsigned grid, size_t lds, hipStream_t st) {
  if (inter)
    rope_kernel<XT, N, VEC, true><<<grid, kRopeThreads, lds, st>>>(a);
  else
    rope_kernel<XT, N, VEC, false><<<grid, kRopeThreads, lds, st>>>(a);
  return check_launch();
}
// N: elements of a piece, 4 or (of 2 bytes) 8.
template <int XT>
int launch_vec(const RopeArgs& a, int N, bool vec, bool inter, unsigned grid, size_t lds, hipStream_t st) {
  if constexpr (XT != XT_F32) {
    if (N == 8) return vec ? launch_xt<XT, 8, true>(a, inter, grid, lds, st) : launch_xt<XT, 8, false>(a, inter, grid, lds, st);
  }
  return vec ? launch_xt<XT, 4, true>(a, inter, grid, lds, st) : launch_xt<XT, 4, false>(a, inter, grid, lds, st);
}

}  // namespace

int launch_rope(const RopeArgs& c, bool inter, int xt, hipStream_t st) {
  RopeArgs a = c;
  a.rows = a.heads + a.kv_heads;
  const int64_t es = xt == XT_F32 ? 4 : 2;
  auto fits = [&](const void* p, int64_t s, int64_t h, int n) {
    return (uintptr_t)p % (n * es) == 0 && s % n == 0 && h % n == 0;
  };
  auto vec = [&](int n) {
    return a.pairs % n == 0 && a.D % n == 0 && fits(a.q, a.q_st, a.q_sh, n) && fits(a.q_out, a.qo_st, a.qo_sh, n) &&
           (a.kv_heads == 0 || (fits(a.k, a.k_st, a.k_sh, n) && fits(a.k_out, a.ko_st, a.ko_sh, n)));
  };
  const int most_n = xt == XT_F32 ? 4 : 8;
  const bool aligned = vec(4);
  const int N = aligned ? (most_n == 8 && vec(8) ? 8 : 4) : a.pairs >= 8 ? most_n : 4;
  const int items = (a.pairs + N - 1) / N + (a.D - 2 * a.pairs + 2 * N - 1) / (2 * N);
  a.lanes = 1;
  while (a.lanes < items) a.lanes <<= 1;
  const int groups = kRopeThreads / a.lanes;
  a.tokens = (int)std::max<int64_t>(1, std::min<int64_t>(kRopeTokens, a.T / 1024));
  // few tokens: a vector a lane group, on as many workgroups as that takes; else a
  // workgroup a token's vectors (40 x 128 bf16: 1, 256, 300, 512 tokens 4.1, 5.2, 5.5,
  // 6.2 us the one way, 5.0, 5.7, 6.0, 6.3 the other)
  a.parts = a.T <= 512 ? (a.rows + groups - 1) / groups : 1;
  const size_t lds = (size_t)a.tokens * ((a.pairs + N - 1) / N) * N * sizeof(float2);
  const int64_t most = kLaunchThreads / kRopeThreads / a.parts * a.tokens;  // tokens of a launch
  for (int64_t t0 = 0; t0 < c.T; t0 += most) {
    a.T = c.T - t0 < most ? c.T - t0 : most;
    a.q = (const char*)c.q + t0 * c.q_st * es, a.k = (const char*)c.k + t0 * c.k_st * es;
    a.q_out = (char*)c.q_out + t0 * c.qo_st * es, a.k_out = (char*)c.k_out + t0 * c.ko_st * es;
    a.first = t0;
    const unsigned grid = (unsigned)((a.T + a.tokens - 1) / a.tokens * a.parts);
    const int rc = xt == XT_F32   ? launch_vec<XT_F32>(a, N, aligned, inter, grid, lds, st)
                   : xt == XT_F16 ? launch_vec<XT_F16>(a, N, aligned, inter, grid, lds, st)
                                  : launch_vec<XT_BF16>(a, N, aligned, inter, grid, lds, st);
    if (rc) return rc;
  }
  return 0;
}

}  // namespace sbq
