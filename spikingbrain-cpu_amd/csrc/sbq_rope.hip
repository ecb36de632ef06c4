// sbq_rope.hip - norms of queries and keys for each head, and the rotation to
// their positions, in one pass.
//
//   y = x / sqrt(mean(x^2) + eps) * w            (where there are weights)
//   (y_a, y_b) <- (y_a cos - y_b sin, y_b cos + y_a sin), angle = pos * f[i],
//
// a pair i being the columns (i, i + F) or (2i, 2i + 1).  Every vector is read
// and written once, which is what bounds a long prompt; a step's few rows are
// bound by the latency of one load after the launch.  A lane holds four pairs
// (or eight columns that are not rotated), so that a vector of 128 columns lies
// in 16 lanes, four vectors in a wave, and the rotation crosses no lanes.
//
// The angle's product is exact and reduced in 64 bits: at position 131072 an
// fp32 product is off by up to 2^-8 of a radian.  The cosines of a workgroup's
// tokens are computed once, a pair a thread, and kept in LDS for all heads.
#include "sbq_common.h"
#include "sbq_launch.h"

namespace sbq {

namespace {

constexpr int kRopeThreads = 256, kRopeTokens = 4;  // threads, and at most so many tokens a workgroup

// cos and sin of pos * f.  The product as a sum of two doubles, its distance
// from the nearest quarter turn (pi / 2 in two doubles), then the Taylor series
// over [-pi/4, pi/4] (next terms 2e-9 and 1e-10 of the result's scale).
__device__ __forceinline__ float2 turn(int64_t pos, float f) {
  const double a = (double)pos, b = (double)f;
  const double hi = a * b, lo = __builtin_fma(a, b, -hi);
  const double n = __builtin_rint(hi * 0.63661977236758134308);
  double r = __builtin_fma(-n, 1.57079632679489655800, hi);
  r = __builtin_fma(-n, 6.12323399573676603587e-17, r) + lo;
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
  const int quarter = (int)(int64_t)n & 3;  // (of an n past 2^63 nothing is left anyway)
  const float cs = quarter & 1 ? s : c, sn = quarter & 1 ? c : s;
  return make_float2(quarter == 1 || quarter == 2 ? -cs : cs, quarter >= 2 ? -sn : sn);
}

__device__ __forceinline__ void rotate(float a, float b, float2 t, float& ya, float& yb) {
  ya = __builtin_fmaf(a, t.x, -(b * t.y));
  yb = __builtin_fmaf(b, t.x, a * t.y);
}

// Four consecutive elements, n of them there (VEC: 0 or 4, aligned).
template <int XT, bool VEC>
__device__ __forceinline__ void load4(const typename XElem<XT>::T* p, int n, float (&x)[4]) {
  typedef typename XElem<XT>::T T;
  typedef T V __attribute__((ext_vector_type(4)));
  if constexpr (VEC) {
    if (n > 0) {
      const V v = *(const V*)p;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = (float)v[j];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = 0.0f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = j < n ? (float)p[j] : 0.0f;
  }
}

template <int XT, bool VEC, bool INTER>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(RopeArgs a) {
  typedef typename XElem<XT>::T T;
  extern __shared__ __align__(16) float2 cs[];  // [tokens][items * 4]
  const int lane = threadIdx.x & (a.lanes - 1), group = threadIdx.x / a.lanes, groups = kRopeThreads / a.lanes;
  const int64_t token0 = (int64_t)(blockIdx.x / a.parts) * a.tokens;
  const int part = blockIdx.x % a.parts, n_tok = (int)min((int64_t)a.tokens, a.T - token0);
  const int rows = n_tok * a.rows;  // a.rows: vectors of a token
  const int pair_items = (a.pairs + 3) / 4;

  // the lane's two pieces of four columns: from column pa and pb on, na and nb of them there
  int pa, pb, na, nb;
  const bool rotated = lane < pair_items;
  if (!rotated) {
    pa = 2 * a.pairs + 8 * (lane - pair_items), pb = pa + 4;
    na = a.D - pa, nb = a.D - pb;
  } else if (INTER) {
    pa = 8 * lane, pb = pa + 4;
    na = 2 * a.pairs - pa, nb = 2 * a.pairs - pb;
  } else {
    pa = 4 * lane, pb = a.pairs + pa;
    na = nb = a.pairs - pa;
  }
  na = na < 0 ? 0 : na > 4 ? 4 : na, nb = nb < 0 ? 0 : nb > 4 ? 4 : nb;

  const int step = groups * a.parts;
  int row = part * groups + group;
  float xa[4], xb[4];
  auto fetch = [&](int row) {
    const int tok = row / a.rows, h = row % a.rows;
    const bool key = h >= a.heads;
    const T* p = (const T*)(key ? a.k : a.q) + (token0 + tok) * (key ? a.k_st : a.q_st) + (key ? (h - a.heads) * a.k_sh : h * a.q_sh);
    load4<XT, VEC>(p + pa, na, xa);
    load4<XT, VEC>(p + pb, nb, xb);
  };
  if (row < rows) fetch(row);  // (the first vector's load goes ahead of the angles)

  for (int i = threadIdx.x; i < n_tok * a.pairs; i += kRopeThreads) {
    const int tok = i / a.pairs, f = i - tok * a.pairs;
    const int64_t t = a.first + token0 + tok;
    cs[tok * pair_items * 4 + f] = turn(a.positions[t / a.per] + t % a.per, a.inv_freq[f]);
  }
  __syncthreads();

  for (; row < rows; row += step) {
    const int tok = row / a.rows, h = row % a.rows;
    const bool key = h >= a.heads;
    const void* const w = key ? a.k_weight : a.q_weight;
    if (w) {
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) sum = __builtin_fmaf(xa[j], xa[j], __builtin_fmaf(xb[j], xb[j], sum));
      for (int o = 1; o < a.lanes; o <<= 1) sum += __shfl_xor(sum, o, 64);
      const float r = 1.0f / __builtin_sqrtf(sum / (float)a.D + a.eps);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j < na) xa[j] = xa[j] * r * load_elem(w, a.wt, pa + j);
        if (j < nb) xb[j] = xb[j] * r * load_elem(w, a.wt, pb + j);
      }
    }
    float ya[4], yb[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) ya[j] = xa[j], yb[j] = xb[j];
    if (rotated) {
      const float2* const t = cs + (tok * pair_items + lane) * 4;
      if constexpr (INTER) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {  // (entries past the last pair meet columns past it)
          const float2 u = t[j], v = t[j + 2];
          rotate(xa[2 * j], xa[2 * j + 1], u, ya[2 * j], ya[2 * j + 1]);
          rotate(xb[2 * j], xb[2 * j + 1], v, yb[2 * j], yb[2 * j + 1]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) rotate(xa[j], xb[j], t[j], ya[j], yb[j]);
      }
    }
    const int64_t to = (token0 + tok) * (key ? a.ko_st : a.qo_st) + (key ? (h - a.heads) * a.ko_sh : h * a.qo_sh);
    void* const out = key ? a.k_out : a.q_out;
    store_y4(out, XT, to + pa, (f32x4){ya[0], ya[1], ya[2], ya[3]}, VEC && na == 4, na);
    store_y4(out, XT, to + pb, (f32x4){yb[0], yb[1], yb[2], yb[3]}, VEC && nb == 4, nb);
    if (row + step < rows) fetch(row + step);
  }
}

template <int XT, bool VEC>
int launch_xt(const RopeArgs& a, bool inter, unsigned grid, size_t lds, hipStream_t st) {
  if (inter)
    rope_kernel<XT, VEC, true><<<grid, kRopeThreads, lds, st>>>(a);
  else
    rope_kernel<XT, VEC, false><<<grid, kRopeThreads, lds, st>>>(a);
  return check_launch();
}

}  // namespace

int launch_rope(const RopeArgs& c, bool inter, int xt, hipStream_t st) {
  RopeArgs a = c;
  a.rows = a.heads + a.kv_heads;
  const int items = (a.pairs + 3) / 4 + (a.D - 2 * a.pairs + 7) / 8;
  a.lanes = 1;
  while (a.lanes < items) a.lanes <<= 1;
  const int groups = kRopeThreads / a.lanes;
  a.tokens = a.T >= 1024 ? kRopeTokens : 1;
  // few tokens: a vector a lane group, on as many workgroups as that takes
  a.parts = a.T < 512 ? (a.rows + groups - 1) / groups : 1;
  const int64_t es = xt == XT_F32 ? 4 : 2, n = 4 * es;
  auto vec = [&](const void* p, int64_t s, int64_t h) { return (uintptr_t)p % n == 0 && s % 4 == 0 && h % 4 == 0; };
  const bool v = a.pairs % 4 == 0 && a.D % 4 == 0 && vec(a.q, a.q_st, a.q_sh) && vec(a.q_out, a.qo_st, a.qo_sh) &&
                 (a.kv_heads == 0 || (vec(a.k, a.k_st, a.k_sh) && vec(a.k_out, a.ko_st, a.ko_sh)));
  const size_t lds = (size_t)a.tokens * ((a.pairs + 3) / 4) * 4 * sizeof(float2);
  const int64_t most = kLaunchThreads / kRopeThreads / a.parts * a.tokens;  // tokens of a launch
  for (int64_t t0 = 0; t0 < c.T; t0 += most) {
    a.T = c.T - t0 < most ? c.T - t0 : most;
    a.q = (const char*)c.q + t0 * c.q_st * es, a.k = (const char*)c.k + t0 * c.k_st * es;
    a.q_out = (char*)c.q_out + t0 * c.qo_st * es, a.k_out = (char*)c.k_out + t0 * c.ko_st * es;
    a.first = t0;
    const unsigned grid = (unsigned)((a.T + a.tokens - 1) / a.tokens * a.parts);
    const int rc = xt == XT_F32   ? v ? launch_xt<XT_F32, true>(a, inter, grid, lds, st) : launch_xt<XT_F32, false>(a, inter, grid, lds, st)
                   : xt == XT_F16 ? v ? launch_xt<XT_F16, true>(a, inter, grid, lds, st) : launch_xt<XT_F16, false>(a, inter, grid, lds, st)
                   : v ? launch_xt<XT_BF16, true>(a, inter, grid, lds, st) : launch_xt<XT_BF16, false>(a, inter, grid, lds, st);
    if (rc) return rc;
  }
  return 0;
}

}  // namespace sbq
