// sbq_w4.hip - linears with 4-bit weights and one scale per group of columns.
//
//   y[m,n] = sum_G s[n,G] * (sum_{k in G} q[n,k] x[m,k]) (+ bias[n]),
//   q in -8..7, G = groups of 32, 64 or 128 columns, s in bf16.
//
// What bounds it: at one row the conversions of the weights (some 140 vector
// instructions a tile and wave; 151936 x 2560: fp16 54 us, fp32 73 us, 39 us
// for the bytes at a large copy's rate); at many rows reading x, once per
// workgroup (64 rows over 12288 x 4096, groups of 128: bf16 17 us, fp32 32;
// of 64: 18 and 43), and at fp32 splitting it.  (Times of replayed graphs, four
// weights in turn.)  A packed tile is 16 rows x
// 128 columns in 1 KiB, one 16-byte load per lane, in the order of the MFMA A
// operand: lane = g*16 + r holds row r, dword s the columns 32 s + 8 g + 0..7
// of the tile, so that each group of 32 columns is one 16x16x32 MFMA step and
// the scale is applied to the fp32 partial sums of its group (a weight
// rounded with its scale to 16 bits would lose half of the bits of fp32
// activations).
//
// A workgroup of KS waves owns G 16-row tiles of the weight; its waves take
// the K tiles in turn and are summed through LDS in wave order.
//
// Activations: fp16 and bf16 are the MFMA's own operands (weights converted to
// the same type, exactly).  fp32 is split into two fp16 planes after a
// power-of-two scaling per row and K tile: 22 significant bits, 2^-39 of the
// tile's maximum at least, below the rounding of an fp32 sum.
//   STAGE   up to 8 rows: the wave converts its K tiles once into LDS, 16 lanes
//           per row and tile (a single row: four tiles at a time), and reads
//           fragments from there; a fragment read straight from memory would be
//           converted 16 times over at one row
//   rows    more: rows are copied into LDS as they are (rows_w4_kernel)
//   direct  more, and not aligned for those copies: each lane reads the
//           fragment it multiplies
#include "sbq_common.h"
#include "sbq_dma.h"
#include "sbq_launch.h"

namespace sbq {

namespace {

constexpr int kW4MaxWaves = 8;
// rows_w4_kernel: weight tiles (of 16 rows) up to which a workgroup takes one;
// two up to twice as many, then three.  A CU holds one workgroup, each of which
// reads all of x.  64 bf16 rows, K 4096: 256 tiles 13 us by one each, 18 by
// three; 512 tiles 24 by one, 16 by two, 18 by three; 768 tiles 33, 28 and 19.
constexpr int kW4RowGroups = 256;
constexpr int kW4WideTiles = 2048;  // 16-row tiles from which a decode workgroup takes two

// 8 nibbles u = q + 8 -> fp16 q: element 2i in nibble i, 2i + 1 in nibble
// i + 4; 0x6400 | u is 1024 + u.
__device__ __forceinline__ f16x8 w4_to_f16(uint32_t w) {
  const f16x2 bias = {(_Float16)1032.0f, (_Float16)1032.0f};
  f16x8 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f16x2 p = __builtin_bit_cast(f16x2, ((w >> (4 * i)) & 0x000f000fu) | 0x64006400u) - bias;
    o[2 * i] = p.x;
    o[2 * i + 1] = p.y;
  }
  return o;
}

// ... -> bf16 q / 16, exactly: v_cvt_off_f32_i4 gives the fp32 value of a
// two's complement nibble over 16 (u ^ 8), the upper halves of two pair up.
// The 16 comes back at the end (W4Math::kBack).
__device__ __forceinline__ bf16x8 w4_to_bf16(uint32_t w) {
  u32x4 o;
  w ^= 0x88888888u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t p = w >> (4 * i);
    const uint32_t lo = __float_as_uint(__builtin_amdgcn_cvt_off_f32_i4((int)p));
    const uint32_t hi = __float_as_uint(__builtin_amdgcn_cvt_off_f32_i4((int)(p >> 16)));
    o[i] = __builtin_amdgcn_perm(hi, lo, 0x07060302u);
  }
  return __builtin_bit_cast(bf16x8, o);
}

template <int XT>
struct W4Math {
  typedef f16x8 V;
  static constexpr float kBack = 1.0f;
  static __device__ __forceinline__ V weight(uint32_t w) { return w4_to_f16(w); }
  static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct W4Math<XT_BF16> {
  typedef bf16x8 V;
  static constexpr float kBack = 16.0f;
  static __device__ __forceinline__ V weight(uint32_t w) { return w4_to_bf16(w); }
  static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

// 8 consecutive activations, as they are in memory.
template <int XT>
struct X8 {
  typedef typename XElem<XT>::T T;
  typedef T V __attribute__((ext_vector_type(8)));
  V v;
  // VEC: the row is 16-byte aligned and K a multiple of 16 bytes.  Columns from
  // K on are zero, by selection: with a branch per piece one row over 151936 x
  // 2560 took 87 us, without 79.
  template <bool VEC>
  __device__ __forceinline__ void load(const T* row, int k0, int K) {
    constexpr int N = VEC ? 16 / sizeof(T) : 1;
    typedef T Part __attribute__((ext_vector_type(N)));
    Part p[8 / N];
#pragma unroll
    for (int j = 0; j < 8; j += N) p[j / N] = *(const Part*)(row + (k0 + j < K ? k0 + j : 0));
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k0 + j / N * N < K ? p[j / N][j % N] : (T)0.0f;
  }
};

// Largest magnitude of 8 fp32 values (NaN left out; FINITE: infinities too).
template <bool FINITE>
__device__ __forceinline__ float max_abs8(const X8<XT_F32>::V& v) {
  float m = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float a = __builtin_fabsf(v[j]);
    m = !FINITE || a <= 3.4028235e38f ? __builtin_fmaxf(m, a) : m;
  }
  return m;
}

// Two fp16 planes of v * 2^e (s = 2^e): hi rounded to nearest, lo the
// remainder.  An infinity stays one (ODD; its remainder would be NaN).  Two
// values at a time: this conversion is most of a wave's work at fp32.
template <bool ODD>
__device__ __forceinline__ void split_f16(const X8<XT_F32>::V& v, float s, f16x8& hi, f16x8& lo) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const f32x2 t = {v[j] * s, v[j + 1] * s};
    const f16x2 h = __builtin_convertvector(t, f16x2);
    f32x2 r = {__builtin_fmaf(v[j], s, -(float)h.x), __builtin_fmaf(v[j + 1], s, -(float)h.y)};
    if (ODD) r = f32x2{__builtin_fabsf(t.x) > 3.4028235e38f ? 0.0f : r.x, __builtin_fabsf(t.y) > 3.4028235e38f ? 0.0f : r.y};
    const f16x2 l = __builtin_convertvector(r, f16x2);
    hi[j] = h.x, hi[j + 1] = h.y, lo[j] = l.x, lo[j + 1] = l.y;
  }
}

__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Exponent for a tile's maximum (>= 0, finite): it lands in [2^14, 2^15), or
// below where the maximum is under 2^-106.  (-113 at least, for the largest
// values; exp2i holds it and its inverse.)
__device__ __forceinline__ int tile_exp(float mx) {
  const int e = 141 - (int)(__float_as_uint(mx) >> 23);
  return mx > 0.0f ? min(e, 120) : 0;
}

__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// The two planes of the lane's N pieces of a row's K tile, whose maximum
// `across` takes over the lanes that share the row; the factor to multiply the
// products by.
template <int N, class F>
__device__ __forceinline__ float split_tile(const X8<XT_F32> (&raw)[N], f16x8 (&hi)[N], f16x8 (&lo)[N], F across) {
  float mx = 0.0f;
#pragma unroll
  for (int s = 0; s < N; ++s) mx = __builtin_fmaxf(mx, max_abs8<false>(raw[s].v));
  mx = across(mx);
  const bool odd = __any(mx == __builtin_inff());
  if (__builtin_expect(odd, false)) {
    mx = 0.0f;
#pragma unroll
    for (int s = 0; s < N; ++s) mx = __builtin_fmaxf(mx, max_abs8<true>(raw[s].v));
    mx = across(mx);
  }
  const int e = tile_exp(mx);
  if (__builtin_expect(odd, false)) {
#pragma unroll
    for (int s = 0; s < N; ++s) split_f16<true>(raw[s].v, exp2i(e), hi[s], lo[s]);
  } else {
#pragma unroll
    for (int s = 0; s < N; ++s) split_f16<false>(raw[s].v, exp2i(e), hi[s], lo[s]);
  }
  return exp2i(-e);
}
// ... over the lane groups of a fragment's row
__device__ __forceinline__ float max_groups(float mx) {
  mx = __builtin_fmaxf(mx, __shfl_xor(mx, 16, 64));
  return __builtin_fmaxf(mx, __shfl_xor(mx, 32, 64));
}

// acc += one 16x16 tile over a K tile: each group's partial sums times its
// scales (b: bf16, four rows of the weight) and the row's factor f.
template <int XT, int GS, int P>
__device__ __forceinline__ void add_tile(const typename W4Math<XT>::V (&wv)[4], const typename W4Math<XT>::V (&xv)[P][4],
                                         const u32x2 (&b)[4 / GS], float f, f32x4& acc) {
#pragma unroll
  for (int q = 0; q < 4 / GS; ++q) {
    f32x4 part = (f32x4)(0.0f);
#pragma unroll
    for (int s = q * GS; s < q * GS + GS; ++s)
#pragma unroll
      for (int p = 0; p < P; ++p) part = W4Math<XT>::mfma(wv[s], xv[p][s], part);
    const f32x4 s4 = {__uint_as_float(b[q].x << 16), __uint_as_float(b[q].x & 0xffff0000u),
                      __uint_as_float(b[q].y << 16), __uint_as_float(b[q].y & 0xffff0000u)};
#pragma unroll
    for (int v = 0; v < 4; ++v) acc[v] = __builtin_fmaf(part[v], s4[v] * f, acc[v]);
  }
}

struct W4Args {
  const void* x;
  const uint8_t* packed;
  const uint16_t* gscale;
  const float* bias;
  void* y;
  int64_t ldx, ldy;
  int M, N, K, Nt, Kc, yt;
  bool yvec;
};

// The waves' partial sums, added in wave order, and the rows out.  lds is free
// once every wave is here.
template <int XT, int G, int MT>
__device__ __forceinline__ void join_w4(const W4Args& a, const f32x4 (&acc)[G][MT], uint8_t* lds, int nt0, int m0) {
  const int lane = threadIdx.x & 63, ks = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), KS = blockDim.x >> 6;
  const int c = lane & 15, g = lane >> 4, M = min(a.M - m0, MT * 16);
  if (KS > 1) {
    f32x4* const red = (f32x4*)lds;
    __syncthreads();  // (the staging area is done with)
#pragma unroll
    for (int i = 0; i < G; ++i)
#pragma unroll
      for (int t = 0; t < MT; ++t) red[(ks * G * MT + i * MT + t) * 64 + lane] = acc[i][t];
    __syncthreads();
  }
  for (int u = ks; u < G * MT; u += KS) {
    const int i = u / MT, t = u % MT;
    f32x4 v;
    if (KS > 1) {
      const f32x4* const red = (const f32x4*)lds;
      v = red[u * 64 + lane];
      for (int k = 1; k < KS; ++k) v += red[(k * G * MT + u) * 64 + lane];
    } else {
#pragma unroll
      for (int ii = 0; ii < G; ++ii)
#pragma unroll
        for (int tt = 0; tt < MT; ++tt)
          if (ii == i && tt == t) v = acc[ii][tt];
    }
    const int m = t * 16 + c, n = (nt0 + i) * 16 + 4 * g;
    if (m >= M || n >= a.N) continue;
    v *= W4Math<XT>::kBack;
    if (a.bias) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += n + j < a.N ? a.bias[n + j] : 0.0f;
    }
    store_y4(a.y, a.yt, (int64_t)(m0 + m) * a.ldy + n, v, a.yvec, a.N - n);
  }
}

// XT: activations; MT: 16-row tiles of x; G: 16-row tiles of the weight; GS:
// MFMA steps per group (1, 2, 4); ROWS: 0 direct, else STAGE of 1, 2, 4 or 8
// rows; D: K tiles loaded together; VEC: as X8::load.
template <int XT, int MT, int G, int GS, int ROWS, int D, bool VEC>
__global__ __launch_bounds__(kW4MaxWaves * 64) void linear_w4_kernel(W4Args a) {
  typedef typename XElem<XT>::T T;
  typedef W4Math<XT> Math;
  typedef typename Math::V V;
  constexpr int P = XT == XT_F32 ? 2 : 1;  // planes of x
  constexpr int GPT = 4 / GS;              // groups per tile
  // STAGE: the D tiles' ROWS rows are staged 4 (row, tile) pairs at a time
  constexpr int PASSES = D * ROWS / 4;
  constexpr int STAGE = P * D * ROWS * 256;  // bytes of a wave, then the pairs' factors
  static_assert(ROWS == 0 || (MT == 1 && D * ROWS % 4 == 0), "staging serves one row tile, four pairs at a time");
  extern __shared__ __align__(16) uint8_t lds[];
  const int lane = threadIdx.x & 63, ks = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), KS = blockDim.x >> 6;
  const int c = lane & 15, g = lane >> 4;
  const int m0 = blockIdx.y * (MT * 16), M = min(a.M - m0, MT * 16);
  const int nt0 = blockIdx.x * G;
  const T* const x = (const T*)a.x + (int64_t)m0 * a.ldx;

  f32x4 acc[G][MT];
#pragma unroll
  for (int i = 0; i < G; ++i)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[i][t] = (f32x4)(0.0f);

  uint8_t* const stage = lds + ks * (STAGE + (P == 2 ? D * ROWS * 4 : 0));
  float* const factor = (float*)(stage + STAGE);

  for (int kb = ks; kb < a.Kc; kb += D * KS) {
    u32x4 w[D][G];
    u32x2 sc[D][G][GPT];
    X8<XT> raw[ROWS ? PASSES : D][ROWS ? 1 : MT][ROWS ? 1 : 4];
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int kt = min(kb + d * KS, a.Kc - 1);  // (a surplus tile is loaded again, not used)
#pragma unroll
      for (int i = 0; i < G; ++i) {
        const int64_t nt = min(nt0 + i, a.Nt - 1);
        w[d][i] = *(const u32x4*)(a.packed + ((nt * a.Kc + kt) * 64 + lane) * 16);
#pragma unroll
        for (int q = 0; q < GPT; ++q)
          sc[d][i][q] = *(const u32x2*)(a.gscale + ((nt * a.Kc + kt) * GPT + q) * 16 + 4 * g);
      }
      if constexpr (ROWS == 0) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int s = 0; s < 4; ++s)
            raw[d][t][s].template load<VEC>(x + (int64_t)min(t * 16 + c, M - 1) * a.ldx, kt * 128 + s * 32 + g * 8, a.K);
      }
    }
    if constexpr (ROWS > 0) {
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {  // lane group g: pair p * 4 + g = (tile, row)
        const int pair = p * 4 + g, kt = min(kb + pair / ROWS * KS, a.Kc - 1);
        raw[p][0][0].template load<VEC>(x + (int64_t)min(pair % ROWS, M - 1) * a.ldx, kt * 128 + c * 8, a.K);
      }
      wave_lds_fence();
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const int pair = p * 4 + g;
        uint8_t* const to = stage + pair * 256 + ((c ^ pair) & 15) * 16;
        if constexpr (XT == XT_F32) {
          f16x8 hi[1], lo[1];
          const float f = split_tile(raw[p][0], hi, lo, [](float mx) {
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) mx = __builtin_fmaxf(mx, __shfl_xor(mx, o, 64));
            return mx;
          });
          *(f16x8*)to = hi[0];
          *(f16x8*)(to + D * ROWS * 256) = lo[0];
          if (c == 0) factor[pair] = f;
        } else {
          *(V*)to = __builtin_bit_cast(V, raw[p][0][0].v);
        }
      }
      wave_lds_fence();
    }
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int kt = kb + d * KS;
      if (kt >= a.Kc) break;
      V wv[G][4];
#pragma unroll
      for (int i = 0; i < G; ++i)
#pragma unroll
        for (int s = 0; s < 4; ++s) wv[i][s] = Math::weight(w[d][i][s]);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        V xv[P][4];
        float f = 1.0f;
        if constexpr (ROWS > 0) {
          const int pair = d * ROWS + min(c, M - 1);
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const uint8_t* const from = stage + pair * 256 + (((s * 4 + g) ^ pair) & 15) * 16;
#pragma unroll
            for (int p = 0; p < P; ++p) xv[p][s] = *(const V*)(from + p * D * ROWS * 256);
          }
          if constexpr (XT == XT_F32) f = factor[pair];
        } else if constexpr (XT == XT_F32) {
          f = split_tile(raw[d][t], xv[0], xv[1], max_groups);
        } else {
#pragma unroll
          for (int s = 0; s < 4; ++s) xv[0][s] = __builtin_bit_cast(V, raw[d][t][s].v);
        }
#pragma unroll
        for (int i = 0; i < G; ++i) add_tile<XT, GS>(wv[i], xv, sc[d][i], f, acc[i][t]);
      }
    }
  }

  join_w4<XT, G, MT>(a, acc, lds, nt0, m0);
}

// More than 8 rows, aligned.  A fragment read straight from memory takes one
// line per lane (its lanes are 16 rows), four times the time of the bytes, so
// the wave copies its K tiles' rows into LDS 8 KiB at a time (whole rows' 256
// or 512 bytes, two chunks under way, their 16-byte pieces permuted by the row)
// and reads fragments there: 64 rows over 12288 x 4096, bf16, 39.5 us without,
// 19 with.  Two chunks and one K tile's weights are always under way; the last
// ones of a wave once more.
// Order of issue, a K tile's weights w(i) and chunks c(i): w0 c0 c1, w1 after
// w0 is read, then a chunk after each one read.  With two or more chunks a K
// tile, w(i) is older than the two chunks under way; with one it is between
// them, and only the compiler's own wait for its registers retires it.
template <int XT, int MT, int G, int GS>
__global__ __launch_bounds__(kW4MaxWaves * 64) void rows_w4_kernel(W4Args a) {
  typedef typename XElem<XT>::T T;
  typedef W4Math<XT> Math;
  typedef typename Math::V V;
  constexpr int P = XT == XT_F32 ? 2 : 1, ES = sizeof(T), GPT = 4 / GS;
  constexpr int CT = MT < 4 / ES ? MT : 4 / ES, NCH = MT / CT;  // row tiles of a chunk, chunks of a K tile
  constexpr int PPR = 8 * ES, NDMA = CT * 2 * ES, CHUNK = CT * 16 * 128 * ES, NW = G * (1 + GPT);
  extern __shared__ __align__(16) uint8_t lds[];
  const int lane = threadIdx.x & 63, ks = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), KS = blockDim.x >> 6;
  const int c = lane & 15, g = lane >> 4;
  const int m0 = blockIdx.y * (MT * 16), M = min(a.M - m0, MT * 16);
  const int nt0 = blockIdx.x * G;
  const T* const x = (const T*)a.x + (int64_t)m0 * a.ldx;
  uint8_t* const own = lds + ks * (2 * CHUNK);

  f32x4 acc[G][MT];
#pragma unroll
  for (int i = 0; i < G; ++i)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[i][t] = (f32x4)(0.0f);

  u32x4 w[G];
  u32x2 sc[2][G][GPT];
  auto load = [&](int kt, u32x2 (&sc)[G][GPT]) {
    asm volatile("" ::: "memory");  // (their order among the copies is counted on)
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const int64_t at = (int64_t)min(nt0 + i, a.Nt - 1) * a.Kc + kt;
      w[i] = *(const u32x4*)(a.packed + (at * 64 + lane) * 16);
#pragma unroll
      for (int q = 0; q < GPT; ++q) sc[i][q] = *(const u32x2*)(a.gscale + (at * GPT + q) * 16 + 4 * g);
    }
    asm volatile("" ::: "memory");
  };
  auto copy = [&](int kt, int ch, int buf) {
    int l = lane;
    asm volatile("" : "+v"(l));  // (else the addresses of all copies are kept in registers)
#pragma unroll
    for (int i = 0; i < NDMA; ++i) {
      const int row = i * (64 / PPR) + l / PPR, k = kt * 128 + ((l % PPR) ^ (row & 15)) * (16 / ES);
      const T* const src = x + (int64_t)min(ch * CT * 16 + row, M - 1) * a.ldx + (k < a.K ? k : 0);
      __builtin_amdgcn_global_load_lds((const void*)src,
                                       (__attribute__((address_space(3))) void*)(own + buf * CHUNK + i * 1024), 16, 0, 0);
    }
    asm volatile("" ::: "memory");
  };

  int buf = 0;
  auto tile = [&](int kt, const u32x2 (&b)[G][GPT], u32x2 (&next)[G][GPT]) {
    wait_vmcnt<2 * NDMA>();  // the weights where NCH > 1; the two chunks after them stay under way
    asm volatile("" ::: "memory");
    V wv[G][4];
#pragma unroll
    for (int i = 0; i < G; ++i)
#pragma unroll
      for (int s = 0; s < 4; ++s) wv[i][s] = Math::weight(w[i][s]);
    load(min(kt + KS, a.Kc - 1), next);
    const bool tail = kt * 128 + 128 > a.K;
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch) {
      if (ch < 2)  // all but the next chunk, and the next weights where they came after this one
        wait_vmcnt<NDMA + NW>();
      else
        wait_vmcnt<NDMA>();
      asm volatile("" ::: "memory");
#pragma unroll
      for (int tc = 0; tc < CT; ++tc) {
        const int t = ch * CT + tc;
        X8<XT> raw[4];
        const uint8_t* const from = own + buf * CHUNK + (tc * 16 + c) * (128 * ES);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          u32x4 piece[ES / 2];
#pragma unroll
          for (int h = 0; h < ES / 2; ++h) {
            const int p = (s * 4 + g) * (ES / 2) + h;
            piece[h] = *(const u32x4*)(from + (p ^ c) * 16);
            if (tail && kt * 128 + p * (16 / ES) >= a.K) piece[h] = (u32x4)(0u);
          }
          __builtin_memcpy(&raw[s].v, piece, sizeof(piece));
        }
        V xv[P][4];
        float f = 1.0f;
        if constexpr (XT == XT_F32) {
          f = split_tile(raw, xv[0], xv[1], max_groups);
        } else {
#pragma unroll
          for (int s = 0; s < 4; ++s) xv[0][s] = __builtin_bit_cast(V, raw[s].v);
        }
#pragma unroll
        for (int i = 0; i < G; ++i) add_tile<XT, GS>(wv[i], xv, b[i], f, acc[i][t]);
      }
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): the chunk is read
      asm volatile("" ::: "memory");
      copy(min(kt + (ch + 2) / NCH * KS, a.Kc - 1), (ch + 2) % NCH, buf);
      buf ^= 1;
    }
  };
  load(ks, sc[0]);
  copy(ks, 0, 0);
  copy(NCH == 1 ? min(ks + KS, a.Kc - 1) : ks, NCH == 1 ? 0 : 1, 1);
#pragma unroll 1
  for (int kt = ks; kt < a.Kc; kt += 2 * KS) {
    tile(kt, sc[0], sc[1]);
    if (kt + KS < a.Kc) tile(kt + KS, sc[1], sc[0]);
  }
  wait_vmcnt<0>();  // (no copy outlives the area)
  join_w4<XT, G, MT>(a, acc, lds, nt0, m0);
}

// ---------------------------------------------------------------------------
// quantizing and packing (once per weight)
// ---------------------------------------------------------------------------
// One group per 32 lanes: s = bf16(max(max |w|, 1e-8) / 7), q = rint(w / s)
// clamped to -7..7, so the rounding of the scale to bf16 costs nothing: q is
// taken against the rounded one.
template <int XT>
__global__ __launch_bounds__(256) void quantize_groups_kernel(const void* w, int64_t ldw, int N, int K, int group, int Gn,
                                                              int8_t* q, int64_t ldq, uint16_t* scale) {
  typedef typename XElem<XT>::T T;
  const int64_t id = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (id >= (int64_t)N * Gn) return;
  const int n = (int)(id / Gn), G = (int)(id % Gn), l = threadIdx.x & 31;
  const T* const row = (const T*)w + n * ldw;
  float v[4], mx = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int k = G * group + i * 32 + l;
    v[i] = i * 32 < group && k < K ? XElem<XT>::to_f32(row[k]) : 0.0f;
    mx = __builtin_fmaxf(mx, __builtin_fabsf(v[i]));
  }
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) mx = __builtin_fmaxf(mx, __shfl_xor(mx, o, 64));
  const __bf16 sb = (__bf16)(__builtin_fmaxf(mx, 1e-8f) / 7.0f);
  const float s = (float)sb;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int k = G * group + i * 32 + l;
    if (i * 32 < group && k < K)
      q[n * ldq + k] = (int8_t)__builtin_fminf(__builtin_fmaxf(__builtin_rintf(v[i] / s), -7.0f), 7.0f);
  }
  if (l == 0) scale[id] = __builtin_bit_cast(uint16_t, sb);
}

// One dword (8 columns of one row) of the packed tiles per thread.
__global__ __launch_bounds__(256) void pack_w4_kernel(const int8_t* q, int64_t ldq, int N, int K, int Kc, int64_t count,
                                                      uint32_t* packed) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= count) return;
  const int s = id & 3, lane = (id >> 2) & 63;
  const int64_t tile = id >> 8;
  const int64_t n = tile / Kc * 16 + (lane & 15);
  const int k0 = (int)(tile % Kc) * 128 + s * 32 + (lane >> 4) * 8;
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int v = n < N && k0 + j < K ? min(max((int)q[n * ldq + k0 + j], -8), 7) : 0;
    w |= (uint32_t)(v + 8) << (4 * (j / 2) + 16 * (j % 2));
  }
  packed[id] = w;
}

// Scales [N][Gn] -> [Nt][Gp][16], padding 0 (Gp: the groups of whole tiles).
__global__ __launch_bounds__(256) void pack_scale_kernel(const uint16_t* scale, int N, int Gn, int Gp, int64_t count,
                                                         uint16_t* gscale) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= count) return;
  const int64_t n = id / 16 / Gp * 16 + (id & 15);
  const int G = (int)(id / 16 % Gp);
  gscale[id] = n < N && G < Gn ? scale[n * Gn + G] : 0;
}

__global__ __launch_bounds__(256) void unpack_w4_kernel(const uint32_t* packed, int N, int K, int Kc, int64_t count,
                                                        int8_t* q, int64_t ldq) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= count) return;
  const int s = id & 3, lane = (id >> 2) & 63;
  const int64_t tile = id >> 8;
  const int64_t n = tile / Kc * 16 + (lane & 15);
  const int k0 = (int)(tile % Kc) * 128 + s * 32 + (lane >> 4) * 8;
  const uint32_t w = packed[id];
  if (n >= N) return;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (k0 + j < K) q[n * ldq + k0 + j] = (int8_t)((int)((w >> (4 * (j / 2) + 16 * (j % 2))) & 15) - 8);
}

__global__ __launch_bounds__(256) void unpack_scale_kernel(const uint16_t* gscale, int Gn, int Gp, int64_t count,
                                                           uint16_t* scale) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= count) return;
  const int64_t n = id / Gn;
  scale[id] = gscale[(n / 16 * Gp + id % Gn) * 16 + n % 16];
}

inline unsigned blocks(int64_t count) { return (unsigned)((count + 255) / 256); }

template <int XT, int MT, int G, int ROWS, int D, bool VEC = true>
int launch_w4(const W4Args& a, int group, int KS, hipStream_t st) {
  constexpr int P = XT == XT_F32 ? 2 : 1;
  const int stage = KS * D * ROWS * (P * 256 + (P == 2 ? 4 : 0)), red = KS > 1 ? KS * G * MT * 1024 : 0;
  const size_t lds = (size_t)(stage > red ? stage : red);
  const dim3 grid((unsigned)((a.Nt + G - 1) / G), (unsigned)((a.M + MT * 16 - 1) / (MT * 16)));
  if (group == 32)
    linear_w4_kernel<XT, MT, G, 1, ROWS, D, VEC><<<grid, KS * 64, lds, st>>>(a);
  else if (group == 64)
    linear_w4_kernel<XT, MT, G, 2, ROWS, D, VEC><<<grid, KS * 64, lds, st>>>(a);
  else
    linear_w4_kernel<XT, MT, G, 4, ROWS, D, VEC><<<grid, KS * 64, lds, st>>>(a);
  return check_launch();
}

template <int XT, int MT, int G>
int launch_rows_w4(const W4Args& a, int group, int KS, hipStream_t st) {
  constexpr int ES = XT == XT_F32 ? 4 : 2, CT = MT < 4 / ES ? MT : 4 / ES;
  const int stage = KS * 2 * CT * 16 * 128 * ES, red = KS > 1 ? KS * G * MT * 1024 : 0;
  const size_t lds = (size_t)(stage > red ? stage : red);
  const dim3 grid((unsigned)((a.Nt + G - 1) / G), (unsigned)((a.M + MT * 16 - 1) / (MT * 16)));
  if (group == 32) {
    if constexpr (G < 3 || (MT < 4 && XT != XT_F32))
      rows_w4_kernel<XT, MT, G, 1><<<grid, KS * 64, lds, st>>>(a);
    else
      return -1;  // no such kernel (rows_w4 never asks for it)
  } else if (group == 64) {
    rows_w4_kernel<XT, MT, G, 2><<<grid, KS * 64, lds, st>>>(a);
  } else {
    rows_w4_kernel<XT, MT, G, 4><<<grid, KS * 64, lds, st>>>(a);
  }
  return check_launch();
}
template <int XT, int MT>
int rows_w4(const W4Args& a, int group, int KS, hipStream_t st) {
  if (a.Nt <= kW4RowGroups) return launch_rows_w4<XT, MT, 1>(a, group, KS, st);
  // (three tiles of 32-column groups beside 64 rows, or beside fp32's planes, do not fit the registers)
  if (a.Nt <= 2 * kW4RowGroups || (group == 32 && (MT == 4 || XT == XT_F32))) return launch_rows_w4<XT, MT, 2>(a, group, KS, st);
  return launch_rows_w4<XT, MT, 3>(a, group, KS, st);
}

template <int XT>
int pick_w4(const W4Args& a, bool xvec, int group, hipStream_t st) {
  int KS = 1;
  while (KS < kW4MaxWaves && KS * 2 < a.Kc) KS *= 2;
  if (!xvec) {  // rows that are not aligned: element by element, in the widest form of each kind
    if (a.M == 1) return launch_w4<XT, 1, 1, 1, 4, false>(a, group, KS, st);
    if (a.M <= 8) return launch_w4<XT, 1, 1, 8, 2, false>(a, group, KS, st);
    if (a.M <= 16) return launch_w4<XT, 1, 1, 0, 1, false>(a, group, KS, st);
    return launch_w4<XT, 4, 2, 0, 1, false>(a, group, KS, st);
  }
  const bool wide = a.Nt >= kW4WideTiles;
  if (a.M == 1) return wide ? launch_w4<XT, 1, 2, 1, 4>(a, group, KS, st) : launch_w4<XT, 1, 1, 1, 4>(a, group, KS, st);
  if (a.M == 2) return wide ? launch_w4<XT, 1, 2, 2, 4>(a, group, KS, st) : launch_w4<XT, 1, 1, 2, 4>(a, group, KS, st);
  if (a.M <= 4) return wide ? launch_w4<XT, 1, 2, 4, 2>(a, group, KS, st) : launch_w4<XT, 1, 1, 4, 2>(a, group, KS, st);
  if (a.M <= 8) return launch_w4<XT, 1, 1, 8, 2>(a, group, KS, st);
  if (a.M <= 16) return rows_w4<XT, 1>(a, group, KS, st);
  if (a.M <= 32) return rows_w4<XT, 2>(a, group, KS, st);
  return rows_w4<XT, 4>(a, group, KS, st);
}

}  // namespace

int launch_quantize_groups(const void* w, int wt, int64_t N, int64_t K, int64_t ldw, int group, int8_t* q, int64_t ldq,
                           uint16_t* scale, hipStream_t st) {
  const int Gn = (int)((K + group - 1) / group);
  const int64_t es = wt == XT_F32 ? 4 : 2, step = kLaunchThreads / 32 / Gn > 0 ? kLaunchThreads / 32 / Gn : 1;
  for (int64_t n = 0; n < N; n += step) {
    const int rows = (int)(N - n < step ? N - n : step);
    const unsigned grid = (unsigned)(((int64_t)rows * Gn + 7) / 8);
    const void* const wn = (const uint8_t*)w + n * ldw * es;
    int8_t* const qn = q + n * ldq;
    uint16_t* const sn = scale + n * Gn;
    if (wt == XT_F32)
      quantize_groups_kernel<XT_F32><<<grid, 256, 0, st>>>(wn, ldw, rows, (int)K, group, Gn, qn, ldq, sn);
    else if (wt == XT_F16)
      quantize_groups_kernel<XT_F16><<<grid, 256, 0, st>>>(wn, ldw, rows, (int)K, group, Gn, qn, ldq, sn);
    else
      quantize_groups_kernel<XT_BF16><<<grid, 256, 0, st>>>(wn, ldw, rows, (int)K, group, Gn, qn, ldq, sn);
    const int rc = check_launch();
    if (rc) return rc;
  }
  return 0;
}

// 16-row tiles that a packing launch takes.
static int64_t tiles_step(int64_t Kc) { return kLaunchThreads / 256 / Kc > 0 ? kLaunchThreads / 256 / Kc : 1; }

int launch_repack_w4(const int8_t* q, int64_t N, int64_t K, int64_t ldq, const uint16_t* scale, int group, uint8_t* packed,
                     uint16_t* gscale, hipStream_t st) {
  const int64_t Nt = (N + 15) / 16, Kc = (K + 127) / 128, Gp = Kc * (128 / group), Gn = (K + group - 1) / group;
  const int64_t step = tiles_step(Kc);
  for (int64_t t = 0; t < Nt; t += step) {
    const int64_t tiles = Nt - t < step ? Nt - t : step, words = tiles * Kc * 256, scales = tiles * Gp * 16;
    const int rows = (int)(N - t * 16 < tiles * 16 ? N - t * 16 : tiles * 16);
    pack_w4_kernel<<<blocks(words), 256, 0, st>>>(q + t * 16 * ldq, ldq, rows, (int)K, (int)Kc, words,
                                                  (uint32_t*)packed + t * Kc * 256);
    pack_scale_kernel<<<blocks(scales), 256, 0, st>>>(scale + t * 16 * Gn, rows, (int)Gn, (int)Gp, scales,
                                                      gscale + t * Gp * 16);
    const int rc = check_launch();
    if (rc) return rc;
  }
  return 0;
}

int launch_unpack_w4(const uint8_t* packed, const uint16_t* gscale, int64_t N, int64_t K, int group, int8_t* q, int64_t ldq,
                     uint16_t* scale, hipStream_t st) {
  const int64_t Nt = (N + 15) / 16, Kc = (K + 127) / 128, Gp = Kc * (128 / group), Gn = (K + group - 1) / group;
  const int64_t step = tiles_step(Kc);
  for (int64_t t = 0; t < Nt; t += step) {
    const int64_t tiles = Nt - t < step ? Nt - t : step, words = tiles * Kc * 256;
    const int64_t rows = N - t * 16 < tiles * 16 ? N - t * 16 : tiles * 16, scales = rows * Gn;
    unpack_w4_kernel<<<blocks(words), 256, 0, st>>>((const uint32_t*)packed + t * Kc * 256, (int)rows, (int)K, (int)Kc, words,
                                                    q + t * 16 * ldq, ldq);
    unpack_scale_kernel<<<blocks(scales), 256, 0, st>>>(gscale + t * Gp * 16, (int)Gn, (int)Gp, scales, scale + t * 16 * Gn);
    const int rc = check_launch();
    if (rc) return rc;
  }
  return 0;
}

int launch_linear_w4(const void* x, int xt, int64_t M, int64_t K, int64_t ldx, bool xvec, const uint8_t* packed,
                     const uint16_t* gscale, const float* bias, int64_t N, int group, void* y, int yt, int64_t ldy, bool yvec,
                     hipStream_t st) {
  constexpr int64_t kRows = 1 << 20;  // rows per launch (the grid's second dimension holds 65535 blocks)
  constexpr int64_t kTiles = kLaunchThreads / (kW4MaxWaves * 64);  // weight tiles per launch
  const int64_t xs = xt == XT_F32 ? 4 : 2, ys = yt == XT_F32 ? 4 : 2, Nt = (N + 15) / 16, Kc = (K + 127) / 128;
  xvec = xvec && K * xs % 16 == 0;
  for (int64_t m = 0; m < M; m += kRows)
    for (int64_t t = 0; t < Nt; t += kTiles) {
      const int64_t tiles = Nt - t < kTiles ? Nt - t : kTiles, n = t * 16, rest = N - n < tiles * 16 ? N - n : tiles * 16;
      const W4Args a{(const uint8_t*)x + m * ldx * xs, packed + t * Kc * 1024, gscale + t * Kc * (128 / group) * 16,
                     bias ? bias + n : nullptr, (uint8_t*)y + (m * ldy + n) * ys, ldx, ldy,
                     (int)(M - m < kRows ? M - m : kRows), (int)rest, (int)K, (int)tiles, (int)Kc, yt, yvec};
      const int rc = xt == XT_F32   ? pick_w4<XT_F32>(a, xvec, group, st)
                     : xt == XT_F16 ? pick_w4<XT_F16>(a, xvec, group, st)
                                    : pick_w4<XT_BF16>(a, xvec, group, st);
      if (rc) return rc;
    }
  return 0;
}

}  // namespace sbq
