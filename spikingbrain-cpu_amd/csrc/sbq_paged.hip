// sbq_paged.hip - the paged cache's writing and reading back (sbq_paged.h
// describes the pool).
//
// An 8-bit pool keeps of each token's keys (values) of a head the scale
// max |x| / 127 (int8) or / 448 (e4m3), in fp32, and the nearest codes of x /
// scale (IEEE division, half to even): half a step of 1/127 of the largest
// value, or 2^-4 of each.  Each vector is read once and written once; a lane
// takes 8 columns, so that a vector of 128 lies in 16 lanes and its maximum
// crosses those alone.  A prompt is bound by its bytes (8192 tokens of 8 x 128 bf16
// to e4m3 14 us, 3.6 TB/s, back 12; 32768 fp32 tokens to int8 87 us, 3.9 TB/s), a
// step's few rows by the loads one after another: start, table, row (4.4 us).
#include "sbq_paged.h"

#include <algorithm>

namespace sbq {

namespace {

constexpr int kStoreThreads = 256;
// Vectors of a sequence that one workgroup stores by itself, and moves the length; more
// need a second launch for that (32 vectors of 128 int8 columns 6.3 us the one way, 6.1
// the other, eager 3 us less; 128 vectors 14.8 against 6.0).
constexpr int kStoreAlone = 32;
constexpr int64_t kStoreGroups = 1536;  // workgroups of a launch about (8192 x 8 x 128 bf16 to e4m3, at 1024, 1536, 2048, 4096: 15.2, 14.0, 14.9, 15.9 us)

// Largest code of an 8-bit type.
template <int CT>
__device__ __forceinline__ float largest() {
  return CT == CT_I8 ? 127.0f : 448.0f;
}

// Eight columns as they lie in memory: they become floats where they are used,
// so that nothing waits for them before the next ones are on their way.
template <int XT>
struct Cols {
  typedef typename XElem<XT>::T T;
  typedef T V __attribute__((ext_vector_type(8)));
  V x;
  template <bool VEC>
  __device__ __forceinline__ void load(const T* p, int n) {  // (n of them there; VEC: all or none)
    if constexpr (VEC) {
      if (n > 0) x = *(const V*)p;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < n) x[j] = p[j];
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (T)0.0f;
  }
  __device__ __forceinline__ void floats(float (&to)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) to[j] = (float)x[j];
  }
};

// Eight columns to y from element `at` on, n of them there (vec: eight or none).
__device__ __forceinline__ void store_cols8(void* y, int type, int64_t at, const float (&x)[8], bool vec, int n) {
  if (vec && type != XT_F32) {
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      typedef _Float16 H2 __attribute__((ext_vector_type(2)));
      typedef __bf16 B2 __attribute__((ext_vector_type(2)));
      w[j] = type == XT_F16 ? __builtin_bit_cast(uint32_t, (H2){out_f16(x[2 * j]), out_f16(x[2 * j + 1])})
                            : __builtin_bit_cast(uint32_t, (B2){out_bf16(x[2 * j]), out_bf16(x[2 * j + 1])});
    }
    *(u32x4*)((uint16_t*)y + at) = w;
  } else {
    store_y4(y, type, at, (f32x4){x[0], x[1], x[2], x[3]}, vec, n);
    store_y4(y, type, at + 4, (f32x4){x[4], x[5], x[6], x[7]}, vec, n - 4);
  }
}

// x / scale for eight values, as IEEE division rounds it: the steps of the
// division itself (a refined reciprocal, then the quotient twice by its
// remainder), the reciprocal once for all; where scale is too small or large
// for them to stay in range, the division.
__device__ __forceinline__ void quotients(const float (&x)[8], float scale, float (&q)[8]) {
  if (scale > 0x1p-100f && scale < 0x1p100f) {
    float r = __builtin_amdgcn_rcpf(scale);
    r = __builtin_fmaf(__builtin_fmaf(-scale, r, 1.0f), r, r);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float q0 = x[j] * r, q1 = __builtin_fmaf(__builtin_fmaf(-q0, scale, x[j]), r, q0);
      q[j] = __builtin_fmaf(__builtin_fmaf(-q1, scale, x[j]), r, q1);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = scale > 0.0f ? x[j] / scale : 0.0f;
  }
}

// The nearest codes to eight quotients (scale 0 or NaN: zeros), the first in the low byte.
template <int CT>
__device__ __forceinline__ u32x2 codes(const float (&x)[8], float scale) {
  u32x2 w;
  float y[8];
  quotients(x, scale, y);
#pragma unroll
  for (int j = 0; j < 8; ++j) y[j] = __builtin_amdgcn_fmed3f(y[j], -largest<CT>(), largest<CT>());  // (a subnormal scale's own rounding)
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if constexpr (CT == CT_I8) {
      uint32_t n[4];  // (an integer in the low bits, rounded to even by the addition)
#pragma unroll
      for (int j = 0; j < 4; ++j) n[j] = __float_as_uint(y[4 * h + j] + 12582912.0f);
      w[h] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(n[3], n[2], 0x0c0c0400u), __builtin_amdgcn_perm(n[1], n[0], 0x0c0c0400u),
                                   0x05040100u);
    } else {
      int v = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h], y[4 * h + 1], 0, false);
      w[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h + 2], y[4 * h + 3], v, true);
    }
  }
  return w;
}

// One vector's columns to the pool; the lanes of a vector are neighbours, a
// power of two of them.
template <int CT>
__device__ __forceinline__ void store_cols(const PagedCache& c, bool value, int64_t at, int d, int n, const float (&x)[8],
                                           int lanes) {
  void* const pool = value ? c.v : c.k;
  if constexpr (is_8bit(CT)) {
    uint32_t most = 0;  // the largest magnitude as an integer: infinities and NaN above every number
#pragma unroll
    for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(x[j]) & 0x7fffffffu);
    for (int o = 1; o < lanes; o <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o, 64));
    // (a vector with an infinity or NaN has no codes: it reads back as NaN)
    const float scale = most < 0x7f800000u ? __uint_as_float(most) / largest<CT>() : __builtin_nanf("");
    if (n <= 0) return;
    *(u32x2*)((uint8_t*)pool + at * c.row + d) = codes<CT>(x, scale);  // (columns past D: zeros again)
    if (d == 0) (value ? c.v_scale : c.k_scale)[at] = scale;
  } else {
    if (n <= 0) return;
    store_cols8(pool, CT, at * c.row + d, x, true, 8);
  }
}

// The length after `count` tokens from `start` on.
__device__ __forceinline__ int64_t paged_end(int64_t start, int64_t count, int64_t room) {
  if (start < 0) return 0;
  return start >= room ? room : start + count < room ? start + count : room;
}

// A sequence's vectors, `lanes` lanes each, in tiles of a workgroup's lane
// groups: `tile` neighbouring tokens of a head, which stand side by side in a
// page (as do their scales, that lines of either are written whole), and as
// many heads as there are groups left.
struct PagedTiles {
  int t_in, h_in, heads, across, n;  // the group's token and head of a tile, a tile's heads, tiles across them, tiles in all
  __device__ __forceinline__ explicit PagedTiles(const PagedStore& a) {
    const int group = threadIdx.x / a.lanes;
    t_in = group & (a.tile - 1), h_in = group / a.tile;
    heads = kStoreThreads / a.lanes / a.tile, across = (a.c.Hk + heads - 1) / heads;
    n = (int)((a.T + a.tile - 1) / a.tile) * across;
  }
  // The group's token and head of tile q (token INT32_MAX: none).
  __device__ __forceinline__ void at(const PagedStore& a, int q, int& t, int& h) const {
    const int row = q / across;
    t = row * a.tile + t_in, h = (q - row * across) * heads + h_in;
    if (q >= n || h >= a.c.Hk) t = INT32_MAX;
  }
};

template <int CT, int XT, bool VEC>
__global__ __launch_bounds__(kStoreThreads) void paged_append_kernel(PagedStore a) {
  typedef typename XElem<XT>::T T;
  const PagedCache& c = a.c;
  const int64_t b = blockIdx.x / a.parts, room = (int64_t)c.max_pages << c.page_log;
  const int part = blockIdx.x % a.parts, d = (threadIdx.x & (a.lanes - 1)) * 8, n = c.D - d;
  // A tile's loads go ahead of the one before it: of its rows, whether the
  // sequence has as many or not, and of its page, which the length leads to.
  const PagedTiles tiles(a);
  Cols<XT> k, v;
  int t, h;
  auto fetch = [&](int q) {
    tiles.at(a, q, t, h);
    k.zero(), v.zero();
    if (t >= a.T) return;
    const int64_t from = b * a.n_sb + (int64_t)t * a.n_st + (int64_t)h * a.n_sh + d;
    k.template load<VEC>((const T*)a.kn + from, n);
    v.template load<VEC>((const T*)a.vn + from, n);
  };
  fetch(part);
  const int64_t start = a.start[b], count = paged_count(a.counts, b, a.T);
  int32_t id = -1;
  auto look_up = [&]() {
    const int64_t pos = start + t;
    id = t >= count || start < 0 || start >= room || pos >= room ? -1 : c.table[b * c.max_pages + (pos >> c.page_log)];
  };
  look_up();
  for (int q = part; q < tiles.n; q += a.parts) {
    const Cols<XT> k0 = k, v0 = v;
    const int64_t at = paged_row_of(id, c.pages, start + t, h, c.Hk, c.page_log);
    fetch(q + a.parts);
    look_up();
    if (at < 0) continue;  // (the lanes of a vector go together)
    float x[8];
    k0.floats(x);
    store_cols<CT>(c, false, at, d, n, x, a.lanes);
    v0.floats(x);
    store_cols<CT>(c, true, at, d, n, x, a.lanes);
  }
  if (a.set_length && part == 0) {
    __syncthreads();  // (start may be the length itself, then with one workgroup a sequence)
    if (threadIdx.x == 0) c.length[b] = paged_end(start, count, room);
  }
}

__global__ __launch_bounds__(kStoreThreads) void paged_length_kernel(PagedStore a) {
  const int64_t b = (int64_t)blockIdx.x * kStoreThreads + threadIdx.x;
  if (b >= a.c.B) return;
  const int64_t room = (int64_t)a.c.max_pages << a.c.page_log, start = a.start[b];
  a.c.length[b] = paged_end(start, paged_count(a.counts, b, a.T), room);
}

// Eight columns of a row of the pool, and its scale.
template <int CT>
struct Held : Cols<CT> {
  __device__ __forceinline__ void zero() { Cols<CT>::zero(); }
  __device__ __forceinline__ void load(const PagedCache& c, bool value, int64_t at, int d) {
    Cols<CT>::template load<true>((const typename XElem<CT>::T*)(value ? c.v : c.k) + at * c.row + d, 8);
  }
};
template <>
struct Held<CT_I8> {
  u32x2 w;
  float scale;
  __device__ __forceinline__ void zero() { w = (u32x2){0, 0}, scale = 0.0f; }
  __device__ __forceinline__ void load(const PagedCache& c, bool value, int64_t at, int d) {
    w = *(const u32x2*)((const uint8_t*)(value ? c.v : c.k) + at * c.row + d);
    scale = (value ? c.v_scale : c.k_scale)[at];
  }
  __device__ __forceinline__ void floats(float (&x)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (float)(int8_t)(w[j / 4] >> (8 * (j % 4))) * scale;
  }
};
template <>
struct Held<CT_E4M3> : Held<CT_I8> {
  __device__ __forceinline__ void floats(float (&x)[8]) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int v = (int)w[h];
      x[4 * h + 0] = __builtin_amdgcn_cvt_f32_fp8(v, 0) * scale;
      x[4 * h + 1] = __builtin_amdgcn_cvt_f32_fp8(v, 1) * scale;
      x[4 * h + 2] = __builtin_amdgcn_cvt_f32_fp8(v, 2) * scale;
      x[4 * h + 3] = __builtin_amdgcn_cvt_f32_fp8(v, 3) * scale;
    }
  }
};

// Positions start .. start + T - 1 of each sequence, zeros for those it does not hold.
template <int CT>
__global__ __launch_bounds__(kStoreThreads) void paged_read_kernel(PagedStore a) {
  const PagedCache& c = a.c;
  const int64_t b = blockIdx.x / a.parts, room = (int64_t)c.max_pages << c.page_log;
  const int part = blockIdx.x % a.parts, d = (threadIdx.x & (a.lanes - 1)) * 8, n = c.D - d;
  const int64_t start = a.start[b], held = c.length[b] < room ? c.length[b] : room;
  if (n <= 0) return;
  // A tile's rows are on their way before the one ahead of it is written, its page before that.
  const PagedTiles tiles(a);
  int32_t id;
  auto look_up = [&](int q) {
    int t, h;
    tiles.at(a, q, t, h);
    const int64_t pos = start + t;
    id = t >= a.T || pos < 0 || pos >= held ? -1 : c.table[b * c.max_pages + (pos >> c.page_log)];
  };
  Held<CT> k, v;
  auto fetch = [&](int q) {
    int t, h;
    tiles.at(a, q, t, h);
    k.zero(), v.zero();
    const int64_t at = paged_row_of(id, c.pages, start + t, h, c.Hk, c.page_log);
    if (at < 0) return;
    k.load(c, false, at, d);
    v.load(c, true, at, d);
  };
  look_up(part);
  fetch(part);
  look_up(part + a.parts);
  for (int q = part; q < tiles.n; q += a.parts) {
    const Held<CT> k0 = k, v0 = v;
    fetch(q + a.parts);
    look_up(q + 2 * a.parts);
    int t, h;
    tiles.at(a, q, t, h);
    if (t >= a.T) continue;
    const int64_t to = b * a.n_sb + (int64_t)t * a.n_st + (int64_t)h * a.n_sh + d;
    float x[8];
    k0.floats(x);
    store_cols8(a.k_out, a.xt, to, x, a.vec && n >= 8, n);
    v0.floats(x);
    store_cols8(a.v_out, a.xt, to, x, a.vec && n >= 8, n);
  }
}

template <int CT, int XT>
int launch_append_xt(const PagedStore& a, unsigned grid, hipStream_t st) {
  if (a.vec)
    paged_append_kernel<CT, XT, true><<<grid, kStoreThreads, 0, st>>>(a);
  else
    paged_append_kernel<CT, XT, false><<<grid, kStoreThreads, 0, st>>>(a);
  return check_launch();
}
template <int CT>
int launch_append_ct(const PagedStore& a, unsigned grid, hipStream_t st) {
  return a.xt == XT_F32   ? launch_append_xt<CT, XT_F32>(a, grid, st)
         : a.xt == XT_F16 ? launch_append_xt<CT, XT_F16>(a, grid, st)
                          : launch_append_xt<CT, XT_BF16>(a, grid, st);
}
template <int CT>
int launch_read_ct(const PagedStore& a, unsigned grid, hipStream_t st) {
  paged_read_kernel<CT><<<grid, kStoreThreads, 0, st>>>(a);
  return check_launch();
}

// Lanes of a vector, and how many workgroups share a sequence's vectors: each
// wave a few, up to about 6 workgroups a CU.
void plan(PagedStore& a) {
  a.lanes = 1;
  while (a.lanes * 8 < a.c.D) a.lanes <<= 1;
  const int64_t groups = kStoreThreads / a.lanes;
  a.tile = 1;
  while (a.tile < groups && a.tile < a.T) a.tile <<= 1;
  const int64_t heads = groups / a.tile, want = (a.T + a.tile - 1) / a.tile * ((a.c.Hk + heads - 1) / heads);
  const int64_t room = std::max<int64_t>(1, kStoreGroups / a.c.B);
  a.parts = (int)std::max<int64_t>(1, std::min(want, room));
}

// One row's splits joined: the maximum over their maxima and the sum of weights
// against it by every wave, then the means by their shares of that sum (no more
// than the values themselves, whatever their number), independent loads eight at
// a time.
template <int DP>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a) {
  constexpr int ND = DP / 4, NG = 256 / ND, U = 8;
  __shared__ __align__(16) f32x4 lds[NG][ND];
  const int R = a.rep * a.T, lane = threadIdx.x & 63, d = threadIdx.x % ND * 4, grp = threadIdx.x / ND;
  const int r = blockIdx.x, kvh = blockIdx.y, t = a.T > 1 ? r / a.rep : 0;
  const int64_t b = a.first + blockIdx.z;
  const int2 places = a.joins[r / a.tile_rows * a.n + (int)blockIdx.z];
  PagedSpan span;
  span.of<true>(a, b);
  const int used = places.y;
  if (used == 1) return;  // (written by the one workgroup)
  // the s-th of its partial results
  auto at = [&](int s) { return ((int64_t)kvh * a.places + paged_part_place(places.x + s, places.x)) * R + r; };
  float2 mine = make_float2(-__builtin_inff(), 0.0f);
  if (lane < used) mine = a.part_ml[at(lane)];
  f32x4 x[U], sum = (f32x4)(0.0f);
  float2 y[U];
  auto fetch = [&](int s0) {
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int s = min(s0 + k * NG, used - 1);
      x[k] = *(const f32x4*)(a.part_o + at(s) * DP + d);
      y[k] = a.part_ml[at(s)];
    }
  };
  fetch(grp);  // (on their way while the maximum is found)
  float top = mine.x;
  for (int s = lane + 64; s < used; s += 64) top = __builtin_fmaxf(top, a.part_ml[at(s)].x);
  top = wave_max(top);
  const float from = top == -__builtin_inff() ? 0.0f : top;
  // (a split that saw nothing adds nothing)
  auto weight = [&](float2 v) { return v.y != 0.0f ? __builtin_amdgcn_exp2f(v.x - from) * v.y : 0.0f; };
  float l = weight(mine);
  for (int s = lane + 64; s < used; s += 64) l += weight(a.part_ml[at(s)]);
  l = wave_sum(l);
  const float inv = l != 0.0f ? 1.0f / l : 0.0f;
  for (int s0 = grp; s0 < used; s0 += U * NG) {
    if (s0 != grp) fetch(s0);
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const float f = weight(y[k]);
      if (s0 + k * NG < used && y[k].y != 0.0f) sum += x[k] * (f * inv);
    }
  }
  lds[grp][threadIdx.x % ND] = sum;
  __syncthreads();
  if (grp) return;
#pragma unroll
  for (int k = 1; k < NG; ++k) sum += lds[k][threadIdx.x];
  if (span.last(t) < span.first(t, a.window)) sum = (f32x4)(0.0f);
  const int64_t out = b * a.o_sb + (int64_t)t * a.o_st + (int64_t)(kvh * a.rep + r - t * a.rep) * a.o_sh + d;
  if (d < a.c.D) store_y4(a.out, a.qt, out, sum, a.ovec && d + 4 <= a.c.D, a.c.D - d);
}

// Rounds of a wave's blocks up to which a workgroup takes a whole sequence, which
// saves the joining and, where a workgroup would do several sequences' parts in
// turn, the way to each one's first keys; what it costs is the wait for the longest.
// So: kPagedWhole rounds, and kPagedWholeFull more (kPagedWholeMost in all) for each
// time that the sequences' workgroups fill the chip.  8 key heads of 128 columns,
// e4m3, all sequences full / of lengths spread evenly / one full among short ones,
// whole against split in us: 16 x 512 positions 10.8 against 14.2 (all full), 16 x 1024
// 17.4, 14.9, 14.7 against 16.9, 14.1, 11.2; 64 x 2048 47, 35, 23 against 50, 45, 17;
// 256 x 2048 191, 121, 25 against 202, 127, 37; 256 x 4096 371, 219, 44 against 382,
// 217, 37.
constexpr int64_t kPagedWhole = 4, kPagedWholeFull = 12, kPagedWholeMost = 16;
// Rounds of all workgroups' blocks, in times the chip, from which a workgroup takes two
// sixteens of rows (half of that where workgroups of whole sequences fill the chip): the
// way to and from a part's blocks is 3 to 5 us longer with them, the blocks are read
// and converted half as often.  32 query heads over 8 x 128, two sixteens against one
// in us (bf16 queries, a pool of zeros): 16 x 1024 e4m3 positions, 8 tokens 33 against
// 20; 16 x 2048 38 against 37; 16 x 4096 47 against 49, bf16 63 against 62; 16 x 8192 69
// against 81, bf16 118 against 119; 64 x 512 e4m3 27 against 30; a chunk of 512 tokens
// over 2048 bf16 positions 47 against 77, over 8192 153 against 286, e4m3 145 against 212.
constexpr int64_t kPagedTiles = 8;
constexpr int64_t kPagedGroup = 512;   // sequences of a launch that are split at most (each workgroup scans their lengths)
constexpr int64_t kPagedRows = 65535;  // ... of one that are not: the grid's limit

struct PagedPlan {
  int DP, SB, tile_rows;
  int64_t rtiles, n, slots, places;
  bool joins;  // can a sequence have several parts?
};
// How many workgroups there are goes by the table's room: how much of it is
// filled is known on the device alone, where workgroups without a part leave
// at once.
PagedPlan paged_plan(int64_t B, int64_t T, int64_t R, int64_t Hk, int64_t D, int64_t room, int64_t window, int ct, bool wide) {
  PagedPlan p;
  p.DP = D <= 64 ? 64 : D <= 128 ? 128 : 256;
  p.SB = ct == XT_F32 ? 16 : 32;
  if (window > 0 && window < room - T) room = window + T;  // (what the tokens of a call can look at)
  const int64_t blocks = (room + p.SB - 1) / p.SB + (window > 0), fours = (blocks + kAttnWaves - 1) / kAttnWaves;
  const int64_t groups = 256 * paged_occupancy(ct, wide ? XT_F32 : XT_F16, p.DP);
  const int64_t most = 16 * paged_tiles(wide ? XT_F32 : XT_F16, p.DP), tiles = B * Hk * ((R + most - 1) / most);
  p.tile_rows = R > 16 && tiles * fours >= (tiles >= groups ? kPagedTiles / 2 : kPagedTiles) * groups ? (int)most : 16;
  p.rtiles = (R + p.tile_rows - 1) / p.tile_rows;
  const int64_t one = Hk * p.rtiles;
  p.n = std::min(B, kPagedGroup);
  p.n = std::max<int64_t>(1, std::min(p.n, ((int64_t)1 << 29) / (fours * kAttnWaves)));  // (all blocks fit an int, in whole parts too)
  p.slots = std::max<int64_t>(1, std::min(groups / one, p.n * fours));
  if (fours <= std::min(kPagedWhole + kPagedWholeFull * B * one / groups, kPagedWholeMost)) p.slots = 0, p.n = std::min(B, kPagedRows);
  p.places = 2 * p.slots;
  p.joins = p.slots > 1;
  return p;
}

int64_t round256(int64_t n) { return (n + 255) & ~(int64_t)255; }

}  // namespace

int64_t paged_attn_workspace_bytes(int64_t B, int64_t T, int64_t heads, int64_t Hk, int64_t D, int64_t room, int64_t window, int ct) {
  const int64_t R = heads / Hk * T;
  int64_t n = 0;
  for (bool wide : {false, true}) {  // (the queries' type is not known here)
    const PagedPlan p = paged_plan(B, T, R, Hk, D, room, window, ct, wide);
    const int64_t parts = Hk * R * p.places;
    if (p.joins) n = std::max(n, round256(parts * p.DP * 4) + round256(parts * 8) + p.rtiles * p.n * 8);
  }
  return n;
}

int launch_paged_attention(const PagedCall& c, hipStream_t st) {
  const int64_t Hk = c.c.Hk, rep = c.heads / Hk, R = rep * c.T, B = c.c.B;
  const PagedPlan p = paged_plan(B, c.T, R, Hk, c.c.D, (int64_t)c.c.max_pages << c.c.page_log, c.window, c.ct, c.qt == XT_F32);
  PagedArgs a{};
  a.c = c.c, a.q = c.q, a.start = c.start, a.counts = c.counts, a.out = c.out;
  a.q_sb = c.q_sb, a.q_st = c.q_st, a.q_sh = c.q_sh, a.o_sb = c.o_sb, a.o_st = c.o_st, a.o_sh = c.o_sh;
  a.window = c.window, a.T = (int)c.T, a.rep = (int)rep, a.qt = c.qt, a.tile_rows = p.tile_rows, a.slots = (int)p.slots, a.per_slot = p.slots ? 1.0f / (float)p.slots : 0.0f;
  a.places = (int)p.places;
  a.scale = c.scale * 1.44269504f;
  const int64_t eq = c.qt == XT_F32 ? 4 : 2;
  a.ovec = (uintptr_t)c.out % (4 * eq) == 0 && c.o_sb % 4 == 0 && c.o_st % 4 == 0 && c.o_sh % 4 == 0;
  if (p.joins) {
    a.part_o = (float*)c.ws;
    a.part_ml = (float2*)((uint8_t*)c.ws + round256(Hk * R * p.places * p.DP * 4));
    a.joins = (int2*)((uint8_t*)a.part_ml + round256(Hk * R * p.places * 8));
  }
  for (a.first = 0; a.first < B; a.first += p.n) {
    a.n = (int)std::min(p.n, B - a.first);
    const dim3 grid((unsigned)(Hk * p.rtiles), (unsigned)(p.slots ? p.slots : a.n));
    int rc = c.ct == XT_F32    ? launch_paged_attn_f32(a, p.DP, grid, st)
             : c.ct == XT_F16  ? launch_paged_attn_f16(a, p.DP, grid, st)
             : c.ct == XT_BF16 ? launch_paged_attn_bf16(a, p.DP, grid, st)
             : c.ct == CT_I8   ? launch_paged_attn_i8(a, p.DP, grid, st)
                               : launch_paged_attn_e4m3(a, p.DP, grid, st);
    if (rc) return rc;
    if (!p.joins) continue;
    const dim3 joins((unsigned)R, (unsigned)Hk, (unsigned)a.n);
    if (p.DP == 64)
      paged_join_kernel<64><<<joins, 256, 0, st>>>(a);
    else if (p.DP == 128)
      paged_join_kernel<128><<<joins, 256, 0, st>>>(a);
    else
      paged_join_kernel<256><<<joins, 256, 0, st>>>(a);
    if ((rc = check_launch())) return rc;
  }
  return 0;
}

int launch_paged_append(const PagedStore& c, hipStream_t st) {
  PagedStore a = c;
  plan(a);
  const int64_t es = a.xt == XT_F32 ? 4 : 2;
  auto vec = [&](const void* p) { return (uintptr_t)p % 16 == 0; };
  a.vec = a.c.D % 8 == 0 && vec(a.kn) && vec(a.vn) && a.n_sb * es % 16 == 0 && a.n_st * es % 16 == 0 && a.n_sh * es % 16 == 0;
  const bool own = a.start == a.c.length;  // the length is read by every workgroup: moved by one that no other reads after
  if (own && a.T * a.c.Hk <= kStoreAlone) a.parts = 1;
  a.set_length = !own || a.parts == 1;
  const int64_t B = a.c.B, most = std::max<int64_t>(1, kLaunchThreads / kStoreThreads / a.parts);
  for (int64_t b0 = 0; b0 < B; b0 += most) {
    PagedStore s = a;
    s.c.B = std::min(most, B - b0);
    s.c.table += b0 * a.c.max_pages, s.c.length += b0, s.start += b0;
    if (s.counts) s.counts += b0;
    s.kn = (const char*)a.kn + b0 * a.n_sb * es, s.vn = (const char*)a.vn + b0 * a.n_sb * es;
    const unsigned grid = (unsigned)(s.c.B * s.parts);
    const int rc = a.ct == XT_F32    ? launch_append_ct<XT_F32>(s, grid, st)
                   : a.ct == XT_F16  ? launch_append_ct<XT_F16>(s, grid, st)
                   : a.ct == XT_BF16 ? launch_append_ct<XT_BF16>(s, grid, st)
                   : a.ct == CT_I8   ? launch_append_ct<CT_I8>(s, grid, st)
                                     : launch_append_ct<CT_E4M3>(s, grid, st);
    if (rc) return rc;
  }
  if (a.set_length) return 0;
  paged_length_kernel<<<(unsigned)((B + kStoreThreads - 1) / kStoreThreads), kStoreThreads, 0, st>>>(a);
  return check_launch();
}

int launch_paged_read(const PagedStore& c, hipStream_t st) {
  PagedStore a = c;
  plan(a);
  const int64_t es = a.xt == XT_F32 ? 4 : 2, n = 16 / es;
  a.vec = (uintptr_t)a.k_out % 16 == 0 && (uintptr_t)a.v_out % 16 == 0 && a.n_sb % n == 0 && a.n_st % n == 0 && a.n_sh % n == 0;
  const int64_t B = a.c.B, most = std::max<int64_t>(1, kLaunchThreads / kStoreThreads / a.parts);
  for (int64_t b0 = 0; b0 < B; b0 += most) {
    PagedStore s = a;
    s.c.B = std::min(most, B - b0);
    s.c.table += b0 * a.c.max_pages, s.c.length += b0, s.start += b0;
    s.k_out = (char*)a.k_out + b0 * a.n_sb * es, s.v_out = (char*)a.v_out + b0 * a.n_sb * es;
    const unsigned grid = (unsigned)(s.c.B * s.parts);
    const int rc = a.ct == XT_F32    ? launch_read_ct<XT_F32>(s, grid, st)
                   : a.ct == XT_F16  ? launch_read_ct<XT_F16>(s, grid, st)
                   : a.ct == XT_BF16 ? launch_read_ct<XT_BF16>(s, grid, st)
                   : a.ct == CT_I8   ? launch_read_ct<CT_I8>(s, grid, st)
                                     : launch_read_ct<CT_E4M3>(s, grid, st);
    if (rc) return rc;
  }
  return 0;
}

}  // namespace sbq
