// sbq_paged.h - the paged cache of several sequences: what its kernels share,
// and the attention over it, included by the files that instantiate it.
//
// The pool holds pages of `page` positions (a power of two, 16 to 1024) of
// every key head: k, v [pages][Hk][page][row], row the D columns rounded up
// to 16 (those past D are zero), so that one head's positions of a page lie
// side by side and every row takes 16-byte loads.  8-bit pools have one fp32
// scale for each row, [pages][Hk][page].  Sequence b's position p stands in
// page table[b][p / page], row p % page; a table entry that names no page of
// the pool holds nothing.
#pragma once

#include "sbq_attn.h"
#include "sbq_common.h"
#include "sbq_launch.h"

namespace sbq {

// Cache element types beside XType's first three.
enum { CT_I8 = 3, CT_E4M3 = 4 };
constexpr bool is_8bit(int ct) { return ct >= CT_I8; }
constexpr int ct_bytes(int ct) { return ct == XT_F32 ? 4 : is_8bit(ct) ? 1 : 2; }

__device__ __forceinline__ bool valid_page(const PagedCache& c, int32_t id) { return id >= 0 && id < c.pages; }

// Tokens of a sequence's T that are there.
__device__ __forceinline__ int64_t paged_count(const int64_t* counts, int64_t b, int64_t T) {
  if (!counts) return T;
  const int64_t n = counts[b];
  return n < 0 ? 0 : n > T ? T : n;
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------
// out[b,t,h] = sum_p softmax_p(scale q[b,t,h] . k[b,p,h/rep]) v[b,p,h/rep] over
// the positions p that token t, at start[b] + t, sees: those up to its own,
// below the length, within the window, in a page of the pool.
//
// The products are attn_kernel's (sbq_attn.h): S^T = K Q^T puts the rep * T
// rows of a key head in the matrix instruction's columns and leaves lane (g, c)
// four slots of row c, the operand that O^T = V^T P^T needs.  A wave walks
// blocks of SB positions, loads their keys and values straight to registers
// and keeps a running maximum and sum; the blocks of a sequence's length are
// dealt in turn to the waves of its `splits` workgroups, so that the split
// follows the length on the device and no call depends on a length known to
// the host.  The cache's bytes, read once, bound it.
//
// Types of the products:
//   fp32 cache: fp32 (16x16x4).
//   fp16, bf16 cache with its own type's queries: that type (16x16x32); fp32
//     queries in pieces of it (2 of fp16, each row scaled by a power of two, 3
//     of bf16), which hold 22 and 24 bits.
//   8-bit cache: its codes are exact in fp16; queries in fp16 likewise, one
//     piece of 2-byte ones (bf16: each row scaled by a power of two), two of
//     fp32.  A position's scales multiply its score and its weight.
// The weights are rounded for the product with V: one piece of fp16 (against
// 2^14 at the maximum, so that one 2^-28 of it keeps its bits) or two of bf16
// with 2-byte queries, as many pieces as the queries' with fp32 ones.
struct PagedArgs {
  PagedCache c;
  const void* q;
  const int64_t *start, *counts;
  void* out;
  float* part_o;    // [B][Hk][R][splits][DP]
  float2* part_ml;  // [B][Hk][R][splits]
  int64_t q_sb, q_st, q_sh, o_sb, o_st, o_sh, window, first;
  int T, rep, splits, rtiles, qt;
  float scale;  // times log2(e)
  bool qvec, ovec;
};

// What the rows of one sequence see; a row sees lo..hi, none where hi < lo.
struct PagedSpan {
  int64_t start;
  int count, held;
  __device__ __forceinline__ PagedSpan(const PagedArgs& a, int64_t b) {
    const int64_t room = (int64_t)a.c.max_pages << a.c.page_log, len = a.c.length[b];
    count = (int)paged_count(a.counts, b, a.T);
    start = a.start ? a.start[b] : len - count;
    start = min(max(start, -((int64_t)1 << 40)), (int64_t)1 << 40);  // (past every position)
    held = (int)(len < 0 ? 0 : len < room ? len : room);
  }
  __device__ __forceinline__ void of(const PagedArgs& a, int t, int& lo, int& hi) const {
    const int64_t pos = start + t, from = a.window > 0 ? pos - a.window + 1 : 0;
    hi = t < count ? (int)(pos < held ? pos < -1 ? -1 : pos : held - 1) : -1;
    lo = (int)(from < 0 ? 0 : from < held ? from : held);
  }
  // first and last position that any row of tokens t0..t1 sees
  __device__ __forceinline__ void all(const PagedArgs& a, int t0, int t1, int& lo, int& hi) const {
    int x;
    of(a, t0, lo, x);
    of(a, min(t1, count - 1), x, hi);
    if (count <= t0) hi = -1;
  }
};

template <int CT>
struct PagedMath : AttnMath<CT == XT_BF16 ? XT_BF16 : XT_F16> {
  typedef typename XElem<CT == XT_BF16 ? XT_BF16 : XT_F16>::T T;
};

// 8 columns of an 8-bit row in two words to fp16, in the order column_of().
template <int CT>
__device__ __forceinline__ f16x8 codes_f16(uint32_t w0, uint32_t w1) {
  u32x4 t;
  if constexpr (CT == CT_I8) {  // 1024 + (q + 128) in fp16's bits, less 1152
    w0 ^= 0x80808080u, w1 ^= 0x80808080u;
    t[0] = (w0 & 0x00ff00ffu) | 0x64006400u, t[1] = (w0 >> 8 & 0x00ff00ffu) | 0x64006400u;
    t[2] = (w1 & 0x00ff00ffu) | 0x64006400u, t[3] = (w1 >> 8 & 0x00ff00ffu) | 0x64006400u;
    const f16x2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t x = t[j];  // (a bit cast of a vector's element itself reads the first one)
      t[j] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, x) - off);
    }
  } else {
    t[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w0, 1.0f, false));
    t[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w0, 1.0f, true));
    t[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w1, 1.0f, false));
    t[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w1, 1.0f, true));
  }
  return __builtin_bit_cast(f16x8, t);
}
template <int CT>
__device__ __forceinline__ constexpr int column_of(int j) {
  return CT == CT_I8 ? (j & 4) | (j & 1) << 1 | (j >> 1 & 1) : j;
}

// Bytes e of the words of two positions to fp16, side by side.
template <int CT>
__device__ __forceinline__ uint32_t pair_i8(uint32_t hi, uint32_t lo, int e) {
  const uint32_t sel = 0x0c000c00u | (uint32_t)(4 + e) << 16 | (uint32_t)e;
  const uint32_t t = __builtin_amdgcn_perm(hi, lo, sel) | 0x64006400u;
  const f16x2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, t) - off);
}

// N values split into pieces of T, the first the nearest value, each next the
// nearest to what is left.
template <int N, class T>
__device__ __forceinline__ void pieces(float x, T (&to)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    to[i] = (T)x;
    x -= (float)to[i];
  }
}

// Eight consecutive columns of a query row.
__device__ __forceinline__ void load_q8(const PagedArgs& a, int64_t at, int d, float (&x)[8]) {
  if (a.qvec && d + 8 <= a.c.D) {
    if (a.qt == XT_F32)
      load8_f32_vec<XT_F32>((const float*)a.q + at + d, x);
    else if (a.qt == XT_F16)
      load8_f32_vec<XT_F16>((const _Float16*)a.q + at + d, x);
    else
      load8_f32_vec<XT_BF16>((const __bf16*)a.q + at + d, x);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = d + j < a.c.D ? load_elem(a.q, a.qt, at + d + j) : 0.0f;
  }
}

// CT: the cache's type, NQ: pieces of a query (fp32 products: 1), NP: pieces of
// a weight, DP: columns the registers hold (64, 128, 256), EXACT: row == DP.
template <int CT, int NQ, int NP, int DP, bool EXACT>
__global__ __launch_bounds__(kAttnWaves * 64, DP == 256 ? 1 : 2) void paged_attn_kernel(PagedArgs a) {
  constexpr bool B8 = is_8bit(CT), F32 = CT == XT_F32;
  constexpr int ES = ct_bytes(CT), E = 16 / ES, NCH = DP / (4 * E);  // columns in 16 bytes, key loads of a lane's row
  constexpr int SUB = F32 ? 1 : B8 ? 4 : 2, SB = 16 * SUB;
  constexpr int EV = E < DP / 16 ? E : DP / 16, DB = DP / (16 * EV), NF = DP / 16;  // columns of a value load, loads
  constexpr int NFR = DP / 32;                                                       // 16x16x32 steps of a score
  constexpr int HP = DP < 128 ? DP : 128, OLD = HP + 4;
  constexpr float kNone = -__builtin_inff();
  typedef typename PagedMath<CT>::T M;
  typedef typename PagedMath<CT>::V MV;
  typedef uint32_t KV __attribute__((ext_vector_type(4)));
  typedef uint32_t VW __attribute__((ext_vector_type(EV * ES / 4)));
  __shared__ __align__(16) float lds_o[kAttnWaves * 16 * OLD];
  __shared__ float lds_m[kAttnWaves][16], lds_l[kAttnWaves][16];

  const PagedCache& pc = a.c;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
  unsigned bid = blockIdx.x;
  const int kvh = bid % pc.Hk;
  bid /= pc.Hk;
  const int rtile = bid % a.rtiles;
  bid /= a.rtiles;
  const int split = bid % a.splits;
  const int64_t b = a.first + bid / a.splits;
  const int R = a.rep * a.T, row0 = rtile * 16;

  const PagedSpan span(a, b);
  int lo_min, hi_max;
  span.all(a, row0 / a.rep, min(row0 + 15, R - 1) / a.rep, lo_min, hi_max);
  const int b0 = lo_min / SB, blocks = hi_max >= lo_min ? hi_max / SB + 1 - b0 : 0;
  const int used = max(1, min(a.splits, (blocks + kAttnWaves - 1) / kAttnWaves));
  if (split >= used) return;

  const int row = min(row0 + c, R - 1), tok = row / a.rep;
  int lo, hi;
  span.of(a, tok, lo, hi);
  // what every row that sees anything sees
  int lo_max = lo, hi_min = hi < lo ? INT32_MAX : hi;
  if (hi < lo) lo_max = 0;
  if (a.T > 1) {
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
      lo_max = max(lo_max, __shfl_xor(lo_max, o, 64));
      hi_min = min(hi_min, __shfl_xor(hi_min, o, 64));
    }
  }
  lo_max = __builtin_amdgcn_readfirstlane(lo_max), hi_min = __builtin_amdgcn_readfirstlane(hi_min);

  // the lane's share of its row of Q
  const int64_t q_at = b * a.q_sb + (int64_t)tok * a.q_st + (int64_t)(kvh * a.rep + row % a.rep) * a.q_sh;
  MV qm[F32 ? 1 : NFR][NQ];
  float qf[F32 ? NCH : 1][4];
  float factor = a.scale;
  if constexpr (F32) {
#pragma unroll
    for (int ch = 0; ch < NCH; ch += 2) {  // (two loads of four columns each lie 16 apart)
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int d = (ch + k) * 16 + g * 4 + j;
          qf[ch + k][j] = d < pc.D ? load_elem(a.q, a.qt, q_at + d) : 0.0f;
        }
    }
  } else {
    float x[NFR][8];
    constexpr bool SCALED = (B8 || CT == XT_F16) && (NQ > 1 || B8);
    float most = 0.0f;
#pragma unroll
    for (int f = 0; f < NFR; ++f) {
      const int d = B8 ? f / 2 * 64 + g * 16 + f % 2 * 8 : f * 32 + g * 8;
      load_q8(a, q_at, d, x[f]);
      if constexpr (SCALED) {
#pragma unroll
        for (int j = 0; j < 8; ++j) most = __builtin_fmaxf(most, __builtin_fabsf(x[f][j]));
      }
    }
    if constexpr (SCALED) {
      most = __builtin_fmaxf(most, __shfl_xor(most, 16, 64));
      most = __builtin_fmaxf(most, __shfl_xor(most, 32, 64));
      const int e = row_scale_exp(most);
      factor = __builtin_ldexpf(factor, -e);
#pragma unroll
      for (int f = 0; f < NFR; ++f)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[f][j] = __builtin_ldexpf(x[f][j], e);
    }
#pragma unroll
    for (int f = 0; f < NFR; ++f)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        M p[NQ];
        pieces(x[f][column_of<CT>(j)], p);
#pragma unroll
        for (int i = 0; i < NQ; ++i) qm[f][i][j] = p[i];
      }
  }

  f32x4 o[NF];
#pragma unroll
  for (int f = 0; f < NF; ++f) o[f] = (f32x4)(0.0f);
  float m = kNone, l = 0.0f;
  float vref = 1.17549435e-38f;  // 8-bit: O's unit, the largest value scale that the row saw so far

  const int32_t* const table = pc.table + b * pc.max_pages;
  const int page_mask = (1 << pc.page_log) - 1, stride = used * kAttnWaves;
  // lane offsets in bytes inside a page of a head: its key row (c) and value rows (4g + j)
  const uint32_t row_bytes = pc.row * ES, k_lane = c * row_bytes + g * 16, v_lane = 4 * g * row_bytes + c * EV * ES;
  const int64_t page_bytes = (int64_t)row_bytes << pc.page_log;

  for (int n = split * kAttnWaves + w; n < blocks; n += stride) {
    const int s0 = (b0 + n) * SB;
    KV kf[SUB][NCH];
    VW vf[4 * SUB][DB];
    f32x4 ks[B8 ? SUB : 1], vs[B8 ? SUB : 1];
    uint32_t held = 0;  // sub-blocks whose page is there
#pragma unroll
    for (int st = 0; st < SUB; ++st) {
      const int s = s0 + st * 16, page = s >> pc.page_log;
      int32_t id = page < pc.max_pages ? table[page] : -1;
      if (valid_page(pc, id)) held |= 1u << st;
      else id = 0;
      const int64_t at = ((int64_t)id * pc.Hk + kvh) * page_bytes + (int64_t)(s & page_mask) * row_bytes;
      const char *const kp = (const char*)pc.k + at, *const vp = (const char*)pc.v + at;
#pragma unroll
      for (int ch = 0; ch < NCH; ++ch) {
        if (EXACT || ch * 4 * E + g * E < pc.row)
          kf[st][ch] = *(const KV*)(kp + k_lane + ch * 64);
        else
          kf[st][ch] = (KV)(0u);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          if (EXACT || db * 16 * EV + c * EV < pc.row)
            vf[st * 4 + j][db] = *(const VW*)(vp + v_lane + j * row_bytes + db * 16 * EV * ES);
          else
            vf[st * 4 + j][db] = (VW)(0u);
        }
      if constexpr (B8) {
        const int64_t sc = (((int64_t)id * pc.Hk + kvh) << pc.page_log) + (s & page_mask) + 4 * g;
        ks[st] = *(const f32x4*)(pc.k_scale + sc);
        vs[st] = *(const f32x4*)(pc.v_scale + sc);
      }
    }
    const bool full = held == (1u << SUB) - 1 && s0 >= lo_max && s0 + SB - 1 <= hi_min;

    // scores, in powers of two
    float p[SUB][4];
#pragma unroll
    for (int st = 0; st < SUB; ++st) {
      f32x4 s = (f32x4)(0.0f);
      if constexpr (F32) {
        f32x4 t[4] = {(f32x4)(0.0f), (f32x4)(0.0f), (f32x4)(0.0f), (f32x4)(0.0f)};
#pragma unroll
        for (int ch = 0; ch < NCH; ++ch) {
          const f32x4 kk = __builtin_bit_cast(f32x4, kf[st][ch]);
#pragma unroll
          for (int j = 0; j < 4; ++j) t[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(kk[j], qf[ch][j], t[j], 0, 0, 0);
        }
        s = (t[0] + t[1]) + (t[2] + t[3]);
      } else {
        f32x4 t[NQ];
#pragma unroll
        for (int i = 0; i < NQ; ++i) t[i] = (f32x4)(0.0f);
#pragma unroll
        for (int f = 0; f < NFR; ++f) {
          MV kk;
          if constexpr (B8)
            kk = codes_f16<CT>(kf[st][f / 2][f % 2 * 2], kf[st][f / 2][f % 2 * 2 + 1]);
          else
            kk = __builtin_bit_cast(MV, kf[st][f]);
#pragma unroll
          for (int i = 0; i < NQ; ++i) t[i] = PagedMath<CT>::mfma(kk, qm[f][i], t[i]);
        }
#pragma unroll
        for (int i = NQ - 1; i > 0; --i) t[i - 1] += t[i];
        s = t[0];
      }
#pragma unroll
      for (int v = 0; v < 4; ++v) p[st][v] = s[v] * (B8 ? factor * ks[st][v] : factor);
    }

    uint32_t seen = ~0u;  // bit st * 4 + v: the lane's row sees that position
    if (!full) {
      seen = 0;
#pragma unroll
      for (int st = 0; st < SUB; ++st)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const int s = s0 + st * 16 + 4 * g + v;
          if (s >= lo && s <= hi && (held >> st & 1)) seen |= 1u << (st * 4 + v);
        }
    }
    float mx = kNone;
#pragma unroll
    for (int st = 0; st < SUB; ++st)
#pragma unroll
      for (int v = 0; v < 4; ++v) mx = full || (seen >> (st * 4 + v) & 1) ? __builtin_fmaxf(mx, p[st][v]) : mx;
    mx = reference<XT_F16, !F32 && CT != XT_BF16>(mx);
    if (__any(mx > m)) {
      mx = __builtin_fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = __builtin_fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float up = __builtin_fmaxf(m, mx), alpha = up == kNone ? 1.0f : __builtin_amdgcn_exp2f(m - up);
      m = up;
      l *= alpha;
#pragma unroll
      for (int f = 0; f < NF; ++f) o[f] *= alpha;
    }
    const float from = m == kNone ? 0.0f : m;
#pragma unroll
    for (int st = 0; st < SUB; ++st)
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        float e = __builtin_amdgcn_exp2f(p[st][v] - from);
        if (!full) e = seen >> (st * 4 + v) & 1 ? e : 0.0f;
        p[st][v] = e;
        l += e;
      }

    if constexpr (B8) {  // the weights times the values' scales, in units of vref
      float top = 0.0f;
#pragma unroll
      for (int st = 0; st < SUB; ++st)
#pragma unroll
        for (int v = 0; v < 4; ++v)
          top = finite(vs[st][v]) && (full || (seen >> (st * 4 + v) & 1)) ? __builtin_fmaxf(top, vs[st][v]) : top;
      if (__any(top > vref)) {
        top = __builtin_fmaxf(top, __shfl_xor(top, 16, 64));
        top = __builtin_fmaxf(top, __shfl_xor(top, 32, 64));
        const float up = __builtin_fmaxf(vref, top), alpha = vref / up;
        vref = up;
#pragma unroll
        for (int f = 0; f < NF; ++f) o[f] *= alpha;
      }
      const float inv = 1.0f / vref;
#pragma unroll
      for (int st = 0; st < SUB; ++st)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float e = p[st][v] * (vs[st][v] * inv);
          p[st][v] = full || (seen >> (st * 4 + v) & 1) ? e : 0.0f;
        }
    }

    // infinities and NaN in values that not every row sees (codes have none)
    bool odd = false;
    if constexpr (!B8) {
      if (!full) {
#pragma unroll
        for (int j = 0; j < 4 * SUB; ++j)
#pragma unroll
          for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int e = 0; e < EV * ES / 4; ++e) {
              if constexpr (F32)
                odd |= !finite(__uint_as_float(vf[j][db][e]));
              else
                odd |= Odd2<CT>::any(vf[j][db][e]);
            }
        odd = __any(odd);
      }
    }

    // O^T += V^T P^T
    if constexpr (F32) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int e = 0; e < EV; ++e) {
            float x = __uint_as_float(vf[j][db][e]);
            if (odd) {
#pragma unroll 1
              for (int kind = 0; kind < 3; ++kind) {
                const f32x4 cnt = __builtin_amdgcn_mfma_f32_16x16x4f32(odd_one(x, kind), seen >> j & 1 ? 1.0f : 0.0f,
                                                                       (f32x4)(0.0f), 0, 0, 0);
#pragma unroll
                for (int v = 0; v < 4; ++v)
                  if (cnt[v] > 0.0f) o[db * EV + e][v] += odd_value(kind);
              }
              x = finite(x) ? x : 0.0f;
            }
            o[db * EV + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(x, p[0][j], o[db * EV + e], 0, 0, 0);
          }
    } else {
#pragma unroll
      for (int h = 0; h < SUB / 2; ++h) {  // 32 positions a step
        MV pf[NP];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          M x[NP];
          pieces(p[h * 2 + (j >> 2)][j & 3], x);
#pragma unroll
          for (int i = 0; i < NP; ++i) pf[i][j] = x[i];
        }
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          VW vw[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            vw[j] = vf[h * 8 + j][db];
            if constexpr (CT == CT_I8) vw[j] ^= 0x80808080u;
          }
#pragma unroll
          for (int e0 = 0; e0 < EV; e0 += 2) {  // two columns at a time
            u32x4 t[2];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if constexpr (CT == CT_I8) {
                t[0][j] = pair_i8<CT>(vw[2 * j + 1][e0 / 4], vw[2 * j][e0 / 4], e0 % 4);
                t[1][j] = pair_i8<CT>(vw[2 * j + 1][e0 / 4], vw[2 * j][e0 / 4], e0 % 4 + 1);
              } else {
                uint32_t x, y;
                if constexpr (CT == CT_E4M3) {
                  x = __builtin_bit_cast(uint32_t, e0 % 4 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)vw[2 * j][e0 / 4], 1.0f, true)
                                                          : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)vw[2 * j][e0 / 4], 1.0f, false));
                  y = __builtin_bit_cast(uint32_t, e0 % 4 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)vw[2 * j + 1][e0 / 4], 1.0f, true)
                                                          : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)vw[2 * j + 1][e0 / 4], 1.0f, false));
                } else {
                  x = vw[2 * j][e0 / 2], y = vw[2 * j + 1][e0 / 2];
                }
                t[0][j] = __builtin_amdgcn_perm(y, x, 0x05040100u);
                t[1][j] = __builtin_amdgcn_perm(y, x, 0x07060302u);
              }
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int f = db * EV + e0 + k;
              if constexpr (!B8) {
                if (odd) {
#pragma unroll 1
                  for (int kind = 0; kind < 3; ++kind) {
                    u32x4 ones;
                    MV sees;
#pragma unroll
                    for (int j = 0; j < 4; ++j) ones[j] = Odd2<CT>::ones(t[k][j], kind);
#pragma unroll
                    for (int j = 0; j < 8; ++j) sees[j] = (M)(seen >> (h * 8 + j) & 1 ? 1.0f : 0.0f);
                    const f32x4 cnt = PagedMath<CT>::mfma(__builtin_bit_cast(MV, ones), sees, (f32x4)(0.0f));
#pragma unroll
                    for (int v = 0; v < 4; ++v)
                      if (cnt[v] > 0.0f) o[f][v] += odd_value(kind);
                  }
#pragma unroll
                  for (int j = 0; j < 4; ++j) t[k][j] = Odd2<CT>::finite(t[k][j]);
                }
              }
              const MV vt = __builtin_bit_cast(MV, t[k]);
#pragma unroll
              for (int i = 0; i < NP; ++i) o[f] = PagedMath<CT>::mfma(vt, pf[i], o[f]);
            }
          }
        }
      }
    }
  }

  // the workgroup's waves joined
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (g == 0) lds_m[w][c] = m, lds_l[w][c] = l;
  const float unit = B8 ? vref : 1.0f;
#pragma unroll
  for (int h0 = 0; h0 < DP; h0 += HP) {
    if (h0) __syncthreads();  // (lds_o is free)
    float* const to = lds_o + (w * 16 + c) * OLD;
#pragma unroll
    for (int db = h0 / (16 * EV); db < (h0 + HP) / (16 * EV); ++db)
#pragma unroll
      for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int e = 0; e < EV; ++e) to[db * 16 * EV - h0 + (4 * g + v) * EV + e] = o[db * EV + e][v] * unit;
    __syncthreads();
    for (int u = threadIdx.x; u < 16 * (HP / 4); u += kAttnWaves * 64) {
      const int rr = u / (HP / 4), d = h0 + u % (HP / 4) * 4;
      if (row0 + rr >= R) continue;
      float top = kNone;
#pragma unroll
      for (int k = 0; k < kAttnWaves; ++k) top = __builtin_fmaxf(top, lds_m[k][rr]);
      const float from = top == kNone ? 0.0f : top;
      f32x4 sum = (f32x4)(0.0f);
      float ls = 0.0f;
#pragma unroll
      for (int k = 0; k < kAttnWaves; ++k) {
        const float f = __builtin_amdgcn_exp2f(lds_m[k][rr] - from);
        if (lds_l[k][rr] != 0.0f) {  // (a wave that saw nothing adds nothing)
          sum += *(const f32x4*)(lds_o + (k * 16 + rr) * OLD + d - h0) * f;
          ls += lds_l[k][rr] * f;
        }
      }
      const int r = row0 + rr, t = r / a.rep;
      if (used > 1) {
        const int64_t at = ((b * pc.Hk + kvh) * R + r) * a.splits + split;
        *(f32x4*)(a.part_o + at * DP + d) = sum;
        if (d == 0) a.part_ml[at] = make_float2(top, ls);
      } else {
        int row_lo, row_hi;
        span.of(a, t, row_lo, row_hi);
        const float inv = ls != 0.0f && row_hi >= row_lo ? 1.0f / ls : 0.0f;
        if (row_hi < row_lo) sum = (f32x4)(0.0f);
        const int64_t out = b * a.o_sb + (int64_t)t * a.o_st + (int64_t)(kvh * a.rep + r % a.rep) * a.o_sh + d;
        if (d < pc.D) store_y4(a.out, a.qt, out, sum * inv, a.ovec && d + 4 <= pc.D, pc.D - d);
      }
    }
  }
}

template <int CT, int NQ, int NP>
int launch_paged_types(const PagedArgs& a, int DP, unsigned grid, hipStream_t st) {
  constexpr int threads = kAttnWaves * 64;
  const bool exact = a.c.row == DP;
  if (DP == 64)
    exact ? paged_attn_kernel<CT, NQ, NP, 64, true><<<grid, threads, 0, st>>>(a)
          : paged_attn_kernel<CT, NQ, NP, 64, false><<<grid, threads, 0, st>>>(a);
  else if (DP == 128)
    exact ? paged_attn_kernel<CT, NQ, NP, 128, true><<<grid, threads, 0, st>>>(a)
          : paged_attn_kernel<CT, NQ, NP, 128, false><<<grid, threads, 0, st>>>(a);
  else
    exact ? paged_attn_kernel<CT, NQ, NP, 256, true><<<grid, threads, 0, st>>>(a)
          : paged_attn_kernel<CT, NQ, NP, 256, false><<<grid, threads, 0, st>>>(a);
  return check_launch();
}

int launch_paged_attn_f32(const PagedArgs& a, int DP, unsigned grid, hipStream_t st);
int launch_paged_attn_f16(const PagedArgs& a, int DP, unsigned grid, hipStream_t st);
int launch_paged_attn_bf16(const PagedArgs& a, int DP, unsigned grid, hipStream_t st);
int launch_paged_attn_i8(const PagedArgs& a, int DP, unsigned grid, hipStream_t st);
int launch_paged_attn_e4m3(const PagedArgs& a, int DP, unsigned grid, hipStream_t st);

}  // namespace sbq
