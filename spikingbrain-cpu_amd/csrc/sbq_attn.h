// sbq_attn.h - attention of a few query tokens over a cache of keys and values
// and over each other's (a tree of drafted tokens): the kernel and its
// arguments, included by the files that instantiate it.
//
//   o[t,h] = sum_s softmax_s(scale * q[t,h] . k[s,h/rep]) v[s,h/rep]
//
// over the cached slots whose position lies in (q_pos[t] - window, q_pos[t]]
// and the drafts that tree[t] names.  The cache is read once, which is what
// bounds it at a few tokens; the rep = H / Hk query heads of a key head and
// the T tokens make R = rep * T rows that share every key and value.
//
// A wave owns RT tiles of 16 rows and walks blocks of slots.  Both products
// put the rows in the matrix instruction's columns: S^T = K Q^T leaves lane
// (g, c) the scores of row c and four slots 4g + v, which is exactly the
// operand that O^T = V^T P^T needs (k = the lane group's own slots), so the
// softmax's weights go from one product to the other in their registers, a
// row's running maximum and sum belong to its lanes, and its rescaling needs
// no lane crossing.  V^T's operand holds one column of V for the lane
// group's slots: a lane loads 16 bytes of a V row per slot and the 2-byte
// types pair up two slots with one byte permute per register.  K and V go
// from memory straight to registers; LDS only joins the waves.
//
// M16: 2-byte cache and queries of one type on 16x16x32, the weights rounded
// to that type (half a step each, averaged over the slots of a sum, see
// reference(); the sum of weights itself stays in fp32).  Otherwise all products are fp32
// (16x16x4), whatever the cache holds.
//
// The blocks are dealt in turn to the waves of all `splits` workgroups of a
// row tile, so that a cache that is filled only at its front still keeps
// every workgroup busy; a block that no row sees is left out after a look at
// its positions.  A decode step of 32 heads over 2048 slots of 8 x 128 fp32
// takes 10 us and 4.3 for the joining (kernel trace; the latency of a few loads
// after each other; 3.3 us for the bytes), over 65536 bf16 47 us with the
// joining (replayed graph), 5.7 TB/s.
#pragma once

#include "sbq_common.h"
#include "sbq_dma.h"
#include "sbq_launch.h"

namespace sbq {

constexpr int kAttnWaves = 4;
constexpr int kTileSlots = 64, kTileWaves = 8, kTileBufs = 4;  // attn_tile_kernel: slots per step, tiles in LDS

template <int N>
struct Const {
  static constexpr int value = N;
};

struct AttnArgs {
  const void *q, *k, *v, *kn, *vn;
  const int64_t *slot_pos, *q_pos;
  const uint8_t* tree;          // [T][tree_ld], null: draft j is seen by t >= j
  void* out;
  float* part_o;                // [Hk*R][splits][DP]; null: a workgroup has the whole row
  float2* part_ml;              // [Hk*R][splits]
  float* scores;                // [Hk*R][score_ld] of the cached slots, where they are kept for the slots' weights
  float2* row_ml;               // [Hk*R] (maximum, 1 / sum), where the slots' weights are wanted
  int64_t q_st, q_sh, k_ss, k_sh, n_ss, n_sh, o_st, o_sh, tree_ld, score_ld;
  int64_t window;               // 0: none
  int T, Hk, rep, D, slots, Tn, splits, rtiles, qt;
  float scale;                  // times log2(e), >= 0 (`neg`: q is negated instead)
  bool neg, qvec, ovec;         // q's rows take 16-byte loads, out's rows stores of 4 elements
};

__device__ __forceinline__ void wait_lds() { __builtin_amdgcn_s_waitcnt(0xc07f); }  // lgkmcnt(0) alone

template <int CT>
struct CElem {
  typedef typename XElem<CT>::T T;
  static constexpr int E = CT == XT_F32 ? 4 : 8;  // elements in 16 bytes
};

// N consecutive elements from d on; MODE 2: all inside D and aligned, 1: all
// or none inside D, aligned, 0: any.  Elements from D on are zero.
template <int CT, int N, int MODE>
struct Piece {
  typedef typename XElem<CT>::T T;
  typedef T V __attribute__((ext_vector_type(N)));
  V v;
  __device__ __forceinline__ void load(const T* row, int d, int D) {
    if constexpr (MODE == 2) {
      v = *(const V*)(row + d);
    } else if constexpr (MODE == 1) {
      if (d < D) {
        v = *(const V*)(row + d);
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = (T)0.0f;
      }
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = d + j < D ? row[d + j] : (T)0.0f;
    }
  }
};

template <int CT>
struct AttnMath;
template <>
struct AttnMath<XT_F16> {
  typedef f16x8 V;
  static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct AttnMath<XT_BF16> {
  typedef bf16x8 V;
  static __device__ __forceinline__ f32x4 mfma(V a, V b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct AttnMath<XT_F32> {
  typedef f32x4 V;
};

// What a block's weights are taken against, from its largest score: fp16 weights
// against 2^-14 of it, up to 2^14.  Rounded for the product with V, one far
// below the largest (many slots beside one that takes most of the weight) keeps
// all bits down to 2^-28 of it, where against the maximum itself they end at
// 2^-14 and the weight at 2^-25.  Sums and partial results carry the factor
// until the sum of weights divides it out.  From 2^23 on the maximum's own
// rounding is half a power and more, which the room above 2^14 is left to.
// bf16 has fp32's exponents.
template <int CT, bool M16>
__device__ __forceinline__ float reference(float mx) {
  if constexpr (M16 && CT == XT_F16) return __builtin_fabsf(mx) < 8388608.0f ? mx - 14.0f : mx;
  return mx;
}

__device__ __forceinline__ float load_q(const void* q, int qt, int64_t i) {
  return qt == XT_F32 ? ((const float*)q)[i] : qt == XT_F16 ? (float)((const _Float16*)q)[i] : (float)((const __bf16*)q)[i];
}

__device__ __forceinline__ bool finite(float v) { return __builtin_fabsf(v) <= 3.4028235e38f; }

// Which of N slots token `tok` sees, one bit each; slot(v) is the v-th one's
// index in the cache (or among the drafts), valid up to `last`.  All loads
// before the first comparison: one after the other they would cost a memory
// latency each.
template <int N, class F>
__device__ __forceinline__ uint32_t sees(const AttnArgs& a, bool fresh, int tok, int last, F slot) {
  const int64_t hi = a.q_pos[tok], lo = a.window > 0 && hi - a.window + 1 > 0 ? hi - a.window + 1 : 0;
  uint32_t bits = 0;
  if (!fresh) {
    int64_t sp[N];
#pragma unroll
    for (int v = 0; v < N; ++v) sp[v] = a.slot_pos[min(slot(v), last)];
#pragma unroll
    for (int v = 0; v < N; ++v) bits |= slot(v) <= last && sp[v] >= lo && sp[v] <= hi ? 1u << v : 0u;
    return bits;
  }
  if (a.tree) {
    uint8_t t[N];
#pragma unroll
    for (int v = 0; v < N; ++v) t[v] = a.tree[(int64_t)tok * a.tree_ld + min(slot(v), last)];
#pragma unroll
    for (int v = 0; v < N; ++v) bits |= slot(v) <= last && t[v] ? 1u << v : 0u;
  } else {
#pragma unroll
    for (int v = 0; v < N; ++v) bits |= slot(v) <= tok ? 1u << v : 0u;  // (tok <= last)
  }
  if (a.window > 0) {
    int64_t qp[N];
#pragma unroll
    for (int v = 0; v < N; ++v) qp[v] = a.q_pos[min(slot(v), last)];
#pragma unroll
    for (int v = 0; v < N; ++v)
      if (qp[v] <= hi - a.window) bits &= ~(1u << v);
  }
  return bits;
}

// Infinities and NaN of V.  Where a row does not see every slot of a block,
// such a value must not reach it as 0 * inf: the block's product takes the
// finite values only, and the others are counted by a product of zeros and
// ones (V's element is of the kind, the row sees the slot): a row that sees
// one has it added.  kind: 0 +inf, 1 -inf, 2 NaN.
__device__ __forceinline__ float odd_value(int kind) {
  return kind == 0 ? __builtin_inff() : kind == 1 ? -__builtin_inff() : __builtin_nanf("");
}
__device__ __forceinline__ float odd_one(float x, int kind) {
  const bool is = kind == 0 ? x == __builtin_inff() : kind == 1 ? x == -__builtin_inff() : x != x;
  return is ? 1.0f : 0.0f;
}
// ... on two 2-byte values side by side
template <int CT>
struct Odd2 {
  static constexpr uint32_t kExp = CT == XT_F16 ? 0x7c00u : 0x7f80u, kOne = CT == XT_F16 ? 0x3c00u : 0x3f80u;
  static __device__ __forceinline__ bool any(uint32_t w) {
    return (w & kExp) == kExp || (w >> 16 & kExp) == kExp;
  }
  static __device__ __forceinline__ uint32_t finite(uint32_t w) {
    return ((w & kExp) == kExp ? 0u : w & 0xffffu) | ((w >> 16 & kExp) == kExp ? 0u : w & 0xffff0000u);
  }
  static __device__ __forceinline__ bool is(uint32_t x, int kind) {
    return kind == 2 ? (x & 0x7fffu) > kExp : x == (kind ? kExp | 0x8000u : kExp);
  }
  static __device__ __forceinline__ uint32_t ones(uint32_t w, int kind) {
    return (is(w & 0xffffu, kind) ? kOne : 0u) | (is(w >> 16, kind) ? kOne << 16 : 0u);
  }
};

// One row of Q as the S^T product's operand: lane group g holds the columns
// ch * 4E + g * E + 0..E-1 of every piece ch.
template <int CT, bool M16, int DP, int MODE>
struct QRow {
  static constexpr int E = CElem<CT>::E, NCH = DP / (4 * E);
  typename AttnMath<CT>::V v[M16 ? NCH : 1];
  float f[M16 ? 1 : NCH][E];
  __device__ __forceinline__ void load(const AttnArgs& a, int kvh, int r, int g) {
    typedef typename XElem<CT>::T T;
    const int64_t at = (int64_t)(r / a.rep) * a.q_st + (int64_t)(kvh * a.rep + r % a.rep) * a.q_sh;
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch) {
      const int d = ch * 4 * E + g * E;
      if constexpr (M16) {
        Piece<CT, E, MODE> x;
        if (a.qvec) {
          x.load((const T*)a.q + at, d, a.D);
        } else {
          Piece<CT, E, 0> y;
          y.load((const T*)a.q + at, d, a.D);
          x.v = y.v;
        }
        u32x4 bits = __builtin_bit_cast(u32x4, x.v);
        if (a.neg) bits ^= 0x80008000u;
        v[ch] = __builtin_bit_cast(typename AttnMath<CT>::V, bits);
      } else if (a.qvec) {
#pragma unroll
        for (int j = 0; j < E; j += 4) {
          Piece<XT_F32, 4, MODE == 2 ? 2 : 1> x;
          x.load((const float*)a.q + at, d + j, a.D);
#pragma unroll
          for (int k = 0; k < 4; ++k) f[ch][j + k] = a.neg ? -x.v[k] : x.v[k];
        }
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const float x = d + j < a.D ? load_q(a.q, a.qt, at + d + j) : 0.0f;
          f[ch][j] = a.neg ? -x : x;
        }
      }
    }
  }
};

// A block's scores in fp32, four sums side by side: the products wait less for
// each other and the rounding errors of a score of many columns halve.
template <int E, class P, int NCH>
__device__ __forceinline__ f32x4 fp32_scores(const P (&k)[NCH], const float (&q)[NCH][E]) {
  f32x4 s[4] = {(f32x4)(0.0f), (f32x4)(0.0f), (f32x4)(0.0f), (f32x4)(0.0f)};
#pragma unroll
  for (int ch = 0; ch < NCH; ++ch)
#pragma unroll
    for (int j = 0; j < E; ++j)
      s[j % 4] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)k[ch].v[j], q[ch][j], s[j % 4], 0, 0, 0);
  return (s[0] + s[1]) + (s[2] + s[3]);
}

template <int CT, bool M16, int DP, int MODE, int RT>
__global__ __launch_bounds__(kAttnWaves * 64, DP == 256 ? (RT == 2 ? 1 : 2) : RT == 2 ? 2 : 3) void attn_kernel(AttnArgs a) {
  typedef typename XElem<CT>::T T;
  typedef AttnMath<CT> Math;
  constexpr int E = CElem<CT>::E, NCH = DP / (4 * E);
  constexpr int SUB = M16 ? 2 : 1, SB = 16 * SUB, VS = M16 ? 8 : 4;
  constexpr int EV = E < DP / 16 ? E : DP / 16, DB = DP / (16 * EV), NF = DB * EV;
  constexpr int HP = DP < 128 ? DP : 128, OLD = HP + 4;  // columns of O joined at a time, LDS row of them
  constexpr float kNone = -__builtin_inff();
  __shared__ __align__(16) float lds_o[kAttnWaves * 16 * OLD];
  __shared__ float lds_m[kAttnWaves][16], lds_l[kAttnWaves][16];

  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
  const int kvh = blockIdx.x % a.Hk, rtile = blockIdx.x / a.Hk % a.rtiles, split = blockIdx.x / a.Hk / a.rtiles;
  const int R = a.rep * a.T, row0 = rtile * (16 * RT);

  const int nbc = (a.slots + SB - 1) / SB, nb = nbc + (a.Tn + SB - 1) / SB, W = a.splits * kAttnWaves;
  // position of the lane's slot (lane % SB) of block b; -1 past the cache
  auto position = [&](int b) -> int64_t {
    const int s = b * SB + (lane & (SB - 1));
    return s < a.slots ? a.slot_pos[s] : -1;
  };
  int b = split * kAttnWaves + w;
  int64_t sp = position(b);

  // the lane's rows and what they see: positions lo..hi
  int row[RT], tok[RT];
  int64_t lo[RT], hi[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    row[i] = row0 + i * 16 + c;
    tok[i] = min(row[i], R - 1) / a.rep;
    hi[i] = a.q_pos[tok[i]];
  }

  QRow<CT, M16, DP, MODE> qr[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) qr[i].load(a, kvh, min(row[i], R - 1), g);

  int64_t lo_min = INT64_MAX, lo_max = 0, hi_min = INT64_MAX, hi_max = -1;
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    lo[i] = a.window > 0 && hi[i] - a.window + 1 > 0 ? hi[i] - a.window + 1 : 0;
    // (a row past the last one is the last one again)
    lo_min = min(lo_min, lo[i]), lo_max = max(lo_max, lo[i]), hi_min = min(hi_min, hi[i]), hi_max = max(hi_max, hi[i]);
  }
  if (a.T > 1) {
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
      lo_min = min(lo_min, (int64_t)__shfl_xor((long long)lo_min, o, 64));
      lo_max = max(lo_max, (int64_t)__shfl_xor((long long)lo_max, o, 64));
      hi_min = min(hi_min, (int64_t)__shfl_xor((long long)hi_min, o, 64));
      hi_max = max(hi_max, (int64_t)__shfl_xor((long long)hi_max, o, 64));
    }
  }

  f32x4 o[RT][NF];
  float m[RT], l[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    m[i] = kNone, l[i] = 0.0f;
#pragma unroll
    for (int f = 0; f < NF; ++f) o[i][f] = (f32x4)(0.0f);
  }

  // Block b of the cache (b < nbc) or of the drafts; FULL: of the cache, and
  // every row sees all of it.
  auto block = [&](int b, auto FULL) {
    constexpr bool full = decltype(FULL)::value != 0;
    const bool fresh = !full && b >= nbc;
    const int base = (fresh ? b - nbc : b) * SB, last = (fresh ? a.Tn : a.slots) - 1;
    const int64_t ss = fresh ? a.n_ss : a.k_ss, head = (int64_t)kvh * (fresh ? a.n_sh : a.k_sh);
    const T* const kp = (const T*)(fresh ? a.kn : a.k) + head;
    const T* const vp = (const T*)(fresh ? a.vn : a.v) + head;

    Piece<CT, E, MODE> kf[SUB][NCH];
    Piece<CT, EV, MODE> vf[VS][DB];
#pragma unroll
    for (int st = 0; st < SUB; ++st) {
      const T* const kr = kp + min(base + st * 16 + c, last) * ss;
#pragma unroll
      for (int ch = 0; ch < NCH; ++ch) kf[st][ch].load(kr, ch * 4 * E + g * E, a.D);
    }
#pragma unroll
    for (int j = 0; j < VS; ++j) {
      const T* const vr = vp + min(base + (j >> 2) * 16 + 4 * g + (j & 3), last) * ss;
#pragma unroll
      for (int db = 0; db < DB; ++db) vf[j][db].load(vr, db * 16 * EV + c * EV, a.D);
    }

    float p[RT][SUB][4];
    uint32_t seen[RT] = {};  // bit st * 4 + v (= V's slot j of the lane), where not every row sees every slot
#pragma unroll
    for (int i = 0; i < RT; ++i) {
#pragma unroll
      for (int st = 0; st < SUB; ++st) {
        f32x4 s = (f32x4)(0.0f);
#pragma unroll
        for (int ch = 0; ch < NCH; ++ch) {
          if constexpr (M16) {
            s = Math::mfma(__builtin_bit_cast(typename Math::V, kf[st][ch].v), qr[i].v[ch], s);
          }
        }
        if constexpr (!M16) s = fp32_scores<E>(kf[st], qr[i].f);
#pragma unroll
        for (int v = 0; v < 4; ++v) p[i][st][v] = s[v];
        if (RT == 1 && a.scores && !fresh && row[i] < R)  // (as many as fit whole blocks have room)
          *(f32x4*)(a.scores + ((int64_t)kvh * R + row[i]) * a.score_ld + base + st * 16 + 4 * g) = s;
      }
      float mx = kNone;
      if constexpr (full) {
#pragma unroll
        for (int st = 0; st < SUB; ++st)
#pragma unroll
          for (int v = 0; v < 4; ++v) mx = __builtin_fmaxf(mx, p[i][st][v]);
      } else {
        seen[i] = sees<SUB * 4>(a, fresh, tok[i], last, [&](int v) { return base + (v >> 2) * 16 + 4 * g + (v & 3); });
#pragma unroll
        for (int st = 0; st < SUB; ++st)
#pragma unroll
          for (int v = 0; v < 4; ++v) mx = seen[i] >> (st * 4 + v) & 1 ? __builtin_fmaxf(mx, p[i][st][v]) : mx;
      }
      mx = reference<CT, M16>(mx * a.scale);
      if (__any(mx > m[i])) {
        mx = __builtin_fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = __builtin_fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float up = __builtin_fmaxf(m[i], mx);
        const float alpha = up == kNone ? 1.0f : __builtin_amdgcn_exp2f(m[i] - up);
        m[i] = up;
        l[i] *= alpha;
#pragma unroll
        for (int f = 0; f < NF; ++f) o[i][f] *= alpha;
      }
      const float from = m[i] == kNone ? 0.0f : m[i];
#pragma unroll
      for (int st = 0; st < SUB; ++st)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          float e = __builtin_amdgcn_exp2f(__builtin_fmaf(p[i][st][v], a.scale, -from));
          if constexpr (!full) e = seen[i] >> (st * 4 + v) & 1 ? e : 0.0f;
          p[i][st][v] = e;
          l[i] += e;
        }
    }

    bool odd = false;  // infinities or NaN in V, and rows that do not see every slot
    if constexpr (!full) {
#pragma unroll
      for (int j = 0; j < VS; ++j)
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int e = 0; e < EV; ++e) odd |= !finite((float)vf[j][db].v[e]);
      odd = __any(odd);
    }

    // O^T += V^T P^T
    if constexpr (M16) {
      typename Math::V pf[RT];
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) pf[i][j] = (T)p[i][j >> 2][j & 3];
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        typedef uint32_t Words __attribute__((ext_vector_type(EV / 2)));
        Words vw[VS];
#pragma unroll
        for (int j = 0; j < VS; ++j) vw[j] = __builtin_bit_cast(Words, vf[j][db].v);
#pragma unroll
        for (int e = 0; e < EV; ++e) {
          u32x4 t;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            t[j] = __builtin_amdgcn_perm(vw[2 * j + 1][e / 2], vw[2 * j][e / 2], e % 2 ? 0x07060302u : 0x05040100u);
          if (!full && odd) {
#pragma unroll 1
            for (int kind = 0; kind < 3; ++kind) {
              u32x4 ones;
#pragma unroll
              for (int j = 0; j < 4; ++j) ones[j] = Odd2<CT>::ones(t[j], kind);
#pragma unroll
              for (int i = 0; i < RT; ++i) {
                typename Math::V sees;
#pragma unroll
                for (int j = 0; j < 8; ++j) sees[j] = (T)(seen[i] >> j & 1 ? 1.0f : 0.0f);
                const f32x4 n = Math::mfma(__builtin_bit_cast(typename Math::V, ones), sees, (f32x4)(0.0f));
#pragma unroll
                for (int v = 0; v < 4; ++v)
                  if (n[v] > 0.0f) o[i][db * EV + e][v] += odd_value(kind);
              }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) t[j] = Odd2<CT>::finite(t[j]);
          }
          const typename Math::V vt = __builtin_bit_cast(typename Math::V, t);
#pragma unroll
          for (int i = 0; i < RT; ++i) o[i][db * EV + e] = Math::mfma(vt, pf[i], o[i][db * EV + e]);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int e = 0; e < EV; ++e) {
            float x = (float)vf[j][db].v[e];
            if (!full && odd) {
#pragma unroll 1
              for (int kind = 0; kind < 3; ++kind)
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                  const f32x4 n = __builtin_amdgcn_mfma_f32_16x16x4f32(odd_one(x, kind), seen[i] >> j & 1 ? 1.0f : 0.0f,
                                                                       (f32x4)(0.0f), 0, 0, 0);
#pragma unroll
                  for (int v = 0; v < 4; ++v)
                    if (n[v] > 0.0f) o[i][db * EV + e][v] += odd_value(kind);
                }
              x = finite(x) ? x : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < RT; ++i)
              o[i][db * EV + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(x, p[i][0][j], o[i][db * EV + e], 0, 0, 0);
          }
    }
  };

  // The wave's blocks, 64 at a time: those that every row sees whole, then the
  // others; a loop each, so that the masks of the second cost the first no
  // registers.
#pragma unroll 1
  while (b < nb) {
    const int b0 = b;
    uint64_t later = 0;
#pragma unroll 1
    for (int i = 0; i < 64 && b < nb; ++i) {
      const int at = b;
      const bool fresh = at >= nbc, any = fresh || __any(sp >= lo_min && sp <= hi_max);
      const bool full = !fresh && __all(sp >= lo_max && sp <= hi_min);
      b += W;
      if (b < nbc) sp = position(b);
      if (full)
        block(at, Const<1>{});
      else
        later |= (uint64_t)any << i;
    }
#pragma unroll 1
    for (; later; later &= later - 1) block(b0 + __builtin_ctzll(later) * W, Const<0>{});
  }

  // the workgroup's waves joined, one row tile at a time
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    l[i] += __shfl_xor(l[i], 16, 64);
    l[i] += __shfl_xor(l[i], 32, 64);
#pragma unroll
    for (int h0 = 0; h0 < DP; h0 += HP) {
      __syncthreads();  // (lds_o is free)
      if (g == 0) lds_m[w][c] = m[i], lds_l[w][c] = l[i];
      float* const to = lds_o + (w * 16 + c) * OLD;
#pragma unroll
      for (int db = h0 / (16 * EV); db < (h0 + HP) / (16 * EV); ++db)
#pragma unroll
        for (int v = 0; v < 4; ++v)
#pragma unroll
          for (int e = 0; e < EV; ++e) to[db * 16 * EV - h0 + (4 * g + v) * EV + e] = o[i][db * EV + e][v];
      __syncthreads();
      const int r0 = row0 + i * 16;
      for (int u = threadIdx.x; u < 16 * (HP / 4); u += kAttnWaves * 64) {
        const int rr = u / (HP / 4), d = h0 + u % (HP / 4) * 4;
        if (r0 + rr >= R) continue;
        float top = kNone;
#pragma unroll
        for (int k = 0; k < kAttnWaves; ++k) top = __builtin_fmaxf(top, lds_m[k][rr]);
        const float from = top == kNone ? 0.0f : top;
        f32x4 sum = (f32x4)(0.0f);
        float ls = 0.0f;
#pragma unroll
        for (int k = 0; k < kAttnWaves; ++k) {
          const float f = __builtin_amdgcn_exp2f(lds_m[k][rr] - from);
          const f32x4 x = *(const f32x4*)(lds_o + (k * 16 + rr) * OLD + d - h0);
          if (lds_l[k][rr] != 0.0f) {  // (a wave that saw nothing adds nothing)
            sum += x * f;
            ls += lds_l[k][rr] * f;
          }
        }
        const int64_t at = (int64_t)kvh * R + r0 + rr;
        if (a.part_o) {
          *(f32x4*)(a.part_o + (at * a.splits + split) * DP + d) = sum;
          if (d == 0) a.part_ml[at * a.splits + split] = make_float2(top, ls);
        } else {
          const float inv = ls != 0.0f ? 1.0f / ls : 0.0f;
          const int t = (r0 + rr) / a.rep, h = kvh * a.rep + (r0 + rr) % a.rep;
          const int64_t out = (int64_t)t * a.o_st + (int64_t)h * a.o_sh + d;
          if (d < a.D) store_y4(a.out, a.qt, out, sum * inv, a.ovec && d + 4 <= a.D, a.D - d);
          if (d == 0 && a.row_ml) a.row_ml[at] = make_float2(from, inv);
        }
      }
    }
  }
}

// The same for many rows (256 and more of a key head) over 2-byte caches of
// 64 or 128 columns: a wave owns 32 rows, the workgroup's waves share every
// tile of 64 slots through LDS (global -> LDS copies of the next NBUF - 1 tiles
// run under the products of this one), and 32x32x16 products halve the operand
// reads per product.  K and V rows lie in LDS as in memory, their
// 16-byte pieces permuted by the row (source side: the copy writes lane after
// lane), so that the operand reads of 32 rows meet all banks.  S^T and O^T as
// above: lane (h, r) holds the scores of row r and the slots 8 (v / 4) + 4 h +
// v % 4, which 16 at a time are the operand of V^T's product in that slot
// order.  What bounds it: per 64 scores 32 cycles of products and some 30 of
// exponentials and sums per SIMD, two waves of which overlap.  64 tokens of 32
// heads over 65000 slots of 8 x 128 bf16: 115 us with the joining (replayed
// graph), 590 TFLOP/s.
template <int CT, int DP>
__global__ __launch_bounds__(kTileWaves * 64, 2) void attn_tile_kernel(AttnArgs a) {
  typedef typename XElem<CT>::T T;
  typedef AttnMath<CT> Math;
  typedef typename Math::V V;
  typedef float f32x16 __attribute__((ext_vector_type(16)));
  constexpr int NW = kTileWaves, NBUF = kTileBufs, TS = kTileSlots, KK = DP / 16, EV = DP / 32, CPR = DP / 8, ROWB = DP * 2;
  constexpr int TILEB = TS * ROWB, BUFB = 2 * TILEB;  // K then V
  constexpr float kNone = -__builtin_inff();
  extern __shared__ __align__(16) uint8_t lds[];  // NBUF tiles
  auto product = [](V x, V y, f32x16 z) {
    if constexpr (CT == XT_F16)
      return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, z, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, z, 0, 0, 0);
  };
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r = lane & 31, h = lane >> 5;
  const int kvh = blockIdx.x % a.Hk, rtile = blockIdx.x / a.Hk % a.rtiles, split = blockIdx.x / a.Hk / a.rtiles;
  const int R = a.rep * a.T, row = (rtile * NW + w) * 32 + r, rowc = min(row, R - 1), tok = rowc / a.rep;

  const int nbc = (a.slots + TS - 1) / TS, nb = nbc + (a.Tn + TS - 1) / TS;
  // what the tokens of the whole call see (the workgroup's skipping is uniform)
  int64_t lo_min = INT64_MAX, lo_max = 0, hi_min = INT64_MAX, hi_max = -1;
  for (int t = lane; t < a.T; t += 64) {
    const int64_t hi = a.q_pos[t], lo = a.window > 0 && hi - a.window + 1 > 0 ? hi - a.window + 1 : 0;
    lo_min = min(lo_min, lo), lo_max = max(lo_max, lo), hi_min = min(hi_min, hi), hi_max = max(hi_max, hi);
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    lo_min = min(lo_min, (int64_t)__shfl_xor((long long)lo_min, o, 64));
    lo_max = max(lo_max, (int64_t)__shfl_xor((long long)lo_max, o, 64));
    hi_min = min(hi_min, (int64_t)__shfl_xor((long long)hi_min, o, 64));
    hi_max = max(hi_max, (int64_t)__shfl_xor((long long)hi_max, o, 64));
  }

  // Q^T operand: lane (h, r) holds columns 16 kk + 8 h + 0..7 of row r
  V qf[KK];
  {
    const int64_t at = (int64_t)tok * a.q_st + (int64_t)(kvh * a.rep + rowc % a.rep) * a.q_sh;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      u32x4 bits;
      if (a.qvec) {
        bits = *(const u32x4*)((const T*)a.q + at + kk * 16 + h * 8);
      } else {
        Piece<CT, 8, 0> y;
        y.load((const T*)a.q + at, kk * 16 + h * 8, DP);
        bits = __builtin_bit_cast(u32x4, y.v);
      }
      if (a.neg) bits ^= 0x80008000u;
      qf[kk] = __builtin_bit_cast(V, bits);
    }
  }

  // Copies of a tile: COPIES pieces of 16 bytes a lane, the same number by
  // every call, so that counting them is enough to wait for a tile.
  constexpr int COPIES = BUFB / 1024 / NW;
  static_assert(BUFB % (1024 * NW) == 0, "whole copies per wave");
  static_assert(COPIES % 2 == 0, "as many of K as of V");
  uint32_t piece_at[COPIES / 2];  // bytes from a tile's start to the lane's pieces, the same in K and V
#pragma unroll
  for (int i = 0; i < COPIES / 2; ++i) {
    const int u = (i * NW + w) * 64 + lane, s = u / CPR;
    piece_at[i] = (uint32_t)(s * a.k_ss + ((u ^ s) & (CPR - 1)) * 8) * 2;
  }
  const bool near = a.k_ss < (1 << 23);  // (the offsets fit 32 bits)
  auto copy_tile = [&](int b, int buf) {
    uint8_t* const to = lds + buf * BUFB + w * 1024;
    if (near && (b + 1) * TS <= a.slots) {
      const int64_t first = (int64_t)kvh * a.k_sh + (int64_t)b * TS * a.k_ss;
      const uint8_t* const kp = (const uint8_t*)((const T*)a.k + first);
      const uint8_t* const vp = (const uint8_t*)((const T*)a.v + first);
#pragma unroll
      for (int i = 0; i < COPIES; ++i)
        __builtin_amdgcn_global_load_lds((const void*)((i < COPIES / 2 ? kp : vp) + piece_at[i % (COPIES / 2)]),
                                         (__attribute__((address_space(3))) void*)(to + i * NW * 1024), 16, 0, 0);
    } else {  // the cache's end, or drafts: slots past the last one are the last one again
      const bool fresh = b >= nbc;
      const int base = (fresh ? b - nbc : b) * TS, last = (fresh ? a.Tn : a.slots) - 1;
      const int64_t ss = fresh ? a.n_ss : a.k_ss, head = (int64_t)kvh * (fresh ? a.n_sh : a.k_sh);
#pragma unroll
      for (int i = 0; i < COPIES; ++i) {
        const int q = i * NW + w, u = (q * 64 + lane) & (TS * CPR - 1), s = u / CPR;
        const void* const p = q >= TILEB / 1024 ? (fresh ? a.vn : a.v) : (fresh ? a.kn : a.k);
        const T* const src = (const T*)p + head + min(base + s, last) * ss + ((u ^ s) & (CPR - 1)) * 8;
        __builtin_amdgcn_global_load_lds((const void*)src, (__attribute__((address_space(3))) void*)(to + i * NW * 1024), 16, 0, 0);
      }
    }
  };

  f32x16 o[EV];
  float m = kNone, l = 0.0f;
#pragma unroll
  for (int e = 0; e < EV; ++e) o[e] = (f32x16)(0.0f);

  // Offsets in a tile of the lane's K pieces of its first 32 slots and V pieces
  // of its first 16 (the permutation depends on the slot modulo CPR alone).
  uint32_t koff[KK], voff[8];
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) koff[kk] = r * ROWB + (((kk * 2 + h) ^ r) & (CPR - 1)) * 16;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int sl = (j >> 2) * 8 + 4 * h + (j & 3), byte = r * EV * 2;
    voff[j] = TILEB + sl * ROWB + (((byte >> 4) ^ sl) & (CPR - 1)) * 16 + (byte & 15);
  }
  // Scores of the 32 slots that lie from `at` on in LDS.
  auto scores = [&](uint32_t at) {
    f32x16 s = (f32x16)(0.0f);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) s = product(*(const V*)(lds + at + koff[kk]), qf[kk], s);
    return s;
  };
  // ... of tile b, taken in; FULL: every row sees all of them.
  auto half = [&](f32x16 s, int b, uint32_t at, auto FULL) {
    constexpr bool kFull = decltype(FULL)::value != 0;
    uint32_t seen = 0;
    float mx = kNone;
    if constexpr (kFull) {
#pragma unroll
      for (int v = 0; v < 16; ++v) mx = __builtin_fmaxf(mx, s[v]);
    } else {
      const bool fresh = b >= nbc;
      const int base = (fresh ? b - nbc : b) * TS + (at & (TILEB - 1) ? 32 : 0), last = (fresh ? a.Tn : a.slots) - 1;
      seen = sees<16>(a, fresh, tok, last, [&](int v) { return base + (v / 4) * 8 + 4 * h + v % 4; });
#pragma unroll
      for (int v = 0; v < 16; ++v) mx = seen >> v & 1 ? __builtin_fmaxf(mx, s[v]) : mx;
    }
    mx = reference<CT, true>(mx * a.scale);
    if (__any(mx > m)) {
      mx = __builtin_fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float up = __builtin_fmaxf(m, mx);
      const float alpha = up == kNone ? 1.0f : __builtin_amdgcn_exp2f(m - up);
      m = up;
      l *= alpha;
#pragma unroll
      for (int e = 0; e < EV; ++e)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          float x = o[e][v];
          asm("v_mul_f32 %0, %1, %0" : "+v"(x) : "v"(alpha));  // (in place: the compiler would copy all of o for the branch)
          o[e][v] = x;
        }
    }
    const float from = m == kNone ? 0.0f : m;
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[v], a.scale, -from));
      if constexpr (!kFull) p = seen >> v & 1 ? p : 0.0f;
      s[v] = p;
      l += p;
    }
    // V^T's operand for 16 slots: 8 of the lane's slots, EV columns each
#pragma unroll
    for (int kc = 0; kc < 2; ++kc) {
      uint32_t vw[8][EV / 2];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint8_t* const x = lds + at + kc * 16 * ROWB + voff[j];
        if constexpr (EV == 4) {
          const u32x2 y = *(const u32x2*)x;
          vw[j][0] = y.x, vw[j][1] = y.y;
        } else {
          vw[j][0] = *(const uint32_t*)x;
        }
      }
      bool odd = false;
      if constexpr (!kFull) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int e = 0; e < EV / 2; ++e) odd |= Odd2<CT>::any(vw[j][e]);
        odd = __any(odd);
      }
      V pf;
#pragma unroll
      for (int j = 0; j < 8; ++j) pf[j] = (T)s[kc * 8 + j];
#pragma unroll
      for (int e = 0; e < EV; ++e) {
        u32x4 t;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          t[j] = __builtin_amdgcn_perm(vw[2 * j + 1][e / 2], vw[2 * j][e / 2], e % 2 ? 0x07060302u : 0x05040100u);
        if constexpr (!kFull) {
          if (odd) {
#pragma unroll 1
            for (int kind = 0; kind < 3; ++kind) {
              u32x4 ones;
              V sees;
#pragma unroll
              for (int j = 0; j < 4; ++j) ones[j] = Odd2<CT>::ones(t[j], kind);
#pragma unroll
              for (int j = 0; j < 8; ++j) sees[j] = (T)(seen >> (kc * 8 + j) & 1 ? 1.0f : 0.0f);
              const f32x16 n = product(__builtin_bit_cast(V, ones), sees, (f32x16)(0.0f));
#pragma unroll
              for (int v = 0; v < 16; ++v)
                if (n[v] > 0.0f) o[e][v] += odd_value(kind);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) t[j] = Odd2<CT>::finite(t[j]);
          }
        }
        o[e] = product(__builtin_bit_cast(V, t), pf, o[e]);
      }
    }
  };

  // 64 of the workgroup's tiles from b0 on, one bit each: `part` of them are
  // seen by some token, `whole` by every token in every slot (the waves look at
  // 64 / NW each; positions loaded between the copies would drain them).
  auto look = [&](int64_t b0, uint64_t& part, uint64_t& whole) {
    uint64_t some = 0, every = 0;
    int64_t sp[64 / NW];  // (all loads before the first comparison)
#pragma unroll
    for (int i = 0; i < 64 / NW; ++i) {
      const int64_t at = (b0 + (int64_t)(w * (64 / NW) + i) * a.splits) * TS + lane;
      sp[i] = a.slot_pos[at < a.slots ? at : a.slots - 1];
    }
#pragma unroll
    for (int i = 0; i < 64 / NW; ++i) {
      const int64_t b = b0 + (int64_t)(w * (64 / NW) + i) * a.splits;
      const int64_t pos = b * TS + lane < a.slots ? sp[i] : -1;
      const bool any = __any(pos >= lo_min && pos <= hi_max), all = __all(pos >= lo_max && pos <= hi_min);
      some |= (uint64_t)(b < nbc ? any : b < nb) << i;
      every |= (uint64_t)(b < nbc && all) << i;
    }
    uint64_t* const flags = (uint64_t*)lds;  // [2][NW]
    __syncthreads();                         // (the tiles before are done with)
    if (lane == 0) flags[w] = some, flags[NW + w] = every;
    __syncthreads();
    some = every = 0;
#pragma unroll
    for (int k = 0; k < NW; ++k) {
      some |= flags[k] << (k * (64 / NW));
      every |= flags[NW + k] << (k * (64 / NW));
    }
    __syncthreads();  // (the flags are read)
    part = (uint64_t)__builtin_amdgcn_readfirstlane((int)(some >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)some);
    whole = (uint64_t)__builtin_amdgcn_readfirstlane((int)(every >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)every);
  };

  // Tiles that every row sees whole, then the others: one loop each, so that
  // the masks of the second cost the first no registers.
  uint64_t part = 0, whole = 0;
  const bool once = nb <= split + (int64_t)64 * a.splits;  // (one look covers all)
#pragma unroll 1
  for (int64_t b0 = split; b0 < nb; b0 += (int64_t)64 * a.splits) {
    look(b0, part, whole);
    uint64_t todo = whole;
    if (!todo) continue;
    uint64_t coming = todo;  // tiles not copied yet
    int last_copied = 0;
    auto copy_next = [&](int buf) {  // (past the last one it copies that again)
      if (coming) last_copied = __builtin_ctzll(coming);
      coming &= coming - 1;
      copy_tile((int)(b0 + (int64_t)last_copied * a.splits), buf);
    };
#pragma unroll
    for (int i = 0; i < NBUF - 1; ++i) copy_next(i);
    auto step = [&](auto BUF) {  // (a constant buffer, whose offsets are then the reads' own)
      constexpr int buf = decltype(BUF)::value;
      // This wave's copies of the current tile have arrived (loads return in
      // order; those of the NBUF - 2 tiles after it may be under way), and
      // behind the barrier everyone's; everyone is also done with the tile
      // before, whose place the next copy takes.
      wait_vmcnt<(NBUF - 2) * COPIES>();
      wait_lds();
      barrier_nofence();
      copy_next((buf + NBUF - 1) % NBUF);
      // the second half's scores are on their way while the first is taken in
      const f32x16 s0 = scores(buf * BUFB), s1 = scores(buf * BUFB + 32 * ROWB);
      half(s0, 0, buf * BUFB, Const<1>{});
      __builtin_amdgcn_sched_barrier(0);  // (both at once do not fit the registers)
      half(s1, 0, buf * BUFB + 32 * ROWB, Const<1>{});
      todo &= todo - 1;
      return todo != 0;
    };
    static_assert(NBUF == 4, "a step per buffer");
#pragma unroll 1
    while (step(Const<0>{}) && step(Const<1>{}) && step(Const<2>{}) && step(Const<3>{})) {
    }
    wait_vmcnt<0>();  // (no copy outlives its buffer)
  }
#pragma unroll 1
  for (int64_t b0 = split; b0 < nb; b0 += (int64_t)64 * a.splits) {
    if (!once) look(b0, part, whole);
#pragma unroll 1
    for (part &= ~whole; part; part &= part - 1) {
      const int b = (int)(b0 + (int64_t)__builtin_ctzll(part) * a.splits);
      __syncthreads();  // (the tile before is done with)
      copy_tile(b, 0);
      wait_vmcnt<0>();
      __syncthreads();
#pragma unroll 1
      for (int sub = 0; sub < 2; ++sub) half(scores(sub * 32 * ROWB), b, sub * 32 * ROWB, Const<0>{});
    }
  }

  l += __shfl_xor(l, 32, 64);
  const int tile = rtile * NW + w;  // of 32 rows
  if (tile * 32 >= R) return;
  if (a.splits > 1) {  // as they lie in the registers: [head][tile][split][v][lane][EV], maxima and sums [32]
    const int64_t at = ((int64_t)kvh * (a.rtiles * NW) + tile) * a.splits + split;
    typedef float Row __attribute__((ext_vector_type(EV)));
    Row* const to = (Row*)a.part_o + at * 1024 + lane;
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      Row x;
#pragma unroll
      for (int e = 0; e < EV; ++e) x[e] = o[e][v];
      to[v * 64] = x;
    }
    if (h == 0) a.part_ml[at * 32 + r] = make_float2(m, l);
    return;
  }
  if (row >= R) return;
  const float inv = l != 0.0f ? 1.0f / l : 0.0f;
  if (l == 0.0f) {  // (scores of -infinity alone; infinities of V have made its sums NaN)
#pragma unroll
    for (int e = 0; e < EV; ++e) o[e] = (f32x16)(0.0f);
  }
  const int64_t out = (int64_t)tok * a.o_st + (int64_t)(kvh * a.rep + row % a.rep) * a.o_sh;
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    const int d = ((v / 4) * 8 + 4 * h + v % 4) * EV;
    if constexpr (EV == 4) {
      store_y4(a.out, a.qt, out + d, (f32x4){o[0][v], o[1][v], o[2][v], o[3][v]} * inv, a.ovec, 4);
    } else {
      store_y(a.out, a.qt, out + d, o[0][v] * inv);
      store_y(a.out, a.qt, out + d + 1, o[1][v] * inv);
    }
  }
  if (h == 0 && a.row_ml) a.row_ml[(int64_t)kvh * R + row] = make_float2(m == kNone ? 0.0f : m, inv);
}

// The splits of attn_tile_kernel's rows joined: a wave per (key head, tile of
// 32 rows, v), which reads the partial sums as they were written.
template <int DP>
__global__ __launch_bounds__(64) void attn_tile_join_kernel(AttnArgs a) {
  constexpr int EV = DP / 32, NW = kTileWaves;
  typedef float Row __attribute__((ext_vector_type(EV)));
  const int R = a.rep * a.T, tiles = (R + 31) / 32, lane = threadIdx.x, r = lane & 31, h = lane >> 5;
  const int v = blockIdx.x & 15, tile = (blockIdx.x >> 4) % tiles, kvh = (blockIdx.x >> 4) / tiles;
  const int64_t at = ((int64_t)kvh * (a.rtiles * NW) + tile) * a.splits;
  const Row* const from = (const Row*)a.part_o + at * 1024 + v * 64 + lane;
  const float2* const ml = a.part_ml + at * 32 + r;
  float top = -__builtin_inff(), l = 0.0f;
  for (int s0 = 0; s0 < a.splits; s0 += 8) {
    float x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = ml[min(s0 + k, a.splits - 1) * 32].x;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = __builtin_fmaxf(top, x[k]);
  }
  const float base = top == -__builtin_inff() ? 0.0f : top;
  Row sum = (Row)(0.0f);
  for (int s0 = 0; s0 < a.splits; s0 += 4) {
    Row x[4];
    float2 y[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int s = min(s0 + k, a.splits - 1);
      x[k] = from[(int64_t)s * 1024];
      y[k] = ml[s * 32];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float f = __builtin_amdgcn_exp2f(y[k].x - base);
      if (s0 + k < a.splits && y[k].y != 0.0f) {  // (a split that saw nothing adds nothing)
        sum += x[k] * f;
        l += y[k].y * f;
      }
    }
  }
  const int row = tile * 32 + r;
  if (row >= R) return;
  const float inv = l != 0.0f ? 1.0f / l : 0.0f;
  const int64_t out = (int64_t)(row / a.rep) * a.o_st + (int64_t)(kvh * a.rep + row % a.rep) * a.o_sh +
                      ((v / 4) * 8 + 4 * h + v % 4) * EV;
  if constexpr (EV == 4) {
    store_y4(a.out, a.qt, out, sum * inv, a.ovec, 4);
  } else {
    store_y(a.out, a.qt, out, sum[0] * inv);
    store_y(a.out, a.qt, out + 1, sum[1] * inv);
  }
  if (v == 0 && h == 0 && a.row_ml) a.row_ml[(int64_t)kvh * R + row] = make_float2(base, inv);
}

// weight[s] += sum over the rows that see slot s of exp2(score - maximum) /
// sum, for more rows than attn_join_weight_kernel takes: the scores are computed
// once more, as storing them would move 8 bytes per row and slot, more than a
// key's own bytes, and hold them in memory.  A workgroup takes SB slots and every row; its waves share the
// (key head, 16-row tile) pairs, keep the slots' keys in registers while the
// head stays, and add up in wave order.
constexpr int kWeightWaves = 8, kWeightBufs = 4;
// attn_weight_tile_kernel: rows of a key head, and slots, from which it is taken
constexpr int kWeightTileRows = 256, kWeightTileSlots = 28 * 1024;
template <int CT, bool M16, int DP, int MODE>
__global__ __launch_bounds__(kWeightWaves * 64) void attn_weight_kernel(AttnArgs a, float* weight) {
  typedef typename XElem<CT>::T T;
  typedef AttnMath<CT> Math;
  constexpr int E = CElem<CT>::E, NCH = DP / (4 * E), SUB = M16 ? 2 : 1, SB = 16 * SUB;
  __shared__ float sums[kWeightWaves][SB];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
  const int R = a.rep * a.T, tiles = (R + 15) / 16, base = blockIdx.x * SB, last = a.slots - 1;

  // is there a row that sees any of the slots, do all rows see all of them?
  const int own = base + (lane & (SB - 1));
  const int64_t sp = own <= last ? a.slot_pos[own] : -1;
  int64_t lo_min = INT64_MAX, lo_max = 0, hi_min = INT64_MAX, hi_max = -1;
  for (int t = lane; t < a.T; t += 64) {
    const int64_t hi = a.q_pos[t], lo = a.window > 0 && hi - a.window + 1 > 0 ? hi - a.window + 1 : 0;
    lo_min = min(lo_min, lo), lo_max = max(lo_max, lo), hi_min = min(hi_min, hi), hi_max = max(hi_max, hi);
  }
  for (int o = 1; o < 64 && o < a.T; o <<= 1) {
    lo_min = min(lo_min, (int64_t)__shfl_xor((long long)lo_min, o, 64));
    lo_max = max(lo_max, (int64_t)__shfl_xor((long long)lo_max, o, 64));
    hi_min = min(hi_min, (int64_t)__shfl_xor((long long)hi_min, o, 64));
    hi_max = max(hi_max, (int64_t)__shfl_xor((long long)hi_max, o, 64));
  }
  lo_min = __shfl((long long)lo_min, 0, 64), lo_max = __shfl((long long)lo_max, 0, 64);
  hi_min = __shfl((long long)hi_min, 0, 64), hi_max = __shfl((long long)hi_max, 0, 64);
  if (!__any(sp >= lo_min && sp <= hi_max)) return;  // (the same for every wave)
  const bool full = __all(sp < 0 || (sp >= lo_max && sp <= hi_min));  // (an empty slot's sum is not written)

  Piece<CT, E, MODE> kf[SUB][NCH];
  float acc[SUB][4] = {};
  const int units = a.Hk * tiles, u1 = (int)((int64_t)(w + 1) * units / kWeightWaves);
  int held = -1;
  for (int u = (int)((int64_t)w * units / kWeightWaves); u < u1; ++u) {
    const int kvh = u / tiles, r = u % tiles * 16 + c, rc = min(r, R - 1);
    QRow<CT, M16, DP, MODE> qr;
    qr.load(a, kvh, rc, g);
    const float2 ml = a.row_ml[(int64_t)kvh * R + rc];
    uint32_t seen = r < R ? ~0u : 0u;
    if (!full) seen &= sees<SUB * 4>(a, false, rc / a.rep, last, [&](int v) { return base + (v >> 2) * 16 + 4 * g + (v & 3); });
    if (kvh != held) {
      held = kvh;
#pragma unroll
      for (int st = 0; st < SUB; ++st) {
        const T* const kr = (const T*)a.k + (int64_t)kvh * a.k_sh + min(base + st * 16 + c, last) * a.k_ss;
#pragma unroll
        for (int ch = 0; ch < NCH; ++ch) kf[st][ch].load(kr, ch * 4 * E + g * E, a.D);
      }
    }
#pragma unroll
    for (int st = 0; st < SUB; ++st) {
      f32x4 s = (f32x4)(0.0f);
#pragma unroll
      for (int ch = 0; ch < NCH; ++ch) {
        if constexpr (M16) {
          s = Math::mfma(__builtin_bit_cast(typename Math::V, kf[st][ch].v), qr.v[ch], s);
        }
      }
      if constexpr (!M16) s = fp32_scores<E>(kf[st], qr.f);
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[v], a.scale, -ml.x)) * ml.y;
        acc[st][v] += seen >> (st * 4 + v) & 1 ? p : 0.0f;
      }
    }
  }
#pragma unroll
  for (int st = 0; st < SUB; ++st)
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      float x = acc[st][v];
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) x += __shfl_xor(x, o, 64);
      if (c == 0) sums[w][st * 16 + 4 * g + v] = x;
    }
  __syncthreads();
  if (threadIdx.x < SB && base + (int)threadIdx.x <= last) {
    float x = sums[0][threadIdx.x];
#pragma unroll
    for (int k = 1; k < kWeightWaves; ++k) x += sums[k][threadIdx.x];
    if (a.slot_pos[base + threadIdx.x] >= 0) weight[base + threadIdx.x] += x;
  }
}

// The same for many rows over 2-byte caches of 64 or 128 columns: a wave
// takes 32 slots (their keys of one head in registers, the next head's on
// their way), the workgroup's 8 waves share every 64 rows of Q through LDS, so
// that Q is read once per 256 slots, and work on the two halves of the rows
// side by side.  It pays from 256 rows of a key head and enough slots to fill
// many CUs 256 at a time: 64 tokens of 32 heads over 65000 slots of 8 x 128
// bf16 71 us against 143 us for attn_weight_kernel, over 40000 63 / 89, over
// 32768 63 / 73, over 24576 62 / 56, over 8192 61 / 23; 128 tokens over 24576
// 105 / 100 (replayed graphs, a call with weights less one without; other
// numbers of key heads are not measured).  The workgroups whose slots not every
// row sees look at positions per row and take longest: a chunk of 64 tokens
// whose own slots are the last of 32768 takes 108 us / 81, of 65000 119 / 151.
template <int CT, int DP>
__global__ __launch_bounds__(kWeightWaves * 64, 2) void attn_weight_tile_kernel(AttnArgs a, float* weight) {
  typedef typename XElem<CT>::T T;
  typedef typename AttnMath<CT>::V V;
  typedef float f32x16 __attribute__((ext_vector_type(16)));
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  constexpr int KK = DP / 16, CPR = DP / 8, ROWB = DP * 2, TILEB = 64 * ROWB, NBUF = kWeightBufs;
  constexpr int PARTS = TILEB / 1024 / kWeightWaves;  // copies of a wave, of 64 pieces of 16 bytes
  // (one dynamic object: before a read of a static one the compiler waits for every copy under way)
  extern __shared__ __align__(16) uint8_t lds[];  // NBUF tiles of rows, then their maxima and sums
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r = lane & 31, h = lane >> 5;
  const int R = a.rep * a.T;
  const int base = blockIdx.x * (32 * kWeightWaves) + w * 32, last = a.slots - 1;

  const int64_t sp = base + r <= last ? a.slot_pos[base + r] : -1;
  int64_t lo_min = INT64_MAX, lo_max = 0, hi_min = INT64_MAX, hi_max = -1;
  for (int t = lane; t < a.T; t += 64) {
    const int64_t hi = a.q_pos[t], lo = a.window > 0 && hi - a.window + 1 > 0 ? hi - a.window + 1 : 0;
    lo_min = min(lo_min, lo), lo_max = max(lo_max, lo), hi_min = min(hi_min, hi), hi_max = max(hi_max, hi);
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    lo_min = min(lo_min, (int64_t)__shfl_xor((long long)lo_min, o, 64));
    lo_max = max(lo_max, (int64_t)__shfl_xor((long long)lo_max, o, 64));
    hi_min = min(hi_min, (int64_t)__shfl_xor((long long)hi_min, o, 64));
    hi_max = max(hi_max, (int64_t)__shfl_xor((long long)hi_max, o, 64));
  }
  const bool any = __any(sp >= lo_min && sp <= hi_max), full = __all(sp < 0 || (sp >= lo_max && sp <= hi_min));
  if (!__syncthreads_or(any)) return;  // (full: an empty slot's sum is not written)

  // The rows that are copied next, 64 of a key head, and their maxima and sums
  // (by every wave, so that all have as many copies under way).
  int rs[PARTS], chunk[PARTS], t0[PARTS], j0[PARTS], c_tok[PARTS], c_sub[PARTS];  // (sub: the row's head among the key head's)
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    const int piece = (i * kWeightWaves + w) * 64 + lane;
    rs[i] = piece / CPR, chunk[i] = ((piece ^ rs[i]) & (CPR - 1)) * 8;
    c_tok[i] = t0[i] = min(rs[i], R - 1) / a.rep, c_sub[i] = j0[i] = min(rs[i], R - 1) % a.rep;
  }
  const int tl = (R - 1) / a.rep, jl = (R - 1) % a.rep, dt = 64 / a.rep, dj = 64 % a.rep;
  int c_head = 0, c_row = 0, c_buf = 0;
  auto copy_rows = [&]() {
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
      const bool in = c_row + rs[i] < R;
      const T* const src = (const T*)a.q + (int64_t)(in ? c_tok[i] : tl) * a.q_st +
                           (int64_t)(c_head * a.rep + (in ? c_sub[i] : jl)) * a.q_sh + chunk[i];
      __builtin_amdgcn_global_load_lds(
          (const void*)src, (__attribute__((address_space(3))) void*)(lds + c_buf * TILEB + (i * kWeightWaves + w) * 1024), 16, 0, 0);
      c_tok[i] += dt, c_sub[i] += dj;
      if (c_sub[i] >= a.rep) c_sub[i] -= a.rep, ++c_tok[i];
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float* const ml = (const float*)(a.row_ml + (int64_t)c_head * R + min(c_row + i * 32 + (lane >> 1), R - 1));
      __builtin_amdgcn_global_load_lds((const void*)(ml + (lane & 1)),
                                       (__attribute__((address_space(3))) void*)(lds + NBUF * TILEB + c_buf * 512 + i * 256), 4, 0, 0);
    }
    c_buf = c_buf + 1 == NBUF ? 0 : c_buf + 1;
    c_row += 64;
    if (c_row >= R) {  // the next key head; past the last one its rows once more
      c_head = min(c_head + 1, a.Hk - 1);
      c_row = 0;
#pragma unroll
      for (int i = 0; i < PARTS; ++i) c_tok[i] = t0[i], c_sub[i] = j0[i];
    }
  };
  const T* kr = (const T*)a.k + min(base + r, last) * a.k_ss + h * 8;  // the lane's slot, of the head loaded next
  auto load_k = [&](V (&to)[KK]) {
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) to[kk] = *(const V*)(kr + kk * 16);
  };

  V kf[KK], kn[KK];
  load_k(kn);
  float acc[16] = {};
  const float scale = a.neg ? -a.scale : a.scale;
#pragma unroll
  for (int i = 0; i < NBUF - 1; ++i) copy_rows();
  int buf = 0;
#pragma unroll 1
  for (int kvh = 0; kvh < a.Hk; ++kvh) {
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) kf[kk] = kn[kk];
    kr += kvh + 1 < a.Hk ? a.k_sh : 0;
    load_k(kn);
#pragma unroll 1
    for (int row0 = 0; row0 < R; row0 += 64) {
      // as in attn_tile_kernel: these rows are there, the place of the rows before is free
      wait_vmcnt<(NBUF - 2) * (PARTS + 2)>();
      wait_lds();
      barrier_nofence();
      copy_rows();
      const uint8_t* const qt = lds + buf * TILEB + r * ROWB;
      const uint8_t* const mt = lds + NBUF * TILEB + buf * 512 + r * 8;
      buf = buf + 1 == NBUF ? 0 : buf + 1;
      if (!any) continue;
      f32x16 s[2] = {(f32x16)(0.0f), (f32x16)(0.0f)};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const V qf = *(const V*)(qt + i * 32 * ROWB + (((kk * 2 + h) ^ r) & (CPR - 1)) * 16);
          if constexpr (CT == XT_F16)
            s[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[kk], qf, s[i], 0, 0, 0);
          else
            s[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[kk], qf, s[i], 0, 0, 0);
        }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = row0 + i * 32 + r;
        const f32x2 ml = *(const f32x2*)(mt + i * 256);
        const float inv = row < R ? ml.y : 0.0f;
        if (full) {
#pragma unroll
          for (int v = 0; v < 16; ++v)
            acc[v] = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(s[i][v], scale, -ml.x)), inv, acc[v]);
        } else {
          const uint32_t seen = sees<16>(a, false, min(row, R - 1) / a.rep, last,
                                         [&](int v) { return base + (v / 4) * 8 + 4 * h + v % 4; });
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][v], scale, -ml.x)) * inv;
            acc[v] += row < R && (seen >> v & 1) ? p : 0.0f;
          }
        }
      }
    }
  }
  __builtin_amdgcn_s_waitcnt(0);  // (no copy outlives the workgroup's LDS)
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    float x = acc[v];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) x += __shfl_xor(x, o, 64);
    const int at = base + (v / 4) * 8 + 4 * h + v % 4;
    if (r == 0 && at <= last && a.slot_pos[at] >= 0) weight[at] += x;
  }
}

// One attention launch of a configuration; defined per pair (cache type,
// 2-byte products) in the files that instantiate the kernel.
template <int CT, bool M16, int DP>
int launch_attn_dp(const AttnArgs& a, int mode, int RT, hipStream_t st) {
  const dim3 grid((unsigned)(a.Hk * a.rtiles * a.splits));
  if (RT == 2) {
    if constexpr (M16 || DP < 256) {  // (two tiles of 256 fp32 columns do not fit the registers)
      if (mode != 2) return -1;
      attn_kernel<CT, M16, DP, 2, 2><<<grid, kAttnWaves * 64, 0, st>>>(a);
    } else {
      return -1;  // no such kernel (the plan never asks for it)
    }
  } else if (RT != 1) {
    return -1;
  } else if (mode == 2) {
    attn_kernel<CT, M16, DP, 2, 1><<<grid, kAttnWaves * 64, 0, st>>>(a);
  } else if (mode == 1) {
    attn_kernel<CT, M16, DP, 1, 1><<<grid, kAttnWaves * 64, 0, st>>>(a);
  } else if constexpr (!M16) {
    attn_kernel<CT, M16, DP, 0, 1><<<grid, kAttnWaves * 64, 0, st>>>(a);
  } else {
    return -1;
  }
  return check_launch();
}

template <int CT, int DP>
int launch_tile_dp(const AttnArgs& a, hipStream_t st) {
  constexpr int lds = kTileBufs * 2 * kTileSlots * DP * 2;
  attn_tile_kernel<CT, DP><<<dim3((unsigned)(a.Hk * a.rtiles * a.splits)), kTileWaves * 64, lds, st>>>(a);
  const int rc = check_launch();
  if (rc) return rc;
  if (a.splits > 1)
    attn_tile_join_kernel<DP><<<dim3((unsigned)(a.Hk * ((a.rep * a.T + 31) / 32) * 16)), 64, 0, st>>>(a);
  return check_launch();
}

template <int CT, bool M16, int DP>
int launch_weight_dp(const AttnArgs& a, int mode, float* weight, hipStream_t st) {
  constexpr int SB = M16 ? 32 : 16, threads = kWeightWaves * 64;
  if constexpr (M16 && DP <= 128) {
    if (mode == 2 && a.qvec && a.rep * a.T >= kWeightTileRows && a.slots >= kWeightTileSlots) {
      attn_weight_tile_kernel<CT, DP><<<(unsigned)((a.slots + 255) / 256), threads, kWeightBufs * (64 * DP * 2 + 512), st>>>(a, weight);
      return check_launch();
    }
  }
  constexpr int64_t kStep = kLaunchThreads / threads * SB;  // slots per launch
  for (int64_t s = 0; s < a.slots; s += kStep) {
    AttnArgs part = a;
    part.k = (const typename XElem<CT>::T*)a.k + s * a.k_ss;
    part.slot_pos = a.slot_pos + s;
    part.slots = (int)(a.slots - s < kStep ? a.slots - s : kStep);
    const dim3 grid((unsigned)((part.slots + SB - 1) / SB));
    if (mode == 2)
      attn_weight_kernel<CT, M16, DP, 2><<<grid, threads, 0, st>>>(part, weight + s);
    else if (mode == 1)
      attn_weight_kernel<CT, M16, DP, 1><<<grid, threads, 0, st>>>(part, weight + s);
    else if constexpr (!M16)
      attn_weight_kernel<CT, M16, DP, 0><<<grid, threads, 0, st>>>(part, weight + s);
    else
      return -1;
    const int rc = check_launch();
    if (rc) return rc;
  }
  return 0;
}

// `weight` null: the attention (RT 0: attn_tile_kernel); else the slots'
// weights after it.
template <int CT, bool M16>
int launch_attn_ct(const AttnArgs& a, int DP, int mode, int RT, float* weight, hipStream_t st) {
  if (weight)
    return DP == 64 ? launch_weight_dp<CT, M16, 64>(a, mode, weight, st)
           : DP == 128 ? launch_weight_dp<CT, M16, 128>(a, mode, weight, st)
                       : launch_weight_dp<CT, M16, 256>(a, mode, weight, st);
  if constexpr (M16) {
    if (RT == 0) return DP == 64 ? launch_tile_dp<CT, 64>(a, st) : launch_tile_dp<CT, 128>(a, st);
  }
  return DP == 64 ? launch_attn_dp<CT, M16, 64>(a, mode, RT, st)
         : DP == 128 ? launch_attn_dp<CT, M16, 128>(a, mode, RT, st)
                     : launch_attn_dp<CT, M16, 256>(a, mode, RT, st);
}

int launch_attn_f32(const AttnArgs& a, int DP, int mode, int RT, float* weight, hipStream_t st);
int launch_attn_f16(const AttnArgs& a, bool m16, int DP, int mode, int RT, float* weight, hipStream_t st);
int launch_attn_bf16(const AttnArgs& a, bool m16, int DP, int mode, int RT, float* weight, hipStream_t st);

}  // namespace sbq
