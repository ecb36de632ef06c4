// sbq_attn.hip - attention over a cache with a tree of drafted tokens: the
// instances for an fp32 cache, the plan, the joining of the splits and the
// attention weight that each slot received (sbq_attn.h holds the kernel).
#include "sbq_attn.h"

#include "sbq_launch.h"

namespace sbq {

int launch_attn_f32(const AttnArgs& a, int DP, int mode, int RT, float* weight, hipStream_t st) {
  return launch_attn_ct<XT_F32, false>(a, DP, mode, RT, weight, st);
}

namespace {

// One row's splits joined: the maximum over their maxima, then the partial
// sums scaled to it.  A thread's loads are independent, eight at a time.
template <int DP>
__device__ __forceinline__ void join_row(const AttnArgs& a, int64_t at) {
  constexpr int ND = DP / 4, NG = 256 / ND, U = 8;
  __shared__ __align__(16) f32x4 lds[NG][ND];
  __shared__ float lds_l[NG];
  const int R = a.rep * a.T, lane = threadIdx.x & 63, d = threadIdx.x % ND * 4, grp = threadIdx.x / ND;
  const float2* const ml = a.part_ml + at * a.splits;
  float top = -__builtin_inff();
  for (int s = lane; s < a.splits; s += 64) top = __builtin_fmaxf(top, ml[s].x);
  top = wave_max(top);
  const float from = top == -__builtin_inff() ? 0.0f : top;
  f32x4 sum = (f32x4)(0.0f);
  float l = 0.0f;
  for (int s0 = grp; s0 < a.splits; s0 += U * NG) {
    f32x4 x[U];
    float2 y[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int s = min(s0 + k * NG, a.splits - 1);
      x[k] = *(const f32x4*)(a.part_o + (at * a.splits + s) * DP + d);
      y[k] = ml[s];
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const float f = __builtin_amdgcn_exp2f(y[k].x - from);
      if (s0 + k * NG < a.splits && y[k].y != 0.0f) {  // (a split that saw nothing adds nothing)
        sum += x[k] * f;
        l += y[k].y * f;
      }
    }
  }
  lds[grp][threadIdx.x % ND] = sum;
  if (d == 0) lds_l[grp] = l;
  __syncthreads();
  if (grp) return;
  l = lds_l[0];
#pragma unroll
  for (int k = 1; k < NG; ++k) {
    sum += lds[k][threadIdx.x];
    l += lds_l[k];
  }
  const float inv = l != 0.0f ? 1.0f / l : 0.0f;
  const int kvh = (int)(at / R), r = (int)(at % R);
  const int64_t out = (int64_t)(r / a.rep) * a.o_st + (int64_t)(kvh * a.rep + r % a.rep) * a.o_sh + d;
  if (d < a.D) store_y4(a.out, a.qt, out, sum * inv, a.ovec && d + 4 <= a.D, a.D - d);
  if (d == 0 && a.row_ml) a.row_ml[at] = make_float2(from, inv);
}

template <int DP>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a) {
  join_row<DP>(a, blockIdx.x);
}

// The joining and, in further workgroups of the same launch, what every slot
// received: weight[s] += sum over the rows that see slot s of exp2(score -
// maximum) / sum, from the scores that the attention kept.  Each of these
// workgroups takes the rows' maxima and sums from the partial ones itself, so
// that none waits for a joined row.  A wave adds up every fourth row, the waves
// are added in order.  What bounds it is the latency of two loads after another
// (few rows: 32 rows over 2304 slots take 0.3 MB).
constexpr int kScoreR = 8, kScoreRows = 256, kScoreStats = 4096;  // rows of a key head, of all; all rows x splits
constexpr int kScoreSlots = 64;  // slots of a step
template <int DP>
__global__ __launch_bounds__(256) void attn_join_weight_kernel(AttnArgs a, float* weight, int strips) {
  __shared__ float2 ml[kScoreRows];
  __shared__ int64_t top_pos[kScoreRows];
  __shared__ float sums[4][kScoreSlots];
  const int R = a.rep * a.T, rows = a.Hk * R, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  if ((int)blockIdx.x < rows) {
    join_row<DP>(a, blockIdx.x);
    return;
  }
  constexpr int U = 8;
  float s[U];
  auto load = [&](int slot, int row0) {
#pragma unroll
    for (int k = 0; k < U; ++k)
      s[k] = a.scores[(int64_t)min(row0 + 4 * k, rows - 1) * a.score_ld + slot];  // (slot < score_ld)
  };
  const int strip0 = ((int)blockIdx.x - rows) * strips;
  load(min(strip0 * kScoreSlots + lane, (int)a.score_ld - 1), w);  // (the first strip's, under the maxima)

  for (int row = threadIdx.x >> 3; row < rows; row += 32) {  // 8 lanes a row
    const float2* const part = a.part_ml + (int64_t)row * a.splits;
    const int first = threadIdx.x & 7;
    float top = -__builtin_inff(), l = 0.0f;
#pragma unroll 1
    for (int s0 = 0; s0 < a.splits; s0 += 8 * U) {  // (the loads of a step together)
      float2 y[U];
#pragma unroll
      for (int k = 0; k < U; ++k) y[k] = part[min(s0 + first + 8 * k, a.splits - 1)];
      float up = top;
#pragma unroll
      for (int k = 0; k < U; ++k) up = __builtin_fmaxf(up, y[k].x);
      const float from = up == -__builtin_inff() ? 0.0f : up;
      l *= __builtin_amdgcn_exp2f(top - from);
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (s0 + first + 8 * k < a.splits && y[k].y != 0.0f) l += y[k].y * __builtin_amdgcn_exp2f(y[k].x - from);
      top = up;
    }
    const float own = top;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) top = __builtin_fmaxf(top, __shfl_xor(top, o, 64));
    const float from = top == -__builtin_inff() ? 0.0f : top;
    l *= __builtin_amdgcn_exp2f(own - from);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) l += __shfl_xor(l, o, 64);
    if (first == 0) {
      ml[row] = make_float2(from, l != 0.0f ? 1.0f / l : 0.0f);
      top_pos[row] = a.q_pos[row % R / a.rep];
    }
  }
  for (int strip = strip0; strip < strip0 + strips && strip * kScoreSlots < a.slots; ++strip) {
    const int slot = strip * kScoreSlots + lane;
    const int64_t pos = slot < a.slots ? a.slot_pos[slot] : -1;
    if (strip > strip0) load(min(slot, (int)a.score_ld - 1), w);
    __syncthreads();  // the maxima are there, the last strip's sums are read
    float sum = 0.0f;
    for (int row0 = w;;) {
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int row = row0 + 4 * k;
        if (row >= rows) break;
        const int64_t hi = top_pos[row], lo = a.window > 0 && hi - a.window + 1 > 0 ? hi - a.window + 1 : 0;
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k], a.scale, -ml[row].x)) * ml[row].y;
        sum += pos >= lo && pos <= hi ? p : 0.0f;
      }
      row0 += 4 * U;
      if (row0 >= rows) break;
      load(min(slot, (int)a.score_ld - 1), row0);
    }
    sums[w][lane] = sum;
    __syncthreads();
    if (w == 0 && slot < a.slots) weight[slot] += sums[0][lane] + sums[1][lane] + sums[2][lane] + sums[3][lane];
  }
}

constexpr int kAttnGroups = 512;    // workgroups aimed at
// attn_tile_kernel: workgroups aimed at (one a CU), and the rows of a key head
// and rows times slots from which it is taken.  8 key heads of 128 bf16
// columns, 256 rows each: 65536 slots 122 us against attn_kernel's 185, 32768
// 74 / 93, 8192 44 / 37; 512 rows: 8192 slots 49 / 58; 128 rows: 65536 slots
// (with 4 waves) 120 / 106.  Other numbers of key heads are not measured.
constexpr int kTileGroups = 256;
constexpr int64_t kTileRows = 256, kTileScores = 1 << 22;

// Scores from which a wave takes two row tiles: they share its loads of keys and
// values, but fewer waves fit a CU, which costs more while a wave has only a few
// blocks.  8 key heads of 128 columns, two tiles against one: 64 rows over 4096
// slots 19.5 us / 15.9 (bf16), 34 / 29 (fp32), over 8192 21.6 / 21.3 and 45 / 44,
// over 16384 26.7 / 31.1 and 65 / 73; 32 rows over 16384 25.5 / 22.3 and 49 / 45.
constexpr int64_t kPairScores = 1 << 22;

int attn_dp(int64_t D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }

struct AttnPlan {
  int RT, rtiles, splits;  // RT: row tiles per wave, 0 for attn_tile_kernel
  int64_t rows;            // rows of a key head that partial sums are kept for
};
// vec: rows of exactly DP columns by 16-byte loads; m16: 2-byte products.
AttnPlan attn_plan(int64_t R, int64_t Hk, int64_t slots, int64_t Tn, int DP, bool vec, bool m16) {
  AttnPlan p;
  int64_t groups = kAttnGroups, each = kAttnWaves, SB = m16 ? 32 : 16;
  if (vec && m16 && DP <= 128 && R >= kTileRows && R * slots >= kTileScores) {
    p.RT = 0;
    p.rtiles = (int)((R + 32 * kTileWaves - 1) / (32 * kTileWaves));
    groups = kTileGroups;
    each = 1, SB = kTileSlots;
  } else {
    // (two tiles of 256 fp32 columns do not fit the registers)
    p.RT = vec && R > 16 && Hk * R * slots > kPairScores && (m16 || DP < 256) ? 2 : 1;
    p.rtiles = (int)((R + 16 * p.RT - 1) / (16 * p.RT));
  }
  p.rows = p.RT == 0 ? (int64_t)p.rtiles * kTileWaves * 32 : R;
  const int64_t room = groups / (Hk * p.rtiles) < 1 ? 1 : groups / (Hk * p.rtiles);
  const int64_t blocks = (slots + SB - 1) / SB + (Tn + SB - 1) / SB;
  const int64_t most = (blocks + each * room - 1) / (each * room);  // blocks of a wave (of a workgroup) at most
  p.splits = (int)((blocks + each * most - 1) / (each * most));
  return p;
}

// Are the scores kept for the slots' weights, [Hk * R][score_ld], and the partial
// results always?  For so few rows that every workgroup can join their maxima.
// 8 key heads of 128 bf16 columns, the weights' share of a call, kept against
// computed again (and a launch less): 4 rows each, 65536 slots 11 us / 32 us,
// 32768 6 / 18; 8 rows 24 / 34 and 13 / 18; 16 rows 49 / 36 and 26 / 19.
bool keeps_scores(const AttnPlan& p, int64_t R, int64_t Hk, bool weight) {
  return weight && p.RT == 1 && R <= kScoreR && Hk * R <= kScoreRows && Hk * R * p.splits <= kScoreStats;
}
int64_t score_ld(int64_t slots) { return (slots + 31) & ~(int64_t)31; }

int64_t round256(int64_t n) { return (n + 255) & ~(int64_t)255; }

}  // namespace

int64_t attn_workspace_bytes(int64_t T, int64_t heads, int64_t Hk, int64_t D, int64_t slots, bool weight) {
  const int64_t R = heads / Hk * T;
  int64_t n = 0;
  for (int way = 0; way < 8; ++way) {  // types, alignment and drafts are not known here
    const AttnPlan p = attn_plan(R, Hk, slots, way & 4 ? T : 0, attn_dp(D), way & 1, way & 2);
    const int64_t parts = Hk * p.rows * p.splits;
    const bool kept = keeps_scores(p, R, Hk, weight);
    int64_t need = p.splits > 1 || kept ? round256(parts * attn_dp(D) * 4) + round256(parts * 8) : 0;
    if (kept) need += round256(Hk * R * score_ld(slots) * 4);
    n = need > n ? need : n;
  }
  if (weight) n += round256(Hk * R * 8);
  return n;
}

int launch_tree_attention(const AttnCall& c, hipStream_t st) {
  const int64_t es = c.ct == XT_F32 ? 4 : 2;
  auto vec = [&](const void* p, int64_t a, int64_t b) {
    return (uintptr_t)p % 16 == 0 && a * es % 16 == 0 && b * es % 16 == 0;
  };
  const int DP = attn_dp(c.D);
  const bool aligned = c.D * es % 16 == 0 && vec(c.k, c.k_ss, c.k_sh) && vec(c.v, c.k_ss, c.k_sh) &&
                       (c.Tn == 0 || (vec(c.kn, c.n_ss, c.n_sh) && vec(c.vn, c.n_ss, c.n_sh)));
  const int mode = !aligned ? 0 : c.D == DP ? 2 : 1;
  const bool m16 = c.ct != XT_F32 && c.qt == c.ct && mode > 0;
  const int64_t Hk = c.Hk, rep = c.heads / Hk, R = rep * c.T;
  const AttnPlan p = attn_plan(R, Hk, c.slots, c.Tn, DP, mode == 2, m16);
  AttnArgs a{};
  a.q = c.q, a.k = c.k, a.v = c.v, a.kn = c.kn, a.vn = c.vn, a.slot_pos = c.slot_pos, a.q_pos = c.q_pos, a.tree = c.tree;
  a.out = c.out;
  a.q_st = c.q_st, a.q_sh = c.q_sh, a.k_ss = c.k_ss, a.k_sh = c.k_sh, a.n_ss = c.n_ss, a.n_sh = c.n_sh;
  a.o_st = c.o_st, a.o_sh = c.o_sh, a.tree_ld = c.tree_ld, a.window = c.window;
  a.T = (int)c.T, a.Hk = (int)Hk, a.rep = (int)rep, a.D = (int)c.D, a.slots = (int)c.slots, a.Tn = (int)c.Tn;
  a.splits = p.splits, a.rtiles = p.rtiles, a.qt = c.qt;
  a.neg = c.scale < 0.0f;
  a.scale = (a.neg ? -c.scale : c.scale) * 1.44269504f;
  const int64_t eq = c.qt == XT_F32 ? 4 : 2;
  a.qvec = (m16 || c.qt == XT_F32) && c.D * eq % 16 == 0 && (uintptr_t)c.q % 16 == 0 && c.q_st * eq % 16 == 0 &&
           c.q_sh * eq % 16 == 0;
  a.ovec = (uintptr_t)c.out % (4 * eq) == 0 && c.o_st % 4 == 0 && c.o_sh % 4 == 0;
  uint8_t* ws = (uint8_t*)c.ws;
  const bool kept = keeps_scores(p, R, Hk, c.weight);
  if (p.splits > 1 || kept) {
    a.part_o = (float*)ws;
    ws += round256(Hk * p.rows * p.splits * DP * 4);
    a.part_ml = (float2*)ws;
    ws += round256(Hk * p.rows * p.splits * 8);
  }
  if (kept) {
    a.scores = (float*)ws;
    a.score_ld = score_ld(c.slots);
  } else if (c.weight) {
    a.row_ml = (float2*)ws;
  }
  auto launch = [&](float* weight) {
    return c.ct == XT_F32   ? launch_attn_f32(a, DP, mode, p.RT, weight, st)
           : c.ct == XT_F16 ? launch_attn_f16(a, m16, DP, mode, p.RT, weight, st)
                            : launch_attn_bf16(a, m16, DP, mode, p.RT, weight, st);
  };
  int rc = launch(nullptr);
  if (rc) return rc;
  if (kept) {
    const int64_t all = (c.slots + kScoreSlots - 1) / kScoreSlots;
    const int strips = (int)((all + 255) / 256);
    const unsigned grid = (unsigned)(Hk * R + (all + strips - 1) / strips);
    if (DP == 64)
      attn_join_weight_kernel<64><<<grid, 256, 0, st>>>(a, c.weight, strips);
    else if (DP == 128)
      attn_join_weight_kernel<128><<<grid, 256, 0, st>>>(a, c.weight, strips);
    else
      attn_join_weight_kernel<256><<<grid, 256, 0, st>>>(a, c.weight, strips);
    return check_launch();
  }
  if (p.splits > 1 && p.RT != 0) {  // (attn_tile_kernel's launch joins its own)
    const unsigned grid = (unsigned)(Hk * R);
    if (DP == 64)
      attn_join_kernel<64><<<grid, 256, 0, st>>>(a);
    else if (DP == 128)
      attn_join_kernel<128><<<grid, 256, 0, st>>>(a);
    else
      attn_join_kernel<256><<<grid, 256, 0, st>>>(a);
    if ((rc = check_launch())) return rc;
  }
  return c.weight ? launch(c.weight) : 0;
}

}  // namespace sbq
