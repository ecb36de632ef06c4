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

// A value that no kernel of the launch writes, at an address the wave shares: by a scalar load.
template <class T>
__device__ __forceinline__ T uniform_load(const T* p) {
  typedef const __attribute__((address_space(4))) T* Const;
  return *(Const)(uintptr_t)p;
}

static_assert(kPagedWaves == kAttnWaves, "the cut deals blocks to a workgroup's waves");

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
// four positions of row c, the operand that O^T = V^T P^T needs.  A wave walks
// blocks of SB positions, loads their keys and values straight to registers
// and keeps a running maximum and sum; LDS only joins a workgroup's waves.
// The cache's bytes, read once, bound long sequences (32 query heads over 8 x 128:
// 65536 bf16 positions 54 us, 5.0 TB/s with the joining; 64 sequences of up to 16384
// e4m3 ones 119 us, 4.8 TB/s); short ones the way to the first keys (launch, lengths,
// page: 3 us) and from the last ones (3 us, and 4 for the joining).
//
// Types of the products:
//   fp32 cache: fp32 (16x16x4).
//   fp16, bf16 cache with its own type's queries: that type (16x16x32); fp32
//     queries in pieces of it (2 of fp16, each row scaled by a power of two, 3
//     of bf16), which hold 22 and 24 bits.
//   8-bit cache: its codes are exact in fp16; queries in fp16 likewise, each
//     row scaled by a power of two, one piece of 2-byte ones, two of fp32.  A
//     position's scales multiply its score and its weight.
// The weights are rounded for the product with V: as many pieces as the queries
// with fp32 ones; else two, whose error stays far below the output's rounding
// (one would add to it: the sum of weights is not rounded with them).  fp16 pieces
// are of what is multiplied, against 2^14 at the row's largest so far: of the
// weight, or with 8 bits of the weight times the value's scale (against the largest
// scale, one far above the others would take their bits with no weight of its own).
// So 2^-28 of the largest keeps 11 bits, and what is lost is 2^-39 of it.  bf16 and
// fp32 ones are against a power of two below it that their number makes up for, or
// large values' sums overflowed on the way to a mean that does not.
struct PagedArgs {
  PagedCache c;
  const void* q;
  const int64_t *start, *counts;
  void* out;
  float* part_o;    // [Hk][places][R][DP]: a part's mean of the values
  float2* part_ml;  // [Hk][places][R]: its largest score, and its sum of weights against that
  int2* joins;      // [tiles of tile_rows rows][n]: a sequence's first slot, and how many
  int64_t q_sb, q_st, q_sh, o_sb, o_st, o_sh, window, first;
  int T, rep, qt, tile_rows;
  int n, slots, places;  // sequences of the launch, workgroups of a key head and row tile (0: one each), their places
  float per_slot;        // 1 / slots
  float scale;               // times log2(e)
  bool ovec;
};

// What the rows of one sequence see: token t the positions first..last, none
// where last < first.
struct PagedSpan {
  int64_t start;
  int count, held;
  // UNIFORM: the same sequence in every lane
  template <bool UNIFORM>
  __device__ __forceinline__ void of(const PagedArgs& a, int64_t b) {
    auto load = [&](const int64_t* p) { return UNIFORM ? uniform_load(p + b) : p[b]; };
    const int64_t room = (int64_t)a.c.max_pages << a.c.page_log, len = load(a.c.length);
    count = a.T;
    if (a.counts) {
      const int64_t n = load(a.counts);
      count = (int)(n < 0 ? 0 : n < a.T ? n : a.T);
    }
    start = len - count;
    if (a.start) start = min(max(load(a.start), -((int64_t)1 << 40)), (int64_t)1 << 40);  // (past every position)
    held = (int)(len < 0 ? 0 : len < room ? len : room);
  }
  __device__ __forceinline__ int last(int t) const {
    const int64_t pos = start + t;
    return t < count && pos >= 0 ? (int)(pos < held ? pos : held - 1) : -1;
  }
  __device__ __forceinline__ int first(int t, int64_t window) const {
    if (window == 0) return 0;
    const int64_t from = start + t - window + 1;
    return (int)(from < 0 ? 0 : from < held ? from : held);
  }
};

// The inclusive sum over the lanes up to this one, by lane moves.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);   // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);   // row_shr:2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);   // row_shr:4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);   // row_shr:8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return v;
}

// How the slots, the workgroups of a key head and row tile, share a launch's
// sequences (the arithmetic is in sbq_index.h).  All sequences' blocks, one
// sequence after another and each in whole fours (one block for each wave), are
// cut into equal parts of four blocks or more, one for each slot: a long
// sequence among short ones has as much of the chip as its length asks for,
// whatever the host knows of lengths.  A part that meets several does them in
// turn, which costs it the way to the first keys and the joining of its waves
// again (about what kPagedLonger fours cost): where parts of up to so many more
// are enough for the sequences to begin with a part each, they do.  A slot has
// at most two pieces of sequences that others share, its first and its last, and
// two places for their partial results (paged_part_place).
// Every workgroup finds its part by a scan over the lengths; which slots a
// sequence has the workgroup of its first block notes for the joining.  Where no
// sequence is long (kPagedWhole), each has a workgroup of its own, and nothing is
// joined.
struct PagedPlace {
  int b, from, blocks;  // the sequence (n: none), its first block and how many (0: sees nothing)
  int before, own;      // the parts' blocks before it, and its own
  int each, total;      // a part's, and all
};
constexpr int kPagedLonger = 3;

template <bool UNIFORM>
__device__ __forceinline__ void paged_look(const PagedArgs& a, int b, int t0, int t1, int SB, PagedPlace& p) {
  PagedSpan span;
  span.of<UNIFORM>(a, a.first + b);
  const int lo = span.first(t0, a.window), hi = span.count > t0 ? span.last(min(t1, span.count - 1)) : -1;
  p.from = lo / SB;
  p.blocks = hi >= lo ? hi / SB + 1 - p.from : 0;
  p.own = paged_own(p.blocks);
}
// The sequence that a slot's part begins in.  t0, t1: the row tile's first and last token.
__device__ __forceinline__ PagedPlace paged_place(const PagedArgs& a, int slot, int t0, int t1, int SB) {
  PagedPlace p;
  p.before = 0;
  if (a.slots == 0) {  // a slot for every sequence
    p.b = slot;
    paged_look<true>(a, slot, t0, t1, SB, p);
    p.total = p.each = p.own;
    return p;
  }
  if (a.n == 1) {
    paged_look<true>(a, 0, t0, t1, SB, p);
    p.total = p.own;
    p.each = paged_each(p.total, a.slots, a.per_slot);
    p.b = (int64_t)slot * p.each >= p.total ? 1 : 0;
    return p;
  }
  const int lane = threadIdx.x & 63;
  PagedPlace l;
  int sum;
  auto look = [&](int b0) {
    paged_look<false>(a, min(b0 + lane, a.n - 1), t0, t1, SB, l);
    if (b0 + lane >= a.n) l.own = 0;
    sum = wave_scan(l.own);
  };
  p.total = 0;
  for (int b0 = 0; b0 < a.n; b0 += 64) {
    look(b0);
    p.total += __builtin_amdgcn_readlane(sum, 63);
  }
  p.each = paged_each(p.total, a.slots, a.per_slot);
  if (a.n <= 64 && 2 * a.n <= a.slots && p.each > kPagedWaves) {  // (parts of one four hold one sequence anyway)
    const int e0 = (p.each + kPagedWaves - 1) & ~(kPagedWaves - 1);
    for (int e = e0; e < e0 + kPagedLonger * kPagedWaves; e += kPagedWaves) {
      const int own = paged_padded(l.own, e), before = wave_scan(own), all = __builtin_amdgcn_readlane(before, 63);
      if (all <= (int64_t)a.slots * e) {
        l.own = own, sum = before, p.total = all, p.each = e;
        break;
      }
    }
  }
  p.b = a.n;
  if ((int64_t)slot * p.each >= p.total) return p;
  const int at = slot * p.each;
  for (int b0 = 0; b0 < a.n; b0 += 64) {
    if (a.n > 64) look(b0);
    const int i = __builtin_popcountll(__ballot(p.before + sum <= at));
    if (i < 64) {
      p.b = b0 + i;
      p.own = __builtin_amdgcn_readlane(l.own, i), p.from = __builtin_amdgcn_readlane(l.from, i);
      p.blocks = __builtin_amdgcn_readlane(l.blocks, i);
      p.before += __builtin_amdgcn_readlane(sum, i) - p.own;
      return p;
    }
    p.before += __builtin_amdgcn_readlane(sum, 63);
  }
  return p;
}
template <int CT>
struct PagedMath : AttnMath<CT == XT_BF16 ? XT_BF16 : XT_F16> {
  typedef typename XElem<CT == XT_BF16 ? XT_BF16 : XT_F16>::T T;
};

// Columns e and e + 1 (e 0 or 2) of a word of e4m3 codes to fp16.
__device__ __forceinline__ uint32_t pair_e4m3(uint32_t w, int e) {
  return e ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, true))
           : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, false));
}

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
    t[0] = pair_e4m3(w0, 0), t[1] = pair_e4m3(w0, 2), t[2] = pair_e4m3(w1, 0), t[3] = pair_e4m3(w1, 2);
  }
  return __builtin_bit_cast(f16x8, t);
}
template <int CT>
__device__ __forceinline__ constexpr int column_of(int j) {
  return CT == CT_I8 ? (j & 4) | (j & 1) << 1 | (j >> 1 & 1) : j;
}

// Bytes e of the words of two positions to fp16, side by side.
__device__ __forceinline__ uint32_t pair_i8(uint32_t hi, uint32_t lo, int e) {
  const uint32_t sel = 0x0c000c00u | (uint32_t)(4 + e) << 16 | (uint32_t)e;
  const uint32_t t = __builtin_amdgcn_perm(hi, lo, sel) | 0x64006400u;
  const f16x2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, t) - off);
}

// Two values in pieces of T, side by side: the nearest first, each next the
// nearest to what is left.
template <class T>
struct Pair {
  typedef T V __attribute__((ext_vector_type(2)));
  template <int N>
  static __device__ __forceinline__ void pieces(float x, float y, uint32_t (&to)[N]) {
    typedef float F2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const V h = __builtin_convertvector(((F2){x, y}), V);
      to[i] = __builtin_bit_cast(uint32_t, h);
      x -= (float)h[0], y -= (float)h[1];
    }
  }
};

// Workgroups of a CU that the registers are bounded for, as many as a launch has: the
// next block's keys and values lie in them (128 columns: 160 to 235 registers; three
// workgroups a CU, in fewer registers or waiting for their turn, 33.6 us for 16 x 8192
// int8 positions, two 27.6).
constexpr int paged_occupancy(int ct, int qt, int DP) {
  return DP == 256 ? is_8bit(ct) && qt != XT_F32 ? 2 : 1 : DP == 128 ? 2 : 3;
}

// Sixteens of rows that a workgroup can take: two where the registers hold them (fp32
// queries and 256 columns spill: 16 x 8192 int8 positions, 8 tokens 122 us against 95).
constexpr int paged_tiles(int qt, int DP) { return qt == XT_F32 || DP > 128 ? 1 : 2; }

// CT: the cache's type, QT: the queries', DP: columns the registers hold (64,
// 128, 256), EXACT: row == DP, RT: sixteens of rows that a block serves (its keys and
// values are loaded and converted once for them).  Grid: key heads of every RT
// sixteens x slots.
template <int CT, int QT, int DP, bool EXACT, int RT>
__global__ __launch_bounds__(kAttnWaves * 64, paged_occupancy(CT, QT, DP)) void paged_attn_kernel(PagedArgs a) {
  constexpr bool B8 = is_8bit(CT), F32 = CT == XT_F32, WIDE = QT == XT_F32 && !F32;
  // pieces of a query and of a weight
  constexpr int NQ = !WIDE ? 1 : CT == XT_BF16 ? 3 : 2, NP = WIDE ? NQ : 2;
  constexpr int ES = ct_bytes(CT), E = 16 / ES, NCH = DP / (4 * E);  // columns in 16 bytes, key loads of a lane's row
  constexpr int SUB = F32 ? 1 : 2, SB = 16 * SUB;
  constexpr int EV = E < DP / 16 ? E : DP / 16, DB = DP / (16 * EV), NF = DP / 16;  // columns of a value load, loads
  constexpr int NFR = DP / 32;                                                       // 16x16x32 steps of a score
  constexpr int HP = 16 * EV > 128 || DP < 128 ? DP : 128, OLD = HP + 4;  // columns joined at a time: whole value loads
  static_assert(HP % (16 * EV) == 0 && DP % HP == 0, "the joining takes whole value loads");
  constexpr float kNone = -__builtin_inff(), kUnitMin = 0x1p-112f;
  typedef typename PagedMath<CT>::T M;
  typedef typename PagedMath<CT>::V MV;
  typedef uint32_t KV __attribute__((ext_vector_type(4)));
  typedef uint32_t VW __attribute__((ext_vector_type(EV * ES / 4)));
  __shared__ __align__(16) float lds_o[kAttnWaves * 16 * OLD];
  __shared__ float lds_m[RT][kAttnWaves][16], lds_l[RT][kAttnWaves][16];
  static_assert(16 * RT * (DP + 4) <= kAttnWaves * 16 * OLD, "the rows of Q fit");

  const PagedCache& pc = a.c;
  const int slot = blockIdx.y, R = a.rep * a.T;
  int kvh = blockIdx.x, row0 = 0;
  if (R > 16 * RT) row0 = kvh / pc.Hk * (16 * RT), kvh %= pc.Hk;
  int t0 = 0, t1 = 0;
  if (a.T > 1) t0 = row0 / a.rep, t1 = min(row0 + 16 * RT - 1, R - 1) / a.rep;
  PagedPlace p = paged_place(a, slot, t0, t1, SB);
  if (p.b >= a.n) return;

  for (;;) {
    int n0, n1;
    paged_piece(a.slots ? slot : 0, p.each, p.before, p.blocks, n0, n1);
    if (n0 < n1) {
      int tid = threadIdx.x;
      asm volatile("" : "+v"(tid));  // (or what depends on it is kept in registers across the sequences)
      const int lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
      const int page_mask = (1 << pc.page_log) - 1;
      // lane offsets in bytes inside a page of a head: its key row (c) and value rows (4g + j)
      const uint32_t row_bytes = pc.row * ES, k_lane = c * row_bytes + g * 16, v_lane = 4 * g * row_bytes + c * EV * ES;
      const int64_t head_bytes = (int64_t)row_bytes << pc.page_log;
      const int64_t b = a.first + p.b;
      PagedSpan span;
      span.of<true>(a, b);
      // the lane's rows' positions, and what every row that sees anything sees
      int lo[RT], hi[RT], lo_max = 0, hi_min = INT32_MAX;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int row = min(row0 + rt * 16 + c, R - 1), tok = a.T > 1 ? row / a.rep : 0;
        lo[rt] = span.first(tok, a.window), hi[rt] = span.last(tok);
        if (hi[rt] >= lo[rt]) lo_max = max(lo_max, lo[rt]), hi_min = min(hi_min, hi[rt]);
      }
      if (a.T > 1) {
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) {
          lo_max = max(lo_max, __shfl_xor(lo_max, o, 64));
          hi_min = min(hi_min, __shfl_xor(hi_min, o, 64));
        }
      }
      lo_max = __builtin_amdgcn_readfirstlane(lo_max), hi_min = __builtin_amdgcn_readfirstlane(hi_min);

      // A block's keys and values, straight to registers.  The next block's follow as
      // soon as this one's are used, so that they are on their way meanwhile; the
      // first one's go ahead of the queries.
      KV kf[SUB][NCH];
      VW vf[4 * SUB][DB];
      f32x4 ks[B8 ? SUB : 1], vs[B8 ? SUB : 1];
      uint32_t held_k = 0;  // sixteens whose page is there
      const int32_t* const table = pc.table + b * pc.max_pages;
      int32_t ids[SUB], ids_v[SUB];
      auto look_up = [&](int n) {  // (past the table's last page: past the length too, whichever page is read)
#pragma unroll
        for (int st = 0; st < SUB; ++st)
          ids[st] = uniform_load(table + min(((p.from + n) * SB + st * 16) >> pc.page_log, pc.max_pages - 1));
      };
      // (sixteen rows of a page through a buffer each: the lane's offset in one
      // register, what the wave shares in scalar ones; past the sixteen rows zeros)
      auto rows_at = [&](const void* pool, int st, int n) {
        const int64_t block = (int64_t)ids_v[st] * pc.Hk + kvh;
        const uint32_t in_page = ((p.from + n) * SB + st * 16) & page_mask;
        return raw_rsrc((const char*)pool + block * head_bytes + in_page * row_bytes, 16 * row_bytes);
      };
      auto scales_at = [&](const float* scale, int st, int n) {
        const int64_t block = (int64_t)ids_v[st] * pc.Hk + kvh;
        const uint32_t in_page = ((p.from + n) * SB + st * 16) & page_mask;
        return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                             raw_rsrc(scale + (block << pc.page_log) + in_page, 64), 16 * g, 0, 0));
      };
      auto load_k = [&](int n) {
        held_k = 0;
#pragma unroll
        for (int st = 0; st < SUB; ++st) {
          if (valid_page(pc, ids[st])) held_k |= 1u << st;
          ids_v[st] = valid_page(pc, ids[st]) ? ids[st] : 0;
          const __amdgpu_buffer_rsrc_t rs = rows_at(pc.k, st, n);
#pragma unroll
          for (int ch = 0; ch < NCH; ++ch)
            kf[st][ch] = __builtin_amdgcn_raw_buffer_load_b128(
                rs, EXACT || ch * 4 * E + g * E < pc.row ? k_lane + ch * 64 : ~0u, 0, 0);
          if constexpr (B8) ks[st] = scales_at(pc.k_scale, st, n);
        }
      };
      auto load_v = [&](int n) {
#pragma unroll
        for (int st = 0; st < SUB; ++st) {
          const __amdgpu_buffer_rsrc_t rs = rows_at(pc.v, st, n);
          if constexpr (B8) vs[st] = scales_at(pc.v_scale, st, n);
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int db = 0; db < DB; ++db) {
              const uint32_t at = EXACT                            ? v_lane + db * 16 * EV * ES
                                  : db * 16 * EV + c * EV < pc.row ? v_lane + j * row_bytes + db * 16 * EV * ES
                                                                   : ~0u;
              VW& to = vf[st * 4 + j][db];
              if constexpr (EV * ES == 16)
                to = __builtin_amdgcn_raw_buffer_load_b128(rs, at, EXACT ? j * row_bytes : 0, 0);
              else if constexpr (EV * ES == 8)
                to = __builtin_amdgcn_raw_buffer_load_b64(rs, at, EXACT ? j * row_bytes : 0, 0);
              else
                to[0] = __builtin_amdgcn_raw_buffer_load_b32(rs, at, EXACT ? j * row_bytes : 0, 0);
            }
        }
      };
      if (n0 + w < n1) {
        look_up(n0 + w);
        load_k(n0 + w);
        load_v(n0 + w);
        look_up(min(n0 + w + kAttnWaves, n1 - 1));
      }

      // the rows of Q by all threads to LDS, and the lane's share of its own
      MV qm[RT][F32 ? 1 : NFR][NQ];
      f32x4 qf[RT][F32 ? NCH : 1];
      float factor[RT];
      const int rows = min(R - row0, 16 * RT);
      {
        typedef typename XElem<QT>::T T;
        constexpr int LD = DP + 4, STEP = kAttnWaves * 64 / DP;
        const int d = tid & (DP - 1);
        const T* const q = (const T*)a.q + b * a.q_sb + (int64_t)kvh * a.rep * a.q_sh + min(d, pc.D - 1);
        __syncthreads();  // (LDS is free of the last sequence)
#pragma unroll 1
        for (int r = tid / DP; r < rows; r += 4 * STEP) {  // four loads at a time
          int tt[4] = {}, hh[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) hh[i] = min(row0 + r + i * STEP, R - 1);
          if (a.T > 1) {
#pragma unroll
            for (int i = 0; i < 4; ++i) tt[i] = hh[i] / a.rep, hh[i] -= tt[i] * a.rep;
          }
          T x[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = q[(int64_t)tt[i] * a.q_st + (int64_t)hh[i] * a.q_sh];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (r + i * STEP < rows) lds_o[(r + i * STEP) * LD + d] = d < pc.D ? (float)x[i] : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const float* const mine = lds_o + min(rt * 16 + c, rows - 1) * LD;
          factor[rt] = a.scale;
          if constexpr (F32) {
#pragma unroll
            for (int ch = 0; ch < NCH; ++ch) qf[rt][ch] = *(const f32x4*)(mine + ch * 16 + g * 4);
          } else {
            constexpr bool SCALED = B8 || (CT == XT_F16 && WIDE);
            f32x4 x[NFR][2];
            float most = 0.0f;
#pragma unroll
            for (int f = 0; f < NFR; ++f)
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                x[f][k] = *(const f32x4*)(mine + (B8 ? f / 2 * 64 + g * 16 + f % 2 * 8 : f * 32 + g * 8) + k * 4);
                if constexpr (SCALED) {
#pragma unroll
                  for (int j = 0; j < 4; ++j) most = __builtin_fmaxf(most, __builtin_fabsf(x[f][k][j]));
                }
              }
            float unit = 1.0f;
            if constexpr (SCALED) {
              most = __builtin_fmaxf(most, __shfl_xor(most, 16, 64));
              most = __builtin_fmaxf(most, __shfl_xor(most, 32, 64));
              const int e = row_scale_exp(most);
              unit = __builtin_ldexpf(1.0f, e);
              factor[rt] = __builtin_ldexpf(a.scale, -e);
            }
#pragma unroll
            for (int f = 0; f < NFR; ++f) {
              u32x4 words[NQ];
#pragma unroll
              for (int j = 0; j < 8; j += 2) {
                uint32_t to[NQ];
                const float y = x[f][column_of<CT>(j) / 4][column_of<CT>(j) % 4];
                const float z = x[f][column_of<CT>(j + 1) / 4][column_of<CT>(j + 1) % 4];
                Pair<M>::pieces(SCALED ? y * unit : y, SCALED ? z * unit : z, to);
#pragma unroll
                for (int i = 0; i < NQ; ++i) words[i][j / 2] = to[i];
              }
#pragma unroll
              for (int i = 0; i < NQ; ++i) qm[rt][f][i] = __builtin_bit_cast(MV, words[i]);
            }
          }
        }
      }

      f32x4 o[RT][NF];
      float m[RT], l[RT];
      float vref[RT], vinv[RT];  // 8-bit: O's unit, the row's largest weight times value scale so far, and 2^14 of its inverse
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int f = 0; f < NF; ++f) o[rt][f] = (f32x4)(0.0f);
        m[rt] = kNone, l[rt] = 0.0f;
        vref[rt] = kUnitMin, vinv[rt] = 0x1p14f / kUnitMin;
      }
      // fp32's exponents: weights against 2^-k of the largest, for fewer than 2^k positions
      const float less_than_all = F32 || CT == XT_BF16 ? (float)(32 - __builtin_clz((unsigned)((n1 - n0) * SB))) : 0.0f;
#pragma unroll 1
      for (int n = n0 + w; n < n1; n += kAttnWaves) {
        const int s0 = (p.from + n) * SB;
        const uint32_t held = held_k;
        const bool full = held == (1u << SUB) - 1 && s0 >= lo_max && s0 + SB - 1 <= hi_min;

        // scores, in powers of two
        float e[RT][SUB][4];
#pragma unroll
        for (int st = 0; st < SUB; ++st) {
          f32x4 s[RT];
          if constexpr (F32) {
            f32x4 t[RT][4];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
              for (int j = 0; j < 4; ++j) t[rt][j] = (f32x4)(0.0f);
#pragma unroll
            for (int ch = 0; ch < NCH; ++ch) {
              const f32x4 kk = __builtin_bit_cast(f32x4, kf[st][ch]);
#pragma unroll
              for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  t[rt][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(kk[j], qf[rt][ch][j], t[rt][j], 0, 0, 0);
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) s[rt] = (t[rt][0] + t[rt][1]) + (t[rt][2] + t[rt][3]);
          } else {
            f32x4 t[RT][NQ];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
              for (int i = 0; i < NQ; ++i) t[rt][i] = (f32x4)(0.0f);
#pragma unroll
            for (int f = 0; f < NFR; ++f) {
              MV kk;
              if constexpr (B8)
                kk = codes_f16<CT>(kf[st][f / 2][f % 2 * 2], kf[st][f / 2][f % 2 * 2 + 1]);
              else
                kk = __builtin_bit_cast(MV, kf[st][f]);
#pragma unroll
              for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int i = 0; i < NQ; ++i) t[rt][i] = PagedMath<CT>::mfma(kk, qm[rt][f][i], t[rt][i]);
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
              for (int i = NQ - 1; i > 0; --i) t[rt][i - 1] += t[rt][i];
              s[rt] = t[rt][0];
            }
          }
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int v = 0; v < 4; ++v) e[rt][st][v] = s[rt][v] * (B8 ? factor[rt] * ks[st][v] : factor[rt]);
        }
        const bool more = n + kAttnWaves < n1;
        if (more) load_k(n + kAttnWaves);

        uint32_t seen[RT];  // bit st * 4 + v: the lane's row sees that position
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          seen[rt] = ~0u;
          f32x4 vr[B8 ? SUB : 1];  // the values' scales, as far as the row sees them
          if constexpr (B8) {
#pragma unroll
            for (int st = 0; st < SUB; ++st) vr[st] = vs[st];
          }
          if (!full) {
            seen[rt] = 0;
#pragma unroll
            for (int st = 0; st < SUB; ++st)
#pragma unroll
              for (int v = 0; v < 4; ++v) {
                const int at = s0 + st * 16 + 4 * g + v;
                if (at >= lo[rt] && at <= hi[rt] && (held >> st & 1)) seen[rt] |= 1u << (st * 4 + v);
                e[rt][st][v] = seen[rt] >> (st * 4 + v) & 1 ? e[rt][st][v] : kNone;
                if constexpr (B8) vr[st][v] = seen[rt] >> (st * 4 + v) & 1 ? vr[st][v] : 0.0f;
              }
          }
          float mx = kNone;
#pragma unroll
          for (int st = 0; st < SUB; ++st)
#pragma unroll
            for (int v = 0; v < 4; ++v) mx = __builtin_fmaxf(mx, e[rt][st][v]);
          mx = reference<XT_F16, CT == XT_F16>(mx) + less_than_all;
          float kept = 1.0f;  // 8-bit: what of the unit is left
          if (__any(mx > m[rt])) {
            mx = __builtin_fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = __builtin_fmaxf(mx, __shfl_xor(mx, 32, 64));
            const float up = __builtin_fmaxf(m[rt], mx), alpha = up == kNone ? 1.0f : __builtin_amdgcn_exp2f(m[rt] - up);
            m[rt] = up;
            l[rt] *= alpha;
            if constexpr (B8) {
              kept = alpha;
            } else {
#pragma unroll
              for (int f = 0; f < NF; ++f) o[rt][f] *= alpha;
            }
          }
          const float from = m[rt] == kNone ? 0.0f : m[rt];
#pragma unroll
          for (int st = 0; st < SUB; ++st)
#pragma unroll
            for (int v = 0; v < 4; ++v) {  // (exp2 of -infinity: what is not seen has weight 0)
              e[rt][st][v] = __builtin_amdgcn_exp2f(e[rt][st][v] - from);
              l[rt] += e[rt][st][v];
            }

          if constexpr (B8) {  // the weights times the values' scales, against 2^14 at the largest of them
            float top = 0.0f;
#pragma unroll
            for (int st = 0; st < SUB; ++st)
#pragma unroll
              for (int v = 0; v < 4; ++v) {
                e[rt][st][v] *= vr[st][v];
                top = __builtin_fmaxf(top, e[rt][st][v]);  // (NaN: the other one)
              }
            const float unit = vref[rt] * kept;
            if (__any(kept != 1.0f || top > unit)) {
              top = __builtin_fmaxf(top, __shfl_xor(top, 16, 64));
              top = __builtin_fmaxf(top, __shfl_xor(top, 32, 64));
              const float up = __builtin_fmaxf(__builtin_fmaxf(unit, top), kUnitMin), alpha = unit / up;
              vref[rt] = up, vinv[rt] = 0x1p14f / up;
#pragma unroll
              for (int f = 0; f < NF; ++f) o[rt][f] *= alpha;
            }
#pragma unroll
            for (int st = 0; st < SUB; ++st)
#pragma unroll
              for (int v = 0; v < 4; ++v) e[rt][st][v] *= vinv[rt];
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
                for (int k = 0; k < EV * ES / 4; ++k) {
                  if constexpr (F32)
                    odd |= !finite(__uint_as_float(vf[j][db][k]));
                  else
                    odd |= Odd2<CT>::any(vf[j][db][k]);
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
              for (int k = 0; k < EV; ++k) {
                float x = __uint_as_float(vf[j][db][k]);
                if (odd) {
#pragma unroll
                  for (int rt = 0; rt < RT; ++rt) {
#pragma unroll 1
                    for (int kind = 0; kind < 3; ++kind) {
                      const f32x4 cnt = __builtin_amdgcn_mfma_f32_16x16x4f32(odd_one(x, kind), seen[rt] >> j & 1 ? 1.0f : 0.0f,
                                                                             (f32x4)(0.0f), 0, 0, 0);
#pragma unroll
                      for (int v = 0; v < 4; ++v)
                        if (cnt[v] > 0.0f) o[rt][db * EV + k][v] += odd_value(kind);
                    }
                  }
                  x = finite(x) ? x : 0.0f;
                }
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                  o[rt][db * EV + k] = __builtin_amdgcn_mfma_f32_16x16x4f32(x, e[rt][0][j], o[rt][db * EV + k], 0, 0, 0);
              }
        } else {
          MV pf[RT][NP];
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            u32x4 words[NP];
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
              uint32_t to[NP];
              Pair<M>::pieces(e[rt][j >> 2][j & 3], e[rt][j >> 2][(j & 3) + 1], to);
#pragma unroll
              for (int i = 0; i < NP; ++i) words[i][j / 2] = to[i];
            }
#pragma unroll
            for (int i = 0; i < NP; ++i) pf[rt][i] = __builtin_bit_cast(MV, words[i]);
          }
#pragma unroll
          for (int db = 0; db < DB; ++db) {
            VW vw[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              vw[j] = vf[j][db];
              if constexpr (CT == CT_I8) vw[j] ^= 0x80808080u;
            }
#pragma unroll
            for (int e0 = 0; e0 < EV; e0 += 2) {  // two columns at a time
              u32x4 t[2];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                if constexpr (CT == CT_I8) {
                  t[0][j] = pair_i8(vw[2 * j + 1][e0 / 4], vw[2 * j][e0 / 4], e0 % 4);
                  t[1][j] = pair_i8(vw[2 * j + 1][e0 / 4], vw[2 * j][e0 / 4], e0 % 4 + 1);
                } else {
                  uint32_t x, y;
                  if constexpr (CT == CT_E4M3) {
                    x = pair_e4m3(vw[2 * j][e0 / 4], e0 % 4), y = pair_e4m3(vw[2 * j + 1][e0 / 4], e0 % 4);
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
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll 1
                      for (int kind = 0; kind < 3; ++kind) {
                        u32x4 ones;
                        MV sees;
#pragma unroll
                        for (int j = 0; j < 4; ++j) ones[j] = Odd2<CT>::ones(t[k][j], kind);
#pragma unroll
                        for (int j = 0; j < 8; ++j) sees[j] = (M)(seen[rt] >> j & 1 ? 1.0f : 0.0f);
                        const f32x4 cnt = PagedMath<CT>::mfma(__builtin_bit_cast(MV, ones), sees, (f32x4)(0.0f));
#pragma unroll
                        for (int v = 0; v < 4; ++v)
                          if (cnt[v] > 0.0f) o[rt][f][v] += odd_value(kind);
                      }
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) t[k][j] = Odd2<CT>::finite(t[k][j]);
                  }
                }
                const MV vt = __builtin_bit_cast(MV, t[k]);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                  for (int i = 0; i < NP; ++i) o[rt][f] = PagedMath<CT>::mfma(vt, pf[rt][i], o[rt][f]);
              }
            }
          }
        }
        if (more) {
          load_v(n + kAttnWaves);
          look_up(min(n + 2 * kAttnWaves, n1 - 1));
        }
      }

      // the workgroup's waves joined: each one's mean of the values, which is never
      // larger than they are, and its sum of weights
      int first = 0, places = 1;
      if (a.slots) places = paged_places(p.b, p.each, p.before, p.blocks, first), first -= p.b;
      const int place = paged_part_place(slot, first);
      const bool alone = places == 1;
      if (a.joins && n0 == 0 && kvh == 0 && tid == 0) a.joins[row0 / (16 * RT) * a.n + p.b] = make_int2(first, places);
      __syncthreads();  // (every wave has read its Q)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        l[rt] += __shfl_xor(l[rt], 16, 64);
        l[rt] += __shfl_xor(l[rt], 32, 64);
        if (g == 0) lds_m[rt][w][c] = m[rt], lds_l[rt][w][c] = l[rt];
        const float less = (B8 ? 0x1p-14f : 1.0f) * (l[rt] != 0.0f ? 1.0f / l[rt] : 0.0f);
        const float unit = B8 ? vref[rt] : 1.0f;  // (after `less`: the product of both can underflow)
        const int here = min(rows - rt * 16, 16);  // (none: nothing is copied or joined)
#pragma unroll
        for (int h0 = 0; h0 < DP; h0 += HP) {
          if (h0 || rt) __syncthreads();
          float* const to = lds_o + (w * 16 + c) * OLD;
          if (c < here) {
#pragma unroll
            for (int db = h0 / (16 * EV); db < (h0 + HP) / (16 * EV); ++db)
#pragma unroll
              for (int v = 0; v < 4; ++v)
#pragma unroll
                for (int k = 0; k < EV; ++k) to[db * 16 * EV - h0 + (4 * g + v) * EV + k] = o[rt][db * EV + k][v] * less * unit;
          }
          __syncthreads();
          for (int u = tid; u < here * (HP / 4); u += kAttnWaves * 64) {
            const int rr = u / (HP / 4), d = h0 + u % (HP / 4) * 4;
            float top = kNone;
#pragma unroll
            for (int k = 0; k < kAttnWaves; ++k) top = __builtin_fmaxf(top, lds_m[rt][k][rr]);
            const float ref = top == kNone ? 0.0f : top;
            f32x4 sum = (f32x4)(0.0f);
            float part[kAttnWaves], ls = 0.0f;
#pragma unroll
            for (int k = 0; k < kAttnWaves; ++k) {  // (a wave that saw nothing adds nothing)
              const float lk = lds_l[rt][k][rr];
              part[k] = lk != 0.0f ? __builtin_amdgcn_exp2f(lds_m[rt][k][rr] - ref) * lk : 0.0f;
              ls += part[k];
            }
            const float inv = ls != 0.0f ? 1.0f / ls : 0.0f;
#pragma unroll
            for (int k = 0; k < kAttnWaves; ++k) {
              const f32x4 x = *(const f32x4*)(lds_o + (k * 16 + rr) * OLD + d - h0);
              if (lds_l[rt][k][rr] != 0.0f) sum += x * (part[k] * inv);  // (an infinity also where its weight is below fp32's)
            }
            const int r = row0 + rt * 16 + rr;
            if (!alone) {
              const int64_t at = ((int64_t)kvh * a.places + place) * R + r;
              *(f32x4*)(a.part_o + at * DP + d) = sum;
              if (d == 0) a.part_ml[at] = make_float2(top, ls);
            } else {
              int t = 0, h = r;
              if (a.T > 1) t = r / a.rep, h = r - t * a.rep;
              const bool any = span.last(t) >= span.first(t, a.window);
              const int64_t out = b * a.o_sb + (int64_t)t * a.o_st + (int64_t)(kvh * a.rep + h) * a.o_sh + d;
              if (d < pc.D) store_y4(a.out, QT, out, any ? sum : (f32x4)(0.0f), a.ovec && d + 4 <= pc.D, pc.D - d);
            }
          }
        }
      }
    }
    p.before += p.own;
    if (p.before >= p.total || p.before >= (int64_t)(slot + 1) * p.each) break;  // (at once where a slot has one sequence)
    ++p.b;
    paged_look<true>(a, p.b, t0, t1, SB, p);
  }
}

template <int CT, int QT, int DP>
int launch_paged_dp(const PagedArgs& a, dim3 grid, hipStream_t st) {
  constexpr int threads = kAttnWaves * 64, RT = paged_tiles(QT, DP);
  const bool exact = a.c.row == DP;
  if constexpr (RT > 1) {
    if (a.tile_rows > 16) {
      exact ? paged_attn_kernel<CT, QT, DP, true, RT><<<grid, threads, 0, st>>>(a)
            : paged_attn_kernel<CT, QT, DP, false, RT><<<grid, threads, 0, st>>>(a);
      return check_launch();
    }
  }
  exact ? paged_attn_kernel<CT, QT, DP, true, 1><<<grid, threads, 0, st>>>(a)
        : paged_attn_kernel<CT, QT, DP, false, 1><<<grid, threads, 0, st>>>(a);
  return check_launch();
}
template <int CT, int QT>
int launch_paged_types(const PagedArgs& a, int DP, dim3 grid, hipStream_t st) {
  return DP == 64    ? launch_paged_dp<CT, QT, 64>(a, grid, st)
         : DP == 128 ? launch_paged_dp<CT, QT, 128>(a, grid, st)
                     : launch_paged_dp<CT, QT, 256>(a, grid, st);
}

int launch_paged_attn_f32(const PagedArgs& a, int DP, dim3 grid, hipStream_t st);
int launch_paged_attn_f16(const PagedArgs& a, int DP, dim3 grid, hipStream_t st);
int launch_paged_attn_bf16(const PagedArgs& a, int DP, dim3 grid, hipStream_t st);
int launch_paged_attn_i8(const PagedArgs& a, int DP, dim3 grid, hipStream_t st);
int launch_paged_attn_e4m3(const PagedArgs& a, int DP, dim3 grid, hipStream_t st);

}  // namespace sbq
