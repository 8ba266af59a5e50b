// Attention over paged latents for a batch whose sequences begin with the same tokens, for gfx950.
//
// MLA-absorb as the sparse attention (value = key, one key head): for head row h (a query row and
// one of its heads) and its tokens t < limit(h),
//   score = (q . k_t + q_rope . k_rope_t) * scale,   out = softmax(score) . k
// with tokens below `prefix` found through block-table row 0 for every sequence, the others through
// the sequence's own row.
//
// What bounds it: one latent row of D + 64 values serves 2 (2 D + 64) operations per head row, so from
// about 300 head rows on the matrix units are the bound, below it the bytes of the latents. The
// work is cut accordingly:
//  * split: the prefix is a matrix product for all the batch's head rows at once (tiles of 128 of
//    them, whichever sequences they belong to), the own tokens a second one per sequence;
//  * joined: where a sequence fills such tiles by itself, its tile runs over prefix and own tokens.
// Both kinds of item, each over a range of tokens, run in one launch; a second one joins the ranges'
// (max, sum, output) per head row, unless every row had a single range.
//
// An item is one work-group of four waves and 32, 64 or 128 head rows (MT 32-row blocks). Tiles of 32
// tokens go direct to a ring of three LDS buffers, two tiles ahead. S^T = K Q^T has the tokens as M and
// 32 head rows as N, the contraction split over the 4 / MT waves of a block (summed through LDS); the
// online softmax runs in each lane's 16 scores of its head row plus one exchange between lane halves,
// and its result is already the B operand of O^T += V^T P^T, whose columns the block's waves share.
#include <algorithm>
#include <climits>
#include <cmath>

#include "dsa_common.hpp"

namespace dsa {
namespace {

constexpr int DR = 64;
constexpr float LOG2E = 1.4426950408889634f;
constexpr int NWV = 4;
constexpr int BN = 32;      // tokens per tile
constexpr int NBUF = 3;

struct PfxK {
  const uint16_t* q;
  const uint16_t* qr;
  const uint16_t* k;
  const uint16_t* kr;
  const int32_t* table;
  const int32_t* row_start;
  const int32_t* act_q;
  const int32_t* act_k;
  int max_blocks, page;
  uint32_t blocks, page_mul;   // page_mul, page_shift: t / page for t < 2^31
  int page_shift;
  int batch, rows, n1, prefix, s2, guess_rows, mode;
  float scale;
  uint16_t* out;
  float* sm_max;
  float* sm_sum;
  float* part_o;    // [slots][rows * n1][D]
  float4* part_s;   // [rows * n1][slots]: reference maximum, true maximum, sum
  int p_mt, p_tiles, p_splits, p_chunk, p_items;   // prefix items
  int o_mt, o_tiles, o_splits, o_chunk, o_base;    // own items (o_base: first token, 0 joined)
  int slots;
};

// A row of zeros, the source of tokens whose block is missing (never written)
__device__ const uint4 g_zero_row[(512 + 8) * 2 / 16] = {};

// 4-byte direct-to-LDS load: lane l writes lds_base + 4 l (see lds_dma16_untracked)
__device__ __forceinline__ void lds_dma4_untracked(const void* gptr, void* lds_base) {
  const uint32_t m0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)lds_base;
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" : : "v"(gptr), "s"(m0) : "memory", "m0");
}

// e^TAU is the largest P relative to the reference maximum: finite in the io type (bf16 has fp32's
// exponents; fp16 ends at e^11.09), so the output is rescaled only when a tile exceeds it
template <int IO> constexpr float lazy_tau() { return IO == IO_F16 ? 8.f : 40.f; }

template <int D> struct Tile {
  static constexpr int KSN = D / 16;           // 32x32x16 steps of the latent part
  static constexpr int KS = (D + DR) / 16;     // and with the rotary part
  static constexpr int ROW = D * 2 + 128;      // LDS bytes of a token's row: 128 modulo 256
  static constexpr int NOPE = BN * ROW;
  static constexpr int ROPE = BN * DR * 2;
  static constexpr int GPW = 10;               // direct-to-LDS loads per wave and tile: 8 rows, rope, ids
};
// Start of token t's row. In the LDS's 64 banks (256 bytes) it lies at 128 (t % 2) + 64 (t / 2 % 2) + 16
// (t / 4 % 4): the operand reads (16 tokens, 16 bytes of one column) and the transposed reads (4
// tokens, 64 bytes) both touch every bank once.
template <int D> __host__ __device__ constexpr int nope_off(int t) {
  return t * Tile<D>::ROW + 64 * ((t >> 1) & 1) + 16 * ((t >> 2) & 3);
}
__device__ __forceinline__ int rope_off(int t, int c) { return (t >> 3) * 1024 + (c * 8 + (t & 7)) * 16; }

// o *= f on an accumulator element in an AGPR, which the VALU cannot use directly
__device__ __forceinline__ float agpr_scale(float o, float f) {
  float t;
  asm volatile("v_accvgpr_read_b32 %1, %0\n\tv_mul_f32 %1, %1, %2\n\tv_accvgpr_write_b32 %0, %1"
               : "+a"(o), "=&v"(t)
               : "v"(f));
  return o;
}

// v_max3 without the quieting of each operand that fmaxf needs (a NaN score reaches the output
// through its exponential either way)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

template <int D> struct PfxLds {
  uint8_t nope[NBUF][Tile<D>::NOPE];
  uint8_t rope[NBUF][Tile<D>::ROPE];
  union {
    uint16_t qr[128 * (DR + 8)];      // MT = 4: the query's rotary part
    float x[NWV][16 * 64];            // MT < 4: partial scores
  };
  int32_t ids[4][BN];
  int red[2][NWV];
  uint32_t bad[2][NWV];               // tokens of the tile (bit) with values that are not finite
};

// limit(h): how many tokens of its sequence head row h's query sees
__device__ __forceinline__ int row_limit(const PfxK& a, int row, int b) {
  const int s1 = row - a.row_start[b], aq = a.act_q[b], ak = a.act_k[b];
  if (s1 >= aq || row >= a.row_start[b + 1]) return 0;
  const int64_t thr = a.mode == 0 ? (int64_t)ak : (int64_t)ak - aq + s1 + 1;
  return (int)(thr < 0 ? 0 : thr > a.s2 ? a.s2 : thr);
}
__device__ __forceinline__ int batch_of(const PfxK& a, int r) {
  const int g = min(r / a.guess_rows, a.batch - 1);
  if (a.row_start[g] <= r && r < a.row_start[g + 1]) return g;
  return batch_of_row(a.row_start, a.batch, r);
}

struct Item {
  int h0, h_end;   // head rows [h0, min(h0 + 32 MT, h_end))
  int b;           // own items: the sequence; -1: prefix
  int t_lo, t_hi;  // tokens, before the rows' limits
  int slot;
};

template <int IO, int D, int MT>
__device__ __forceinline__ void run_item(const PfxK& a, const Item& it, PfxLds<D>& L) {
  using C = Tile<D>;
  constexpr int KSPL = NWV / MT;             // waves of a row block
  constexpr int KSH = C::KS / KSPL;          // their steps of S^T: wave kh takes steps j * KSPL + kh
  constexpr int KNH = C::KSN / KSPL;         // of which in the latent part
  static_assert(C::KS % KSPL == 0 && C::KSN % KSPL == 0 && KSH >= 3, "contraction split");
  constexpr int ON = D / 32 / KSPL;          // their 32-column tiles of O
  constexpr bool QLDS = MT == 4;             // the rotary part of Q stays in LDS
  constexpr int QF = QLDS ? KNH : KSH;       // Q fragments in registers
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rb = wave % MT, kh = wave / MT;
  const int kg = lane >> 5, rr = lane & 31;
  const int h = it.h0 + rb * 32 + rr;
  const bool valid = h < it.h_end;
  const int m_rows = a.rows * a.n1;
  // the softmax works on raw scores times a positive factor: a negative scale negates the query, a
  // zero one becomes 1e-30 (scores round to 0, masked ones stay -inf)
  const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
  const float cpos = a.scale > 0.f ? a.scale : a.scale < 0.f ? -a.scale : 1e-30f;
  const float cl2 = cpos * LOG2E;

  // ---- Q^T fragments (B operand: this lane's head row, 8 values at 16 ks + 8 kg)
  uint4 qf[QF];
  {
    const int hc = valid ? h : it.h_end - 1;
    const uint16_t* qn = a.q + (int64_t)hc * D + kh * 16 + kg * 8;
    const uint16_t* qr = a.qr + (int64_t)hc * DR + kh * 16 + kg * 8;
    auto flipped = [&](uint4 v) { return make_uint4(v.x ^ flip, v.y ^ flip, v.z ^ flip, v.w ^ flip); };
#pragma unroll
    for (int j = 0; j < QF; ++j) qf[j] = flipped(ldg16(j < KNH ? qn + j * KSPL * 16 : qr + (j - KNH) * KSPL * 16));
    if constexpr (QLDS)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<uint4*>(L.qr + (rb * 32 + rr) * (DR + 8) + j * 16 + kg * 8) = flipped(ldg16(qr + j * 16));
  }

  // ---- this head row's tokens: a row that sees none of the item's is dead: it runs along unmasked
  // and leaves a sum of 0
  int lim = 0;
  if (valid) {
    const int row = h / a.n1;
    lim = row_limit(a, row, it.b >= 0 ? it.b : batch_of(a, row));
  }
  const bool dead = lim <= it.t_lo;
  lim = dead ? INT_MAX : min(lim, it.t_hi);   // within the item
  int hi, min_lim;
  {
    int mx = dead ? 0 : lim, mn = lim;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      mx = max(mx, __shfl_xor(mx, o));
      mn = min(mn, __shfl_xor(mn, o));
    }
    if (lane == 0) {
      L.red[0][wave] = mx;
      L.red[1][wave] = mn;
    }
    __syncthreads();   // (and the rotary part of Q)
    mx = max(max(L.red[0][0], L.red[0][1]), max(L.red[0][2], L.red[0][3]));
    mn = min(min(L.red[1][0], L.red[1][1]), min(L.red[1][2], L.red[1][3]));
    hi = __builtin_amdgcn_readfirstlane(mx);        // end of the item's tokens
    min_lim = __builtin_amdgcn_readfirstlane(mn);   // from here on some row is masked
  }
  const bool direct = a.slots == 1;
  const bool writer = kh == 0 && lane < 32 && valid;   // one lane per head row
  if (hi <= it.t_lo) {   // no row sees any token
    if (direct) {
      for (int i = threadIdx.x; i < 32 * MT * (D / 8); i += NWV * 64) {
        const int hr = it.h0 + i / (D / 8);
        if (hr < it.h_end) stg16(a.out + (int64_t)hr * D + (i % (D / 8)) * 8, make_uint4(0, 0, 0, 0));
      }
      if (writer && a.sm_max) a.sm_max[h] = a.sm_sum[h] = 0.f;
    } else if (writer) {
      a.part_s[(int64_t)h * a.slots + it.slot] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    return;
  }
  const int ntiles = (hi - it.t_lo + BN - 1) / BN;

  // ---- ids and gathers. Wave w copies tokens 8 w .. 8 w + 7 of each tile; their block ids travel the
  // same ordered path four tiles ahead, so nothing waits for them. Tokens past the end repeat the last
  // one, tiles past the end the last tile: every wave issues the same GPW loads per tile.
  auto token = [&](int u) { return min(it.t_lo + min(u, ntiles - 1) * BN + wave * 8 + (lane & 7), hi - 1); };
  auto page_of = [&](int t) { return (int)(((uint64_t)(uint32_t)t * a.page_mul) >> (31 + a.page_shift)); };
  auto ids_dma = [&](int u) __attribute__((always_inline)) {
    const int t = token(u);
    const int32_t* src = a.table + (t < a.prefix || it.b < 0 ? 0 : (int64_t)it.b * a.max_blocks) + page_of(t);
    if (lane < 8) lds_dma4_untracked(src, &L.ids[u & 3][wave * 8]);
  };
  // cache row of token 8 w + lane % 8 of tile u, -1: its block is missing
  auto tile_rows = [&](int u) __attribute__((always_inline)) {
    const int t = token(u);
    const int32_t id = L.ids[u & 3][wave * 8 + (lane & 7)];
    return (uint32_t)id < a.blocks ? id * a.page + (t - page_of(t) * a.page) : -1;
  };
  // one of the GPW - 1 gathers of a tile: the latent of token 8 w + j, or (j = 8) the wave's rotary
  // parts. The empty asm keeps the address arithmetic here, among the MFMAs it is issued with.
  auto gather_part = [&](int j, int row, uint8_t* nope, uint8_t* rope) __attribute__((always_inline)) {
    if (j < 8) {
      int r = __builtin_amdgcn_readlane(row, j);
      asm volatile("" : "+s"(r));
      const uint16_t* src = r >= 0 ? a.k + (int64_t)r * D : reinterpret_cast<const uint16_t*>(g_zero_row);
      if (lane < D / 8) lds_dma16_sbase_untracked(src, lane * 16, nope + nope_off<D>(wave * 8 + j));
    } else {
      int r = row;
      asm volatile("" : "+v"(r));
      const uint16_t* src = r >= 0 ? a.kr + (int64_t)r * DR : reinterpret_cast<const uint16_t*>(g_zero_row);
      lds_dma16_untracked(src + (lane >> 3) * 8, rope + wave * 1024);
    }
  };
  // A tile that some of the head rows see only in part: a masked token has P = 0, but 0 times a value
  // that is not finite would still reach the rows that do not see it. Such values become 0 in LDS, and
  // the token's score NaN for the rows that do see it. (Each wave its own rows, landed by now.)
  auto is_mixed = [&](int u) { return min_lim < hi && it.t_lo + u * BN + BN > min_lim; };
  auto sanitize = [&](int u) __attribute__((always_inline)) {
    uint32_t bad = 0;
#pragma unroll 1
    for (int j = 0; j < 8; ++j) {
      uint4* p = reinterpret_cast<uint4*>(L.nope[u % NBUF] + nope_off<D>(wave * 8 + j) + (lane % (D / 8)) * 16);
      uint4 v = *p;
      bool any = false;
      constexpr uint32_t EXP = IO == IO_BF16 ? 0x7F80u : 0x7C00u;
      auto clean = [&](uint32_t w) {
        if ((w & EXP) == EXP) w &= 0xFFFF0000u, any = true;
        if (((w >> 16) & EXP) == EXP) w &= 0xFFFFu, any = true;
        return w;
      };
      v = make_uint4(clean(v.x), clean(v.y), clean(v.z), clean(v.w));
      if (any && lane < D / 8) *p = v;
      if (__builtin_amdgcn_ballot_w64(any)) bad |= 1u << (wave * 8 + j);
    }
    if (lane == 0) L.bad[u & 1][wave] = bad;
  };
#pragma unroll
  for (int u = 0; u < 4; ++u) ids_dma(u);
  wait_vmcnt<0>();
  asm volatile("" ::: "memory");
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int row = tile_rows(u);
#pragma unroll
    for (int j = 0; j < 9; ++j) gather_part(j, row, L.nope[u], L.rope[u]);
  }

  {   // an AGPR operand makes the compiler keep the MFMA accumulators there, the VGPRs free for operands
    float agpr_hint = 0.f;
    asm volatile("" : "+a"(agpr_hint));
  }
  f32x16 o[ON];
#pragma unroll
  for (int n = 0; n < ON; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[n][i] = 0.f;

  // ---- S^T of tile u. Its rows are permuted so that a lane's 16 scores are tokens 16 (i / 8) + 8 kg +
  // i % 8: the order of the B operand of the PV product. Operands are read KPF steps ahead; `spread(j)`
  // issues what rides on step j, `pre()` what covers the first operands' latency.
  const int tk = 16 * (rr >> 4) + 8 * ((rr >> 2) & 1) + 4 * ((rr >> 3) & 1) + (rr & 3);
  constexpr int KPF = KSH < 5 ? KSH : 5;
  auto s_tile = [&](int u, auto&& spread, auto&& pre) __attribute__((always_inline)) -> f32x16 {
    const uint8_t* arow = L.nope[u % NBUF] + nope_off<D>(tk) + kg * 16 + kh * 32;
    const uint8_t* rrow = L.rope[u % NBUF] + rope_off(tk, kh * 2 + kg);
    auto a_frag = [&](int j) -> uint4 {
      return j < KNH ? *reinterpret_cast<const uint4*>(arow + j * KSPL * 32)
                     : *reinterpret_cast<const uint4*>(rrow + (j - KNH) * KSPL * 256);
    };
    constexpr int NR = QLDS ? KSH - KNH : 1;
    uint4 qr[NR];
    auto qr_frag = [&](int j) -> uint4 {
      return *reinterpret_cast<const uint4*>(L.qr + (rb * 32 + rr) * (DR + 8) + j * 16 + kg * 8);
    };
    uint4 af[KPF];
#pragma unroll
    for (int j = 0; j < KPF; ++j) af[j] = a_frag(j);
    pre();
    f32x16 acc;
#pragma unroll
    for (int j = 0; j < KSH; ++j) {
      uint4 bq;
      if constexpr (QLDS) bq = j < KNH ? qf[j < QF ? j : 0] : qr[j >= KNH ? j - KNH : 0];
      else bq = qf[j];
      if (j == 0) acc = mfma32_vacc_first<IO>(af[0], bq);
      else if (j < KSH - 1) mfma32_vacc<IO>(acc, af[j % KPF], bq);
      else acc = mfma32_vacc_last_to<IO>(acc, af[j % KPF], bq);
      if (j + KPF < KSH) af[j % KPF] = a_frag(j + KPF);
      if constexpr (QLDS)
        if (j + KPF < KSH && j + KPF >= KNH) qr[j + KPF - KNH] = qr_frag(j + KPF - KNH);
      spread(j);
      __builtin_amdgcn_sched_barrier(0);
    }
    return acc;
  };
  // several waves of a row block add their parts in one order: the same bits in each
  auto put_part = [&](const f32x16& sv) __attribute__((always_inline)) {
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<float4*>(&L.x[wave][(g * 64 + lane) * 4]) =
          make_float4(sv[4 * g], sv[4 * g + 1], sv[4 * g + 2], sv[4 * g + 3]);
  };
  auto sum_parts = [&]() __attribute__((always_inline)) -> f32x16 {
    f32x16 sv;
#pragma unroll
    for (int w = 0; w < KSPL; ++w)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 p = *reinterpret_cast<const float4*>(&L.x[rb + MT * w][(g * 64 + lane) * 4]);
        sv[4 * g] = w == 0 ? p.x : sv[4 * g] + p.x;
        sv[4 * g + 1] = w == 0 ? p.y : sv[4 * g + 1] + p.y;
        sv[4 * g + 2] = w == 0 ? p.z : sv[4 * g + 2] + p.z;
        sv[4 * g + 3] = w == 0 ? p.w : sv[4 * g + 3] + p.w;
      }
    return sv;
  };
  auto mask = [&](int u, f32x16& sv) __attribute__((always_inline)) {
    const int t0 = it.t_lo + u * BN;
    if (t0 + BN <= min_lim) return;
    if (is_mixed(u)) {
      const uint32_t bad = L.bad[u & 1][0] | L.bad[u & 1][1] | L.bad[u & 1][2] | L.bad[u & 1][3];
      if (bad)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if ((bad >> (16 * (i >> 3) + 8 * kg + (i & 7))) & 1u) sv[i] = __builtin_nanf("");
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) sv[i] = t0 + 16 * (i >> 3) + 8 * kg + (i & 7) < lim ? sv[i] : -INFINITY;
  };

  // ---- online softmax in NST stages of a few VALU operations each, placed among the previous tile's
  // PV MFMAs: 0-3 the maximum, 4 the reference maximum, 5-12 two exponentials each, 13 the sum and the
  // B operands of the two 16-token steps. Raw scores; max(c s) = c max(s) as c > 0. The reference m_used
  // moves only past the lazy threshold, so the output's factor alpha is nearly always 1.
  float m_used = -INFINITY, m_true = -INFINITY, l_part = 0.f, alpha = 1.f;
  float sm_mx = 0.f, sm_mb = 0.f, sm_sum = 0.f;
  uint32_t sm_d[4][2];
  uint4 pb[2], pn[2];   // P of the tile whose PV runs, and of the next one
  constexpr int NST = 14;
  auto smx = [&](int st, const f32x16& sv) __attribute__((always_inline)) {
    if (st < 4) {
      const int b = 4 * st;
      sm_mx = st == 0 ? max3(sv[0], sv[1], sv[2]) : max3(sm_mx, sv[b], sv[b + 1]);
      sm_mx = st == 0 ? max3(sm_mx, sv[3], sv[3]) : max3(sm_mx, sv[b + 2], sv[b + 3]);
    } else if (st == 4) {
      const float mx = max_half_swap(sm_mx) * cpos;
      m_true = max3(m_true, mx, mx);
      const float m_new = mx > m_used + lazy_tau<IO>() ? mx : m_used;
      alpha = m_used == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m_used - m_new) * LOG2E);
      m_used = m_new;
      sm_mb = m_used * LOG2E;
      sm_sum = 0.f;
    } else if (st < NST - 1) {
      const int i = 2 * (st - 5);
      const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[i], cl2, -sm_mb));
      const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[i + 1], cl2, -sm_mb));
      sm_sum += p0;
      sm_sum += p1;
      sm_d[i >> 2][(i >> 1) & 1] = pack2<IO>(p0, p1);
    } else {
      l_part = l_part * alpha + sm_sum;
      pn[0] = make_uint4(sm_d[0][0], sm_d[0][1], sm_d[1][0], sm_d[1][1]);
      pn[1] = make_uint4(sm_d[2][0], sm_d[2][1], sm_d[3][0], sm_d[3][1]);
    }
  };
  auto rescale = [&]() __attribute__((always_inline)) {
    if (__builtin_amdgcn_ballot_w64(alpha != 1.f)) {
#pragma unroll
      for (int n = 0; n < ON; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[n][i] = agpr_scale(o[n][i], alpha);
    }
  };

  // ---- O^T += V^T P^T: MFMA m is column tile m % ON of 16-token step m / ON. The transposed operands
  // run VR MFMAs ahead in one ring across tiles: past a tile's last MFMA the reads go on with the next
  // tile's first operands, resident since the barrier before.
  const int g16 = lane >> 4, c16 = lane & 15;
  // (tok0 has bit 2 clear: four tokens on is 4 ROW + 16 bytes on)
  const int vlane = nope_off<D>((g16 >> 1) * 8 + (c16 >> 2)) + ((g16 & 1) * 16 + 4 * (c16 & 3)) * 2 + kh * (D / KSPL) * 2;
  constexpr int NPV = 2 * ON;
  constexpr int VR = NPV < 8 ? NPV : 8;
  constexpr int NPRE = NPV >= 16 ? 6 : NPV / 4;                       // before the next tile's S^T
  constexpr int NMID = KSPL > 1 ? NPRE + (NPV - NPRE) / 2 : NPRE;     // before its partial sums are read
  uint4 vb[VR];
  auto v_base = [&](int u) __attribute__((always_inline)) -> uint32_t {
    uint32_t b = lds_addr(L.nope[u % NBUF]) + vlane;
    asm volatile("" : "+v"(b));   // constant offsets then go into the reads
    return b;
  };
  auto v_frag = [&](uint32_t b, int m) __attribute__((always_inline)) -> uint4 {
    const uint32_t p = b + (m / ON) * 16 * C::ROW + (m % ON) * 64;
    const uint2 lo = ds_read_tr_at(p), hi2 = ds_read_tr_at(p + 4 * C::ROW + 16);
    return make_uint4(lo.x, lo.y, hi2.x, hi2.y);
  };
  auto pv_run = [&](int m0, int m1, uint32_t vbase, uint32_t vnext, bool next, auto&& between)
      __attribute__((always_inline)) {
#pragma unroll
    for (int m = m0; m < m1; ++m) {
      o[m % ON] = Mfma<IO>::m32(vb[m % VR], pb[m / ON], o[m % ON]);
      if (m + VR < NPV) vb[m % VR] = v_frag(vbase, m + VR);
      else if (next) vb[m % VR] = v_frag(vnext, m + VR - NPV);
      between(m);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  wait_vmcnt<C::GPW - 1>();   // tile 0 here, tile 1 may be under way
  if (is_mixed(0)) sanitize(0);
  lds_barrier();
  {
    f32x16 s0 = s_tile(0, [](int) {}, [] {});
    if constexpr (KSPL > 1) {
      put_part(s0);
      lds_barrier();
      s0 = sum_parts();
    }
    mask(0, s0);
#pragma unroll
    for (int st = 0; st < NST; ++st) smx(st, s0);
    const uint32_t vb0 = v_base(0);
#pragma unroll
    for (int m = 0; m < VR; ++m) vb[m] = v_frag(vb0, m);
  }
  // Iteration t: PV of tile t around S^T of tile t + 1, on whose steps the gathers of tile t + 2 ride; the
  // softmax of tile t + 1 runs among the last PV MFMAs.
  for (int tv = 0; tv + 1 < ntiles; ++tv) {
    const int t = __builtin_amdgcn_readfirstlane(tv);   // (the compiler may keep the counter in a VGPR)
    pb[0] = pn[0];
    pb[1] = pn[1];
    rescale();
    if (t == 0) wait_vmcnt<0>();   // this wave's part of tile t + 1 (its ids copy may be under way)
    else wait_vmcnt<1>();
    if (is_mixed(t + 1)) sanitize(t + 1);
    lds_barrier();   // tile t + 1 resident; every wave done with tile t - 1, whose buffer is free
    const int row = tile_rows(t + 2);
    const int gb = __builtin_amdgcn_readfirstlane((t + 2) % NBUF);   // the free buffer
    uint8_t* const gnope = L.nope[gb];
    uint8_t* const grope = L.rope[gb];
    const uint32_t vbase = v_base(t), vnext = v_base(t + 1);
    f32x16 s1 = s_tile(
        t + 1,
        [&](int ks) __attribute__((always_inline)) {
#pragma unroll
          for (int j = 0; j < C::GPW; ++j)
            if (j * KSH / C::GPW == ks) {
              if (j < C::GPW - 1) gather_part(j, row, gnope, grope);
              else ids_dma(t + 4);   // the slot of tile t's ids, read two iterations ago
            }
        },
        [&]() __attribute__((always_inline)) { pv_run(0, NPRE, vbase, vnext, true, [](int) {}); });
    if constexpr (KSPL > 1) {
      put_part(s1);
      pv_run(NPRE, NMID, vbase, vnext, true, [](int) {});
      lds_barrier();
      s1 = sum_parts();
    }
    mask(t + 1, s1);
    pv_run(NMID, NPV, vbase, vnext, true, [&](int m) __attribute__((always_inline)) {
#pragma unroll
      for (int st = 0; st < NST; ++st)
        if (st * (NPV - NMID) / NST == m - NMID) smx(st, s1);
    });
    __builtin_amdgcn_sched_barrier(0);
  }
  pb[0] = pn[0];
  pb[1] = pn[1];
  rescale();
  pv_run(0, NPV, v_base(ntiles - 1), 0u, false, [](int) {});
  wait_vmcnt<0>();   // the ring's last (unused) gathers land before the LDS is released

  // ---- epilogue: lane l holds head row h, columns n * 32 + 8 g + 4 kg + j of o[n][4 g + j]
  const float l_tot = add_half_swap(l_part);
  if (a.scale == 0.f) m_true *= 0.f;
  if (writer) {
    if (!direct) {
      a.part_s[(int64_t)h * a.slots + it.slot] = make_float4(m_used, m_true, dead ? 0.f : l_tot, 0.f);
    } else if (a.sm_max) {
      a.sm_max[h] = dead ? 0.f : m_true;
      a.sm_sum[h] = dead ? 0.f : l_tot * exp2f((m_used - m_true) * LOG2E);
    }
  }
  if (!direct) {
    if (!valid || dead) return;
    float* dst = a.part_o + ((int64_t)it.slot * m_rows + h) * D + kh * (D / KSPL) + 4 * kg;
#pragma unroll
    for (int n = 0; n < ON; ++n)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4*>(dst + n * 32 + 8 * g) =
            make_float4(o[n][4 * g], o[n][4 * g + 1], o[n][4 * g + 2], o[n][4 * g + 3]);
    return;
  }
  // two exchanges between lane halves leave lanes 0-31 with columns [0, 8) and [16, 24) of a 32-column
  // tile, the others with [8, 16) and [24, 32): 16-byte stores
  const float inv = 1.f / l_tot;
  uint16_t* dst = a.out + (int64_t)(valid ? h : 0) * D + kh * (D / KSPL) + 8 * kg;
#pragma unroll
  for (int n = 0; n < ON; ++n) {
    uint32_t d[4][2];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      d[g][0] = dead ? 0u : pack2<IO>(o[n][4 * g] * inv, o[n][4 * g + 1] * inv);
      d[g][1] = dead ? 0u : pack2<IO>(o[n][4 * g + 2] * inv, o[n][4 * g + 3] * inv);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      swap_halves(d[0][j], d[1][j]);
      swap_halves(d[2][j], d[3][j]);
    }
    if (valid) {
      stg16(dst + n * 32, make_uint4(d[0][0], d[0][1], d[1][0], d[1][1]));
      stg16(dst + n * 32 + 16, make_uint4(d[2][0], d[2][1], d[3][0], d[3][1]));
    }
  }
}

template <int IO, int D>
__global__ __launch_bounds__(NWV * 64) void prefix_attn_kernel(PfxK a) {
  __shared__ __attribute__((aligned(16))) PfxLds<D> L;
  Item it;
  int i = blockIdx.x;
  int mt;
  if (i < a.p_items) {
    const int sp = i / a.p_tiles, tile = i - sp * a.p_tiles;
    mt = a.p_mt;
    it.h0 = tile * 32 * mt;
    it.h_end = a.rows * a.n1;
    it.b = -1;
    it.t_lo = sp * a.p_chunk;
    it.t_hi = sp == a.p_splits - 1 ? a.prefix : min(a.prefix, it.t_lo + a.p_chunk);
    it.slot = sp;
  } else {
    i -= a.p_items;
    const int per = a.o_tiles * a.o_splits;
    const int b = i / per;
    i -= b * per;
    const int sp = i / a.o_tiles, tile = a.o_tiles - 1 - (i - sp * a.o_tiles);
    mt = a.o_mt;
    const int r0 = a.row_start[b], r1 = a.row_start[b + 1];
    it.h0 = r0 * a.n1 + tile * 32 * mt;
    it.h_end = r1 * a.n1;
    if (a.slots == 1 && b == a.batch - 1) {   // rows behind the last sequence: zeros
      const int64_t end = (int64_t)a.rows * a.n1 * (D / 8);
      for (int64_t j = (int64_t)it.h_end * (D / 8) + tile * (NWV * 64) + threadIdx.x; j < end; j += a.o_tiles * (NWV * 64)) {
        stg16(a.out + j * 8, make_uint4(0, 0, 0, 0));
        if (a.sm_max && j % (D / 8) == 0) a.sm_max[j / (D / 8)] = a.sm_sum[j / (D / 8)] = 0.f;
      }
    }
    if (it.h0 >= it.h_end) return;
    it.b = b;
    it.t_lo = a.o_base + sp * a.o_chunk;
    it.t_hi = sp == a.o_splits - 1 ? INT_MAX : it.t_lo + a.o_chunk;
    it.slot = a.p_splits + sp;
  }
  if (mt == 1) run_item<IO, D, 1>(a, it, L);
  else if (mt == 2) run_item<IO, D, 2>(a, it, L);
  else run_item<IO, D, 4>(a, it, L);
}

// Joins the ranges of a head row: M = max m_s, out = sum O_s 2^(m_s - M) / sum l_s 2^(m_s - M), and the
// rows of no sequence get zeros. 64 lanes hold the row's statistics (a slot each, in turns), D / 4
// threads its columns.
template <int IO, int D>
__global__ __launch_bounds__(256) void prefix_merge_kernel(PfxK a) {
  constexpr int TPR = D / 4;           // threads a row: 128, 64, 32
  const int m_rows = a.rows * a.n1;
  const int h = blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  const int c = (threadIdx.x % TPR) * 4;
  if (h >= m_rows) return;
  const int row = h / a.n1;
  const bool live = row_limit(a, row, batch_of(a, row)) > 0;
  const float4* ps = a.part_s + (int64_t)h * a.slots;
  float M = -INFINITY, mt = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (live) {
    for (int s = 0; s < a.slots; ++s) {
      const float4 st = ps[s];
      if (st.z != 0.f) {   // (NaN sums take part)
        M = fmaxf(M, st.x);
        mt = fmaxf(mt, st.y);
      }
    }
    for (int s = 0; s < a.slots; ++s) {
      const float4 st = ps[s];
      if (st.z == 0.f) continue;
      const float w = exp2f((st.x - M) * LOG2E);
      const float4 v = *reinterpret_cast<const float4*>(a.part_o + ((int64_t)s * m_rows + h) * D + c);
      l += st.z * w;
      acc.x += v.x * w;
      acc.y += v.y * w;
      acc.z += v.z * w;
      acc.w += v.w * w;
    }
    const float inv = 1.f / l;
    acc.x *= inv;
    acc.y *= inv;
    acc.z *= inv;
    acc.w *= inv;
  }
  *reinterpret_cast<uint2*>(a.out + (int64_t)h * D + c) = make_uint2(pack2<IO>(acc.x, acc.y), pack2<IO>(acc.z, acc.w));
  if (c == 0 && a.sm_max) {
    a.sm_max[h] = live ? mt : 0.f;
    a.sm_sum[h] = live ? l * exp2f((M - mt) * LOG2E) : 0.f;
  }
}

constexpr int MAX_SLOTS = 256;

// How a call is cut. Counts are host-known bounds; the kernel's ranges are right for any lengths.
struct Cut {
  int p_mt, p_tiles, p_splits, p_chunk;
  int o_mt, o_tiles, o_splits, o_chunk, o_base;
  int slots;
};

int mt_for(int64_t head_rows) { return head_rows > 64 ? 4 : head_rows > 32 ? 2 : 1; }
int up(int x, int to) { return (x + to - 1) / to * to; }

Cut make_cut(int batch, int rows, int n1, int prefix, int max_rows, int max_kv, int kv_splits) {
  Cut c{};
  const int64_t m = (int64_t)rows * n1;
  const int own = max_kv > prefix ? max_kv - prefix : 0;
  c.o_mt = mt_for((int64_t)max_rows * n1);
  c.o_tiles = (int)(((int64_t)max_rows * n1 + 32 * c.o_mt - 1) / (32 * c.o_mt));
  const int64_t o_all = std::min<int64_t>((int64_t)batch * c.o_tiles, m / (32 * c.o_mt) + batch);
  c.p_mt = mt_for(m);
  c.p_tiles = (int)((m + 32 * c.p_mt - 1) / (32 * c.p_mt));
  const bool joined = prefix == 0 || o_all * c.o_mt * 8 <= (int64_t)c.p_tiles * c.p_mt * 9;
  constexpr int CUS = 256;
  if (joined) {
    c.p_tiles = 0;
    c.o_base = 0;
    const int64_t tiles = std::max<int64_t>(o_all, 1);
    const int all = std::max(max_kv, 1);
    int best = 1;
    double least = 1e30;
    for (int s = 1; s <= 64 && (s == 1 || (s - 1) * BN < all); ++s) {
      const int chunk = up((all + s - 1) / s, BN);
      // rounds of items, each its tiles and a fixed part of about four; the join reads and writes
      const double cost = (double)((tiles * s + CUS - 1) / CUS) * (chunk / BN + 4) + (s > 1 ? 3.0 + tiles * s * 0.01 : 0.0);
      if (cost < least) least = cost, best = s;
    }
    if (kv_splits > 0) best = kv_splits;
    c.o_splits = best;
    c.o_chunk = up((all + best - 1) / best, BN);
    c.slots = best;
    return c;
  }
  c.o_base = prefix;
  // split: ranges of one length for both kinds, as many items as keep the CUs busy
  int best = BN;
  double least = 1e30;
  for (int chunk = BN; chunk <= std::max(prefix, own) + BN; chunk += up(chunk / 8, BN)) {
    const int64_t np = (prefix + chunk - 1) / chunk, no = (own + chunk - 1) / chunk;
    if (np + no > MAX_SLOTS) continue;
    const int64_t items = np * c.p_tiles + no * o_all;
    const double cost = (double)((items + CUS - 1) / CUS) * (std::min(chunk, std::max(prefix, own)) / (double)BN + 4) +
                        3.0 + (double)(np + no) * m / 128 * 0.01;
    if (cost < least) least = cost, best = chunk;
  }
  if (kv_splits > 0) best = up((prefix + kv_splits - 1) / kv_splits, BN);
  c.p_chunk = c.o_chunk = best;
  c.p_splits = (prefix + best - 1) / best;
  c.o_splits = std::max(1, std::min((own + best - 1) / best, MAX_SLOTS - c.p_splits));
  c.slots = c.p_splits + c.o_splits;
  return c;
}

template <int IO>
hipError_t launch_io(const PfxK& k, int d, hipStream_t s) {
  const int64_t items = (int64_t)k.p_items + (int64_t)k.batch * k.o_tiles * k.o_splits;
  const int64_t m = (int64_t)k.rows * k.n1;
#define DSA_PFX(DD)                                                                                               \
  hipLaunchKernelGGL((prefix_attn_kernel<IO, DD>), dim3((unsigned)items), dim3(NWV * 64), 0, s, k);                \
  if (k.slots > 1)                                                                                                 \
    hipLaunchKernelGGL((prefix_merge_kernel<IO, DD>), dim3((unsigned)((m * (DD / 4) + 255) / 256)), dim3(256), 0, s, k)
  if (d == 512) {
    DSA_PFX(512);
  } else if (d == 256) {
    DSA_PFX(256);
  } else {
    DSA_PFX(128);
  }
#undef DSA_PFX
  return hipGetLastError();
}

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }
}  // namespace
}  // namespace dsa

using namespace dsa;

size_t prefix_attn_workspace_bytes(int batch, int rows, int n1, int d, int prefix, int max_rows, int max_kv, int kv_splits) {
  const Cut c = make_cut(batch, rows, n1, prefix, max_rows, max_kv, kv_splits);
  if (c.slots == 1) return 0;
  const size_t m = (size_t)rows * n1;
  return align256(m * c.slots * sizeof(float4)) + m * c.slots * d * sizeof(float);
}

hipError_t launch_prefix_attn(const PrefixArgs& a, hipStream_t s) {
  const Cut c = make_cut(a.batch, a.total_rows, a.n1, a.prefix, a.max_rows, a.max_kv, a.kv_splits);
  PfxK k{};
  k.q = (const uint16_t*)a.q;
  k.qr = (const uint16_t*)a.qr;
  k.k = (const uint16_t*)a.k;
  k.kr = (const uint16_t*)a.kr;
  k.table = a.table;
  k.row_start = a.row_start;
  k.act_q = a.act_q;
  k.act_k = a.act_k;
  k.max_blocks = a.max_blocks;
  k.page = a.page;
  k.blocks = (uint32_t)a.blocks;
  k.page_shift = 0;
  while ((1ll << k.page_shift) < a.page) ++k.page_shift;
  k.page_mul = (uint32_t)(((1ull << (31 + k.page_shift)) + a.page - 1) / a.page);
  k.batch = a.batch;
  k.rows = a.total_rows;
  k.n1 = a.n1;
  k.prefix = a.prefix;
  k.s2 = (int)((int64_t)a.max_blocks * a.page);
  k.guess_rows = a.max_rows > 0 ? a.max_rows : 1;
  k.mode = a.sparse_mode;
  k.scale = a.scale;
  k.out = (uint16_t*)a.out;
  k.sm_max = a.sm_max;
  k.sm_sum = a.sm_sum;
  k.part_s = (float4*)a.ws;
  k.part_o = c.slots > 1 ? (float*)((char*)a.ws + align256((size_t)a.total_rows * a.n1 * c.slots * sizeof(float4))) : nullptr;
  k.p_mt = c.p_mt;
  k.p_tiles = c.p_tiles;
  k.p_splits = c.p_splits;
  k.p_chunk = c.p_chunk;
  k.p_items = c.p_tiles * c.p_splits;
  k.o_mt = c.o_mt;
  k.o_tiles = c.o_tiles;
  k.o_splits = c.o_splits;
  k.o_chunk = c.o_chunk;
  k.o_base = c.o_base;
  k.slots = c.slots;
  return a.io == DSA_DTYPE_BF16 ? launch_io<IO_BF16>(k, a.d, s) : launch_io<IO_F16>(k, a.d, s);
}
