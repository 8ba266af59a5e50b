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
  static constexpr int ROW = D * 2 + 128;      // LDS bytes of a token's row
  static constexpr int NOPE = BN * ROW;
  static constexpr int ROPE = BN * DR * 2;
  static constexpr int GPW = 10;               // direct-to-LDS loads per wave and tile: 8 rows, rope, ids
};
// Start of token t's row: shifted so that the operand reads (8 tokens, one column) and the
// transposed reads (4 tokens, 32 bytes) land on distinct banks
template <int D> __device__ __forceinline__ int nope_off(int t) {
  return t * Tile<D>::ROW + 32 * (t & 3) + 16 * ((t >> 2) & 1);
}
__device__ __forceinline__ int rope_off(int t, int c) { return (t >> 3) * 1024 + (c * 8 + (t & 7)) * 16; }

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
  constexpr int KSH = C::KS / KSPL;          // their steps of S^T
  static_assert(C::KS % KSPL == 0, "contraction split");
  constexpr int ON = D / 32 / KSPL;          // their 32-column tiles of O
  constexpr bool QLDS = MT == 4;             // the rotary part of Q stays in LDS
  constexpr int QF = QLDS ? C::KSN : KSH;    // Q fragments in registers
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rb = wave % MT, kh = wave / MT;
  const int kg = lane >> 5;
  const int h = it.h0 + rb * 32 + (lane & 31);
  const bool valid = h < it.h_end;
  const int hc = valid ? h : it.h_end - 1;
  const int m_rows = a.rows * a.n1;

  // ---- Q^T fragments (B operand: this lane's head row, 8 values at 16 ks + 8 kg)
  uint4 qf[QF];
  {
    const uint16_t* qn = a.q + (int64_t)hc * D;
    const uint16_t* qr = a.qr + (int64_t)hc * DR;
    if constexpr (QLDS) {
#pragma unroll
      for (int j = 0; j < QF; ++j) qf[j] = ldg16(qn + j * 16 + kg * 8);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<uint4*>(L.qr + (rb * 32 + (lane & 31)) * (DR + 8) + j * 16 + kg * 8) = ldg16(qr + j * 16 + kg * 8);
    } else {
#pragma unroll
      for (int j = 0; j < QF; ++j) {
        const int ks = kh * KSH + j;
        qf[j] = ldg16((ks < C::KSN ? qn + ks * 16 : qr + (ks - C::KSN) * 16) + kg * 8);
      }
    }
  }
  // the softmax works on raw scores times a positive factor: a negative scale negates the query, a
  // zero one becomes 1e-30 (scores round to 0, masked ones stay -inf)
  const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
  const float cpos = a.scale > 0.f ? a.scale : a.scale < 0.f ? -a.scale : 1e-30f;
  const float cl2 = cpos * LOG2E;
#pragma unroll
  for (int j = 0; j < QF; ++j) {
    qf[j].x ^= flip;
    qf[j].y ^= flip;
    qf[j].z ^= flip;
    qf[j].w ^= flip;
  }

  // ---- this head row's tokens: a row that sees none of the item's is dead: it runs along unmasked
  // and leaves a sum of 0
  int lim = 0;
  if (valid) {
    const int row = h / a.n1;
    lim = row_limit(a, row, it.b >= 0 ? it.b : batch_of(a, row));
  }
  const bool dead = lim <= it.t_lo;
  int hi = dead ? 0 : min(lim, it.t_hi), lo = dead ? INT_MAX : hi;
  {
    int mx = hi, mn = lo;
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
    lim = lo;          // own limit within the item, INT_MAX for dead rows
    hi = 0;
    lo = INT_MAX;
#pragma unroll
    for (int w = 0; w < NWV; ++w) {
      hi = max(hi, L.red[0][w]);
      lo = min(lo, L.red[1][w]);
    }
  }
  hi = __builtin_amdgcn_readfirstlane(hi);          // end of the item's tokens
  const int min_lim = __builtin_amdgcn_readfirstlane(lo);
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
  // one, tiles past the end the last tile: every wave issues the same loads per tile.
  auto token = [&](int u, int j) { return min(it.t_lo + min(u, ntiles - 1) * BN + wave * 8 + j, hi - 1); };
  auto page_of = [&](int t) { return (int)(((uint64_t)(uint32_t)t * a.page_mul) >> (31 + a.page_shift)); };
  auto ids_dma = [&](int u) {
    const int t = token(u, lane & 7);
    const int32_t* src = a.table + (t < a.prefix || it.b < 0 ? 0 : (int64_t)it.b * a.max_blocks) + page_of(t);
    if (lane < 8) lds_dma4_untracked(src, &L.ids[u & 3][wave * 8]);
  };
  auto gather = [&](int u) {
    const int t = token(u, lane & 7);
    const int32_t id = L.ids[u & 3][wave * 8 + (lane & 7)];
    const int row = (uint32_t)id < a.blocks ? id * a.page + (t - page_of(t) * a.page) : -1;
    uint8_t* nope = L.nope[u % NBUF];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int r = __builtin_amdgcn_readlane(row, j);
      const uint16_t* src = r >= 0 ? a.k + (int64_t)r * D : reinterpret_cast<const uint16_t*>(g_zero_row);
      if (lane < D / 8) lds_dma16_sbase_untracked(src, lane * 16, nope + nope_off<D>(wave * 8 + j));
    }
    const uint16_t* src = row >= 0 ? a.kr + (int64_t)row * DR : reinterpret_cast<const uint16_t*>(g_zero_row);
    lds_dma16_untracked(src + (lane >> 3) * 8, L.rope[u % NBUF] + wave * 1024);
  };
  // A tile that some of the head rows see only in part: a masked token has P = 0, but 0 times a value
  // that is not finite would still reach the rows that do not see it. Such values become 0 in LDS, and
  // the token's score NaN for the rows that do see it. (Each wave its own rows, landed by now.)
  auto sanitize = [&](int u) {
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
  gather(0);
  gather(1);

  f32x16 o[ON];
#pragma unroll
  for (int n = 0; n < ON; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[n][i] = 0.f;
  float m_used = -INFINITY, m_true = -INFINITY, l_part = 0.f;

  // S^T rows are permuted so that a lane's 16 scores are tokens 16 (i / 8) + 8 kg + i % 8: the order of
  // the B operand of the PV product
  const int rr = lane & 31;
  const int tk = 16 * (rr >> 4) + 8 * ((rr >> 2) & 1) + 4 * ((rr >> 3) & 1) + (rr & 3);
  const int g16 = lane >> 4, c16 = lane & 15;
  const int vlane = nope_off<D>((g16 >> 1) * 8 + (c16 >> 2)) + ((g16 & 1) * 16 + 4 * (c16 & 3)) * 2 + kh * (D / KSPL) * 2;

  for (int t = 0; t < ntiles; ++t) {
    if (t == 0) wait_vmcnt<C::GPW - 1>();   // tile 0 here, tile 1 may be under way
    else wait_vmcnt<C::GPW>();
    const int t0 = it.t_lo + t * BN;
    uint8_t* nope = L.nope[t % NBUF];
    uint8_t* rope = L.rope[t % NBUF];
    const bool mixed = min_lim < hi && t0 + BN > min_lim;
    if (mixed) sanitize(t);
    lds_barrier();   // tile t resident, every wave done with tile t - 1
    gather(t + 2);
    ids_dma(t + 4);

    // ---- S^T
    f32x16 sv;
#pragma unroll
    for (int i = 0; i < 16; ++i) sv[i] = 0.f;
#pragma unroll
    for (int j = 0; j < KSH; ++j) {
      const int ks = kh * KSH + j;
      const uint4 kf = *reinterpret_cast<const uint4*>(ks < C::KSN ? nope + nope_off<D>(tk) + kg * 16 + ks * 32
                                                                   : rope + rope_off(tk, (ks - C::KSN) * 2 + kg));
      uint4 qv;
      if (QLDS && j >= C::KSN) {
        qv = *reinterpret_cast<const uint4*>(L.qr + (rb * 32 + rr) * (DR + 8) + (j - C::KSN) * 16 + kg * 8);
        qv.x ^= flip, qv.y ^= flip, qv.z ^= flip, qv.w ^= flip;
      } else {
        qv = qf[j < QF ? j : 0];
      }
      sv = Mfma<IO>::m32(kf, qv, sv);
    }
    if constexpr (KSPL > 1) {   // the waves of a block add their parts in one order: the same bits in each
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4*>(&L.x[wave][(g * 64 + lane) * 4]) =
            make_float4(sv[4 * g], sv[4 * g + 1], sv[4 * g + 2], sv[4 * g + 3]);
      lds_barrier();
#pragma unroll
      for (int i = 0; i < 16; ++i) sv[i] = 0.f;
#pragma unroll
      for (int w = 0; w < KSPL; ++w)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float4 p = *reinterpret_cast<const float4*>(&L.x[rb + MT * w][(g * 64 + lane) * 4]);
          sv[4 * g] += p.x;
          sv[4 * g + 1] += p.y;
          sv[4 * g + 2] += p.z;
          sv[4 * g + 3] += p.w;
        }
    }
    if (mixed) {
      const uint32_t bad = L.bad[t & 1][0] | L.bad[t & 1][1] | L.bad[t & 1][2] | L.bad[t & 1][3];
      if (bad)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if ((bad >> (16 * (i >> 3) + 8 * kg + (i & 7))) & 1u) sv[i] = __builtin_nanf("");
    }
    if (t0 + BN > min_lim) {
#pragma unroll
      for (int i = 0; i < 16; ++i) sv[i] = t0 + 16 * (i >> 3) + 8 * kg + (i & 7) < lim ? sv[i] : -INFINITY;
    }
    // ---- online softmax
    float mx = max3(sv[0], sv[1], sv[2]);
#pragma unroll
    for (int i = 3; i < 15; i += 2) mx = max3(mx, sv[i], sv[i + 1]);
    mx = max_half_swap(fmaxf(mx, sv[15])) * cpos;
    m_true = fmaxf(m_true, mx);
    const float m_new = mx > m_used + lazy_tau<IO>() || m_used == -INFINITY ? mx : m_used;
    const float alpha = m_used == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m_used - m_new) * LOG2E);
    m_used = m_new;
    const float mb = m_used * LOG2E;
    float p[16], sum = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[i], cl2, -mb));
      sum += p[i];
    }
    l_part = l_part * alpha + sum;
    if (__builtin_amdgcn_ballot_w64(alpha != 1.f)) {
#pragma unroll
      for (int n = 0; n < ON; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[n][i] *= alpha;
    }
    // ---- O^T += V^T P^T
#pragma unroll
    for (int kq = 0; kq < 2; ++kq) {
      const uint4 pb = make_uint4(pack2<IO>(p[8 * kq], p[8 * kq + 1]), pack2<IO>(p[8 * kq + 2], p[8 * kq + 3]),
                                  pack2<IO>(p[8 * kq + 4], p[8 * kq + 5]), pack2<IO>(p[8 * kq + 6], p[8 * kq + 7]));
#pragma unroll
      for (int n = 0; n < ON; ++n) {
        const uint8_t* v = nope + vlane + kq * 16 * C::ROW + n * 64;
        const uint2 lo2 = ds_read_tr(v), hi2 = ds_read_tr(v + 4 * C::ROW + 16);
        o[n] = Mfma<IO>::m32(make_uint4(lo2.x, lo2.y, hi2.x, hi2.y), pb, o[n]);
      }
    }
  }
  wait_vmcnt<0>();   // the ring's last gathers land before the LDS is released

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
  if (!valid) return;
  const int c0 = kh * (D / KSPL) + 4 * kg;
  if (!direct) {
    if (dead) return;
    float* dst = a.part_o + ((int64_t)it.slot * m_rows + h) * D + c0;
#pragma unroll
    for (int n = 0; n < ON; ++n)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4*>(dst + n * 32 + 8 * g) =
            make_float4(o[n][4 * g], o[n][4 * g + 1], o[n][4 * g + 2], o[n][4 * g + 3]);
  } else {
    const float inv = dead ? 0.f : 1.f / l_tot;
    uint16_t* dst = a.out + (int64_t)h * D + c0;
#pragma unroll
    for (int n = 0; n < ON; ++n)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = dead ? 0.f : o[n][4 * g + j] * inv;
        *reinterpret_cast<uint2*>(dst + n * 32 + 8 * g) = make_uint2(pack2<IO>(v[0], v[1]), pack2<IO>(v[2], v[3]));
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
