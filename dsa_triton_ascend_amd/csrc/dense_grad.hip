// Gradients of the dense attention of whole prompts, for gfx950.
//
// With P = e^(score - max) / sum, dP = dO . v, delta = dO . O (both per head row), dS = P (dP - delta):
//   dV = P^T dO,   dK = scale dS^T Q,   dQ = scale dS K,
// dK and dV summed over the queries and heads that read them. P is made again from the scores and the statistics:
// keeping it would cost more bytes than its product costs time.
//
// Three launches, without atomics, so results do not depend on timing:
//  * rows: delta and the logarithm of the sum for every head row (fp16: also the norms that bound dS);
//  * queries: 128 head rows, 32 a wave, Q and dO in registers, running over the tokens: S^T = K Q^T, dP^T = V dO^T,
//    dQ^T += K^T dS^T; on its way it makes delta anew, without the rounding of O, and sum P K, which corrects dQ for it;
//  * keys: a work-group has 128 tokens of one key head, 32 a wave, K and V in registers, and runs over the head rows
//    that see them (the group's heads are rows side by side): S = Q K^T and dP = dO V^T with the head rows as M, whose
//    results are already the B operands of dV^T += dO^T P and dK^T += Q^T dS.
// Few tokens or rows are cut into ranges over the other axis, whose sums a further launch adds.
//
// S and dP are computed in both, with sum P K 8 products instead of 5; what that saves is the addition of dQ from many
// work-groups, in 32 bits and an order of its own. P and dS are rounded to the io type for their products.
//
// Bound by the issue of instructions beside the matrix ones: a wave holds two operands and up to 10 accumulators, so there is
// one to a SIMD, and P and dS of one half tile are placed among the products of the half before it and the scores of
// the one after (8192 tokens, 32 heads on 8 of 128, bf16: 3079 -> 2189 us). Loads whose addresses need no branch: 1954;
// all work-groups of a key head at the same head rows at the same time, and dP that starts from -delta: 1836;
// levels turned (pair_of) and twice the work-groups for the rows: 1770; with sum P K: 1900 (rows 29, queries 920, keys 950;
// 1150 TFLOP/s of the 8 products). Two waves to 32 tokens, one for dV and one for dK, each with the scores of both, were no
// faster than one for both (1954).
#include <algorithm>

#include "dense_attn.hpp"

namespace dsa {
namespace {

constexpr int NWV = 4;
constexpr int BN = 64;     // rows of a tile in LDS
constexpr int NBUF = 3;
constexpr int TOK = NWV * 32;     // tokens, or head rows, of a work-group
constexpr int PREP = 1024;        // work-groups of the first launch

// fp16 keeps 11 bits down to 2^-14 and none below 2^-25. P <= 1 is multiplied by 2^15 for its product. dS is bounded by
// 2 max|dO| max|v| (row norms), and multiplied by the power of two that takes this bound to 2^15.
template <int IO> constexpr float p_shift() { return IO == IO_F16 ? 15.f : 0.f; }

struct GradK {
  Rows q, qr, k, kr, v, d, o;
  Lens len;
  int heads, key_heads, per;
  uint32_t per_mul;        // r / per for r < 2^31: see rows_of
  int per_shift;
  int linear;              // the heads of a group divide 16: see the loads of the keys' kernel
  int q_seqs, k_seqs;      // sequences, with what lies behind the last
  int q_even, k_even;      // tiles of the longest, 0: numbered through
  float scale;
  int64_t stat_head;
  int stat_padded, s1;     // s1: rows of a sequence of padded statistics
  const float* sm_max;
  const float* sm_sum;
  float* lse;              // [key heads][rows * per]: log2 of the sum of e^score, +inf for rows that see nothing
  float* delta;            // -delta
  float* norms;            // fp16: [2][PREP] largest |dO|^2 and |v|^2
  uint16_t* dq;
  uint16_t* dqr;
  uint16_t* dk;
  uint16_t* dkr;
  uint16_t* dv;
  int k_splits, k_chunk, k_blocks;   // ranges of head rows; blocks of 32 tokens, all key heads
  int q_splits, q_chunk, q_blocks;   // ranges of tokens; blocks of 32 head rows
  float4* k_part;
  float4* q_part;
  float* q_sum;            // [splits][blocks][32]: a range's sum of P dP
};

__device__ __forceinline__ int row_div(const GradK& a, int r) { return (int)(((uint64_t)(uint32_t)r * a.per_mul) >> (31 + a.per_shift)); }

// ---------------------------------------------------------------- rows
template <int IO, int D>
__global__ __launch_bounds__(256) void dense_prep_kernel(GradK a) {
  constexpr int LPR = D / 8;   // lanes a row
  const int lane = threadIdx.x & 63;
  const int slot = threadIdx.x / LPR, c = (threadIdx.x % LPR) * 8;
  auto values = [&](const uint16_t* p, float (&x)[8]) {
    const uint4 u = ldg16(p + c);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = to_f32<IO>((uint16_t)w[i]), x[2 * i + 1] = to_f32<IO>((uint16_t)(w[i] >> 16));
  };
  auto row_sum = [&](float x) {
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) x += __shfl_xor(x, o);
    return x;
  };
  constexpr int SLOTS = 256 / LPR;
  float most_d = 0.f, most_v = 0.f;
  const int64_t total = (int64_t)a.len.rows * a.heads;
  for (int64_t i = (int64_t)blockIdx.x * SLOTS + slot; i < total; i += (int64_t)gridDim.x * SLOTS) {
    const int64_t row = i / a.heads;
    const int h = (int)(i - row * a.heads);
    const int n = row_div(a, h), g = h - n * a.per;
    float d[8], o[8], s = 0.f, q = 0.f;
    int64_t b = 0, r = row;   // where it lies: row r of sequence b, or of all
    if (a.len.apart) b = row / a.s1, r = row - b * a.s1;
    values(a.d.p + b * a.d.batch + r * a.d.row + h * a.d.head, d);
    values(a.o.p + b * a.o.batch + r * a.o.row + h * a.o.head, o);
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(d[e], o[e], s), q = fmaf(d[e], d[e], q);
    const int64_t at = n * (int64_t)a.len.rows * a.per + row * a.per + g;
    int64_t st = at;
    if (a.stat_padded) {
      b = row / a.s1;
      st = ((b * a.key_heads + n) * a.s1 + (row - b * a.s1)) * a.per + g;
    }
    const float m = a.sm_max[st], l = a.sm_sum[st];
    s = row_sum(s);
    if constexpr (IO == IO_F16) {
      q = row_sum(q);
      // (rows that see nothing, padding among them, do not count; those that are not finite give NaN whatever the factor)
      if (l != 0.f && q < INFINITY) most_d = fmaxf(most_d, q);
    }
    if (c == 0) {
      a.lse[at] = l == 0.f ? INFINITY : m * LOG2E + log2f(l) - p_shift<IO>();
      a.delta[at] = -s;
    }
  }
  if constexpr (IO == IO_F16) {
    const int64_t keys = (int64_t)a.len.keys * a.key_heads;
    for (int64_t i = (int64_t)blockIdx.x * SLOTS + slot; i < keys; i += (int64_t)gridDim.x * SLOTS) {
      const int64_t row = i / a.key_heads;
      const int b = batch_of_row(a.len.key_start, a.len.batch, (int)row);
      if (row - a.len.key_start[b] >= a.len.act_k[b]) continue;   // padding
      float v[8], q = 0.f;
      const int k0 = a.len.key_start[b];
      values(first_of(a.len, a.v, b, k0) + (row - k0) * a.v.row + (i - row * a.key_heads) * a.v.head, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) q = fmaf(v[e], v[e], q);
      q = row_sum(q);
      if (q < INFINITY) most_v = fmaxf(most_v, q);
    }
    __shared__ float red[2][4];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      most_d = fmaxf(most_d, __shfl_xor(most_d, o));
      most_v = fmaxf(most_v, __shfl_xor(most_v, o));
    }
    if (lane == 0) red[0][threadIdx.x >> 6] = most_d, red[1][threadIdx.x >> 6] = most_v;
    __syncthreads();
    if (threadIdx.x < 2) {
      const float* r = red[threadIdx.x];
      a.norms[threadIdx.x * PREP + blockIdx.x] = fmaxf(fmaxf(r[0], r[1]), fmaxf(r[2], r[3]));
    }
  }
}

// The factor of dS (a power of two) and the one that undoes it, by the whole work-group
template <int IO, int NWV>
__device__ __forceinline__ float2 ds_factor(const GradK& a, float (*red)[NWV]) {
  if constexpr (IO != IO_F16) return make_float2(1.f, 1.f);
  float m[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    m[w] = 0.f;
#pragma unroll
    for (int i = 0; i < PREP; i += NWV * 64) m[w] = fmaxf(m[w], a.norms[w * PREP + i + threadIdx.x]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m[w] = fmaxf(m[w], __shfl_xor(m[w], o));
    if ((threadIdx.x & 63) == 0) red[w][threadIdx.x >> 6] = m[w];
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    m[w] = red[w][0];
#pragma unroll
    for (int i = 1; i < NWV; ++i) m[w] = fmaxf(m[w], red[w][i]);
  }
  // 2 |dO| |v| 2^e <= 2^15: 2^e = 2^floor(14 - log2(|dO| |v|)); no more than fp32's exponents hold
  const float e = floorf(14.f - 0.5f * (log2f(fmaxf(m[0], 1e-30f)) + log2f(fmaxf(m[1], 1e-30f))));
  const float f = exp2f(fminf(fmaxf(e, -100.f), 100.f));
  return make_float2(f, 1.f / f);
}

// ---------------------------------------------------------------- which tile
// i: the work-group; count(q) rows (or tokens) of a sequence, per of them a position of starts[]. Returns the sequence,
// the tile's number from the sequence's first and the key head; tile < 0: none.
struct Place {
  int b, n, tile, sp;
};
template <typename F>
__device__ __forceinline__ Place place_of(int i, int seqs, int heads, int splits, int even, const int32_t* starts, int per, F&& tiles_of) {
  Place p;
  if (even) {
    const int pairs = seqs * heads, level = i / pairs;
    i = pair_of(i, level, pairs, splits);
    p.b = i / heads;
    p.n = i - p.b * heads;
    p.sp = level % splits;
    p.tile = level / splits;
    if (p.tile >= tiles_of(p.b)) p.tile = -1;
    return p;
  }
  p.sp = i % splits;
  i /= splits;
  p.n = i % heads;
  i /= heads;
  int lo = 0, hi = seqs - 1;
  auto first = [&](int s) { return (int)((int64_t)starts[s] * per / TOK) + s; };
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first(mid) <= i) lo = mid; else hi = mid - 1;
  }
  p.b = lo;
  p.tile = i - first(lo);
  if (p.tile >= tiles_of(lo)) p.tile = -1;
  return p;
}

// ---------------------------------------------------------------- keys
template <int D, int DR> struct KeyLds {
  struct {
    uint8_t q[BN * D * 2];   // (d lies at a constant offset from q)
    uint8_t d[BN * D * 2];
  } t[NBUF];
  uint8_t qr[NBUF][DR ? BN * DR * 2 : 16];
  float lse[NBUF][BN];
  float delta[NBUF][BN];
  uint64_t bad[NBUF][NWV];
  float red[2][NWV];
};

__device__ __forceinline__ void lds_dma4(const void* gptr, void* lds_base) {
  const uint32_t m0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)lds_base;
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" : : "v"(gptr), "s"(m0) : "memory", "m0");
}

template <int IO, int D, int DR, bool LINEAR>
__global__ __launch_bounds__(NWV * 64) void dense_keys_kernel(GradK a) {
  constexpr int KSN = D / 16, KS = (D + DR) / 16, ON = D / 32, RN = DR / 32, RB = D * 2;
  __shared__ __attribute__((aligned(16))) KeyLds<D, DR> L;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = lane >> 5, rr = lane & 31;
  const Place at = place_of(blockIdx.x, a.k_seqs, a.key_heads, a.k_splits, a.k_even, a.len.key_start, 1, [&](int b) {
    const Seq q = seq_of(a.len, b);
    return (q.keys + TOK - 1) / TOK;
  });
  if (at.tile < 0) return;
  const int b = at.b, n = at.n;
  const Seq seq = seq_of(a.len, b);
  const float2 factor = ds_factor<IO, NWV>(a, L.red);

  const int t0 = at.tile * TOK, t_end = min(seq.keys, t0 + TOK), t_seen = min(t_end, seq.ak);
  const int t = t0 + wave * 32 + rr;
  // head rows [r_lo, r_hi) see some of these tokens, from r_full on all of them; this range's share
  const int r_end = seq.aq * a.per;
  const int r_lo = __builtin_amdgcn_readfirstlane(max(first_query(a.len, seq, t0) * a.per, at.sp * a.k_chunk));
  const int r_hi = __builtin_amdgcn_readfirstlane(at.sp == a.k_splits - 1 ? r_end : min(r_end, (at.sp + 1) * a.k_chunk));
  const int r_full = t_seen > t0 ? first_query(a.len, seq, t_seen - 1) * a.per : 0;
  const int my_first = t < t_seen ? first_query(a.len, seq, t) * a.per : INT_MAX;
  const int ntiles = t_seen > t0 && r_hi > r_lo ? (r_hi - r_lo + BN - 1) / BN : 0;

  f32x16 dk[ON + RN], dv[ON];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
#pragma unroll
    for (int c = 0; c < ON + RN; ++c) dk[c][i] = 0.f;
#pragma unroll
    for (int c = 0; c < ON; ++c) dv[c][i] = 0.f;
  }

  if (ntiles > 0) {
    const float sl2 = a.scale * LOG2E;
    // ---- tiles of head rows: each wave loads a share, in GPW loads (past the last tile it again, into buffers that nobody
    // reads: no load then depends on a branch). Tile u has the rows from first_row(u) on: the last rows first, which
    // all work-groups of a key head see, so that they read the same ones at the same time (from the first on, each began at
    // rows of its own, and 63% of the loads missed the L2). Rows past the last repeat it (they are masked); only tile 0
    // has any. LINEAR: the group's heads divide 16, so that a lane's rows of all tiles are of one head and evenly spaced.
    auto first_row = [&](int u) { return r_lo + (ntiles - 1 - u) * BN; };
    using Sh = Share<RB, BN, NWV>;
    using ShR = Share<DR ? DR * 2 : 128, BN, NWV>;
    const Sh sh(wave, lane);
    const ShR shr(wave, lane);
    constexpr int CQ = Sh::CNT, CR = DR ? ShR::CNT : 0, GPW = 2 * CQ + CR + 1;
    auto place = [&](const Rows& x, int r) {   // of head row r, in bytes
      const int s = row_div(a, r);
      return ((int64_t)s * x.row + (int64_t)(r - s * a.per) * x.head) * 2;
    };
    auto base_of = [&](const Rows& x) {
      return reinterpret_cast<const char*>(first_of(a.len, x, b, seq.r0) + (int64_t)n * a.per * x.head);
    };
    const char* const qb = base_of(a.q);
    const char* const db = base_of(a.d);
    const char* const qrb = DR ? base_of(a.qr) : nullptr;
    const int64_t stat0 = n * (int64_t)a.len.rows * a.per + (int64_t)seq.r0 * a.per;
    const float* const stat = ((wave & 1) ? a.delta : a.lse) + stat0;   // (two waves each, the same values)
    const uint32_t q_lds = lds_addr(L.t[0].q) + wave * 1024, r_lds = lds_addr(L.qr[0]) + wave * 1024;
    const uint32_t s_lds = lds_addr((wave & 1) ? L.delta[0] : L.lse[0]);
    // (linear) of the tile that is loaded next: bases, and this lane's offsets from them
    const int64_t q_step = (int64_t)(BN >> a.per_shift) * a.q.row * 2, d_step = (int64_t)(BN >> a.per_shift) * a.d.row * 2,
                  r_step = DR ? (int64_t)(BN >> a.per_shift) * a.qr.row * 2 : 0;
    const char* qn = qb + (int64_t)(first_row(0) >> a.per_shift) * a.q.row * 2;
    const char* dn = db + (int64_t)(first_row(0) >> a.per_shift) * a.d.row * 2;
    const char* rn = DR ? qrb + (int64_t)(first_row(0) >> a.per_shift) * a.qr.row * 2 : nullptr;
    uint32_t q_off[CQ], d_off[CQ], r_off[CR ? CR : 1];
    int load_row = first_row(0);
    auto aim = [&]() __attribute__((always_inline)) {
      if constexpr (LINEAR) {
        const int last = r_hi - 1 - load_row;
#pragma unroll
        for (int i = 0; i < CQ; ++i) {
          const int r = min(i * Sh::STEP + sh.row, last);
          q_off[i] = (uint32_t)place(a.q, r) + sh.col;
          d_off[i] = (uint32_t)place(a.d, r) + sh.col;
        }
        if constexpr (DR > 0)
#pragma unroll
          for (int i = 0; i < CR; ++i) r_off[i] = (uint32_t)place(a.qr, min(i * ShR::STEP + shr.row, last)) + shr.col;
      }
    };
    auto load_part = [&](auto jc, int buf) __attribute__((always_inline)) {
      constexpr int j = decltype(jc)::value;
      constexpr int what = j == GPW - 1 ? 3 : j < CQ ? 0 : j < 2 * CQ ? 1 : 2, i = what == 0 ? j : what == 1 ? j - CQ : what == 2 ? j - 2 * CQ : 0;
      if constexpr (what == 3) {
        lds_dma4(stat + min(load_row + lane, r_hi - 1), (void*)(__attribute__((address_space(3))) void*)(uintptr_t)(s_lds + buf * (BN * 4)));
      } else {
        const uint32_t dst = what == 2 ? r_lds + buf * (BN * 128) : q_lds + buf * (2 * BN * RB);
        constexpr int at = (what == 1 ? BN * RB : 0) + i * NWV * 1024;
        if constexpr (LINEAR) {
          lds_dma16_at<at>(what == 0 ? qn : what == 1 ? dn : rn, what == 0 ? q_off[what == 0 ? i : 0] : what == 1 ? d_off[what == 1 ? i : 0] : r_off[what == 2 ? i : 0], dst);
        } else {
          const int r = min(load_row + i * (what == 2 ? ShR::STEP : Sh::STEP) + (what == 2 ? shr.row : sh.row), r_hi - 1);
          lds_dma16_untracked((what == 0 ? qb : what == 1 ? db : qrb) + place(what == 0 ? a.q : what == 1 ? a.d : a.qr, r) + (what == 2 ? shr.col : sh.col),
                              (void*)(__attribute__((address_space(3))) void*)(uintptr_t)(dst + at));
        }
      }
    };
    auto load_tile = [&](int buf) __attribute__((always_inline)) {
      static_for<0, GPW>([&](auto j) __attribute__((always_inline)) { load_part(j, buf); });
    };
    // from tile u - 1 to tile u
    auto advance = [&](int u) __attribute__((always_inline)) {
      if (u >= ntiles) return;
      load_row -= BN;
      if constexpr (LINEAR) {
        qn = uniform(qn - q_step);
        dn = uniform(dn - d_step);
        if constexpr (DR > 0) rn = uniform(rn - r_step);
      }
      if (u == 1) aim();   // (whole from here on)
    };
    // (a masked pair has P = dS = 0, but 0 times a value that is not finite would reach tokens that the row does not see)
    auto is_mixed = [&](int u) { return first_row(u) < r_full || first_row(u) + BN > r_hi; };
    auto sanitize = [&](int u, int buf) __attribute__((always_inline)) {
      if (!is_mixed(u)) return;
      uint64_t bad = clean_share<IO, RB, BN, NWV>(lds_addr(L.t[buf].q), wave, lane) |
                     clean_share<IO, RB, BN, NWV>(lds_addr(L.t[buf].d), wave, lane);
      if constexpr (DR > 0) bad |= clean_share<IO, 128, BN, NWV>(lds_addr(L.qr[buf]), wave, lane);
      if (lane == 0) L.bad[buf][wave] = bad;
    };
    aim();
    load_tile(0);
    uint4 kf[KS], vf[KSN];
    {
      const int64_t tt = min(t, t_seen - 1);
      const uint16_t* kp = first_of(a.len, a.k, b, seq.k0) + tt * a.k.row + n * a.k.head + kg * 8;
      const uint16_t* vp = first_of(a.len, a.v, b, seq.k0) + tt * a.v.row + n * a.v.head + kg * 8;
#pragma unroll
      for (int j = 0; j < KSN; ++j) kf[j] = ldg16(kp + j * 16), vf[j] = ldg16(vp + j * 16);
      if constexpr (DR > 0) {
        const uint16_t* rp = first_of(a.len, a.kr, b, seq.k0) + tt * a.kr.row + n * a.kr.head + kg * 8;
#pragma unroll
        for (int j = KSN; j < KS; ++j) kf[j] = ldg16(rp + (j - KSN) * 16);
      }
#pragma unroll
      for (int j = 0; j < KS; ++j) kf[j] = in_agprs(kf[j]);
#pragma unroll
      for (int j = 0; j < KSN; ++j) vf[j] = in_agprs(vf[j]);
    }

    // ---- operands
    constexpr int DOFF = BN * D * 2;   // from a place in q to the same in d
    const int qk = s_row(rr), g16 = lane >> 4, c16 = lane & 15;
    const int r4 = (g16 >> 1) * 8 + (c16 >> 2), vc = (g16 & 1) * 2 + ((c16 & 3) >> 1), o8 = (c16 & 1) * 8;
    const uint32_t op_lane = tile_off<RB>(qk, kg), opr_lane = tile_off<128>(qk, kg);
    const uint32_t tr_lo = tile_off<RB>(r4, vc) + o8, tr_hi = tile_off<RB>(r4 + 4, vc) + o8;
    const uint32_t trr_lo = tile_off<128>(r4, vc) + o8, trr_hi = tile_off<128>(r4 + 4, vc) + o8;
    OpAddr<RB> op;
    OpAddr<128> opr;
    TrAddr<RB> tr;
    TrAddr<128> trr;
    auto point_op = [&](int buf) __attribute__((always_inline)) {
      op.point(lds_addr(L.t[buf].q), op_lane);
      if constexpr (DR > 0) opr.point(lds_addr(L.qr[buf]), opr_lane);
    };
    auto point_tr = [&](int buf) __attribute__((always_inline)) {
      tr.point(lds_addr(L.t[buf].q), tr_lo, tr_hi);
      if constexpr (DR > 0) trr.point(lds_addr(L.qr[buf]), trr_lo, trr_hi);
    };
    auto q_frag = [&](int j, int h) __attribute__((always_inline)) -> uint4 {
      return lds_read16_at(j < KSN ? op.a[j < KSN ? j : 0] + h * 32 * RB : opr.a[j >= KSN ? j - KSN : 0] + h * 32 * 128);
    };
    auto d_frag = [&](int j, int h) __attribute__((always_inline)) -> uint4 { return lds_read16_at(op.a[j] + h * 32 * RB + DOFF); };
    // product i of a half's NP: column tiles of dV, dK and dK's rotary part for 16 rows, then for the next 16
    constexpr int NC = 2 * ON + RN, NP = 2 * NC;
    auto t_frag = [&](int i, int h) __attribute__((always_inline)) -> uint4 {
      const int st = i / NC, c = i % NC;
      if (c < ON) return tr.frag(c < ON ? c : 0, (h * 32 + st * 16) * RB + DOFF);
      if (c < 2 * ON) return tr.frag(c >= ON && c < 2 * ON ? c - ON : 0, (h * 32 + st * 16) * RB);
      return trr.frag(c >= 2 * ON ? c - 2 * ON : 0, (h * 32 + st * 16) * 128);
    };

    // ---- P and dS of 32 rows in NST stages of two rows each, placed among the products before and after them
    constexpr int NST = 8;
    struct Four {
      float4 v[4];   // rows 16 x + 8 kg + 4 y + 0 .. 3 at [2 x + y]
    };
    auto four = [&](const float* p, int e) __attribute__((always_inline)) {
      return *reinterpret_cast<const float4*>(p + 16 * (e >> 1) + 8 * kg + 4 * (e & 1));
    };
    // dP starts from -delta
    auto start = [&](f32x16& d, const float* p, int e) __attribute__((always_inline)) {
      const float4 v = four(p, e);
      d[4 * e] = v.x, d[4 * e + 1] = v.y, d[4 * e + 2] = v.z, d[4 * e + 3] = v.w;
    };
    const float f16 = factor.x * 0x1p-15f;   // (fp16's P has the factor 2^15)
    auto stage = [&](int st, f32x16& sv, f32x16& dp, Four& lse, uint32_t (&pw)[8], uint32_t (&sw)[8]) __attribute__((always_inline)) {
      const int i = 2 * st;
      const float4 l4 = lse.v[i >> 2];
      const float l0 = i & 2 ? l4.z : l4.x, l1 = i & 2 ? l4.w : l4.y;
      const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[i], sl2, -l0));
      const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[i + 1], sl2, -l1));
      float w0 = p0 * dp[i], w1 = p1 * dp[i + 1];
      if constexpr (IO == IO_F16) w0 *= f16, w1 *= f16;
      pw[st] = pack2<IO>(p0, p1);
      sw[st] = pack2<IO>(w0, w1);
      asm volatile("" : "+v"(pw[st]), "+v"(sw[st]));   // here, not where the next step needs them
    };
    auto mask = [&](int u, int buf, int h, uint32_t (&pw)[8], uint32_t (&sw)[8]) __attribute__((always_inline)) {
      if (!is_mixed(u)) return;
      const uint64_t all = L.bad[buf][0] | L.bad[buf][1] | L.bad[buf][2] | L.bad[buf][3];
      const uint32_t bad = (uint32_t)(all >> (h * 32));
      const int r0 = first_row(u) + h * 32, first = my_first - r0, last = r_hi - r0;   // rows [first, last) see the token
      int k = kg;
      asm volatile("" : "+v"(k));   // (what follows from it is not kept in registers for these few tiles)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int x = s_token(2 * i, k);
        const uint32_t nan = ((bad >> x) & 1u ? 0x7FFFu : 0u) | ((bad >> (x + 1)) & 1u ? 0x7FFF0000u : 0u);
        const uint32_t keep = (x >= first && x < last ? 0xFFFFu : 0u) | (x + 1 >= first && x + 1 < last ? 0xFFFF0000u : 0u);
        pw[i] = (pw[i] | nan) & keep;
        sw[i] = (sw[i] | nan) & keep;
      }
    };

    // ---- One step handles 32 rows: the products of the rows before them, S and dP of the rows after them, each MFMA
    // followed by a part of this one's P and dS. Fragments are read a few MFMAs ahead.
    constexpr int LAG = KS - KSN, NS = KS + KSN;   // S and dP end together
    constexpr int TR = 4, QR = 4, DRING = 4;
    uint4 tf[TR], qf[QR], df[DRING];
    // (nbuf: the buffer of the rows whose S and dP are made here)
    auto step = [&](auto pvc, auto sc, auto hc, int nbuf, f32x16& cs, f32x16& cd, Four& cl, f32x16& ns, f32x16& nd, Four& nl,
                    uint32_t (&pb)[8], uint32_t (&sb)[8], uint32_t (&pn)[8], uint32_t (&sn)[8], auto&& between, auto&& ride) __attribute__((always_inline)) {
      constexpr bool PV = decltype(pvc)::value, S = decltype(sc)::value;
      constexpr int H = decltype(hc)::value;
      constexpr int M0 = PV ? NP : 0, NMM = M0 + (S ? NS : 0), LEAD = NMM > 8 ? 2 : 0;
      auto values_at = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
        for (int st = 0; st < NST; ++st)
          if (LEAD + st * (NMM - LEAD) / NST == slot) stage(st, cs, cd, cl, pn, sn);
      };
      if constexpr (PV)
        static_for<0, NP>([&](auto ic) __attribute__((always_inline)) {
          constexpr int i = decltype(ic)::value, st = i / NC, c = i % NC;
          const uint4 b = c < ON ? make_uint4(pb[4 * st], pb[4 * st + 1], pb[4 * st + 2], pb[4 * st + 3])
                                 : make_uint4(sb[4 * st], sb[4 * st + 1], sb[4 * st + 2], sb[4 * st + 3]);
          if constexpr (c < ON) dv[c] = Mfma<IO>::m32(tf[i % TR], b, dv[c]);
          else dk[c - ON] = Mfma<IO>::m32(tf[i % TR], b, dk[c - ON]);
          if constexpr (i + TR < NP) tf[i % TR] = t_frag(i + TR, H);
          if constexpr (S)   // meanwhile, what the next ones begin with
            static_for<0, 4 + QR + DRING>([&](auto gc) __attribute__((always_inline)) {
              constexpr int g = decltype(gc)::value;
              if constexpr (g * NP / (4 + QR + DRING) == i) {
                if constexpr (g < 4) start(nd, &L.delta[nbuf][H * 32], g);
                else if constexpr (g < 4 + QR) qf[g - 4] = q_frag(g - 4, H);
                else df[g - 4 - QR] = d_frag(g - 4 - QR, H);
              }
            });
          values_at(i);
          __builtin_amdgcn_sched_barrier(0);
        });
      between();
      if constexpr (S)
        static_for<0, NS>([&](auto jc) __attribute__((always_inline)) {
          constexpr int j = decltype(jc)::value;
          constexpr bool is_s = j < LAG || (j - LAG) % 2 == 0;
          constexpr int i = j < LAG ? j : is_s ? LAG + (j - LAG) / 2 : (j - LAG) / 2;   // step of its chain
          if constexpr (j == NS - 1) mfma32_va_end2<IO>(ns, qf[(KS - 1) % QR], kf[KS - 1], nd, df[(KSN - 1) % DRING], vf[KSN - 1]);
          else if constexpr (is_s && i < KS - 1) {
            mfma32_va<IO, i == 0>(ns, qf[i % QR], kf[i]);
            if constexpr (i + QR < KS) qf[i % QR] = q_frag(i + QR, H);
          } else if constexpr (!is_s) {
            mfma32_va<IO, false>(nd, df[i % DRING], vf[i]);
            if constexpr (i + DRING < KSN) df[i % DRING] = d_frag(i + DRING, H);
          }
          if constexpr (j >= NS - TR) tf[j - (NS - TR)] = t_frag(j - (NS - TR), 1 - H);
          else if constexpr (j >= NS - TR - 4) nl.v[j - (NS - TR - 4)] = four(&L.lse[nbuf][H * 32], j - (NS - TR - 4));
          ride(jc);
          values_at(M0 + j);
          __builtin_amdgcn_sched_barrier(0);
        });
    };
    std::true_type yes;
    std::false_type no;
    std::integral_constant<int, 0> h0;
    std::integral_constant<int, 1> h1;
    auto nothing = [](auto...) __attribute__((always_inline)) {};

    wait_vmcnt<0>();
    asm volatile("" ::: "memory");
    sanitize(0, 0);
    lds_barrier();
    advance(1);
    load_tile(1);
    f32x16 s0, s1, d0, d1;
    Four l0, l1;
    uint32_t p0[8], p1[8], w0[8], w1[8];
    point_op(0);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      start(d0, L.delta[0], e);
      start(d1, &L.delta[0][32], e);
      l0.v[e] = four(L.lse[0], e);
    }
#pragma unroll
    for (int j = 0; j < KS - 1; ++j) {
      const uint4 f = q_frag(j, 0);
      if (j == 0) mfma32_va<IO, true>(s0, f, kf[j]);
      else mfma32_va<IO, false>(s0, f, kf[j]);
    }
#pragma unroll
    for (int j = 0; j < KSN - 1; ++j) mfma32_va<IO, false>(d0, d_frag(j, 0), vf[j]);
    mfma32_va_end2<IO>(s0, q_frag(KS - 1, 0), kf[KS - 1], d0, d_frag(KSN - 1, 0), vf[KSN - 1]);
#pragma unroll
    for (int j = 0; j < QR; ++j) qf[j] = q_frag(j, 1);
#pragma unroll
    for (int j = 0; j < DRING; ++j) df[j] = d_frag(j, 1);
    int buf = 0;   // of tile u
    // Step (u, 0): tile u + 1 has landed by the middle of it, when nobody needs tile u - 1 any more
    auto half0 = [&](auto pvc, int u) __attribute__((always_inline)) {
      const int nb = buf == NBUF - 1 ? 0 : buf + 1, lb = buf == 0 ? NBUF - 1 : buf - 1;   // of tiles u + 1 and u - 1 (u + 2)
      advance(u + 2);
      step(pvc, yes, h1, buf, s0, d0, l0, s1, d1, l1, p1, w1, p0, w0,
           [&]() __attribute__((always_inline)) {
             wait_vmcnt<0>();
             asm volatile("" ::: "memory");
             if (u + 1 < ntiles) sanitize(u + 1, nb);
             lds_barrier();
             point_tr(buf);
           },
           [&](auto jc) __attribute__((always_inline)) {
             constexpr int j = decltype(jc)::value;
             static_for<0, GPW>([&](auto g) __attribute__((always_inline)) {
               if constexpr (g * NS / GPW == j) load_part(g, lb);
             });
           });
      mask(u, buf, 0, p0, w0);
    };
    half0(no, 0);
    if (ntiles > 1) {
      int u = 0;
      do {
        u = __builtin_amdgcn_readfirstlane(u);
        const int nb = buf == NBUF - 1 ? 0 : buf + 1;
        point_op(nb);
        step(yes, yes, h0, nb, s1, d1, l1, s0, d0, l0, p0, w0, p1, w1, nothing, nothing);
        mask(u, buf, 1, p1, w1);
        buf = nb;
        half0(yes, u + 1);
      } while (++u + 1 < ntiles);
    }
    step(yes, no, h0, 0, s1, d1, l1, s0, d0, l0, p0, w0, p1, w1, nothing, nothing);
    mask(ntiles - 1, buf, 1, p1, w1);
#pragma unroll
    for (int i = 0; i < TR; ++i) tf[i] = t_frag(i, 1);
    static_for<0, NP>([&](auto ic) __attribute__((always_inline)) {
      constexpr int i = decltype(ic)::value, st = i / NC, c = i % NC;
      const uint4 b = c < ON ? make_uint4(p1[4 * st], p1[4 * st + 1], p1[4 * st + 2], p1[4 * st + 3])
                             : make_uint4(w1[4 * st], w1[4 * st + 1], w1[4 * st + 2], w1[4 * st + 3]);
      if constexpr (c < ON) dv[c] = Mfma<IO>::m32(tf[i % TR], b, dv[c]);
      else dk[c - ON] = Mfma<IO>::m32(tf[i % TR], b, dk[c - ON]);
      if constexpr (i + TR < NP) tf[i % TR] = t_frag(i + TR, 1);
    });
    wait_vmcnt<0>();   // the last (unused) loads land before the LDS is released
  }

  // lane l: token t, columns c * 32 + 8 g + 4 kg + j
  const float fk = a.scale * factor.y, fv = IO == IO_F16 ? 0x1p-15f : 1.f;
  if (a.k_splits > 1) {
    const int blk = n * (a.k_blocks / a.key_heads) + seq.k0 / 32 + b + at.tile * NWV + wave;
    if (t0 + wave * 32 >= seq.keys) return;
    float4* dst = a.k_part + ((int64_t)at.sp * a.k_blocks + blk) * ((2 * D + DR) / 8) * 64 + lane;
#pragma unroll
    for (int c = 0; c < ON + RN + ON; ++c) {
      const f32x16& v = c < ON + RN ? dk[c < ON + RN ? c : 0] : dv[c >= ON + RN ? c - ON - RN : 0];
      const float f = c < ON + RN ? fk : fv;
#pragma unroll
      for (int g = 0; g < 4; ++g)
        dst[(c * 4 + g) * 64] = make_float4(v[4 * g] * f, v[4 * g + 1] * f, v[4 * g + 2] * f, v[4 * g + 3] * f);
    }
    return;
  }
  const bool live = t < t_seen, valid = t < t_end;
  const int64_t tt = (int64_t)(seq.k0 + t) * a.key_heads + n;
  auto store = [&](const f32x16& v, float f, uint16_t* dst) __attribute__((always_inline)) {
    uint4 w[2];
    pack_tile<IO>(v, f, w);
    if (valid) {
      stg16(dst + 8 * kg, live ? w[0] : make_uint4(0, 0, 0, 0));
      stg16(dst + 8 * kg + 16, live ? w[1] : make_uint4(0, 0, 0, 0));
    }
  };
#pragma unroll
  for (int c = 0; c < ON; ++c) store(dk[c], fk, a.dk + tt * D + c * 32);
#pragma unroll
  for (int c = 0; c < RN; ++c) store(dk[ON + c], fk, a.dkr + tt * DR + c * 32);
#pragma unroll
  for (int c = 0; c < ON; ++c) store(dv[c], fv, a.dv + tt * D + c * 32);
}

// ---------------------------------------------------------------- queries
template <int D, int DR> struct QueryLds {
  struct {
    uint8_t k[BN * D * 2];   // (v lies at a constant offset from k)
    uint8_t v[BN * D * 2];
  } t[NBUF];
  uint8_t kr[NBUF][DR ? BN * DR * 2 : 16];
  uint64_t bad[NBUF][NWV];
  float red[2][NWV];
};

// delta = dO . O takes the rounded output, off by half a step of it on every token of the row alike: that adds up along what
// the keys have in common, and where dP and delta cancel it is all there is (keys and values with a common part as large as
// the rest, bf16, 4100 tokens: dQ's error 38 times that of rounding the exact dS). The sum of P dP over the row's tokens is
// the same number without that error, known at the end: sum P K comes along, and dQ gets its share of the difference. It
// needs no fragment of its own, but a third product, D / 32 accumulators and a rounding of P.
template <int IO, int D, int DR>
__global__ __launch_bounds__(NWV * 64) void dense_queries_kernel(GradK a) {
  constexpr int KSN = D / 16, KS = (D + DR) / 16, ON = D / 32, RN = DR / 32, RB = D * 2;
  __shared__ __attribute__((aligned(16))) QueryLds<D, DR> L;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = lane >> 5, rr = lane & 31;
  Place at = place_of(blockIdx.x, a.q_seqs, a.key_heads, a.q_splits, a.q_even, a.len.row_start, a.per, [&](int b) {
    const Seq q = seq_of(a.len, b);
    return (q.rows * a.per + TOK - 1) / TOK;
  });
  if (at.tile < 0) return;
  const int b = at.b, n = at.n;
  const Seq seq = seq_of(a.len, b);
  at.tile = (seq.rows * a.per + TOK - 1) / TOK - 1 - at.tile;   // the last, which see most, first
  const float2 factor = ds_factor<IO, NWV>(a, L.red);

  const int r_base = at.tile * TOK, r_end = min(seq.rows * a.per, r_base + TOK);
  const int t_lo = at.sp * a.q_chunk, t_hi = at.sp == a.q_splits - 1 ? INT_MAX : t_lo + a.q_chunk;
  auto seen = [&](int x, int y) {
    return x >= y || x / a.per >= seq.aq ? 0 : min(limit_of(a.len, seq, min((y - 1) / a.per, seq.aq - 1)), t_hi);
  };
  const int hi = seen(r_base, r_end);
  const int min_lim = max(t_lo + 1, limit_of(a.len, seq, r_base / a.per));
  const int ntiles = hi > t_lo ? (hi - t_lo + BN - 1) / BN : 0;
  const int w_base = r_base + wave * 32;
  const int row = w_base + rr;
  const bool valid = row < r_end;
  const int r = valid ? row : r_end - 1, s = r / a.per, g = r - s * a.per;
  const int lim = valid ? min(limit_of(a.len, seq, s), t_hi) : 0;
  const bool dead = lim <= t_lo;

  f32x16 dq[ON + RN], pk[ON + RN];
#pragma unroll
  for (int c = 0; c < ON + RN; ++c)
#pragma unroll
    for (int i = 0; i < 16; ++i) dq[c][i] = pk[c][i] = 0.f;
  float sum = 0.f;   // of P dP

  if (ntiles > 0) {
    // (a zero scale becomes 1e-30: scores round to 0, and a masked one, of the sign that makes it so, to P = 0)
    const float sl2 = (a.scale == 0.f ? 1e-30f : a.scale) * LOG2E;
    const float masked = sl2 > 0.f ? -INFINITY : INFINITY;
    // (as in the forward: past the last tile it again)
    Stream<RB, BN, NWV> ks(first_of(a.len, a.k, b, seq.k0) + t_lo * a.k.row + n * a.k.head, (uint32_t)a.k.row * 2, L.t[0].k, wave, lane);
    Stream<RB, BN, NWV> vs(first_of(a.len, a.v, b, seq.k0) + t_lo * a.v.row + n * a.v.head, (uint32_t)a.v.row * 2, L.t[0].v, wave, lane);
    Stream<128, BN, NWV> rs(DR ? first_of(a.len, a.kr, b, seq.k0) + t_lo * a.kr.row + n * a.kr.head : nullptr, (uint32_t)a.kr.row * 2, L.kr[0], wave, lane);
    constexpr int CK = ks.sh.CNT, CR = DR ? rs.sh.CNT : 0, GPW = 2 * CK + CR;
    auto load_part = [&](auto jc, int buf) __attribute__((always_inline)) {
      constexpr int j = decltype(jc)::value;
      if constexpr (j < CK) ks.template load<j>(buf * (2 * BN * RB));
      else if constexpr (j < 2 * CK) vs.template load<j - CK>(buf * (2 * BN * RB));
      else rs.template load<j - 2 * CK>(buf * (BN * 128));
    };
    auto aim = [&](int u) __attribute__((always_inline)) {
      const int last = seq.ak - 1 - (t_lo + u * BN);
      ks.aim(last);
      vs.aim(last);
      if constexpr (DR > 0) rs.aim(last);
    };
    // the streams to tile u, from the tile before it
    auto advance = [&](int u) __attribute__((always_inline)) {
      if (u >= ntiles) return;
      ks.base = uniform(ks.base + (int64_t)BN * ks.row_bytes);
      vs.base = uniform(vs.base + (int64_t)BN * vs.row_bytes);
      if constexpr (DR > 0) rs.base = uniform(rs.base + (int64_t)BN * rs.row_bytes);
      if (t_lo + (u + 1) * BN > seq.ak) aim(u);
    };
    auto load_tile = [&](int buf) __attribute__((always_inline)) {
      static_for<0, GPW>([&](auto j) __attribute__((always_inline)) { load_part(j, buf); });
    };
    // (a masked token has dS = 0, but 0 times a value that is not finite would reach rows that do not see it)
    auto is_mixed = [&](int u) { return t_lo + u * BN + BN > min_lim; };
    auto sanitize = [&](int u, int buf) __attribute__((always_inline)) {
      if (!is_mixed(u)) return;
      uint64_t bad = clean_share<IO, RB, BN, NWV>(lds_addr(L.t[buf].k), wave, lane);
      if constexpr (DR > 0) bad |= clean_share<IO, 128, BN, NWV>(lds_addr(L.kr[buf]), wave, lane);
      if (lane == 0) L.bad[buf][wave] = bad;
    };
    aim(0);
    load_tile(0);
    constexpr int QA = KSN;   // of Q's fragments in AGPRs: the accumulators leave room for no more
    uint4 qf[KS], df[KSN];
    const int64_t stat = n * (int64_t)a.len.rows * a.per + (int64_t)seq.r0 * a.per + r;
    const float lse = a.lse[stat];
    const float delta = -a.delta[stat];
    {
      const int64_t head = n * a.per + g;
      const uint16_t* qp = first_of(a.len, a.q, b, seq.r0) + s * a.q.row + head * a.q.head + kg * 8;
      const uint16_t* dp = first_of(a.len, a.d, b, seq.r0) + s * a.d.row + head * a.d.head + kg * 8;
#pragma unroll
      for (int j = 0; j < KSN; ++j) qf[j] = ldg16(qp + j * 16), df[j] = ldg16(dp + j * 16);
      if constexpr (DR > 0) {
        const uint16_t* rp = first_of(a.len, a.qr, b, seq.r0) + s * a.qr.row + head * a.qr.head + kg * 8;
#pragma unroll
        for (int j = KSN; j < KS; ++j) qf[j] = ldg16(rp + (j - KSN) * 16);
      }
#pragma unroll
      for (int j = 0; j < QA; ++j) qf[j] = in_agprs(qf[j]);
#pragma unroll
      for (int j = 0; j < KSN; ++j) df[j] = in_agprs(df[j]);
    }

    // ---- operands
    constexpr int VOFF = BN * D * 2;   // from a place in k to the same in v
    const int tk = s_row(rr), g16 = lane >> 4, c16 = lane & 15;
    const int r4 = (g16 >> 1) * 8 + (c16 >> 2), vc = (g16 & 1) * 2 + ((c16 & 3) >> 1), o8 = (c16 & 1) * 8;
    const uint32_t op_lane = tile_off<RB>(tk, kg), opr_lane = tile_off<128>(tk, kg);
    const uint32_t tr_lo = tile_off<RB>(r4, vc) + o8, tr_hi = tile_off<RB>(r4 + 4, vc) + o8;
    const uint32_t trr_lo = tile_off<128>(r4, vc) + o8, trr_hi = tile_off<128>(r4 + 4, vc) + o8;
    OpAddr<RB> op;
    OpAddr<128> opr;
    TrAddr<RB> tr;
    TrAddr<128> trr;
    auto point_op = [&](int buf) __attribute__((always_inline)) {
      op.point(lds_addr(L.t[buf].k), op_lane);
      if constexpr (DR > 0) opr.point(lds_addr(L.kr[buf]), opr_lane);
    };
    auto point_tr = [&](int buf) __attribute__((always_inline)) {
      tr.point(lds_addr(L.t[buf].k), tr_lo, tr_hi);
      if constexpr (DR > 0) trr.point(lds_addr(L.kr[buf]), trr_lo, trr_hi);
    };
    auto k_frag = [&](int j, int h) __attribute__((always_inline)) -> uint4 {
      return lds_read16_at(j < KSN ? op.a[j < KSN ? j : 0] + h * 32 * RB : opr.a[j >= KSN ? j - KSN : 0] + h * 32 * 128);
    };
    auto v_frag = [&](int j, int h) __attribute__((always_inline)) -> uint4 { return lds_read16_at(op.a[j] + h * 32 * RB + VOFF); };
    // product i of a half's NP: column tiles of dQ and its rotary part for 16 tokens, then for the next 16
    constexpr int NC = ON + RN, NP = 2 * NC;
    auto t_frag = [&](int i, int h) __attribute__((always_inline)) -> uint4 {
      const int st = i / NC, c = i % NC;
      if (c < ON) return tr.frag(c < ON ? c : 0, (h * 32 + st * 16) * RB);
      return trr.frag(c >= ON ? c - ON : 0, (h * 32 + st * 16) * 128);
    };
    // S^T and dP^T of half h of the tile that op points to, by themselves
    auto scores = [&](int h, f32x16& sv, f32x16& dp) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < KS - 1; ++j) {
        const uint4 f = k_frag(j, h);
        if (j == 0) mfma32_va<IO, true>(sv, f, qf[j]);
        else if (j < QA) mfma32_va<IO, false>(sv, f, qf[j]);
        else mfma32_vv<IO>(sv, f, qf[j]);
      }
#pragma unroll
      for (int j = 0; j < KSN - 1; ++j) {
        const uint4 f = v_frag(j, h);
        if (j == 0) mfma32_va<IO, true>(dp, f, df[j]);
        else mfma32_va<IO, false>(dp, f, df[j]);
      }
      if constexpr (QA < KS) mfma32_vv_va_end2<IO>(sv, k_frag(KS - 1, h), qf[KS - 1], dp, v_frag(KSN - 1, h), df[KSN - 1]);
      else mfma32_va_end2<IO>(sv, k_frag(KS - 1, h), qf[KS - 1], dp, v_frag(KSN - 1, h), df[KSN - 1]);
    };
    auto mask = [&](int u, int buf, int h, f32x16& sv, f32x16& dp) __attribute__((always_inline)) {
      if (!is_mixed(u)) return;
      const int l = lim - (t_lo + u * BN + h * 32);
      const uint64_t all = L.bad[buf][0] | L.bad[buf][1] | L.bad[buf][2] | L.bad[buf][3];
      const uint32_t bad = (uint32_t)(all >> (h * 32));
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if ((bad >> s_token(i, kg)) & 1u) sv[i] = __builtin_nanf("");
        if (s_token(i, kg) >= l) sv[i] = masked, dp[i] = 0.f;
      }
    };
    // ---- P and dS of 32 tokens in NST stages of two each, placed among the products before and after them
    constexpr int NST = 8;
    const float fs = factor.x * 0x1p-15f;   // (fp16's P has the factor 2^15)
    auto stage = [&](int st, f32x16& sv, f32x16& dp, uint32_t (&pn)[8], uint32_t (&wn)[8]) __attribute__((always_inline)) {
      const int i = 2 * st;
      const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[i], sl2, -lse));
      const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[i + 1], sl2, -lse));
      sum = fmaf(p0, dp[i], sum);
      sum = fmaf(p1, dp[i + 1], sum);
      float x0 = p0 * (dp[i] - delta), x1 = p1 * (dp[i + 1] - delta);
      if constexpr (IO == IO_F16) x0 *= fs, x1 *= fs;
      pn[st] = pack2<IO>(p0, p1);
      wn[st] = pack2<IO>(x0, x1);
      asm volatile("" : "+v"(pn[st]), "+v"(wn[st]), "+v"(sum));   // here, not where the next step needs them
    };

    // ---- One step handles 32 tokens: the products of those before them, S and dP of those after them, each MFMA
    // followed by a part of this one's P and dS. Fragments are read a few MFMAs ahead.
    constexpr int LAG = KS - KSN, NS = KS + KSN;   // S and dP end together
    constexpr int TR = 4, KR = D == 64 ? 2 : 4, VR = KR;   // (heads of 64: 254 registers, two work-groups on a CU)
    uint4 tf[TR], kf[KR], vf[VR];
    auto step = [&](auto pvc, auto sc, auto hc, f32x16& cs, f32x16& cd, f32x16& ns, f32x16& nd, uint32_t (&pb)[8], uint32_t (&wb)[8],
                    uint32_t (&pn)[8], uint32_t (&wn)[8], auto&& between, auto&& ride) __attribute__((always_inline)) {
      constexpr bool PV = decltype(pvc)::value, S = decltype(sc)::value;
      constexpr int H = decltype(hc)::value;
      constexpr int M0 = PV ? 2 * NP : 0, NMM = M0 + (S ? NS : 0), LEAD = NMM > 8 ? 2 : 0;
      auto values_at = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
        for (int st = 0; st < NST; ++st)
          if (LEAD + st * (NMM - LEAD) / NST == slot) stage(st, cs, cd, pn, wn);
      };
      if constexpr (PV)
        static_for<0, 2 * NP>([&](auto ic) __attribute__((always_inline)) {
          constexpr int i = decltype(ic)::value / 2, st = i / NC, c = i % NC;
          if constexpr (decltype(ic)::value % 2 == 0) {
            dq[c] = Mfma<IO>::m32(tf[i % TR], make_uint4(wb[4 * st], wb[4 * st + 1], wb[4 * st + 2], wb[4 * st + 3]), dq[c]);
          } else {
            pk[c] = Mfma<IO>::m32(tf[i % TR], make_uint4(pb[4 * st], pb[4 * st + 1], pb[4 * st + 2], pb[4 * st + 3]), pk[c]);
            if constexpr (i + TR < NP) tf[i % TR] = t_frag(i + TR, H);
          }
          if constexpr (S)
            static_for<0, KR + VR>([&](auto gc) __attribute__((always_inline)) {
              constexpr int g = decltype(gc)::value;
              if constexpr (g * 2 * NP / (KR + VR) == decltype(ic)::value) {
                if constexpr (g < KR) kf[g] = k_frag(g, H);
                else vf[g - KR] = v_frag(g - KR, H);
              }
            });
          values_at(decltype(ic)::value);
          __builtin_amdgcn_sched_barrier(0);
        });
      between();
      if constexpr (S)
        static_for<0, NS>([&](auto jc) __attribute__((always_inline)) {
          constexpr int j = decltype(jc)::value;
          constexpr bool is_s = j < LAG || (j - LAG) % 2 == 0;
          constexpr int i = j < LAG ? j : is_s ? LAG + (j - LAG) / 2 : (j - LAG) / 2;   // step of its chain
          if constexpr (j == NS - 1 && QA < KS) mfma32_vv_va_end2<IO>(ns, kf[(KS - 1) % KR], qf[KS - 1], nd, vf[(KSN - 1) % VR], df[KSN - 1]);
          else if constexpr (j == NS - 1) mfma32_va_end2<IO>(ns, kf[(KS - 1) % KR], qf[KS - 1], nd, vf[(KSN - 1) % VR], df[KSN - 1]);
          else if constexpr (is_s && i < KS - 1) {
            if constexpr (i < QA) mfma32_va<IO, i == 0>(ns, kf[i % KR], qf[i]);
            else mfma32_vv<IO>(ns, kf[i % KR], qf[i]);
            if constexpr (i + KR < KS) kf[i % KR] = k_frag(i + KR, H);
          } else if constexpr (!is_s) {
            mfma32_va<IO, i == 0>(nd, vf[i % VR], df[i]);
            if constexpr (i + VR < KSN) vf[i % VR] = v_frag(i + VR, H);
          }
          if constexpr (j >= NS - TR) tf[j - (NS - TR)] = t_frag(j - (NS - TR), 1 - H);
          ride(jc);
          values_at(M0 + j);
          __builtin_amdgcn_sched_barrier(0);
        });
    };
    std::true_type yes;
    std::false_type no;
    std::integral_constant<int, 0> h0;
    std::integral_constant<int, 1> h1;
    auto nothing = [](auto...) __attribute__((always_inline)) {};

    wait_vmcnt<0>();
    asm volatile("" ::: "memory");
    sanitize(0, 0);
    lds_barrier();
    advance(1);
    load_tile(1);
    f32x16 s0, s1, d0, d1;
    uint32_t p0[8], p1[8], w0[8], w1[8];
    point_op(0);
    scores(0, s0, d0);
#pragma unroll
    for (int j = 0; j < KR; ++j) kf[j] = k_frag(j, 1);
#pragma unroll
    for (int j = 0; j < VR; ++j) vf[j] = v_frag(j, 1);
    int buf = 0;   // of tile u
    // Step (u, 0): tile u + 1 has landed by the middle of it, when nobody needs tile u - 1 any more
    auto half0 = [&](auto pvc, int u) __attribute__((always_inline)) {
      const int nb = buf == NBUF - 1 ? 0 : buf + 1, lb = buf == 0 ? NBUF - 1 : buf - 1;   // of tiles u + 1 and u - 1 (u + 2)
      mask(u, buf, 0, s0, d0);
      advance(u + 2);
      step(pvc, yes, h1, s0, d0, s1, d1, p1, w1, p0, w0,
           [&]() __attribute__((always_inline)) {
             wait_vmcnt<0>();
             asm volatile("" ::: "memory");
             if (u + 1 < ntiles) sanitize(u + 1, nb);
             lds_barrier();
             point_tr(buf);
           },
           [&](auto jc) __attribute__((always_inline)) {
             constexpr int j = decltype(jc)::value;
             static_for<0, GPW>([&](auto g) __attribute__((always_inline)) {
               if constexpr (g * NS / GPW == j) load_part(g, lb);
             });
           });
    };
    half0(no, 0);
    for (int uv = 0; uv + 1 < ntiles; ++uv) {
      const int u = __builtin_amdgcn_readfirstlane(uv);
      const int nb = buf == NBUF - 1 ? 0 : buf + 1;
      point_op(nb);
      mask(u, buf, 1, s1, d1);
      step(yes, yes, h0, s1, d1, s0, d0, p0, w0, p1, w1, nothing, nothing);
      buf = nb;
      half0(yes, u + 1);
    }
    mask(ntiles - 1, buf, 1, s1, d1);
    step(yes, no, h0, s1, d1, s0, d0, p0, w0, p1, w1, nothing, nothing);
#pragma unroll
    for (int i = 0; i < TR; ++i) tf[i] = t_frag(i, 1);
    static_for<0, NP>([&](auto ic) __attribute__((always_inline)) {
      constexpr int i = decltype(ic)::value, st = i / NC, c = i % NC;
      dq[c] = Mfma<IO>::m32(tf[i % TR], make_uint4(w1[4 * st], w1[4 * st + 1], w1[4 * st + 2], w1[4 * st + 3]), dq[c]);
      pk[c] = Mfma<IO>::m32(tf[i % TR], make_uint4(p1[4 * st], p1[4 * st + 1], p1[4 * st + 2], p1[4 * st + 3]), pk[c]);
      if constexpr (i + TR < NP) tf[i % TR] = t_frag(i + TR, 1);
    });
    wait_vmcnt<0>();   // the last (unused) loads land before the LDS is released
    sum = add_half_swap(sum) * (IO == IO_F16 ? 0x1p-15f : 1.f);
    if (a.q_splits == 1) {
      if (lane < 32 && valid && !dead) a.delta[stat] = -sum;
      const float more = (delta - sum) * (IO == IO_F16 ? fs : 1.f);
#pragma unroll
      for (int c = 0; c < ON + RN; ++c)
#pragma unroll
        for (int i = 0; i < 16; ++i) dq[c][i] = fmaf(more, pk[c][i], dq[c][i]);
    }
  }

  const float f = a.scale * factor.y;
  if (a.q_splits > 1) {
    if (w_base >= r_end) return;
    const int blk = n * (a.q_blocks / a.key_heads) + (int)((int64_t)seq.r0 * a.per / 32) + b + w_base / 32;
    // both sums and that of P dP: the join knows all of it
    if (lane < 32) a.q_sum[((int64_t)at.sp * a.q_blocks + blk) * 32 + rr] = dead ? 0.f : sum;
    float4* dst = a.q_part + ((int64_t)at.sp * a.q_blocks + blk) * (2 * (D + DR) / 8) * 64 + lane;
    const float fp = a.scale * (IO == IO_F16 ? 0x1p-15f : 1.f);
#pragma unroll
    for (int c = 0; c < 2 * (ON + RN); ++c) {
      const f32x16& v = c < ON + RN ? dq[c < ON + RN ? c : 0] : pk[c >= ON + RN ? c - ON - RN : 0];
      const float x = c < ON + RN ? f : fp;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        dst[(c * 4 + e) * 64] = dead ? make_float4(0.f, 0.f, 0.f, 0.f)
                                     : make_float4(v[4 * e] * x, v[4 * e + 1] * x, v[4 * e + 2] * x, v[4 * e + 3] * x);
    }
    return;
  }
  const int64_t head_row = (int64_t)(seq.r0 + s) * a.heads + n * a.per + g;
  auto store = [&](const f32x16& v, uint16_t* dst) __attribute__((always_inline)) {
    uint4 w[2];
    pack_tile<IO>(v, f, w);
    if (valid) {
      stg16(dst + 8 * kg, dead ? make_uint4(0, 0, 0, 0) : w[0]);
      stg16(dst + 8 * kg + 16, dead ? make_uint4(0, 0, 0, 0) : w[1]);
    }
  };
#pragma unroll
  for (int c = 0; c < ON; ++c) store(dq[c], a.dq + head_row * D + c * 32);
#pragma unroll
  for (int c = 0; c < RN; ++c) store(dq[ON + c], a.dqr + head_row * DR + c * 32);
}

// ---------------------------------------------------------------- joins
// Adds the ranges' blocks of 32 rows (tokens or head rows), in order. The columns are those of one, two or three
// outputs side by side: D + DR (+ D); the queries' blocks have those of sum P K behind them, whose share goes by the sum of
// P dP over all ranges, which is left for the keys' kernel.
template <int IO, int D, int DR, bool KEYS>
__global__ __launch_bounds__(256) void dense_join_kernel(GradK a) {
  constexpr int W8 = ((KEYS ? 2 * D : D) + DR) / 8;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, rr = lane & 31, kg = lane >> 5;
  const int blocks = KEYS ? a.k_blocks : a.q_blocks, splits = KEYS ? a.k_splits : a.q_splits, per = KEYS ? 1 : a.per;
  const int seqs = KEYS ? a.k_seqs : a.q_seqs;
  const int32_t* starts = KEYS ? a.len.key_start : a.len.row_start;
  const int per_head = blocks / a.key_heads, n = (int)blockIdx.x / per_head, i = (int)blockIdx.x - n * per_head;
  auto first = [&](int s) { return (int)((int64_t)starts[s] * per / 32) + s; };
  int lo = 0, up = seqs - 1;
  while (lo < up) {
    const int mid = (lo + up + 1) >> 1;
    if (first(mid) <= i) lo = mid; else up = mid - 1;
  }
  const Seq seq = seq_of(a.len, lo);
  const int count = KEYS ? seq.keys : seq.rows * a.per, row = (i - first(lo)) * 32 + rr;
  if (row - rr >= count) return;
  const bool seen = KEYS ? row < seq.ak : true;
  int64_t out_row;
  if constexpr (KEYS) out_row = (int64_t)(seq.k0 + row) * a.key_heads + n;
  else {
    const int s = row / a.per;
    out_row = (int64_t)(seq.r0 + s) * a.heads + n * a.per + (row - s * a.per);
  }
  constexpr int ALL8 = KEYS ? W8 : 2 * W8;
  float more = 0.f;
  if constexpr (!KEYS) {
    const int64_t stat = n * (int64_t)a.len.rows * a.per + (int64_t)seq.r0 * a.per + min(row, count - 1);
    const float delta = -a.delta[stat];
    float sum = 0.f;
#pragma unroll 4
    for (int k = 0; k < splits; ++k) sum += a.q_sum[((int64_t)k * blocks + blockIdx.x) * 32 + rr];
    more = delta - sum;
    __syncthreads();   // every wave has read it
    if (threadIdx.x < 32 && row < count) a.delta[stat] = -sum;
  }
  for (int grp = wave; grp < W8; grp += 4) {
    auto total = [&](int g) {
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      const float4* p = (KEYS ? a.k_part : a.q_part) + ((int64_t)blockIdx.x * ALL8 + g) * 64 + lane;
#pragma unroll 4
      for (int k = 0; k < splits; ++k) {
        const uint4 v = ldg16(p + (int64_t)k * blocks * ALL8 * 64);
        acc.x += __uint_as_float(v.x);
        acc.y += __uint_as_float(v.y);
        acc.z += __uint_as_float(v.z);
        acc.w += __uint_as_float(v.w);
      }
      return acc;
    };
    float4 acc = total(grp);
    if constexpr (!KEYS) {
      const float4 pk = total(W8 + grp);
      acc.x = fmaf(more, pk.x, acc.x), acc.y = fmaf(more, pk.y, acc.y), acc.z = fmaf(more, pk.z, acc.z), acc.w = fmaf(more, pk.w, acc.w);
    }
    if (row >= count) continue;
    const int c = grp * 8;
    uint16_t* dst;
    if (c < D) dst = (KEYS ? a.dk : a.dq) + out_row * D + c;
    else if (c < D + DR) dst = (KEYS ? a.dkr : a.dqr) + out_row * DR + (c - D);
    else dst = a.dv + out_row * D + (c - D - DR);
    *reinterpret_cast<uint2*>(dst + kg * 4) = seen ? make_uint2(pack2<IO>(acc.x, acc.y), pack2<IO>(acc.z, acc.w)) : make_uint2(0, 0);
  }
}

// ---------------------------------------------------------------- how a call is cut
int64_t div_up(int64_t x, int64_t y) { return (x + y - 1) / y; }
struct Part {   // one of the two main launches
  int even, splits, chunk, blocks, seqs;
  int64_t groups;
};
// Tiles of TOK rows (or tokens) of every sequence: by levels of the longest's number (the heaviest of all first), or
// numbered through where that is more than half as many again (1.9 times: 1069 and 1033 us, 4.1: 160 and 140, 24: 6068
// and 1975; 1.25: 1042 and 1113, 1.2: 445 and 466. Two sequences of 8 key heads, whose pairs turn by half a round, are the
// exception: 1.3: 882 and 755). Ranges of the other axis where there are fewer tiles than CUs: each loads its operands
// anew, and a launch adds their sums; of 512 rows, two rounds' worth, or up to four of 128 (a sample of 2048, 8 heads on 4:
// one range 159 us, 4 109, 8 149, as chosen 106; one of 300: 50, 53, 51, as chosen 50).
Part make_part(int64_t total, int64_t longest, int batch, bool behind, int heads, int64_t other, int forced) {
  Part p{};
  const int64_t seqs = batch + (behind ? 1 : 0);
  const int64_t tiles = std::max<int64_t>(1, div_up(longest, TOK));
  const int64_t even = tiles * seqs, through = total / TOK + seqs;
  const int64_t real = (total / TOK + batch) * heads;
  int64_t splits = forced;
  if (splits <= 0) splits = real >= 256 ? 1 : std::max<int64_t>(1, std::min(512 / real, std::max(other / 512, std::min<int64_t>(4, other / 128))));
  splits = std::min<int64_t>(splits, 64);
  p.chunk = (int)(div_up(std::max<int64_t>(div_up(other, splits), 1), BN) * BN);
  p.splits = (int)std::max<int64_t>(1, div_up(other, p.chunk));
  const bool compact = 2 * even > 3 * through || even * heads * p.splits * NWV * 64 >= MAX_THREADS;
  p.even = compact ? 0 : (int)tiles;
  p.seqs = (int)seqs;
  p.groups = (compact ? through : even) * heads * p.splits;
  p.blocks = (int)((total / 32 + seqs + 1) * heads);
  return p;
}
struct Cut {
  Part keys, queries;
  size_t stats, norms, k_part, q_part, q_sum, bytes;
};
size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }
Cut make_cut(const DenseGradArgs& g) {
  const DenseArgs& a = g.f;
  const int64_t per = a.n1 / a.n2, w = 8;
  Cut c{};
  c.keys = make_part(a.total_keys, g.max_keys, a.batch, g.keys_behind > 0, a.n2, a.max_rows * per, a.kv_splits);
  c.queries = make_part((int64_t)a.total_rows * per, a.max_rows * per, a.batch, a.rows_behind > 0, a.n2, a.max_kv, a.kv_splits);
  c.stats = align256((size_t)a.total_rows * a.n1 * sizeof(float));
  c.norms = 2 * PREP * sizeof(float);
  if (c.keys.splits > 1) c.k_part = (size_t)c.keys.splits * c.keys.blocks * (size_t)((2 * a.d + a.dr) / w) * 64 * sizeof(float4);
  if (c.queries.splits > 1) {
    c.q_part = (size_t)c.queries.splits * c.queries.blocks * (size_t)(2 * (a.d + a.dr) / w) * 64 * sizeof(float4);
    c.q_sum = align256((size_t)c.queries.splits * c.queries.blocks * 32 * sizeof(float));
  }
  c.bytes = 2 * c.stats + c.norms + c.k_part + c.q_part + c.q_sum;
  return c;
}

template <int IO, int D, int DR>
hipError_t launch_d(const GradK& k, const Cut& c, hipStream_t s) {
  hipLaunchKernelGGL((dense_prep_kernel<IO, D>), dim3(PREP), dim3(256), 0, s, k);
  hipLaunchKernelGGL((dense_queries_kernel<IO, D, DR>), dim3((unsigned)c.queries.groups), dim3(NWV * 64), 0, s, k);
  if (c.queries.splits > 1)
    hipLaunchKernelGGL((dense_join_kernel<IO, D, DR, false>), dim3((unsigned)c.queries.blocks), dim3(256), 0, s, k);
  if (k.linear) hipLaunchKernelGGL((dense_keys_kernel<IO, D, DR, true>), dim3((unsigned)c.keys.groups), dim3(NWV * 64), 0, s, k);
  else hipLaunchKernelGGL((dense_keys_kernel<IO, D, DR, false>), dim3((unsigned)c.keys.groups), dim3(NWV * 64), 0, s, k);
  if (c.keys.splits > 1)
    hipLaunchKernelGGL((dense_join_kernel<IO, D, DR, true>), dim3((unsigned)c.keys.blocks), dim3(256), 0, s, k);
  return hipGetLastError();
}
template <int IO>
hipError_t launch_io(const GradK& k, const Cut& c, int d, int dr, hipStream_t s) {
  if (d == 64) return launch_d<IO, 64, 0>(k, c, s);
  return dr ? launch_d<IO, 128, 64>(k, c, s) : launch_d<IO, 128, 0>(k, c, s);
}

}  // namespace
}  // namespace dsa

using namespace dsa;

size_t dense_grad_workspace_bytes(const DenseGradArgs& a) { return make_cut(a).bytes; }

hipError_t launch_dense_grad(const DenseGradArgs& g, size_t* lacking, hipStream_t s) {
  const DenseArgs& a = g.f;
  const Cut c = make_cut(g);
  *lacking = !a.ws || a.ws_bytes < c.bytes || ((uintptr_t)a.ws & 15) != 0 ? c.bytes : 0;
  if (*lacking) return hipSuccess;
  for (const Part* p : {&c.keys, &c.queries})
    if (p->groups * NWV * 64 >= MAX_THREADS || (p->splits > 1 && (int64_t)p->blocks * 256 >= MAX_THREADS)) return hipErrorInvalidConfiguration;
  GradK k{};
  auto rows = [](const DenseTensor& t) { return Rows{(const uint16_t*)t.p, t.row, t.head, t.batch}; };
  k.q = rows(a.q), k.qr = rows(a.qr), k.k = rows(a.k), k.kr = rows(a.kr), k.v = rows(a.v), k.d = rows(g.d_out), k.o = rows(g.out);
  k.len = {a.row_start, a.key_start, a.act_q, a.act_k, a.batch, a.total_rows, a.total_keys, a.sparse_mode, a.apart};
  k.heads = a.n1;
  k.key_heads = a.n2;
  k.per = a.n1 / a.n2;
  while ((1 << k.per_shift) < k.per) ++k.per_shift;
  k.per_mul = (uint32_t)(((1ull << (31 + k.per_shift)) + k.per - 1) / k.per);
  k.linear = 16 % k.per == 0;
  for (const DenseTensor* t : {&a.q, &a.qr, &g.d_out})   // (a lane's offset has 32 bits)
    if ((a.dr > 0 || t != &a.qr) && (16 * t->row + k.per * t->head) * 2 >= (1ll << 31)) k.linear = 0;
  k.q_seqs = c.queries.seqs, k.k_seqs = c.keys.seqs, k.q_even = c.queries.even, k.k_even = c.keys.even;
  k.scale = a.scale;
  k.stat_padded = a.stat_padded;
  k.s1 = std::max(1, a.total_rows / a.batch);
  k.sm_max = a.sm_max;
  k.sm_sum = a.sm_sum;
  char* ws = (char*)a.ws;
  k.lse = (float*)ws;
  k.delta = (float*)(ws + c.stats);
  k.norms = (float*)(ws + 2 * c.stats);
  k.k_part = (float4*)(ws + 2 * c.stats + c.norms);
  k.q_part = (float4*)(ws + 2 * c.stats + c.norms + c.k_part);
  k.q_sum = (float*)(ws + 2 * c.stats + c.norms + c.k_part + c.q_part);
  k.dq = (uint16_t*)g.dq, k.dqr = (uint16_t*)g.dqr, k.dk = (uint16_t*)g.dk, k.dkr = (uint16_t*)g.dkr, k.dv = (uint16_t*)g.dv;
  k.k_splits = c.keys.splits, k.k_chunk = c.keys.chunk, k.k_blocks = c.keys.blocks;
  k.q_splits = c.queries.splits, k.q_chunk = c.queries.chunk, k.q_blocks = c.queries.blocks;
  return a.io == DSA_DTYPE_BF16 ? launch_io<IO_BF16>(k, c, a.d, a.dr, s) : launch_io<IO_F16>(k, c, a.d, a.dr, s);
}
