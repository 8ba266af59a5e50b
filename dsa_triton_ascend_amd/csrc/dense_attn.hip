// Dense attention of whole prompts over keys and values of their own, for gfx950: forward.
//
// Head row r = (query s, head g of a group) of a sequence and key head sees the tokens t < limit(s):
//   score = (q . k_t + q_rope . k_rope_t) * scale,   out = softmax(score) . v
// limit(s) = act_k - act_q + s + 1 (causal, the last query is the last token) or act_k.
//
// A work-group has 256 or 128 head rows of one key head: the heads of a group lie side by side as rows, so keys and
// values are read once for all of them, and a single token's group still fills the MFMA's columns. Each wave owns 32 RT
// rows. Tiles of 64 tokens go direct to LDS, into a ring of three. S^T = K Q^T has the tokens as M; the online softmax
// runs in each lane's scores of its own head row plus one exchange between lane halves, and its result is already
// the B operand of O^T += V^T P^T. P is rounded to the io type for that product; scores, sums and O have 32 bits.
//
// Bound by the matrix instructions, and by the issue of all others beside them: the softmax of one half tile (32 tokens)
// is placed, a few operations at a time, among the products O += V P of the half before it and S of the one after (8192
// tokens, 32 heads on 8 of 128, bf16: 898 -> 621 us). Eight waves of 32 rows, two a SIMD, pass the time of each other's
// waits where the registers allow it (621 -> 553; heads of 64: 490 -> 372); with 192 wide scores Q alone would take the
// registers, and four waves of 64 rows read each fragment half as often. Loads whose addresses need no branch: 533 -> 513,
// 1070 TFLOP/s of those that the mask leaves.
#include <algorithm>

#include "dense_attn.hpp"

namespace dsa {
namespace {

constexpr int BN = 64;     // tokens a tile
constexpr int NBUF = 3;

// P = e^(score - reference). The reference moves, and the output is rescaled, only when a tile's P would exceed
// e^LIMIT, which is finite in the io type (bf16 has fp32's exponents; fp16 ends at e^11.09); it moves to GAP below
// that tile's maximum: fp16 rounds P below 2^-14 = e^-9.7 to steps of 2^-24, and with the gap a weight is off by at
// most 2^-25 e^-6 of the row's largest.
template <int IO> constexpr float lazy_limit() { return IO == IO_F16 ? 10.5f : 40.f; }
template <int IO> constexpr float lazy_gap() { return IO == IO_F16 ? 6.f : 0.f; }

struct DenseK {
  Rows q, qr, k, kr, v;
  Lens len;
  Tiles tiles;
  int per;                 // heads of a group
  int heads;               // query heads
  int64_t stat_head;       // statistics: elements from one key head to the next
  int stat_padded;         // [B, N2, S, G] (rows evenly split), else [N2, T, G]
  float scale;
  uint16_t* out;           // [rows, heads, D]
  float* sm_max;
  float* sm_sum;
  // ranges of tokens
  int splits, chunk;
  float4* part;            // [splits][blocks][D / 8][64]: 32 head rows as the MFMAs leave them
  float4* part_s;          // [splits][blocks][32]: reference maximum, true maximum, sum, NaN where a value is not finite
  int blocks;              // of 32 head rows, all key heads
};

// First block of 32 head rows of a sequence and key head
__device__ __forceinline__ int first_block(const DenseK& a, int b, const Seq& q, int n) {
  return n * (a.blocks / a.tiles.heads) + (int)((int64_t)q.r0 * a.per / 32) + b;
}
__device__ __forceinline__ int64_t stat_at(const DenseK& a, const Seq& q, int n, int r) {
  const int64_t first = (int64_t)q.r0 * a.per;
  return (a.stat_padded ? first * a.tiles.heads : first) + n * a.stat_head + r;
}

template <int D, int DR> struct FwdLds {
  uint8_t k[NBUF][BN * D * 2];
  uint8_t v[NBUF][BN * D * 2];
  uint8_t kr[NBUF][DR ? BN * DR * 2 : 16];
  uint64_t bad[NBUF][8];
};

template <int IO, int D, int DR, int NWV, int RT>
__global__ __launch_bounds__(NWV * 64) void dense_attn_kernel(DenseK a) {
  constexpr int KSN = D / 16, KS = (D + DR) / 16, ON = D / 32, RB = D * 2;
  constexpr int ROWS = NWV * 32 * RT;
  __shared__ __attribute__((aligned(16))) FwdLds<D, DR> L;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = lane >> 5, rr = lane & 31;

  // ---- which tile
  int b, n, tile, sp;
  Seq seq;
  {
    const int pairs = a.tiles.seqs * a.tiles.heads;
    int i = blockIdx.x;
    sp = 0;
    if (a.tiles.even) {
      const int level = i / pairs;
      i = pair_of(i, level, pairs, a.splits);
      b = i / a.tiles.heads;
      n = i - b * a.tiles.heads;
      sp = level % a.splits;
      seq = seq_of(a.len, b);
      const int nt = (int)(((int64_t)seq.rows * a.per + ROWS - 1) / ROWS);
      const int behind = a.tiles.even - 1 - level / a.splits;   // the longest sequence's last tile first
      if (behind >= nt) return;
      tile = behind;
    } else {
      sp = i % a.splits;
      i /= a.splits;
      n = i % a.tiles.heads;
      i /= a.tiles.heads;
      int lo = 0, hi = a.tiles.seqs - 1;
      auto first = [&](int s) { return (int)((int64_t)a.len.row_start[s] * a.per / ROWS) + s; };
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first(mid) <= i) lo = mid; else hi = mid - 1;
      }
      b = lo;
      seq = seq_of(a.len, b);
      const int nt = (int)(((int64_t)seq.rows * a.per + ROWS - 1) / ROWS);
      tile = nt - 1 - (i - first(b));
      if (tile < 0) return;
    }
  }
  const int r_base = tile * ROWS, r_end = min((int)min((int64_t)INT_MAX, (int64_t)seq.rows * a.per), r_base + ROWS);
  const int t_lo = sp * a.chunk;
  const int t_hi = sp == a.splits - 1 ? INT_MAX : t_lo + a.chunk;
  // how far tokens are seen: the limits grow with the row
  auto seen = [&](int x, int y) {   // by the queries of the rows [x, y)
    return x >= y || x / a.per >= seq.aq ? 0 : min(limit_of(a.len, seq, min((y - 1) / a.per, seq.aq - 1)), t_hi);
  };
  const int hi = seen(r_base, r_end);
  const int min_lim = max(t_lo + 1, limit_of(a.len, seq, r_base / a.per));   // from here on some row is masked
  const int ntiles = hi > t_lo ? (hi - t_lo + BN - 1) / BN : 0;

  // ---- this lane's head rows
  int row[RT], lim[RT];
  bool valid[RT], dead[RT];
  const uint16_t* qp[RT];
  const uint16_t* qrp[RT];
#pragma unroll
  for (int m = 0; m < RT; ++m) {
    row[m] = r_base + (wave * RT + m) * 32 + rr;
    valid[m] = row[m] < r_end;
    const int r = valid[m] ? row[m] : r_end - 1, s = r / a.per, g = r - s * a.per;
    lim[m] = valid[m] ? min(limit_of(a.len, seq, s), t_hi) : 0;
    dead[m] = lim[m] <= t_lo;
    qp[m] = first_of(a.len, a.q, b, seq.r0) + s * a.q.row + (n * a.per + g) * a.q.head;
    if constexpr (DR > 0) qrp[m] = first_of(a.len, a.qr, b, seq.r0) + s * a.qr.row + (n * a.per + g) * a.qr.head;
  }

  f32x16 o[RT][ON];
  float m_used[RT], m_true[RT], l_part[RT], alpha[RT];
  float taint[RT];   // NaN: a value that this row sees was not finite
#pragma unroll
  for (int m = 0; m < RT; ++m) {
    m_used[m] = m_true[m] = -INFINITY;
    l_part[m] = taint[m] = 0.f;
    alpha[m] = 1.f;
#pragma unroll
    for (int c = 0; c < ON; ++c)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[m][c][i] = 0.f;
  }

  if (ntiles > 0) {
    // the softmax works on raw scores times a positive factor: a negative scale negates the query, a
    // zero one becomes 1e-30 (scores round to 0, masked ones stay -inf)
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
    const float cpos = a.scale == 0.f ? 1e-30f : fabsf(a.scale);
    const float cl2 = cpos * LOG2E;

    // ---- tiles: each wave loads a share, in GPW loads, one tile after another (past the last one it again, into
    // buffers that nobody reads: no load then depends on a branch)
    Stream<RB, BN, NWV> ks(first_of(a.len, a.k, b, seq.k0) + t_lo * a.k.row + n * a.k.head, (uint32_t)a.k.row * 2, L.k[0], wave, lane);
    Stream<RB, BN, NWV> vs(first_of(a.len, a.v, b, seq.k0) + t_lo * a.v.row + n * a.v.head, (uint32_t)a.v.row * 2, L.v[0], wave, lane);
    Stream<128, BN, NWV> rs(DR ? first_of(a.len, a.kr, b, seq.k0) + t_lo * a.kr.row + n * a.kr.head : nullptr, (uint32_t)a.kr.row * 2, L.kr[0], wave, lane);
    constexpr int CK = ks.sh.CNT, CR = DR ? rs.sh.CNT : 0, GPW = 2 * CK + CR;
    auto load_part = [&](auto jc, int buf) __attribute__((always_inline)) {
      constexpr int j = decltype(jc)::value;
      if constexpr (j < CK) ks.template load<j>(buf * (BN * RB));
      else if constexpr (j < 2 * CK) vs.template load<j - CK>(buf * (BN * RB));
      else rs.template load<j - 2 * CK>(buf * (BN * 128));
    };
    // the streams to tile u, from the tile before it
    auto aim = [&](int u) __attribute__((always_inline)) {
      const int last = seq.ak - 1 - (t_lo + u * BN);
      ks.aim(last);
      vs.aim(last);
      if constexpr (DR > 0) rs.aim(last);
    };
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
    // A tile that some rows see only in part: a masked token has P = 0, but 0 times a value that is not finite would
    // still reach the rows that do not see it. Such values become 0 in LDS, and the output of the rows that do see them
    // NaN; the statistics are of the scores alone.
    auto is_mixed = [&](int u) { return t_lo + u * BN + BN > min_lim; };
    auto sanitize = [&](int u, int buf) __attribute__((always_inline)) {
      if (!is_mixed(u)) return;
      const uint64_t bad = clean_share<IO, RB, BN, NWV>(lds_addr(L.v[buf]), wave, lane);
      if (lane == 0) L.bad[buf][wave] = bad;
    };
    aim(0);
    load_tile(0);
    uint4 qf[RT][KS];
#pragma unroll
    for (int m = 0; m < RT; ++m)
#pragma unroll
      for (int j = 0; j < KS; ++j)
        qf[m][j] = flipped(j < KSN ? ldg16(qp[m] + j * 16 + kg * 8) : ldg16(qrp[m] + (j - KSN) * 16 + kg * 8), flip);
#pragma unroll
    for (int m = 0; m < RT; ++m)
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        i32x4v v = __builtin_bit_cast(i32x4v, qf[m][j]);
        asm volatile("" : "+a"(v));
        qf[m][j] = __builtin_bit_cast(uint4, v);
      }

    // ---- operand addresses of this lane in a buffer; those of the other fragments differ by an exclusive or of
    // constants in the chunk bits, kept in registers and moved to another buffer once a tile
    const int tk = s_row(rr), g16 = lane >> 4, c16 = lane & 15;
    const int t4 = (g16 >> 1) * 8 + (c16 >> 2), vc = (g16 & 1) * 2 + ((c16 & 3) >> 1);
    const uint32_t k_lane = tile_off<RB>(tk, kg), r_lane = tile_off<128>(tk, kg);
    const uint32_t v_lo = tile_off<RB>(t4, vc) + (c16 & 1) * 8, v_hi = tile_off<RB>(t4 + 4, vc) + (c16 & 1) * 8;
    uint32_t ka[KSN], ra[DR ? KS - KSN : 1], va[ON], vh[ON];
    auto point_k = [&](int buf) __attribute__((always_inline)) {
      const uint32_t kt = lds_addr(L.k[buf]), rt = lds_addr(L.kr[buf]);
#pragma unroll
      for (int j = 0; j < KSN; ++j) {
        ka[j] = kt + (k_lane ^ (j << 5));
        asm volatile("" : "+v"(ka[j]));
      }
      if constexpr (DR > 0)
#pragma unroll
        for (int j = 0; j < KS - KSN; ++j) {
          ra[j] = rt + (r_lane ^ (j << 5));
          asm volatile("" : "+v"(ra[j]));
        }
    };
    auto point_v = [&](int buf) __attribute__((always_inline)) {
      const uint32_t vt = lds_addr(L.v[buf]);
#pragma unroll
      for (int c = 0; c < ON; ++c) {
        va[c] = vt + (v_lo ^ (c << 6));
        vh[c] = vt + (v_hi ^ (c << 6));
        asm volatile("" : "+v"(va[c]), "+v"(vh[c]));
      }
    };
    auto k_frag = [&](int j, int h) __attribute__((always_inline)) -> uint4 {
      return lds_read16_at(j < KSN ? ka[j < KSN ? j : 0] + h * 32 * RB : ra[j >= KSN ? j - KSN : 0] + h * 32 * 128);
    };
    // column tile i % ON of the 16 tokens i / ON of half h
    auto v_frag = [&](int i, int h) __attribute__((always_inline)) -> uint4 {
      const int off = (h * 32 + (i / ON) * 16) * RB;
      const uint2 lo = ds_read_tr_at(va[i % ON] + off), hi2 = ds_read_tr_at(vh[i % ON] + off);
      return make_uint4(lo.x, lo.y, hi2.x, hi2.y);
    };

    // ---- online softmax of 32 tokens in NST stages of a few VALU operations, placed among the MFMAs of the products
    // before and after it. Raw scores; max(c s) = c max(s) as c > 0. The reference m_used moves only past the
    // lazy threshold, so the output's factor alpha is nearly always 1.
    constexpr int NST = 13;
    float sm_mx[RT], sm_mb[RT], sm_sum[RT], sm_p[RT];
    auto stage = [&](int st, int m, f32x16& sv, uint4 (&pn)[2]) __attribute__((always_inline)) {
      if (st < 2) {
        float mx = st == 0 ? max3(sv[0], sv[1], sv[2]) : max3(sm_mx[m], sv[9], sv[10]);
        mx = st == 0 ? max3(mx, sv[3], sv[4]) : max3(mx, sv[11], sv[12]);
        mx = st == 0 ? max3(mx, sv[5], sv[6]) : max3(mx, sv[13], sv[14]);
        sm_mx[m] = st == 0 ? max3(mx, sv[7], sv[8]) : max3(mx, sv[15], sv[15]);
      } else if (st == 2) {
        sm_mx[m] = max_half_swap(sm_mx[m]) * cpos;
        m_true[m] = max3(m_true[m], sm_mx[m], sm_mx[m]);
      } else if (st == 3) {
        const float m_new = sm_mx[m] > m_used[m] + lazy_limit<IO>() ? sm_mx[m] - lazy_gap<IO>() : m_used[m];
        alpha[m] = m_used[m] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m_used[m] - m_new) * LOG2E);
        m_used[m] = m_new;
        sm_mb[m] = m_new == -INFINITY ? 0.f : m_new * LOG2E;
        sm_sum[m] = 0.f;
      } else if (st < 12) {
        const int i = st - 4;
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[2 * i], cl2, -sm_mb[m]));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[2 * i + 1], cl2, -sm_mb[m]));
        sm_sum[m] += p0;
        sm_sum[m] += p1;
        uint32_t w = pack2<IO>(p0, p1);
        asm volatile("" : "+v"(w));   // here, not where the next step needs it
        uint4& q = pn[i >> 2];
        if ((i & 3) == 0) q.x = w;
        else if ((i & 3) == 1) q.y = w;
        else if ((i & 3) == 2) q.z = w;
        else q.w = w;
      } else {
        l_part[m] = l_part[m] * alpha[m] + sm_sum[m];
      }
    };
    auto mask = [&](int u, int buf, int h, f32x16 (&sv)[RT]) __attribute__((always_inline)) {
      if (!is_mixed(u)) return;
      const int t0 = t_lo + u * BN + h * 32;
      uint64_t all = 0;
#pragma unroll
      for (int w = 0; w < NWV; ++w) all |= L.bad[buf][w];
      const uint32_t bad = (uint32_t)(all >> (h * 32));
#pragma unroll
      for (int m = 0; m < RT; ++m) {
        const int l = dead[m] ? INT_MAX : lim[m] - t0;
        if (l > 0 && (bad & (0xFFFFFFFFu >> (l < 32 ? 32 - l : 0)))) taint[m] = __builtin_nanf("");
#pragma unroll
        for (int i = 0; i < 16; ++i) sv[m][i] = s_token(i, kg) < l ? sv[m][i] : -INFINITY;
      }
    };
    auto rescale = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int m = 0; m < RT; ++m)
        if (__builtin_amdgcn_ballot_w64(alpha[m] != 1.f)) {
#pragma unroll
          for (int c = 0; c < ON; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[m][c][i] = agpr_scale(o[m][c][i], alpha[m]);
        }
#pragma unroll
      for (int m = 0; m < RT; ++m)
#pragma unroll
        for (int c = 0; c < ON; ++c) asm volatile("" : "+a"(o[m][c]));   // whole accumulators, in AGPRs, across the branch
    };

    // ---- One step handles the 32 tokens i = (tile u, half h): O += V P of the tokens before them, then S of the tokens
    // after them, each MFMA followed by a stage of this one's softmax. Fragments are read a few MFMAs ahead, past the
    // end of one product for the next.
    constexpr int NPV = 2 * ON, NM = (NPV + KS) * RT;
    constexpr int RING = NWV == 8 ? 2 : 4, VR = NPV < RING ? NPV : RING, KR = KS < RING ? KS : RING;
    uint4 vfr[VR], kfr[KR];
    auto step = [&](auto pvc, auto sc, auto hc, f32x16 (&cur)[RT], f32x16 (&next)[RT], uint4 (&pb)[RT][2], uint4 (&pn)[RT][2],
                    auto&& between, auto&& ride) __attribute__((always_inline)) {
      constexpr bool PV = decltype(pvc)::value, S = decltype(sc)::value;
      constexpr int H = decltype(hc)::value;   // half of the product's tokens: V's and the next S's are the same
      constexpr int M0 = PV ? NPV * RT : 0, NMM = M0 + (S ? KS * RT : 0);
      constexpr int LEAD = NMM > 8 ? 2 : 0;   // (the scores' last products are on their way)
      auto softmax_at = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
        for (int st = 0; st < NST; ++st)
#pragma unroll
          for (int m = 0; m < RT; ++m)
            if (LEAD + (st * RT + m) * (NMM - LEAD) / (NST * RT) == slot) stage(st, m, cur[m], pn[m]);
      };
      if constexpr (NMM == 0) {
#pragma unroll
        for (int st = 0; st < NST; ++st)
#pragma unroll
          for (int m = 0; m < RT; ++m) stage(st, m, cur[m], pn[m]);
      }
      if constexpr (PV)
        static_for<0, M0>([&](auto jc) __attribute__((always_inline)) {
          constexpr int j = decltype(jc)::value, i = j / RT, m = j % RT;
          o[m][i % ON] = Mfma<IO>::m32(vfr[i % VR], pb[m][i / ON], o[m][i % ON]);
          if constexpr (m == RT - 1 && i + VR < NPV) vfr[i % VR] = v_frag(i + VR, H);
          if constexpr (S && m == 0 && i < KR) kfr[i] = k_frag(i, H);
          softmax_at(j);
          __builtin_amdgcn_sched_barrier(0);
        });
      between();
      if constexpr (S)
        static_for<0, KS * RT>([&](auto jc) __attribute__((always_inline)) {
          constexpr int j = decltype(jc)::value, i = j / RT, m = j % RT;
          if constexpr (i < KS - 1) mfma32_va<IO, i == 0>(next[m], kfr[i % KR], qf[m][i]);
          else if constexpr (m == RT - 1 && RT == 2) mfma32_va_last2<IO>(next[0], next[1], kfr[i % KR], qf[0][i], qf[1][i]);
          else if constexpr (RT == 1) mfma32_va_last<IO>(next[0], kfr[i % KR], qf[0][i]);
          if constexpr (m == RT - 1 && i + KR < KS) kfr[i % KR] = k_frag(i + KR, H);
          if constexpr (m == 0 && i >= KS - VR) vfr[i - (KS - VR)] = v_frag(i - (KS - VR), 1 - H);
          ride(jc);
          softmax_at(M0 + j);
          __builtin_amdgcn_sched_barrier(0);
        });
    };
    auto first_k = [&](int h) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < KR; ++i) kfr[i] = k_frag(i, h);
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
    f32x16 s0[RT], s1[RT];
    uint4 p0[RT][2], p1[RT][2];
    point_k(0);
    first_k(0);
    static_for<0, KS>([&](auto ic) __attribute__((always_inline)) {
      constexpr int i = decltype(ic)::value;
      if constexpr (i < KS - 1)
#pragma unroll
        for (int m = 0; m < RT; ++m) mfma32_va<IO, i == 0>(s0[m], kfr[i % KR], qf[m][i]);
      else if constexpr (RT == 2) mfma32_va_last2<IO>(s0[0], s0[1], kfr[i % KR], qf[0][i], qf[1][i]);
      else mfma32_va_last<IO>(s0[0], kfr[i % KR], qf[0][i]);
      if constexpr (i + KR < KS) kfr[i % KR] = k_frag(i + KR, 0);
    });
    first_k(1);
    int buf = 0;   // of tile u
    // Step (u, 0): tile u + 1 has landed by the middle of it, when nobody needs tile u - 1 any more
    auto middle = [&](int u) __attribute__((always_inline)) {
      const int nb = buf == NBUF - 1 ? 0 : buf + 1;
      wait_vmcnt<0>();
      asm volatile("" ::: "memory");
      if (u + 1 < ntiles) sanitize(u + 1, nb);
      lds_barrier();
    };
    auto half0 = [&](auto pvc, int u) __attribute__((always_inline)) {
      mask(u, buf, 0, s0);
      const int lb = buf == 0 ? NBUF - 1 : buf - 1;   // tile u - 1's, for tile u + 2
      advance(u + 2);
      step(pvc, yes, h1, s0, s1, p1, p0, [&]() __attribute__((always_inline)) {
             middle(u);
             point_v(buf);
           },
           [&](auto jc) __attribute__((always_inline)) {
             constexpr int j = decltype(jc)::value;
             static_for<0, GPW>([&](auto g) __attribute__((always_inline)) {
               if constexpr (g * (KS * RT) / GPW == j) load_part(g, lb);
             });
           });
      rescale();
    };
    half0(no, 0);
    for (int uv = 0; uv + 1 < ntiles; ++uv) {
      const int u = __builtin_amdgcn_readfirstlane(uv);
      const int nb = buf == NBUF - 1 ? 0 : buf + 1;
      point_k(nb);
      mask(u, buf, 1, s1);
      step(yes, yes, h0, s1, s0, p0, p1, nothing, nothing);
      rescale();
      buf = nb;
      half0(yes, u + 1);
    }
    mask(ntiles - 1, buf, 1, s1);
    step(yes, no, h0, s1, s0, p0, p1, nothing, nothing);
    rescale();
#pragma unroll
    for (int i = 0; i < VR; ++i) vfr[i] = v_frag(i, 1);
#pragma unroll
    for (int i = 0; i < NPV; ++i) {
#pragma unroll
      for (int m = 0; m < RT; ++m) o[m][i % ON] = Mfma<IO>::m32(vfr[i % VR], p1[m][i / ON], o[m][i % ON]);
      if (i + VR < NPV) vfr[i % VR] = v_frag(i + VR, 1);
    }
    wait_vmcnt<0>();   // the last (unused) loads land before the LDS is released
  }

  // ---- lane l holds head row rr, columns c * 32 + 8 g + 4 kg + j of o[c][4 g + j]
#pragma unroll
  for (int m = 0; m < RT; ++m) {
    const float l_tot = add_half_swap(l_part[m]);
    float top = m_true[m];
    if (a.scale == 0.f) top *= 0.f;
    if (a.splits > 1) {
      const int blk = first_block(a, b, seq, n) + r_base / 32 + wave * RT + m;
      const int64_t at = (int64_t)sp * a.blocks + blk;
      if (lane < 32 && valid[m])
        a.part_s[at * 32 + rr] = make_float4(m_used[m], top, dead[m] ? 0.f : l_tot, dead[m] ? 0.f : taint[m]);
      if (valid[m] && !dead[m]) {
        float4* dst = a.part + at * (D / 8) * 64 + lane;
#pragma unroll
        for (int c = 0; c < ON; ++c)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            dst[(c * 4 + g) * 64] = make_float4(o[m][c][4 * g], o[m][c][4 * g + 1], o[m][c][4 * g + 2], o[m][c][4 * g + 3]);
      }
      continue;
    }
    const int s = row[m] / a.per, g = row[m] - s * a.per;
    if (a.sm_max && lane < 32 && valid[m]) {
      const int64_t at = stat_at(a, seq, n, row[m]);
      a.sm_max[at] = dead[m] ? 0.f : top;
      a.sm_sum[at] = dead[m] ? 0.f : l_tot * exp2f((m_used[m] - top) * LOG2E);
    }
    const float inv = 1.f / l_tot + taint[m];
    uint16_t* dst = a.out + ((int64_t)(seq.r0 + s) * a.heads + n * a.per + g) * D + 8 * kg;
#pragma unroll
    for (int c = 0; c < ON; ++c) {
      uint4 w[2];
      pack_tile<IO>(o[m][c], inv, w);
      if (valid[m]) {
        stg16(dst + c * 32, dead[m] ? make_uint4(0, 0, 0, 0) : w[0]);
        stg16(dst + c * 32 + 16, dead[m] ? make_uint4(0, 0, 0, 0) : w[1]);
      }
    }
  }
}

// Joins the ranges of 32 head rows: M = max m_s, out = sum O_s 2^(m_s - M) / sum l_s 2^(m_s - M); rows that see nothing
// get zeros. A work-group has 32 columns of a block of 32 head rows. All its threads fetch the ranges' statistics at once,
// its waves take every fourth range, and their sums are added in the order of the waves.
constexpr int MAX_SPLITS = 64;
template <int IO, int D>
__global__ __launch_bounds__(256) void dense_merge_kernel(DenseK a) {
  __shared__ float s_w[MAX_SPLITS][32];
  __shared__ float2 s_top[8][32];   // of the ranges that 32 threads have: largest reference, true maximum
  __shared__ float s_sum[8][32];
  __shared__ float4 s_part[3][4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, rr = lane & 31, kg = lane >> 5;
  // the sequence of this block
  const int block = blockIdx.x / (D / 32), col = blockIdx.x % (D / 32);
  const int per_head = a.blocks / a.tiles.heads, n = block / per_head, i = block - n * per_head;
  auto first = [&](int s) { return (int)((int64_t)a.len.row_start[s] * a.per / 32) + s; };
  int lo = 0, up = a.tiles.seqs - 1;
  while (lo < up) {
    const int mid = (lo + up + 1) >> 1;
    if (first(mid) <= i) lo = mid; else up = mid - 1;
  }
  const Seq seq = seq_of(a.len, lo);
  const int r0 = (i - first(lo)) * 32;
  if (r0 >= (int64_t)seq.rows * a.per) return;   // (no such rows: the numbering leaves room)
  const int row = r0 + rr, s = row / a.per, g = row - s * a.per;
  const bool valid = row < (int64_t)seq.rows * a.per;
  const int lim = valid ? limit_of(a.len, seq, s) : 0;
  const int most = lim > 0 ? min(a.splits, (lim + a.chunk - 1) / a.chunk) : 0;   // ranges that this row sees
  const int k8 = threadIdx.x >> 5;
  float4 st[MAX_SPLITS / 8];
#pragma unroll
  for (int j = 0; j < MAX_SPLITS / 8; ++j) {
    const int k = k8 + 8 * j;
    st[j] = make_float4(-INFINITY, -INFINITY, 0.f, 0.f);
    if (k < most) st[j] = a.part_s[((int64_t)k * a.blocks + block) * 32 + rr];
  }
  float M = -INFINITY, top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int j = 0; j < MAX_SPLITS / 8; ++j)
    if (st[j].z != 0.f) M = fmaxf(M, st[j].x), top = fmaxf(top, st[j].y);
  s_top[k8][rr] = make_float2(M, top);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 8; ++j) M = fmaxf(M, s_top[j][rr].x), top = fmaxf(top, s_top[j][rr].y);
#pragma unroll
  for (int j = 0; j < MAX_SPLITS / 8; ++j) {
    // (a range whose scores are all NaN has no maximum: its weight is its sum, or the NaN would be left out)
    const float w = st[j].z != st[j].z ? st[j].z : st[j].z != 0.f ? exp2f((st[j].x - M) * LOG2E) : 0.f;
    if (w != 0.f) sum += w * st[j].z;
    s_w[k8 + 8 * j][rr] = w + st[j].w;
  }
  s_sum[k8][rr] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) sum += s_sum[j][rr];
  if (a.sm_max && col == 0 && threadIdx.x < 32 && valid) {
    const int64_t at = stat_at(a, seq, n, row);
    a.sm_max[at] = lim > 0 ? top : 0.f;
    a.sm_sum[at] = lim > 0 ? sum * exp2f((M - top) * LOG2E) : 0.f;
  }
  float4 acc[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) acc[c] = make_float4(0.f, 0.f, 0.f, 0.f);
  const float4* p = a.part + ((int64_t)block * (D / 8) + col * 4) * 64 + lane;
  const int64_t step = (int64_t)a.blocks * (D / 8) * 64;
  for (int k0 = wave; k0 < a.splits; k0 += 16) {
    float w[4];
    uint4 v[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = k0 + 4 * j < a.splits ? s_w[k0 + 4 * j][rr] : 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) v[j][c] = make_uint4(0, 0, 0, 0);
      if (w[j] != 0.f)
#pragma unroll
        for (int c = 0; c < 4; ++c) v[j][c] = ldg16(p + (k0 + 4 * j) * step + c * 64);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        acc[c].x += w[j] * __uint_as_float(v[j][c].x);
        acc[c].y += w[j] * __uint_as_float(v[j][c].y);
        acc[c].z += w[j] * __uint_as_float(v[j][c].z);
        acc[c].w += w[j] * __uint_as_float(v[j][c].w);
      }
  }
  if (wave)
#pragma unroll
    for (int c = 0; c < 4; ++c) s_part[wave - 1][c][lane] = acc[c];
  __syncthreads();
  if (wave || !valid) return;
  const float inv = lim > 0 ? 1.f / sum : 0.f;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
#pragma unroll
    for (int w = 0; w < 3; ++w) {
      const float4 v = s_part[w][c][lane];
      acc[c].x += v.x, acc[c].y += v.y, acc[c].z += v.z, acc[c].w += v.w;
    }
    *reinterpret_cast<uint2*>(a.out + ((int64_t)(seq.r0 + s) * a.heads + n * a.per + g) * D + (col * 4 + c) * 8 + kg * 4) =
        lim > 0 ? make_uint2(pack2<IO>(acc[c].x * inv, acc[c].y * inv), pack2<IO>(acc[c].z * inv, acc[c].w * inv)) : make_uint2(0, 0);
  }
}

// ---------------------------------------------------------------- how a call is cut
struct Cut {
  int rt, even, splits, chunk, blocks;
  int64_t groups;
};
int64_t div_up(int64_t x, int64_t y) { return (x + y - 1) / y; }

Cut make_cut(const DenseArgs& a) {
  const int64_t seqs = a.batch + (a.rows_behind > 0), per = a.n1 / a.n2;
  Cut c{};
  auto tiles = [&](int rows) { return div_up((int64_t)a.max_rows * per, rows); };
  // Work-groups of 256 rows read each tile half as often as those of 128, which balance better. With all items about as
  // long (no mask, or a chunk after many tokens; 16 heads, bf16, us of 256 and of 128 rows): those of 128 as long as they are one
  // round of the CUs (128 items: one sequence 54 and 43, 16 sequences 10.2 and 9.3; rotary, 100 items, 56 and 37), those of 256
  // from there on (129 items: 57 and 82, 12.6 and 18.7; 155: 66 and 96, rotary 85 and 109; 260: 220 and 225, 33 and 39; 1030:
  // 2339 and 2641, 197 and 236). Heads of 64, several of whose work-groups a CU holds: 128 items 42 and 36, 129 43 and 45,
  // 200 62 and 64, 240 76 and 81, 260 157 and 136, 1030 1552 and 1443; a chunk after twice as many tokens, 200 items 175 and
  // 153, 1030 items 10,987 and 10,191 (after six times as many). Below a diagonal, where the longest has twice the mean: 256
  // items 199 and 167, 320 items 75 and 83, 1024 items 504 and 631 (rotary 637 and 753); heads of 64 344 and 335.
  const bool flat = a.sparse_mode == 0 || a.max_kv >= 2 * (int64_t)a.max_rows;
  const int64_t items256 = (int64_t)a.total_rows * per * a.n2 / 256;
  c.rt = a.d == 128 ? (items256 > (flat ? 128 : 256) ? 2 : 1) : (a.sparse_mode == 0 && items256 > 128 && items256 <= 256 ? 2 : 1);
  const int rows = 128 * c.rt;
  const int64_t even = std::max<int64_t>(1, tiles(rows)) * seqs, through = (int64_t)a.total_rows * per / rows + seqs;
  const int64_t real = std::min(even, (int64_t)a.total_rows * per / rows + a.batch) * a.n2;   // about so many have rows
  // Fewer items than CUs: ranges of tokens that make one round of them, of two tiles at least (a work-group's LDS fills its
  // CU; four single tokens, 4 key heads, 8190 keys: 8, 16, 32 ranges take 29.9, 22.9, 27.8 us with their join), from
  // 512 tokens on (600 keys: 16.2 us in one range, 11.8 in four; 333: 10.0 in one, 13.0 in two).
  int splits = a.kv_splits;
  if (splits <= 0) {
    splits = 1;
    if (real < 256 && a.max_kv >= 512) splits = (int)std::max<int64_t>(1, std::min<int64_t>(256 / std::max<int64_t>(real, 1), a.max_kv / 128));
  }
  splits = std::min(splits, MAX_SPLITS);
  c.chunk = (int)div_up(std::max<int64_t>(div_up(a.max_kv, splits), 1), BN) * BN;
  c.splits = (int)std::max<int64_t>(1, div_up(a.max_kv, c.chunk));
  // All sequences get the longest's tiles, by levels, the last, which see most, first. Numbered through, that order is
  // lost: 43 sequences, the longest 512, 3.3 times as many even items: 32 and 38 us; 9, the longest 4096, 5.5 times: 161 and 152.
  const bool compact = even > 4 * through || even * a.n2 * c.splits * 2 * rows >= MAX_THREADS;
  c.even = compact ? 0 : (int)std::max<int64_t>(1, tiles(rows));
  c.groups = (compact ? through : even) * a.n2 * c.splits;
  c.blocks = (int)(((int64_t)a.total_rows * per / 32 + seqs + 1) * a.n2);
  return c;
}

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }
size_t workspace_bytes(const Cut& c, int d) {
  if (c.splits == 1) return 0;
  return (size_t)c.splits * c.blocks * (align256(32 * sizeof(float4)) + (size_t)32 * d * sizeof(float));
}

template <int IO, int D, int DR>
hipError_t launch_d(const DenseK& k, const Cut& c, hipStream_t s) {
  // 256 rows: eight waves of 32, two a SIMD, or (192 wide scores: their queries leave no room for that) four of 64
  if (c.rt == 2) hipLaunchKernelGGL((dense_attn_kernel<IO, D, DR, DR ? 4 : 8, DR ? 2 : 1>), dim3((unsigned)c.groups), dim3(DR ? 256 : 512), 0, s, k);
  else hipLaunchKernelGGL((dense_attn_kernel<IO, D, DR, 4, 1>), dim3((unsigned)c.groups), dim3(256), 0, s, k);
  if (c.splits > 1) hipLaunchKernelGGL((dense_merge_kernel<IO, D>), dim3((unsigned)c.blocks * (D / 32)), dim3(256), 0, s, k);
  return hipGetLastError();
}
template <int IO>
hipError_t launch_io(const DenseK& k, const Cut& c, int d, int dr, hipStream_t s) {
  if (d == 64) return launch_d<IO, 64, 0>(k, c, s);
  return dr ? launch_d<IO, 128, 64>(k, c, s) : launch_d<IO, 128, 0>(k, c, s);
}

}  // namespace
}  // namespace dsa

using namespace dsa;

size_t dense_attn_workspace_bytes(const DenseArgs& a) { return workspace_bytes(make_cut(a), a.d); }

hipError_t launch_dense_attn(const DenseArgs& a, size_t* lacking, hipStream_t s) {
  const Cut c = make_cut(a);
  const size_t need = workspace_bytes(c, a.d);
  *lacking = need > 0 && (!a.ws || a.ws_bytes < need || ((uintptr_t)a.ws & 15) != 0) ? need : 0;
  if (*lacking) return hipSuccess;
  if (c.groups * (c.rt == 2 && a.dr == 0 ? 512 : 256) >= MAX_THREADS || (c.splits > 1 && (int64_t)c.blocks * (a.d / 32) * 256 >= MAX_THREADS))
    return hipErrorInvalidConfiguration;
  DenseK k{};
  auto rows = [](const DenseTensor& t) { return Rows{(const uint16_t*)t.p, t.row, t.head, t.batch}; };
  k.q = rows(a.q), k.qr = rows(a.qr), k.k = rows(a.k), k.kr = rows(a.kr), k.v = rows(a.v);
  k.len = {a.row_start, a.key_start, a.act_q, a.act_k, a.batch, a.total_rows, a.total_keys, a.sparse_mode, a.apart};
  k.tiles = {a.batch + (a.rows_behind > 0), a.n2, c.even};
  k.per = a.n1 / a.n2;
  k.heads = a.n1;
  k.stat_padded = a.stat_padded;
  k.stat_head = (int64_t)(a.stat_padded ? a.total_rows / a.batch : a.total_rows) * k.per;
  k.scale = a.scale;
  k.out = (uint16_t*)a.out;
  k.sm_max = a.sm_max;
  k.sm_sum = a.sm_sum;
  k.splits = c.splits;
  k.chunk = c.chunk;
  k.blocks = c.blocks;
  k.part = (float4*)a.ws;
  k.part_s = k.part + (size_t)c.splits * c.blocks * (a.d / 8) * 64;
  return a.io == DSA_DTYPE_BF16 ? launch_io<IO_BF16>(k, c, a.d, a.dr, s) : launch_io<IO_F16>(k, c, a.d, a.dr, s);
}
