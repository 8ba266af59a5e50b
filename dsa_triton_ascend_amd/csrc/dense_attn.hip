// Dense attention of whole prompts over keys and values of their own, for gfx950: forward.
//
// Head row r = (query s, head g of a group) of a sequence and key head sees the tokens t < limit(s):
//   score = (q . k_t + q_rope . k_rope_t) * scale,   out = softmax(score) . v
// limit(s) = act_k - act_q + s + 1 (causal, the last query is the last token) or act_k.
//
// A work-group of four waves has 128 RT head rows of one key head: the heads of a group lie side by side as rows,
// so keys and values are read once for all of them, and a single token's group still fills the MFMA's columns. Each wave
// owns 32 RT rows. Tiles of 64 tokens go direct to LDS. S^T = K Q^T has the tokens as M; the online softmax
// runs in each lane's scores of its own head row plus one exchange between lane halves, and its result is already
// the B operand of O^T += V^T P^T. P is rounded to the io type for that product; scores, sums and O have 32 bits.
#include <algorithm>

#include "dense_attn.hpp"

namespace dsa {
namespace {

constexpr int NWV = 4;
constexpr int BN = 64;     // tokens a tile
constexpr int NBUF = 2;

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
  float4* part_s;          // [splits][blocks][32]: reference maximum, true maximum, sum
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
  uint64_t bad[NBUF][NWV];
};

template <int IO, int D, int DR, int RT>
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
      i -= level * pairs;
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
    qp[m] = a.q.p + (seq.r0 + s) * a.q.row + (n * a.per + g) * a.q.head;
    if constexpr (DR > 0) qrp[m] = a.qr.p + (seq.r0 + s) * a.qr.row + (n * a.per + g) * a.qr.head;
  }
  const int w_base = r_base + wave * RT * 32, w_hi = seen(w_base, min(r_end, w_base + RT * 32));

  f32x16 o[RT][ON];
  float m_used[RT], m_true[RT], l_part[RT];
#pragma unroll
  for (int m = 0; m < RT; ++m) {
    m_used[m] = m_true[m] = -INFINITY;
    l_part[m] = 0.f;
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

    const Share<RB, BN, NWV> sh(wave, lane);
    const Share<DR ? DR * 2 : 128, BN, NWV> shr(wave, lane);
    const uint16_t* const kb = a.k.p + (int64_t)seq.k0 * a.k.row + n * a.k.head;
    const uint16_t* const vb = a.v.p + (int64_t)seq.k0 * a.v.row + n * a.v.head;
    const uint16_t* const krb = DR ? a.kr.p + (int64_t)seq.k0 * a.kr.row + n * a.kr.head : nullptr;
    const uint32_t k_row = (uint32_t)a.k.row * 2, v_row = (uint32_t)a.v.row * 2, kr_row = (uint32_t)a.kr.row * 2;
    // (rows past the last token repeat it; they are masked)
    auto load_rows = [&](auto share, const uint16_t* base, uint32_t row_bytes, int t0, uint8_t* dst) __attribute__((always_inline)) {
      const char* p = reinterpret_cast<const char*>(base) + (int64_t)t0 * row_bytes;
#pragma unroll
      for (int j = 0; j < share.CNT; ++j) {
        const int t = min(j * share.STEP + share.row, seq.ak - 1 - t0);
        lds_dma16_sbase_untracked(p, (uint32_t)t * row_bytes + share.col, dst + (j * NWV + wave) * 1024);
      }
    };
    auto load_tile = [&](int u) __attribute__((always_inline)) {
      const int t0 = t_lo + u * BN, buf = u % NBUF;
      load_rows(sh, kb, k_row, t0, L.k[buf]);
      load_rows(sh, vb, v_row, t0, L.v[buf]);
      if constexpr (DR > 0) load_rows(shr, krb, kr_row, t0, L.kr[buf]);
    };
    load_tile(0);
    uint4 qf[RT][KS];
#pragma unroll
    for (int m = 0; m < RT; ++m)
#pragma unroll
      for (int j = 0; j < KS; ++j)
        qf[m][j] = flipped(j < KSN ? ldg16(qp[m] + j * 16 + kg * 8) : ldg16(qrp[m] + (j - KSN) * 16 + kg * 8), flip);

    const int tk = s_row(rr);
    for (int u = 0; u < ntiles; ++u) {
      const int t0 = t_lo + u * BN, buf = u % NBUF;
      // A tile that some rows see only in part: a masked token has P = 0, but 0 times a value that is not finite would
      // still reach the rows that do not see it. Such values become 0 in LDS, and the token's score NaN for the
      // rows that do see it.
      const bool mixed = t0 + BN > min_lim;
      wait_vmcnt<0>();
      asm volatile("" ::: "memory");
      if (mixed) {
        const uint64_t bad = clean_share<IO, RB, BN, NWV>(lds_addr(L.v[buf]), wave, lane);
        if (lane == 0) L.bad[buf][wave] = bad;
      }
      lds_barrier();   // tile u is here, tile u - 1 done with
      if (u + 1 < ntiles) load_tile(u + 1);
      if (t0 >= w_hi) continue;
      uint64_t bad = 0;
      if (mixed) bad = L.bad[buf][0] | L.bad[buf][1] | L.bad[buf][2] | L.bad[buf][3];
      const uint32_t kt = lds_addr(L.k[buf]), vt = lds_addr(L.v[buf]), krt = lds_addr(L.kr[buf]);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        f32x16 sv[RT];
#pragma unroll
        for (int m = 0; m < RT; ++m)
#pragma unroll
          for (int i = 0; i < 16; ++i) sv[m][i] = 0.f;
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          const uint4 af = j < KSN ? op_frag<RB>(kt, h * 32 + tk, j, kg) : op_frag<128>(krt, h * 32 + tk, j - KSN, kg);
#pragma unroll
          for (int m = 0; m < RT; ++m) sv[m] = Mfma<IO>::m32(af, qf[m][j], sv[m]);
        }
        uint4 pb[RT][2];
#pragma unroll
        for (int m = 0; m < RT; ++m) {
          if (bad)
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if ((bad >> (h * 32 + s_token(i, kg))) & 1u) sv[m][i] = __builtin_nanf("");
          if (t0 + h * 32 + 32 > min_lim)
#pragma unroll
            for (int i = 0; i < 16; ++i)
              sv[m][i] = t0 + h * 32 + s_token(i, kg) < lim[m] || dead[m] ? sv[m][i] : -INFINITY;
          float mx = max3(sv[m][0], sv[m][1], sv[m][2]);
#pragma unroll
          for (int i = 3; i < 15; i += 2) mx = max3(mx, sv[m][i], sv[m][i + 1]);
          mx = max_half_swap(max3(mx, sv[m][15], sv[m][15])) * cpos;
          m_true[m] = max3(m_true[m], mx, mx);
          const float m_new = mx > m_used[m] + lazy_limit<IO>() ? mx - lazy_gap<IO>() : m_used[m];
          const float alpha = m_used[m] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m_used[m] - m_new) * LOG2E);
          m_used[m] = m_new;
          const float mb = m_new == -INFINITY ? 0.f : m_new * LOG2E;
          uint32_t d[8];
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[m][2 * i], cl2, -mb));
            const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[m][2 * i + 1], cl2, -mb));
            sum += p0;
            sum += p1;
            d[i] = pack2<IO>(p0, p1);
          }
          l_part[m] = l_part[m] * alpha + sum;
          pb[m][0] = make_uint4(d[0], d[1], d[2], d[3]);
          pb[m][1] = make_uint4(d[4], d[5], d[6], d[7]);
          if (__builtin_amdgcn_ballot_w64(alpha != 1.f)) {
#pragma unroll
            for (int c = 0; c < ON; ++c)
#pragma unroll
              for (int i = 0; i < 16; ++i) o[m][c][i] *= alpha;
          }
        }
#pragma unroll
        for (int st = 0; st < 2; ++st)
#pragma unroll
          for (int c = 0; c < ON; ++c) {
            const uint4 vf = tr_frag<RB>(vt, h * 32 + st * 16, c, lane);
#pragma unroll
            for (int m = 0; m < RT; ++m) o[m][c] = Mfma<IO>::m32(vf, pb[m][st], o[m][c]);
          }
      }
    }
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
        a.part_s[at * 32 + rr] = make_float4(m_used[m], top, dead[m] ? 0.f : l_tot, 0.f);
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
    const float inv = 1.f / l_tot;
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
// get zeros. A work-group has a block of 32 head rows; its waves take the D / 8 groups of 8 columns.
constexpr int MAX_SPLITS = 64;
template <int IO, int D>
__global__ __launch_bounds__(256) void dense_merge_kernel(DenseK a) {
  __shared__ float s_w[MAX_SPLITS][32];
  __shared__ float s_inv[32];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, rr = lane & 31, kg = lane >> 5;
  // the sequence of this block
  const int per_head = a.blocks / a.tiles.heads, n = (int)blockIdx.x / per_head, i = (int)blockIdx.x - n * per_head;
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
  if (threadIdx.x < 32) {
    const float4* ps = a.part_s + (int64_t)blockIdx.x * 32 + rr;
    const int64_t step = (int64_t)a.blocks * 32;
    float M = -INFINITY, top = -INFINITY, sum = 0.f;
    const int most = lim > 0 ? min(a.splits, (lim + a.chunk - 1) / a.chunk) : 0;   // ranges that this row sees
    for (int k = 0; k < most; ++k) {
      const float4 st = ps[k * step];
      if (st.z != 0.f) M = fmaxf(M, st.x), top = fmaxf(top, st.y);
    }
    for (int k = 0; k < a.splits; ++k) {
      float w = 0.f;
      if (k < most) {
        const float4 st = ps[k * step];
        // (a range whose scores are all NaN has no maximum: its weight is its sum, or the NaN would be left out)
        w = st.z != st.z ? st.z : st.z != 0.f ? exp2f((st.x - M) * LOG2E) : 0.f;
        if (w != 0.f) sum += w * st.z;
      }
      s_w[k][rr] = w;
    }
    s_inv[rr] = lim > 0 ? 1.f / sum : 0.f;
    if (a.sm_max && valid) {
      const int64_t at = stat_at(a, seq, n, row);
      a.sm_max[at] = lim > 0 ? top : 0.f;
      a.sm_sum[at] = lim > 0 ? sum * exp2f((M - top) * LOG2E) : 0.f;
    }
  }
  __syncthreads();
  const float inv = s_inv[rr];
  for (int grp = wave; grp < D / 8; grp += 4) {
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    const float4* p = a.part + ((int64_t)blockIdx.x * (D / 8) + grp) * 64 + lane;
    const int64_t step = (int64_t)a.blocks * (D / 8) * 64;
#pragma unroll 4
    for (int k = 0; k < a.splits; ++k) {
      const float w = s_w[k][rr];
      if (w != 0.f) {
        const uint4 v = ldg16(p + k * step);
        acc.x += w * __uint_as_float(v.x);
        acc.y += w * __uint_as_float(v.y);
        acc.z += w * __uint_as_float(v.z);
        acc.w += w * __uint_as_float(v.w);
      }
    }
    if (valid)
      *reinterpret_cast<uint2*>(a.out + ((int64_t)(seq.r0 + s) * a.heads + n * a.per + g) * D + grp * 8 + kg * 4) =
          lim > 0 ? make_uint2(pack2<IO>(acc.x * inv, acc.y * inv), pack2<IO>(acc.z * inv, acc.w * inv)) : make_uint2(0, 0);
  }
}

// ---------------------------------------------------------------- how a call is cut
struct Cut {
  int rt, even, through, splits, chunk, blocks;
  int64_t groups;
};
int64_t div_up(int64_t x, int64_t y) { return (x + y - 1) / y; }

Cut make_cut(const DenseArgs& a) {
  const int64_t seqs = a.batch + (a.rows_behind > 0), per = a.n1 / a.n2;
  Cut c{};
  // 256 rows a work-group where that leaves two rounds of the CUs, else 128
  auto tiles = [&](int rows) { return div_up((int64_t)a.max_rows * per, rows); };
  c.rt = (int64_t)a.total_rows * per / 256 * a.n2 >= 512 ? 2 : 1;
  const int rows = 128 * c.rt;
  const int64_t even = std::max<int64_t>(1, tiles(rows)) * seqs, through = (int64_t)a.total_rows * per / rows + seqs;
  const bool compact = even > through + through / 2;
  const int64_t items = (compact ? through : even) * a.n2;
  const int64_t real = ((int64_t)a.total_rows * per / rows + a.batch) * a.n2;   // about so many have rows
  int splits = a.kv_splits;
  if (splits <= 0) {
    splits = 1;
    if (real < 256) splits = (int)std::max<int64_t>(1, std::min<int64_t>(512 / std::max<int64_t>(real, 1), a.max_kv / 256));
  }
  splits = std::min(splits, MAX_SPLITS);
  c.chunk = (int)div_up(std::max<int64_t>(div_up(a.max_kv, splits), 1), BN) * BN;
  c.splits = (int)std::max<int64_t>(1, div_up(a.max_kv, c.chunk));
  c.even = compact ? 0 : (int)std::max<int64_t>(1, tiles(rows));
  c.through = (int)through;
  c.groups = items * c.splits;
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
  if (c.rt == 2) hipLaunchKernelGGL((dense_attn_kernel<IO, D, DR, 2>), dim3((unsigned)c.groups), dim3(NWV * 64), 0, s, k);
  else hipLaunchKernelGGL((dense_attn_kernel<IO, D, DR, 1>), dim3((unsigned)c.groups), dim3(NWV * 64), 0, s, k);
  if (c.splits > 1) hipLaunchKernelGGL((dense_merge_kernel<IO, D>), dim3((unsigned)c.blocks), dim3(256), 0, s, k);
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
  if (c.groups >= (1 << 24)) return hipErrorInvalidConfiguration;   // 2^32 threads
  DenseK k{};
  auto rows = [](const DenseTensor& t) { return Rows{(const uint16_t*)t.p, t.row, t.head}; };
  k.q = rows(a.q), k.qr = rows(a.qr), k.k = rows(a.k), k.kr = rows(a.kr), k.v = rows(a.v);
  k.len = {a.row_start, a.key_start, a.act_q, a.act_k, a.batch, a.total_rows, a.total_keys, a.sparse_mode};
  k.tiles = {a.batch + (a.rows_behind > 0), a.n2, c.even, c.through};
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
