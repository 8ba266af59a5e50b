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
// An item is one work-group of four waves and 32, 64 or 128 head rows. Tiles of 32 tokens go direct to LDS.
// S^T = K Q^T has the tokens as M and 32 head rows as N; the online softmax runs in each lane's 16 scores
// of its head row plus one exchange between lane halves, and its result is already the B operand of
// O^T += V^T P^T, over all columns. P is rounded to the io type for that product, as the sparse attention's is (more
// bits of it would take a second product): the output's errors against 64 bits are 3 to 30% above those of 32-bit P.
// The sums of P, the scores and O are in 32 bits.
// With 128 head rows the matrix units are the bound: a wave for each block of 32, the tiles in a ring of three
// buffers shared by them. With fewer the bytes are, or the latency: the waves split the tokens and join their
// outputs through LDS at the end.
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
  // Partial outputs of 32 head rows x D values each, a block: as the MFMAs leave them, so that every store
  // and load is 1 KB in a row (row-major ones, 32 rows x 32 bytes an instruction, took 9.6 us a
  // work-group of 256 KB). Prefix range s holds block s * p_blocks + h / 32; own range s block s * o_blocks +
  // (row_start[b] * n1) / 32 + b + (h - row_start[b] * n1) / 32.
  float4* p_part;
  float4* o_part;
  float4* part_s;   // [rows * n1][slots]: reference maximum, true maximum, sum
  int p_blocks, o_blocks, n1_shift;
  int p_mt, p_tiles, p_splits, p_chunk;            // prefix items
  int o_mt, o_tiles, o_splits, o_chunk, o_base;    // own items (o_base: first token, 0 joined)
  int per_xcd, o_by_range;                         // work-groups per XCD; own items of a range on one XCD
  int o_items, o_compact;                          // own items of a range; numbered through (uneven sequences)
  int slots;
};

// A row of zeros, the source of tokens whose block is missing (never written)
__device__ const uint4 g_zero_row[(512 + 8) * 2 / 16] = {};

// 4-byte direct-to-LDS load: lane l writes lds_base + 4 l (see lds_dma16_untracked)
__device__ __forceinline__ void lds_dma4_untracked(const void* gptr, void* lds_base) {
  const uint32_t m0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)lds_base;
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" : : "v"(gptr), "s"(m0) : "memory", "m0");
}

// 16-byte direct-to-LDS load as lds_dma16_sbase_untracked, to LDS address lds + OFF: the sum goes into M0
// in one instruction (a wave here has its SIMD to itself, so each one it saves shortens the tile)
template <int OFF>
__device__ __forceinline__ void lds_dma16_at(uint64_t sbase, uint32_t voff, uint32_t lds) {
  asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :
               : "v"(voff), "s"(sbase), "s"(lds), "n"(OFF)
               : "memory", "m0", "scc");
}

// P = e^(score - reference). The reference moves, and the output is rescaled, only when a tile's P would exceed
// e^LIMIT, which is finite in the io type (bf16 has fp32's exponents; fp16 ends at e^11.09); it moves to GAP below
// that tile's maximum. fp16 rounds P below 2^-14 = e^-9.7 to steps of 2^-24: with the gap a weight is off by at most
// 2^-25 e^-6 of the row's largest, 3e-5 of it for 400,000 tokens together (without one, 60,000 tokens 17.5 below a
// single one were lost altogether, and with them values of 1.5e-3).
template <int IO> constexpr float lazy_limit() { return IO == IO_F16 ? 10.5f : 40.f; }
template <int IO> constexpr float lazy_gap() { return IO == IO_F16 ? 6.f : 0.f; }

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
  union {
    struct {                              // 128 head rows: a ring of tiles for the work-group
      uint8_t nope[NBUF][Tile<D>::NOPE];
      uint8_t rope[NBUF][Tile<D>::ROPE];
      uint16_t qr[128 * (DR + 8)];        // the query's rotary part
    };
    struct {                              // 32 or 64: the waves' or the groups' tiles; any: Q on its way to registers
      uint8_t own_nope[NWV][BN * D * 2];
      uint8_t own_rope[NWV][BN * DR * 2];
    };
    float4 join[NWV][D > 128 ? 32 : 16][64];   // the waves' outputs, up to 256 columns at a time
  };
  int32_t ids[4][BN];
  int red[2][NWV];
  uint32_t bad[2][NWV];                   // tokens of the tile (bit) with values that are not finite
  float4 stat[NWV][32];                   // 32 or 64 head rows: the waves' maxima and sums
};

// limit(h): how many tokens of its sequence head row h's query sees
struct Seq {
  int r0, r1, aq, ak;
};
__device__ __forceinline__ Seq seq_of(const PfxK& a, int b) { return {a.row_start[b], a.row_start[b + 1], a.act_q[b], a.act_k[b]}; }
__device__ __forceinline__ int row_limit(const PfxK& a, int row, const Seq& q) {
  const int s1 = row - q.r0;
  if (s1 < 0 || s1 >= q.aq || row >= q.r1) return 0;
  const int64_t thr = a.mode == 0 ? (int64_t)q.ak : (int64_t)q.ak - q.aq + s1 + 1;
  return (int)(thr < 0 ? 0 : thr > a.s2 ? a.s2 : thr);
}
// Sequence of a packed row: that of evenly split ones (all its values in one round of loads), a search
// where the guess is wrong
__device__ __forceinline__ int batch_guess(const PfxK& a, int row) { return min(row / a.guess_rows, a.batch - 1); }
__device__ __forceinline__ void batch_fix(const PfxK& a, int row, int& b, Seq& q) {
  if (q.r0 <= row && row < q.r1) return;
  b = batch_of_row(a.row_start, a.batch, row);
  q = seq_of(a, b);
}

struct Item {
  int h0, h_end;   // head rows [h0, min(h0 + 32 MT, h_end))
  int b;           // own items: the sequence; -1: prefix
  Seq seq;         // own items
  int t_lo, t_hi;  // tokens, before the rows' limits
  int slot;
  float4* part;    // the item's first block
};

// Copies head rows [h, h + 32) (rows past the last repeat it) to LDS, whole rows an instruction; chunk c of
// row r goes to c ^ (r % 16), so that a fragment read (16 rows, one chunk) touches every bank once.
template <int D>
__device__ __forceinline__ void stage_q(const uint16_t* q, int64_t h, int rows, uint8_t* dst, int lane) {
  constexpr int LPR = D / 8, RPI = 64 / LPR;   // lanes a row, rows an instruction
#pragma unroll 4
  for (int j = 0; j < 32 / RPI; ++j) {
    const int r = j * RPI + lane / LPR;
    lds_dma16_untracked(q + (h + min(r, rows - 1)) * D + ((lane % LPR) ^ (r & 15)) * 8, dst + j * 1024);
  }
}
__device__ __forceinline__ uint4 flipped(uint4 v, uint32_t f) { return make_uint4(v.x ^ f, v.y ^ f, v.z ^ f, v.w ^ f); }
template <int D>
__device__ __forceinline__ uint4 staged_q(const uint8_t* src, int ks, int rr, int kg) {
  return *reinterpret_cast<const uint4*>(src + rr * (D * 2) + (((2 * ks + kg) ^ (rr & 15)) << 4));
}

// 128 head rows: wave w has rows 32 w .. 32 w + 31, the tiles are shared.
template <int IO, int D>
__device__ __forceinline__ void run_item(const PfxK& a, const Item& it, PfxLds<D>& L) {
  using C = Tile<D>;
  constexpr int KS = C::KS, KSN = C::KSN;    // steps of S^T, of which in the latent part
  constexpr int ON = D / 32;                 // 32-column tiles of O
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = lane >> 5, rr = lane & 31;
  const int h = it.h0 + wave * 32 + rr;
  const bool valid = h < it.h_end;
  // the softmax works on raw scores times a positive factor: a negative scale negates the query, a
  // zero one becomes 1e-30 (scores round to 0, masked ones stay -inf)
  const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
  const float cpos = a.scale == 0.f ? 1e-30f : fabsf(a.scale);
  const float cl2 = cpos * LOG2E;

  // ---- block ids of the first tiles, requested before the item's end is known. Wave w copies tokens 8 w ..
  // 8 w + 7 of each tile; their block ids travel the same ordered path four tiles ahead, so nothing waits for
  // them. Tokens past the end (and tiles: every wave issues the same GPW loads per tile) read zeros.
  auto token = [&](int u) { return it.t_lo + u * BN + wave * 8 + (lane & 7); };
  auto page_of = [&](int t) { return (int)(((uint64_t)(uint32_t)t * a.page_mul) >> (31 + a.page_shift)); };
  auto ids_dma = [&](int u) __attribute__((always_inline)) {
    const int t = min(token(u), a.s2 - 1);
    const int32_t* src = a.table + (t < a.prefix || it.b < 0 ? 0 : (int64_t)it.b * a.max_blocks) + page_of(t);
    if (lane < 8) lds_dma4_untracked(src, &L.ids[u & 3][wave * 8]);
  };
#pragma unroll
  for (int u = 0; u < 4; ++u) ids_dma(u);
  // ---- this head row's sequence, requested first; then Q^T fragments (B operand: this lane's head row, 8
  // values at 16 ks + 8 kg), through LDS
  const int row = (valid ? h : it.h_end - 1) >> a.n1_shift;
  int b = it.b >= 0 ? it.b : batch_guess(a, row);
  Seq seq = it.b >= 0 ? it.seq : seq_of(a, b);
  asm volatile("" ::: "memory");
  uint4 qf[KSN];   // the latent part; the rotary part stays in LDS
  uint8_t* const qs = L.own_nope[wave];
  const int hb = it.h0 + wave * 32;
  // (a wave behind the last head row takes that one: the scores of whatever the LDS holds would grow, and
  // rescale the outputs, every few tiles, 2.7 us a tile instead of 1.5)
  const int hq = min(hb, it.h_end - 1);
  stage_q<D>(a.q, hq, min(32, it.h_end - hq), qs, lane);
  uint4 qrv[4];
  {
    const uint16_t* qr = a.qr + (int64_t)(valid ? h : it.h_end - 1) * DR + kg * 8;
#pragma unroll
    for (int j = 0; j < 4; ++j) qrv[j] = ldg16(qr + j * 16);
  }

  // ---- this head row's tokens: a row that sees none of the item's is dead: it runs along unmasked
  // and leaves a sum of 0
  if (it.b < 0) batch_fix(a, row, b, seq);
  int lim = valid ? row_limit(a, row, seq) : 0;
  const bool dead = lim <= it.t_lo;
  lim = dead ? INT_MAX : min(lim, it.t_hi);   // within the item
  int hi, min_lim;
  {
    // (VALU scans; the last lane has the wave's. Limits are not negative.)
    int mx = __builtin_amdgcn_readlane((int)wave_incl_max(dead ? 0u : (uint32_t)lim), 63);
    int mn = __builtin_amdgcn_readlane(wave_incl_min_i32(lim), 63);
    if (lane == 0) {
      L.red[0][wave] = mx;
      L.red[1][wave] = mn;
    }
    wait_vmcnt<0>();   // Q and the first ids
    asm volatile("" ::: "memory");
#pragma unroll
    for (int j = 0; j < KSN; ++j) qf[j] = flipped(staged_q<D>(qs, j, rr, kg), flip);
    __syncthreads();   // every wave has its Q: the staging area becomes the ring
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<uint4*>(L.qr + (wave * 32 + rr) * (DR + 8) + j * 16 + kg * 8) = flipped(qrv[j], flip);
    mx = max(max(L.red[0][0], L.red[0][1]), max(L.red[0][2], L.red[0][3]));
    mn = min(min(L.red[1][0], L.red[1][1]), min(L.red[1][2], L.red[1][3]));
    hi = __builtin_amdgcn_readfirstlane(mx);        // end of the item's tokens
    min_lim = __builtin_amdgcn_readfirstlane(mn);   // from here on some row is masked
  }
  const bool direct = a.slots == 1;
  const bool writer = lane < 32 && valid;   // one lane per head row
  if (hi <= it.t_lo) {   // no row sees any token
    if (direct) {
      for (int i = threadIdx.x; i < 128 * (D / 8); i += NWV * 64) {
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

  // where the latent and the rotary part of token 8 w + lane % 8 of tile u lie (a missing block: zeros)
  struct Source {
    uint32_t lo, hi;
    const uint16_t* rope;
  };
  auto tile_id = [&](int u) { return L.ids[u & 3][wave * 8 + (lane & 7)]; };
  auto tile_rows = [&](int u, int32_t id) __attribute__((always_inline)) -> Source {
    const int t = token(u);
    const bool ok = (uint32_t)id < a.blocks && t < hi;
    const int row = id * a.page + (t - page_of(t) * a.page);
    const uint16_t* zero = reinterpret_cast<const uint16_t*>(g_zero_row);
    const uint64_t p = (uint64_t)(ok ? a.k + (int64_t)row * D : zero);
    return {(uint32_t)p, (uint32_t)(p >> 32), (ok ? a.kr + (int64_t)row * DR : zero) + (lane >> 3) * 8};
  };
  // one of the GPW - 1 gathers of a tile: the latent of token 8 w + j, or (j = 8) the wave's rotary
  // parts, to the LDS addresses nope and rope (of the tile's buffer, this wave's rows)
  auto gather_part = [&](auto jc, const Source& src, uint32_t nope, uint32_t rope) __attribute__((always_inline)) {
    constexpr int j = decltype(jc)::value;
    if constexpr (j < 8) {
      const uint64_t p = (uint32_t)__builtin_amdgcn_readlane(src.lo, j) |
                         (uint64_t)(uint32_t)__builtin_amdgcn_readlane(src.hi, j) << 32;
      if (lane < D / 8) lds_dma16_at<nope_off<D>(j)>(p, lane * 16, nope);
    } else {
      lds_dma16_untracked(src.rope, (void*)(__attribute__((address_space(3))) void*)(uintptr_t)rope);
    }
  };
  // LDS addresses of this wave's rows in buffer b (8 w has token bits 0 and 1 clear)
  auto nope_at = [&](int b) { return (uint32_t)__builtin_amdgcn_readfirstlane(lds_addr(L.nope[b]) + nope_off<D>(wave * 8)); };
  auto rope_at = [&](int b) { return (uint32_t)__builtin_amdgcn_readfirstlane(lds_addr(L.rope[b]) + wave * 1024); };
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
  for (int u = 0; u < 2; ++u) {
    const Source src = tile_rows(u, tile_id(u));
    const uint32_t gnope = nope_at(u), grope = rope_at(u);
    static_for<0, C::GPW - 1>([&](auto j) { gather_part(j, src, gnope, grope); });
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
  constexpr int KPF = 5;
  auto s_tile = [&](int u, auto&& spread, auto&& pre) __attribute__((always_inline)) -> f32x16 {
    const uint8_t* arow = L.nope[u % NBUF] + nope_off<D>(tk) + kg * 16;
    const uint8_t* rrow = L.rope[u % NBUF] + rope_off(tk, kg);
    auto a_frag = [&](int j) -> uint4 {
      return j < KSN ? *reinterpret_cast<const uint4*>(arow + j * 32) : *reinterpret_cast<const uint4*>(rrow + (j - KSN) * 256);
    };
    uint4 qr[KS - KSN];
    auto qr_frag = [&](int j) -> uint4 {
      return *reinterpret_cast<const uint4*>(L.qr + (wave * 32 + rr) * (DR + 8) + j * 16 + kg * 8);
    };
    uint4 af[KPF];
#pragma unroll
    for (int j = 0; j < KPF; ++j) af[j] = a_frag(j);
    pre();
    f32x16 acc;
#pragma unroll
    for (int j = 0; j < KS; ++j) {
      const uint4 bq = j < KSN ? qf[j < KSN ? j : 0] : qr[j >= KSN ? j - KSN : 0];
      if (j == 0) acc = mfma32_vacc_first<IO>(af[0], bq);
      else if (j < KS - 1) mfma32_vacc<IO>(acc, af[j % KPF], bq);
      else acc = mfma32_vacc_last_to<IO>(acc, af[j % KPF], bq);
      if (j + KPF < KS) af[j % KPF] = a_frag(j + KPF);
      if (j + KPF < KS && j + KPF >= KSN) qr[j + KPF - KSN] = qr_frag(j + KPF - KSN);
      spread(j);
      __builtin_amdgcn_sched_barrier(0);
    }
    return acc;
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
      const float m_new = mx > m_used + lazy_limit<IO>() ? mx - lazy_gap<IO>() : m_used;
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
  const int vlane = nope_off<D>((g16 >> 1) * 8 + (c16 >> 2)) + ((g16 & 1) * 16 + 4 * (c16 & 3)) * 2;
  constexpr int NPV = 2 * ON;
  constexpr int VR = NPV < 8 ? NPV : 8;
  constexpr int NPRE = NPV >= 16 ? 6 : NPV / 4;   // before the next tile's S^T
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
    const int32_t id = tile_id(t + 2);
    if (is_mixed(t + 1)) sanitize(t + 1);
    lds_barrier();   // tile t + 1 resident; every wave done with tile t - 1, whose buffer is free
    Source src;   // (computed behind the chain's first MFMA)
    const uint32_t gnope = nope_at((t + 2) % NBUF), grope = rope_at((t + 2) % NBUF);   // the free buffer
    const uint32_t vbase = v_base(t), vnext = v_base(t + 1);
    f32x16 s1 = s_tile(
        t + 1,
        [&](int ks) __attribute__((always_inline)) {
          if (ks == 0) src = tile_rows(t + 2, id);
          static_for<0, C::GPW>([&](auto j) __attribute__((always_inline)) {
            if (1 + j * (KS - 1) / C::GPW == ks) {
              if constexpr (j < C::GPW - 1) gather_part(j, src, gnope, grope);
              else ids_dma(t + 4);   // the slot of tile t's ids, read two iterations ago
            }
          });
        },
        [&]() __attribute__((always_inline)) { pv_run(0, NPRE, vbase, vnext, true, [](int) {}); });
    mask(t + 1, s1);
    pv_run(NPRE, NPV, vbase, vnext, true, [&](int m) __attribute__((always_inline)) {
#pragma unroll
      for (int st = 0; st < NST; ++st)
        if (st * (NPV - NPRE) / NST == m - NPRE) smx(st, s1);
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
    float4* dst = it.part + (int64_t)wave * (D / 8) * 64 + lane;
#pragma unroll
    for (int n = 0; n < ON; ++n)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        dst[(n * 4 + g) * 64] = make_float4(o[n][4 * g], o[n][4 * g + 1], o[n][4 * g + 2], o[n][4 * g + 3]);
    return;
  }
  // two exchanges between lane halves leave lanes 0-31 with columns [0, 8) and [16, 24) of a 32-column
  // tile, the others with [8, 16) and [24, 32): 16-byte stores
  const float inv = 1.f / l_tot;
  uint16_t* dst = a.out + (int64_t)(valid ? h : 0) * D + 8 * kg;
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

// 32 or 64 head rows (MT = 1, 2 blocks): the waves split the tokens, NG = 4 / MT groups taking every NG-th
// tile, each wave with all of the contraction and of the columns of its row block.
//  * MT = 1: a wave's tile is loaded, then used, without a barrier; the four waves' loads and products
//    overlap, with up to four tiles (147 KB at D = 512) under way on a CU.
//  * MT = 2: the two waves of a group share its tile, each copying half of the next one into a second buffer
//    while they use this one: a barrier a tile. (Four waves on one tile, the contraction split and summed
//    through LDS, took 3285 cycles per 32 tokens, as long as 128 head rows do.)
template <int IO, int D, int MT>
__device__ __forceinline__ void run_tokens(const PfxK& a, const Item& it, PfxLds<D>& L) {
  constexpr int KSN = D / 16, KS = (D + DR) / 16, ON = D / 32, ROW = D * 2;
  constexpr int NG = NWV / MT, OWN = BN / MT;   // token groups; tokens of a tile that a wave copies
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rb = wave % MT, grp = wave / MT;
  const int kg = lane >> 5, rr = lane & 31;
  const int hb = it.h0 + rb * 32, h = hb + rr;
  const bool valid = h < it.h_end;
  const float cpos = a.scale == 0.f ? 1e-30f : fabsf(a.scale);
  const float cl2 = cpos * LOG2E;

  // the token that this lane looks up, its block requested before the item's end is known (tokens past it,
  // and tiles, read zeros)
  auto page_of = [&](int t) { return (int)(((uint64_t)(uint32_t)t * a.page_mul) >> (31 + a.page_shift)); };
  auto token = [&](int u) { return it.t_lo + u * BN + rb * OWN + (lane & (OWN - 1)); };
  auto block_id = [&](int u) {
    const int t = min(token(u), a.s2 - 1);
    return a.table[(t < a.prefix || it.b < 0 ? 0 : (int64_t)it.b * a.max_blocks) + page_of(t)];
  };
  int32_t id = block_id(grp);
  const int row = (valid ? h : it.h_end - 1) >> a.n1_shift;
  int b = it.b >= 0 ? it.b : batch_guess(a, row);
  Seq seq = it.b >= 0 ? it.seq : seq_of(a, b);
  asm volatile("" ::: "memory");
  const int hq = min(hb, it.h_end - 1);   // (as in run_item)
  stage_q<D>(a.q, hq, min(32, it.h_end - hq), L.own_nope[wave], lane);   // each wave for itself
  uint4 qf[KS];
  {
    const uint16_t* qr = a.qr + (int64_t)(valid ? h : it.h_end - 1) * DR + kg * 8;
#pragma unroll
    for (int j = KSN; j < KS; ++j) qf[j] = ldg16(qr + (j - KSN) * 16);
  }
  if (it.b < 0) batch_fix(a, row, b, seq);
  int lim = valid ? row_limit(a, row, seq) : 0;
  const bool dead = lim <= it.t_lo;
  lim = dead ? INT_MAX : min(lim, it.t_hi);
  int hi, min_lim;
  {
    // (VALU scans; the last lane has the wave's. Limits are not negative.)
    int mx = __builtin_amdgcn_readlane((int)wave_incl_max(dead ? 0u : (uint32_t)lim), 63);
    int mn = __builtin_amdgcn_readlane(wave_incl_min_i32(lim), 63);
    wait_vmcnt<0>();   // Q
    asm volatile("" ::: "memory");
#pragma unroll
    for (int j = 0; j < KSN; ++j) qf[j] = staged_q<D>(L.own_nope[wave], j, rr, kg);
    if (__builtin_expect(a.scale < 0.f, 0))
#pragma unroll
      for (int j = 0; j < KS; ++j) qf[j] = flipped(qf[j], 0x80008000u);
    if constexpr (MT > 1) {
      if (lane == 0) {
        L.red[0][wave] = mx;
        L.red[1][wave] = mn;
      }
      __syncthreads();   // (and every wave has its Q: the staging area becomes the tiles' buffers)
      mx = max(L.red[0][0], L.red[0][1]);
      mn = min(L.red[1][0], L.red[1][1]);
    }
    hi = __builtin_amdgcn_readfirstlane(mx);
    min_lim = __builtin_amdgcn_readfirstlane(mn);
  }
  const bool direct = a.slots == 1;
  const bool writer = grp == 0 && lane < 32 && valid;
  if (hi <= it.t_lo) {   // no row sees any token (every wave finds the same)
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

  // the group's buffers: one (MT = 1), or two in turn
  const uint32_t nope_lds = __builtin_amdgcn_readfirstlane(lds_addr(L.own_nope[grp * MT]));
  const uint32_t rope_lds = __builtin_amdgcn_readfirstlane(lds_addr(L.own_rope[grp * MT]));

  {
    float agpr_hint = 0.f;
    asm volatile("" : "+a"(agpr_hint));
  }
  f32x16 o[ON];
#pragma unroll
  for (int n = 0; n < ON; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[n][i] = 0.f;
  float m_used = -INFINITY, m_true = -INFINITY, l_part = 0.f;

  // Rows are unpadded: 16-byte chunk c of token t lies at c ^ kv_swz(t), so both readers' addresses are
  // a few fixed ones per lane plus constants. Operand read: chunk 2 ks + kg of token tk; transposed read:
  // tokens t4 (and + 4), chunk 4 n + vc.
  const int tk = 16 * (rr >> 4) + 8 * ((rr >> 2) & 1) + 4 * ((rr >> 3) & 1) + (rr & 3);
  const int g16 = lane >> 4, c16 = lane & 15;
  const int t4 = (g16 >> 1) * 8 + (c16 >> 2), vc = (g16 & 1) * 2 + ((c16 & 3) >> 1);
  const uint32_t k_at = nope_lds + tk * ROW + ((kg ^ kv_swz(tk & 15)) << 4);
  const uint32_t v_lo = nope_lds + t4 * ROW + ((vc ^ kv_swz(t4)) << 4) + (c16 & 1) * 8;
  const uint32_t v_hi = nope_lds + (t4 + 4) * ROW + ((vc ^ kv_swz(t4 + 4)) << 4) + (c16 & 1) * 8;
  const uint32_t r_at = rope_lds + rope_off(tk, kg);
  struct Base {
    uint32_t k, r, lo, hi;
  };
  // the lane's addresses in a buffer, opaque to the compiler: it would keep each of their combinations with
  // the constants in a register of its own
  auto base_of = [&](uint32_t buf) __attribute__((always_inline)) -> Base {
    Base b{k_at + buf * (BN * ROW), r_at + buf * (BN * DR * 2), v_lo + buf * (BN * ROW), v_hi + buf * (BN * ROW)};
    asm volatile("" : "+v"(b.k), "+v"(b.r), "+v"(b.lo), "+v"(b.hi));
    return b;
  };
  auto k_frag = [&](int j, const Base& b) __attribute__((always_inline)) -> uint4 {
    return lds_read16_at(j < KSN ? (b.k ^ ((j & 7) << 5)) + (j >> 3) * 256 : b.r + (j - KSN) * 256);
  };
  auto v_frag = [&](int m, const Base& b) __attribute__((always_inline)) -> uint4 {
    const int n = m % ON, off = (m / ON) * 16 * ROW + (n >> 2) * 256;
    const uint2 lo = ds_read_tr_at((b.lo ^ ((n & 3) << 6)) + off), hi2 = ds_read_tr_at((b.hi ^ ((n & 3) << 6)) + off);
    return make_uint4(lo.x, lo.y, hi2.x, hi2.y);
  };
  // This wave's part of tile u to buffer buf, in OWN + OWN / 8 loads: lane l holds where token OWN rb + l % OWN
  // lies (a missing block: zeros).
  struct Source {
    uint32_t lo, hi, rlo, rhi, dst, rdst;
  };
  auto source_of = [&](int u, int32_t id, uint32_t buf) __attribute__((always_inline)) -> Source {
    const int t = token(u);
    const bool ok = (uint32_t)id < a.blocks && t < hi;
    const int row = id * a.page + (t - page_of(t) * a.page);
    const uint16_t* zero = reinterpret_cast<const uint16_t*>(g_zero_row);
    const uint64_t p = (uint64_t)(ok ? a.k + (int64_t)row * D : zero);
    const uint64_t pr = (uint64_t)(ok ? a.kr + (int64_t)row * DR : zero);
    return {(uint32_t)p, (uint32_t)(p >> 32), (uint32_t)pr, (uint32_t)(pr >> 32),
            (uint32_t)__builtin_amdgcn_readfirstlane(nope_lds + buf * (BN * ROW) + rb * OWN * ROW),
            (uint32_t)__builtin_amdgcn_readfirstlane(rope_lds + buf * (BN * DR * 2) + rb * (OWN / 8) * 1024)};
  };
  constexpr int NLD = OWN + OWN / 8;
  auto load_part = [&](auto jc, const Source& s) __attribute__((always_inline)) {
    constexpr int j = decltype(jc)::value;
    if constexpr (j < OWN) {   // (OWN rb is a multiple of 16: the same permutation for every wave)
      const uint64_t src = (uint32_t)__builtin_amdgcn_readlane(s.lo, j) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane(s.hi, j) << 32;
      if (lane < D / 8) lds_dma16_at<j * ROW>(src, (lane * 16) ^ (kv_swz(j & 15) << 4), s.dst);
    } else {   // tokens 8 g + lane % 8, chunk lane / 8
      constexpr int g = j - OWN;
      const uint32_t lo = __shfl(s.rlo, 8 * g + (lane & 7)), hi2 = __shfl(s.rhi, 8 * g + (lane & 7));
      lds_dma16_untracked((const uint16_t*)(lo | (uint64_t)hi2 << 32) + (lane >> 3) * 8,
                          (void*)(__attribute__((address_space(3))) void*)(uintptr_t)(s.rdst + g * 1024));
    }
  };
  // values that are not finite, masked for some rows (see run_item): this wave's tokens of the tile
  auto sanitize = [&](uint32_t buf) __attribute__((always_inline)) -> uint32_t {
    uint32_t bad = 0;
#pragma unroll 1
    for (int j = rb * OWN; j < rb * OWN + OWN; ++j) {
      uint4* p = reinterpret_cast<uint4*>(L.own_nope[grp * MT + buf] + j * ROW + (lane % (D / 8)) * 16);
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
      if (__builtin_amdgcn_ballot_w64(any)) bad |= 1u << j;
    }
    return bad;
  };

  // MT = 1: the wave's own tiles only; MT = 2: every wave the same number of turns, for their barriers
  if constexpr (MT > 1) {
    const Source src = source_of(grp, id, 0);
    static_for<0, NLD>([&](auto j) __attribute__((always_inline)) { load_part(j, src); });
    id = block_id(grp + NG);
  }
  for (int uv = MT > 1 ? 0 : grp; uv < ntiles; uv += NG) {
    const int u0 = __builtin_amdgcn_readfirstlane(uv);
    const int u = MT > 1 ? u0 + grp : u0;
    const uint32_t buf = MT > 1 ? (u0 / NG) & 1 : 0;
    const int t0 = it.t_lo + u * BN;
    Source src;
    if constexpr (MT == 1) {
      // the last tile's reads are done (its products waited for them) before this one overwrites it
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      src = source_of(u, id, 0);
      static_for<0, NLD>([&](auto j) __attribute__((always_inline)) { load_part(j, src); });
      id = block_id(u + NG);
    }
    wait_vmcnt<0>();
    asm volatile("" ::: "memory");
    const bool mixed = min_lim < hi && t0 + BN > min_lim;
    uint32_t bad = mixed ? sanitize(buf) : 0;
    if constexpr (MT > 1) {
      if (mixed && lane == 0) L.bad[buf][wave] = bad;
      lds_barrier();   // the tile is here; both waves are done with the other buffer
      src = source_of(u + NG, id, buf ^ 1);
      if (mixed) bad = L.bad[buf][grp * MT] | L.bad[buf][grp * MT + 1];
    }
    // ---- S^T
    constexpr int KPF = 5;
    const Base at = base_of(buf);
    uint4 af[KPF];
#pragma unroll
    for (int j = 0; j < KPF; ++j) af[j] = k_frag(j, at);
    f32x16 sv;
#pragma unroll
    for (int j = 0; j < KS; ++j) {
      if (j == 0) sv = mfma32_vacc_first<IO>(af[0], qf[0]);
      else if (j < KS - 1) mfma32_vacc<IO>(sv, af[j % KPF], qf[j]);
      else sv = mfma32_vacc_last_to<IO>(sv, af[j % KPF], qf[j]);
      if (j + KPF < KS) af[j % KPF] = k_frag(j + KPF, at);
      if constexpr (MT > 1)   // the next tile's loads ride on the chain
        static_for<0, NLD>([&](auto i) __attribute__((always_inline)) {
          if (i * KS / NLD == j) load_part(i, src);
        });
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (MT > 1) id = block_id(u + 2 * NG);
    constexpr int VR = 4;
    uint4 vb[VR];
#pragma unroll
    for (int m = 0; m < VR; ++m) vb[m] = v_frag(m, at);
    if (bad)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if ((bad >> (16 * (i >> 3) + 8 * kg + (i & 7))) & 1u) sv[i] = __builtin_nanf("");
    if (t0 + BN > min_lim)
#pragma unroll
      for (int i = 0; i < 16; ++i) sv[i] = t0 + 16 * (i >> 3) + 8 * kg + (i & 7) < lim ? sv[i] : -INFINITY;
    // ---- softmax; a row may see nothing of a wave's first tiles
    float mx = max3(sv[0], sv[1], sv[2]);
#pragma unroll
    for (int i = 3; i < 15; i += 2) mx = max3(mx, sv[i], sv[i + 1]);
    mx = max_half_swap(max3(mx, sv[15], sv[15])) * cpos;
    m_true = max3(m_true, mx, mx);
    const float m_new = mx > m_used + lazy_limit<IO>() ? mx - lazy_gap<IO>() : m_used;
    const float alpha = m_used == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m_used - m_new) * LOG2E);
    m_used = m_new;
    const float mb = m_used == -INFINITY ? 0.f : m_used * LOG2E;
    uint32_t d[8];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[2 * i], cl2, -mb));
      const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[2 * i + 1], cl2, -mb));
      sum += p0;
      sum += p1;
      d[i] = pack2<IO>(p0, p1);
    }
    l_part = l_part * alpha + sum;
    if (__builtin_amdgcn_ballot_w64(alpha != 1.f)) {
#pragma unroll
      for (int n = 0; n < ON; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[n][i] = agpr_scale(o[n][i], alpha);
    }
    const uint4 pb[2] = {make_uint4(d[0], d[1], d[2], d[3]), make_uint4(d[4], d[5], d[6], d[7])};
#pragma unroll
    for (int m = 0; m < 2 * ON; ++m) {
      o[m % ON] = Mfma<IO>::m32(vb[m % VR], pb[m / ON], o[m % ON]);
      if (m + VR < 2 * ON) vb[m % VR] = v_frag(m + VR, at);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  if constexpr (MT > 1) wait_vmcnt<0>();   // the last (unused) loads land before their buffer is used again

  // ---- the groups' outputs joined, up to 256 columns at a time: sum over the groups of O_g 2^(m_g - M). The
  // outputs go to LDS as they are and a rolled loop scales and adds them: little code for what runs once (with
  // this, less of it in the prologue, and two groups a barrier, 16.2 us a call instead of 17.1 for 4 rows of 16
  // heads after 304 tokens).
  const float l_wave = add_half_swap(l_part);
  if (lane < 32) L.stat[wave][rr] = make_float4(m_used, m_true, l_wave, 0.f);
  __syncthreads();   // (also: every wave is done with its tiles)
  float M = -INFINITY, top = -INFINITY, l_tot = 0.f, f[NG];
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const float4 st = L.stat[rb + MT * g][rr];
    M = fmaxf(M, st.x);
    top = fmaxf(top, st.y);
  }
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const float4 st = L.stat[rb + MT * g][rr];
    f[g] = st.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((st.x - M) * LOG2E);   // (O and l are 0 with -inf)
    l_tot += st.z * f[g];
  }
  if (a.scale == 0.f) top *= 0.f;
  if (writer) {
    if (!direct) {
      a.part_s[(int64_t)h * a.slots + it.slot] = make_float4(M, top, dead ? 0.f : l_tot, 0.f);
    } else if (a.sm_max) {
      a.sm_max[h] = dead ? 0.f : top;
      a.sm_sum[h] = dead ? 0.f : l_tot * exp2f((M - top) * LOG2E);
    }
  }
  const float inv = dead ? 0.f : 1.f / l_tot;
  constexpr int NC = ON < 8 ? ON : 8;   // column tiles at a time
  float4* const part = it.part + (int64_t)rb * (D / 8) * 64 + lane;
  uint16_t* const out = a.out + (int64_t)(valid ? h : 0) * D + 4 * kg;
#pragma unroll
  for (int c = 0; c < ON; c += NC) {
    if (c > 0) lds_barrier();
    if (valid)   // (a mask: fewer lanes, fewer LDS cycles)
#pragma unroll
      for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x16& v = o[c + n];
          L.join[wave][n * 4 + g][lane] = make_float4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
        }
    lds_barrier();
    if (valid && !(dead && !direct))
#pragma unroll 2
      for (int e = grp; e < NC * 4; e += NG) {   // groups of 8 columns
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const float4 p = L.join[rb + MT * g][e][lane];
          v.x += p.x * f[g];
          v.y += p.y * f[g];
          v.z += p.z * f[g];
          v.w += p.w * f[g];
        }
        if (direct)
          *reinterpret_cast<uint2*>(out + (c * 4 + e) * 8) =
              dead ? make_uint2(0, 0) : make_uint2(pack2<IO>(v.x * inv, v.y * inv), pack2<IO>(v.z * inv, v.w * inv));
        else
          part[(c * 4 + e) * 64] = v;
      }
  }
}

template <int IO, int D>
__global__ __launch_bounds__(NWV * 64) void prefix_attn_kernel(PfxK a) {
  __shared__ __attribute__((aligned(16))) PfxLds<D> L;
  Item it;
  int mt;
  // Work-groups go round the eight XCDs, each with an L2 of its own and 32 CUs: XCD x takes an eighth of the
  // prefix items, numbered range by range (so a range's latents come from HBM once or twice, and no XCD has
  // an item more than another, which cost a round of them where whole ranges went to one: 84 us instead of 58
  // for 34 ranges of 7 tiles), then own items up to an even count: dense indexes row by row, or (joined, at
  // least eight ranges) a run of ranges per XCD.
  const int x = blockIdx.x & 7, j = blockIdx.x >> 3;
  const int np = a.p_splits * a.p_tiles, rem = np & 7, lo = np >> 3, hi = lo + (rem ? 1 : 0);
  if (j < (x < rem ? hi : lo)) {
    const int i = x * lo + min(x, rem) + j;
    const int sp = i / a.p_tiles, tile = i - sp * a.p_tiles;
    mt = a.p_mt;
    it.h0 = tile * 32 * mt;
    it.h_end = a.rows * a.n1;
    it.b = -1;
    it.seq = {0, 0, 0, 0};
    it.t_lo = sp * a.p_chunk;
    it.t_hi = sp == a.p_splits - 1 ? a.prefix : min(a.prefix, it.t_lo + a.p_chunk);
    it.slot = sp;
    it.part = a.p_part + ((int64_t)sp * a.p_blocks + tile * mt) * (D / 8) * 64;
  } else {
    int i = a.o_by_range ? x * a.per_xcd + j : j < hi ? (j - lo) * (8 - rem) + (x - rem) : (hi - lo) * (8 - rem) + (j - hi) * 8 + x;
    const int sp = i / a.o_items;
    if (sp >= a.o_splits) return;
    i -= sp * a.o_items;
    mt = a.o_mt;
    // o_tiles items a sequence, or (sequences much shorter than the longest) numbered through: those of
    // sequence b begin at row_start[b] * n1 / (32 mt) + b, which leaves each enough
    int b, n;   // the sequence, how many of its items are before this one
    if (a.o_compact) {
      auto first_item = [&](int q) { return a.row_start[q] * a.n1 / (32 * mt) + q; };
      int below = 0, above = a.batch - 1;
      while (below < above) {
        const int mid = (below + above + 1) >> 1;
        if (first_item(mid) <= i) below = mid; else above = mid - 1;
      }
      b = below;
      n = i - first_item(b);
    } else {
      b = i / a.o_tiles;
      n = i - b * a.o_tiles;
    }
    it.seq = seq_of(a, b);
    const int first = it.seq.r0 * a.n1;
    it.h_end = it.seq.r1 * a.n1;
    const int tiles = (it.h_end - first + 32 * mt - 1) / (32 * mt);
    const int tile = tiles - 1 - n;   // (causal: the longest first)
    it.h0 = first + tile * 32 * mt;
    it.b = b;
    it.t_lo = a.o_base + sp * a.o_chunk;
    it.t_hi = sp == a.o_splits - 1 ? INT_MAX : it.t_lo + a.o_chunk;
    it.slot = a.p_splits + sp;
    it.part = a.o_part + ((int64_t)sp * a.o_blocks + first / 32 + b + tile * mt) * (D / 8) * 64;
    if (a.slots == 1 && b == a.batch - 1) {   // rows behind the last sequence: zeros, by its items
      const int share = a.o_compact ? a.o_items - (i - n) : a.o_tiles;
      const int64_t end = (int64_t)a.rows * a.n1 * (D / 8);
      for (int64_t q = (int64_t)it.h_end * (D / 8) + n * (NWV * 64) + threadIdx.x; q < end; q += (int64_t)share * (NWV * 64)) {
        stg16(a.out + q * 8, make_uint4(0, 0, 0, 0));
        if (a.sm_max && q % (D / 8) == 0) a.sm_max[q / (D / 8)] = a.sm_sum[q / (D / 8)] = 0.f;
      }
    }
    if (tile < 0) return;
  }
  if (mt == 1) run_tokens<IO, D, 1>(a, it, L);
  else if (mt == 2) run_tokens<IO, D, 2>(a, it, L);
  else run_item<IO, D>(a, it, L);
}

constexpr int MAX_SLOTS = 256;

// Joins the ranges of 32 head rows: M = max m_s, out = sum O_s 2^(m_s - M) / sum l_s 2^(m_s - M); rows that
// see nothing get zeros. Bound by the partials' bytes where there are many rows, by latency where there
// are few, so the first PF ranges' partials are requested before the weights are known (a range that a row
// saw nothing of has weight 0: its partial, whatever it holds, is left out), later ones UN at a time; with
// few rows and many ranges, SG waves take every SG-th one. A wave's lanes are the 32 rows and two column
// groups of one of the D / 8 groups of 8 columns: 1 KB of a block.
template <int IO, int D, int SG>
__global__ __launch_bounds__(SG > 1 ? SG * 64 : 256) void prefix_merge_kernel(PfxK a) {
  constexpr int TPB = SG > 1 ? SG * 64 : 256;
  constexpr int LPR = TPB / 32;   // threads a row for the statistics
  constexpr int PF = 12, UN = 8;
  __shared__ float s_w[MAX_SLOTS][32];
  __shared__ float s_inv[32];
  __shared__ float4 s_acc[SG > 1 ? SG : 1][64];
  const int m_rows = a.rows * a.n1;
  const int h0 = blockIdx.x * 32;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int rr = lane & 31, kg = lane >> 5;
  const int grp = SG > 1 ? blockIdx.y : blockIdx.y * 4 + wave;   // group of 8 columns
  const int sg = SG > 1 ? wave : 0;
  // the sequences of this thread's row of the statistics and of this lane's row of the output
  const int sr = threadIdx.x / LPR, j = threadIdx.x % LPR;
  const int sh = min(h0 + sr, m_rows - 1), oh = min(h0 + rr, m_rows - 1);
  int sb = batch_guess(a, sh >> a.n1_shift), ob = batch_guess(a, oh >> a.n1_shift);
  Seq sq = seq_of(a, sb), oq = seq_of(a, ob);
  batch_fix(a, sh >> a.n1_shift, sb, sq);
  batch_fix(a, oh >> a.n1_shift, ob, oq);
  const bool live = row_limit(a, sh >> a.n1_shift, sq) > 0, o_live = row_limit(a, oh >> a.n1_shift, oq) > 0;
  const int own = oh - oq.r0 * a.n1;
  const float4* pp = a.p_part + ((int64_t)blockIdx.x * (D / 8) + grp) * 64 + lane;
  const float4* op = a.o_part + ((int64_t)(oq.r0 * a.n1 / 32 + ob + own / 32) * (D / 8) + grp) * 64 + kg * 32 + own % 32;
  const int64_t p_step = (int64_t)a.p_blocks * (D / 8) * 64, o_step = (int64_t)a.o_blocks * (D / 8) * 64;
  auto part = [&](int s) { return s < a.p_splits ? pp + s * p_step : op + (s - a.p_splits) * o_step; };
  uint4 first[PF];
#pragma unroll
  for (int i = 0; i < PF; ++i) {
    const int s = sg + i * SG;
    first[i] = ldg16_or0(o_live && s < a.slots, part(s));
  }
  {
    const float4* ps = a.part_s + (int64_t)sh * a.slots;
    float M = -INFINITY, top = -INFINITY, sum = 0.f;
    for (int s = j; s < a.slots; s += LPR) {
      const float4 st = live ? ps[s] : make_float4(0.f, 0.f, 0.f, 0.f);
      if (st.z != 0.f) {   // (NaN sums take part)
        M = fmaxf(M, st.x);
        top = fmaxf(top, st.y);
      }
    }
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) {
      M = fmaxf(M, __shfl_xor(M, o));
      top = fmaxf(top, __shfl_xor(top, o));
    }
    for (int s = j; s < a.slots; s += LPR) {
      const float4 st = live ? ps[s] : make_float4(0.f, 0.f, 0.f, 0.f);
      // (a range whose scores are all NaN has no maximum, -inf: its weight is its sum, or the NaN would be left out)
      const float w = st.z != st.z ? st.z : st.z != 0.f ? exp2f((st.x - M) * LOG2E) : 0.f;
      s_w[s][sr] = w;
      if (w != 0.f) sum += w * st.z;
    }
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if (j == 0) {
      s_inv[sr] = live ? 1.f / sum : 0.f;
      if (blockIdx.y == 0 && a.sm_max && h0 + sr < m_rows) {
        a.sm_max[sh] = live ? top : 0.f;
        a.sm_sum[sh] = live ? sum * exp2f((M - top) * LOG2E) : 0.f;
      }
    }
  }
  __syncthreads();
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float w, const uint4& v) {
    if (w != 0.f) {
      acc.x += w * __uint_as_float(v.x);
      acc.y += w * __uint_as_float(v.y);
      acc.z += w * __uint_as_float(v.z);
      acc.w += w * __uint_as_float(v.w);
    }
  };
#pragma unroll
  for (int i = 0; i < PF; ++i) {
    const int s = sg + i * SG;
    if (s < a.slots) add(s_w[s][rr], first[i]);
  }
  for (int s0 = sg + PF * SG; s0 < a.slots; s0 += SG * UN) {
    float w[UN];
    uint4 v[UN];
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const int s = s0 + i * SG;
      w[i] = s < a.slots ? s_w[s][rr] : 0.f;
      v[i] = ldg16_or0(w[i] != 0.f, part(s));
    }
#pragma unroll
    for (int i = 0; i < UN; ++i) add(w[i], v[i]);
  }
  if constexpr (SG > 1) {
    s_acc[sg][lane] = acc;
    __syncthreads();
    if (sg != 0) return;
#pragma unroll
    for (int g = 1; g < SG; ++g) {
      const float4 v = s_acc[g][lane];
      acc.x += v.x;
      acc.y += v.y;
      acc.z += v.z;
      acc.w += v.w;
    }
  }
  if (h0 + rr >= m_rows) return;
  const float inv = s_inv[rr];
  *reinterpret_cast<uint2*>(a.out + (int64_t)(h0 + rr) * D + grp * 8 + kg * 4) =
      make_uint2(pack2<IO>(acc.x * inv, acc.y * inv), pack2<IO>(acc.z * inv, acc.w * inv));
}

// How a call is cut. Lengths are what the caller expects; the kernels' ranges are right for any.
struct Cut {
  int p_mt, p_tiles, p_splits, p_chunk;
  int o_mt, o_tiles, o_splits, o_chunk, o_base;
  int slots;
};

int mt_for(int64_t head_rows) { return head_rows > 64 ? 4 : head_rows > 32 ? 2 : 1; }
int up(int x, int to) { return (x + to - 1) / to * to; }

// Microseconds of a call by a simple model of what was measured (256 CUs, one item each at a time): an item
// costs 6 (its rows' sequences, Q, first tile, ends) and, at D = 512 / 128, per 32 tokens 1.55 / 0.93 for 128
// head rows (D = 512: 1.4 where few items run, 1.9 with all CUs busy, whose clock is 2.0 GHz then), 0.95 / 0.71
// for 64, or per 128 tokens 3.7 / 3.0 for 32 (narrow latents: the tile's chain of loads, softmax and waits, not its
// products); the latents come at 4.9 TB/s; partial outputs are written at 7 TB/s,
// and the join is a launch of 6 that reads them at 6 TB/s. It is there to weigh rounds of items against
// partials: at 64 x 16 heads after 8192 tokens 16 prefix ranges take 47 us, 8 take 65 and 32 take 65 as well.
struct Model {
  int d;
  double tokens32(int mt) const {   // 32 tokens of an item
    return mt == 4 ? 0.72 + 1.62e-3 * d : mt == 2 ? 0.63 + 6.25e-4 * d : 0.6875 + 4.6e-4 * d;
  }
  double item(int mt, int tokens) const {
    const int gran = mt == 1 ? 4 * BN : BN;
    return 6.0 + tokens32(mt) * ((tokens + gran - 1) / gran * (gran / BN));
  }
};

double cut_cost(const Model& md, const Cut& c, int d, double own_tiles, int own_max, double own_mean,
                double latents_mb) {
  const double np = (double)c.p_splits * c.p_tiles;
  const double tp = c.p_splits ? md.item(c.p_mt, c.p_chunk) : 0.0;
  const double no = own_tiles * std::min((double)c.o_splits, own_mean / c.o_chunk + (c.o_splits > 1 ? 0.5 : 1.0));
  const double to = own_max > 0 ? md.item(c.o_mt, std::min(c.o_chunk, own_max)) : 3.0;
  // items past the CUs wait for whole ones, also where others end at once (18 prefix ranges instead of 16
  // in the example, 272 work-groups: 47 -> 61 us): half an item at least
  const double n = np + no, grid = np + own_tiles * c.o_splits, longest = std::max(tp, to);
  const double mean = (np * tp + no * to) / std::max(n, 1.0);
  double us = longest + (grid > 256.0 ? mean * std::max(std::max(n, 256.0) / 256.0 - 1.0, 0.45) : 0.0);
  // the later of both, and more where they are near
  const double hbm = 6.0 + latents_mb / 4.9;
  us = std::max(us, hbm) + 0.25 * std::min(us, hbm);
  if (c.slots > 1) {
    const double mb = (np * c.p_mt + no * c.o_mt) * 32.0 * d * 4.0 * 1e-6;
    us += mb / 7.0 + 6.0 + mb / 6.0;
  }
  return us;
}

// total_kv: the sum of the lengths
Cut make_cut(int batch, int rows, int n1, int d, int prefix, int max_rows, int max_kv, int64_t total_kv, int kv_splits) {
  const int64_t m = (int64_t)rows * n1;
  const double mean = (double)total_kv / batch;
  const Model md{d};
  const double latents_mb = (prefix + std::max(mean - prefix, 0.0) * batch) * (d + 64) * 2e-6;
  Cut c{}, best{};
  double least = 1e300;
  c.o_mt = mt_for((int64_t)max_rows * n1);
  c.o_tiles = (int)(((int64_t)max_rows * n1 + 32 * c.o_mt - 1) / (32 * c.o_mt));
  c.o_tiles = std::max(c.o_tiles, 1);
  const double own_tiles = (double)std::min<int64_t>((int64_t)batch * c.o_tiles, m / (32 * c.o_mt) + batch);
  auto consider = [&](int own_max, double own_mean, int o_splits) {
    c.o_splits = std::min(std::max(o_splits, 1), std::max(1, MAX_SLOTS - c.p_splits));
    c.o_chunk = up(std::max((own_max + c.o_splits - 1) / c.o_splits, 1), c.o_mt == 1 ? 4 * BN : BN);
    c.o_splits = std::max(1, (own_max + c.o_chunk - 1) / c.o_chunk);
    c.slots = c.p_splits + c.o_splits;
    const double us = cut_cost(md, c, d, own_tiles, own_max, own_mean, latents_mb);
    if (us < least) least = us, best = c;
  };
  auto more = [](int s) { return s < 24 ? 1 : s < 48 ? 4 : 8; };
  // joined: each tile over the prefix and its own tokens
  c.p_mt = mt_for(m);
  c.o_base = 0;
  for (int s = kv_splits > 0 ? kv_splits : 1; s <= (kv_splits > 0 ? kv_splits : 192); s += more(s)) consider(max_kv, mean, s);
  if (prefix == 0) return best;
  // split: the prefix for all head rows at once, in ranges
  const int own = std::max(max_kv - prefix, 0);
  const double own_mean = std::max(mean - prefix, 0.0);
  c.o_base = prefix;
  c.p_tiles = (int)((m + 32 * c.p_mt - 1) / (32 * c.p_mt));
  const int gran = c.p_mt == 1 ? 4 * BN : BN;
  for (int s = kv_splits > 0 ? kv_splits : 1; s <= (kv_splits > 0 ? kv_splits : 192); s += more(s)) {
    c.p_chunk = up((prefix + s - 1) / s, gran);
    c.p_splits = (prefix + c.p_chunk - 1) / c.p_chunk;
    // own ranges as long as a prefix range takes, or one
    const double fit = md.item(c.p_mt, c.p_chunk) - 6.0;
    const double per = md.tokens32(c.o_mt) / BN;
    consider(own, own_mean, (int)std::ceil(own * per / std::max(fit, per * BN)));
    if (c.o_splits > 1) consider(own, own_mean, 1);
    if (s > 1 && c.p_chunk == gran) break;
  }
  return best;
}

template <int IO>
hipError_t launch_io(const PfxK& k, int d, hipStream_t s) {
  const int64_t items = 8 * (int64_t)k.per_xcd;
  const int64_t m = (int64_t)k.rows * k.n1;
  const unsigned blocks = (unsigned)((m + 31) / 32);
  // Few rows: eight waves share a row group's ranges (a work-group a group of 8 columns), up to three such work-groups a
  // CU. Calls of 16 heads, us with one / eight waves a range group: D = 512, 4 sequences, 17 ranges 20.8 / 19.2, 129: 49.7
  // / 32; 16 sequences, 9: 18.4 / 18.3, 104: 56.3 / 48.6; 24 (768 work-groups), 12: 22.9 / 23.2, 70: 58.0 / 55.7; 32: 12:
  // 24.0 / 26.1, 33: 38.5 / 41.9. D = 128, 40, 23: 18.5 / 16.8; 64 (512), 12: 15.7 / 15.6, 25: 28.8 / 27.4; 128, 17: 39.6
  // / 41.7. Up to eight ranges it makes no difference with few rows (4 sequences, 7: 18.0 / 17.8) and costs with more
  // (24, 5: 17.9 / 19.4).
  const bool wide = k.slots > 8 && blocks * (d / 8) <= 768;
#define DSA_PFX(DD)                                                                                               \
  hipLaunchKernelGGL((prefix_attn_kernel<IO, DD>), dim3((unsigned)items), dim3(NWV * 64), 0, s, k);                \
  if (k.slots > 1 && wide)                                                                                         \
    hipLaunchKernelGGL((prefix_merge_kernel<IO, DD, 8>), dim3(blocks, DD / 8), dim3(512), 0, s, k);                \
  else if (k.slots > 1)                                                                                            \
    hipLaunchKernelGGL((prefix_merge_kernel<IO, DD, 1>), dim3(blocks, DD / 32), dim3(256), 0, s, k)
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

// Blocks of 32 head rows: the prefix's, of whole tiles, and the sequences' own, each from a block of its own
int prefix_blocks(const Cut& c) { return c.p_tiles * c.p_mt; }
int own_blocks(int batch, int64_t m) { return (int)(m / 32) + batch + 1; }
size_t block_bytes(int d) { return (size_t)32 * d * sizeof(float); }
size_t workspace_bytes(const Cut& c, int batch, size_t m, int d) {
  if (c.slots == 1) return 0;
  return align256(m * c.slots * sizeof(float4)) +
         ((size_t)c.p_splits * prefix_blocks(c) + (size_t)c.o_splits * own_blocks(batch, m)) * block_bytes(d);
}
}  // namespace
}  // namespace dsa

using namespace dsa;

size_t prefix_attn_workspace_bytes(int batch, int rows, int n1, int d, int prefix, int max_rows, int max_kv, int64_t total_kv,
                                   int kv_splits) {
  return workspace_bytes(make_cut(batch, rows, n1, d, prefix, max_rows, max_kv, total_kv, kv_splits), batch, (size_t)rows * n1, d);
}

// (the search for the cut takes 1 to 4 us, so that a call makes one: it checks the workspace too)
hipError_t launch_prefix_attn(const PrefixArgs& a, size_t* lacking, hipStream_t s) {
  const Cut c = make_cut(a.batch, a.total_rows, a.n1, a.d, a.prefix, a.max_rows, a.max_kv, a.total_kv, a.kv_splits);
  const size_t need = workspace_bytes(c, a.batch, (size_t)a.total_rows * a.n1, a.d);
  *lacking = need > 0 && (!a.ws || a.ws_bytes < need || ((uintptr_t)a.ws & 15) != 0) ? need : 0;
  if (*lacking) return hipSuccess;
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
  k.p_blocks = prefix_blocks(c);
  k.o_blocks = own_blocks(a.batch, (int64_t)a.total_rows * a.n1);
  k.p_part = c.slots > 1 ? (float4*)((char*)a.ws + align256((size_t)a.total_rows * a.n1 * c.slots * sizeof(float4))) : nullptr;
  k.o_part = c.slots > 1 ? k.p_part + (size_t)c.p_splits * k.p_blocks * (block_bytes(a.d) / sizeof(float4)) : nullptr;
  while ((1 << k.n1_shift) < a.n1) ++k.n1_shift;
  k.p_mt = c.p_mt;
  k.p_tiles = c.p_tiles;
  k.p_splits = c.p_splits;
  k.p_chunk = c.p_chunk;
  k.o_mt = c.o_mt;
  k.o_tiles = c.o_tiles;
  k.o_splits = c.o_splits;
  k.o_chunk = c.o_chunk;
  k.o_base = c.o_base;
  k.slots = c.slots;
  const int64_t even = (int64_t)a.batch * c.o_tiles, through = (int64_t)a.total_rows * a.n1 / (32 * c.o_mt) + a.batch;
  // Numbering through costs a search, and items that are not there cost a work-group each. One prompt and up to 64 of an
  // eighth of it (16 heads, D = 512), us without / with it: 1.45 times the items 22.8 / 23.0, 1.7: 37.7 / 36.7, 2.9: 28.9 /
  // 27.5, 4.8: 74 / 39, 5.9: 215 / 58.
  k.o_compact = even > through + through / 2;
  const int64_t own = k.o_compact ? through : even, all = (int64_t)c.p_splits * c.p_tiles + own * c.o_splits;
  if (all >= (1 << 24) - 8) return hipErrorInvalidConfiguration;   // 2^32 threads, before anything is launched
  k.o_items = (int)own;
  k.per_xcd = (int)((all + 7) / 8);
  k.o_by_range = c.p_splits == 0 && c.o_splits >= 8;
  return a.io == DSA_DTYPE_BF16 ? launch_io<IO_BF16>(k, a.d, s) : launch_io<IO_F16>(k, a.d, s);
}
