// What the dense attention's forward and backward kernels share: sequences and their masks, tiles of keys,
// values, queries or output gradients in LDS, and the reading of MFMA operands from them.
#pragma once

#include <climits>
#include <cmath>

#include "dsa_common.hpp"

namespace dsa {

constexpr float LOG2E = 1.4426950408889634f;

// A tensor [rows, heads, width], or [sequences, rows, heads, width], by strides in elements
struct Rows {
  const uint16_t* p;
  int64_t row, head, batch;
};

// Lengths of a call. Sequence b's query rows begin at row_start[b], its keys at key_start[b]; sequence `batch` is
// what lies behind the last one, nothing of which is seen.
struct Lens {
  const int32_t* row_start;
  const int32_t* key_start;
  const int32_t* act_q;
  const int32_t* act_k;
  int batch, rows, keys, mode;   // rows, keys: of the tensors
  int apart;                     // operands' sequences lie batch strides apart, else their rows follow each other
};
// where the rows of sequence b, whose first one is row r0 of all, begin in an operand
__device__ __forceinline__ const uint16_t* first_of(const Lens& l, const Rows& x, int b, int r0) {
  return x.p + (l.apart ? (int64_t)b * x.batch : (int64_t)r0 * x.row);
}
struct Seq {
  int r0, rows;   // first query row, rows that belong to it (act_q of them are queries)
  int k0, keys;
  int aq, ak;
};
__device__ __forceinline__ Seq seq_of(const Lens& l, int b) {
  Seq q;
  q.r0 = l.row_start[b];
  q.k0 = l.key_start[b];
  const bool tail = b >= l.batch;
  q.rows = (tail ? l.rows : l.row_start[b + 1]) - q.r0;
  q.keys = (tail ? l.keys : l.key_start[b + 1]) - q.k0;
  q.aq = tail ? 0 : min(l.act_q[b], q.rows);
  q.ak = tail ? 0 : min(l.act_k[b], q.keys);
  return q;
}
// how many of its tokens query s of a sequence sees
__device__ __forceinline__ int limit_of(const Lens& l, const Seq& q, int s) {
  if (s >= q.aq) return 0;
  return l.mode == 0 ? q.ak : max(0, q.ak - q.aq + s + 1);
}
// the first query that sees token t (aq if none does)
__device__ __forceinline__ int first_query(const Lens& l, const Seq& q, int t) {
  if (t >= q.ak) return q.aq;
  return l.mode == 0 ? 0 : min(q.aq, max(0, t - (q.ak - q.aq)));
}

// ---------------------------------------------------------------- tiles in LDS
// Rows of RB = 256 or 128 bytes, unpadded, so that direct-to-LDS loads fill them (a wave's 64 lanes 1 KB in a row). A
// row's 16-byte chunks are permuted: c lies at c ^ swizzle(row). Operand reads (16 rows, one chunk) and
// transposed reads (4 rows, 64 bytes) both touch every bank once. Rows of 128 bytes share a line of the banks by twos.
__host__ __device__ constexpr int line_swz(int l) { return ((l & 1) << 2) | (l & 2) | ((l >> 2) & 1); }
template <int RB>
__device__ __forceinline__ constexpr uint32_t tile_off(int t, int c) {
  if constexpr (RB == 256) return (uint32_t)(t * 256 + ((c ^ kv_swz(t & 15)) << 4));
  else return (uint32_t)(t * 128 + ((c ^ line_swz((t >> 1) & 7)) << 4));
}

// One wave's share of the loads of a tile of BN rows by NW waves: CNT loads; load j covers the rows STEP j + first ..
template <int RB, int BN, int NW> struct Share {
  static constexpr int RPL = 1024 / RB;          // rows a load
  static constexpr int STEP = RPL * NW;
  static constexpr int CNT = BN / STEP;
  static_assert(BN % STEP == 0 && STEP % 16 == 0, "every load of a wave has the same permutation");
  int row;        // this lane's row of load 0
  uint32_t col;   // byte of its chunk in the row
  __device__ __forceinline__ Share(int wave, int lane) {
    row = wave * RPL + lane / (RB / 16);
    const int c = lane & (RB / 16 - 1);
    col = (uint32_t)((RB == 256 ? c ^ kv_swz(row & 15) : c ^ line_swz((row >> 1) & 7)) << 4);
  }
};

// 16-byte direct-to-LDS load as lds_dma16_sbase_untracked, to LDS address lds + OFF: the sum goes into M0 in one
// instruction
template <int OFF>
__device__ __forceinline__ void lds_dma16_at(const void* sbase, uint32_t voff, uint32_t lds) {
  asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :
               : "v"(voff), "s"(sbase), "s"(lds), "n"(OFF)
               : "memory", "m0", "scc");
}

// p, which is the same in all lanes, in scalar registers
__device__ __forceinline__ const char* uniform(const char* p) {
  const uint64_t v = (uint64_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return (const char*)(lo | (uint64_t)hi << 32);
}

// The loads of one array's tiles, one tile after another: this wave's share as offsets from a base that moves from
// tile to tile. Rows past the last repeat it (they are masked); as only the last tile has any, the offsets are
// made anew for that one and stay.
template <int RB, int BN, int NW> struct Stream {
  using Sh = Share<RB, BN, NW>;
  Sh sh;
  const char* base;      // of the next tile
  uint32_t row_bytes;
  uint32_t lds;          // this wave's first place in buffer 0
  uint32_t off[Sh::CNT];
  __device__ __forceinline__ Stream(const uint16_t* p, uint32_t row_bytes_, const void* buf, int wave, int lane)
      : sh(wave, lane), base(reinterpret_cast<const char*>(p)), row_bytes(row_bytes_), lds(lds_addr(buf) + wave * 1024) {}
  __device__ __forceinline__ void aim(int last) {   // last: the last row there is, from the tile's first
#pragma unroll
    for (int i = 0; i < Sh::CNT; ++i) off[i] = (uint32_t)min(i * Sh::STEP + sh.row, last) * row_bytes + sh.col;
  }
  template <int I> __device__ __forceinline__ void load(uint32_t buf_bytes) const {
    lds_dma16_at<I * NW * 1024>(base, off[I], lds + buf_bytes);
  }
};

// Token order of the S tiles: with row m of the operand at token tk(m), a lane's 16 accumulators of a 32-row tile
// are tokens 16 (i / 8) + 8 (lane / 32) + i % 8, the order in which the next product takes them as an operand.
__device__ __forceinline__ int s_row(int m) { return 16 * (m >> 4) + 8 * ((m >> 2) & 1) + 4 * ((m >> 3) & 1) + (m & 3); }
__device__ __forceinline__ int s_token(int i, int kg) { return 16 * (i >> 3) + 8 * kg + (i & 7); }

// Values that are not finite become zeros in this wave's share of a tile (its loads have landed); returns the rows
// (bit) that held one.
template <int IO, int RB, int BN, int NW>
__device__ __forceinline__ uint64_t clean_share(uint32_t tile, int wave, int lane) {
  static_assert(BN <= 64, "a bit a row");
  using Sh = Share<RB, BN, NW>;
  constexpr uint32_t EXP = IO == IO_BF16 ? 0x7F80u : 0x7C00u;
  uint64_t bad = 0;
#pragma unroll 1
  for (int j = 0; j < Sh::CNT; ++j) {
    const uint32_t at = tile + (uint32_t)((j * NW + wave) * 1024 + lane * 16);
    const uint4 v = lds_read16_at(at);
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if ((w[i] & EXP) == EXP) w[i] &= 0xFFFF0000u, any = true;
      if (((w[i] >> 16) & EXP) == EXP) w[i] &= 0xFFFFu, any = true;
    }
    if (any) *(__attribute__((address_space(3))) u32x4v*)(uintptr_t)at = __builtin_bit_cast(u32x4v, make_uint4(w[0], w[1], w[2], w[3]));
    const uint64_t lanes = __builtin_amdgcn_ballot_w64(any);
    if (lanes) {
#pragma unroll
      for (int r = 0; r < Sh::RPL; ++r)
        if ((lanes >> (r * (RB / 16))) & ((1ull << (RB / 16)) - 1)) bad |= 1ull << (j * Sh::STEP + wave * Sh::RPL + r);
    }
  }
  return bad;
}

// 32x32x16 chains whose accumulators stay in VGPRs (their results go to the VALU) and whose second operand, loaded
// once, lies in AGPRs. The compiler does not see these as MFMAs: the last ones of a chain end with the wait states that a
// VALU read of their results needs (8 passes: 12; 16 are waited), in the same statement, as the compiler may copy an
// accumulator between two of them.
template <int IO, bool FIRST>
__device__ __forceinline__ void mfma32_va(f32x16& c, uint4 a, uint4 b) {
  const i32x4v av = __builtin_bit_cast(i32x4v, a), bv = __builtin_bit_cast(i32x4v, b);
  if constexpr (IO == IO_BF16 && FIRST) asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(c) : "v"(av), "a"(bv));
  else if constexpr (IO == IO_BF16) asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(av), "a"(bv));
  else if constexpr (FIRST) asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, 0" : "=&v"(c) : "v"(av), "a"(bv));
  else asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+v"(c) : "v"(av), "a"(bv));
}
template <int IO>
__device__ __forceinline__ void mfma32_va_last(f32x16& c, uint4 a, uint4 b) {
  const i32x4v av = __builtin_bit_cast(i32x4v, a), bv = __builtin_bit_cast(i32x4v, b);
  if constexpr (IO == IO_BF16) asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0\n\ts_nop 15" : "+v"(c) : "v"(av), "a"(bv));
  else asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0\n\ts_nop 15" : "+v"(c) : "v"(av), "a"(bv));
}
// the last step of two chains with the same first operand
template <int IO>
__device__ __forceinline__ void mfma32_va_last2(f32x16& c0, f32x16& c1, uint4 a, uint4 b0, uint4 b1) {
  const i32x4v av = __builtin_bit_cast(i32x4v, a), v0 = __builtin_bit_cast(i32x4v, b0), v1 = __builtin_bit_cast(i32x4v, b1);
  if constexpr (IO == IO_BF16)
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %2, %3, %0\n\tv_mfma_f32_32x32x16_bf16 %1, %2, %4, %1\n\ts_nop 15"
                 : "+v"(c0), "+v"(c1) : "v"(av), "a"(v0), "a"(v1));
  else
    asm volatile("v_mfma_f32_32x32x16_f16 %0, %2, %3, %0\n\tv_mfma_f32_32x32x16_f16 %1, %2, %4, %1\n\ts_nop 15"
                 : "+v"(c0), "+v"(c1) : "v"(av), "a"(v0), "a"(v1));
}

// the last steps of two chains
template <int IO>
__device__ __forceinline__ void mfma32_va_end2(f32x16& c0, uint4 a0, uint4 b0, f32x16& c1, uint4 a1, uint4 b1) {
  const i32x4v p0 = __builtin_bit_cast(i32x4v, a0), p1 = __builtin_bit_cast(i32x4v, a1);
  const i32x4v v0 = __builtin_bit_cast(i32x4v, b0), v1 = __builtin_bit_cast(i32x4v, b1);
  if constexpr (IO == IO_BF16)
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %2, %4, %0\n\tv_mfma_f32_32x32x16_bf16 %1, %3, %5, %1\n\ts_nop 15"
                 : "+v"(c0), "+v"(c1) : "v"(p0), "v"(p1), "a"(v0), "a"(v1));
  else
    asm volatile("v_mfma_f32_32x32x16_f16 %0, %2, %4, %0\n\tv_mfma_f32_32x32x16_f16 %1, %3, %5, %1\n\ts_nop 15"
                 : "+v"(c0), "+v"(c1) : "v"(p0), "v"(p1), "a"(v0), "a"(v1));
}
// the same with operands that lie in VGPRs, where the AGPRs are full
template <int IO>
__device__ __forceinline__ void mfma32_vv(f32x16& c, uint4 a, uint4 b) {
  const i32x4v av = __builtin_bit_cast(i32x4v, a), bv = __builtin_bit_cast(i32x4v, b);
  if constexpr (IO == IO_BF16) asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(av), "v"(bv));
  else asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+v"(c) : "v"(av), "v"(bv));
}
template <int IO>
__device__ __forceinline__ void mfma32_vv_va_end2(f32x16& c0, uint4 a0, uint4 b0, f32x16& c1, uint4 a1, uint4 b1) {
  const i32x4v p0 = __builtin_bit_cast(i32x4v, a0), p1 = __builtin_bit_cast(i32x4v, a1);
  const i32x4v v0 = __builtin_bit_cast(i32x4v, b0), v1 = __builtin_bit_cast(i32x4v, b1);
  if constexpr (IO == IO_BF16)
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %2, %4, %0\n\tv_mfma_f32_32x32x16_bf16 %1, %3, %5, %1\n\ts_nop 15"
                 : "+v"(c0), "+v"(c1) : "v"(p0), "v"(p1), "v"(v0), "a"(v1));
  else
    asm volatile("v_mfma_f32_32x32x16_f16 %0, %2, %4, %0\n\tv_mfma_f32_32x32x16_f16 %1, %3, %5, %1\n\ts_nop 15"
                 : "+v"(c0), "+v"(c1) : "v"(p0), "v"(p1), "v"(v0), "a"(v1));
}
// v in AGPRs from here on
__device__ __forceinline__ uint4 in_agprs(uint4 u) {
  i32x4v v = __builtin_bit_cast(i32x4v, u);
  asm volatile("" : "+a"(v));
  return __builtin_bit_cast(uint4, v);
}

// Addresses of a lane's operand fragments in a tile: those of one row (tk) or of one group of rows (transposed) differ by
// an exclusive or of constants in the chunk bits. Kept in registers and moved to another buffer once a tile, so that
// halves of a tile and other arrays of the same layout are constant offsets.
template <int RB> struct OpAddr {
  uint32_t a[RB / 32];
  __device__ __forceinline__ void point(uint32_t tile, uint32_t lane) {
#pragma unroll
    for (int j = 0; j < RB / 32; ++j) {
      a[j] = tile + (lane ^ (j << 5));
      asm volatile("" : "+v"(a[j]));
    }
  }
};
template <int RB> struct TrAddr {
  uint32_t lo[RB / 64], hi[RB / 64];
  __device__ __forceinline__ void point(uint32_t tile, uint32_t lane_lo, uint32_t lane_hi) {
#pragma unroll
    for (int c = 0; c < RB / 64; ++c) {
      lo[c] = tile + (lane_lo ^ (c << 6));
      hi[c] = tile + (lane_hi ^ (c << 6));
      asm volatile("" : "+v"(lo[c]), "+v"(hi[c]));
    }
  }
  // column tile c of the 16 rows at byte offset off
  __device__ __forceinline__ uint4 frag(int c, int off) const {
    const uint2 l = ds_read_tr_at(lo[c] + off), h = ds_read_tr_at(hi[c] + off);
    return make_uint4(l.x, l.y, h.x, h.y);
  }
};

// o *= f on an accumulator element in an AGPR, which the VALU cannot use directly
__device__ __forceinline__ float agpr_scale(float o, float f) {
  float t;
  asm volatile("v_accvgpr_read_b32 %1, %0\n\tv_mul_f32 %1, %1, %2\n\tv_accvgpr_write_b32 %0, %1"
               : "+a"(o), "=&v"(t)
               : "v"(f));
  return o;
}

__device__ __forceinline__ uint4 flipped(uint4 v, uint32_t f) { return make_uint4(v.x ^ f, v.y ^ f, v.z ^ f, v.w ^ f); }

// v_max3 without the quieting of each operand that fmaxf needs (a NaN score reaches the output
// through its exponential either way)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// The four groups of four accumulators of a 32-column tile, packed, exchanged between lane halves: lanes 0-31
// then hold columns [0, 8) and [16, 24), the others [8, 16) and [24, 32), each 16 bytes.
template <int IO>
__device__ __forceinline__ void pack_tile(const f32x16& v, float f, uint4 (&out)[2]) {
  uint32_t d[4][2];
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    d[g][0] = pack2<IO>(v[4 * g] * f, v[4 * g + 1] * f);
    d[g][1] = pack2<IO>(v[4 * g + 2] * f, v[4 * g + 3] * f);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    swap_halves(d[0][j], d[1][j]);
    swap_halves(d[2][j], d[3][j]);
  }
  out[0] = make_uint4(d[0][0], d[0][1], d[1][0], d[1][1]);
  out[1] = make_uint4(d[2][0], d[2][1], d[3][0], d[3][1]);
}

// A launch has fewer than 2^32 threads
constexpr int64_t MAX_THREADS = 1ll << 32;

// Work-groups of a launch: tiles of rows of every sequence and key head. Even numbering, levels of one tile of
// each (the last, which see most, first); or numbered through, where sequences are much shorter than the longest:
// those of sequence b begin at start(b) * per / tile + b, which leaves each enough.
struct Tiles {
  int seqs, heads;       // sequences (with what lies behind the last), key heads
  int even;              // tiles of the longest, 0: numbered through
};
// Work-group i's sequence and key head within its level. Work-groups go to the 8 XCDs in turn, and there to groups of CUs
// in turn, so a number of pairs that 8 or 32 divides gives the same CUs the same pairs in every level, long and short ones
// alike: levels are turned, by 8 (a key head's tiles stay on one XCD, whose L2 they share) or, as ranges share nothing, by one.
// Samples of 4093 and 2100, 16 heads of 128 + 64: forward 161 -> 141 us, backward (without sum P K) 548 -> 443.
__device__ __forceinline__ int pair_of(int i, int level, int pairs, int splits) {
  return (int)(((uint32_t)(i - level * pairs) + (uint32_t)level * (splits > 1 ? 1u : 8u)) % (uint32_t)pairs);
}

}  // namespace dsa
