// Rotary positions and the appends to the paged caches, for gfx950.
//
// Rotation by position p of a pair (a, b) with inverse frequency f: theta = p f,
// (a cos theta - b sin theta, a sin theta + b cos theta). The gradient of a rotation is the
// rotation back (theta negated). Pairs are neighbours (2 i, 2 i + 1) or half the rotary width
// apart (i, i + R / 2); with several position axes (time, height, width), consecutive runs of
// pairs take their position from one axis each.
//
// All kernels here are bound by memory (6 operations per pair), so each value is read once and
// written once with 16-byte accesses. What is worth computing once is the angle: it needs 64 bits
// (position 10^5 times a frequency of 1 leaves 2^-7 of a radian in 32-bit arithmetic), so a
// work-group turns its tokens' angles into a table of (cos, sin) in LDS, shared by all heads.
#include <algorithm>
#include <cstring>

#include "elements.hpp"

namespace dsa {
namespace {

constexpr int TPB = 256;
constexpr double INV_2PI = 0.15915494309189533577;

// A launch holds fewer than 2^32 threads in x: work-groups past GRID_X of them go on in z. (Rows end 4096 short of
// 2^31, so that the last group's row numbers do not overflow: the entries refuse more.)
constexpr int GRID_X = 1 << 23;
__device__ __forceinline__ int group_id() { return (int)blockIdx.z * GRID_X + (int)blockIdx.x; }
dim3 grid_of(int64_t groups, unsigned y) {
  return dim3((unsigned)std::min<int64_t>(groups, GRID_X), y, (unsigned)((groups + GRID_X - 1) / GRID_X));
}

// Rows of a [batch, rows_per_batch, heads, width] view: elements between them
struct View {
  int64_t batch, row, head;
  int rows_per_batch;
};
__device__ __forceinline__ int64_t row_offset(const View& v, int r) {
  if (v.batch == v.row * v.rows_per_batch) return r * v.row;   // evenly spaced rows: no division
  const int b = r / v.rows_per_batch;
  return b * v.batch + (r - b * v.rows_per_batch) * v.row;
}

// Which axis each pair belongs to: axis a takes the pairs [end[a-1], end[a])
struct Axes {
  int n;
  int end[4];
};
struct Positions {
  const void* p;   // [axes, rows], int32 or int64; NULL: the caller's own
  int wide;        // int64
  int rows;
  Axes axes;
};
__device__ __forceinline__ int64_t position_of(const Positions& ps, int row, int pair) {
  int a = 0;
#pragma unroll
  for (int k = 0; k < 3; ++k) a += (k + 1 < ps.axes.n && pair >= ps.axes.end[k]) ? 1 : 0;
  const int64_t at = (int64_t)a * ps.rows + row;
  return ps.wide ? reinterpret_cast<const int64_t*>(ps.p)[at] : (int64_t) reinterpret_cast<const int32_t*>(ps.p)[at];
}

// (cos, sin) of position * frequency. Turns in 64 bits, less the whole ones: what is left, in
// [-1/2, 1/2], keeps 24 bits, so the angle is as good as 32-bit cos and sin are.
__device__ __forceinline__ float2 cos_sin(int64_t pos, float freq) {
  double turns = (double)pos * ((double)freq * INV_2PI);
  turns -= rint(turns);
  float s, c;
  sincospif(2.f * (float)turns, &s, &c);
  return make_float2(c, s);
}

// ------------------------------------------------------------------ rotary
struct RotaryK {
  const void* x;
  void* out;       // contiguous
  View view;
  Positions pos;
  const float* freq;
  int rows, heads, width, start, rdim, inverse;
  int uph;         // units per head
  uint32_t uph_magic;   // ceil(2^32 / uph)
  int group;       // rows per work-group
};

// A unit is what one thread moves at a time: V elements (INTER, and those that do not turn), or
// the two groups of V elements whose pairs are half the rotary width apart. V = 1: any alignment
// and any even rotary width (INTER: the two elements of a pair).
// A work-group takes `group` whole rows where a row has fewer units than threads, else
// UPT * TPB units of one row (8192 rows of 128 heads of 64, bf16: 50.7 us a call, 5.3 TB/s).
template <int IO, int V, bool INTER, int UPT>
__global__ __launch_bounds__(TPB) void rotary_kernel(RotaryK a) {
  using T = typename Elem<IO>::T;
  constexpr bool TWO = !INTER || V == 1;            // a rotating unit has two parts
  extern __shared__ float2 tab[];                   // [group][rdim / 2]
  const int half = a.rdim / 2;
  const int upr = a.heads * a.uph;
  if ((int64_t)group_id() * a.group >= a.rows) return;   // (of the last z, the whole group)
  const int r0 = group_id() * a.group;
  const int nrot = V == 1 ? half : INTER ? a.rdim / V : half / V;   // rotating units of a head
  const T* x = reinterpret_cast<const T*>(a.x);
  T* out = reinterpret_cast<T*>(a.out);

  float v0[UPT][V], v1[UPT][V];
  int64_t src[UPT];
  // where the unit's second part lies (elements)
  const int second = V == 1 && INTER ? 1 : half;
  int lrow[UPT], unit[UPT];
  bool ok[UPT];
#pragma unroll
  for (int i = 0; i < UPT; ++i) {
    int u = (int)blockIdx.y * (TPB * UPT) + i * TPB + (int)threadIdx.x;
    lrow[i] = 0;
    if (a.group > 1) {
      lrow[i] = u / upr;
      u -= lrow[i] * upr;
    }
    ok[i] = lrow[i] < a.group && r0 + lrow[i] < a.rows && u < upr;
    const int h = a.uph == 1 ? u : (int)__umulhi((uint32_t)u, a.uph_magic);
    const int j = u - h * a.uph;
    unit[i] = j;
    int e;   // first element of the unit in the head
    if (j < nrot) e = a.start + (V == 1 && INTER ? 2 * j : j * V);
    else {
      e = (j - nrot) * V;
      if (e >= a.start) e += a.rdim;
    }
    src[i] = (int64_t)h * a.view.head + e;
    if (ok[i]) {
      const T* p = x + row_offset(a.view, r0 + lrow[i]) + src[i];
      load_vec<IO, V>(p, v0[i]);
      if (TWO && j < nrot) load_vec<IO, V>(p + second, v1[i]);
    }
    src[i] = ((int64_t)(r0 + lrow[i]) * a.heads + h) * a.width + e;
  }
  // the table, while the loads are under way
  for (int i = threadIdx.x; i < a.group * half; i += TPB) {
    const int lr = i / half, pair = i - lr * half;
    if (r0 + lr < a.rows) {
      float2 cs = cos_sin(position_of(a.pos, r0 + lr, pair), a.freq[pair]);
      if (a.inverse) cs.y = -cs.y;
      tab[i] = cs;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < UPT; ++i) {
    if (!ok[i]) continue;
    T* p = out + src[i];
    if (unit[i] >= nrot) {
      store_vec<IO, V>(p, v0[i]);
      continue;
    }
    const float2* t = tab + lrow[i] * half;
    if constexpr (TWO) {
      t += unit[i] * V;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float x0 = v0[i][e], x1 = v1[i][e];
        v0[i][e] = x0 * t[e].x - x1 * t[e].y;
        v1[i][e] = x0 * t[e].y + x1 * t[e].x;
      }
      store_vec<IO, V>(p, v0[i]);
      store_vec<IO, V>(p + second, v1[i]);
    } else {
      t += unit[i] * (V / 2);
#pragma unroll
      for (int e = 0; e < V / 2; ++e) {
        const float x0 = v0[i][2 * e], x1 = v0[i][2 * e + 1];
        v0[i][2 * e] = x0 * t[e].x - x1 * t[e].y;
        v0[i][2 * e + 1] = x0 * t[e].y + x1 * t[e].x;
      }
      store_vec<IO, V>(p, v0[i]);
    }
  }
}

// (rows of a single batch are evenly spaced, whatever its stride)
View make_view(int64_t batch, int64_t row, int64_t head, int rows_per_batch, int rows) {
  return {rows <= rows_per_batch ? row * rows_per_batch : batch, row, head, rows_per_batch};
}

Positions make_positions(const void* p, int wide, int rows, int axes, const int32_t* sections, int pairs) {
  Positions ps{p, wide, rows, {axes, {pairs, pairs, pairs, pairs}}};
  int end = 0;
  for (int i = 0; i < axes && sections; ++i) ps.axes.end[i] = end += sections[i];
  return ps;
}

template <int IO, int V, bool INTER>
hipError_t launch_rotary_v(RotaryK k, hipStream_t s) {
  const int half = k.rdim / 2;
  k.uph = (k.width - k.rdim) / V + (V == 1 ? half : INTER ? k.rdim / V : half / V);
  k.uph_magic = (uint32_t)(((1ull << 32) + k.uph - 1) / k.uph);
  const int upr = k.heads * k.uph;
  k.group = upr >= TPB ? 1 : TPB / upr;
  const size_t lds = (size_t)k.group * half * sizeof(float2);
  const int64_t groups = ((int64_t)k.rows + k.group - 1) / k.group;
  // Four units a thread, 64 bytes in flight each, for 2^24 units or more of 16-bit neighbours (bf16, inputs from HBM,
  // one unit's time first): rows of 128 heads of 64, 16,384: 103 -> 101 us, 32,768: 197 -> 190; of 128, 8192: 103.4 ->
  // 102.4, 32,768: 395 -> 375. Below that they lose (4096 rows of 64: 28.5 -> 29.7), and so they do with pairs half a
  // width apart (16,384: 101 -> 104) and in fp32 (16,384: 194 -> 201).
  if constexpr (INTER && V == 8) {
    if (upr >= 4 * TPB && (int64_t)k.rows * upr >= 1 << 24) {
      const dim3 grid = grid_of(groups, (upr + 4 * TPB - 1) / (4 * TPB));
      hipLaunchKernelGGL((rotary_kernel<IO, V, INTER, 4>), grid, dim3(TPB), lds, s, k);
      return hipGetLastError();
    }
  }
  const dim3 grid = grid_of(groups, upr >= TPB ? (upr + TPB - 1) / TPB : 1);
  hipLaunchKernelGGL((rotary_kernel<IO, V, INTER, 1>), grid, dim3(TPB), lds, s, k);
  return hipGetLastError();
}

template <int IO>
hipError_t launch_rotary_io(const RotaryK& k, bool inter, hipStream_t s) {
  using T = typename Elem<IO>::T;
  constexpr int V = Elem<IO>::V;
  // 16-byte accesses: every row, head and unit starts on a 16-byte border
  const bool vec = ((uintptr_t)k.x & 15) == 0 && ((uintptr_t)k.out & 15) == 0 && k.width % V == 0 && k.start % V == 0 &&
                   k.rdim % (2 * V) == 0 && (k.view.batch * (int64_t)sizeof(T)) % 16 == 0 &&
                   (k.view.row * (int64_t)sizeof(T)) % 16 == 0 && (k.view.head * (int64_t)sizeof(T)) % 16 == 0;
  if (vec) return inter ? launch_rotary_v<IO, V, true>(k, s) : launch_rotary_v<IO, V, false>(k, s);
  return inter ? launch_rotary_v<IO, 1, true>(k, s) : launch_rotary_v<IO, 1, false>(k, s);
}

// Each packed row's place in its sequence (0 for rows behind the last): what a prefill turns its rows by. Made
// here from the sequences' starts, as a list of them on the host took 0.9 ms for 8192 rows and a copy that
// waits for the stream.
__global__ __launch_bounds__(TPB) void row_positions_kernel(const int32_t* row_start, int batch, int rows, int32_t* positions) {
  const int64_t at = (int64_t)blockIdx.x * TPB + threadIdx.x;
  if (at >= rows) return;
  const int r = (int)at, b = batch_of_row(row_start, batch, r);
  positions[r] = r < row_start[b + 1] ? r - row_start[b] : 0;
}

// ------------------------------------------------------------------ appends
// A work-group takes NTOK tokens: one thread each finds its token's place in the cache, all of them
// fill the table of angles, and the tokens' vectors are normed, rotated and stored, LPV lanes of 8
// elements to a vector. A decode step's few tokens wait for a chain of memory accesses: so the vectors,
// the norm's weights, the frequencies and the lengths (of the sequence that evenly split ones give) are
// all requested first, and only the block table is left behind them.
// Tokens a work-group: 4 up to this many, else 8. Launches of a replayed graph, four sequences, us with 4 / 8 tokens,
// latents of 512, of 128, and keys of two heads of 128: 256 tokens 4.3 / 4.9, 4.0 / 4.1, 5.4 / 5.6; 2048: 4.6 / 5.2,
// 4.3 / 4.2, 5.8 / 5.7; 4096: 5.1 / 5.7, 4.5 / 4.4, 6.6 / 6.1; 6926: 6.5 / 6.7, 5.3 / 4.8, 8.2 / 7.1; 18,216: 13.5 /
// 12.4, 10.2 / 7.6, 17.0 / 11.8. (One border for all: latents of 512 have theirs near 8000, the others near 1500.)
constexpr int APPEND_FEW = 2048;

// The lengths of a call, [row_start | act_q | act_k], from device memory or as a kernel argument (a one-shot
// call of few sequences: no upload before it)
struct DeviceLens {
  const int32_t* row_start;
  const int32_t* act_q;
  const int32_t* act_k;
  __device__ __forceinline__ int rs(int b) const { return row_start[b]; }
  __device__ __forceinline__ int aq(int b) const { return act_q[b]; }
  __device__ __forceinline__ int ak(int b) const { return act_k[b]; }
};
struct ArgLens {
  int32_t v[APPEND_ARG_LENGTHS];
  int batch;
  __device__ __forceinline__ int rs(int b) const { return v[b]; }
  __device__ __forceinline__ int aq(int b) const { return v[batch + 1 + b]; }
  __device__ __forceinline__ int ak(int b) const { return v[2 * batch + 1 + b]; }
};

struct Norm {
  int kind;   // 0 none, 1 root mean square, 2 mean and variance
  const void* w;
  const void* b;
  int wdt, w_aligned, b_aligned;
  float eps;
};

struct AppendPart {
  const void* x;
  View view;
  int aligned;   // 16-byte loads
  int heads, width;
  void* cache;   // [cache rows, heads, width], 16-byte aligned
};

struct AppendK {
  AppendPart a, b;   // b: the rotary keys beside latents
  Norm norm;         // of part a
  int start, rdim;   // rotated dimensions, of part a (index keys) or part b (latents)
  int inter;
  const float* freq;
  Positions pos;     // pos.p NULL: a token's place in its sequence
  const int32_t* table;
  int batch, total_rows, max_blocks, page, rows_per_batch;
  int64_t blocks;
};

// Eight of the norm's parameters from element e on, by 16-byte loads where they may be
__device__ __forceinline__ void norm_params(const void* p, int dt, int aligned, int e, float (&w)[8]) {
  if (dt == DSA_DTYPE_F32) {
    const float* f = reinterpret_cast<const float*>(p) + e;
    if (aligned) {
      const uint4 u = ldg16(f), v = ldg16(f + 4);
      const uint32_t b[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = __uint_as_float(b[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = f[i];
    }
    return;
  }
  const uint16_t* h = reinterpret_cast<const uint16_t*>(p) + e;
  uint16_t b[8];
  if (aligned) {
    const uint4 u = ldg16(h);
    const uint32_t d[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = (uint16_t)(d[i / 2] >> (16 * (i & 1)));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = h[i];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = dt == DSA_DTYPE_BF16 ? bf16_to_f32(b[i]) : f16_to_f32(b[i]);
}

template <int IO>
__device__ __forceinline__ void load8(const uint16_t* p, int aligned, float (&x)[8]) {
  if (aligned) load_vec<IO, 8>(p, x);
  else
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32<IO>(p[i]);
}

template <int LPV>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = LPV / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// Norm and rotation of one vector: lane `li` of its LPV lanes holds elements 8 li .. 8 li + 7 (zeros
// past the width). Statistics, weights and rotation in 32 bits; the caller rounds once.
template <int LPV>
__device__ __forceinline__ void norm_vec(const Norm& n, const float (&w)[8], const float (&b)[8], int width, int li,
                                         float (&x)[8]) {
  if (n.kind == 0) return;
  const bool in = 8 * li < width;
  float mean = 0.f;
  if (n.kind == 2) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += x[i];
    mean = group_sum<LPV>(s) / width;
  }
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] -= mean;
    q += x[i] * x[i];
  }
  q = group_sum<LPV>(in ? q : 0.f) / width;
  const float inv = 1.f / sqrtf(q + n.eps);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * w[i] + b[i];
}

template <int LPV>
__device__ __forceinline__ void rotate_vec(const float2* t, int start, int rdim, int inter, int li, float (&x)[8]) {
  const int e = 8 * li - start;   // first element's place in the rotary part
  const bool in = e >= 0 && e < rdim;
  if (inter) {
    if (!in) return;
    t += e / 2;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = x[2 * i], b = x[2 * i + 1];
      x[2 * i] = a * t[i].x - b * t[i].y;
      x[2 * i + 1] = a * t[i].y + b * t[i].x;
    }
    return;
  }
  // the other half of the pairs is rdim / 16 lanes away (every lane takes part in the exchange)
  const bool low = e < rdim / 2;
  const int other = (threadIdx.x & 63) + (in ? (low ? rdim / 16 : -(rdim / 16)) : 0);
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = __shfl(x[i], other);
  if (!in) return;
  t += low ? e : e - rdim / 2;
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = low ? x[i] * t[i].x - y[i] * t[i].y : y[i] * t[i].y + x[i] * t[i].x;
}

template <int IO, int LPV, bool LATENT, int NTOK, typename Lens>
__global__ __launch_bounds__(TPB) void append_kernel(AppendK a, Lens lens) {
  extern __shared__ float2 tab[];   // [NTOK][rdim / 2]
  __shared__ int64_t s_row[NTOK];   // the token's cache row, -1: it has none
  __shared__ int s_pos[NTOK];
  constexpr int VPP = TPB / LPV;    // vectors a pass of the work-group
  if ((int64_t)group_id() * NTOK >= a.total_rows) return;
  const int r0 = group_id() * NTOK;
  const int li = threadIdx.x % LPV, vi = threadIdx.x / LPV;
  const int heads = LATENT ? 1 : a.a.heads, half = LATENT ? 32 : a.rdim / 2;
  const int nvec = NTOK * heads;
  auto load_a = [&](int v, float (&x)[8]) __attribute__((always_inline)) {
    const int tok = heads == 1 ? v : v / heads, h = v - tok * heads;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 0.f;
    if (v < nvec && r0 + tok < a.total_rows && 8 * li < a.a.width)
      load8<IO>(reinterpret_cast<const uint16_t*>(a.a.x) + row_offset(a.a.view, r0 + tok) + h * a.a.view.head + 8 * li,
                a.a.aligned, x);
  };
  float x[8], xb[8];
  load_a(vi, x);
  // part b (64 wide): 8 lanes a token, the last waves
  const int bt = ((int)threadIdx.x - (TPB - 8 * NTOK)) >> 3, bl = threadIdx.x & 7;
  const bool bwave = LATENT && (int)threadIdx.x >= TPB - 8 * NTOK;
#pragma unroll
  for (int i = 0; i < 8; ++i) xb[i] = 0.f;
  if (bwave && r0 + bt < a.total_rows)
    load8<IO>(reinterpret_cast<const uint16_t*>(a.b.x) + row_offset(a.b.view, r0 + bt) + 8 * bl, a.b.aligned, xb);

  float nw[8], nb[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) nw[i] = nb[i] = 0.f;
  if (a.norm.kind != 0 && 8 * li < a.a.width) {
    norm_params(a.norm.w, a.norm.wdt, a.norm.w_aligned, 8 * li, nw);
    if (a.norm.b) norm_params(a.norm.b, a.norm.wdt, a.norm.b_aligned, 8 * li, nb);
  }
  // pair threadIdx.x % half of the table's token threadIdx.x / half (32 pairs: one a thread)
  const float freq0 = a.freq[(int)threadIdx.x % half];
  if (threadIdx.x < NTOK) {
    const int r = min(r0 + (int)threadIdx.x, a.total_rows - 1);
    int b = a.rows_per_batch > 0 ? min(r / a.rows_per_batch, a.batch - 1) : 0;
    int rs = lens.rs(b), re = lens.rs(b + 1), aq = lens.aq(b), ak = lens.ak(b);
    if (r < rs || r >= re) {   // the last sequence that begins at or before r
      int lo = 0, hi = a.batch - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (lens.rs(mid) <= r) lo = mid; else hi = mid - 1;
      }
      b = lo;
      rs = lens.rs(b), re = lens.rs(b + 1), aq = lens.aq(b), ak = lens.ak(b);
    }
    int64_t row = -1;
    const int s1 = r - rs, pos = ak - aq + s1;
    // rows past the batch's queries (or past the last batch), and tokens before position 0, have no place
    if (r0 + (int)threadIdx.x < a.total_rows && s1 >= 0 && s1 < aq && r < re && pos >= 0) {
      const int pg = pos / a.page;
      if (pg < a.max_blocks) {
        const int blk = a.table[(int64_t)b * a.max_blocks + pg];
        if (blk >= 0 && blk < a.blocks) row = (int64_t)blk * a.page + (pos - pg * a.page);
      }
    }
    s_row[threadIdx.x] = row;
    s_pos[threadIdx.x] = pos;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < NTOK * half; i += TPB) {
    const int tok = i / half, pair = i - tok * half;
    if (s_row[tok] >= 0) {
      const int64_t p = a.pos.p ? position_of(a.pos, r0 + tok, pair) : (int64_t)s_pos[tok];
      tab[i] = cos_sin(p, i == (int)threadIdx.x ? freq0 : a.freq[pair]);
    } else {
      tab[i] = make_float2(1.f, 0.f);
    }
  }
  __syncthreads();
  for (int v0 = 0; v0 < nvec; v0 += VPP) {
    const int v = v0 + vi;
    const int tok = min(heads == 1 ? v : v / heads, NTOK - 1), h = v - tok * heads;
    norm_vec<LPV>(a.norm, nw, nb, a.a.width, li, x);
    if (!LATENT) rotate_vec<LPV>(tab + tok * half, a.start, a.rdim, a.inter, li, x);
    if (v < nvec && 8 * li < a.a.width && s_row[tok] >= 0)
      store_vec<IO, 8>(reinterpret_cast<uint16_t*>(a.a.cache) + (s_row[tok] * heads + h) * a.a.width + 8 * li, x);
    // (requesting it before this pass's norm and store took longer: 16 x 32 heads of 128 17.9 us instead of 17.1)
    if (v0 + VPP < nvec) load_a(v + VPP, x);
  }
  if (bwave) {
    rotate_vec<8>(tab + bt * half, 0, a.rdim, a.inter, bl, xb);
    if (s_row[bt] >= 0) store_vec<IO, 8>(reinterpret_cast<uint16_t*>(a.b.cache) + s_row[bt] * a.b.width + 8 * bl, xb);
  }
}

template <int IO, bool LATENT, int NTOK, typename Lens>
hipError_t launch_append_n(const AppendK& k, const Lens& l, hipStream_t s) {
  const dim3 grid = grid_of(((int64_t)k.total_rows + NTOK - 1) / NTOK, 1);
  const size_t lds = (size_t)NTOK * (k.rdim / 2) * sizeof(float2);
  if (!LATENT && k.a.width <= 64) hipLaunchKernelGGL((append_kernel<IO, 8, LATENT, NTOK, Lens>), grid, dim3(TPB), lds, s, k, l);
  else if (k.a.width <= 128) hipLaunchKernelGGL((append_kernel<IO, 16, LATENT, NTOK, Lens>), grid, dim3(TPB), lds, s, k, l);
  else if (k.a.width <= 256) hipLaunchKernelGGL((append_kernel<IO, 32, LATENT, NTOK, Lens>), grid, dim3(TPB), lds, s, k, l);
  else hipLaunchKernelGGL((append_kernel<IO, 64, LATENT, NTOK, Lens>), grid, dim3(TPB), lds, s, k, l);
  return hipGetLastError();
}
template <int IO, bool LATENT>
hipError_t launch_append_io(const AppendK& k, const AppendArgs& a, hipStream_t s) {
  if (a.lengths_host) {
    ArgLens l{};
    std::memcpy(l.v, a.row_start, sizeof(int32_t) * (a.batch + 1));
    std::memcpy(l.v + a.batch + 1, a.act_q, sizeof(int32_t) * a.batch);
    std::memcpy(l.v + 2 * a.batch + 1, a.act_k, sizeof(int32_t) * a.batch);
    l.batch = a.batch;
    return k.total_rows > APPEND_FEW ? launch_append_n<IO, LATENT, 8>(k, l, s) : launch_append_n<IO, LATENT, 4>(k, l, s);
  }
  const DeviceLens l{a.row_start, a.act_q, a.act_k};
  return k.total_rows > APPEND_FEW ? launch_append_n<IO, LATENT, 8>(k, l, s) : launch_append_n<IO, LATENT, 4>(k, l, s);
}

int is_aligned(const void* p, const View& v) {
  return ((uintptr_t)p & 15) == 0 && v.batch % 8 == 0 && v.row % 8 == 0 && v.head % 8 == 0;
}
}  // namespace
}  // namespace dsa

using namespace dsa;

hipError_t launch_rotary(const RotaryArgs& a, hipStream_t s) {
  RotaryK k{};
  k.x = a.x;
  k.out = a.out;
  k.view = make_view(a.batch_stride, a.row_stride, a.head_stride, a.rows_per_batch, a.rows);
  k.pos = make_positions(a.positions, a.wide, a.rows, a.axes, a.sections, a.rdim / 2);
  k.freq = a.freq;
  k.rows = a.rows;
  k.heads = a.heads;
  k.width = a.width;
  k.start = a.start;
  k.rdim = a.rdim;
  k.inverse = a.inverse;
  if (a.io == DSA_DTYPE_BF16) return launch_rotary_io<DSA_DTYPE_BF16>(k, a.interleaved, s);
  if (a.io == DSA_DTYPE_F16) return launch_rotary_io<DSA_DTYPE_F16>(k, a.interleaved, s);
  return launch_rotary_io<DSA_DTYPE_F32>(k, a.interleaved, s);
}

hipError_t launch_row_positions(const int32_t* row_start, int batch, int rows, int32_t* positions, hipStream_t s) {
  hipLaunchKernelGGL(row_positions_kernel, dim3((unsigned)(((int64_t)rows + TPB - 1) / TPB)), dim3(TPB), 0, s, row_start, batch, rows,
                     positions);
  return hipGetLastError();
}

hipError_t launch_cache_append(const AppendArgs& a, hipStream_t s) {
  AppendK k{};
  const View va = make_view(a.batch_stride, a.row_stride, a.head_stride, a.rows_per_batch, a.total_rows);
  k.a = {a.x, va, is_aligned(a.x, va), a.heads, a.width, a.cache};
  const bool latent = a.rope != nullptr;
  if (latent) {
    const View vb = make_view(a.rope_batch_stride, a.rope_row_stride, 0, a.rows_per_batch, a.total_rows);
    k.b = {a.rope, vb, is_aligned(a.rope, vb), 1, 64, a.rope_cache};
  }
  k.norm = {a.norm_kind, a.norm_w, a.norm_b, a.wdt, ((uintptr_t)a.norm_w & 15) == 0, ((uintptr_t)a.norm_b & 15) == 0, a.eps};
  k.start = a.start;
  k.rdim = a.rdim;
  k.inter = a.interleaved;
  k.freq = a.freq;
  k.pos = make_positions(a.positions, a.wide, a.total_rows, a.axes, a.sections, a.rdim / 2);
  k.table = a.table;
  k.batch = a.batch;
  k.total_rows = a.total_rows;
  k.max_blocks = a.max_blocks;
  k.page = a.page;
  k.rows_per_batch = std::max(1, a.total_rows / a.batch);
  k.blocks = a.blocks;
  if (a.io == DSA_DTYPE_BF16)
    return latent ? launch_append_io<DSA_DTYPE_BF16, true>(k, a, s) : launch_append_io<DSA_DTYPE_BF16, false>(k, a, s);
  return latent ? launch_append_io<DSA_DTYPE_F16, true>(k, a, s) : launch_append_io<DSA_DTYPE_F16, false>(k, a, s);
}
