// Layer norm over the last dimension and its gradients, for gfx950.
//
//   mean = sum x / n, rstd = 1 / sqrt(sum (x - mean)^2 / n + eps), h = (x - mean) rstd, y = h w + b
// and with g = d w (d the gradient of y):
//   dx = (g - sum g / n - h sum(g h) / n) rstd,   dw = sum over rows of d h,   db = sum over rows of d
//
// Bound by memory: a row is read once into registers, and all its sums are made there: the mean, then the squares of what is
// left without it. Where the row lies far from zero, what is left has a sum as well: the rounding of the mean, which would
// stay in each value (a constant row of 10^4 in fp32 gave outputs up to 0.6 where they are 0); it corrects mean, variance and
// output. (For every row: 8192 rows of 8192 in bf16 45 us for 44, 4096 of 16384 57 for 50.) Statistics and sums are 32-bit, each output is
// rounded once. A row has TR threads: up to a wave's 64 (a power of two) they sum by VALU lane exchanges, a work-group
// then taking several rows at a time; wider rows add through LDS. The next row is loaded before this one's sums, which
// wait for each other. 16383 rows of 4096 in bf16: forward 44 us (6.1 TB/s; 48 right before the gradient), gradient 83
// (4.8); in fp32 100 (5.4) and 154 (5.2).
//
// Rows of an odd width, or strided ones, begin anywhere: the accesses are of 16 bytes all the same, which the hardware
// takes at any alignment (8192 rows of 2049 in bf16: 126 -> 20 us against single elements, the gradient 139 -> 32).
//
// The sums over rows: each work-group adds up its rows' d h and d in registers (a thread's columns are the
// same in every row), joins its row slots in LDS and leaves one row of partial sums; a second launch adds those, in
// a fixed order, so the results do not depend on timing.
#include <algorithm>

#include "elements.hpp"

namespace dsa {
namespace {

constexpr int MAX_GROUPS = 512;   // of the gradient, each leaving a row of partial sums

struct NormK {
  const void* x;
  const void* d;        // gradient: of y
  int64_t x_stride, d_stride;
  int64_t rows;
  int width, tr;        // threads a row: a power of two, or the whole work-group's waves
  const void* w;
  const void* b;
  int wdt;
  float eps, inv_n;
  void* y;              // forward: y; gradient: dx (contiguous)
  float* mean;
  float* rstd;
  float* part;          // gradient: [groups][2][width], NULL: no weights' gradient wanted
  int* groups;          // host: how many work-groups the gradient's launch has
};

// The same 16-byte accesses whatever the alignment: rows of an odd width begin anywhere
template <int IO, int V>
__device__ __forceinline__ typename Raw<IO, V>::T load_any(const typename Elem<IO>::T* p) {
  typename Raw<IO, V>::T u;
  __builtin_memcpy(&u, p, sizeof(u));
  return u;
}
template <int IO, int V>
__device__ __forceinline__ void store_any(typename Elem<IO>::T* p, const float (&x)[V]) {
  typename Elem<IO>::T v[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    if constexpr (IO == DSA_DTYPE_F32) v[e] = x[e];
    else v[e] = from_f32<IO>(x[e]);
  }
  __builtin_memcpy(p, v, sizeof(v));
}

// V parameters from column c on
template <int V>
__device__ __forceinline__ void params(const void* p, int dt, int c, float (&w)[V]) {
  if (dt == DSA_DTYPE_F32) {
    __builtin_memcpy(w, reinterpret_cast<const float*>(p) + c, sizeof(w));
  } else {
    uint16_t v[V];
    __builtin_memcpy(v, reinterpret_cast<const uint16_t*>(p) + c, sizeof(v));
#pragma unroll
    for (int e = 0; e < V; ++e) w[e] = dt == DSA_DTYPE_BF16 ? bf16_to_f32(v[e]) : f16_to_f32(v[e]);
  }
}

template <int CTRL>
__device__ __forceinline__ float dpp_add(float x) {
  return x + __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), CTRL, 0xF, 0xF, false));
}
// The sum over each aligned run of min(tr, 64) lanes, on all of them (tr a power of two, uniform)
__device__ __forceinline__ float lane_sum(float x, int tr) {
  if (tr > 1) x = dpp_add<0xB1>(x);    // quad_perm: the neighbour
  if (tr > 2) x = dpp_add<0x4E>(x);    // quad_perm: two on
  if (tr > 4) x = dpp_add<0x141>(x);   // row_half_mirror: the other quad of eight lanes
  if (tr > 8) x = dpp_add<0x140>(x);   // row_mirror: the other eight of sixteen
  if (tr > 16) {
    float a = x, b = x;
    swap_rows16(a, b);
    x = a + b;
  }
  if (tr > 32) x = add_half_swap(x);
  return x;
}

// Sums of N values over a row's threads. Rows wider than a wave go through LDS, in two buffers by turns: one
// barrier a sum.
template <int N>
__device__ __forceinline__ void row_sums(float (&v)[N], int tr, float (*red)[16][N], int& turn) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lane_sum(v[i], tr);
  if (tr <= 64) return;
  float (*buf)[N] = red[turn & 1];
  ++turn;
  const int wave = threadIdx.x >> 6, first = tr < (int)blockDim.x ? wave & ~((tr >> 6) - 1) : 0;
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) buf[wave][i] = v[i];
  lds_barrier();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = 0.f;
  for (int k = 0; k < tr >> 6; ++k)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += buf[first + k][i];
}

// A row in units of V columns, UPT of them to a thread. The last unit ends with the row, so it may begin with columns of
// the one before it: both make the same outputs of those, but only the other one adds them to sums.
template <int V>
struct Columns {
  int t, tr, width;
  __device__ __forceinline__ int of(int i) const { return (t + i * tr) * V; }
  __device__ __forceinline__ int at(int i) const { return min(of(i), width - V); }   // where unit i lies
  __device__ __forceinline__ int skip(int i) const { return max(0, of(i) - at(i)); }   // not added; V or more: no unit
};

// x as it is rounded: the compiler would otherwise take a product into the sums that use it in some of a row's units and
// not in others, which then differ by the product's rounding, columns that two units hold too
__device__ __forceinline__ float rounded(float x) {
  asm volatile("" : "+v"(x));
  return x;
}

constexpr float FAR = 4.f;
__device__ __forceinline__ bool far_from_zero(float mean, float rstd) { return fabsf(mean) * rstd > FAR; }

// UPT units of V elements a thread; T threads a work-group at most
template <int IO, int V, int UPT, int T>
__global__ __launch_bounds__(T) void layer_norm_kernel(NormK a) {
  using E = typename Elem<IO>::T;
  __shared__ float red[2][16][1];
  const int slots = (int)blockDim.x / a.tr, slot = (int)threadIdx.x / a.tr;
  const Columns<V> col{(int)threadIdx.x - slot * a.tr, a.tr, a.width};
  int turn = 0;
  float w[UPT][V], b[UPT][V];
#pragma unroll
  for (int i = 0; i < UPT; ++i) {
#pragma unroll
    for (int e = 0; e < V; ++e) w[i][e] = 1.f, b[i][e] = 0.f;
    if (a.w) params<V>(a.w, a.wdt, col.at(i), w[i]);
    if (a.b) params<V>(a.b, a.wdt, col.at(i), b[i]);
  }
  typename Raw<IO, V>::T next[UPT];
  auto fetch = [&](int64_t r) {
    const E* x = reinterpret_cast<const E*>(a.x) + min(r, a.rows - 1) * a.x_stride;
#pragma unroll
    for (int i = 0; i < UPT; ++i) next[i] = load_any<IO, V>(x + col.at(i));
  };
  fetch((int64_t)blockIdx.x * slots + slot);
  for (int64_t base = (int64_t)blockIdx.x * slots; base < a.rows; base += (int64_t)gridDim.x * slots) {
    const int64_t r = base + slot;
    float v[UPT][V], s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < UPT; ++i) widen<IO, V>(next[i], v[i]);
    fetch(r + (int64_t)gridDim.x * slots);
#pragma unroll
    for (int i = 0; i < UPT; ++i) {
      const int skip = col.skip(i);
      if (skip == 0) {
#pragma unroll
        for (int e = 0; e < V; ++e) s[0] += v[i][e];
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) s[0] += e >= skip ? v[i][e] : 0.f;
      }
    }
    row_sums<1>(s, a.tr, red, turn);
    const float first = rounded(s[0] * a.inv_n);
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < UPT; ++i) {
      const int skip = col.skip(i);
#pragma unroll
      for (int e = 0; e < V; ++e) v[i][e] -= first;
      if (skip == 0) {
#pragma unroll
        for (int e = 0; e < V; ++e) s[0] = fmaf(v[i][e], v[i][e], s[0]);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) s[0] += e >= skip ? v[i][e] * v[i][e] : 0.f;
      }
    }
    row_sums<1>(s, a.tr, red, turn);
    float mean = first, var = s[0] * a.inv_n, off = 0.f;
    // (within FAR deviations the mean's rounding is that of the sums; a work-group's rows that share barriers go together)
    const bool far = first * first > FAR * FAR * (var + a.eps);
    if (a.tr <= 64 ? __builtin_amdgcn_ballot_w64(far) != 0 : far || slots > 1) {
      s[0] = 0.f;
#pragma unroll
      for (int i = 0; i < UPT; ++i) {
        const int skip = col.skip(i);
#pragma unroll
        for (int e = 0; e < V; ++e) s[0] += e >= skip ? v[i][e] : 0.f;
      }
      row_sums<1>(s, a.tr, red, turn);
      if (far) {
        off = s[0] * a.inv_n;
        mean = first + off;
        var = fmaf(-off, off, var);
        var = var < 0.f ? 0.f : var;   // (NaN stays)
      }
    }
    const float rstd = 1.f / sqrtf(var + a.eps), shift = rounded(-off * rstd);
    if (r >= a.rows) continue;   // (the slots' trips through the barriers are the same: base is the work-group's)
    if (col.t == 0 && a.mean) {
      a.mean[r] = mean;
      a.rstd[r] = rstd;
    }
    E* y = reinterpret_cast<E*>(a.y) + r * a.width;
#pragma unroll
    for (int i = 0; i < UPT; ++i) {
      if (col.of(i) >= a.width) continue;
#pragma unroll
      for (int e = 0; e < V; ++e) v[i][e] = fmaf(fmaf(v[i][e], rstd, shift), w[i][e], b[i][e]);
      store_any<IO, V>(y + col.at(i), v[i]);
    }
  }
}

template <int IO, int V, int UPT, int T>
__global__ __launch_bounds__(T) void layer_norm_grad_kernel(NormK a) {
  using E = typename Elem<IO>::T;
  __shared__ float red[2][16][2], red1[2][16][1];
  extern __shared__ float join[];   // [slots][2][width], where a work-group has several
  const int slots = (int)blockDim.x / a.tr, slot = (int)threadIdx.x / a.tr;
  const Columns<V> col{(int)threadIdx.x - slot * a.tr, a.tr, a.width};
  int turn = 0, turn1 = 0;
  // the parameters in registers; 1024 threads in 32 bits, which have too few, read them for each row (6000 rows of 9000: 189 ->
  // 158 us, 4096 of 16384: 212 -> 201)
  constexpr bool HOLD = T < 1024 || IO != DSA_DTYPE_F32;
  float w[HOLD ? UPT : 1][V], dw[UPT][V], db[UPT][V];
  auto parameters = [&](int i, float (&p)[V]) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < V; ++e) p[e] = 1.f;
    if (a.w) params<V>(a.w, a.wdt, col.at(i), p);
  };
#pragma unroll
  for (int i = 0; i < UPT; ++i) {
#pragma unroll
    for (int e = 0; e < V; ++e) dw[i][e] = db[i][e] = 0.f;
    if constexpr (HOLD) parameters(i, w[i]);
  }
  // the next row's elements are on their way while this one's sums are made (16383 rows of 4096 in bf16: 157 -> 83 us),
  // but where 1024 threads leave no registers for them
  constexpr bool AHEAD = T < 1024 || IO != DSA_DTYPE_F32;
  typename Raw<IO, V>::T xn[UPT], dn[UPT];
  float mean_n, rstd_n;
  auto fetch = [&](int64_t r) {
    const int64_t rr = min(r, a.rows - 1);
    const E* x = reinterpret_cast<const E*>(a.x) + rr * a.x_stride;
    const E* d = reinterpret_cast<const E*>(a.d) + rr * a.d_stride;
#pragma unroll
    for (int i = 0; i < UPT; ++i) {
      xn[i] = load_any<IO, V>(x + col.at(i));
      dn[i] = load_any<IO, V>(d + col.at(i));
    }
    mean_n = a.mean[rr], rstd_n = a.rstd[rr];
  };
  if constexpr (AHEAD) fetch((int64_t)blockIdx.x * slots + slot);
  for (int64_t base = (int64_t)blockIdx.x * slots; base < a.rows; base += (int64_t)gridDim.x * slots) {
    const int64_t r = base + slot;
    const bool ok = r < a.rows;
    float h[UPT][V], g[UPT][V], s[2] = {0.f, 0.f};
    if constexpr (!AHEAD) fetch(r);
#pragma unroll
    for (int i = 0; i < UPT; ++i) {
      widen<IO, V>(xn[i], h[i]);
      widen<IO, V>(dn[i], g[i]);
    }
    const float mean = mean_n, rstd = rstd_n;
#pragma unroll
    for (int i = 0; i < UPT; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) h[i][e] -= mean;
    if constexpr (AHEAD) fetch(r + (int64_t)gridDim.x * slots);
    // far from zero, the mean as it was handed over is rounded too much (as in the forward); rows that share barriers go together
    float shift = 0.f;
    const bool far = far_from_zero(mean, rstd);
    bool any = far;
    if constexpr (T == 256) {   // (wider work-groups have one row)
      if (a.tr <= 64) any = __builtin_amdgcn_ballot_w64(far) != 0;
      else if (slots > 1) {     // two rows of 128 threads
        const int64_t other = min(base + 1 - slot, a.rows - 1);
        any = any || far_from_zero(a.mean[other], a.rstd[other]);
      }
    }
    if (any) {
      float t[1] = {0.f};
#pragma unroll
      for (int i = 0; i < UPT; ++i) {
        const int skip = col.skip(i);
#pragma unroll
        for (int e = 0; e < V; ++e) t[0] += e >= skip ? h[i][e] : 0.f;
      }
      row_sums<1>(t, a.tr, red1, turn1);
      if (far) shift = -t[0] * a.inv_n * rstd;
    }
    shift = rounded(shift);
#pragma unroll
    for (int i = 0; i < UPT; ++i) {
      const int skip = ok ? col.skip(i) : V;
      if constexpr (!HOLD) parameters(i, w[0]);
      float(&wi)[V] = w[HOLD ? i : 0];
      if (skip == 0) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          h[i][e] = fmaf(h[i][e], rstd, shift);
          dw[i][e] = fmaf(g[i][e], h[i][e], dw[i][e]);
          db[i][e] += g[i][e];
          g[i][e] *= wi[e];
          s[0] += g[i][e];
          s[1] = fmaf(g[i][e], h[i][e], s[1]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          h[i][e] = fmaf(h[i][e], rstd, shift);
          dw[i][e] += e >= skip ? g[i][e] * h[i][e] : 0.f;
          db[i][e] += e >= skip ? g[i][e] : 0.f;
          g[i][e] *= wi[e];
          s[0] += e >= skip ? g[i][e] : 0.f;
          s[1] += e >= skip ? g[i][e] * h[i][e] : 0.f;
        }
      }
    }
    row_sums<2>(s, a.tr, red, turn);
    if (!ok) continue;
    const float c0 = rounded(s[0] * a.inv_n), c1 = rounded(s[1] * a.inv_n);
    E* dx = reinterpret_cast<E*>(a.y) + r * a.width;
#pragma unroll
    for (int i = 0; i < UPT; ++i) {
      if (col.of(i) >= a.width) continue;
#pragma unroll
      for (int e = 0; e < V; ++e) g[i][e] = (g[i][e] - c0 - h[i][e] * c1) * rstd;
      store_any<IO, V>(dx + col.at(i), g[i]);
    }
  }
  if (!a.part) return;
  // the work-group's sums: a slot's straight from the registers, of several through LDS
  float* out = a.part + (int64_t)blockIdx.x * 2 * a.width;
  float* to = slots > 1 ? join + slot * 2 * a.width : out;
#pragma unroll
  for (int i = 0; i < UPT; ++i) {
    const int skip = col.skip(i), c = col.at(i);
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e >= skip) {
        to[c + e] = dw[i][e];
        to[a.width + c + e] = db[i][e];
      }
  }
  if (slots == 1) return;
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * a.width; c += blockDim.x) {
    float p = join[c];
    for (int k = 1; k < slots; ++k) p += join[k * 2 * a.width + c];
    out[c] = p;
  }
}

// Column sums of the partial rows: 32 columns a work-group, 32 threads to a column. blockIdx.y: dw or db.
template <int WDT>
__global__ __launch_bounds__(1024) void layer_norm_join_kernel(const float* part, int groups, int width, void* dw, void* db) {
  __shared__ float red[32][33];
  using E = typename Elem<WDT>::T;
  E* out = reinterpret_cast<E*>(blockIdx.y ? db : dw);
  if (!out) return;
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5, c = (int)blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < width) {
    const float* p = part + (int64_t)blockIdx.y * width + c;
#pragma unroll 8
    for (int g = row; g < groups; g += 32) s += p[(int64_t)g * 2 * width];
  }
  red[row][lane] = s;
  __syncthreads();
  if (row) return;
#pragma unroll
  for (int k = 1; k < 32; ++k) s += red[k][lane];
  if (c < width) {
    const float v[1] = {s};
    store_vec<WDT, 1>(out + c, v);
  }
}

int pow2_above(int n) {
  int p = 1;
  while (p < n) p <<= 1;
  return p;
}

template <int IO, int V, int UPT, int T>
hipError_t launch(const NormK& k, bool grad, hipStream_t s) {
  const int slots = k.tr > 128 ? 1 : 256 / k.tr, threads = slots * k.tr;
  const int64_t trips = (k.rows + slots - 1) / slots;
  if (!grad) {
    // Four work-groups a CU, or two wide ones, that stay, so that a row's loads hide behind the one before it and the
    // parameters are read once: 16383 rows of 4096 in bf16 take 57, 43, 44, 48 us with 512, 1024, 4096, 8192 work-groups
    // of 256 threads; 8192 rows of 8192 43, 44, 53, 61 with 512 threads; 100,000 rows of 128 14, 11, 11, 11. In fp32, whose
    // rows of 4096 are two loads a thread longer, 1024 against 4096 take 100 and 97
    const unsigned groups = (unsigned)std::min<int64_t>(trips, threads <= 320 ? 1024 : 512);
    hipLaunchKernelGGL((layer_norm_kernel<IO, V, UPT, T>), dim3(groups), dim3(threads), 0, s, k);
  } else {
    // a work-group's row of partial sums costs as much as some rows of the input: eight trips for it (2048 rows of 4096 in
    // bf16: 512 work-groups 25.5 us, 256 22.1; 512 rows: 512 23.5, 128 17.8), four of several narrow rows (16384 of
    // 128: 128 work-groups 9.9, 256 7.6), but no fewer than half the CUs, or all
    const int64_t few = slots > 1 ? (trips + 3) / 4 : (trips + 7) / 8;
    *k.groups = (int)std::min<int64_t>(std::max(few, std::min<int64_t>(trips, slots > 1 ? 256 : 128)), MAX_GROUPS);
    const size_t lds = slots > 1 && k.part ? (size_t)slots * k.width * 2 * sizeof(float) : 0;
    hipLaunchKernelGGL((layer_norm_grad_kernel<IO, V, UPT, T>), dim3(*k.groups), dim3(threads), lds, s, k);
  }
  return hipGetLastError();
}

template <int IO>
hipError_t launch_io(NormK k, bool grad, hipStream_t s) {
  constexpr int V = Elem<IO>::V;
  if (k.width < V) {
    k.tr = pow2_above(k.width);
    return launch<IO, 1, 1, 256>(k, grad, s);
  }
  // One unit a thread up to a wave a row; then 16 columns a thread, from 256 threads on as many waves as that takes.
  const int units = (k.width + V - 1) / V;
  k.tr = pow2_above(units);
  if (k.tr <= 64) return launch<IO, V, 1, 256>(k, grad, s);
  constexpr int UPT = 16 / V;
  const int threads = ((units + UPT - 1) / UPT + 63) / 64 * 64;
  k.tr = threads <= 128 ? pow2_above(threads) : threads;
  if (k.tr <= 256) return launch<IO, V, UPT, 256>(k, grad, s);
  if (k.tr <= 512) return launch<IO, V, UPT, 512>(k, grad, s);
  // (two work-groups of 512 threads on a CU pass the time of each other's barriers, one of 1024 has nobody to: 4096 rows of
  // 16384 in bf16 take 83 against 88 us at a work-group a row, their gradient 112 against 124. In 32 bits 512 threads
  // would have twice the registers.)
  if constexpr (V == 8) {
    k.tr = ((units + 3) / 4 + 63) / 64 * 64;
    return launch<IO, V, 4, 512>(k, grad, s);
  } else {
    return launch<IO, V, UPT, 1024>(k, grad, s);
  }
}

hipError_t launch_any(NormK k, int io, bool grad, hipStream_t s) {
  k.inv_n = 1.f / (float)k.width;
  switch (io) {
    case DSA_DTYPE_F16: return launch_io<DSA_DTYPE_F16>(k, grad, s);
    case DSA_DTYPE_BF16: return launch_io<DSA_DTYPE_BF16>(k, grad, s);
    default: return launch_io<DSA_DTYPE_F32>(k, grad, s);
  }
}

}  // namespace
}  // namespace dsa

using namespace dsa;

hipError_t launch_layer_norm(const NormArgs& a, hipStream_t s) {
  NormK k{};
  k.x = a.x, k.x_stride = a.x_stride, k.rows = a.rows, k.width = a.width, k.w = a.w, k.b = a.b, k.wdt = a.wdt, k.eps = a.eps;
  k.y = a.y, k.mean = a.mean, k.rstd = a.rstd;
  return launch_any(k, a.io, false, s);
}

size_t layer_norm_grad_workspace_bytes(int64_t rows, int width) {
  return (size_t)std::min<int64_t>(rows, MAX_GROUPS) * 2 * (size_t)width * sizeof(float);
}

hipError_t launch_layer_norm_grad(const NormArgs& a, hipStream_t s) {
  NormK k{};
  k.x = a.x, k.x_stride = a.x_stride, k.d = a.d, k.d_stride = a.d_stride, k.rows = a.rows, k.width = a.width, k.w = a.w;
  k.wdt = a.wdt, k.y = a.y, k.mean = a.mean, k.rstd = a.rstd;
  const bool sums = a.dw || a.db;
  k.part = sums ? a.part : nullptr;
  int groups = 0;   // no rows: the sums are zero
  k.groups = &groups;
  if (a.rows > 0) {
    const hipError_t e = launch_any(k, a.io, true, s);
    if (e != hipSuccess) return e;
  }
  if (!sums) return hipSuccess;
  const dim3 grid((unsigned)((a.width + 31) / 32), 2);
  if (a.wdt == DSA_DTYPE_F16)
    hipLaunchKernelGGL(layer_norm_join_kernel<DSA_DTYPE_F16>, grid, dim3(1024), 0, s, a.part, groups, a.width, a.dw, a.db);
  else if (a.wdt == DSA_DTYPE_BF16)
    hipLaunchKernelGGL(layer_norm_join_kernel<DSA_DTYPE_BF16>, grid, dim3(1024), 0, s, a.part, groups, a.width, a.dw, a.db);
  else
    hipLaunchKernelGGL(layer_norm_join_kernel<DSA_DTYPE_F32>, grid, dim3(1024), 0, s, a.part, groups, a.width, a.dw, a.db);
  return hipGetLastError();
}
