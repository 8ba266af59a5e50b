// Layer norm over the last dimension and its gradients, for gfx950.
//
//   mean = sum x / n, rstd = 1 / sqrt(sum (x - mean)^2 / n + eps), h = (x - mean) rstd, y = h w + b
// and with g = d w (d the gradient of y):
//   dx = (g - sum g / n - h sum(g h) / n) rstd,   dw = sum over rows of d h,   db = sum over rows of d
//
// Bound by memory: a row is read once into registers, and all its sums are made there (the variance from
// the centered values, so a large mean costs no bits). Statistics and sums are 32-bit, each output is
// rounded once. A row has TR threads, a power of two: up to a wave's 64 they sum by VALU lane exchanges,
// a work-group then taking several rows at a time; wider rows add through LDS.
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
  int width, tr;        // threads a row
  const void* w;
  const void* b;
  int wdt, w_vec;       // w_vec: w and b by 16 (8) byte loads
  float eps, inv_n;
  void* y;              // forward: y; gradient: dx (contiguous)
  float* mean;
  float* rstd;
  float* part;          // gradient: [groups][2][width], NULL: no weights' gradient wanted
  int* groups;          // host: how many work-groups the gradient's launch has
};

// V parameters from column c on (c + V <= width)
template <int V>
__device__ __forceinline__ void params(const void* p, int dt, int vec, int c, float (&w)[V]) {
  if (V > 1 && vec) {
    if (dt == DSA_DTYPE_F32) {
      const float* f = reinterpret_cast<const float*>(p) + c;
#pragma unroll
      for (int i = 0; i + 4 <= V; i += 4) {
        const uint4 u = ldg16(f + i);
        w[i] = __uint_as_float(u.x), w[i + 1] = __uint_as_float(u.y), w[i + 2] = __uint_as_float(u.z),
        w[i + 3] = __uint_as_float(u.w);
      }
    } else {
      const uint16_t* h = reinterpret_cast<const uint16_t*>(p) + c;
      uint2 u[V / 4 + 1];
#pragma unroll
      for (int i = 0; i + 4 <= V; i += 4) u[i / 4] = *reinterpret_cast<const uint2*>(h + i);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const uint16_t v = (uint16_t)((i & 2 ? u[i / 4].y : u[i / 4].x) >> (16 * (i & 1)));
        w[i] = dt == DSA_DTYPE_BF16 ? bf16_to_f32(v) : f16_to_f32(v);
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (dt == DSA_DTYPE_F32) w[i] = reinterpret_cast<const float*>(p)[c + i];
    else {
      const uint16_t v = reinterpret_cast<const uint16_t*>(p)[c + i];
      w[i] = dt == DSA_DTYPE_BF16 ? bf16_to_f32(v) : f16_to_f32(v);
    }
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
  const int wave = threadIdx.x >> 6, first = wave & ~((tr >> 6) - 1);
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

// UPT units of V elements a thread; T threads a work-group at most
template <int IO, int V, int UPT, int T>
__global__ __launch_bounds__(T) void layer_norm_kernel(NormK a) {
  using E = typename Elem<IO>::T;
  __shared__ float red[2][16][1];
  const int slots = (int)blockDim.x / a.tr, slot = (int)threadIdx.x / a.tr, t = (int)threadIdx.x & (a.tr - 1);
  int turn = 0;
  auto col = [&](int i) { return (t + i * a.tr) * V; };
  // the parameters stay in registers from row to row where they are few, else each row reads them (from a
  // cache) when it needs them; the opaque zero keeps the compiler from holding them all the same
  constexpr bool HOLD = UPT * V <= 16;
  const void* const wp = a.w;
  const void* const bp = a.b;
  float w[HOLD ? UPT : 1][V], b[HOLD ? UPT : 1][V];
  if constexpr (HOLD) {
#pragma unroll
    for (int i = 0; i < UPT; ++i) {
#pragma unroll
      for (int e = 0; e < V; ++e) w[i][e] = 1.f, b[i][e] = 0.f;
      if (wp && col(i) < a.width) params<V>(wp, a.wdt, a.w_vec, col(i), w[i]);
      if (bp && col(i) < a.width) params<V>(bp, a.wdt, a.w_vec, col(i), b[i]);
    }
  }
  for (int64_t base = (int64_t)blockIdx.x * slots; base < a.rows; base += (int64_t)gridDim.x * slots) {
    const int64_t r = base + slot;
    const bool ok = r < a.rows;
    const E* x = reinterpret_cast<const E*>(a.x) + (ok ? r : a.rows - 1) * a.x_stride;
    float v[UPT][V], s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < UPT; ++i) {
      if (col(i) < a.width) load_vec<IO, V>(x + col(i), v[i]);
      else
#pragma unroll
        for (int e = 0; e < V; ++e) v[i][e] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < UPT; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) s[0] += v[i][e];
    row_sums<1>(s, a.tr, red, turn);
    const float mean = s[0] * a.inv_n;
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < UPT; ++i)
      if (col(i) < a.width)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          v[i][e] -= mean;
          s[0] = fmaf(v[i][e], v[i][e], s[0]);
        }
    row_sums<1>(s, a.tr, red, turn);
    const float rstd = 1.f / sqrtf(s[0] * a.inv_n + a.eps);
    if (!ok) continue;   // (the slots' trips through the barriers are the same: base is the work-group's)
    if (t == 0 && a.mean) {
      a.mean[r] = mean;
      a.rstd[r] = rstd;
    }
    E* y = reinterpret_cast<E*>(a.y) + r * a.width;
    int again = 0;   // opaque
    asm volatile("" : "+v"(again));
#pragma unroll
    for (int i = 0; i < UPT; ++i) {
      if (col(i) >= a.width) continue;
      if constexpr (HOLD) {
#pragma unroll
        for (int e = 0; e < V; ++e) v[i][e] = fmaf(v[i][e] * rstd, w[i][e], b[i][e]);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) w[0][e] = 1.f, b[0][e] = 0.f;
        if (wp) params<V>(wp, a.wdt, a.w_vec, col(i) + again, w[0]);
        if (bp) params<V>(bp, a.wdt, a.w_vec, col(i) + again, b[0]);
#pragma unroll
        for (int e = 0; e < V; ++e) v[i][e] = fmaf(v[i][e] * rstd, w[0][e], b[0][e]);
      }
      store_vec<IO, V>(y + col(i), v[i]);
    }
  }
}

template <int IO, int V, int UPT, int T>
__global__ __launch_bounds__(T) void layer_norm_grad_kernel(NormK a) {
  using E = typename Elem<IO>::T;
  __shared__ float red[2][16][2];
  extern __shared__ float join[];   // [2][width] of one slot, where a work-group has several
  const int slots = (int)blockDim.x / a.tr, slot = (int)threadIdx.x / a.tr, t = (int)threadIdx.x & (a.tr - 1);
  int turn = 0;
  auto col = [&](int i) { return (t + i * a.tr) * V; };
  float w[UPT][V], dw[UPT][V], db[UPT][V];
#pragma unroll
  for (int i = 0; i < UPT; ++i) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      w[i][e] = 1.f;
      dw[i][e] = db[i][e] = 0.f;
    }
    if (a.w && col(i) < a.width) params<V>(a.w, a.wdt, a.w_vec, col(i), w[i]);
  }
  for (int64_t base = (int64_t)blockIdx.x * slots; base < a.rows; base += (int64_t)gridDim.x * slots) {
    const int64_t r = base + slot;
    const bool ok = r < a.rows;
    const int64_t rr = ok ? r : a.rows - 1;
    const E* x = reinterpret_cast<const E*>(a.x) + rr * a.x_stride;
    const E* d = reinterpret_cast<const E*>(a.d) + rr * a.d_stride;
    float h[UPT][V], g[UPT][V], s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < UPT; ++i) {
      if (ok && col(i) < a.width) {
        load_vec<IO, V>(x + col(i), h[i]);
        load_vec<IO, V>(d + col(i), g[i]);
      }
    }
    const float mean = a.mean[rr], rstd = a.rstd[rr];
#pragma unroll
    for (int i = 0; i < UPT; ++i)
      if (ok && col(i) < a.width)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          h[i][e] = (h[i][e] - mean) * rstd;
          dw[i][e] = fmaf(g[i][e], h[i][e], dw[i][e]);
          db[i][e] += g[i][e];
          g[i][e] *= w[i][e];
          s[0] += g[i][e];
          s[1] = fmaf(g[i][e], h[i][e], s[1]);
        }
    row_sums<2>(s, a.tr, red, turn);
    if (!ok) continue;
    const float c0 = s[0] * a.inv_n, c1 = s[1] * a.inv_n;
    E* dx = reinterpret_cast<E*>(a.y) + r * a.width;
#pragma unroll
    for (int i = 0; i < UPT; ++i) {
      if (col(i) >= a.width) continue;
#pragma unroll
      for (int e = 0; e < V; ++e) g[i][e] = (g[i][e] - c0 - h[i][e] * c1) * rstd;
      store_vec<IO, V>(dx + col(i), g[i]);
    }
  }
  if (!a.part) return;
  // the slots one after another, the last one leaves the work-group's sums
  float* out = a.part + (int64_t)blockIdx.x * 2 * a.width;
  for (int k = 0; k < slots; ++k) {
    if (slot == k) {
#pragma unroll
      for (int i = 0; i < UPT; ++i) {
        if (col(i) >= a.width) continue;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int c = col(i) + e;
          float p = dw[i][e], q = db[i][e];
          if (k > 0) {
            p += join[c];
            q += join[a.width + c];
          }
          if (k + 1 < slots) {
            join[c] = p;
            join[a.width + c] = q;
          } else {
            out[c] = p;
            out[a.width + c] = q;
          }
        }
      }
    }
    if (slots > 1) __syncthreads();
  }
}

// Column sums of the partial rows: 64 columns a work-group, 16 threads to a column. blockIdx.y: dw or db.
template <int WDT>
__global__ __launch_bounds__(1024) void layer_norm_join_kernel(const float* part, int groups, int width, void* dw, void* db) {
  __shared__ float red[16][64];
  using E = typename Elem<WDT>::T;
  E* out = reinterpret_cast<E*>(blockIdx.y ? db : dw);
  if (!out) return;
  const int lane = threadIdx.x & 63, row = threadIdx.x >> 6, c = (int)blockIdx.x * 64 + lane;
  float s = 0.f;
  if (c < width)
    for (int g = row; g < groups; g += 16) s += part[((int64_t)g * 2 + blockIdx.y) * width + c];
  red[row][lane] = s;
  __syncthreads();
  if (row == 0 && c < width) {
#pragma unroll
    for (int k = 1; k < 16; ++k) s += red[k][lane];
    const float v[1] = {s};
    store_vec<WDT, 1>(out + c, v);
  }
}

// Threads a row, and units of V elements a thread
struct Shape {
  int tr, upt, threads;
};
int pow2_above(int n) {
  int p = 1;
  while (p < n) p <<= 1;
  return p;
}
Shape shape_of(int units, int v) {
  if (units <= 64) return {pow2_above(units), 1, 256};
  if (v == 1) {
    if (units <= 256) return {64, 4, 256};
    if (units <= 1024) return {256, 4, 256};
    return {1024, 16, 1024};
  }
  if (units <= 128) return {64, 2, 256};
  if (units <= 256) return {64, 4, 256};
  if (units <= 512) return {256, 2, 256};
  if (units <= 1024) return {256, 4, 256};
  return {pow2_above((units + 3) / 4), 4, 1024};   // (fp32 to 16384 columns, 16 bits to 16384 in 512 threads)
}

template <int IO, int V, int UPT, int T>
hipError_t launch(const NormK& k, bool grad, int threads, hipStream_t s) {
  const int slots = threads / k.tr;
  if (!grad) {
    const int64_t groups = std::min<int64_t>((k.rows + slots - 1) / slots, 4096);
    hipLaunchKernelGGL((layer_norm_kernel<IO, V, UPT, T>), dim3((unsigned)groups), dim3(threads), 0, s, k);
  } else {
    const size_t lds = slots > 1 && k.part ? (size_t)k.width * 2 * sizeof(float) : 0;
    *k.groups = (int)std::min<int64_t>((k.rows + slots - 1) / slots, MAX_GROUPS);
    hipLaunchKernelGGL((layer_norm_grad_kernel<IO, V, UPT, T>), dim3(*k.groups), dim3(threads), lds, s, k);
  }
  return hipGetLastError();
}

template <int IO, int V>
hipError_t launch_v(NormK k, bool grad, hipStream_t s) {
  const Shape sh = shape_of((k.width + V - 1) / V, V);
  k.tr = sh.tr;
  switch (sh.upt) {
    case 1: return launch<IO, V, 1, 256>(k, grad, sh.threads, s);
    case 2: if constexpr (V > 1) return launch<IO, V, 2, 256>(k, grad, sh.threads, s); break;
    case 4:
      if (sh.threads == 256) return launch<IO, V, 4, 256>(k, grad, sh.threads, s);
      // rows of more than 256 threads: one to a work-group
      if constexpr (V == 8) return launch<IO, V, 4, 512>(k, grad, k.tr, s);
      if constexpr (V == 4) return launch<IO, V, 4, 1024>(k, grad, k.tr, s);
      break;
    case 16: if constexpr (V == 1) return launch<IO, V, 16, 1024>(k, grad, sh.threads, s); break;
  }
  return hipErrorInvalidValue;
}

template <int IO>
hipError_t launch_io(NormK k, bool grad, hipStream_t s) {
  using T = typename Elem<IO>::T;
  constexpr int V = Elem<IO>::V;
  auto on16 = [](const void* p, int64_t stride) { return ((uintptr_t)p & 15) == 0 && stride * (int64_t)sizeof(T) % 16 == 0; };
  const bool vec = k.width % V == 0 && on16(k.x, k.x_stride) && on16(k.y, k.width) && (!grad || on16(k.d, k.d_stride));
  return vec ? launch_v<IO, V>(k, grad, s) : launch_v<IO, 1>(k, grad, s);
}

hipError_t launch_any(NormK k, int io, bool grad, hipStream_t s) {
  k.w_vec = (((uintptr_t)k.w | (uintptr_t)k.b) & 15) == 0;
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
  const dim3 grid((unsigned)((a.width + 63) / 64), 2);
  if (a.wdt == DSA_DTYPE_F16)
    hipLaunchKernelGGL(layer_norm_join_kernel<DSA_DTYPE_F16>, grid, dim3(1024), 0, s, a.part, groups, a.width, a.dw, a.db);
  else if (a.wdt == DSA_DTYPE_BF16)
    hipLaunchKernelGGL(layer_norm_join_kernel<DSA_DTYPE_BF16>, grid, dim3(1024), 0, s, a.part, groups, a.width, a.dw, a.db);
  else
    hipLaunchKernelGGL(layer_norm_join_kernel<DSA_DTYPE_F32>, grid, dim3(1024), 0, s, a.part, groups, a.width, a.dw, a.db);
  return hipGetLastError();
}
