// Elements of fp16, bf16 and fp32 tensors, moved V at a time (16 bytes, or single elements where the
// alignment asks for it) as 32-bit values.
#pragma once

#include "dsa_common.hpp"

namespace dsa {

template <int IO> struct Elem { using T = uint16_t; static constexpr int V = 8; };
template <> struct Elem<DSA_DTYPE_F32> { using T = float; static constexpr int V = 4; };

// V elements as they lie in memory
template <int IO, int V> struct Raw { using T = uint4; };
template <int IO> struct Raw<IO, 1> { using T = typename Elem<IO>::T; };
template <int IO, int V>
__device__ __forceinline__ void widen(typename Raw<IO, V>::T u, float (&x)[V]) {
  if constexpr (V == 1) {
    if constexpr (IO == DSA_DTYPE_F32) x[0] = u;
    else x[0] = to_f32<IO>(u);
  } else if constexpr (IO == DSA_DTYPE_F32) {
    x[0] = __uint_as_float(u.x), x[1] = __uint_as_float(u.y), x[2] = __uint_as_float(u.z), x[3] = __uint_as_float(u.w);
  } else {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = to_f32<IO>((uint16_t)(w[i] & 0xFFFFu));
      x[2 * i + 1] = to_f32<IO>((uint16_t)(w[i] >> 16));
    }
  }
}

template <int IO, int V>
__device__ __forceinline__ void load_vec(const typename Elem<IO>::T* p, float (&x)[V]) {
  if constexpr (V == 1) widen<IO, V>(p[0], x);
  else widen<IO, V>(ldg16(p), x);
}
template <int IO, int V>
__device__ __forceinline__ void store_vec(typename Elem<IO>::T* p, const float (&x)[V]) {
  if constexpr (V == 1) {
    if constexpr (IO == DSA_DTYPE_F32) p[0] = x[0];
    else p[0] = from_f32<IO>(x[0]);
  } else if constexpr (IO == DSA_DTYPE_F32) {
    stg16(p, make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])));
  } else {
    stg16(p, make_uint4(pack2<IO>(x[0], x[1]), pack2<IO>(x[2], x[3]), pack2<IO>(x[4], x[5]), pack2<IO>(x[6], x[7])));
  }
}

}  // namespace dsa
