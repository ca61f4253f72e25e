// Device helpers shared by the serving kernels (short convolution, single tokens, norm, state space scan).
#pragma once

#include "pf_device.h"

namespace pf {

// A launch counts its workgroups over x and y: a grid dimension holds fewer than 2^32 threads.
constexpr long kGridX = 1L << 20, kGridY = 65535;

__device__ __forceinline__ long block_id() { return (long)blockIdx.y * gridDim.x + blockIdx.x; }

// sigmoid(v) v.  exp(-v) = inf gives v * 0, so the far negative side ends in -0 and not in NaN.
__device__ __forceinline__ float silu(float v) { return v * __builtin_amdgcn_rcpf(1.f + __expf(-v)); }

// log(1 + e^v) = max(v, 0) + log(1 + u), u = e^-|v|.  1 + u keeps few digits of a small u (a step of 1e-3 would have
// four): the logarithm of the rounded w = 1 + u is scaled by u / (w - 1), which is exact to first order (Kahan's log1p).
__device__ __forceinline__ float softplus(float v) {
  const float u = __expf(-fabsf(v)), w = 1.f + u, d = w - 1.f;
  const float l = __logf(w) * (u * __builtin_amdgcn_rcpf(d));
  return fmaxf(v, 0.f) + (d == 0.f ? u : l);
}

// One value of a tensor that is fp32 or the operands' type.
template <typename E>
__device__ __forceinline__ float load_any(const void* p, size_t i, bool f32) {
  return f32 ? static_cast<const float*>(p)[i] : to_f32(static_cast<const E*>(p)[i]);
}

// V consecutive values at an address that promises an element's alignment only.
template <typename E, int V> struct VecAny {
  typedef E T __attribute__((ext_vector_type(V), aligned(sizeof(E))));
};
template <typename E> struct VecAny<E, 1> { typedef E T; };

template <typename E, int V>
__device__ __forceinline__ void expand(const typename VecAny<E, V>::T& x, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = to_f32(x);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = to_f32((E)x[i]);
  }
}

template <int V, typename E>
__device__ __forceinline__ void load_vec(const E* p, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = to_f32(*p);
  } else {
    const typename VecAny<E, V>::T x = *reinterpret_cast<const typename VecAny<E, V>::T*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = to_f32((E)x[i]);
  }
}

template <int V, typename E>
__device__ __forceinline__ void store_vec(E* p, const float (&v)[V]) {
  if constexpr (V == 1) {
    *p = from_f32<E>(v[0]);
  } else {
    typename VecAny<E, V>::T x;
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = from_f32<E>(v[i]);
    *reinterpret_cast<typename VecAny<E, V>::T*>(p) = x;
  }
}

}  // namespace pf
