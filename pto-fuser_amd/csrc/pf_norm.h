// Root-mean-square norm with the residual's addition:
//   h = x + residual,  y = h * rsqrt(mean(h^2) + eps) * w,
// y rounded to the output's type, or to 8 bits (e4m3) with one fp32 scale a row or a block of 128 columns:
//   top = max |y|,  scale = top / 448,  code = e4m3(y * (448 / top)).
//
// One pass: a row stays in the registers of the threads that loaded it (VPT vectors of 16 bytes each), the sum of
// squares and the maximum are reduced across them in fp32, and y and h leave from the same registers.  h is rounded
// once, when it is stored; the norm is of the sum before that.
// Memory bound.  Measured, bf16 with a residual: 16384 x 2048, a wave a row, 50.5 us, 5.3 TB/s, a copy's rate;
// 8191 x 6144 to 8 bits in blocks of 128, a workgroup a row, 76 us, 4.7 TB/s.  Four rows: 5 us, latency.
#pragma once

#include "pf_serving.h"

namespace pf {

struct NormArgs {
  const void* x;
  const void* residual;   // may be null
  const void* w;
  void* y;                // output rows, or codes
  float* scales;          // fp8 only
  void* h;                // null without residual
  long x_row, r_row, y_row, h_row;
  int rows, D;
  int w_f32;
  float eps;
};

enum class NormOut { kPlain, kFp8Row, kFp8Block };

constexpr float kFp8Max = 448.f;

// Sum and maximum over the lanes of a segment of `lanes` (a power of two, at most 64).
__device__ __forceinline__ float lanes_sum(float v, int lanes) {
  for (int m = 1; m < lanes; m <<= 1) v += __shfl_xor(v, m);
  return v;
}
// Of the bits of |v|: as integers they order like the values, with NaN above infinity, so a NaN is kept.
__device__ __forceinline__ uint32_t lanes_max(uint32_t v, int lanes) {
  for (int m = 1; m < lanes; m <<= 1) v = max(v, (uint32_t)__shfl_xor((int)v, m));
  return v;
}

// TPR threads a row: a wave (four rows a workgroup) or a workgroup of its own.
template <typename E, typename R, typename O, NormOut OUT, int TPR, int VPT>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void norm_kernel(NormArgs a) {
  constexpr int V = 16 / sizeof(E);
  constexpr int ROWS = TPR < 256 ? 256 / TPR : 1, WAVES = TPR / 64;
  __shared__ uint32_t red[2 * (TPR / 64)];
  const int t = threadIdx.x % TPR;
  const long row = block_id() * ROWS + threadIdx.x / TPR;
  if (row >= a.rows) return;                        // whole waves, and with one row a workgroup whole workgroups
  const E* x = static_cast<const E*>(a.x) + row * a.x_row;
  const R* r = a.residual ? static_cast<const R*>(a.residual) + row * a.r_row : nullptr;
  const int D = a.D;

  float v[VPT][V];
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int d = (j * TPR + t) * V;
    if (d + V <= D) {
      load_vec<V>(x + d, v[j]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) v[j][i] = d + i < D ? to_f32(x[d + i]) : 0.f;
    }
  }
  if (r) {
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int d = (j * TPR + t) * V;
      if (d + V <= D) {
        float q[V];
        load_vec<V>(r + d, q);
#pragma unroll
        for (int i = 0; i < V; ++i) v[j][i] += q[i];
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (d + i < D) v[j][i] += to_f32(r[d + i]);
      }
    }
  }
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < VPT; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) sum = fmaf(v[j][i], v[j][i], sum);
  sum = lanes_sum(sum, 64);
  if constexpr (WAVES > 1) {
    if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = __float_as_uint(sum);
    __syncthreads();
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) sum += __uint_as_float(red[i]);
  }
  if (a.h) {
    R* h = static_cast<R*>(a.h) + row * a.h_row;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int d = (j * TPR + t) * V;
      if (d + V <= D) {
        store_vec<V>(h + d, v[j]);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (d + i < D) h[d + i] = from_f32<R>(v[j][i]);
      }
    }
  }
  const float inv = 1.f / sqrtf(sum / (float)D + a.eps);
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int d = (j * TPR + t) * V;
    if (d + V <= D) {
      float w[V];
      if (a.w_f32) load_vec<V>(static_cast<const float*>(a.w) + d, w);
      else load_vec<V>(static_cast<const E*>(a.w) + d, w);
#pragma unroll
      for (int i = 0; i < V; ++i) v[j][i] = v[j][i] * inv * w[i];
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (d + i < D) v[j][i] = v[j][i] * inv * load_any<E>(a.w, d + i, a.w_f32);
    }
  }

  if constexpr (OUT == NormOut::kPlain) {
    O* y = static_cast<O*>(a.y) + row * a.y_row;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int d = (j * TPR + t) * V;
      if (d + V <= D) {
        store_vec<V>(y + d, v[j]);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (d + i < D) y[d + i] = from_f32<O>(v[j][i]);
      }
    }
  } else {
    uint32_t top[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      top[j] = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) top[j] = max(top[j], __float_as_uint(v[j][i]) & 0x7fffffffu);
    }
    if constexpr (OUT == NormOut::kFp8Row) {
#pragma unroll
      for (int j = 1; j < VPT; ++j) top[0] = max(top[0], top[j]);
      top[0] = lanes_max(top[0], 64);
      if constexpr (WAVES > 1) {
        if (threadIdx.x % 64 == 0) red[WAVES + threadIdx.x / 64] = top[0];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WAVES; ++i) top[0] = max(top[0], red[WAVES + i]);
      }
      if (t == 0) a.scales[row] = __uint_as_float(top[0]) / kFp8Max;
    } else {
      constexpr int LANES = 128 / V;                // lanes that hold one block of 128 columns (D % 128 == 0)
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        top[j] = lanes_max(top[j], LANES);
        const int d = (j * TPR + t) * V;
        if (d < D && t % LANES == 0) a.scales[row * (D / 128) + d / 128] = __uint_as_float(top[j]) / kFp8Max;
      }
    }
    uint8_t* y = static_cast<uint8_t*>(a.y) + row * a.y_row;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int d = (j * TPR + t) * V;
      const float m = __uint_as_float(top[OUT == NormOut::kFp8Row ? 0 : j]);
      // a NaN stays one; a maximum so small that 448 / m overflows keeps its zeros zero
      float s = m == 0.f ? 0.f : kFp8Max / m;
      s = s > 3.4028235e38f ? 3.4028235e38f : s;
      uint32_t code[V / 4];
#pragma unroll
      for (int q = 0; q < V / 4; ++q) {
        const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[j][4 * q] * s, v[j][4 * q + 1] * s, 0, false);
        code[q] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[j][4 * q + 2] * s, v[j][4 * q + 3] * s, lo, true);
      }
      if (d + V <= D) {
        typedef uint32_t CodeVec __attribute__((ext_vector_type(V / 4), aligned(1)));
        CodeVec c;
#pragma unroll
        for (int q = 0; q < V / 4; ++q) c[q] = code[q];
        *reinterpret_cast<CodeVec*>(y + d) = c;
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (d + i < D) y[d + i] = (uint8_t)(code[i / 4] >> (8 * (i % 4)));
      }
    }
  }
}

}  // namespace pf
