// Short causal convolution along the tokens, one filter of K taps a channel (depthwise), and its single-token form:
//   y[t] = act( bias + sum_k w[k] x[t - (K-1) + k] ),   act = silu or none,
// where tokens before the first are the rows of the state (the last K-1 inputs of what came before) or zero.
//
// Memory bound: 2K + 5 operations for two elements moved.  A thread owns VEC neighbouring channels (16 bytes) and TT
// consecutive tokens: all its rows are loaded before the first is used, the window of K rows slides through registers,
// and the K-1 rows before its tokens are read again (from the caches: the neighbouring thread's rows).
// Measured, 4 x 4096 x 6144 bf16, K = 4: 91 us, 4.4 TB/s of the 403 MB it cannot do without (a copy of that size reaches
// 5.3).  4 / 8 / 16 tokens a thread 105 / 92 / 91 us there, 11.6 / 12.7 / 15.9 at 3 x 1471 x 1920 fp32: 8.  The
// activation's exponential and quotient are what is left beside the memory.  One token of 64 sequences: 4.1 us, launch.
#pragma once

#include "pf_serving.h"

namespace pf {

struct ConvArgs {
  const void* x;
  const void* w;          // [W, K]
  const void* bias;       // [W] or null
  const void* state_in;   // [B, K-1, W] or null
  const int* lengths;     // [B] or null
  void* y;
  void* state_out;        // [B, K-1, W] or null; may be state_in
  long x_b, x_t, y_b, y_t;
  long si_b, so_b;
  long threads;           // B * tiles * vectors
  long blocks;            // of 256 threads
  int B, T, W;
  int vectors, tiles;
  int w_f32, act;
};

// The filters of VEC neighbouring channels: their K taps lie side by side, K vectors of VEC values.
template <typename E, int K, int VEC>
__device__ __forceinline__ void load_taps(const void* w, int c, bool f32, float (&tap)[K][VEC]) {
  float flat[K][VEC];
#pragma unroll
  for (int j = 0; j < K; ++j) {
    if (f32) load_vec<VEC>(static_cast<const float*>(w) + (size_t)c * K + j * VEC, flat[j]);
    else load_vec<VEC>(static_cast<const E*>(w) + (size_t)c * K + j * VEC, flat[j]);
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i)
#pragma unroll
    for (int k = 0; k < K; ++k) tap[k][i] = flat[(i * K + k) / VEC][(i * K + k) % VEC];
}
template <typename E, int VEC>
__device__ __forceinline__ void load_bias(const void* bias, int c, bool f32, float (&v)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = 0.f;
  if (bias) {
    if (f32) load_vec<VEC>(static_cast<const float*>(bias) + c, v);
    else load_vec<VEC>(static_cast<const E*>(bias) + c, v);
  }
}

template <typename E, int K, int VEC, int TT>
__global__ __launch_bounds__(256) void conv_kernel(ConvArgs a) {
  typedef typename VecAny<E, VEC>::T Vec;
  // Workgroups go round robin over the eight XCDs: each takes a run of them, so that the rows that two neighbouring
  // tiles both read come through one L2.
  const long per = (a.blocks + 7) / 8, block = (block_id() & 7) * per + (block_id() >> 3);
  const long id = block * 256 + threadIdx.x;
  if (block_id() >> 3 >= per || id >= a.threads) return;
  const int cv = (int)(id % a.vectors);
  const long rest = id / a.vectors;
  const int tile = (int)(rest % a.tiles), b = (int)(rest / a.tiles);
  const int c = cv * VEC, t0 = tile * TT;
  int n = a.T;
  if (a.lengths) n = min(max(a.lengths[b], 0), a.T);

  const E* x = static_cast<const E*>(a.x) + b * a.x_b + c;
  const E* si = a.state_in ? static_cast<const E*>(a.state_in) + b * a.si_b + c : nullptr;

  // rows t0 - (K-1) .. t0 + TT - 1, as they are stored
  Vec row[TT + K - 1];
  if (t0 >= K - 1 && t0 + TT <= n) {
    const E* p = x + (long)(t0 - (K - 1)) * a.x_t;
#pragma unroll
    for (int j = 0; j < TT + K - 1; ++j) row[j] = *reinterpret_cast<const Vec*>(p + j * a.x_t);
  } else {
#pragma unroll
    for (int j = 0; j < TT + K - 1; ++j) {
      const int t = t0 - (K - 1) + j;
      row[j] = Vec{};
      if (t >= 0) {
        if (t < n) row[j] = *reinterpret_cast<const Vec*>(x + t * a.x_t);
      } else if (si) {
        row[j] = *reinterpret_cast<const Vec*>(si + (long)(t + K - 1) * a.W);
      }
    }
  }
  float w[K][VEC], bias[VEC];
  load_taps<E, K, VEC>(a.w, c, a.w_f32, w);
  load_bias<E, VEC>(a.bias, c, a.w_f32, bias);
  float win[K][VEC];                            // the K rows of a token, in 32 bits; row j is at j % K
#pragma unroll
  for (int j = 0; j < K - 1; ++j) expand<E, VEC>(row[j], win[j]);
  E* y = static_cast<E*>(a.y) + b * a.y_b + c;
#pragma unroll
  for (int j = 0; j < TT; ++j) {
    const int t = t0 + j;
    expand<E, VEC>(row[j + K - 1], win[(j + K - 1) % K]);
    float o[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      o[i] = bias[i];
#pragma unroll
      for (int k = 0; k < K; ++k) o[i] = fmaf(w[k][i], win[(j + k) % K][i], o[i]);
      if (a.act) o[i] = silu(o[i]);
    }
    if (t >= n) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) o[i] = 0.f;
    }
    if (t < a.T) store_vec<VEC>(y + t * a.y_t, o);
  }
  // The state after the last token.  The thread of the first tile writes it: it is the only one that reads the state
  // before, whose rows a prompt shorter than K-1 tokens still needs, and has them in its first registers.
  if (tile == 0 && a.state_out) {
    E* so = static_cast<E*>(a.state_out) + b * a.so_b + c;
#pragma unroll
    for (int r = 0; r < K - 1; ++r) {
      const int t = n - (K - 1) + r;
      Vec v{};
      if (t >= 0) {
        v = *reinterpret_cast<const Vec*>(x + t * a.x_t);
      } else {
#pragma unroll
        for (int j = 0; j < K - 1; ++j)
          if (j == t + K - 1) v = row[j];
      }
      *reinterpret_cast<Vec*>(so + (long)r * a.W) = v;
    }
  }
}

struct ConvStepArgs {
  const void* x;          // [B, W]
  const void* w;
  const void* bias;
  void* state;            // [S, K-1, W], updated
  const int* slots;       // [B] or null (sequence b in slot b)
  void* y;                // [B, W]
  long x_b, y_b, s_b;
  long threads;
  int B, S, W, vectors;
  int w_f32, act;
};

// One token of each of B sequences.  A slot outside the pool is skipped, its y zero.
template <typename E, int K, int VEC>
__global__ __launch_bounds__(256) void conv_step_kernel(ConvStepArgs a) {
  const long id = block_id() * 256 + threadIdx.x;
  if (id >= a.threads) return;
  const int c = (int)(id % a.vectors) * VEC;
  const long b = id / a.vectors;
  const long slot = a.slots ? a.slots[b] : b;
  const bool live = slot >= 0 && slot < a.S;
  float o[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) o[i] = 0.f;
  if (live) {
    float row[K][VEC];
    E* s = static_cast<E*>(a.state) + slot * a.s_b + c;
#pragma unroll
    for (int k = 0; k < K - 1; ++k) load_vec<VEC>(s + (long)k * a.W, row[k]);
    load_vec<VEC>(static_cast<const E*>(a.x) + b * a.x_b + c, row[K - 1]);
    float w[K][VEC];
    load_taps<E, K, VEC>(a.w, c, a.w_f32, w);
    load_bias<E, VEC>(a.bias, c, a.w_f32, o);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
#pragma unroll
      for (int k = 0; k < K; ++k) o[i] = fmaf(w[k][i], row[k][i], o[i]);
      if (a.act) o[i] = silu(o[i]);
    }
#pragma unroll
    for (int k = 1; k < K; ++k) store_vec<VEC>(s + (long)(k - 1) * a.W, row[k]);
  }
  store_vec<VEC>(static_cast<E*>(a.y) + b * a.y_b + c, o);
}

}  // namespace pf
