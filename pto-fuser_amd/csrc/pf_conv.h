// Short causal convolution along the tokens, one filter of K taps a channel (depthwise), and its single-token form:
//   y[t] = act( bias + sum_k w[k] x[t - (K-1) + k] ),   act = silu or none,
// where tokens before the first are the rows of the state (the last K-1 inputs of what came before) or zero.
//
// Memory bound: 2K + 5 operations for two elements moved.  A thread owns VEC neighbouring channels (16 bytes) and TT
// consecutive tokens: all its rows are loaded before the first is used, the window of K rows slides through registers,
// and the K-1 rows before its tokens are read again (from the caches: the neighbouring thread's rows).
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
  int B, T, W;
  int vectors, tiles;
  int w_f32, act;
};

template <typename E, int K, int VEC, int TT>
__global__ __launch_bounds__(256) void conv_kernel(ConvArgs a) {
  const long id = block_id() * 256 + threadIdx.x;
  if (id >= a.threads) return;
  const int cv = (int)(id % a.vectors);
  const long rest = id / a.vectors;
  const int tile = (int)(rest % a.tiles), b = (int)(rest / a.tiles);
  const int c = cv * VEC, t0 = tile * TT;
  int n = a.T;
  if (a.lengths) n = min(max(a.lengths[b], 0), a.T);

  const E* x = static_cast<const E*>(a.x) + b * a.x_b + c;
  const E* si = a.state_in ? static_cast<const E*>(a.state_in) + b * a.si_b + c : nullptr;

  // rows t0 - (K-1) .. t0 + TT - 1
  float row[TT + K - 1][VEC];
#pragma unroll
  for (int j = 0; j < TT + K - 1; ++j) {
    const int t = t0 - (K - 1) + j;
#pragma unroll
    for (int i = 0; i < VEC; ++i) row[j][i] = 0.f;
    if (t >= 0) {
      if (t < n) load_vec<VEC>(x + t * a.x_t, row[j]);
    } else if (si) {
      load_vec<VEC>(si + (long)(t + K - 1) * a.W, row[j]);
    }
  }
  float w[K][VEC], bias[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
#pragma unroll
    for (int k = 0; k < K; ++k) w[k][i] = load_any<E>(a.w, (size_t)(c + i) * K + k, a.w_f32);
    bias[i] = a.bias ? load_any<E>(a.bias, c + i, a.w_f32) : 0.f;
  }
  E* y = static_cast<E*>(a.y) + b * a.y_b + c;
#pragma unroll
  for (int j = 0; j < TT; ++j) {
    const int t = t0 + j;
    if (t >= a.T) break;
    float o[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      o[i] = bias[i];
#pragma unroll
      for (int k = 0; k < K; ++k) o[i] = fmaf(w[k][i], row[j + k][i], o[i]);
      if (a.act) o[i] = silu(o[i]);
      if (t >= n) o[i] = 0.f;
    }
    store_vec<VEC>(y + t * a.y_t, o);
  }
  // The state after the last token.  The thread of the first tile writes it: it is the only one that reads the state
  // before, whose rows a prompt shorter than K-1 tokens still needs, and has them in its first registers.
  if (tile == 0 && a.state_out) {
    E* so = static_cast<E*>(a.state_out) + b * a.so_b + c;
#pragma unroll
    for (int r = 0; r < K - 1; ++r) {
      const int t = n - (K - 1) + r;
      float v[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = 0.f;
      if (t >= 0) {
        load_vec<VEC>(x + t * a.x_t, v);
      } else {
#pragma unroll
        for (int j = 0; j < K - 1; ++j)
          if (j == t + K - 1) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[i] = row[j][i];
          }
      }
      store_vec<VEC>(so + (long)r * a.W, v);
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
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      o[i] = a.bias ? load_any<E>(a.bias, c + i, a.w_f32) : 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k) o[i] = fmaf(load_any<E>(a.w, (size_t)(c + i) * K + k, a.w_f32), row[k][i], o[i]);
      if (a.act) o[i] = silu(o[i]);
    }
#pragma unroll
    for (int k = 1; k < K; ++k) store_vec<VEC>(s + (long)(k - 1) * a.W, row[k]);
  }
  store_vec<VEC>(static_cast<E*>(a.y) + b * a.y_b + c, o);
}

}  // namespace pf
