// One token of the recurrences with a matrix state S [rows, cols] per sequence and head (fp32, updated in place):
//   state space   S <- e^{dt A} S + B (dt x)^T,                       y = C^T S + D x  (times silu(z))
//   delta rule    S <- e^g S,  r = beta (v - k^T S),  S <- S + k r^T,  o = scale q^T S  (g of the head or of the row)
//
// Memory bound: 8 bytes of state move for 5 to 7 operations.  The columns of S are independent, so a workgroup takes
// all rows of 4 * LPR columns, holds them in registers (one read and one write of the state), and needs one exchange
// between its threads.  The products with the new state come from the decayed one, S' = e^g S, without a second exchange:
//   C^T S = C^T S' + (C . B) dt x,     q^T S = q^T S' + (q . k) r.
// Measured: state space, 64 sequences x 32 heads of 128 x 64: 28.4 us, 4.8 TB/s of state (a copy of its size reaches 5.3);
// delta rule, 64 x 16 heads of 128 x 128: 30.3 us, 4.5 TB/s; a single sequence of 32 heads 6 us, latency.  Workgroups of
// 16 / 32 / 64 columns: 44.5 / 28.4 / 39.5 us and 40.1 / 30.3 / 40.3: half a line a row is too little to ask for at once, and
// 64 columns leave each thread eight rows, whose registers halve the waves in flight.  32.
#pragma once

#include "pf_serving.h"

namespace pf {

struct StepArgs {
  float* state;           // [S, H, N, P]
  const int* slots;       // [B] or null
  const void* v;          // x or v   [B, H, P]
  const void* k;          // B or k   [B, G, N]
  const void* q;          // C or q   [B, G, N]
  void* y;                // [B, H, P]: E (state space) or fp32 (delta rule)
  const void* dt;         // state space: [B, H], E or fp32
  const void* z;          // state space: [B, H, P] or null
  const float* a;         // state space: A [H]
  const float* d;         // state space: D [H] or null
  const float* dt_bias;   // state space: [H] or null
  const float* beta;      // delta rule: [B, H]
  const float* g;         // delta rule: [B, H], or [B, H, N] with g_rows, or null
  long v_b, v_h, k_b, k_h, q_b, q_h, y_b, y_h, dt_b, dt_h, z_b, z_h;
  long s_b;               // state elements of one slot
  long blocks;            // B * H * slices
  int S, H, G, N, P;
  int slices;             // column slices of one head
  int dt_f32, softplus, g_rows;
  float scale;
};

template <typename E, bool DELTA, int LPR, int RPT>
__global__ __launch_bounds__(256) void step_kernel(StepArgs a) {
  constexpr int COLS = 4 * LPR, RP = 256 / LPR;      // columns of the slice, rows of one pass
  __shared__ floatx4 part[2][4][LPR];
  __shared__ float dots[4];
  const long block = block_id();
  if (block >= a.blocks) return;
  const int slice = (int)(block % a.slices);
  const long bh = block / a.slices;
  const int h = (int)(bh % a.H);
  const long b = bh / a.H;
  const int col = threadIdx.x % LPR, row0 = threadIdx.x / LPR, wave = threadIdx.x / 64;
  const int p = slice * COLS + 4 * col;
  const bool in = p < a.P;                           // P % 4 == 0: a thread's four columns are in or out together
  const long slot = a.slots ? a.slots[b] : b;
  if (slot < 0 || slot >= a.S) {                     // not a slot of the pool: skipped, y zero
    if (row0 == 0 && in) {
      const float zero[4] = {0.f, 0.f, 0.f, 0.f};
      if constexpr (DELTA) store_vec<4>(static_cast<float*>(a.y) + b * a.y_b + h * a.y_h + p, zero);
      else store_vec<4>(static_cast<E*>(a.y) + b * a.y_b + h * a.y_h + p, zero);
    }
    return;
  }
  const int g = h / (a.H / a.G);
  float* st = a.state + slot * a.s_b + (long)h * a.N * a.P + p;
  const E* kp = static_cast<const E*>(a.k) + b * a.k_b + g * a.k_h;
  const E* qp = static_cast<const E*>(a.q) + b * a.q_b + g * a.q_h;

  floatx4 s[RPT];
  float k[RPT], q[RPT];
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int n = row0 + i * RP;
    s[i] = zero4();
    if (in && n < a.N) s[i] = *reinterpret_cast<const floatx4_any*>(st + (long)n * a.P);
  }
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int n = row0 + i * RP;
    k[i] = n < a.N ? to_f32(kp[n]) : 0.f;
    q[i] = n < a.N ? to_f32(qp[n]) : 0.f;
  }
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  if (in) load_vec<4>(static_cast<const E*>(a.v) + b * a.v_b + h * a.v_h + p, x);
  float decay = 1.f, dt = 0.f;
  if constexpr (!DELTA) {
    dt = load_any<E>(a.dt, b * a.dt_b + h * a.dt_h, a.dt_f32);
    if (a.dt_bias) dt += a.dt_bias[h];
    if (a.softplus) dt = softplus(dt);
    decay = __expf(dt * a.a[h]);
  } else if (a.g && !a.g_rows) {
    decay = __expf(a.g[bh]);
  }
  floatx4 ks = zero4(), qs = zero4();
  float kq = 0.f;
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    float e = decay;
    if constexpr (DELTA) {
      if (a.g_rows) {
        const int n = row0 + i * RP;
        e = n < a.N ? __expf(a.g[bh * a.N + n]) : 0.f;
      }
    }
    s[i] *= e;
    if constexpr (DELTA) ks += s[i] * k[i];
    qs += s[i] * q[i];
    kq = fmaf(k[i], q[i], kq);
  }
  // Sums over the rows: of one wave by exchange between its lanes, of the four waves through LDS.
#pragma unroll
  for (int m = LPR; m < 64; m <<= 1) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (DELTA) ks[j] += __shfl_xor(ks[j], m);
      qs[j] += __shfl_xor(qs[j], m);
    }
    kq += __shfl_xor(kq, m);
  }
  if (threadIdx.x % 64 < LPR) {
    if constexpr (DELTA) part[0][wave][col] = ks;
    part[1][wave][col] = qs;
    if (col == 0) dots[wave] = kq;
  }
  __syncthreads();
  kq = dots[0] + dots[1] + dots[2] + dots[3];
  qs = part[1][0][col] + part[1][1][col] + part[1][2][col] + part[1][3][col];
  floatx4 r;
  if constexpr (DELTA) {
    ks = part[0][0][col] + part[0][1][col] + part[0][2][col] + part[0][3][col];
    const float beta = a.beta[bh];
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = beta * (x[j] - ks[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = dt * x[j];
  }
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int n = row0 + i * RP;
    s[i] += r * k[i];
    if (in && n < a.N) *reinterpret_cast<floatx4_any*>(st + (long)n * a.P) = s[i];
  }
  if (row0 == 0 && in) {
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = fmaf(kq, r[j], qs[j]);
    if constexpr (DELTA) {
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] *= a.scale;
      store_vec<4>(static_cast<float*>(a.y) + b * a.y_b + h * a.y_h + p, y);
    } else {
      if (a.d) {
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = fmaf(a.d[h], x[j], y[j]);
      }
      if (a.z) {
        float z[4];
        load_vec<4>(static_cast<const E*>(a.z) + b * a.z_b + h * a.z_h + p, z);
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] *= silu(z[j]);
      }
      store_vec<4>(static_cast<E*>(a.y) + b * a.y_b + h * a.y_h + p, y);
    }
  }
}

}  // namespace pf
