// Selective state space scan over prompts, in chunks of Q = 64 tokens.  Per head, with dt the (softplus of the) step,
// G = cumulative sum of dt A within the chunk and S [N, P] the state in fp32:
//   y_i = e^{G_i} (C_i^T S) + sum_{j <= i} e^{G_i - G_j} dt_j (C_i . B_j) x_j + D x_i,     y *= silu(z)
//   S  <- e^{G_last} S + sum_t B_t (e^{G_last - G_t} dt_t x_t)^T
// B and C belong to a group of heads, so the score C B^T is the same for all of them.
//
// A workgroup walks the chunks of one (sequence, group, block of heads): NW waves, each the owner of 32 columns of one
// head.  A wave's state stays in its registers as MFMA results S[n, p] (rows n, column p a lane), which are at once the
// operand of y^T = S^T C^T; y^T = x^T P^T takes the score tiles the same way, so the only exchanges are the staged rows
// of B and C and the score tiles, which the waves compute together.  (Permuted K: see pf_device.h.)
//
// Few sequences do not fill the chip with whole walks.  A sequence then runs as segments side by side, in three launches:
// the state each segment adds by itself (kStates: no C, no score), the states that enter the segments (a sum along the
// segments, ssm_prefix_kernel), and the outputs (kOutput from those states).
#pragma once

#include "pf_gfx950.h"
#include "pf_serving.h"

namespace pf {

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

constexpr int kSsmChunk = 64;

struct SsmArgs {
  const void* x;
  const void* dt;
  const void* b;
  const void* c;
  const void* z;           // or null
  const float* a;
  const float* d;          // or null
  const float* dt_bias;    // or null
  const float* h0;         // [B, H, N, P] or null
  const int* lengths;      // [B] or null
  void* y;
  float* h_final;          // or null; may be h0
  float* seg_state;        // [B, H, segs, N, P]: what a segment adds, then what enters it
  float* seg_decay;        // [B, H, segs]: log2 of a segment's decay
  long x_b, x_h, x_t, dt_b, dt_h, dt_t, b_b, b_g, b_t, c_b, c_g, c_t, z_b, z_h, z_t, y_b, y_h, y_t;
  long tasks;              // B * G * head blocks * segments
  int B, H, G, T, N, P;
  int heads;               // heads of a workgroup
  int blocks;              // blocks of heads of a group
  int segs, seg_chunks;
  int dt_f32, softplus;
};

enum class SsmMode { kStates, kOutput };

// ---- one MFMA operand of 32 contraction rows: eight values a lane ---------------------------
template <typename E> struct Frag;
template <> struct Frag<bf16> { bf16x8 v; };
template <> struct Frag<float> { floatx4 lo, hi; };

__device__ __forceinline__ floatx4 mfma32(const Frag<bf16>& a, const Frag<bf16>& b, floatx4 acc) {
  return mfma_bf16(a.v, b.v, acc);
}
__device__ __forceinline__ floatx4 mfma32(const Frag<float>& a, const Frag<float>& b, floatx4 acc) {
#pragma unroll
  for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.lo[i], b.lo[i], acc, 0, 0, 0);
#pragma unroll
  for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.hi[i], b.hi[i], acc, 0, 0, 0);
  return acc;
}

// Two MFMA results as the operand that contracts over their 32 rows.
template <typename E> __device__ __forceinline__ Frag<E> frag_of(const floatx4& lo, const floatx4& hi);
template <> __device__ __forceinline__ Frag<bf16> frag_of<bf16>(const floatx4& lo, const floatx4& hi) { return {pack8(lo, hi)}; }
template <> __device__ __forceinline__ Frag<float> frag_of<float>(const floatx4& lo, const floatx4& hi) { return {lo, hi}; }

// ---- LDS tiles ------------------------------------------------------------------------------
// Rows of B or C, [64][NT].  bf16: within each 32 columns the eight 4-column units are stored in the order 0 4 1 5 2 6 3 7,
// so that lane group g finds its two units (4g.., 16 + 4g..) side by side; the rows are 16 bytes apart modulo the banks.
template <typename E, int NT> struct RowTile {
  static constexpr int LD = NT + 16 / (int)sizeof(E);
  static constexpr int ELEMS = kSsmChunk * LD;
  // 16 bytes of row `row`, column vector `vec`
  __device__ __forceinline__ static void put(E* s, int row, int vec, const u32x4& v) {
    if constexpr (sizeof(E) == 2) {
      const int q = vec & 3;                               // units 2q and 2q + 1
      E* p = s + row * LD + (vec >> 2) * 32 + 4 * ((q & 1) * 4 + (q >> 1));
      *reinterpret_cast<u32x2*>(p) = u32x2{v[0], v[1]};
      *reinterpret_cast<u32x2*>(p + 8) = u32x2{v[2], v[3]};
    } else {
      *reinterpret_cast<u32x4*>(s + row * LD + vec * 4) = v;
    }
  }
  // operand: lane c holds row `row`, lane group g its eight of columns 32 kb ..
  __device__ __forceinline__ static Frag<E> rows(const E* s, int row, int kb, int g) {
    if constexpr (sizeof(E) == 2) {
      return {*reinterpret_cast<const bf16x8*>(s + row * LD + kb * 32 + g * 8)};
    } else {
      const E* p = s + row * LD + kb * 32 + g * 4;
      return {*reinterpret_cast<const floatx4*>(p), *reinterpret_cast<const floatx4*>(p + 16)};
    }
  }
  // transposed operand: lane c holds column 16 nt + c, lane group g its eight of rows 32 kb ..
  __device__ __forceinline__ static Frag<E> cols(const E* s, int nt, int kb, int c, int g) {
    if constexpr (sizeof(E) == 2) {
      const E* p = s + (32 * kb + 4 * g + (c >> 2)) * LD + (nt >> 1) * 32 + 4 * (2 * (c & 3) + (nt & 1));
      return {cat8(lds_read_tr(p), lds_read_tr(p + 16 * LD))};
    } else {
      const E* p = s + (32 * kb + 4 * g) * LD + 16 * nt + c;
      Frag<E> f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f.lo[i] = p[i * LD];
        f.hi[i] = p[(16 + i) * LD];
      }
      return f;
    }
  }
};

// A wave's 32 columns of x, [64][32].
template <typename E> struct XTile {
  static constexpr int LD = 32 + 16 / (int)sizeof(E);
  static constexpr int ELEMS = kSsmChunk * LD;
  // operand: lane c holds column 16 pt + c, lane group g its eight of rows 32 kb ..
  __device__ __forceinline__ static Frag<E> cols(const E* s, int pt, int kb, int c, int g) {
    if constexpr (sizeof(E) == 2) {
      const E* p = s + (32 * kb + 4 * g + (c >> 2)) * LD + 16 * pt + 4 * (c & 3);
      return {cat8(lds_read_tr(p), lds_read_tr(p + 16 * LD))};
    } else {
      const E* p = s + (32 * kb + 4 * g) * LD + 16 * pt + c;
      Frag<E> f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f.lo[i] = p[i * LD];
        f.hi[i] = p[(16 + i) * LD];
      }
      return f;
    }
  }
};

// acc += A (x scaled by its rows' weights): the weighted operand in SPLIT bf16 terms, each the rounding of what the ones
// before it left (8, 16 or 24 bits of the product); fp32 needs none.
template <int SPLIT> struct Weighted {
  Frag<bf16> t[SPLIT];
  __device__ __forceinline__ Weighted(const Frag<bf16>& x, const floatx4& w0, const floatx4& w1) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v = (float)x.v[i] * (i < 4 ? w0[i & 3] : w1[i & 3]);
#pragma unroll
      for (int k = 0; k < SPLIT; ++k) {
        const bf16 r = (bf16)v;
        t[k].v[i] = r;
        v -= (float)r;
      }
    }
  }
  __device__ __forceinline__ floatx4 times(const Frag<bf16>& a, floatx4 acc) const {
#pragma unroll
    for (int k = SPLIT - 1; k >= 0; --k) acc = mfma32(a, t[k], acc);
    return acc;
  }
};
struct WeightedF32 {
  Frag<float> t;
  __device__ __forceinline__ WeightedF32(const Frag<float>& x, const floatx4& w0, const floatx4& w1) : t{x.lo * w0, x.hi * w1} {}
  __device__ __forceinline__ floatx4 times(const Frag<float>& a, floatx4 acc) const { return mfma32(a, t, acc); }
};
template <typename E, int SPLIT> struct WeightedOf { typedef Weighted<SPLIT> T; };
template <int SPLIT> struct WeightedOf<float, SPLIT> { typedef WeightedF32 T; };

template <typename E, int NT, int NW> struct SsmLds {
  E b[RowTile<E, NT>::ELEMS];
  E c[RowTile<E, NT>::ELEMS];
  E x[NW][XTile<E>::ELEMS];
  floatx4 score[10][64];            // C B^T, tile (ib, jb): lane (c, g) holds rows j = 16 jb + 4 g .. of column i = 16 ib + c
  float tab[NW][4][kSsmChunk];      // per token: G, dt, dt 2^(G_m - G) (m: last token of its 16), dt 2^(G_last - G)
};

// SPLIT: bf16 terms of the weighted x in the state's update.  Three keep the state a sum in 24 bits, as it has to be where
// it is returned; two where it only enters y, whose operand S is rounded to 8 bits anyway.
template <typename E, int NT, int NW, SsmMode MODE, int SPLIT>
__global__ __launch_bounds__(NW * 64) void ssm_kernel(SsmArgs a) {
  using Rows = RowTile<E, NT>;
  using Xs = XTile<E>;
  constexpr int Q = kSsmChunk, V = 16 / (int)sizeof(E), TH = NW * 64;
  constexpr int RV = NT / V;                   // vectors of a row of B or C
  constexpr int NB = Q * RV / TH;              // of them a thread
  constexpr int XV = 32 / V;                   // vectors of a row of a wave's x
  constexpr int NX = Q * XV / 64;
  constexpr bool OUT = MODE == SsmMode::kOutput;
  __shared__ __attribute__((aligned(16))) SsmLds<E, NT, NW> s;

  // Workgroups go round robin over the eight XCDs: each XCD takes a run of tasks, whose neighbours (the blocks of heads
  // of one group's segment) read the same B and C through its L2.
  const long per = (a.tasks + 7) / 8;
  const long task = (block_id() % 8) * per + block_id() / 8;
  if (block_id() / 8 >= per || task >= a.tasks) return;
  const int hb = (int)(task % a.blocks);
  long rest = task / a.blocks;
  const int seg = (int)(rest % a.segs);
  rest /= a.segs;
  const int grp = (int)(rest % a.G);
  const long bi = rest / a.G;

  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
  const int R = a.H / a.G;
  const int hl = w * 32 / a.P, p0 = w * 32 % a.P;
  const bool active = hl < a.heads && hb * a.heads + hl < R;
  const int h = grp * R + (active ? hb * a.heads + hl : 0);
  const int N = a.N, P = a.P;
  int len = a.T;
  if (a.lengths) len = min(max(a.lengths[bi], 0), a.T);

  const E* xg = static_cast<const E*>(a.x) + bi * a.x_b + h * a.x_h + p0;
  const E* bg = static_cast<const E*>(a.b) + bi * a.b_b + grp * a.b_g;
  const E* cg = static_cast<const E*>(a.c) + bi * a.c_b + grp * a.c_g;
  const float a2 = active ? a.a[h] * 1.44269504f : 0.f;
  const float dbias = active && a.dt_bias ? a.dt_bias[h] : 0.f;

  // ---- what a chunk loads: rows of B and C by all threads, its x by each wave, dt a token a lane
  u32x4 rb[NB], rc[NB], rx[NX];
  float rdt = 0.f;
  auto load = [&](int t0) {
    const int valid = len - t0;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int v = threadIdx.x + i * TH, row = v / RV, col = (v % RV) * V;
      rb[i] = u32x4{0, 0, 0, 0};
      if (OUT) rc[i] = u32x4{0, 0, 0, 0};
      if (row < valid && col < N) {
        rb[i] = *reinterpret_cast<const u32x4_any*>(bg + (t0 + row) * a.b_t + col);
        if (OUT) rc[i] = *reinterpret_cast<const u32x4_any*>(cg + (t0 + row) * a.c_t + col);
      }
    }
#pragma unroll
    for (int i = 0; i < NX; ++i) {
      const int v = lane + i * 64, row = v / XV, col = (v % XV) * V;
      rx[i] = u32x4{0, 0, 0, 0};
      if (active && row < valid) rx[i] = *reinterpret_cast<const u32x4_any*>(xg + (t0 + row) * a.x_t + col);
    }
    rdt = 0.f;
    if (active && lane < valid) rdt = load_any<E>(a.dt, bi * a.dt_b + h * a.dt_h + (t0 + lane) * a.dt_t, a.dt_f32);
  };

  floatx4 S[NT / 16][2];
#pragma unroll
  for (int nt = 0; nt < NT / 16; ++nt)
#pragma unroll
    for (int pt = 0; pt < 2; ++pt) S[nt][pt] = zero4();
  if (OUT && active) {
    const float* in = a.segs > 1 ? a.seg_state + (((long)bi * a.H + h) * a.segs + seg) * N * P
                                 : (a.h0 ? a.h0 + ((long)bi * a.H + h) * N * P : nullptr);
    if (in) {
#pragma unroll
      for (int nt = 0; nt < NT / 16; ++nt)
#pragma unroll
        for (int pt = 0; pt < 2; ++pt)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int n = 16 * nt + 4 * g + r;
            if (n < N) S[nt][pt][r] = in[(long)n * P + p0 + 16 * pt + c];
          }
    }
  }

  const int chunks = (a.T + Q - 1) / Q;
  const int first = seg * a.seg_chunks, end = min(first + a.seg_chunks, chunks);
  float decay2 = 0.f;                          // kStates: log2 of the segment's decay
  if (first < end) load(first * Q);
  for (int ch = first; ch < end; ++ch) {
    const int t0 = ch * Q;
    lds_barrier();                             // the last chunk's reads are done
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int v = threadIdx.x + i * TH;
      Rows::put(s.b, v / RV, v % RV, rb[i]);
      if (OUT) Rows::put(s.c, v / RV, v % RV, rc[i]);
    }
#pragma unroll
    for (int i = 0; i < NX; ++i) {
      const int v = lane + i * 64;
      *reinterpret_cast<u32x4*>(&s.x[w][(v / XV) * Xs::LD + (v % XV) * V]) = rx[i];
    }
    // the chunk's step sizes and decays, a token a lane, in log2
    float dt = rdt + dbias;
    if (a.softplus) dt = softplus(dt);
    if (t0 + lane >= len) dt = 0.f;
    const float gate = dt * a2;
    float G = gate, after = gate;              // sums up to here, and from here on
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const float up = __shfl_up(G, m), down = __shfl_down(after, m);
      if (lane >= m) G += up;
      if (lane + m < 64) after += down;
    }
    const float total = __shfl(G, 63);
    s.tab[w][0][lane] = G;
    s.tab[w][1][lane] = dt;
    s.tab[w][2][lane] = dt * exp2f(__shfl(G, lane | 15) - G);
    s.tab[w][3][lane] = dt * exp2f(after - gate);
    lds_barrier();
    if (ch + 1 < end) load(t0 + Q);

    Frag<E> xf[2][2];
#pragma unroll
    for (int pt = 0; pt < 2; ++pt)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) xf[pt][kb] = Xs::cols(s.x[w], pt, kb, c, g);

    if constexpr (OUT) {
      // the score's tiles, dealt over the waves
#pragma unroll
      for (int k = 0; k < (10 + NW - 1) / NW; ++k) {
        const int tile = w + k * NW;
        if (tile < 10) {
          const int ib = tile >= 6 ? 3 : tile >= 3 ? 2 : tile >= 1 ? 1 : 0, jb = tile - ib * (ib + 1) / 2;
          floatx4 acc = zero4();
#pragma unroll
          for (int kb = 0; kb < NT / 32; ++kb)
            acc = mfma32(Rows::rows(s.b, 16 * jb + c, kb, g), Rows::rows(s.c, 16 * ib + c, kb, g), acc);
          s.score[tile][lane] = acc;
        }
      }
      // y^T = S^T C^T
      floatx4 y[2][4];
#pragma unroll
      for (int pt = 0; pt < 2; ++pt)
#pragma unroll
        for (int ib = 0; ib < 4; ++ib) y[pt][ib] = zero4();
#pragma unroll
      for (int kb = 0; kb < NT / 32; ++kb) {
        const Frag<E> s0 = frag_of<E>(S[2 * kb][0], S[2 * kb + 1][0]), s1 = frag_of<E>(S[2 * kb][1], S[2 * kb + 1][1]);
#pragma unroll
        for (int ib = 0; ib < 4; ++ib) {
          const Frag<E> cf = Rows::rows(s.c, 16 * ib + c, kb, g);
          y[0][ib] = mfma32(s0, cf, y[0][ib]);
          y[1][ib] = mfma32(s1, cf, y[1][ib]);
        }
      }
      lds_barrier();                           // the score is whole
      floatx4 u[4];
#pragma unroll
      for (int jb = 0; jb < 4; ++jb) u[jb] = *reinterpret_cast<const floatx4*>(&s.tab[w][2][16 * jb + 4 * g]);
#pragma unroll
      for (int ib = 0; ib < 4; ++ib) {
        const float Gi = s.tab[w][0][16 * ib + c];
        const float e = exp2f(Gi);
        y[0][ib] *= e;
        y[1][ib] *= e;
        floatx4 pr[4];
#pragma unroll
        for (int jb = 0; jb < 4; ++jb) {
          pr[jb] = zero4();
          if (jb < ib) {
            const float f = exp2f(Gi - s.tab[w][0][16 * jb + 15]);
            pr[jb] = s.score[ib * (ib + 1) / 2 + jb][lane] * (u[jb] * f);
          } else if (jb == ib) {
            const floatx4 sc = s.score[ib * (ib + 1) / 2 + jb][lane];
            const floatx4 Gj = *reinterpret_cast<const floatx4*>(&s.tab[w][0][16 * jb + 4 * g]);
            const floatx4 dj = *reinterpret_cast<const floatx4*>(&s.tab[w][1][16 * jb + 4 * g]);
#pragma unroll
            for (int r = 0; r < 4; ++r) pr[jb][r] = 4 * g + r <= c ? sc[r] * (dj[r] * exp2f(Gi - Gj[r])) : 0.f;
          }
        }
#pragma unroll
        for (int kb = 0; kb <= ib / 2; ++kb) {
          const Frag<E> pf = frag_of<E>(pr[2 * kb], pr[2 * kb + 1]);
          y[0][ib] = mfma32(xf[0][kb], pf, y[0][ib]);
          y[1][ib] = mfma32(xf[1][kb], pf, y[1][ib]);
        }
      }
      // y out: lane c's token, four columns of each tile
      if (active) {
        const float dd = a.d ? a.d[h] : 0.f;
#pragma unroll
        for (int ib = 0; ib < 4; ++ib) {
          const int t = t0 + 16 * ib + c;
          if (t < a.T) {
#pragma unroll
            for (int pt = 0; pt < 2; ++pt) {
              float v[4], xr[4];
#pragma unroll
              for (int r = 0; r < 4; ++r) xr[r] = to_f32(s.x[w][(16 * ib + c) * Xs::LD + 16 * pt + 4 * g + r]);
#pragma unroll
              for (int r = 0; r < 4; ++r) v[r] = fmaf(dd, xr[r], y[pt][ib][r]);
              if (a.z) {
                float z[4];
                load_vec<4>(static_cast<const E*>(a.z) + bi * a.z_b + h * a.z_h + t * a.z_t + p0 + 16 * pt + 4 * g, z);
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] *= silu(z[r]);
              }
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (t >= len) v[r] = 0.f;
              store_vec<4>(static_cast<E*>(a.y) + bi * a.y_b + h * a.y_h + t * a.y_t + p0 + 16 * pt + 4 * g, v);
            }
          }
        }
      }
    }

    // S <- e^{G_last} S + B^T (w x)
    const float e = exp2f(total);
    decay2 += total;
#pragma unroll
    for (int nt = 0; nt < NT / 16; ++nt) {
      S[nt][0] *= e;
      S[nt][1] *= e;
    }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const floatx4 w0 = *reinterpret_cast<const floatx4*>(&s.tab[w][3][32 * kb + 4 * g]);
      const floatx4 w1 = *reinterpret_cast<const floatx4*>(&s.tab[w][3][32 * kb + 16 + 4 * g]);
      const typename WeightedOf<E, SPLIT>::T wx0(xf[0][kb], w0, w1), wx1(xf[1][kb], w0, w1);
#pragma unroll
      for (int nt = 0; nt < NT / 16; ++nt) {
        const Frag<E> bf = Rows::cols(s.b, nt, kb, c, g);
        S[nt][0] = wx0.times(bf, S[nt][0]);
        S[nt][1] = wx1.times(bf, S[nt][1]);
      }
    }
  }

  float* out = nullptr;
  if (OUT) {
    if (a.segs == 1 && a.h_final) out = a.h_final + ((long)bi * a.H + h) * N * P;
  } else {
    out = a.seg_state + (((long)bi * a.H + h) * a.segs + seg) * N * P;
    if (active && p0 == 0 && lane == 0) a.seg_decay[((long)bi * a.H + h) * a.segs + seg] = decay2;
  }
  if (active && out) {
#pragma unroll
    for (int nt = 0; nt < NT / 16; ++nt)
#pragma unroll
      for (int pt = 0; pt < 2; ++pt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int n = 16 * nt + 4 * g + r;
          if (n < N) out[(long)n * P + p0 + 16 * pt + c] = S[nt][pt][r];
        }
  }
}

// The states that enter the segments, in place of what each adds: H_0 = h0, H_{s+1} = decay_s H_s + D_s; the last is the
// final state.  A thread owns four neighbouring elements; the segments' values are loaded eight ahead of the sum.
__global__ __launch_bounds__(256) void ssm_prefix_kernel(SsmArgs a) {
  const long vecs = (long)a.N * a.P / 4, id = block_id() * 256 + threadIdx.x;
  if (id >= vecs * a.B * a.H) return;
  const long bh = id / vecs, at = id % vecs * 4;
  const long step = (long)a.N * a.P;
  float* st = a.seg_state + bh * a.segs * step + at;
  const float* decay = a.seg_decay + bh * a.segs;
  floatx4 H = zero4();
  if (a.h0) H = *reinterpret_cast<const floatx4_any*>(a.h0 + bh * step + at);
  constexpr int AHEAD = 8;
  for (int s0 = 0; s0 < a.segs; s0 += AHEAD) {
    floatx4 D[AHEAD];
    float e[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (s0 + i < a.segs) {
        D[i] = *reinterpret_cast<const floatx4*>(st + (s0 + i) * step);
        e[i] = exp2f(decay[s0 + i]);
      }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (s0 + i < a.segs) {
        *reinterpret_cast<floatx4*>(st + (s0 + i) * step) = H;
        H = H * e[i] + D[i];
      }
  }
  if (a.h_final) *reinterpret_cast<floatx4_any*>(a.h_final + bh * step + at) = H;
}

}  // namespace pf
