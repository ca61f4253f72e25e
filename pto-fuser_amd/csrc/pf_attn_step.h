// One new token of each of B sequences over a cache of keys and values in pages:
//   o = sum_j 2^{c (q . k_j - m)} v_j / l over the sequence's tokens j,  c = scale log2(e),  m a bound,  l the sum of weights.
//
// Bound by the bytes of the cache, each read once: the query heads that share a head of keys are the columns of one 16-wide
// product (transposed as in pf_attn.h: S^T = K Q^T, O^T = V^T P^T).  The walk is cut evenly, whatever the lengths: the keys
// of all sequences and heads, in units of 64, are one line of which each workgroup takes an equal run.  A (sequence, head)
// that ends up in several workgroups leaves partial sums there, which a second kernel joins.  Each wave walks its own 32 keys
// of a unit, through buffers of its own, the next ones under way to LDS; waves meet only at a segment's end.  With bf16
// operands the weights enter the second product in two terms of bf16, which costs nothing beside the memory (1 %).  Sums that
// are not finite are made again (step_keys); that they are looked for costs a short call 0.1 to 0.3 us, a long one nothing.
//
// Measured, bf16, D = 128: 64 sequences of up to 8192, 4 heads of keys, 504 MB, 99 to 104 us and 4.5 to 5.7 the join (4.6 to 4.8
// TB/s together; a copy moves 5.05); 1 of 131072, 8 heads, 537 MB, 101 to 105 and 4.8.  Two workgroups of two waves a CU;
// one of four: 114 and 130.  A short call is a chain of latencies: 1 of 512 tokens 6.4 us and 2.9 us the join, and 13.4 us
// in one workgroup a head.  When a walk is shared out: step_shares in pf_attn.hip.
#pragma once

#include "pf_attn.h"

namespace pf {

constexpr int kStepWaves = 2;
constexpr int kStepUnit = 32 * kStepWaves;           // keys: 32 of each wave

struct AttnStepArgs {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  const int* tables;       // [S, M]: a sequence's pages
  const int* lengths;      // [B]
  const int* slots;        // [B] or null
  float* part;             // [2 wgs][16][DP + 4]: sums, then the bound and the weights' sum
  int* spread;             // [rows][4]: of a (sequence, head, block) its first part, the workgroups of the first and last one
  long q_b, q_h, o_b, o_h, k_p, k_r, k_h, v_p, v_r, v_h;
  int B, S, H, G, D, M, pages, page_log;
  int blocks;              // of 16 of a group's query heads
  int wgs;                 // that share the walk; 0: a workgroup a (sequence, head, block)
  float scale_log2;
};

// Tokens of a sequence that the cache holds.
__device__ __forceinline__ int cached(const AttnStepArgs& a, int b) {
  if (a.slots) {
    const int s = a.slots[b];
    if (s < 0 || s >= a.S) return 0;
  }
  return a.pages > 0 ? (int)min((long)max(a.lengths[b], 0), (long)a.M << a.page_log) : 0;
}
// Its units, one of them of an empty sequence, whose output somebody has to write.
__device__ __forceinline__ int units_of(int len) { return max((len - 1) / kStepUnit + 1, 1); }

// A workgroup's run on the line of units, and where it begins.  (The host keeps the line to 2^30 units.)
struct StepRun {
  int per, begin, end;     // units of a run; this one's
  int b, before, len;      // the sequence that the first of them lies in, the units before that, its tokens
};
// Up to 64 sequences, a lane each: their lengths are asked for once.  More: once for all, then 64 at a time up to the one.
__device__ __forceinline__ StepRun find_run(const AttnStepArgs& a, int wg) {
  const int lane = threadIdx.x & 63, each = a.G * a.blocks;
  StepRun r{};
  int len = lane < a.B ? cached(a, lane) : 0;
  int n = lane < a.B ? units_of(len) : 0, upto = wave_sums(n), total = __builtin_amdgcn_readlane(upto, 63);
  if (a.B > 64) {
    int rest = 0;
#pragma unroll 4
    for (int b = 64 + lane; b < a.B; b += 64) rest += units_of(cached(a, b));
    total += wave_sum(rest);
  }
  total *= each;
  r.per = (total + a.wgs - 1) / a.wgs;
  if ((long)wg * r.per >= total) return r;
  const int x = wg * r.per / each;                   // in units of all heads
  int before = 0;
  for (int b0 = 0; b0 < a.B;) {
    const unsigned long long behind = __ballot(before + upto > x);
    if (behind) {
      const int l = __builtin_ctzll(behind);
      r.begin = wg * r.per;
      r.end = min(r.begin + r.per, total);
      r.b = b0 + l;
      r.before = (before + __builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(n, l)) * each;
      r.len = __builtin_amdgcn_readlane(len, l);
      return r;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
    b0 += 64;
    len = b0 + lane < a.B ? cached(a, b0 + lane) : 0;
    n = b0 + lane < a.B ? units_of(len) : 0;
    upto = wave_sums(n);
  }
  return r;
}

template <typename E, int DP> struct StepLds {
  static constexpr int KEYS = sizeof(E) == 2 ? 32 : 16;    // of a wave's step
  E k[kStepWaves][2][KEYS * DP];
  union {
    E v[kStepWaves][2][KEYS * DP];
    float o[kStepWaves][16 * (DP + 4)];                      // the waves' sums
  };
  float m[kStepWaves][16], l[kStepWaves][16];
  int again;                                                 // a sum came out not finite
};

// The keys [k0, k1) of one (sequence, head, block) by a workgroup; len: the sequence's.  Returns whether a sum came out not
// finite.  A value of v that is not finite meets weights that are no token's (0 times it is no number), and the second term of
// a weight, which may have the other sign (inf - inf): the keys are then walked AGAIN, where keys that are no token's have
// no values, and the second term no value that is not finite.
template <typename E, int DP, bool AGAIN>
__device__ __forceinline__ bool step_keys(const AttnStepArgs& a, StepLds<E, DP>& s, const int b, const int g, const int hb,
                                          const int len, const int k0, const int k1, float* part) {
  using R = Rows<E, DP>;
  constexpr bool kBf = sizeof(E) == 2;
  constexpr int ES = sizeof(E), KEYS = StepLds<E, DP>::KEYS, KG = KEYS / 16, DT = DP / 16;
  constexpr int QV = DP / (kBf ? 32 : 16);
  constexpr int FIRST = 1024 / R::RB, LOADS = 16 / FIRST;   // rows of a load; loads of a 16-key group
  constexpr int N = LOADS > 4 ? 4 : LOADS;
  const int tid = threadIdx.x, lane = tid & 63, w = wave_int(tid >> 6), c = lane & 15, gr = lane >> 4;
  const int share = a.H / a.G, heads = min(16, share - 16 * hb);
  const int slot = wave_int(a.slots ? a.slots[b] : b);
  // (through the scalar cache, whose loads are not counted with those of keys and values)
  const auto* table = (const __attribute__((address_space(4))) int*)(a.tables + (long)slot * a.M);

  u32x4 q[QV];
  const E* qp = static_cast<const E*>(a.q) + b * a.q_b + (g * share + 16 * hb + min(c, heads - 1)) * a.q_h;
#pragma unroll
  for (int kb = 0; kb < QV; ++kb) {
    const int col = (kb * 4 + gr) * R::V;
    q[kb] = col < a.D ? *reinterpret_cast<const u32x4*>(qp + col) : u32x4{0, 0, 0, 0};
  }
  floatx4 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = zero4();
  float m = -INFINITY, l = 0.f;
  const float sc = a.scale_log2;
  const char* kg = static_cast<const char*>(a.k) + g * a.k_h * ES;
  const char* vg = static_cast<const char*>(a.v) + g * a.v_h * ES;
  const uint32_t kr = (uint32_t)a.k_r * ES, vr = (uint32_t)a.v_r * ES;

  // A lane's place in a group's loads.  Columns past D repeat the first ones; they are left out where K is read.
  uint32_t l_row[LOADS], l_chunk[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    l_row[i] = i * FIRST + lane / R::CHUNKS;
    l_chunk[i] = (lane % R::CHUNKS) ^ R::swizzle(l_row[i]);
    if ((int)l_chunk[i] * R::V >= a.D) l_chunk[i] = 0;
  }

  struct Stage {
    int j;
    bool ok[KG], any;
  };
  // The pages of a step's groups: -1 past the sequence's end and where a page is outside the pool.
  const auto entries = [&](int j, int (&page)[KG]) {
#pragma unroll
    for (int t = 0; t < KG; ++t) {
      const int key = j + 16 * t;
      page[t] = key < len ? table[key >> a.page_log] : -1;
      if (page[t] >= a.pages) page[t] = -1;
    }
  };
  // A step's loads.  A group without a page takes the rows of the other, and weighs nothing; without either, page 0's.
  const auto issue = [&](int j, const int (&page)[KG], int buf, Stage& st) {
    st.j = j;
    st.any = false;
#pragma unroll
    for (int t = 0; t < KG; ++t) {
      st.ok[t] = page[t] >= 0;
      st.any |= st.ok[t];
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);              // this wave's reads of the buffer
#pragma unroll
    for (int t = 0; t < KG; ++t) {
      const int u = st.ok[t] ? t : KG - 1 - t, key = j + 16 * u;
      const long p = st.any ? page[st.ok[t] ? t : KG - 1 - t] : 0;
      const int row = st.any ? key & ((1 << a.page_log) - 1) : 0, last = st.any ? len - 1 - key : 15;
      const char* kp = kg + (p * a.k_p + row * a.k_r) * ES;
      const char* vp = vg + (p * a.v_p + row * a.v_r) * ES;
      uint32_t ko[LOADS], vo[LOADS];
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const uint32_t r = min((int)l_row[i], last);
        ko[i] = r * kr + l_chunk[i] * 16;
        vo[i] = r * vr + l_chunk[i] * 16;
      }
      const uint32_t kl = lds_address(&s.k[w][buf][16 * t * DP]), vl = lds_address(&s.v[w][buf][16 * t * DP]);
#pragma unroll
      for (int i = 0; i < LOADS; i += N) {
        uint32_t kn[N], vn[N];
#pragma unroll
        for (int x = 0; x < N; ++x) {
          kn[x] = ko[i + x];
          vn[x] = vo[i + x];
        }
        async_loads<N, 1024>(kp, kl + i * 1024, kn);
        async_loads<N, 1024>(vp, vl + i * 1024, vn);
      }
    }
  };

  const auto is_token = [&](const Stage& stage, int t, int i) { return stage.ok[t] && stage.j + 16 * t + 4 * gr + i < len; };
  const auto compute = [&](const Stage& stage, int buf) {
    if (!stage.any) return;
    const E* ks = s.k[w][buf];
    const E* vs = s.v[w][buf];
    floatx4 st[KG];
#pragma unroll
    for (int t = 0; t < KG; ++t) {
      st[t] = zero4();
#pragma unroll
      for (int kb = 0; kb < QV; ++kb) {
        u32x4 f = *reinterpret_cast<const u32x4*>(ks + R::at(16 * t + c, (kb * 4 + gr) * R::V));
        if ((kb * 4 + gr) * R::V >= a.D) f = u32x4{0, 0, 0, 0};
        if constexpr (kBf) {
          st[t] = mfma_bf16(__builtin_bit_cast(bf16x8, f), __builtin_bit_cast(bf16x8, q[kb]), st[t]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            st[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(f[i]), __uint_as_float(q[kb][i]), st[t], 0, 0, 0);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (!is_token(stage, t, i)) st[t][i] = -INFINITY;
    }
    float top = st[0][0];
#pragma unroll
    for (int t = 0; t < KG; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, st[t][i]);
    top = fmaxf(top, __shfl_xor(top, 16));
    top = half_max(top);
    if (__ballot((top - m) * sc > kAttnRescale)) {
      const float up = fmaxf(top, m), f = m == -INFINITY ? 0.f : pow2((m - up) * sc);
      m = up;
      l *= f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] *= f;
    }
    const float off = m == -INFINITY ? 0.f : m * sc;
    floatx4 p[KG];
#pragma unroll
    for (int t = 0; t < KG; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[t][i] = pow2(__builtin_fmaf(st[t][i], sc, -off));
        l += p[t][i];
      }
    bf16x8 hi, lo;                                   // the weights in two terms of bf16
    if constexpr (kBf) {
      hi = pack8(p[0], p[KG - 1]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[0][i] -= (float)hi[i];
        p[KG - 1][i] -= (float)hi[4 + i];
      }
      lo = pack8(p[0], p[KG - 1]);
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      if constexpr (kBf) {
        const int row = 4 * gr + (c >> 2), col = 16 * dt + 4 * (c & 3);
        bf16x8 f = cat8(lds_read_tr(vs + R::at(row, col)), lds_read_tr(vs + R::at(row + 16, col))), finite = f;
        if constexpr (AGAIN) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (!is_token(stage, i / 4, i % 4)) f[i] = (bf16)0.f;
            finite[i] = __builtin_isfinite((float)f[i]) ? f[i] : (bf16)0.f;
          }
        }
        o[dt] = mfma_bf16(f, hi, mfma_bf16(finite, lo, o[dt]));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float f = vs[R::at(4 * gr + i, 16 * dt + c)];
          if (AGAIN && !is_token(stage, 0, i)) f = 0.f;
          o[dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(f, p[0][i], o[dt], 0, 0, 0);
        }
      }
    }
  };

  // Two steps in flight: while one is worked on the next is loaded, whose pages were asked for a step before.
  const int first = k0 + w * KEYS, count = first < k1 ? (k1 - first + kStepWaves * KEYS - 1) / (kStepWaves * KEYS) : 0;
  if (count > 0) {
    int page[KG];
    Stage now, next;
    entries(first, page);
    wait_loads();                                    // (the query: the compiler counts its own loads)
    issue(first, page, 0, now);
    if (count > 1) entries(first + kStepWaves * KEYS, page);
    for (int i = 0; i < count; ++i) {
      const int buf = i & 1;
      if (i + 1 < count) {
        const int j = first + (i + 1) * kStepWaves * KEYS;
        issue(j, page, buf ^ 1, next);
        if (i + 2 < count) entries(j + kStepWaves * KEYS, page);
        wait_all_but<2 * KG * LOADS>();
      } else {
        wait_all_but<0>();
      }
      compute(now, buf);
      now = next;
    }
  }

  // The waves' sums over their keys, at one bound.
  l += __shfl_xor(l, 16);
  l = half_sum(l);
  __syncthreads();                                   // (the sums take the place of V)
  if (gr == 0) {
    s.m[w][c] = m;
    s.l[w][c] = l;
  }
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<floatx4*>(&s.o[w][c * (DP + 4) + 16 * dt + 4 * gr]) = o[dt];
  if (tid == 0) s.again = 0;
  __syncthreads();
  float spoilt = 0.f;                                // 0 of finite sums, else NaN
  for (int i = tid; i < heads * (DP / 4); i += 64 * kStepWaves) {
    const int r = i / (DP / 4), col = i % (DP / 4) * 4;
    float up = s.m[0][r];
#pragma unroll
    for (int k = 1; k < kStepWaves; ++k) up = fmaxf(up, s.m[k][r]);
    floatx4 sum = zero4();
    float weight = 0.f;
#pragma unroll
    for (int k = 0; k < kStepWaves; ++k) {
      const float f = s.m[k][r] == -INFINITY ? 1.f : pow2((s.m[k][r] - up) * sc);
      sum += *reinterpret_cast<const floatx4*>(&s.o[k][r * (DP + 4) + col]) * f;
      weight += s.l[k][r] * f;
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) spoilt = __builtin_fmaf(sum[x], 0.f, spoilt);
    if (part) {
      *reinterpret_cast<floatx4*>(part + r * (DP + 4) + col) = sum;
      if (col == 0) {
        part[r * (DP + 4) + DP] = up;
        part[r * (DP + 4) + DP + 1] = weight;
      }
    } else if (col < a.D) {
      const float inv = weight == 0.f ? 0.f : 1.f / weight;
      const float out[4] = {sum[0] * inv, sum[1] * inv, sum[2] * inv, sum[3] * inv};
      store_vec<4>(static_cast<E*>(a.o) + b * a.o_b + (g * share + 16 * hb + r) * a.o_h + col, out);
    }
  }
  if (spoilt != 0.f) s.again = 1;                    // (NaN is unequal)
  __syncthreads();
  return s.again;                                    // (set to 0 next behind another barrier)
}

template <typename E, int DP>
__device__ __forceinline__ void step_segment(const AttnStepArgs& a, StepLds<E, DP>& s, const int b, const int g, const int hb,
                                             const int len, const int k0, const int k1, float* part) {
  if (step_keys<E, DP, false>(a, s, b, g, hb, len, k0, k1, part)) step_keys<E, DP, true>(a, s, b, g, hb, len, k0, k1, part);
}

template <int DP> __device__ __forceinline__ float* part_of(const AttnStepArgs& a, long i) { return a.part + i * 16 * (DP + 4); }

template <typename E, int DP>
__global__ __launch_bounds__(64 * kStepWaves) void attn_step_kernel(AttnStepArgs a) {
  __shared__ StepLds<E, DP> s;
  const int each = a.G * a.blocks, wg = (int)block_id();
  if (!a.wgs) {
    const int b = wg / each, u = wg % each;
    if (b >= a.B) return;
    const int len = wave_int(cached(a, b));
    step_segment<E, DP>(a, s, b, u / a.blocks, u % a.blocks, len, 0, len, nullptr);
    return;
  }
  if (wg >= a.wgs) return;
  const StepRun run = find_run(a, wg);
  int x = run.begin, b = run.b, len = run.len, off = x - run.before;
  while (x < run.end && b < a.B) {
    const int n = units_of(len), u = off / n, i0 = off % n, count = min(n - i0, run.end - x);
    const int mine = 2 * wg + (x == run.begin ? 0 : 1);
    float* part = count == n ? nullptr : part_of<DP>(a, mine);
    if (i0 == 0 && threadIdx.x == 0) {               // (for the kernel that joins)
      int* to = a.spread + 4L * (b * each + u);
      to[0] = mine;
      to[1] = wg;
      to[2] = (x + n - 1) / run.per;
    }
    step_segment<E, DP>(a, s, b, u / a.blocks, u % a.blocks, len, i0 * kStepUnit, min(len, (i0 + count) * kStepUnit), part);
    x += count;
    off += count;
    if (off == n * each) {
      off = 0;
      ++b;
      if (x < run.end && b < a.B) len = wave_int(cached(a, b));
    }
  }
}

// A query head of a (sequence, head, block) that lies in several workgroups' runs: their partial sums, joined.  The parts are
// shared out over eight groups of lanes, each of which holds a row, and the groups' sums meet in LDS.
template <typename E, int DP>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnStepArgs a) {
  constexpr int LANES = DP / 4, GROUPS = 256 / LANES;
  __shared__ floatx4 sums[GROUPS][LANES];
  __shared__ float bounds[GROUPS], weights[GROUPS];
  const int share = a.H / a.G, each = a.G * a.blocks;
  const int head = (int)block_id(), b = head / a.H, g = head % a.H / share, hr = head % share, hb = hr / 16, r = hr % 16;
  if (b >= a.B) return;
  // The first part is its workgroup's last piece, unless it begins that run; in the others it is the first.
  const int* spread = a.spread + 4L * (b * each + g * a.blocks + hb);
  const int p0 = spread[0], w0 = spread[1], w1 = spread[2], grp = threadIdx.x / LANES, col = threadIdx.x % LANES * 4;
  if (w0 == w1) return;
  const float sc = a.scale_log2;
  floatx4 sum = zero4();
  float up = -INFINITY, weight = 0.f;
#pragma unroll 4
  for (int w = w0 + grp; w <= w1; w += GROUPS) {
    const float* p = part_of<DP>(a, w == w0 ? p0 : 2 * w) + r * (DP + 4);
    const float m = p[DP], l = p[DP + 1];
    const floatx4 x = *reinterpret_cast<const floatx4*>(p + col);
    const float top = fmaxf(up, m);
    const float f = up == -INFINITY ? 1.f : pow2((up - top) * sc), fw = m == -INFINITY ? 1.f : pow2((m - top) * sc);
    sum = sum * f + x * fw;
    weight = weight * f + l * fw;
    up = top;
  }
  sums[grp][threadIdx.x % LANES] = sum;
  if (col == 0) {
    bounds[grp] = up;
    weights[grp] = weight;
  }
  __syncthreads();
  if (grp != 0) return;
  float top = up;
#pragma unroll
  for (int i = 1; i < GROUPS; ++i) top = fmaxf(top, bounds[i]);
  sum = zero4();
  weight = 0.f;
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) {
    const float f = bounds[i] == -INFINITY ? 1.f : pow2((bounds[i] - top) * sc);
    sum += sums[i][threadIdx.x] * f;
    weight += weights[i] * f;
  }
  if (col < a.D) {
    const float inv = weight == 0.f ? 0.f : 1.f / weight;
    const float out[4] = {sum[0] * inv, sum[1] * inv, sum[2] * inv, sum[3] * inv};
    store_vec<4>(static_cast<E*>(a.o) + b * a.o_b + (g * share + hr) * a.o_h + col, out);
  }
}

}  // namespace pf
