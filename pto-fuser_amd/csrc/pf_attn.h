// Causal attention over packed prompts.  For query row i of a prompt, over its rows j <= i, with c = scale log2(e):
//   o_i = sum_j 2^{c (q_i . k_j - m_i)} v_j / l_i,     m_i a bound of q_i . k_j so far,  l_i = sum_j 2^{..}
// in one pass over the keys: m_i, l_i and o_i are carried, and o_i and l_i are scaled down when m_i has to grow.
//
// A workgroup's four waves own 32 query rows each: of four heads that share keys where there are as many, so that all four see
// as many keys, else of two heads or one; it walks the keys up to its last row in tiles.  The products are made
// transposed, S^T = K Q^T and O^T = V^T P^T, so that a lane holds ONE query's column of S^T: the maximum and the sum over
// keys are sums over its registers (and one swap with the other half of the wave), and the registers of P^T are at once the
// operand of the second product (permuted K: see pf_device.h).  K and V tiles go from global memory to LDS directly, double
// buffered, one barrier a tile.
//
// Rounding: scores, bounds, sums and outputs are fp32; with bf16 operands the weights enter the second product in bf16 (one
// rounding of 2^-9 to 2^-8 each: the output is 2.0e-3 of its norm off, 1.7e-3 by its own rounding alone).  A second term for
// them would cost half of that product again, which bounds the kernel; single tokens have it (pf_attn_step.h).
//
// Measured, bf16, D = 128: 1 prompt of 32768, 32 heads over 8 of keys, 7.57 to 8.12 ms by machine, 1085 to 1160 TFLOP/s; the library's
// product of 8192^3 reaches 1213 to 1224 on the same card.  Under it the shader clock falls to 1.6 GHz (12.3 million cycles a
// pass), of which the matrix pipes work 8.4 million, the vector port 7.4; L2 answers 96 % of the tiles.  4 x 4096 x 16 heads
// 262 to 281 us (980 to 1050 TFLOP/s): the diagonal's tiles and each workgroup's start and end.  D = 64: 2.2 ms for 1 x 32768 x
// 16, 1000 TFLOP/s: the vector port, with as many weights to half the products.  fp32, D = 128: 1.13 ms for 2 x 4096 x 16, 121 of
// the library's 154 TFLOP/s.  D = 256, a wave a SIMD (492 registers; fp32 512 and 36 spilled): bf16 610 TFLOP/s for 1 x 4096 x 16,
// 630 for 4 x 4096, 705 for 1 x 32768, fp32 103 to 107.  Tried on the way (4 x 4096 x 16, us): one wave a SIMD 603, two 297, loads
// in flight past the compiler's waits 274, tiles of 32 keys and three waves (168 registers, 9 spilled) 262; the diagonal's second half left out by a branch (spills, 310),
// the weights' sum by dot products of bf16 pairs (no gain), 128 rows of one head a workgroup instead of 32 of four (the
// same here, 48 prompts of up to 512 tokens 48 to 43).
#pragma once

#include "pf_gfx950.h"
#include "pf_serving.h"

#include <type_traits>

namespace pf {

typedef float floatx16 __attribute__((ext_vector_type(16)));

struct AttnArgs {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  const int* cu;           // [B + 1]: the prompts' rows
  const int* lengths;      // [B] or null: live rows of each
  long q_t, q_h, k_t, k_h, v_t, v_h, o_t, o_h;
  int N, B, H, G, D;
  int heads_log;           // log2 of the heads, that share one of keys, of a workgroup
  int rows_log;            // log2 of its query rows
  int tiles;               // of those rows, at most, plus one or more that find none
  int zero_rest;           // rows of no live token are written zero
  float scale_log2;
};

__device__ __forceinline__ floatx16 zero16() {
  floatx16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// The larger / the sum of a value in the two halves of a wave.
__device__ __forceinline__ float half_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Loads from global memory to LDS, N of 1 KiB each by a wave, 16 bytes a lane in order of the lanes, APART bytes of LDS from one
// to the next.  In assembly, since the compiler would wait for all of them before the next read of LDS, whatever buffer that is
// of; the caller waits (wait_loads) before it reads what they bring.  They write no register.  (s_nop: the distance from a
// scalar that a vector instruction has just written, and from m0, to a load.)
template <int N, int APART>
__device__ __forceinline__ void async_loads(const void* base, uint32_t lds, const uint32_t (&off)[N]) {
  const uint64_t at = (uint64_t)base;
  const u32x4 r = {(uint32_t)wave_int((int)at), (uint32_t)wave_int((int)(at >> 32)) & 0xffffu, 0x7fffffffu, 0x00020000u};
  const uint32_t m = (uint32_t)wave_int((int)lds);
  if constexpr (N == 1) {
    __asm__ __volatile__("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %2, %1, 0 offen lds"
                         :: "s"(m), "s"(r), "v"(off[0]) : "memory", "m0");
  } else if constexpr (N == 4) {
    __asm__ __volatile__(
        "s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %2, %1, 0 offen lds\n\t"
        "s_add_u32 m0, %0, %6\n\ts_nop 0\n\tbuffer_load_dwordx4 %3, %1, 0 offen lds\n\t"
        "s_add_u32 m0, %0, %7\n\ts_nop 0\n\tbuffer_load_dwordx4 %4, %1, 0 offen lds\n\t"
        "s_add_u32 m0, %0, %8\n\ts_nop 0\n\tbuffer_load_dwordx4 %5, %1, 0 offen lds"
        :: "s"(m), "s"(r), "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "n"(APART), "n"(2 * APART), "n"(3 * APART)
        : "memory", "m0", "scc");
  } else if constexpr (N == 8) {
    async_loads<4, APART>(base, lds, {off[0], off[1], off[2], off[3]});
    async_loads<4, APART>(base, lds + 4 * APART, {off[4], off[5], off[6], off[7]});
  } else {
    static_assert(N == 2, "one, two, four or eight loads");
    __asm__ __volatile__(
        "s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %2, %1, 0 offen lds\n\t"
        "s_add_u32 m0, %0, %4\n\ts_nop 0\n\tbuffer_load_dwordx4 %3, %1, 0 offen lds"
        :: "s"(m), "s"(r), "v"(off[0]), "v"(off[1]), "n"(APART) : "memory", "m0", "scc");
  }
}
// All of them, and this wave's reads of LDS.
__device__ __forceinline__ void wait_loads() {
  __asm__ __volatile__("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070);                // vmcnt 0, lgkmcnt 0
  __asm__ __volatile__("" ::: "memory");
}

// All but the last N.
template <int N> __device__ __forceinline__ void wait_all_but() {
  static_assert(N < 64, "six bits");
  __asm__ __volatile__("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | (N >> 4) << 14);
  __asm__ __volatile__("" ::: "memory");
}

__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}

// Rows of DP elements in LDS, their 16-byte chunks permuted by XOR with a function of the row, so that sixteen rows at one
// chunk (the operand of S^T) and four rows at four neighbouring chunks (the transposed one of O^T) meet no bank twice.
template <typename E, int DP> struct Rows {
  static constexpr int V = 16 / (int)sizeof(E), RB = DP * (int)sizeof(E), CHUNKS = RB / 16;
  __device__ __forceinline__ static constexpr int swizzle(int row) {
    if constexpr (RB > 512) return (row & 3) << 2;
    if constexpr (RB > 256) return ((row & 3) << 2) | ((row >> 2) & 1);     // (wide rows: two or four of 16 meet, beside products enough)
    if constexpr (RB == 256) return ((row & 3) << 2) | ((row >> 2) & 3);
    else return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
  }
  __device__ __forceinline__ static int at(int row, int col) { return row * DP + ((col / V) ^ swizzle(row)) * V + col % V; }
};

constexpr float kAttnRescale = 8.f;      // log2 by which scores may pass the carried maximum before it is moved

// Sums over the lanes of a wave up to each (inclusive): within rows of 16, then from row to row.
__device__ __forceinline__ int wave_sums(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);      // a row's last lane to the next row, of rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);      // lane 31 to rows 2 and 3
  return v;
}
__device__ __forceinline__ int wave_sum(int v) { return __builtin_amdgcn_readlane(wave_sums(v), 63); }

// Where a tile of the grid lies: prompt, first row within it.
struct AttnTile {
  int start, extent, len, row0;          // extent: rows up to the next prompt; len: live ones
  int excess, first, last;               // of a tile past all prompts: its number among those; the rows that prompts cover
  bool found, past;
};

// The longest tiles are to come first, and the shortest last, when the chip runs empty.  Up to 64 prompts, a lane each: the
// tiles are numbered by their place in the prompt, the last place first, over all prompts, and a search over places finds the
// tile.  More prompts: prompt b has tiles from cu[b] / rows + b on, which leaves it as many as it needs and one too many at most,
// so that a search in cu finds it.  (Offsets that fall find some prompt or none, inside the rows.)
__device__ __forceinline__ AttnTile find_tile(const AttnArgs& a, int tile) {
  const int lane = threadIdx.x & 63, log = a.rows_log, up = (1 << log) - 1;
  AttnTile t{};
  int b, place;
  if (a.B <= 64) {
    const int start = min(max(a.cu[min(lane, a.B)], 0), a.N), end = min(max(a.cu[min(lane + 1, a.B)], start), a.N);
    const int n = lane < a.B ? (end - start + up) >> log : 0;
    const auto from = [&](int p) { return wave_sum(max(n - p, 0)); };     // tiles at place p and later
    const int all = from(0);
    t.excess = tile - all;
    if (t.excess >= 0) {
      t.past = true;
      t.first = __builtin_amdgcn_readlane(start, 0);
      t.last = max(min(max(wave_int(a.cu[a.B]), 0), a.N), t.first);
      return t;
    }
    int lo = 0, hi = (a.N >> log) + 1, behind = 0;       // tiles from lo on are more than this one's number, from hi on `behind`
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2, count = from(mid);
      if (count > tile) {
        lo = mid;
      } else {
        hi = mid;
        behind = count;
      }
    }
    const unsigned long long here = __ballot(n > lo);
    const int rank = __builtin_amdgcn_mbcnt_hi((unsigned)(here >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)here, 0));
    const unsigned long long mine = __ballot(n > lo && rank == tile - behind);
    if (!mine) return t;
    b = __builtin_ctzll(mine);
    place = lo;
    t.start = __builtin_amdgcn_readlane(start, b);
    t.extent = __builtin_amdgcn_readlane(end, b) - t.start;
    t.found = true;
  } else {
    int lo = 0, count = a.B + 1;                     // entries of cu, the last of which at or before the tile is sought
    while (count > 1) {
      const int run = (count + 63) / 64, i = lo + min(lane * run, count - 1);
      const unsigned long long before = __ballot((min(max(a.cu[i], 0), a.N) >> log) + i <= tile && lane * run < count);
      const int l = before ? 63 - __builtin_clzll(before) : 0;
      lo += l * run;
      count = min(run, count - l * run);
    }
    const int start = min(max(wave_int(a.cu[lo]), 0), a.N), rank = tile - ((start >> log) + lo);
    if (lo == a.B) {
      t.past = true;
      t.excess = max(rank, 0);
      t.first = min(max(wave_int(a.cu[0]), 0), a.N);
      t.last = max(start, t.first);
      return t;
    }
    b = lo;
    t.start = start;
    t.extent = min(max(wave_int(a.cu[lo + 1]), start), a.N) - start;
    const int tiles = (t.extent + up) >> log;
    t.found = rank >= 0 && rank < tiles;
    place = tiles - 1 - rank;
  }
  t.row0 = place << log;
  t.len = t.extent;
  if (a.lengths) t.len = min(max(wave_int(a.lengths[b]), 0), t.extent);
  return t;
}

// Zeros in rows [from, to) of the output's heads from h on, by a workgroup.
template <typename E>
__device__ __forceinline__ void zero_rows(const AttnArgs& a, int h, long from, long to, long step, long rows) {
#pragma unroll 1
  for (long r0 = from; r0 < to; r0 += step) {
    const long n = min(to - r0, rows);
#pragma unroll 1
    for (long i = threadIdx.x; i < n * a.D << a.heads_log; i += blockDim.x) {
      const long r = i / a.D;
      static_cast<E*>(a.o)[(r0 + (r >> a.heads_log)) * a.o_t + (h + (r & ((1 << a.heads_log) - 1))) * a.o_h + i % a.D] = from_f32<E>(0.f);
    }
  }
}

template <typename E, int DP, int KW> struct AttnLds {
  static constexpr int BN = 32 * KW;                 // keys of a tile
  static constexpr int BUFS = KW == 4 ? 1 : 2;
  E k[BUFS][BN * DP], v[BUFS][BN * DP];
  float bounds[4][2][64];                            // of waves that share rows
};

// One workgroup's walk.  Returns whether an output came out not finite.  A value of v that is not finite reaches the queries
// before it through the products with the zeros above the diagonal: the walk is then made AGAIN, which leaves such values of
// the diagonal's tiles out of the products and adds them to the queries that see them.
template <typename E, int DP, int KW, bool AGAIN>
__device__ __forceinline__ bool attn_walk(const AttnArgs& a, AttnLds<E, DP, KW>& s, const AttnTile& t, const int h0) {
  using R = Rows<E, DP>;
  constexpr bool kBf = sizeof(E) == 2;
  constexpr int NW = 4, BN = AttnLds<E, DP, KW>::BN, RW = NW / KW, DT = DP / 32, ES = sizeof(E);
  constexpr int LOADS = BN * R::RB / 1024 / NW;      // 1 KiB each, of a wave and operand
  constexpr int QV = DP / (kBf ? 16 : 8);            // 16-byte vectors of a lane's query
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, hf = lane >> 5;
  const int g = wave_int(h0 / (a.H / a.G));
  // The wave's part of a tile's keys, its head and its first query.
  const int kw = w / RW, h = h0 + (w % RW & ((1 << a.heads_log) - 1)), q0 = t.row0 + (w % RW >> a.heads_log) * 32;

  const char* kg = reinterpret_cast<const char*>(static_cast<const E*>(a.k) + (long)t.start * a.k_t + g * a.k_h);
  const char* vg = reinterpret_cast<const char*>(static_cast<const E*>(a.v) + (long)t.start * a.v_t + g * a.v_h);
  const uint32_t kt = (uint32_t)a.k_t * ES, vt = (uint32_t)a.v_t * ES;
  const int rows_end = min(t.row0 + (1 << a.rows_log), t.len);      // keys that any query here sees
  const int n_tiles = (rows_end + BN - 1) / BN;

  // A lane's place in the loads of a tile: row and (swizzled) chunk, the same chunk for all LOADS.  Rows past the last live one
  // repeat it: they are masked.  Lanes whose columns lie past D stay out, and what they would fill stays zero.
  constexpr int FIRST = 1024 / R::RB;                // rows of a load
  const int l_row = w * FIRST + lane / R::CHUNKS, l_chunk = (lane % R::CHUNKS) ^ R::swizzle(l_row);
  static_assert(R::swizzle(NW * FIRST) == 0, "the swizzle is the same for a lane's rows");
  const uint32_t k_lds = lds_address(s.k[0]) + w * 1024, v_lds = lds_address(s.v[0]) + w * 1024;
  uint32_t k_off[LOADS], v_off[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    k_off[i] = (l_row + i * NW * FIRST) * kt + l_chunk * 16;
    v_off[i] = (l_row + i * NW * FIRST) * vt + l_chunk * 16;
  }
  const auto load = [&](int tile, int buf) {
    const int j0 = tile * BN, last = t.len - 1 - j0;
    if (l_chunk * R::V >= a.D) return;
    if (last >= BN - 1) {
      async_loads<LOADS, NW * 1024>(kg + (long)j0 * kt, k_lds + buf * BN * R::RB, k_off);
      async_loads<LOADS, NW * 1024>(vg + (long)j0 * vt, v_lds + buf * BN * R::RB, v_off);
    } else {
      uint32_t ko[LOADS], vo[LOADS];
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const uint32_t row = min(l_row + i * NW * FIRST, last);
        ko[i] = row * kt + l_chunk * 16;
        vo[i] = row * vt + l_chunk * 16;
      }
      async_loads<LOADS, NW * 1024>(kg + (long)j0 * kt, k_lds + buf * BN * R::RB, ko);
      async_loads<LOADS, NW * 1024>(vg + (long)j0 * vt, v_lds + buf * BN * R::RB, vo);
    }
  };

  // Four waves that share rows read nothing of each other's keys: each loads its own, K again as soon as the scores are made
  // and V as soon as the products are, into the one buffer of it, and there is no barrier.  Columns past D repeat the first.
  constexpr int OWN = KW == 4 ? 32 * R::RB / 1024 : 1;     // loads of a wave's 32 keys
  const int own_tiles = q0 >= 32 * kw ? (q0 - 32 * kw) / BN + 1 : 0;
  const auto own_load = [&](const char* from, uint32_t pitch, E* to, int tile) {
    const int j0 = tile * BN + 32 * kw, last = t.len - 1 - j0;
    uint32_t off[OWN];
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      const int row = i * FIRST + lane / R::CHUNKS, chunk = (lane % R::CHUNKS) ^ R::swizzle(row);
      off[i] = (uint32_t)min(row, last) * pitch + (chunk * R::V < a.D ? chunk * 16 : 0);
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);              // this wave's reads of the buffer
    async_loads<OWN, 1024>(from + (long)j0 * pitch, lds_address(to + 32 * kw * DP), off);
  };

  if constexpr (KW == 4) {
    if (own_tiles > 0) {
      own_load(kg, kt, s.k[0], 0);
      own_load(vg, vt, s.v[0], 0);
    }
  } else {
    load(0, 0);
  }

  // Q: a lane has row q0 + c; columns 16 kb + 8 hf .. (fp32: 8 kb + 4 hf ..)
  u32x4 q[QV];
  const E* qp = static_cast<const E*>(a.q) + (t.start + min(q0 + c, t.len - 1)) * a.q_t + h * a.q_h;
#pragma unroll
  for (int kb = 0; kb < QV; ++kb) {
    const int col = (kb * 2 + hf) * R::V;
    q[kb] = col < a.D ? *reinterpret_cast<const u32x4*>(qp + col) : u32x4{0, 0, 0, 0};
  }

  floatx16 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = zero16();
  float m = -INFINITY, l = 0.f;
  const float sc = a.scale_log2;

  // The wave's keys from jw on, in rows 32 kw .. of a tile; the hooks stand where its reads of K are made, before those of V
  // and after them.
  const auto work = [&](const int jw, const E* ks, const E* vs, auto k_read, auto v_next, auto v_read) {
    int row0 = 32 * kw;
    if constexpr (!kBf && DP == 256) __asm__ __volatile__("" : "+v"(row0));     // (places in LDS made anew: kept, they would spill)
    // With bf16 the operands are asked for AHEAD of the products, those of V before the weights, where registers allow it: at
    // D = 64, and at D = 128 where two waves share rows.  Else at D = 128 three waves a SIMD hide LDS for each other and
    // have no registers for that.  Past 128 columns it is not done (nor tried), nor with fp32, whose products outlast LDS.
    constexpr bool AHEAD = kBf && DP <= 128 && (KW > 1 || DP == 64);
    const auto k_at = [&](int kb) {
      const int col = (kb * 2 + hf) * R::V;
      const u32x4 f = *reinterpret_cast<const u32x4*>(ks + R::at(row0 + c, col));
      return KW == 4 && col >= a.D ? u32x4{0, 0, 0, 0} : f;
    };
    const int v_row = row0 + 4 * hf + ((lane & 15) >> 2), v_col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    const auto v_at = [&](int j, int dt) {
      const bf16* v = reinterpret_cast<const bf16*>(vs);
      return cat8(lds_read_tr(v + R::at(v_row + 16 * j, v_col + 32 * dt)), lds_read_tr(v + R::at(v_row + 16 * j + 8, v_col + 32 * dt)));
    };
    floatx16 st = zero16();
    u32x4 kf[AHEAD ? QV : 1];
    bf16x8 vf[AHEAD ? 2 : 1][AHEAD ? DT : 1];
    if constexpr (AHEAD) {
#pragma unroll
      for (int kb = 0; kb < QV; ++kb) kf[kb] = k_at(kb);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int kb = 0; kb < QV; ++kb) {
      const u32x4 f = AHEAD ? kf[AHEAD ? kb : 0] : k_at(kb);
      if constexpr (kBf) {
        st = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, f), __builtin_bit_cast(bf16x8, q[kb]), st, 0, 0, 0);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          st = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(f[i]), __uint_as_float(q[kb][i]), st, 0, 0, 0);
      }
    }
    k_read();
    if constexpr (AHEAD) {
      v_next();
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) vf[j][dt] = v_at(j, dt);
      __builtin_amdgcn_sched_barrier(0);
    }
    const bool masked = jw == q0;                    // on the diagonal
    if (masked) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (8 * (i / 4) + i % 4 > c - 4 * hf) st[i] = -INFINITY;
    }
    float top = st[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top = fmaxf(top, st[i]);
    top = half_max(top);
    if (__ballot((top - m) * sc > kAttnRescale)) {   // (-inf - -inf is no number and asks for nothing)
      const float up = fmaxf(top, m);
      const float f = m == -INFINITY ? 0.f : pow2((m - up) * sc);
      m = up;
      l *= f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] *= f;
    }
    const float off = m == -INFINITY ? 0.f : m * sc;
    float p[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      p[i] = pow2(__builtin_fmaf(st[i], sc, -off));
      l += p[i];
    }
    if constexpr (!AHEAD) v_next();
    if constexpr (kBf) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        bf16x8 pb;
#pragma unroll
        for (int i = 0; i < 8; ++i) pb[i] = (bf16)p[8 * j + i];
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          bf16x8 f = AHEAD ? vf[AHEAD ? j : 0][AHEAD ? dt : 0] : v_at(j, dt);
          if (AGAIN && masked) {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = __builtin_isfinite((float)f[i]) ? f[i] : (bf16)0.f;
          }
          o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f, pb, o[dt], 0, 0, 0);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int row = row0 + 8 * (i / 4) + 4 * hf + i % 4;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          float f = vs[R::at(row, 32 * dt + c)];
          if (AGAIN && masked) f = __builtin_isfinite(f) ? f : 0.f;
          o[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(f, p[i], o[dt], 0, 0, 0);
        }
      }
    }
    if (AGAIN && masked) {
#pragma unroll 1
      for (int j = 0; j < 32; ++j)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float x = to_f32(vs[R::at(row0 + j, 32 * dt + 8 * (i / 4) + 4 * hf + i % 4)]);
            if (!__builtin_isfinite(x) && j <= c) o[dt][i] += x;
          }
    }
    v_read();
  };
  if constexpr (KW == 4) {
    wait_loads();                                    // (the query: the compiler counts its own loads)
    for (int tile = 0; tile < own_tiles; ++tile) {
      const bool more = tile + 1 < own_tiles;
      wait_all_but<OWN>();                           // V is under way
      work(tile * BN + 32 * kw, s.k[0], s.v[0], [&] { if (more) own_load(kg, kt, s.k[0], tile + 1); },
           [&] { if (more) wait_all_but<OWN>(); else wait_all_but<0>(); },
           [&] { if (more) own_load(vg, vt, s.v[0], tile + 1); });
    }
  } else {
    const auto step = [&](const int tile, auto parity) {
      constexpr int buf = decltype(parity)::value;
      wait_loads();
      __builtin_amdgcn_s_barrier();
      __asm__ __volatile__("" ::: "memory");
      if (tile + 1 < n_tiles) load(tile + 1, buf ^ 1);
      const int jw = tile * BN + 32 * kw;
      const auto nothing = [] {};
      if (jw <= q0) work(jw, s.k[buf], s.v[buf], nothing, nothing, nothing);   // (multiples of 32: else nothing is visible)
    };
    for (int tile = 0; tile < n_tiles; tile += 2) {  // (twice, so that the buffers' addresses are constants)
      step(tile, std::integral_constant<int, 0>{});
      if (tile + 1 < n_tiles) step(tile + 1, std::integral_constant<int, 1>{});
    }
  }

  // Waves that share the rows: their sums at one bound, in the first of them.
  lds_barrier();
  l = half_sum(l);
  if constexpr (KW > 1) {
    floatx4* const sums = reinterpret_cast<floatx4*>(&s);
    static_assert((KW - 1) * RW * DT * 4 * 64 * 16 <= (int)sizeof(s) - (int)sizeof(s.bounds), "the sums fit");
    if (kw > 0) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4)
          sums[(((w - RW) * DT + dt) * 4 + i4) * 64 + lane] = floatx4{o[dt][4 * i4], o[dt][4 * i4 + 1], o[dt][4 * i4 + 2], o[dt][4 * i4 + 3]};
      s.bounds[w][0][lane] = m;
      s.bounds[w][1][lane] = l;
    }
    lds_barrier();
    if (kw == 0) {
      float up = m;
#pragma unroll
      for (int k = 1; k < KW; ++k) up = fmaxf(up, s.bounds[k * RW + w][0][lane]);
      const float own = m == -INFINITY ? 1.f : pow2((m - up) * sc);
      l *= own;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] *= own;
#pragma unroll
      for (int k = 1; k < KW; ++k) {
        const float mk = s.bounds[k * RW + w][0][lane], f = mk == -INFINITY ? 1.f : pow2((mk - up) * sc);
        l += s.bounds[k * RW + w][1][lane] * f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int i4 = 0; i4 < 4; ++i4) {
            const floatx4 x = sums[((((k - 1) * RW + w) * DT + dt) * 4 + i4) * 64 + lane];
#pragma unroll
            for (int i = 0; i < 4; ++i) o[dt][4 * i4 + i] = __builtin_fmaf(x[i], f, o[dt][4 * i4 + i]);
          }
      }
    }
    lds_barrier();
    if (kw > 0) return false;
  }
  // The output by way of LDS, where each wave has a quarter, so that it is stored in whole rows.
  E* const place = reinterpret_cast<E*>(&s) + w * BN * DP;
  typedef typename VecAny<E, R::V>::T Out;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  float spoilt = inv * 0.f;                          // 0 of finite values, else NaN
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4) {
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = o[dt][4 * i4 + i] * inv;
        spoilt = __builtin_fmaf(x[i], 0.f, spoilt);
      }
      store4(place + R::at(c, 32 * dt + 8 * i4 + 4 * hf), x[0], x[1], x[2], x[3]);
    }
  const bool bad = q0 + c < t.len && spoilt != 0.f;  // (NaN is unequal)
  const int rows = min(32, (a.zero_rest ? t.extent : t.len) - q0), live = t.len - q0;
  E* const to = static_cast<E*>(a.o) + (long)(t.start + q0) * a.o_t + h * a.o_h;
#pragma unroll
  for (int i = 0; i < 32 / FIRST; ++i) {
    const int r = i * FIRST + lane / R::CHUNKS, col = lane % R::CHUNKS * R::V;
    u32x4 x = *reinterpret_cast<const u32x4*>(place + R::at(r, col));
    if (r >= live) x = u32x4{0, 0, 0, 0};
    if (r < rows && col < a.D) *reinterpret_cast<Out*>(to + r * a.o_t + col) = __builtin_bit_cast(Out, x);
  }
  return bad;
}

template <typename E, int DP, int KW>
__global__ __launch_bounds__(256, DP == 256 || (sizeof(E) == 4 && DP == 128) ? 1 : KW > 1 ? 2 : 3) void attn_kernel(AttnArgs a) {
  __shared__ AttnLds<E, DP, KW> s;
  __shared__ int again;
  // Heads vary fastest, those of keys before those that share one, and go round robin over the eight XCDs: the workgroups that
  // read the same keys at the same time meet in few L2s.
  const uint32_t sets = (uint32_t)a.H >> a.heads_log, bid = block_id(), hi = bid % sets, tile = bid / sets;
  if (tile >= (uint32_t)a.tiles) return;
  const int h = wave_int(hi % (uint32_t)a.G * (a.H / a.G) + (hi / (uint32_t)a.G << a.heads_log));
  const AttnTile t = find_tile(a, wave_int(tile));
  if (t.past && a.zero_rest) {
    const long each = 64, step = (long)(a.tiles - ((int)tile - t.excess)) * each;
    zero_rows<E>(a, h, t.excess * each, t.first, step, each);
    zero_rows<E>(a, h, t.last + t.excess * each, a.N, step, each);
  }
  if (!t.found) return;
  if (t.row0 >= t.len) {
    if (a.zero_rest) {
      const long r = t.start + t.row0, n = min(t.extent - t.row0, 1 << a.rows_log);
      zero_rows<E>(a, h, r, r + n, n, n);
    }
    return;
  }
  const auto clear = [&] {                           // columns past D: no load writes them
    if (a.D == DP) return;
    u32x4* z = reinterpret_cast<u32x4*>(&s);
    for (int i = threadIdx.x; i < (int)(sizeof(s) / 16); i += 256) z[i] = u32x4{0, 0, 0, 0};
    lds_barrier();
  };
  clear();
  if (threadIdx.x == 0) again = 0;                   // (the walk's barriers lie between this and the next line)
  if (attn_walk<E, DP, KW, false>(a, s, t, h)) again = 1;
  lds_barrier();                                     // (the stores are under way: nobody waits for them)
  if (!again) return;
  __syncthreads();
  clear();
  attn_walk<E, DP, KW, true>(a, s, t, h);
}

}  // namespace pf
