// Selective state space scan over prompts, in chunks of Q = 64 tokens.  Per head, with dt the (softplus of the) step,
// G = cumulative sum of dt A within the chunk and S [N, P] the state in fp32:
//   y_i = e^{G_i} (C_i^T S) + sum_{j <= i} e^{G_i - G_j} dt_j (C_i . B_j) x_j + D x_i,     y *= silu(z)
//   S  <- e^{G_last} S + sum_t B_t (e^{G_last - G_t} dt_t x_t)^T
// B and C belong to a group of heads, so the score C B^T is the same for all of them.
//
// A workgroup walks the chunks of one (sequence, group, block of columns): NW waves, each the owner of 16 or 32 columns
// of one head.  A wave's state stays in its registers as MFMA results S[n, p] (rows n, column p a lane), which are at once the
// operand of y^T = S^T C^T; y^T = x^T P^T takes the score tiles the same way, so the only exchanges are the staged rows
// of B and C and the score tiles, which the waves compute together.  (Permuted K: see pf_device.h.)
//
// Few sequences do not fill the chip with whole walks.  A sequence then runs as segments side by side, in three launches:
// the state each segment adds by itself (kStates: no C, no score), the states that enter the segments (a sum along the
// segments, ssm_prefix_kernel), and the outputs (kOutput from those states).
//
// Rounding, bf16 operands: S and the decayed score enter the products for y in two bf16 terms each, 16 bits, so that y is
// off by its own rounding to 8 bits (1.66e-3 of its norm; with one term each 1.75e-3 where D x is most of y, 2.0e-3 to
// 2.4e-3 else, at 100 and 204 us against 105 and 215 for 2 x 8192 and 32768 tokens); the state is a sum in fp32 of
// products whose weighted operand has 16 or 24 bits (SPLIT).
// fp32 operands: fp32 matrix instructions throughout.
//
// Measured, bf16, N = 128, P = 64 (kernel times of a trace; together they take 105 us): 2 x 32 heads x 8192 tokens, 16
// segments: states 36.5 us (67 MB of x and 34 MB of states moved, 2.8 TB/s), sum 11.2 us (67 MB, 6.0 TB/s), outputs 67 us
// (170 MB, 2.5 TB/s).  Bound by neither the memory nor the products: with every matrix instruction taken out the states'
// kernel takes 26 us and the outputs' 50.  A chunk step of a workgroup takes some 8 500 and 16 800 cycles, of which the
// matrix pipes work 3 580 and 6 180, the vector port 2 990 and 6 800 and LDS 2 670 and 5 460.  The rest is waiting, which
// two waves a SIMD (the states and the chunk in flight fill its registers) do not fill for each other: the outputs have
// three barriers a step, and the phases between them use one of the three at a time.  Measured and left out, in times of one bf16 term for y (states 39, outputs 58 us): 64 columns a wave with one
// wave a SIMD (states 50, outputs 75 us: the halved LDS traffic is lost to moves between the register files), two workgroups
// of 128 columns a CU (outputs 88 us with the score shared or not), 16 columns a wave (states 47 us), the waves of one SIMD in
// opposite phases (spills, 147 us), operands fetched half a chunk ahead (states 39 us), the first chunk's loads before the
// state's (outputs 63 us).
#pragma once

#include "pf_gfx950.h"
#include "pf_serving.h"

namespace pf {

constexpr int kSsmChunk = 64;
// A thread's offset inside a chunk is 32-bit: 64 tokens of this many 4-byte elements.
constexpr long kMaxTokenStride = 1L << 22;

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
  float* seg_state;        // what a segment adds, then what enters it: per task the registers of its waves, as they lie
  float* seg_decay;        // [B, H, segs]: log2 of a segment's decay
  long x_b, x_h, x_t, dt_b, dt_h, dt_t, b_b, b_g, b_t, c_b, c_g, c_t, z_b, z_h, z_t, y_b, y_h, y_t;
  uint32_t tasks;          // B * G * column blocks * segments
  int B, H, G, T, N, P;
  int blocks;              // blocks of columns of a group's heads
  int segs, seg_chunks;
  int dt_f32, softplus;
};

enum class SsmMode { kStates, kOutput };

// A buffer offset past the end of any: reads as zero, is not written.
constexpr uint32_t kPastEnd = 0x80000000u;

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

__device__ __forceinline__ void only_finite(Frag<bf16>& f) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f.v[i] = __builtin_isfinite((float)f.v[i]) ? f.v[i] : (bf16)0.f;
}
__device__ __forceinline__ void only_finite(Frag<float>& f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f.lo[i] = __builtin_isfinite(f.lo[i]) ? f.lo[i] : 0.f;
    f.hi[i] = __builtin_isfinite(f.hi[i]) ? f.hi[i] : 0.f;
  }
}

template <typename E, typename V> __device__ __forceinline__ Frag<E> frag_cat(const V& lo, const V& hi);
template <> __device__ __forceinline__ Frag<bf16> frag_cat<bf16, bf16x4>(const bf16x4& lo, const bf16x4& hi) { return {cat8(lo, hi)}; }
template <> __device__ __forceinline__ Frag<float> frag_cat<float, floatx4>(const floatx4& lo, const floatx4& hi) { return {lo, hi}; }

// Two MFMA results as the operand that contracts over their 32 rows, in bf16 terms: each the rounding of what the ones before
// it left (8, 16 or 24 bits); fp32 needs one.  A term is taken off by subtractions, or (BY_PRODUCT) by a product with minus
// the identity, exact as well: one product and zeros.  (That also spoils the column of a value that is not finite, as the sums
// to come do.)  Where two waves share a SIMD the vector port is the fuller one: 2 x 32 heads x 8192 tokens 108.5 us by
// subtractions, 105.5 by products.  A wave alone on its SIMD waits for its products: 64 columns, 1 x 512 tokens whole 47
// against 53, 128 columns, 16 x 1024 92 against 97.
template <typename E, bool BY_PRODUCT> struct Terms;
template <bool BY_PRODUCT> struct Terms<bf16, BY_PRODUCT> {
  static constexpr int N = 2;        // for y
  Frag<bf16> lo, hi;                 // minus the identity for the first 16 and for the second 16 of 32 rows
  __device__ __forceinline__ Terms(int c, int g) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lo.v[i] = hi.v[4 + i] = 4 * g + i == c ? (bf16)-1.f : (bf16)0.f;
      lo.v[4 + i] = hi.v[i] = (bf16)0.f;
    }
  }
  template <int COUNT>
  __device__ __forceinline__ void of(floatx4 l, floatx4 h, Frag<bf16> (&t)[COUNT]) const {
#pragma unroll
    for (int k = 0; k < COUNT; ++k) {
      t[k].v = pack8(l, h);
      if (k + 1 == COUNT) break;
      if constexpr (BY_PRODUCT) {
        l = mfma32(lo, t[k], l);
        h = mfma32(hi, t[k], h);
      } else {
        const u32x4 o = __builtin_bit_cast(u32x4, t[k].v);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          l[2 * i] -= __uint_as_float(o[i] << 16);
          l[2 * i + 1] -= __uint_as_float(o[i] & 0xffff0000u);
          h[2 * i] -= __uint_as_float(o[2 + i] << 16);
          h[2 * i + 1] -= __uint_as_float(o[2 + i] & 0xffff0000u);
        }
      }
    }
  }
};
template <bool BY_PRODUCT> struct Terms<float, BY_PRODUCT> {
  static constexpr int N = 1;
  __device__ __forceinline__ Terms(int, int) {}
  __device__ __forceinline__ void of(const floatx4& l, const floatx4& h, Frag<float> (&t)[N]) const { t[0] = {l, h}; }
};

// ---- LDS tiles: 64 token rows, PAD elements longer than they are ----------------------------
// Rows 16 bytes apart modulo the banks suit the operand that reads sixteen rows at one place; 32 bytes the transposed one,
// which reads eight rows at four neighbouring 8-byte places in half a wave.  fp32 rows are 16 bytes apart.
template <typename E, int W, int PAD> struct Tile {
  static constexpr int LD = W + PAD;
  static constexpr int ELEMS = kSsmChunk * LD;
  // operand: lane c holds row `row`, lane group g the eight columns 32 kb + 8g ..
  __device__ __forceinline__ static Frag<E> rows(const E* s, int row, int kb, int g) {
    const E* p = s + row * LD + kb * 32 + g * 8;
    if constexpr (sizeof(E) == 2) {
      return {*reinterpret_cast<const bf16x8*>(p)};
    } else {
      return {*reinterpret_cast<const floatx4*>(p), *reinterpret_cast<const floatx4*>(p + 4)};
    }
  }
  // transposed operand: lane c holds column col + c (APART = 4), or col + 8 (c / 4) + c % 4 (APART = 8); lane group g rows
  // 32 kb + 4g .. and 32 kb + 16 + 4g ..
  template <int APART>
  __device__ __forceinline__ static Frag<E> cols(const E* s, int col, int kb, int c, int g) {
    if constexpr (sizeof(E) == 2) {
      const E* p = s + (32 * kb + 4 * g + (c >> 2)) * LD + col + APART * (c & 3);
      return {cat8(lds_read_tr(p), lds_read_tr(p + 16 * LD))};
    } else {
      const E* p = s + (32 * kb + 4 * g) * LD + col + APART * (c >> 2) + (c & 3);
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
// Row of the state that lane group g holds as register r of tile nt.  The tiles of a pair interleave, four rows each, so
// that a lane group's rows in the two are the eight neighbouring columns of B or C it reads as one vector.
__device__ __forceinline__ constexpr int state_row(int nt, int g, int r) { return 32 * (nt >> 1) + 8 * g + 4 * (nt & 1) + r; }

// Column, of a wave's 16 PT, that lane c holds in tile pt: interleaved the same way, so that the rows 4g .. of the PT tiles
// of y^T are 4 PT neighbouring columns, one vector.
template <int PT> __device__ __forceinline__ constexpr int state_col(int pt, int c) { return 4 * PT * (c >> 2) + 4 * pt + (c & 3); }

// x scaled by its rows' weights, in SPLIT terms.
template <typename T, int SPLIT>
__device__ __forceinline__ void weigh(const T& terms, const Frag<bf16>& x, const floatx4& w0, const floatx4& w1,
                                      Frag<bf16> (&t)[SPLIT]) {
  const u32x4 xb = __builtin_bit_cast(u32x4, x.v);
  floatx4 l, h;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l[2 * i] = __uint_as_float(xb[i] << 16) * w0[2 * i];
    l[2 * i + 1] = __uint_as_float(xb[i] & 0xffff0000u) * w0[2 * i + 1];
    h[2 * i] = __uint_as_float(xb[2 + i] << 16) * w1[2 * i];
    h[2 * i + 1] = __uint_as_float(xb[2 + i] & 0xffff0000u) * w1[2 * i + 1];
  }
  terms.of(l, h, t);
}
template <typename T>
__device__ __forceinline__ void weigh(const T&, const Frag<float>& x, const floatx4& w0, const floatx4& w1,
                                      Frag<float> (&t)[1]) {
  t[0] = {x.lo * w0, x.hi * w1};
}

// A value that all lanes hold, in a scalar register.  (Quotients come in vector registers, and what is made of them stays there.)
__device__ __forceinline__ int wave_int(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ float wave_value(float v) {
  return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v)));
}

// 2^x of the hardware: results below 2^-126 are zero.
__device__ __forceinline__ float pow2(float x) { return __builtin_amdgcn_exp2f(x); }

// v of the lane N before (SHR) or behind (SHL) within a row of 16 lanes, zero past its end.
template <int CTRL> __device__ __forceinline__ float row_move(float v) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, 0xf, 0xf, true));
}
// Sums over a row's lanes up to each (inclusive).
__device__ __forceinline__ float row_sums(float v) {
  v += row_move<0x111>(v);
  v += row_move<0x112>(v);
  v += row_move<0x114>(v);
  v += row_move<0x118>(v);
  return v;
}
// The value of a row's last lane.
__device__ __forceinline__ float row_last(float v) { return row_move<0x15f>(v); }

constexpr float kGateFloor = -256.f;                     // log2 of a token's decay

// The weight of one token for another is 2 to the sum of the gates between them, whose rounding has to be of its own size,
// not of what came before it in the chunk (weak tokens behind strong ones).  Between 16s these are sums from a 16's end or
// start; inside one, differences of the running sum, which is held in two parts for it: the high ones are multiples of 2^-10
// and at most 16 * 2^8, so that they and their differences are exact, the low ones stay under 16 * 2^-11.
constexpr float kGateGrain = 1.f / 1024;

// The tables of a chunk and head.  Of each token: dt times the decay to the chunk's end; the running sum of gates within its
// 16, in two parts; dt; dt times the decay to the end of its 16 (not of the last 16, where none comes after it); and the
// decays over the 16s that end in it: its own up to it, and one, two or three before that, as far as there are any.
enum SsmTab {
  kToEnd = 0, kHigh = 64, kLow = 128, kStep = 192, kToTile = 256, kDecay1 = 304, kDecay2 = 368 - 16, kDecay3 = 416 - 32,
  kDecay4 = 448 - 48, kTabEnd = 464
};
__device__ __forceinline__ constexpr int decay_over(int tiles) {
  return tiles == 1 ? kDecay1 : tiles == 2 ? kDecay2 : tiles == 3 ? kDecay3 : kDecay4;
}

// (chunk, head) pairs of a batch of tables that a wave makes.
constexpr int kSsmShare = 2;

// The outputs keep one chunk and what only they need; the states' kernel two chunks.
template <typename E, int NT, int NW, int PT, bool OUT> struct SsmLds {
  static constexpr int SLOTS = kSsmShare * NW, BUF = OUT ? 1 : 2;
  typedef Tile<E, NT, (OUT ? 32 : 16) / (int)sizeof(E)> B;
  typedef Tile<E, NT, 16 / (int)sizeof(E)> C;
  typedef Tile<E, 16 * PT, 16 / (int)sizeof(E)> X;
  E b[BUF][B::ELEMS];
  E x[BUF][NW][X::ELEMS];
  E c[OUT ? C::ELEMS : 1];
  // C B^T, tile (ib, jb) transposed: lane (c, g) holds rows j = 16 jb + 4g .. of column i = 16 ib + c.
  floatx4 score[OUT ? 10 : 1][64];
  float tab[SLOTS][OUT ? (int)kTabEnd : kSsmChunk];    // SsmTab, per (chunk, head) of a batch
  float total[SLOTS];                                  // log2 of the chunk's decay
};

// SPLIT: bf16 terms of the weighted x in the state's update.  Three keep the state a sum in 24 bits, as it has to be where
// it is returned; two where it only enters y, whose operand S has two terms itself.
// PT: 16-column tiles of a wave.
// One workgroup's walk.  Returns whether it has to be made AGAIN: a value of x that is not finite reaches the tokens before it
// in its chunk, through the products with the zeros above the score's diagonal.  The second walk leaves such values out of the
// products for y, and makes every token from theirs on NaN.
template <typename E, int NT, int NW, int PT, SsmMode MODE, int SPLIT, bool HAS_Z, bool AGAIN>
__device__ __forceinline__ bool ssm_walk(const SsmArgs& a, SsmLds<E, NT, NW, PT, MODE == SsmMode::kOutput>& s, const uint32_t tid,
                                         const uint32_t bid) {
  constexpr int Q = kSsmChunk, ES = (int)sizeof(E), V = 16 / ES, TH = NW * 64, NTS = NT / 16;
  constexpr int COLS = NW * 16 * PT;           // columns of a workgroup
  constexpr int RV = NT / V;                   // vectors of a row of B or C
  constexpr int NB = Q * RV < TH ? 1 : Q * RV / TH;   // of them a thread, TH / RV rows apart
  constexpr int XV = 16 * PT / V;              // vectors of a row of a wave's x
  constexpr int NX = Q * XV / 64;
  constexpr bool OUT = MODE == SsmMode::kOutput;
  using Lds = SsmLds<E, NT, NW, PT, OUT>;
  using Bs = typename Lds::B;
  using Cs = typename Lds::C;
  using Xs = typename Lds::X;

  // Workgroups go round robin over the eight XCDs: each XCD takes a run of tasks, so that the segments of one block of
  // columns, and the sum along them, meet in its L2.
  const uint32_t per = (a.tasks + 7) / 8, task = (bid & 7) * per + (bid >> 3);
  if (bid >> 3 >= per || task >= a.tasks) return false;
  const int seg = wave_int(task % (uint32_t)a.segs);
  uint32_t rest = wave_int(task / (uint32_t)a.segs);
  const int cb = wave_int(rest % (uint32_t)a.blocks);
  rest = wave_int(rest / (uint32_t)a.blocks);
  const int grp = wave_int(rest % (uint32_t)a.G);
  const long bi = wave_int(rest / (uint32_t)a.G);

  const int lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int R = wave_int(a.H / a.G);
  // The columns of a group's heads lie end to end, and the workgroup has COLS of them: P is a multiple of 32, so that a
  // wave's are of one head.
  const int col = cb * COLS + w * 16 * PT;
  const bool active = col < R * a.P;
  const int hr = wave_int(active ? col / a.P : 0), p0 = wave_int(active ? col - hr * a.P : 0);
  const int h = grp * R + hr, hl = active ? hr - wave_int(cb * COLS / a.P) : 0;
  const int N = a.N, P = a.P;
  int len = a.T;
  if (a.lengths) len = __builtin_amdgcn_readfirstlane(min(max(a.lengths[bi], 0), a.T));

  const int chunks = (a.T + Q - 1) / Q;
  const int first = seg * a.seg_chunks, end = min(first + a.seg_chunks, chunks);

  // ---- what a chunk loads: rows of B and C by all threads, its own columns of x by each wave.  The buffers end after the
  // last live token of the chunk (a token's stride covers its row), so that what lies past it reads as zero.
  const char* xg = reinterpret_cast<const char*>(static_cast<const E*>(a.x) + bi * a.x_b + h * a.x_h + p0);
  const char* bg = reinterpret_cast<const char*>(static_cast<const E*>(a.b) + bi * a.b_b + grp * a.b_g);
  const char* cg = reinterpret_cast<const char*>(static_cast<const E*>(a.c) + bi * a.c_b + grp * a.c_g);
  const int xt = (int)a.x_t * ES, bt = (int)a.b_t * ES, ct = (int)a.c_t * ES;
  const int b_row = tid / RV, b_col = tid % RV * V, x_row = lane / XV, x_col = lane % XV * V;
  const bool stages = Q * RV >= TH || tid < Q * RV;
  const uint32_t b_off = b_col < N ? (uint32_t)(b_row * bt + b_col * ES) : kPastEnd;
  const uint32_t c_off = b_col < N ? (uint32_t)(b_row * ct + b_col * ES) : kPastEnd;
  const uint32_t x_off = active ? (uint32_t)(x_row * xt + x_col * ES) : kPastEnd;
  u32x4 rb[NB], rc[NB], rx[NX];
  auto load = [&](int t0) {
    const int valid = __builtin_amdgcn_readfirstlane(min(max(len - t0, 0), Q));
    const auto xr = make_rsrc(xg + (long)t0 * xt, (uint32_t)(valid * xt)), br = make_rsrc(bg + (long)t0 * bt, (uint32_t)(valid * bt)),
               cr = make_rsrc(cg + (long)t0 * ct, (uint32_t)(valid * ct));
    if (stages) {
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        rb[i] = __builtin_amdgcn_raw_buffer_load_b128(br, b_off + i * (TH / RV) * bt, 0, 0);
        if (OUT) rc[i] = __builtin_amdgcn_raw_buffer_load_b128(cr, c_off + i * (TH / RV) * ct, 0, 0);
      }
    }
#pragma unroll
    for (int i = 0; i < NX; ++i) rx[i] = __builtin_amdgcn_raw_buffer_load_b128(xr, x_off + i * (64 / XV) * xt, 0, 0);
  };
  auto stage = [&](int buf) {
    if (stages) {
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int row = b_row + i * (TH / RV);
        *reinterpret_cast<u32x4*>(&s.b[buf][row * Bs::LD + b_col]) = rb[i];
        if (OUT) *reinterpret_cast<u32x4*>(&s.c[row * Cs::LD + b_col]) = rc[i];
      }
    }
#pragma unroll
    for (int i = 0; i < NX; ++i) *reinterpret_cast<u32x4*>(&s.x[buf][w][(x_row + i * (64 / XV)) * Xs::LD + x_col]) = rx[i];
  };
  // ---- the chunks' step sizes and decays, a token a lane, in log2.  A batch of chunks at a time: its (chunk, head) pairs
  // are dealt over the waves, the steps loaded a batch ahead.
  const int h_first = wave_int(cb * COLS / P), heads = min(R, wave_int((cb * COLS + COLS - 1) / P) + 1) - h_first,
            batch = wave_int(Lds::SLOTS / heads);
  // The steps' bits as stored: a conversion beside the load would wait for it and for all before it (2 x 32 heads x 8192
  // tokens: states 40 us against 39, outputs 60 against 58).
  uint32_t rdt[kSsmShare];
  float ra[kSsmShare], rbias[kSsmShare];
#pragma unroll
  for (int i = 0; i < kSsmShare; ++i) {
    const int head = grp * R + h_first + (w + i * NW) % heads;
    ra[i] = wave_value(a.a[head] * 1.44269504f);
    rbias[i] = wave_value(a.dt_bias ? a.dt_bias[head] : 0.f);
  }
  auto load_dt = [&](int ch) {
#pragma unroll
    for (int i = 0; i < kSsmShare; ++i) {
      const int slot = w + i * NW, t = (ch + slot / heads) * Q + lane;
      rdt[i] = 0;
      if (slot / heads < batch && t < len) {
        const size_t at = bi * a.dt_b + (grp * R + h_first + slot % heads) * a.dt_h + t * a.dt_t;
        if (ES == 4 || a.dt_f32) rdt[i] = static_cast<const uint32_t*>(a.dt)[at];
        else rdt[i] = static_cast<const uint16_t*>(a.dt)[at];
      }
    }
  };
  auto tabulate = [&](int ch) {
#pragma unroll
    for (int i = 0; i < kSsmShare; ++i) {
      const int slot = w + i * NW;
      if (slot / heads >= batch) continue;
      float dt = __uint_as_float(ES == 4 || a.dt_f32 ? rdt[i] : rdt[i] << 16) + rbias[i];
      if (a.softplus) dt = softplus(dt);
      if ((ch + slot / heads) * Q + lane >= len) dt = 0.f;
      // 2^-256 of anything is zero; the floor bounds the sums.
      float gate = dt * ra[i];
      gate = gate < kGateFloor ? kGateFloor : gate;
      const float coarse = rintf(gate * (1 / kGateGrain)) * kGateGrain;
      const float high = row_sums(coarse), low = row_sums(gate - coarse), sum = high + low;
      float t[4];                              // a 16's gates
#pragma unroll
      for (int k = 0; k < 4; ++k) t[k] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sum), 16 * k + 15));
      const float to_tile = (row_last(high) - high) + (row_last(low) - low);
      const float after = g == 0 ? t[1] + t[2] + t[3] : g == 1 ? t[2] + t[3] : g == 2 ? t[3] : 0.f;
      float* tab = s.tab[slot] + lane;
      tab[kToEnd] = dt * pow2(to_tile + after);
      if constexpr (OUT) {
        tab[kHigh] = high;
        tab[kLow] = low;
        tab[kStep] = dt;
        tab[kDecay1] = pow2(sum);
        if (g < 3) tab[kToTile] = dt * pow2(to_tile);
        if (g > 0) tab[kDecay2] = pow2(sum + (g == 1 ? t[0] : g == 2 ? t[1] : t[2]));
        if (g > 1) tab[kDecay3] = pow2(sum + (g == 2 ? t[0] + t[1] : t[1] + t[2]));
        if (g > 2) tab[kDecay4] = pow2(sum + (t[0] + t[1] + t[2]));
      }
      if (lane == 63) s.total[slot] = t[0] + t[1] + t[2] + t[3];
    }
  };
  float decay2 = 0.f;                          // log2 of the segment's decay

  floatx4 S[NTS][PT];
#pragma unroll
  for (int nt = 0; nt < NTS; ++nt)
#pragma unroll
    for (int pt = 0; pt < PT; ++pt) S[nt][pt] = zero4();
  floatx4* const slab = reinterpret_cast<floatx4*>(a.seg_state) + ((size_t)task * NW + w) * NTS * PT * 64 + lane;
  if (OUT && active) {
    if (a.segs > 1) {
#pragma unroll
      for (int nt = 0; nt < NTS; ++nt)
#pragma unroll
        for (int pt = 0; pt < PT; ++pt) S[nt][pt] = slab[(nt * PT + pt) * 64];
    } else if (a.h0) {
      const float* in = a.h0 + ((long)bi * a.H + h) * N * P + p0;
#pragma unroll
      for (int nt = 0; nt < NTS; ++nt)
#pragma unroll
        for (int pt = 0; pt < PT; ++pt)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int n = state_row(nt, g, r);
            if (n < N) S[nt][pt][r] = in[n * P + state_col<PT>(pt, c)];
          }
    }
  }

  const int yt = (int)a.y_t * ES, zt = (int)a.z_t * ES;
  char* yg = reinterpret_cast<char*>(static_cast<E*>(a.y) + bi * a.y_b + h * a.y_h + p0);
  const char* zg = reinterpret_cast<const char*>(static_cast<const E*>(a.z) + bi * a.z_b + h * a.z_h + p0);
  const uint32_t y_off = active ? (uint32_t)(c * yt + 4 * PT * g * ES) : kPastEnd;
  const uint32_t z_off = active ? (uint32_t)(c * zt + 4 * PT * g * ES) : kPastEnd;
  static_assert(4 * PT == V, "a lane's columns of y are one vector");
  const float dd = wave_value(active && a.d ? a.d[h] : 0.f);

  const Terms<E, NW * 16 * PT == 256> terms(c, g);
  int slot0 = -heads;                          // of this chunk's tables
  if (first < end) {
    load_dt(first);
    load(first * Q);
    if (!OUT) {
      tabulate(first);
      load_dt(first + batch);
      stage(first & 1);
      load((first + 1) * Q);                   // past the last chunk: nothing is valid, nothing is read
      lds_barrier();
    }
  }
  for (int ch = first; ch < end; ++ch) {
    const int t0 = ch * Q, buf = OUT ? 0 : ch & 1;
    slot0 += heads;
    if (slot0 + heads > Lds::SLOTS) slot0 = 0;
    const float* tab = s.tab[slot0 + hl];
    if (OUT) {
      lds_barrier();                           // the last chunk's reads are done
      stage(0);
      if (slot0 == 0) {
        tabulate(ch);
        load_dt(ch + batch);
      }
      lds_barrier();
      if (ch + 1 < end) load(t0 + Q);
    }
    const E* sb = s.b[buf];
    const E* sx = s.x[buf][w];

    Frag<E> xf[PT][2];
#pragma unroll
    for (int pt = 0; pt < PT; ++pt)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        xf[pt][kb] = Xs::template cols<4 * PT>(sx, 4 * pt, kb, c, g);
        if (AGAIN) only_finite(xf[pt][kb]);
      }

    if constexpr (OUT) {
      // the score's tiles, dealt over the waves
#pragma unroll
      for (int k = 0; k < (10 + NW - 1) / NW; ++k) {
        const int tile = w + k * NW;
        if ((k + 1) * NW <= 10 || tile < 10) {
          const int ib = tile >= 6 ? 3 : tile >= 3 ? 2 : tile >= 1 ? 1 : 0, jb = tile - ib * (ib + 1) / 2;
          floatx4 acc = zero4();
#pragma unroll
          for (int kb = 0; kb < NT / 32; ++kb)
            acc = mfma32(Bs::rows(sb, 16 * jb + c, kb, g), Cs::rows(s.c, 16 * ib + c, kb, g), acc);
          s.score[tile][lane] = acc;
        }
      }
      // y^T = S^T C^T
      floatx4 y[PT][4];
#pragma unroll
      for (int pt = 0; pt < PT; ++pt)
#pragma unroll
        for (int ib = 0; ib < 4; ++ib) y[pt][ib] = zero4();
#pragma unroll
      for (int kb = 0; kb < NT / 32; ++kb) {
        Frag<E> sf[PT][terms.N];
#pragma unroll
        for (int pt = 0; pt < PT; ++pt) terms.of(S[2 * kb][pt], S[2 * kb + 1][pt], sf[pt]);
#pragma unroll
        for (int ib = 0; ib < 4; ++ib) {
          const Frag<E> cf = Cs::rows(s.c, 16 * ib + c, kb, g);
#pragma unroll
          for (int pt = 0; pt < PT; ++pt)
#pragma unroll
            for (int k = terms.N - 1; k >= 0; --k) y[pt][ib] = mfma32(sf[pt][k], cf, y[pt][ib]);
        }
      }
      const int valid = __builtin_amdgcn_readfirstlane(min(max(len - t0, 0), Q));
      lds_barrier();                           // the score is whole
#pragma unroll
      for (int ib = 0; ib < 4; ++ib) {
        const float e = tab[decay_over(ib + 1) + 16 * ib + c];
#pragma unroll
        for (int pt = 0; pt < PT; ++pt) y[pt][ib] *= e;
        floatx4 pr[4];
#pragma unroll
        for (int jb = 0; jb < 4; ++jb) {
          pr[jb] = zero4();
          if (jb < ib) {
            const float f = tab[decay_over(ib - jb) + 16 * ib + c];
            const floatx4 u = *reinterpret_cast<const floatx4*>(&tab[kToTile + 16 * jb + 4 * g]);
            pr[jb] = s.score[ib * (ib + 1) / 2 + jb][lane] * (u * f);
          } else if (jb == ib) {
            const floatx4 sc = s.score[ib * (ib + 1) / 2 + jb][lane];
            const float Gi = tab[kHigh + 16 * ib + c], li = tab[kLow + 16 * ib + c];
            const floatx4 Gj = *reinterpret_cast<const floatx4*>(&tab[kHigh + 16 * jb + 4 * g]);
            const floatx4 lj = *reinterpret_cast<const floatx4*>(&tab[kLow + 16 * jb + 4 * g]);
            const floatx4 dj = *reinterpret_cast<const floatx4*>(&tab[kStep + 16 * jb + 4 * g]);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              float v = sc[r] * (dj[r] * pow2((Gi - Gj[r]) + (li - lj[r])));
              __asm__ volatile("" : "+v"(v));  // made here, or the select becomes a branch around the exponential
              pr[jb][r] = 4 * g + r <= c ? v : 0.f;
            }
          }
        }
#pragma unroll
        for (int kb = 0; kb <= ib / 2; ++kb) {
          Frag<E> pf[terms.N];
          terms.of(pr[2 * kb], pr[2 * kb + 1], pf);
#pragma unroll
          for (int pt = 0; pt < PT; ++pt)
#pragma unroll
            for (int k = terms.N - 1; k >= 0; --k) y[pt][ib] = mfma32(xf[pt][kb], pf[k], y[pt][ib]);
        }
      }
      if (AGAIN) {                             // 0 x, summed along the tokens: NaN from a value that is not finite on
#pragma unroll
        for (int i = 0; i < 4 * PT; ++i) {
          float before = 0.f;
#pragma unroll
          for (int ib = 0; ib < 4; ++ib) {
            const float upto = row_sums(0.f * to_f32(sx[(16 * ib + c) * Xs::LD + 4 * PT * g + i]));
            y[i / 4][ib][i % 4] += before + upto;
            before += row_last(upto);
          }
        }
#pragma unroll
        for (int pt = 0; pt < PT; ++pt)
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) xf[pt][kb] = Xs::template cols<4 * PT>(sx, 4 * pt, kb, c, g);
      }
      // z of this chunk.  (Asked for before the barrier, its registers cost more in spills than its latency does here:
      // 32768 tokens 186 us against 150.)
      u32x4 rz[HAS_Z ? 4 : 1];
      if (HAS_Z) {
        const auto zr = make_rsrc(zg + (long)t0 * zt, (uint32_t)(valid * zt));
#pragma unroll
        for (int ib = 0; ib < 4; ++ib) rz[ib] = __builtin_amdgcn_raw_buffer_load_b128(zr, z_off + 16 * ib * zt, 0, 0);
      }
      // y out: lane c's token, the lane group's 4 PT columns as one vector
      const auto yr = make_rsrc(yg + (long)t0 * yt, (uint32_t)(min(a.T - t0, Q) * yt));
#pragma unroll
      for (int ib = 0; ib < 4; ++ib) {
        float v[4 * PT];
        load_vec<4 * PT>(&sx[(16 * ib + c) * Xs::LD + 4 * PT * g], v);
#pragma unroll
        for (int i = 0; i < 4 * PT; ++i) v[i] = fmaf(dd, v[i], y[i / 4][ib][i % 4]);
        if (HAS_Z) {
          float z[4 * PT];
          expand<E, V>(__builtin_bit_cast(typename VecAny<E, V>::T, rz[ib]), z);
#pragma unroll
          for (int i = 0; i < 4 * PT; ++i) v[i] *= silu(z[i]);
        }
        typename VecAny<E, V>::T o;
#pragma unroll
        for (int i = 0; i < 4 * PT; ++i) o[i] = from_f32<E>(v[i]);
        u32x4 bits = __builtin_bit_cast(u32x4, o);
        if (valid < Q && 16 * ib + c >= valid) bits = u32x4{0, 0, 0, 0};
        __builtin_amdgcn_raw_buffer_store_b128(bits, yr, y_off + 16 * ib * yt, 0, 0);
      }
    }
    // S <- e^{G_last} S + B^T (w x), a tile column and half of the chunk at a time: the products of one while the next one's
    // x is weighed.
    const float total = s.total[slot0 + hl], e = pow2(total);
    decay2 += total;
    floatx4 wt[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) wt[q] = *reinterpret_cast<const floatx4*>(&tab[kToEnd + 16 * q + 4 * g]);
    Frag<E> bf[NTS], wx[2][SPLIT];
#pragma unroll
    for (int nt = 0; nt < NTS; ++nt) bf[nt] = Bs::template cols<8>(sb, 32 * (nt >> 1) + 4 * (nt & 1), 0, c, g);
    weigh(terms, xf[0][0], wt[0], wt[1], wx[0]);
#pragma unroll
    for (int st = 0; st < 2 * PT; ++st) {
      const int kb = st / PT, pt = st % PT, nx = st + 1;
      if (nx < 2 * PT) weigh(terms, xf[nx % PT][nx / PT], wt[2 * (nx / PT)], wt[2 * (nx / PT) + 1], wx[nx & 1]);
      if (kb == 0) {
#pragma unroll
        for (int nt = 0; nt < NTS; ++nt) S[nt][pt] *= e;
      }
#pragma unroll
      for (int k = SPLIT - 1; k >= 0; --k)
#pragma unroll
        for (int nt = 0; nt < NTS; ++nt) {
          S[nt][pt] = mfma32(bf[nt], wx[st & 1][k], S[nt][pt]);
          if (k == 0 && pt == PT - 1 && kb == 0) bf[nt] = Bs::template cols<8>(sb, 32 * (nt >> 1) + 4 * (nt & 1), 1, c, g);
        }
    }
    if (!OUT && ch + 1 < end) {
      stage((ch + 1) & 1);
      load(t0 + 2 * Q);
      if (slot0 + 2 * heads > Lds::SLOTS) {    // the next chunk begins a batch
        lds_barrier();                         // the last batch's reads are done
        tabulate(ch + 1);
        load_dt(ch + 1 + batch);
      }
      lds_barrier();
    }
  }

  if (OUT && !AGAIN) {
    // A value of x that is not finite stays in its column of the state, in all rows of it.
    float bad = 0.f;
#pragma unroll
    for (int pt = 0; pt < PT; ++pt) bad += 0.f * S[0][pt][0];
    bad = __any(bad != 0.f) ? 1.f : 0.f;
    lds_barrier();                             // the last chunk's reads are done
    if (lane == 0) s.total[w] = bad;
    lds_barrier();
    for (int i = 0; i < NW; ++i) bad += s.total[i];
    if (__builtin_expect(wave_value(bad) != 0.f, 0)) return true;
  }
  if (!active) return false;
  if (!OUT) {
    if (p0 == 0 && lane == 0) a.seg_decay[((long)bi * a.H + h) * a.segs + seg] = decay2;
#pragma unroll
    for (int nt = 0; nt < NTS; ++nt)
#pragma unroll
      for (int pt = 0; pt < PT; ++pt) slab[(nt * PT + pt) * 64] = S[nt][pt];
  } else if (a.segs == 1 && a.h_final) {
    float* out = a.h_final + ((long)bi * a.H + h) * N * P + p0;
#pragma unroll
    for (int nt = 0; nt < NTS; ++nt)
#pragma unroll
      for (int pt = 0; pt < PT; ++pt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int n = state_row(nt, g, r);
          if (n < N) out[n * P + state_col<PT>(pt, c)] = S[nt][pt][r];
        }
  }
  return false;
}

template <typename E, int NT, int NW, int PT, SsmMode MODE, int SPLIT, bool HAS_Z>
__global__ __launch_bounds__(NW * 64) __attribute__((
    amdgpu_waves_per_eu(sizeof(E) == 4 || NW * 16 * PT < 256 ? 1 : 2))) void ssm_kernel(SsmArgs a) {
  __shared__ __attribute__((aligned(16))) SsmLds<E, NT, NW, PT, MODE == SsmMode::kOutput> s;
  uint32_t tid = threadIdx.x, bid = blockIdx.x;
  const bool again = ssm_walk<E, NT, NW, PT, MODE, SPLIT, HAS_Z, false>(a, s, tid, bid);
  if constexpr (MODE == SsmMode::kOutput) {
    if (__builtin_expect(again, 0)) {
      __builtin_amdgcn_s_waitcnt(0);                   // the first walk's stores of y are done
      // The second walk makes all it needs anew, arguments too: what it kept of the first would cost that one registers.
      typedef const SsmArgs __attribute__((address_space(4)))* Args;
      Args args = (Args)__builtin_amdgcn_kernarg_segment_ptr();
      __asm__ volatile("" : "+v"(tid), "+s"(bid), "+s"(args));
      ssm_walk<E, NT, NW, PT, MODE, SPLIT, HAS_Z, true>(*(const SsmArgs*)args, s, tid, bid);
    }
  }
}

// The states that enter the segments, in place of what each adds: H_0 = h0, H_{s+1} = decay_s H_s + D_s; the last is the
// final state.  A thread owns the four elements of one register of a segment's waves (four rows of one column); the
// segments' values are loaded four ahead of the sum.  The workgroups of one column block run where its segments' did.
// Bound by memory (2 x 32 heads x 8192 tokens: 67 MB, 5.8 TB/s, part of it from the cache).  One / two / four / eight / sixteen
// ahead, us: that shape 13.4 / 11.4 / 11.5 / 11.8 / 11.7, 32 segments of one context 16.4 / 13.0 / 12.8 / 13.4 / 13.7, 12 of
// small states 7.0 / 5.1 / 4.6 / 4.6 / 4.5.
template <int NT, int PT, int COLS>
__global__ __launch_bounds__(256) void ssm_prefix_kernel(SsmArgs a) {
  constexpr int SLAB = COLS * NT / 4, NTS = NT / 16;       // vectors of a segment
  const long blocks = (long)(a.tasks / (uint32_t)a.segs) * (SLAB / 256), per = (blocks + 7) / 8;
  const long block = (block_id() & 7) * per + (block_id() >> 3);
  if (block_id() >> 3 >= per || block >= blocks) return;
  const int at = (int)(block % (SLAB / 256)) * 256 + threadIdx.x;
  const long unit = block / (SLAB / 256);
  const int lane = at & 63, c = lane & 15, g = lane >> 4, pt = at / 64 % PT, nt = at / (64 * PT) % NTS, w = at / (64 * PT * NTS);
  const int col = (int)(unit % a.blocks) * COLS + w * 16 * PT + state_col<PT>(pt, c), R = a.H / a.G;
  if (col >= R * a.P) return;
  const long bg = unit / a.blocks, bh = bg / a.G * a.H + bg % a.G * R + col / a.P;
  const long h_at = bh * a.N * a.P + col % a.P;
  const int n = state_row(nt, g, 0);                       // and the three after it
  const float* decay = a.seg_decay + bh * a.segs;
  floatx4* st = reinterpret_cast<floatx4*>(a.seg_state) + (size_t)unit * a.segs * SLAB + at;
  floatx4 H = zero4();
  if (a.h0) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (n + r < a.N) H[r] = a.h0[h_at + (long)(n + r) * a.P];
  }
  constexpr int AHEAD = 4;
  for (int s0 = 0; s0 < a.segs; s0 += AHEAD) {
    floatx4 D[AHEAD];
    float e[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (s0 + i < a.segs) {
        D[i] = st[(size_t)(s0 + i) * SLAB];
        e[i] = decay[s0 + i];                              // raw: its power taken here would wait for each load in turn
      }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (s0 + i < a.segs) {
        st[(size_t)(s0 + i) * SLAB] = H;
        H = H * pow2(e[i]) + D[i];
      }
  }
  if (a.h_final) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (n + r < a.N) a.h_final[h_at + (long)(n + r) * a.P] = H[r];
  }
}

}  // namespace pf
