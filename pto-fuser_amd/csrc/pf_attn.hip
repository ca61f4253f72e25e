// extern "C" entry points of attention over prompts and over a paged cache (declared in include/pto_fuser_hip.h): checks on
// the host, then one launch, or two where the walk over a cache is shared out.
#include <hip/hip_runtime.h>

#include "../../include/pto_fuser_hip.h"
#include "pf_attn.h"
#include "pf_attn_step.h"
#include "pf_status.h"

namespace {

using pf::bf16;

constexpr int kMaxRows = 1 << 30;
constexpr long long kMaxRowStride = 1LL << 22;   // elements: offsets inside a tile are 32-bit

bool heads_ok(int H, int G, int D, int dtype) {
  return H > 0 && G > 0 && H % G == 0 && H <= 65536 && D > 0 && D <= 256 && D % 8 == 0 &&
         (dtype == PF_DTYPE_F32 || dtype == PF_DTYPE_BF16);
}

// Whole 16-byte vectors: base addresses, and strides that are multiples of one.
template <typename... S>
bool vectors(int dtype, const void* p, S... strides) {
  const long long v = dtype == PF_DTYPE_BF16 ? 8 : 4;
  return ((size_t)p & 15) == 0 && ((strides >= 0 && strides % v == 0) && ...);
}

bool grid_of(double workgroups, dim3& grid) {
  if (workgroups > (double)pf::kGridX * (pf::kGridY - 1)) return false;
  const long n = (long)workgroups;
  grid = dim3((unsigned)(n < pf::kGridX ? n : pf::kGridX), (unsigned)((n + pf::kGridX - 1) / pf::kGridX));
  return true;
}

// ---- prompts -------------------------------------------------------------------------------
template <typename E, int DP, int KW>
int attn_launch(pf::AttnArgs& a, hipStream_t s) {
  const int share = a.H / a.G;
  a.heads_log = KW <= 1 && share % 4 == 0 ? 2 : KW <= 2 && share % 2 == 0 ? 1 : 0;
  a.rows_log = (KW == 1 ? 7 : KW == 2 ? 6 : 5) - a.heads_log;
  const double tiles = (double)(a.N >> a.rows_log) + a.B + 1;      // a prompt's last tile is ragged; and one that finds none
  const double workgroups = tiles * (a.H >> a.heads_log);
  dim3 grid;
  if (workgroups >= 2147483648.0 || !grid_of(workgroups, grid)) return PF_ERR_ARG;
  a.tiles = (int)tiles;
  pf::LaunchScope scope;
  pf::attn_kernel<E, DP, KW><<<grid, dim3(256), 0, s>>>(a);
  return scope.status();
}

// Waves that share a query row, each with a part of every tile's keys.  Alone a wave walks all of them, and three workgroups a CU
// hide each other's waiting; sharing makes two or four times as many workgroups of as many times fewer steps, which is better
// where workgroups are few, or where the longest one is what is waited for.  By the number of workgroups without sharing (rows x
// heads / 128) and the prompts' mean length; us alone / two / four, prompts x rows x heads, 4 (fp32 ragged: 3) heads to one of keys:
//   bf16, D = 128: 1 x 2048 x 16 (256) 55 / 32.3, 4 x 512 x 16 (256) 19.0 / 13.8, 6 x 512 (384) 21.1 / 22.1, 2 x 2048 (512) 61 / 54,
//                  8 x 512 (512) 23.5 / 26, 1 x 6144 (768) 188 / 178, 3 x 2048 (768) 69 / 72, 1 x 8192 (1024) 288 / 306;
//                  four are not built: they were nowhere faster than two by more than a twentieth
//   bf16, D = 256: 1 x 1024 x 8 (64) 58.5 / 40.3, 1 x 2048 x 16 (256) 107 / 83, 4 x 512 (256) 36 / 38, 8 x 512 45 / 72, 1 x 4096 226 / 276
//   bf16, D = 64:  1 x 1024 x 16 (128) 20.2 / 13.8 / 11.7, 1 x 1536 (192) 27.7 / 18.3 / 15.0, 1 x 2048 35.5 / 22.4 / 24.8, 3 x 512
//                  (192) 12.5 / 11.1 / 11.3, 4 x 512 12.7 / 11.2 / 15.0, 12 x 512 (768) 14.8 / 18.5, 1 x 6144 110 / 100
//   fp32, D = 128: 1 x 2048 x 16 274 / 169, 3 x 2048 x 8 (384) 274 / 270, 1 x 4096 x 16 (512) 580 / 620
//   fp32, D = 64:  1 x 1024 x 16 73 / 41 / 34, 3 x 512 (192) 40.3 / 29.8 / 30.5, 1 x 2048 143 / 104 / 93, 3 x 2048 x 8 178 / 124 / 127, a
//                  padded batch of 3 x 1471 x 6 with 61 % live rows (207) 103 / 71.6 / 50.3, 12 x 512 72 / 74, 2 x 4096 (1024) 562 / 542,
//                  4 x 4096 1026 / 1067
template <typename E, int DP>
int attn_width(pf::AttnArgs& a, hipStream_t s) {
  constexpr bool kBf = sizeof(E) == 2;
  const double alone = (double)a.N / 128 * a.H, mean = a.B > 0 ? (double)a.N / a.B : 0;
  if (DP == 256 && !kBf) return attn_launch<E, DP, 1>(a, s);      // (two would have 256 KB of LDS)
  if (alone > (DP == 256 ? 128 + mean / 16 : kBf ? 384 + mean / 16 : DP == 64 ? 768 + mean / 16 : 384)) return attn_launch<E, DP, 1>(a, s);
  if constexpr (DP == 64) {
    if (alone <= (mean < 1024 ? 128 : kBf ? 192 : 256)) return attn_launch<E, DP, 4>(a, s);
  }
  if constexpr (kBf || DP < 256) return attn_launch<E, DP, 2>(a, s);
  return PF_ERR_ARG;
}

// The kernels' widths: a head's columns up to the next are zero.
template <typename E>
int attn_heads(pf::AttnArgs& a, hipStream_t s) {
  return a.D <= 64 ? attn_width<E, 64>(a, s) : a.D <= 128 ? attn_width<E, 128>(a, s) : attn_width<E, 256>(a, s);
}
int padded(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }

// ---- single tokens -------------------------------------------------------------------------
constexpr int kStepWgs = 512;          // workgroups that share a walk: two a CU, which their LDS fills (heads up to 64: four; past 128: one)

struct StepPlan {
  int rows, wgs, blocks;
  size_t parts, bytes;
};

// Whether the walk is shared out, by what the host knows: the tables' width in tokens, and the rows, (sequence, head, block).
// Whole rows need no second kernel, so they are faster where a row is a few steps; from there on a row is a chain of steps that
// sharing cuts, while rows are few.  us as nodes of a graph, a workgroup a row / shared, rows x tokens, all of them in use:
//   bf16, D = 128: 4 x 128 6.3 / 8.9, 4 x 256 8.9 / 9.0, 4 x 512 14.3 / 9.1, 64 x 512 14.9 / 11.8, 128 x 512 15.6 / 15.6, 256 x 512 16.6 / 19.9
//   bf16, D = 64:  4 x 256 7.2 / 8.2, 4 x 512 11.5 / 8.4, 128 x 512 12.2 / 11.9, 256 x 512 12.9 / 14.8 (uneven lengths 11.8 / 11.2)
//   bf16, D = 256: 4 x 256 12.7 / 10.4, 4 x 512 20.8 / 10.8, 64 x 512 21.7 / 16.5, 128 x 512 22.4 / 21.9, 256 x 512 26.4 / 32.0
//   fp32, D = 64:  4 x 128 8.0 / 9.8, 4 x 256 12.9 / 9.8, 128 x 256 13.5 / 13.3, 256 x 256 14.1 / 15.7, 256 x 512 24.6 / 21.6
//   fp32, D = 128: 4 x 128 12.4 / 12.7, 4 x 256 20.9 / 12.7, 128 x 256 21.6 / 17.9, 128 x 512 38.7 / 24.0, 256 x 512 40.0 / 35.7
// Past 512 tokens hundreds of even rows are 2 to 16 % faster whole (512 x 2048, bf16, D = 128: 98.5 / 103.4), few rows up to
// ten times slower (4 x 2048 45.4 / 9.4), and one long row among many short ones alone takes as long as it does whole: shared.
bool step_shares(double rows, double tokens, double wgs, int dtype) {
  return tokens > 512 || (tokens > (dtype == PF_DTYPE_BF16 ? 256 : 128) && rows * 4 <= wgs);
}

bool step_plan(int B, int H, int G, int D, int M, int page, int dtype, StepPlan& p) {
  p.blocks = (H / G + 15) / 16;
  const double rows = (double)B * G * p.blocks, tokens = (double)M * page;
  const double units = rows * ((tokens + pf::kStepUnit - 1) / pf::kStepUnit + 1);
  if (tokens > kMaxRows || units > kMaxRows) return false;       // (a run's end stays an int)
  p.rows = (int)rows;
  const double wgs = (double)kStepWgs * 128 / padded(D);
  p.wgs = step_shares(rows, tokens, wgs, dtype) ? (int)(units < wgs ? units : wgs) : 0;
  p.parts = (size_t)p.wgs * 2 * 16 * (padded(D) + 4);
  p.bytes = p.wgs ? p.parts * sizeof(float) + (size_t)p.rows * 4 * sizeof(int) : 0;
  return true;
}

template <typename E, int DP>
int step_launch(const pf::AttnStepArgs& a, const StepPlan& p, hipStream_t s) {
  dim3 grid, rows;
  if (!grid_of(p.wgs ? p.wgs : p.rows, grid) || !grid_of((double)a.B * a.H, rows)) return PF_ERR_ARG;
  pf::LaunchScope scope;
  pf::attn_step_kernel<E, DP><<<grid, dim3(64 * pf::kStepWaves), 0, s>>>(a);
  if (p.wgs) pf::attn_join_kernel<E, DP><<<rows, dim3(256), 0, s>>>(a);
  return scope.status();
}

template <typename E>
int step_heads(const pf::AttnStepArgs& a, const StepPlan& p, hipStream_t s) {
  return a.D <= 64 ? step_launch<E, 64>(a, p, s) : a.D <= 128 ? step_launch<E, 128>(a, p, s) : step_launch<E, 256>(a, p, s);
}

int log2_of(int page) {
  if (page < 16 || page > 65536 || (page & (page - 1))) return -1;
  return __builtin_ctz((unsigned)page);
}

}  // namespace

extern "C" {

int pf_attn_exec(const pf_attn_args* p, void* stream) {
  if (!p || p->size != sizeof *p || !heads_ok(p->H, p->G, p->D, p->dtype)) return PF_ERR_ARG;
  if (p->N < 0 || p->N > kMaxRows || p->B < 0 || p->B > kMaxRows || !p->cu || !(p->scale > 0.f)) return PF_ERR_ARG;
  if (p->N == 0) return PF_OK;
  if (!p->q || !p->k || !p->v || !p->o) return PF_ERR_ARG;
  if (!vectors(p->dtype, p->q, p->q_t, p->q_h) || !vectors(p->dtype, p->k, p->k_t, p->k_h) || !vectors(p->dtype, p->v, p->v_t, p->v_h))
    return PF_ERR_ARG;
  if (p->q_t > kMaxRowStride || p->k_t > kMaxRowStride || p->v_t > kMaxRowStride || p->o_t < 0 || p->o_h < 0) return PF_ERR_ARG;
  pf::AttnArgs a{};
  a.q = p->q; a.k = p->k; a.v = p->v; a.o = p->o; a.cu = p->cu; a.lengths = p->lengths;
  a.q_t = p->q_t; a.q_h = p->q_h; a.k_t = p->k_t; a.k_h = p->k_h; a.v_t = p->v_t; a.v_h = p->v_h; a.o_t = p->o_t; a.o_h = p->o_h;
  a.N = p->N; a.B = p->B; a.H = p->H; a.G = p->G; a.D = p->D; a.zero_rest = p->zero_rest;
  a.scale_log2 = p->scale * 1.44269504088896340736f;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return p->dtype == PF_DTYPE_BF16 ? attn_heads<bf16>(a, s) : attn_heads<float>(a, s);
}

size_t pf_attn_step_workspace_bytes(int B, int H, int G, int D, int M, int page, int dtype) {
  StepPlan pl;
  if (B <= 0 || M < 0 || !heads_ok(H, G, D, dtype) || log2_of(page) < 0 || !step_plan(B, H, G, D, M, page, dtype, pl)) return 0;
  return pl.bytes;
}

int pf_attn_step_exec(const pf_attn_step_args* p, void* stream) {
  if (!p || p->size != sizeof *p || !heads_ok(p->H, p->G, p->D, p->dtype) || log2_of(p->page) < 0) return PF_ERR_ARG;
  if (p->B < 0 || p->S < 0 || p->M < 0 || p->pages < 0 || !(p->scale > 0.f) || (!p->slots && p->B > p->S)) return PF_ERR_ARG;
  StepPlan pl;
  if (!step_plan(p->B, p->H, p->G, p->D, p->M, p->page, p->dtype, pl)) return PF_ERR_ARG;
  if (p->B == 0) return PF_OK;
  if (!p->q || !p->o || !p->lengths || (p->pages > 0 && (!p->k || !p->v)) || (!p->tables && p->S > 0 && p->M > 0)) return PF_ERR_ARG;
  if (!vectors(p->dtype, p->q, p->q_b, p->q_h) || !vectors(p->dtype, p->k, p->k_p, p->k_r, p->k_h) ||
      !vectors(p->dtype, p->v, p->v_p, p->v_r, p->v_h))
    return PF_ERR_ARG;
  if (p->k_r > kMaxRowStride || p->v_r > kMaxRowStride || p->o_b < 0 || p->o_h < 0) return PF_ERR_ARG;
  if (pl.bytes && (!p->workspace || p->workspace_bytes < pl.bytes || ((size_t)p->workspace & 15))) return PF_ERR_WORKSPACE;
  pf::AttnStepArgs a{};
  a.q = p->q; a.k = p->k; a.v = p->v; a.o = p->o; a.tables = p->tables; a.lengths = p->lengths; a.slots = p->slots;
  a.part = static_cast<float*>(p->workspace);
  a.spread = reinterpret_cast<int*>(a.part + pl.parts);
  a.q_b = p->q_b; a.q_h = p->q_h; a.o_b = p->o_b; a.o_h = p->o_h;
  a.k_p = p->k_p; a.k_r = p->k_r; a.k_h = p->k_h; a.v_p = p->v_p; a.v_r = p->v_r; a.v_h = p->v_h;
  a.B = p->B; a.S = p->S; a.H = p->H; a.G = p->G; a.D = p->D; a.M = p->M; a.pages = p->pages; a.page_log = log2_of(p->page);
  a.blocks = pl.blocks; a.wgs = pl.wgs;
  a.scale_log2 = p->scale * 1.44269504088896340736f;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return p->dtype == PF_DTYPE_BF16 ? step_heads<bf16>(a, pl, s) : step_heads<float>(a, pl, s);
}

}  // extern "C"
