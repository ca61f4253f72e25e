// extern "C" entry points of the short convolution, the single-token steps and the norm (declared in
// include/pto_fuser_hip.h): checks on the host, then one launch on the caller's stream.
#include <hip/hip_runtime.h>

#include "../../include/pto_fuser_hip.h"
#include "pf_conv.h"
#include "pf_norm.h"
#include "pf_status.h"
#include "pf_step.h"

namespace {

using pf::bf16;

bool known(int dtype) { return dtype == PF_DTYPE_F32 || dtype == PF_DTYPE_BF16; }

// The largest prompt and head: what is rounded up to whole tiles and counted past the end stays an int.
constexpr int kMaxSize = 1 << 30;

template <typename... S>
bool strides_ok(S... s) { return ((s >= 0) && ...); }

// The grid of `a` x `b` x `c` / `d` workgroups, and whether there is one.
bool grid_of(double a, double b, double c, double d, dim3& grid, long& blocks) {
  if (a * b * c / d > (double)pf::kGridX * (pf::kGridY - 1)) return false;
  blocks = ((long)a * (long)b * (long)c + (long)d - 1) / (long)d;
  grid = dim3((unsigned)(blocks < pf::kGridX ? blocks : pf::kGridX), (unsigned)((blocks + pf::kGridX - 1) / pf::kGridX));
  return true;
}

// ---- convolution ---------------------------------------------------------------------------
constexpr int kConvTokens = 8;      // tokens of a thread

template <typename E, int K, int VEC>
int conv_launch(pf::ConvArgs& a, hipStream_t s) {
  a.vectors = a.W / VEC;
  a.tiles = a.T ? (a.T + kConvTokens - 1) / kConvTokens : 1;
  dim3 grid;
  long launched;
  if (!grid_of(a.B, a.tiles, a.vectors, 256, grid, a.blocks)) return PF_ERR_ARG;
  grid_of((double)((a.blocks + 7) / 8 * 8), 1, 1, 1, grid, launched);
  a.threads = (long)a.B * a.tiles * a.vectors;
  pf::LaunchScope scope;
  pf::conv_kernel<E, K, VEC, kConvTokens><<<grid, dim3(256), 0, s>>>(a);
  return scope.status();
}

template <typename E, int K, int VEC>
int conv_launch(pf::ConvStepArgs& a, hipStream_t s) {
  a.vectors = a.W / VEC;
  dim3 grid;
  long blocks;
  if (!grid_of(a.B, 1, a.vectors, 256, grid, blocks)) return PF_ERR_ARG;
  a.threads = (long)a.B * a.vectors;
  pf::LaunchScope scope;
  pf::conv_step_kernel<E, K, VEC><<<grid, dim3(256), 0, s>>>(a);
  return scope.status();
}

// 16-byte vectors of channels where the width is a whole number of them, else single channels.
template <typename E, typename A>
int conv_width(A& a, int K, hipStream_t s) {
  constexpr int V = 16 / sizeof(E);
  const bool wide = a.W % V == 0;
  switch (K) {
    case 2: return wide ? conv_launch<E, 2, V>(a, s) : conv_launch<E, 2, 1>(a, s);
    case 3: return wide ? conv_launch<E, 3, V>(a, s) : conv_launch<E, 3, 1>(a, s);
    case 4: return wide ? conv_launch<E, 4, V>(a, s) : conv_launch<E, 4, 1>(a, s);
  }
  return PF_ERR_ARG;
}

// ---- single tokens -------------------------------------------------------------------------
template <typename E, bool DELTA, int LPR>
int step_rows(pf::StepArgs& a, int B, hipStream_t s) {
  constexpr int RP = 256 / LPR;
  a.slices = (a.P + 4 * LPR - 1) / (4 * LPR);
  dim3 grid, block(256);
  if (!grid_of(B, a.H, a.slices, 1, grid, a.blocks)) return PF_ERR_ARG;
  pf::LaunchScope scope;
  if (a.N <= 2 * RP) pf::step_kernel<E, DELTA, LPR, 2><<<grid, block, 0, s>>>(a);
  else if (a.N <= 4 * RP) pf::step_kernel<E, DELTA, LPR, 4><<<grid, block, 0, s>>>(a);
  else pf::step_kernel<E, DELTA, LPR, 8><<<grid, block, 0, s>>>(a);
  return scope.status();
}

template <bool DELTA>
int step(const pf_step_args* p, void* stream) {
  if (!p || p->size != sizeof *p || !known(p->dtype)) return PF_ERR_ARG;
  if (p->B < 0 || p->S < 0 || p->H <= 0 || p->G <= 0 || p->H % p->G || p->N <= 0 || p->N > 256 || p->P <= 0 || p->P % 4 || p->P > kMaxSize)
    return PF_ERR_ARG;
  if (DELTA && p->G != p->H) return PF_ERR_ARG;
  if (!strides_ok(p->v_b, p->v_h, p->k_b, p->k_h, p->q_b, p->q_h, p->y_b, p->y_h, p->dt_b, p->dt_h, p->z_b, p->z_h, p->state_b))
    return PF_ERR_ARG;
  if (!p->slots && p->B > p->S) return PF_ERR_ARG;
  if (p->B == 0) return PF_OK;                // (of no elements a pointer may be null)
  if (DELTA ? !p->beta : !p->dt || !p->a) return PF_ERR_ARG;
  if ((!p->state && p->S > 0) || !p->v || !p->k || !p->q || !p->y) return PF_ERR_ARG;
  pf::StepArgs a{};
  a.state = p->state; a.slots = p->slots; a.v = p->v; a.k = p->k; a.q = p->q; a.y = p->y;
  a.dt = p->dt; a.z = p->z; a.a = p->a; a.d = p->d; a.dt_bias = p->dt_bias; a.beta = p->beta; a.g = p->g;
  a.v_b = p->v_b; a.v_h = p->v_h; a.k_b = p->k_b; a.k_h = p->k_h; a.q_b = p->q_b; a.q_h = p->q_h;
  a.y_b = p->y_b; a.y_h = p->y_h; a.dt_b = p->dt_b; a.dt_h = p->dt_h; a.z_b = p->z_b; a.z_h = p->z_h;
  a.s_b = p->state_b;
  a.S = p->S; a.H = p->H; a.G = p->G; a.N = p->N; a.P = p->P;
  a.dt_f32 = p->dt_f32; a.softplus = p->softplus; a.g_rows = p->g_rows; a.scale = p->scale;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return p->dtype == PF_DTYPE_BF16 ? step_rows<bf16, DELTA, 8>(a, p->B, s) : step_rows<float, DELTA, 8>(a, p->B, s);
}

// ---- norm ----------------------------------------------------------------------------------
template <typename E, typename R, typename O, pf::NormOut OUT>
int norm_launch(const pf::NormArgs& a, hipStream_t s) {
  constexpr int V = 16 / sizeof(E);
  const int vectors = (a.D + V - 1) / V;
  const bool waves = vectors <= 256;       // a wave a row while four vectors a lane hold it, else a workgroup
  dim3 grid;
  long blocks;
  if (!grid_of(a.rows, 1, 1, waves ? 4 : 1, grid, blocks)) return PF_ERR_ARG;
  pf::LaunchScope scope;
  if (vectors <= 64) pf::norm_kernel<E, R, O, OUT, 64, 1><<<grid, 256, 0, s>>>(a);
  else if (vectors <= 128) pf::norm_kernel<E, R, O, OUT, 64, 2><<<grid, 256, 0, s>>>(a);
  else if (vectors <= 256) pf::norm_kernel<E, R, O, OUT, 64, 4><<<grid, 256, 0, s>>>(a);
  else if (vectors <= 512) pf::norm_kernel<E, R, O, OUT, 256, 2><<<grid, 256, 0, s>>>(a);
  else if (vectors <= 1024) pf::norm_kernel<E, R, O, OUT, 256, 4><<<grid, 256, 0, s>>>(a);
  else if (vectors <= 2048) pf::norm_kernel<E, R, O, OUT, 512, 4><<<grid, 512, 0, s>>>(a);
  else if (vectors <= 4096) pf::norm_kernel<E, R, O, OUT, 1024, 4><<<grid, 1024, 0, s>>>(a);
  else pf::norm_kernel<E, R, O, OUT, 1024, 8><<<grid, 1024, 0, s>>>(a);
  return scope.status();
}

template <typename E, typename R>
int norm_out(const pf::NormArgs& a, int y_dtype, int block, hipStream_t s) {
  if (y_dtype == PF_NORM_FP8)
    return block ? norm_launch<E, R, E, pf::NormOut::kFp8Block>(a, s) : norm_launch<E, R, E, pf::NormOut::kFp8Row>(a, s);
  return y_dtype == PF_DTYPE_BF16 ? norm_launch<E, R, bf16, pf::NormOut::kPlain>(a, s)
                                  : norm_launch<E, R, E, pf::NormOut::kPlain>(a, s);
}

}  // namespace

extern "C" {

int pf_conv_exec(const pf_conv_args* p, void* stream) {
  if (!p || p->size != sizeof *p || !known(p->dtype)) return PF_ERR_ARG;
  if (p->B < 0 || p->T < 0 || p->T > kMaxSize || p->W <= 0 || p->K < 2 || p->K > 4 || !p->w) return PF_ERR_ARG;
  if (p->T > 0 && p->B > 0 && (!p->x || !p->y)) return PF_ERR_ARG;
  if (!strides_ok(p->x_b, p->x_t, p->y_b, p->y_t, p->state_in_b, p->state_out_b)) return PF_ERR_ARG;
  if (p->B == 0) return PF_OK;
  pf::ConvArgs a{};
  a.x = p->x; a.w = p->w; a.bias = p->bias; a.state_in = p->state_in; a.lengths = p->lengths; a.y = p->y;
  a.state_out = p->state_out;
  a.x_b = p->x_b; a.x_t = p->x_t; a.y_b = p->y_b; a.y_t = p->y_t; a.si_b = p->state_in_b; a.so_b = p->state_out_b;
  a.B = p->B; a.T = p->T; a.W = p->W; a.w_f32 = p->w_f32; a.act = p->act;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return p->dtype == PF_DTYPE_BF16 ? conv_width<bf16>(a, p->K, s) : conv_width<float>(a, p->K, s);
}

int pf_conv_step_exec(const pf_conv_step_args* p, void* stream) {
  if (!p || p->size != sizeof *p || !known(p->dtype)) return PF_ERR_ARG;
  if (p->B < 0 || p->S < 0 || p->W <= 0 || p->K < 2 || p->K > 4 || !p->w) return PF_ERR_ARG;
  if (p->B > 0 && (!p->x || !p->y || (!p->state && p->S > 0))) return PF_ERR_ARG;
  if (!strides_ok(p->x_b, p->y_b, p->state_b) || (!p->slots && p->B > p->S)) return PF_ERR_ARG;
  if (p->B == 0) return PF_OK;
  pf::ConvStepArgs a{};
  a.x = p->x; a.w = p->w; a.bias = p->bias; a.state = p->state; a.slots = p->slots; a.y = p->y;
  a.x_b = p->x_b; a.y_b = p->y_b; a.s_b = p->state_b;
  a.B = p->B; a.S = p->S; a.W = p->W; a.w_f32 = p->w_f32; a.act = p->act;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  return p->dtype == PF_DTYPE_BF16 ? conv_width<bf16>(a, p->K, s) : conv_width<float>(a, p->K, s);
}

int pf_ssm_step_exec(const pf_step_args* args, void* stream) { return step<false>(args, stream); }
int pf_gdn_step_exec(const pf_step_args* args, void* stream) { return step<true>(args, stream); }

int pf_norm_exec(const pf_norm_args* p, void* stream) {
  if (!p || p->size != sizeof *p || !known(p->dtype)) return PF_ERR_ARG;
  if (p->rows < 0 || p->D <= 0 || p->D > 32768) return PF_ERR_ARG;
  const bool fp8 = p->y_dtype == PF_NORM_FP8;
  if (!fp8 && p->y_dtype != p->dtype && p->y_dtype != PF_DTYPE_BF16) return PF_ERR_ARG;
  if (p->scale_block != 0 && (!fp8 || p->scale_block != 128 || p->D % 128)) return PF_ERR_ARG;
  if (!strides_ok(p->x_row, p->residual_row, p->y_row, p->h_row)) return PF_ERR_ARG;
  if (p->rows == 0) return PF_OK;
  if (!p->x || !p->w || !p->y || (fp8 && !p->scales) || (p->h_out && !p->residual)) return PF_ERR_ARG;
  pf::NormArgs a{};
  a.x = p->x; a.residual = p->residual; a.w = p->w; a.y = p->y; a.scales = p->scales; a.h = p->h_out;
  a.x_row = p->x_row; a.r_row = p->residual_row; a.y_row = p->y_row; a.h_row = p->h_row;
  a.rows = p->rows; a.D = p->D; a.w_f32 = p->w_f32; a.eps = p->eps;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (p->dtype == PF_DTYPE_F32) return norm_out<float, float>(a, p->y_dtype, p->scale_block, s);
  return p->r_f32 ? norm_out<bf16, float>(a, p->y_dtype, p->scale_block, s)
                  : norm_out<bf16, bf16>(a, p->y_dtype, p->scale_block, s);
}

}  // extern "C"
