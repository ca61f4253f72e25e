// extern "C" entry points of the selective state space scan (declared in include/pto_fuser_hip.h): checks and the number
// of segments on the host, then one launch, or three for segmented sequences.
#include <hip/hip_runtime.h>

#include "../../include/pto_fuser_hip.h"
#include "pf_segments.h"
#include "pf_ssm.h"
#include "pf_status.h"

namespace {

using pf::bf16;
using pf::SsmMode;

// How a shape is cut: waves of a workgroup, heads of a workgroup, blocks of heads of a group, segments of a sequence.
struct SsmPlan {
  int waves, heads, blocks, segs, seg_chunks;
  size_t bytes;              // workspace of the segments
};

bool shape_ok(int B, int H, int G, int T, int N, int P, int dtype) {
  return B >= 0 && H > 0 && G > 0 && H % G == 0 && T >= 0 && T <= (1 << 30) && N > 0 && N <= 128 && N % 16 == 0 && P > 0 &&
         P <= 256 && P % 32 == 0 && (dtype == PF_DTYPE_F32 || dtype == PF_DTYPE_BF16);
}

size_t state_bytes(long chains, int segs, int N, int P) {
  return (size_t)chains * segs * N * P * sizeof(float) + (size_t)chains * segs * sizeof(float);
}

SsmPlan plan(int B, int H, int G, int T, int N, int P) {
  SsmPlan p{};
  const int R = H / G, per_head = P / 32;
  const long need = (long)R * per_head;
  p.waves = need <= 2 && per_head <= 2 ? 2 : need <= 4 && per_head <= 4 ? 4 : 8;
  p.heads = p.waves / per_head < R ? p.waves / per_head : R;
  p.blocks = (R + p.heads - 1) / p.heads;
  const int chunks = (T + pf::kSsmChunk - 1) / pf::kSsmChunk;
  const long units = (long)B * G * p.blocks;
  // Segments while they fit one generation of workgroups, of two chunks at least.
  long segs = units > 0 ? pf::kCus / units : 1;
  if (segs > chunks / 2) segs = chunks / 2;
  if (segs < 2) segs = 1;
  p.seg_chunks = chunks ? (int)((chunks + segs - 1) / segs) : 1;
  p.segs = chunks ? (chunks + p.seg_chunks - 1) / p.seg_chunks : 1;
  p.bytes = p.segs > 1 ? state_bytes((long)B * H, p.segs, N, P) : 0;
  return p;
}

bool grid_of(double workgroups, dim3& grid) {
  if (workgroups > (double)pf::kGridX * (pf::kGridY - 1)) return false;
  const long n = (long)workgroups;
  grid = dim3((unsigned)(n < pf::kGridX ? n : pf::kGridX), (unsigned)((n + pf::kGridX - 1) / pf::kGridX));
  return true;
}

template <typename E, int NT, int NW, SsmMode MODE, int SPLIT>
void scan(const pf::SsmArgs& a, dim3 grid, hipStream_t s) {
  pf::ssm_kernel<E, NT, NW, MODE, SPLIT><<<grid, dim3(NW * 64), 0, s>>>(a);
}

template <typename E, int NT, int NW>
int launch(pf::SsmArgs& a, hipStream_t s) {
  constexpr bool kF32 = std::is_same<E, float>::value;
  a.tasks = (long)a.B * a.G * a.blocks * a.segs;
  const long per = (a.tasks + 7) / 8;
  dim3 grid, prefix;
  if (!grid_of(8. * per, grid) || !grid_of(((double)a.N * a.P / 4 * a.B * a.H + 255) / 256, prefix)) return PF_ERR_ARG;
  pf::LaunchScope scope;
  if (a.segs > 1) {
    scan<E, NT, NW, SsmMode::kStates, kF32 ? 1 : 3>(a, grid, s);
    pf::ssm_prefix_kernel<<<prefix, dim3(256), 0, s>>>(a);
    scan<E, NT, NW, SsmMode::kOutput, kF32 ? 1 : 2>(a, grid, s);
  } else {
    scan<E, NT, NW, SsmMode::kOutput, kF32 ? 1 : 3>(a, grid, s);
  }
  return scope.status();
}

template <typename E, int NT>
int launch_waves(pf::SsmArgs& a, int waves, hipStream_t s) {
  return waves == 2 ? launch<E, NT, 2>(a, s) : waves == 4 ? launch<E, NT, 4>(a, s) : launch<E, NT, 8>(a, s);
}

}  // namespace

extern "C" {

size_t pf_ssm_workspace_bytes(int B, int H, int G, int T, int N, int P, int dtype) {
  if (!shape_ok(B, H, G, T, N, P, dtype) || (double)B * H * N * P > 1e12) return 0;
  return plan(B, H, G, T, N, P).bytes;
}

int pf_ssm_exec(const pf_ssm_args* p, void* stream) {
  if (!p || p->size != sizeof *p || !shape_ok(p->B, p->H, p->G, p->T, p->N, p->P, p->dtype)) return PF_ERR_ARG;
  if ((double)p->B * p->H * p->N * p->P > 1e12 || !p->a) return PF_ERR_ARG;
  if (p->T > 0 && p->B > 0 && (!p->x || !p->dt || !p->b || !p->c || !p->y)) return PF_ERR_ARG;
  for (long long st : {p->x_b, p->x_h, p->x_t, p->dt_b, p->dt_h, p->dt_t, p->b_b, p->b_g, p->b_t, p->c_b, p->c_g, p->c_t,
                       p->z_b, p->z_h, p->z_t, p->y_b, p->y_h, p->y_t})
    if (st < 0) return PF_ERR_ARG;
  if (p->B == 0) return PF_OK;
  SsmPlan pl = plan(p->B, p->H, p->G, p->T, p->N, p->P);
  if (!p->workspace || p->workspace_bytes < pl.bytes || ((size_t)p->workspace & 15)) {   // whole sequences
    pl.segs = 1;
    pl.seg_chunks = (p->T + pf::kSsmChunk - 1) / pf::kSsmChunk;
  }
  pf::SsmArgs a{};
  a.x = p->x; a.dt = p->dt; a.b = p->b; a.c = p->c; a.z = p->z; a.a = p->a; a.d = p->d; a.dt_bias = p->dt_bias;
  a.h0 = p->h0; a.lengths = p->lengths; a.y = p->y; a.h_final = p->h_final;
  a.seg_state = static_cast<float*>(p->workspace);
  a.seg_decay = a.seg_state + (size_t)p->B * p->H * pl.segs * p->N * p->P;
  a.x_b = p->x_b; a.x_h = p->x_h; a.x_t = p->x_t; a.dt_b = p->dt_b; a.dt_h = p->dt_h; a.dt_t = p->dt_t;
  a.b_b = p->b_b; a.b_g = p->b_g; a.b_t = p->b_t; a.c_b = p->c_b; a.c_g = p->c_g; a.c_t = p->c_t;
  a.z_b = p->z_b; a.z_h = p->z_h; a.z_t = p->z_t; a.y_b = p->y_b; a.y_h = p->y_h; a.y_t = p->y_t;
  a.B = p->B; a.H = p->H; a.G = p->G; a.T = p->T; a.N = p->N; a.P = p->P;
  a.heads = pl.heads; a.blocks = pl.blocks; a.segs = pl.segs; a.seg_chunks = pl.seg_chunks;
  a.dt_f32 = p->dt_f32; a.softplus = p->softplus;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (p->dtype == PF_DTYPE_BF16)
    return p->N <= 64 ? launch_waves<bf16, 64>(a, pl.waves, s) : launch_waves<bf16, 128>(a, pl.waves, s);
  return p->N <= 64 ? launch_waves<float, 64>(a, pl.waves, s) : launch_waves<float, 128>(a, pl.waves, s);
}

}  // extern "C"
