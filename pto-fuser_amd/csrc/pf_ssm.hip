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

// How a shape is cut: columns of a workgroup, blocks of them in a group's heads, segments of a sequence.
struct SsmPlan {
  int cols, blocks, segs, seg_chunks;
  size_t bytes;              // workspace of the segments
};

bool shape_ok(int B, int H, int G, int T, int N, int P, int dtype) {
  return B >= 0 && H > 0 && G > 0 && H % G == 0 && T >= 0 && T <= (1 << 30) && N > 0 && N <= 128 && N % 16 == 0 && P > 0 &&
         P <= 256 && P % 32 == 0 && (dtype == PF_DTYPE_F32 || dtype == PF_DTYPE_BF16);
}

int padded_rows(int N) { return N <= 64 ? 64 : 128; }

// The segments' states lie as the waves hold them: whole blocks of columns, rows padded.
size_t state_floats(long units, int segs, int cols, int N) { return (size_t)units * segs * cols * padded_rows(N); }

// What a plan takes in microseconds, to choose among plans by (one workgroup a CU, N = 128): whole sequences a fixed part and
// a step a chunk; segments a fixed part for three launches, a step of both kernels a chunk of a segment, the sum along the
// segments and the traffic of their states.  A step of 64 columns takes nearly as long as one of 256 (it is latency, not
// throughput), so wide blocks win once there are enough of them to fill the chip, narrow ones before.  32 heads of 64, bf16,
// us at 64 / 128 / 256 columns: 1 x 512 tokens 24.4 / 24.3 / 25.1 (8 segments; whole 46 / 47 / 57), 4 x 2048 79 / 78 / 67
// (whole 166 / 168 / 209), 16 x 256 whole 31 / 30 / 36 (two segments of 256 columns 49), 16 x 1024 92 / 91 / 111 whole, 105 in
// two segments of 256, 2 x 8192 133 / 133 / 105 in 8, 8 and 16 segments.
// As a time it is right to 5 % at the long ones of these (4 x 2048 67 for 67, 16 x 1024 90 for 91, 2 x 8192 104 for 105), and not
// elsewhere: 28 for 24 at 1 x 512, 177 for 217 at 1 x 32768 with z, which it does not know, 44 for 31 at 3 x 1471 fp32 with
// 64 rows, which it takes for 128.
struct SsmCost {
  int cols;
  double whole0, whole_step, seg0, seg_step;
};
constexpr SsmCost kCost[2][3] = {{{64, 10, 8.5, 15, 11.5}, {128, 10, 12.5, 17, 17}, {0, 0, 0, 0, 0}},
                                 {{64, 10, 5, 13, 8}, {128, 10, 5, 14, 8}, {256, 12, 6, 15, 8.5}}};

SsmPlan plan(int B, int H, int G, int T, int N, int P, int dtype) {
  const int chunks = (T + pf::kSsmChunk - 1) / pf::kSsmChunk;
  const long width = (long)(H / G) * P;
  SsmPlan best{};
  double least = 0;
  for (const SsmCost& c : kCost[dtype == PF_DTYPE_BF16]) {
    if (!c.cols || (c.cols > 64 && width <= c.cols / 2)) continue;
    SsmPlan p{};
    p.cols = c.cols;
    p.blocks = (int)((width + c.cols - 1) / c.cols);
    const long units = (long)B * G * p.blocks;
    const auto consider = [&](int seg_chunks, double us) {
      if (best.cols && us >= least) return;
      p.seg_chunks = seg_chunks;
      p.segs = chunks ? (chunks + seg_chunks - 1) / seg_chunks : 1;
      best = p;
      least = us;
    };
    consider(chunks ? chunks : 1, (double)((units + pf::kCus - 1) / pf::kCus) * (c.whole0 + c.whole_step * chunks));
    long most = units > 0 ? pf::kCus / units : 1;       // one generation of workgroups
    if (most > chunks) most = chunks;
    for (; most >= 2; most /= 2) {
      const int each = (int)((chunks + most - 1) / most), segs = (chunks + each - 1) / each;
      if (segs < 2) break;
      consider(each, c.seg0 + c.seg_step * each + 0.35 * segs + (double)units * segs * c.cols * padded_rows(N) * 16 / 9e6);
    }
  }
  const long units = (long)B * G * best.blocks;
  best.bytes = best.segs > 1 ? (state_floats(units, best.segs, best.cols, N) + (size_t)B * H * best.segs) * sizeof(float) : 0;
  return best;
}

constexpr double kMaxTasks = 1 << 22;   // workgroups of up to 1024 threads in one grid dimension

bool grid_of(double workgroups, dim3& grid) {
  if (workgroups > (double)pf::kGridX * (pf::kGridY - 1)) return false;
  const long n = (long)workgroups;
  grid = dim3((unsigned)(n < pf::kGridX ? n : pf::kGridX), (unsigned)((n + pf::kGridX - 1) / pf::kGridX));
  return true;
}

template <typename E, int NT, int NW, int PT, int SPLIT>
void outputs(const pf::SsmArgs& a, dim3 grid, hipStream_t s) {
  if (a.z) pf::ssm_kernel<E, NT, NW, PT, SsmMode::kOutput, SPLIT, true><<<grid, dim3(NW * 64), 0, s>>>(a);
  else pf::ssm_kernel<E, NT, NW, PT, SsmMode::kOutput, SPLIT, false><<<grid, dim3(NW * 64), 0, s>>>(a);
}

template <typename E, int NT, int COLS>
int launch(pf::SsmArgs& a, hipStream_t s) {
  constexpr bool kF32 = std::is_same<E, float>::value;
  constexpr int PT = kF32 ? 1 : 2, NW = COLS / (16 * PT);
  const double tasks = (double)a.B * a.G * a.blocks * a.segs;
  if (tasks > kMaxTasks) return PF_ERR_ARG;
  a.tasks = (uint32_t)tasks;
  const dim3 grid((a.tasks + 7) / 8 * 8);
  dim3 prefix;
  const double prefix_blocks = tasks / a.segs * (COLS * NT / 4 / 256);
  if (!grid_of((double)((long)(prefix_blocks + 7) / 8 * 8), prefix)) return PF_ERR_ARG;
  pf::LaunchScope scope;
  if (a.segs > 1) {
    pf::ssm_kernel<E, NT, NW, PT, SsmMode::kStates, kF32 ? 1 : 3, false><<<grid, dim3(NW * 64), 0, s>>>(a);
    pf::ssm_prefix_kernel<NT, PT, COLS><<<prefix, dim3(256), 0, s>>>(a);
    outputs<E, NT, NW, PT, kF32 ? 1 : 2>(a, grid, s);
  } else {
    outputs<E, NT, NW, PT, kF32 ? 1 : 3>(a, grid, s);
  }
  return scope.status();
}

template <typename E, int NT>
int launch_cols(pf::SsmArgs& a, int cols, hipStream_t s) {
  if constexpr (std::is_same<E, bf16>::value)
    if (cols == 256) return launch<E, NT, 256>(a, s);
  return cols == 128 ? launch<E, NT, 128>(a, s) : launch<E, NT, 64>(a, s);
}

}  // namespace

extern "C" {

size_t pf_ssm_workspace_bytes(int B, int H, int G, int T, int N, int P, int dtype) {
  if (!shape_ok(B, H, G, T, N, P, dtype) || (double)B * H * N * P > 1e12) return 0;
  return plan(B, H, G, T, N, P, dtype).bytes;
}

int pf_ssm_exec(const pf_ssm_args* p, void* stream) {
  if (!p || p->size != sizeof *p || !shape_ok(p->B, p->H, p->G, p->T, p->N, p->P, p->dtype)) return PF_ERR_ARG;
  if ((double)p->B * p->H * p->N * p->P > 1e12 || !p->a) return PF_ERR_ARG;
  if (p->B == 0) return PF_OK;
  if (p->T > 0 && p->B > 0 && (!p->x || !p->dt || !p->b || !p->c || !p->y)) return PF_ERR_ARG;
  for (long long st : {p->x_b, p->x_h, p->x_t, p->dt_b, p->dt_h, p->dt_t, p->b_b, p->b_g, p->b_t, p->c_b, p->c_g, p->c_t,
                       p->z_b, p->z_h, p->z_t, p->y_b, p->y_h, p->y_t})
    if (st < 0) return PF_ERR_ARG;
  // A chunk's rows are read up to the end of the last live one: a token's stride covers its row, whatever it is of one token.
  const bool many = p->T > 1;
  const long long x_t = many ? p->x_t : p->P, y_t = many ? p->y_t : p->P, z_t = many && p->z ? p->z_t : p->P,
                  b_t = many ? p->b_t : p->N, c_t = many ? p->c_t : p->N;
  if (x_t < p->P || y_t < p->P || z_t < p->P || b_t < p->N || c_t < p->N) return PF_ERR_ARG;
  for (long long st : {x_t, y_t, z_t, b_t, c_t})
    if (st > pf::kMaxTokenStride) return PF_ERR_ARG;
  SsmPlan pl = plan(p->B, p->H, p->G, p->T, p->N, p->P, p->dtype);
  if (!p->workspace || p->workspace_bytes < pl.bytes || ((size_t)p->workspace & 15)) {   // whole sequences
    pl.segs = 1;
    pl.seg_chunks = (p->T + pf::kSsmChunk - 1) / pf::kSsmChunk;
  }
  pf::SsmArgs a{};
  a.x = p->x; a.dt = p->dt; a.b = p->b; a.c = p->c; a.z = p->z; a.a = p->a; a.d = p->d; a.dt_bias = p->dt_bias;
  a.h0 = p->h0; a.lengths = p->lengths; a.y = p->y; a.h_final = p->h_final;
  a.seg_state = static_cast<float*>(p->workspace);
  a.seg_decay = a.seg_state + state_floats((long)p->B * p->G * pl.blocks, pl.segs, pl.cols, p->N);
  a.x_b = p->x_b; a.x_h = p->x_h; a.x_t = x_t; a.dt_b = p->dt_b; a.dt_h = p->dt_h; a.dt_t = p->dt_t;
  a.b_b = p->b_b; a.b_g = p->b_g; a.b_t = b_t; a.c_b = p->c_b; a.c_g = p->c_g; a.c_t = c_t;
  a.z_b = p->z_b; a.z_h = p->z_h; a.z_t = z_t; a.y_b = p->y_b; a.y_h = p->y_h; a.y_t = y_t;
  a.B = p->B; a.H = p->H; a.G = p->G; a.T = p->T; a.N = p->N; a.P = p->P;
  a.blocks = pl.blocks; a.segs = pl.segs; a.seg_chunks = pl.seg_chunks;
  a.dt_f32 = p->dt_f32; a.softplus = p->softplus;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (p->dtype == PF_DTYPE_BF16)
    return padded_rows(p->N) == 64 ? launch_cols<bf16, 64>(a, pl.cols, s) : launch_cols<bf16, 128>(a, pl.cols, s);
  return padded_rows(p->N) == 64 ? launch_cols<float, 64>(a, pl.cols, s) : launch_cols<float, 128>(a, pl.cols, s);
}

}  // extern "C"
