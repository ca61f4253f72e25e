// extern "C" entry points of the paged cache's bookkeeping (declared in include/pto_fuser_hip.h).
#include <hip/hip_runtime.h>

#include "../../include/pto_fuser_hip.h"
#include "pf_pages.h"
#include "pf_status.h"

namespace {

using pf::bf16;

int log2_of(int page) {
  if (page < 16 || page > 65536 || (page & (page - 1))) return -1;
  return __builtin_ctz((unsigned)page);
}

bool grid_of(double workgroups, dim3& grid) {
  if (workgroups > (double)pf::kGridX * (pf::kGridY - 1)) return false;
  const long n = (long)workgroups;
  grid = dim3((unsigned)(n < pf::kGridX ? n : pf::kGridX), (unsigned)((n + pf::kGridX - 1) / pf::kGridX));
  return true;
}

}  // namespace

extern "C" {

int pf_assign_exec(const pf_assign_args* p, void* stream) {
  if (!p || p->size != sizeof *p || log2_of(p->page) < 0) return PF_ERR_ARG;
  if (p->B < 0 || p->S < 0 || p->M < 0 || p->F < 0 || p->capacity < 0 || (!p->slots && p->B > p->S)) return PF_ERR_ARG;
  if ((double)p->M * p->page > (double)(1 << 30) || p->B == 0x7fffffff) return PF_ERR_ARG;
  if (!p->cu || !p->taken || !p->taken_out || (p->capacity > 0 && !p->rows)) return PF_ERR_ARG;
  if (p->B > 0 && (!p->lengths || !p->lengths_out)) return PF_ERR_ARG;
  if ((p->F > 0 && !p->free) || (p->S > 0 && p->M > 0 && !p->tables)) return PF_ERR_ARG;
  pf::AssignArgs a{};
  a.tables = p->tables; a.lengths = p->lengths; a.tokens = p->tokens; a.slots = p->slots; a.free = p->free; a.taken = p->taken;
  a.rows = p->rows; a.cu = p->cu; a.lengths_out = p->lengths_out; a.taken_out = p->taken_out;
  a.B = p->B; a.S = p->S; a.M = p->M; a.F = p->F; a.capacity = p->capacity; a.page_log = log2_of(p->page);
  dim3 grid;
  if (!grid_of(a.capacity ? ((double)a.capacity + pf::kAssignTokens - 1) / pf::kAssignTokens : 1, grid)) return PF_ERR_ARG;
  pf::LaunchScope scope;
  pf::assign_kernel<<<grid, 256, 0, static_cast<hipStream_t>(stream)>>>(a);
  return scope.status();
}

int pf_release_exec(const pf_release_args* p, void* stream) {
  if (!p || p->size != sizeof *p || log2_of(p->page) < 0) return PF_ERR_ARG;
  if (p->B < 0 || p->S < 0 || p->M < 0 || p->F < 0 || (!p->slots && p->B > p->S)) return PF_ERR_ARG;
  if (!p->taken || !p->taken_out || (p->B > 0 && !p->lengths) || (p->F > 0 && !p->free)) return PF_ERR_ARG;
  if (p->S > 0 && p->M > 0 && !p->tables) return PF_ERR_ARG;
  dim3 grid;
  if (!grid_of((double)p->B + 1, grid)) return PF_ERR_ARG;
  pf::ReleaseArgs a{};
  a.tables = p->tables; a.lengths = p->lengths; a.slots = p->slots; a.free = p->free; a.taken = p->taken; a.taken_out = p->taken_out;
  a.B = p->B; a.S = p->S; a.M = p->M; a.F = p->F; a.page_log = log2_of(p->page);
  pf::LaunchScope scope;
  pf::release_kernel<<<grid, 256, 0, static_cast<hipStream_t>(stream)>>>(a);
  return scope.status();
}

int pf_refuse_exec(const pf_refuse_args* p, void* stream) {
  if (!p || p->size != sizeof *p || (p->dtype != PF_DTYPE_F32 && p->dtype != PF_DTYPE_BF16)) return PF_ERR_ARG;
  if (p->N < 0 || p->B < 0 || p->B == 0x7fffffff || p->G <= 0 || p->G > 65536 || p->k_t < 0 || p->k_h < 0) return PF_ERR_ARG;
  if (p->N == 0 || p->B == 0) return PF_OK;
  if (!p->cu || !p->lengths || !p->rows || !p->k) return PF_ERR_ARG;
  pf::RefuseArgs a{};
  a.cu = p->cu; a.lengths = p->lengths; a.rows = p->rows; a.k = p->k; a.k_t = p->k_t; a.k_h = p->k_h;
  a.N = p->N; a.B = p->B; a.G = p->G;
  dim3 grid;
  if (!grid_of(((double)a.B + 255) / 256, grid)) return PF_ERR_ARG;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  pf::LaunchScope scope;
  if (p->dtype == PF_DTYPE_BF16) pf::refuse_kernel<bf16><<<grid, 256, 0, s>>>(a);
  else pf::refuse_kernel<float><<<grid, 256, 0, s>>>(a);
  return scope.status();
}

int pf_store_exec(const pf_store_args* p, void* stream) {
  if (!p || p->size != sizeof *p || log2_of(p->page) < 0 || (p->dtype != PF_DTYPE_F32 && p->dtype != PF_DTYPE_BF16)) return PF_ERR_ARG;
  if (p->N < 0 || p->G <= 0 || p->G > 65536 || p->D <= 0 || p->D > 65536 || p->D % 8 || p->pages < 0) return PF_ERR_ARG;
  for (long long st : {p->k_t, p->k_h, p->v_t, p->v_h, p->kc_p, p->kc_r, p->kc_h, p->vc_p, p->vc_r, p->vc_h})
    if (st < 0) return PF_ERR_ARG;
  if (p->N == 0 || p->pages == 0) return PF_OK;
  if (!p->k || !p->v || !p->k_cache || !p->v_cache || !p->rows) return PF_ERR_ARG;
  pf::StoreArgs a{};
  a.k = p->k; a.v = p->v; a.k_cache = p->k_cache; a.v_cache = p->v_cache; a.rows = p->rows;
  a.k_t = p->k_t; a.k_h = p->k_h; a.v_t = p->v_t; a.v_h = p->v_h;
  a.kc_p = p->kc_p; a.kc_r = p->kc_r; a.kc_h = p->kc_h; a.vc_p = p->vc_p; a.vc_r = p->vc_r; a.vc_h = p->vc_h;
  a.N = p->N; a.G = p->G; a.D = p->D; a.pages = p->pages; a.page_log = log2_of(p->page);
  const int V = p->dtype == PF_DTYPE_BF16 ? 8 : 4;
  dim3 grid;
  if (!grid_of(((double)a.N * a.G * (a.D / V) + 255) / 256, grid)) return PF_ERR_ARG;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  pf::LaunchScope scope;
  if (p->dtype == PF_DTYPE_BF16) pf::store_kernel<bf16><<<grid, 256, 0, s>>>(a);
  else pf::store_kernel<float><<<grid, 256, 0, s>>>(a);
  return scope.status();
}

}  // extern "C"
