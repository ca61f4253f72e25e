// The bookkeeping of a cache in pages of 2^page_log rows, on the device: which pages new tokens take and which row each token
// has, and the storing of keys and values into those rows.
//
// Requests are served in order.  With c tokens in the cache and n new ones, request b needs ceil((c + n) / page) - ceil(c /
// page) pages: free[taken + those of all before it ..].  One that the rest of the pool does not hold gets none, and no later
// one that needs any does; so the ones served are a prefix, and a sum over the requests before gives each its place.
//
// Latency, not bytes: 64 prompts of up to 1024 tokens 4.4 us, 256 requests of a token each 3.4 us (a launch of nothing takes 2.4);
// as one workgroup and a second launch for the rows they took 9.4 and 7.3.  Storing: 16384 tokens of 4 heads of 128, 67 MB
// 11.4 us, 5.9 TB/s (what the last pass wrote is partly still in the memory-side cache).  Marking requests that held tokens: 1.4 us
// for 64.
#pragma once

#include "pf_serving.h"

#include <type_traits>

namespace pf {

struct AssignArgs {
  int* tables;             // [S, M]
  const int* lengths;      // [B]: c
  const int* tokens;       // [B]: n, or null: one each
  const int* slots;        // [B] or null
  const int* free;         // [F]
  const int* taken;        // [1]
  long long* rows;         // [capacity]
  int* cu;                 // [B + 1]
  int* lengths_out;        // [B]
  int* taken_out;          // [1]
  int B, S, M, F, capacity, page_log;
};

// (tokens up to 2^31)
__device__ __forceinline__ uint32_t pages_of(uint32_t tokens, int page_log) {
  return (tokens >> page_log) + ((tokens & ((1u << page_log) - 1)) != 0);
}

// Sums that stay at 2^32 - 1 once they reach it, which is past every capacity and pool.
__device__ __forceinline__ uint32_t sat_add(uint32_t x, uint32_t y) { return __builtin_elementwise_add_sat(x, y); }

// A value's sum over the threads before each, added to `carry`, which then takes them all in.
__device__ __forceinline__ uint32_t block_sums(uint32_t v, uint32_t& carry, uint32_t (&s)[4]) {
  const int w = threadIdx.x >> 6;
  const auto moved = [](uint32_t x, auto ctrl, auto rows) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, decltype(rows)::value, 0xf, decltype(rows)::value == 0xf);
  };
  uint32_t u = v;
  u = sat_add(u, moved(u, std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xf>{}));
  u = sat_add(u, moved(u, std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xf>{}));
  u = sat_add(u, moved(u, std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xf>{}));
  u = sat_add(u, moved(u, std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xf>{}));
  u = sat_add(u, moved(u, std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{}));   // from row to row of 16
  u = sat_add(u, moved(u, std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{}));
  __syncthreads();
  if ((threadIdx.x & 63) == 63) s[w] = u;
  __syncthreads();
  // (the lane before's inclusive sum: a saturated sum less its own value would not be one)
  uint32_t before = (uint32_t)__shfl_up((int)u, 1);
  if ((threadIdx.x & 63) == 0) before = 0;
  uint32_t sum = carry;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i == w) before = sat_add(sum, before);
    sum = sat_add(sum, s[i]);
  }
  carry = sum;
  return before;
}

constexpr int kAssignTokens = 512;       // of a workgroup

// Every workgroup goes through all requests, 256 at a time, and fills the rows of its own tokens from them; the first also
// writes what is of requests.  So there is one launch, and none waits for another.
__global__ __launch_bounds__(256) void assign_kernel(AssignArgs a) {
  __shared__ uint32_t sums[4];
  __shared__ int s_cu[257], s_place[256], s_c[256], s_slot[256];
  const int tid = threadIdx.x;
  const uint32_t taken = (uint32_t)min(max(a.taken[0], 0), a.F), left = a.F - taken;
  const long mine = block_id() * kAssignTokens;
  const int t0 = (int)min(mine, (long)a.capacity), t1 = (int)min(mine + kAssignTokens, (long)a.capacity);
  const bool leads = blockIdx.x == 0 && blockIdx.y == 0;
  uint32_t rows = 0, pages = 0, used = 0;            // new tokens and pages of the requests so far; pages that were given
  for (int b0 = 0; b0 < a.B; b0 += 256) {
    const int b = b0 + tid;
    uint32_t c = 0, n = 0;
    int slot = -1;
    if (b < a.B) {
      c = (uint32_t)max(a.lengths[b], 0);
      n = a.tokens ? (uint32_t)max(a.tokens[b], 0) : 1u;
      slot = a.slots ? a.slots[b] : b;
    }
    const uint32_t first = block_sums(n, rows, sums);
    const bool fits = slot >= 0 && slot < a.S && c + n <= (uint32_t)a.M << a.page_log && sat_add(first, n) <= (uint32_t)a.capacity;
    const uint32_t need = fits ? pages_of(c + n, a.page_log) - pages_of(c, a.page_log) : 0;
    const uint32_t before = block_sums(need, pages, sums);
    const bool served = fits && (need == 0 || sat_add(before, need) <= left);
    if (served && need) used = before + need;
    const int start = (int)min(first, (uint32_t)a.capacity), after = (int)(served ? c + n : c);
    s_cu[tid] = start;
    s_place[tid] = served ? (int)(taken + min(before, left)) : -1;
    s_c[tid] = (int)c;
    s_slot[tid] = slot;
    if (tid == 0) s_cu[256] = (int)min(rows, (uint32_t)a.capacity);
    if (leads && b < a.B) {
      a.cu[b] = start;
      a.lengths_out[b] = after;
    }
    __syncthreads();
    for (int t = max(t0, s_cu[0]) + tid; t < min(t1, s_cu[256]); t += 256) {
      int lo = 0, hi = 256;                          // the last request that begins at t or before has it
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int mid = (lo + hi) / 2;
        (s_cu[mid] <= t ? lo : hi) = mid;
      }
      long row = -1;
      const int place = s_place[lo];
      if (place >= 0) {
        const int at = s_c[lo] + t - s_cu[lo], index = at >> a.page_log, have = (int)pages_of((uint32_t)s_c[lo], a.page_log);
        const int off = at & ((1 << a.page_log) - 1);
        int* entry = a.tables + (long)s_slot[lo] * a.M + index;
        int page;
        if (index >= have) {
          page = a.free[place + index - have];
          if (off == 0) *entry = page;               // (every new page begins with a new token)
        } else {
          page = *entry;
        }
        if (page >= 0) row = ((long)page << a.page_log) + off;
      }
      a.rows[t] = row;
    }
  }
  for (int t = max(t0, (int)min(rows, (uint32_t)a.capacity)) + tid; t < t1; t += 256) a.rows[t] = -1;
  if (!leads) return;
  // (pages given: up to the end of the last request that got any)
#pragma unroll
  for (int d = 32; d > 0; d /= 2) used = max(used, (uint32_t)__shfl_xor((int)used, d));
  __syncthreads();
  if ((tid & 63) == 0) sums[tid >> 6] = used;
  __syncthreads();
  if (tid == 0) {
    a.cu[a.B] = (int)min(rows, (uint32_t)a.capacity);
    a.taken_out[0] = (int)(taken + max(max(sums[0], sums[1]), max(sums[2], sums[3])));
  }
}

struct ReleaseArgs {
  const int* tables;
  const int* lengths;
  const int* slots;
  int* free;
  const int* taken;
  int* taken_out;
  int B, S, M, F, page_log;
};

// Request b's pages go back to free[taken - 1 - those of all before it ..] downwards; one that more pages come before than
// were taken (a request released twice) keeps them.  A workgroup a request, and one for what all give back.
__global__ __launch_bounds__(256) void release_kernel(ReleaseArgs a) {
  __shared__ uint32_t sums[4];
  const int mine = (int)block_id(), tid = threadIdx.x;
  if (mine > a.B) return;
  const uint32_t taken = (uint32_t)min(max(a.taken[0], 0), a.F);
  const auto pages = [&](int b) {
    const int slot = a.slots ? a.slots[b] : b;
    return slot < 0 || slot >= a.S ? 0u : min(pages_of((uint32_t)max(a.lengths[b], 0), a.page_log), (uint32_t)a.M);
  };
  uint32_t before = 0, back = 0;                     // pages of the requests before this one; of those, that go back
  for (int b0 = 0; b0 < mine; b0 += 256) {
    const uint32_t own = b0 + tid < mine ? pages(b0 + tid) : 0;
    const uint32_t x = block_sums(own, before, sums);
    if (own && sat_add(x, own) <= taken) back = x + own;
  }
  if (mine == a.B) {
#pragma unroll
    for (int d = 32; d > 0; d /= 2) back = max(back, (uint32_t)__shfl_xor((int)back, d));
    __syncthreads();
    if ((tid & 63) == 0) sums[tid >> 6] = back;
    __syncthreads();
    if (tid == 0) a.taken_out[0] = (int)(taken - max(max(sums[0], sums[1]), max(sums[2], sums[3])));
    return;
  }
  const uint32_t n = pages(mine);
  if (sat_add(before, n) > taken) return;
  const int* row = a.tables + (long)(a.slots ? a.slots[mine] : mine) * a.M;
  for (uint32_t i = tid; i < n; i += 256) a.free[taken - 1 - before - i] = row[i];
}

struct RefuseArgs {
  const int* cu;           // [B + 1]
  const int* lengths;      // [B]: after the plan
  const long long* rows;   // [N]
  void* k;
  long k_t, k_h;
  int N, B, G;
};

// A request held tokens before a plan where more are in the cache after it than the plan brought: all its new ones if its
// first has a row, else none.  Its first new key becomes NaN, in every head, which reaches each of its rows.
template <typename E>
__global__ __launch_bounds__(256) void refuse_kernel(RefuseArgs a) {
  const long b = block_id() * 256 + threadIdx.x;
  if (b >= a.B) return;
  const int first = a.cu[b], end = a.cu[b + 1];
  if (first < 0 || first >= min(end, a.N) || a.lengths[b] <= (a.rows[first] >= 0 ? end - first : 0)) return;
  for (int g = 0; g < a.G; ++g) static_cast<E*>(a.k)[first * a.k_t + g * a.k_h] = from_f32<E>(__builtin_nanf(""));
}

struct StoreArgs {
  const void* k;
  const void* v;
  void* k_cache;
  void* v_cache;
  const long long* rows;   // [N]
  long k_t, k_h, v_t, v_h, kc_p, kc_r, kc_h, vc_p, vc_r, vc_h;
  int N, G, D, pages, page_log;
};

// A 16-byte vector a thread, of k and of v.  Bound by memory.
template <typename E>
__global__ __launch_bounds__(256) void store_kernel(StoreArgs a) {
  constexpr int V = 16 / (int)sizeof(E);
  typedef typename VecAny<E, V>::T Vec;
  const uint32_t per = a.G * (a.D / V);
  const long i = block_id() * 256 + threadIdx.x;
  const long t = i / per;
  if (t >= a.N) return;
  const uint32_t u = (uint32_t)(i - t * per), g = u / (uint32_t)(a.D / V), col = u % (uint32_t)(a.D / V) * V;
  const long row = a.rows[t], page = row >> a.page_log, off = row & ((1L << a.page_log) - 1);
  if (row < 0 || page >= a.pages) return;
  const Vec x = *reinterpret_cast<const Vec*>(static_cast<const E*>(a.k) + t * a.k_t + g * a.k_h + col);
  const Vec y = *reinterpret_cast<const Vec*>(static_cast<const E*>(a.v) + t * a.v_t + g * a.v_h + col);
  *reinterpret_cast<Vec*>(static_cast<E*>(a.k_cache) + page * a.kc_p + off * a.kc_r + g * a.kc_h + col) = x;
  *reinterpret_cast<Vec*>(static_cast<E*>(a.v_cache) + page * a.vc_p + off * a.vc_r + g * a.vc_h + col) = y;
}

}  // namespace pf
