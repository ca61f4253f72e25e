// The bookkeeping of a cache in pages of 2^page_log rows, on the device: which pages new tokens take and which row each token
// has, and the storing of keys and values into those rows.
//
// Requests are served in order.  With c tokens in the cache and n new ones, request b needs ceil((c + n) / page) - ceil(c /
// page) pages: free[taken + those of all before it ..].  One that the rest of the pool does not hold gets none, and no later
// one that needs any does; so the ones served are a prefix, and a sum over the requests before gives each its place.
#pragma once

#include "pf_serving.h"

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
  int* place;              // [B] scratch: the first of a request's new pages in free; -1: it is not served
  int B, S, M, F, capacity, page_log;
  int fill;                // the first kernel's workgroup fills the rows too
};

__device__ __forceinline__ int pages_of(long tokens, int page_log) { return (int)((tokens + (1L << page_log) - 1) >> page_log); }

// Sums of two values over a workgroup's threads before each, and of all.
template <int THREADS>
__device__ __forceinline__ void scan2(long& x, long& y, long& all_x, long& all_y, long (*s)[THREADS / 64]) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  long ux = x, uy = y;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const long ox = __shfl_up(ux, d), oy = __shfl_up(uy, d);
    if (lane >= d) {
      ux += ox;
      uy += oy;
    }
  }
  if (lane == 63) {
    s[0][w] = ux;
    s[1][w] = uy;
  }
  __syncthreads();
  long bx = 0, by = 0;
  all_x = all_y = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 64; ++i) {
    if (i < w) {
      bx += s[0][i];
      by += s[1][i];
    }
    all_x += s[0][i];
    all_y += s[1][i];
  }
  __syncthreads();
  x = bx + ux - x;
  y = by + uy - y;
}

// The row of new token t, and the entry of a page that begins with it.
__device__ __forceinline__ void fill_row(const AssignArgs& a, int t) {
  long row = -1;
  if (t < a.cu[a.B]) {
    int lo = 0, hi = a.B;                            // the last request that begins at t or before has it
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      (a.cu[mid] <= t ? lo : hi) = mid;
    }
    const int place = a.place[lo];
    if (place >= 0) {
      const int c = max(a.lengths[lo], 0), at = c + t - a.cu[lo], index = at >> a.page_log, have = pages_of(c, a.page_log);
      const int off = at & ((1 << a.page_log) - 1);
      int* entry = a.tables + (long)(a.slots ? a.slots[lo] : lo) * a.M + index;
      int page;
      if (index >= have) {
        page = a.free[place + index - have];
        if (off == 0) *entry = page;
      } else {
        page = *entry;
      }
      if (page >= 0) row = ((long)page << a.page_log) + off;
    }
  }
  a.rows[t] = row;
}

template <int THREADS>
__global__ __launch_bounds__(THREADS) void assign_kernel(AssignArgs a) {
  __shared__ long s[2][THREADS / 64];
  const int tid = threadIdx.x;
  const long taken = min(max(a.taken[0], 0), a.F);
  long rows = 0, pages = 0, used = 0;                // new tokens and pages of the requests so far; pages that were given
  for (int b0 = 0; b0 < a.B; b0 += THREADS) {
    const int b = b0 + tid;
    long c = 0, n = 0, need = 0, limit = 0;
    if (b < a.B) {
      c = max(a.lengths[b], 0);
      n = a.tokens ? max(a.tokens[b], 0) : 1;
      limit = (long)a.M << a.page_log;
      const int slot = a.slots ? a.slots[b] : b;
      if (slot < 0 || slot >= a.S || c + n > limit) limit = -1;
      need = limit < 0 ? 0 : pages_of(c + n, a.page_log) - pages_of(c, a.page_log);
    }
    // (a request that its rows' capacity cuts off is not served either, and its need does not count: all that come before it
    // within the capacity are known from the first sum alone)
    long first = n, none = 0, all_n, all_none;
    scan2<THREADS>(first, none, all_n, all_none, s);
    first += rows;
    const bool fits = b < a.B && limit >= 0 && first + n <= a.capacity;
    long before = fits ? need : 0, given = 0, all_need, all_given;
    scan2<THREADS>(before, given, all_need, all_given, s);
    before += pages;
    const bool served = fits && (need == 0 || taken + before + need <= a.F);
    given = served ? need : 0;
    none = 0;
    scan2<THREADS>(given, none, all_given, all_none, s);
    used += all_given;
    if (b < a.B) {
      a.cu[b] = (int)min(first, (long)a.capacity);
      a.lengths_out[b] = (int)(served ? c + n : c);
      a.place[b] = served ? (int)(taken + min(before, a.F - taken)) : -1;
    }
    rows += all_n;
    pages += all_need;
  }
  if (tid == 0) {
    a.cu[a.B] = (int)min(rows, (long)a.capacity);
    a.taken_out[0] = (int)(taken + used);
  }
  if (!a.fill) return;
  __syncthreads();
  for (int t = tid; t < a.capacity; t += THREADS) fill_row(a, t);
}

__global__ __launch_bounds__(256) void assign_rows_kernel(AssignArgs a) {
  const long t = block_id() * 256 + threadIdx.x;
  if (t < a.capacity) fill_row(a, (int)t);
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
// were taken (a request released twice) keeps them.  A workgroup a request.
__global__ __launch_bounds__(256) void release_kernel(ReleaseArgs a) {
  __shared__ long s[2][4];
  const int mine = (int)block_id();
  const long taken = min(max(a.taken[0], 0), a.F);
  const auto pages = [&](int b) {
    const int slot = a.slots ? a.slots[b] : b;
    return slot < 0 || slot >= a.S ? 0L : (long)min(pages_of(max(a.lengths[b], 0), a.page_log), a.M);
  };
  // Of the requests up to this one (the last workgroup: of all, and of those that are released).
  long before = 0, n = 0;
  const bool last = mine == a.B;
  for (int b0 = 0; b0 < mine; b0 += 256) {
    const int b = b0 + threadIdx.x;
    long x = b < mine ? pages(b) : 0, y = 0, all, none;
    const long own = x;
    scan2<256>(x, y, all, none, s);
    if (last) {
      y = before + x + own <= taken ? own : 0;
      x = 0;
      long all_x;
      scan2<256>(x, y, all_x, none, s);
      n += none;
    }
    before += all;
  }
  if (last) {
    if (threadIdx.x == 0) a.taken_out[0] = (int)(taken - n);
    return;
  }
  n = pages(mine);
  if (before + n > taken) return;
  const int* row = a.tables + (long)(a.slots ? a.slots[mine] : mine) * a.M;
  for (long i = threadIdx.x; i < n; i += 256) a.free[taken - 1 - before - i] = row[i];
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
