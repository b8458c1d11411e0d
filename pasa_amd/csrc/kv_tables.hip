// Block tables, slots and positions of a step, from the requests' lengths.
//
// Request r has lens[r] cached tokens and new_tokens[r] new ones.  With page size P:
//   cu[r + 1] = min(tokens, cu[r] + new[r])                     first new token of each request
//   need[r]   = ceil((len + new) / P) - ceil(len / P)           pages it takes from the free list, in order of r
//   pages come from the end of free_pages[0 .. num_free)
//   token t of request r: position = len + t - cu[r], slot = table[r][position / P] * P + position % P
// Where the free list or the table's width ends, the tokens without a page have slot -1 and lens_out counts those
// that have one.  Tokens behind the last request have slot and position -1.
//
// A handful of integers a token: bound by the launch and by the two prefix sums.  One kernel: every workgroup sums
// over the requests by itself (8 bytes a request, from L2) rather than waiting for a first kernel to do it, then
// takes its share of the tokens; the token at the start of a page writes the page's table entry.
#include "common.h"
#include "kv_cache.h"

namespace pasa {

namespace {

constexpr int kThreads = 256;

// Exclusive prefix sum of x over the workgroup; the total in *total.
__device__ __forceinline__ int64_t scan_excl(int64_t x, int64_t* tmp, int64_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t s = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t y = __shfl_up(s, d, 64);
    if (lane >= d) s += y;
  }
  __syncthreads();
  if (lane == 63) tmp[wave] = s;
  __syncthreads();
  int64_t base = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w < wave) base += tmp[w];
    sum += tmp[w];
  }
  *total = sum;
  return base + s - x;
}

__global__ __launch_bounds__(kThreads) void kv_tables(KvTablesParams p, int per_wg) {
  extern __shared__ int32_t sh[];  // cu[requests + 1], before[requests]
  __shared__ int64_t tmp[kThreads / 64];
  const int R = p.requests;
  int32_t* cu = sh;
  int32_t* before = sh + R + 1;
  const int tid = threadIdx.x;
  const int each = (R + kThreads - 1) / kThreads;
  const int r0 = min(R, tid * each), r1 = min(R, r0 + each);
  const int64_t cap = min(p.width << p.page_log2, (int64_t)0x7fffffff);
  const int page_mask = (1 << p.page_log2) - 1;
  auto len_of = [&](int r) { return min(max((int64_t)p.lens[r], (int64_t)0), cap); };
  auto pages = [&](int64_t n) { return (n + page_mask) >> p.page_log2; };

  int64_t sum = 0, total;
  for (int r = r0; r < r1; ++r) sum += max(p.new_tokens[r], 0);
  int64_t at = scan_excl(sum, tmp, &total);
  for (int r = r0; r < r1; ++r) {
    cu[r] = (int32_t)min(at, p.tokens);
    at += max(p.new_tokens[r], 0);
  }
  if (tid == 0) cu[R] = (int32_t)min(total, p.tokens);
  __syncthreads();
  sum = 0;
  for (int r = r0; r < r1; ++r) {
    const int64_t len = len_of(r);
    sum += pages(min(len + cu[r + 1] - cu[r], cap)) - pages(len);
  }
  at = scan_excl(sum, tmp, &total);
  const int64_t num_free = min(max((int64_t)p.num_free[0], (int64_t)0), p.free_cap);
  for (int r = r0; r < r1; ++r) {
    const int64_t len = len_of(r), want = len + cu[r + 1] - cu[r];
    const int64_t had = pages(len), need = pages(min(want, cap)) - had;
    before[r] = (int32_t)min(at, (int64_t)0x7fffffff);
    if (blockIdx.x == 0) {
      const int64_t got = min(max(num_free - at, (int64_t)0), need);
      p.cu_q[r] = cu[r];
      p.lens_out[r] = (int32_t)min(want, (had + got) << p.page_log2);
    }
    at += need;
  }
  if (blockIdx.x == 0 && tid == 0) {
    p.cu_q[R] = cu[R];
    p.num_free_out[0] = (int32_t)max(num_free - total, (int64_t)0);
  }
  __syncthreads();

  const int64_t t0 = (int64_t)blockIdx.x * per_wg;
  const int64_t t1 = min(p.tokens, t0 + per_wg);
  for (int64_t t = t0 + tid; t < t1; t += kThreads) {
    if (t >= cu[R]) {
      p.slots[t] = -1;
      p.positions[t] = -1;
      continue;
    }
    int lo = 0, hi = R;  // the last request whose first token is at or before t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (cu[mid] <= t) lo = mid;
      else hi = mid;
    }
    const int64_t len = len_of(lo);
    const int64_t pos = len + t - cu[lo], lp = pos >> p.page_log2, had = pages(len);
    int64_t id = -1;
    if (lp < p.width) {
      if (lp < had) {
        id = p.tables[lo * p.stride + lp];
      } else {
        const int64_t i = num_free - 1 - (before[lo] + lp - had);
        if (i >= 0) {
          id = p.free_pages[i];
          if ((pos & page_mask) == 0) p.tables[lo * p.stride + lp] = (int32_t)id;
        }
      }
    }
    p.slots[t] = id < 0 ? -1 : (id << p.page_log2) + (pos & page_mask);
    p.positions[t] = (int32_t)min(pos, (int64_t)0x7fffffff);
  }
}

}  // namespace

hipError_t launch_kv_tables(const KvTablesParams& p, hipStream_t stream) {
  if (p.requests < 1 || p.requests > kMaxTableRequests) return hipErrorInvalidValue;
  const int64_t per_wg = 1024;
  const int64_t wgs = max((int64_t)1, (p.tokens + per_wg - 1) / per_wg);
  if (wgs > 0x7fffffff) return hipErrorInvalidValue;
  const size_t lds = (size_t)(2 * p.requests + 1) * sizeof(int32_t);
  hipLaunchKernelGGL(kv_tables, dim3((unsigned)wgs), dim3(kThreads), lds, stream, p, (int)per_wg);
  return hipGetLastError();
}

}  // namespace pasa
