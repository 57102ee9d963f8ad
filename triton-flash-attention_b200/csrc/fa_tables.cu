// fa_tables.cu -- what one serving step over a paged K/V cache needs, built
// on the GPU from the requests' lengths: new pages in the block table, the
// query offsets, key counts, positions and cache slots of the new tokens.
//
// Request r has cached[r] tokens and brings fresh[r].  With P = page size it
// owns ceil(cached / P) pages and wants ceil((cached + fresh) / P).  Prefix
// sums over the requests place its tokens in the packed batch and its new
// pages in the free list.  A request fits when its pages fit its table row,
// its tokens the batch, and its new pages what the free list still holds.
//
// Integers only, some 8 bytes a token and 8 a page, so a call is its latency.
// Every block does the prefix sums over all requests for itself, 512 at a
// time, instead of waiting for another launch to do them, and then writes
// its share of the tokens and pages; a binary search in shared memory finds
// the request of each.  Adjacent threads write adjacent entries.  16 requests
// of one token: 4.3 us; 256 of up to 2,048 tokens (269,000 in all): 7.4 us.
#include "fa_kernels.h"

namespace fa {
namespace {

constexpr int THREADS = 512;  // and requests a chunk
constexpr int WARPS = THREADS / 32;

// Inclusive sum over the block; total gets the block's.
__device__ __forceinline__ long long block_scan(long long v, long long* warp_sums, long long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const long long o = __shfl_up_sync(0xffffffffu, v, m);
    if (lane >= m) v += o;
  }
  __syncthreads();  // the previous scan's sums are read
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  long long before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    const long long s = warp_sums[w];
    if (w < warp) before += s;
    all += s;
  }
  *total = all;
  return v + before;
}

// First index in [0, n) whose end is above x (the ends never fall).
__device__ __forceinline__ int upper(const int* ends, int n, int x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (ends[mid] > x) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

__global__ void __launch_bounds__(THREADS) fa_extend_table_kernel(const __grid_constant__ TableArgs a) {
  __shared__ long long warp_sums[WARPS];
  __shared__ int tok_start[THREADS], tok_end[THREADS];  // rows of the packed batch
  __shared__ int page_end[THREADS];                     // new pages up to and with the request
  __shared__ int have[THREADS], first[THREADS], cached[THREADS];
  __shared__ unsigned char fit[THREADS];
  const int tid = threadIdx.x;
  let_next_begin();
  begin_after_previous();
  const long long page = 1LL << a.page_log2;
  long long start = *a.free_start;
  if (start < 0) start = 0;
  const long long left = (long long)a.n_free - start;  // may be negative: nothing fits
  long long tok_base = 0, page_base = 0, used = 0;
  for (int r0 = 0; r0 < a.requests; r0 += THREADS) {
    const int r = r0 + tid;
    const int m = min(THREADS, a.requests - r0);
    long long c = 0, f = 0;
    if (r < a.requests) {
      c = max(0, a.cached[r]);
      f = max(0, a.fresh[r]);
    }
    long long toks, pages;
    const long long t_end = tok_base + block_scan(f, warp_sums, &toks);
    const long long t_start = t_end - f;
    const long long had = (c + page - 1) >> a.page_log2, want = (c + f + page - 1) >> a.page_log2;
    const bool placed = want <= a.width && t_end <= a.total;
    const long long need = (r < a.requests && placed) ? want - had : 0;
    const long long p_end = page_base + block_scan(need, warp_sums, &pages);
    const bool fits = placed && p_end <= left;
    tok_start[tid] = int(min(t_start, (long long)a.total));
    tok_end[tid] = int(min(t_end, (long long)a.total));
    page_end[tid] = int(min(p_end, max(left, 0LL)));
    first[tid] = int(min(p_end - need, max(left, 0LL)));
    have[tid] = int(min(had, (long long)a.width));
    cached[tid] = int(c);
    fit[tid] = fits;
    __syncthreads();
    if (blockIdx.x == 0 && r < a.requests) {
      if (r == 0) a.cu[0] = 0;
      a.cu[r + 1] = int(min(t_end, (long long)a.total));
      a.seqlens[r] = int(fits ? c + f : c);
      a.fits[r] = fits;
      if (fits) used = p_end;
    }
    // tokens of this chunk
    const int t_last = int(min(tok_base + toks, (long long)a.total));
    for (long long t = min(tok_base, (long long)a.total) + blockIdx.x * THREADS + tid; t < t_last;
         t += (long long)gridDim.x * THREADS) {
      const int i = upper(tok_end, m, int(t));
      const long long pos = (long long)cached[i] + (t - tok_start[i]);
      long long slot = -1;
      if (fit[i]) {
        const int lp = int(pos >> a.page_log2);
        const int id = lp < have[i] ? a.table[(long long)(r0 + i) * a.width + lp]
                                    : a.free_pages[start + first[i] + (lp - have[i])];
        slot = (long long)id * page + (pos & (page - 1));
        if (id < 0 || slot > 0x7fffffffLL) slot = -1;
      }
      a.pos[t] = int(min(pos, 0x7fffffffLL));
      a.slots[t] = int(slot);
    }
    // new pages of this chunk
    const long long p_last = min(page_base + pages, max(left, 0LL));
    for (long long p = page_base + blockIdx.x * THREADS + tid; p < p_last; p += (long long)gridDim.x * THREADS) {
      const int i = upper(page_end, m, int(p));
      if (i < m && fit[i])
        a.table[(long long)(r0 + i) * a.width + have[i] + (p - first[i])] = a.free_pages[start + p];
    }
    tok_base += toks;
    page_base += pages;
    __syncthreads();  // the chunk's entries are used up
  }
  // rows behind the last request
  for (long long t = min(tok_base, (long long)a.total) + blockIdx.x * THREADS + tid; t < a.total;
       t += (long long)gridDim.x * THREADS) {
    a.pos[t] = 0;
    a.slots[t] = -1;
  }
  if (blockIdx.x == 0) {  // `used` is the largest prefix among a thread's requests that fit
    __shared__ long long top[WARPS];
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) used = max(used, __shfl_xor_sync(0xffffffffu, used, m));
    if ((tid & 31) == 0) top[tid >> 5] = used;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < WARPS; ++w) used = max(used, top[w]);
      *a.free_next = int(start + used);
    }
  }
}

}  // namespace

int launch_extend_table(const TableArgs& a) {
  // two tokens a thread, up to one block a SM (a new page holds a new token, so pages are fewer)
  long long ctas = ((long long)a.total + 2 * THREADS - 1) / (2 * THREADS);
  if (ctas < 1) ctas = 1;
  const int sms = device_sm_count();
  if (ctas > sms) ctas = sms;
  return launch_early(fa_extend_table_kernel, dim3(unsigned(ctas)), THREADS, 0, 1, a.stream, a);
}

}  // namespace fa
