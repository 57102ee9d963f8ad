// fa_sparse.cu -- attention of new tokens over a few pages of a paged K/V
// cache, chosen for each token and K/V head by a cheap score.
//
//  * fa_page_means_kernel: the mean key of every page that a step's tokens
//    completed;
//  * fa_select_pages_kernel: score(p) = max over the group's query heads of
//    q . mean key of page p, and the top pages by it;
//  * fa_sparse_decode_kernel: softmax attention over the keys of the listed
//    pages that the token may see.
//
// Means and scores decide which pages are kept, and two pages' scores may be
// as near as their roundings, so both are defined by 64-bit sums, rounded once
// to what they are kept in (means: to fp32 and then the cache's type; scores:
// to fp32).  The kept pages then depend on the inputs alone, not on the order
// of a sum.  (Scores are summed in fp32 first, and in 64 bits where that could
// change which pages are kept.)
#include <atomic>

#include "fa_kernels.h"

namespace fa {
namespace {

// Sequence of packed row t: the last b with cu[b] <= t, by 32 probes a step.
// Every lane of the warp calls and gets it.
__device__ __forceinline__ int warp_find_seq(const int* cu, int B, int t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, len = B;
  while (len > 1) {
    const int step = (len + 31) / 32;
    const int i = lane * step;
    const bool ok = i < len && cu[lo + i] <= t;
    const int c = __popc(__ballot_sync(0xffffffffu, ok));
    const int at = c > 0 ? (c - 1) * step : 0;
    lo += at;
    len = min(step, len - at);
  }
  return lo;
}

template <int DT>
__device__ __forceinline__ float to_f32(uint16_t v) {
  return unpack2<DT>(uint32_t(v)).x;
}

template <int DT>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (DT == 0) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

// ---------------------------------------------------------------------------
// Means of completed pages.
//
// Sequence b brings rows cu[b] .. cu[b+1] - 1, its last keys, and so completes
// pages (nk - nq) / P .. nk / P - 1: at most floor(nq / P) + 1 of them.  Unit
// u of the launch is page u - off(b) of them with off(b) = cu[b] / P + b, which
// leaves room enough for every b and needs no sum over the sequences.
//
// A block takes one page: P rows of W = Hkv D neighbouring columns.  A thread
// sums 8 columns of every n-th row; the partial sums meet in shared memory.
// 16 pages of 64 x 8 x 128 that a decode step completed: 5 us, latency.  3,840 of
// them from prompts: 102 us, of which their bytes take 77; every value is
// converted to 64 bits, at 16 a clock and SM.
constexpr int MEAN_THREADS = 512;

template <int DT>
__global__ void __launch_bounds__(MEAN_THREADS) fa_page_means_kernel(const __grid_constant__ PageArgs a, int units) {
  extern __shared__ double part[];  // [row groups][8 * columns of a pass]
  const int W8 = a.Hkv * a.D / 8;   // 16-byte column chunks of a row
  const int cols = min(W8, MEAN_THREADS);
  const int groups = min(MEAN_THREADS / cols, 8);
  const int P = 1 << a.page_log2;
  let_next_begin();
  begin_after_previous();
  units = min(units, (a.cu[a.B] >> a.page_log2) + a.B);  // the step's own rows
  for (int u = blockIdx.x; u < units; u += gridDim.x) {
    // last b with off(b) <= u.  A decode step's first guess is b = u, loaded at
    // once; the search with its dependent loads is for other batches
    int b = min(u, a.B - 1);
    int q0 = a.cu[b], q1 = a.cu[b + 1], nk = a.seqlens[b];
    if ((q0 >> a.page_log2) + b > u || (b + 1 < a.B && (q1 >> a.page_log2) + b + 1 <= u)) {
      const int lane = threadIdx.x & 31;
      int lo = 0, len = a.B;
      while (len > 1) {
        const int step = (len + 31) / 32;
        const int i = lane * step;
        const bool ok = i < len && (a.cu[lo + i] >> a.page_log2) + lo + i <= u;
        const int c = __popc(__ballot_sync(0xffffffffu, ok));
        const int at = c > 0 ? (c - 1) * step : 0;
        lo += at;
        len = min(step, len - at);
      }
      b = lo;
      q0 = a.cu[b];
      q1 = a.cu[b + 1];
      nk = a.seqlens[b];
    }
    const int nq = q1 - q0;
    if (nq <= 0 || nk <= 0) continue;
    if (nk > (a.width << a.page_log2)) {  // its table row cannot hold it: refused whole, as place_row does
      if (threadIdx.x == 0) refuse_index(a.status, FA_SITE_PAGE);
      continue;
    }
    const int from = max(nk - nq, 0) >> a.page_log2;
    const long long p = (long long)from + (u - ((q0 >> a.page_log2) + b));
    if (p < from || p >= (nk >> a.page_log2)) continue;  // uniform in the block
    const int id = a.table[(long long)b * a.width + p];
    if (id < 0 || id >= a.num_pages) {
      if (threadIdx.x == 0) refuse_index(a.status, FA_SITE_PAGE);
      continue;
    }
    const uint16_t* src = static_cast<const uint16_t*>(a.k_cache) + (long long)id * P * a.Hkv * a.D;
    uint16_t* dst = static_cast<uint16_t*>(a.means) + (long long)id * a.Hkv * a.D;
    const int g = threadIdx.x / cols, c0 = threadIdx.x % cols;
    for (int base = 0; base < W8; base += cols) {
      const int c = base + c0;
      const bool mine = g < groups && c < W8;
      double s[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] = 0.0;
      if (mine) {
#pragma unroll 8
        for (int r = g; r < P; r += groups) {
          const uint4 v = *(reinterpret_cast<const uint4*>(src + (long long)r * a.Hkv * a.D) + c);
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = unpack2<DT>(w[j]);
            s[2 * j] += double(f.x);
            s[2 * j + 1] += double(f.y);
          }
        }
      }
      __syncthreads();  // the last pass's sums are read
      if (mine && g > 0)
#pragma unroll
        for (int j = 0; j < 8; ++j) part[((g - 1) * 8 + j) * cols + c0] = s[j];
      __syncthreads();
      if (mine && g == 0) {
        for (int o = 1; o < groups; ++o)
#pragma unroll
          for (int j = 0; j < 8; ++j) s[j] += part[((o - 1) * 8 + j) * cols + c0];
        float f[8];
        const double inv = 1.0 / double(P);  // a power of two: exact
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = __double2float_rn(s[j] * inv);
        reinterpret_cast<uint4*>(dst)[c] = make_uint4(pack2<DT>(f[0], f[1]), pack2<DT>(f[2], f[3]),
                                                      pack2<DT>(f[4], f[5]), pack2<DT>(f[6], f[7]));
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Cluster helpers: `S` blocks of one launch cluster share a unit's work.
constexpr int MAX_CLUSTER = 8;
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// All threads of all blocks of the cluster; shared-memory writes before it
// are seen after it.  It ends as soon as every block has come to it.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Address of this block's shared variable at saddr in block `rank`.
__device__ __forceinline__ uint32_t cluster_map(uint32_t saddr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
  return r;
}
__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// The packed row's sequence and its position there: keys 0 .. pos are seen.
// pos < 0: a row behind the last sequence, or one whose sequence has no key
// for it.  Every lane of the warp calls.
struct RowPlace {
  int b;
  int pos;
};
__device__ __forceinline__ RowPlace place_row(const int* cu, const int* seqlens, int B, int t, int key_cap,
                                              int* status) {
  RowPlace r;
  // a decode step brings one row a sequence: that guess is loaded at once,
  // and the search with its dependent loads is for other batches
  r.b = min(t, B - 1);
  int q0 = cu[r.b], q1 = cu[r.b + 1], nk = seqlens[r.b];
  if (t < q0 || t >= q1) {
    r.b = warp_find_seq(cu, B, t);
    q0 = cu[r.b];
    q1 = cu[r.b + 1];
    nk = seqlens[r.b];
  }
  const long long pos = (long long)nk - (q1 - t);  // the rows are the sequence's last
  const bool too_long = nk > key_cap;  // its table row cannot hold it
  if (too_long) refuse_index(status, FA_SITE_PAGE);
  r.pos = (t < q0 || t >= q1 || too_long) ? -1 : int(pos < 0 ? -1 : pos);
  return r;
}

// ---------------------------------------------------------------------------
// Page selection.  A cluster of S blocks takes one (token, K/V head): every
// block scores its share of the pages into the first block's shared memory,
// which then finds the top ones.
//
// Scoring: matrix instructions, 16 pages a warp as their rows, 8 of the group's
// heads as columns.  A lane's share of a row are 8 neighbouring columns at a
// time, straight from global memory to registers (a second set of registers for
// the pages to come gained nothing); the queries lie in shared memory.  The
// products are exact and PTX has their sums in at least single precision, so
// that a score is off by at most 5/4 D 2^-23 of the sum of sizes |q| . |k|,
// which the same instructions give.
//
// Selection: keys are the scores' bits in an order that whole numbers have,
// neighbouring keys a thread.  T, the kk-th largest, is found by counting the
// keys in bins of equal width and ranking those of its bin; where scores lie
// in heaps, two bits a round by counts of the keys at and above three
// candidates.  If more than one key lies so near T that its score's roundings
// may decide, the pages of all such keys are scored again in 64 bits.  The
// pages above T, and of those at T the first ones, are written in order of
// their index.
//
// Bound: latency.  64 (token, K/V head) units of 2,048 pages, 4 heads each,
// D 128: 15.5 us, of which 2 go before the first page, 4 for the scores (the
// means' bytes alone take 5 from HBM, here they lie in L2), 1 to meet, 2.5 for
// T, 1 for the pages near it and 1 to write; 128 units of 128 pages: 7.2 us.
// 124 rows x 4 heads of 129 pages (D 64, drafted tokens): 11.7 us.
// Where more than 256 pages lie within the bound of each other, the first block
// scores all of those again, a warp a page: 2,048 equal pages 250 us, 16,384
// 1.8 ms.  A large part common to all means does not reach it (19 us).
// fp32 multiply-adds took 8 us for the scores (they are short of shared memory
// bandwidth for the queries), 64-bit ones 15, and rounds of two bits alone 5
// for T.
constexpr int SEL_THREADS = 256;
constexpr int SEL_WARPS = SEL_THREADS / 32;
constexpr int SEL_STEP = SEL_WARPS * 16;  // pages of the block's step
template <int D>
constexpr int sel_pitch() {  // bytes of a query's row in shared memory: two neighbours on different banks
  return D == 32 ? 64 : 2 * D + 64;
}

__device__ __forceinline__ uint32_t order_key(float f) {
  if (f != f) return 0u;  // NaN: behind everything
  const uint32_t u = __float_as_uint(f + 0.f);  // zeros are equal
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_score(uint32_t k) {  // of a key that is not 0
  return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}

__device__ __forceinline__ float max_nan(float x, float y) {  // NaN if either is
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(x), "f"(y));
  return m;
}

// fp32 scores of the block's pn pages, as keys to keys_at.  ids holds their
// pages and may be where the keys go: a page's key replaces its id, which is
// read by then.  Returns the bits of the largest |q| . |k| that this thread has
// seen (NaN is the largest), 0 only where every k is 0.
template <int D, int DT>
__device__ __forceinline__ uint32_t score_pages(const SelectArgs& a, const unsigned char* qs, const int* ids, int h,
                                                int G, int pn, uint32_t keys_at) {
  constexpr int CH = D / 32;  // 16-byte chunks of a lane and row
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g8 = lane >> 2, t4 = lane & 3;
  const uint16_t* means = static_cast<const uint16_t*>(a.means) + (long long)h * D + 8 * t4;
  const long long page_stride = (long long)a.Hkv * D;
  // 16 pages of the warp: rows g8 and g8 + 8 are this lane's, its chunk c of
  // them columns 32 c + 8 t4 .. + 7
  struct Pages {
    uint4 v[2][CH];
    bool ok[2];
  };
  auto load = [&](Pages& x, int base) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = base + g8 + 8 * i;
      const int id = at < pn ? ids[at] : -1;
      x.ok[i] = id >= 0;
#pragma unroll
      for (int c = 0; c < CH; ++c)
        x.v[i][c] = id >= 0 ? *reinterpret_cast<const uint4*>(means + id * page_stride + c * 32)
                            : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  constexpr uint32_t ABS = 0x7fff7fffu;
  float most = 0.f;
  uint32_t any = 0u;  // of k, whose products may all be too small to see
  Pages here;
  load(here, warp * 16);
  for (int base = warp * 16; base < pn; base += SEL_STEP) {
    float best[2] = {-INFINITY, -INFINITY};
    for (int g0 = 0; g0 < G; g0 += 8) {
      float even[4] = {0.f, 0.f, 0.f, 0.f}, odd[4] = {0.f, 0.f, 0.f, 0.f}, size[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        // a sum does not care which column is which k: both operands take the
        // lane's 8 neighbouring ones as two products' shares
        const uint4 q = *reinterpret_cast<const uint4*>(qs + (g0 + g8) * sel_pitch<D>() + c * 64 + t4 * 16);
        const uint4 r0 = here.v[0][c], r1 = here.v[1][c];
        const uint32_t lo[4] = {r0.x, r1.x, r0.y, r1.y}, hi[4] = {r0.z, r1.z, r0.w, r1.w};
        mma16816<DT>(even, lo, q.x, q.y);
        mma16816<DT>(odd, hi, q.z, q.w);
        const uint32_t lo_abs[4] = {lo[0] & ABS, lo[1] & ABS, lo[2] & ABS, lo[3] & ABS};
        const uint32_t hi_abs[4] = {hi[0] & ABS, hi[1] & ABS, hi[2] & ABS, hi[3] & ABS};
        mma16816<DT>(size, lo_abs, q.x & ABS, q.y & ABS);
        mma16816<DT>(size, hi_abs, q.z & ABS, q.w & ABS);
        any |= lo_abs[0] | lo_abs[1] | lo_abs[2] | lo_abs[3] | hi_abs[0] | hi_abs[1] | hi_abs[2] | hi_abs[3];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)  // page g8 + 8 (j / 2), head g0 + 2 t4 + j % 2
        if (g0 + 2 * t4 + j % 2 < G) best[j / 2] = max_nan(best[j / 2], even[j] + odd[j]);
      most = max_nan(most, max_nan(max_nan(size[0], size[1]), max_nan(size[2], size[3])));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      best[i] = max_nan(best[i], __shfl_xor_sync(0xffffffffu, best[i], 1));
      best[i] = max_nan(best[i], __shfl_xor_sync(0xffffffffu, best[i], 2));
    }
    const int mine = base + g8 + 8 * t4;  // of lanes t4 = 0 and 1
    const bool ok = t4 ? here.ok[1] : here.ok[0];
    load(here, base + SEL_STEP);
    __syncwarp();  // the step's ids are read
    if (t4 < 2 && mine < pn)
      st_cluster_u32(keys_at + 4u * uint32_t(mine), ok ? order_key(t4 ? best[1] : best[0]) : 0u);
  }
  return max(__float_as_uint(most) & 0x7fffffffu, any != 0u ? 1u : 0u);
}

// The score of page `id` by its definition: 64-bit sums, rounded to fp32.  One
// warp; a lane's D / 32 neighbouring columns against the queries in shared
// memory, which hold the operands exactly.
template <int D, int DT>
__device__ __forceinline__ uint32_t exact_key(const SelectArgs& a, const unsigned char* qs, int h, int G, int id) {
  constexpr int N = D / 32;
  const int d0 = (threadIdx.x & 31) * N;
  const uint16_t* k = static_cast<const uint16_t*>(a.means) + ((long long)id * a.Hkv + h) * D + d0;
  double kd[N];
#pragma unroll
  for (int i = 0; i < N; ++i) kd[i] = double(to_f32<DT>(k[i]));
  float best = -INFINITY;
  bool nan = false;
#pragma unroll 4
  for (int g = 0; g < G; ++g) {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(qs + g * sel_pitch<D>()) + d0;
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < N; ++i) s = fma(double(to_f32<DT>(q[i])), kd[i], s);
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
    const float f = __double2float_rn(s);
    nan |= f != f;
    best = fmaxf(best, f);
  }
  return nan ? 0u : order_key(best);
}

// Shared memory of the selection.
struct SelectShared {
  uint2 counts[2][SEL_WARPS];
  uint32_t list[SEL_THREADS];
  int pages[SEL_THREADS];
  uint32_t found;
  int listed;
  int bin, above, active;
};

// The rank-th largest (from 1) of n <= SEL_THREADS values; v has zeros up to a
// multiple of 4.  All threads; ends with a barrier.
__device__ __forceinline__ uint32_t ranked(SelectShared& sh, const uint32_t* v, int n, int rank) {
  const int me = threadIdx.x;
  if ((me & ~31) < n) {
    const uint32_t mine = me < n ? v[me] : 0u;
    int above = 0, from = 0;  // values > mine, >= mine
#pragma unroll 4
    for (int i = 0; i < n; i += 4) {
      const uint4 k = *reinterpret_cast<const uint4*>(v + i);
      above += (k.x > mine) + (k.y > mine) + (k.z > mine) + (k.w > mine);
      from += (k.x >= mine) + (k.y >= mine) + (k.z >= mine) + (k.w >= mine);
    }
    if (me < n && above < rank && rank <= from) sh.found = mine;
  }
  __syncthreads();
  return sh.found;
}

// A thread's neighbouring keys: E of them in registers, or (E = 0) read again
// from shared memory.
template <int E>
struct Held {
  const uint32_t* keys;
  int k0, k1;
  uint32_t v[E > 0 ? E : 1];
  __device__ __forceinline__ Held(const uint32_t* all, int M) : keys(all) {
    const int each = E > 0 ? E : (M + SEL_THREADS - 1) / SEL_THREADS;
    k0 = min(M, int(threadIdx.x) * each);
    k1 = min(M, k0 + each);
    if constexpr (E > 0) {
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] = k0 + i < k1 ? keys[k0 + i] : 0u;
    }
  }
  template <class F>
  __device__ __forceinline__ void each(F f) const {  // f(index, key)
    if constexpr (E > 0) {
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (k0 + i < k1) f(k0 + i, v[i]);
    } else {
      for (int i = k0; i < k1; ++i) f(i, keys[i]);
    }
  }
};
// Block-wide sums of two counts below 2^16 each a thread; one barrier.
__device__ __forceinline__ uint2 block_counts(SelectShared& sh, int turn, uint32_t x, uint32_t y) {
  x = __reduce_add_sync(0xffffffffu, x);
  y = __reduce_add_sync(0xffffffffu, y);
  uint2* slot = sh.counts[turn & 1];
  if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = make_uint2(x, y);
  __syncthreads();
  x = y = 0;
#pragma unroll
  for (int w = 0; w < SEL_WARPS; ++w) x += slot[w].x, y += slot[w].y;
  return make_uint2(x, y);
}

// The rank-th largest of the n <= SEL_THREADS held keys that `in` picks.  All
// threads.
template <int E, class In>
__device__ __forceinline__ uint32_t ranked_of(SelectShared& sh, const Held<E>& held, int n, int rank, In in) {
  if (threadIdx.x == 0) sh.listed = 0;
  sh.list[threadIdx.x] = 0u;
  __syncthreads();
  held.each([&](int, uint32_t k) {
    if (in(k)) sh.list[atomicAdd(&sh.listed, 1)] = k;
  });
  __syncthreads();
  return ranked(sh, sh.list, n, rank);
}

// The kk-th largest of the M keys (below 2^16 of them).
template <int E>
__device__ __forceinline__ uint32_t kth_largest(SelectShared& sh, const Held<E>& held, int M, int kk) {
  // SEL_THREADS bins of equal width between the smallest and the largest
  // score: a larger score's bin is never below a smaller one's, whatever the
  // roundings, so a count of each finds T's, and its few keys are ranked
  uint32_t lo = 0xffffffffu, hi = 0u;
  held.each([&](int, uint32_t k) { lo = k != 0u ? min(lo, k) : lo, hi = max(hi, k); });
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (lane == 0) sh.counts[0][warp] = make_uint2(lo, hi);
  sh.list[threadIdx.x] = 0u;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < SEL_WARPS; ++w) lo = min(lo, sh.counts[0][w].x), hi = max(hi, sh.counts[0][w].y);
  if (lo < hi && fabsf(key_score(lo)) < INFINITY && fabsf(key_score(hi)) < INFINITY) {  // uniform
    const float low = key_score(lo), scale = (SEL_THREADS - 0.5f) / (key_score(hi) - low);
    auto bin_of = [&](uint32_t k) {
      return k == 0u ? 0 : min(SEL_THREADS - 1, int((key_score(k) - low) * scale));
    };
    held.each([&](int, uint32_t k) { atomicAdd(&sh.list[bin_of(k)], 1u); });
    __syncthreads();
    const int bin = SEL_THREADS - 1 - int(threadIdx.x);  // from the top
    const int n = int(sh.list[bin]);
    int sum = n;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, sum, m);
      if (lane >= m) sum += x;
    }
    if (lane == 31) sh.counts[1][warp].x = uint32_t(sum);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SEL_WARPS; ++w) sum += w < warp ? int(sh.counts[1][w].x) : 0;
    if (sum - n < kk && kk <= sum) sh.bin = bin, sh.above = sum - n, sh.active = n;
    __syncthreads();
    if (sh.active <= SEL_THREADS) {
      const int mine = sh.bin;
      return ranked_of(sh, held, sh.active, kk - sh.above, [&](uint32_t k) { return bin_of(k) == mine; });
    }
  }
  // scores that lie in heaps: two bits of T a round
  uint32_t T = 0;
  int above = 0, active = M;  // keys above T's range, keys in it
#pragma unroll 1
  for (int bit = 30; bit >= 0; bit -= 2) {
    if (bit <= 20 && active <= SEL_THREADS) {  // few keys agree with T so far
      const uint32_t low = bit + 1 >= 31 ? 0xffffffffu : (4u << bit) - 1u;
      return ranked_of(sh, held, active, kk - above, [&](uint32_t k) { return (k & ~low) == T; });
    }
    const uint32_t t1 = T | (1u << bit), t2 = T | (2u << bit), t3 = T | (3u << bit);
    uint32_t c12 = 0, c3 = 0;
    held.each([&](int, uint32_t k) { c12 += (k >= t1) + ((k >= t2) << 16), c3 += k >= t3; });
    const uint2 c = block_counts(sh, bit >> 1, c12, c3);
    const int c1 = int(c.x & 0xffffu), c2 = int(c.x >> 16), n3 = int(c.y);
    // the range that T is in, the keys above it and from it on
    if (n3 >= kk) T = t3, active = n3 - above;
    else if (c2 >= kk) T = t2, active = c2 - n3, above = n3;
    else if (c1 >= kk) T = t1, active = c1 - c2, above = c2;
    else active -= c1 - above, above = c1;
  }
  return T;
}

// Writes the kk largest of the M keys, to out in order of their index, plus
// off.  slack: how far an fp32 score may be from the one by definition; where
// that leaves a choice, rescore(page, key) gives the key by definition.
template <int E, class Rescore>
__device__ __forceinline__ void write_top(SelectShared& sh, uint32_t* keys, int M, int kk, int off, int* out,
                                          float slack, Rescore rescore) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Held<E> held(keys, M);
  uint32_t T = E == 1 ? ranked(sh, keys, M, kk) : kth_largest(sh, held, M, kk);
  // keys whose scores by definition may lie on either side of the kk-th
  uint32_t lo = 0u, hi = 0xffffffffu;
  bool all_open = !(slack < INFINITY);  // infinities or NaN: any key
  if (!all_open && slack > 0.f && T != 0u) {
    lo = order_key(__fsub_rd(key_score(T), 2.f * slack));
    hi = order_key(__fadd_ru(key_score(T), 2.f * slack));
    uint32_t near = 0, over = 0;
    held.each([&](int, uint32_t k) { near += k >= lo && k <= hi, over += k > hi; });
    const uint2 c = block_counts(sh, 1, near, over);
    const int n = int(c.x), want = kk - int(c.y);  // pages near T, and how many of them are kept
    all_open = n > SEL_THREADS;
    if (n > 1 && !all_open) {
      if (threadIdx.x == 0) sh.listed = 0;
      __syncthreads();
      held.each([&](int i, uint32_t k) {
        if (k >= lo && k <= hi) sh.pages[atomicAdd(&sh.listed, 1)] = i;
      });
      __syncthreads();
      for (int i = warp; i < n; i += SEL_WARPS) {
        const uint32_t key = rescore(sh.pages[i]);
        if (lane == 0) sh.list[i] = key;
      }
      __syncthreads();
      if (int(threadIdx.x) < n) {
        const uint32_t mine = sh.list[threadIdx.x];
        const int page = sh.pages[threadIdx.x];
        int before = 0;
        for (int i = 0; i < n; ++i) before += sh.list[i] > mine || (sh.list[i] == mine && sh.pages[i] < page);
        keys[page] = before < want ? 0xffffffffu : 0u;  // kept: above every other, or not: below
      }
      __syncthreads();
      held = Held<E>(keys, M);
      T = hi;
    }
  }
  if (all_open) {  // uniform
    __syncthreads();
    for (int p0 = warp * 32; p0 < M; p0 += SEL_THREADS) {
      const uint32_t k = p0 + lane < M ? keys[p0 + lane] : 0u;
      uint32_t todo = __ballot_sync(0xffffffffu, p0 + lane < M && k >= lo && k <= hi);
      while (todo) {
        const int j = __ffs(todo) - 1;
        todo &= todo - 1;
        const uint32_t key = rescore(p0 + j);
        if (lane == 0) keys[p0 + j] = key;
      }
    }
    __syncthreads();
    held = Held<E>(keys, M);
    T = E == 1 ? ranked(sh, keys, M, kk) : kth_largest(sh, held, M, kk);
  }
  int gt = 0, eq = 0;
  held.each([&](int, uint32_t k) { gt += k > T, eq += k == T; });
  const uint32_t both = uint32_t(gt) | (uint32_t(eq) << 16);
  uint32_t sum = both;
#pragma unroll
  for (int m = 1; m < 32; m <<= 1) {
    const uint32_t x = __shfl_up_sync(0xffffffffu, sum, m);
    if (lane >= m) sum += x;
  }
  __syncthreads();
  if (lane == 31) sh.counts[0][warp].x = sum;
  __syncthreads();
  uint32_t before = sum - both, all = 0;
#pragma unroll
  for (int w = 0; w < SEL_WARPS; ++w) {
    const uint32_t x = sh.counts[0][w].x;
    before += w < warp ? x : 0u;
    all += x;
  }
  int gs = int(before & 0xffffu), es = int(before >> 16);
  const int want_eq = kk - int(all & 0xffffu);
  held.each([&](int i, uint32_t key) {
    if (key > T || (key == T && es < want_eq)) out[gs + min(es, want_eq)] = off + i;
    gs += key > T;
    es += key == T;
  });
}

template <int D, int DT>
__global__ void __launch_bounds__(SEL_THREADS, 2) fa_select_pages_kernel(const __grid_constant__ SelectArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ SelectShared sh;
  __shared__ uint32_t size, sizes[MAX_CLUSTER];  // largest |q| . |k| of the block; of all blocks
  constexpr int PITCH = sel_pitch<D>();
  const int S = a.cluster;
  const int rank = S > 1 ? int(cluster_rank()) : 0;
  const int unit = blockIdx.x / S;
  const int t = unit / a.Hkv, h = unit - t * a.Hkv;
  const int G = a.Hq / a.Hkv;
  const int lane = threadIdx.x & 31;
  // the group's queries, zeros up to a whole 8 of them; then page ids and keys
  const int G8 = (G + 7) / 8 * 8;
  unsigned char* qs = smem;
  uint32_t* keys = reinterpret_cast<uint32_t*>(smem + size_t(G8) * PITCH);
  int* ids = reinterpret_cast<int*>(keys);  // until their scores are known
  if (threadIdx.x == 0) size = 0u;
  let_next_begin();
  begin_after_previous();

  const uint16_t* q = static_cast<const uint16_t*>(a.q) + t * a.q_st + (long long)h * G * a.q_sh;
  for (int i = threadIdx.x; i < G8 * (D / 8); i += SEL_THREADS) {
    const int g = i / (D / 8), d = i % (D / 8) * 8;
    *reinterpret_cast<uint4*>(qs + g * PITCH + d * 2) =
        g < G ? *reinterpret_cast<const uint4*>(q + g * a.q_sh + d) : make_uint4(0u, 0u, 0u, 0u);
  }
  const RowPlace row = place_row(a.cu, a.seqlens, a.B, t, a.width << a.page_log2, a.status);
  int* out = a.out + (long long)unit * a.top;
  const int n = row.pos < 0 ? 0 : (row.pos >> a.page_log2) + 1;  // pages up to the token's own
  if (n <= a.top) {  // all of them (uniform over the cluster)
    if (rank == 0)
      for (int i = threadIdx.x; i < a.top; i += SEL_THREADS) out[i] = i < n ? i : -1;
    return;
  }
  const int M = n - a.sink - a.local;  // pages to choose from, the first at index sink
  const int kk = a.top - a.sink - a.local;
  if (rank == 0)
    for (int i = threadIdx.x; i < a.sink + a.local; i += SEL_THREADS) {
      if (i < a.sink) out[i] = i;
      else out[a.top - a.local + (i - a.sink)] = n - a.local + (i - a.sink);
    }
  if (kk == 0) return;

  // this block's pages: a contiguous share
  const int share = (M + S - 1) / S;
  const int p0 = rank * share, pn = max(0, min(share, M - p0));
  const int* pages = a.table + (long long)row.b * a.width + a.sink;
  for (int i = threadIdx.x; i < pn; i += SEL_THREADS) {
    const int id = pages[p0 + i];
    const bool ok = id >= 0 && id < a.num_pages;
    if (!ok) refuse_index(a.status, FA_SITE_PAGE);
    ids[i] = ok ? id : -1;
  }
  if (S > 1) cluster_sync();  // and the first block has begun, so that its shared memory may be written
  else __syncthreads();
  const uint32_t keys0 = smem_u32(keys) + 4u * uint32_t(p0);
  const uint32_t top = score_pages<D, DT>(a, qs, ids, h, G, pn, S > 1 ? cluster_map(keys0, 0) : keys0);
  const uint32_t top_bits = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) atomicMax(&size, top_bits);  // sizes' bits have their order
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t to = smem_u32(sizes + rank);
    st_cluster_u32(S > 1 ? cluster_map(to, 0) : to, size);
  }
  if (threadIdx.x < 4 && rank == 0 && M + int(threadIdx.x) < (M + 3) / 4 * 4) keys[M + threadIdx.x] = 0u;
  if (S > 1) {
    cluster_sync();
    if (rank != 0) return;
  } else {
    __syncthreads();
  }
  uint32_t bits = 0u;
  for (int i = 0; i < S; ++i) bits = max(bits, sizes[i]);
  // D products and D / 16 accumulators are added with at least single
  // precision, in whatever order and rounding: 2^-23 of the sum of sizes each,
  // or 2^-126 below the normal numbers; two roundings more join the halves and
  // are the definition's, and the sum of sizes is as inexact.  5 D / 4 + 1
  // covers them.  Near the end of the range no bound
  const float most = __uint_as_float(bits);
  const float slack = bits == 0u     ? 0.f  // as every k and score is
                      : most < 1e38f ? most * ((5 * D / 4 + 1) / 8388608.f) + 2e-36f
                                     : INFINITY;
  auto rescore = [&](int p) {
    const int id = pages[p];
    return id >= 0 && id < a.num_pages ? exact_key<D, DT>(a, qs, h, G, id) : 0u;
  };
  out += a.sink;
  if (M <= SEL_THREADS) write_top<1>(sh, keys, M, kk, a.sink, out, slack, rescore);
  else if (M <= 4 * SEL_THREADS) write_top<4>(sh, keys, M, kk, a.sink, out, slack, rescore);
  else if (M <= 8 * SEL_THREADS) write_top<8>(sh, keys, M, kk, a.sink, out, slack, rescore);
  else if (M <= 16 * SEL_THREADS) write_top<16>(sh, keys, M, kk, a.sink, out, slack, rescore);
  else write_top<0>(sh, keys, M, kk, a.sink, out, slack, rescore);
}

// ---------------------------------------------------------------------------
// Attention over the listed pages.
//
// A cluster of S blocks takes one (token, K/V head, up to 8 of its query
// heads).  The list is cut into 64-key tiles; block r takes tiles r, r + S,
// ...  Two producer warps copy a tile's K and V rows by TMA, one copy a piece
// of a page, into a ring of tiles.  Four warps take 16 keys of every tile
// each, with softmax state of their own, so nothing is exchanged until the
// end: then the warps' states are joined in shared memory and the blocks' over
// the cluster's.
//
// Both products are m16n8k16 matrix instructions.  S = Q K^T has the heads as
// rows (8 of 16) and the keys as columns; what a thread then holds of the
// weights is just what it has to hold of P^T, as two numbers of the operand type
// a weight, as the second operand of O^T = V^T P^T, whose rows are 16 of the D columns and whose columns are the
// 8 heads.  That takes half of the instructions and accumulators of O = P V
// with 16 rows of heads.
//
// Bound: HBM, 4 D bytes a key.  For a key the products take some 3 clocks of
// the 22 that its bytes take an SM's share of HBM; tcgen05's 128 rows would
// be 15 of 16 parts empty for a group's heads.  16 sequences x 8 K/V heads x
// 2,048 keys at D 128: 27 us (134 MB: 20.5 us of HBM), of which 4 go before the
// first keys arrive and 2.5 behind the last; without the products it takes 24.
// 2 sequences x 8 x 8,192 keys in pages of 16: 19.6 us (10.3 of HBM).
// Groups above 8 heads read their keys once for each 8: 16 x 8 x 2,048 keys with
// groups of 8, 9, 16 and 32 heads take 26.5, 30, 30 and 57 us.
constexpr int DEC_WARPS = 4;
constexpr int DEC_THREADS = (DEC_WARPS + 2) * 32;
constexpr int DEC_TILE = 64;
constexpr int NO_KEY = 0x7fffffff;

template <int D>
constexpr int dec_stages() {
  return D == 32 ? 6 : 3;
}
template <int D>
constexpr int dec_tile_bytes() {
  return DEC_TILE * D * 2;
}
template <int D>
struct DecSmem {
  static constexpr int ST = dec_stages<D>();
  static constexpr int RING = ST * 2 * dec_tile_bytes<D>();
  static constexpr int BASE = RING;                      // first logical key of each 16 of a tile
  static constexpr int BARS = BASE + ST * 4 * 4;         // K full, V full, empty
  static constexpr int BYTES = BARS + ST * 3 * 8 + 64 + 1024;  // control block; room to align the ring
  // after the last tile: joined state of the block, then the warps' states
  static constexpr int O_PITCH = D + 4;                               // floats of a head's row
  static constexpr int O_BLOCK = 0;                                   // [8][O_PITCH] fp32
  static constexpr int ML_BLOCK = O_BLOCK + 8 * O_PITCH * 4;          // [2][8]
  static constexpr int O_WARP = ML_BLOCK + 64;                        // [4][8][O_PITCH]
  static constexpr int ML_WARP = O_WARP + DEC_WARPS * 8 * O_PITCH * 4;  // [4][2][8]
  static_assert(ML_WARP + DEC_WARPS * 64 <= RING, "the states reuse the ring");
};

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// Byte offset of 16-byte chunk c (8 columns) of row r of 16 rows that start at
// a multiple of 8 rows of a piece, as the TMA's swizzle leaves it.  box: bytes
// between the first 64 columns and the last 64 of a piece.
template <int D>
__device__ __forceinline__ uint32_t tile_off(int r, int c, uint32_t box) {
  if constexpr (D == 32) return uint32_t(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
  else return (D == 128 && (c & 8) ? box : 0u) + uint32_t(r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// Two weights, none negative, as numbers of the operand type whose sum they
// are: hi, the largest below the weight, and lo, the rest.  A weight is then
// off by lo's rounding, half a step of a number below 2^-7 (bf16) or 2^-10
// (fp16) of it: 2^-15 or 2^-21.  Rounded once it would be 2^-8 or 2^-11, which
// showed in the result (error of 16 x 2,048 keys in fp16 2.5e-4 of the result,
// 2.1e-4 with fp32 weights and with these).  No part is negative, and of a
// weight that the type can hold none is zero, so that a value of infinity
// gives infinity.
template <int DT>
__device__ __forceinline__ void split_weights(float w0, float w1, uint32_t& hi, uint32_t& lo) {
  // the fp32 numbers before them, cut off
  const uint32_t b0 = max(__float_as_uint(w0), 1u) - 1u, b1 = max(__float_as_uint(w1), 1u) - 1u;
  float2 h;
  if constexpr (DT == DT_F16) {
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(__uint_as_float(b1)), "f"(__uint_as_float(b0)));
    h = unpack2<DT>(hi);
  } else {
    hi = __byte_perm(b0, b1, 0x7632);
    h = make_float2(__uint_as_float(b0 & 0xffff0000u), __uint_as_float(b1 & 0xffff0000u));
  }
  lo = pack2<DT>(w0 - h.x, w1 - h.y);
}
// The weights' factor, which the result loses with their sum: fp16 has no
// exponents for weights below 2^-24 of the largest.
template <int DT>
constexpr float weight_lift() {
  return DT == DT_F16 ? 16384.f : 1.f;
}

// Blocks a SM, with what dec_stages takes of shared memory.  D 64, 4 drafted
// tokens of 31 sequences (496 units): 4 blocks x 3 stages hold all units at
// once, 27 us; 3 x 3 35, 2 x 6 33, in two waves.  D 128, 2 blocks: 3 stages
// 27 us, 2 stages and 3 blocks 29 (16 sequences, 128 units in clusters of 2;
// in clusters of 1, 4 and 8: 28, 33 and 45).
template <int D>
constexpr int dec_per_sm() {
  return D == 128 ? 2 : 4;
}
template <int D, int DT>
__global__ void __launch_bounds__(DEC_THREADS, dec_per_sm<D>())
    fa_sparse_decode_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                            const __grid_constant__ SparseArgs a) {
  using M = DecSmem<D>;
  constexpr int ST = M::ST;
  constexpr int KS = D / 16;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  int* key_base = reinterpret_cast<int*>(smem + M::BASE);
  uint64_t* full_k = reinterpret_cast<uint64_t*>(smem + M::BARS);
  uint64_t* full_v = full_k + ST;
  uint64_t* empty = full_v + ST;
  CtaCtl* ctl = reinterpret_cast<CtaCtl*>(empty + ST);
  const int S = a.cluster;
  const int rank = S > 1 ? int(cluster_rank()) : 0;
  const int G = a.Hq / a.Hkv;
  const int hblocks = (G + 7) / 8;
  const int unit = blockIdx.x / S;  // (token, K/V head, block of 8 heads)
  const int hb = unit % hblocks;
  const int th = unit / hblocks;
  const int t = th / a.Hkv, h = th - t * a.Hkv;
  const int rows = min(8, G - hb * 8);
  // Up to 4 heads leave columns 4 to 7 of the second product free: those take
  // the weights' second parts (their heads' queries are there twice), one
  // product instead of two.  At 4 heads and D 128, 16 x 2,048 keys 27.0
  // us against 27.1, 2 x 8,192 keys 19.6 against 20.1.
  const bool few = rows <= 4;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int PR = min(1 << a.page_log2, DEC_TILE);  // rows of a piece

  if (threadIdx.x == 0) {
    ctl->abort = 0;
    ctl->status = a.status;
    for (int i = 0; i < ST; ++i) {
      mbar_init(full_k + i, 1);
      mbar_init(full_v + i, 1);
      mbar_init(empty + i, DEC_WARPS);
    }
    fence_mbar_init();
  }
  let_next_begin();
  begin_after_previous();
  // the producers' first list entries do not wait for the row's place
  const int PT = DEC_TILE / PR;                  // pieces of a tile
  const int sub_log2 = max(0, a.page_log2 - 6);  // pieces of a page
  const int pieces = a.top << sub_log2;
  const int* list = a.idx + ((long long)t * a.Hkv + h) * a.top;
  // lane j: piece j % PT of tile t0 + j / PT of the block's
  auto list_entry = [&](int t0) {
    const int piece = ((t0 + lane / PT) * S + rank) * PT + lane % PT;
    return piece < pieces ? list[piece >> sub_log2] : -1;
  };
  int entry = warp >= DEC_WARPS ? list_entry(0) : -1;
  const RowPlace row = place_row(a.cu, a.seqlens, a.B, t, a.width << a.page_log2, a.status);
  const int pos = row.pos;
  __syncthreads();

  const int g8 = lane >> 2, t4 = lane & 3;
  // O^T: columns 16 i + g8 (values 0, 1) and + 8 (2, 3) of heads 2 t4, 2 t4 + 1;
  // maximum and this thread's sum of head g8
  float o[D / 16][4];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

  if (warp >= DEC_WARPS) {
    // ---- producers: K rows, V rows ----
    const bool is_k = warp == DEC_WARPS;
    uint64_t* full = is_k ? full_k : full_v;
    const CUtensorMap* map = is_k ? &tmap_k : &tmap_v;
    const int tiles = pos < 0 ? 0 : (pieces + PT - 1) / PT;
    const int mine = tiles > rank ? (tiles - rank + S - 1) / S : 0;  // tiles rank, rank + S, ...
    const int per_batch = 32 / PT;  // tiles whose pieces the warp's lanes look up at once
    int it = 0;
    bool ok = true;
    for (int t0 = 0; t0 < mine && ok; t0 += per_batch) {
      // lane j: piece j % PT of tile t0 + j / PT
      const int sub = (((t0 + lane / PT) * S + rank) * PT + lane % PT) & ((1 << sub_log2) - 1);
      int base = NO_KEY, at = 0;  // first logical key; row in the cache
      if (entry >= 0 && entry < a.width) {
        const int first = (entry << a.page_log2) + sub * DEC_TILE;
        if (first <= pos) {
          const int id = a.table[(long long)row.b * a.width + entry];
          if (id >= 0 && id < a.num_pages) {
            base = first;
            at = (id << a.page_log2) + sub * DEC_TILE;
          } else {
            refuse_index(a.status, FA_SITE_PAGE);
          }
        }
      }
      if (t0 + per_batch < mine) entry = list_entry(t0 + per_batch);  // the next look-up's
      const uint32_t there = __ballot_sync(0xffffffffu, base != NO_KEY);
      for (int i = 0; i < per_batch && t0 + i < mine; ++i) {
        const uint32_t have = (there >> (i * PT)) & ((1u << PT) - 1u);
        if (have == 0) continue;
        const int s = it % ST;
        if (it >= ST && !mbar_wait_warp(empty + s, uint32_t(it / ST - 1) & 1, ctl, 96)) {
          ok = false;
          break;
        }
        if (is_k) {
          const int b16 = __shfl_sync(0xffffffffu, base, i * PT + min(lane * 16 / PR, PT - 1));
          if (lane < 4) key_base[s * 4 + lane] = b16 == NO_KEY ? NO_KEY : b16 + (lane * 16) % PR;
          __syncwarp();
        }
        unsigned char* tile = smem + (s * 2 + (is_k ? 0 : 1)) * dec_tile_bytes<D>();
        if (lane == 0) mbar_arrive_expect_tx(full + s, uint32_t(__popc(have)) * uint32_t(PR * D * 2));
        for (int p = 0; p < PT; ++p) {
          const int row_at = __shfl_sync(0xffffffffu, at, i * PT + p);
          if (lane == 0 && ((have >> p) & 1u)) tma_load_4d(tile + p * PR * D * 2, map, full + s, 0, row_at, 0, h);
        }
        ++it;
      }
    }
    // one more turn of the ring that says there is nothing more
    if (ok) {
      const int s = it % ST;
      if (it < ST || mbar_wait_warp(empty + s, uint32_t(it / ST - 1) & 1, ctl, 97)) {
        if (is_k) {
          if (lane < 4) key_base[s * 4 + lane] = -1;
          __syncwarp();
          if (lane == 0) mbar_arrive(full + s);
        }
      } else {
        ok = false;
      }
    }
    if (!ok || *(volatile int*)&ctl->abort) {
      for (int i = it > ST ? it - ST : 0; i < it; ++i)  // its copies land before the block goes
        mbar_wait_drain(full + i % ST, uint32_t(i / ST) & 1, ctl, 98);
      __syncwarp();
    }
  } else {
    // ---- consumers: keys 16 warp .. of each tile ----
    uint32_t qf[KS][2];  // head g8's columns 16 ks + 2 t4 and + 8
    {
      const int head = few ? g8 & 3 : g8;
      const uint16_t* q = static_cast<const uint16_t*>(a.q) + t * a.q_st + ((long long)h * G + hb * 8 + head) * a.q_sh;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          qf[ks][j] =
              head < rows && pos >= 0 ? *(reinterpret_cast<const uint32_t*>(q + ks * 16 + j * 8 + t4 * 2)) : 0u;
    }
    // the warp's 16 rows: their piece, and their place in it
    const uint32_t box = uint32_t(PR) * 128u;
    const uint32_t rows_at = uint32_t(warp * 16 / PR * PR * D * 2 + warp * 16 % PR * (D == 32 ? 64 : 128));
    const int mi = lane >> 3, mr = lane & 7;
    for (int it = 0;; ++it) {
      const int s = it % ST;
      const uint32_t parity = uint32_t(it / ST) & 1;
      if (!mbar_wait_warp(full_k + s, parity, ctl, 99)) break;
      const int base = key_base[s * 4 + warp];
      if (base == -1) break;
      const int seen = base == NO_KEY ? 0 : max(0, min(16, pos - base + 1));
      unsigned char* vt = smem + (s * 2 + 1) * dec_tile_bytes<D>() + rows_at;
      const uint32_t va = smem_u32(vt), ka = va - dec_tile_bytes<D>();
      float sc[2][2][4];  // [k-steps even, odd][keys 0-7, 8-15][head g8's keys 2 t4, + 1; two of no head]
      if (seen > 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) sc[i >> 1][i & 1][j] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          uint32_t b[4];
          ldmatrix4(ka + tile_off<D>((mi >> 1) * 8 + mr, ks * 2 + (mi & 1), box), b);
          const uint32_t af[4] = {qf[ks][0], 0u, qf[ks][1], 0u};
          mma16816<DT>(sc[ks & 1][0], af, b[0], b[1]);
          mma16816<DT>(sc[ks & 1][1], af, b[2], b[3]);
        }
      }
      if (!mbar_wait_warp(full_v + s, parity, ctl, 100)) break;
      if (seen > 0) {
        if (seen < 16) {
          // values behind the token's position may be anything and would meet
          // a zero weight: zeros in their place
          for (int i = lane; i < (16 - seen) * (D / 8); i += 32)
            *reinterpret_cast<uint4*>(vt + tile_off<D>(seen + i / (D / 8), i % (D / 8), box)) = make_uint4(0, 0, 0, 0);
          __syncwarp();
        }
        uint32_t vf[D / 16][4];  // V^T: 16 columns x 16 keys each
#pragma unroll
        for (int np = 0; np < D / 16; ++np)
          ldmatrix4_t(va + tile_off<D>((mi >> 1) * 8 + mr, np * 2 + (mi & 1), box), vf[np]);
        float w[4];  // scores, then weights of keys 2 t4, + 1, + 8, + 9
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          w[j] = (sc[0][j >> 1][j & 1] + sc[1][j >> 1][j & 1]) * a.scale_log2;
          if (seen < 16 && (j >> 1) * 8 + t4 * 2 + (j & 1) >= seen) w[j] = -INFINITY;
        }
        float x = fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3]));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
        x = fmaxf(m, x);
        const float ref = x == -INFINITY ? 0.f : x;  // no finite score so far: weights of zero
        if (__any_sync(0xffffffffu, x != m)) {
          const float al = ex2(m - ref);
          m = x;
          l *= al;
          const float a0 = __shfl_sync(0xffffffffu, al, t4 * 8), a1 = __shfl_sync(0xffffffffu, al, t4 * 8 + 4);
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            o[i][0] *= a0, o[i][1] *= a1;
            o[i][2] *= a0, o[i][3] *= a1;
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          w[j] = ex2(w[j] - ref) * weight_lift<DT>();
          l += w[j];
        }
        uint32_t p0, p1, r0, r1;  // the second product's operand, twice
        split_weights<DT>(w[0], w[1], p0, r0);
        split_weights<DT>(w[2], w[3], p1, r1);
        if (few && g8 >= 4) p0 = r0, p1 = r1;
#pragma unroll
        for (int np = 0; np < D / 16; ++np) mma16816<DT>(o[np], vf[np], p0, p1);
        if (!few)
#pragma unroll
          for (int np = 0; np < D / 16; ++np) mma16816<DT>(o[np], vf[np], r0, r1);
        if (seen < 16) fence_proxy_async_smem();  // zeros written before the next copy lands there
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + s);
    }
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
  }
  __syncthreads();  // the ring is free
  float* ml_warp = reinterpret_cast<float*>(smem + M::ML_WARP);
  float* o_warp = reinterpret_cast<float*>(smem + M::O_WARP);
  float* ml_block = reinterpret_cast<float*>(smem + M::ML_BLOCK);
  float* o_block = reinterpret_cast<float*>(smem + M::O_BLOCK);
  constexpr int OP = M::O_PITCH;
  if (warp < DEC_WARPS) {
    if (t4 == 0) {
      ml_warp[warp * 16 + g8] = m;
      ml_warp[warp * 16 + 8 + g8] = l;
    }
    float* dst = o_warp + (warp * 8 + t4 * 2) * OP + g8;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      dst[i * 16] = o[i][0], dst[i * 16 + OP] = o[i][1];
      dst[i * 16 + 8] = o[i][2], dst[i * 16 + 8 + OP] = o[i][3];
    }
  }
  __syncthreads();
  // the block's state: rows x D / 4 vectors over the threads
  for (int i = threadIdx.x; i < rows * (D / 4); i += DEC_THREADS) {
    const int r = i / (D / 4), c = i % (D / 4) * 4;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < DEC_WARPS; ++w) mm = fmaxf(mm, ml_warp[w * 16 + r]);
    const float ref = mm == -INFINITY ? 0.f : mm;
    float ll = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < DEC_WARPS; ++w) {
      const float x = ex2(ml_warp[w * 16 + r] - ref);
      ll += x * ml_warp[w * 16 + 8 + r];
      float4 v = *reinterpret_cast<const float4*>(o_warp + (w * 8 + r) * OP + c);
      if (few) {  // the second parts' product
        const float4 u = *reinterpret_cast<const float4*>(o_warp + (w * 8 + r + 4) * OP + c);
        v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
      }
      acc.x += x * v.x, acc.y += x * v.y, acc.z += x * v.z, acc.w += x * v.w;
    }
    *reinterpret_cast<float4*>(o_block + r * OP + c) = acc;
    if (c == 0) {
      ml_block[r] = mm;
      ml_block[8 + r] = ll;
    }
  }
  if (S > 1) cluster_sync();
  else __syncthreads();
  // the cluster's state: each block joins its share of the columns
  uint16_t* out = static_cast<uint16_t*>(a.o) + ((long long)t * a.Hq + h * G + hb * 8) * D;
  const uint32_t o_addr = smem_u32(o_block), ml_addr = smem_u32(ml_block);
  const int vecs = rows * (D / 4);
  for (int i = rank + S * int(threadIdx.x); i < vecs; i += S * DEC_THREADS) {
    const int r = i / (D / 4), c = i % (D / 4) * 4;
    float ll = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (S > 1) {
      // all blocks' values at once: one trip through the cluster's network
      float mk[MAX_CLUSTER], lk[MAX_CLUSTER];
      float4 v[MAX_CLUSTER];
#pragma unroll
      for (int k = 0; k < MAX_CLUSTER; ++k) {
        const uint32_t from = uint32_t(k < S ? k : rank);
        mk[k] = ld_cluster_f32(cluster_map(ml_addr + r * 4, from));
        lk[k] = ld_cluster_f32(cluster_map(ml_addr + 32 + r * 4, from));
        v[k] = ld_cluster_f4(cluster_map(o_addr + (r * OP + c) * 4, from));
      }
      float mm = -INFINITY;
#pragma unroll
      for (int k = 0; k < MAX_CLUSTER; ++k) mm = fmaxf(mm, k < S ? mk[k] : -INFINITY);
      const float ref = mm == -INFINITY ? 0.f : mm;
#pragma unroll
      for (int k = 0; k < MAX_CLUSTER; ++k)
        if (k < S) {
          const float x = ex2(mk[k] - ref);
          ll += x * lk[k];
          acc.x += x * v[k].x, acc.y += x * v[k].y, acc.z += x * v[k].z, acc.w += x * v[k].w;
        }
    } else {
      ll = ml_block[8 + r];
      acc = *reinterpret_cast<const float4*>(o_block + r * OP + c);
    }
    const float inv = ll > 0.f ? 1.f / ll : (ll == 0.f ? 0.f : ll);  // no key: zeros; NaN stays
    *reinterpret_cast<uint2*>(out + r * D + c) =
        make_uint2(pack2<DT>(acc.x * inv, acc.y * inv), pack2<DT>(acc.z * inv, acc.w * inv));
  }
  if (S > 1) cluster_sync();  // the others have read this block's state
}

// Raises a kernel's dynamic shared memory limit, once per device.
template <auto* Kernel>
int allow_smem(int bytes) {
  static std::atomic<bool> done[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return FA_ERR_LAUNCH;
  if (!done[dev].load(std::memory_order_acquire)) {
    if (cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
      return FA_ERR_LAUNCH;
    done[dev].store(true, std::memory_order_release);
  }
  return FA_OK;
}

template <int D, int DT>
int run_sparse(const SparseArgs& a, const CUtensorMap& k, const CUtensorMap& v) {
  auto* kernel = fa_sparse_decode_kernel<D, DT>;
  const int smem = DecSmem<D>::BYTES;
  if (int rc = allow_smem<fa_sparse_decode_kernel<D, DT>>(smem)) return rc;
  const int G = a.Hq / a.Hkv;
  const long long units = (long long)a.total_q * a.Hkv * ((G + 7) / 8);
  if (units * a.cluster > 0x7fffffffLL) return FA_ERR_BAD_SHAPE;
  return launch_early(kernel, dim3(unsigned(units * a.cluster)), DEC_THREADS, size_t(smem), a.cluster, a.stream, k, v, a);
}

template <int D, int DT>
int run_select(const SelectArgs& a) {
  auto* kernel = fa_select_pages_kernel<D, DT>;
  const int G = a.Hq / a.Hkv;
  const size_t smem = size_t((G + 7) / 8 * 8) * sel_pitch<D>() + (size_t(a.width) * 4 + 15) / 16 * 16;
  constexpr size_t most = size_t(220) << 10;  // of an SM's 227 KB, the static part left out
  if (smem > most) return FA_ERR_BAD_SHAPE;
  if (int rc = allow_smem<fa_select_pages_kernel<D, DT>>(int(most))) return rc;
  const long long units = (long long)a.total_q * a.Hkv;
  if (units * a.cluster > 0x7fffffffLL) return FA_ERR_BAD_SHAPE;
  return launch_early(kernel, dim3(unsigned(units * a.cluster)), SEL_THREADS, smem, a.cluster, a.stream, a);
}

// Blocks that share a unit: the largest power of two up to 8 with which all
// units are on the GPU at once (per_sm blocks a SM) and every block has
// `least` pieces of its unit's work.
int cluster_for(long long units, long long pieces, int least, int per_sm) {
  const long long slots = (long long)device_sm_count() * per_sm;
  int S = 1;
  while (S < MAX_CLUSTER && units * S * 2 <= slots && pieces >= 2LL * S * least) S *= 2;
  return S;
}

}  // namespace

int launch_page_means(const PageArgs& a, int total_q) {
  const long long units = (long long)(total_q >> a.page_log2) + a.B;
  const long long cap = (long long)device_sm_count() * 2;
  const unsigned ctas = unsigned(units < cap ? units : cap);
  const int W8 = a.Hkv * a.D / 8;
  const int cols = W8 < MEAN_THREADS ? W8 : MEAN_THREADS;
  const int groups = MEAN_THREADS / cols < 8 ? MEAN_THREADS / cols : 8;
  const size_t smem = size_t(groups - 1) * 8 * cols * 8;
  if (units > 0x7fffffffLL) return FA_ERR_BAD_SHAPE;
  return launch_early(a.dtype == DT_BF16 ? fa_page_means_kernel<DT_BF16> : fa_page_means_kernel<DT_F16>, dim3(ctas),
                      MEAN_THREADS, smem, 1, a.stream, a, int(units));
}

int launch_select_pages(SelectArgs a, int D) {
  a.cluster = cluster_for((long long)a.total_q * a.Hkv, a.width, 64, 2);
  if (a.dtype == DT_BF16)
    return D == 32 ? run_select<32, DT_BF16>(a) : D == 64 ? run_select<64, DT_BF16>(a) : run_select<128, DT_BF16>(a);
  return D == 32 ? run_select<32, DT_F16>(a) : D == 64 ? run_select<64, DT_F16>(a) : run_select<128, DT_F16>(a);
}

int launch_sparse_decode(SparseArgs a, const CUtensorMap& k, const CUtensorMap& v, int D) {
  const int G = a.Hq / a.Hkv;
  const long long tiles = (((long long)a.top << a.page_log2) + DEC_TILE - 1) / DEC_TILE;
  a.cluster = cluster_for((long long)a.total_q * a.Hkv * ((G + 7) / 8), tiles, 2,
                          D == 128 ? dec_per_sm<128>() : dec_per_sm<64>());
  if (a.dtype == DT_BF16)
    return D == 32 ? run_sparse<32, DT_BF16>(a, k, v)
                   : D == 64 ? run_sparse<64, DT_BF16>(a, k, v) : run_sparse<128, DT_BF16>(a, k, v);
  return D == 32 ? run_sparse<32, DT_F16>(a, k, v)
                 : D == 64 ? run_sparse<64, DT_F16>(a, k, v) : run_sparse<128, DT_F16>(a, k, v);
}

}  // namespace fa
