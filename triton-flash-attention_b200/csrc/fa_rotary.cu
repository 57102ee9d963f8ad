// fa_rotary.cu -- per-head RMS norm of queries and keys and the rotation by
// their positions in one pass, forward and backward, and the serving form
// that writes the prepared keys and the values into a paged cache.
//
// A row is one head of one token, x of D values.  With r = rsqrt(mean(x^2) +
// eps) and weights w the normed row is y = x r w, and a pair (a, b) of its
// first rd columns turns by the angle of its position:
//   a' = a cos - b sin,  b' = b cos + a sin.
// Pair i is columns (i, i + rd/2), or (2i, 2i + 1) when interleaved; columns
// past rd are not turned.  Backward, with dy the incoming gradient turned
// back and g = dy w:
//   dx = r (g - x r^2 mean(g x)),   dw = sum over rows of dy x r.
//
// All arithmetic is fp32 on registers and each result is rounded once.  The
// table holds fp32 cosines and sines made from 64-bit angles.
//
// Bound: HBM.  A forward moves 4 bytes an element, a backward 6.  D / 16
// lanes own a row, each lane 8 + 8 of its columns placed so that a lane
// holds both halves of its pairs: the rotation needs no exchange and the
// mean of squares log2(D / 16) shuffles.  A group of lanes takes several
// heads of one token, so that its cosines and sines are read once for all of
// them and that many 16-byte load pairs are in flight.
#include "fa_kernels.h"

namespace fa {
namespace {

// 16 bytes read once.
__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

template <int DT>
__device__ __forceinline__ void unpack8(const uint4& v, float* f) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = unpack2<DT>(u[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
template <int DT>
__device__ __forceinline__ uint4 pack8(const float* f) {
  return make_uint4(pack2<DT>(f[0], f[1]), pack2<DT>(f[2], f[3]), pack2<DT>(f[4], f[5]), pack2<DT>(f[6], f[7]));
}

// Columns [a, a + 8) and [b, b + 8) of a row belong to lane l of its group.
// Halves: the lanes below rd / 16 hold pair i's two columns at the same
// place of a and b; interleaved: 16 neighbouring columns a lane.
struct LaneCols {
  int a, b;
  bool turned;
};
template <bool INTER>
__device__ __forceinline__ LaneCols lane_cols(int l, int rd) {
  LaneCols c;
  c.turned = l < rd / 16;
  if (INTER || !c.turned) {
    c.a = 16 * l;
    c.b = 16 * l + 8;
  } else {
    c.a = 8 * l;
    c.b = rd / 2 + 8 * l;
  }
  return c;
}

// This lane's 8 cosines and sines of position p: pairs 8 l .. 8 l + 7.
__device__ __forceinline__ void load_trig(const float* __restrict__ table, int rd, int p, int l, float (&cs)[8],
                                          float (&sn)[8]) {
  const float* t = table + (long long)p * rd + 8 * l;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 c = __ldg(reinterpret_cast<const float4*>(t) + i);
    const float4 s = __ldg(reinterpret_cast<const float4*>(t + rd / 2) + i);
    cs[4 * i] = c.x, cs[4 * i + 1] = c.y, cs[4 * i + 2] = c.z, cs[4 * i + 3] = c.w;
    sn[4 * i] = s.x, sn[4 * i + 1] = s.y, sn[4 * i + 2] = s.z, sn[4 * i + 3] = s.w;
  }
}

// Turns the lane's columns by (cs, sgn * sn).
template <bool INTER>
__device__ __forceinline__ void turn(float (&a)[8], float (&b)[8], const float (&cs)[8], const float (&sn)[8],
                                     float sgn) {
  if constexpr (INTER) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float s0 = sgn * sn[i], s1 = sgn * sn[4 + i];
      const float x0 = a[2 * i], y0 = a[2 * i + 1], x1 = b[2 * i], y1 = b[2 * i + 1];
      a[2 * i] = x0 * cs[i] - y0 * s0;
      a[2 * i + 1] = y0 * cs[i] + x0 * s0;
      b[2 * i] = x1 * cs[4 + i] - y1 * s1;
      b[2 * i + 1] = y1 * cs[4 + i] + x1 * s1;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float s = sgn * sn[i];
      const float x = a[i], y = b[i];
      a[i] = x * cs[i] - y * s;
      b[i] = y * cs[i] + x * s;
    }
  }
}

// 8 consecutive weights from column c, in the operand type or fp32.
template <int DT>
__device__ __forceinline__ void load_w(const void* w, int w_fp32, int c, float (&f)[8]) {
  if (w_fp32) {
    const float* p = static_cast<const float*>(w) + c;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __ldg(p + i);
  } else {
    const uint16_t* p = static_cast<const uint16_t*>(w) + c;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = unpack2<DT>(uint32_t(__ldg(p + i))).x;
  }
}

template <int L>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int m = L / 2; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}

// Position of token (b, n), or -1 (with the device status word set) when it
// has no row in the table.
__device__ __forceinline__ int checked_pos(const RotaryArgs& a, int b, int n) {
  const int p = a.pos ? __ldg(a.pos + (long long)b * a.pos_sb + n) : n;
  if (p >= 0 && p < a.max_pos) return p;
  if (a.status) atomicCAS(a.status, 0, (FA_SITE_POSITION << 8) | FA_ERR_BAD_INDEX);
  return -1;
}
__device__ __forceinline__ void load_trig_checked(const RotaryArgs& a, int p, int l, float (&cs)[8], float (&sn)[8]) {
  if (p >= 0) {
    load_trig(a.table, a.rd, p, l, cs, sn);
  } else {  // no such position: the turned columns come out NaN
#pragma unroll
    for (int i = 0; i < 8; ++i) cs[i] = sn[i] = __int_as_float(0x7fc00000);
  }
}

constexpr int FWD_THREADS = 256;
constexpr int HB = 4;  // heads a group of lanes takes of one token

// One group of D / 16 lanes per (token, HB heads of q, of k or -- APPEND --
// of v); groups of one token are neighbours, so that they share its table
// row in L1.  APPEND: k and v rows go to row slots[n] of the caches.
template <int D, int DT, bool INTER, bool APPEND>
__global__ void __launch_bounds__(FWD_THREADS) fa_rotary_fwd_kernel(const __grid_constant__ RotaryArgs a) {
  constexpr int L = D / 16;
  const uint32_t item = (blockIdx.x * uint32_t(FWD_THREADS) + threadIdx.x) / L;
  const int l = threadIdx.x % L;
  const int q_blocks = (a.Hq + HB - 1) / HB, k_blocks = (a.Hkv + HB - 1) / HB;
  const uint32_t per_token = q_blocks + k_blocks * (APPEND ? 2 : 1);
  const uint32_t token = item / per_token;
  int blk = int(item - token * per_token);
  // groups past the end stay for the shuffles and touch nothing
  const bool live = token < uint32_t(a.B) * uint32_t(a.N);
  const int b = live ? int(token / uint32_t(a.N)) : 0;
  const int n = live ? int(token - uint32_t(b) * uint32_t(a.N)) : 0;
  const int which = blk < q_blocks ? 0 : blk < q_blocks + k_blocks ? 1 : 2;
  blk -= which == 0 ? 0 : which == 1 ? q_blocks : q_blocks + k_blocks;
  const int h0 = blk * HB;
  const int heads = live ? min(HB, (which == 0 ? a.Hq : a.Hkv) - h0) : 0;
  const uint16_t* src = static_cast<const uint16_t*>(which == 0 ? a.q : which == 1 ? a.k : a.v);
  const RowStrides si = which == 0 ? a.qs : which == 1 ? a.ks : a.vs;
  uint16_t* dst;
  RowStrides so;
  int stored = heads;
  if (which == 0 || !APPEND) {
    dst = static_cast<uint16_t*>(which == 0 ? a.qo : a.ko);
    so = which == 0 ? a.qos : a.kos;
    dst += (long long)b * so.b + (long long)n * so.n + (long long)h0 * so.h;
  } else {
    so.h = D;
    long long slot = live ? __ldg(a.slots + n) : -1;
    if (slot >= a.n_slots) {
      if (a.status) atomicCAS(a.status, 0, (FA_SITE_SLOT << 8) | FA_ERR_BAD_INDEX);
      slot = -1;
    }
    if (slot < 0) stored = 0, slot = 0;
    dst = static_cast<uint16_t*>(which == 1 ? a.ko : a.vo) + (slot * a.Hkv + h0) * D;
  }
  src += (long long)b * si.b + (long long)n * si.n + (long long)h0 * si.h;
  const LaneCols c = lane_cols<INTER>(l, which == 2 ? 0 : a.rd);
  uint4 va[HB], vb[HB];
#pragma unroll
  for (int i = 0; i < HB; ++i)
    if (i < heads) {
      va[i] = ld_stream(src + (long long)i * si.h + c.a);
      vb[i] = ld_stream(src + (long long)i * si.h + c.b);
    }
  if (APPEND && which == 2) {
#pragma unroll
    for (int i = 0; i < HB; ++i)
      if (i < stored) {
        *reinterpret_cast<uint4*>(dst + (long long)i * so.h + c.a) = va[i];
        *reinterpret_cast<uint4*>(dst + (long long)i * so.h + c.b) = vb[i];
      }
  }
  float cs[8], sn[8];
  if (c.turned && which != 2 && heads > 0) load_trig_checked(a, checked_pos(a, b, n), l, cs, sn);
  const void* w = which == 0 ? a.wq : a.wk;
  const bool norm = w != nullptr && which != 2;
  float wa[8], wb[8];
  if (norm) {
    load_w<DT>(w, a.w_fp32, c.a, wa);
    load_w<DT>(w, a.w_fp32, c.b, wb);
  }
#pragma unroll
  for (int i = 0; i < HB; ++i) {
    float x[8], y[8];
    if (i < heads) {
      unpack8<DT>(va[i], x);
      unpack8<DT>(vb[i], y);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = y[j] = 0.f;
    }
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], fmaf(y[j], y[j], ss));
    ss = group_sum<L>(ss);  // all lanes of the warp come here
    if (norm) {
      const float r = rsqrtf(ss * (1.f / D) + a.eps);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] *= r * wa[j], y[j] *= r * wb[j];
    }
    if (c.turned) turn<INTER>(x, y, cs, sn, 1.f);
    if (i < stored && which != 2) {
      *reinterpret_cast<uint4*>(dst + (long long)i * so.h + c.a) = pack8<DT>(x);
      *reinterpret_cast<uint4*>(dst + (long long)i * so.h + c.b) = pack8<DT>(y);
    }
  }
}

constexpr int BWD_THREADS = 256;
constexpr int BWD_HB = 2;

// Backward.  The first q_ctas blocks take the query rows, the others the key
// rows, so that a lane's weight-gradient sums (16 fp32 registers) are of one
// weight; each block loops over its (token, BWD_HB heads) items and leaves
// its sums in w_part[block][D] for the reduction that follows.  The sums run
// in an order that the launch alone decides, so gradients repeat bit for bit.
template <int D, int DT, bool INTER>
__global__ void __launch_bounds__(BWD_THREADS) fa_rotary_bwd_kernel(const __grid_constant__ RotaryArgs a) {
  constexpr int L = D / 16;
  constexpr int GROUPS = BWD_THREADS / L;
  const bool is_q = int(blockIdx.x) < a.q_ctas;
  const uint32_t cta = is_q ? blockIdx.x : blockIdx.x - a.q_ctas;
  const uint32_t ctas = is_q ? a.q_ctas : gridDim.x - a.q_ctas;
  const int l = threadIdx.x % L;
  const int H = is_q ? a.Hq : a.Hkv;
  const uint32_t blocks = (H + BWD_HB - 1) / BWD_HB;
  const uint32_t items = uint32_t(a.B) * uint32_t(a.N) * blocks;
  const uint16_t* xb = static_cast<const uint16_t*>(is_q ? a.q : a.k);
  const uint16_t* gb = static_cast<const uint16_t*>(is_q ? a.gq : a.gk);
  uint16_t* ob = static_cast<uint16_t*>(is_q ? a.qo : a.ko);
  const RowStrides sx = is_q ? a.qs : a.ks, sg = is_q ? a.gqs : a.gks, so = is_q ? a.qos : a.kos;
  const void* w = is_q ? a.wq : a.wk;
  const bool norm = w != nullptr;
  const LaneCols c = lane_cols<INTER>(l, a.rd);
  float wa[8], wb[8], dwa[8], dwb[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) dwa[j] = dwb[j] = 0.f;
  if (norm) {
    load_w<DT>(w, a.w_fp32, c.a, wa);
    load_w<DT>(w, a.w_fp32, c.b, wb);
  }
  // the trip count is the block's, so that its warps stay whole for the shuffles
  for (uint32_t base = cta * GROUPS; base < items; base += ctas * GROUPS) {
    const uint32_t item = base + threadIdx.x / L;
    const bool live = item < items;
    const uint32_t token = live ? item / blocks : 0;
    const int h0 = live ? int(item - token * blocks) * BWD_HB : 0;
    const int heads = live ? min(BWD_HB, H - h0) : 0;
    const int b = int(token / uint32_t(a.N));
    const int n = int(token - uint32_t(b) * uint32_t(a.N));
    const uint16_t* xp = xb + (long long)b * sx.b + (long long)n * sx.n + (long long)h0 * sx.h;
    const uint16_t* gp = gb + (long long)b * sg.b + (long long)n * sg.n + (long long)h0 * sg.h;
    uint16_t* op = ob + (long long)b * so.b + (long long)n * so.n + (long long)h0 * so.h;
    uint4 xa[BWD_HB], xv[BWD_HB], ga[BWD_HB], gv[BWD_HB];
#pragma unroll
    for (int i = 0; i < BWD_HB; ++i)
      if (i < heads) {
        ga[i] = ld_stream(gp + (long long)i * sg.h + c.a);
        gv[i] = ld_stream(gp + (long long)i * sg.h + c.b);
        if (norm) {
          xa[i] = ld_stream(xp + (long long)i * sx.h + c.a);
          xv[i] = ld_stream(xp + (long long)i * sx.h + c.b);
        }
      }
    float cs[8], sn[8];
    if (c.turned && heads > 0) load_trig_checked(a, checked_pos(a, b, n), l, cs, sn);
#pragma unroll
    for (int i = 0; i < BWD_HB; ++i) {
      float ya[8], yb[8];
      if (i < heads) {
        unpack8<DT>(ga[i], ya);
        unpack8<DT>(gv[i], yb);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) ya[j] = yb[j] = 0.f;
      }
      if (c.turned && i < heads) turn<INTER>(ya, yb, cs, sn, -1.f);
      if (norm) {
        float x[8], y[8];
        if (i < heads) {
          unpack8<DT>(xa[i], x);
          unpack8<DT>(xv[i], y);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = y[j] = 0.f;
        }
        float ss = 0.f, gx = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          ss = fmaf(x[j], x[j], fmaf(y[j], y[j], ss));
          gx = fmaf(ya[j] * wa[j], x[j], fmaf(yb[j] * wb[j], y[j], gx));
        }
        ss = group_sum<L>(ss);
        gx = group_sum<L>(gx);
        const float r = rsqrtf(ss * (1.f / D) + a.eps);
        const float m = gx * (1.f / D) * r * r;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          dwa[j] = fmaf(ya[j], x[j] * r, dwa[j]);
          dwb[j] = fmaf(yb[j], y[j] * r, dwb[j]);
          ya[j] = r * (ya[j] * wa[j] - x[j] * m);
          yb[j] = r * (yb[j] * wb[j] - y[j] * m);
        }
      }
      if (i < heads) {
        *reinterpret_cast<uint4*>(op + (long long)i * so.h + c.a) = pack8<DT>(ya);
        *reinterpret_cast<uint4*>(op + (long long)i * so.h + c.b) = pack8<DT>(yb);
      }
    }
  }
  if (!norm || a.w_part == nullptr) return;
  __shared__ float sums[GROUPS][D + 4];
  float* mine = sums[threadIdx.x / L];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    mine[c.a + j] = dwa[j];
    mine[c.b + j] = dwb[j];
  }
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += BWD_THREADS) {
    float s = 0.f;
    for (int g = 0; g < GROUPS; ++g) s += sums[g][d];
    a.w_part[(long long)blockIdx.x * D + d] = s;
  }
}

// Weight gradients: block 0 sums the query blocks' partial sums, block 1 the
// key blocks', each in a fixed order.
template <int D, int DT>
__global__ void __launch_bounds__(1024) fa_rotary_dw_kernel(const float* __restrict__ part, int q_ctas, int ctas,
                                                            void* dwq, void* dwk, int w_fp32) {
  constexpr int SLICES = 1024 / D;
  __shared__ float sums[SLICES][D];
  const int first = blockIdx.x == 0 ? 0 : q_ctas;
  const int last = blockIdx.x == 0 ? q_ctas : ctas;
  const int d = threadIdx.x % D, s = threadIdx.x / D;
  float v = 0.f;
  for (int i = first + s; i < last; i += SLICES) v += part[(long long)i * D + d];
  sums[s][d] = v;
  __syncthreads();
  if (s != 0) return;
  v = 0.f;
#pragma unroll
  for (int i = 0; i < SLICES; ++i) v += sums[i][d];
  void* out = blockIdx.x == 0 ? dwq : dwk;
  if (w_fp32)
    static_cast<float*>(out)[d] = v;
  else
    static_cast<uint16_t*>(out)[d] = uint16_t(pack2<DT>(v, 0.f) & 0xffffu);
}

template <int D, int DT, bool INTER, bool APPEND>
int run_fwd(const RotaryArgs& a) {
  const long long per = (a.Hq + HB - 1) / HB + (long long)((a.Hkv + HB - 1) / HB) * (APPEND ? 2 : 1);
  const long long items = per * a.B * a.N;
  constexpr int GROUPS = FWD_THREADS / (D / 16);
  if (items > 0x7fffffffLL * GROUPS || items + GROUPS > 0xffffffffLL) return FA_ERR_BAD_SHAPE;
  fa_rotary_fwd_kernel<D, DT, INTER, APPEND>
      <<<unsigned((items + GROUPS - 1) / GROUPS), FWD_THREADS, 0, a.stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? FA_OK : FA_ERR_LAUNCH;
}

template <int D, int DT, bool INTER>
int run_bwd(RotaryArgs a) {
  constexpr int GROUPS = BWD_THREADS / (D / 16);
  const long long rows = (long long)a.B * a.N;
  const long long q_items = rows * ((a.Hq + BWD_HB - 1) / BWD_HB), k_items = rows * ((a.Hkv + BWD_HB - 1) / BWD_HB);
  if (q_items + 4096LL * GROUPS > 0xffffffffLL || k_items + 4096LL * GROUPS > 0xffffffffLL) return FA_ERR_BAD_SHAPE;
  int q_ctas, k_ctas;
  rotary_bwd_ctas(a.Hq, a.Hkv, rows, D, &q_ctas, &k_ctas);
  a.q_ctas = q_ctas;
  fa_rotary_bwd_kernel<D, DT, INTER><<<q_ctas + k_ctas, BWD_THREADS, 0, a.stream>>>(a);
  if (cudaGetLastError() != cudaSuccess) return FA_ERR_LAUNCH;
  if (a.w_part) {
    fa_rotary_dw_kernel<D, DT><<<2, 1024, 0, a.stream>>>(a.w_part, q_ctas, q_ctas + k_ctas, a.dwq, a.dwk, a.w_fp32);
    if (cudaGetLastError() != cudaSuccess) return FA_ERR_LAUNCH;
  }
  return FA_OK;
}

template <int DT, bool INTER, bool APPEND>
int by_d(const RotaryArgs& a, int D, bool bwd) {
  if constexpr (!APPEND)
    if (bwd) {
      if (D == 32) return run_bwd<32, DT, INTER>(a);
      if (D == 64) return run_bwd<64, DT, INTER>(a);
      return run_bwd<128, DT, INTER>(a);
    }
  if (D == 32) return run_fwd<32, DT, INTER, APPEND>(a);
  if (D == 64) return run_fwd<64, DT, INTER, APPEND>(a);
  return run_fwd<128, DT, INTER, APPEND>(a);
}
template <bool APPEND>
int by_type(const RotaryArgs& a, int D, bool bwd) {
  if (a.dtype == DT_BF16)
    return a.interleaved ? by_d<DT_BF16, true, APPEND>(a, D, bwd) : by_d<DT_BF16, false, APPEND>(a, D, bwd);
  return a.interleaved ? by_d<DT_F16, true, APPEND>(a, D, bwd) : by_d<DT_F16, false, APPEND>(a, D, bwd);
}

}  // namespace

// Blocks of the backward: four a SM at most, shared between queries and keys
// by their heads, none without a full turn of work.
void rotary_bwd_ctas(int Hq, int Hkv, long long rows, int D, int* q_ctas, int* k_ctas) {
  const long long groups = BWD_THREADS / (D / 16);
  const long long most = ROTARY_BWD_CTAS;
  const long long q_need = (rows * ((Hq + BWD_HB - 1) / BWD_HB) + groups - 1) / groups;
  const long long k_need = (rows * ((Hkv + BWD_HB - 1) / BWD_HB) + groups - 1) / groups;
  long long k = most * Hkv / (Hq + Hkv);
  if (k < 1) k = 1;
  const long long q = most - k;
  *q_ctas = int(q < q_need ? q : q_need);
  *k_ctas = int(k < k_need ? k : k_need);
}

int launch_rotary_fwd(const RotaryArgs& a, int D) { return by_type<false>(a, D, false); }
int launch_rotary_bwd(const RotaryArgs& a, int D) { return by_type<false>(a, D, true); }
int launch_paged_append(const RotaryArgs& a, int D) { return by_type<true>(a, D, false); }

}  // namespace fa
