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
// Bound: HBM.  A forward moves 4 bytes an element, a backward 6.  D / 8
// lanes own a row, each lane 4 + 4 of its columns placed so that a lane
// holds both halves of its pairs: the rotation needs no exchange and the
// mean of squares log2(D / 8) shuffles.  A group of lanes takes several
// heads of one token, so that its cosines and sines are read once for all of
// them and that many 8-byte load pairs are in flight.  (8 + 8 columns a lane
// halve the loads but double what a lane keeps -- angles, weights, weight
// gradients --, and with fewer warps a SM ran slower.)
#include "fa_kernels.h"

namespace fa {
namespace {

// A lane's run of C columns as fp32 pairs: packed instructions take two of
// them at once (the forward issued 70 % of its slots without them).
template <int C>
struct Run {
  uint64_t p[C / 2];
};
template <int C>
struct Raw {  // the same run in the operand type
  uint32_t u[C / 2];
};

// C elements, read once.
template <int C>
__device__ __forceinline__ Raw<C> ld_stream(const void* p) {
  Raw<C> r;
  if constexpr (C == 8)
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r.u[0]), "=r"(r.u[1]), "=r"(r.u[2]), "=r"(r.u[3])
                 : "l"(p));
  else
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(r.u[0]), "=r"(r.u[1]) : "l"(p));
  return r;
}
template <int C>
__device__ __forceinline__ void st_run(void* p, const Raw<C>& r) {
  if constexpr (C == 8) *static_cast<uint4*>(p) = make_uint4(r.u[0], r.u[1], r.u[2], r.u[3]);
  else *static_cast<uint2*>(p) = make_uint2(r.u[0], r.u[1]);
}
template <int DT, int C>
__device__ __forceinline__ Run<C> widen(const Raw<C>& r) {
  Run<C> f;
#pragma unroll
  for (int i = 0; i < C / 2; ++i) {
    const float2 t = unpack2<DT>(r.u[i]);
    f.p[i] = f2pack(t.x, t.y);
  }
  return f;
}
template <int DT, int C>
__device__ __forceinline__ Raw<C> narrow(const Run<C>& f) {
  Raw<C> r;
#pragma unroll
  for (int i = 0; i < C / 2; ++i) r.u[i] = pack2_f2<DT>(f.p[i]);
  return r;
}
template <int C>
__device__ __forceinline__ Run<C> zero_run() {
  Run<C> f;
#pragma unroll
  for (int i = 0; i < C / 2; ++i) f.p[i] = 0;
  return f;
}
__device__ __forceinline__ uint64_t both(float v) { return f2pack(v, v); }
__device__ __forceinline__ uint64_t neg2(uint64_t v) { return v ^ 0x8000000080000000ull; }
__device__ __forceinline__ uint64_t swap2(uint64_t v) {
  float lo, hi;
  f2unpack(v, lo, hi);
  return f2pack(hi, lo);
}
__device__ __forceinline__ float add_halves(uint64_t v) {
  float lo, hi;
  f2unpack(v, lo, hi);
  return lo + hi;
}

// Columns [a, a + C) and [b, b + C) of a row belong to lane l of its group.
// Halves: the lanes below rd / 2 C hold pair i's two columns at the same
// place of a and b; interleaved: 2 C neighbouring columns a lane.
struct LaneCols {
  int a, b;
  bool turned;
};
template <bool INTER, int C>
__device__ __forceinline__ LaneCols lane_cols(int l, int rd) {
  LaneCols c;
  c.turned = l < rd / (2 * C);
  if (INTER || !c.turned) {
    c.a = 2 * C * l;
    c.b = 2 * C * l + C;
  } else {
    c.a = C * l;
    c.b = rd / 2 + C * l;
  }
  return c;
}

// C consecutive floats.
template <int C>
__device__ __forceinline__ Run<C> ld_floats(const float* p) {
  Run<C> f;
#pragma unroll
  for (int i = 0; i < C / 4; ++i) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(p) + i);
    f.p[2 * i] = f2pack(v.x, v.y);
    f.p[2 * i + 1] = f2pack(v.z, v.w);
  }
  return f;
}

// A lane's angles, laid out for turn(): cosines and sines of its C pairs.
// Halves: cs and sn of pair i at place i.  Interleaved: pair i is one packed
// value, so cs and sn hold (c, c) and (-s, s) of the pairs of run a, then b
// (C / 2 each, in ca, sa and cb, sb).
template <bool INTER, int C>
struct Angles {
  Run<C> ca, sa;
  Run<INTER ? C : 2> cb, sb;
};
template <bool INTER, int C>
__device__ __forceinline__ Angles<INTER, C> arrange(const Run<C>& cs, const Run<C>& sn) {
  Angles<INTER, C> g;
  if constexpr (INTER) {
#pragma unroll
    for (int i = 0; i < C / 2; ++i) {  // pairs 2 i and 2 i + 1 of the lane's C
      float c0, c1, s0, s1;
      f2unpack(cs.p[i], c0, c1);
      f2unpack(sn.p[i], s0, s1);
      Run<C>& c = 2 * i < C / 2 ? g.ca : g.cb;
      Run<C>& s = 2 * i < C / 2 ? g.sa : g.sb;
      const int at = (2 * i) % (C / 2);
      c.p[at] = both(c0);
      c.p[at + 1] = both(c1);
      s.p[at] = f2pack(-s0, s0);
      s.p[at + 1] = f2pack(-s1, s1);
    }
  } else {
    g.ca = cs;
    g.sa = sn;
    g.cb.p[0] = g.sb.p[0] = 0;
  }
  return g;
}
// Turns the runs; BACK: the other way.
template <bool INTER, bool BACK, int C>
__device__ __forceinline__ void turn(Run<C>& a, Run<C>& b, const Angles<INTER, C>& g) {
#pragma unroll
  for (int i = 0; i < C / 2; ++i) {
    const uint64_t x = a.p[i], y = b.p[i];
    if constexpr (INTER) {
      const uint64_t sx = BACK ? neg2(g.sa.p[i]) : g.sa.p[i], sy = BACK ? neg2(g.sb.p[i]) : g.sb.p[i];
      a.p[i] = ffma2(x, g.ca.p[i], fmul2(swap2(x), sx));
      b.p[i] = ffma2(y, g.cb.p[i], fmul2(swap2(y), sy));
    } else {
      const uint64_t s = BACK ? neg2(g.sa.p[i]) : g.sa.p[i];
      a.p[i] = ffma2(x, g.ca.p[i], fmul2(neg2(y), s));
      b.p[i] = ffma2(y, g.ca.p[i], fmul2(x, s));
    }
  }
}

// C consecutive weights from column c, in the operand type or fp32.
template <int DT, int C>
__device__ __forceinline__ Run<C> load_w(const void* w, int w_fp32, int c) {
  Run<C> f;
#pragma unroll
  for (int i = 0; i < C / 2; ++i) {
    if (w_fp32) {
      const float* p = static_cast<const float*>(w) + c + 2 * i;
      f.p[i] = f2pack(__ldg(p), __ldg(p + 1));
    } else {
      const uint16_t* p = static_cast<const uint16_t*>(w) + c + 2 * i;
      f.p[i] = f2pack(unpack2<DT>(uint32_t(__ldg(p))).x, unpack2<DT>(uint32_t(__ldg(p + 1))).x);
    }
  }
  return f;
}

template <int L>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int m = L / 2; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}
template <int L>
__device__ __forceinline__ uint64_t group_sum2(uint64_t v) {
#pragma unroll
  for (int m = L / 2; m > 0; m >>= 1) v = fadd2(v, __shfl_xor_sync(0xffffffffu, v, m));
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
template <bool INTER, int C>
__device__ __forceinline__ Angles<INTER, C> load_angles(const RotaryArgs& a, int p, int l) {
  Run<C> cs, sn;
  if (p >= 0) {
    const float* t = a.table + (long long)p * a.rd + C * l;
    cs = ld_floats<C>(t);
    sn = ld_floats<C>(t + a.rd / 2);
  } else {  // no such position: the turned columns come out NaN
#pragma unroll
    for (int i = 0; i < C / 2; ++i) cs.p[i] = sn.p[i] = both(__int_as_float(0x7fc00000));
  }
  return arrange<INTER, C>(cs, sn);
}

#ifndef T_FC
#define T_FC 8
#endif
#ifndef T_BC
#define T_BC 4
#endif
#ifndef T_HB
#define T_HB 4
#endif
#ifndef T_BHB
#define T_BHB 4
#endif
#ifndef T_FMIN
#define T_FMIN 2
#endif
#ifndef T_BMIN
#define T_BMIN 2
#endif
#ifndef T_BCTAS
#define T_BCTAS 296
#endif
#ifndef T_FT
#define T_FT 256
#endif
#ifndef T_BT
#define T_BT 256
#endif
constexpr int FWD_THREADS = T_FT;
constexpr int FC = T_FC;  // columns of a lane's run
constexpr int HB = T_HB;  // heads a group of lanes takes of one token

// One group of D / 2 C lanes per (token, HB heads of q, of k or -- APPEND --
// of v); groups of one token are neighbours, so that they share its table
// row in L1.  APPEND: k and v rows go to row slots[n] of the caches.
template <int D, int DT, bool INTER, bool APPEND>
__global__ void __launch_bounds__(FWD_THREADS, T_FMIN) fa_rotary_fwd_kernel(const __grid_constant__ RotaryArgs a) {
  constexpr int C = FC;
  constexpr int L = D / (2 * C);
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
  const LaneCols c = lane_cols<INTER, C>(l, a.rd);
  src += (long long)b * si.b + (long long)n * si.n + (long long)h0 * si.h;
  Raw<C> va[HB], vb[HB];
#pragma unroll
  for (int i = 0; i < HB; ++i)
    if (i < heads) {
      va[i] = ld_stream<C>(src + (long long)i * si.h + c.a);
      vb[i] = ld_stream<C>(src + (long long)i * si.h + c.b);
    }
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
  if (APPEND && which == 2) {
#pragma unroll
    for (int i = 0; i < HB; ++i)
      if (i < stored) {
        st_run<C>(dst + (long long)i * so.h + c.a, va[i]);
        st_run<C>(dst + (long long)i * so.h + c.b, vb[i]);
      }
    stored = 0;
  }
  if (APPEND && __all_sync(0xffffffffu, which == 2)) return;
  Angles<INTER, C> g;
  const bool turned = c.turned && which != 2 && heads > 0;
  if (turned) g = load_angles<INTER, C>(a, checked_pos(a, b, n), l);
  const bool norm = a.wq != nullptr;  // of every row of the launch
  Run<C> wa, wb;
  if (norm) {
    const void* w = which == 0 ? a.wq : a.wk;
    wa = load_w<DT, C>(w, a.w_fp32, c.a);
    wb = load_w<DT, C>(w, a.w_fp32, c.b);
  }
#pragma unroll
  for (int i = 0; i < HB; ++i) {
    Run<C> x, y;
    if (i < heads) {
      x = widen<DT, C>(va[i]);
      y = widen<DT, C>(vb[i]);
    } else {
      x = y = zero_run<C>();
    }
    if (norm) {
      uint64_t ss = 0;
#pragma unroll
      for (int j = 0; j < C / 2; ++j) ss = ffma2(x.p[j], x.p[j], ffma2(y.p[j], y.p[j], ss));
      const float s = group_sum<L>(add_halves(ss));  // all lanes of the warp come here
      const uint64_t r = both(rsqrtf(s * (1.f / D) + a.eps));
#pragma unroll
      for (int j = 0; j < C / 2; ++j) {
        x.p[j] = fmul2(x.p[j], fmul2(r, wa.p[j]));
        y.p[j] = fmul2(y.p[j], fmul2(r, wb.p[j]));
      }
    }
    if (turned) turn<INTER, false, C>(x, y, g);
    if (i < stored) {
      st_run<C>(dst + (long long)i * so.h + c.a, narrow<DT, C>(x));
      st_run<C>(dst + (long long)i * so.h + c.b, narrow<DT, C>(y));
    }
  }
}

constexpr int BWD_THREADS = T_BT;
constexpr int BC = T_BC;
constexpr int BWD_HB = T_BHB;

// Backward.  The first q_ctas blocks take the query rows, the others the key
// rows, so that a lane's weight-gradient sums (2 C fp32 registers) are of one
// weight; each block loops over its (token, BWD_HB heads) items and leaves
// its sums in w_part[block][D] for the reduction that follows.  The sums run
// in an order that the launch alone decides, so gradients repeat bit for bit.
template <int D, int DT, bool INTER>
__global__ void __launch_bounds__(BWD_THREADS, T_BMIN) fa_rotary_bwd_kernel(const __grid_constant__ RotaryArgs a) {
  constexpr int C = BC;
  constexpr int L = D / (2 * C);
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
  const LaneCols c = lane_cols<INTER, C>(l, a.rd);
  Run<C> wa, wb, dwa = zero_run<C>(), dwb = zero_run<C>();
  if (norm) {
    wa = load_w<DT, C>(w, a.w_fp32, c.a);
    wb = load_w<DT, C>(w, a.w_fp32, c.b);
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
    Raw<C> xa[BWD_HB], xv[BWD_HB], ga[BWD_HB], gv[BWD_HB];
#pragma unroll
    for (int i = 0; i < BWD_HB; ++i)
      if (i < heads) {
        ga[i] = ld_stream<C>(gp + (long long)i * sg.h + c.a);
        gv[i] = ld_stream<C>(gp + (long long)i * sg.h + c.b);
        if (norm) {
          xa[i] = ld_stream<C>(xp + (long long)i * sx.h + c.a);
          xv[i] = ld_stream<C>(xp + (long long)i * sx.h + c.b);
        }
      }
    Angles<INTER, C> g;
    const bool turned = c.turned && heads > 0;
    if (turned) g = load_angles<INTER, C>(a, checked_pos(a, b, n), l);
#pragma unroll
    for (int i = 0; i < BWD_HB; ++i) {
      Run<C> ya, yb;
      if (i < heads) {
        ya = widen<DT, C>(ga[i]);
        yb = widen<DT, C>(gv[i]);
      } else {
        ya = yb = zero_run<C>();
      }
      if (turned && i < heads) turn<INTER, true, C>(ya, yb, g);
      if (norm) {
        Run<C> x, y;
        if (i < heads) {
          x = widen<DT, C>(xa[i]);
          y = widen<DT, C>(xv[i]);
        } else {
          x = y = zero_run<C>();
        }
        uint64_t ss = 0, gx = 0;
        Run<C> ta, tb;  // dy w
#pragma unroll
        for (int j = 0; j < C / 2; ++j) {
          ta.p[j] = fmul2(ya.p[j], wa.p[j]);
          tb.p[j] = fmul2(yb.p[j], wb.p[j]);
          ss = ffma2(x.p[j], x.p[j], ffma2(y.p[j], y.p[j], ss));
          gx = ffma2(ta.p[j], x.p[j], ffma2(tb.p[j], y.p[j], gx));
        }
        float s, t;
        f2unpack(group_sum2<L>(f2pack(add_halves(ss), add_halves(gx))), s, t);
        const float r = rsqrtf(s * (1.f / D) + a.eps);
        const uint64_t rr = both(r), m = both(-t * (1.f / D) * r * r);
#pragma unroll
        for (int j = 0; j < C / 2; ++j) {
          const uint64_t xr = fmul2(x.p[j], rr), yr = fmul2(y.p[j], rr);
          dwa.p[j] = ffma2(ya.p[j], xr, dwa.p[j]);
          dwb.p[j] = ffma2(yb.p[j], yr, dwb.p[j]);
          ya.p[j] = ffma2(xr, m, fmul2(ta.p[j], rr));
          yb.p[j] = ffma2(yr, m, fmul2(tb.p[j], rr));
        }
      }
      if (i < heads) {
        st_run<C>(op + (long long)i * so.h + c.a, narrow<DT, C>(ya));
        st_run<C>(op + (long long)i * so.h + c.b, narrow<DT, C>(yb));
      }
    }
  }
  if (!norm || a.w_part == nullptr) return;
  __shared__ float sums[GROUPS][D + 4];
  float* mine = sums[threadIdx.x / L];
#pragma unroll
  for (int j = 0; j < C / 2; ++j) {
    f2unpack(dwa.p[j], mine[c.a + 2 * j], mine[c.a + 2 * j + 1]);
    f2unpack(dwb.p[j], mine[c.b + 2 * j], mine[c.b + 2 * j + 1]);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += BWD_THREADS) {
    float s = 0.f;
    for (int g = 0; g < GROUPS; ++g) s += sums[g][d];
    a.w_part[(long long)blockIdx.x * D + d] = s;
  }
}

// Weight gradients: block (x, y) sums columns 32 x .. of the query blocks'
// partial sums (y = 0) or the key blocks' (y = 1), 32 rows of them a pass, in
// a fixed order.
template <int DT>
__global__ void __launch_bounds__(1024) fa_rotary_dw_kernel(const float* __restrict__ part, int D, int q_ctas, int ctas,
                                                            void* dwq, void* dwk, int w_fp32) {
  __shared__ float sums[32][33];
  const int first = blockIdx.y == 0 ? 0 : q_ctas;
  const int last = blockIdx.y == 0 ? q_ctas : ctas;
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int d = blockIdx.x * 32 + lane;
  float v = 0.f;
#pragma unroll 8
  for (int i = first + row; i < last; i += 32) v += part[(long long)i * D + d];
  sums[row][lane] = v;
  __syncthreads();
  v = sums[lane][row];  // warp `row` sums column `row` of the 32
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  if (lane != 0) return;
  void* out = blockIdx.y == 0 ? dwq : dwk;
  const int c = blockIdx.x * 32 + row;
  if (w_fp32)
    static_cast<float*>(out)[c] = v;
  else
    static_cast<uint16_t*>(out)[c] = uint16_t(pack2<DT>(v, 0.f) & 0xffffu);
}

template <int D, int DT, bool INTER, bool APPEND>
int run_fwd(const RotaryArgs& a) {
  const long long per = (a.Hq + HB - 1) / HB + (long long)((a.Hkv + HB - 1) / HB) * (APPEND ? 2 : 1);
  const long long items = per * a.B * a.N;
  constexpr int GROUPS = FWD_THREADS / (D / (2 * FC));
  if (items > 0x7fffffffLL * GROUPS || items + GROUPS > 0xffffffffLL) return FA_ERR_BAD_SHAPE;
  fa_rotary_fwd_kernel<D, DT, INTER, APPEND>
      <<<unsigned((items + GROUPS - 1) / GROUPS), FWD_THREADS, 0, a.stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? FA_OK : FA_ERR_LAUNCH;
}

template <int D, int DT, bool INTER>
int run_bwd(RotaryArgs a) {
  constexpr int GROUPS = BWD_THREADS / (D / (2 * BC));
  const long long rows = (long long)a.B * a.N;
  const long long q_items = rows * ((a.Hq + BWD_HB - 1) / BWD_HB), k_items = rows * ((a.Hkv + BWD_HB - 1) / BWD_HB);
  if (q_items + 4096LL * GROUPS > 0xffffffffLL || k_items + 4096LL * GROUPS > 0xffffffffLL) return FA_ERR_BAD_SHAPE;
  int q_ctas, k_ctas;
  rotary_bwd_ctas(a.Hq, a.Hkv, rows, D, &q_ctas, &k_ctas);
  a.q_ctas = q_ctas;
  fa_rotary_bwd_kernel<D, DT, INTER><<<q_ctas + k_ctas, BWD_THREADS, 0, a.stream>>>(a);
  if (cudaGetLastError() != cudaSuccess) return FA_ERR_LAUNCH;
  if (a.w_part) {
    fa_rotary_dw_kernel<DT><<<dim3(D / 32, 2), 1024, 0, a.stream>>>(a.w_part, D, q_ctas, q_ctas + k_ctas, a.dwq, a.dwk, a.w_fp32);
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
  const long long groups = BWD_THREADS / (D / (2 * BC));
  const long long most = T_BCTAS;
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
