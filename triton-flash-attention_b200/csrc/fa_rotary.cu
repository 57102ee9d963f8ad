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
// Bound: HBM.  A forward moves 4 bytes an element, a backward 6.  D / 2 C
// lanes own a row, each lane C + C of its columns placed so that a lane holds
// both halves of its pairs: the rotation needs no exchange and the mean of
// squares log2(D / 2 C) shuffles.  A warp takes GW = 64 C / D neighbouring
// heads of all tokens of a range, one token a step, so that its weights and
// strides stay in registers and a step adds to its pointers and no more.  At
// D 128 that takes two thirds of the issue slots; forms that worked out a
// token's place or a kind of row at every step had 260 to 305 instructions in
// it and ran out of them first.  Asynchronous copies bring the next steps' rows
// and angles into a ring of the warp's own in shared memory, so that no
// register waits for them.  B2 H32/8 N8191 D128 bf16: forward 58 us (51 of
// HBM), backward 88 with the weights' sums (77); without a norm 57 and 61 (51
// each).  Further from their bytes: D 32 (B4 H32/8 N8191) 39 and 60 us (26 and
// 38), whose copies are 8 bytes a lane, and interleaved pairs (B8 H16 N4097
// D64) 73 and 118 us (41 and 62; halves 50 and 73): a lane's two runs lie beside
// each other there, an access of the warp touches half of every 32 bytes, and
// the memory pipe is what it waits for.
#include "fa_kernels.h"

namespace fa {
namespace {

// A lane's run of C columns in fp32.  (Packed pairs, f32x2, were slower: they
// cost more moves than they save.)
template <int C>
struct Run {
  float v[C];
};
template <int C>
struct Raw {  // the same run in the operand type
  uint32_t u[C / 2];
};

// C elements of a row into shared memory, asynchronously; nothing where !valid.
template <int C>
__device__ __forceinline__ void copy_run(uint32_t saddr, const void* p, bool valid) {
  if (valid) {
    if constexpr (C == 8)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(saddr), "l"(p) : "memory");
    else
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(saddr), "l"(p) : "memory");
  }
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
template <int C>
__device__ __forceinline__ Raw<C> ld_run(uint32_t saddr) {
  Raw<C> r;
  if constexpr (C == 8)
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r.u[0]), "=r"(r.u[1]), "=r"(r.u[2]), "=r"(r.u[3])
                 : "r"(saddr)
                 : "memory");
  else
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r.u[0]), "=r"(r.u[1]) : "r"(saddr) : "memory");
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
    f.v[2 * i] = t.x;
    f.v[2 * i + 1] = t.y;
  }
  return f;
}
template <int DT, int C>
__device__ __forceinline__ Raw<C> narrow(const Run<C>& f) {
  Raw<C> r;
#pragma unroll
  for (int i = 0; i < C / 2; ++i) r.u[i] = pack2<DT>(f.v[2 * i], f.v[2 * i + 1]);
  return r;
}
template <int C>
__device__ __forceinline__ Run<C> fill_run(float v) {
  Run<C> f;
#pragma unroll
  for (int i = 0; i < C; ++i) f.v[i] = v;
  return f;
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

// Cosines and sines of the C pairs of a lane's runs a, b: pair i is (a i, b i),
// or interleaved (a 2 i, a 2 i + 1) and from C / 2 on those of b.
template <int C>
struct Angles {
  Run<C> c, s;
};
// Turns the runs; BACK: the other way.
template <bool INTER, bool BACK, int C>
__device__ __forceinline__ void turn(Run<C>& a, Run<C>& b, const Angles<C>& g) {
#pragma unroll
  for (int i = 0; i < C; ++i) {
    float& x = INTER ? (2 * i < C ? a.v[(2 * i) % C] : b.v[(2 * i) % C]) : a.v[i];
    float& y = INTER ? (2 * i < C ? a.v[(2 * i + 1) % C] : b.v[(2 * i + 1) % C]) : b.v[i];
    const float c = g.c.v[i], s = BACK ? -g.s.v[i] : g.s.v[i];
    const float t = x * c - y * s;
    y = y * c + x * s;
    x = t;
  }
}

// C consecutive weights from column c, in the operand type or fp32.
template <int DT, int C>
__device__ __forceinline__ Run<C> load_w(const void* w, int w_fp32, int c) {
  Run<C> f;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    f.v[i] = w_fp32 ? *(static_cast<const float*>(w) + c + i)
                    : unpack2<DT>(uint32_t(*(static_cast<const uint16_t*>(w) + c + i))).x;
  }
  return f;
}

template <int L>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int m = L / 2; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}
// bf16 rows reach from 2^-133 to 2^128, and their squares past both ends of
// fp32.  A root r = rsqrt(mean(x^2) + eps) below 2^-50 or above 2^50 tells (0
// and infinity do too; NaN stays what it is).  fp16 rows stay within.
template <int DT>
__device__ __forceinline__ bool out_of_range(float r) {
  constexpr uint32_t lo = (127u - 50u) << 23, hi = (127u + 50u) << 23;
  return DT == DT_BF16 && __float_as_uint(r) - lo > hi - lo;
}
// Brings such a row (of a warp's rows those that are; all lanes call) by a power
// of two, 2^-72 or 2^72, to where its squares are normal numbers, with eps
// alike; returns the power.  r becomes the scaled row's.
template <int DT, int D, int L, int C>
__device__ __forceinline__ float bring_in_range(Run<C>& x, Run<C>& y, float& r, float eps) {
  const float k = !out_of_range<DT>(r) ? 1.f : r > 1.f ? 0x1p72f : 0x1p-72f;
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < C; ++j) {
    x.v[j] *= k, y.v[j] *= k;
    ss = fmaf(x.v[j], x.v[j], fmaf(y.v[j], y.v[j], ss));
  }
  r = rsqrtf(group_sum<L>(ss) * (1.f / D) + eps * k * k);
  return k;
}
__device__ __forceinline__ int raw_pos(const RotaryArgs& a, int b, int n) {
  return a.pos ? a.pos[(long long)b * a.pos_sb + n] : n;
}
// The position, or -1 when it has no row in the table: an error (the device
// status is set), but for an appended token without a slot, as those of a
// request are that found no room.
template <bool APPEND>
__device__ __forceinline__ int checked_pos(const RotaryArgs& a, int p, int n) {
  if (p >= 0 && p < a.max_pos) return p;
  if (!(APPEND && a.slots[n] < 0)) refuse_index(a.status, FA_SITE_POSITION);
  return -1;
}
constexpr int THREADS = 128;
constexpr int WARPS = THREADS / 32;
// Steps of a ring and blocks a SM.  Measured at B2 H32/8 N8191 D128 bf16 (HBM
// alone takes 51 and 77 us): forward 4 steps x 5 blocks 58 us, 6 x 4 60, 5 x 6
// 59; backward 3 x 4 85 us, 4 x 4 87, 4 x 3 87 (and 113 with C = 4).
constexpr int FWD_STEPS = 4, FWD_BLOCKS = 5;
// One backward form (D 64, bf16, halves) spills 12 bytes a thread.
constexpr int BWD_STEPS = 3, BWD_BLOCKS = 4;
template <int D>
constexpr int run_cols() {  // C: of narrow rows fewer, so that a step is 8 rows at most
  return D == 32 ? 4 : 8;
}

// A warp's ring of ST steps in shared memory: a step's rows (STREAMS runs a and
// b of 32 lanes) and its token's angles (cosines, sines of a row's lanes).
template <int D, int C, int ST, int STREAMS>
struct Ring {
  static constexpr uint32_t RUN = 2 * C;                    // bytes
  static constexpr uint32_t LANES = D / (2 * C);            // of a row
  static constexpr uint32_t ANGLES = 32 * 2 * RUN * STREAMS;  // where they begin
  static constexpr uint32_t STEP = ANGLES + LANES * 8 * C;
  static constexpr uint32_t BYTES = ST * STEP;
  static_assert(STEP % 16 == 0, "16-byte copies");
};

// Fetches a token's angles, 16 bytes a copy, by the lanes of the first group.
// A position without a row in the table gives NaN.
template <int D, int C>
__device__ __forceinline__ void fetch_angles(const RotaryArgs& a, uint32_t to, int p, int lane) {
  constexpr uint32_t LANES = D / (2 * C);
  if (lane < int(LANES) && lane < a.rd / (2 * C)) {
    const float* t = a.table + (long long)max(p, 0) * a.rd + C * lane;
#pragma unroll
    for (int i = 0; i < C / 4; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {  // cosines, sines
        const uint32_t at = to + uint32_t(j * (C / 4) + i) * (LANES * 16) + lane * 16;
        if (p >= 0)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(at), "l"(t + j * (a.rd / 2) + 4 * i)
                       : "memory");
        else
          st_shared_v4(at, 0x7fc00000u, 0x7fc00000u, 0x7fc00000u, 0x7fc00000u);
      }
  }
}
template <int D, int C>
__device__ __forceinline__ Angles<C> read_angles(uint32_t from, int l) {
  constexpr uint32_t LANES = D / (2 * C);
  Angles<C> g;
#pragma unroll
  for (int i = 0; i < C / 4; ++i) {
    const float4 c = ld_shared_f4(from + uint32_t(i) * (LANES * 16) + l * 16);
    const float4 s = ld_shared_f4(from + uint32_t(C / 4 + i) * (LANES * 16) + l * 16);
    g.c.v[4 * i] = c.x, g.c.v[4 * i + 1] = c.y, g.c.v[4 * i + 2] = c.z, g.c.v[4 * i + 3] = c.w;
    g.s.v[4 * i] = s.x, g.s.v[4 * i + 1] = s.y, g.s.v[4 * i + 2] = s.z, g.s.v[4 * i + 3] = s.w;
  }
  return g;
}

// The tokens of a warp's range, one after the other: where a token's row of
// head h lies in a tensor, and its position.
struct Rows {
  const uint16_t* p;
  long long sn, sb;  // to the next token; from a batch's last token to the next batch's first
  __device__ __forceinline__ Rows(const void* base, const RowStrides& s, int N, int b, int n, int h, int col)
      : p(static_cast<const uint16_t*>(base) + (b * s.b + n * s.n + h * s.h + col)),
        sn(s.n),
        sb(s.b - (N - 1) * s.n) {}
  __device__ __forceinline__ void next(bool batch_ends) { p += batch_ends ? sb : sn; }
};

// Range of a warp: `parts` warps share all tokens for the same heads.
struct Range {
  int count, b, n;
  __device__ __forceinline__ Range(const RotaryArgs& a, int part, int per_part) {
    const long long tokens = (long long)a.B * a.N, first = (long long)part * per_part;
    count = int(min((long long)per_part, tokens - first));
    b = int(first / a.N);
    n = int(first - (long long)b * a.N);
  }
};

// Forward.  Chunks of GW heads: the query's, the key's and -- APPEND -- the
// value's, which are copied as they are; k and v rows go to row slots[n] of
// the caches.  Warps of a block take neighbouring chunks of the same tokens.
template <int D, int DT, bool INTER, bool NORM, bool APPEND>
__global__ void __launch_bounds__(THREADS, FWD_BLOCKS) fa_rotary_fwd_kernel(const __grid_constant__ RotaryArgs a) {
  constexpr int C = run_cols<D>();
  constexpr int L = D / (2 * C);
  constexpr int GW = 32 / L;
  constexpr int ST = FWD_STEPS;
  using R = Ring<D, C, ST, 1>;
  extern __shared__ __align__(16) unsigned char ring[];
  const int lane = threadIdx.x & 31, l = lane % L;
  const uint32_t mem = smem_u32(ring) + (threadIdx.x / 32) * R::BYTES;
  const LaneCols c = lane_cols<INTER, C>(l, a.rd);
  const int ab = c.b - c.a;
  const int q_chunks = (a.Hq + GW - 1) / GW, k_chunks = (a.Hkv + GW - 1) / GW;
  const int chunks = q_chunks + k_chunks * (APPEND ? 2 : 1);
  const int wid = blockIdx.x * WARPS + threadIdx.x / 32;
  const int part = wid / chunks, chunk = wid - part * chunks;
  begin_after_previous();
  if (part >= a.parts) return;
  const int kind = chunk < q_chunks ? 0 : chunk < q_chunks + k_chunks ? 1 : 2;
  const int h = (chunk - (kind == 0 ? 0 : kind == 1 ? q_chunks : q_chunks + k_chunks)) * GW + lane / L;
  const bool valid = h < (kind == 0 ? a.Hq : a.Hkv);
  const Range range(a, part, a.per_part);

  // rows and angles to come: one group of copies a step, empty behind the end
  Rows src(kind == 0 ? a.q : kind == 1 ? a.k : a.v, kind == 0 ? a.qs : kind == 1 ? a.ks : a.vs, a.N, range.b, range.n,
           h, c.a);
  int to_come = range.count, src_b = range.b, src_n = range.n;
  int pos = raw_pos(a, src_b, src_n);
  auto fetch = [&](uint32_t to) {
    if (to_come > 0) {
      copy_run<C>(to + lane * R::RUN, src.p, valid);
      copy_run<C>(to + (32 + lane) * R::RUN, src.p + ab, valid);
      if (!APPEND || kind != 2) fetch_angles<D, C>(a, to + R::ANGLES, checked_pos<APPEND>(a, pos, src_n), lane);
      const bool ends = src_n + 1 == a.N;
      src.next(ends);
      src_n = ends ? 0 : src_n + 1;
      src_b += ends;
      if (--to_come > 0) pos = raw_pos(a, src_b, src_n);
    }
    copies_commit();
  };
#pragma unroll 1
  for (int i = 0; i < ST - 1; ++i) fetch(mem + i * R::STEP);

  const bool cached = APPEND && kind != 0;
  Rows dst(kind == 0 ? a.qo : kind == 1 ? a.ko : a.vo, kind == 0 ? a.qos : a.kos, a.N, cached ? 0 : range.b,
           cached ? 0 : range.n, h, c.a);
  Run<C> wa, wb;
  if (NORM && kind != 2) {
    wa = load_w<DT, C>(kind == 0 ? a.wq : a.wk, a.w_fp32, c.a);
    wb = load_w<DT, C>(kind == 0 ? a.wq : a.wk, a.w_fp32, c.b);
  }
  int slot = cached ? a.slots[range.n] : 0;
  int n = range.n;
  uint32_t here = mem;
  for (int left = range.count; left > 0; --left) {
    copies_wait<ST - 2>();
    __syncwarp();  // the angles were copied by some lanes for all, and those of the step before are read
    Raw<C> ra = ld_run<C>(here + lane * R::RUN), rb = ld_run<C>(here + (32 + lane) * R::RUN);
    if (!APPEND || kind != 2) {
      Run<C> x = widen<DT, C>(ra), y = widen<DT, C>(rb);
      if (NORM) {
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int j = 0; j < C; ++j) s0 = fmaf(x.v[j], x.v[j], s0), s1 = fmaf(y.v[j], y.v[j], s1);
        float r = rsqrtf(group_sum<L>(s0 + s1) * (1.f / D) + a.eps);
        if (__any_sync(0xffffffffu, out_of_range<DT>(r))) bring_in_range<DT, D, L, C>(x, y, r, a.eps);
#pragma unroll
        for (int j = 0; j < C; ++j) x.v[j] *= r * wa.v[j], y.v[j] *= r * wb.v[j];
      }
      if (c.turned) turn<INTER, false, C>(x, y, read_angles<D, C>(here + R::ANGLES, l));
      ra = narrow<DT, C>(x);
      rb = narrow<DT, C>(y);
    }
    if (cached) {
      const bool in = slot >= 0 && slot < a.n_slots;
      if (slot >= a.n_slots) refuse_index(a.status, FA_SITE_SLOT);
      uint16_t* p = const_cast<uint16_t*>(dst.p) + (in ? (long long)slot * (a.Hkv * D) : 0);
      if (valid && in) {
        st_run<C>(p, ra);
        st_run<C>(p + ab, rb);
      }
      if (left > 1) slot = a.slots[++n];
    } else {
      if (valid) {
        st_run<C>(const_cast<uint16_t*>(dst.p), ra);
        st_run<C>(const_cast<uint16_t*>(dst.p) + ab, rb);
      }
      const bool ends = n + 1 == a.N;
      dst.next(ends);
      n = ends ? 0 : n + 1;
    }
    // into the place of the step before, which every lane has read
    fetch(here == mem ? mem + (ST - 1) * R::STEP : here - R::STEP);
    here = here == mem + (ST - 1) * R::STEP ? mem : here + R::STEP;
  }
  copies_wait<0>();
}

// Backward.  The first q_ctas blocks take the query rows, the others the key
// rows, so that a block's weight-gradient sums (2 C fp32 registers a lane) are
// of one weight; it leaves them in w_part[block][D] for the reduction that
// follows.  The sums run in an order that the launch alone decides, so
// gradients repeat bit for bit.
template <int D, int DT, bool INTER, bool NORM>
__global__ void __launch_bounds__(THREADS, BWD_BLOCKS) fa_rotary_bwd_kernel(const __grid_constant__ RotaryArgs a) {
  constexpr int C = run_cols<D>();
  constexpr int L = D / (2 * C);
  constexpr int GW = 32 / L;
  constexpr int ST = BWD_STEPS;
  using R = Ring<D, C, ST, 2>;  // gradients, then rows
  extern __shared__ __align__(16) unsigned char ring[];
  const bool is_q = int(blockIdx.x) < a.q_ctas;
  const int lane = threadIdx.x & 31, l = lane % L;
  const uint32_t mem = smem_u32(ring) + (threadIdx.x / 32) * R::BYTES;
  const LaneCols c = lane_cols<INTER, C>(l, a.rd);
  const int ab = c.b - c.a;
  const int H = is_q ? a.Hq : a.Hkv;
  const int chunks = (H + GW - 1) / GW;
  const int wid = (is_q ? blockIdx.x : blockIdx.x - a.q_ctas) * WARPS + threadIdx.x / 32;
  const int part = wid / chunks, h = (wid - part * chunks) * GW + lane / L;
  const bool valid = h < H;
  const int per_part = is_q ? a.per_part : a.k_per_part;
  Run<C> dwa = fill_run<C>(0.f), dwb = dwa;
  begin_after_previous();
  if (part < (is_q ? a.parts : a.k_parts)) {
    const Range range(a, part, per_part);
    Rows gp(is_q ? a.gq : a.gk, is_q ? a.gqs : a.gks, a.N, range.b, range.n, h, c.a);
    Rows xp(is_q ? a.q : a.k, is_q ? a.qs : a.ks, a.N, range.b, range.n, h, c.a);
    Rows dst(is_q ? a.qo : a.ko, is_q ? a.qos : a.kos, a.N, range.b, range.n, h, c.a);
    int to_come = range.count, src_b = range.b, src_n = range.n;
    int pos = raw_pos(a, src_b, src_n);
    auto fetch = [&](uint32_t to) {
      if (to_come > 0) {
        copy_run<C>(to + lane * R::RUN, gp.p, valid);
        copy_run<C>(to + (32 + lane) * R::RUN, gp.p + ab, valid);
        copy_run<C>(to + (64 + lane) * R::RUN, xp.p, NORM && valid);
        copy_run<C>(to + (96 + lane) * R::RUN, xp.p + ab, NORM && valid);
        fetch_angles<D, C>(a, to + R::ANGLES, checked_pos<false>(a, pos, src_n), lane);
        const bool ends = src_n + 1 == a.N;
        gp.next(ends);
        xp.next(ends);
        src_n = ends ? 0 : src_n + 1;
        src_b += ends;
        if (--to_come > 0) pos = raw_pos(a, src_b, src_n);
      }
      copies_commit();
    };
#pragma unroll 1
    for (int i = 0; i < ST - 1; ++i) fetch(mem + i * R::STEP);
    Run<C> wa, wb;
    if (NORM) {
      wa = load_w<DT, C>(is_q ? a.wq : a.wk, a.w_fp32, c.a);
      wb = load_w<DT, C>(is_q ? a.wq : a.wk, a.w_fp32, c.b);
    }
    int n = range.n;
    uint32_t here = mem;
    for (int left = range.count; left > 0; --left) {
      copies_wait<ST - 2>();
      __syncwarp();
      Run<C> ya = widen<DT, C>(ld_run<C>(here + lane * R::RUN));
      Run<C> yb = widen<DT, C>(ld_run<C>(here + (32 + lane) * R::RUN));
      if (c.turned) turn<INTER, true, C>(ya, yb, read_angles<D, C>(here + R::ANGLES, l));
      if (NORM) {
        Run<C> x = widen<DT, C>(ld_run<C>(here + (64 + lane) * R::RUN));
        Run<C> y = widen<DT, C>(ld_run<C>(here + (96 + lane) * R::RUN));
        float ss = 0.f, gx = 0.f;
        Run<C> ta, tb;  // dy w
#pragma unroll
        for (int j = 0; j < C; ++j) {
          ta.v[j] = ya.v[j] * wa.v[j];
          tb.v[j] = yb.v[j] * wb.v[j];
          ss = fmaf(x.v[j], x.v[j], fmaf(y.v[j], y.v[j], ss));
          gx = fmaf(ta.v[j], x.v[j], fmaf(tb.v[j], y.v[j], gx));
        }
        float r = rsqrtf(group_sum<L>(ss) * (1.f / D) + a.eps);
        float k = 1.f;  // what the row is scaled by, and its gradient then too
        if (__any_sync(0xffffffffu, out_of_range<DT>(r))) {
          k = bring_in_range<DT, D, L, C>(x, y, r, a.eps);
          gx = 0.f;
#pragma unroll
          for (int j = 0; j < C; ++j) gx = fmaf(ta.v[j], x.v[j], fmaf(tb.v[j], y.v[j], gx));
        }
        gx = group_sum<L>(gx);
        const float rk = r * k;
        const float m = -gx * (1.f / D) * r * rk;
#pragma unroll
        for (int j = 0; j < C; ++j) {
          const float xr = x.v[j] * r, yr = y.v[j] * r;
          dwa.v[j] = fmaf(ya.v[j], xr, dwa.v[j]);
          dwb.v[j] = fmaf(yb.v[j], yr, dwb.v[j]);
          ya.v[j] = fmaf(xr, m, ta.v[j] * rk);
          yb.v[j] = fmaf(yr, m, tb.v[j] * rk);
        }
      }
      if (valid) {
        st_run<C>(const_cast<uint16_t*>(dst.p), narrow<DT, C>(ya));
        st_run<C>(const_cast<uint16_t*>(dst.p) + ab, narrow<DT, C>(yb));
      }
      const bool ends = n + 1 == a.N;
      dst.next(ends);
      n = ends ? 0 : n + 1;
      fetch(here == mem ? mem + (ST - 1) * R::STEP : here - R::STEP);
      here = here == mem + (ST - 1) * R::STEP ? mem : here + R::STEP;
    }
    copies_wait<0>();
  }
  if (!NORM || a.w_part == nullptr) return;
  static_assert(WARPS * GW * (D + 4) * 4 <= WARPS * R::BYTES, "the sums reuse the ring");
  float(*sums)[D + 4] = reinterpret_cast<float(*)[D + 4]>(ring);
  __syncthreads();  // every warp is done with its part of the ring
  float* mine = sums[threadIdx.x / L];
#pragma unroll
  for (int j = 0; j < C; ++j) {
    mine[c.a + j] = valid ? dwa.v[j] : 0.f;  // what lanes without a head worked on is nothing
    mine[c.b + j] = valid ? dwb.v[j] : 0.f;
  }
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += THREADS) {
    float s = 0.f;
    for (int r = 0; r < WARPS * GW; ++r) s += sums[r][d];
    a.w_part[(long long)blockIdx.x * D + d] = s;
  }
}

// Weight gradients: block (x, y) sums columns 32 x .. of the query blocks'
// partial sums (y = 0) or the key blocks' (y = 1), 32 rows of them a pass, in
// a fixed order.
template <int DT>
__global__ void __launch_bounds__(1024) fa_rotary_dw_kernel(const float* part, int D, int q_ctas, int ctas,
                                                            void* dwq, void* dwk, int w_fp32) {
  __shared__ float sums[32][33];
  const int first = blockIdx.y == 0 ? 0 : q_ctas;
  const int last = blockIdx.y == 0 ? q_ctas : ctas;
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int d = blockIdx.x * 32 + lane;
  begin_after_previous();
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

// Ranges of tokens for `warps` warps that share `chunks` chunks of heads:
// returns how many, each per_part long.
int cut_tokens(long long tokens, int chunks, long long warps, int* per_part) {
  long long parts = warps / chunks;
  if (parts < 1) parts = 1;
  if (parts > tokens) parts = tokens;
  *per_part = int((tokens + parts - 1) / parts);
  return int((tokens + *per_part - 1) / *per_part);
}

template <int D, int DT, bool INTER, bool NORM, bool APPEND>
int run_fwd(RotaryArgs a) {
  constexpr int GW = 64 * run_cols<D>() / D;
  constexpr int smem = WARPS * Ring<D, run_cols<D>(), FWD_STEPS, 1>::BYTES;
  static_assert(smem <= 48 * 1024, "no larger than any kernel may have");
  const long long tokens = (long long)a.B * a.N, most = (long long)device_sm_count() * FWD_BLOCKS;
  const int chunks = (a.Hq + GW - 1) / GW + (a.Hkv + GW - 1) / GW * (APPEND ? 2 : 1);
  a.parts = cut_tokens(tokens, chunks, most * WARPS, &a.per_part);
  const long long ctas = ((long long)a.parts * chunks + WARPS - 1) / WARPS;
  if (ctas * WARPS > 0x7fffffffLL) return FA_ERR_BAD_SHAPE;
  return launch_early(fa_rotary_fwd_kernel<D, DT, INTER, NORM, APPEND>, dim3(unsigned(ctas)), THREADS, smem, 1, a.stream,
                      a);
}

template <int D, int DT, bool INTER, bool NORM>
int run_bwd(RotaryArgs a) {
  constexpr int GW = 64 * run_cols<D>() / D;
  constexpr int smem = WARPS * Ring<D, run_cols<D>(), BWD_STEPS, 2>::BYTES;
  static_assert(smem <= 48 * 1024, "no larger than any kernel may have");
  // blocks shared between queries and keys by their chunks of heads
  const long long tokens = (long long)a.B * a.N;
  long long most = (long long)device_sm_count() * BWD_BLOCKS;
  if (most > ROTARY_BWD_CTAS) most = ROTARY_BWD_CTAS;
  const int q_chunks = (a.Hq + GW - 1) / GW, k_chunks = (a.Hkv + GW - 1) / GW;
  long long k_most = most * k_chunks / (q_chunks + k_chunks);
  if (k_most < 1) k_most = 1;
  a.parts = cut_tokens(tokens, q_chunks, (most - k_most) * WARPS, &a.per_part);
  a.k_parts = cut_tokens(tokens, k_chunks, k_most * WARPS, &a.k_per_part);
  const long long q_ctas = ((long long)a.parts * q_chunks + WARPS - 1) / WARPS;
  const long long k_ctas = ((long long)a.k_parts * k_chunks + WARPS - 1) / WARPS;
  // thousands of heads: more chunks than warps, which would take more rows of
  // w_part than there are
  if (q_ctas + k_ctas > ROTARY_BWD_CTAS) return FA_ERR_BAD_SHAPE;
  a.q_ctas = int(q_ctas);
  if (int rc = launch_early(fa_rotary_bwd_kernel<D, DT, INTER, NORM>, dim3(unsigned(q_ctas + k_ctas)), THREADS, smem, 1,
                            a.stream, a))
    return rc;
  if (!a.w_part) return FA_OK;
  return launch_early(fa_rotary_dw_kernel<DT>, dim3(D / 32, 2), 1024, 0, 1, a.stream, (const float*)a.w_part, D,
                      int(q_ctas), int(q_ctas + k_ctas), a.dwq, a.dwk, a.w_fp32);
}

// Instantiated for the head dims, operand types, pairings and with and
// without a norm.
enum class Op { kForward, kBackward, kAppend };
template <Op OP, int D, int DT, bool INTER, bool NORM>
int run(const RotaryArgs& a) {
  if constexpr (OP == Op::kBackward) return run_bwd<D, DT, INTER, NORM>(a);
  else return run_fwd<D, DT, INTER, NORM, OP == Op::kAppend>(a);
}
template <Op OP, int D, int DT>
int by_form(const RotaryArgs& a) {
  if (a.wq) return a.interleaved ? run<OP, D, DT, true, true>(a) : run<OP, D, DT, false, true>(a);
  return a.interleaved ? run<OP, D, DT, true, false>(a) : run<OP, D, DT, false, false>(a);
}
template <Op OP>
int by_type(const RotaryArgs& a, int D) {
  if (a.dtype == DT_BF16)
    return D == 32 ? by_form<OP, 32, DT_BF16>(a) : D == 64 ? by_form<OP, 64, DT_BF16>(a) : by_form<OP, 128, DT_BF16>(a);
  return D == 32 ? by_form<OP, 32, DT_F16>(a) : D == 64 ? by_form<OP, 64, DT_F16>(a) : by_form<OP, 128, DT_F16>(a);
}

}  // namespace

int launch_rotary_fwd(const RotaryArgs& a, int D) { return by_type<Op::kForward>(a, D); }
int launch_rotary_bwd(const RotaryArgs& a, int D) { return by_type<Op::kBackward>(a, D); }
int launch_paged_append(const RotaryArgs& a, int D) { return by_type<Op::kAppend>(a, D); }

}  // namespace fa
