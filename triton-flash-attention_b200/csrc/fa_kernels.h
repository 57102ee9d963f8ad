// fa_kernels.h -- internal launch interface between the C ABI (fa_capi.cu)
// and the kernel translation units.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <cuda_fp16.h>

#include "../../include/fa_b200.h"
#include "fa_common.cuh"
#include "fa_status.h"

namespace fa {

// Operand element types (dtype fields below).
enum : int { DT_F16 = 0, DT_BF16 = 1 };

struct FwdArgs {
  CUtensorMap tmap_q, tmap_k, tmap_v;  // 4-D {D, N, H, B}, box {<=64, 128, 1, 1}
  AttnShape shape;
  int dtype;  // DT_F16 or DT_BF16: q, k, v and o
  void* o;
  long long o_sb, o_sh, o_sn;
  float* lse;
  MaskBits mask;  // dense boolean mask (bits == nullptr: none)
  DropArgs drop;  // attention dropout (t == 0: none)
  SplitArgs split;  // split-KV partial outputs (n == 1: none)
  cudaStream_t stream;
};

struct BwdArgs {
  CUtensorMap tmap_q, tmap_k, tmap_v, tmap_do;  // 4-D maps of the operand type
  AttnShape shape;
  int dtype;  // DT_F16 or DT_BF16: q, k, v, dO and the non-fp32 outputs
  const float* lse;
  const float* delta;
  void* dq;  // fa_bwd_dq output (operand type, or fp32 when accumulate_fp32)
  long long dq_sb, dq_sh, dq_sn;
  void* dk;
  void* dv;
  long long dk_sb, dk_sh, dk_sn;
  long long dv_sb, dv_sh, dv_sn;
  int accumulate_fp32;
  MaskBits mask;  // dense boolean mask (bits == nullptr: none)
  DropArgs drop;  // attention dropout (t == 0: none)
  cudaStream_t stream;
};

// Number of SMs of the current device (cached per device); persistent
// kernels launch at most one CTA per SM.
inline int device_sm_count() {
  static int cache[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (cache[dev] == 0) {
    int n = 0;
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    cache[dev] = n > 0 ? n : 148;
  }
  return cache[dev];
}

// The text of the CUDA runtime error behind the last FA_ERR_CUDA status
// (cudaGetErrorString's static string), for fa_status_string.
void record_cuda_error(cudaError_t e);
const char* last_cuda_error_text();

int launch_fwd(const FwdArgs& a, int D);
int launch_bwd_dq(const BwdArgs& a, int D);
int launch_bwd_dkdv(const BwdArgs& a, int D);
// zero_acc: when not null, the contiguous [B, H, N, D] fp32 buffer is zeroed
// on the way (the fused backward's dQ accumulator).
int launch_bwd_delta(const void* o, long long o_sb, long long o_sh, long long o_sn, const void* dO,
                     long long do_sb, long long do_sh, long long do_sn, float* delta, float* zero_acc, int B, int H,
                     int N, int D, int dtype, cudaStream_t stream);
// Fused dK/dV + dQ backward (every D; D = 128 runs fa_bwd_fused128.cu, with
// no boolean mask or dropout).  The fp32 dQ accumulator is a.dq; the D = 128
// kernel reduce-adds into it through tmap_dq, the D <= 64 kernels add into it
// directly (tmap_dq unused).
int launch_bwd_fused(const BwdArgs& a, const CUtensorMap& tmap_dq, int D);
int launch_bwd_fused128(const BwdArgs& a, const CUtensorMap& tmap_dq);
// acc_w: the accumulator's row width (0: D); dq receives its first D columns.
int launch_dq_convert(const float* acc, void* dq, long long sb, long long sh, long long sn, int B, int H, int N, int D,
                      int dtype, cudaStream_t stream, int acc_w = 0);
// Dense boolean mask (bytes, element strides {sb, sh, sq, sk}, Bm x Hm x Nq x
// Nk) -> bits (Bm, Hm, Nq, roundup(Nk, 128) / 32) and bits_t (Bm, Hm, Nk,
// roundup(Nq, 128) / 32) uint32 words, contiguous.
int launch_mask_pack(const void* mask, long long sb, long long sh, long long sq, long long sk, int Bm, int Hm, int Nq,
                     int Nk, uint32_t* bits, uint32_t* bits_t, cudaStream_t stream);
int launch_combine_splits(const void* o_part, const float* lse_part, void* o, float* lse, int S, int total_q, int H,
                          int D, int dtype, cudaStream_t stream);
int launch_merge_partial(float* o_acc, float* lse_acc, const void* o_part, const float* lse_part, long long rows,
                         int D, int dtype, cudaStream_t stream);

// ---------------------------------------------------------------------------
// Query/key preparation and the paged cache (fa_rotary.cu, fa_tables.cu,
// fa_sparse.cu; no counterpart in the reference).

// Sites of FA_ERR_BAD_INDEX in the device status (bits 8..15 of its word): a
// position, a slot, a page or a length that a kernel refused.
enum : int { FA_SITE_POSITION = 224, FA_SITE_SLOT = 225, FA_SITE_PAGE = 226 };
__device__ __forceinline__ void refuse_index(int* status, int site) {
  if (status) atomicCAS(status + STATUS_REFUSED, 0, (site << 8) | FA_ERR_BAD_INDEX);
}

struct RowStrides {
  long long b, h, n;  // elements
};
// Norm and rotation of query and key rows (B batches x N tokens x heads).
struct RotaryArgs {
  const void *q, *k, *v;  // v: append only
  RowStrides qs, ks, vs;
  const void *gq, *gk;  // backward: gradients of the outputs
  RowStrides gqs, gks;
  void *qo, *ko, *vo;  // outputs; append: packed q, k cache, v cache
  RowStrides qos, kos;
  const float* table;  // (max_pos, rd): cosines, then sines
  const int* pos;      // nullptr: the token's index
  long long pos_sb;
  const int* slots;  // append: a cache row for each token, -1 for none
  const void *wq, *wk;  // nullptr: no norm
  void *dwq, *dwk;
  float* w_part;  // (ROTARY_BWD_CTAS, D) partial weight gradients
  float eps;
  int max_pos, rd, interleaved, w_fp32, n_slots;
  int B, N, Hq, Hkv, dtype;
  // set by the launches: ranges of tokens and their length (backward: the query
  // rows' and the key rows'), blocks of the query rows
  int parts, per_part, k_parts, k_per_part, q_ctas;
  int* status;
  cudaStream_t stream;
};
constexpr int ROTARY_BWD_CTAS = FA_ROTARY_PARTIALS;
int launch_rotary_fwd(const RotaryArgs& a, int D);
int launch_rotary_bwd(const RotaryArgs& a, int D);
int launch_paged_append(const RotaryArgs& a, int D);

struct TableArgs {
  int* table;  // (requests, width)
  const int *cached, *fresh;
  const int *free_pages, *free_start;
  int *cu, *seqlens, *pos, *slots;
  unsigned char* fits;
  int* free_next;
  int requests, width, n_free, page_log2, total;
  cudaStream_t stream;
};
int launch_extend_table(const TableArgs& a);

struct PageArgs {
  const void* k_cache;
  void* means;  // (num_pages, Hkv, D)
  const int *table, *cu, *seqlens;
  int B, Hkv, D, num_pages, page_log2, width, dtype;
  int* status;
  cudaStream_t stream;
};
int launch_page_means(const PageArgs& a, int total_q);

struct SelectArgs {
  const void *q, *means;
  long long q_sh, q_st;  // element strides of heads and rows
  const int *table, *cu, *seqlens;
  int* out;  // (total_q, Hkv, top)
  int B, Hq, Hkv, total_q, num_pages, page_log2, width, top, sink, local, dtype;
  int cluster;  // set by the launch
  int* status;
  cudaStream_t stream;
};
int launch_select_pages(SelectArgs a, int D);

struct SparseArgs {
  const void* q;
  void* o;
  long long q_sh, q_st;
  const int *table, *cu, *seqlens, *idx;
  int B, Hq, Hkv, total_q, num_pages, page_log2, width, top, dtype;
  int cluster;  // set by the launch
  float scale_log2;
  int* status;
  cudaStream_t stream;
};
int launch_sparse_decode(SparseArgs a, const CUtensorMap& k, const CUtensorMap& v, int D);

// The kernels above may come onto the GPU while the kernel before them on the
// stream is still ending (programmatic dependent launch): that hides 1 to 3 us
// of a launch.  Each calls begin_after_previous(), in every thread and before
// it reads or writes any global memory: it waits until all earlier kernels of
// the stream are done and their writes are seen.  (Their loads are plain ones:
// read-only loads, __ldg and __restrict__ to const, promise data that nobody
// writes while the kernel lives, which starts before that wait.)
__device__ __forceinline__ void begin_after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// Lets the stream's next kernel come on once every block has called it, not
// when the last one has ended.  The kernels of a serving step call it at once
// (sparse attention over 16 x 8192 tokens 28.7 -> 26.8 us).  The rotary ones do
// not: their blocks fill the GPU for a long time, the next kernel's first
// blocks then sit where there happens to be room, and a forward and backward
// pass over 8192 tokens took 213 us instead of 156.
__device__ __forceinline__ void let_next_begin() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
// Such a launch, in clusters of S blocks (1: none).
template <class... Params, class... Args>
int launch_early(void (*kernel)(Params...), dim3 blocks, unsigned threads, size_t smem, int S, cudaStream_t stream,
                 const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = blocks;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = unsigned(S);
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = S > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? FA_OK : FA_ERR_LAUNCH;
}

// The device status words, and a tensor map over a (num_pages, page_size, Hkv,
// D) cache whose box is `rows` rows of one head, all D columns: dimensions
// {min(D, 64) columns, cache rows, D / 64 runs of columns, heads}, so that one
// copy leaves a row's runs of 64 columns behind each other (fa_capi.cu).
int* device_status_words();
int make_cache_map(CUtensorMap* map, const void* cache, int cache_rows, int Hkv, int D, int rows, int dtype);

// Query-tile / key-tile sizes the host needs for TMA box shapes.
namespace dq_cfg {
constexpr int BM = 128;  // query rows per tile
constexpr int BN = 128;  // keys per key tile
}  // namespace dq_cfg
namespace dkdv_cfg {
constexpr int BM = 128;  // key rows per tile (the MMA M dimension)
constexpr int BQ = 64;   // query rows per tile (D = 128)
constexpr int BQ_WIDE = 128;  // query rows per item (D <= 64)
}  // namespace dkdv_cfg
// Query rows per item of the fused backward (its Q / dO tensor-map boxes).
constexpr int fused_item_rows(int D) { return D <= 64 ? dkdv_cfg::BQ_WIDE : dkdv_cfg::BQ; }

}  // namespace fa
