// fa_serving_capi.cu -- extern "C" entries of the query/key preparation and of
// the paged cache's tables, appends and page-sparse attention
// (include/fa_b200.h).  As in fa_capi.cu: arguments are checked before any
// CUDA call, nothing is thrown, and every entry returns an FA_ERR_* code.
#include <cmath>
#include <cstring>
#include <tuple>
#include <type_traits>
#include <utility>

#include "fa_kernels.h"

namespace fa {
namespace {

bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
bool head_dim_ok(int D) { return D == 32 || D == 64 || D == 128; }

// log2 of a page size, or -1 when it is not a power of two of at least 16
int page_log2(int page_size) {
  if (page_size < 16 || (page_size & (page_size - 1)) != 0) return -1;
  int l = 0;
  while ((1 << l) < page_size) ++l;
  return l;
}

// 16-byte loads of rows: the pointer and every stride; zero strides are for inputs.
bool rows_ok(const void* p, const int64_t* s, bool input) {
  if (!aligned(p, 16)) return false;
  for (int i = 0; i < 3; ++i)
    if (s[i] < 0 || s[i] % 8 != 0 || (!input && s[i] == 0)) return false;
  return true;
}
RowStrides strides(const int64_t* s) { return RowStrides{s[0], s[1], s[2]}; }

int rotary_common(RotaryArgs* a, const float* table, const int* positions, const void* wq, const void* wk, int B,
                  int Hq, int Hkv, int N, int D, int max_positions, int rd, int interleaved, int w_fp32,
                  int64_t pos_batch_stride, float eps, void* stream, int dtype) {
  if (!head_dim_ok(D)) return FA_ERR_UNSUPPORTED_HEAD_DIM;
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || N <= 0 || max_positions <= 0) return FA_ERR_BAD_SHAPE;
  if ((long long)B * N > 0x7fffffffLL || pos_batch_stride < 0) return FA_ERR_BAD_SHAPE;
  if (rd <= 0 || rd > D || rd % 16 != 0 || !table) return FA_ERR_BAD_SHAPE;
  if ((wq == nullptr) != (wk == nullptr) || !std::isfinite(eps) || eps < 0.f) return FA_ERR_BAD_SHAPE;
  if (!aligned(table, 16)) return FA_ERR_MISALIGNED;
  *a = RotaryArgs{};
  a->table = table;
  a->pos = positions;
  a->pos_sb = pos_batch_stride;
  a->wq = wq;
  a->wk = wk;
  a->eps = eps;
  a->max_pos = max_positions;
  a->rd = rd;
  a->interleaved = interleaved ? 1 : 0;
  a->w_fp32 = w_fp32 ? 1 : 0;
  a->B = B;
  a->N = N;
  a->Hq = Hq;
  a->Hkv = Hkv;
  a->dtype = dtype;
  a->status = device_status_words();
  a->stream = static_cast<cudaStream_t>(stream);
  return FA_OK;
}

int rotary_fwd_impl(const void* q, const void* k, void* q_out, void* k_out, const float* table, const int* positions,
                    const void* wq, const void* wk, int B, int Hq, int Hkv, int N, int D, int max_positions, int rd,
                    int interleaved, int w_fp32, const int64_t* qs, const int64_t* ks, const int64_t* qos,
                    const int64_t* kos, int64_t pos_sb, float eps, void* stream, int dtype) {
  if (!q || !k || !q_out || !k_out || !qs || !ks || !qos || !kos) return FA_ERR_BAD_SHAPE;
  RotaryArgs a;
  if (int rc = rotary_common(&a, table, positions, wq, wk, B, Hq, Hkv, N, D, max_positions, rd, interleaved, w_fp32,
                             pos_sb, eps, stream, dtype))
    return rc;
  if (!rows_ok(q, qs, true) || !rows_ok(k, ks, true) || !rows_ok(q_out, qos, false) || !rows_ok(k_out, kos, false))
    return FA_ERR_MISALIGNED;
  a.q = q;
  a.k = k;
  a.qs = strides(qs);
  a.ks = strides(ks);
  a.qo = q_out;
  a.ko = k_out;
  a.qos = strides(qos);
  a.kos = strides(kos);
  return launch_rotary_fwd(a, D);
}

int rotary_bwd_impl(const void* q, const void* k, const void* gq, const void* gk, void* dq, void* dk, void* dwq,
                    void* dwk, float* w_part, const float* table, const int* positions, const void* wq,
                    const void* wk, int B, int Hq, int Hkv, int N, int D, int max_positions, int rd, int interleaved,
                    int w_fp32, const int64_t* qs, const int64_t* ks, const int64_t* gqs, const int64_t* gks,
                    const int64_t* dqs, const int64_t* dks, int64_t pos_sb, float eps, void* stream, int dtype) {
  if (!q || !k || !gq || !gk || !dq || !dk || !qs || !ks || !gqs || !gks || !dqs || !dks) return FA_ERR_BAD_SHAPE;
  if ((dwq == nullptr) != (dwk == nullptr) || (dwq && (!w_part || !wq))) return FA_ERR_BAD_SHAPE;
  RotaryArgs a;
  if (int rc = rotary_common(&a, table, positions, wq, wk, B, Hq, Hkv, N, D, max_positions, rd, interleaved, w_fp32,
                             pos_sb, eps, stream, dtype))
    return rc;
  if (!rows_ok(q, qs, true) || !rows_ok(k, ks, true) || !rows_ok(gq, gqs, true) || !rows_ok(gk, gks, true) ||
      !rows_ok(dq, dqs, false) || !rows_ok(dk, dks, false))
    return FA_ERR_MISALIGNED;
  a.q = q;
  a.k = k;
  a.qs = strides(qs);
  a.ks = strides(ks);
  a.gq = gq;
  a.gk = gk;
  a.gqs = strides(gqs);
  a.gks = strides(gks);
  a.qo = dq;
  a.ko = dk;
  a.qos = strides(dqs);
  a.kos = strides(dks);
  a.dwq = dwq;
  a.dwk = dwk;
  a.w_part = dwq ? w_part : nullptr;
  return launch_rotary_bwd(a, D);
}

int append_impl(const void* q, const void* k, const void* v, void* q_out, void* k_cache, void* v_cache,
                const int* slots, const float* table, const int* positions, const void* wq, const void* wk, int total,
                int Hq, int Hkv, int D, int num_slots, int max_positions, int rd, int interleaved, int w_fp32,
                const int64_t* qs, const int64_t* ks, const int64_t* vs, float eps, void* stream, int dtype) {
  if (!q || !k || !v || !q_out || !k_cache || !v_cache || !slots || !positions || !qs || !ks || !vs || num_slots <= 0)
    return FA_ERR_BAD_SHAPE;
  RotaryArgs a;
  if (int rc = rotary_common(&a, table, positions, wq, wk, 1, Hq, Hkv, total, D, max_positions, rd, interleaved,
                             w_fp32, 0, eps, stream, dtype))
    return rc;
  if (!rows_ok(q, qs, true) || !rows_ok(k, ks, true) || !rows_ok(v, vs, true) || !aligned(q_out, 16) ||
      !aligned(k_cache, 16) || !aligned(v_cache, 16))
    return FA_ERR_MISALIGNED;
  a.q = q;
  a.k = k;
  a.v = v;
  a.qs = strides(qs);
  a.ks = strides(ks);
  a.vs = strides(vs);
  a.qo = q_out;
  a.qos = RowStrides{0, D, (long long)Hq * D};
  a.kos = RowStrides{0, D, (long long)Hkv * D};  // of a cache's rows
  a.ko = k_cache;
  a.vo = v_cache;
  a.slots = slots;
  a.n_slots = num_slots;
  return launch_paged_append(a, D);
}

int means_impl(const void* k_cache, void* means, const int* table, const int* cu, const int* seqlens, int B, int Hkv,
               int D, int num_pages, int page_size, int width, int total_q, void* stream, int dtype) {
  if (!head_dim_ok(D)) return FA_ERR_UNSUPPORTED_HEAD_DIM;
  const int pl = page_log2(page_size);
  if (pl < 0 || B <= 0 || Hkv <= 0 || num_pages <= 0 || width <= 0 || total_q <= 0) return FA_ERR_BAD_SHAPE;
  if ((long long)num_pages * page_size > 0x7fffffffLL || (long long)width * page_size > 0x7fffffffLL)
    return FA_ERR_BAD_SHAPE;
  if (!k_cache || !means || !table || !cu || !seqlens) return FA_ERR_BAD_SHAPE;
  if (!aligned(k_cache, 16) || !aligned(means, 16)) return FA_ERR_MISALIGNED;
  PageArgs a{};
  a.k_cache = k_cache;
  a.means = means;
  a.table = table;
  a.cu = cu;
  a.seqlens = seqlens;
  a.B = B;
  a.Hkv = Hkv;
  a.D = D;
  a.num_pages = num_pages;
  a.page_log2 = pl;
  a.width = width;
  a.dtype = dtype;
  a.status = device_status_words();
  a.stream = static_cast<cudaStream_t>(stream);
  return launch_page_means(a, total_q);
}

int sparse_shape(int B, int Hq, int Hkv, int D, int total_q, int num_pages, int page_size, int width, int top) {
  if (!head_dim_ok(D)) return FA_ERR_UNSUPPORTED_HEAD_DIM;
  if (page_log2(page_size) < 0 || B <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || total_q <= 0 || num_pages <= 0 ||
      width <= 0 || top <= 0)
    return FA_ERR_BAD_SHAPE;
  if ((long long)num_pages * page_size > 0x7fffffffLL || (long long)width * page_size > 0x7fffffffLL ||
      (long long)top * page_size > 0x3fffffffLL)
    return FA_ERR_BAD_SHAPE;
  return FA_OK;
}

int select_impl(const void* q, const void* means, const int* table, const int* cu, const int* seqlens, int* selected,
                int B, int Hq, int Hkv, int D, int total_q, int num_pages, int page_size, int width, int top, int sink,
                int local, const int64_t* qs, void* stream, int dtype) {
  if (int rc = sparse_shape(B, Hq, Hkv, D, total_q, num_pages, page_size, width, top)) return rc;
  if (width > FA_MAX_SELECT_PAGES || sink < 0 || local < 1 || sink > top || local > top - sink) return FA_ERR_BAD_SHAPE;
  if (!q || !means || !table || !cu || !seqlens || !selected || !qs) return FA_ERR_BAD_SHAPE;
  if (!rows_ok(q, qs, true) || !aligned(means, 16)) return FA_ERR_MISALIGNED;
  SelectArgs a{};
  a.q = q;
  a.means = means;
  a.q_sh = qs[1];
  a.q_st = qs[2];
  a.table = table;
  a.cu = cu;
  a.seqlens = seqlens;
  a.out = selected;
  a.B = B;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.total_q = total_q;
  a.num_pages = num_pages;
  a.page_log2 = page_log2(page_size);
  a.width = width;
  a.top = top;
  a.sink = sink;
  a.local = local;
  a.dtype = dtype;
  a.status = device_status_words();
  a.stream = static_cast<cudaStream_t>(stream);
  return launch_select_pages(a, D);
}

int sparse_impl(const void* q, const void* k_cache, const void* v_cache, void* o, const int* table, const int* cu,
                const int* seqlens, const int* pages, int B, int Hq, int Hkv, int D, int total_q, int num_pages,
                int page_size, int width, int top, float softmax_scale, const int64_t* qs, void* stream, int dtype) {
  if (int rc = sparse_shape(B, Hq, Hkv, D, total_q, num_pages, page_size, width, top)) return rc;
  if (!q || !k_cache || !v_cache || !o || !table || !cu || !seqlens || !pages || !qs) return FA_ERR_BAD_SHAPE;
  if (!std::isfinite(softmax_scale)) return FA_ERR_BAD_SHAPE;
  if (!rows_ok(q, qs, true) || !aligned(o, 16)) return FA_ERR_MISALIGNED;
  SparseArgs a{};
  CUtensorMap mk, mv;
  const int rows = page_size < 64 ? page_size : 64;
  if (int rc = make_cache_map(&mk, k_cache, num_pages * page_size, Hkv, D, rows, dtype)) return rc;
  if (int rc = make_cache_map(&mv, v_cache, num_pages * page_size, Hkv, D, rows, dtype)) return rc;
  a.q = q;
  a.o = o;
  a.q_sh = qs[1];
  a.q_st = qs[2];
  a.table = table;
  a.cu = cu;
  a.seqlens = seqlens;
  a.idx = pages;
  a.B = B;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.total_q = total_q;
  a.num_pages = num_pages;
  a.page_log2 = page_log2(page_size);
  a.width = width;
  a.top = top;
  a.dtype = dtype;
  a.scale_log2 = float(double(softmax_scale) * 1.4426950408889634);
  a.status = device_status_words();
  a.stream = static_cast<cudaStream_t>(stream);
  return launch_sparse_decode(a, mk, mv, D);
}

}  // namespace
}  // namespace fa

using namespace fa;

#define FA_ROTARY_FWD(NAME, DTYPE)                                                                                    \
  extern "C" int NAME(const void* q, const void* k, void* q_out, void* k_out, const float* table,                    \
                      const int* positions, const void* wq, const void* wk, int B, int Hq, int Hkv, int N, int D,     \
                      int max_positions, int rotary_dim, int interleaved, int w_fp32, const int64_t* q_strides,       \
                      const int64_t* k_strides, const int64_t* qo_strides, const int64_t* ko_strides,                 \
                      int64_t pos_batch_stride, float eps, void* stream) {                                            \
    return rotary_fwd_impl(q, k, q_out, k_out, table, positions, wq, wk, B, Hq, Hkv, N, D, max_positions, rotary_dim, \
                           interleaved, w_fp32, q_strides, k_strides, qo_strides, ko_strides, pos_batch_stride, eps,  \
                           stream, DTYPE);                                                                            \
  }
FA_ROTARY_FWD(fa_qk_norm_rotary, DT_F16)
FA_ROTARY_FWD(fa_qk_norm_rotary_bf16, DT_BF16)

#define FA_ROTARY_BWD(NAME, DTYPE)                                                                                   \
  extern "C" int NAME(const void* q, const void* k, const void* gq, const void* gk, void* dq, void* dk, void* dwq,   \
                      void* dwk, float* w_part, const float* table, const int* positions, const void* wq,            \
                      const void* wk, int B, int Hq, int Hkv, int N, int D, int max_positions, int rotary_dim,       \
                      int interleaved, int w_fp32, const int64_t* q_strides, const int64_t* k_strides,               \
                      const int64_t* gq_strides, const int64_t* gk_strides, const int64_t* dq_strides,               \
                      const int64_t* dk_strides, int64_t pos_batch_stride, float eps, void* stream) {                \
    return rotary_bwd_impl(q, k, gq, gk, dq, dk, dwq, dwk, w_part, table, positions, wq, wk, B, Hq, Hkv, N, D,       \
                           max_positions, rotary_dim, interleaved, w_fp32, q_strides, k_strides, gq_strides,         \
                           gk_strides, dq_strides, dk_strides, pos_batch_stride, eps, stream, DTYPE);                \
  }
FA_ROTARY_BWD(fa_qk_norm_rotary_bwd, DT_F16)
FA_ROTARY_BWD(fa_qk_norm_rotary_bwd_bf16, DT_BF16)

#define FA_APPEND(NAME, DTYPE)                                                                                     \
  extern "C" int NAME(const void* q, const void* k, const void* v, void* q_out, void* k_cache, void* v_cache,      \
                      const int* slots, const float* table, const int* positions, const void* wq, const void* wk,  \
                      int total, int Hq, int Hkv, int D, int num_slots, int max_positions, int rotary_dim,         \
                      int interleaved, int w_fp32, const int64_t* q_strides, const int64_t* k_strides,             \
                      const int64_t* v_strides, float eps, void* stream) {                                         \
    return append_impl(q, k, v, q_out, k_cache, v_cache, slots, table, positions, wq, wk, total, Hq, Hkv, D,       \
                       num_slots, max_positions, rotary_dim, interleaved, w_fp32, q_strides, k_strides, v_strides, \
                       eps, stream, DTYPE);                                                                        \
  }
FA_APPEND(fa_paged_append, DT_F16)
FA_APPEND(fa_paged_append_bf16, DT_BF16)

extern "C" int fa_extend_block_table(int* block_table, const int* cached, const int* fresh, const int* free_pages,
                                     const int* free_start, int* cu_seqlens_q, int* seqlens_k, int* positions,
                                     int* slots, uint8_t* fits, int* free_next, int requests, int max_pages,
                                     int n_free, int page_size, int total_q, void* stream) {
  const int pl = page_log2(page_size);
  if (pl < 0 || requests <= 0 || max_pages <= 0 || n_free < 0 || total_q < 0) return FA_ERR_BAD_SHAPE;
  if ((long long)max_pages * page_size > 0x7fffffffLL) return FA_ERR_BAD_SHAPE;
  if (!block_table || !cached || !fresh || !free_start || !cu_seqlens_q || !seqlens_k || !fits || !free_next ||
      (n_free > 0 && !free_pages) || (total_q > 0 && (!positions || !slots)))
    return FA_ERR_BAD_SHAPE;
  TableArgs a{};
  a.table = block_table;
  a.cached = cached;
  a.fresh = fresh;
  a.free_pages = free_pages;
  a.free_start = free_start;
  a.cu = cu_seqlens_q;
  a.seqlens = seqlens_k;
  a.pos = positions;
  a.slots = slots;
  a.fits = fits;
  a.free_next = free_next;
  a.requests = requests;
  a.width = max_pages;
  a.n_free = n_free;
  a.page_log2 = pl;
  a.total = total_q;
  a.stream = static_cast<cudaStream_t>(stream);
  return launch_extend_table(a);
}

#define FA_MEANS(NAME, DTYPE)                                                                                       \
  extern "C" int NAME(const void* k_cache, void* page_means, const int* block_table, const int* cu_seqlens_q,       \
                      const int* seqlens_k, int B, int Hkv, int D, int num_pages, int page_size,                    \
                      int max_pages_per_seq, int total_q, void* stream) {                                           \
    return means_impl(k_cache, page_means, block_table, cu_seqlens_q, seqlens_k, B, Hkv, D, num_pages, page_size,   \
                      max_pages_per_seq, total_q, stream, DTYPE);                                                   \
  }
FA_MEANS(fa_page_means, DT_F16)
FA_MEANS(fa_page_means_bf16, DT_BF16)

#define FA_SELECT(NAME, DTYPE)                                                                                       \
  extern "C" int NAME(const void* q, const void* page_means, const int* block_table, const int* cu_seqlens_q,        \
                      const int* seqlens_k, int* selected, int B, int Hq, int Hkv, int D, int total_q,               \
                      int num_pages, int page_size, int max_pages_per_seq, int top, int sink, int local,             \
                      const int64_t* q_strides, void* stream) {                                                      \
    return select_impl(q, page_means, block_table, cu_seqlens_q, seqlens_k, selected, B, Hq, Hkv, D, total_q,        \
                       num_pages, page_size, max_pages_per_seq, top, sink, local, q_strides, stream, DTYPE);         \
  }
FA_SELECT(fa_select_pages, DT_F16)
FA_SELECT(fa_select_pages_bf16, DT_BF16)

#define FA_SPARSE(NAME, DTYPE)                                                                                    \
  extern "C" int NAME(const void* q, const void* k_cache, const void* v_cache, void* o, const int* block_table,   \
                      const int* cu_seqlens_q, const int* seqlens_k, const int* pages, int B, int Hq, int Hkv,    \
                      int D, int total_q, int num_pages, int page_size, int max_pages_per_seq, int top,           \
                      float softmax_scale, const int64_t* q_strides, void* stream) {                              \
    return sparse_impl(q, k_cache, v_cache, o, block_table, cu_seqlens_q, seqlens_k, pages, B, Hq, Hkv, D,        \
                       total_q, num_pages, page_size, max_pages_per_seq, top, softmax_scale, q_strides, stream,   \
                       DTYPE);                                                                                    \
  }
FA_SPARSE(fa_fwd_paged_sparse, DT_F16)
FA_SPARSE(fa_fwd_paged_sparse_bf16, DT_BF16)

namespace fa {
namespace {

// One argument from its 8-byte word; an int that is none clears ok.
template <class T>
T from_word(uint64_t w, bool* ok) {
  if constexpr (std::is_pointer_v<T>) {
    return reinterpret_cast<T>(uintptr_t(w));
  } else if constexpr (std::is_same_v<T, float>) {
    double d;
    std::memcpy(&d, &w, sizeof d);
    return float(d);
  } else {
    const int64_t v = int64_t(w);
    if (int64_t(T(v)) != v) *ok = false;
    return T(v);
  }
}
template <class... A, size_t... I>
int call_words(int (*fn)(A...), const void* words, std::index_sequence<I...>) {
  if (!words) return FA_ERR_BAD_SHAPE;
  uint64_t w[sizeof...(A)];
  std::memcpy(w, words, sizeof w);
  bool ok = true;
  const std::tuple<A...> args{from_word<A>(w[I], &ok)...};
  return ok ? fn(std::get<I>(args)...) : FA_ERR_BAD_SHAPE;
}
template <class... A>
constexpr std::index_sequence_for<A...> indices(int (*)(A...)) {
  return {};
}
template <auto* Fn>
int packed(const void* words) {
  return call_words(Fn, words, indices(Fn));
}

#define FA_PACKED(NAME) {#NAME, packed<&NAME>}
#define FA_PACKED2(NAME) FA_PACKED(NAME), FA_PACKED(NAME##_bf16)
const struct {
  const char* name;
  int (*call)(const void*);
} packed_entries[] = {FA_PACKED2(fa_qk_norm_rotary), FA_PACKED2(fa_qk_norm_rotary_bwd), FA_PACKED2(fa_paged_append),
                      FA_PACKED(fa_extend_block_table), FA_PACKED2(fa_page_means), FA_PACKED2(fa_select_pages),
                      FA_PACKED2(fa_fwd_paged_sparse)};

}  // namespace
}  // namespace fa

extern "C" void* fa_packed_entry(const char* name) {
  for (const auto& e : packed_entries)
    if (name && std::strcmp(e.name, name) == 0) return reinterpret_cast<void*>(e.call);
  return nullptr;
}
