// extern "C" entry points of the operators of an attention layer: argument validation + kernel launches.
// No allocation, no synchronisation, no exceptions cross this boundary.

#include <atomic>

#include "common.cuh"

namespace gdn2 {

int launch_rotary(const void*, const void*, void*, void*, const float*, const float*, const int64_t*, const int64_t*,
                  int64_t, int64_t, int64_t, int, int, int, int, int64_t, int, int, int, cudaStream_t);
int launch_append(const void*, const void*, void*, void*, const int64_t*, int64_t, const int64_t*, int64_t, int, int, int,
                  cudaStream_t);
int tree_ctas(int*);
int64_t tree_workspace_bytes(int64_t, int, int);
int launch_tree(const void*, const void*, const void*, const void*, const void*, const int*, const int*, const uint8_t*,
                void*, void*, const int64_t*, int64_t, int64_t, int, int, int, int, int, int64_t, int, int, int, float,
                cudaStream_t);
namespace attn {
static std::atomic<uint32_t> g_wait_polls{GDN2_ATTENTION_WAIT_POLLS};
uint32_t wait_polls() { return g_wait_polls.load(std::memory_order_relaxed); }
int64_t attention_stat_rows(const int64_t*, int64_t, int64_t);
int launch_attention_forward(const void*, const void*, const void*, void*, float*, const int64_t*, const int64_t*, int64_t,
                             int64_t, int, int, int, int, float, cudaStream_t);
int64_t attention_backward_bytes(const int64_t*, int64_t, int64_t, int, int, int);
int launch_attention_backward(const void*, const void*, const void*, const void*, const void*, const float*, void*, void*,
                              void*, void*, const int64_t*, const int64_t*, int64_t, int64_t, int, int, int, int, float,
                              cudaStream_t);
}  // namespace attn

namespace {

constexpr int64_t kMost = 0x7fffffff;

bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
int element_size(int dtype) { return dtype == GDN2_FP32 ? 4 : 2; }

int check_heads(int64_t heads, int64_t kv_heads, int64_t dim) {
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0) return GDN2_ERR_BAD_SHAPE;
  if (dim <= 0 || dim > GDN2_ATTENTION_MAX_DIM || dim % 8 != 0) return GDN2_ERR_BAD_SHAPE;
  if (heads > 65535) return GDN2_ERR_TOO_LARGE;
  return GDN2_OK;
}

// Rows, heads and channels of tensors that the tiled copies read: strides of whole 16 bytes
int check_strides(const int64_t* strides, int count) {
  for (int i = 0; i < count; ++i) {
    if (strides[i] <= 0 || strides[i] % 8 != 0 || strides[i] >= (int64_t(1) << 39)) return GDN2_ERR_ALIGNMENT;
  }
  return GDN2_OK;
}

int check_sequences(const int64_t* bounds, int64_t n_seq, int64_t time, int64_t heads) {
  if (n_seq <= 0 || time <= 0) return GDN2_ERR_BAD_SHAPE;
  const int64_t rows = bounds != nullptr ? time : n_seq;
  if (rows > kMost / 2 || time > kMost / 2 || n_seq > kMost / 2) return GDN2_ERR_TOO_LARGE;
  if (bounds != nullptr) {
    for (int64_t i = 0; i < n_seq; ++i) {
      if (bounds[i] < 0 || bounds[i + 1] < bounds[i] || bounds[i + 1] > time) return GDN2_ERR_BAD_RANGE;
    }
  }
  // pieces of 64 rows are numbered with 31 bits
  const int64_t stat = attn::attention_stat_rows(bounds, n_seq, time);
  return stat / 64 > kMost / heads ? GDN2_ERR_TOO_LARGE : GDN2_OK;
}

}  // namespace
}  // namespace gdn2

using namespace gdn2;

extern "C" {

int gdn2_rotary(const void* q, const void* k, void* q_out, void* k_out, const float* cos, const float* sin,
                const int64_t* positions, const int64_t* strides, int64_t position_stride, int64_t batch, int64_t time,
                int64_t q_heads, int64_t k_heads, int64_t dim, int64_t pairs, int64_t table, int interleaved, int inverse,
                int dtype, void* stream) {
  if (!q || !k || !q_out || !k_out || !cos || !sin || !strides) return GDN2_ERR_NULL_POINTER;
  if (batch <= 0 || time <= 0 || q_heads <= 0 || k_heads <= 0 || table <= 0) return GDN2_ERR_BAD_SHAPE;
  if (dim <= 0 || dim > 512 || dim % 2 != 0 || pairs <= 0 || 2 * pairs > dim) return GDN2_ERR_BAD_SHAPE;
  if (dtype != GDN2_BF16 && dtype != GDN2_FP16 && dtype != GDN2_FP32) return GDN2_ERR_BAD_DTYPE;
  if (batch > kMost || time > kMost || batch * time > kMost || q_heads > 65535 || k_heads > 65535) return GDN2_ERR_TOO_LARGE;
  const void* need[] = {q, k, q_out, k_out};
  for (const void* p : need) {
    if (!aligned(p, uintptr_t(element_size(dtype)))) return GDN2_ERR_ALIGNMENT;
  }
  if (!aligned(cos, 4) || !aligned(sin, 4) || !aligned(positions, 8)) return GDN2_ERR_ALIGNMENT;
  return launch_rotary(q, k, q_out, k_out, cos, sin, positions, strides, position_stride, batch, time, int(q_heads),
                       int(k_heads), int(dim), int(pairs), table, interleaved != 0, inverse != 0, dtype,
                       static_cast<cudaStream_t>(stream));
}

int gdn2_append_tokens(const void* k, const void* v, void* k_pages, void* v_pages, const int64_t* slots,
                       const int64_t* strides, int64_t tokens, int64_t pages, int64_t page, int64_t kv_heads, int64_t dim,
                       int dtype, void* stream) {
  if (!k || !v || !k_pages || !v_pages || !slots || !strides) return GDN2_ERR_NULL_POINTER;
  if (tokens <= 0 || pages <= 0 || page <= 0 || kv_heads <= 0 || dim <= 0) return GDN2_ERR_BAD_SHAPE;
  if (dtype != GDN2_BF16 && dtype != GDN2_FP16 && dtype != GDN2_FP32) return GDN2_ERR_BAD_DTYPE;
  if (pages > kMost || page > kMost || kv_heads > 65535 || dim > 65535 || kv_heads * dim > kMost / 4) return GDN2_ERR_TOO_LARGE;
  const uintptr_t es = uintptr_t(element_size(dtype));
  if (!aligned(k, es) || !aligned(v, es) || !aligned(k_pages, es) || !aligned(v_pages, es) || !aligned(slots, 8)) {
    return GDN2_ERR_ALIGNMENT;
  }
  return launch_append(k, v, k_pages, v_pages, slots, tokens, strides, pages * page, int(kv_heads), int(dim), int(es),
                       static_cast<cudaStream_t>(stream));
}

int64_t gdn2_tree_workspace_bytes(int64_t drafted, int64_t heads, int64_t kv_heads, int64_t dim) {
  if (check_heads(heads, kv_heads, dim) != GDN2_OK || drafted <= 0 || drafted > kMost / heads) return GDN2_ERR_BAD_SHAPE;
  int ctas = 0;
  const int status = tree_ctas(&ctas);
  return status != GDN2_OK ? status : tree_workspace_bytes(drafted * (heads / kv_heads), int(dim), ctas);
}

int gdn2_tree_attention(const void* q, const void* k, const void* v, const void* k_pages, const void* v_pages,
                        const int* page_table, const int* lengths, const void* mask, void* out, void* workspace,
                        const int64_t* strides, int64_t table_stride, int64_t mask_stride, int64_t batch, int64_t drafted,
                        int64_t heads, int64_t kv_heads, int64_t dim, int64_t pages, int64_t page, int64_t columns,
                        int dtype, float scale, void* stream) {
  if (!q || !k || !v || !k_pages || !v_pages || !page_table || !lengths || !out || !workspace || !strides) {
    return GDN2_ERR_NULL_POINTER;
  }
  int status = check_heads(heads, kv_heads, dim);
  if (status != GDN2_OK) return status;
  if (batch <= 0 || drafted <= 0 || pages <= 0 || page <= 0 || columns < 0) return GDN2_ERR_BAD_SHAPE;
  if (!valid_seq_dtype(dtype)) return GDN2_ERR_BAD_DTYPE;
  // a sequence's tokens, cached and drafted, are numbered with 31 bits
  if (batch > kMost || drafted > kMost / 2 / heads || pages > kMost || page > kMost || columns > (kMost / 2 - 128) / page) {
    return GDN2_ERR_TOO_LARGE;
  }
  if ((status = check_strides(strides, 9)) != GDN2_OK) return status;
  const void* need16[] = {q, k, v, k_pages, v_pages, out, workspace};
  for (const void* p : need16) {
    if (!aligned(p, 16)) return GDN2_ERR_ALIGNMENT;
  }
  if (!aligned(page_table, 4) || !aligned(lengths, 4)) return GDN2_ERR_ALIGNMENT;
  return launch_tree(q, k, v, k_pages, v_pages, page_table, lengths, static_cast<const uint8_t*>(mask), out, workspace,
                     strides, table_stride, mask_stride, int(batch), int(drafted), int(heads), int(kv_heads), int(dim),
                     pages, int(page), int(columns), dtype, scale, static_cast<cudaStream_t>(stream));
}

int64_t gdn2_attention_stat_rows(const int64_t* bounds, int64_t n_seq, int64_t time) {
  const int status = check_sequences(bounds, n_seq, time, 1);
  return status != GDN2_OK ? status : attn::attention_stat_rows(bounds, n_seq, time);
}

int gdn2_attention_forward(const void* q, const void* k, const void* v, void* out, float* statistics,
                           const int64_t* strides, const int64_t* bounds, int64_t n_seq, int64_t time, int64_t heads,
                           int64_t kv_heads, int64_t dim, int dtype, float scale, void* stream) {
  if (!q || !k || !v || !out || !strides) return GDN2_ERR_NULL_POINTER;
  int status = check_heads(heads, kv_heads, dim);
  if (status != GDN2_OK) return status;
  if (!valid_seq_dtype(dtype)) return GDN2_ERR_BAD_DTYPE;
  if ((status = check_sequences(bounds, n_seq, time, heads)) != GDN2_OK) return status;
  if ((status = check_strides(strides, 9)) != GDN2_OK) return status;
  const void* need16[] = {q, k, v, out, statistics};
  for (const void* p : need16) {
    if (!aligned(p, 16)) return GDN2_ERR_ALIGNMENT;
  }
  return attn::launch_attention_forward(q, k, v, out, statistics, strides, bounds, n_seq, time, int(heads), int(kv_heads),
                                        int(dim), dtype, scale, static_cast<cudaStream_t>(stream));
}

int64_t gdn2_attention_backward_bytes(const int64_t* bounds, int64_t n_seq, int64_t time, int64_t heads, int64_t kv_heads,
                                      int64_t dim) {
  int status = check_heads(heads, kv_heads, dim);
  if (status == GDN2_OK) status = check_sequences(bounds, n_seq, time, heads);
  return status != GDN2_OK ? status : attn::attention_backward_bytes(bounds, n_seq, time, int(heads), int(kv_heads), int(dim));
}

int gdn2_attention_backward(const void* q, const void* k, const void* v, const void* out, const void* d_out,
                            const float* statistics, void* scratch, void* dq, void* dk, void* dv, const int64_t* strides,
                            const int64_t* bounds, int64_t n_seq, int64_t time, int64_t heads, int64_t kv_heads, int64_t dim,
                            int dtype, float scale, void* stream) {
  if (!q || !k || !v || !out || !d_out || !statistics || !scratch || !dq || !dk || !dv || !strides) {
    return GDN2_ERR_NULL_POINTER;
  }
  int status = check_heads(heads, kv_heads, dim);
  if (status != GDN2_OK) return status;
  if (!valid_seq_dtype(dtype)) return GDN2_ERR_BAD_DTYPE;
  if ((status = check_sequences(bounds, n_seq, time, heads)) != GDN2_OK) return status;
  if ((status = check_strides(strides, 12)) != GDN2_OK) return status;
  const void* need16[] = {q, k, v, out, d_out, statistics, scratch, dq, dk, dv};
  for (const void* p : need16) {
    if (!aligned(p, 16)) return GDN2_ERR_ALIGNMENT;
  }
  return attn::launch_attention_backward(q, k, v, out, d_out, statistics, scratch, dq, dk, dv, strides, bounds, n_seq, time,
                                         int(heads), int(kv_heads), int(dim), dtype, scale,
                                         static_cast<cudaStream_t>(stream));
}

int gdn2_debug_wait_limit(int64_t polls) {
  if (polls > GDN2_ATTENTION_WAIT_POLLS) return GDN2_ERR_TOO_LARGE;
  attn::g_wait_polls.store(polls < 0 ? GDN2_ATTENTION_WAIT_POLLS : uint32_t(polls), std::memory_order_relaxed);
  return GDN2_OK;
}

}  // extern "C"
