// extern "C" entry points of the operators of an attention layer: argument validation + kernel launches.
// No allocation, no synchronisation, no exceptions cross this boundary.

#include <algorithm>
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
                void*, void*, const int64_t*, int64_t, int64_t, int, int, int, int, int, int64_t, int, int, const int*, int64_t, int,
                int, int, float, cudaStream_t);
int64_t weighed_workspace_bytes(int, int, int, int, int, int, int);
int launch_weighed(const void*, const void*, const void*, const void*, const void*, float*, const int*, const int*, const int64_t*,
                   void*, void*, const int64_t*, int64_t, int, int, int, int, int, int64_t, int, int, float, int, float, cudaStream_t);
int64_t evict_workspace_bytes(int64_t, int64_t, int64_t);
int launch_evict(void*, void*, float*, const int*, const int*, const int*, int*, void*, int64_t, int64_t, int, int64_t, int, int, int,
                 int, int, int, int, int, cudaStream_t);
namespace attn {
static std::atomic<uint32_t> g_wait_polls{GDN2_ATTENTION_WAIT_POLLS};
uint32_t wait_polls() { return g_wait_polls.load(std::memory_order_relaxed); }
int64_t attention_stat_rows(const int64_t*, int64_t, int64_t);
int launch_attention_forward(const void*, const void*, const void*, void*, float*, void*, const int64_t*, const int64_t*, int64_t,
                             int64_t, int, int, int, int, float, int64_t, int64_t, cudaStream_t);
int64_t attention_backward_bytes(const int64_t*, int64_t, int64_t, int, int, int, int64_t, int64_t);
int launch_attention_backward(const void*, const void*, const void*, const void*, const void*, const void*, const float*, void*, void*,
                              void*, void*, const int64_t*, const int64_t*, int64_t, int64_t, int, int, int, int, float,
                              int64_t, int64_t, cudaStream_t);
int64_t attention_weights_bytes(const int64_t*, int64_t, int64_t, int, int);
int launch_attention_weights(const void*, const void*, const float*, float*, void*, const int64_t*, const int64_t*, int64_t, int64_t,
                             int, int, int, int, float, cudaStream_t);
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

// Attention over a paged cache, with a window of 0 for none
int tree_attention(const void* q, const void* k, const void* v, const void* k_pages, const void* v_pages,
                   const int* page_table, const int* lengths, const void* mask, const int* depths, void* out,
                   void* workspace, const int64_t* strides, int64_t table_stride, int64_t mask_stride, int64_t depth_stride,
                   int64_t batch, int64_t drafted, int64_t heads, int64_t kv_heads, int64_t dim, int64_t pages, int64_t page,
                   int64_t columns, int64_t window, int64_t sinks, int dtype, float scale, void* stream) {
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
  if (!aligned(page_table, 4) || !aligned(lengths, 4) || !aligned(depths, 4)) return GDN2_ERR_ALIGNMENT;
  return launch_tree(q, k, v, k_pages, v_pages, page_table, lengths, static_cast<const uint8_t*>(mask), out, workspace,
                     strides, table_stride, mask_stride, int(batch), int(drafted), int(heads), int(kv_heads), int(dim),
                     pages, int(page), int(columns), depths, depth_stride, int(std::min(window, kMost / 2)),
                     int(std::min(sinks, kMost / 2)), dtype, scale, static_cast<cudaStream_t>(stream));
}

int check_weighed(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim, int64_t page, int64_t columns) {
  const int status = check_heads(heads, kv_heads, dim);
  if (status != GDN2_OK) return status;
  if (batch <= 0 || tokens <= 0 || page <= 0 || columns <= 0) return GDN2_ERR_BAD_SHAPE;
  // a sequence's tokens, cached and new, are numbered with 31 bits
  if (batch > kMost / heads || tokens > GDN2_WEIGHED_MAX_ROWS / (heads / kv_heads) || page > kMost || columns > (kMost / 2 - 512) / page) {
    return GDN2_ERR_TOO_LARGE;
  }
  return GDN2_OK;
}

// Causal attention, with a window of 0 for none
int attention_forward(const void* q, const void* k, const void* v, void* out, float* statistics, void* rest, const int64_t* strides,
                      const int64_t* bounds, int64_t n_seq, int64_t time, int64_t heads, int64_t kv_heads, int64_t dim,
                      int64_t window, int64_t sinks, int dtype, float scale, void* stream) {
  if (!q || !k || !v || !out || !strides) return GDN2_ERR_NULL_POINTER;
  int status = check_heads(heads, kv_heads, dim);
  if (status != GDN2_OK) return status;
  if (!valid_seq_dtype(dtype)) return GDN2_ERR_BAD_DTYPE;
  if ((status = check_sequences(bounds, n_seq, time, heads)) != GDN2_OK) return status;
  if ((status = check_strides(strides, 9)) != GDN2_OK) return status;
  const void* need16[] = {q, k, v, out, statistics, rest};
  for (const void* p : need16) {
    if (!aligned(p, 16)) return GDN2_ERR_ALIGNMENT;
  }
  return attn::launch_attention_forward(q, k, v, out, statistics, rest, strides, bounds, n_seq, time, int(heads), int(kv_heads),
                                        int(dim), dtype, scale, window, sinks, static_cast<cudaStream_t>(stream));
}

int64_t attention_backward_bytes(const int64_t* bounds, int64_t n_seq, int64_t time, int64_t heads, int64_t kv_heads,
                                 int64_t dim, int64_t window, int64_t sinks) {
  int status = check_heads(heads, kv_heads, dim);
  if (status == GDN2_OK) status = check_sequences(bounds, n_seq, time, heads);
  return status != GDN2_OK ? status : attn::attention_backward_bytes(bounds, n_seq, time, int(heads), int(kv_heads), int(dim), window, sinks);
}

int attention_backward(const void* q, const void* k, const void* v, const void* out, const void* rest, const void* d_out, const float* statistics,
                       void* scratch, void* dq, void* dk, void* dv, const int64_t* strides, const int64_t* bounds, int64_t n_seq,
                       int64_t time, int64_t heads, int64_t kv_heads, int64_t dim, int64_t window, int64_t sinks, int dtype,
                       float scale, void* stream) {
  if (!q || !k || !v || !out || !d_out || !statistics || !scratch || !dq || !dk || !dv || !strides) {
    return GDN2_ERR_NULL_POINTER;
  }
  int status = check_heads(heads, kv_heads, dim);
  if (status != GDN2_OK) return status;
  if (!valid_seq_dtype(dtype)) return GDN2_ERR_BAD_DTYPE;
  if ((status = check_sequences(bounds, n_seq, time, heads)) != GDN2_OK) return status;
  if ((status = check_strides(strides, 12)) != GDN2_OK) return status;
  const void* need16[] = {q, k, v, out, rest, d_out, statistics, scratch, dq, dk, dv};
  for (const void* p : need16) {
    if (!aligned(p, 16)) return GDN2_ERR_ALIGNMENT;
  }
  return attn::launch_attention_backward(q, k, v, out, rest, d_out, statistics, scratch, dq, dk, dv, strides, bounds, n_seq, time,
                                         int(heads), int(kv_heads), int(dim), dtype, scale, window, sinks,
                                         static_cast<cudaStream_t>(stream));
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
  return tree_attention(q, k, v, k_pages, v_pages, page_table, lengths, mask, nullptr, out, workspace, strides, table_stride,
                        mask_stride, 0, batch, drafted, heads, kv_heads, dim, pages, page, columns, 0, 0, dtype, scale, stream);
}

int gdn2_window_tree_attention(const void* q, const void* k, const void* v, const void* k_pages, const void* v_pages,
                               const int* page_table, const int* lengths, const void* mask, const int* depths, void* out,
                               void* workspace, const int64_t* strides, int64_t table_stride, int64_t mask_stride,
                               int64_t depth_stride, int64_t batch, int64_t drafted, int64_t heads, int64_t kv_heads, int64_t dim,
                               int64_t pages, int64_t page, int64_t columns, int64_t window, int64_t sinks, int dtype, float scale,
                               void* stream) {
  if (window <= 0 || sinks < 0 || (mask != nullptr && depths == nullptr)) return GDN2_ERR_BAD_RANGE;
  return tree_attention(q, k, v, k_pages, v_pages, page_table, lengths, mask, depths, out, workspace, strides, table_stride,
                        mask_stride, depth_stride, batch, drafted, heads, kv_heads, dim, pages, page, columns, window, sinks, dtype,
                        scale, stream);
}

int64_t gdn2_attention_stat_rows(const int64_t* bounds, int64_t n_seq, int64_t time) {
  const int status = check_sequences(bounds, n_seq, time, 1);
  return status != GDN2_OK ? status : attn::attention_stat_rows(bounds, n_seq, time);
}

int gdn2_attention_forward(const void* q, const void* k, const void* v, void* out, float* statistics,
                           const int64_t* strides, const int64_t* bounds, int64_t n_seq, int64_t time, int64_t heads,
                           int64_t kv_heads, int64_t dim, int dtype, float scale, void* stream) {
  return attention_forward(q, k, v, out, statistics, nullptr, strides, bounds, n_seq, time, heads, kv_heads, dim, 0, 0, dtype, scale, stream);
}

int64_t gdn2_attention_backward_bytes(const int64_t* bounds, int64_t n_seq, int64_t time, int64_t heads, int64_t kv_heads,
                                      int64_t dim) {
  return attention_backward_bytes(bounds, n_seq, time, heads, kv_heads, dim, 0, 0);
}

int gdn2_attention_backward(const void* q, const void* k, const void* v, const void* out, const void* d_out,
                            const float* statistics, void* scratch, void* dq, void* dk, void* dv, const int64_t* strides,
                            const int64_t* bounds, int64_t n_seq, int64_t time, int64_t heads, int64_t kv_heads, int64_t dim,
                            int dtype, float scale, void* stream) {
  return attention_backward(q, k, v, out, nullptr, d_out, statistics, scratch, dq, dk, dv, strides, bounds, n_seq, time, heads, kv_heads, dim,
                            0, 0, dtype, scale, stream);
}

int gdn2_window_attention_forward(const void* q, const void* k, const void* v, void* out, float* statistics, void* rest,
                                  const int64_t* strides, const int64_t* bounds, int64_t n_seq, int64_t time, int64_t heads,
                                  int64_t kv_heads, int64_t dim, int64_t window, int64_t sinks, int dtype, float scale,
                                  void* stream) {
  if (window <= 0 || sinks < 0) return GDN2_ERR_BAD_RANGE;
  return attention_forward(q, k, v, out, statistics, rest, strides, bounds, n_seq, time, heads, kv_heads, dim, window, sinks, dtype, scale,
                           stream);
}

int64_t gdn2_window_attention_backward_bytes(const int64_t* bounds, int64_t n_seq, int64_t time, int64_t heads, int64_t kv_heads,
                                             int64_t dim, int64_t window, int64_t sinks) {
  if (window <= 0 || sinks < 0) return GDN2_ERR_BAD_RANGE;
  return attention_backward_bytes(bounds, n_seq, time, heads, kv_heads, dim, window, sinks);
}

int gdn2_window_attention_backward(const void* q, const void* k, const void* v, const void* out, const void* rest,
                                   const void* d_out, const float* statistics, void* scratch, void* dq, void* dk, void* dv, const int64_t* strides,
                                   const int64_t* bounds, int64_t n_seq, int64_t time, int64_t heads, int64_t kv_heads,
                                   int64_t dim, int64_t window, int64_t sinks, int dtype, float scale, void* stream) {
  if (window <= 0 || sinks < 0) return GDN2_ERR_BAD_RANGE;
  return attention_backward(q, k, v, out, rest, d_out, statistics, scratch, dq, dk, dv, strides, bounds, n_seq, time, heads, kv_heads, dim,
                            window, sinks, dtype, scale, stream);
}

int64_t gdn2_attention_weights_bytes(const int64_t* bounds, int64_t n_seq, int64_t time, int64_t heads, int64_t kv_heads) {
  int status = check_heads(heads, kv_heads, 8);
  if (status == GDN2_OK) status = check_sequences(bounds, n_seq, time, heads);
  return status != GDN2_OK ? status : attn::attention_weights_bytes(bounds, n_seq, time, int(heads), int(kv_heads));
}

int gdn2_attention_weights(const void* q, const void* k, const float* statistics, float* weights, void* scratch,
                           const int64_t* strides, const int64_t* bounds, int64_t n_seq, int64_t time, int64_t heads,
                           int64_t kv_heads, int64_t dim, int dtype, float scale, void* stream) {
  if (!q || !k || !statistics || !weights || !strides) return GDN2_ERR_NULL_POINTER;
  int status = check_heads(heads, kv_heads, dim);
  if (status != GDN2_OK) return status;
  if (!valid_seq_dtype(dtype)) return GDN2_ERR_BAD_DTYPE;
  if ((status = check_sequences(bounds, n_seq, time, heads)) != GDN2_OK) return status;
  if ((status = check_strides(strides, 6)) != GDN2_OK) return status;
  const void* need16[] = {q, k, statistics};
  for (const void* p : need16) {
    if (!aligned(p, 16)) return GDN2_ERR_ALIGNMENT;
  }
  if (!aligned(weights, 4) || !aligned(scratch, 4)) return GDN2_ERR_ALIGNMENT;
  return attn::launch_attention_weights(q, k, statistics, weights, scratch, strides, bounds, n_seq, time, int(heads), int(kv_heads),
                                        int(dim), dtype, scale, static_cast<cudaStream_t>(stream));
}

int64_t gdn2_weighed_token_workspace_bytes(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim,
                                           int64_t page, int64_t columns) {
  const int status = check_weighed(batch, tokens, heads, kv_heads, dim, page, columns);
  return status != GDN2_OK ? status
                           : weighed_workspace_bytes(int(batch), int(tokens), int(heads), int(kv_heads), int(dim), int(page), int(columns));
}

int gdn2_weighed_token_attention(const void* q, const void* k, const void* v, const void* k_pages, const void* v_pages,
                                 float* weight_pages, const int* page_table, const int* lengths, const int64_t* slots, void* out,
                                 void* workspace, const int64_t* strides, int64_t table_stride, int64_t batch, int64_t tokens,
                                 int64_t heads, int64_t kv_heads, int64_t dim, int64_t pages, int64_t page, int64_t columns,
                                 float decay, int dtype, float scale, void* stream) {
  if (!q || !k || !v || !k_pages || !v_pages || !weight_pages || !page_table || !lengths || !slots || !out || !workspace || !strides) {
    return GDN2_ERR_NULL_POINTER;
  }
  int status = check_weighed(batch, tokens, heads, kv_heads, dim, page, columns);
  if (status != GDN2_OK) return status;
  if (pages <= 0) return GDN2_ERR_BAD_SHAPE;
  if (pages > kMost) return GDN2_ERR_TOO_LARGE;
  if (!valid_seq_dtype(dtype)) return GDN2_ERR_BAD_DTYPE;
  if ((status = check_strides(strides, 9)) != GDN2_OK) return status;
  const void* need16[] = {q, k, v, k_pages, v_pages, out, workspace};
  for (const void* p : need16) {
    if (!aligned(p, 16)) return GDN2_ERR_ALIGNMENT;
  }
  if (!aligned(page_table, 4) || !aligned(lengths, 4) || !aligned(weight_pages, 4) || !aligned(slots, 8)) return GDN2_ERR_ALIGNMENT;
  return launch_weighed(q, k, v, k_pages, v_pages, weight_pages, page_table, lengths, slots, out, workspace, strides, table_stride,
                        int(batch), int(tokens), int(heads), int(kv_heads), int(dim), pages, int(page), int(columns), decay, dtype,
                        scale, static_cast<cudaStream_t>(stream));
}

int64_t gdn2_evict_workspace_bytes(int64_t batch, int64_t kv_heads, int64_t keep) {
  if (batch <= 0 || kv_heads <= 0 || keep <= 0) return GDN2_ERR_BAD_SHAPE;
  if (keep > kMost / 2 || batch > kMost / kv_heads) return GDN2_ERR_TOO_LARGE;
  return evict_workspace_bytes(batch, kv_heads, keep);
}

int gdn2_evict_tokens(void* k_pages, void* v_pages, float* weight_pages, const int* page_table, const int* lengths,
                      const int* new_table, int* new_lengths, void* workspace, int64_t table_stride, int64_t new_stride,
                      int64_t batch, int64_t pages, int64_t page, int64_t kv_heads, int64_t dim, int64_t columns,
                      int64_t new_columns, int64_t keep, int64_t sinks, int64_t recent, int dtype, void* stream) {
  if (!k_pages || !v_pages || !weight_pages || !page_table || !lengths || !new_table || !new_lengths || !workspace) {
    return GDN2_ERR_NULL_POINTER;
  }
  if (batch <= 0 || pages <= 0 || page <= 0 || kv_heads <= 0 || dim <= 0 || columns <= 0 || new_columns <= 0) return GDN2_ERR_BAD_SHAPE;
  if (dtype != GDN2_BF16 && dtype != GDN2_FP16 && dtype != GDN2_FP32) return GDN2_ERR_BAD_DTYPE;
  if (pages > kMost || page > kMost || kv_heads > 65535 || dim > 65535 || kv_heads * dim > kMost / 4 || batch > kMost / kv_heads ||
      columns > kMost / 2 / page || new_columns > kMost / 2 / page) {
    return GDN2_ERR_TOO_LARGE;
  }
  if (keep <= 0 || sinks < 0 || recent < 0 || sinks > keep || recent > keep - sinks || keep > new_columns * page) return GDN2_ERR_BAD_RANGE;
  const uintptr_t es = uintptr_t(element_size(dtype));
  if (!aligned(k_pages, es) || !aligned(v_pages, es) || !aligned(weight_pages, 4) || !aligned(page_table, 4) || !aligned(lengths, 4) ||
      !aligned(new_table, 4) || !aligned(new_lengths, 4) || !aligned(workspace, 4)) {
    return GDN2_ERR_ALIGNMENT;
  }
  return launch_evict(k_pages, v_pages, weight_pages, page_table, lengths, new_table, new_lengths, workspace, table_stride, new_stride,
                      int(batch), pages, int(page), int(kv_heads), int(dim), int(columns), int(keep), int(sinks), int(recent), int(es),
                      static_cast<cudaStream_t>(stream));
}

int gdn2_debug_wait_limit(int64_t polls) {
  if (polls > GDN2_ATTENTION_WAIT_POLLS) return GDN2_ERR_TOO_LARGE;
  attn::g_wait_polls.store(polls < 0 ? GDN2_ATTENTION_WAIT_POLLS : uint32_t(polls), std::memory_order_relaxed);
  return GDN2_OK;
}

}  // extern "C"
