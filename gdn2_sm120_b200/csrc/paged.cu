// A paged cache of keys and values: writing tokens into it, and attention of drafted tokens over it.
//
// The cache is two tensors [pages][page][kv heads][dim]; a sequence's cached token t lies in page
// page_table[sequence][t / page] at t % page, whatever the page size.
//
// append_kernel   copies the keys and values of tokens to their slots (slot = page number * page size + place in the
//                 page; a slot that is not in the cache is left out).  Bound by HBM.
//
// Attention over it: paged_tree.cuh (drafted tokens, any number of rows), paged_tiles.cuh (up to 16 rows, and what all kernels
// share), paged_window.cu (with a window), paged_weigh.cu (with the weights that tokens get).

#include "paged_tree.cuh"

namespace gdn2 {
namespace paged {

int launch_tree_window(const TreeParams& p, int dtype, cudaStream_t stream);

}  // namespace paged

namespace {

// ---- append ------------------------------------------------------------------------------------------
struct AppendParams {
  const uint8_t *k, *v;
  uint8_t *k_pages, *v_pages;
  const int64_t* slots;
  int64_t k_token, k_head, v_token, v_head;  // strides in bytes
  int64_t tokens, capacity;
  int per_head, per_token;                   // packs of a head, of a token
};

// 16411 tokens of 8 heads of 128, keys and values (121 MB both ways, half of it in L2): 18 us, 6.5 TB/s.
template <typename P>
__global__ void __launch_bounds__(256) append_kernel(const AppendParams p) {
  const int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t token = i / p.per_token;
  if (token >= p.tokens) return;
  const int at = int(i - token * p.per_token), head = at / p.per_head, c = at - head * p.per_head;
  const int64_t slot = p.slots[token];
  if (slot < 0 || slot >= p.capacity) return;
  const P k = *reinterpret_cast<const P*>(p.k + token * p.k_token + head * p.k_head + c * int64_t(sizeof(P)));
  const P v = *reinterpret_cast<const P*>(p.v + token * p.v_token + head * p.v_head + c * int64_t(sizeof(P)));
  const int64_t to = (slot * p.per_token + at) * int64_t(sizeof(P));
  *reinterpret_cast<P*>(p.k_pages + to) = k;
  *reinterpret_cast<P*>(p.v_pages + to) = v;
}

}  // namespace

int launch_append(const void* k, const void* v, void* k_pages, void* v_pages, const int64_t* slots, int64_t tokens,
                  const int64_t* strides, int64_t capacity, int kv_heads, int dim, int element, cudaStream_t stream) {
  AppendParams p{};
  p.k = static_cast<const uint8_t*>(k); p.v = static_cast<const uint8_t*>(v);
  p.k_pages = static_cast<uint8_t*>(k_pages); p.v_pages = static_cast<uint8_t*>(v_pages);
  p.slots = slots;
  p.k_token = strides[0] * element; p.k_head = strides[1] * element;
  p.v_token = strides[2] * element; p.v_head = strides[3] * element;
  p.tokens = tokens; p.capacity = capacity;
  // 16 bytes at a time where every row begins on such a boundary, or else an element
  const uintptr_t bits = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                         reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages) |
                         uintptr_t(p.k_token) | uintptr_t(p.k_head) | uintptr_t(p.v_token) | uintptr_t(p.v_head) |
                         uintptr_t(int64_t(dim) * element);
  const int pack = bits % 16 == 0 ? 16 : element;
  p.per_head = dim * element / pack;
  p.per_token = p.per_head * kv_heads;
  const int64_t blocks = (tokens * p.per_token + 255) / 256;
  if (blocks <= 0 || blocks > int64_t(0x7fffffff)) return GDN2_ERR_TOO_LARGE;
  if (pack == 16) append_kernel<uint4><<<unsigned(blocks), 256, 0, stream>>>(p);
  else if (pack == 4) append_kernel<uint32_t><<<unsigned(blocks), 256, 0, stream>>>(p);
  else append_kernel<uint16_t><<<unsigned(blocks), 256, 0, stream>>>(p);
  return check_launch();
}

int tree_ctas(int* ctas) { return multiprocessors(ctas); }

int64_t tree_workspace_bytes(int64_t rows, int dim, int ctas) {
  return int64_t(ctas) * 2 * paged::block_rows(rows) * ((dim <= 64 ? 64 : 128) + 2) * 4;
}

int launch_tree(const void* q, const void* k, const void* v, const void* k_pages, const void* v_pages, const int* table,
                const int* lengths, const uint8_t* mask, void* out, void* workspace, const int64_t* strides,
                int64_t table_stride, int64_t mask_stride, int batch, int drafted, int heads, int kv_heads, int dim,
                int64_t pages, int page, int columns, const int* depths, int64_t depth_stride, int window, int sinks, int dtype, float scale,
                cudaStream_t stream) {
  using namespace paged;
  TreeParams p{};
  const int per_block = block_rows(int64_t(drafted) * (heads / kv_heads));
  const int status = fill_tree(&p, q, k, v, k_pages, v_pages, table, lengths, out, strides, table_stride, batch, drafted, heads, kv_heads,
                               dim, pages, page, columns, dtype, scale, per_block);
  if (status != GDN2_OK) return status;
  p.mask = mask; p.mask_stride = mask_stride;
  p.partials = static_cast<float*>(workspace);
  p.depths = depths; p.depth_stride = depth_stride; p.window = window; p.sinks = sinks;
  if (int64_t(batch) * kv_heads * p.row_blocks > int64_t(0x7fffffff) / joining_ctas(p, per_block)) return GDN2_ERR_TOO_LARGE;
  if (window > 0) return launch_tree_window(p, dtype, stream);
  return dtype == GDN2_BF16 ? launch_tree_dim<__nv_bfloat16, false>(p, stream) : launch_tree_dim<__half, false>(p, stream);
}

}  // namespace gdn2
