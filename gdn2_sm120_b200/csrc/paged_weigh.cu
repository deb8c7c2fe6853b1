// Attention of new tokens over a paged cache, and the weight that every token of it got from them: tree_few_kernel, which leaves
// its scores, and weigh_kernel.
#include "paged_tiles.cuh"

namespace gdn2 {
namespace paged {
namespace {

// What weight the tokens of a sequence got from the rows of a key head, a thread a token:
//
//   w_t = sum_r exp(s_rt - m_r) / l_r
//
// which joins the weight that cached tokens have so far, times `decay`, and is put into their slots for the new tokens.  The
// rows' statistics are joined first, by every CTA of a sequence and head for itself, and the values of parted rows by them
// in turn.  Bound by L2, in which the scores (4 bytes a row and token, against 4 * dim of keys and values) mostly still are:
// TODO-FIGURES
constexpr int kWeighThreads = 256, kWeighCtas = 4;   // of an SM
constexpr int kWeighRows = GDN2_WEIGHED_MAX_ROWS;   // of a key head: new tokens times heads of a group
template <typename T, int DP>
__global__ void __launch_bounds__(kWeighThreads, kWeighCtas) weigh_kernel(const __grid_constant__ TreeParams p) {
  constexpr int kWarps = kWeighThreads / 32;
  __shared__ float4 rows[kWeighRows];   // shift, scaled, 1 / l
  const int unit = int(blockIdx.x) / p.slices, slice = int(blockIdx.x) - unit * p.slices;
  const int head = unit % p.kv_heads, b = unit / p.kv_heads;
  const int lane = threadIdx.x & 31;
  int64_t total = 0, from = 0;   // tiles of all sequences, of those before this one: by every warp
  for (int x = lane; x < p.batch; x += 32) {
    const int64_t own = tiles_of<false>(p, x);
    total += own;
    from += x < b ? own : 0;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, d);
    from += __shfl_xor_sync(0xffffffffu, from, d);
  }
  Unit u{b, 0, 0, 0, 0, false, 0, 0, 0};
  read_length<false>(p, u);
  const int64_t ctas = sharing(p, total);
  // Four tokens a thread at a time.  Their pages are looked up a round ahead, the first ones' while the other kernel still
  // runs: a round's loads wait for nothing but one another's arrival.
  const int* table = p.table + b * p.table_stride;
  const int end = u.length + p.drafted, round = p.slices * kWeighThreads * 4;
  struct Pages { int of[4]; };   // of cached tokens, -1 for none
  auto pages_of = [&](int t0) {
    Pages x;
#pragma unroll
    for (int y = 0; y < 4; ++y) x.of[y] = t0 + y < u.length ? table[p.by_page.quotient(t0 + y)] : -1;
    return x;
  };
  int t0 = (slice * kWeighThreads + int(threadIdx.x)) * 4;
  Pages pages = pages_of(t0);
  // Until here nothing was read that the other kernel writes
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int r = threadIdx.x >> 5; r < p.rows; r += kWarps) {
    const int block = r / 16;
    const int64_t t0 = from + (int64_t(head) * p.row_blocks + block) * u.tiles, t1 = t0 + u.tiles;
    const RowParts x{((t0 + 1) * ctas - 1) / total, (t1 * ctas - 1) / total, 16, r - block * 16};
    float acc[DP / 32];
    const bool parted = x.c0 != x.c1, mine = r % p.slices == slice;
    const float2 ml = parted ? join_row<DP>(p, x, mine, acc) : p.stats[(int64_t(b) * p.kv_heads + head) * p.rows + r];
    const float inv = ml.y == 0.f ? 0.f : 1.f / ml.y;
    if (parted && mine) store_joined<T, DP>(p, b, head, r, acc, inv);
    if (lane == 0) {
      const attn::Reference ref = attn::reference(ml.x, p.scale_log2);
      rows[r] = make_float4(ref.shift, ref.scaled, inv, 0.f);
    }
  }
  __syncthreads();
  // (whole float4s of a row: its width is a multiple of 32)
  const float* scores = p.scores + (int64_t(b) * p.kv_heads + head) * p.rows * p.width;
  for (; t0 < end; t0 += round) {
    float* at[4];      // of the weights, null for none
    float old[4], weight[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int page = pages.of[y];
      int place;
      p.by_page.split(t0 + y, &place);
      at[y] = page < 0 || page >= p.pages ? nullptr : p.weight_pages + (int64_t(page) * p.kv_heads + head) * p.page + place;
      old[y] = 0.f;
      if (p.decay != 0.f && at[y] != nullptr) old[y] = *at[y];
    }
    pages = pages_of(t0 + round);
#pragma unroll 4
    for (int r = 0; r < p.rows; ++r) {
      const float4 row = rows[r], s = __ldcs(reinterpret_cast<const float4*>(scores + int64_t(r) * p.width + t0));
      weight[0] = fmaf(exp2_approx(fmaf(s.x - row.x, p.scale_log2, -row.y)), row.z, weight[0]);
      weight[1] = fmaf(exp2_approx(fmaf(s.y - row.x, p.scale_log2, -row.y)), row.z, weight[1]);
      weight[2] = fmaf(exp2_approx(fmaf(s.z - row.x, p.scale_log2, -row.y)), row.z, weight[2]);
      weight[3] = fmaf(exp2_approx(fmaf(s.w - row.x, p.scale_log2, -row.y)), row.z, weight[3]);
    }
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      if (at[y] != nullptr) *at[y] = p.decay != 0.f ? fmaf(old[y], p.decay, weight[y]) : weight[y];
    }
    if (t0 + 4 > u.length) {   // new tokens
      for (int y = 0; y < 4; ++y) {
        const int i = t0 + y - u.length;
        if (i < 0 || i >= p.drafted) continue;
        const int64_t slot = p.slots[int64_t(b) * p.drafted + i], page = slot < 0 ? -1 : slot / p.page;
        if (page >= 0 && page < p.pages) p.weight_pages[(page * p.kv_heads + head) * p.page + slot % p.page] = weight[y];
      }
    }
  }
}

template <typename T, int DP>
int launch_weigh(const TreeParams& p, cudaStream_t stream) {
  return launch_beside(&weigh_kernel<T, DP>, unsigned(p.batch * p.kv_heads * p.slices), kWeighThreads, 0, stream, p);
}

template <typename T, int DP>
int launch_typed(const TreeParams& p, cudaStream_t stream) {
  const int status = launch_few<T, DP, false, true>(p, stream);
  return status != GDN2_OK ? status : launch_weigh<T, DP>(p, stream);
}

}  // namespace
}  // namespace paged

// parts of rows that several CTAs have, statistics of the others, scores
struct WeighBytes { int64_t parts, stats, scores; int width; };
static WeighBytes weigh_bytes(int batch, int tokens, int heads, int kv_heads, int dim, int page, int columns, int ctas) {
  const int64_t rows = int64_t(batch) * tokens * heads;
  const int64_t width = (int64_t(page) * columns + tokens + 31) / 32 * 32;
  return {int64_t(ctas) * 2 * 16 * ((dim <= 64 ? 64 : 128) + 2) * 4, (rows * 8 + 15) / 16 * 16, rows * width * 4, int(width)};
}

int64_t weighed_workspace_bytes(int batch, int tokens, int heads, int kv_heads, int dim, int page, int columns) {
  int ctas = 0;
  const int status = tree_ctas(&ctas);
  if (status != GDN2_OK) return status;
  const WeighBytes x = weigh_bytes(batch, tokens, heads, kv_heads, dim, page, columns, ctas);
  return x.parts + x.stats + x.scores;
}

int launch_weighed(const void* q, const void* k, const void* v, const void* k_pages, const void* v_pages, float* weight_pages,
                   const int* table, const int* lengths, const int64_t* slots, void* out, void* workspace, const int64_t* strides,
                   int64_t table_stride, int batch, int tokens, int heads, int kv_heads, int dim, int64_t pages, int page, int columns,
                   float decay, int dtype, float scale, cudaStream_t stream) {
  using namespace paged;
  TreeParams p{};
  int status = fill_tree(&p, q, k, v, k_pages, v_pages, table, lengths, out, strides, table_stride, batch, tokens, heads, kv_heads, dim,
                         pages, page, columns, dtype, scale, kFewRows);
  if (status != GDN2_OK) return status;
  const WeighBytes x = weigh_bytes(batch, tokens, heads, kv_heads, dim, page, columns, p.ctas);
  uint8_t* at = static_cast<uint8_t*>(workspace);
  p.partials = reinterpret_cast<float*>(at);
  p.stats = reinterpret_cast<float2*>(at + x.parts);
  p.scores = reinterpret_cast<float*>(at + x.parts + x.stats);
  p.width = x.width;
  p.weight_pages = weight_pages; p.slots = slots; p.decay = decay;
  p.by_page = divisor(page);
  // CTAs of weigh_kernel: four times what the SMs hold at once, since sequences are not equally long, but not more than a round
  // of its threads at the most tokens that there can be
  const int64_t units = int64_t(batch) * kv_heads;
  const int64_t most = (int64_t(page) * columns + tokens + 4 * kWeighThreads - 1) / (4 * kWeighThreads);
  p.slices = int(std::max<int64_t>(1, std::min(most, 4 * kWeighCtas * p.ctas / units)));
  if (units > int64_t(0x7fffffff) / p.slices) return GDN2_ERR_TOO_LARGE;
  if (dtype == GDN2_BF16) return dim <= 64 ? launch_typed<__nv_bfloat16, 64>(p, stream) : launch_typed<__nv_bfloat16, 128>(p, stream);
  return dim <= 64 ? launch_typed<__half, 64>(p, stream) : launch_typed<__half, 128>(p, stream);
}

}  // namespace gdn2
