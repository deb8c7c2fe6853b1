// Attention of new tokens over a paged cache, and the weight that every token of it got from them: tree_few_kernel, which leaves
// its scores, and weigh_kernel.
#include "paged_tiles.cuh"

namespace gdn2 {
namespace paged {
namespace {

// What weight the tokens of a sequence got from the rows of a key head, four tokens a thread:
//
//   w_t = sum_r exp(s_rt - m_r) / l_r
//
// which joins the weight that cached tokens have so far, times `decay`, and is put into their slots for the new tokens.  The
// rows' statistics are joined first, by every CTA that has tokens of a sequence and head, and the values of parted rows by the one
// that has the first.  It has to read 4 bytes of scores a row and token, against 4 * dim bytes of keys and values that the main kernel
// read (which leave L2 first, to let the scores stay), and 4 to 8 bytes of weights.  64 sequences of up to 8192 tokens, 32 / 8
// heads (42 MB of scores): 17 us behind the main kernel's end, five rounds of 1.9 us, a round being as long as its loads take;
// the main kernel takes 230 us, 15 more than without the scores.
constexpr int kWeighThreads = 256, kWeighCtas = 4;   // of an SM
constexpr int kWeighRows = GDN2_WEIGHED_MAX_ROWS;   // of a key head: new tokens times heads of a group
template <typename T, int DP>
__global__ void __launch_bounds__(kWeighThreads, kWeighCtas) weigh_kernel(const __grid_constant__ TreeParams p) {
  constexpr int kWarps = kWeighThreads / 32;
  __shared__ float4 rows[kWeighRows];   // shift, scaled, 1 / l
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // All tiles of 128 tokens, of all sequences and heads, are one list that the CTAs share evenly.  Every warp looks for its
  // CTA's first one by itself.
  auto tiles = [&](int b) {
    Unit x{b, 0, 0, 0, 0, false, 0, 0, 0};
    read_length<false>(p, x);
    return x.tiles;
  };
  int all = 0;         // tiles of the sequences
  for (int x = lane; x < p.batch; x += 32) all += tiles(x);
  all = int(__reduce_add_sync(0xffffffffu, unsigned(all)));
  const int list = all * p.kv_heads, ctas = min(list, int(gridDim.x)), cta = int(blockIdx.x);
  if (cta >= ctas) return;
  const int least = list / ctas, more = list - least * ctas;   // the first `more` CTAs have one more
  int at_tile = cta * least + min(cta, more), rest = least + (cta < more);
  int from = 0;        // tiles of the sequences before b
  int b = 0;
  for (int b0 = 0;; b0 += 32) {
    const int own = b0 + lane < p.batch ? tiles(b0 + lane) : 0;
    int up_to = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, up_to, d);
      if (lane >= d) up_to += y;
    }
    const uint32_t behind = __ballot_sync(0xffffffffu, (from + up_to) * p.kv_heads > at_tile);
    if (behind != 0) {
      b = b0 + __ffs(behind) - 1;
      from += __shfl_sync(0xffffffffu, up_to - own, b - b0);
      break;
    }
    from += __shfl_sync(0xffffffffu, up_to, 31);
  }
  Unit u{b, 0, 0, 0, 0, false, 0, 0, 0};
  read_length<false>(p, u);
  at_tile -= from * p.kv_heads;
  u.head = at_tile / u.tiles;
  int tile = at_tile - u.head * u.tiles;

  // Four tokens a thread at a time.  Their pages are looked up a round ahead, the first ones' while the other kernel still
  // runs: a round's loads wait for nothing but one another's arrival.
  struct Pages { int of[4]; };   // of cached tokens, -1 for none
  auto pages_of = [&](const Unit& x, int t0, int last) {
    Pages r;
#pragma unroll
    for (int y = 0; y < 4; ++y) r.of[y] = t0 + y < x.length && t0 < last ? p.table[x.b * p.table_stride + p.by_page.quotient(t0 + y)] : -1;
    return r;
  };
  Pages pages = pages_of(u, tile * kTile + int(threadIdx.x) * 4, (tile + min(rest, u.tiles - tile)) * kTile);
  // Until here nothing was read that the other kernel writes
  asm volatile("griddepcontrol.wait;" ::: "memory");
  while (rest > 0) {
    const int n = min(rest, u.tiles - tile), last = (tile + n) * kTile, end = min(u.length + p.drafted, last);
    for (int r = warp; r < p.rows; r += kWarps) {
      const int block = r / 16;
      const int2 ctas = p.ends[(int64_t(u.b) * p.kv_heads + u.head) * p.row_blocks + block];
      const RowParts x{ctas.x, ctas.y, 16, r - block * 16};
      float acc[DP / 32];
      const bool several = x.c0 != x.c1, mine = tile == 0;   // the values by the CTA that has the first tile
      const float2 ml = several ? join_row<DP>(p, x, mine, acc) : p.stats[(int64_t(u.b) * p.kv_heads + u.head) * p.rows + r];
      const float inv = ml.y == 0.f ? 0.f : 1.f / ml.y;
      if (several && mine) store_joined<T, DP>(p, u.b, u.head, r, acc, inv);
      if (lane == 0) {
        const attn::Reference ref = attn::reference(ml.x, p.scale_log2);
        rows[r] = make_float4(ref.shift, ref.scaled, inv, 0.f);
      }
    }
    __syncthreads();
    // (whole float4s of a row: its width is a multiple of 32)
    const float* scores = p.scores + (int64_t(u.b) * p.kv_heads + u.head) * p.rows * p.width;
    for (int t0 = tile * kTile + int(threadIdx.x) * 4; t0 < end; t0 += kWeighThreads * 4) {
      float* at[4];      // of the weights, null for none
      float old[4], weight[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int page = pages.of[y];
        int place;
        p.by_page.split(t0 + y, &place);
        at[y] = page < 0 || page >= p.pages ? nullptr : p.weight_pages + (int64_t(page) * p.kv_heads + u.head) * p.page + place;
        old[y] = 0.f;
        if (p.decay != 0.f && at[y] != nullptr) old[y] = *at[y];
      }
      pages = pages_of(u, t0 + kWeighThreads * 4, last);
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
          const int64_t slot = p.slots[int64_t(u.b) * p.drafted + i];
          if (slot < 0 || slot >= p.pages * p.page) continue;
          const int64_t page = slot <= 0x7fffffff ? p.by_page.quotient(int(slot)) : slot / p.page;   // (64-bit quotients take long)
          p.weight_pages[(page * p.kv_heads + u.head) * p.page + (slot - page * p.page)] = weight[y];
        }
      }
    }
    rest -= n;
    if (rest == 0) break;
    tile = 0;
    if (++u.head == p.kv_heads) {
      u.head = 0;
      ++u.b;
      read_length<false>(p, u);
    }
    pages = pages_of(u, int(threadIdx.x) * 4, min(rest, u.tiles) * kTile);
    __syncthreads();   // the rows have been read
  }
}

template <typename T, int DP>
int launch_weigh(const TreeParams& p, cudaStream_t stream) {
  return launch_beside(&weigh_kernel<T, DP>, unsigned(p.slices), kWeighThreads, 0, stream, p);
}

template <typename T, int DP>
int launch_typed(const TreeParams& p, cudaStream_t stream) {
  const int status = launch_few<T, DP, false, true>(p, stream);
  return status != GDN2_OK ? status : launch_weigh<T, DP>(p, stream);
}

}  // namespace
}  // namespace paged

// parts of rows that several CTAs have, statistics of the others, which CTAs those are, scores
struct WeighBytes { int64_t parts, stats, ends, scores; int width; };
static WeighBytes weigh_bytes(int batch, int tokens, int heads, int kv_heads, int dim, int page, int columns, int ctas) {
  const int64_t rows = int64_t(batch) * tokens * heads;
  const int64_t width = (int64_t(page) * columns + tokens + 31) / 32 * 32;
  return {int64_t(ctas) * 2 * 16 * ((dim <= 64 ? 64 : 128) + 2) * 4, (rows * 8 + 15) / 16 * 16,
          (int64_t(batch) * kv_heads * ((tokens * (heads / kv_heads) + 15) / 16) * 8 + 15) / 16 * 16, rows * width * 4, int(width)};
}

int64_t weighed_workspace_bytes(int batch, int tokens, int heads, int kv_heads, int dim, int page, int columns) {
  int ctas = 0;
  const int status = tree_ctas(&ctas);
  if (status != GDN2_OK) return status;
  const WeighBytes x = weigh_bytes(batch, tokens, heads, kv_heads, dim, page, columns, ctas);
  return x.parts + x.stats + x.ends + x.scores;
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
  p.ends = reinterpret_cast<int2*>(at + x.parts + x.stats);
  p.scores = reinterpret_cast<float*>(at + x.parts + x.stats + x.ends);
  p.width = x.width;
  p.weight_pages = weight_pages; p.slots = slots; p.decay = decay;
  p.by_page = divisor(page);
  // CTAs of weigh_kernel: what the SMs hold at once, but no more than there can be tiles
  const int64_t most = (int64_t(page) * columns + tokens + kTile - 1) / kTile;
  if (int64_t(batch) * kv_heads * most > int64_t(0x7fffffff)) return GDN2_ERR_TOO_LARGE;
  p.slices = int(std::min<int64_t>(kWeighCtas * p.ctas, int64_t(batch) * kv_heads * most));
  if (dtype == GDN2_BF16) return dim <= 64 ? launch_typed<__nv_bfloat16, 64>(p, stream) : launch_typed<__nv_bfloat16, 128>(p, stream);
  return dim <= 64 ? launch_typed<__half, 64>(p, stream) : launch_typed<__half, 128>(p, stream);
}

}  // namespace gdn2
