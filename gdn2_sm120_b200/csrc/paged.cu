// A paged cache of keys and values: writing tokens into it, and attention of drafted tokens over it.
//
// The cache is two tensors [pages][page][kv heads][dim]; a sequence's cached token t lies in page
// page_table[sequence][t / page] at t % page, whatever the page size.
//
// append_kernel   copies the keys and values of tokens to their slots (slot = page number * page size + place in the
//                 page; a slot that is not in the cache is left out).  Bound by HBM.
//
// tree_kernel     N drafted tokens of each sequence, given beside the cache, see all its cached tokens and those
//                 drafted ones that their mask row names (their ancestors in a tree of drafts); N = 1 is plain decoding:
//
//                   o_i = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i),   s_ij = scale q_i . k_j,  m_i = max_j s_ij
//
//                 and 0 where nothing is seen.  One pass with a running maximum and sum.  The heads of a group are rows
//                 of one product with their shared key head, so a key is read once for 256 rows (drafted tokens x heads
//                 of a group).  Bound by HBM: the 64 KiB of a tile of 128 tokens take an SM's share of HBM 2700 clocks,
//                 its products 1024 for up to 128 rows and 2048 for up to 256, the few rows of plain decoding too.
//                 All (sequence, key head, block of rows, tile) are one list that the CTAs share evenly, so neither
//                 unequal lengths nor few sequences leave SMs idle, and the host need not know the lengths.  A CTA
//                 whose part begins or ends inside a sequence leaves (O, m, l) in the workspace; tree_join_kernel joins
//                 these in the order of the tiles: the same inputs give the same bits.
//
// A CTA of tree_kernel: two chains of four warps turn scores into weights, a row a thread.  Up to 128 rows both work on the
// same rows, on every other tile, and their (O, m, l) are joined at the end; above, each has 128 rows and all tiles.  Four
// warps bring in keys and values, in boxes of a tiled copy where the pages allow it and row by row with 16-byte asynchronous
// copies elsewhere; one brings queries, one issues the products.  TMEM: S0 S1 O0 O1, 128 columns each, P over S.  48 drafted
// tokens of 8 sequences over up to 16000 cached ones, 4 heads a group (192 rows): 106 us, 3.4 TB/s (a call in a loop, with the
// join of the parts, 128 to 132); what bounds it is a chain's round trip between the tensor cores and its warps (of an older form
// that took 142 us, 108 remained without the copies, 116 without the weights).
// tree_few_kernel has up to 16 rows (below).

#include <algorithm>

#include "attention_common.cuh"

namespace gdn2 {

using attn::Format;
using attn::pack_pair;
using attn::place_of;

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

// ---- tree attention ----------------------------------------------------------------------------------
constexpr int kTile = 128;     // tokens of a tile
constexpr int kThreads = 512;  // warps 0-3, 4-7: weights; 8-11: keys and values; 12: products; 13: queries
constexpr int kJoinThreads = 128;
struct TreeParams {
  const void *q, *k, *v;
  const void *k_pages, *v_pages;
  void* out;
  const int *table, *lengths;
  const uint8_t* mask;                       // [batch or 1][drafted][drafted], or null: j <= i
  float* partials;                           // [CTA][2][rows of a block][DP], then [CTA][2][rows of a block][m, l]
  int64_t q_stride[3], k_stride[3], v_stride[3];  // batch, token, head, in elements
  int64_t table_stride, mask_stride, pages;
  int batch, drafted, heads, kv_heads, group, dim, page, columns;
  int rows, row_blocks, ctas;
  int box;                                   // rows of a tiled copy, or 0: none fits the pages
  CUtensorMap k_map, v_map;
  float scale_log2;                          // positive
  uint32_t negate;                           // the scale is negative: Q counts with its sign changed
  uint32_t polls;                            // of a wait
  bool wide;                                 // rows of the output are 32-byte aligned
  // With a window a drafted token's place is its sequence's length and its depth; it sees the last `window` places, its own
  // among them, and the first `sinks`.
  int window, sinks;
  const int* depths;                         // [batch or 1][drafted], or null: i
  int64_t depth_stride;
};

// A sequence's cached tokens and then its drafted ones, in tiles; kRows rows of one key head
struct Unit {
  int b, head, block;
  int length, tiles;
  bool bad;             // the sequence's length is none that its page table can hold
  // with a window: tiles of sinks, how many tiles behind them nobody sees, the first token that a token of depth 0 sees
  int sink_tiles, skipped, from;
};

template <bool kWindow>
__device__ __forceinline__ void read_length(const TreeParams& p, Unit& u) {
  const int n = u.b < p.batch ? p.lengths[u.b] : 0;
  u.bad = n < 0 || n > p.columns * p.page;
  u.length = u.bad ? 0 : n;
  u.tiles = (u.length + p.drafted + kTile - 1) / kTile;
  if (kWindow) {
    u.from = max(0, u.length - p.window + 1);
    u.sink_tiles = min((p.sinks - 1) / kTile + (p.sinks > 0), u.from / kTile);
    u.skipped = u.from / kTile - u.sink_tiles;
    u.tiles -= u.skipped;
  }
}

// where a unit's tile begins in its sequence
template <bool kWindow>
__device__ __forceinline__ int tile_token(const Unit& u, int tile) {
  return kTile * (!kWindow || tile < u.sink_tiles ? tile : tile + u.skipped);
}

// with a window: the drafted token's depth, and the first token that it sees but for the sinks
__device__ __forceinline__ int depth_of(const TreeParams& p, int b, int i) {
  return p.depths == nullptr ? i : min(max(p.depths[b * p.depth_stride + i], 0), (1 << 30) - 1);
}
__device__ __forceinline__ int seen_from(const TreeParams& p, const Unit& u, int depth) { return u.length + depth - p.window + 1; }
// ... whether it sees drafted token d, which its mask names
__device__ __forceinline__ bool reaches(const TreeParams& p, const Unit& u, int depth, int d) {
  const int at = depth_of(p, u.b, d);
  return depth - at < p.window || u.length + at < p.sinks;
}
// Whether drafted token `token` sees the cached or drafted token t of its sequence; d = t - length, the drafted one's number
template <bool kWindow>
__device__ __forceinline__ bool sees_token(const TreeParams& p, const Unit& u, const uint8_t* mask, int token, int depth, int d) {
  if (d < 0) return !kWindow || u.length + d >= seen_from(p, u, depth) || u.length + d < p.sinks;
  if (d >= p.drafted || token < 0) return false;
  return (mask == nullptr ? d <= token : mask[d] != 0) && (!kWindow || reaches(p, u, depth, d));
}
// ... the first token from `from` on that all drafted ones of a warp's sequence see: tokens before it are not seen by the deepest
__device__ __forceinline__ int seen_by_all(const TreeParams& p, const Unit& u) {
  int most = p.depths == nullptr ? p.drafted - 1 : 0;
  if (p.depths != nullptr) {
    for (int i = threadIdx.x & 31; i < p.drafted; i += 32) most = max(most, depth_of(p, u.b, i));
    most = int(__reduce_max_sync(0xffffffffu, unsigned(most)));
  }
  return max(0, seen_from(p, u, most));
}

template <bool kWindow>
__device__ __forceinline__ void next_unit(const TreeParams& p, Unit& u) {
  if (++u.block < p.row_blocks) return;
  u.block = 0;
  if (++u.head < p.kv_heads) return;
  u.head = 0;
  ++u.b;
  read_length<kWindow>(p, u);
}

// tiles of sequence b, for all its key heads and blocks of rows
template <bool kWindow>
__device__ __forceinline__ int64_t tiles_of(const TreeParams& p, int b) {
  Unit u{b, 0, 0, 0, 0, false, 0, 0, 0};
  read_length<kWindow>(p, u);
  return int64_t(u.tiles) * p.kv_heads * p.row_blocks;
}

// CTAs that have a part of `total` tiles: each of them a tile at least
__device__ __forceinline__ int64_t sharing(const TreeParams& p, int64_t total) { return total < p.ctas ? total : p.ctas; }

// Sum over all threads of the CTA (every one of them gets it) and of those before this one
template <int kWarps>
__device__ __forceinline__ int64_t cta_scan(int64_t x, int64_t* before, int64_t* shared) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t sum = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += y;
  }
  __syncthreads();
  if (lane == 31) shared[warp] = sum;
  __syncthreads();
  int64_t total = 0, earlier = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w == warp) earlier = total;
    total += shared[w];
  }
  *before = earlier + sum - x;
  return total;
}

// This CTA's part of all tiles: its first unit and tile, and how many tiles; false if there are fewer tiles than CTAs.
template <int kWarps>
struct Share { int64_t scan[kWarps], found[2]; };
template <bool kWindow, int kWarps>
__device__ __forceinline__ bool part_of_cta(const TreeParams& p, Share<kWarps>& shared, Unit& u, int& tile, int& rest) {
  const int tid = threadIdx.x;
  int64_t total = 0, before, own = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 32 * kWarps) {
    own = b0 + tid < p.batch ? tiles_of<kWindow>(p, b0 + tid) : 0;
    total += cta_scan<kWarps>(own, &before, shared.scan);
  }
  const int64_t ctas = sharing(p, total);
  if (blockIdx.x >= ctas) return false;
  const int64_t begin = total * blockIdx.x / ctas, end = total * (blockIdx.x + 1) / ctas;
  int64_t base = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 32 * kWarps) {
    int64_t sum = total;
    if (p.batch > 32 * kWarps) {   // otherwise all of them have just been looked at
      own = b0 + tid < p.batch ? tiles_of<kWindow>(p, b0 + tid) : 0;
      sum = cta_scan<kWarps>(own, &before, shared.scan);
    }
    const int64_t from = base + before;
    if (own > 0 && begin >= from && begin < from + own) {  // one thread of all
      shared.found[0] = b0 + tid;
      shared.found[1] = begin - from;
    }
    base += sum;
    if (begin < base) break;
  }
  __syncthreads();
  u = Unit{int(shared.found[0]), 0, 0, 0, 0, false, 0, 0, 0};
  read_length<kWindow>(p, u);
  const int64_t unit = shared.found[1] / u.tiles;
  tile = int(shared.found[1] - unit * u.tiles);
  u.head = int(unit / p.row_blocks);
  u.block = int(unit - int64_t(u.head) * p.row_blocks);
  rest = int(end - begin);
  return true;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// Arrives on an mbarrier, which counts on it, when all copies of this thread so far have.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(tc::smem_u32(bar)) : "memory");
}

// both chains
__device__ __forceinline__ void sync_chains() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// The key of a page number outside the cache: 128 channels of NaN, in either type
#define GDN2_NAN4 {~0u, ~0u, ~0u, ~0u}
__device__ const uint4 g_nan_row[16] = {GDN2_NAN4, GDN2_NAN4, GDN2_NAN4, GDN2_NAN4, GDN2_NAN4, GDN2_NAN4, GDN2_NAN4, GDN2_NAN4,
                                        GDN2_NAN4, GDN2_NAN4, GDN2_NAN4, GDN2_NAN4, GDN2_NAN4, GDN2_NAN4, GDN2_NAN4, GDN2_NAN4};
#undef GDN2_NAN4

// A warp copies 32 rows of DP channels, half of it or a quarter a row at a time: `at` is where row `first + lane` is, null
// for zeros.
template <int DP>
__device__ __forceinline__ void copy_rows(uint32_t base, uint32_t slab, int first, int dim, const void* at) {
  constexpr int kPieces = DP / 8, kAtOnce = 32 / kPieces;
  const int lane = threadIdx.x & 31, piece = lane % kPieces, sub = lane / kPieces;
  const uint64_t anything = reinterpret_cast<uintptr_t>(g_nan_row);   // an address for copies of nothing
  const uint32_t lo = uint32_t(reinterpret_cast<uintptr_t>(at)), hi = uint32_t(reinterpret_cast<uintptr_t>(at) >> 32);
#pragma unroll
  for (int i = 0; i < 32; i += 8 * kAtOnce) {
    uint64_t row[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const int r = i + x * kAtOnce + sub;
      row[x] = (uint64_t(__shfl_sync(0xffffffffu, hi, r)) << 32) | __shfl_sync(0xffffffffu, lo, r);
    }
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const bool there = piece * 8 < dim && row[x] != 0;
      cp_async16(place_of<DP>(base, slab, first + i + x * kAtOnce + sub, piece),
                 reinterpret_cast<const uint8_t*>(there ? row[x] : anything) + piece * 16, there);
    }
  }
}

// a tiled copy into shared memory that is given by its address there
__device__ __forceinline__ void tma_load_page(uint32_t to, const CUtensorMap* map, int c, int head, int row, int page,
                                              uint64_t* full, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %7, 0;\n\t"
      "@q cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
      "[%1, {%2, %3, %4, %5}], [%6];\n\t}"
      ::"r"(to), "l"(map), "r"(c), "r"(head), "r"(row), "r"(page), "r"(tc::smem_u32(full)), "r"(leader)
      : "memory");
}

// The keys and values of all tiles of a CTA, brought in by kWarps warps that share the rows of every tile, in the order K0,
// K1 V0, K2 V1, ... of a unit, into kStages places by turns.  full[] counts all their threads, empty[] says that a place has
// been used.  *strange says that a drafted token had a value that is not finite, strange_rows (may be null) which: a bit for
// every token modulo kStrangeRows.  With a window the cached tokens that some of the drafted ones see and some do not are
// looked at like these (numbered back from the first drafted one), and those that none of them sees are not read.
constexpr int kStrangeRows = 2048;
template <typename T, int DP, bool kWindow, int kStages, int kWarps>
__device__ __forceinline__ void bring_tiles(const TreeParams& p, Unit u, int tile, int rest, int warp, uint32_t kv_base, uint64_t* full,
                                            uint64_t* empty, const attn::Waiter& waiter, int* strange, uint32_t* strange_rows) {
  constexpr int kTileBytes = kTile * DP * 2;
  constexpr uint32_t kSlab = kTile * 128;
  constexpr int kMine = kTile / kWarps, kParts = kMine / 32;
  const int mine = warp * kMine, lane = threadIdx.x & 31;
  const uint32_t leader = tc::elect_leader();
  int filled = 0;
  bool ok = true;
  int all_from = kWindow ? seen_by_all(p, u) : 0;
  struct Pages { int of[kParts]; };    // of rows mine + lane, mine + 32 + lane, ... of a tile
  auto pages_of = [&](const Unit& x, int tile) {
    Pages r;
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const int t = tile_token<kWindow>(x, tile) + mine + i * 32 + lane;
      r.of[i] = t < x.length ? p.table[x.b * p.table_stride + t / p.page] : 0;
    }
    return r;
  };
  auto fetch = [&](bool keys, int tile, const Pages& pages) {
    const int s = filled % kStages;
    if (filled >= kStages) ok = waiter.wait(&empty[s], (filled / kStages - 1) & 1);
    if (!ok) return;
    ++filled;
    const uint32_t base = kv_base + s * kTileBytes;
    const int t0 = tile_token<kWindow>(u, tile) + mine;
    // whether some of these tokens are not seen by all drafted ones, whether some of those are seen by some
    const bool edge = kWindow && t0 < all_from && t0 + kMine > p.sinks;
    const bool sifted = edge && max(t0, max(u.from, p.sinks)) < min(t0 + kMine, all_from);
    bool good = !edge;
#pragma unroll
    for (int i = 0; i < kParts; ++i) good = good && pages.of[i] >= 0 && pages.of[i] < p.pages;
    if (p.box > 0 && t0 + kMine <= u.length && __all_sync(0xffffffffu, good)) {
      // all cached: boxes of p.box rows, of which none reaches into another page
      if (leader) tc::mbar_arrive_expect_tx(&full[s], kMine * DP * 2);
      else tc::mbar_arrive(&full[s]);
#pragma unroll
      for (int i = 0; i < kParts; ++i) {
        for (int r = 0; r < 32; r += p.box) {
          const int page = __shfl_sync(0xffffffffu, pages.of[i], r), row = (t0 + i * 32 + r) % p.page;
#pragma unroll
          for (int slab = 0; slab < DP / 64; ++slab) {
            tma_load_page(base + slab * kSlab + uint32_t(mine + i * 32 + r) * 128u, keys ? &p.k_map : &p.v_map, slab * 64, u.head, row, page, &full[s],
                          leader);
          }
        }
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      const int t = t0 + i * 32 + lane, j = t - u.length;
      const uint8_t* at = nullptr;
      if (edge && t < u.from && t >= p.sinks) {
        // zeros
      } else if (j < 0) {
        const int64_t row = (int64_t(pages.of[i]) * p.page + t % p.page) * p.kv_heads + u.head;
        if (pages.of[i] >= 0 && pages.of[i] < p.pages) at = static_cast<const uint8_t*>(keys ? p.k_pages : p.v_pages) + row * p.dim * 2;
        else if (keys) at = reinterpret_cast<const uint8_t*>(g_nan_row);
      } else if (j < p.drafted) {
        const int64_t* stride = keys ? p.k_stride : p.v_stride;
        at = static_cast<const uint8_t*>(keys ? p.k : p.v) + 2 * (u.b * stride[0] + j * stride[1] + u.head * stride[2]);
      }
      copy_rows<DP>(base, kSlab, mine + i * 32, p.dim, at);
    }
    if (!keys && (sifted || t0 + kMine > u.length)) {
      cp_async_wait_all();
      // a drafted token's values that are not finite are added to the rows that see them
      attn::sift<T, DP>(base, kSlab, mine + (sifted ? 0 : max(0, u.length - t0)), mine + kMine, [&](int row) {
        *static_cast<volatile int*>(strange) = 1;
        const int d = t0 - mine + row - u.length;
        if (strange_rows != nullptr) atomicOr(&strange_rows[(d & (kStrangeRows - 1)) >> 5], 1u << (d & 31));
      });
      tc::mbar_arrive(&full[s]);
    } else {
      cp_async_arrive(&full[s]);
    }
  };
  Pages pages = pages_of(u, tile);
  while (rest > 0 && ok) {
    const int n = min(rest, u.tiles - tile);
    Unit next = u;
    if (rest > n) next_unit<kWindow>(p, next);
    Pages before = pages;
    for (int x = 0; x <= n && ok; ++x) {
      const Pages now = pages;
      if (x < n) {
        pages = x + 1 < n ? pages_of(u, tile + x + 1) : pages_of(next, 0);   // looked up a tile ahead
        fetch(true, tile + x, now);
      }
      if (x > 0 && ok) fetch(false, tile + x - 1, before);
      before = now;
    }
    rest -= n;
    tile = 0;
    if (kWindow && next.b != u.b && rest > 0) all_from = seen_by_all(p, next);
    u = next;
  }
  cp_async_wait_all();
  if (!ok) {  // tiled copies under way end before the CTA does
    for (int back = 1; back <= kStages && back <= filled; ++back) {
      const int x = filled - back;
      for (int i = 0; i < 4096 && !tc::mbar_try_wait(&full[x % kStages], (x / kStages) & 1); ++i) {}
    }
  }
}

// With a window: where the values of token d (counted from the first drafted one) are, if drafted token `token` sees it, if it
// is one that not all see (only those were taken out of their tiles) and in the tiles tile .. tile + n - 1; null otherwise
template <typename T>
__device__ __noinline__ const T* strange_value(const TreeParams& p, const Unit& u, const uint8_t* mask, int token, int depth, int d, int tile,
                                               int n) {
  const int t = u.length + d, t0 = t / kTile * kTile;
  // its tile is one of the unit's, and this CTA's
  const int of_unit = t0 / kTile < u.sink_tiles ? t0 / kTile : t0 / kTile - u.skipped;
  if (of_unit < tile || of_unit >= tile + n || tile_token<true>(u, of_unit) != t0) return nullptr;
  if (!sees_token<true>(p, u, mask, token, depth, d)) return nullptr;
  if (d >= 0) return static_cast<const T*>(p.v) + u.b * p.v_stride[0] + d * p.v_stride[1] + u.head * p.v_stride[2];
  const int page = p.table[u.b * p.table_stride + t / p.page];
  if (page < 0 || page >= p.pages) return nullptr;
  return static_cast<const T*>(p.v_pages) + ((int64_t(page) * p.page + t % p.page) * p.kv_heads + u.head) * p.dim;
}

template <int DP, int RT>   // RT: tiles of 128 rows that a CTA has, 1 or 2
struct TreeConfig {
  static constexpr int kTileBytes = kTile * DP * 2;
  static constexpr int kSlab = kTile * 128;                    // 64 channels of 128 rows
  static constexpr int kRows = 128 * RT;
  // Queries of two units, so that the copies need not wait between two; those of 256 rows of 128 channels leave no room.
  static constexpr int kQueries = RT == 2 ? 1 : 2;
  static constexpr int kStages = DP == 64 ? 8 : 5;
  static constexpr int kBytes = RT * kQueries * kTileBytes + kStages * kTileBytes + 768 + 2048;
};

struct TreeBars {
  uint64_t s_full[2], p_ready[2], o_full[2], q_full[2], q_empty[2], drained;
  uint64_t kv_full[8], kv_empty[8];
  Share<kThreads / 32> share;
  uint32_t tmem;
  int failed;
  int strange;          // a drafted value was infinite or NaN
  uint32_t strange_rows[kStrangeRows / 32];
};
static_assert(sizeof(TreeBars) <= 768, "");

template <typename T, int DP, int RT, bool kWindow>
__global__ void __launch_bounds__(kThreads, 1) tree_kernel(const __grid_constant__ TreeParams p) {
  using C = TreeConfig<DP, RT>;
  extern __shared__ __align__(1024) uint8_t smem[];   // swizzled tiles: 1024-byte aligned, there is no static shared memory
  const uint32_t q_base = tc::smem_u32(smem), kv_base = q_base + RT * C::kQueries * C::kTileBytes;
  TreeBars& bar = *reinterpret_cast<TreeBars*>(smem + RT * C::kQueries * C::kTileBytes + C::kStages * C::kTileBytes);
  // (m, l) of the rows of two chains
  float2(*told)[128] = reinterpret_cast<float2(*)[128]>(smem + RT * C::kQueries * C::kTileBytes + C::kStages * C::kTileBytes + 768);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (tid == 0) {
    for (int t = 0; t < 2; ++t) {
      tc::mbar_init(&bar.s_full[t], 1);
      tc::mbar_init(&bar.p_ready[t], 4);
      tc::mbar_init(&bar.o_full[t], 1);
    }
    for (int x = 0; x < C::kQueries; ++x) {
      tc::mbar_init(&bar.q_full[x], 32);
      tc::mbar_init(&bar.q_empty[x], 1);
    }
    tc::mbar_init(&bar.drained, 1);
    for (int s = 0; s < C::kStages; ++s) {
      tc::mbar_init(&bar.kv_full[s], 128);
      tc::mbar_init(&bar.kv_empty[s], 1);
    }
    bar.failed = bar.strange = 0;
    tc::fence_mbar_init();
  }
  if (tid < kStrangeRows / 32) bar.strange_rows[tid] = 0;
  if (warp == 12) {
    tc::tmem_alloc(&bar.tmem, 512);
    tc::tmem_relinquish();
  }
  Unit u;
  int tile, rest;   // the first of this CTA's tiles of the unit; how many there are left of all its tiles
  const bool idle = !part_of_cta<kWindow, kThreads / 32>(p, bar.share, u, tile, rest);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = bar.tmem;
  if (idle) {
    if (warp == 12) tc::tmem_dealloc(tmem, 512);
    return;
  }
  const attn::Waiter waiter{&bar.failed, p.polls};
  // tiles of 128 rows that a unit has
  auto row_tiles = [&](const Unit& x) { return RT == 2 && p.rows - x.block * C::kRows > 128 ? 2 : 1; };

  // 512 threads of 128 registers = 256 of 168 + 256 of 88
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 12) {
      // ---- products --------------------------------------------------------------------------------------
      const uint32_t leader = tc::elect_leader();
      const uint32_t id_s = tc::idesc(128, 128, Format<T>::code, tc::kMajorK, tc::kMajorK, p.negate);
      const uint32_t id_o = tc::idesc(128, DP, Format<T>::code, tc::kMajorK, tc::kMajorMN);
      int used = 0, p_used[2] = {0, 0}, units = 0, queries = 0;   // which of the kQueries
      bool ok = true;
      auto full = [&](int x) {
        const bool r = waiter.wait(&bar.kv_full[x % C::kStages], (x / C::kStages) & 1);
        tc::fence_async_smem();   // what the copies wrote is read by the products
        return r;
      };
      auto scores = [&](int t, int x) {   // S_t from the keys in stage x
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
          attn::mma_ss(tmem + t * 128, attn::desc_k(q_base + (RT == 2 ? t : queries) * C::kTileBytes, C::kSlab, ks),
                       attn::desc_k(kv_base + (x % C::kStages) * C::kTileBytes, C::kSlab, ks), id_s, ks > 0, leader);
        }
        tc::mma_commit(&bar.s_full[t], leader);
      };
      auto outputs = [&](int t, int x, bool first) {   // O_t += P_t V
        if (!waiter.wait(&bar.p_ready[t], p_used[t] & 1)) return false;
        ++p_used[t];
        tc::tc_fence_after();
#pragma unroll
        for (int ks = 0; ks < kTile / 16; ++ks) {
          attn::mma_ts(tmem + 256 + t * 128, tmem + t * 128 + ks * 8, attn::desc_mn(kv_base + (x % C::kStages) * C::kTileBytes, C::kSlab, ks),
                       id_o, !first || ks > 0, leader);
        }
        return true;
      };
      while (rest > 0 && ok) {
        const int n = min(rest, u.tiles - tile), chains = row_tiles(u);
        // the order of the copies is that of use: K0, K1 V0, K2 V1, ...
        auto k_of = [&](int j) { return used + max(2 * j - 1, 0); };
        auto v_of = [&](int j) { return used + min(2 * j + 2, 2 * n - 1); };
        if (!(ok = waiter.wait(&bar.q_full[queries], (units / C::kQueries) & 1))) break;
        if (RT == 1) {
          // chains by turns: S(j + 2) is issued behind O += P(j) V, whose P lies in its place
          for (int j = 0; j < min(n, 2) && ok; ++j) {
            if (!(ok = full(k_of(j)))) break;
            scores(j, k_of(j));
            tc::mma_commit(&bar.kv_empty[k_of(j) % C::kStages], leader);
          }
          if (n <= 2) tc::mma_commit(&bar.q_empty[queries], leader);
          for (int j = 0; j < n && ok; ++j) {
            const int t = j & 1, xv = v_of(j), xk = k_of(j + 2);
            if (!(ok = full(xv)) || !(ok = outputs(t, xv, j < 2))) break;
            tc::mma_commit(&bar.kv_empty[xv % C::kStages], leader);
            if (j + 2 >= n) {
              tc::mma_commit(&bar.o_full[t], leader);
            } else {
              if (!(ok = full(xk))) break;
              scores(t, xk);
              tc::mma_commit(&bar.kv_empty[xk % C::kStages], leader);
              if (j + 3 == n) tc::mma_commit(&bar.q_empty[queries], leader);
            }
          }
        } else {
          if (!(ok = full(used))) break;
          for (int t = 0; t < chains; ++t) scores(t, used);
          tc::mma_commit(&bar.kv_empty[used % C::kStages], leader);
          if (n == 1) tc::mma_commit(&bar.q_empty[queries], leader);
          for (int j = 0; j < n && ok; ++j) {
            const int xv = v_of(j), xk = k_of(j + 1);
            if ((j + 1 < n && !(ok = full(xk))) || !(ok = full(xv))) break;
            for (int t = 0; t < chains && ok; ++t) {
              if (!(ok = outputs(t, xv, j == 0))) break;
              if (j + 1 == n) tc::mma_commit(&bar.o_full[t], leader);
              if (t + 1 == chains) tc::mma_commit(&bar.kv_empty[xv % C::kStages], leader);
              if (j + 1 < n) scores(t, xk);
            }
            if (j + 1 < n) tc::mma_commit(&bar.kv_empty[xk % C::kStages], leader);
            if (j + 2 == n) tc::mma_commit(&bar.q_empty[queries], leader);
          }
        }
        used += 2 * n;
        ++units;
        if (++queries == C::kQueries) queries = 0;
        rest -= n;
        tile = 0;
        if (rest > 0) next_unit<kWindow>(p, u);
      }
      if (!ok) {  // products under way end before the CTA does
        tc::mma_commit(&bar.drained, leader);
        for (int i = 0; i < 4096 && !tc::mbar_try_wait(&bar.drained, 0); ++i) {}
      }
      __syncwarp();
    } else if (warp == 13) {
      // ---- queries ---------------------------------------------------------------------------------------
      int units = 0;
      while (rest > 0) {
        const int n = min(rest, u.tiles - tile), place = units % C::kQueries;
        if (units >= C::kQueries && !waiter.wait(&bar.q_empty[place], (units / C::kQueries - 1) & 1)) break;
        ++units;
        for (int x = 0; x < RT * 128; x += 32) {
          const int r = u.block * C::kRows + x + lane;
          const int i = r / p.group, g = r - i * p.group;
          const T* at = static_cast<const T*>(p.q) + u.b * p.q_stride[0] + i * p.q_stride[1] + int64_t(u.head * p.group + g) * p.q_stride[2];
          copy_rows<DP>(q_base + (RT == 2 ? x / 128 : place) * C::kTileBytes, C::kSlab, x % 128, p.dim, r < p.rows ? at : nullptr);
        }
        cp_async_arrive(&bar.q_full[place]);
        rest -= n;
        tile = 0;
        if (rest > 0) next_unit<kWindow>(p, u);
      }
      cp_async_wait_all();
    } else if (warp < 12) {
      bring_tiles<T, DP, kWindow, C::kStages, 4>(p, u, tile, rest, warp - 8, kv_base, bar.kv_full, bar.kv_empty, waiter, &bar.strange,
                                                 bar.strange_rows);
    }
  } else {
    // ---- weights: a row a thread ---------------------------------------------------------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    const int t = warp >> 2, row = tid & 127;
    const uint32_t lane_base = uint32_t(warp & 3) << 21;   // 32 lanes of TMEM, in bits 16 and up
    const uint32_t s_at = tmem + lane_base + t * 128, o_at = tmem + lane_base + 256 + t * 128;
    int seen = 0, outs = 0;
    bool ok = true, split = tile != 0;   // the unit began in another CTA
    while (rest > 0) {
      const int n = min(rest, u.tiles - tile), chains = row_tiles(u);
      const int local = (RT == 2 ? t * 128 : 0) + row, r = u.block * C::kRows + local;   // row in the block, of all
      const int token = r / p.group;
      const bool there = r < p.rows, any_there = r - lane < p.rows;
      const bool takes_part = RT == 1 || t < chains;
      const int depth = kWindow && there ? depth_of(p, u.b, token) : 0;
      // a tile of tokens of which no warp's row misses any: behind the window's beginning and before the drafted ones
      const int all_from = kWindow ? max(0, seen_from(p, u, int(__reduce_max_sync(0xffffffffu, unsigned(depth))))) : 0;
      float m = -INFINITY;
      float sum = 0.f;
      int mine = 0;
      for (int j = RT == 1 ? t : 0; j < n && takes_part; j += RT == 1 ? 2 : 1) {
        if (!ok || !(ok = waiter.wait(&bar.s_full[t], seen & 1))) break;
        ++seen;
        tc::tc_fence_after();
        if (any_there) {   // warps without a row have nothing to do but to keep count
          const int first_token = tile_token<kWindow>(u, tile + j);
          attn::soften<T, DP>(s_at, o_at, p.scale_log2, m, sum, [&](int x, uint32_t (&s)[32]) {
            if (first_token + x * 32 + 32 <= u.length) {
              if (!kWindow || first_token + x * 32 >= all_from || first_token + x * 32 + 32 <= p.sinks) return;
              // (rows that are not there have a depth of 0; nothing but their zeros comes of them)
              const attn::Span span{p.window, p.sinks};
              span.hide(u.length + depth, first_token + x * 32, s);
              return;
            }
            // drafted tokens, or the end
            const uint8_t* mask = p.mask == nullptr || !there ? nullptr : p.mask + u.b * p.mask_stride + int64_t(token) * p.drafted;
            uint32_t sees = 0;
#pragma unroll 8
            for (int y = 0; y < 32; ++y) {
              const int d = first_token + x * 32 + y - u.length;
              bool see = d < 0;
              if (kWindow) see = sees_token<true>(p, u, mask, there ? token : -1, depth, d);
              else if (!see && d < p.drafted && there) see = p.mask == nullptr ? d <= token : mask[d] != 0;
              sees |= uint32_t(see) << y;
            }
#pragma unroll
            for (int y = 0; y < 32; ++y) {
              if (!((sees >> y) & 1)) s[y] = 0xff800000u;
            }
          });
        }
        ++mine;
        tc::tc_fence_before();
        __syncwarp();
        tc::mbar_arrive(&bar.p_ready[t], lane == 0);
      }
      if (mine > 0) {
        if (ok) ok = waiter.wait(&bar.o_full[t], outs & 1);
        ++outs;
      }
      tc::tc_fence_after();
      // the columns of this thread: all of its row's, or where both chains have the row a half of the sum of both
      constexpr int kCols = RT == 1 ? DP / 2 : DP;
      const int col0 = RT == 1 ? t * kCols : 0;
      float f[2] = {1.f, 1.f};
      bool has[2] = {true, true};
      if (RT == 1) {
        told[t][row] = make_float2(m, sum);
        tc::tc_fence_before();
        sync_chains();
        tc::tc_fence_after();
        const float m0 = told[0][row].x, m1 = told[1][row].x, l0 = told[0][row].y, l1 = told[1][row].y;
        m = fmaxf(m0, m1);
        has[1] = n > 1;
        f[0] = attn::factor_to(m0, m, p.scale_log2);
        f[1] = attn::factor_to(m1, m, p.scale_log2);
        sum = l0 * f[0] + l1 * f[1];
        if (isnan(l0) || isnan(l1)) sum = NAN;
      }
      ok = ok && waiter.nobody_failed();
      const bool whole = !split && tile + n == u.tiles;
      // nothing seen: the sum is 0 and so is the output
      const float inv = !ok || u.bad ? NAN : !whole ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
      const int64_t slot = int64_t(blockIdx.x) * 2 + (split ? 0 : 1);
      float* part = p.partials + (slot * C::kRows + local) * DP;
      const bool strange = *static_cast<volatile int*>(&bar.strange) != 0;
      if (takes_part && any_there) {
        const int g = r - token * p.group;
        T* to = static_cast<T*>(p.out) + (int64_t(u.b) * p.drafted + token) * p.heads * p.dim + int64_t(u.head * p.group + g) * p.dim;
#pragma unroll 1
        for (int x = col0; x < col0 + kCols; x += 16) {
          uint32_t raw[16];
          float o[16];
          tc::tmem_ld16(tmem + lane_base + 256 + (RT == 1 ? 0 : t * 128) + x, raw);
          tc::tmem_wait_ld();
#pragma unroll
          for (int y = 0; y < 16; ++y) o[y] = __uint_as_float(raw[y]);
          if (RT == 1) {
#pragma unroll
            for (int y = 0; y < 16; ++y) o[y] *= f[0];
            if (has[1]) {
              tc::tmem_ld16(tmem + lane_base + 256 + 128 + x, raw);
              tc::tmem_wait_ld();
#pragma unroll
              for (int y = 0; y < 16; ++y) o[y] = fmaf(__uint_as_float(raw[y]), f[1], o[y]);
            }
          }
          if (!there) continue;
          if (strange) {
            // of the drafted tokens in this CTA's tiles of the unit those that had such a value in some unit; with a window
            // the cached ones, too, that not all of the drafted ones see
            const int first = kWindow ? max(u.from - 31, 0) - u.length : max(0, tile_token<kWindow>(u, tile) - u.length);
            const int last = min(p.mask == nullptr ? token + 1 : p.drafted, tile_token<kWindow>(u, tile + n - 1) + kTile - u.length);
            const uint8_t* mask = p.mask == nullptr ? nullptr : p.mask + u.b * p.mask_stride + int64_t(token) * p.drafted;
            bool done = false;          // all channels are NaN
            for (int d0 = first & ~31; d0 < last && !done; d0 += 32) {
              for (uint32_t bits = bar.strange_rows[(d0 & (kStrangeRows - 1)) >> 5]; bits != 0 && !done; bits &= bits - 1) {
                const int d = d0 + __ffs(bits) - 1;
                if (d < first || d >= last) continue;
                const T* v = nullptr;
                if (kWindow) {
                  v = strange_value<T>(p, u, mask, token, depth, d, tile, n);
                  if (v == nullptr) continue;
                  v += x;
                } else {
                  if (mask != nullptr && mask[d] == 0) continue;
                  v = static_cast<const T*>(p.v) + u.b * p.v_stride[0] + d * p.v_stride[1] + u.head * p.v_stride[2] + x;
                }
#pragma unroll
                for (int y = 0; y < 16; y += 8) {
                  if (x + y >= p.dim) continue;
                  const uint4 raw = *reinterpret_cast<const uint4*>(v + y);
                  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                  for (int z = 0; z < 4; ++z) {
                    const float2 value = unpack2<T>(w[z]);
                    if (!isfinite(value.x)) o[y + 2 * z] += value.x;
                    if (!isfinite(value.y)) o[y + 2 * z + 1] += value.y;
                  }
                }
                done = true;
#pragma unroll
                for (int y = 0; y < 16; ++y) done = done && isnan(o[y]);
              }
            }
          }
          if (whole) {
            attn::store_row16<T>(to + x, o, inv, p.dim - x, p.wide);
          } else {
#pragma unroll
            for (int y = 0; y < 16; y += 4) *reinterpret_cast<float4*>(part + x + y) = make_float4(o[y], o[y + 1], o[y + 2], o[y + 3]);
          }
        }
        if (!whole && there && col0 == 0) {
          float* ml = p.partials + int64_t(p.ctas) * 2 * C::kRows * DP + (slot * C::kRows + local) * 2;
          *reinterpret_cast<float2*>(ml) = make_float2(m, inv * sum);
        }
      }
      tc::tc_fence_before();
      if (RT == 1) sync_chains();   // the other chain has read this one's O, m and l
      rest -= n;
      tile = 0;
      split = false;
      if (rest > 0) next_unit<kWindow>(p, u);
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

// ---- few rows ------------------------------------------------------------------------------------------
// Up to 16 rows (plain decoding, small trees of small groups): mma.sync m16n8k16, whose sums are in registers: no product has
// more rows than there are, and no score goes through TMEM to a few lanes.  Eight warps have 16 tokens of every tile each and
// go through them on their own; what they have of a unit is joined at its end.  Decoding 64 sequences of up to 8192 tokens,
// 8 key heads: 210 us, 6.45 TB/s of the copy rate's 6.53 (a call in a loop, with the join of the parts, 217 to 227).  (Copies
// by the computing warps themselves: 31 us more.)
constexpr int kFewThreads = 384;   // warps 0-7: 16 tokens of every tile each; 8-11: copies

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int DP>
struct FewConfig {
  static constexpr int kTileBytes = kTile * DP * 2;
  static constexpr uint32_t kSlab = kTile * 128;
  static constexpr int kStages = DP == 128 ? 6 : 10;
  static constexpr int kJoinBytes = 4 * 16 * DP * 4;   // what four warps leave for four others
  static constexpr int kBytes = kStages * kTileBytes + kJoinBytes + 2048;
};
struct FewBars {
  uint64_t kv_full[10], kv_empty[10];
  Share<kFewThreads / 32> share;
  int failed, strange;
  float m[8][16], l[8][16];
};
static_assert(sizeof(FewBars) <= 2048, "");

template <typename T, int DP, bool kWindow>
__global__ void __launch_bounds__(kFewThreads, 1) tree_few_kernel(const __grid_constant__ TreeParams p) {
  using C = FewConfig<DP>;
  constexpr int kKSteps = DP / 16, kDB = DP / 8;
  extern __shared__ __align__(1024) uint8_t smem[];   // swizzled tiles: 1024-byte aligned, there is no static shared memory
  const uint32_t kv_base = tc::smem_u32(smem);
  float* join = reinterpret_cast<float*>(smem + C::kStages * C::kTileBytes);
  FewBars& bar = *reinterpret_cast<FewBars*>(smem + C::kStages * C::kTileBytes + C::kJoinBytes);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int quad = lane >> 2, in_quad = lane & 3;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      tc::mbar_init(&bar.kv_full[s], 128);
      tc::mbar_init(&bar.kv_empty[s], 8);
    }
    bar.failed = bar.strange = 0;
    tc::fence_mbar_init();
  }
  Unit u;
  int tile, rest;
  if (!part_of_cta<kWindow, kFewThreads / 32>(p, bar.share, u, tile, rest)) return;
  const attn::Waiter waiter{&bar.failed, p.polls};
  if (warp >= 8) {
    bring_tiles<T, DP, kWindow, C::kStages, 4>(p, u, tile, rest, warp - 8, kv_base, bar.kv_full, bar.kv_empty, waiter, &bar.strange, nullptr);
    return;
  }

  uint32_t qf[kKSteps][4];
  const uint32_t sign = p.negate ? 0x80008000u : 0u;   // the scale's goes to the queries
  int token_of[2];
  int depth[2] = {0, 0}, all_from = 0;   // with a window: depths of the two tokens, the first token that all rows see
  auto queries = [&](const Unit& x) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int r = quad + 8 * half;
      const bool there = r < p.rows;
      const int n = there ? r / p.group : 0, g = there ? r - n * p.group : 0;
      token_of[half] = there ? n : -1;
      if (kWindow) depth[half] = there ? depth_of(p, x.b, n) : 0;
      const T* row = static_cast<const T*>(p.q) + x.b * p.q_stride[0] + n * p.q_stride[1] + int64_t(x.head * p.group + g) * p.q_stride[2];
#pragma unroll
      for (int s = 0; s < kKSteps; ++s) {
#pragma unroll
        for (int kh = 0; kh < 2; ++kh) {
          const int col = s * 16 + kh * 8 + in_quad * 2;
          qf[s][kh * 2 + half] = (there && col < p.dim ? *reinterpret_cast<const uint32_t*>(row + col) : 0u) ^ sign;
        }
      }
    }
    if (kWindow) all_from = max(0, seen_from(p, x, int(__reduce_max_sync(0xffffffffu, unsigned(max(depth[0], depth[1]))))));
  };
  queries(u);
  const float c = p.scale_log2;
  // where this lane's part of an ldmatrix begins: rows of this warp's 16 tokens
  const int k_row = warp * 16 + (lane & 7) + ((lane >> 4) << 3), v_row = warp * 16 + (lane & 15);
  int used = 0;
  bool ok = true, split = tile != 0;   // the unit began in another CTA
  while (rest > 0) {
    const int n = min(rest, u.tiles - tile);
    float o[kDB][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int d = 0; d < kDB; ++d) { o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f; }
    for (int j = 0; j < n && ok; ++j) {
      const int xk = used + max(2 * j - 1, 0), xv = used + min(2 * j + 2, 2 * n - 1);
      if (!(ok = waiter.wait(&bar.kv_full[xk % C::kStages], (xk / C::kStages) & 1))) break;
      const uint32_t k_tile = kv_base + (xk % C::kStages) * C::kTileBytes, v_tile = kv_base + (xv % C::kStages) * C::kTileBytes;
      // S = Q K^T: two blocks of 8 tokens, two sums each
      float s2[2][2][4];
#pragma unroll
      for (int x = 0; x < 16; ++x) s2[x >> 3][(x >> 2) & 1][x & 3] = 0.f;
#pragma unroll
      for (int ks = 0; ks < kKSteps; ++ks) {
        uint32_t kf[4];  // tokens 0..7 and 8..15, channels ks*16 + 0..7 and 8..15
        ldmatrix4(kf, place_of<DP>(k_tile, C::kSlab, k_row, ks * 2 + ((lane >> 3) & 1)));
        mma16816<T>(s2[ks & 1][0], qf[ks], kf[0], kf[1]);
        mma16816<T>(s2[ks & 1][1], qf[ks], kf[2], kf[3]);
      }
      __syncwarp();
      tc::mbar_arrive(&bar.kv_empty[xk % C::kStages], lane == 0);
      const int first_token = tile_token<kWindow>(u, tile + j) + warp * 16;
      float s[2][4];
#pragma unroll
      for (int x = 0; x < 8; ++x) s[x >> 2][x & 3] = s2[0][x >> 2][x & 3] + s2[1][x >> 2][x & 3];
      // drafted tokens, or the end; tokens that not all rows see
      if (first_token + 16 > u.length || (kWindow && first_token < all_from && first_token + 16 > p.sinks)) {
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const int d = first_token + (x >> 2) * 8 + in_quad * 2 + (x & 1) - u.length, token = token_of[(x >> 1) & 1];
          bool see = d < 0;
          if (kWindow) {
            const uint8_t* mask = p.mask == nullptr ? nullptr : p.mask + u.b * p.mask_stride + int64_t(max(token, 0)) * p.drafted;
            see = sees_token<true>(p, u, mask, token, depth[(x >> 1) & 1], d);
          } else if (!see && d < p.drafted && token >= 0) {
            see = p.mask == nullptr ? d <= token : p.mask[u.b * p.mask_stride + int64_t(token) * p.drafted + d] != 0;
          }
          if (!see) s[x >> 2][x & 3] = -INFINITY;
        }
      }
      // running maximum and sum of the two rows of this thread's quad
      uint32_t pa[4];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float top = fmaxf(fmaxf(s[0][2 * half], s[0][2 * half + 1]), fmaxf(s[1][2 * half], s[1][2 * half + 1]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        if (__any_sync(0xffffffffu, top > m[half])) {
          const float now = fmaxf(m[half], top), keep = attn::factor_to(m[half], now, c);
          l[half] *= keep;
#pragma unroll
          for (int d = 0; d < kDB; ++d) { o[d][2 * half] *= keep; o[d][2 * half + 1] *= keep; }
          m[half] = now;
        }
        const attn::Reference ref = attn::reference(m[half], c);
        float w[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) w[x] = exp2_approx(fmaf(s[x >> 1][2 * half + (x & 1)] - ref.shift, c, -ref.scaled));
        l[half] += (w[0] + w[1]) + (w[2] + w[3]);   // (of this thread's columns; the quad's are added at the end)
        pa[half] = pack_pair<T>(w[0], w[1]);       // weights at most 1, rounded to the values' type for the product
        pa[2 + half] = pack_pair<T>(w[2], w[3]);
      }
      // O += P V
      if (!(ok = waiter.wait(&bar.kv_full[xv % C::kStages], (xv / C::kStages) & 1))) break;
#pragma unroll
      for (int d = 0; d < kDB; d += 2) {
        uint32_t vf[4];  // channels d*8.. (tokens 0..7, 8..15), channels (d+1)*8.. (the same)
        ldmatrix4_trans(vf, place_of<DP>(v_tile, C::kSlab, v_row, d + (lane >> 4)));
        mma16816<T>(o[d], pa, vf[0], vf[1]);
        mma16816<T>(o[d + 1], pa, vf[2], vf[3]);
      }
      __syncwarp();
      tc::mbar_arrive(&bar.kv_empty[xv % C::kStages], lane == 0);
    }
    used += 2 * n;
    Unit next = u;
    if (rest > n) {
      next_unit<kWindow>(p, next);
      queries(next);   // on their way while the warps join
    }

    // the eight warps' sums
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
      l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
      if (in_quad == 0) bar.m[warp][quad + 8 * half] = m[half];
    }
    auto sync = [] { asm volatile("bar.sync 1, 256;" ::: "memory"); };
    sync();
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int r = quad + 8 * half;
      float top = bar.m[0][r];
#pragma unroll
      for (int w = 1; w < 8; ++w) top = fmaxf(top, bar.m[w][r]);
      const float f = attn::factor_to(m[half], top, c);
      m[half] = top;
#pragma unroll
      for (int d = 0; d < kDB; ++d) { o[d][2 * half] *= f; o[d][2 * half + 1] *= f; }
      if (in_quad == 0) bar.l[warp][r] = isnan(l[half]) ? l[half] : l[half] * f;
    }
#pragma unroll
    for (int with = 4; with > 0; with >>= 1) {
      float2* at = reinterpret_cast<float2*>(join + (warp & (with - 1)) * 16 * DP);
      if (warp >= with && warp < 2 * with) {
#pragma unroll
        for (int x = 0; x < 2 * kDB; ++x) at[x * 32 + lane] = make_float2(o[x >> 1][2 * (x & 1)], o[x >> 1][2 * (x & 1) + 1]);
      }
      sync();
      if (warp < with) {
#pragma unroll
        for (int x = 0; x < 2 * kDB; ++x) {
          const float2 y = at[x * 32 + lane];
          o[x >> 1][2 * (x & 1)] += y.x;
          o[x >> 1][2 * (x & 1) + 1] += y.y;
        }
      }
      if (with > 1) sync();
    }
    if (warp == 0) {
      const bool whole = !split && tile + n == u.tiles, strange = *static_cast<volatile int*>(&bar.strange) != 0;
      const int64_t slot = int64_t(blockIdx.x) * 2 + (split ? 0 : 1);
      ok = ok && waiter.nobody_failed();   // none of the eight
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int r = quad + 8 * half;
        if (r >= p.rows) continue;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) sum += bar.l[w][r];
        // nothing seen: the sum is 0 and so is the output
        const float inv = !ok || u.bad ? NAN : !whole ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
        const int i = r / p.group, g = r - i * p.group;
        if (strange) {
          const int first = kWindow ? max(u.from - 31, 0) - u.length : max(0, tile * kTile - u.length);
          const int last = min(p.drafted, tile_token<kWindow>(u, tile + n - 1) + kTile - u.length);
          for (int d = first; d < last; ++d) {
            const uint8_t* mask = p.mask == nullptr ? nullptr : p.mask + u.b * p.mask_stride + int64_t(i) * p.drafted;
            const T* v;
            if (kWindow) {
              v = strange_value<T>(p, u, mask, i, depth_of(p, u.b, i), d, tile, n);
              if (v == nullptr) continue;
            } else {
              if (!(mask == nullptr ? d <= i : mask[d] != 0)) continue;
              v = static_cast<const T*>(p.v) + u.b * p.v_stride[0] + d * p.v_stride[1] + u.head * p.v_stride[2];
            }
#pragma unroll
            for (int x = 0; x < 2 * kDB; ++x) {
              const int col = (x >> 1) * 8 + in_quad * 2 + (x & 1);
              const float value = col < p.dim ? to_float(v[col]) : 0.f;
              if (!isfinite(value)) o[x >> 1][2 * half + (x & 1)] += value;
            }
          }
        }
        T* to = static_cast<T*>(p.out) + (int64_t(u.b) * p.drafted + i) * p.heads * p.dim + int64_t(u.head * p.group + g) * p.dim;
        float* part = p.partials + (slot * 16 + r) * DP;
#pragma unroll
        for (int d = 0; d < kDB; ++d) {
          const int col = d * 8 + in_quad * 2;
          const float2 y = make_float2(o[d][2 * half], o[d][2 * half + 1]);
          if (!whole) *reinterpret_cast<float2*>(part + col) = y;
          else if (col < p.dim) *reinterpret_cast<uint32_t*>(to + col) = pack_pair<T>(y.x * inv, y.y * inv);
        }
        if (!whole && in_quad == 0) {
          *reinterpret_cast<float2*>(p.partials + int64_t(p.ctas) * 2 * 16 * DP + (slot * 16 + r) * 2) = make_float2(m[half], inv * sum);
        }
      }
    }
    sync();   // what the warps told each other has been read
    rest -= n;
    tile = 0;
    split = false;
    u = next;
  }
}

// Joins what several CTAs have of a unit: a warp a row, in the order of the tiles.
template <typename T, int DP, bool kWindow>
__global__ void __launch_bounds__(kJoinThreads) tree_join_kernel(const __grid_constant__ TreeParams p, int block_rows, int ctas_of_unit) {
  __shared__ int64_t scan[kJoinThreads / 32];
  const int unit = int(blockIdx.x) / ctas_of_unit;
  const int block = unit % p.row_blocks, head = unit / p.row_blocks % p.kv_heads, b = unit / p.row_blocks / p.kv_heads;
  int64_t total = 0, from = 0, before;
  for (int b0 = 0; b0 < p.batch; b0 += kJoinThreads) {
    const int x = b0 + int(threadIdx.x);
    const int64_t own = x < p.batch ? tiles_of<kWindow>(p, x) : 0;
    total += cta_scan<kJoinThreads / 32>(own, &before, scan);
    from += cta_scan<kJoinThreads / 32>(x < b ? own : 0, &before, scan);
  }
  Unit u{b, 0, 0, 0, 0, false, 0, 0, 0};
  read_length<kWindow>(p, u);
  const int64_t t0 = from + (int64_t(head) * p.row_blocks + block) * u.tiles, t1 = t0 + u.tiles;
  const int64_t ctas = sharing(p, total), c0 = ((t0 + 1) * ctas - 1) / total, c1 = (t1 * ctas - 1) / total;
  // Until here only lengths were read, which stood before the other kernel began; the parts are there when it has ended
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (c0 == c1) return;   // one CTA had it all
  const int lane = threadIdx.x & 31;
  const int local = (int(blockIdx.x) - unit * ctas_of_unit) * (kJoinThreads / 32) + int(threadIdx.x >> 5);
  const int r = block * block_rows + local;
  if (local >= block_rows || r >= p.rows) return;
  const float* all_ml = p.partials + int64_t(p.ctas) * 2 * block_rows * DP;
  // the part of CTA i: its last unit where the unit began there, its first one otherwise
  auto row_of = [&](int64_t i) { return (i * 2 + (i == c0 ? 1 : 0)) * block_rows + local; };
  // a part a lane: the first 32 parts' m and l stay
  const float2 none = make_float2(-INFINITY, 0.f);
  auto part_ml = [&](int64_t i) { return i <= c1 ? *reinterpret_cast<const float2*>(all_ml + row_of(i) * 2) : none; };
  const float2 ml0 = part_ml(c0 + lane);
  float top = ml0.x;
  for (int64_t i = c0 + 32 + lane; i <= c1; i += 32) top = fmaxf(top, part_ml(i).x);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  constexpr int kOwn = DP / 32;
  float sum = 0.f, acc[kOwn];
#pragma unroll
  for (int y = 0; y < kOwn; ++y) acc[y] = 0.f;
  for (int64_t i0 = c0; i0 <= c1; i0 += 32) {
    const float2 ml = i0 == c0 ? ml0 : part_ml(i0 + lane);
    const float f = attn::factor_to(ml.x, top, p.scale_log2);
    sum += isnan(ml.y) ? ml.y : ml.y * f;
    const int count = int(c1 - i0 < 32 ? c1 - i0 + 1 : 32);
#pragma unroll 4
    for (int j = 0; j < count; ++j) {
      const float by = __shfl_sync(0xffffffffu, f, j);
      const float* o = p.partials + row_of(i0 + j) * DP + lane * kOwn;
#pragma unroll
      for (int y = 0; y < kOwn; ++y) acc[y] = fmaf(o[y], by, acc[y]);
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int n = r / p.group, g = r - n * p.group, d = lane * kOwn;
  if (d >= p.dim) return;
  T* to = static_cast<T*>(p.out) + (int64_t(b) * p.drafted + n) * p.heads * p.dim + int64_t(head * p.group + g) * p.dim + d;
#pragma unroll
  for (int y = 0; y < kOwn; y += 2) *reinterpret_cast<uint32_t*>(to + y) = pack_pair<T>(acc[y] * inv, acc[y + 1] * inv);
}

// Where tree_few_kernel is taken: all the rows that one of its products has.  4 drafted tokens, 4 heads a group (16 rows): 4
// sequences of 500 tokens 19 us, with tree_kernel 28; 32 of 8192 142 us, 146.
constexpr int kFewRows = 16;
// rows of a block
int block_rows(int64_t rows) { return rows <= kFewRows ? kFewRows : rows <= 128 ? 128 : 256; }

// the CTAs of tree_join_kernel for a unit
int joining_ctas(const TreeParams& p, int rows) { return (std::min(p.rows, rows) + kJoinThreads / 32 - 1) / (kJoinThreads / 32); }

template <typename T, int DP, bool kWindow>
int launch_join(const TreeParams& p, int rows, cudaStream_t stream) {
  const int per_unit = joining_ctas(p, rows);
  return launch_beside(&tree_join_kernel<T, DP, kWindow>, unsigned(p.batch * p.kv_heads * p.row_blocks * per_unit), kJoinThreads, 0, stream, p,
                       rows, per_unit);
}

template <typename T, int DP, bool kWindow>
int launch_few(const TreeParams& p, cudaStream_t stream) {
  constexpr int kBytes = FewConfig<DP>::kBytes;
  const cudaError_t err = ensure_dynamic_smem(reinterpret_cast<const void*>(&tree_few_kernel<T, DP, kWindow>), kBytes);
  if (err != cudaSuccess) { record_cuda_error(err); return GDN2_ERR_LAUNCH; }
  tree_few_kernel<T, DP, kWindow><<<unsigned(p.ctas), kFewThreads, kBytes, stream>>>(p);
  const int status = check_launch();
  return status != GDN2_OK ? status : launch_join<T, DP, kWindow>(p, kFewRows, stream);
}

template <typename T, int DP, int RT, bool kWindow>
int launch_tree_typed(const TreeParams& p, cudaStream_t stream) {
  using C = TreeConfig<DP, RT>;
  const void* kernel = reinterpret_cast<const void*>(&tree_kernel<T, DP, RT, kWindow>);
  const cudaError_t err = ensure_dynamic_smem(kernel, C::kBytes);
  if (err != cudaSuccess) { record_cuda_error(err); return GDN2_ERR_LAUNCH; }
  tree_kernel<T, DP, RT, kWindow><<<unsigned(p.ctas), kThreads, C::kBytes, stream>>>(p);
  const int status = check_launch();
  return status != GDN2_OK ? status : launch_join<T, DP, kWindow>(p, C::kRows, stream);
}

template <typename T, bool kWindow>
int launch_tree_dim(const TreeParams& p, cudaStream_t stream) {
  if (p.rows <= kFewRows) return p.dim <= 64 ? launch_few<T, 64, kWindow>(p, stream) : launch_few<T, 128, kWindow>(p, stream);
  if (p.dim <= 64) return p.rows <= 128 ? launch_tree_typed<T, 64, 1, kWindow>(p, stream) : launch_tree_typed<T, 64, 2, kWindow>(p, stream);
  return p.rows <= 128 ? launch_tree_typed<T, 128, 1, kWindow>(p, stream) : launch_tree_typed<T, 128, 2, kWindow>(p, stream);
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

// CTAs of a call: one an SM, which the tiles share whatever their number
int tree_ctas(int* ctas) { return multiprocessors(ctas); }

int64_t tree_workspace_bytes(int64_t rows, int dim, int ctas) {
  return int64_t(ctas) * 2 * block_rows(rows) * ((dim <= 64 ? 64 : 128) + 2) * 4;
}

int launch_tree(const void* q, const void* k, const void* v, const void* k_pages, const void* v_pages, const int* table,
                const int* lengths, const uint8_t* mask, void* out, void* workspace, const int64_t* strides,
                int64_t table_stride, int64_t mask_stride, int batch, int drafted, int heads, int kv_heads, int dim,
                int64_t pages, int page, int columns, const int* depths, int64_t depth_stride, int window, int sinks, int dtype, float scale,
                cudaStream_t stream) {
  TreeParams p{};
  p.q = q; p.k = k; p.v = v; p.k_pages = k_pages; p.v_pages = v_pages; p.out = out;
  p.table = table; p.lengths = lengths; p.mask = mask;
  p.partials = static_cast<float*>(workspace);
  for (int i = 0; i < 3; ++i) { p.q_stride[i] = strides[i]; p.k_stride[i] = strides[3 + i]; p.v_stride[i] = strides[6 + i]; }
  p.table_stride = table_stride; p.mask_stride = mask_stride; p.pages = pages;
  p.depths = depths; p.depth_stride = depth_stride; p.window = window; p.sinks = sinks;
  p.batch = batch; p.drafted = drafted; p.heads = heads; p.kv_heads = kv_heads; p.group = heads / kv_heads;
  p.dim = dim; p.page = page; p.columns = columns;
  p.rows = drafted * p.group;
  // Whole boxes of tiled copies come out of a page only where it has 8 or 16 rows, or a multiple of 32; pages of other
  // sizes, and tiles that a sequence ends in, are copied row by row.  Calls in a loop, decoding as above, pages of 64: 220
  // us with boxes, 242 row by row; of 16 225 and 249.  Trees of 48 drafts as above, pages of 64: 124 and 126; of 16 124 and 128.
  p.box = page % 32 == 0 ? 32 : page == 16 || page == 8 ? page : 0;
  if (p.box > 0) {
    const int64_t page_strides[3] = {int64_t(page) * kv_heads * dim, int64_t(kv_heads) * dim, dim};
    if (!attn::encode_heads_map(&p.k_map, k_pages, page_strides, pages, page, kv_heads, dim, dtype, p.box) ||
        !attn::encode_heads_map(&p.v_map, v_pages, page_strides, pages, page, kv_heads, dim, dtype, p.box)) {
      return GDN2_ERR_LAUNCH;
    }
  }
  const int per_block = block_rows(p.rows);
  p.row_blocks = (p.rows + per_block - 1) / per_block;
  const int status = tree_ctas(&p.ctas);
  if (status != GDN2_OK) return status;
  if (int64_t(batch) * kv_heads * p.row_blocks > int64_t(0x7fffffff) / joining_ctas(p, per_block)) return GDN2_ERR_TOO_LARGE;
  p.negate = scale < 0.f;
  p.polls = attn::wait_polls();
  p.wide = attn::wide_rows(out, dim);
  p.scale_log2 = attn::positive_scale(scale);
  if (window > 0) return dtype == GDN2_BF16 ? launch_tree_dim<__nv_bfloat16, true>(p, stream) : launch_tree_dim<__half, true>(p, stream);
  return dtype == GDN2_BF16 ? launch_tree_dim<__nv_bfloat16, false>(p, stream) : launch_tree_dim<__half, false>(p, stream);
}

}  // namespace gdn2
