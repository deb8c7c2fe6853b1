// What the kernels of attention over a paged cache share: the units and tiles of a call, the copies of their keys and values,
// the kernel for few rows, and the joining of what several CTAs have of a row.
#pragma once

#include <algorithm>

#include "attention_common.cuh"

namespace gdn2 {

int tree_ctas(int* ctas);   // CTAs of a call: one an SM, which the tiles share whatever their number

namespace paged {

using attn::Format;
using attn::pack_pair;
using attn::place_of;

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
  // weights that tokens get
  float* scores;                             // [batch][kv head][row][width], as they come out of Q K^T
  float2* stats;                             // [batch][kv head][row]: (m, l) where one CTA had all of a row
  int2* ends;                                // [batch][kv head][block of rows]: the first and last CTA that had a part of it
  float* weight_pages;                       // [pages][kv head][page]
  const int64_t* slots;                      // [batch][drafted]
  float decay;
  Divisor by_page;
  int width, slices;                         // floats of a row of scores; CTAs of weigh_kernel
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
  if (depth < p.window) return true;   // (no depth is below 0)
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
static __device__ const uint4 g_nan_row[16] = {GDN2_NAN4, GDN2_NAN4, GDN2_NAN4, GDN2_NAN4, GDN2_NAN4, GDN2_NAN4, GDN2_NAN4, GDN2_NAN4,
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
// (kOnce: it leaves L2 before anything else)
template <bool kOnce>
__device__ __forceinline__ void tma_load_page(uint32_t to, const CUtensorMap* map, int c, int head, int row, int page,
                                              uint64_t* full, uint32_t leader) {
  if (kOnce) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t.reg .b64 once;\n\tsetp.ne.b32 q, %7, 0;\n\tcreatepolicy.fractional.L2::evict_first.b64 once, 1.0;\n\t"
        "@q cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], "
        "[%1, {%2, %3, %4, %5}], [%6], once;\n\t}"
        ::"r"(to), "l"(map), "r"(c), "r"(head), "r"(row), "r"(page), "r"(tc::smem_u32(full)), "r"(leader)
        : "memory");
    return;
  }
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
template <typename T, int DP, bool kWindow, bool kOnce, int kStages, int kWarps>
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
            tma_load_page<kOnce>(base + slab * kSlab + uint32_t(mine + i * 32 + r) * 128u, keys ? &p.k_map : &p.v_map, slab * 64, u.head, row, page, &full[s],
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

// With a window: behind which token, counted from the first drafted one, no cached one was taken out of a unit's tiles: a warp's 32
// are looked at where any of them is not seen by all drafted ones.  By whole warps.
__device__ __forceinline__ int edge_of(const TreeParams& p, const Unit& u) { return min(0, seen_by_all(p, u) + 31 - u.length); }

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
  uint32_t strange_rows[kStrangeRows / 32];
  float m[8][16], l[8][16];
};
static_assert(sizeof(FewBars) <= 2048, "");

// kWeigh: scores and statistics are left for weigh_kernel, which makes of them what weight the tokens got; more rows than 16
// are several blocks of them.
template <typename T, int DP, bool kWindow, bool kWeigh>
__global__ void __launch_bounds__(kFewThreads, 1) tree_few_kernel(const __grid_constant__ TreeParams p) {
  using C = FewConfig<DP>;
  constexpr int kKSteps = DP / 16, kDB = DP / 8;
  constexpr bool kBits = kWindow || kWeigh;   // more tokens than a few to look through for values that are not finite
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
  if (kBits && tid < kStrangeRows / 32) bar.strange_rows[tid] = 0;
  Unit u;
  int tile, rest;
  if (!part_of_cta<kWindow, kFewThreads / 32>(p, bar.share, u, tile, rest)) return;
  const attn::Waiter waiter{&bar.failed, p.polls};
  if (warp >= 8) {
    bring_tiles<T, DP, kWindow, kWeigh, C::kStages, 4>(p, u, tile, rest, warp - 8, kv_base, bar.kv_full, bar.kv_empty, waiter, &bar.strange,
                                                       kBits ? bar.strange_rows : nullptr);
    return;
  }

  uint32_t qf[kKSteps][4];
  const uint32_t sign = p.negate ? 0x80008000u : 0u;   // the scale's goes to the queries
  int token_of[2];
  int depth[2] = {0, 0}, all_from = 0;   // with a window: depths of the two tokens, the first token that all rows see
  auto queries = [&](const Unit& x) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int r = quad + 8 * half + (kWeigh ? x.block * 16 : 0);
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
    float* scores = kWeigh ? p.scores + ((int64_t(u.b) * p.kv_heads + u.head) * p.rows + u.block * 16 + quad) * p.width : nullptr;
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
      if (kWeigh) {   // scores of all tokens that there are, of rows that there are (whose widths are even)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int t = first_token + (x >> 1) * 8 + in_quad * 2;
          if (token_of[x & 1] >= 0 && t < u.length + p.drafted) {
            *reinterpret_cast<float2*>(scores + (x & 1) * 8 * int64_t(p.width) + t) = make_float2(s[x >> 1][2 * (x & 1)], s[x >> 1][2 * (x & 1) + 1]);
          }
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
      const bool whole = !split && tile + n == u.tiles;
      const bool told = *static_cast<volatile int*>(&bar.strange) != 0, strange = kWindow ? __any_sync(0xffffffffu, told) : told;
      const int edge = kWindow && strange ? edge_of(p, u) : 0;
      const int64_t slot = int64_t(blockIdx.x) * 2 + (split ? 0 : 1);
      ok = ok && waiter.nobody_failed();   // none of the eight
      if (kWeigh && lane == 0) {
        int2* ends = p.ends + (int64_t(u.b) * p.kv_heads + u.head) * p.row_blocks + u.block;
        if (!split) ends->x = int(blockIdx.x);
        if (tile + n == u.tiles) ends->y = int(blockIdx.x);
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int local = quad + 8 * half, r = local + (kWeigh ? u.block * 16 : 0);
        if (r >= p.rows) continue;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) sum += bar.l[w][local];
        // nothing seen: the sum is 0 and so is the output
        const float inv = !ok || u.bad ? NAN : !whole ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
        const int i = r / p.group, g = r - i * p.group;
        if (strange) {
          const int first = kWindow ? max(u.from - 31, 0) - u.length : max(0, tile * kTile - u.length);
          const int last = min(p.drafted, tile_token<kWindow>(u, tile + n - 1) + kTile - u.length);
          const int deep = kWindow ? depth_of(p, u.b, i) : 0;
          auto add = [&](int d) {
            const uint8_t* mask = kWeigh || p.mask == nullptr ? nullptr : p.mask + u.b * p.mask_stride + int64_t(i) * p.drafted;
            const T* v;
            if (kWindow) {
              v = strange_value<T>(p, u, mask, i, deep, d, tile, n);
              if (v == nullptr) return;
            } else {
              if (!(mask == nullptr ? d <= i : mask[d] != 0)) return;
              v = static_cast<const T*>(p.v) + u.b * p.v_stride[0] + d * p.v_stride[1] + u.head * p.v_stride[2];
            }
#pragma unroll
            for (int x = 0; x < 2 * kDB; ++x) {
              const int col = (x >> 1) * 8 + in_quad * 2 + (x & 1);
              const float value = col < p.dim ? to_float(v[col]) : 0.f;
              if (!isfinite(value)) o[x >> 1][2 * half + (x & 1)] += value;
            }
          };
          if (kBits) {   // those that had such a value in some unit of the CTA, but for cached ones behind the window's edge
            for (int d0 = first & ~31; d0 < last; d0 += 32) {
              if (kWindow && d0 >= edge && d0 < 0) d0 = 0;
              for (uint32_t bits = bar.strange_rows[(d0 & (kStrangeRows - 1)) >> 5]; bits != 0; bits &= bits - 1) {
                const int d = d0 + __ffs(bits) - 1;
                if (d >= first && d < last) add(d);
              }
            }
          } else {
            for (int d = first; d < last; ++d) add(d);
          }
        }
        T* to = static_cast<T*>(p.out) + (int64_t(u.b) * p.drafted + i) * p.heads * p.dim + int64_t(u.head * p.group + g) * p.dim;
        float* part = p.partials + (slot * 16 + local) * DP;
#pragma unroll
        for (int d = 0; d < kDB; ++d) {
          const int col = d * 8 + in_quad * 2;
          const float2 y = make_float2(o[d][2 * half], o[d][2 * half + 1]);
          if (!whole) *reinterpret_cast<float2*>(part + col) = y;
          else if (col < p.dim) *reinterpret_cast<uint32_t*>(to + col) = pack_pair<T>(y.x * inv, y.y * inv);
        }
        if (!whole && in_quad == 0) {
          *reinterpret_cast<float2*>(p.partials + int64_t(p.ctas) * 2 * 16 * DP + (slot * 16 + local) * 2) = make_float2(m[half], inv * sum);
        }
        if (kWeigh && whole && in_quad == 0) {
          p.stats[(int64_t(u.b) * p.kv_heads + u.head) * p.rows + r] = make_float2(m[half], isnan(inv) ? inv : sum);
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

// The parts of a row that several CTAs have: where they are, and in how many of them
struct RowParts {
  int64_t c0, c1;    // CTAs
  int rows, local;   // of a block; the row's number in its block
  // the part of CTA i: its last unit where the unit began there, its first one otherwise
  __device__ __forceinline__ int64_t row_of(int64_t i) const { return (i * 2 + (i == c0 ? 1 : 0)) * rows + local; }
};

// A row's maximum and sum of all parts, by a warp, and the sums of DP / 32 channels a lane
template <int DP>
__device__ __forceinline__ float2 join_row(const TreeParams& p, const RowParts& x, bool values, float (&acc)[DP / 32]) {
  const int lane = threadIdx.x & 31;
  const float* all_ml = p.partials + int64_t(p.ctas) * 2 * x.rows * DP;
  // a part a lane: the first 32 parts' m and l stay
  const float2 none = make_float2(-INFINITY, 0.f);
  auto part_ml = [&](int64_t i) { return i <= x.c1 ? *reinterpret_cast<const float2*>(all_ml + x.row_of(i) * 2) : none; };
  const float2 ml0 = part_ml(x.c0 + lane);
  float top = ml0.x;
  for (int64_t i = x.c0 + 32 + lane; i <= x.c1; i += 32) top = fmaxf(top, part_ml(i).x);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  constexpr int kOwn = DP / 32;
  float sum = 0.f;
#pragma unroll
  for (int y = 0; y < kOwn; ++y) acc[y] = 0.f;
  for (int64_t i0 = x.c0; i0 <= x.c1; i0 += 32) {
    const float2 ml = i0 == x.c0 ? ml0 : part_ml(i0 + lane);
    const float f = attn::factor_to(ml.x, top, p.scale_log2);
    sum += isnan(ml.y) ? ml.y : ml.y * f;
    const int count = values ? int(x.c1 - i0 < 32 ? x.c1 - i0 + 1 : 32) : 0;
#pragma unroll 4
    for (int j = 0; j < count; ++j) {
      const float by = __shfl_sync(0xffffffffu, f, j);
      const float* o = p.partials + x.row_of(i0 + j) * DP + lane * kOwn;
#pragma unroll
      for (int y = 0; y < kOwn; ++y) acc[y] = fmaf(o[y], by, acc[y]);
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  return make_float2(top, sum);
}

template <typename T, int DP>
__device__ __forceinline__ void store_joined(const TreeParams& p, int b, int head, int r, const float (&acc)[DP / 32], float inv) {
  constexpr int kOwn = DP / 32;
  const int n = r / p.group, g = r - n * p.group, d = (threadIdx.x & 31) * kOwn;
  if (d >= p.dim) return;
  T* to = static_cast<T*>(p.out) + (int64_t(b) * p.drafted + n) * p.heads * p.dim + int64_t(head * p.group + g) * p.dim + d;
#pragma unroll
  for (int y = 0; y < kOwn; y += 2) *reinterpret_cast<uint32_t*>(to + y) = pack_pair<T>(acc[y] * inv, acc[y + 1] * inv);
}

// Where tree_few_kernel is taken: all the rows that one of its products has.  4 drafted tokens, 4 heads a group (16 rows): 4
// sequences of 500 tokens 19 us, with tree_kernel 28; 32 of 8192 142 us, 146.
constexpr int kFewRows = 16;

template <typename T, int DP, bool kWindow, bool kWeigh>
int launch_few(const TreeParams& p, cudaStream_t stream) {
  constexpr int kBytes = FewConfig<DP>::kBytes;
  const cudaError_t err = ensure_dynamic_smem(reinterpret_cast<const void*>(&tree_few_kernel<T, DP, kWindow, kWeigh>), kBytes);
  if (err != cudaSuccess) { record_cuda_error(err); return GDN2_ERR_LAUNCH; }
  tree_few_kernel<T, DP, kWindow, kWeigh><<<unsigned(p.ctas), kFewThreads, kBytes, stream>>>(p);
  return check_launch();
}

// What both ways have in common; rows of a block: `per_block`
inline int fill_tree(TreeParams* to, const void* q, const void* k, const void* v, const void* k_pages, const void* v_pages, const int* table,
              const int* lengths, void* out, const int64_t* strides, int64_t table_stride, int batch, int drafted, int heads, int kv_heads,
              int dim, int64_t pages, int page, int columns, int dtype, float scale, int per_block) {
  TreeParams& p = *to;
  p.q = q; p.k = k; p.v = v; p.k_pages = k_pages; p.v_pages = v_pages; p.out = out;
  p.table = table; p.lengths = lengths;
  for (int i = 0; i < 3; ++i) { p.q_stride[i] = strides[i]; p.k_stride[i] = strides[3 + i]; p.v_stride[i] = strides[6 + i]; }
  p.table_stride = table_stride; p.pages = pages;
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
  p.row_blocks = (p.rows + per_block - 1) / per_block;
  const int status = tree_ctas(&p.ctas);
  if (status != GDN2_OK) return status;
  p.negate = scale < 0.f;
  p.polls = attn::wait_polls();
  p.wide = attn::wide_rows(out, dim);
  p.scale_log2 = attn::positive_scale(scale);
  return GDN2_OK;
}

}  // namespace paged
}  // namespace gdn2
