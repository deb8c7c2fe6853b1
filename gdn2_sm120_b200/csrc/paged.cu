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
// A CTA: two chains of four warps turn scores into weights, a row a thread.  Up to 128 rows both work on the same rows,
// on every other tile, and their (O, m, l) are joined at the end; above, each has 128 rows and all tiles.  Four warps
// bring in rows with 16-byte asynchronous copies, since pages of any size make no box for a tiled copy; one issues the
// products.  TMEM: S0 S1 O0 O1, 128 columns each, P over S.

#include <algorithm>

#include "attention_common.cuh"

namespace gdn2 {

using attn::Format;
using attn::pack_pair;

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
constexpr int kThreads = 512;  // warps 0-3, 4-7: weights; 8-11: copies; 12: products
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
  float scale_log2;                          // positive
  uint32_t negate;                           // the scale is negative: Q counts with its sign changed
};

// A sequence's cached tokens and then its drafted ones, in tiles; kRows rows of one key head
struct Unit {
  int b, head, block;
  int length, tiles;
  bool bad;             // the sequence's length is none that its page table can hold
};

__device__ __forceinline__ void read_length(const TreeParams& p, Unit& u) {
  const int n = u.b < p.batch ? p.lengths[u.b] : 0;
  u.bad = n < 0 || n > p.columns * p.page;
  u.length = u.bad ? 0 : n;
  u.tiles = (u.length + p.drafted + kTile - 1) / kTile;
}

__device__ __forceinline__ void next_unit(const TreeParams& p, Unit& u) {
  if (++u.block < p.row_blocks) return;
  u.block = 0;
  if (++u.head < p.kv_heads) return;
  u.head = 0;
  ++u.b;
  read_length(p, u);
}

// tiles of sequence b, for all its key heads and blocks of rows
__device__ __forceinline__ int64_t tiles_of(const TreeParams& p, int b) {
  Unit u{b, 0, 0, 0, 0, false};
  read_length(p, u);
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

// RT: tiles of 128 rows that a CTA has, 1 or 2; QR: rows of queries that a tile has in shared memory.  Where that is 32
// the product reads on behind them: what its other rows are nobody looks at.
template <int DP, int RT, int QR>
struct TreeConfig {
  static constexpr int kTileBytes = kTile * DP * 2;
  static constexpr int kSlab = kTile * 128;                    // 64 channels of 128 rows
  static constexpr int kRows = 128 * RT;
  static constexpr int kQuerySlab = QR * 128, kQueryBytes = QR * DP * 2;
  // Queries of two units, so that the copies need not wait between two; those of 256 rows of 128 channels leave no room.
  static constexpr int kQueries = RT == 2 ? 1 : 2;
  static constexpr int kStages = DP == 64 ? 8 : QR == 32 ? 6 : 5;
  static constexpr int kBytes = RT * kQueries * kQueryBytes + kStages * kTileBytes + 2560;
};

struct TreeBars {
  uint64_t s_full[2], p_ready[2], o_full[2], q_empty[2], drained;
  uint64_t kv_full[8], kv_empty[8];
  int64_t scan[kThreads / 32], found[2];
  uint32_t tmem;
  int failed;
  int strange;          // a drafted value was infinite or NaN
  float2 ml[2][128];    // what the chains of the same rows tell each other
};
static_assert(sizeof(TreeBars) <= 2560, "");

template <typename T, int DP, int RT, int QR>
__global__ void __launch_bounds__(kThreads, 1) tree_kernel(const __grid_constant__ TreeParams p) {
  using C = TreeConfig<DP, RT, QR>;
  extern __shared__ __align__(1024) uint8_t smem[];   // swizzled tiles: 1024-byte aligned, there is no static shared memory
  const uint32_t q_base = tc::smem_u32(smem), kv_base = q_base + RT * C::kQueries * C::kQueryBytes;
  TreeBars& bar = *reinterpret_cast<TreeBars*>(smem + RT * C::kQueries * C::kQueryBytes + C::kStages * C::kTileBytes);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (tid == 0) {
    for (int t = 0; t < 2; ++t) {
      tc::mbar_init(&bar.s_full[t], 1);
      tc::mbar_init(&bar.p_ready[t], 4);
      tc::mbar_init(&bar.o_full[t], 1);
    }
    for (int x = 0; x < C::kQueries; ++x) tc::mbar_init(&bar.q_empty[x], 1);
    tc::mbar_init(&bar.drained, 1);
    for (int s = 0; s < C::kStages; ++s) {
      tc::mbar_init(&bar.kv_full[s], 128);
      tc::mbar_init(&bar.kv_empty[s], 1);
    }
    bar.failed = bar.strange = 0;
    tc::fence_mbar_init();
  }
  if (warp == 12) {
    tc::tmem_alloc(&bar.tmem, 512);
    tc::tmem_relinquish();
  }
  // this CTA's part of all tiles
  int64_t total = 0, before, own = 0;
  for (int b0 = 0; b0 < p.batch; b0 += kThreads) {
    own = b0 + tid < p.batch ? tiles_of(p, b0 + tid) : 0;
    total += cta_scan<kThreads / 32>(own, &before, bar.scan);
  }
  const int64_t ctas = sharing(p, total);
  const bool idle = blockIdx.x >= ctas;
  const int64_t begin = total * blockIdx.x / ctas, end = total * (blockIdx.x + 1) / ctas;
  if (!idle) {
    int64_t base = 0;
    for (int b0 = 0; b0 < p.batch; b0 += kThreads) {
      int64_t sum = total;
      if (p.batch > kThreads) {
        own = b0 + tid < p.batch ? tiles_of(p, b0 + tid) : 0;
        sum = cta_scan<kThreads / 32>(own, &before, bar.scan);
      }
      const int64_t from = base + before;
      if (own > 0 && begin >= from && begin < from + own) {  // one thread of all
        bar.found[0] = b0 + tid;
        bar.found[1] = begin - from;
      }
      base += sum;
      if (begin < base) break;
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = bar.tmem;
  if (idle) {
    if (warp == 12) tc::tmem_dealloc(tmem, 512);
    return;
  }
  const attn::Waiter waiter{&bar.failed};
  Unit u{int(bar.found[0]), 0, 0, 0, 0, false};
  read_length(p, u);
  const int64_t unit0 = bar.found[1] / u.tiles;
  int tile = int(bar.found[1] - unit0 * u.tiles);     // the first of this CTA's tiles of the unit
  u.head = int(unit0 / p.row_blocks);
  u.block = int(unit0 - int64_t(u.head) * p.row_blocks);
  int rest = int(end - begin);                        // tiles of this CTA that are left
  // tiles of 128 rows that a unit has
  auto row_tiles = [&](const Unit& x) { return RT == 2 && p.rows - x.block * C::kRows > 128 ? 2 : 1; };

  // 512 threads of 128 registers = 256 of 200 + 128 of 64 + 128 of 48
  if (warp >= 12) {
    attn::give_registers<48>();
    if (warp == 12) {
      // ---- products --------------------------------------------------------------------------------------
      const uint32_t leader = tc::elect_leader();
      const uint32_t id_s = tc::idesc(128, 128, Format<T>::code, tc::kMajorK, tc::kMajorK, p.negate);
      const uint32_t id_o = tc::idesc(128, DP, Format<T>::code, tc::kMajorK, tc::kMajorMN);
      int used = 0, p_used[2] = {0, 0}, queries = 0;   // which of the kQueries
      bool ok = true;
      auto full = [&](int x) {
        const bool r = waiter.wait(&bar.kv_full[x % C::kStages], (x / C::kStages) & 1);
        tc::fence_async_smem();   // what the copies wrote is read by the products
        return r;
      };
      auto scores = [&](int t, int x) {   // S_t from the keys in stage x
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
          attn::mma_ss(tmem + t * 128, attn::desc_k(q_base + (RT == 2 ? t : queries) * C::kQueryBytes, C::kQuerySlab, ks),
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
        if (++queries == C::kQueries) queries = 0;
        rest -= n;
        tile = 0;
        if (rest > 0) next_unit(p, u);
      }
      if (!ok) {  // products under way end before the CTA does
        tc::mma_commit(&bar.drained, leader);
        for (int i = 0; i < 4096 && !tc::mbar_try_wait(&bar.drained, 0); ++i) {}
      }
      __syncwarp();
    }
  } else if (warp >= 8) {
    // ---- copies: a warp has 32 rows of every tile, half a warp (128 channels) or a quarter copies a row at a time -----
    attn::give_registers<64>();
    constexpr int kPieces = DP / 8, kAtOnce = 32 / kPieces;
    const int mine = (warp - 8) * 32, piece = lane % kPieces, sub = lane / kPieces;
    const bool piece_there = piece * 8 < p.dim;
    const uint64_t anything = reinterpret_cast<uintptr_t>(g_nan_row);   // an address for copies of nothing
    int filled = 0, units = 0;
    bool ok = true;
    // a row of 16-byte pieces, lines of 128 bytes permuted by the row
    auto to = [&](uint32_t base, uint32_t slab, int row) {
      return base + uint32_t(piece >> 3) * slab + uint32_t(row) * 128u + ((uint32_t(piece ^ row) & 7u) << 4);
    };
    // copies this warp's rows of a tile; `at` is where row `mine + lane` is, null for zeros
    auto copy = [&](uint32_t base, uint32_t slab, const void* at) {
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
          const bool there = piece_there && row[x] != 0;
          cp_async16(to(base, slab, mine + i + x * kAtOnce + sub), reinterpret_cast<const uint8_t*>(there ? row[x] : anything) + piece * 16, there);
        }
      }
    };
    // An infinite or NaN value of a drafted token (this warp's rows from `first` on) must reach the rows that see it and no
    // others, but in the product it would meet every row (0 * NaN): it leaves the tile, and is added to those rows at the end.
    auto sift = [&](uint32_t base, int first) {
      for (int i = 0; i < 32; i += kAtOnce) {
        if (i + sub < first) continue;
        const uint32_t at = to(base, C::kSlab, mine + i + sub);
        uint32_t w[4];
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
        bool any = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if ((w[j] & Format<T>::exponent) == Format<T>::exponent) { w[j] &= 0xffff0000u; any = true; }
          if (((w[j] >> 16) & Format<T>::exponent) == Format<T>::exponent) { w[j] &= 0xffffu; any = true; }
        }
        if (any) {
          asm volatile("st.shared.v4.b32 [%4], {%0, %1, %2, %3};" ::"r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(at) : "memory");
          *static_cast<volatile int*>(&bar.strange) = 1;
        }
      }
    };
    auto page_of = [&](const Unit& x, int tile) {   // the page of row mine + lane, looked up a tile ahead
      const int t = tile * kTile + mine + lane;
      return t < x.length ? p.table[x.b * p.table_stride + t / p.page] : 0;
    };
    // the stage of the next copy, when its tile has been used
    auto stage = [&]() {
      const int s = filled % C::kStages;
      if (filled >= C::kStages) ok = waiter.wait(&bar.kv_empty[s], (filled / C::kStages - 1) & 1);
      ++filled;
      return s;
    };
    int page = page_of(u, tile);
    while (rest > 0 && ok) {
      const int n = min(rest, u.tiles - tile);
      Unit next = u;
      if (rest > n) next_unit(p, next);
      // the queries come with the first keys
      const int place = units % C::kQueries;
      if (units >= C::kQueries && !(ok = waiter.wait(&bar.q_empty[place], (units / C::kQueries - 1) & 1))) break;
      ++units;
      for (int x = 0; x < RT; ++x) {
        if (mine >= QR) break;
        const int r = u.block * C::kRows + x * 128 + mine + lane;
        const int i = r / p.group, g = r - i * p.group;
        const T* at = static_cast<const T*>(p.q) + u.b * p.q_stride[0] + i * p.q_stride[1] + int64_t(u.head * p.group + g) * p.q_stride[2];
        copy(q_base + (RT == 2 ? x : place) * C::kQueryBytes, C::kQuerySlab, r < p.rows ? at : nullptr);
      }
      const uint8_t* v_at = nullptr;
      int first = 32;     // of this warp's rows of values, the first drafted one
      for (int x = 0; x <= n && ok; ++x) {
        const uint8_t *k_now = nullptr, *v_now = nullptr;
        int first_now = 32;
        if (x < n) {
          const int t = (tile + x) * kTile + mine + lane, j = t - u.length;
          if (j < 0) {
            const int64_t row = (int64_t(page) * p.page + t % p.page) * p.kv_heads + u.head;
            const bool there = page >= 0 && page < p.pages;
            k_now = there ? static_cast<const uint8_t*>(p.k_pages) + row * p.dim * 2 : reinterpret_cast<const uint8_t*>(g_nan_row);
            v_now = there ? static_cast<const uint8_t*>(p.v_pages) + row * p.dim * 2 : nullptr;
          } else if (j < p.drafted) {
            k_now = static_cast<const uint8_t*>(p.k) + 2 * (u.b * p.k_stride[0] + j * p.k_stride[1] + u.head * p.k_stride[2]);
            v_now = static_cast<const uint8_t*>(p.v) + 2 * (u.b * p.v_stride[0] + j * p.v_stride[1] + u.head * p.v_stride[2]);
          }
          first_now = u.length - (tile + x) * kTile - mine;
          page = x + 1 < n ? page_of(u, tile + x + 1) : page_of(next, 0);
          const int s = stage();
          if (!ok) break;
          copy(kv_base + s * C::kTileBytes, C::kSlab, k_now);
          cp_async_arrive(&bar.kv_full[s]);
        }
        if (x > 0) {
          const int s = stage();
          if (!ok) break;
          copy(kv_base + s * C::kTileBytes, C::kSlab, v_at);
          if (first < 32) {
            cp_async_wait_all();
            sift(kv_base + s * C::kTileBytes, first);
            tc::mbar_arrive(&bar.kv_full[s]);
          } else {
            cp_async_arrive(&bar.kv_full[s]);
          }
        }
        v_at = v_now;
        first = first_now;
      }
      rest -= n;
      tile = 0;
      u = next;
    }
    cp_async_wait_all();
  } else {
    // ---- weights: a row a thread ---------------------------------------------------------------------------
    attn::take_registers<200>();
    const int t = warp >> 2, row = tid & 127;
    const uint32_t lane_base = uint32_t(warp & 3) << 21;   // 32 lanes of TMEM, in bits 16 and up
    const uint32_t s_at = tmem + lane_base + t * 128, o_at = tmem + lane_base + 256 + t * 128;
    int seen = 0, outs = 0;
    bool ok = true, split = false;   // the unit began in another CTA
    split = tile != 0;
    while (rest > 0) {
      const int n = min(rest, u.tiles - tile), chains = row_tiles(u);
      const int local = (RT == 2 ? t * 128 : 0) + row, r = u.block * C::kRows + local;   // row in the block, of all
      const int token = r / p.group;
      const bool there = r < p.rows, any_there = r - lane < p.rows;
      const bool takes_part = RT == 1 || t < chains;
      float m = -INFINITY;
      float2 sum2[2] = {{0.f, 0.f}, {0.f, 0.f}};
      int mine = 0;
      for (int j = RT == 1 ? t : 0; j < n && takes_part; j += RT == 1 ? 2 : 1) {
        if (!ok || !(ok = waiter.wait(&bar.s_full[t], seen & 1))) break;
        ++seen;
        tc::tc_fence_after();
        if (any_there) {
          const int first_token = (tile + j) * kTile;
          attn::soften<T, DP>(s_at, o_at, p.scale_log2, mine == 0, m, sum2, [&](uint32_t (&s)[4][32]) {
            if (first_token + kTile <= u.length) return;
            // drafted tokens, or the end
            const uint8_t* mask = p.mask == nullptr || !there ? nullptr : p.mask + u.b * p.mask_stride + int64_t(token) * p.drafted;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              uint32_t sees = 0;
#pragma unroll 8
              for (int y = 0; y < 32; ++y) {
                const int d = first_token + x * 32 + y - u.length;
                bool see = d < 0;
                if (!see && d < p.drafted && there) see = p.mask == nullptr ? d <= token : mask[d] != 0;
                sees |= uint32_t(see) << y;
              }
#pragma unroll
              for (int y = 0; y < 32; ++y) {
                if (!((sees >> y) & 1)) s[x][y] = 0xff800000u;
              }
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
      float sum = (sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y);
      // the columns of this thread: all, or where both chains have its row a half of the sum of both
      constexpr int kCols = RT == 1 ? DP / 2 : DP;
      const int col0 = RT == 1 ? t * kCols : 0;
      float f[2] = {1.f, 1.f};
      bool has[2] = {true, true};
      if (RT == 1) {
        bar.ml[t][row] = make_float2(mine > 0 ? m : -INFINITY, mine > 0 ? sum : 0.f);
        tc::tc_fence_before();
        sync_chains();
        tc::tc_fence_after();
        const float2 a = bar.ml[0][row], b = bar.ml[1][row];
        m = fmaxf(a.x, b.x);
        has[1] = n > 1;
        f[0] = m == -INFINITY ? 0.f : exp2_approx((a.x - m) * p.scale_log2);
        f[1] = m == -INFINITY ? 0.f : exp2_approx((b.x - m) * p.scale_log2);
        sum = a.y * f[0] + b.y * f[1];
        if (isnan(a.y) || isnan(b.y)) sum = NAN;
      }
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
        for (int x = col0; x < col0 + kCols; x += 32) {
          uint32_t raw[32];
          float o[32];
          tc::tmem_ld32(tmem + lane_base + 256 + (RT == 1 ? 0 : t * 128) + x, raw);
          tc::tmem_wait_ld();
#pragma unroll
          for (int y = 0; y < 32; ++y) o[y] = __uint_as_float(raw[y]);
          if (RT == 1) {
#pragma unroll
            for (int y = 0; y < 32; ++y) o[y] *= f[0];
            if (has[1]) {
              tc::tmem_ld32(tmem + lane_base + 256 + 128 + x, raw);
              tc::tmem_wait_ld();
#pragma unroll
              for (int y = 0; y < 32; ++y) o[y] = fmaf(__uint_as_float(raw[y]), f[1], o[y]);
            }
          }
          if (!there) continue;
          if (strange) {
            for (int d = max(0, tile * kTile - u.length); d < min(p.drafted, (tile + n) * kTile - u.length); ++d) {
              if (!(p.mask == nullptr ? d <= token : p.mask[u.b * p.mask_stride + int64_t(token) * p.drafted + d] != 0)) continue;
              const T* v = static_cast<const T*>(p.v) + u.b * p.v_stride[0] + d * p.v_stride[1] + u.head * p.v_stride[2];
#pragma unroll
              for (int y = 0; y < 32; ++y) {
                const float value = x + y < p.dim ? to_float(v[x + y]) : 0.f;
                if (!isfinite(value)) o[y] += value;
              }
            }
          }
          if (whole) {
#pragma unroll
            for (int y = 0; y < 32; y += 8) {
              if (x + y < p.dim) {
                uint4 w;
                w.x = pack_pair<T>(o[y] * inv, o[y + 1] * inv);
                w.y = pack_pair<T>(o[y + 2] * inv, o[y + 3] * inv);
                w.z = pack_pair<T>(o[y + 4] * inv, o[y + 5] * inv);
                w.w = pack_pair<T>(o[y + 6] * inv, o[y + 7] * inv);
                *reinterpret_cast<uint4*>(to + x + y) = w;
              }
            }
          } else {
#pragma unroll
            for (int y = 0; y < 32; y += 4) *reinterpret_cast<float4*>(part + x + y) = make_float4(o[y], o[y + 1], o[y + 2], o[y + 3]);
          }
        }
        if (!whole && there && col0 == 0) {
          float* ml = p.partials + int64_t(p.ctas) * 2 * C::kRows * DP + (slot * C::kRows + local) * 2;
          *reinterpret_cast<float2*>(ml) = make_float2(m == -INFINITY ? m : m * p.scale_log2, inv * sum);
        }
      }
      tc::tc_fence_before();
      if (RT == 1) sync_chains();   // the other chain has read this one's O
      rest -= n;
      tile = 0;
      split = false;
      if (rest > 0) next_unit(p, u);
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

// Joins what several CTAs have of a unit: a warp a row, in the order of the tiles.
template <typename T, int DP>
__global__ void __launch_bounds__(kJoinThreads) tree_join_kernel(const __grid_constant__ TreeParams p, int block_rows, int ctas_of_unit) {
  __shared__ int64_t scan[kJoinThreads / 32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int unit = int(blockIdx.x) / ctas_of_unit;
  const int block = unit % p.row_blocks, head = unit / p.row_blocks % p.kv_heads, b = unit / p.row_blocks / p.kv_heads;
  int64_t total = 0, from = 0, before;
  for (int b0 = 0; b0 < p.batch; b0 += kJoinThreads) {
    const int x = b0 + int(threadIdx.x);
    const int64_t own = x < p.batch ? tiles_of(p, x) : 0;
    total += cta_scan<kJoinThreads / 32>(own, &before, scan);
    from += cta_scan<kJoinThreads / 32>(x < b ? own : 0, &before, scan);
  }
  Unit u{b, 0, 0, 0, 0, false};
  read_length(p, u);
  const int64_t t0 = from + (int64_t(head) * p.row_blocks + block) * u.tiles, t1 = t0 + u.tiles;
  const int64_t ctas = sharing(p, total), c0 = ((t0 + 1) * ctas - 1) / total, c1 = (t1 * ctas - 1) / total;
  if (c0 == c1) return;   // one CTA had it all
  const int lane = threadIdx.x & 31;
  const int local = (int(blockIdx.x) - unit * ctas_of_unit) * (kJoinThreads / 32) + int(threadIdx.x >> 5);
  const int r = block * block_rows + local;
  if (local >= block_rows || r >= p.rows) return;
  const float* all_ml = p.partials + int64_t(p.ctas) * 2 * block_rows * DP;
  // the part of CTA i: its last unit where the unit began there, its first one otherwise
  auto row_of = [&](int64_t i) { return (i * 2 + (i == c0 ? 1 : 0)) * block_rows + local; };
  float top = -INFINITY;
  for (int64_t i = c0 + lane; i <= c1; i += 32) top = fmaxf(top, all_ml[row_of(i) * 2]);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  constexpr int kOwn = DP / 32;
  float sum = 0.f, acc[kOwn];
#pragma unroll
  for (int y = 0; y < kOwn; ++y) acc[y] = 0.f;
#pragma unroll 4
  for (int64_t i = c0; i <= c1; ++i) {
    const float2 ml = *reinterpret_cast<const float2*>(all_ml + row_of(i) * 2);
    const float f = ml.x == -INFINITY ? 0.f : exp2_approx(ml.x - top);
    sum += isnan(ml.y) ? ml.y : ml.y * f;
    const float* o = p.partials + row_of(i) * DP + lane * kOwn;
#pragma unroll
    for (int y = 0; y < kOwn; ++y) acc[y] = fmaf(o[y], f, acc[y]);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int n = r / p.group, g = r - n * p.group, d = lane * kOwn;
  if (d >= p.dim) return;
  T* to = static_cast<T*>(p.out) + (int64_t(b) * p.drafted + n) * p.heads * p.dim + int64_t(head * p.group + g) * p.dim + d;
#pragma unroll
  for (int y = 0; y < kOwn; y += 2) *reinterpret_cast<uint32_t*>(to + y) = pack_pair<T>(acc[y] * inv, acc[y + 1] * inv);
}

// rows of a block
int block_rows(int64_t rows) { return rows <= 128 ? 128 : 256; }

template <typename T, int DP, int RT, int QR>
int launch_tree_typed(const TreeParams& p, cudaStream_t stream) {
  using C = TreeConfig<DP, RT, QR>;
  const void* kernel = reinterpret_cast<const void*>(&tree_kernel<T, DP, RT, QR>);
  const cudaError_t err = ensure_dynamic_smem(kernel, C::kBytes);
  if (err != cudaSuccess) { record_cuda_error(err); return GDN2_ERR_LAUNCH; }
  const int per_unit = (std::min(p.rows, C::kRows) + kJoinThreads / 32 - 1) / (kJoinThreads / 32);
  const int64_t joining = int64_t(p.batch) * p.kv_heads * p.row_blocks * per_unit;
  if (joining > int64_t(0x7fffffff)) return GDN2_ERR_TOO_LARGE;
  tree_kernel<T, DP, RT, QR><<<unsigned(p.ctas), kThreads, C::kBytes, stream>>>(p);
  const int status = check_launch();
  if (status != GDN2_OK) return status;
  return launch_beside(&tree_join_kernel<T, DP>, unsigned(joining), kJoinThreads, 0, stream, p, C::kRows, per_unit);
}

template <typename T>
int launch_tree_dim(const TreeParams& p, cudaStream_t stream) {
  if (p.dim <= 64) {
    return p.rows <= 128 ? launch_tree_typed<T, 64, 1, 128>(p, stream) : launch_tree_typed<T, 64, 2, 128>(p, stream);
  }
  return p.rows <= 32 ? launch_tree_typed<T, 128, 1, 32>(p, stream)
                      : p.rows <= 128 ? launch_tree_typed<T, 128, 1, 128>(p, stream) : launch_tree_typed<T, 128, 2, 128>(p, stream);
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
                int64_t pages, int page, int columns, int dtype, float scale, cudaStream_t stream) {
  TreeParams p{};
  p.q = q; p.k = k; p.v = v; p.k_pages = k_pages; p.v_pages = v_pages; p.out = out;
  p.table = table; p.lengths = lengths; p.mask = mask;
  p.partials = static_cast<float*>(workspace);
  for (int i = 0; i < 3; ++i) { p.q_stride[i] = strides[i]; p.k_stride[i] = strides[3 + i]; p.v_stride[i] = strides[6 + i]; }
  p.table_stride = table_stride; p.mask_stride = mask_stride; p.pages = pages;
  p.batch = batch; p.drafted = drafted; p.heads = heads; p.kv_heads = kv_heads; p.group = heads / kv_heads;
  p.dim = dim; p.page = page; p.columns = columns;
  p.rows = drafted * p.group;
  const int per_block = block_rows(p.rows);
  p.row_blocks = (p.rows + per_block - 1) / per_block;
  const int status = tree_ctas(&p.ctas);
  if (status != GDN2_OK) return status;
  if (int64_t(batch) * kv_heads * p.row_blocks > int64_t(0x7fffffff)) return GDN2_ERR_TOO_LARGE;
  // the sign goes to the product, and a scale of 0 stays a positive number, so that -inf * scale masks as ever
  p.negate = scale < 0.f;
  p.scale_log2 = fmaxf(fabsf(scale) * attn::kLog2e, 1e-30f);
  return dtype == GDN2_BF16 ? launch_tree_dim<__nv_bfloat16>(p, stream) : launch_tree_dim<__half>(p, stream);
}

}  // namespace gdn2
