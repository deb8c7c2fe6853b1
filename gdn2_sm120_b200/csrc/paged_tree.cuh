// Attention of drafted tokens over a paged cache: the kernel for any number of rows, the joining of what several CTAs have, and the
// launches, without a window and with one.
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
// With a window the tiles between the sinks and the first token that any row sees are passed over (which of them, the drafted tokens'
// number does not say: their depths move the window's edge, so that a tile at the edge is masked row by row).
#pragma once

#include "paged_tiles.cuh"

namespace gdn2 {
namespace paged {

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
      bring_tiles<T, DP, kWindow, false, C::kStages, 4>(p, u, tile, rest, warp - 8, kv_base, bar.kv_full, bar.kv_empty, waiter, &bar.strange,
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
            const int key = first_token + x * 32;
            if (key + 32 <= u.length && (!kWindow || key >= all_from || key + 32 <= p.sinks)) return;
            if (kWindow && (key + 32 <= u.length || (p.mask == nullptr && p.depths == nullptr))) {
              // cached tokens, or a chain's, whose places are those behind them.  (Rows that are not there have a depth of 0;
              // nothing but their zeros comes of them.)
              attn::Span{p.window, p.sinks}.hide(u.length + depth, key, s);
              return;
            }
            // drafted tokens, or the end
            const uint8_t* mask = p.mask == nullptr || !there ? nullptr : p.mask + u.b * p.mask_stride + int64_t(token) * p.drafted;
            uint32_t sees = 0;
            if (kWindow) {
              const int d0 = key - u.length;
              if (there && d0 < p.drafted) {
#pragma unroll
                for (int y = 0; y < 32; ++y) {   // (all loads at once)
                  const int d = d0 + y;
                  if (d >= 0 && d < p.drafted) sees |= uint32_t(p.mask == nullptr ? d <= token : mask[d] != 0) << y;
                }
              }
              if (depth >= p.window) {           // some of them may lie a window behind
                for (uint32_t bits = sees; bits != 0; bits &= bits - 1) {
                  if (!reaches(p, u, depth, d0 + __ffs(bits) - 1)) sees &= ~(bits & -bits);
                }
              }
              if (d0 < 0) sees |= attn::Span{p.window, p.sinks}.sees(u.length + depth, key) & ((1u << -d0) - 1u);   // cached ones
            } else {
#pragma unroll 8
              for (int y = 0; y < 32; ++y) {
                const int d = key + y - u.length;
                bool see = d < 0;
                if (!see && d < p.drafted && there) see = p.mask == nullptr ? d <= token : mask[d] != 0;
                sees |= uint32_t(see) << y;
              }
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
      const bool told_strange = *static_cast<volatile int*>(&bar.strange) != 0, strange = kWindow ? __any_sync(0xffffffffu, told_strange) : told_strange;
      const int edge = kWindow && strange ? edge_of(p, u) : 0;
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
              if (kWindow && d0 >= edge && d0 < 0) d0 = 0;
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
  const int local = (int(blockIdx.x) - unit * ctas_of_unit) * (kJoinThreads / 32) + int(threadIdx.x >> 5);
  const int r = block * block_rows + local;
  if (local >= block_rows || r >= p.rows) return;
  float acc[DP / 32];
  const float sum = join_row<DP>(p, RowParts{c0, c1, block_rows, local}, true, acc).y;
  store_joined<T, DP>(p, b, head, r, acc, sum == 0.f ? 0.f : 1.f / sum);
}

// rows of a block
inline int block_rows(int64_t rows) { return rows <= kFewRows ? kFewRows : rows <= 128 ? 128 : 256; }

// the CTAs of tree_join_kernel for a unit
inline int joining_ctas(const TreeParams& p, int rows) { return (std::min(p.rows, rows) + kJoinThreads / 32 - 1) / (kJoinThreads / 32); }

template <typename T, int DP, bool kWindow>
int launch_join(const TreeParams& p, int rows, cudaStream_t stream) {
  const int per_unit = joining_ctas(p, rows);
  return launch_beside(&tree_join_kernel<T, DP, kWindow>, unsigned(p.batch * p.kv_heads * p.row_blocks * per_unit), kJoinThreads, 0, stream, p,
                       rows, per_unit);
}

template <typename T, int DP, bool kWindow>
int launch_few_typed(const TreeParams& p, cudaStream_t stream) {
  const int status = launch_few<T, DP, kWindow, false>(p, stream);
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
  if (p.rows <= kFewRows) return p.dim <= 64 ? launch_few_typed<T, 64, kWindow>(p, stream) : launch_few_typed<T, 128, kWindow>(p, stream);
  if (p.dim <= 64) return p.rows <= 128 ? launch_tree_typed<T, 64, 1, kWindow>(p, stream) : launch_tree_typed<T, 64, 2, kWindow>(p, stream);
  return p.rows <= 128 ? launch_tree_typed<T, 128, 1, kWindow>(p, stream) : launch_tree_typed<T, 128, 2, kWindow>(p, stream);
}

}  // namespace paged
}  // namespace gdn2
