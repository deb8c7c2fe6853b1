// Causal attention, backward, on the tensor cores.  With the forward's statistics lse_i = m_i + log l_i:
//
//   p_ij = exp(scale q_i . k_j - lse_i)      delta_i = do_i . o_i      ds_ij = p_ij (do_i . v_j - delta_i)
//   dv_j = sum_i p_ij do_i      dk_j = scale sum_i ds_ij q_i      dq_i = scale sum_j ds_ij k_j
//
// Three kernels: delta (bound by HBM), one that sums dk and dv of 128 keys over the queries that see them, and one that sums
// dq of 128 queries over the keys that they see.  Each of the two sums its rows' gradients by itself, over all query heads of
// a group too: no atomics, the same bits every time, at the price of forming S and dP twice (seven products in place of
// five).
//
// p and ds are rounded to the inputs' type for their products, which is as near as a 16-bit operand comes: a gradient's
// error in the 2-norm is that of its own rounding and of one of these, 1.4 times a rounding of the exact gradient, 1.5 with
// the output's rounding in delta, and up to 1.8 in sequences of a few tokens, where that counts as much.
//
// P and dS are 0 by selection where a row does not see a key.  In the tiles on the diagonal their products meet those rows of k,
// q and do all the same, and 0 * inf and 0 * NaN are not 0: a key that is not finite reaches dq, in its channel, of the rows
// before it in its tile, a query dk and a cotangent dv of the keys behind it there.  (Another sequence's rows never.)
//
// Training 4 x 2048 tokens, 16 heads of 128 channels, 4 heads a group, each kernel by itself: delta 11 us, keys 121, queries 120, forward 73.
//
// With a window (kWindow) delta is taken from the output and what its rounding has left over: where rows see few tokens delta's
// own error counts most.  Gradients' errors in the 2-norm without it and with it, in roundings: a window of 2 tokens 2.3 and 1.5, 4
// 1.8 and 1.5, 10 1.6 and 1.45, 100 1.48 and 1.43; it costs 13 us of the 242 of the training step below (in 8 bits, whose rows are
// half sectors, 18).  Each of the two goes over the tiles that its rows see or are seen by, and those of the sinks: 4 x 2048
// tokens as above, a window of 512 and 16 sinks: keys and queries 155 us together, forward 69, delta 16.  Where a
// window reaches over everything, the gradients of sequences of one tile have their delta taken that way, too; the rest is as
// without one.

#include <algorithm>
#include <climits>

#include "attention_common.cuh"

namespace gdn2 {
namespace attn {

namespace {

constexpr int kThreads = 640;    // warps 0-7: even steps; 8-15: odd ones; 16: products; 17: copies
constexpr int kStep = 64;        // rows of a step

// Queries: q and do of 128 queries stay, in TMEM; keys and values go by, 64 at a time, by turns in two sets of S and dP:
// while the tensor cores form one, eight warps make dS of the other, two threads a row.  TMEM: dq 128 columns, q and do 64
// each, two sets of 64 + 64; dS (16-bit) overlays its dP.  What bounds it is the round trip of a set: 1635 clocks a step, of
// which its products take the tensor cores 768; with q and do in shared memory 1900.
template <int DP>
struct QueryConfig {
  static constexpr int kStayBytes = 128 * DP * 2, kStaySlab = 128 * 128;
  static constexpr int kGoBytes = kStep * DP * 2, kGoSlab = kStep * 128;
  static constexpr int kStages = DP == 128 ? 4 : 6;
  static constexpr int kBytes = 2 * kStayBytes + kStages * 2 * kGoBytes + 512;
};

struct BwdParams {
  CUtensorMap q_tile, do_tile, k_tile, v_tile, k_step, v_step;   // 128 rows, 64 rows
  void *dq, *dk, *dv;
  const float *lse, *delta;  // -(m + log2 l) in powers of two, -delta
  const float* shifts;       // references that are far away, where lse says so
  float* partials;           // dk and dv of the parts of an item, [part][dk, dv][row][kv head][dim]
  int64_t partial_rows;      // rows * kv heads
  int parts;                 // of an item of the key kernel
  // With a window: the sums of keys that are sinks go on where those of others have ended, over all later queries.  Their
  // tiles are items of their own, `sink_tiles` of every sequence, in `sink_parts` parts, [part][dk, dv][sequence, row][kv
  // head][dim] behind the others'.
  int sink_tiles, sink_parts;
  float* sink_partials;
  int64_t sink_items;
  Span span;
  int heads, kv_heads, group, dim, turns;
  int64_t items;
  float scale, scale_log2;   // scale_log2 is positive
  uint32_t negate;
  uint32_t polls;            // of a wait
  bool wide;                 // rows of the gradients are 32-byte aligned
  Sequences seq;
};

struct QueryBars {
  uint64_t stay_full, stay_empty, in_tmem, acc_full, acc_empty, raw, drained;
  uint64_t s_full[2], ds_ready[2], go_full[6], go_empty[6];
  uint32_t tmem;
  int failed;
};

struct BwdItem {
  Item at;
  int head, tile;       // of queries, or of keys; 128-row tile in the sequence
  int first, per_head, steps;  // keys: first 128-row step, steps of a query head, of this part; queries: 64-row steps
  int part, begin;             // keys: which part, its first step of the item's
  int sinks;                   // queries, with a window: steps over sinks ahead of those from `first` on; keys: the sinks' sequence or -1
  // queries: the first key of a step
  template <bool kWindow>
  __device__ __forceinline__ int key_of(int step) const { return kStep * (!kWindow || step < sinks ? step : first + step - sinks); }
};

// The weight of a score s of a query whose statistic is l and whose reference, if that is far away, is *shift.  Scores are
// formed anew, so that one may lie above the forward's maximum by an ulp, which is powers of two for large ones: no weight is
// above 1.
__device__ __forceinline__ float far_weight(uint32_t s, float l, const float* shift, float c) {
  const float x = __uint_as_float(s);
  return exp2_approx(l > kFarFrom ? min_nan(fmaf(x - *shift, c, l - kFarMark), 0.f) : fmaf(x, c, l));
}

// dS of half a row of the query kernel whose warp has a row with such a reference, formed and left over dP: the row sees its
// columns that have a bit
template <typename T>
__device__ __noinline__ void far_slopes(uint32_t s_at, uint32_t dp_at, float l, const float* shift, float minus_delta, float c, uint32_t sees) {
  uint32_t w[16];
#pragma unroll
  for (int x = 0; x < 32; x += 16) {
    uint32_t s[16], dp[16];
    tc::tmem_ld16(s_at + x, s);
    tc::tmem_ld16(dp_at + x, dp);
    tc::tmem_wait_ld();
#pragma unroll
    for (int y = 0; y < 16; y += 2) {
      float ds[2];
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        ds[z] = ((sees >> (x + y + z)) & 1) == 0 ? 0.f : far_weight(s[y + z], l, shift, c) * (__uint_as_float(dp[y + z]) + minus_delta);
      }
      w[(x + y) / 2] = pack_pair<T>(ds[0], ds[1]);
    }
  }
  tc::tmem_st16(dp_at, w);
}

// the first step of a part of an item of the key kernel
__device__ __forceinline__ int part_begin(int steps, int part, int parts) { return int(int64_t(steps) * part / parts); }

// tiles of 128 queries that see some key of a tile of 128, of which no key is a sink: all from the tile's own on, as many as
// the window reaches
__device__ __forceinline__ int seeing_tiles(int len, int tile, int window) {
  return min((len + 127) / 128 - tile, (126 + window) / 128 + 1);
}

template <bool kKeys, bool kWindow>
__device__ __forceinline__ bool bwd_item(const BwdParams& p, int turn, BwdItem* w) {
  int64_t index = item_of_turn(turn);
  if (index >= p.items) return false;
  if (kKeys && kWindow) {
    w->sinks = -1;
    if (index < p.sink_items) {
      const int part = int(index % p.sink_parts);
      index /= p.sink_parts;
      w->head = int(index % p.kv_heads);
      index /= p.kv_heads;
      w->tile = int(index % p.sink_tiles);
      w->sinks = int(index / p.sink_tiles);
      w->at = find_sequence(p.seq, w->sinks);
      if (w->tile * 128 >= w->at.len) return false;
      w->first = w->tile;
      w->per_head = (w->at.len + 127) / 128 - w->tile;
      w->part = part;
      w->begin = part_begin(w->per_head * p.group, part, p.sink_parts);
      w->steps = part_begin(w->per_head * p.group, part + 1, p.sink_parts) - w->begin;
      return w->steps > 0;
    }
    index -= p.sink_items;
  }
  const int parts = kKeys ? p.parts : 1, heads = (kKeys ? p.kv_heads : p.heads) * parts;
  const int u = int(index / heads), in_tile = int(index - int64_t(u) * heads);
  w->head = in_tile / parts;
  w->part = in_tile - w->head * parts;
  w->at = find_item(p.seq, u >> 1, !kKeys);
  w->tile = 2 * w->at.tile + (kKeys ? u & 1 : 1 - (u & 1));
  if (w->tile * 128 >= w->at.len) return false;
  w->first = kKeys ? w->tile : 0;
  w->per_head = kKeys ? (w->at.len + 127) / 128 - w->tile : min(2 * w->tile + 2, (w->at.len + kStep - 1) / kStep);
  if (kWindow && kKeys) {
    if (w->tile < p.sink_tiles) return false;
    w->per_head = seeing_tiles(w->at.len, w->tile, p.span.window);
  } else if (kWindow) {
    w->first = p.span.first_tile(w->tile * 128, kStep, &w->sinks);
    w->per_head += w->sinks - w->first;
  }
  w->begin = kKeys ? part_begin(w->per_head * p.group, w->part, parts) : 0;
  w->steps = kKeys ? part_begin(w->per_head * p.group, w->part + 1, parts) - w->begin : w->per_head;
  return w->steps > 0;
}

template <typename T, int DP, bool kWindow>
__global__ void __launch_bounds__(kThreads, 1) attention_queries_kernel(const __grid_constant__ BwdParams p) {
  using C = QueryConfig<DP>;
  extern __shared__ __align__(1024) uint8_t smem[];   // swizzled tiles: 1024-byte aligned, there is no static shared memory
  uint8_t* stay = smem;
  uint8_t* go = smem + 2 * C::kStayBytes;
  QueryBars& bar = *reinterpret_cast<QueryBars*>(go + C::kStages * 2 * C::kGoBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    tc::mbar_init(&bar.stay_full, 1);
    tc::mbar_init(&bar.stay_empty, 16);
    tc::mbar_init(&bar.in_tmem, 16);
    tc::mbar_init(&bar.acc_full, 1);
    tc::mbar_init(&bar.acc_empty, 16);
    tc::mbar_init(&bar.raw, 1);
    tc::mbar_init(&bar.drained, 1);
    for (int b = 0; b < 2; ++b) {
      tc::mbar_init(&bar.s_full[b], 1);
      tc::mbar_init(&bar.ds_ready[b], 8);
    }
    for (int s = 0; s < C::kStages; ++s) {
      tc::mbar_init(&bar.go_full[s], 1);
      tc::mbar_init(&bar.go_empty[s], 1);
    }
    bar.failed = 0;
    tc::fence_mbar_init();
  }
  if (warp == 16) {
    tc::tmem_alloc(&bar.tmem, 512);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = bar.tmem;
  const Waiter waiter{&bar.failed, p.polls};

  if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");   // 640 threads of 96 registers = 512 of 104 + 128 of 64
    if (warp == 17) {
      // ---- copies ----------------------------------------------------------------------------------------
      const uint32_t leader = tc::elect_leader();
      int filled = 0, stayed = 0, mended = 0;
      bool ok = true;
      for (int turn = 0; turn < p.turns && ok; ++turn) {
        BwdItem w;
        if (!bwd_item<false, kWindow>(p, turn, &w)) continue;
        const int kv_head = w.head / p.group;
        if (stayed > 0) ok = waiter.wait(&bar.stay_empty, (stayed - 1) & 1);
        if (!ok) break;
        tc::mbar_arrive_expect_tx(&bar.stay_full, 2 * C::kStayBytes, leader);
#pragma unroll
        for (int slab = 0; slab < DP / 64; ++slab) {
          const int row = w.at.row0 + w.tile * 128;
          tc::tma_load_4d(stay + slab * C::kStaySlab, &p.q_tile, slab * 64, w.head, row, w.at.batch, &bar.stay_full, leader);
          tc::tma_load_4d(stay + C::kStayBytes + slab * C::kStaySlab, &p.do_tile, slab * 64, w.head, row, w.at.batch,
                          &bar.stay_full, leader);
        }
        ++stayed;
        for (int i = 0; i < w.steps && ok; ++i) {
          const int s = filled % C::kStages;
          if (filled >= C::kStages) ok = waiter.wait(&bar.go_empty[s], (filled / C::kStages - 1) & 1);
          if (!ok) break;
          const int at = w.key_of<kWindow>(i);
          uint8_t* to = go + s * 2 * C::kGoBytes;
          // rows of the next sequence would meet weights of 0, but 0 * inf and 0 * NaN are not 0
          const int valid = w.at.len - at;
          const bool mend = p.seq.packed && valid < kStep;
          uint64_t* full = mend ? &bar.raw : &bar.go_full[s];
          tc::mbar_arrive_expect_tx(full, 2 * C::kGoBytes, leader);
#pragma unroll
          for (int slab = 0; slab < DP / 64; ++slab) {
            tc::tma_load_4d(to + slab * C::kGoSlab, &p.k_step, slab * 64, kv_head, w.at.row0 + at, w.at.batch, full, leader);
            tc::tma_load_4d(to + C::kGoBytes + slab * C::kGoSlab, &p.v_step, slab * 64, kv_head, w.at.row0 + at, w.at.batch,
                            full, leader);
          }
          if (mend) {
            ok = waiter.wait(&bar.raw, mended & 1);
            ++mended;
#pragma unroll
            for (int slab = 0; slab < 2 * DP / 64; ++slab) {
              uint4* lines = reinterpret_cast<uint4*>(to + slab * C::kGoSlab);
              for (int x = valid * 8 + lane; x < kStep * 8; x += 32) lines[x] = make_uint4(0, 0, 0, 0);
            }
            tc::fence_async_smem();
            __syncwarp();
            tc::mbar_arrive(&bar.go_full[s], leader);
          }
          ++filled;
        }
      }
      if (!ok) {  // copies under way end before the CTA does
        for (int back = 1; back <= C::kStages && back <= filled; ++back) {
          const int x = filled - back;
          for (int i = 0; i < 4096 && !tc::mbar_try_wait(&bar.go_full[x % C::kStages], (x / C::kStages) & 1); ++i) {}
        }
        for (int i = 0; stayed > 0 && i < 4096 && !tc::mbar_try_wait(&bar.stay_full, (stayed - 1) & 1); ++i) {}
        for (int i = 0; mended > 0 && i < 4096 && !tc::mbar_try_wait(&bar.raw, (mended - 1) & 1); ++i) {}
      }
    } else if (warp == 16) {
      // ---- products --------------------------------------------------------------------------------------
      const uint32_t leader = tc::elect_leader();
      const uint32_t id_s = tc::idesc(128, kStep, Format<T>::code, tc::kMajorK, tc::kMajorK, p.negate);
      const uint32_t id_dp = tc::idesc(128, kStep, Format<T>::code, tc::kMajorK, tc::kMajorK);
      const uint32_t id_acc = tc::idesc(128, DP, Format<T>::code, tc::kMajorK, tc::kMajorMN);
      const uint32_t go_base = tc::smem_u32(go);
      int used = 0, stayed = 0, ready[2] = {0, 0};
      bool ok = true;
      auto both = [&](int b, int x) {   // S and dP of the step in stage x
        if (!waiter.wait(&bar.go_full[x % C::kStages], (x / C::kStages) & 1)) return false;
        tc::tc_fence_after();
        const uint32_t xs = go_base + (x % C::kStages) * 2 * C::kGoBytes, ys = xs + C::kGoBytes;
        const uint32_t s_at = tmem + 256 + b * 128, dp_at = s_at + 64;
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) mma_ts(s_at, tmem + 128 + ks * 8, desc_k(xs, C::kGoSlab, ks), id_s, ks > 0, leader);
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) mma_ts(dp_at, tmem + 192 + ks * 8, desc_k(ys, C::kGoSlab, ks), id_dp, ks > 0, leader);
        tc::mma_commit(&bar.s_full[b], leader);
        return true;
      };
      for (int turn = 0; turn < p.turns && ok; ++turn) {
        BwdItem w;
        if (!bwd_item<false, kWindow>(p, turn, &w)) continue;
        ok = waiter.wait(&bar.in_tmem, stayed & 1);
        if (ok) ok = both(0, used);
        if (ok && w.steps > 1) ok = both(1, used + 1);
        for (int i = 0; i < w.steps && ok; ++i) {
          const int b = i & 1, x = used + i;
          if (i == 0 && stayed > 0 && !(ok = waiter.wait(&bar.acc_empty, (stayed - 1) & 1))) break;
          if (!(ok = waiter.wait(&bar.ds_ready[b], ready[b] & 1))) break;
          ++ready[b];
          tc::tc_fence_after();
          const uint32_t xs = go_base + (x % C::kStages) * 2 * C::kGoBytes, ds_at = tmem + 256 + b * 128 + 64;
#pragma unroll
          for (int ks = 0; ks < kStep / 16; ++ks) mma_ts(tmem, ds_at + (ks >> 1) * 32 + (ks & 1) * 8, desc_mn(xs, C::kGoSlab, ks), id_acc, i > 0 || ks > 0, leader);
          tc::mma_commit(&bar.go_empty[x % C::kStages], leader);
          if (i + 1 == w.steps) tc::mma_commit(&bar.acc_full, leader);
          if (i + 2 < w.steps) ok = both(b, x + 2);
        }
        used += w.steps;
        ++stayed;
      }
      if (!ok) {  // products under way end before the CTA does
        tc::mma_commit(&bar.drained, leader);
        for (int i = 0; i < 4096 && !tc::mbar_try_wait(&bar.drained, 0); ++i) {}
      }
      __syncwarp();
    }
  } else {
    // ---- weights: two threads a row ------------------------------------------------------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    const int b = warp >> 3, half = (warp >> 2) & 1, row = threadIdx.x & 127;   // two threads a row, 32 columns each
    const uint32_t lane_base = uint32_t(warp & 3) << 21;   // 32 lanes of TMEM, in bits 16 and up
    const uint32_t s_at = tmem + lane_base + 256 + b * 128 + half * 32, dp_at = s_at + 64;
    int seen = 0, outs = 0, stayed = 0, all[2] = {0, 0};   // steps of this set, items, items in TMEM, steps of both sets
    bool ok = true;
    // A product whose first operand comes from TMEM reads a third of the shared memory (16 KiB of the rows that go
    // by, and not 32 KiB of those that stay), which is what bounds it.  A thread brings half a row of q and of do there.
    auto into_tmem = [&]() {
      if (ok) ok = waiter.wait(&bar.stay_full, stayed & 1);
      ++stayed;
      tc::tc_fence_after();
      constexpr int kWords = DP / 4;   // of half a row
#pragma unroll
      for (int which = 0; which < 2; ++which) {
#pragma unroll
        for (int x = 0; x < kWords; x += 16) {
          uint32_t w[16];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const int piece = (half * kWords + x) / 4 + y;
            const uint4 v = *reinterpret_cast<const uint4*>(stay + which * C::kStayBytes + (piece >> 3) * C::kStaySlab + row * 128 +
                                                            ((piece ^ row) & 7) * 16);
            w[4 * y] = v.x; w[4 * y + 1] = v.y; w[4 * y + 2] = v.z; w[4 * y + 3] = v.w;
          }
          tc::tmem_st16(tmem + lane_base + 128 + which * 64 + half * kWords + x, w);
        }
      }
      tc::tmem_wait_st();
      tc::tc_fence_before();
      __syncwarp();
      tc::mbar_arrive(&bar.stay_empty, lane == 0 && ok);
      tc::mbar_arrive(&bar.in_tmem, lane == 0 && ok);
    };
    for (int turn = 0; turn < p.turns; ++turn) {
      BwdItem w;
      if (!bwd_item<false, kWindow>(p, turn, &w)) continue;
      if (stayed == outs) into_tmem();
      const int64_t stat = w.head * p.seq.stat_rows + w.at.stat + w.tile * 128 + row;
      const float lse = p.lse[stat];
      const bool far = __any_sync(0xffffffffu, lse > kFarFrom);
      const float2 minus_lse = twice(lse), minus_delta = twice(p.delta[stat]), by_scale = twice(p.scale_log2);
      for (int i = b; i < w.steps && ok; i += 2) {
        if (!(ok = waiter.wait(&bar.s_full[b], seen & 1))) break;
        ++seen;
        tc::tc_fence_after();
        // a query sees keys up to itself: of those that go by the first to `last`
        const int last = w.tile * 128 + row - i * kStep;
        const bool diagonal = kWindow ? !p.span.whole(w.tile * 128, 128, w.key_of<kWindow>(i), kStep) : (i + 1) * kStep > w.tile * 128;
        uint32_t sees = ~0u;
        if (kWindow && diagonal) sees = p.span.sees(w.tile * 128 + row, w.key_of<kWindow>(i) + half * 32);
        uint32_t s[32], dp[32], dsw[16];
        tc::tmem_ld32(s_at, s);
        tc::tmem_ld32(dp_at, dp);
        tc::tmem_wait_ld();
#pragma unroll
        for (int y = 0; y < 32; y += 2) {
          const int x = half * 32 + y;
          const float2 z = fma2(make_float2(__uint_as_float(s[y]), __uint_as_float(s[y + 1])), by_scale, minus_lse);
          const float2 e = exp2_2(z);
          float2 ds = mul2(e, add2(make_float2(__uint_as_float(dp[y]), __uint_as_float(dp[y + 1])), minus_delta));
          if (diagonal) {
            if (kWindow ? ((sees >> y) & 1) == 0 : x > last) ds.x = 0.f;
            if (kWindow ? ((sees >> (y + 1)) & 1) == 0 : x + 1 > last) ds.y = 0.f;
          }
          dsw[y / 2] = pack_pair<T>(ds.x, ds.y);   // rounded to the inputs' type for its product, whose sums are in 32 bits
        }
        if (far) {
          if (!kWindow && diagonal) sees = last - half * 32 >= 31 ? ~0u : last < half * 32 ? 0u : (2u << (last - half * 32)) - 1u;
          far_slopes<T>(s_at, dp_at, lse, p.shifts + stat, minus_delta.x, p.scale_log2, sees);
        } else {
          tc::tmem_st16(dp_at, dsw);
        }
        tc::tmem_wait_st();
        tc::tc_fence_before();
        __syncwarp();
        tc::mbar_arrive(&bar.ds_ready[b], lane == 0);
      }
      // When the last S has arrived nobody reads this item's q and do any more: the next item's take their place, and its
      // first products begin, ahead of this one's stores.
      const int last_set = (w.steps - 1) & 1;
      all[0] += (w.steps + 1) / 2;
      all[1] += w.steps / 2;
      if (ok) ok = waiter.wait(&bar.s_full[last_set], (all[last_set] - 1) & 1);
      BwdItem next;
      for (int later = turn + 1; later < p.turns; ++later) {
        if (bwd_item<false, kWindow>(p, later, &next)) {
          into_tmem();
          break;
        }
      }
      if (ok) ok = waiter.wait(&bar.acc_full, outs & 1) && waiter.nobody_failed();
      ++outs;
      tc::tc_fence_after();
      // a thread has a quarter of its row's channels
      const int i = w.tile * 128 + row;
      const bool there = i < w.at.len;
      const float by = ok ? p.scale : NAN;
      T* to = static_cast<T*>(p.dq) + ((w.at.row + i) * p.heads + w.head) * p.dim;
      constexpr int kCols = DP / 4;
      const int col0 = (2 * b + half) * kCols;
#pragma unroll
      for (int x = 0; x < kCols; x += 16) {
        uint32_t raw[16];
        float o[16];
        tc::tmem_ld16(tmem + lane_base + col0 + x, raw);
        tc::tmem_wait_ld();
#pragma unroll
        for (int y = 0; y < 16; ++y) o[y] = __uint_as_float(raw[y]);
        if (there) store_row16<T>(to + col0 + x, o, by, p.dim - col0 - x, p.wide);
      }
      tc::tc_fence_before();
      __syncwarp();
      tc::mbar_arrive(&bar.acc_empty, lane == 0 && ok);
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 16) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
  outlast_others();   // the key kernel
}

// Keys: K and V of 128 keys stay; q and do of all queries that see them go by, 128 at a time, for every head of the group.
// One set of S^T and dP^T (128 columns each; the two sums have the rest of TMEM), in two phases that overlap the products:
//
//   products   dv += P^T do, S^T(i + 1) | dk += dS^T q, dP^T(i + 1) | ...
//   threads    dS(i) from dP^T(i)       | P(i + 1) from S^T(i + 1)  | ...
//
// P and dS (16-bit) overlay S^T and dP^T.  Sixteen warps, a quarter of a row a thread: its weights stay in registers from the
// first phase to the second.  A quarter of the exponentials is made on the FMA units.  3600 clocks a step of 128 queries, of
// which its products take the tensor cores 2048; what bounds it is the threads' two phases (1300 and 900) and the products
// between them.  (Two sets of 64 queries by turns, as for the queries: 146 us and not 129; P through shared memory, so that
// S^T need not wait for dv: 144 against 139.)
template <int DP>
struct KeyConfig {
  static constexpr int kTileBytes = 128 * DP * 2, kSlab = 128 * 128;
  static constexpr int kStages = DP == 128 ? 4 : 8;       // tiles of q and of do by turns
  static constexpr int kStats = kStages / 2;              // steps whose statistics are there
  static constexpr int kBytes = (2 + kStages) * kTileBytes + kStats * 2 * 128 * 4 + 512;
};

struct KeyBars {
  uint64_t stay_full, stay_empty, acc_full, acc_empty, raw, drained;
  uint64_t s_full, dp_full, p_ready, ds_ready, go_full[8], go_empty[8];
  uint32_t tmem;
  int failed;
};

// A thread's share of a step in which a query's reference is far away: P and dS as below, with weights as in far_weight.  `seen`
// is the first of its queries that sees the key, or with kBits has a bit for every one that does.  False where a wait ran out.
template <typename T, bool kBits>
__device__ __noinline__ bool far_step(KeyBars& bar, const Waiter& waiter, uint32_t parity, uint32_t s_at, uint32_t dp_at, const float* st,
                                      const float* shifts, float c, uint32_t seen) {
  float e[32];
  uint32_t w[16], x[32];
  tc::tmem_ld32(s_at, x);
  tc::tmem_wait_ld();
#pragma unroll
  for (int y = 0; y < 32; ++y) e[y] = (kBits ? ((seen >> y) & 1) == 0 : y < int(seen)) ? 0.f : far_weight(x[y], st[y], shifts + y, c);
#pragma unroll
  for (int y = 0; y < 16; ++y) w[y] = pack_pair<T>(e[2 * y], e[2 * y + 1]);
  tc::tmem_st16(s_at, w);
  tc::tmem_wait_st();
  tc::tc_fence_before();
  __syncwarp();
  tc::mbar_arrive(&bar.p_ready, (threadIdx.x & 31) == 0);
  if (!waiter.wait(&bar.dp_full, parity)) return false;
  tc::tc_fence_after();
  tc::tmem_ld32(dp_at, x);
  tc::tmem_wait_ld();
#pragma unroll
  for (int y = 0; y < 32; ++y) e[y] = (kBits ? ((seen >> y) & 1) == 0 : y < int(seen)) ? 0.f : e[y] * (__uint_as_float(x[y]) + st[128 + y]);
#pragma unroll
  for (int y = 0; y < 16; ++y) w[y] = pack_pair<T>(e[2 * y], e[2 * y + 1]);
  tc::tmem_st16(dp_at, w);
  tc::tmem_wait_st();
  tc::tc_fence_before();
  __syncwarp();
  tc::mbar_arrive(&bar.ds_ready, (threadIdx.x & 31) == 0);
  return true;
}

template <typename T, int DP, bool kWindow>
__global__ void __launch_bounds__(kThreads, 1) attention_keys_kernel(const __grid_constant__ BwdParams p) {
  using C = KeyConfig<DP>;
  extern __shared__ __align__(1024) uint8_t smem[];   // swizzled tiles: 1024-byte aligned, there is no static shared memory
  uint8_t* go = smem + 2 * C::kTileBytes;
  float* stats = reinterpret_cast<float*>(go + C::kStages * C::kTileBytes);   // [step by turns][-lse, -delta][128]
  KeyBars& bar = *reinterpret_cast<KeyBars*>(stats + C::kStats * 2 * 128);
  static_assert(sizeof(KeyBars) <= 512, "");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    tc::mbar_init(&bar.stay_full, 1);
    tc::mbar_init(&bar.stay_empty, 1);
    tc::mbar_init(&bar.acc_full, 1);
    tc::mbar_init(&bar.acc_empty, 16);
    tc::mbar_init(&bar.raw, 1);
    tc::mbar_init(&bar.drained, 1);
    tc::mbar_init(&bar.s_full, 1);
    tc::mbar_init(&bar.dp_full, 1);
    tc::mbar_init(&bar.p_ready, 16);
    tc::mbar_init(&bar.ds_ready, 16);
    for (int s = 0; s < C::kStages; ++s) {
      tc::mbar_init(&bar.go_full[s], 1);
      tc::mbar_init(&bar.go_empty[s], 1);
    }
    bar.failed = 0;
    tc::fence_mbar_init();
  }
  if (warp == 16) {
    tc::tmem_alloc(&bar.tmem, 512);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = bar.tmem;
  const Waiter waiter{&bar.failed, p.polls};
  asm volatile("griddepcontrol.wait;" ::: "memory");   // delta
  let_others_begin();

  if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");   // 640 threads of 96 registers = 512 of 104 + 128 of 64
    if (warp == 17) {
      // ---- copies ----------------------------------------------------------------------------------------
      tc::fence_async_all();   // delta was written by threads, and is read by bulk copies
      const uint32_t leader = tc::elect_leader();
      int filled = 0, stayed = 0, mended = 0;
      bool ok = true;
      for (int turn = 0; turn < p.turns && ok; ++turn) {
        BwdItem w;
        if (!bwd_item<true, kWindow>(p, turn, &w)) continue;
        if (stayed > 0 && !(ok = waiter.wait(&bar.stay_empty, (stayed - 1) & 1))) break;
        tc::mbar_arrive_expect_tx(&bar.stay_full, 2 * C::kTileBytes, leader);
#pragma unroll
        for (int slab = 0; slab < DP / 64; ++slab) {
          const int row = w.at.row0 + w.tile * 128;
          tc::tma_load_4d(smem + slab * C::kSlab, &p.k_tile, slab * 64, w.head, row, w.at.batch, &bar.stay_full, leader);
          tc::tma_load_4d(smem + C::kTileBytes + slab * C::kSlab, &p.v_tile, slab * 64, w.head, row, w.at.batch, &bar.stay_full, leader);
        }
        ++stayed;
        for (int i = 0; i < 2 * w.steps && ok; ++i) {   // q and do by turns
          const int s = filled % C::kStages, step = w.begin + (i >> 1);
          if (filled >= C::kStages && !(ok = waiter.wait(&bar.go_empty[s], (filled / C::kStages - 1) & 1))) break;
          const int g = step / w.per_head, at = (w.first + step - g * w.per_head) * 128;
          const int head = w.head * p.group + g;
          uint8_t* to = go + s * C::kTileBytes;
          // rows of the next sequence would meet weights of 0, but 0 * inf and 0 * NaN are not 0
          const int valid = w.at.len - at;
          const bool mend = p.seq.packed && valid < 128, queries = (i & 1) == 0;
          uint64_t* full = mend ? &bar.raw : &bar.go_full[s];
          tc::mbar_arrive_expect_tx(full, C::kTileBytes + (queries ? 2 * 128 * 4 : 0), leader);
#pragma unroll
          for (int slab = 0; slab < DP / 64; ++slab) {
            tc::tma_load_4d(to + slab * C::kSlab, queries ? &p.q_tile : &p.do_tile, slab * 64, head, w.at.row0 + at, w.at.batch, full, leader);
          }
          if (queries) {
            const int64_t from = head * p.seq.stat_rows + w.at.stat + at;
            float* st = stats + (filled >> 1) % C::kStats * 2 * 128;
            tc::bulk_g2s(st, p.lse + from, 128 * 4, full, leader);
            tc::bulk_g2s(st + 128, p.delta + from, 128 * 4, full, leader);
          }
          if (mend) {
            ok = waiter.wait(&bar.raw, mended & 1);
            ++mended;
#pragma unroll
            for (int slab = 0; slab < DP / 64; ++slab) {
              uint4* lines = reinterpret_cast<uint4*>(to + slab * C::kSlab);
              for (int x = valid * 8 + lane; x < 128 * 8; x += 32) lines[x] = make_uint4(0, 0, 0, 0);
            }
            tc::fence_async_smem();
            __syncwarp();
            tc::mbar_arrive(&bar.go_full[s], leader);
          }
          ++filled;
        }
      }
      if (!ok) {  // copies under way end before the CTA does
        for (int back = 1; back <= C::kStages && back <= filled; ++back) {
          const int x = filled - back;
          for (int i = 0; i < 4096 && !tc::mbar_try_wait(&bar.go_full[x % C::kStages], (x / C::kStages) & 1); ++i) {}
        }
        for (int i = 0; stayed > 0 && i < 4096 && !tc::mbar_try_wait(&bar.stay_full, (stayed - 1) & 1); ++i) {}
        for (int i = 0; mended > 0 && i < 4096 && !tc::mbar_try_wait(&bar.raw, (mended - 1) & 1); ++i) {}
      }
    } else if (warp == 16) {
      // ---- products --------------------------------------------------------------------------------------
      const uint32_t leader = tc::elect_leader();
      const uint32_t id_s = tc::idesc(128, 128, Format<T>::code, tc::kMajorK, tc::kMajorK, p.negate);
      const uint32_t id_dp = tc::idesc(128, 128, Format<T>::code, tc::kMajorK, tc::kMajorK);
      const uint32_t id_acc = tc::idesc(128, DP, Format<T>::code, tc::kMajorK, tc::kMajorMN);
      const uint32_t k_base = tc::smem_u32(smem), v_base = k_base + C::kTileBytes, go_base = tc::smem_u32(go);
      int used = 0, stayed = 0, steps = 0;   // tiles, items, steps
      bool ok = true;
      auto full = [&](int x) { return waiter.wait(&bar.go_full[x % C::kStages], (x / C::kStages) & 1); };
      auto scores = [&](int x) {   // S^T from the queries in stage x
        if (!full(x)) return false;
        tc::tc_fence_after();
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
          mma_ss(tmem + 256, desc_k(k_base, C::kSlab, ks), desc_k(go_base + (x % C::kStages) * C::kTileBytes, C::kSlab, ks), id_s, ks > 0, leader);
        }
        tc::mma_commit(&bar.s_full, leader);
        return true;
      };
      auto slopes = [&](int x) {   // dP^T
        if (!full(x)) return false;
        tc::tc_fence_after();
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
          mma_ss(tmem + 384, desc_k(v_base, C::kSlab, ks), desc_k(go_base + (x % C::kStages) * C::kTileBytes, C::kSlab, ks), id_dp, ks > 0, leader);
        }
        tc::mma_commit(&bar.dp_full, leader);
        return true;
      };
      for (int turn = 0; turn < p.turns && ok; ++turn) {
        BwdItem w;
        if (!bwd_item<true, kWindow>(p, turn, &w)) continue;
        if (!(ok = waiter.wait(&bar.stay_full, stayed & 1))) break;
        if (!(ok = scores(used)) || !(ok = slopes(used + 1))) break;
        for (int i = 0; i < w.steps && ok; ++i) {
          const int x = used + 2 * i;
          const bool more = i + 1 < w.steps;
          if (i == 0 && stayed > 0 && !(ok = waiter.wait(&bar.acc_empty, (stayed - 1) & 1))) break;
          if (!(ok = waiter.wait(&bar.p_ready, steps & 1))) break;
          tc::tc_fence_after();
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {   // the 16-bit numbers of a quarter of the queries are 32 columns apart
            mma_ts(tmem, tmem + 256 + (ks >> 1) * 32 + (ks & 1) * 8, desc_mn(go_base + ((x + 1) % C::kStages) * C::kTileBytes, C::kSlab, ks),
                   id_acc, i > 0 || ks > 0, leader);
          }
          tc::mma_commit(&bar.go_empty[(x + 1) % C::kStages], leader);
          if (more && !(ok = scores(x + 2))) break;
          if (!(ok = waiter.wait(&bar.ds_ready, steps & 1))) break;
          tc::tc_fence_after();
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {
            mma_ts(tmem + 128, tmem + 384 + (ks >> 1) * 32 + (ks & 1) * 8, desc_mn(go_base + (x % C::kStages) * C::kTileBytes, C::kSlab, ks),
                   id_acc, i > 0 || ks > 0, leader);
          }
          tc::mma_commit(&bar.go_empty[x % C::kStages], leader);
          if (more && !(ok = slopes(x + 3))) break;
          ++steps;
        }
        if (!ok) break;   // dk and dv lack a product, and are not reported
        tc::mma_commit(&bar.acc_full, leader);
        tc::mma_commit(&bar.stay_empty, leader);
        used += 2 * w.steps;
        ++stayed;
      }
      if (!ok) {  // products under way end before the CTA does
        tc::mma_commit(&bar.drained, leader);
        for (int i = 0; i < 4096 && !tc::mbar_try_wait(&bar.drained, 0); ++i) {}
      }
      __syncwarp();
    }
  } else {
    // ---- weights: four threads a row -----------------------------------------------------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    const int part = warp >> 2, row = threadIdx.x & 127;   // 32 of a step's queries, key
    const uint32_t lane_base = uint32_t(warp & 3) << 21;   // 32 lanes of TMEM, in bits 16 and up
    const uint32_t s_at = tmem + lane_base + 256 + part * 32, dp_at = s_at + 128;
    const float2 by_scale = twice(p.scale_log2);
    int steps = 0, outs = 0;
    bool ok = true;
    for (int turn = 0; turn < p.turns; ++turn) {
      BwdItem w;
      if (!bwd_item<true, kWindow>(p, turn, &w)) continue;
      int in_head = w.begin % w.per_head;
      for (int i = 0; i < w.steps && ok; ++i, ++steps) {
        const float* st = stats + steps % C::kStats * 2 * 128 + part * 32;
        // queries see keys up to themselves; a head's first step is the one on the diagonal
        const int from = row - part * 32, query = (w.first + in_head) * 128 + part * 32;
        const bool diagonal = kWindow ? !p.span.whole((w.first + in_head) * 128, 128, w.tile * 128, 128) : in_head == 0;
        uint32_t seen = ~0u;   // by which of its queries
        if (kWindow && diagonal) seen = p.span.seen(w.tile * 128 + row, query);
        if (++in_head == w.per_head) in_head = 0;
        if (!(ok = waiter.wait(&bar.s_full, steps & 1))) break;
        tc::tc_fence_after();
        uint32_t s[32], w16[16];
        float2 e[16];
        tc::tmem_ld32(s_at, s);
        const bool far = __any_sync(0xffffffffu, st[lane] > kFarFrom);
        tc::tmem_wait_ld();
        if (far) {
          const float* shifts = p.shifts + (w.head * p.group + (w.begin + i) / w.per_head) * p.seq.stat_rows + w.at.stat + query;
          if (!(ok = far_step<T, kWindow>(bar, waiter, steps & 1, s_at, dp_at, st, shifts, p.scale_log2,
                                          kWindow ? seen : uint32_t(diagonal ? from : 0)))) break;
          continue;
        }
#pragma unroll
        for (int y = 0; y < 16; y += 2) {
          const float4 l = *reinterpret_cast<const float4*>(st + 2 * y);
          const float2 a = fma2(make_float2(__uint_as_float(s[2 * y]), __uint_as_float(s[2 * y + 1])), by_scale, make_float2(l.x, l.y));
          const float2 b = fma2(make_float2(__uint_as_float(s[2 * y + 2]), __uint_as_float(s[2 * y + 3])), by_scale, make_float2(l.z, l.w));
          e[y] = exp2_2(a);
          e[y + 1] = (y & 2) != 0 ? exp2_fma(b) : exp2_2(b);
        }
        if (diagonal) {
#pragma unroll
          for (int y = 0; y < 16; ++y) {
            if (kWindow ? ((seen >> (2 * y)) & 1) == 0 : 2 * y < from) e[y].x = 0.f;
            if (kWindow ? ((seen >> (2 * y + 1)) & 1) == 0 : 2 * y + 1 < from) e[y].y = 0.f;
          }
        }
        // rounded to the inputs' type for their product, whose sums are in 32 bits
#pragma unroll
        for (int y = 0; y < 16; ++y) w16[y] = pack_pair<T>(e[y].x, e[y].y);
        tc::tmem_st16(s_at, w16);
        tc::tmem_wait_st();
        tc::tc_fence_before();
        __syncwarp();
        tc::mbar_arrive(&bar.p_ready, lane == 0);

        if (!(ok = waiter.wait(&bar.dp_full, steps & 1))) break;
        tc::tc_fence_after();
        tc::tmem_ld32(dp_at, s);
        tc::tmem_wait_ld();
#pragma unroll
        for (int y = 0; y < 16; y += 2) {
          const float4 d = *reinterpret_cast<const float4*>(st + 128 + 2 * y);
          e[y] = mul2(e[y], add2(make_float2(__uint_as_float(s[2 * y]), __uint_as_float(s[2 * y + 1])), make_float2(d.x, d.y)));
          e[y + 1] = mul2(e[y + 1], add2(make_float2(__uint_as_float(s[2 * y + 2]), __uint_as_float(s[2 * y + 3])), make_float2(d.z, d.w)));
        }
        if (diagonal) {   // 0 times what is not finite
#pragma unroll
          for (int y = 0; y < 16; ++y) {
            if (kWindow ? ((seen >> (2 * y)) & 1) == 0 : 2 * y < from) e[y].x = 0.f;
            if (kWindow ? ((seen >> (2 * y + 1)) & 1) == 0 : 2 * y + 1 < from) e[y].y = 0.f;
          }
        }
#pragma unroll
        for (int y = 0; y < 16; ++y) w16[y] = pack_pair<T>(e[y].x, e[y].y);
        tc::tmem_st16(dp_at, w16);
        tc::tmem_wait_st();
        tc::tc_fence_before();
        __syncwarp();
        tc::mbar_arrive(&bar.ds_ready, lane == 0);
      }
      if (ok) ok = waiter.wait(&bar.acc_full, outs & 1) && waiter.nobody_failed();
      ++outs;
      tc::tc_fence_after();
      // a thread has half of its row of dv or of dk
      const int i = w.tile * 128 + row;
      const bool there = i < w.at.len;
      const float by = !ok ? NAN : part < 2 ? 1.f : p.scale;
      const int64_t out_row = (w.at.row + i) * p.kv_heads + w.head;
      T* to = static_cast<T*>(part < 2 ? p.dv : p.dk) + out_row * p.dim;
      const bool sink = kWindow && w.sinks >= 0, whole = (sink ? p.sink_parts : p.parts) == 1;
      float* partial = p.partials + ((2 * w.part + (part < 2)) * p.partial_rows + out_row) * p.dim;
      if (sink) {
        const int64_t rows = int64_t(p.sink_tiles) * 128;
        partial = p.sink_partials + (((2 * w.part + (part < 2)) * p.seq.n * rows + w.sinks * rows + i) * p.kv_heads + w.head) * p.dim;
      }
      const int col0 = (part & 1) * (DP / 2);
#pragma unroll
      for (int x = 0; x < DP / 2; x += 16) {
        uint32_t raw[16];
        float o[16];
        tc::tmem_ld16(tmem + lane_base + (part >> 1) * 128 + col0 + x, raw);
        tc::tmem_wait_ld();
#pragma unroll
        for (int y = 0; y < 16; ++y) o[y] = __uint_as_float(raw[y]);
        if (!there) continue;
        if (whole) {
          store_row16<T>(to + col0 + x, o, by, p.dim - col0 - x, p.wide);
        } else {
#pragma unroll
          for (int y = 0; y < 16; y += 4) {
            if (col0 + x + y < p.dim) *reinterpret_cast<float4*>(partial + col0 + x + y) = make_float4(o[y] * by, o[y + 1] * by, o[y + 2] * by, o[y + 3] * by);
          }
        }
      }
      tc::tc_fence_before();
      __syncwarp();
      tc::mbar_arrive(&bar.acc_empty, lane == 0 && ok);
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 16) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

// -delta_i = -do_i . o_i in 32 bits, 0 for the rows behind a sequence's end: a CTA has 64 rows of a head, half a warp a row
constexpr int kDeltaRows = 64;
struct DeltaParams {
  const void *out, *d_out, *rest;   // rest: what the rounding of `out` has left over, or null
  int64_t do_stride[3];
  float* delta;
  int heads, dim;
  int rest_rows;                    // of sequences of up to so many rows
  Sequences seq;
};

template <typename T, bool kRest>
__global__ void __launch_bounds__(256) attention_delta_kernel(const __grid_constant__ DeltaParams p) {
  let_others_begin();
  const int unit = int(blockIdx.x) / p.heads, head = int(blockIdx.x) - unit * p.heads;
  const Item it = find_item(p.seq, unit / (kTileRows / kDeltaRows), false);
  const int first = it.tile * kTileRows + unit % (kTileRows / kDeltaRows) * kDeltaRows;
  const int part = threadIdx.x & 15, group = threadIdx.x >> 4;
  constexpr int kEach = kDeltaRows / 16;
  uint4 a[kEach], b[kEach], c[kEach];
#pragma unroll
  for (int x = 0; x < kEach; ++x) {
    const int i = first + x * 16 + group;
    a[x] = b[x] = c[x] = make_uint4(0, 0, 0, 0);
    if (i < it.len && part * 8 < p.dim) {
      a[x] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.out) + ((it.row + i) * p.heads + head) * p.dim + part * 8);
      b[x] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.d_out) + it.batch * p.do_stride[0] + int64_t(it.row0 + i) * p.do_stride[1] +
                                             head * p.do_stride[2] + part * 8);
      if (kRest && it.len <= p.rest_rows) c[x] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.rest) + ((it.row + i) * p.heads + head) * p.dim + part * 8);
    }
  }
#pragma unroll
  for (int x = 0; x < kEach; ++x) {
    const uint32_t aw[4] = {a[x].x, a[x].y, a[x].z, a[x].w}, bw[4] = {b[x].x, b[x].y, b[x].z, b[x].w}, cw[4] = {c[x].x, c[x].y, c[x].z, c[x].w};
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float2 u = unpack2<T>(aw[j]);
      const float2 v = unpack2<T>(bw[j]);
      if (kRest) u = add2(u, unpack2<T>(cw[j]));
      sum = fmaf(u.x, v.x, sum);
      sum = fmaf(u.y, v.y, sum);
    }
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (part == 0) p.delta[head * p.seq.stat_rows + it.stat + first + x * 16 + group] = -sum;
  }
}

// Where single items of the keys would take longer than all the rest (key_parts), each is cut into parts that sum over some
// of its steps (heads and queries) and leave their sums in 32 bits; these are added up here in the order of the parts, four
// channels a thread.
// CTAs behind those of all tiles have the tiles of the sinks.
template <typename T, bool kWindow>
__global__ void __launch_bounds__(256) attention_parts_kernel(const __grid_constant__ BwdParams p) {
  const int pieces = p.dim / 4;
  const int64_t x = int64_t(blockIdx.y) * blockDim.x + threadIdx.x;   // (row of the tile, kv head, piece)
  const int unit = int(blockIdx.x), others = kWindow && p.parts == 1 ? 0 : 2 * p.seq.tiles;
  const bool sink = kWindow && unit >= others;
  const int sequence = sink ? (unit - others) / p.sink_tiles : 0;
  const Item it = sink ? find_sequence(p.seq, sequence) : find_item(p.seq, unit >> 1, false);
  const int tile = sink ? unit - others - sequence * p.sink_tiles : 2 * it.tile + (unit & 1);
  const int i = tile * 128 + int(x / (p.kv_heads * pieces));
  if (i >= it.len || x >= int64_t(128) * p.kv_heads * pieces || (kWindow && !sink && tile < p.sink_tiles)) return;
  const int64_t at = ((it.row + tile * 128) * p.kv_heads * pieces + x) * 4;
  const int steps = (kWindow && !sink ? seeing_tiles(it.len, tile, p.span.window) : (it.len + 127) / 128 - tile) * p.group;
  const int parts = sink ? p.sink_parts : p.parts;
  const int64_t sink_rows = int64_t(p.sink_tiles) * 128;
  const float* from = sink ? p.sink_partials + ((sequence * sink_rows + tile * 128) * p.kv_heads * pieces + x) * 4 : p.partials + at;
  const int64_t next = (sink ? p.seq.n * sink_rows * p.kv_heads : p.partial_rows) * p.dim;
#pragma unroll
  for (int which = 0; which < 2; ++which) {   // dk, dv
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int part = 0; part < parts; ++part) {
      if (part_begin(steps, part, parts) == part_begin(steps, part + 1, parts)) continue;
      const float4 y = *reinterpret_cast<const float4*>(from + (2 * part + which) * next);
      sum.x += y.x; sum.y += y.y; sum.z += y.z; sum.w += y.w;
    }
    *reinterpret_cast<uint2*>(static_cast<T*>(which ? p.dv : p.dk) + at) = make_uint2(pack_pair<T>(sum.x, sum.y), pack_pair<T>(sum.z, sum.w));
  }
}

// One after the other, but a kernel begins on the SMs that the one before it has left: the key kernel waits for delta, and
// nobody's results are read by the query kernel, which begins after that wait.
template <typename Kernel>
int launch_half(Kernel kernel, int bytes, const BwdParams& base, int64_t items, cudaStream_t stream) {
  const cudaError_t err = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), bytes);
  if (err != cudaSuccess) { record_cuda_error(err); return GDN2_ERR_LAUNCH; }
  int sms = 0;
  const int status = multiprocessors(&sms);
  if (status != GDN2_OK) return status;
  BwdParams p = base;
  p.items = items;
  const int64_t grid = p.items < sms ? p.items : sms;
  p.turns = int((p.items + grid - 1) / grid);
  return launch_beside(kernel, unsigned(grid), kThreads, bytes, stream, p);
}

template <typename T, int DP, bool kWindow>
int launch_typed(BwdParams& p, const DeltaParams& d, cudaStream_t stream) {
  const unsigned ctas = unsigned(p.seq.tiles * (kTileRows / kDeltaRows) * p.heads);
  if (d.rest != nullptr) attention_delta_kernel<T, true><<<ctas, 256, 0, stream>>>(d);
  else attention_delta_kernel<T, false><<<ctas, 256, 0, stream>>>(d);
  int status = check_launch();
  if (status != GDN2_OK) return status;
  const int64_t tiles = int64_t(p.seq.tiles) * 2;
  p.sink_items = kWindow ? int64_t(p.seq.n) * p.sink_tiles * p.kv_heads * p.sink_parts : 0;
  status = launch_half(&attention_keys_kernel<T, DP, kWindow>, KeyConfig<DP>::kBytes, p, tiles * p.kv_heads * p.parts + p.sink_items, stream);
  if (status != GDN2_OK) return status;
  status = launch_half(&attention_queries_kernel<T, DP, kWindow>, QueryConfig<DP>::kBytes, p, tiles * p.heads, stream);
  if (status != GDN2_OK) return status;
  const unsigned per_tile = unsigned((int64_t(128) * p.kv_heads * (p.dim / 4) + 255) / 256);
  const int64_t joined = (p.parts > 1 ? tiles : 0) + (p.sink_parts > 1 ? int64_t(p.seq.n) * p.sink_tiles : 0);
  if (joined == 0) return GDN2_OK;
  attention_parts_kernel<T, kWindow><<<dim3(unsigned(joined), per_tile), 256, 0, stream>>>(p);
  return check_launch();
}

template <typename T>
int launch_dim(BwdParams& p, const DeltaParams& d, cudaStream_t stream) {
  if (p.span.window > 0) return p.dim <= 64 ? launch_typed<T, 64, true>(p, d, stream) : launch_typed<T, 128, true>(p, d, stream);
  return p.dim <= 64 ? launch_typed<T, 64, false>(p, d, stream) : launch_typed<T, 128, false>(p, d, stream);
}

}  // namespace

// Parts of the key kernel's items.  The first tile of the longest sequence has the most steps, and the other SMs have the
// rest of the keys and then the queries, about as many steps again, to do meanwhile: parts as many as bring it down to an
// SM's share of both.  16 heads; whole items / parts: 1 x 2048 tokens, 2 key heads (128 steps, a share of 29) 259 / 134 us;
// packed 700, 1200, 300 tokens, 2 key heads (80, 18) 173 / 128; 2 x 2048, 4 key heads (64, 118) 178 / 188; below sixteen
// steps, 1 x 1000 tokens, 8 heads (8, 4) 122 / 126.
// With a window of W tokens an item has a group's heads times the tiles that the window reaches, and the tiles of the sinks
// have all; those are cut by the same rule, but not finer than the others.
struct KeyParts { int parts, sink_tiles, sink_parts; };
static KeyParts key_parts(const int64_t* bounds, int64_t n_seq, int64_t time, int heads, int kv_heads, const Span& span, int sms) {
  const int group = heads / kv_heads;
  const int64_t reach = span.window > 0 ? (126 + span.window) / 128 + 1 : int64_t(1) << 40;   // tiles
  const int64_t sink_tiles = span.window > 0 ? (span.sinks + 127) / 128 : 0;
  int64_t longest = 0, all = 0;
  for (int64_t i = 0; i < (bounds != nullptr ? n_seq : 1); ++i) {
    const int64_t tiles = ((bounds != nullptr ? bounds[i + 1] - bounds[i] : time) + 127) / 128;
    longest = std::max(longest, tiles * group);
    const int64_t up = std::min(tiles, reach);   // items that have 1, 2, ... tiles of queries; the others have as many as is most
    all += (up * (up + 1) / 2 + (tiles - up) * up + std::min(sink_tiles, tiles) * (tiles - up)) * heads;
  }
  if (bounds == nullptr) all *= n_seq;
  const int64_t share = std::max<int64_t>(1, 2 * all / sms);
  auto parts = [&](int64_t steps, int64_t least) { return steps < 16 ? 1 : int(std::max<int64_t>(1, steps / std::max(share, least))); };
  const int64_t windowed = std::min(longest, span.window > 0 ? reach * group : longest);
  const int of_others = parts(windowed, 1);
  return {of_others, int(sink_tiles), sink_tiles > 0 ? parts(longest, std::max<int64_t>(1, windowed / of_others)) : 1};
}

// delta, then the parts' sums, then those of the sinks
struct BackwardBytes { int64_t delta, parts, sinks; };
static int backward_bytes(const int64_t* bounds, int64_t n_seq, int64_t time, int heads, int kv_heads, int dim, const Span& span, KeyParts* k,
                          BackwardBytes* bytes) {
  int sms = 0;
  const int status = multiprocessors(&sms);
  if (status != GDN2_OK) return status;
  *k = key_parts(bounds, n_seq, time, heads, kv_heads, span, sms);
  bytes->delta = (stat_rows(bounds, n_seq, time) * heads * 4 + 15) / 16 * 16;
  bytes->parts = k->parts == 1 ? 0 : int64_t(k->parts) * 2 * (bounds != nullptr ? time : n_seq * time) * kv_heads * dim * 4;
  const int64_t sequences = bounds != nullptr ? std::min<int64_t>(n_seq, kMaxSequences) : n_seq;   // of a launch
  bytes->sinks = k->sink_parts == 1 ? 0 : int64_t(k->sink_parts) * 2 * sequences * k->sink_tiles * 128 * kv_heads * dim * 4;
  return GDN2_OK;
}

int64_t attention_backward_bytes(const int64_t* bounds, int64_t n_seq, int64_t time, int heads, int kv_heads, int dim, int64_t window,
                                 int64_t sinks) {
  KeyParts k;
  BackwardBytes bytes;
  const int status = backward_bytes(bounds, n_seq, time, heads, kv_heads, dim, ways_of(window, sinks, bounds, n_seq, time, false).span, &k, &bytes);
  return status != GDN2_OK ? status : bytes.delta + bytes.parts + bytes.sinks;
}

int64_t attention_stat_rows(const int64_t* bounds, int64_t n_seq, int64_t time) { return stat_rows(bounds, n_seq, time); }

int launch_attention_backward(const void* q, const void* k, const void* v, const void* out, const void* rest, const void* d_out,
                              const float* lse, void* scratch, void* dq, void* dk, void* dv, const int64_t* strides,
                              const int64_t* bounds, int64_t n_seq, int64_t time, int heads, int kv_heads, int dim,
                              int dtype, float scale, int64_t window, int64_t sinks, cudaStream_t stream) {
  BwdParams p;
  const int64_t batch = bounds != nullptr ? 1 : n_seq;
  struct { CUtensorMap* map; const void* base; const int64_t* strides; int heads, rows; } maps[] = {
      {&p.q_tile, q, strides, heads, 128},         {&p.k_tile, k, strides + 3, kv_heads, 128},
      {&p.v_tile, v, strides + 6, kv_heads, 128},  {&p.do_tile, d_out, strides + 9, heads, 128},
      {&p.k_step, k, strides + 3, kv_heads, kStep}, {&p.v_step, v, strides + 6, kv_heads, kStep}};
  for (const auto& m : maps) {
    if (!encode_heads_map(m.map, m.base, m.strides, batch, time, m.heads, dim, dtype, m.rows)) return GDN2_ERR_LAUNCH;
  }
  p.dq = dq; p.dk = dk; p.dv = dv;
  float* delta = static_cast<float*>(scratch);
  p.lse = lse; p.delta = delta;
  p.shifts = lse + stat_rows(bounds, n_seq, time) * heads;
  const Ways ways = ways_of(window, sinks, bounds, n_seq, time, rest != nullptr);
  p.span = ways.span;
  KeyParts cut;
  BackwardBytes bytes;
  const int status = backward_bytes(bounds, n_seq, time, heads, kv_heads, dim, ways.span, &cut, &bytes);
  if (status != GDN2_OK) return status;
  p.parts = cut.parts;
  p.sink_tiles = cut.sink_tiles;
  p.sink_parts = cut.sink_parts;
  p.partials = delta + bytes.delta / 4;
  p.sink_partials = p.partials + bytes.parts / 4;
  p.partial_rows = batch * time * kv_heads;
  p.heads = heads; p.kv_heads = kv_heads; p.group = heads / kv_heads; p.dim = dim;
  p.scale = scale;
  p.negate = scale < 0.f;
  p.polls = wait_polls();
  p.wide = wide_rows(dq, dim) && wide_rows(dk, dim) && wide_rows(dv, dim);
  p.scale_log2 = positive_scale(scale);
  return for_groups(bounds, n_seq, time, false, &p.seq, [&](bool) -> int {
    DeltaParams d{out, d_out, rest, {strides[9], strides[10], strides[11]}, delta, heads, dim, ways.apart ? kShortRows : INT_MAX, p.seq};
    return dtype == GDN2_BF16 ? launch_dim<__nv_bfloat16>(p, d, stream) : launch_dim<__half>(p, d, stream);
  });
}

}  // namespace attn
}  // namespace gdn2
