// Causal attention, backward, on the tensor cores.  With the forward's statistics lse_i = m_i + log l_i:
//
//   p_ij = exp(scale q_i . k_j - lse_i)      delta_i = do_i . o_i      ds_ij = p_ij (do_i . v_j - delta_i)
//   dv_j = sum_i p_ij do_i      dk_j = scale sum_i ds_ij q_i      dq_i = scale sum_j ds_ij k_j
//
// Three kernels: delta (bound by HBM), then two of one shape.  A work item has 128 rows that stay, of two tensors X and
// Y, and goes through the rows that meet them, 64 at a time, of Xs and Ys:
//
//                   stay     go by       product 1   product 2    sums in TMEM
//   keys            k, v     q, do       S^T = X Xs^T  dP^T = Y Ys^T   dv += P^T Ys, dk += dS^T Xs
//   queries         q, do    k, v        S = X Xs^T    dP = Y Ys^T     dq += dS Xs
//
// Each of the two sums its rows' gradients by itself, over all query heads of a group too: no atomics, the same bits
// every time, at the price of forming S and dP twice (seven products in place of five).  The rows that go by alternate
// between two sets of S and dP: four warps make weights of one (a row a thread) while the tensor cores form the other.
//
// TMEM: keys: two sums of 128 columns, queries: one, and the rows that stay, 64 columns each; two sets of S and dP of 64
// each; P and dS (16-bit) overlay theirs.

#include "attention_common.cuh"

namespace gdn2 {
namespace attn {

namespace {

constexpr int kThreads = 640;    // warps 0-7: even steps; 8-15: odd ones; 16: products; 17: copies
constexpr int kStep = 64;        // rows of a step

template <int DP>
struct BwdConfig {
  static constexpr int kStayBytes = 128 * DP * 2, kStaySlab = 128 * 128;
  static constexpr int kGoBytes = kStep * DP * 2, kGoSlab = kStep * 128;
  static constexpr int kStages = DP == 128 ? 4 : 6;
  static constexpr int kBytes = 2 * kStayBytes + kStages * (2 * kGoBytes + 2 * kStep * 4) + 512;
};

struct BwdParams {
  CUtensorMap q_stay, do_stay, k_stay, v_stay, q_go, do_go, k_go, v_go;
  void *dq, *dk, *dv;
  const float *lse, *delta;
  int heads, kv_heads, group, dim, turns;
  int64_t items;
  float scale, scale_log2;   // scale_log2 is positive
  uint32_t negate;
  bool wide;                 // rows of the gradients are 32-byte aligned
  Sequences seq;
};

struct BwdBars {
  uint64_t stay_full, stay_empty, in_tmem, acc_full, acc_empty, raw, drained;
  uint64_t s_full[2], ds_ready[2], go_full[6], go_empty[6];
  uint32_t tmem;
  int failed;
};

struct BwdItem {
  Item at;
  int head, tile;       // of queries, or of keys; 128-row tile in the sequence
  int first, per_head, steps;  // first 64-row step, steps of a query head, of all
};

template <bool kKeys>
__device__ __forceinline__ bool bwd_item(const BwdParams& p, int turn, BwdItem* w) {
  const int64_t index = item_of_turn(turn);
  if (index >= p.items) return false;
  const int heads = kKeys ? p.kv_heads : p.heads;
  const int u = int(index / heads);
  w->head = int(index - int64_t(u) * heads);
  w->at = find_item(p.seq, u >> 1, !kKeys);
  w->tile = 2 * w->at.tile + (kKeys ? u & 1 : 1 - (u & 1));
  if (w->tile * 128 >= w->at.len) return false;
  const int all = (w->at.len + kStep - 1) / kStep;
  w->first = kKeys ? 2 * w->tile : 0;
  w->per_head = kKeys ? all - w->first : min(2 * w->tile + 2, all);
  w->steps = kKeys ? w->per_head * p.group : w->per_head;
  return true;
}

template <typename T, int DP, bool kKeys>
__global__ void __launch_bounds__(kThreads, 1) attention_backward_kernel(const __grid_constant__ BwdParams p) {
  using C = BwdConfig<DP>;
  extern __shared__ __align__(1024) uint8_t smem[];   // swizzled tiles: 1024-byte aligned, there is no static shared memory
  uint8_t* stay = smem;
  uint8_t* go = smem + 2 * C::kStayBytes;
  float* stats = reinterpret_cast<float*>(go + C::kStages * 2 * C::kGoBytes);   // [stage][lse, delta][64]
  BwdBars& bar = *reinterpret_cast<BwdBars*>(stats + C::kStages * 2 * kStep);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    tc::mbar_init(&bar.stay_full, 1);
    tc::mbar_init(&bar.stay_empty, kKeys ? 1 : 16);
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
  const Waiter waiter{&bar.failed};

  if (warp >= 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");   // 640 threads of 96 registers = 512 of 104 + 128 of 64
    if (warp == 17) {
      // ---- copies ----------------------------------------------------------------------------------------
      const uint32_t leader = tc::elect_leader();
      int filled = 0, stayed = 0, mended = 0;
      bool ok = true;
      for (int turn = 0; turn < p.turns && ok; ++turn) {
        BwdItem w;
        if (!bwd_item<kKeys>(p, turn, &w)) continue;
        const int kv_head = kKeys ? w.head : w.head / p.group;
        if (stayed > 0) ok = waiter.wait(&bar.stay_empty, (stayed - 1) & 1);
        if (!ok) break;
        tc::mbar_arrive_expect_tx(&bar.stay_full, 2 * C::kStayBytes, leader);
#pragma unroll
        for (int slab = 0; slab < DP / 64; ++slab) {
          const int row = w.at.row0 + w.tile * 128;
          tc::tma_load_4d(stay + slab * C::kStaySlab, kKeys ? &p.k_stay : &p.q_stay, slab * 64, w.head, row, w.at.batch, &bar.stay_full, leader);
          tc::tma_load_4d(stay + C::kStayBytes + slab * C::kStaySlab, kKeys ? &p.v_stay : &p.do_stay, slab * 64, w.head, row, w.at.batch,
                          &bar.stay_full, leader);
        }
        ++stayed;
        for (int i = 0; i < w.steps && ok; ++i) {
          const int s = filled % C::kStages;
          if (filled >= C::kStages) ok = waiter.wait(&bar.go_empty[s], (filled / C::kStages - 1) & 1);
          if (!ok) break;
          const int g = i / w.per_head, at = (w.first + i - g * w.per_head) * kStep;
          const int head = kKeys ? w.head * p.group + g : kv_head;
          uint8_t* to = go + s * 2 * C::kGoBytes;
          // rows of the next sequence would meet weights of 0, but 0 * inf and 0 * NaN are not 0
          const int valid = w.at.len - at;
          const bool mend = p.seq.packed && valid < kStep;
          uint64_t* full = mend ? &bar.raw : &bar.go_full[s];
          tc::mbar_arrive_expect_tx(full, 2 * C::kGoBytes + (kKeys ? 2 * kStep * 4 : 0), leader);
#pragma unroll
          for (int slab = 0; slab < DP / 64; ++slab) {
            tc::tma_load_4d(to + slab * C::kGoSlab, kKeys ? &p.q_go : &p.k_go, slab * 64, head, w.at.row0 + at, w.at.batch, full, leader);
            tc::tma_load_4d(to + C::kGoBytes + slab * C::kGoSlab, kKeys ? &p.do_go : &p.v_go, slab * 64, head, w.at.row0 + at, w.at.batch,
                            full, leader);
          }
          if (kKeys) {
            const int64_t from = head * p.seq.stat_rows + w.at.stat + at;
            tc::bulk_g2s(stats + s * 2 * kStep, p.lse + from, kStep * 4, full, leader);
            tc::bulk_g2s(stats + s * 2 * kStep + kStep, p.delta + from, kStep * 4, full, leader);
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
      }
    } else if (warp == 16) {
      // ---- products --------------------------------------------------------------------------------------
      const uint32_t leader = tc::elect_leader();
      const uint32_t id_s = tc::idesc(128, kStep, Format<T>::code, tc::kMajorK, tc::kMajorK, p.negate);
      const uint32_t id_dp = tc::idesc(128, kStep, Format<T>::code, tc::kMajorK, tc::kMajorK);
      const uint32_t id_acc = tc::idesc(128, DP, Format<T>::code, tc::kMajorK, tc::kMajorMN);
      const uint32_t x_base = tc::smem_u32(stay), y_base = x_base + C::kStayBytes, go_base = tc::smem_u32(go);
      int used = 0, stayed = 0, ready[2] = {0, 0};
      bool ok = true;
      auto both = [&](int b, int x) {   // S and dP of the step in stage x
        if (!waiter.wait(&bar.go_full[x % C::kStages], (x / C::kStages) & 1)) return false;
        tc::tc_fence_after();
        const uint32_t xs = go_base + (x % C::kStages) * 2 * C::kGoBytes, ys = xs + C::kGoBytes;
        const uint32_t s_at = tmem + 256 + b * 128, dp_at = s_at + 64;
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
          if (kKeys) mma_ss(s_at, desc_k(x_base, C::kStaySlab, ks), desc_k(xs, C::kGoSlab, ks), id_s, ks > 0, leader);
          else mma_ts(s_at, tmem + 128 + ks * 8, desc_k(xs, C::kGoSlab, ks), id_s, ks > 0, leader);
        }
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
          if (kKeys) mma_ss(dp_at, desc_k(y_base, C::kStaySlab, ks), desc_k(ys, C::kGoSlab, ks), id_dp, ks > 0, leader);
          else mma_ts(dp_at, tmem + 192 + ks * 8, desc_k(ys, C::kGoSlab, ks), id_dp, ks > 0, leader);
        }
        tc::mma_commit(&bar.s_full[b], leader);
        return true;
      };
      for (int turn = 0; turn < p.turns && ok; ++turn) {
        BwdItem w;
        if (!bwd_item<kKeys>(p, turn, &w)) continue;
        ok = waiter.wait(kKeys ? &bar.stay_full : &bar.in_tmem, stayed & 1);
        if (ok) ok = both(0, used);
        if (ok && w.steps > 1) ok = both(1, used + 1);
        for (int i = 0; i < w.steps && ok; ++i) {
          const int b = i & 1, x = used + i;
          if (i == 0 && stayed > 0 && !(ok = waiter.wait(&bar.acc_empty, (stayed - 1) & 1))) break;
          if (!(ok = waiter.wait(&bar.ds_ready[b], ready[b] & 1))) break;
          ++ready[b];
          tc::tc_fence_after();
          const uint32_t xs = go_base + (x % C::kStages) * 2 * C::kGoBytes, ys = xs + C::kGoBytes;
          const uint32_t p_at = tmem + 256 + b * 128, ds_at = p_at + 64;
          if (kKeys) {
#pragma unroll
            for (int ks = 0; ks < kStep / 16; ++ks) mma_ts(tmem, p_at + (ks >> 1) * 32 + (ks & 1) * 8, desc_mn(ys, C::kGoSlab, ks), id_acc, i > 0 || ks > 0, leader);
          }
#pragma unroll
          for (int ks = 0; ks < kStep / 16; ++ks) mma_ts(kKeys ? tmem + 128 : tmem, ds_at + (ks >> 1) * 32 + (ks & 1) * 8, desc_mn(xs, C::kGoSlab, ks), id_acc, i > 0 || ks > 0, leader);
          tc::mma_commit(&bar.go_empty[x % C::kStages], leader);
          if (i + 1 == w.steps) {
            tc::mma_commit(&bar.acc_full, leader);
            if (kKeys) tc::mma_commit(&bar.stay_empty, leader);
          }
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
    int used = 0, seen = 0, outs = 0, stayed = 0;
    bool ok = true;
    // Queries: a product whose first operand comes from TMEM reads a third of the shared memory (16 KiB of the rows that go
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
      tc::mbar_arrive(&bar.stay_empty, lane == 0);
      tc::mbar_arrive(&bar.in_tmem, lane == 0);
    };
    for (int turn = 0; turn < p.turns; ++turn) {
      BwdItem w;
      if (!bwd_item<kKeys>(p, turn, &w)) continue;
      float lse = 0.f, delta = 0.f;
      if (!kKeys) {
        if (stayed == outs) into_tmem();
        const int64_t at = w.head * p.seq.stat_rows + w.at.stat + w.tile * 128 + row;
        lse = p.lse[at];
        delta = p.delta[at];
      }
      for (int i = b; i < w.steps && ok; i += 2) {
        if (!(ok = waiter.wait(&bar.s_full[b], seen & 1))) break;
        ++seen;
        tc::tc_fence_after();
        const int g = i / w.per_head, at = (w.first + i - g * w.per_head) * kStep;
        // queries see keys up to themselves: of the rows that go by, x from `from` on (keys), up to `from` (queries)
        const int from = w.tile * 128 + row - at;
        const bool diagonal = kKeys ? at < w.tile * 128 + 128 : at + kStep > w.tile * 128;
        const float* st = stats + ((used + i) % C::kStages) * 2 * kStep;
        uint32_t s[32], dp[32], pw[16], dsw[16];
        tc::tmem_ld32(s_at, s);
        tc::tmem_ld32(dp_at, dp);
        tc::tmem_wait_ld();
#pragma unroll
        for (int y = 0; y < 32; y += 2) {
          const int x = half * 32 + y;
          float2 l = twice(lse), d = twice(delta);
          if (kKeys) {
            l = *reinterpret_cast<const float2*>(st + x);
            d = *reinterpret_cast<const float2*>(st + kStep + x);
          }
          const float2 sc = fma2(make_float2(__uint_as_float(s[y]), __uint_as_float(s[y + 1])), twice(p.scale_log2), minus2(make_float2(0.f, 0.f), l));
          float2 e = exp2_2(sc);
          float2 ds = mul2(e, minus2(make_float2(__uint_as_float(dp[y]), __uint_as_float(dp[y + 1])), d));
          if (diagonal) {
            if (kKeys ? x < from : x > from) { e.x = 0.f; ds.x = 0.f; }
            if (kKeys ? x + 1 < from : x + 1 > from) { e.y = 0.f; ds.y = 0.f; }
          }
          // both are rounded to the inputs' type for their products, the sums are in 32 bits
          if (kKeys) pw[y / 2] = pack_pair<T>(e.x, e.y);
          dsw[y / 2] = pack_pair<T>(ds.x, ds.y);
        }
        if (kKeys) tc::tmem_st16(s_at, pw);
        tc::tmem_st16(dp_at, dsw);
        tc::tmem_wait_st();
        tc::tc_fence_before();
        __syncwarp();
        tc::mbar_arrive(&bar.ds_ready[b], lane == 0);
      }
      used += w.steps;
      if (ok) ok = waiter.wait(&bar.acc_full, outs & 1);
      ++outs;
      tc::tc_fence_after();
      if (!kKeys) {   // the next item's, ahead of this one's stores
        BwdItem next;
        for (int later = turn + 1; later < p.turns; ++later) {
          if (bwd_item<kKeys>(p, later, &next)) {
            into_tmem();
            break;
          }
        }
      }
      // keys: eight warps have dv, the others dk, a thread half of a row's channels; queries: a quarter of dq's
      const int i = w.tile * 128 + row;
      const bool there = i < w.at.len;
      const float by = !ok ? NAN : kKeys && b == 0 ? 1.f : p.scale;
      const int64_t out_row = ((w.at.row + i) * (kKeys ? p.kv_heads : p.heads) + w.head) * p.dim;
      T* to = static_cast<T*>(kKeys ? (b == 0 ? p.dv : p.dk) : p.dq) + out_row;
      const uint32_t acc = tmem + lane_base + (kKeys ? b * 128 : 0);
      constexpr int kCols = kKeys ? DP / 2 : DP / 4;
      const int col0 = kKeys ? half * kCols : (2 * b + half) * kCols;
#pragma unroll
      for (int x = 0; x < kCols; x += 16) {
        uint32_t raw[16];
        float o[16];
        tc::tmem_ld16(acc + col0 + x, raw);
        tc::tmem_wait_ld();
#pragma unroll
        for (int y = 0; y < 16; ++y) o[y] = __uint_as_float(raw[y]);
        if (there) store_row16<T>(to + col0 + x, o, by, p.dim - col0 - x, p.wide);
      }
      tc::tc_fence_before();
      __syncwarp();
      tc::mbar_arrive(&bar.acc_empty, lane == 0);
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 16) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

// delta_i = do_i . o_i in 32 bits, 0 for the rows behind a sequence's end: a CTA has 256 rows of a head, half a warp a row
struct DeltaParams {
  const void *out, *d_out;
  int64_t do_stride[3];
  float* delta;
  int heads, dim;
  Sequences seq;
};

template <typename T>
__global__ void __launch_bounds__(256) attention_delta_kernel(const __grid_constant__ DeltaParams p) {
  const int t = int(blockIdx.x) / p.heads, head = int(blockIdx.x) - t * p.heads;
  const Item it = find_item(p.seq, t, false);
  const int part = threadIdx.x & 15, group = threadIdx.x >> 4;
  float* to = p.delta + head * p.seq.stat_rows + it.stat + it.tile * kTileRows;
#pragma unroll 4
  for (int r = group; r < kTileRows; r += 16) {
    const int i = it.tile * kTileRows + r;
    float sum = 0.f;
    if (i < it.len && part * 8 < p.dim) {
      const T* o = static_cast<const T*>(p.out) + ((it.row + i) * p.heads + head) * p.dim;
      const T* d = static_cast<const T*>(p.d_out) + it.batch * p.do_stride[0] + int64_t(it.row0 + i) * p.do_stride[1] + head * p.do_stride[2];
      const uint4 a = *reinterpret_cast<const uint4*>(o + part * 8), b = *reinterpret_cast<const uint4*>(d + part * 8);
      const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 x = unpack2<T>(aw[j]), y = unpack2<T>(bw[j]);
        sum = fmaf(x.x, y.x, sum);
        sum = fmaf(x.y, y.y, sum);
      }
    }
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (part == 0) to[r] = sum;
  }
}

template <typename T, int DP, bool kKeys>
int launch_half(const BwdParams& base, cudaStream_t stream) {
  using C = BwdConfig<DP>;
  const void* kernel = reinterpret_cast<const void*>(&attention_backward_kernel<T, DP, kKeys>);
  const cudaError_t err = ensure_dynamic_smem(kernel, C::kBytes);
  if (err != cudaSuccess) { record_cuda_error(err); return GDN2_ERR_LAUNCH; }
  int sms = 0;
  const int status = multiprocessors(&sms);
  if (status != GDN2_OK) return status;
  BwdParams p = base;
  p.items = int64_t(p.seq.tiles) * 2 * (kKeys ? p.kv_heads : p.heads);
  const int64_t grid = p.items < sms ? p.items : sms;
  p.turns = int((p.items + grid - 1) / grid);
  attention_backward_kernel<T, DP, kKeys><<<unsigned(grid), kThreads, C::kBytes, stream>>>(p);
  return check_launch();
}

template <typename T, int DP>
int launch_typed(const BwdParams& p, const DeltaParams& d, cudaStream_t stream) {
  attention_delta_kernel<T><<<unsigned(p.seq.tiles * p.heads), 256, 0, stream>>>(d);
  int status = check_launch();
  if (status != GDN2_OK) return status;
  status = launch_half<T, DP, true>(p, stream);
  return status != GDN2_OK ? status : launch_half<T, DP, false>(p, stream);
}

}  // namespace

int64_t attention_stat_rows(const int64_t* bounds, int64_t n_seq, int64_t time) { return stat_rows(bounds, n_seq, time); }

int launch_attention_backward(const void* q, const void* k, const void* v, const void* out, const void* d_out,
                              const float* lse, float* delta, void* dq, void* dk, void* dv, const int64_t* strides,
                              const int64_t* bounds, int64_t n_seq, int64_t time, int heads, int kv_heads, int dim,
                              int dtype, float scale, cudaStream_t stream) {
  BwdParams p;
  const int64_t batch = bounds != nullptr ? 1 : n_seq;
  struct { CUtensorMap* map; const void* base; const int64_t* strides; int heads, rows; } maps[] = {
      {&p.q_stay, q, strides, heads, 128},         {&p.k_stay, k, strides + 3, kv_heads, 128},
      {&p.v_stay, v, strides + 6, kv_heads, 128},  {&p.do_stay, d_out, strides + 9, heads, 128},
      {&p.q_go, q, strides, heads, kStep},         {&p.k_go, k, strides + 3, kv_heads, kStep},
      {&p.v_go, v, strides + 6, kv_heads, kStep},  {&p.do_go, d_out, strides + 9, heads, kStep}};
  for (const auto& m : maps) {
    if (!encode_heads_map(m.map, m.base, m.strides, batch, time, m.heads, dim, dtype, m.rows)) return GDN2_ERR_LAUNCH;
  }
  p.dq = dq; p.dk = dk; p.dv = dv;
  p.lse = lse; p.delta = delta;
  p.heads = heads; p.kv_heads = kv_heads; p.group = heads / kv_heads; p.dim = dim;
  p.scale = scale;
  p.negate = scale < 0.f;
  p.wide = wide_rows(dq, dim) && wide_rows(dk, dim) && wide_rows(dv, dim);
  p.scale_log2 = fmaxf(fabsf(scale) * kLog2e, 1e-30f);
  return for_groups(bounds, n_seq, time, &p.seq, [&]() -> int {
    DeltaParams d{out, d_out, {strides[9], strides[10], strides[11]}, delta, heads, dim, p.seq};
    if (dtype == GDN2_BF16) {
      return dim <= 64 ? launch_typed<__nv_bfloat16, 64>(p, d, stream) : launch_typed<__nv_bfloat16, 128>(p, d, stream);
    }
    return dim <= 64 ? launch_typed<__half, 64>(p, d, stream) : launch_typed<__half, 128>(p, d, stream);
  });
}

}  // namespace attn
}  // namespace gdn2
