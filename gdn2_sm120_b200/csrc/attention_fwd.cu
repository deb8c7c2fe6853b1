// Causal attention over whole prompts, forward, on the tensor cores.
//
//   s_ij = scale q_i . k_j (j <= i)    m_i = max_j s_ij    o_i = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i)
//
// One pass over keys and values with a running reference and sum.  A work item is 256 query rows of one head, two tiles of
// 128, against tiles of 128 keys.  The two tiles take turns: while the tensor cores form one's O += P V and next S = Q K^T,
// eight warps turn the other's S into P, two threads a row.  A tile of 128 x 128 x 128 takes the tensor cores 1024 clocks for
// its two products, the shared memory that they read as long (64 KiB for S, 32 for P V, 64 arrive for both tiles), and the
// special-function unit 1024 for its exponentials, less a quarter on the FMA units.
//
// 8 prompts of 4096 tokens, 16 heads of 128 channels, 4 heads a group: 461 to 474 us alone (by the machine), 1.17 PFLOP/s (72 %
// of the measured 1.63); one of 16381 tokens, 8 heads 424 us, 1.30.  Back to back under the power cap 550 to 565 and 505 us.
// The products by themselves, with nobody waiting for anybody, take 376 us of them: what bounds it is the tensor cores' own rate
// with operands from shared memory, then the round trip of a chain.
//
// TMEM (512 columns): S0 S1 O0 O1, 128 each; P (16-bit) overlays the first 32 of its half's 64 columns of S and is the A
// operand of P V from there.  Products are issued in an order that needs no further waits: S_t(j+1) after O_t += P_t(j) V, so
// an S that has arrived says that the O before it has, too.  The items are shared by turns that go up and down the list of
// them, the longest first.

#include "attention_common.cuh"

namespace gdn2 {
namespace attn {

namespace {

constexpr int kThreads = 576;    // warps 0-7, 8-15: the rows of the two tiles; 16: products; 17: copies

template <int DP>
struct FwdConfig {
  static constexpr int kTileBytes = 128 * DP * 2;
  static constexpr int kSlab = 128 * 128;               // 64 channels of 128 rows
  static constexpr int kStages = DP == 128 ? 5 : 8;
  static constexpr int kBarBytes = 1024;
  static constexpr int kBytes = (2 + kStages) * kTileBytes + kBarBytes + 2 * 2 * 128 * 4;
};

struct FwdParams {
  CUtensorMap q, k, v;
  const void* values;
  int64_t strides[3];  // of the values: batch, token and head, in elements
  void* out;
  float* lse;          // [heads][stat rows]: -(m + log2 l) in powers of two, then far references; or null
  int heads, kv_heads, group, dim, turns;
  int64_t items;
  float scale_log2;    // positive
  uint32_t negate;     // the scale is negative: Q counts with its sign changed
  uint32_t polls;      // of a wait
  bool wide;           // rows of the output are 32-byte aligned
  Sequences seq;
};

struct FwdBars {
  uint64_t q_full[2], q_empty[2], s_full[2], p_ready[2], o_full[2];
  uint64_t raw;        // a tile that is mended before the products may read it
  uint64_t drained;
  uint64_t kv_full[8], kv_empty[8];
};
struct FwdMarks {
  uint32_t again[32];      // items to be done once more, a bit a turn modulo 1024 (another one of that bit is done for nothing)
  uint32_t strange[4][8];  // rows of an item's two diagonal tiles with values that are not finite, of the last four such items
  uint32_t tmem;
  int failed;
};

// In the tile on the diagonal a row meets values that it does not see, with weights of 0; but 0 * inf and 0 * NaN are not 0.
// Nothing is looked for in advance: where a row comes out infinite or NaN, its item is marked, and the CTA goes through its
// marked items once more when it has done them all.  Then values that are not finite leave the tiles on the diagonals, and
// are added here to the rows that see them: `to` is a row's output, the last of the rows `seen` of these tiles; strange[] has
// a bit for every row of the two tiles from v on that held such a value.
template <typename T>
__device__ __noinline__ void add_strange(const T* v, int64_t stride, const uint32_t* strange, int seen, T* to, int channels) {
#pragma unroll 1
  for (int x = 0; x < channels; x += 8) {
    uint4 out = *reinterpret_cast<const uint4*>(to + x);
    uint32_t(&w)[4] = reinterpret_cast<uint32_t(&)[4]>(out);
    float o[8];
#pragma unroll
    for (int y = 0; y < 4; ++y) { const float2 u = unpack2<T>(w[y]); o[2 * y] = u.x; o[2 * y + 1] = u.y; }
    bool done = false;      // all of them are NaN
    for (int j0 = 0; j0 <= seen; j0 += 32) {
      uint32_t bits = strange[j0 >> 5];
      if (seen - j0 < 31) bits &= (2u << (seen - j0)) - 1u;
      for (; bits != 0 && !done; bits &= bits - 1) {
        const uint4 raw = *reinterpret_cast<const uint4*>(v + (j0 + __ffs(bits) - 1) * stride + x);
        const uint32_t r[4] = {raw.x, raw.y, raw.z, raw.w};
        done = true;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const float2 u = unpack2<T>(r[y]);
          if (!isfinite(u.x)) o[2 * y] += u.x;
          if (!isfinite(u.y)) o[2 * y + 1] += u.y;
          done = done && isnan(o[2 * y]) && isnan(o[2 * y + 1]);
        }
      }
    }
#pragma unroll
    for (int y = 0; y < 4; ++y) w[y] = pack_pair<T>(o[2 * y], o[2 * y + 1]);
    *reinterpret_cast<uint4*>(to + x) = out;
  }
}

template <int kStages>
__device__ __forceinline__ void init_bars(FwdBars& bar) {
  for (int t = 0; t < 2; ++t) {
    tc::mbar_init(&bar.q_full[t], 1);
    tc::mbar_init(&bar.q_empty[t], 1);
    tc::mbar_init(&bar.s_full[t], 1);
    tc::mbar_init(&bar.p_ready[t], 8);
    tc::mbar_init(&bar.o_full[t], 1);
  }
  tc::mbar_init(&bar.raw, 1);
  tc::mbar_init(&bar.drained, 1);
  for (int s = 0; s < kStages; ++s) {
    tc::mbar_init(&bar.kv_full[s], 1);
    tc::mbar_init(&bar.kv_empty[s], 1);
  }
  tc::fence_mbar_init();
}

// All items of the CTA, or the marked ones once more
template <typename T, int DP, bool kAgain>
__device__ __forceinline__ void forward_items(const FwdParams& p, uint8_t* smem, FwdBars& bar, FwdMarks& marks, float (*told)[2][128],
                                              uint32_t tmem) {
  using C = FwdConfig<DP>;
  uint8_t* q_tiles = smem;
  uint8_t* kv_tiles = smem + 2 * C::kTileBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Waiter waiter{&marks.failed, p.polls};

  // an item's head, rows and numbers of key tiles
  auto item_at = [&](int64_t index, int* head) {
    const int t = int(index / p.heads);
    *head = int(index - int64_t(t) * p.heads);
    return find_item(p.seq, t, true);
  };
  auto key_tiles = [](const Item& it, int t) {  // of the first or second query tile
    const int tile = 2 * it.tile + t;
    return tile * 128 < it.len ? tile + 1 : 0;
  };

  auto marked = [&](int turn) { return ((marks.again[(turn >> 5) & 31] >> (turn & 31)) & 1) != 0; };

  if (warp >= 16) {
    if (warp == 17) {
      // ---- copies ------------------------------------------------------------------------------------------
      const uint32_t leader = tc::elect_leader();
      int filled = 0, loaded[2] = {0, 0}, mended = 0, redone = 0;
      bool ok = true;
      auto load = [&](const CUtensorMap* map, uint8_t* to, int head, int row, int batch, uint64_t* full) {
        tc::mbar_arrive_expect_tx(full, C::kTileBytes, leader);
  #pragma unroll
        for (int slab = 0; slab < DP / 64; ++slab) {
          tc::tma_load_4d(to + slab * C::kSlab, map, slab * 64, head, row, batch, full, leader);
        }
      };
      for (int turn = 0; turn < p.turns && ok; ++turn) {
        const int64_t index = item_of_turn(turn);
        if (index >= p.items || (kAgain && !marked(turn))) continue;
        redone += kAgain;
        int head;
        const Item it = item_at(index, &head);
        const int kv_head = head / p.group;
        const int n = max(key_tiles(it, 0), key_tiles(it, 1));
        for (int j = 0; j < n && ok; ++j) {
          if (j == 0) {
            for (int t = 0; t < 2 && ok; ++t) {
              if (key_tiles(it, t) == 0) continue;
              if (loaded[t] > 0) ok = waiter.wait(&bar.q_empty[t], (loaded[t] - 1) & 1);
              if (!ok) break;
              load(&p.q, q_tiles + t * C::kTileBytes, head, it.row0 + (2 * it.tile + t) * 128, it.batch, &bar.q_full[t]);
              ++loaded[t];
              if (t == 0) {  // the first product needs no more than this
                const int s = filled % C::kStages;
                if (filled >= C::kStages) ok = waiter.wait(&bar.kv_empty[s], (filled / C::kStages - 1) & 1);
                if (!ok) break;
                load(&p.k, kv_tiles + s * C::kTileBytes, kv_head, it.row0, it.batch, &bar.kv_full[s]);
                ++filled;
              }
            }
          } else {
            const int s = filled % C::kStages;
            if (filled >= C::kStages) ok = waiter.wait(&bar.kv_empty[s], (filled / C::kStages - 1) & 1);
            if (!ok) break;
            load(&p.k, kv_tiles + s * C::kTileBytes, kv_head, it.row0 + j * 128, it.batch, &bar.kv_full[s]);
            ++filled;
          }
          if (!ok) break;
          const int s = filled % C::kStages;
          if (filled >= C::kStages) ok = waiter.wait(&bar.kv_empty[s], (filled / C::kStages - 1) & 1);
          if (!ok) break;
          uint8_t* to = kv_tiles + s * C::kTileBytes;
          const int valid = it.len - j * 128;   // rows of the sequence
          const bool diagonal = kAgain && j >= 2 * it.tile;   // of one of the two tiles of queries
          if (diagonal || (p.seq.packed && valid < 128)) {
            // rows of the next sequence: their weights are 0, but 0 * inf and 0 * NaN are not
            load(&p.v, to, kv_head, it.row0 + j * 128, it.batch, &bar.raw);
            ok = waiter.wait(&bar.raw, mended & 1);
            ++mended;
  #pragma unroll
            for (int slab = 0; slab < DP / 64; ++slab) {
              uint4* lines = reinterpret_cast<uint4*>(to + slab * C::kSlab);
              for (int x = valid * 8 + lane; x < 128 * 8; x += 32) lines[x] = make_uint4(0, 0, 0, 0);
            }
            if (diagonal) {
              // (when an item's queries could be loaded, nobody reads the rows of the one three before it any more)
              uint32_t* strange = marks.strange[redone & 3];
              if (j == 2 * it.tile && lane < 8) strange[lane] = 0;
              sift<T, DP>(tc::smem_u32(to), C::kSlab, 0, min(valid, 128),
                          [&](int row) { atomicOr(&strange[(j - 2 * it.tile) * 4 + (row >> 5)], 1u << (row & 31)); });
            }
            tc::fence_async_smem();
            __syncwarp();
            tc::mbar_arrive(&bar.kv_full[s], leader);
          } else {
            load(&p.v, to, kv_head, it.row0 + j * 128, it.batch, &bar.kv_full[s]);
          }
          ++filled;
        }
      }
      if (!ok) {  // copies under way end before the CTA does
        for (int back = 1; back <= C::kStages && back <= filled; ++back) {
          const int x = filled - back;
          for (int i = 0; i < 4096 && !tc::mbar_try_wait(&bar.kv_full[x % C::kStages], (x / C::kStages) & 1); ++i) {}
        }
        for (int t = 0; t < 2; ++t) {
          for (int i = 0; loaded[t] > 0 && i < 4096 && !tc::mbar_try_wait(&bar.q_full[t], (loaded[t] - 1) & 1); ++i) {}
        }
        for (int i = 0; mended > 0 && i < 4096 && !tc::mbar_try_wait(&bar.raw, (mended - 1) & 1); ++i) {}
      }
    } else if (warp == 16) {
      // ---- products ----------------------------------------------------------------------------------------
      const uint32_t leader = tc::elect_leader();
      const uint32_t id_s = tc::idesc(128, 128, Format<T>::code, tc::kMajorK, tc::kMajorK, p.negate);
      const uint32_t id_o = tc::idesc(128, DP, Format<T>::code, tc::kMajorK, tc::kMajorMN);
      const uint32_t q_base = tc::smem_u32(q_tiles), kv_base = tc::smem_u32(kv_tiles);
      int used = 0, q_used[2] = {0, 0}, p_used[2] = {0, 0};
      bool ok = true;
      auto scores = [&](int t, int s) {
  #pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
          mma_ss(tmem + t * 128, desc_k(q_base + t * C::kTileBytes, C::kSlab, ks), desc_k(kv_base + s * C::kTileBytes, C::kSlab, ks),
                 id_s, ks > 0, leader);
        }
        tc::mma_commit(&bar.s_full[t], leader);
      };
      for (int turn = 0; turn < p.turns && ok; ++turn) {
        const int64_t index = item_of_turn(turn);
        if (index >= p.items || (kAgain && !marked(turn))) continue;
        int head;
        const Item it = item_at(index, &head);
        const int n_t[2] = {key_tiles(it, 0), key_tiles(it, 1)};
        const int n = max(n_t[0], n_t[1]);
        auto full = [&](int x) { return waiter.wait(&bar.kv_full[x % C::kStages], (x / C::kStages) & 1); };
        if (!(ok = full(used))) break;
  #pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (n_t[t] == 0 || !ok) continue;
          if (!(ok = waiter.wait(&bar.q_full[t], q_used[t] & 1))) continue;
          tc::tc_fence_after();
          scores(t, used % C::kStages);
          if (n_t[t] == 1) tc::mma_commit(&bar.q_empty[t], leader);
        }
        if (!ok) break;
        tc::mma_commit(&bar.kv_empty[used % C::kStages], leader);
        for (int j = 0; j < n && ok; ++j) {
          const int xv = used + 2 * j + 1, xk = xv + 1;
          if (!(ok = full(xv))) break;
          if (j + 1 < n && !(ok = full(xk))) break;
          const uint32_t v_tile = kv_base + (xv % C::kStages) * C::kTileBytes;
  #pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (j < n_t[t] && ok) {
              if (!(ok = waiter.wait(&bar.p_ready[t], p_used[t] & 1))) continue;
              ++p_used[t];
              tc::tc_fence_after();
  #pragma unroll
              for (int ks = 0; ks < 8; ++ks) {
                mma_ts(tmem + 256 + t * 128, tmem + t * 128 + (ks >> 2) * 64 + (ks & 3) * 8, desc_mn(v_tile, C::kSlab, ks), id_o, j > 0 || ks > 0, leader);
              }
              if (j + 1 == n_t[t]) tc::mma_commit(&bar.o_full[t], leader);
            }
            if (t == 1) tc::mma_commit(&bar.kv_empty[xv % C::kStages], leader);
            if (j + 1 < n_t[t]) {
              scores(t, xk % C::kStages);
              if (j + 2 == n_t[t]) tc::mma_commit(&bar.q_empty[t], leader);
            }
          }
          if (j + 1 < n) tc::mma_commit(&bar.kv_empty[xk % C::kStages], leader);
        }
        used += 2 * n;
        for (int t = 0; t < 2; ++t) q_used[t] += n_t[t] > 0;
      }
      if (!ok) {  // products under way end before the CTA does
        tc::mma_commit(&bar.drained, leader);
        for (int i = 0; i < 4096 && !tc::mbar_try_wait(&bar.drained, 0); ++i) {}
      }
      __syncwarp();
    }
  } else {
    // ---- weights: two threads a row ------------------------------------------------------------------------
    const int t = warp >> 3, half = (warp >> 2) & 1, row = threadIdx.x & 127;
    const uint32_t lane_base = uint32_t(warp & 3) << 21;   // 32 lanes of TMEM, in bits 16 and up
    const uint32_t s_at = tmem + lane_base + t * 128 + half * 64, o_at = tmem + lane_base + 256 + t * 128 + half * (DP / 2);
    const Pair pair{t, half, row, told[t]};
    const float c = p.scale_log2;
    int seen = 0, outs = 0, redone = 0;
    for (int turn = 0; turn < p.turns; ++turn) {
      const int64_t index = item_of_turn(turn);
      if (index >= p.items || (kAgain && !marked(turn))) continue;
      redone += kAgain;
      int head;
      const Item it = item_at(index, &head);
      const int n = key_tiles(it, t);
      if (n == 0) {
        if (p.lse != nullptr && half == 0) p.lse[head * p.seq.stat_rows + it.stat + (2 * it.tile + t) * 128 + row] = -INFINITY;
        continue;
      }
      float m = 0.f;
      float sum = 0.f;
      bool far = false;
      // The warps of a chain meet in barriers: one that waited in vain goes on as the others do, and what came of all waits is
      // asked behind the last of them.
      for (int j = 0; j < n; ++j) {
        waiter.wait(&bar.s_full[t], seen & 1);
        ++seen;
        tc::tc_fence_after();
        soften_half<T, DP>(pair, s_at, o_at, c, j == 0, m, sum, far, [&](int x, uint32_t (&s)[32]) {
          if (j + 1 == n) {   // the tile on the diagonal; what lies behind the sequence's end lies behind every row
#pragma unroll
            for (int y = 0; y < 32; ++y) {
              if (half * 64 + x * 32 + y > row) s[y] = 0xff800000u;
            }
          }
        });
        tc::tc_fence_before();
        __syncwarp();
        tc::mbar_arrive(&bar.p_ready[t], lane == 0);
      }
      waiter.wait(&bar.o_full[t], outs & 1);
      ++outs;
      tc::tc_fence_after();
      sum += pair.other(sum);
      const bool ok = waiter.nobody_failed();
      const int i = (2 * it.tile + t) * 128 + row, col0 = half * (DP / 2);
      const bool there = i < it.len;
      const float inv = ok ? 1.f / sum : NAN;
      T* to = static_cast<T*>(p.out) + ((it.row + i) * p.heads + head) * p.dim;
      float strange = 0.f;   // NaN if a channel is infinite or NaN
#pragma unroll
      for (int x = 0; x < DP / 2; x += 16) {
        uint32_t raw[16];
        float o[16];
        tc::tmem_ld16(o_at + x, raw);
        tc::tmem_wait_ld();
#pragma unroll
        for (int y = 0; y < 16; ++y) {
          o[y] = __uint_as_float(raw[y]);
          strange = fmaf(o[y], 0.f, strange);
        }
        if (there) store_row16<T>(to + col0 + x, o, inv, p.dim - col0 - x, p.wide);
      }
      if (!kAgain) {
        if (strange != 0.f && there && ok && isfinite(sum)) atomicOr(&marks.again[(turn >> 5) & 31], 1u << (turn & 31));
      } else if (there && ok && col0 < p.dim) {
        const T* v = static_cast<const T*>(p.values) + it.batch * p.strides[0] + (it.row0 + int64_t(it.tile) * kTileRows) * p.strides[1] +
                     head / p.group * p.strides[2] + col0;
        add_strange<T>(v, p.strides[1], marks.strange[redone & 3], t * 128 + row, to + col0, min(p.dim - col0, DP / 2));
      }
      tc::tc_fence_before();
      // rows behind the end: a backward gives them weights exp2(0 - inf) = 0
      if (p.lse != nullptr && half == 0) {
        const Reference ref = reference(m, c);
        const int64_t at = head * p.seq.stat_rows + it.stat + i;
        const float lse = ref.shift != 0.f ? kFarMark - log2f(sum) : -(ref.scaled + log2f(sum));
        p.lse[at] = !there ? -INFINITY : ok ? lse : NAN;
        if (there && lse > kFarFrom) p.lse[p.heads * p.seq.stat_rows + at] = ref.shift;
      }
    }
  }
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1) attention_forward_kernel(const __grid_constant__ FwdParams p) {
  using C = FwdConfig<DP>;
  extern __shared__ __align__(1024) uint8_t smem[];   // swizzled tiles: 1024-byte aligned, there is no static shared memory
  FwdBars* bars = reinterpret_cast<FwdBars*>(smem + (2 + C::kStages) * C::kTileBytes);
  FwdMarks& marks = *reinterpret_cast<FwdMarks*>(bars + 2);
  float(*told)[2][128] = reinterpret_cast<float(*)[2][128]>(smem + (2 + C::kStages) * C::kTileBytes + C::kBarBytes);
  static_assert(2 * sizeof(FwdBars) + sizeof(FwdMarks) <= C::kBarBytes, "");
  const int warp = threadIdx.x >> 5;

  if (threadIdx.x == 0) {
    init_bars<C::kStages>(bars[0]);
    marks.failed = 0;
  }
  if (threadIdx.x < 32) marks.again[threadIdx.x] = 0;
  if (warp == 16) {
    tc::tmem_alloc(&marks.tmem, 512);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = marks.tmem;
  forward_items<T, DP, false>(p, smem, bars[0], marks, told, tmem);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  // (a CTA in which a wait ran out leaves it at that)
  if (__any_sync(0xffffffffu, marks.again[threadIdx.x & 31] != 0) && marks.failed == 0) {
    if (threadIdx.x == 0) init_bars<C::kStages>(bars[1]);
    __syncthreads();
    forward_items<T, DP, true>(p, smem, bars[1], marks, told, tmem);
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
  }
  if (warp == 16) tc::tmem_dealloc(tmem, 512);
}

template <typename T, int DP>
int launch_typed(const FwdParams& p, cudaStream_t stream) {
  using C = FwdConfig<DP>;
  const void* kernel = reinterpret_cast<const void*>(&attention_forward_kernel<T, DP>);
  const cudaError_t err = ensure_dynamic_smem(kernel, C::kBytes);
  if (err != cudaSuccess) { record_cuda_error(err); return GDN2_ERR_LAUNCH; }
  int sms = 0;
  const int status = multiprocessors(&sms);
  if (status != GDN2_OK) return status;
  FwdParams q = p;
  const int64_t grid = p.items < sms ? p.items : sms;
  q.turns = int((p.items + grid - 1) / grid);
  attention_forward_kernel<T, DP><<<unsigned(grid), kThreads, C::kBytes, stream>>>(q);
  return check_launch();
}

}  // namespace

int launch_attention_forward(const void* q, const void* k, const void* v, void* out, float* lse, const int64_t* strides,
                             const int64_t* bounds, int64_t n_seq, int64_t time, int heads, int kv_heads, int dim,
                             int dtype, float scale, cudaStream_t stream) {
  FwdParams p;
  const int64_t batch = bounds != nullptr ? 1 : n_seq;
  if (!encode_heads_map(&p.q, q, strides, batch, time, heads, dim, dtype, 128) ||
      !encode_heads_map(&p.k, k, strides + 3, batch, time, kv_heads, dim, dtype, 128) ||
      !encode_heads_map(&p.v, v, strides + 6, batch, time, kv_heads, dim, dtype, 128)) {
    return GDN2_ERR_LAUNCH;
  }
  p.values = v;
  for (int i = 0; i < 3; ++i) p.strides[i] = strides[6 + i];
  p.out = out; p.lse = lse;
  p.heads = heads; p.kv_heads = kv_heads; p.group = heads / kv_heads; p.dim = dim;
  p.negate = scale < 0.f;
  p.polls = wait_polls();
  p.wide = wide_rows(out, dim);
  p.scale_log2 = positive_scale(scale);
  return for_groups(bounds, n_seq, time, &p.seq, [&]() -> int {
    p.items = int64_t(p.seq.tiles) * heads;
    if (dtype == GDN2_BF16) return dim <= 64 ? launch_typed<__nv_bfloat16, 64>(p, stream) : launch_typed<__nv_bfloat16, 128>(p, stream);
    return dim <= 64 ? launch_typed<__half, 64>(p, stream) : launch_typed<__half, 128>(p, stream);
  });
}

}  // namespace attn
}  // namespace gdn2
