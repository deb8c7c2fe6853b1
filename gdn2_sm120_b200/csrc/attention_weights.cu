// What weight every token of a prompt gets from the queries that see it, summed over the heads of a group.  With the
// forward's statistics lse_i = m_i + log l_i:
//
//   w_j = sum over heads and i >= j of exp(scale q_i . k_j - lse_i)
//
// A work item is 128 keys of a key head; the queries that see them go by, 128 at a time, for every head of the group.  S^T =
// K Q^T comes out of the tensor cores into one of four sets of TMEM columns by turns, so that a set's four warps, a key a thread,
// sum a row of weights while the others' products run; nothing but a sum a key leaves the kernel.  A step's sum is formed for
// itself before it joins the others, so that the roundings of 32-bit sums count by steps and not by queries.
//
// 4 prompts of 4096 tokens, 16 heads of 128 channels, 4 a group: 157 to 163 us, 1320 clocks a tile of 128 x 128, of which its
// exponentials, less a quarter on the FMA units, take the special-function unit 768 (70 % of its time by a capture) and its
// product the tensor cores 512.  None of them on the FMA units 174 us, half of them 174, three eighths 161.

#include "attention_common.cuh"

namespace gdn2 {
namespace attn {

namespace {

constexpr int kSets = 4;         // of TMEM columns, and of warps that sum
constexpr int kThreads = (4 * kSets + 2) * 32;   // the last two: products, copies
constexpr int kRing = 16;        // steps whose statistics are there: more than the steps under way

template <int DP>
struct WeightConfig {
  static constexpr int kTileBytes = 128 * DP * 2, kSlab = 128 * 128;
  static constexpr int kStages = DP == 128 ? 4 : 8;   // tiles of queries
  static constexpr int kBytes = (2 + kStages) * kTileBytes + kRing * 128 * 4 + 2 * kSets * 128 * 4 + 512;
};

struct WeightParams {
  CUtensorMap q, k;
  const float *lse, *shifts;   // as in the backward
  float* weights;              // [rows][kv heads]
  float* partials;             // [part][rows][kv heads]
  int64_t rows;
  int heads, kv_heads, group, parts, turns;
  int64_t items;
  float scale_log2;            // positive
  uint32_t negate;
  uint32_t polls;              // of a wait
  Sequences seq;
};

struct WeightBars {
  uint64_t k_full[2], k_empty[2], q_full[8], q_empty[8], s_full[kSets], s_empty[kSets], drained;
  uint32_t tmem;
  int failed;
};
static_assert(sizeof(WeightBars) <= 512, "");

struct WeightItem {
  Item at;
  int head, tile;               // of keys; 128-row tile in the sequence
  int per_head, begin, steps;   // tiles of queries that see it, for a head; this part's first step, its steps
  int part;
};

__device__ __forceinline__ int part_begin(int steps, int part, int parts) { return int(int64_t(steps) * part / parts); }

// Tiles of the longest rows come first
__device__ __forceinline__ bool weight_item(const WeightParams& p, int turn, WeightItem* w) {
  const int64_t index = item_of_turn(turn);
  if (index >= p.items) return false;
  const int heads = p.kv_heads * p.parts, unit = int(index / heads), in_tile = int(index - int64_t(unit) * heads);
  w->head = in_tile / p.parts;
  w->part = in_tile - w->head * p.parts;
  w->at = find_item(p.seq, unit >> 1, false);
  w->tile = 2 * w->at.tile + (unit & 1);
  if (w->tile * 128 >= w->at.len) return false;
  w->per_head = (w->at.len + 127) / 128 - w->tile;
  w->begin = part_begin(w->per_head * p.group, w->part, p.parts);
  w->steps = part_begin(w->per_head * p.group, w->part + 1, p.parts) - w->begin;
  return w->steps > 0;
}

// The sum of a row's weights in a step in which a query's reference is far away (as in the backward's key kernel); columns
// first .. last - 1 count
__device__ __noinline__ float far_sum(uint32_t s_at, const float* st, const float* shifts, float c, int first, int last) {
  float sum = 0.f;
#pragma unroll 1
  for (int x = 0; x < 128; x += 32) {
    uint32_t s[32];
    tc::tmem_ld32(s_at + x, s);
    tc::tmem_wait_ld();
#pragma unroll
    for (int y = 0; y < 32; ++y) {
      if (x + y < first || x + y >= last) continue;
      const float l = st[x + y], v = __uint_as_float(s[y]);
      sum += exp2_approx(l > kFarFrom ? min_nan(fmaf(v - shifts[x + y], c, l - kFarMark), 0.f) : fmaf(v, c, l));
    }
  }
  return sum;
}

// The sum of a row's weights; kPartial: columns first .. last - 1 count
template <bool kPartial>
__device__ __forceinline__ float row_sum(uint32_t s_at, const float* st, float2 by, int first, int last) {
  float2 sum[4] = {{0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}};
  uint32_t s[2][32];
  tc::tmem_ld32(s_at, s[0]);
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    tc::tmem_wait_ld();
    if (x < 3) tc::tmem_ld32(s_at + (x + 1) * 32, s[(x + 1) & 1]);
    const uint32_t(&v)[32] = s[x & 1];
#pragma unroll
    for (int y = 0; y < 32; y += 4) {
      const float4 l = *reinterpret_cast<const float4*>(st + x * 32 + y);
      const float2 a = fma2(make_float2(__uint_as_float(v[y]), __uint_as_float(v[y + 1])), by, make_float2(l.x, l.y));
      const float2 b = fma2(make_float2(__uint_as_float(v[y + 2]), __uint_as_float(v[y + 3])), by, make_float2(l.z, l.w));
      float2 e = exp2_2(a), f = (y & 4) != 0 ? exp2_fma(b) : exp2_2(b);
      if (kPartial) {
        const int col = x * 32 + y;
        if (col < first || col >= last) e.x = 0.f;
        if (col + 1 < first || col + 1 >= last) e.y = 0.f;
        if (col + 2 < first || col + 2 >= last) f.x = 0.f;
        if (col + 3 < first || col + 3 >= last) f.y = 0.f;
      }
      sum[(y >> 1) & 2] = add2(sum[(y >> 1) & 2], e);
      sum[((y >> 1) & 2) + 1] = add2(sum[((y >> 1) & 2) + 1], f);
    }
  }
  const float2 all = add2(add2(sum[0], sum[1]), add2(sum[2], sum[3]));
  return all.x + all.y;
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1) attention_weights_kernel(const __grid_constant__ WeightParams p) {
  using C = WeightConfig<DP>;
  extern __shared__ __align__(1024) uint8_t smem[];   // swizzled tiles: 1024-byte aligned, there is no static shared memory
  uint8_t* q_tiles = smem + 2 * C::kTileBytes;
  float* stats = reinterpret_cast<float*>(q_tiles + C::kStages * C::kTileBytes);   // [step by turns][128]
  float* told = stats + kRing * 128;                                              // [item by turns][set][128]
  WeightBars& bar = *reinterpret_cast<WeightBars*>(told + 2 * kSets * 128);
  static_assert(kRing >= C::kStages + 2 * kSets, "");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int x = 0; x < 2; ++x) {
      tc::mbar_init(&bar.k_full[x], 1);
      tc::mbar_init(&bar.k_empty[x], 1);
    }
    for (int x = 0; x < C::kStages; ++x) {
      tc::mbar_init(&bar.q_full[x], 1);
      tc::mbar_init(&bar.q_empty[x], 1);
    }
    for (int x = 0; x < kSets; ++x) {
      tc::mbar_init(&bar.s_full[x], 1);
      tc::mbar_init(&bar.s_empty[x], 4);
    }
    tc::mbar_init(&bar.drained, 1);
    bar.failed = 0;
    tc::fence_mbar_init();
  }
  if (warp == 4 * kSets) {
    tc::tmem_alloc(&bar.tmem, 512);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = bar.tmem;
  const Waiter waiter{&bar.failed, p.polls};
  asm volatile("griddepcontrol.wait;" ::: "memory");   // the forward's statistics
  let_others_begin();

  if (warp == 4 * kSets + 1) {
    // ---- copies --------------------------------------------------------------------------------------------
    tc::fence_async_all();   // they were written by threads, and are read by bulk copies
    const uint32_t leader = tc::elect_leader();
    int filled = 0, items = 0;
    bool ok = true;
    for (int turn = 0; turn < p.turns && ok; ++turn) {
      WeightItem w;
      if (!weight_item(p, turn, &w)) continue;
      const int place = items & 1;
      if (items >= 2 && !(ok = waiter.wait(&bar.k_empty[place], (items / 2 - 1) & 1))) break;
      tc::mbar_arrive_expect_tx(&bar.k_full[place], C::kTileBytes, leader);
#pragma unroll
      for (int slab = 0; slab < DP / 64; ++slab) {
        tc::tma_load_4d(smem + place * C::kTileBytes + slab * C::kSlab, &p.k, slab * 64, w.head, w.at.row0 + w.tile * 128, w.at.batch,
                        &bar.k_full[place], leader);
      }
      ++items;
      for (int i = 0; i < w.steps; ++i) {
        const int s = filled % C::kStages, step = w.begin + i;
        if (filled >= C::kStages && !(ok = waiter.wait(&bar.q_empty[s], (filled / C::kStages - 1) & 1))) break;
        const int g = step / w.per_head, at = (w.tile + step - g * w.per_head) * 128, head = w.head * p.group + g;
        tc::mbar_arrive_expect_tx(&bar.q_full[s], C::kTileBytes + 128 * 4, leader);
#pragma unroll
        for (int slab = 0; slab < DP / 64; ++slab) {
          tc::tma_load_4d(q_tiles + s * C::kTileBytes + slab * C::kSlab, &p.q, slab * 64, head, w.at.row0 + at, w.at.batch, &bar.q_full[s],
                          leader);
        }
        tc::bulk_g2s(stats + filled % kRing * 128, p.lse + head * p.seq.stat_rows + w.at.stat + at, 128 * 4, &bar.q_full[s], leader);
        ++filled;
      }
    }
    if (!ok) {  // copies under way end before the CTA does
      for (int back = 1; back <= C::kStages && back <= filled; ++back) {
        const int x = filled - back;
        for (int i = 0; i < 4096 && !tc::mbar_try_wait(&bar.q_full[x % C::kStages], (x / C::kStages) & 1); ++i) {}
      }
      for (int back = 1; back <= 2 && back <= items; ++back) {
        const int x = items - back;
        for (int i = 0; i < 4096 && !tc::mbar_try_wait(&bar.k_full[x & 1], (x >> 1) & 1); ++i) {}
      }
    }
  } else if (warp == 4 * kSets) {
    // ---- products ------------------------------------------------------------------------------------------
    const uint32_t leader = tc::elect_leader();
    const uint32_t id = tc::idesc(128, 128, Format<T>::code, tc::kMajorK, tc::kMajorK, p.negate);
    const uint32_t k_base = tc::smem_u32(smem), q_base = tc::smem_u32(q_tiles);
    int used = 0, items = 0;
    bool ok = true;
    for (int turn = 0; turn < p.turns && ok; ++turn) {
      WeightItem w;
      if (!weight_item(p, turn, &w)) continue;
      const uint32_t k_tile = k_base + (items & 1) * C::kTileBytes;
      if (!(ok = waiter.wait(&bar.k_full[items & 1], (items >> 1) & 1))) break;
      for (int i = 0; i < w.steps; ++i, ++used) {
        const int s = used % C::kStages, set = used % kSets;
        if (!(ok = waiter.wait(&bar.q_full[s], (used / C::kStages) & 1))) break;
        if (used >= kSets && !(ok = waiter.wait(&bar.s_empty[set], (used / kSets - 1) & 1))) break;
        tc::tc_fence_after();
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
          mma_ss(tmem + set * 128, desc_k(k_tile, C::kSlab, ks), desc_k(q_base + s * C::kTileBytes, C::kSlab, ks), id, ks > 0, leader);
        }
        tc::mma_commit(&bar.s_full[set], leader);
        tc::mma_commit(&bar.q_empty[s], leader);
      }
      if (!ok) break;
      tc::mma_commit(&bar.k_empty[items & 1], leader);
      ++items;
    }
    if (!ok) {  // products under way end before the CTA does
      tc::mma_commit(&bar.drained, leader);
      for (int i = 0; i < 4096 && !tc::mbar_try_wait(&bar.drained, 0); ++i) {}
    }
    __syncwarp();
  } else {
    // ---- sums: a key a thread, every fourth step ---------------------------------------------------------------
    const int set = warp >> 2, row = threadIdx.x & 127;
    const uint32_t s_at = tmem + (uint32_t(warp & 3) << 21) + set * 128;   // 32 lanes of TMEM, in bits 16 and up
    const float2 by = twice(p.scale_log2);
    int used = 0, mine = 0, items = 0;
    for (int turn = 0; turn < p.turns; ++turn) {
      WeightItem w;
      if (!weight_item(p, turn, &w)) continue;
      float total = 0.f;
      // (the warps meet in a barrier: one that waited in vain goes on as the others do, and what came of all waits is asked
      // behind it)
      for (int i = (set - used) & (kSets - 1); i < w.steps; i += kSets) {
        const float* st = stats + (used + i) % kRing * 128;
        const int step = w.begin + i, g = step / w.per_head, at = (w.tile + step - g * w.per_head) * 128;
        // queries from the key itself on, up to the sequence's end
        const int first = at == w.tile * 128 ? row : 0, last = min(w.at.len - at, 128);
        const bool partial = at == w.tile * 128 || last < 128;
        waiter.wait(&bar.s_full[set], mine & 1);
        ++mine;
        tc::tc_fence_after();
        const bool far = __any_sync(0xffffffffu, st[lane] > kFarFrom || st[32 + lane] > kFarFrom || st[64 + lane] > kFarFrom ||
                                                     st[96 + lane] > kFarFrom);
        if (__builtin_expect(far, 0)) {
          total += far_sum(s_at, st, p.shifts + (w.head * p.group + g) * p.seq.stat_rows + w.at.stat + at, p.scale_log2, first, last);
        } else {
          total += partial ? row_sum<true>(s_at, st, by, first, last) : row_sum<false>(s_at, st, by, 0, 128);
        }
        tc::tc_fence_before();
        __syncwarp();
        tc::mbar_arrive(&bar.s_empty[set], lane == 0);
      }
      used += w.steps;
      float* sums = told + (items & 1) * kSets * 128;
      ++items;
      sums[set * 128 + row] = total;
      asm volatile("bar.sync 1, %0;" ::"n"(4 * kSets * 32) : "memory");
      if (set == 0) {
        const bool ok = waiter.nobody_failed();
        const int j = w.tile * 128 + row;
        const float weight = (sums[row] + sums[128 + row]) + (sums[256 + row] + sums[384 + row]);
        float* to = (p.parts == 1 ? p.weights : p.partials + w.part * p.rows * p.kv_heads) + (w.at.row + j) * p.kv_heads + w.head;
        if (j < w.at.len) *to = ok ? weight : NAN;
      }
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 4 * kSets) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

// Sums of an item's parts, in their order: a thread a key and head
__global__ void __launch_bounds__(256) attention_weights_parts_kernel(const __grid_constant__ WeightParams p) {
  const int per_tile = (128 * p.kv_heads + 255) / 256, unit = int(blockIdx.x) / per_tile;
  const int x = (int(blockIdx.x) - unit * per_tile) * int(blockDim.x) + int(threadIdx.x);   // (row of the tile, kv head)
  const Item it = find_item(p.seq, unit >> 1, false);
  const int tile = 2 * it.tile + (unit & 1), i = tile * 128 + x / p.kv_heads;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (i >= it.len || x >= 128 * p.kv_heads) return;
  const int64_t at = (it.row + tile * 128) * p.kv_heads + x;
  const int steps = ((it.len + 127) / 128 - tile) * p.group;
  float sum = 0.f;
  for (int part = 0; part < p.parts; ++part) {
    if (part_begin(steps, part, p.parts) < part_begin(steps, part + 1, p.parts)) sum += p.partials[part * p.rows * p.kv_heads + at];
  }
  p.weights[at] = sum;
}

template <typename T, int DP>
int launch_typed(const WeightParams& base, cudaStream_t stream) {
  using C = WeightConfig<DP>;
  const cudaError_t err = ensure_dynamic_smem(reinterpret_cast<const void*>(&attention_weights_kernel<T, DP>), C::kBytes);
  if (err != cudaSuccess) { record_cuda_error(err); return GDN2_ERR_LAUNCH; }
  int sms = 0;
  int status = multiprocessors(&sms);
  if (status != GDN2_OK) return status;
  WeightParams p = base;
  const int64_t tiles = int64_t(p.seq.tiles) * 2;
  p.items = tiles * p.kv_heads * p.parts;
  const int64_t grid = p.items < sms ? p.items : sms;
  p.turns = int((p.items + grid - 1) / grid);
  // each is there when the one before it ends: 20 short packed prompts 37 us and not 39.5
  status = launch_beside(&attention_weights_kernel<T, DP>, unsigned(grid), kThreads, C::kBytes, stream, p);
  if (status != GDN2_OK || p.parts == 1) return status;
  const int64_t ctas = tiles * ((128 * p.kv_heads + 255) / 256);
  if (ctas > int64_t(0x7fffffff)) return GDN2_ERR_TOO_LARGE;
  return launch_beside(&attention_weights_parts_kernel, unsigned(ctas), 256, 0, stream, p);
}

// Parts of an item, as of the backward's items of keys: as many as bring the longest one down to an SM's share
int weight_parts(const int64_t* bounds, int64_t n_seq, int64_t time, int heads, int kv_heads, int sms) {
  int64_t longest = 0, all = 0;
  for (int64_t i = 0; i < (bounds != nullptr ? n_seq : 1); ++i) {
    const int64_t tiles = ((bounds != nullptr ? bounds[i + 1] - bounds[i] : time) + 127) / 128;
    longest = std::max(longest, tiles * (heads / kv_heads));
    all += tiles * (tiles + 1) / 2 * heads;
  }
  if (bounds == nullptr) all *= n_seq;
  return longest < 16 ? 1 : int(std::max<int64_t>(1, longest / std::max<int64_t>(1, all / sms)));
}

}  // namespace

int64_t attention_weights_bytes(const int64_t* bounds, int64_t n_seq, int64_t time, int heads, int kv_heads) {
  int sms = 0;
  const int status = multiprocessors(&sms);
  if (status != GDN2_OK) return status;
  const int parts = weight_parts(bounds, n_seq, time, heads, kv_heads, sms);
  return parts == 1 ? 0 : int64_t(parts) * (bounds != nullptr ? time : n_seq * time) * kv_heads * 4;
}

int launch_attention_weights(const void* q, const void* k, const float* lse, float* weights, void* scratch, const int64_t* strides,
                             const int64_t* bounds, int64_t n_seq, int64_t time, int heads, int kv_heads, int dim, int dtype,
                             float scale, cudaStream_t stream) {
  WeightParams p;
  const int64_t batch = bounds != nullptr ? 1 : n_seq;
  if (!encode_heads_map(&p.q, q, strides, batch, time, heads, dim, dtype, 128) ||
      !encode_heads_map(&p.k, k, strides + 3, batch, time, kv_heads, dim, dtype, 128)) {
    return GDN2_ERR_LAUNCH;
  }
  int sms = 0;
  const int status = multiprocessors(&sms);
  if (status != GDN2_OK) return status;
  p.lse = lse;
  p.shifts = lse + stat_rows(bounds, n_seq, time) * heads;
  p.weights = weights;
  p.partials = static_cast<float*>(scratch);
  p.rows = batch * time;
  p.heads = heads; p.kv_heads = kv_heads; p.group = heads / kv_heads;
  p.parts = weight_parts(bounds, n_seq, time, heads, kv_heads, sms);
  if (p.parts > 1 && scratch == nullptr) return GDN2_ERR_NULL_POINTER;
  p.negate = scale < 0.f;
  p.polls = wait_polls();
  p.scale_log2 = positive_scale(scale);
  return for_groups(bounds, n_seq, time, false, &p.seq, [&](bool) -> int {
    if (dtype == GDN2_BF16) return dim <= 64 ? launch_typed<__nv_bfloat16, 64>(p, stream) : launch_typed<__nv_bfloat16, 128>(p, stream);
    return dim <= 64 ? launch_typed<__half, 64>(p, stream) : launch_typed<__half, 128>(p, stream);
  });
}

}  // namespace attn
}  // namespace gdn2
