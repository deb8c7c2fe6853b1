// Eviction from a paged cache: of every sequence and key head the tokens of the largest accumulated weights are copied, in their
// order, to other pages, and with them their weights.
//
// select_kernel   a CTA has a sequence and head.  Which tokens are kept follows from the keep-th largest weight and, among those
//                 that are equal to it, from their order.  Weights become whole numbers of the same order, and the one looked
//                 for is closed in by counting them in 2048 bins over the range that is left: every pass over the weights, which
//                 lie in shared memory where there is room, narrows the range 2048 times, and the first range reaches from the
//                 smallest weight to the largest, so that the bins are spread where the weights are.  Then a pass writes down
//                 the numbers of the tokens that stay.
// gather_kernel   copies keys, values and weights, 64 tokens of a head a CTA.  Bound by HBM.
// TODO-FIGURES

#include <algorithm>

#include "common.cuh"

namespace gdn2 {

namespace {

constexpr int kSelectThreads = 512, kSelectWarps = kSelectThreads / 32;
constexpr int kBins = 2048, kBinBits = 11;
constexpr int kCached = 49152;        // weights that stay in shared memory
constexpr int kGatherThreads = 256, kGatherTokens = 64;

struct EvictParams {
  uint8_t *k_pages, *v_pages;
  float* weight_pages;                // [pages][kv head][page]
  const int *table, *lengths, *new_table;
  int* new_lengths;
  int* kept;                          // [batch][kv head]: tokens that are copied, or -1
  int* tokens;                        // [batch][kv head][keep]: which
  int64_t table_stride, new_stride, pages;
  int batch, kv_heads, page, columns, keep, sinks, recent, cached;
  int per_row, chunks;                // packs of a row of keys; CTAs of a sequence and head
};

// Whole numbers in the order of the weights: NaN above all, -0 and 0 the same
__device__ __forceinline__ uint32_t order_of(float w) {
  if (isnan(w)) return ~0u;
  const uint32_t x = __float_as_uint(w + 0.f);   // -0 + 0 is 0
  return (x >> 31) != 0 ? ~x : x | 0x80000000u;
}

// Sums over the CTA of two numbers a thread and over the warps before its own, by all threads
struct WarpSums { int a[kSelectWarps], b[kSelectWarps]; };
__device__ __forceinline__ int2 sums_before(WarpSums& shared, int a, int b, int2* all) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();
  if (lane == 0) { shared.a[warp] = a; shared.b[warp] = b; }
  __syncthreads();
  int2 before = make_int2(0, 0), sum = make_int2(0, 0);
#pragma unroll
  for (int w = 0; w < kSelectWarps; ++w) {
    if (w == warp) before = sum;
    sum.x += shared.a[w];
    sum.y += shared.b[w];
  }
  *all = sum;
  return before;
}

__global__ void __launch_bounds__(kSelectThreads, 1) select_kernel(const __grid_constant__ EvictParams p) {
  extern __shared__ uint32_t cache[];
  __shared__ int bins[kBins];
  __shared__ WarpSums sums;
  __shared__ uint32_t range[2];
  __shared__ int found[3];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = int(blockIdx.x) / p.kv_heads, head = int(blockIdx.x) - b * p.kv_heads;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int length = p.lengths[b];
  const bool sized = length >= 0 && length <= p.columns * p.page;
  const int* table = p.table + b * p.table_stride;
  bool good = sized;
  for (int c = tid; sized && c < (length + p.page - 1) / p.page; c += kSelectThreads) good = good && table[c] >= 0 && table[c] < p.pages;
  good = __syncthreads_and(good);
  const int kept = good ? min(length, p.keep) : -1;
  if (tid == 0) {
    p.kept[blockIdx.x] = kept;
    if (head == 0) p.new_lengths[b] = kept;
  }
  if (kept < p.keep || length == p.keep) return;   // all tokens stay, or none can be read

  // candidates: neither sinks nor recent ones
  const int first = p.sinks, last = length - p.recent;
  const bool cached = last - first <= p.cached;
  auto read = [&](int t) { return order_of(p.weight_pages[(int64_t(table[t / p.page]) * p.kv_heads + head) * p.page + t % p.page]); };
  auto key = [&](int t) { return cached ? cache[t - first] : read(t); };
  int wanted = p.keep - p.sinks - p.recent;   // candidates that stay
  uint32_t lo = ~0u, hi = 0;
  for (int t0 = first + tid; t0 < last; t0 += 8 * kSelectThreads) {
    uint32_t x[8];
#pragma unroll
    for (int y = 0; y < 8; ++y) {
      const int t = t0 + y * kSelectThreads;
      x[y] = t < last ? read(t) : 0;
    }
#pragma unroll
    for (int y = 0; y < 8; ++y) {
      const int t = t0 + y * kSelectThreads;
      if (t >= last) break;
      lo = min(lo, x[y]);
      hi = max(hi, x[y]);
      if (cached) cache[t - first] = x[y];
    }
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if (tid < 2) range[tid] = tid == 0 ? ~0u : 0u;
  __syncthreads();
  if (lane == 0) {
    atomicMin(&range[0], lo);
    atomicMax(&range[1], hi);
  }
  __syncthreads();
  lo = range[0];
  hi = range[1];

  // The wanted-th largest is in lo .. hi; what is above hi stays
  int equal = 0;             // of those that are lo in the end, so many stay
  if (wanted == 0) {
    lo = ~0u;
  } else {
    // 2^32 numbers, then at most 2^21, 2^10 and one
    for (int pass = 0; pass < 4; ++pass) {
      if (lo == hi) {
        equal = wanted;
        break;
      }
      const int shift = max(0, 32 - __clz(hi - lo) - kBinBits);
      for (int x = tid; x < kBins; x += kSelectThreads) bins[x] = 0;
      __syncthreads();
      int smallest = 0;      // many weights are often the smallest one: counted without the others' atomics
      for (int t = first + tid; t < last; t += kSelectThreads) {
        const uint32_t x = key(t);
        if (x == lo) ++smallest;
        else if (x > lo && x <= hi) atomicAdd(&bins[(x - lo) >> shift], 1);
      }
      smallest = __reduce_add_sync(0xffffffffu, smallest);
      if (lane == 0 && smallest > 0) atomicAdd(&bins[0], smallest);
      __syncthreads();
      // a thread's bins, from the top down
      constexpr int kEach = kBins / kSelectThreads;
      int mine = 0;
#pragma unroll
      for (int x = 0; x < kEach; ++x) mine += bins[kBins - 1 - (tid * kEach + x)];
      int up_to = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, up_to, d);
        if (lane >= d) up_to += y;
      }
      int2 all;
      int above = sums_before(sums, __shfl_sync(0xffffffffu, up_to, 31), 0, &all).x + up_to - mine;
      if (above < wanted && above + mine >= wanted) {   // one thread of all
#pragma unroll
        for (int x = 0; x < kEach; ++x) {
          const int bin = kBins - 1 - (tid * kEach + x);
          if (above + bins[bin] >= wanted) {
            found[0] = bin;
            found[1] = wanted - above;
            found[2] = bins[bin];
            break;
          }
          above += bins[bin];
        }
      }
      __syncthreads();
      wanted = found[1];
      lo += uint32_t(found[0]) << shift;
      hi = lo + min(hi - lo, (1u << shift) - 1u);   // (lo + 2^shift may pass 2^32)
      if (wanted == found[2]) {   // all of the bin stay
        equal = 0x7fffffff;
        break;
      }
      __syncthreads();
    }
  }

  // A warp has a range of the tokens: how many stay for their weight or their place, how many are equal to the border
  const int each = (length + kSelectThreads - 1) / kSelectThreads * 32, begin = min(length, warp * each), end = min(length, begin + each);
  auto look = [&](int t, bool* stays, bool* even) {
    const bool protected_ = t < first || t >= last, candidate = t < end && !protected_;
    const uint32_t x = candidate ? key(t) : 0;
    *stays = t < end && (protected_ || (equal == 0x7fffffff ? x >= lo : x > lo));
    *even = candidate && equal != 0x7fffffff && x == lo;
  };
  int staying = 0, evens = 0;
  for (int t = begin + lane; t - lane < end; t += 32) {
    bool stays, even;
    look(t, &stays, &even);
    staying += __popc(__ballot_sync(0xffffffffu, stays));
    evens += __popc(__ballot_sync(0xffffffffu, even));
  }
  int2 all;
  int2 before = sums_before(sums, staying, evens, &all);
  int* to = p.tokens + int64_t(blockIdx.x) * p.keep;
  const uint32_t below = (1u << lane) - 1u;
  for (int t = begin + lane; t - lane < end; t += 32) {
    bool stays, even;
    look(t, &stays, &even);
    const uint32_t s = __ballot_sync(0xffffffffu, stays), e = __ballot_sync(0xffffffffu, even);
    const int rank = before.y + __popc(e & below);
    const int at = before.x + __popc(s & below) + min(rank, equal);
    if ((stays || (even && rank < equal)) && at < p.keep) to[at] = t;
    before.x += __popc(s);
    before.y += __popc(e);
  }
}

template <typename P>
__global__ void __launch_bounds__(kGatherThreads) gather_kernel(const __grid_constant__ EvictParams p) {
  __shared__ int64_t from[kGatherTokens], to[kGatherTokens];   // rows of keys, -1 for none
  const int unit = int(blockIdx.x) / p.chunks, chunk = int(blockIdx.x) - unit * p.chunks;
  const int b = unit / p.kv_heads, head = unit - b * p.kv_heads;
  const int length = p.lengths[b];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int kept = p.kept[unit], j0 = chunk * kGatherTokens, count = min(kept - j0, kGatherTokens);
  if (count <= 0) return;
  if (threadIdx.x < kGatherTokens) {
    const int j = j0 + int(threadIdx.x);
    int64_t source = -1, place = -1;
    if (j < kept) {
      const int t = length <= p.keep ? j : p.tokens[int64_t(unit) * p.keep + j];
      const int page = p.new_table[b * p.new_stride + j / p.page];
      if (page >= 0 && page < p.pages) {
        source = p.table[b * p.table_stride + t / p.page];
        place = page;
        p.weight_pages[(place * p.kv_heads + head) * p.page + j % p.page] = p.weight_pages[(source * p.kv_heads + head) * p.page + t % p.page];
        source = (source * p.page + t % p.page) * p.kv_heads + head;
        place = (place * p.page + j % p.page) * p.kv_heads + head;
      }
    }
    from[threadIdx.x] = source;
    to[threadIdx.x] = place;
  }
  __syncthreads();
  constexpr int kAtOnce = 8;
  const int packs = count * p.per_row;   // of keys, then of values
  for (int x0 = threadIdx.x; x0 < 2 * packs; x0 += kAtOnce * kGatherThreads) {
    P data[kAtOnce];
    int64_t place[kAtOnce];
#pragma unroll
    for (int y = 0; y < kAtOnce; ++y) {
      const int x = x0 + y * kGatherThreads;
      place[y] = -1;
      if (x >= 2 * packs) continue;
      const int z = x < packs ? x : x - packs, row = z / p.per_row, pack = z - row * p.per_row;
      if (to[row] < 0) continue;
      place[y] = to[row] * p.per_row + pack;
      data[y] = reinterpret_cast<const P*>(x < packs ? p.k_pages : p.v_pages)[from[row] * p.per_row + pack];
    }
#pragma unroll
    for (int y = 0; y < kAtOnce; ++y) {
      if (place[y] >= 0) reinterpret_cast<P*>(x0 + y * kGatherThreads < packs ? p.k_pages : p.v_pages)[place[y]] = data[y];
    }
  }
}

template <typename P>
int launch_gather(EvictParams& p, int row_bytes, cudaStream_t stream) {
  p.per_row = row_bytes / int(sizeof(P));
  return launch_beside(&gather_kernel<P>, unsigned(p.batch * p.kv_heads * p.chunks), kGatherThreads, 0, stream, p);
}

}  // namespace

int64_t evict_workspace_bytes(int64_t batch, int64_t kv_heads, int64_t keep) { return (batch * kv_heads * (keep + 1) * 4 + 15) / 16 * 16; }

int launch_evict(void* k_pages, void* v_pages, float* weight_pages, const int* table, const int* lengths, const int* new_table,
                 int* new_lengths, void* workspace, int64_t table_stride, int64_t new_stride, int batch, int64_t pages, int page,
                 int kv_heads, int dim, int columns, int keep, int sinks, int recent, int element, cudaStream_t stream) {
  EvictParams p{};
  p.k_pages = static_cast<uint8_t*>(k_pages); p.v_pages = static_cast<uint8_t*>(v_pages);
  p.weight_pages = weight_pages;
  p.table = table; p.lengths = lengths; p.new_table = new_table; p.new_lengths = new_lengths;
  p.kept = static_cast<int*>(workspace);
  p.tokens = p.kept + int64_t(batch) * kv_heads;
  p.table_stride = table_stride; p.new_stride = new_stride; p.pages = pages;
  p.batch = batch; p.kv_heads = kv_heads; p.page = page; p.columns = columns;
  p.keep = keep; p.sinks = sinks; p.recent = recent;
  p.chunks = (keep + kGatherTokens - 1) / kGatherTokens;
  const int64_t units = int64_t(batch) * kv_heads;
  if (units > int64_t(0x7fffffff) / p.chunks) return GDN2_ERR_TOO_LARGE;
  p.cached = int(std::min<int64_t>(int64_t(columns) * page, kCached));
  const cudaError_t err = ensure_dynamic_smem(reinterpret_cast<const void*>(&select_kernel), kCached * 4);
  if (err != cudaSuccess) { record_cuda_error(err); return GDN2_ERR_LAUNCH; }
  select_kernel<<<unsigned(units), kSelectThreads, p.cached * 4, stream>>>(p);
  const int status = check_launch();
  if (status != GDN2_OK) return status;
  const int row_bytes = dim * element;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages) | uintptr_t(row_bytes);
  if (bits % 16 == 0) return launch_gather<uint4>(p, row_bytes, stream);
  if (bits % 4 == 0) return launch_gather<uint32_t>(p, row_bytes, stream);
  return launch_gather<uint16_t>(p, row_bytes, stream);
}

}  // namespace gdn2
