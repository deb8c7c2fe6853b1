// Eviction from a paged cache: of every sequence and key head the tokens of the largest accumulated weights are copied, in their
// order, to other pages, and with them their weights.
//
// select_kernel   a CTA has a sequence and head.  Which tokens are kept follows from the keep-th largest weight and, among those
//                 that are equal to it, from their order.  Weights become whole numbers of the same order, and the one looked
//                 for is closed in by counting them in 2048 bins over the range that is left, which a pass narrows 2048 times; the
//                 first range reaches from the smallest weight to the largest, so that the bins are spread where the weights
//                 are.  When up to 512 are left they are compared with one another.  The weights lie in shared memory where there is
//                 room (49152), and are read once more for every pass otherwise.
// gather_kernel   copies keys, values and weights, 8 tokens of a head a warp.  Bound by HBM.
//
// 8 sequences of up to 16384 tokens, 8 heads of 128 channels, 4096 kept: 14.5 and 46 us, the latter 5.9 TB/s both ways in pieces
// of 256 bytes that lie where the weights have them.  What select_kernel takes is latency: 64 CTAs, of 24 thousand clocks 7
// for the weights' arrival, 4 for the first pass, 5 for what is left of it, 5 for the tokens' numbers.  (Two or four CTAs of a cluster
// for a sequence and head 41 us, where their barriers and one another's bins took more than they saved.)

#include <algorithm>

#include "common.cuh"

namespace gdn2 {

namespace {

constexpr int kSelectThreads = 1024;
constexpr int kBins = 2048, kBinBits = 11;
constexpr int kAll = 0x7fffffff;
constexpr int kCached = 49152;        // weights that stay in shared memory
constexpr int kAtOnce = 4;            // pieces of keys, and of values, that a lane has under way
constexpr int kGatherThreads = 256, kGatherWarp = 8, kGatherTokens = kGatherThreads / 32 * kGatherWarp;
constexpr int kListed = 512;          // candidates near the border that are compared with one another

struct EvictParams {
  uint8_t *k_pages, *v_pages;
  float* weight_pages;                // [pages][kv head][page]
  const int *table, *lengths, *new_table;
  int* new_lengths;
  int* kept;                          // [batch][kv head]: tokens that are copied, or -1
  int* tokens;                        // [batch][kv head][keep]: which
  int64_t table_stride, new_stride, pages;
  int batch, kv_heads, page, columns, keep, sinks, recent;
  int cached;                         // weights that stay in shared memory
  int per_row, chunks;                // packs of a row of keys; CTAs of a sequence and head
  Divisor by_page, by_row;
};

// Whole numbers in the order of the weights: NaN above all, -0 and 0 the same
__device__ __forceinline__ uint32_t order_of(float w) {
  if (isnan(w)) return ~0u;
  const uint32_t x = __float_as_uint(w + 0.f);   // -0 + 0 is 0
  return (x >> 31) != 0 ? ~x : x | 0x80000000u;
}

// Of two numbers a warp, by all threads: the sums over the warps before its own, and over all
struct WarpSums { int a[32], b[32]; };   // those behind the last warp are 0
__device__ __forceinline__ int2 sums_before(WarpSums& shared, int a, int b, int2* all) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();
  if (lane == 0) { shared.a[warp] = a; shared.b[warp] = b; }
  __syncthreads();
  int x = shared.a[lane], y = shared.b[lane];
  const int own_x = x, own_y = y;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, x, d), v = __shfl_up_sync(0xffffffffu, y, d);
    if (lane >= d) { x += u; y += v; }
  }
  *all = make_int2(__shfl_sync(0xffffffffu, x, 31), __shfl_sync(0xffffffffu, y, 31));
  return make_int2(__shfl_sync(0xffffffffu, x - own_x, warp), __shfl_sync(0xffffffffu, y - own_y, warp));
}

__global__ void __launch_bounds__(kSelectThreads, 1) select_kernel(const __grid_constant__ EvictParams p) {
  extern __shared__ uint32_t cache[];   // of the candidates
  __shared__ int bins[kBins];
  __shared__ uint32_t list[kListed];
  __shared__ WarpSums sums;
  __shared__ uint32_t range[2];
  __shared__ int found[3], listed;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = int(blockIdx.x) / p.kv_heads, head = int(blockIdx.x) - b * p.kv_heads;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int length = p.lengths[b];
  const bool sized = length >= 0 && length <= p.columns * p.page;
  const int* table = p.table + b * p.table_stride;
  bool good = sized;
  for (int c = tid; sized && c < (length + p.page - 1) / p.page; c += kSelectThreads) good = good && table[c] >= 0 && table[c] < p.pages;
  auto tell = [&](bool good) {
    if (tid == 0) {
      p.kept[blockIdx.x] = good ? min(length, p.keep) : -1;
      if (head == 0) p.new_lengths[b] = good ? min(length, p.keep) : -1;
    }
  };
  if (length <= p.keep || !sized) {   // all tokens stay, or none can be read
    tell(__syncthreads_and(good));
    return;
  }

  // Candidates are neither sinks nor recent ones
  const int first = p.sinks, last = length - p.recent;
  const bool cached = last - first <= p.cached;
  const float* weights = p.weight_pages + int64_t(head) * p.page;
  const int64_t page_size = int64_t(p.kv_heads) * p.page;
  auto read = [&](int t) {   // (without a branch, so that several are under way)
    int place;
    const int page = table[p.by_page.split(t, &place)];
    const bool there = page >= 0 && page < p.pages;
    const float w = weights[there ? page * page_size + place : 0];
    return order_of(w);
  };
  auto key = [&](int t) { return cached ? cache[t - first] : read(t); };
  int wanted = p.keep - p.sinks - p.recent;   // candidates that stay
  uint32_t lo = ~0u, hi = 0;
  for (int t0 = first + tid; t0 < last; t0 += 8 * kSelectThreads) {
    uint32_t x[8];
#pragma unroll
    for (int y = 0; y < 8; ++y) x[y] = read(min(t0 + y * kSelectThreads, last - 1));
#pragma unroll
    for (int y = 0; y < 8; ++y) {
      const int t = t0 + y * kSelectThreads;
      lo = min(lo, x[y]);
      hi = max(hi, x[y]);
      if (cached && t < last) cache[t - first] = x[y];
    }
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  for (int x = tid; x < kBins; x += kSelectThreads) bins[x] = 0;
  if (tid < 32) {
    sums.a[tid] = sums.b[tid] = 0;
    if (tid < 2) range[tid] = tid == 0 ? ~0u : 0u;
  }
  good = __syncthreads_and(good);
  tell(good);
  if (!good) return;
  if (lane == 0) {
    atomicMin(&range[0], lo);
    atomicMax(&range[1], hi);
  }
  __syncthreads();
  lo = range[0];
  hi = range[1];

  // The wanted-th largest is in lo .. hi; what is above hi stays
  int equal = 0;             // of those that are lo in the end, so many stay
  if (wanted == 0) lo = ~0u;
  // 2^32 numbers, then at most 2^21, 2^10 and one, or few weights in what is left of the range
  for (int pass = 0; wanted > 0 && pass < 4; ++pass) {
    if (lo == hi) {
      equal = wanted;
      break;
    }
    const int shift = max(0, 32 - __clz(hi - lo) - kBinBits);
    int smallest = 0;        // many weights are often the smallest one: counted without the others' atomics
    for (int t = first + tid; t < last; t += kSelectThreads) {
      const uint32_t x = key(t);
      if (x == lo) ++smallest;
      else if (x > lo && x <= hi) atomicAdd(&bins[(x - lo) >> shift], 1);
    }
    smallest = __reduce_add_sync(0xffffffffu, smallest);
    if (lane == 0 && smallest > 0) atomicAdd(&bins[0], smallest);
    if (tid == 0) listed = 0;
    __syncthreads();
    // a thread's bins, from the top down
    int own[kBins / kSelectThreads], mine = 0;
#pragma unroll
    for (int x = 0; x < kBins / kSelectThreads; ++x) {
      const int bin = kBins - 1 - (tid * (kBins / kSelectThreads) + x);
      mine += own[x] = bins[bin];
      bins[bin] = 0;         // for the next pass
    }
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
      for (int x = 0; x < kBins / kSelectThreads; ++x) {
        if (above < wanted && above + own[x] >= wanted) {
          found[0] = kBins - 1 - (tid * (kBins / kSelectThreads) + x);
          found[1] = wanted - above;
          found[2] = own[x];
        }
        above += own[x];
      }
    }
    __syncthreads();
    wanted = found[1];
    const int count = found[2];
    lo += uint32_t(found[0]) << shift;
    hi = lo + min(hi - lo, (1u << shift) - 1u);   // (lo + 2^shift may pass 2^32)
    if (wanted == count) {   // all of the bin stay
      equal = kAll;
      break;
    }
    if (count <= kListed) {  // few are left: the one that wanted - 1 others are above is compared with all of them
      for (int t = first + tid; t < last; t += kSelectThreads) {
        const uint32_t x = key(t);
        if (x >= lo && x <= hi) {
          const int at = atomicAdd(&listed, 1);
          if (at < kListed) list[at] = x;   // (as many as were counted, unless somebody writes weights meanwhile)
        }
      }
      __syncthreads();
      if (tid < count) {
        const uint32_t x = list[tid];
        int larger = 0, as_large = 0;
#pragma unroll 4
        for (int i = 0; i < count; ++i) {
          larger += list[i] > x;
          as_large += list[i] == x;
        }
        if (larger < wanted && larger + as_large >= wanted) {   // one, or some that are equal
          range[0] = x;
          found[1] = wanted - larger;
          found[2] = as_large;
        }
      }
      __syncthreads();
      lo = range[0];
      equal = found[1] == found[2] ? kAll : found[1];
      break;
    }
    __syncthreads();         // found has been read by all
  }

  // The sinks come first and the recent ones last; a warp has a range of the candidates between them: how many stay for their
  // weight, how many are equal to the border.  (No order_of is 0, so that the bound below all of them is no problem.)
  const uint32_t bound = equal == kAll ? lo - 1 : lo;
  const bool border = equal != kAll && equal > 0;
  const int each = (last - first + kSelectThreads - 1) / kSelectThreads * 32, begin = min(last, first + warp * each), end = min(last, begin + each);
  const uint32_t below = (1u << lane) - 1u;
  int* to = p.tokens + int64_t(blockIdx.x) * p.keep;
  for (int j = tid; j < p.sinks; j += kSelectThreads) to[j] = j;
  for (int j = tid; j < p.recent; j += kSelectThreads) to[p.keep - p.recent + j] = last + j;
  int2 all;
  if (cached && !border) {
    // what stays moves together where it is, token numbers in place of weights, and goes out when all warps have counted
    uint32_t* own = cache + (begin - first);
    int staying = 0;
    for (int t = begin + lane; t - lane < end; t += 32) {
      const bool stay = t < end && own[t - begin] > bound;
      const uint32_t stays = __ballot_sync(0xffffffffu, stay);
      __syncwarp();
      if (stay) own[staying + __popc(stays & below)] = uint32_t(t);
      staying += __popc(stays);
    }
    const int at = p.sinks + sums_before(sums, staying, 0, &all).x;
    for (int i = lane; i < staying && at + i < p.keep; i += 32) to[at + i] = int(own[i]);
    return;
  }
  int staying = 0, evens = 0;
  for (int t = begin + lane; t - lane < end; t += 32) {
    const uint32_t x = t < end ? key(t) : 0;
    staying += __popc(__ballot_sync(0xffffffffu, x > bound));
    if (border) evens += __popc(__ballot_sync(0xffffffffu, x == lo));
  }
  const int2 before = sums_before(sums, staying, evens, &all);
  int at = p.sinks + before.x + (border ? min(before.y, equal) : 0);   // where the warp's next one goes
  int level = before.y;
  for (int t = begin + lane; t - lane < end; t += 32) {
    const uint32_t x = t < end ? key(t) : 0;
    uint32_t stays = __ballot_sync(0xffffffffu, x > bound);
    if (border) {
      const uint32_t even = __ballot_sync(0xffffffffu, x == lo);
      stays |= __ballot_sync(0xffffffffu, x == lo && level + __popc(even & below) < equal);
      level += __popc(even);
    }
    const int place = at + __popc(stays & below);
    if (((stays >> lane) & 1) != 0 && place < p.keep) to[place] = t;
    at += __popc(stays);
  }
}

// A warp has 8 tokens of a head, wherever they are: nothing but its own loads stands between it and the next one's.  (8 sequences as
// above: pieces of keys and of values at the same places of both 46 us, one after the other 50; 16 tokens a warp 47, more warps with
// fewer registers 53 to 55.)
template <typename P>
__global__ void __launch_bounds__(kGatherThreads, 4) gather_kernel(const __grid_constant__ EvictParams p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // the heads of 64 places are written one beside the other
  const int head = int(blockIdx.x) % p.kv_heads, chunk = int(blockIdx.x) / p.kv_heads % p.chunks, b = int(blockIdx.x) / p.kv_heads / p.chunks;
  const int unit = b * p.kv_heads + head;
  const int length = p.lengths[b];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int kept = p.kept[unit], j0 = chunk * kGatherTokens + warp * kGatherWarp, count = min(kept - j0, kGatherWarp);
  if (count <= 0) return;
  int64_t from = 0, to = -1;   // rows of keys of token j0 + lane, -1 for none
  if (lane < count) {
    // (a token of the sequence and a page of the cache, unless somebody writes lengths, weights or tables meanwhile)
    const int j = j0 + lane, t = min(max(length <= p.keep ? j : p.tokens[int64_t(unit) * p.keep + j], 0), p.columns * p.page - 1);
    int t_place, j_place;
    const int page = p.new_table[b * p.new_stride + p.by_page.split(j, &j_place)];
    const int64_t source = p.table[b * p.table_stride + p.by_page.split(t, &t_place)];
    if (page >= 0 && page < p.pages && source >= 0 && source < p.pages) {
      p.weight_pages[(int64_t(page) * p.kv_heads + head) * p.page + j_place] = p.weight_pages[(source * p.kv_heads + head) * p.page + t_place];
      from = (source * p.page + t_place) * p.kv_heads + head;
      to = (int64_t(page) * p.page + j_place) * p.kv_heads + head;
    }
  }
  from *= p.per_row;
  to *= p.per_row;   // (of -1 something below 0)
  const int packs = kGatherWarp * p.per_row;
  for (int x0 = 0; x0 < packs; x0 += kAtOnce * 32) {
    P key[kAtOnce], value[kAtOnce];
    int64_t place[kAtOnce];
#pragma unroll
    for (int y = 0; y < kAtOnce; ++y) {
      const int x = x0 + y * 32 + lane, row = min(p.by_row.quotient(x), kGatherWarp - 1), pack = x - row * p.per_row;
      const int64_t source = __shfl_sync(0xffffffffu, from, row) + pack;
      place[y] = __shfl_sync(0xffffffffu, to, row);
      if (x >= packs) place[y] = -1;
      if (place[y] < 0) continue;
      place[y] += pack;
      key[y] = reinterpret_cast<const P*>(p.k_pages)[source];
      value[y] = reinterpret_cast<const P*>(p.v_pages)[source];
    }
#pragma unroll
    for (int y = 0; y < kAtOnce; ++y) {
      if (place[y] < 0) continue;
      reinterpret_cast<P*>(p.k_pages)[place[y]] = key[y];
      reinterpret_cast<P*>(p.v_pages)[place[y]] = value[y];
    }
  }
}

template <typename P>
int launch_gather(EvictParams& p, int row_bytes, cudaStream_t stream) {
  p.per_row = row_bytes / int(sizeof(P));
  p.by_row = divisor(p.per_row);
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
  p.by_page = divisor(page);
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
