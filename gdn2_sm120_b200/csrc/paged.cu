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
//                 and 0 where nothing is seen.  One pass over the cache with a running maximum and sum; the heads of a
//                 group are rows of one product with their shared key head, so the cache is read once for every 64 rows
//                 (drafted tokens x heads of a group).  Bound by HBM up to there: 64 rows take 64 flop a byte.
//                 All (sequence, key head, 64-token tile) are one list that the CTAs share evenly, so neither
//                 unequal lengths nor few sequences leave SMs idle, and the host need not know the lengths.  A CTA
//                 whose part begins or ends inside a sequence leaves (O, m, l) in the workspace; tree_join_kernel joins
//                 these in the order of the tiles: the same inputs give the same bits.
//                 The products are mma.sync m16n8k16: tiles of 16 rows fit one to a few drafted tokens, where an
//                 instruction of the tcgen05 kind has 64 rows at least and its sums in another memory.

#include <algorithm>

#include "common.cuh"

namespace gdn2 {

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
constexpr int kTile = 64;      // tokens of a tile
constexpr int kStages = 3;     // tiles in flight: 96 KiB of keys and values of 128 channels, two CTAs to an SM
constexpr int kThreads = 128;
constexpr float kLog2e = 1.4426950408889634f;

struct TreeParams {
  const void *q, *k, *v;
  const void *k_pages, *v_pages;
  void* out;
  const int *table, *lengths;
  const uint8_t* mask;                       // [batch or 1][drafted][drafted], or null: j <= i
  float* partials;                           // [CTA][2][rows][DP + 2]
  int64_t q_stride[3], k_stride[3], v_stride[3];  // batch, token, head, in elements
  int64_t table_stride, mask_stride, pages;
  int batch, drafted, heads, kv_heads, group, dim, page, columns;
  int rows, row_blocks, ctas;
  float scale_log2;
};

// One (sequence, key head, block of rows) after the other, tile by tile
struct Cursor {
  int b, head, block;   // block of rows
  int tile, tiles, context_tiles, length;
  bool bad;             // the sequence's length is none that its page table can hold
};

__device__ __forceinline__ void read_length(const TreeParams& p, Cursor& c) {
  if (c.b < p.batch) {
    const int n = p.lengths[c.b], most = p.columns * p.page;
    c.bad = n < 0 || n > most;
    c.length = c.bad ? 0 : n;
    c.context_tiles = (c.length + kTile - 1) / kTile;
    c.tiles = c.context_tiles + (p.drafted + kTile - 1) / kTile;
  }
}

__device__ __forceinline__ void advance(const TreeParams& p, Cursor& c) {
  if (++c.tile < c.tiles) return;
  c.tile = 0;
  if (++c.block < p.row_blocks) return;
  c.block = 0;
  if (++c.head < p.kv_heads) return;
  c.head = 0;
  ++c.b;
  read_length(p, c);
}

// tiles of sequence b, for all its key heads and blocks of rows
__device__ __forceinline__ int64_t tiles_of(const TreeParams& p, int b) {
  Cursor c{b, 0, 0, 0, 0, 0, 0, false};
  read_length(p, c);
  return int64_t(c.tiles) * p.kv_heads * p.row_blocks;
}

// CTAs that have a part of `total` tiles: each of them a tile at least
__device__ __forceinline__ int64_t sharing(const TreeParams& p, int64_t total) { return total < p.ctas ? total : p.ctas; }

// Sum over all threads of the CTA (every one of them gets it) and of those before this one
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
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w == warp) earlier = total;
    total += shared[w];
  }
  *before = earlier + sum - x;
  return total;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

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
template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  const typename Pair<T>::type v = Pair<T>::make(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// a 16-bit float that is infinite or NaN: its exponent bits are all ones
template <typename T> struct Exponent;
template <> struct Exponent<__nv_bfloat16> { static constexpr uint32_t bits = 0x7f80; };
template <> struct Exponent<__half> { static constexpr uint32_t bits = 0x7c00; };
template <typename T>
__device__ __forceinline__ bool any_not_finite(uint32_t pair) {
  constexpr uint32_t e = Exponent<T>::bits;
  return (pair & e) == e || ((pair >> 16) & e) == e;
}

// Shared memory of a CTA: kStages of (K, V) tiles, rows of DP channels whose 16-byte pieces are permuted by the row;
// where the rows' addresses are; what the warps that share rows exchange.
template <int DP, int WM>
struct TreeSmem {
  static constexpr int kRows = 16 * WM, kWN = 4 / WM;
  uint8_t kv[kStages][2][kTile * DP * 2];
  const uint8_t* at[kStages + 1][kTile][2];  // addresses of a token's key and value; null: zeros
  int64_t scan[kThreads / 32], found[2];
  int bad[kStages + 1][kTile / 32];          // by locating warp
  float m[kWN][kRows], l[kWN][kRows];
  float o[kWN > 1 ? kRows : 1][DP];
};

template <int DP>
__device__ __forceinline__ uint32_t piece(int row, int c) {  // byte offset of 16-byte piece c of a row
  return uint32_t(row * DP * 2 + ((c ^ (row & 7)) << 4));
}

// 16 * WM rows a CTA; the 4 / WM warps of the same rows share a tile's tokens.
template <typename T, int DP, int WM>
__global__ void __launch_bounds__(kThreads, 2) tree_kernel(const TreeParams p) {
  using Smem = TreeSmem<DP, WM>;
  constexpr int kRows = Smem::kRows, kWN = Smem::kWN;
  constexpr int kOwn = kTile / kWN;       // tokens of a tile that a warp works on
  constexpr int kKSteps = DP / 16, kNB = kOwn / 8, kDB = DP / 8;
  extern __shared__ __align__(128) uint8_t raw[];
  Smem& sm = *reinterpret_cast<Smem*>(raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int wm = warp % WM, wn = warp / WM;
  const int quad = lane >> 2, in_quad = lane & 3;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // this CTA's part of all tiles
  int64_t total = 0, before;
  for (int b0 = 0; b0 < p.batch; b0 += kThreads) {
    const int b = b0 + tid;
    total += cta_scan(b < p.batch ? tiles_of(p, b) : 0, &before, sm.scan);
  }
  const int64_t ctas = sharing(p, total);
  if (blockIdx.x >= ctas) return;
  const int64_t begin = total * blockIdx.x / ctas, end = total * (blockIdx.x + 1) / ctas;
  Cursor first{0, 0, 0, 0, 0, 0, 0, false};
  {
    int64_t base = 0;
    for (int b0 = 0; b0 < p.batch; b0 += kThreads) {
      const int b = b0 + tid;
      const int64_t own = b < p.batch ? tiles_of(p, b) : 0;
      const int64_t sum = cta_scan(own, &before, sm.scan);
      const int64_t from = base + before;
      if (own > 0 && begin >= from && begin < from + own) {  // one thread of all
        sm.found[0] = b;
        sm.found[1] = begin - from;
      }
      base += sum;
      if (begin < base) break;
    }
    __syncthreads();
    first.b = int(sm.found[0]);
    const int64_t rest = sm.found[1];
    read_length(p, first);
    const int64_t unit = rest / first.tiles;
    first.tile = int(rest - unit * first.tiles);
    first.head = int(unit / p.row_blocks);
    first.block = int(unit - int64_t(first.head) * p.row_blocks);
  }
  const int n_tiles = int(end - begin);

  // where the rows of a tile are: a thread a token
  auto locate = [&](const Cursor& c, int slot) {
    if (tid < kTile) {
      const uint8_t *k = nullptr, *v = nullptr;
      bool bad = c.bad;
      if (c.tile < c.context_tiles) {
        const int t = c.tile * kTile + tid;
        if (t < c.length) {
          const int column = t / p.page;
          const int64_t page = p.table[c.b * p.table_stride + column];
          if (page >= 0 && page < p.pages) {
            const int64_t row = (page * p.page + (t - column * p.page)) * p.kv_heads + c.head;
            k = static_cast<const uint8_t*>(p.k_pages) + row * p.dim * 2;
            v = static_cast<const uint8_t*>(p.v_pages) + row * p.dim * 2;
          } else {
            bad = true;
          }
        }
      } else {
        const int j = (c.tile - c.context_tiles) * kTile + tid;
        if (j < p.drafted) {
          k = static_cast<const uint8_t*>(p.k) + 2 * (c.b * p.k_stride[0] + j * p.k_stride[1] + c.head * p.k_stride[2]);
          v = static_cast<const uint8_t*>(p.v) + 2 * (c.b * p.v_stride[0] + j * p.v_stride[1] + c.head * p.v_stride[2]);
        }
      }
      sm.at[slot][tid][0] = k;
      sm.at[slot][tid][1] = v;
      const bool any = __any_sync(0xffffffffu, bad);
      if (lane == 0) sm.bad[slot][warp] = any;
    }
  };
  constexpr int kPieces = DP / 8;              // 16-byte pieces of a row
  const int my_piece = tid % kPieces, my_row = tid / kPieces;
  const bool piece_there = my_piece * 8 < p.dim;
  auto fetch = [&](int stage, int slot) {
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(sm.kv[stage][which]));
#pragma unroll
      for (int r = 0; r < kTile; r += kThreads / kPieces) {
        const uint8_t* row = sm.at[slot][r + my_row][which];
        const bool there = piece_there && row != nullptr;
        cp_async16(to + piece<DP>(r + my_row, my_piece), there ? row + my_piece * 16 : static_cast<const uint8_t*>(p.k), there);
      }
    }
  };

  Cursor ahead = first;   // the tile whose rows are looked up next
  int located = 0;
  for (; located < kStages && located < n_tiles; ++located) {
    locate(ahead, located);
    advance(p, ahead);
  }
  __syncthreads();
  for (int i = 0; i < kStages - 1; ++i) {
    if (i < n_tiles) fetch(i, i);
    cp_async_commit();
  }

  Cursor c = first;
  uint32_t qf[kKSteps][4];
  float o[kDB][4];
  float m[2], l[2];
  int seg_row = 0;        // first of this warp's rows
  bool starts_here = false, fresh_segment = true;

  for (int i = 0; i < n_tiles; ++i) {
    const int stage = i % kStages, slot = i % (kStages + 1);
    if (fresh_segment) {
      fresh_segment = false;
      starts_here = c.tile == 0;
      seg_row = c.block * kRows + 16 * wm;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int r = seg_row + quad + 8 * half;
        const bool there = r < p.rows;
        const int n = there ? r / p.group : 0, g = there ? r - n * p.group : 0;
        const T* row = static_cast<const T*>(p.q) + c.b * p.q_stride[0] + n * p.q_stride[1] +
                       int64_t(c.head * p.group + g) * p.q_stride[2];
#pragma unroll
        for (int s = 0; s < kKSteps; ++s) {
#pragma unroll
          for (int kh = 0; kh < 2; ++kh) {
            const int col = s * 16 + kh * 8 + in_quad * 2;
            qf[s][kh * 2 + half] = there && col < p.dim ? *reinterpret_cast<const uint32_t*>(row + col) : 0u;
          }
        }
        m[half] = -INFINITY;
        l[half] = 0.f;
      }
#pragma unroll
      for (int d = 0; d < kDB; ++d) { o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f; }
    }
    cp_async_wait<kStages - 2>();
    __syncthreads();   // the tile is there, and nobody reads the one before it any more
    if (i + kStages - 1 < n_tiles) fetch((i + kStages - 1) % kStages, (i + kStages - 1) % (kStages + 1));
    cp_async_commit();
    const bool bad = (sm.bad[slot][0] | sm.bad[slot][1]) != 0;
    const bool drafted_tile = c.tile >= c.context_tiles;
    const int first_token = (drafted_tile ? c.tile - c.context_tiles : c.tile) * kTile + wn * kOwn;
    const uint32_t k_tile = static_cast<uint32_t>(__cvta_generic_to_shared(sm.kv[stage][0]));
    const uint32_t v_tile = static_cast<uint32_t>(__cvta_generic_to_shared(sm.kv[stage][1]));

    // S = Q K^T
    float s[kNB][4];
#pragma unroll
    for (int n = 0; n < kNB; ++n) { s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f; }
#pragma unroll
    for (int ks = 0; ks < kKSteps; ++ks) {
#pragma unroll
      for (int n = 0; n < kNB; n += 2) {
        uint32_t kf[4];  // tokens n*8.. and (n+1)*8.., channels ks*16 + 0..7 and 8..15
        ldmatrix4(kf, k_tile + piece<DP>(wn * kOwn + n * 8 + (lane & 7) + ((lane >> 4) << 3), ks * 2 + ((lane >> 3) & 1)));
        mma16816<T>(s[n], qf[ks], kf[0], kf[1]);
        mma16816<T>(s[n + 1], qf[ks], kf[2], kf[3]);
      }
    }
    // what a row sees of the tile
    auto sees = [&](int row, int token) {
      if (!drafted_tile) return token < c.length;
      if (token >= p.drafted || row >= p.rows) return false;
      const int n = row / p.group;
      if (p.mask == nullptr) return token <= n;
      return p.mask[c.b * p.mask_stride + int64_t(n) * p.drafted + token] != 0;
    };
    const bool whole = !drafted_tile && (c.tile + 1) * kTile <= c.length;
#pragma unroll
    for (int n = 0; n < kNB; ++n) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] *= p.scale_log2;
        if (!whole && !sees(seg_row + quad + 8 * (e >> 1), first_token + n * 8 + in_quad * 2 + (e & 1))) s[n][e] = -INFINITY;
      }
    }
    // running maximum and sum of the two rows of this thread's quad
    uint32_t pf[kNB][2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float top = -INFINITY;
#pragma unroll
      for (int n = 0; n < kNB; ++n) top = fmaxf(top, fmaxf(s[n][2 * half], s[n][2 * half + 1]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float now = fmaxf(m[half], top);
      const float base = now == -INFINITY ? 0.f : now;   // nothing seen yet: every weight is exp(-inf) = 0
      const float keep = exp2_approx(m[half] - base);
      m[half] = now;
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < kNB; ++n) {
        const float a = exp2_approx(s[n][2 * half] - base), b = exp2_approx(s[n][2 * half + 1] - base);
        sum += a + b;
        pf[n][half] = pack_pair<T>(a, b);   // weights at most 1, rounded to the values' type for the product
      }
      l[half] = l[half] * keep + sum;       // (of this thread's columns; the quad's are added at the end)
#pragma unroll
      for (int d = 0; d < kDB; ++d) { o[d][2 * half] *= keep; o[d][2 * half + 1] *= keep; }
    }
    if (bad) l[0] = l[1] = NAN;             // a page or a length that cannot be: the sequence's output is NaN
    // An infinite or NaN value of a drafted token must reach the rows that see it and no others, but in the product below
    // it would meet every row (0 * NaN): it is added to those rows here and leaves the tile.
    if (drafted_tile) {
      bool strange = false;
      for (int x = tid; x < kTile * DP / 8; x += kThreads) {
        const uint4 w = *reinterpret_cast<const uint4*>(sm.kv[stage][1] + x * 16);
        strange = strange || any_not_finite<T>(w.x) || any_not_finite<T>(w.y) || any_not_finite<T>(w.z) || any_not_finite<T>(w.w);
      }
      if (__syncthreads_or(strange)) {
        for (int j = 0; j < kOwn; ++j) {
          const int row_in_tile = wn * kOwn + j;
          const bool lo = sees(seg_row + quad, first_token + j), hi = sees(seg_row + quad + 8, first_token + j);
#pragma unroll
          for (int d = 0; d < kDB; ++d) {
            const uint32_t pair = *reinterpret_cast<const uint32_t*>(sm.kv[stage][1] + piece<DP>(row_in_tile, d) + in_quad * 4);
            const float2 x = unpack2<T>(pair);
            if (!isfinite(x.x)) { if (lo) o[d][0] += x.x; if (hi) o[d][2] += x.x; }
            if (!isfinite(x.y)) { if (lo) o[d][1] += x.y; if (hi) o[d][3] += x.y; }
          }
        }
        __syncthreads();
        for (int x = tid; x < kTile * DP; x += kThreads) {
          uint16_t* e = reinterpret_cast<uint16_t*>(sm.kv[stage][1]) + x;
          if ((*e & Exponent<T>::bits) == Exponent<T>::bits) *e = 0;
        }
        __syncthreads();
      }
    }
    // O += P V
#pragma unroll
    for (int ks = 0; ks < kOwn / 16; ++ks) {
      const uint32_t pa[4] = {pf[2 * ks][0], pf[2 * ks][1], pf[2 * ks + 1][0], pf[2 * ks + 1][1]};
#pragma unroll
      for (int d = 0; d < kDB; d += 2) {
        uint32_t vf[4];  // channels d*8.. (tokens 0..7, 8..15), channels (d+1)*8.. (the same)
        ldmatrix4_trans(vf, v_tile + piece<DP>(wn * kOwn + ks * 16 + (lane & 15), d + (lane >> 4)));
        mma16816<T>(o[d], pa, vf[0], vf[1]);
        mma16816<T>(o[d + 1], pa, vf[2], vf[3]);
      }
    }
    const bool last_tile = c.tile + 1 == c.tiles, last = i + 1 == n_tiles;
    if (last_tile || last) {
      // the end of this CTA's part of the segment
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
        l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
      }
      if constexpr (kWN > 1) {   // warps that share the rows
        if (in_quad == 0) {
          sm.m[wn][16 * wm + quad] = m[0];
          sm.m[wn][16 * wm + quad + 8] = m[1];
        }
        __syncthreads();
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int r = 16 * wm + quad + 8 * half;
          float top = -INFINITY;
#pragma unroll
          for (int w = 0; w < kWN; ++w) top = fmaxf(top, sm.m[w][r]);
          const float f = top == -INFINITY ? 0.f : exp2_approx(m[half] - top);
          m[half] = top;
          l[half] *= f;
#pragma unroll
          for (int d = 0; d < kDB; ++d) { o[d][2 * half] *= f; o[d][2 * half + 1] *= f; }
          if (in_quad == 0) sm.l[wn][r] = l[half];
        }
        for (int w = 1; w < kWN; ++w) {
          if (wn == w) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
#pragma unroll
              for (int d = 0; d < kDB; ++d) {
                float2* at = reinterpret_cast<float2*>(&sm.o[16 * wm + quad + 8 * half][d * 8 + in_quad * 2]);
                float2 x = make_float2(o[d][2 * half], o[d][2 * half + 1]);
                if (w > 1) { x.x += at->x; x.y += at->y; }
                *at = x;
              }
            }
          }
          __syncthreads();
        }
        if (wn == 0) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int r = 16 * wm + quad + 8 * half;
            l[half] = 0.f;
#pragma unroll
            for (int w = 0; w < kWN; ++w) l[half] += sm.l[w][r];
#pragma unroll
            for (int d = 0; d < kDB; ++d) {
              const float2 x = *reinterpret_cast<const float2*>(&sm.o[r][d * 8 + in_quad * 2]);
              o[d][2 * half] += x.x;
              o[d][2 * half + 1] += x.y;
            }
          }
        }
      }
      if (wn == 0) {
        const bool whole_segment = starts_here && last_tile;
        float* part = p.partials + (int64_t(blockIdx.x) * 2 + (starts_here ? 1 : 0)) * kRows * (DP + 2);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int r = seg_row + quad + 8 * half;
          if (whole_segment) {
            if (r < p.rows) {
              const int n = r / p.group, g = r - n * p.group;
              // nothing seen: the sum is 0 and so is the output
              const float inv = l[half] == 0.f ? 0.f : 1.f / l[half];
              T* to = static_cast<T*>(p.out) + (int64_t(c.b) * p.drafted + n) * p.heads * p.dim +
                      int64_t(c.head * p.group + g) * p.dim;
#pragma unroll
              for (int d = 0; d < kDB; ++d) {
                const int col = d * 8 + in_quad * 2;
                if (col < p.dim) *reinterpret_cast<uint32_t*>(to + col) = pack_pair<T>(o[d][2 * half] * inv, o[d][2 * half + 1] * inv);
              }
            }
          } else {
            const int lr = 16 * wm + quad + 8 * half;
            float* row = part + int64_t(lr) * DP;
#pragma unroll
            for (int d = 0; d < kDB; ++d) *reinterpret_cast<float2*>(row + d * 8 + in_quad * 2) = make_float2(o[d][2 * half], o[d][2 * half + 1]);
            if (in_quad == 0) *reinterpret_cast<float2*>(part + kRows * DP + 2 * lr) = make_float2(m[half], l[half]);
          }
        }
      }
      fresh_segment = true;
    }
    advance(p, c);
    if (located < n_tiles) {
      // the slot of the tile before this one: every thread has read it before this iteration's barrier
      locate(ahead, located % (kStages + 1));
      advance(p, ahead);
      ++located;
    }
  }
}

// Joins what several CTAs have of one (sequence, key head, block of rows): a CTA each.
template <typename T, int DP>
__global__ void __launch_bounds__(kThreads) tree_join_kernel(const TreeParams p, int rows_of_block) {
  __shared__ int64_t scan[kThreads / 32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int unit = blockIdx.x;
  const int block = unit % p.row_blocks, head = unit / p.row_blocks % p.kv_heads, b = unit / p.row_blocks / p.kv_heads;
  int64_t total = 0, from = 0, before;
  for (int b0 = 0; b0 < p.batch; b0 += kThreads) {
    const int x = b0 + int(threadIdx.x);
    const int64_t own = x < p.batch ? tiles_of(p, x) : 0;
    total += cta_scan(own, &before, scan);
    int64_t sum_before = cta_scan(x < b ? own : 0, &before, scan);
    from += sum_before;
  }
  Cursor c{b, 0, 0, 0, 0, 0, 0, false};
  read_length(p, c);
  const int64_t t0 = from + (int64_t(head) * p.row_blocks + block) * c.tiles, t1 = t0 + c.tiles;
  const int64_t ctas = sharing(p, total), c0 = ((t0 + 1) * ctas - 1) / total, c1 = (t1 * ctas - 1) / total;
  if (c0 == c1) return;   // one CTA had it all
  const int row0 = block * rows_of_block;
  const int64_t size = int64_t(rows_of_block) * (DP + 2);
  constexpr int kQuads = DP / 4;
  for (int x = threadIdx.x; x < rows_of_block * kQuads; x += kThreads) {
    const int lr = x / kQuads, d = (x - lr * kQuads) * 4, r = row0 + lr;
    if (r >= p.rows || d >= p.dim) continue;
    float top = -INFINITY;
    for (int64_t i = c0; i <= c1; ++i) {
      const float* part = p.partials + (i * 2 + (i == c0 ? 1 : 0)) * size;
      top = fmaxf(top, part[rows_of_block * DP + 2 * lr]);
    }
    float sum = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int64_t i = c0; i <= c1; ++i) {
      const float* part = p.partials + (i * 2 + (i == c0 ? 1 : 0)) * size;
      const float2 ml = *reinterpret_cast<const float2*>(part + rows_of_block * DP + 2 * lr);
      const float f = ml.x == -INFINITY ? 0.f : exp2_approx(ml.x - top);
      sum += isnan(ml.y) ? ml.y : ml.y * f;
      const float4 v = *reinterpret_cast<const float4*>(part + int64_t(lr) * DP + d);
      acc[0] += v.x * f; acc[1] += v.y * f; acc[2] += v.z * f; acc[3] += v.w * f;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int n = r / p.group, g = r - n * p.group;
    T* to = static_cast<T*>(p.out) + (int64_t(b) * p.drafted + n) * p.heads * p.dim + int64_t(head * p.group + g) * p.dim + d;
    *reinterpret_cast<uint2*>(to) = make_uint2(pack_pair<T>(acc[0] * inv, acc[1] * inv), pack_pair<T>(acc[2] * inv, acc[3] * inv));
  }
}

// rows of a block: as few as hold all rows, 64 at most
int block_rows(int64_t rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }

template <typename T, int DP, int WM>
int launch_tree_typed(const TreeParams& p, cudaStream_t stream) {
  constexpr int kBytes = int(sizeof(TreeSmem<DP, WM>));
  const void* kernel = reinterpret_cast<const void*>(&tree_kernel<T, DP, WM>);
  const cudaError_t err = ensure_dynamic_smem(kernel, kBytes);
  if (err != cudaSuccess) { record_cuda_error(err); return GDN2_ERR_LAUNCH; }
  tree_kernel<T, DP, WM><<<unsigned(p.ctas), kThreads, kBytes, stream>>>(p);
  const int status = check_launch();
  if (status != GDN2_OK) return status;
  const int64_t units = int64_t(p.batch) * p.kv_heads * p.row_blocks;
  return launch_beside(&tree_join_kernel<T, DP>, unsigned(units), kThreads, 0, stream, p, 16 * WM);
}

template <typename T>
int launch_tree_dim(const TreeParams& p, cudaStream_t stream) {
  const int rows = block_rows(p.rows);
  if (p.dim <= 64) {
    return rows == 16 ? launch_tree_typed<T, 64, 1>(p, stream) : rows == 32 ? launch_tree_typed<T, 64, 2>(p, stream)
                                                                            : launch_tree_typed<T, 64, 4>(p, stream);
  }
  return rows == 16 ? launch_tree_typed<T, 128, 1>(p, stream) : rows == 32 ? launch_tree_typed<T, 128, 2>(p, stream)
                                                                           : launch_tree_typed<T, 128, 4>(p, stream);
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

// CTAs of a call: two an SM, which the tiles share whatever their number
int tree_ctas(int* ctas) {
  int sms = 0;
  const int status = multiprocessors(&sms);
  *ctas = 2 * sms;
  return status;
}

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
  p.scale_log2 = scale * kLog2e;
  return dtype == GDN2_BF16 ? launch_tree_dim<__nv_bfloat16>(p, stream) : launch_tree_dim<__half>(p, stream);
}

}  // namespace gdn2
