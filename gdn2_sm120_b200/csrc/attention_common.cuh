// What the kernels of causal attention share: which rows a work item has, tensor maps, products of 16-bit operands.
#pragma once

#include <cuda.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <limits>

#include "chunk_common.cuh"
#include "tc05.cuh"

namespace gdn2 {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f;
// The scale of scores in powers of two: its sign goes to a product.  One of 0 becomes the smallest positive number, so that
// -inf * scale masks as ever (no score makes more than 2^-21 of it), and the largest ones stay finite.
inline float positive_scale(float scale) {
  return fminf(fmaxf(fabsf(scale) * kLog2e, std::numeric_limits<float>::denorm_min()), FLT_MAX);
}
constexpr int kTileRows = 256;   // query rows of a work item of the forward: two tiles of 128
constexpr int kMaxSequences = GDN2_PACKED_MAX_SEQUENCES;   // in a launch, whose parameters hold their table

// Sequences of one launch: `n` equally long ones (a [n, time] batch), or the entries of a table, longest first.  Row
// statistics (one float a query row) lie per head in tiles of 256 rows; tile numbers run through all sequences.
struct Sequences {
  struct Entry { int row0, len, tile0, pad; };
  int n, time, packed;        // time: rows of a sequence where not packed
  int tiles, tiles_each;      // of all, of one where not packed
  int64_t stat_rows;          // rows of a head's statistics: of all launches of a call
  int64_t stat_row0;          // of this launch
  Entry e[kMaxSequences];
};

struct Item {
  int row0, batch;   // where the sequence's first row is in the tensor maps
  int len, tile;     // of the sequence; number of the 256-row tile in it
  int64_t row;       // first row of the sequence in [rows][heads][dim]
  int64_t stat;      // first row of the sequence's statistics
};

// tile t of the launch; `last_first`: a sequence's last tiles come first
__device__ __forceinline__ Item find_item(const Sequences& s, int t, bool last_first) {
  Item it;
  if (!s.packed) {
    const int tile = t / s.n;
    it.batch = t - tile * s.n;
    it.tile = last_first ? s.tiles_each - 1 - tile : tile;
    it.row0 = 0;
    it.len = s.time;
    it.row = int64_t(it.batch) * s.time;
    it.stat = s.stat_row0 + int64_t(it.batch) * s.tiles_each * kTileRows;
    return it;
  }
  int lo = 0, hi = s.n - 1;
  while (lo < hi) {  // last entry with tile0 <= t
    const int mid = (lo + hi + 1) >> 1;
    if (s.e[mid].tile0 <= t) lo = mid; else hi = mid - 1;
  }
  const Sequences::Entry x = s.e[lo];
  const int each = (x.len + kTileRows - 1) / kTileRows, tile = t - x.tile0;
  it.batch = 0;
  it.tile = last_first ? each - 1 - tile : tile;
  it.row0 = x.row0;
  it.len = x.len;
  it.row = x.row0;
  it.stat = s.stat_row0 + int64_t(x.tile0) * kTileRows;
  return it;
}

// Items are in the order of their work, the longest first.  CTA c of n takes them by turns that go up and down, c,
// 2n - 1 - c, 2n + c, ...: the sums come out nearly equal without a counter.
__device__ __forceinline__ int64_t item_of_turn(int turn) {
  const int64_t n = gridDim.x, c = blockIdx.x;
  return turn * n + ((turn & 1) ? n - 1 - c : c);
}

// How often a wait polls; a test may have fewer.
uint32_t wait_polls();

// Waits of a CTA are bounded: whoever waits in vain says so, and all others stop waiting too.  A poll takes up to 4 us.  What
// is made of data that others waited for is right only where nobody has failed by then: whoever stores results looks at
// that behind the last barrier between them.
struct Waiter {
  volatile int* failed;
  uint32_t polls;
  // by whole warps, whose lanes agree on what came of it
  __device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity) const {
    return __all_sync(0xffffffffu, tc::mbar_test(bar, parity) || wait_on(bar, parity));
  }
  __device__ __forceinline__ bool nobody_failed() const { return __all_sync(0xffffffffu, *failed == 0); }   // by whole warps
  __device__ __forceinline__ bool wait_on(uint64_t* bar, uint32_t parity) const {
#pragma unroll 1
    for (uint32_t i = 0; i < polls; ++i) {
      if (tc::mbar_try_wait(bar, parity)) return true;
      if (*failed) return false;
    }
    *failed = 1;
    return false;
  }
};

// ---- 16-bit products ---------------------------------------------------------------------------------------
// Tiles of [rows][64] channels in lines of 128 bytes whose 16-byte pieces are permuted by the line (the 128-byte
// swizzle of the tiled copies); a tile of 128 channels is two of them.  One copy serves both ways of reading it:
//   K-major (contraction over channels): 8-line atoms, 1024 bytes apart; 16 channels are 32 bytes of a line.
//   MN-major (contraction over rows): an atom is 64 channels x 8 rows; 16 rows are 2048 bytes; the next 64 channels
//   are the next slab.
__device__ __forceinline__ uint64_t desc_k(uint32_t tile, uint32_t slab_bytes, int kstep) {
  return tc::smem_desc_at(tile, uint32_t(kstep >> 2) * slab_bytes + uint32_t(kstep & 3) * 32u, 16, 1024, 2);
}
__device__ __forceinline__ uint64_t desc_mn(uint32_t tile, uint32_t slab_bytes, int kstep) {
  return tc::smem_desc_at(tile, uint32_t(kstep) * 2048u, slab_bytes, 1024, 2);
}
__device__ __forceinline__ void mma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t id, uint32_t accumulate,
                                       uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(id), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t id, uint32_t accumulate,
                                       uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(id), "r"(accumulate), "r"(leader)
      : "memory");
}

template <typename T> struct Format;
template <> struct Format<__nv_bfloat16> { static constexpr uint32_t code = tc::kFmtBF16, exponent = 0x7f80u; };
template <> struct Format<__half> { static constexpr uint32_t code = tc::kFmtF16, exponent = 0x7c00u; };

// Where 8 channels of a row are in a tile: a slab has 64 channels, in lines of 128 bytes whose 16-byte pieces are permuted by
// the line.
template <int DP>
__device__ __forceinline__ uint32_t place_of(uint32_t base, uint32_t slab, int row, int piece) {
  return base + uint32_t(piece >> 3) * slab + uint32_t(row) * 128u + ((uint32_t(piece ^ row) & 7u) << 4);
}

// An infinite or NaN value must reach the rows that see it and no others, but in the product it would meet every row of a
// tile (0 * NaN): it leaves the tile, and is added to those rows at the end.  Rows first .. last - 1, by the warp that copied
// them; found(row) is called by threads that found one.
template <typename T, int DP, typename Found>
__device__ __forceinline__ void sift(uint32_t base, uint32_t slab, int first, int last, Found found) {
  constexpr int kPieces = DP / 8, kAtOnce = 32 / kPieces;
  const int lane = threadIdx.x & 31, piece = lane % kPieces, sub = lane / kPieces;
  __syncwarp();
  for (int r = first + sub; r < last; r += kAtOnce) {
    const uint32_t at = place_of<DP>(base, slab, r, piece);
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
      found(r);
    }
  }
}

template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  const typename Pair<T>::type v = Pair<T>::make(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// 2^x of two numbers, none above 127, on the FMA units, which are idle where the special-function unit is what bounds a
// phase.  Adding 1.5 * 2^23 rounds x to n, whose low bits are then those of the sum; f = x - n is in [-1/2, 1/2], where 2^f is
// 1 + f p(f) with the cubic p that interpolates (2^f - 1) / f at the four Chebyshev nodes (relative error 7e-6, a weight's
// rounding is 2^-9 or 2^-12); 2^n is made of its exponent.  Below -126.5 the result is 0; NaN stays NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 exp2_fma(float2 x) {
  x.x = max_nan(x.x, -127.f);
  x.y = max_nan(x.y, -127.f);
  const float2 t = add2(x, twice(12582912.f));
  const float2 f = minus2(x, add2(t, twice(-12582912.f)));
  float2 r = fma2(f, twice(0.009656711f), twice(0.055838283f));
  r = fma2(f, r, twice(0.2402253f));
  r = fma2(f, r, twice(0.69313675f));
  r = fma2(f, r, twice(1.f));
  return mul2(r, make_float2(__int_as_float((__float_as_int(t.x) << 23) + 0x3f800000), __int_as_float((__float_as_int(t.y) << 23) + 0x3f800000)));
}

// What a row's weights are made against: exp2((s - shift) c - scaled), for a score m that is the maximum of some tile so far.
// A nearby reference (|m c| below kNear) is fl(m c): that weights stand against m c rounded, by a factor of up to 2^(2^-14),
// is the same for all of a row's weights, sums and outputs.  Farther away the rounding of m c would itself be powers of two
// (16 at 2^28), so there the difference s - m comes first, which is 0 for m and negative for what is below it: no weight
// passes 1, however large the scores.
constexpr float kNear = 1024.f;
struct Reference { float shift, scaled; };
__device__ __forceinline__ Reference reference(float m, float c) {
  const float scaled = m * c;
  const bool near = fabsf(scaled) < kNear;
  return {near || m == -INFINITY ? 0.f : m, near ? scaled : 0.f};   // (-inf: nothing but weights of 0 so far, any will do)
}
// A row's statistic for the backward is -(r + log2 l) for a nearby reference r, rounded once; for one that is far away it is
// kFarMark - log2 l, above kFarFrom, and the reference itself is its second number.  (A nearby one with l as large as sums get
// stays within 1024 + 64.)
constexpr float kFarMark = 2048.f, kFarFrom = 1536.f;
// the exponent that takes what was made against the reference of `from` to that of `to`
__device__ __forceinline__ float between(float from, float to, float c) {
  const Reference a = reference(from, c), b = reference(to, c);
  return fmaf(a.shift - b.shift, c, a.scaled - b.scaled);
}
// What a chain, a warp or a CTA has, made against m, to the reference of top >= m; 0 where it has nothing
__device__ __forceinline__ float factor_to(float m, float top, float c) { return m == -INFINITY ? 0.f : exp2_approx(between(m, top, c)); }
// s - shift for kColumns scores of a row a thread, where they are in TMEM
template <int kColumns>
__device__ __noinline__ void take_shift(uint32_t s_at, float shift) {
#pragma unroll 1
  for (int x = 0; x < kColumns; x += 32) {
    uint32_t s[32];
    tc::tmem_ld32(s_at + x, s);
    tc::tmem_wait_ld();
#pragma unroll
    for (int y = 0; y < 32; ++y) s[y] = __float_as_uint(__uint_as_float(s[y]) - shift);
    tc::tmem_st32(s_at + x, s);
  }
  tc::tmem_wait_st();
}

// One tile of scores becomes weights, a row a thread: S (128 columns of TMEM at s_at) is read, masked, and overlaid by
// P in 16 bits, made against the reference of m, a maximum of some tile so far (-inf: nothing but -inf has been seen); `sum` is
// the sum of the row's weights.  No tile but the first looks for its maximum: where the sum of its weights stays below
// kGrowth, so does each of them, and nothing overflows or loses digits in 32 bits or in either 16-bit type.  Otherwise m
// becomes the maximum, sum and O (DP columns at o_at, as it is after all tiles before this one) are scaled down, and the
// tile's weights are made again, none of them above 1: a tile looks once at most.  Rows whose reference is far look at every
// tile, and then the shift is taken off where the scores are.
constexpr float kGrowth = 32768.f;

// mask(x, s): columns 32 x .. 32 x + 31 in s
template <typename Mask>
__device__ __forceinline__ float row_maximum(uint32_t s_at, Mask mask) {
  float top = -INFINITY;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    uint32_t s[32];
    tc::tmem_ld32(s_at + x * 32, s);
    tc::tmem_wait_ld();
    mask(x, s);
    float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int y = 0; y < 32; ++y) tops[y & 3] = fmaxf(tops[y & 3], __uint_as_float(s[y]));
    top = fmaxf(top, fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])));
  }
  return top;
}

template <typename T, typename Mask>
__device__ __forceinline__ float row_weights(uint32_t s_at, float c, float scaled, uint32_t (&w)[2][32], Mask mask) {
  const float2 minus = twice(-scaled), by = twice(c);
  float2 sum[2] = {{0.f, 0.f}, {0.f, 0.f}};
  uint32_t s[2][32];
  tc::tmem_ld32(s_at, s[0]);
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    tc::tmem_wait_ld();
    if (x < 3) tc::tmem_ld32(s_at + (x + 1) * 32, s[(x + 1) & 1]);
    mask(x, s[x & 1]);
#pragma unroll
    for (int y = 0; y < 16; ++y) {
      const float2 z = fma2(make_float2(__uint_as_float(s[x & 1][2 * y]), __uint_as_float(s[x & 1][2 * y + 1])), by, minus);
      const float2 e = exp2_2(z);
      sum[y & 1] = add2(sum[y & 1], e);
      w[x >> 1][(x & 1) * 16 + y] = pack_pair<T>(e.x, e.y);   // the sum has them as they were, the product rounded
    }
  }
  return (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
}

// m is -inf where there has been no tile
template <typename T, int DP, typename Mask>
__device__ __forceinline__ void soften(uint32_t s_at, uint32_t o_at, float c, float& m, float& sum, Mask mask) {
  uint32_t w[2][32];
  float more;
#pragma unroll 1
  for (bool look = __any_sync(0xffffffffu, !(fabsf(m * c) < kNear));;) {   // (-inf is not near)
    if (look) {
      const float top = fmaxf(m, row_maximum(s_at, mask));
      const float f = top > m && m != -INFINITY ? exp2_approx(between(m, top, c)) : 1.f;
      m = top;
      if (__any_sync(0xffffffffu, f != 1.f)) {
        sum *= f;
#pragma unroll
        for (int x = 0; x < DP; x += 16) {
          uint32_t o[16];
          tc::tmem_ld16(o_at + x, o);
          tc::tmem_wait_ld();
#pragma unroll
          for (int y = 0; y < 16; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
          tc::tmem_st16(o_at + x, o);
        }
      }
      const float shift = reference(m, c).shift;
      if (__any_sync(0xffffffffu, shift != 0.f)) take_shift<128>(s_at, shift);
    }
    more = row_weights<T>(s_at, c, reference(m, c).scaled, w, mask);
    if (look) break;
    look = __any_sync(0xffffffffu, more > kGrowth);
    if (!look) break;
  }
  sum += more;
  tc::tmem_st32(s_at, w[0]);
  tc::tmem_st32(s_at + 32, w[1]);
  tc::tmem_wait_st();
}

// 16 channels of a row, scaled and rounded.  Every lane of a warp has a row of its own, and an instruction takes as long as
// it has rows: 32 bytes each where rows are aligned to that (`wide`: 16 channels at a time), 16 otherwise.
template <typename T>
__device__ __forceinline__ void store_row16(T* to, const float (&x)[16], float by, int channels, bool wide) {
  uint32_t w[8];
#pragma unroll
  for (int y = 0; y < 8; ++y) w[y] = pack_pair<T>(x[2 * y] * by, x[2 * y + 1] * by);
  if (wide) {
    if (channels > 0) {
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                   "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                   : "memory");
    }
    return;
  }
  if (channels > 0) *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
  if (channels > 8) *reinterpret_cast<uint4*>(to + 8) = make_uint4(w[4], w[5], w[6], w[7]);
}
inline bool wide_rows(const void* base, int dim) { return dim % 16 == 0 && (reinterpret_cast<uintptr_t>(base) & 31) == 0; }

// The same with two threads a row, 64 columns each (S at s_at, P over the first half of them, DP / 2 columns of O at o_at):
// the latencies of a chain, and not its instructions, are what the tensor cores wait for.  All 256 threads of a chain look
// again together.  A quarter of the weights is made on the FMA units; there a score that is 127 powers of two above the
// reference counts as 127, and the row looks again.  (A reference that moves only where weights grow, and exponentials by a
// polynomial on the FMA units, have been published for other kernels of attention.)  8 x 4096 tokens, 16 heads (and one prompt of 16381, 8 heads): one thread
// a row 517 us (472), two 476 (450), with the FMA units' quarter 474 (427).
struct Pair {
  int chain, half, row;
  float (*told)[128];      // [half][row], what the two tell each other
  __device__ __forceinline__ void sync() const { asm volatile("bar.sync %0, 256;" ::"r"(chain + 1) : "memory"); }
  __device__ __forceinline__ void tell(float mine) const { told[half][row] = mine; sync(); }
  __device__ __forceinline__ float heard() const { return told[half ^ 1][row]; }   // a barrier later the next may be told
  __device__ __forceinline__ float other(float mine) const {
    tell(mine);
    const float r = heard();
    sync();
    return r;
  }
  __device__ __forceinline__ bool any(bool x) const {   // of the chain
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 q, %2, 0;\n\tbar.red.or.pred p, %1, 256, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(r) : "r"(chain + 1), "r"(uint32_t(x)) : "memory");
    return r != 0;
  }
};

// `far` says whether the reference of a row of the chain is; false before the first tile
template <typename T, int DP, typename Mask>
__device__ __forceinline__ void soften_half(const Pair& pair, uint32_t s_at, uint32_t o_at, float c, bool first, float& m, float& sum,
                                            bool& far, Mask mask) {
  uint32_t w[2][16];
  float more = 0.f;
#pragma unroll 1
  for (bool look = first || far;;) {
    if (look) {
      float top = -INFINITY;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        uint32_t s[32];
        tc::tmem_ld32(s_at + x * 32, s);
        tc::tmem_wait_ld();
        mask(x, s);
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int y = 0; y < 32; ++y) tops[y & 3] = fmaxf(tops[y & 3], __uint_as_float(s[y]));
        top = fmaxf(top, fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])));
      }
      pair.tell(top);
      top = fmaxf(top, pair.heard());
      const float before = m;
      m = first ? (top == -INFINITY ? 0.f : top) : fmaxf(m, top);   // (any will do for a row that has seen nothing but -inf)
      const float shift = reference(m, c).shift;
      far = pair.any(shift != 0.f);       // and all have heard
      if (!first) {
        const float f = m > before ? exp2_approx(between(before, m, c)) : 1.f;
        sum *= f;
#pragma unroll
        for (int x = 0; x < DP / 2; x += 16) {
          uint32_t o[16];
          tc::tmem_ld16(o_at + x, o);
          tc::tmem_wait_ld();
#pragma unroll
          for (int y = 0; y < 16; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
          tc::tmem_st16(o_at + x, o);
        }
      }
      if (__builtin_expect(far, 0)) take_shift<64>(s_at, shift);
    }
    const float2 minus = twice(-reference(m, c).scaled), by = twice(c);
    float2 sums[2] = {{0.f, 0.f}, {0.f, 0.f}};
    uint32_t s[2][32];
    tc::tmem_ld32(s_at, s[0]);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      tc::tmem_wait_ld();
      if (x == 0) tc::tmem_ld32(s_at + 32, s[1]);
      mask(x, s[x]);
#pragma unroll
      for (int y = 0; y < 16; ++y) {
        const float2 z = fma2(make_float2(__uint_as_float(s[x][2 * y]), __uint_as_float(s[x][2 * y + 1])), by, minus);
        const float2 e = (y & 3) == 3 ? exp2_fma(make_float2(min_nan(z.x, 127.f), min_nan(z.y, 127.f))) : exp2_2(z);
        sums[y & 1] = add2(sums[y & 1], e);
        w[x][y] = pack_pair<T>(e.x, e.y);   // the sum has them as they were, the product rounded
      }
    }
    more = (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y);
    if (look) break;    // no weight is above 1 (2^(2^-14) against a nearby reference)
    look = pair.any(more > kGrowth);
    if (!look) break;
  }
  sum += more;
  tc::tmem_st16(s_at, w[0]);
  tc::tmem_st16(s_at + 16, w[1]);
  tc::tmem_wait_st();
}

// [batch][rows][heads][dim] with any strides that are multiples of 16 bytes, in boxes of 64 channels x box_rows rows
// of one head.  Channels from dim on and rows behind a batch entry's last one arrive as zeros.
inline bool encode_heads_map(CUtensorMap* tm, const void* base, const int64_t* strides, int64_t batch, int64_t rows,
                             int64_t heads, int dim, int dtype, int box_rows) {
  const cuuint64_t dims[4] = {cuuint64_t(dim), cuuint64_t(heads), cuuint64_t(rows), cuuint64_t(batch)};
  const cuuint64_t bytes[3] = {cuuint64_t(strides[2]) * 2, cuuint64_t(strides[1]) * 2, cuuint64_t(strides[0]) * 2};
  const cuuint32_t box[4] = {64, 1, cuuint32_t(box_rows), 1};
  return encode_cached(tm, 4, dtype == GDN2_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                       base, dims, bytes, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// rows of a head's statistics for all sequences of a call
inline int64_t stat_rows(const int64_t* bounds, int64_t n_seq, int64_t time) {
  auto padded = [](int64_t n) { return (n + kTileRows - 1) / kTileRows * kTileRows; };
  if (bounds == nullptr) return n_seq * padded(time);
  int64_t rows = 0;
  for (int64_t i = 0; i < n_seq; ++i) rows += padded(bounds[i + 1] - bounds[i]);
  return rows;
}

// The launches of a call: one for a batch of equally long sequences (bounds null, `time` rows each), one for every
// kMaxSequences packed ones.  Fills *s for each and calls launch(); it follows from the bounds alone, so that forward
// and backward agree on where a row's statistics are.
template <typename Launch>
inline int for_groups(const int64_t* bounds, int64_t n_seq, int64_t time, Sequences* s, Launch launch) {
  s->stat_rows = stat_rows(bounds, n_seq, time);
  s->stat_row0 = 0;
  if (bounds == nullptr) {
    s->packed = 0;
    s->n = int(n_seq);
    s->time = int(time);
    s->tiles_each = int((time + kTileRows - 1) / kTileRows);
    s->tiles = s->tiles_each * s->n;
    return launch();
  }
  s->packed = 1;
  s->time = 0;
  s->tiles_each = 0;
  for (int64_t first = 0; first < n_seq; first += kMaxSequences) {
    const int count = int(n_seq - first < kMaxSequences ? n_seq - first : kMaxSequences);
    const int64_t* b = bounds + first;
    int order[kMaxSequences];
    for (int i = 0; i < count; ++i) order[i] = i;
    std::stable_sort(order, order + count, [&](int x, int y) { return b[x + 1] - b[x] > b[y + 1] - b[y]; });
    s->n = s->tiles = 0;
    for (int i = 0; i < count; ++i) {
      const int len = int(b[order[i] + 1] - b[order[i]]);
      if (len == 0) break;   // sorted: nothing but empty ones from here on
      s->e[s->n++] = Sequences::Entry{int(b[order[i]]), len, s->tiles, 0};
      s->tiles += (len + kTileRows - 1) / kTileRows;
    }
    if (s->n > 0) {
      const int status = launch();
      if (status != GDN2_OK) return status;
    }
    s->stat_row0 += int64_t(s->tiles) * kTileRows;
  }
  return GDN2_OK;
}

}  // namespace attn
}  // namespace gdn2
