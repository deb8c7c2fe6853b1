// Rotary positions of an attention layer's queries and keys, and their gradient.
//
// Channel pair i of a head at position p turns by the angle whose cosine and sine are cos[p][i], sin[p][i]:
//
//   y_a = x_a c - x_b s        y_b = x_b c + x_a s        (32-bit arithmetic, one rounding)
//
// with (a, b) = (i, i + R/2) in the half layout, (2i, 2i + 1) in the interleaved one; R = 2 * pairs channels turn,
// the others pass.  The gradient is the transposed rotation: the same kernel with -s.
//
// Bound by HBM: every value is read and written once, 20 KiB each way for a token of 40 heads of 128, against 512 B of
// angles, which the heads of a token share.  A thread keeps the angles of its pairs in registers and goes from head to
// head, but where there are few tokens; q and k are one launch.

#include <algorithm>

#include "common.cuh"

namespace gdn2 {

namespace {

// Heads that a thread takes one after the other where that leaves every SM full of threads: what a thread does
// once (its place, its angles) is spread over them.  q and k of 2 x 8192 tokens, 40 heads, forward and backward: 2 heads
// 144 us, 5 136, 10 132.
constexpr int kHeadsInTurn = 10;
constexpr int64_t kManyUnits = int64_t(148) * 2048 * kHeadsInTurn;
// Up to here a call takes as long as one thread does: every unit (two packs of channels of a head) has a thread of its own,
// and is fetched while the position and then the angles are looked up.  40 heads of 128 in a replayed graph, with this and
// with the loop over heads: 64 tokens 2.3 and 2.7 us, 256 3.15 and 3.45, 512 4.15 and 4.0, 1500 8.1 and 7.2.
constexpr int64_t kFewUnits = int64_t(148) * 768;

struct RotaryParams {
  const void* x[2];
  void* y[2];
  int64_t x_stride[2][3], y_stride[2][3];  // batch, token, head, in elements
  int heads[2];
  const float *cos, *sin;                  // [table][pairs]
  const int64_t* positions;                // [batch or 1][time], or null: a token's number in its sequence
  int64_t position_stride, table;
  int64_t time, tokens;                    // below 2^31
  int pairs, units, units_turned, interleaved;
  int heads_at_once, tokens_at_once;
  bool copy_rest;                          // the channels that do not turn have another place to go
  float sign;
};

// V consecutive elements as they lie in memory
template <typename T, int V> struct alignas(sizeof(T) * V) Pack { T v[V]; };

template <typename T, int V>
__device__ __forceinline__ void turn(Pack<T, V>& lo, Pack<T, V>& hi, const float* c, const float* s, bool interleaved) {
  float a[2 * V];
#pragma unroll
  for (int j = 0; j < V; ++j) { a[j] = to_float(lo.v[j]); a[V + j] = to_float(hi.v[j]); }
  if (interleaved) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float u = a[2 * j], w = a[2 * j + 1];
      a[2 * j] = u * c[j] - w * s[j];
      a[2 * j + 1] = w * c[j] + u * s[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float u = a[j], w = a[V + j];
      a[j] = u * c[j] - w * s[j];
      a[V + j] = w * c[j] + u * s[j];
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) { lo.v[j] = from_float<T>(a[j]); hi.v[j] = from_float<T>(a[V + j]); }
}

// kFew: blockIdx.y counts the heads that a CTA begins with, and a thread has one unit
template <typename T, int V, bool kFew>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryParams p) {
  using P = Pack<T, V>;
  const uint32_t per_token = uint32_t(p.units * p.heads_at_once);
  const uint32_t slot = p.tokens_at_once == 1 ? 0 : threadIdx.x / per_token;
  const uint32_t token = blockIdx.x * p.tokens_at_once + slot;
  if (token >= uint32_t(p.tokens)) return;
  const uint32_t at = threadIdx.x - slot * per_token;
  const int in_pass = int(at / uint32_t(p.units)), unit = int(at - uint32_t(in_pass) * uint32_t(p.units));
  const int first_head = kFew ? in_pass + int(blockIdx.y) * p.heads_at_once : in_pass;
  const int64_t b = token / uint32_t(p.time), t = token - uint32_t(b) * uint32_t(p.time);

  // a unit is two packs of a head: those of V pairs, or 2 V channels that pass
  const bool turns = unit < p.units_turned;
  if (!turns && !p.copy_rest) return;
  const int i = unit * V;
  const int c0 = !turns ? 2 * p.pairs + 2 * V * (unit - p.units_turned) : p.interleaved ? 2 * i : i;
  const int c1 = !turns || p.interleaved ? c0 + V : i + p.pairs;
  float c[V], s[V];
  auto angles = [&] {
    const int64_t pos = p.positions != nullptr ? p.positions[b * p.position_stride + t] : t;
    if (pos >= 0 && pos < p.table) {
      const Pack<float, V> pc = *reinterpret_cast<const Pack<float, V>*>(p.cos + pos * p.pairs + i);
      const Pack<float, V> ps = *reinterpret_cast<const Pack<float, V>*>(p.sin + pos * p.pairs + i);
#pragma unroll
      for (int j = 0; j < V; ++j) { c[j] = pc.v[j]; s[j] = p.sign * ps.v[j]; }
    } else {  // no such row in the table: the token's rotated channels become NaN
#pragma unroll
      for (int j = 0; j < V; ++j) c[j] = s[j] = __int_as_float(0x7fffffff);
    }
  };
  // the token's rows of q, then those of k as heads behind them
  const int heads = p.heads[0] + p.heads[1];
  const T *x0[2];
  T *y0[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    x0[x] = static_cast<const T*>(p.x[x]) + b * p.x_stride[x][0] + t * p.x_stride[x][1] - x * p.heads[0] * p.x_stride[x][2];
    y0[x] = static_cast<T*>(p.y[x]) + b * p.y_stride[x][0] + t * p.y_stride[x][1] - x * p.heads[0] * p.y_stride[x][2];
  }
  if (!kFew && turns) angles();
  for (int h = first_head; h < heads; h += p.heads_at_once) {
    const bool of_k = h >= p.heads[0];
    const T* x = (of_k ? x0[1] : x0[0]) + h * (of_k ? p.x_stride[1][2] : p.x_stride[0][2]);
    T* y = (of_k ? y0[1] : y0[0]) + h * (of_k ? p.y_stride[1][2] : p.y_stride[0][2]);
    P lo = *reinterpret_cast<const P*>(x + c0), hi = *reinterpret_cast<const P*>(x + c1);
    if (kFew && turns) angles();
    if (turns) turn(lo, hi, c, s, p.interleaved);
    *reinterpret_cast<P*>(y + c0) = lo;
    *reinterpret_cast<P*>(y + c1) = hi;
    if (kFew) return;
  }
}

template <typename T, int V>
void launch_width(const RotaryParams& p, unsigned blocks, int passes, int threads, cudaStream_t stream) {
  if (passes > 0) rotary_kernel<T, V, true><<<dim3(blocks, unsigned(passes)), threads, 0, stream>>>(p);
  else rotary_kernel<T, V, false><<<blocks, threads, 0, stream>>>(p);
}

template <typename T>
int launch_typed(const RotaryParams& base, int dim, int vec, cudaStream_t stream) {
  RotaryParams p = base;
  p.units_turned = p.pairs / vec;
  p.units = dim / (2 * vec);
  const int heads = p.heads[0] + p.heads[1];
  if (p.units > 256) return GDN2_ERR_BAD_SHAPE;
  // as many heads at once as leave no pass half empty, then as many tokens as fill the block
  const int most = 256 / p.units;
  int passes = (heads + most - 1) / most;
  if (p.tokens * heads * p.units >= kManyUnits) passes = std::max(passes, std::min(heads, kHeadsInTurn));
  p.heads_at_once = (heads + passes - 1) / passes;
  p.tokens_at_once = 256 / (p.units * p.heads_at_once);
  const int threads = p.units * p.heads_at_once * p.tokens_at_once;
  const int64_t blocks = (p.tokens + p.tokens_at_once - 1) / p.tokens_at_once;
  if (blocks <= 0 || blocks > int64_t(0x7fffffff)) return GDN2_ERR_TOO_LARGE;
  const int apart = p.tokens * heads * p.units <= kFewUnits ? (heads + p.heads_at_once - 1) / p.heads_at_once : 0;
  constexpr int kWide = 16 / int(sizeof(T));
  if (vec == kWide) launch_width<T, kWide>(p, unsigned(blocks), apart, threads, stream);
  else if (vec == 4) launch_width<T, 4>(p, unsigned(blocks), apart, threads, stream);
  else launch_width<T, 1>(p, unsigned(blocks), apart, threads, stream);
  return check_launch();
}

}  // namespace

int launch_rotary(const void* q, const void* k, void* q_out, void* k_out, const float* cos, const float* sin,
                  const int64_t* positions, const int64_t* strides, int64_t position_stride, int64_t batch, int64_t time,
                  int q_heads, int k_heads, int dim, int pairs, int64_t table, int interleaved, int inverse, int dtype,
                  cudaStream_t stream) {
  RotaryParams p{};
  p.x[0] = q; p.x[1] = k; p.y[0] = q_out; p.y[1] = k_out;
  for (int i = 0; i < 2; ++i) {
    for (int j = 0; j < 3; ++j) { p.x_stride[i][j] = strides[3 * i + j]; p.y_stride[i][j] = strides[6 + 3 * i + j]; }
  }
  p.heads[0] = q_heads; p.heads[1] = k_heads;
  p.cos = cos; p.sin = sin; p.positions = positions;
  p.position_stride = position_stride; p.table = table;
  p.time = time; p.tokens = batch * time;
  p.pairs = pairs; p.interleaved = interleaved;
  p.copy_rest = q != q_out;
  p.sign = inverse ? -1.f : 1.f;
  // The widest access that every row allows: 16 bytes, or four elements, or one.  (Tables are read in packs of as many
  // floats, 16 bytes at a time for any width but one.)
  const int es = dtype == GDN2_FP32 ? 4 : 2;
  auto fits = [&](int v) {
    if (pairs % v != 0 || (dim - 2 * pairs) % (2 * v) != 0) return false;
    uintptr_t bits = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) |
                     reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(k_out);
    for (int i = 0; i < 12; ++i) bits |= uintptr_t(strides[i]) * uintptr_t(es);
    const uintptr_t tables = reinterpret_cast<uintptr_t>(cos) | reinterpret_cast<uintptr_t>(sin);
    return bits % uintptr_t(v * es) == 0 && tables % uintptr_t(v * 4) == 0;
  };
  const int wide = 16 / es;
  const int vec = fits(wide) ? wide : fits(4) ? 4 : 1;
  if (dtype == GDN2_BF16) return launch_typed<__nv_bfloat16>(p, dim, vec, stream);
  if (dtype == GDN2_FP16) return launch_typed<__half>(p, dim, vec, stream);
  return launch_typed<float>(p, dim, vec, stream);
}

}  // namespace gdn2
