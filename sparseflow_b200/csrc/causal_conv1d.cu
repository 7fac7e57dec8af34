// Short causal convolution along a sequence, one filter per channel, with its
// backward pass and its single-token form.
//
//   pre[t,d] = bias[d] + sum_k w[d,k] x[t - (W-1) + k, d],   y = pre or silu(pre)
//   g = dy act'(pre);  dx[t] = sum_k w[k] g[t + (W-1) - k];
//   dw[k] = sum_t g[t] x[t - (W-1) + k];  dbias = sum_t g[t]
//
// About W + 9 instructions an element forward against 2 |x| bytes, 3 W + 15 backward against 3 |x|: HBM-bound, if
// enough bytes are on their way. A thread owns V neighbouring channels (8 bytes of a row, so a warp reads whole sectors)
// and walks down a slot of rows with the last W rows in registers. The rows ahead are copied asynchronously to a ring in
// shared memory, each thread its own, so no barrier guards it. Every x is read once, but for the W - 1 rows above each
// slot, which come from L2. Products and sums are pairs of fp32 (mul/fma .f32x2).
// Measured (bf16, 16384 rows of 4096 channels, 4 taps, SiLU): forward 58 us, 4.6 TB/s; backward 106 + 10 us (sums),
// 3.8 TB/s: 140 and 240 instructions for 8 channels of a warp's row at 0.6 a cycle, half of them the activation's
// exponentials and divisions and 16-bit conversions.
#include "sequence.cuh"

namespace sf {
namespace {

using seq::fma2;
using seq::pack2;
using seq::Rows;
using seq::Span;
using seq::u64;
using seq::unpack2;

constexpr int kConvThreads = 128;
constexpr int kMaxWidth = 8;
constexpr int kFwdGroup = 8, kBwdGroup = 4;  // rows copied together
constexpr int kFwdStages = 3, kBwdStages = 4;  // groups in the ring

struct ConvArgs {
  const void *x, *weight, *bias, *init, *dy, *dfinal;
  void *y, *final_state, *dx, *dinit;
  float* partial;
  Rows rows;
  long long x_batch, x_row;
  long long slot_rows;
  int dim, width, silu, w_dtype;
};

// V channels of a row as pairs (one channel: a pair whose second half is 0).
template <int V>
constexpr int kPairs = (V + 1) / 2;
template <typename T, int V>
__device__ __forceinline__ void to_pairs(u64 (&o)[kPairs<V>], const seq::Vec<T, V>& v) {
#pragma unroll
  for (int i = 0; i < kPairs<V>; ++i)
    o[i] = pack2(DT<T>::to_f(v.v[2 * i]), 2 * i + 1 < V ? DT<T>::to_f(v.v[(2 * i + 1) % V]) : 0.f);
}
template <typename T, int V>
__device__ __forceinline__ seq::Vec<T, V> from_pairs(const u64 (&p)[kPairs<V>]) {
  seq::Vec<T, V> v;
#pragma unroll
  for (int i = 0; i < kPairs<V>; ++i) {
    float lo, hi;
    unpack2(lo, hi, p[i]);
    v.v[2 * i] = DT<T>::from_f(lo);
    if (2 * i + 1 < V) v.v[(2 * i + 1) % V] = DT<T>::from_f(hi);
  }
  return v;
}
template <typename T, int V>
__device__ __forceinline__ seq::Vec<T, V> load_raw(const T* p) {
  return *reinterpret_cast<const seq::Vec<T, V>*>(p);
}
template <typename T, int V>
__device__ __forceinline__ void store_raw(T* p, const seq::Vec<T, V>& v) {
  *reinterpret_cast<seq::Vec<T, V>*>(p) = v;
}

// A thread's rows on their way: groups of G rows of N arrays. Single 16-bit channels, which no copy fits, are read when
// they are needed.
template <typename T, int V, int N, int G, int STAGES>
struct Ring {
  static constexpr bool ASYNC = V * sizeof(T) >= 4;
  seq::Vec<T, V> v[ASYNC ? STAGES : 1][N][G][kConvThreads];
};

// Row `t` of the sequence (t < 0: of the state before it; rows above that are 0).
template <typename T, int V>
__device__ __forceinline__ seq::Vec<T, V> load_row(const ConvArgs& a, const T* xs, const Span& p, long long t, int d) {
  if (t >= 0) return load_raw<T, V>(xs + t * a.x_row);
  const long long j = t + (a.width - 1);
  if (a.init && j >= 0)
    return load_raw<T, V>(static_cast<const T*>(a.init) + ((long long)p.s * (a.width - 1) + j) * a.dim + d);
  seq::Vec<T, V> z;
#pragma unroll
  for (int i = 0; i < V; ++i) z.v[i] = DT<T>::from_f(0.f);
  return z;
}

// First element of the sequence for channel d, and of its rows in a contiguous tensor.
template <typename T>
__device__ __forceinline__ const T* seq_x(const ConvArgs& a, const Span& p, int d) {
  return static_cast<const T*>(a.x) + (a.rows.offsets ? p.begin * a.x_row : (long long)p.s * a.x_batch) + d;
}
__device__ __forceinline__ long long seq_row0(const ConvArgs& a, const Span& p) {
  return a.rows.offsets ? p.begin : (long long)p.s * a.rows.length;
}

// W taps: WT = W up to 4, else 8, where the taps before the first (k < WT - W) are skipped, not multiplied by 0: the
// row they would meet may hold an infinity.
template <int WT>
__device__ __forceinline__ int skipped(const ConvArgs& a) {
  return WT <= 4 ? 0 : WT - a.width;
}
template <int V, int WT>
__device__ __forceinline__ void load_weights(u64 (&w)[WT][kPairs<V>], u64 (&b)[kPairs<V>], const ConvArgs& a, int d) {
#pragma unroll
  for (int i = 0; i < kPairs<V>; ++i) {
    float v[2];
#pragma unroll
    for (int k = 0; k < WT; ++k) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        v[h] = k >= skipped<WT>(a) && 2 * i + h < V
                   ? seq::load_param(a.weight, (long long)(d + 2 * i + h) * a.width + k - skipped<WT>(a), a.w_dtype)
                   : 0.f;
      w[k][i] = pack2(v[0], v[1]);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
      v[h] = a.bias && 2 * i + h < V ? seq::load_param(a.bias, d + 2 * i + h, a.w_dtype) : 0.f;
    b[i] = pack2(v[0], v[1]);
  }
}

// The same through shared memory, for blocks that walk down many rows: the block's weights [channels][W] are read once,
// in order, and turned to [tap][channel] (a thread's own reads would touch a sector each).
template <int V, int WT>
struct Weights {
  float w[WT][kConvThreads * V], b[kConvThreads * V];
};
template <int V, int WT>
__device__ __forceinline__ void stage_weights(Weights<V, WT>& s, const ConvArgs& a, int d0) {
  const int n = min(kConvThreads * V, a.dim - d0), skip = skipped<WT>(a);
  for (int i = threadIdx.x; i < n * a.width; i += kConvThreads)
    s.w[skip + i % a.width][i / a.width] = seq::load_param(a.weight, (long long)d0 * a.width + i, a.w_dtype);
  for (int i = threadIdx.x; i < n; i += kConvThreads)
    s.b[i] = a.bias ? seq::load_param(a.bias, d0 + i, a.w_dtype) : 0.f;
}
template <int V, int WT>
__device__ __forceinline__ void own_weights(u64 (&w)[WT][kPairs<V>], u64 (&b)[kPairs<V>], const Weights<V, WT>& s,
                                            int skip) {
#pragma unroll
  for (int i = 0; i < kPairs<V>; ++i) {
    const int c = threadIdx.x * V + 2 * i;
#pragma unroll
    for (int k = 0; k < WT; ++k) w[k][i] = k >= skip ? pack2(s.w[k][c], 2 * i + 1 < V ? s.w[k][c + 1] : 0.f) : 0;
    b[i] = pack2(s.b[c], 2 * i + 1 < V ? s.b[c + 1] : 0.f);
  }
}

// bias + sum over the taps of w[k] row[k]
template <int P, int WT>
__device__ __forceinline__ void taps(u64 (&o)[P], const u64 (&b)[P], const u64 (&w)[WT][P], const u64 (&row)[WT][P],
                                     int skip) {
#pragma unroll
  for (int i = 0; i < P; ++i) {
    o[i] = b[i];
#pragma unroll
    for (int k = 0; k < WT; ++k)
      if (k >= skip) o[i] = fma2(w[k][i], row[k][i], o[i]);
  }
}
template <int P, int WT>
__device__ __forceinline__ void shift(u64 (&row)[WT][P]) {
#pragma unroll
  for (int k = 0; k + 1 < WT; ++k)
#pragma unroll
    for (int i = 0; i < P; ++i) row[k][i] = row[k + 1][i];
}

template <typename T, int V, int WT, bool SILU>
__global__ void __launch_bounds__(kConvThreads, WT <= 4 ? 6 : 3) conv_fwd_kernel(ConvArgs a) {
  constexpr int P = kPairs<V>, G = kFwdGroup;
  using R = Ring<T, V, 1, G, kFwdStages>;
  extern __shared__ __align__(16) char smem[];
  R& ring = *reinterpret_cast<R*>(smem);
  Weights<V, WT>& sw = *reinterpret_cast<Weights<V, WT>*>(smem + sizeof(R));
  const int d0 = blockIdx.y * kConvThreads * V, d = d0 + threadIdx.x * V;
  const Span p = seq::slot_span(a.rows, blockIdx.x, a.slot_rows);
  if (p.len < 0) return;
  const T* xs = seq_x<T>(a, p, d);
  const long long r1 = min(p.r0 + a.slot_rows, p.len);
  const T* px = xs + p.r0 * a.x_row;  // the next group to copy
  long long tl = p.r0;
  int put = 0, get = 0;
  auto load = [&]() {
    if (d < a.dim) {
#pragma unroll
      for (int u = 0; u < G; ++u) {
        if (tl + u >= r1) break;
        if constexpr (R::ASYNC) seq::cp_async(&ring.v[put][0][u][threadIdx.x], px + u * a.x_row, V * sizeof(T), true);
      }
    }
    tl += G;
    px += G * a.x_row;
    seq::cp_async_commit();
    put = put + 1 == kFwdStages ? 0 : put + 1;
  };
  if constexpr (R::ASYNC)
    for (int i = 0; i < kFwdStages - 1; ++i) load();
  stage_weights<V, WT>(sw, a, d0);
  __syncthreads();
  if (d >= a.dim) return;
  const int skip = skipped<WT>(a);

  u64 w[WT][P], b[P], win[WT][P];  // win[WT-1]: the newest row
  own_weights<V, WT>(w, b, sw, skip);
#pragma unroll
  for (int k = 1; k < WT; ++k) to_pairs<T, V>(win[k], load_row<T, V>(a, xs, p, p.r0 - WT + k, d));
  T* py = static_cast<T*>(a.y) + (seq_row0(a, p) + p.r0) * a.dim + d;
  auto one = [&](const seq::Vec<T, V>& x, T* y) {
    shift<P, WT>(win);
    to_pairs<T, V>(win[WT - 1], x);
    u64 o[P];
    taps<P, WT>(o, b, w, win, skip);
    if (SILU) {
#pragma unroll
      for (int i = 0; i < P; ++i) {
        float lo, hi;
        unpack2(lo, hi, o[i]);
        o[i] = pack2(seq::silu(lo), seq::silu(hi));
      }
    }
    store_raw<T, V>(y, from_pairs<T, V>(o));
  };
  // Whole groups without conditions, so that the moving window costs no moves, then the rows that are left.
  for (long long t = p.r0; t < r1; t += G) {
    if constexpr (R::ASYNC) {
      seq::cp_async_wait<kFwdStages - 2>();
    } else {
#pragma unroll
      for (int u = 0; u < G; ++u)
        if (t + u < r1) ring.v[0][0][u][threadIdx.x] = load_raw<T, V>(xs + (t + u) * a.x_row);
    }
    if (t + G <= r1) {
#pragma unroll
      for (int u = 0; u < G; ++u) one(ring.v[get][0][u][threadIdx.x], py + (long long)u * a.dim);
    } else {
#pragma unroll
      for (int u = 0; u < G; ++u)
        if (t + u < r1) one(ring.v[get][0][u][threadIdx.x], py + (long long)u * a.dim);
    }
    py += (long long)G * a.dim;
    if constexpr (R::ASYNC) {
      get = get + 1 == kFwdStages ? 0 : get + 1;
      load();
    }
  }
  if (a.final_state && p.r0 == 0) {
    for (int j = 0; j < a.width - 1; ++j)
      store_raw<T, V>(static_cast<T*>(a.final_state) + ((long long)p.s * (a.width - 1) + j) * a.dim + d,
                      load_row<T, V>(a, xs, p, p.len - (a.width - 1) + j, d));
  }
}

// The gradient of pre at a row with gradient dy, from the W rows up to it.
template <typename T, int V, int WT, bool SILU>
__device__ __forceinline__ void pre_grad(u64 (&g)[kPairs<V>], const ConvArgs& a, const u64 (&w)[WT][kPairs<V>],
                                         const u64 (&b)[kPairs<V>], const u64 (&win)[WT][kPairs<V>],
                                         const seq::Vec<T, V>& dy) {
  constexpr int P = kPairs<V>;
  to_pairs<T, V>(g, dy);
  if (!SILU) return;
  u64 o[P];
  taps<P, WT>(o, b, w, win, skipped<WT>(a));
#pragma unroll
  for (int i = 0; i < P; ++i) {
    float lo, hi;
    unpack2(lo, hi, o[i]);
    g[i] = seq::mul2(g[i], pack2(seq::dsilu(lo), seq::dsilu(hi)));
  }
}

// Rows [r0, r1) of a slot: dx of these rows, which needs g up to W - 1 rows further down, and the sums over these
// rows of dw and dbias, written to partial[slot][W + 1][dim] for the reduction kernel. The weights are kept aligned to
// the oldest tap too (wr), so that dx[t - (W-1)] = sum_j wr[j] g[t - j] has constant indices.
template <typename T, int V, int WT, bool SILU>
__global__ void __launch_bounds__(kConvThreads, WT <= 4 ? 4 : 2) conv_bwd_kernel(ConvArgs a) {
  constexpr int P = kPairs<V>, G = kBwdGroup;
  using R = Ring<T, V, 2, G, kBwdStages>;
  extern __shared__ __align__(16) char smem[];
  R& ring = *reinterpret_cast<R*>(smem);
  Weights<V, WT>& sw = *reinterpret_cast<Weights<V, WT>*>(smem + sizeof(R));
  const int d0 = blockIdx.y * kConvThreads * V, d = d0 + threadIdx.x * V;
  const int W = WT <= 4 ? WT : a.width, skip = WT - W;
  float* part = a.partial + (long long)blockIdx.x * (W + 1) * a.dim + d;
  const Span p = seq::slot_span(a.rows, blockIdx.x, a.slot_rows);
  if (p.len >= 0) stage_weights<V, WT>(sw, a, d0);
  __syncthreads();
  if (d >= a.dim) return;
  if (p.len < 0) {  // a slot of no sequence still has a place in the sums
    for (int k = 0; k <= W; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) part[(long long)k * a.dim + i] = 0.f;
    return;
  }
  const T* xs = seq_x<T>(a, p, d);
  const long long row0 = seq_row0(a, p);
  const T* dys = static_cast<const T*>(a.dy) + row0 * a.dim + d;
  T* dxs = static_cast<T*>(a.dx) + row0 * a.dim + d;
  const long long r1 = min(p.r0 + a.slot_rows, p.len);

  u64 w[WT][P], b[P], win[WT][P], gw[WT][P], dw[WT][P], db[P];  // gw[WT-1-j]: g of j rows ago
  own_weights<V, WT>(w, b, sw, skip);
#pragma unroll
  for (int k = 0; k < WT; ++k)
#pragma unroll
    for (int i = 0; i < P; ++i) gw[k][i] = dw[k][i] = db[i] = 0;
#pragma unroll
  for (int k = 1; k < WT; ++k) to_pairs<T, V>(win[k], load_row<T, V>(a, xs, p, p.r0 - WT + k, d));
  const long long end = p.r0 < r1 ? r1 + W - 1 : r1;  // the slot's rows, and those whose gradients its last ones need
  const long long in = min(end, p.len);               // those that there are
  const T *px = xs + p.r0 * a.x_row, *pg = dys + p.r0 * a.dim;  // the next group to copy
  T* po = dxs + (p.r0 - (W - 1)) * a.dim;                       // where the gradient that row t completes goes
  long long tl = p.r0;
  int put_at = 0, get = 0;
  auto load = [&]() {
    if constexpr (R::ASYNC) {
#pragma unroll
      for (int u = 0; u < G; ++u) {
        if (tl + u >= in) break;
        seq::cp_async(&ring.v[put_at][0][u][threadIdx.x], px + u * a.x_row, V * sizeof(T), true);
        seq::cp_async(&ring.v[put_at][1][u][threadIdx.x], pg + (long long)u * a.dim, V * sizeof(T), true);
      }
      seq::cp_async_commit();
      put_at = put_at + 1 == kBwdStages ? 0 : put_at + 1;
      tl += G;
      px += G * a.x_row;
      pg += (long long)G * a.dim;
    }
  };
  for (int i = 0; i < kBwdStages - 1; ++i) load();

  // dx of row t - (W-1), which g of row t (in gw[WT - 1]) completes: sum over taps j of w[j] g[t - j].
  auto dx_row = [&](u64 (&o)[P]) {
#pragma unroll
    for (int i = 0; i < P; ++i) o[i] = 0;
#pragma unroll
    for (int s = 0; s < WT; ++s)
      if (s == skip) {
#pragma unroll
        for (int j = 0; j + s < WT; ++j)
#pragma unroll
          for (int i = 0; i < P; ++i) o[i] = fma2(w[j + s][i], gw[WT - 1 - j][i], o[i]);
      }
  };
  auto row = [&](int u) {
    shift<P, WT>(win);
    shift<P, WT>(gw);
    to_pairs<T, V>(win[WT - 1], ring.v[get][0][u][threadIdx.x]);
    pre_grad<T, V, WT, SILU>(gw[WT - 1], a, w, b, win, ring.v[get][1][u][threadIdx.x]);
  };
  auto add_sums = [&]() {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      db[i] = seq::add2(db[i], gw[WT - 1][i]);
#pragma unroll
      for (int k = 0; k < WT; ++k)
        if (k >= skip) dw[k][i] = fma2(gw[WT - 1][i], win[k][i], dw[k][i]);
    }
  };
  for (long long t = p.r0; t < end; t += G) {
    if constexpr (R::ASYNC) {
      seq::cp_async_wait<kBwdStages - 2>();
    } else {
#pragma unroll
      for (int u = 0; u < G; ++u)
        if (t + u < in) {
          ring.v[0][0][u][threadIdx.x] = load_raw<T, V>(xs + (t + u) * a.x_row);
          ring.v[0][1][u][threadIdx.x] = load_raw<T, V>(dys + (t + u) * a.dim);
        }
    }
    if (t + G <= r1) {  // the slot's own rows, without conditions, so that the moving windows cost no moves
      const int above = (int)(t - p.r0);  // rows of the slot before this group
#pragma unroll
      for (int u = 0; u < G; ++u) {
        u64 o[P];
        row(u);
        add_sums();
        dx_row(o);
        // The first W - 1 gradients complete rows of the slot before, which its own block stores.
        if (above + u >= W - 1) store_raw<T, V>(po + (long long)u * a.dim, from_pairs<T, V>(o));
      }
    } else {
#pragma unroll
      for (int u = 0; u < G; ++u)
        if (t + u < end) {
          if (t + u < p.len) {
            row(u);
          } else {
            shift<P, WT>(win);
            shift<P, WT>(gw);
#pragma unroll
            for (int i = 0; i < P; ++i) gw[WT - 1][i] = 0;
          }
          if (t + u < r1) add_sums();
          const long long v = t + u - (W - 1);
          u64 o[P];
          dx_row(o);
          if (v >= p.r0 && a.dfinal && t + u >= p.len) {
            u64 f[P];
            to_pairs<T, V>(f, load_raw<T, V>(static_cast<const T*>(a.dfinal) +
                                             ((long long)p.s * (W - 1) + t + u - p.len) * a.dim + d));
#pragma unroll
            for (int i = 0; i < P; ++i) o[i] = seq::add2(o[i], f[i]);
          }
          if (v >= p.r0) store_raw<T, V>(po + (long long)u * a.dim, from_pairs<T, V>(o));
        }
    }
    po += (long long)G * a.dim;
    get = !R::ASYNC || get + 1 == kBwdStages ? 0 : get + 1;
    load();
  }
  auto put = [&](int k, const u64 (&v)[P]) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      float lo, hi;
      unpack2(lo, hi, v[i]);
      part[(long long)k * a.dim + 2 * i] = lo;
      if (2 * i + 1 < V) part[(long long)k * a.dim + 2 * i + 1] = hi;
    }
  };
#pragma unroll
  for (int k = 0; k < WT; ++k)
    if (k >= skip) put(k - skip, dw[k]);
  put(W, db);

  // Gradient of the state before the sequence: virtual rows -(W-1) .. -1 under the first W - 1 rows. Row t reaches
  // virtual row v by tap v + (W-1) - t, so each row's g is found once and added to those above it.
  if (a.dinit && p.r0 == 0) {
    T* di = static_cast<T*>(a.dinit) + (long long)p.s * (W - 1) * a.dim + d;
    u64 o[WT - 1][P];  // o[WT - 2 - j]: virtual row -1 - j
#pragma unroll
    for (int j = 0; j < WT - 1; ++j)
#pragma unroll
      for (int i = 0; i < P; ++i) o[j][i] = 0;
#pragma unroll
    for (int t = 0; t < WT - 1; ++t)
      if (t < W - 1 && t < p.len) {
        u64 g[P], wn[WT][P];
#pragma unroll
        for (int k = 0; k < WT; ++k) to_pairs<T, V>(wn[k], load_row<T, V>(a, xs, p, t - (WT - 1) + k, d));
        pre_grad<T, V, WT, SILU>(g, a, w, b, wn, load_raw<T, V>(dys + (long long)t * a.dim));
        // wn[k] is virtual row t - (WT-1) + k, that is o[t + k] where it is below 0
#pragma unroll
        for (int k = 0; k + t < WT - 1; ++k)
          if (k >= skip)
#pragma unroll
            for (int i = 0; i < P; ++i) o[t + k][i] = fma2(w[k][i], g[i], o[t + k][i]);
      }
#pragma unroll
    for (int j = 0; j < WT - 1; ++j)
      if (j >= skip) {
        const int v = j - (WT - 1);  // -(W-1) .. -1
        // A sequence shorter than the state passes part of it on to the final state.
        const long long f0 = v - (p.len - (W - 1));
        if (a.dfinal && f0 >= 0) {
          u64 f[P];
          to_pairs<T, V>(f, load_raw<T, V>(static_cast<const T*>(a.dfinal) +
                                           ((long long)p.s * (W - 1) + f0) * a.dim + d));
#pragma unroll
          for (int i = 0; i < P; ++i) o[j][i] = seq::add2(o[j][i], f[i]);
        }
        store_raw<T, V>(di + (long long)(j - skip) * a.dim, from_pairs<T, V>(o[j]));
      }
  }
}

// Sums partial[slots][W + 1][dim] over the slots: dweight [dim, W] and dbias [dim]. A warp has 32 values and each of
// the block's 8 warps every eighth slot; the order is fixed.
__global__ void __launch_bounds__(256) conv_bwd_reduce_kernel(const float* partial, long long slots, int dim, int W,
                                                              int w_dtype, void* dweight, void* dbias) {
  __shared__ float sums[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long n = (long long)(W + 1) * dim, i = (long long)blockIdx.x * 32 + lane;
  float s = 0.f;
  if (i < n) {
#pragma unroll 8
    for (long long j = warp; j < slots; j += 8) s += partial[j * n + i];
  }
  sums[warp][lane] = s;
  __syncthreads();
  if (warp != 0 || i >= n) return;
#pragma unroll
  for (int w = 1; w < 8; ++w) s += sums[w][lane];
  const int k = (int)(i / dim), d = (int)(i % dim);
  if (k < W) seq::store_param(dweight, (long long)d * W + k, w_dtype, s);
  else if (dbias) seq::store_param(dbias, d, w_dtype, s);
}

template <typename T, int V, int WT>
__global__ void __launch_bounds__(kConvThreads) conv_update_kernel(ConvArgs a, T* pool, const int32_t* idx,
                                                                   int n_slots) {
  constexpr int P = kPairs<V>;
  const int d = (blockIdx.y * kConvThreads + threadIdx.x) * V;
  if (d >= a.dim) return;
  const int row = blockIdx.x, W = WT <= 4 ? WT : a.width, skip = WT - W;
  T* yp = static_cast<T*>(a.y) + (long long)row * a.dim + d;
  const int slot = idx ? idx[row] : row;
  u64 o[P];
  if (slot < 0 || slot >= n_slots) {
#pragma unroll
    for (int i = 0; i < P; ++i) o[i] = 0;
    store_raw<T, V>(yp, from_pairs<T, V>(o));
    return;
  }
  T* st = pool + (long long)slot * (W - 1) * a.dim + d;
  u64 w[WT][P], b[P], win[WT][P];
  seq::Vec<T, V> raw[WT];
  raw[WT - 1] = load_raw<T, V>(static_cast<const T*>(a.x) + (long long)row * a.x_row + d);
#pragma unroll
  for (int k = 0; k + 1 < WT; ++k)
    if (k >= skip) raw[k] = load_raw<T, V>(st + (long long)(k - skip) * a.dim);
  load_weights<V, WT>(w, b, a, d);
#pragma unroll
  for (int k = 0; k < WT; ++k)
    if (k >= skip) to_pairs<T, V>(win[k], raw[k]);
  taps<P, WT>(o, b, w, win, skip);
#pragma unroll
  for (int k = 1; k < WT; ++k)
    if (k > skip) store_raw<T, V>(st + (long long)(k - 1 - skip) * a.dim, raw[k]);
  if (a.silu) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      float lo, hi;
      unpack2(lo, hi, o[i]);
      o[i] = pack2(seq::silu(lo), seq::silu(hi));
    }
  }
  store_raw<T, V>(yp, from_pairs<T, V>(o));
}

bool valid(const sf_causal_conv1d_desc* d) {
  return d && d->length >= 0 && d->n_seq >= 0 && d->dim >= 0 && d->width >= 2 && d->width <= kMaxWidth &&
         dtype_size(d->dtype) != 0 && dtype_size(d->w_dtype) != 0;
}

// Whether every row of every tensor begins where a vector of V channels can be read; else a thread has one channel.
bool vectors_fit(int V, const sf_causal_conv1d_desc* d, bool batched, std::initializer_list<const void*> ptrs) {
  if (d->dim % V || d->x_row_stride % V || (batched && d->n_seq > 1 && d->x_batch_stride % V)) return false;
  for (const void* p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) % (V * dtype_size(d->dtype))) return false;
  return true;
}

ConvArgs base_args(const void* x, const void* weight, const void* bias, const void* init, const int32_t* offsets,
                   const sf_causal_conv1d_desc* d) {
  ConvArgs a = {};
  a.x = x;
  a.weight = weight;
  a.bias = bias;
  a.init = init;
  a.rows = Rows{offsets, d->length, d->n_seq};
  a.x_batch = d->x_batch_stride;
  a.x_row = d->x_row_stride;
  a.dim = d->dim;
  a.width = d->width;
  a.silu = d->silu;
  a.w_dtype = d->w_dtype;
  return a;
}

int channel_blocks(int dim, int V) { return (dim + V * kConvThreads - 1) / (V * kConvThreads); }

// Rows per slot: as many as leave `want` blocks (the W - 1 rows above a slot are read again, and in the backward pass
// its sums are written and read), between 8 and `most`. Forward, three blocks an SM that end together beat more in two
// rounds: 5003 ragged rows of 4096 channels take 25 us in slots of 64 rows, 27 of 32 and 30 of 16.
long long slot_rows(const sf_causal_conv1d_desc* d, int V, long long want, long long most) {
  const long long across = channel_blocks(d->dim, V);
  long long rows = most;
  while (rows > 8 && seq::total_slots(d->length, d->n_seq, d->packed, rows) * across < want) rows /= 2;
  return rows;
}
// Channels a thread: 8 bytes. With 16 there are half as many warps (forward, ragged prompts of 5003 rows: 38 us against
// 29), and the windows of the backward pass and of more than 4 taps would not fit the registers.
constexpr int kVecBytes = 8;
int vec_of(const sf_causal_conv1d_desc* d) { return kVecBytes / (int)dtype_size(d->dtype); }
long long fwd_rows(const sf_causal_conv1d_desc* d) { return slot_rows(d, vec_of(d), seq::kSms * 3, 64); }
long long bwd_rows(const sf_causal_conv1d_desc* d) { return slot_rows(d, vec_of(d), seq::kSms * 6, 128); }

template <typename T, int V, int WT>
sf_status run_fwd(const ConvArgs& a, dim3 grid, cudaStream_t st) {
  grid.y = channel_blocks(a.dim, V);
  constexpr size_t smem = sizeof(Ring<T, V, 1, kFwdGroup, kFwdStages>) + sizeof(Weights<V, WT>);
  auto kernel = a.silu ? conv_fwd_kernel<T, V, WT, true> : conv_fwd_kernel<T, V, WT, false>;
  if (smem > 48 * 1024 && !allow_max_smem(reinterpret_cast<const void*>(kernel))) return SF_ERR_CUDA;
  kernel<<<grid, kConvThreads, smem, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? SF_OK : SF_ERR_CUDA;
}
template <typename T, int V, int WT>
sf_status run_bwd(const ConvArgs& a, dim3 grid, cudaStream_t st) {
  grid.y = channel_blocks(a.dim, V);
  constexpr size_t smem = sizeof(Ring<T, V, 2, kBwdGroup, kBwdStages>) + sizeof(Weights<V, WT>);
  auto kernel = a.silu ? conv_bwd_kernel<T, V, WT, true> : conv_bwd_kernel<T, V, WT, false>;
  if (smem > 48 * 1024 && !allow_max_smem(reinterpret_cast<const void*>(kernel))) return SF_ERR_CUDA;
  kernel<<<grid, kConvThreads, smem, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? SF_OK : SF_ERR_CUDA;
}
template <typename T, int V, int WT>
sf_status run_update(const ConvArgs& a, dim3 grid, void* pool, const int32_t* idx, int n_slots, cudaStream_t st) {
  grid.y = channel_blocks(a.dim, V);
  conv_update_kernel<T, V, WT><<<grid, kConvThreads, 0, st>>>(a, static_cast<T*>(pool), idx, n_slots);
  return cudaGetLastError() == cudaSuccess ? SF_OK : SF_ERR_CUDA;
}

}  // namespace
}  // namespace sf

using namespace sf;

// CALL<T, V, WT> for the data type, with V channels a thread where `fit` (else one channel), 2, 3, 4 taps or up to 8.
#define SF_CONV_TYPE(TYPE, CALL, ...)                                                \
  {                                                                                  \
    using T = TYPE;                                                                  \
    constexpr int V = kVecBytes / (int)sizeof(T);                                    \
    switch (d->width) {                                                              \
      case 2: return fit ? CALL<T, V, 2>(__VA_ARGS__) : CALL<T, 1, 2>(__VA_ARGS__);  \
      case 3: return fit ? CALL<T, V, 3>(__VA_ARGS__) : CALL<T, 1, 3>(__VA_ARGS__);  \
      case 4: return fit ? CALL<T, V, 4>(__VA_ARGS__) : CALL<T, 1, 4>(__VA_ARGS__);  \
      default: return fit ? CALL<T, V, 8>(__VA_ARGS__) : CALL<T, 1, 8>(__VA_ARGS__); \
    }                                                                                \
  }
#define SF_CONV_DISPATCH(CALL, ...)                                 \
  switch (d->dtype) {                                               \
    case SF_DTYPE_F32: SF_CONV_TYPE(float, CALL, __VA_ARGS__)       \
    case SF_DTYPE_F16: SF_CONV_TYPE(__half, CALL, __VA_ARGS__)      \
    default: SF_CONV_TYPE(__nv_bfloat16, CALL, __VA_ARGS__)         \
  }

extern "C" sf_status sf_causal_conv1d(const void* x, const void* weight, const void* bias, const void* initial_state,
                                      const int32_t* seq_offsets, void* y, void* final_state,
                                      const sf_causal_conv1d_desc* d, void* stream) {
  if (!valid(d) || !weight || (seq_offsets != nullptr) != (d->packed != 0)) return SF_ERR_INVALID_ARG;
  if (d->n_seq == 0 || d->dim == 0) return SF_OK;
  if (d->length > 0 && (!x || !y)) return SF_ERR_INVALID_ARG;
  if (d->length == 0 && !final_state) return SF_OK;
  ConvArgs a = base_args(x, weight, bias, initial_state, seq_offsets, d);
  a.y = y;
  a.final_state = final_state;
  const bool fit = vectors_fit(vec_of(d), d, !d->packed, {x, initial_state, y, final_state});
  a.slot_rows = fwd_rows(d);
  const long long slots = seq::total_slots(d->length, d->n_seq, d->packed, a.slot_rows);
  if (slots > INT32_MAX) return SF_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)slots);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  SF_CONV_DISPATCH(run_fwd, a, grid, st)
}

extern "C" size_t sf_causal_conv1d_backward_workspace_size(const sf_causal_conv1d_desc* d) {
  if (!valid(d)) return 0;
  return (size_t)seq::total_slots(d->length, d->n_seq, d->packed, bwd_rows(d)) * (d->width + 1) * d->dim *
         sizeof(float);
}

static sf_status conv_backward(const ConvArgs& a, const sf_causal_conv1d_desc* d, bool fit, dim3 grid,
                               cudaStream_t st) {
  SF_CONV_DISPATCH(run_bwd, a, grid, st)
}

extern "C" sf_status sf_causal_conv1d_backward(const void* x, const void* weight, const void* bias,
                                               const void* initial_state, const int32_t* seq_offsets, const void* dy,
                                               const void* d_final_state, void* dx, void* dweight, void* dbias,
                                               void* d_initial_state, const sf_causal_conv1d_desc* d, void* workspace,
                                               size_t workspace_bytes, void* stream) {
  if (!valid(d) || !weight || !dweight || (d->n_seq > 0 && (seq_offsets != nullptr) != (d->packed != 0)))
    return SF_ERR_INVALID_ARG;
  if (d->dim == 0) return SF_OK;
  if (d->n_seq > 0 && d->length > 0 && (!x || !dy || !dx)) return SF_ERR_INVALID_ARG;
  if (bias && !dbias) return SF_ERR_INVALID_ARG;
  if (d->n_seq > 0 && (!workspace || workspace_bytes < sf_causal_conv1d_backward_workspace_size(d)))
    return SF_ERR_WORKSPACE;
  if (d->n_seq > 0 && !aligned16(workspace)) return SF_ERR_ALIGNMENT;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  ConvArgs a = base_args(x, weight, bias, initial_state, seq_offsets, d);
  long long slots = 0;  // without sequences the sums are 0
  if (d->n_seq > 0) {
    a.dy = dy;
    a.dfinal = d_final_state;
    a.dx = dx;
    a.dinit = d_initial_state;
    a.partial = static_cast<float*>(workspace);
    a.slot_rows = bwd_rows(d);
    slots = seq::total_slots(d->length, d->n_seq, d->packed, a.slot_rows);
    if (slots > INT32_MAX) return SF_ERR_UNSUPPORTED;
    const bool fit = vectors_fit(vec_of(d), d, !d->packed,
                                 {x, initial_state, dy, d_final_state, dx, d_initial_state});
    const sf_status s = conv_backward(a, d, fit, dim3((unsigned)slots), st);
    if (s != SF_OK) return s;
  }
  const long long n = (long long)(d->width + 1) * d->dim;
  conv_bwd_reduce_kernel<<<(unsigned)((n + 31) / 32), 256, 0, st>>>(a.partial, slots, d->dim, d->width, d->w_dtype,
                                                                    dweight, bias ? dbias : nullptr);
  return cudaGetLastError() == cudaSuccess ? SF_OK : SF_ERR_CUDA;
}

extern "C" sf_status sf_causal_conv1d_update(const void* x, void* state_pool, const void* weight, const void* bias,
                                             const int32_t* state_indices, void* y, int32_t n_slots,
                                             const sf_causal_conv1d_desc* d, void* stream) {
  if (!valid(d) || !weight || n_slots < 0) return SF_ERR_INVALID_ARG;
  if (d->n_seq == 0 || d->dim == 0) return SF_OK;
  if (!x || !y || (!state_pool && n_slots > 0)) return SF_ERR_INVALID_ARG;
  ConvArgs a = base_args(x, weight, bias, nullptr, nullptr, d);
  a.y = y;
  const bool fit = vectors_fit(vec_of(d), d, false, {x, state_pool, y});
  const dim3 grid(d->n_seq);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  SF_CONV_DISPATCH(run_update, a, grid, state_pool, state_indices, n_slots, st)
}
