// Short causal convolution along a sequence, one filter per channel, with its
// backward pass and its single-token form.
//
//   pre[t,d] = bias[d] + sum_k w[d,k] x[t - (W-1) + k, d],   y = pre or silu(pre)
//   g = dy act'(pre);  dx[t] = sum_k w[k] g[t + (W-1) - k];
//   dw[k] = sum_t g[t] x[t - (W-1) + k];  dbias = sum_t g[t]
//
// About 2 W + 5 operations an element against 2 |x| bytes: HBM-bound. A thread
// owns V neighbouring channels (16 or 8 bytes of a row, so a warp reads whole
// sectors) and walks down a slot of rows with the last W rows in registers:
// every x is read once, but for the W - 1 rows above each slot.
#include "sequence.cuh"

namespace sf {
namespace {

using seq::Rows;
using seq::Span;

constexpr int kConvThreads = 128;
constexpr int kMaxWidth = 8;

struct ConvArgs {
  const void *x, *weight, *bias, *init, *dy, *dfinal;
  void *y, *final_state, *dx, *dinit;
  float* partial;
  Rows rows;
  long long x_batch, x_row;
  long long slot_rows;
  int dim, width, silu, w_dtype;
};

// Row `t` of the sequence (t < 0: of the state before it; rows above that and channels past dim are 0).
template <typename T, int V>
__device__ __forceinline__ void load_row(float (&out)[V], const ConvArgs& a, const T* xs, const Span& p, long long t,
                                         int d) {
  if (t >= 0) {
    seq::load_vec<T, V>(out, xs + t * a.x_row);
    return;
  }
  const long long j = t + (a.width - 1);
  if (a.init && j >= 0) {
    seq::load_vec<T, V>(out, static_cast<const T*>(a.init) + ((long long)p.s * (a.width - 1) + j) * a.dim + d);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = 0.f;
  }
}

// First element of the sequence for channel d, and of its rows in a contiguous tensor.
template <typename T>
__device__ __forceinline__ const T* seq_x(const ConvArgs& a, const Span& p, int d) {
  return static_cast<const T*>(a.x) + (a.rows.offsets ? p.begin * a.x_row : (long long)p.s * a.x_batch) + d;
}
__device__ __forceinline__ long long seq_row0(const ConvArgs& a, const Span& p) {
  return a.rows.offsets ? p.begin : (long long)p.s * a.rows.length;
}

// W taps; WT is W rounded up to 4 or 8, the taps before the first (k < WT - W) are skipped, not multiplied by 0:
// the row they would meet may hold an infinity.
template <int V, int WT>
__device__ __forceinline__ void load_weights(float (&w)[WT][V], float (&b)[V], const ConvArgs& a, int d) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
#pragma unroll
    for (int k = 0; k < WT; ++k)
      w[k][i] = k >= WT - a.width
                    ? seq::load_param(a.weight, (long long)(d + i) * a.width + k - (WT - a.width), a.w_dtype)
                    : 0.f;
    b[i] = a.bias ? seq::load_param(a.bias, d + i, a.w_dtype) : 0.f;
  }
}

template <typename T, int V, int WT>
__global__ void __launch_bounds__(kConvThreads) conv_fwd_kernel(ConvArgs a) {
  const int d = (blockIdx.y * kConvThreads + threadIdx.x) * V;
  if (d >= a.dim) return;
  const Span p = seq::slot_span(a.rows, blockIdx.x, a.slot_rows);
  if (p.len < 0) return;
  const T* xs = seq_x<T>(a, p, d);
  T* ys = static_cast<T*>(a.y) + seq_row0(a, p) * a.dim + d;
  const long long r1 = min(p.r0 + a.slot_rows, p.len);

  float w[WT][V], b[V], win[WT][V];  // win[WT-1]: the newest row
  load_weights<V, WT>(w, b, a, d);
#pragma unroll
  for (int k = 1; k < WT; ++k) load_row<T, V>(win[k], a, xs, p, p.r0 - WT + k, d);
  for (long long t = p.r0; t < r1; ++t) {
#pragma unroll
    for (int k = 0; k + 1 < WT; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) win[k][i] = win[k + 1][i];
    seq::load_vec<T, V>(win[WT - 1], xs + t * a.x_row);
    float o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      o[i] = b[i];
#pragma unroll
      for (int k = 0; k < WT; ++k)
        if (k >= WT - a.width) o[i] = fmaf(w[k][i], win[k][i], o[i]);
      if (a.silu) o[i] = seq::silu(o[i]);
    }
    seq::store_vec<T, V>(ys + t * a.dim, o);
  }
  if (a.final_state && p.r0 == 0) {
    for (int j = 0; j < a.width - 1; ++j) {
      float o[V];
      load_row<T, V>(o, a, xs, p, p.len - (a.width - 1) + j, d);
      seq::store_vec<T, V>(
          static_cast<T*>(a.final_state) + ((long long)p.s * (a.width - 1) + j) * a.dim + d, o);
    }
  }
}

// The gradient of pre at row t (0 past the sequence's end), from the W rows up to t.
template <typename T, int V, int WT>
__device__ __forceinline__ void pre_grad(float (&g)[V], const ConvArgs& a, const float (&w)[WT][V],
                                         const float (&b)[V], const float (&win)[WT][V], const T* dys, long long t,
                                         long long len) {
  if (t >= len) {
#pragma unroll
    for (int i = 0; i < V; ++i) g[i] = 0.f;
    return;
  }
  seq::load_vec<T, V>(g, dys + t * a.dim);
  if (a.silu) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float o = b[i];
#pragma unroll
      for (int k = 0; k < WT; ++k)
        if (k >= WT - a.width) o = fmaf(w[k][i], win[k][i], o);
      g[i] *= seq::dsilu(o);
    }
  }
}

// Rows [r0, r1) of a slot: dx of these rows, which needs g up to W - 1 rows further down, and the sums over these
// rows of dw and dbias, written to partial[slot][W + 1][dim] for the reduction kernel.
template <typename T, int V, int WT>
__global__ void __launch_bounds__(kConvThreads) conv_bwd_kernel(ConvArgs a) {
  const int d = (blockIdx.y * kConvThreads + threadIdx.x) * V;
  if (d >= a.dim) return;
  const int W = a.width;
  float* part = a.partial + (long long)blockIdx.x * (W + 1) * a.dim + d;
  const Span p = seq::slot_span(a.rows, blockIdx.x, a.slot_rows);
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

  float w[WT][V], b[V], win[WT][V], gw[WT][V], dw[WT][V] = {}, db[V] = {};
  load_weights<V, WT>(w, b, a, d);
#pragma unroll
  for (int k = 0; k < WT; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) gw[k][i] = 0.f;
#pragma unroll
  for (int k = 1; k < WT; ++k) load_row<T, V>(win[k], a, xs, p, p.r0 - WT + k, d);
  if (p.r0 < r1) {
    for (long long t = p.r0; t < r1 + W - 1; ++t) {
#pragma unroll
      for (int k = 0; k + 1 < WT; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          win[k][i] = win[k + 1][i];
          gw[k][i] = gw[k + 1][i];  // gw[WT-1-j]: g of j rows ago
        }
      if (t < p.len) seq::load_vec<T, V>(win[WT - 1], xs + t * a.x_row);
      pre_grad<T, V, WT>(gw[WT - 1], a, w, b, win, dys, t, p.len);
      if (t < r1) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          db[i] += gw[WT - 1][i];
#pragma unroll
          for (int k = 0; k < WT; ++k)
            if (k >= WT - W) dw[k][i] = fmaf(gw[WT - 1][i], win[k][i], dw[k][i]);
        }
      }
      const long long u = t - (W - 1);  // the row whose gradient is complete now
      if (u >= p.r0) {
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = 0.f;
        // dx[u] = sum over taps j = 0..W-1 of w[j] g[u + (W-1) - j] = w[j] g[t - j]
#pragma unroll
        for (int j = 0; j < WT; ++j)
          if (j < W) {
#pragma unroll
            for (int kk = 0; kk < WT; ++kk)
              if (kk == j + WT - W)
#pragma unroll
                for (int i = 0; i < V; ++i) o[i] = fmaf(w[kk][i], gw[WT - 1 - j][i], o[i]);
          }
        if (a.dfinal && u >= p.len - (W - 1)) {
          float f[V];
          seq::load_vec<T, V>(f, static_cast<const T*>(a.dfinal) +
                                     ((long long)p.s * (W - 1) + u - (p.len - (W - 1))) * a.dim + d);
#pragma unroll
          for (int i = 0; i < V; ++i) o[i] += f[i];
        }
        seq::store_vec<T, V>(dxs + u * a.dim, o);
      }
    }
  }
  for (int k = 0; k < W; ++k)
#pragma unroll
    for (int kk = 0; kk < WT; ++kk)
      if (kk == k + WT - W)
#pragma unroll
        for (int i = 0; i < V; ++i) part[(long long)k * a.dim + i] = dw[kk][i];
#pragma unroll
  for (int i = 0; i < V; ++i) part[(long long)W * a.dim + i] = db[i];

  // Gradient of the state before the sequence: virtual rows -(W-1) .. -1 under the first W - 1 rows.
  if (a.dinit && p.r0 == 0) {
    T* di = static_cast<T*>(a.dinit) + (long long)p.s * (W - 1) * a.dim + d;
    for (int j = 0; j < W - 1; ++j) {
      float o[V];
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = 0.f;
      const long long v = j - (W - 1);
      for (long long t = 0; t <= v + W - 1 && t < p.len; ++t) {
        float g[V], wn[WT][V];
#pragma unroll
        for (int k = 0; k < WT; ++k) load_row<T, V>(wn[k], a, xs, p, t - (WT - 1) + k, d);
        pre_grad<T, V, WT>(g, a, w, b, wn, dys, t, p.len);
        const int tap = (int)(v + (W - 1) - t);
#pragma unroll
        for (int kk = 0; kk < WT; ++kk)
          if (kk == tap + WT - W)
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = fmaf(w[kk][i], g[i], o[i]);
      }
      // A sequence shorter than the state passes part of it on to the final state.
      const long long f0 = v - (p.len - (W - 1));
      if (a.dfinal && f0 >= 0) {
        float f[V];
        seq::load_vec<T, V>(f, static_cast<const T*>(a.dfinal) + ((long long)p.s * (W - 1) + f0) * a.dim + d);
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] += f[i];
      }
      seq::store_vec<T, V>(di + (long long)j * a.dim, o);
    }
  }
}

// Sums partial[slots][W + 1][dim] over the slots in order: dweight [dim, W] and dbias [dim].
__global__ void conv_bwd_reduce_kernel(const float* partial, long long slots, int dim, int W, int w_dtype,
                                       void* dweight, void* dbias) {
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= (long long)(W + 1) * dim) return;
  float s = 0.f;
  for (long long j = 0; j < slots; ++j) s += partial[j * (W + 1) * dim + i];
  const int k = (int)(i / dim), d = (int)(i % dim);
  if (k < W) seq::store_param(dweight, (long long)d * W + k, w_dtype, s);
  else if (dbias) seq::store_param(dbias, d, w_dtype, s);
}

template <typename T, int V, int WT>
__global__ void __launch_bounds__(kConvThreads) conv_update_kernel(ConvArgs a, T* pool, const int32_t* idx,
                                                                   int n_slots) {
  const int d = (blockIdx.y * kConvThreads + threadIdx.x) * V;
  if (d >= a.dim) return;
  const int row = blockIdx.x, W = a.width;
  T* yp = static_cast<T*>(a.y) + (long long)row * a.dim + d;
  const int slot = idx ? idx[row] : row;
  float o[V];
  if (slot < 0 || slot >= n_slots) {
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = 0.f;
    seq::store_vec<T, V>(yp, o);
    return;
  }
  T* st = pool + (long long)slot * (W - 1) * a.dim + d;
  float w[WT][V], win[WT][V];
  load_weights<V, WT>(w, o, a, d);
  seq::load_vec<T, V>(win[WT - 1], static_cast<const T*>(a.x) + (long long)row * a.x_row + d);
#pragma unroll
  for (int k = 0; k + 1 < WT; ++k)
    if (k >= WT - W) seq::load_vec<T, V>(win[k], st + (long long)(k - (WT - W)) * a.dim);
#pragma unroll
  for (int k = 0; k < WT; ++k)
    if (k >= WT - W) {
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = fmaf(w[k][i], win[k][i], o[i]);
      if (k > WT - W) seq::store_vec<T, V>(st + (long long)(k - 1 - (WT - W)) * a.dim, win[k]);
    }
  if (a.silu) {
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = seq::silu(o[i]);
  }
  seq::store_vec<T, V>(yp, o);
}

bool valid(const sf_causal_conv1d_desc* d) {
  return d && d->length >= 0 && d->n_seq >= 0 && d->dim >= 0 && d->width >= 2 && d->width <= kMaxWidth &&
         dtype_size(d->dtype) != 0 && dtype_size(d->w_dtype) != 0;
}

// Channels per thread: a 16-byte vector where every row of every tensor begins on one, else one channel.
template <typename T>
bool vectors_fit(int V, const sf_causal_conv1d_desc* d, bool packed, std::initializer_list<const void*> ptrs) {
  if (d->dim % V || d->x_row_stride % V || (!packed && d->n_seq > 1 && d->x_batch_stride % V)) return false;
  for (const void* p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) % (V * sizeof(T))) return false;
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

constexpr long long kFwdRows = 32, kBwdRows = 64;

template <typename T, int V>
sf_status run_fwd(const ConvArgs& a, cudaStream_t st) {
  const dim3 grid((unsigned)seq::total_slots(a.rows.length, a.rows.n_seq, a.rows.offsets != nullptr, a.slot_rows), channel_blocks(a.dim, V));
  if (a.width <= 4) conv_fwd_kernel<T, V, 4><<<grid, kConvThreads, 0, st>>>(a);
  else conv_fwd_kernel<T, V, 8><<<grid, kConvThreads, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? SF_OK : SF_ERR_CUDA;
}
template <typename T, int V>
sf_status run_bwd(const ConvArgs& a, void* dweight, void* dbias, cudaStream_t st) {
  const long long slots = seq::total_slots(a.rows.length, a.rows.n_seq, a.rows.offsets != nullptr, a.slot_rows);
  const dim3 grid((unsigned)slots, channel_blocks(a.dim, V));
  if (a.width <= 4) conv_bwd_kernel<T, V, 4><<<grid, kConvThreads, 0, st>>>(a);
  else conv_bwd_kernel<T, V, 8><<<grid, kConvThreads, 0, st>>>(a);
  const long long n = (long long)(a.width + 1) * a.dim;
  conv_bwd_reduce_kernel<<<(unsigned)((n + 127) / 128), 128, 0, st>>>(a.partial, slots, a.dim, a.width, a.w_dtype,
                                                                      dweight, dbias);
  return cudaGetLastError() == cudaSuccess ? SF_OK : SF_ERR_CUDA;
}
template <typename T, int V>
sf_status run_update(const ConvArgs& a, void* pool, const int32_t* idx, int n_slots, cudaStream_t st) {
  const dim3 grid(a.rows.n_seq, channel_blocks(a.dim, V));
  if (a.width <= 4) conv_update_kernel<T, V, 4><<<grid, kConvThreads, 0, st>>>(a, static_cast<T*>(pool), idx, n_slots);
  else conv_update_kernel<T, V, 8><<<grid, kConvThreads, 0, st>>>(a, static_cast<T*>(pool), idx, n_slots);
  return cudaGetLastError() == cudaSuccess ? SF_OK : SF_ERR_CUDA;
}

}  // namespace
}  // namespace sf

using namespace sf;

// f(type tag, vector width) for the data type: `fits` says whether 16-byte vectors do.
#define SF_SEQ_DISPATCH(DTYPE, FITS, CALL)                                                 \
  switch (DTYPE) {                                                                         \
    case SF_DTYPE_F32: {                                                                   \
      using T = float;                                                                     \
      if (FITS(4)) { constexpr int V = 4; return CALL; }                                   \
      constexpr int V = 1; return CALL;                                                    \
    }                                                                                      \
    case SF_DTYPE_F16: {                                                                   \
      using T = __half;                                                                    \
      if (FITS(8)) { constexpr int V = 8; return CALL; }                                   \
      constexpr int V = 1; return CALL;                                                    \
    }                                                                                      \
    case SF_DTYPE_BF16: {                                                                  \
      using T = __nv_bfloat16;                                                             \
      if (FITS(8)) { constexpr int V = 8; return CALL; }                                   \
      constexpr int V = 1; return CALL;                                                    \
    }                                                                                      \
  }                                                                                        \
  return SF_ERR_INVALID_ARG

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
  a.slot_rows = kFwdRows;
  if (seq::total_slots(a.rows.length, a.rows.n_seq, a.rows.offsets != nullptr, a.slot_rows) > INT32_MAX) return SF_ERR_UNSUPPORTED;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define FITS(n) vectors_fit<T>(n, d, seq_offsets != nullptr, {x, initial_state, y, final_state})
  SF_SEQ_DISPATCH(d->dtype, FITS, (run_fwd<T, V>(a, st)));
#undef FITS
}

extern "C" size_t sf_causal_conv1d_backward_workspace_size(const sf_causal_conv1d_desc* d) {
  if (!valid(d)) return 0;
  return (size_t)seq::total_slots(d->length, d->n_seq, d->packed, kBwdRows) * (d->width + 1) * d->dim *
         sizeof(float);
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
  if (d->n_seq > 0 && (reinterpret_cast<uintptr_t>(workspace) & 15u)) return SF_ERR_ALIGNMENT;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (d->n_seq == 0) {  // no rows: the sums are 0
    const long long n = (long long)(d->width + 1) * d->dim;
    conv_bwd_reduce_kernel<<<(unsigned)((n + 127) / 128), 128, 0, st>>>(nullptr, 0, d->dim, d->width, d->w_dtype,
                                                                        dweight, dbias);
    return cudaGetLastError() == cudaSuccess ? SF_OK : SF_ERR_CUDA;
  }
  ConvArgs a = base_args(x, weight, bias, initial_state, seq_offsets, d);
  a.dy = dy;
  a.dfinal = d_final_state;
  a.dx = dx;
  a.dinit = d_initial_state;
  a.partial = static_cast<float*>(workspace);
  a.slot_rows = kBwdRows;
  if (seq::total_slots(a.rows.length, a.rows.n_seq, a.rows.offsets != nullptr, a.slot_rows) > INT32_MAX) return SF_ERR_UNSUPPORTED;
#define FITS(n) vectors_fit<T>(n, d, seq_offsets != nullptr, {x, initial_state, dy, d_final_state, dx, d_initial_state})
  SF_SEQ_DISPATCH(d->dtype, FITS, (run_bwd<T, V>(a, dweight, bias ? dbias : nullptr, st)));
#undef FITS
}

extern "C" sf_status sf_causal_conv1d_update(const void* x, void* state_pool, const void* weight, const void* bias,
                                             const int32_t* state_indices, void* y, int32_t n_slots,
                                             const sf_causal_conv1d_desc* d, void* stream) {
  if (!valid(d) || !weight || n_slots < 0) return SF_ERR_INVALID_ARG;
  if (d->n_seq == 0 || d->dim == 0) return SF_OK;
  if (!x || !y || !state_pool) return SF_ERR_INVALID_ARG;
  ConvArgs a = base_args(x, weight, bias, nullptr, nullptr, d);
  a.y = y;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define FITS(n) vectors_fit<T>(n, d, true, {x, state_pool, y})
  SF_SEQ_DISPATCH(d->dtype, FITS, (run_update<T, V>(a, state_pool, state_indices, n_slots, st)));
#undef FITS
}
