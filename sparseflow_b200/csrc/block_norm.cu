// The norms around a block, with its gate and residual scale, in one pass:
//
//   u = w_post y rstd1,  rstd1 = rsqrt(mean y^2 + eps)        (norm after the block)
//   r' = alpha residual + scale act(gate) u                   (gate, residual scale, residual)
//   x' = w_pre r' rstd2, rstd2 = rsqrt(mean r'^2 + eps)       (norm before the next block)
//
// Backward, from dr and dx (gradients of r' and x'), with yh = y rstd1, rh = r' rstd2, G = scale act(gate):
//   dt   = dr + rstd2 (w_pre dx - rh c2),   c2 = mean(w_pre dx rh)
//   dres = alpha dt;  dgate = dt scale u act'(gate);  dscale = sum dt act(gate) u
//   du   = dt G;      dy = rstd1 (w_post du - yh c1),  c1 = mean(w_post du yh)
//   dw_post = sum du yh;  dw_pre = sum dx rh
// c1 depends on c2 through dt, but linearly: with e = w_post G yh, c1 = mean(e (dr + rstd2 w_pre dx))
// - c2 rstd2 mean(e rh), so one reduction of three sums serves both.
// r' is computed again from y, residual and gate: the stored one is rounded to the residual's type.
//
// The sums over rows need one accumulator for both weights behind the norm: with Q = sum dt act(gate) yh,
// dscale = w_post Q and dw_post = scale Q.
//
// About 14 operations an element forward and 36 backward against 4 to 7 tensors moved: HBM-bound. A block holds whole
// rows, 8 neighbouring channels a thread, and walks down a range of rows with the weights and the sums over rows in
// registers, while the rows ahead are copied asynchronously to a ring in shared memory, each thread its own channels
// (no barrier guards the ring). Measured (bf16, fp32 residual, 8192 rows of 4096 channels, SiLU gate): forward 93 us, 4.9
// TB/s; backward 178 us, 4.1 TB/s: one block of 512 threads fills an SM's registers, so nothing covers the sum over
// the block between the two halves of a row. Rows of more than kRingDim channels are shared backward by a cluster of two
// or four blocks, which add up through each other's shared memory. Rows that 16-byte copies do not fit, and wider rows
// forward, take the kernels without a ring.
#include <cooperative_groups.h>
#include "sequence.cuh"

namespace sf {
namespace {

using seq::add2;
using seq::fma2;
using seq::mul2;
using seq::pack2;
using seq::u64;
using seq::unpack2;

constexpr int kV = 8;             // channels per vector: 16 bytes of a 16-bit type
constexpr int kRingDim = 4096;    // channels of a row in a block of 512 threads
constexpr int kMaxDim = 16384;    // 1024 threads, two vectors each

struct NormArgs {
  const void *y, *res, *gate, *w_post, *w_pre, *scale;
  void *r_out, *x_out;
  float* rstd;
  const void *dr, *dx;
  void *dy, *dres, *dgate;
  float *part_w, *part_gate;  // backward partial sums: [blocks][2][dim] (Q, dw_pre), [blocks][dim]
  long long rows, y_row, res_row, gate_row, rows_per_gate;
  int dim, w_dtype, gate_kind;
  float alpha, eps;
  int vec;  // whether every row of every tensor takes vector accesses
  int cluster, slice;  // kernels with a ring: blocks that share a row, channels of it in each
};

// 8 channels from column c on as floats; past dim: 0.
template <typename T>
__device__ __forceinline__ void load8(float (&o)[kV], const T* p, int c, int dim, int vec) {
  if (vec) {
    if (c < dim) {
      constexpr int W = 16 / sizeof(T);
#pragma unroll
      for (int h = 0; h < kV; h += W) {
        float t[W];
        seq::load_vec<T, W>(t, p + c + h);
#pragma unroll
        for (int i = 0; i < W; ++i) o[h + i] = t[i];
      }
      return;
    }
  } else if (c < dim) {
#pragma unroll
    for (int i = 0; i < kV; ++i) o[i] = c + i < dim ? DT<T>::to_f(p[c + i]) : 0.f;
    return;
  }
#pragma unroll
  for (int i = 0; i < kV; ++i) o[i] = 0.f;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[kV], int c, int dim, int vec) {
  if (c >= dim) return;
  if (vec) {
    constexpr int W = 16 / sizeof(T);
#pragma unroll
    for (int h = 0; h < kV; h += W) {
      float t[W];
#pragma unroll
      for (int i = 0; i < W; ++i) t[i] = v[h + i];
      seq::store_vec<T, W>(p + c + h, t);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kV; ++i)
      if (c + i < dim) p[c + i] = DT<T>::from_f(v[i]);
  }
}
__device__ __forceinline__ void load_w8(float (&o)[kV], const void* p, int c, int dim, int vec, int dtype) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < kV; ++i) o[i] = 1.f;
  } else if (dtype == SF_DTYPE_F32) {
    load8<float>(o, static_cast<const float*>(p), c, dim, vec);
  } else if (dtype == SF_DTYPE_F16) {
    load8<__half>(o, static_cast<const __half*>(p), c, dim, vec);
  } else {
    load8<__nv_bfloat16>(o, static_cast<const __nv_bfloat16*>(p), c, dim, vec);
  }
}

// act(gate) and its derivative.
__device__ __forceinline__ float gate_act(float g, int kind) {
  if (kind == SF_GATE_SILU) return seq::silu(g);
  if (kind == SF_GATE_SIGMOID) return seq::logistic(g);
  return g;
}
__device__ __forceinline__ float gate_dact(float g, int kind) {
  if (kind == SF_GATE_SILU) return seq::dsilu(g);
  if (kind == SF_GATE_SIGMOID) {
    const float s = seq::logistic(g);
    return s * (1.f - s);
  }
  return 1.f;
}

// Sums of N values over the block, in every thread; the order is fixed.
template <int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float* buf) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
  const int warps = blockDim.x >> 5, w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warps == 1) return;
  __syncthreads();  // buf may still be read from the sum before
  if (lane == 0)
#pragma unroll
    for (int n = 0; n < N; ++n) buf[w * N + n] = v[n];
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    float s = lane < warps ? buf[lane * N + n] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    v[n] = s;
  }
}

template <typename T, typename R, int K>
__global__ void __launch_bounds__(1024) norm_fwd_kernel(NormArgs a) {
  __shared__ float buf[32];
  const float inv = 1.f / (float)a.dim;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* yp = static_cast<const T*>(a.y) + row * a.y_row;
    const long long gate_row = a.rows_per_gate == 1 ? row : row / a.rows_per_gate;
    float r[K][kV];
    float s1[1] = {0.f};
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * blockDim.x + threadIdx.x) * kV;
      load8<T>(r[k], yp, c, a.dim, a.vec);
#pragma unroll
      for (int i = 0; i < kV; ++i) s1[0] = fmaf(r[k][i], r[k][i], s1[0]);
    }
    float rstd1 = 1.f;
    if (a.w_post) {
      block_sum<1>(s1, buf);
      rstd1 = rsqrtf(s1[0] * inv + a.eps);
    }
    float s2[1] = {0.f};
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * blockDim.x + threadIdx.x) * kV;
      float t[kV];
      if (a.w_post) {
        load_w8(t, a.w_post, c, a.dim, a.vec, a.w_dtype);
#pragma unroll
        for (int i = 0; i < kV; ++i) r[k][i] *= rstd1 * t[i];
      }
      if (a.scale) {
        load_w8(t, a.scale, c, a.dim, a.vec, a.w_dtype);
#pragma unroll
        for (int i = 0; i < kV; ++i) r[k][i] *= t[i];
      }
      // Loaded only now: with gate and residual in registers one block of 1024 threads fills an SM (0.28 against 0.20 ms).
      if (a.gate_kind != SF_GATE_NONE) {
        load8<T>(t, static_cast<const T*>(a.gate) + gate_row * a.gate_row, c, a.dim, a.vec);
#pragma unroll
        for (int i = 0; i < kV; ++i) r[k][i] *= gate_act(t[i], a.gate_kind);
      }
      if (a.res) {
        load8<R>(t, static_cast<const R*>(a.res) + row * a.res_row, c, a.dim, a.vec);
#pragma unroll
        for (int i = 0; i < kV; ++i) r[k][i] = fmaf(a.alpha, t[i], r[k][i]);
      }
      if (a.r_out) store8<R>(static_cast<R*>(a.r_out) + row * a.dim, r[k], c, a.dim, a.vec);
      if (c < a.dim)
#pragma unroll
        for (int i = 0; i < kV; ++i) s2[0] = fmaf(r[k][i], r[k][i], s2[0]);
    }
    float rstd2 = 1.f;
    if (a.w_pre) {
      block_sum<1>(s2, buf);
      rstd2 = rsqrtf(s2[0] * inv + a.eps);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (k * blockDim.x + threadIdx.x) * kV;
        float t[kV];
        load_w8(t, a.w_pre, c, a.dim, a.vec, a.w_dtype);
#pragma unroll
        for (int i = 0; i < kV; ++i) t[i] *= r[k][i] * rstd2;
        store8<T>(static_cast<T*>(a.x_out) + row * a.dim, t, c, a.dim, a.vec);
      }
    }
    if (a.rstd && threadIdx.x == 0) {
      a.rstd[row] = rstd1;
      a.rstd[a.rows + row] = rstd2;
    }
  }
}

// Block b of gate group g (block g * blocks + b of the grid): rows g * group_rows + [b * per, (b + 1) * per) of the group.
// The sums over rows of the weights' gradients (and, where one gate row serves many rows, of the gate's) stay in registers.
template <typename T, typename R, int K, int MAXT>
__global__ void __launch_bounds__(MAXT) norm_bwd_kernel(NormArgs a, long long group_rows, long long per,
                                                        unsigned blocks) {
  __shared__ float buf[96];
  const float inv = 1.f / (float)a.dim;
  const long long first = blockIdx.x / blocks * group_rows;
  const long long begin = first + blockIdx.x % blocks * per, end = min(begin + per, first + group_rows);
  const bool shared_gate = a.part_gate != nullptr;
  float Q[K][kV] = {}, gpre[K][kV] = {}, ggate[K][kV] = {};
  for (long long row = begin; row < end; ++row) {
    const float rstd1 = a.w_post ? a.rstd[row] : 1.f, rstd2 = a.w_pre ? a.rstd[a.rows + row] : 0.f;
    float yh[K][kV], rh[K][kV], dt[K][kV], dx[K][kV];
    float s[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * blockDim.x + threadIdx.x) * kV;
      float wpost[kV], g[kV], t[kV];
      load8<T>(yh[k], static_cast<const T*>(a.y) + row * a.y_row, c, a.dim, a.vec);
      load_w8(wpost, a.w_post, c, a.dim, a.vec, a.w_dtype);
      load_w8(g, a.scale, c, a.dim, a.vec, a.w_dtype);
      if (a.gate_kind != SF_GATE_NONE) {
        load8<T>(t, static_cast<const T*>(a.gate) + row / a.rows_per_gate * a.gate_row, c, a.dim, a.vec);
#pragma unroll
        for (int i = 0; i < kV; ++i) g[i] *= gate_act(t[i], a.gate_kind);
      }
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        yh[k][i] *= rstd1;
        rh[k][i] = g[i] * wpost[i] * yh[k][i];  // scale act(gate) u
      }
      if (a.res) {
        load8<R>(t, static_cast<const R*>(a.res) + row * a.res_row, c, a.dim, a.vec);
#pragma unroll
        for (int i = 0; i < kV; ++i) t[i] = fmaf(a.alpha, t[i], rh[k][i]);
      } else {
#pragma unroll
        for (int i = 0; i < kV; ++i) t[i] = rh[k][i];
      }
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        dt[k][i] = 0.f;
        dx[k][i] = 0.f;
      }
      if (a.dr) load8<R>(dt[k], static_cast<const R*>(a.dr) + row * a.dim, c, a.dim, a.vec);
      float wpre[kV];
      load_w8(wpre, a.w_pre, c, a.dim, a.vec, a.w_dtype);
      if (a.dx && a.w_pre) load8<T>(dx[k], static_cast<const T*>(a.dx) + row * a.dim, c, a.dim, a.vec);
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        const float e = rh[k][i];  // w_post G yh
        rh[k][i] = t[i] * rstd2;
        gpre[k][i] = fmaf(dx[k][i], rh[k][i], gpre[k][i]);
        const float q = wpre[i] * dx[k][i];
        s[0] = fmaf(q, rh[k][i], s[0]);
        dt[k][i] = fmaf(rstd2, q, dt[k][i]);
        s[1] = fmaf(e, dt[k][i], s[1]);
        s[2] = fmaf(e, rh[k][i], s[2]);
      }
    }
    block_sum<3>(s, buf);
    const float c2 = s[0] * inv * rstd2, c1 = a.w_post ? (s[1] - c2 * s[2]) * inv : 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * blockDim.x + threadIdx.x) * kV;
      float wpost[kV], sc[kV], z[kV], o[kV], act[kV];
      load_w8(wpost, a.w_post, c, a.dim, a.vec, a.w_dtype);
      load_w8(sc, a.scale, c, a.dim, a.vec, a.w_dtype);
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        act[i] = 1.f;
        dt[k][i] = fmaf(-c2, rh[k][i], dt[k][i]);
      }
      if (a.gate_kind != SF_GATE_NONE) {
        load8<T>(z, static_cast<const T*>(a.gate) + row / a.rows_per_gate * a.gate_row, c, a.dim, a.vec);
#pragma unroll
        for (int i = 0; i < kV; ++i) {
          act[i] = gate_act(z[i], a.gate_kind);
          o[i] = dt[k][i] * sc[i] * wpost[i] * yh[k][i] * gate_dact(z[i], a.gate_kind);
          ggate[k][i] += o[i];
        }
        if (a.dgate && !shared_gate) store8<T>(static_cast<T*>(a.dgate) + row * a.dim, o, c, a.dim, a.vec);
      }
#pragma unroll
      for (int i = 0; i < kV; ++i) {
        const float da = dt[k][i] * act[i], du = da * sc[i];
        Q[k][i] = fmaf(da, yh[k][i], Q[k][i]);
        o[i] = rstd1 * fmaf(wpost[i], du, -yh[k][i] * c1);
      }
      store8<T>(static_cast<T*>(a.dy) + row * a.dim, o, c, a.dim, a.vec);
      if (a.dres) {
#pragma unroll
        for (int i = 0; i < kV; ++i) o[i] = a.alpha * dt[k][i];
        store8<R>(static_cast<R*>(a.dres) + row * a.dim, o, c, a.dim, a.vec);
      }
    }
  }
  const long long block = blockIdx.x;
  float* pw = a.part_w + block * 2 * a.dim;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * blockDim.x + threadIdx.x) * kV;
#pragma unroll
    for (int i = 0; i < kV; ++i)
      if (c + i < a.dim) {
        pw[c + i] = Q[k][i];
        pw[a.dim + c + i] = gpre[k][i];
        if (shared_gate) a.part_gate[block * a.dim + c + i] = ggate[k][i];
      }
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// Kernels with a ring
// ---------------------------------------------------------------------------------------------------------------------

// 8 channels of a row of E: one or two 16-byte words, word h of thread t at [h][t].
template <typename E>
constexpr int kWords = sizeof(E) / 2;
template <typename E>
__device__ __forceinline__ void copy8(float4* slot, const void* base, long long at) {
  const E* p = static_cast<const E*>(base) + at;
#pragma unroll
  for (int h = 0; h < kWords<E>; ++h)
    seq::cp_async(slot + h * blockDim.x + threadIdx.x, p + h * (16 / (int)sizeof(E)), 16, true);
}
template <typename E>
__device__ __forceinline__ void get8(u64 (&o)[4], const float4* slot) {
  float4 w[kWords<E>];
#pragma unroll
  for (int h = 0; h < kWords<E>; ++h) w[h] = slot[h * blockDim.x + threadIdx.x];
  const E* e = reinterpret_cast<const E*>(w);
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = pack2(DT<E>::to_f(e[2 * i]), DT<E>::to_f(e[2 * i + 1]));
}
template <typename E>
__device__ __forceinline__ void put8(void* base, long long at, const u64 (&v)[4]) {
  E e[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float lo, hi;
    unpack2(lo, hi, v[i]);
    e[2 * i] = DT<E>::from_f(lo);
    e[2 * i + 1] = DT<E>::from_f(hi);
  }
  float4* p = reinterpret_cast<float4*>(static_cast<E*>(base) + at);
#pragma unroll
  for (int h = 0; h < kWords<E>; ++h) __stcs(p + h, reinterpret_cast<const float4*>(e)[h]);
}
__device__ __forceinline__ void weights8(u64 (&o)[4], const void* p, int c, const NormArgs& a) {
  float t[kV];
  load_w8(t, p, c, a.dim, a.vec, a.w_dtype);
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = pack2(t[2 * i], t[2 * i + 1]);
}
__device__ __forceinline__ u64 both(float v) { return pack2(v, v); }
// act(gate) of a pair, where sig is what the logistic function gives for it (used for silu and sigmoid), and its derivative.
__device__ __forceinline__ u64 logistic2(u64 g) {
  float lo, hi;
  unpack2(lo, hi, g);
  return pack2(seq::logistic(lo), seq::logistic(hi));
}
template <int KIND>
__device__ __forceinline__ u64 act2(u64 g, u64 sig) {
  return KIND == SF_GATE_SILU ? mul2(g, sig) : KIND == SF_GATE_SIGMOID ? sig : g;
}
template <int KIND>
__device__ __forceinline__ u64 dact2(u64 g, u64 sig) {
  const u64 rest = fma2(sig, both(-1.f), both(1.f));
  return KIND == SF_GATE_SILU ? mul2(sig, fma2(g, rest, both(1.f))) : mul2(sig, rest);
}

// Sums over the block, or over the cluster's blocks that share a row, with one barrier: every warp writes its sums to
// all blocks of the cluster. `buf` alternates between two halves, so the sum before may still be read.
constexpr int kMaxCluster = 4;
template <int N>
using SumBuf = float[16 * kMaxCluster * N];
template <int N>
__device__ __forceinline__ void ring_sum(float (&v)[N], SumBuf<N>* buf, int& half, int cluster) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
  const int warps = blockDim.x >> 5, w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float s[N];
  if (cluster == 1) {
    if (warps == 1) return;
    if (lane == 0)
#pragma unroll
      for (int n = 0; n < N; ++n) buf[half][w * N + n] = v[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) s[n] = lane < warps ? buf[half][lane * N + n] : 0.f;
  } else {
    const auto g = cooperative_groups::this_cluster();
    if (lane < cluster) {
      float* to = g.map_shared_rank(&buf[half][0], lane) + (g.block_rank() * warps + w) * N;
#pragma unroll
      for (int n = 0; n < N; ++n) to[n] = v[n];
    }
    g.sync();
#pragma unroll
    for (int n = 0; n < N; ++n) s[n] = 0.f;
    for (int i = lane; i < cluster * warps; i += 32)
#pragma unroll
      for (int n = 0; n < N; ++n) s[n] += buf[half][i * N + n];
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s[n] += __shfl_xor_sync(0xffffffffu, s[n], o);
    v[n] = s[n];
  }
  half ^= 1;
}
// This block's channels: the first of the thread's eight, and whether they lie in the row. In a cluster, waits until
// all its blocks run, whose shared memory the sums are written to.
__device__ __forceinline__ int ring_channel(const NormArgs& a, bool& own) {
  const int local = threadIdx.x * kV, c = (int)(blockIdx.x % a.cluster) * a.slice + local;
  own = local < a.slice && c < a.dim;
  if (a.cluster > 1) cooperative_groups::this_cluster().sync();
  return c;
}

template <typename T, typename R>
struct FwdRing {
  static constexpr int STAGES = sizeof(T) == 4 ? 2 : 3;
  static constexpr int Y = 0, GATE = kWords<T>, RES = 2 * kWords<T>, WORDS = 2 * kWords<T> + kWords<R>;
};
template <typename T, typename R, int KIND>
__global__ void __launch_bounds__(512, 2) norm_fwd_ring_kernel(NormArgs a) {
  using S = FwdRing<T, R>;
  extern __shared__ __align__(16) float4 ring[];
  const int c = threadIdx.x * kV, n = blockDim.x;
  const bool own = c < a.dim;
  SumBuf<2>* buf = reinterpret_cast<SumBuf<2>*>(ring + S::STAGES * S::WORDS * n);
  const float inv = 1.f / (float)a.dim;
  constexpr bool gated = KIND != SF_GATE_NONE, curved = KIND == SF_GATE_SILU || KIND == SF_GATE_SIGMOID;
  long long ahead = blockIdx.x;
  int put = 0, get = 0, half = 0;
  auto load = [&]() {
    if (ahead < a.rows && own) {
      float4* s = ring + put * S::WORDS * n;
      copy8<T>(s + S::Y * n, a.y, ahead * a.y_row + c);
      if (gated) {
        const long long g = a.rows_per_gate == 1 ? ahead : ahead / a.rows_per_gate;
        copy8<T>(s + S::GATE * n, a.gate, g * a.gate_row + c);
      }
      if (a.res) copy8<R>(s + S::RES * n, a.res, ahead * a.res_row + c);
    }
    seq::cp_async_commit();
    ahead += gridDim.x;
    put = put + 1 == S::STAGES ? 0 : put + 1;
  };
  for (int i = 0; i < S::STAGES - 1; ++i) load();
  u64 ws[4], wpre[4];
  weights8(ws, a.w_post, c, a);
  weights8(wpre, a.scale, c, a);
#pragma unroll
  for (int i = 0; i < 4; ++i) ws[i] = mul2(ws[i], wpre[i]);
  weights8(wpre, a.w_pre, c, a);
  const u64 alpha = both(a.alpha);
  auto squares = [](const u64 (&v)[4]) {
    u64 q = mul2(v[0], v[0]);
#pragma unroll
    for (int i = 1; i < 4; ++i) q = fma2(v[i], v[i], q);
    return seq::sum2(q);
  };
  // One sum over the block for each row serves both norms: that of r' for this row and of y for the next. Its copies
  // have come by then: a row is waited for a turn before its own.
  u64 y[4] = {0, 0, 0, 0};
  float sum[2] = {0.f, 0.f};  // r' of this row, y of the next
  seq::cp_async_wait<S::STAGES - 2>();
  if (own) {
    get8<T>(y, ring + S::Y * n);
    sum[1] = squares(y);
  }
  if (a.w_post) ring_sum<2>(sum, buf, half, 1);
  float rstd1 = a.w_post ? rsqrtf(sum[1] * inv + a.eps) : 1.f;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float4* s = ring + get * S::WORDS * n;
    const long long at = row * a.dim + c;
    u64 r[4] = {0, 0, 0, 0};
    if (own) {
      const u64 k = both(rstd1);
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = mul2(y[i], mul2(k, ws[i]));
      if (gated) {
        u64 g[4];
        get8<T>(g, s + S::GATE * n);
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = mul2(r[i], act2<KIND>(g[i], curved ? logistic2(g[i]) : 0));
      }
      if (a.res) {
        u64 t[4];
        get8<R>(t, s + S::RES * n);
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = fma2(alpha, t[i], r[i]);
      }
      if (a.r_out) put8<R>(a.r_out, at, r);
    }
    get = get + 1 == S::STAGES ? 0 : get + 1;
    load();
    seq::cp_async_wait<S::STAGES - 2>();
    sum[0] = squares(r);
    sum[1] = 0.f;
    if (own) {  // the next row's y; past the last row an earlier one's, which nothing comes of
      get8<T>(y, ring + (get * S::WORDS + S::Y) * n);
      sum[1] = squares(y);
    }
    if (a.w_post || a.w_pre) ring_sum<2>(sum, buf, half, 1);
    const float rstd2 = a.w_pre ? rsqrtf(sum[0] * inv + a.eps) : 1.f;
    if (a.w_pre && own) {
      const u64 k = both(rstd2);
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = mul2(r[i], mul2(k, wpre[i]));
      put8<T>(a.x_out, at, r);
    }
    if (a.rstd && threadIdx.x == 0) {
      a.rstd[row] = rstd1;
      a.rstd[a.rows + row] = rstd2;
    }
    if (a.w_post) rstd1 = rsqrtf(sum[1] * inv + a.eps);
  }
}

template <typename T, typename R>
struct BwdRing {
  static constexpr int STAGES = sizeof(T) == 4 ? 2 : 3;
  static constexpr int Y = 0, GATE = kWords<T>, DX = 2 * kWords<T>, RES = 3 * kWords<T>, DR = RES + kWords<R>;
  static constexpr int WORDS = 3 * kWords<T> + 2 * kWords<R>;
};
// Rows as in norm_bwd_kernel; part_w[block][0]: Q, [1]: dw_pre.
template <typename T, typename R, int KIND>
__global__ void __launch_bounds__(512, 1) norm_bwd_ring_kernel(NormArgs a, long long group_rows, long long per,
                                                              unsigned blocks) {
  using S = BwdRing<T, R>;
  extern __shared__ __align__(16) float4 ring[];
  bool own;
  const int c = ring_channel(a, own), n = blockDim.x;
  SumBuf<3>* buf = reinterpret_cast<SumBuf<3>*>(ring + S::STAGES * S::WORDS * n);
  const float inv = 1.f / (float)a.dim;
  constexpr bool gated = KIND != SF_GATE_NONE, curved = KIND == SF_GATE_SILU || KIND == SF_GATE_SIGMOID;
  const bool shared_gate = a.part_gate != nullptr, pre = a.w_pre && a.dx;
  const unsigned block = blockIdx.x / a.cluster, group = block / blocks;
  const long long first = group * group_rows;
  const long long begin = first + block % blocks * per, end = min(begin + per, first + group_rows);
  long long ahead = begin;
  int put = 0, get = 0, half = 0;
  float next1 = 1.f, next2 = 0.f;
  auto load = [&]() {
    if (ahead < end && own) {
      float4* s = ring + put * S::WORDS * n;
      copy8<T>(s + S::Y * n, a.y, ahead * a.y_row + c);
      // a gate row for many rows: one for the block's group
      if (gated) copy8<T>(s + S::GATE * n, a.gate, (shared_gate ? (long long)group : ahead) * a.gate_row + c);
      if (a.res) copy8<R>(s + S::RES * n, a.res, ahead * a.res_row + c);
      const long long at = ahead * a.dim + c;
      if (pre) copy8<T>(s + S::DX * n, a.dx, at);
      if (a.dr) copy8<R>(s + S::DR * n, a.dr, at);
    }
    seq::cp_async_commit();
    ++ahead;
    put = put + 1 == S::STAGES ? 0 : put + 1;
  };
  auto load_rstd = [&](long long row) {
    if (row >= end) return;
    if (a.w_post) next1 = a.rstd[row];
    if (a.w_pre) next2 = a.rstd[a.rows + row];
  };
  for (int i = 0; i < S::STAGES - 1; ++i) load();
  load_rstd(begin);
  u64 ws[4], wpre[4], Q[4] = {}, gpre[4] = {}, ggate[4] = {};
  weights8(ws, a.w_post, c, a);
  weights8(wpre, a.scale, c, a);
#pragma unroll
  for (int i = 0; i < 4; ++i) ws[i] = mul2(ws[i], wpre[i]);
  weights8(wpre, a.w_pre, c, a);
  const u64 alpha = both(a.alpha);
  for (long long row = begin; row < end; ++row) {
    seq::cp_async_wait<S::STAGES - 2>();
    const float4* s = ring + get * S::WORDS * n;
    const float rstd1 = next1, rstd2 = next2;
    load_rstd(row + 1);
    u64 yh[4], sig[4], rh[4], dt[4], g[4];
    float sum[3] = {0.f, 0.f, 0.f};
    const u64 k1 = both(rstd1), k2 = both(rstd2);
    if (own) {
      get8<T>(yh, s + S::Y * n);
      if (gated) get8<T>(g, s + S::GATE * n);
      u64 dx[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) rh[i] = dt[i] = dx[i] = 0;
      if (a.res) get8<R>(rh, s + S::RES * n);
      if (a.dr) get8<R>(dt, s + S::DR * n);
      if (pre) get8<T>(dx, s + S::DX * n);
      u64 s0 = 0, s1 = 0, s2 = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        yh[i] = mul2(yh[i], k1);
        u64 e = mul2(ws[i], yh[i]);  // scale act(gate) u
        if (curved) sig[i] = logistic2(g[i]);
        if (gated) e = mul2(e, act2<KIND>(g[i], sig[i]));
        rh[i] = mul2(fma2(alpha, rh[i], e), k2);
        gpre[i] = fma2(dx[i], rh[i], gpre[i]);
        const u64 q = mul2(wpre[i], dx[i]);
        s0 = fma2(q, rh[i], s0);
        dt[i] = fma2(k2, q, dt[i]);
        s1 = fma2(e, dt[i], s1);
        s2 = fma2(e, rh[i], s2);
      }
      sum[0] = seq::sum2(s0), sum[1] = seq::sum2(s1), sum[2] = seq::sum2(s2);
    }
    ring_sum<3>(sum, buf, half, a.cluster);
    const float c2 = sum[0] * inv * rstd2, c1 = a.w_post ? (sum[1] - c2 * sum[2]) * inv : 0.f;
    if (own) {
      const u64 m2 = both(-c2), m1 = both(-c1 * rstd1);
      u64 o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        dt[i] = fma2(m2, rh[i], dt[i]);
        const u64 da = gated ? mul2(dt[i], act2<KIND>(g[i], sig[i])) : dt[i];
        Q[i] = fma2(da, yh[i], Q[i]);
        o[i] = fma2(m1, yh[i], mul2(k1, mul2(ws[i], da)));
      }
      const long long at = row * a.dim + c;
      put8<T>(a.dy, at, o);
      if (gated) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          o[i] = mul2(mul2(dt[i], yh[i]), ws[i]);
          if (curved) o[i] = mul2(o[i], dact2<KIND>(g[i], sig[i]));
        }
        if (shared_gate) {
#pragma unroll
          for (int i = 0; i < 4; ++i) ggate[i] = add2(ggate[i], o[i]);
        } else {
          put8<T>(a.dgate, at, o);
        }
      }
      if (a.dres) {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = mul2(alpha, dt[i]);
        put8<R>(a.dres, at, o);
      }
    }
    get = get + 1 == S::STAGES ? 0 : get + 1;
    load();
  }
  if (!own) return;
  put8<float>(a.part_w, 2ll * block * a.dim + c, Q);
  put8<float>(a.part_w, (2ll * block + 1) * a.dim + c, gpre);
  if (shared_gate) put8<float>(a.part_gate, (long long)block * a.dim + c, ggate);
}

// out[g][i] = factor[i] sum over j < blocks of part[g][j][stride] at i, to at most two outputs (a null output is left
// out, a null factor is 1); where blockIdx.y is 1, out2[i] = the sum over j of the n values after those. A block has 32 of
// a group's n values, and each of its 8 warps every eighth j: a fixed order.
__global__ void __launch_bounds__(256) norm_reduce_kernel(const float* part, long long blocks, long long stride, int n,
                                                          int dtype, void* out0, const void* factor0, void* out1,
                                                          const void* factor1, int factor_dtype, void* out2) {
  __shared__ float sums[8][32];
  const unsigned tiles = (n + 31) / 32, g = blockIdx.x / tiles;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i = (int)(blockIdx.x % tiles) * 32 + lane;
  const float* p = part + g * blocks * stride + i;
  if (blockIdx.y == 1) {
    p += n;
    out0 = out2;
    factor0 = nullptr;
    out1 = nullptr;
  }
  float s = 0.f;
  if (i < n) {
#pragma unroll 8
    for (long long j = warp; j < blocks; j += 8) s += p[j * stride];
  }
  sums[warp][lane] = s;
  __syncthreads();
  if (warp != 0 || i >= n) return;
#pragma unroll
  for (int w = 1; w < 8; ++w) s += sums[w][lane];
  const long long o = (long long)g * n + i;
  if (out0) seq::store_param(out0, o, dtype, factor0 ? s * seq::load_param(factor0, i, factor_dtype) : s);
  if (out1) seq::store_param(out1, o, dtype, factor1 ? s * seq::load_param(factor1, i, factor_dtype) : s);
}

bool valid(const sf_block_norm_desc* d) {
  if (!d || d->rows < 0 || d->dim < 1 || d->rows_per_gate < 1) return false;
  if (dtype_size(d->dtype) == 0 || dtype_size(d->res_dtype) == 0 || dtype_size(d->w_dtype) == 0) return false;
  if (d->res_dtype != d->dtype && d->res_dtype != SF_DTYPE_F32) return false;
  if (d->w_dtype != d->dtype && d->w_dtype != SF_DTYPE_F32) return false;
  if (d->gate_kind < SF_GATE_NONE || d->gate_kind > SF_GATE_SIGMOID) return false;
  return d->rows % d->rows_per_gate == 0;
}

bool vectors_fit(const sf_block_norm_desc* d, std::initializer_list<const void*> ptrs) {
  if (d->dim % kV || d->y_row_stride % kV || d->residual_row_stride % kV || d->gate_row_stride % kV) return false;
  for (const void* p : ptrs)
    if (!aligned16(p)) return false;
  return true;
}

// Threads for a row, and vectors per thread.
int vectors_per_thread(int dim) { return dim > 1024 * kV ? 2 : 1; }
int threads_for(int dim, int K) {
  const int t = (dim + kV * K - 1) / (kV * K);
  return (t + 31) / 32 * 32;
}

// Blocks that share a row in the kernels with a ring, as a cluster, and the channels of each.
int cluster_of(int dim) { return dim <= kRingDim ? 1 : dim <= 2 * kRingDim ? 2 : kMaxCluster; }
int slice_of(int dim) {
  const int cl = cluster_of(dim);
  return (dim + cl * kV - 1) / (cl * kV) * kV;
}
// Rows at work at a time that fill the GPU: 512 threads an SM backward (about 126 registers each), 1024 forward.
long long rows_at_work(int dim, int threads_per_sm) {
  const long long rows = (long long)seq::kSms * (threads_per_sm / threads_for(slice_of(dim), 1)) / cluster_of(dim);
  return rows < 1 ? 1 : rows;
}

struct BwdPlan {
  long long groups, group_rows, blocks, per;
  bool shared_gate;
};
BwdPlan bwd_plan(const sf_block_norm_desc* d) {
  BwdPlan p;
  p.shared_gate = d->gate_kind != SF_GATE_NONE && d->rows_per_gate > 1 && d->rows > 0;
  p.groups = p.shared_gate ? d->rows / d->rows_per_gate : 1;
  p.group_rows = p.shared_gate ? d->rows_per_gate : d->rows;
  // Wide rows that no ring takes: blocks of up to 1024 threads, two an SM.
  const long long want = d->dim % kV && d->dim > kRingDim ? 2 * seq::kSms : rows_at_work(d->dim, 512);
  long long blocks = (want + p.groups - 1) / p.groups;
  if (blocks > p.group_rows) blocks = p.group_rows;
  if (blocks < 1) blocks = 1;
  p.per = (p.group_rows + blocks - 1) / blocks;
  p.blocks = p.per > 0 ? (p.group_rows + p.per - 1) / p.per : 1;
  return p;
}

NormArgs base_args(const void* y, const void* residual, const void* gate, const void* w_post, const void* w_pre,
                   const void* scale, const sf_block_norm_desc* d) {
  NormArgs a = {};
  a.y = y;
  a.res = residual;
  a.gate = gate;
  a.w_post = w_post;
  a.w_pre = w_pre;
  a.scale = scale;
  a.rows = d->rows;
  a.y_row = d->y_row_stride;
  a.res_row = d->residual_row_stride;
  a.gate_row = d->gate_row_stride;
  a.rows_per_gate = d->rows_per_gate;
  a.dim = d->dim;
  a.w_dtype = d->w_dtype;
  a.gate_kind = d->gate_kind;
  a.cluster = cluster_of(d->dim);
  a.slice = slice_of(d->dim);
  a.alpha = d->residual_scale;
  a.eps = d->eps;
  return a;
}

// Launches a kernel with a ring on a grid of rows at work, a cluster for each row of several blocks.
template <typename K, typename... Args>
sf_status launch_ring(K kernel, const NormArgs& a, long long rows, size_t words, int sums, cudaStream_t st,
                      Args... args) {
  const int threads = threads_for(a.slice, 1);
  const size_t smem = words * threads * sizeof(float4) + 2 * 16 * kMaxCluster * sums * sizeof(float);
  if (smem > 48 * 1024 && !allow_max_smem(reinterpret_cast<const void*>(kernel))) return SF_ERR_CUDA;
  const dim3 grid((unsigned)(rows * a.cluster));
  if (a.cluster == 1) {
    kernel<<<grid, threads, smem, st>>>(a, args...);
    return cudaGetLastError() == cudaSuccess ? SF_OK : SF_ERR_CUDA;
  }
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = a.cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, a, args...) == cudaSuccess ? SF_OK : SF_ERR_CUDA;
}

template <typename T, typename R>
sf_status run_fwd(const NormArgs& a, cudaStream_t st) {
  // Wider rows: the barrier of a cluster costs more than the ring gives (8192 rows of 8192 channels: 0.24 ms in
  // clusters of two, 0.20 ms without a ring; backward 0.44 against 0.68 ms).
  if (a.vec && a.cluster == 1) {
    using S = FwdRing<T, R>;
    auto kernel = a.gate_kind == SF_GATE_NONE     ? norm_fwd_ring_kernel<T, R, SF_GATE_NONE>
                  : a.gate_kind == SF_GATE_LINEAR ? norm_fwd_ring_kernel<T, R, SF_GATE_LINEAR>
                  : a.gate_kind == SF_GATE_SILU   ? norm_fwd_ring_kernel<T, R, SF_GATE_SILU>
                                                  : norm_fwd_ring_kernel<T, R, SF_GATE_SIGMOID>;
    const long long most = rows_at_work(a.dim, 1024);
    return launch_ring(kernel, a, a.rows < most ? a.rows : most, S::STAGES * S::WORDS, 2, st);
  }
  const int K = vectors_per_thread(a.dim), threads = threads_for(a.dim, K);
  const unsigned grid = (unsigned)(a.rows < INT32_MAX ? a.rows : INT32_MAX);
  if (K == 1) norm_fwd_kernel<T, R, 1><<<grid, threads, 0, st>>>(a);
  else norm_fwd_kernel<T, R, 2><<<grid, threads, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? SF_OK : SF_ERR_CUDA;
}
template <typename T, typename R>
sf_status run_bwd(const NormArgs& a, const BwdPlan& p, cudaStream_t st) {
  const unsigned blocks = (unsigned)p.blocks;
  if (a.vec) {
    using S = BwdRing<T, R>;
    auto kernel = a.gate_kind == SF_GATE_NONE     ? norm_bwd_ring_kernel<T, R, SF_GATE_NONE>
                  : a.gate_kind == SF_GATE_LINEAR ? norm_bwd_ring_kernel<T, R, SF_GATE_LINEAR>
                  : a.gate_kind == SF_GATE_SILU   ? norm_bwd_ring_kernel<T, R, SF_GATE_SILU>
                                                  : norm_bwd_ring_kernel<T, R, SF_GATE_SIGMOID>;
    return launch_ring(kernel, a, p.blocks * p.groups, S::STAGES * S::WORDS, 3, st, p.group_rows, p.per, blocks);
  }
  // The kernel wants about 90 registers with one vector a thread and 160 with two.
  const int K = a.dim > 512 * kV ? 2 : 1, threads = threads_for(a.dim, K);
  const unsigned grid = (unsigned)(p.blocks * p.groups);
  if (K == 1) norm_bwd_kernel<T, R, 1, 512><<<grid, threads, 0, st>>>(a, p.group_rows, p.per, blocks);
  else if (threads <= 512) norm_bwd_kernel<T, R, 2, 512><<<grid, threads, 0, st>>>(a, p.group_rows, p.per, blocks);
  else norm_bwd_kernel<T, R, 2, 1024><<<grid, threads, 0, st>>>(a, p.group_rows, p.per, blocks);
  return cudaGetLastError() == cudaSuccess ? SF_OK : SF_ERR_CUDA;
}

}  // namespace
}  // namespace sf

using namespace sf;

#define SF_NORM_DISPATCH(D, CALL)                                                          \
  do {                                                                                     \
    if ((D)->dtype == SF_DTYPE_F32) { using T = float; using R = float; status = CALL; }   \
    else if ((D)->dtype == SF_DTYPE_F16) {                                                 \
      using T = __half;                                                                    \
      if ((D)->res_dtype == SF_DTYPE_F32) { using R = float; status = CALL; }              \
      else { using R = __half; status = CALL; }                                            \
    } else {                                                                               \
      using T = __nv_bfloat16;                                                             \
      if ((D)->res_dtype == SF_DTYPE_F32) { using R = float; status = CALL; }              \
      else { using R = __nv_bfloat16; status = CALL; }                                     \
    }                                                                                      \
  } while (0)

extern "C" sf_status sf_block_norm(const void* y, const void* residual, const void* gate, const void* post_weight,
                                   const void* pre_weight, const void* scale, void* residual_out, void* normed,
                                   float* rstd, const sf_block_norm_desc* d, void* stream) {
  if (!valid(d)) return SF_ERR_INVALID_ARG;
  if (d->dim > kMaxDim) return SF_ERR_UNSUPPORTED;
  if (d->rows == 0) return SF_OK;
  if (!y || (!residual_out && !normed) || (normed && !pre_weight)) return SF_ERR_INVALID_ARG;
  if ((d->gate_kind != SF_GATE_NONE) != (gate != nullptr)) return SF_ERR_INVALID_ARG;
  NormArgs a = base_args(y, residual, gate, post_weight, normed ? pre_weight : nullptr, scale, d);
  a.r_out = residual_out;
  a.x_out = normed;
  a.rstd = rstd;
  a.vec = vectors_fit(d, {y, residual, gate, post_weight, pre_weight, scale, residual_out, normed});
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  sf_status status;
  SF_NORM_DISPATCH(d, (run_fwd<T, R>(a, st)));
  return status;
}

extern "C" size_t sf_block_norm_backward_workspace_size(const sf_block_norm_desc* d) {
  if (!valid(d) || d->dim > kMaxDim) return 0;
  const BwdPlan p = bwd_plan(d);
  return (size_t)(p.blocks * p.groups) * d->dim * (p.shared_gate ? 3 : 2) * sizeof(float);
}

extern "C" sf_status sf_block_norm_backward(const void* y, const void* residual, const void* gate,
                                            const void* post_weight, const void* pre_weight, const void* scale,
                                            const float* rstd, const void* d_residual_out, const void* d_normed,
                                            void* dy, void* d_residual, void* d_gate, void* d_post_weight,
                                            void* d_pre_weight, void* d_scale, const sf_block_norm_desc* d,
                                            void* workspace, size_t workspace_bytes, void* stream) {
  if (!valid(d)) return SF_ERR_INVALID_ARG;
  if (d->dim > kMaxDim) return SF_ERR_UNSUPPORTED;
  if (d->rows > 0 && (!y || !rstd || !dy)) return SF_ERR_INVALID_ARG;
  if ((d->gate_kind != SF_GATE_NONE) != (gate != nullptr) && d->rows > 0) return SF_ERR_INVALID_ARG;
  if (d->rows > 0 && (!workspace || workspace_bytes < sf_block_norm_backward_workspace_size(d)))
    return SF_ERR_WORKSPACE;
  if (d->rows > 0 && !aligned16(workspace)) return SF_ERR_ALIGNMENT;
  const BwdPlan p = bwd_plan(d);
  const unsigned tiles = (d->dim + 31) / 32;  // of the sums over blocks
  if (p.blocks * p.groups > INT32_MAX / kMaxCluster || p.groups > INT32_MAX / tiles) return SF_ERR_UNSUPPORTED;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const long long blocks = d->rows > 0 ? p.blocks * p.groups : 0;
  float* part = static_cast<float*>(workspace);
  NormArgs a = base_args(y, residual, gate, post_weight, pre_weight, scale, d);
  a.rstd = const_cast<float*>(rstd);
  a.dr = d_residual_out;
  a.dx = d_normed;
  a.dy = dy;
  a.dres = d_residual;
  a.dgate = d_gate;
  a.part_w = part;
  a.part_gate = p.shared_gate ? part + blocks * 2 * d->dim : nullptr;
  a.vec = vectors_fit(d, {y, residual, gate, post_weight, pre_weight, scale, d_residual_out, d_normed, dy, d_residual,
                          p.shared_gate ? nullptr : d_gate});
  if (d->rows > 0) {
    sf_status status;
    SF_NORM_DISPATCH(d, (run_bwd<T, R>(a, p, st)));
    if (status != SF_OK) return status;
  }
  if (d_post_weight || d_scale || d_pre_weight)
    norm_reduce_kernel<<<dim3(tiles, 2), 256, 0, st>>>(part, blocks, 2ll * d->dim, d->dim, d->w_dtype, d_post_weight,
                                                         scale, d_scale, post_weight, d->w_dtype, d_pre_weight);
  if (p.shared_gate && d_gate && d->rows > 0)
    norm_reduce_kernel<<<tiles * (unsigned)p.groups, 256, 0, st>>>(a.part_gate, p.blocks, d->dim, d->dim, d->dtype,
                                                                       d_gate, nullptr, nullptr, nullptr, d->w_dtype, nullptr);
  return cudaGetLastError() == cudaSuccess ? SF_OK : SF_ERR_CUDA;
}
