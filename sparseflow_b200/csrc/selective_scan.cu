// Selective state space scan: a learned linear recurrence along a sequence,
//
//   a_t = exp(dt_t A),  h_t = a_t h_(t-1) + dt_t x_t B_t,  p_t = C_t . h_t + D x_t,  y_t = p_t silu(z_t)
//
// for every channel d and state n (A [dim, state]; B_t, C_t shared by the channels of a group), its backward pass
// and its single-token form. Backward, with gp = dy silu(z):
//   gh_t = gp_t C_t + a_(t+1) gh_(t+1);  gC_t = sum_d gp h;  gB_t = sum_d gh dt x;  S = sum_n gh B
//   gx = dt S + D gp;  q = gh h_(t-1) a_t;  gdt = x S + sum_n q A;  gA = sum_t q dt;  gD = sum gp x
//   gz = dy p silu'(z);  gdt_raw = gdt softplus'(dt_raw + bias);  gbias = sum gdt_raw;  gh0 = a_1 gh_1
//
// A thread owns 4 states of one channel; the LPC = ceil(state / 4) (a power of two) lanes of a channel lie next to
// each other and add up C . h by shuffles. States past `state` have A = B = C = 0 and stay 0.
#include "sequence.cuh"

namespace sf {
namespace {

using seq::Rows;
using seq::Span;

constexpr int kThreads = 128;
constexpr int kS = 4;       // states per lane
constexpr int kMaxState = 128;
constexpr int kChunk = 16;  // rows per checkpoint, and per staged tile
constexpr float kLog2e = 1.4426950408889634f;

struct ScanArgs {
  const void *x, *dt, *B, *C, *z, *dy;
  const float *A, *D, *dt_bias, *init, *dfinal, *ck;
  void *y, *dx, *ddt, *dz;
  float *final_state, *ck_out, *dinit;
  float *part_bc, *part_a, *part_d;  // backward partial sums
  Rows rows;
  long long x_batch, x_row, dt_batch, dt_row, z_batch, z_row, b_batch, b_row, c_batch, c_row;
  int dim, state, groups, softplus;
};

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

template <typename T>
__device__ __forceinline__ const T* at(const void* p, const ScanArgs& a, const Span& s, long long batch,
                                       long long row) {
  return static_cast<const T*>(p) + (a.rows.offsets ? s.begin * row : (long long)s.s * batch);
}
__device__ __forceinline__ long long row0(const ScanArgs& a, const Span& s) {
  return a.rows.offsets ? s.begin : (long long)s.s * a.rows.length;
}

// Four values of a [.., state] row of floats from state n on, 0 past the end.
__device__ __forceinline__ void load4(float (&o)[kS], const float* p, int n, int state) {
#pragma unroll
  for (int i = 0; i < kS; ++i) o[i] = n + i < state ? p[n + i] : 0.f;
}
__device__ __forceinline__ void store4(float* p, const float (&v)[kS], int n, int state) {
#pragma unroll
  for (int i = 0; i < kS; ++i)
    if (n + i < state) p[n + i] = v[i];
}

template <int LPC>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = LPC / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One block: one sequence and kThreads / LPC channels of one group.
template <typename T, int LPC>
__global__ void __launch_bounds__(kThreads) scan_fwd_kernel(ScanArgs a) {
  constexpr int CH = kThreads / LPC, NP = LPC * kS;
  __shared__ float sB[kChunk][NP], sC[kChunk][NP];
  __shared__ float sx[kChunk][CH], sdt[kChunk][CH], sz[kChunk][CH];
  const int per = a.dim / a.groups, tiles = (per + CH - 1) / CH;
  const int g = blockIdx.x / tiles, d0 = g * per + (blockIdx.x % tiles) * CH, dend = (g + 1) * per;
  const Span p = seq::seq_span(a.rows, blockIdx.y, kChunk);
  const int q = threadIdx.x % LPC, c = threadIdx.x / LPC, d = d0 + c, n = q * kS;
  const bool own = d < dend;
  const T* xs = at<T>(a.x, a, p, a.x_batch, a.x_row);
  const T* dts = at<T>(a.dt, a, p, a.dt_batch, a.dt_row);
  const T* zs = a.z ? at<T>(a.z, a, p, a.z_batch, a.z_row) : nullptr;
  const T* Bs = at<T>(a.B, a, p, a.b_batch, a.b_row) + (long long)g * a.state;
  const T* Cs = at<T>(a.C, a, p, a.c_batch, a.c_row) + (long long)g * a.state;
  T* ys = static_cast<T*>(a.y) + row0(a, p) * a.dim;

  float A2[kS] = {}, h[kS] = {};
  float D = 0.f;
  if (own) {
    load4(A2, a.A + (long long)d * a.state, n, a.state);
#pragma unroll
    for (int i = 0; i < kS; ++i) A2[i] *= kLog2e;
    if (a.init) load4(h, a.init + ((long long)p.s * a.dim + d) * a.state, n, a.state);
    if (a.D) D = a.D[d];
  }
  for (long long t0 = 0; t0 < p.len; t0 += kChunk) {
    const int rows = (int)min((long long)kChunk, p.len - t0);
    if (a.ck_out && own)
      store4(a.ck_out + ((p.slot0 + t0 / kChunk) * a.dim + d) * a.state, h, n, a.state);
    __syncthreads();
    for (int i = threadIdx.x; i < rows * NP; i += kThreads) {
      const int r = i / NP, m = i % NP;
      sB[r][m] = m < a.state ? DT<T>::to_f(Bs[(t0 + r) * a.b_row + m]) : 0.f;
      sC[r][m] = m < a.state ? DT<T>::to_f(Cs[(t0 + r) * a.c_row + m]) : 0.f;
    }
    for (int i = threadIdx.x; i < rows * CH; i += kThreads) {
      const int r = i / CH, m = i % CH;
      if (d0 + m < dend) {
        sx[r][m] = DT<T>::to_f(xs[(t0 + r) * a.x_row + d0 + m]);
        float v = DT<T>::to_f(dts[(t0 + r) * a.dt_row + d0 + m]);
        if (a.dt_bias) v += a.dt_bias[d0 + m];
        sdt[r][m] = a.softplus ? seq::softplus(v) : v;
        sz[r][m] = zs ? DT<T>::to_f(zs[(t0 + r) * a.z_row + d0 + m]) : 0.f;
      } else {
        sx[r][m] = sdt[r][m] = sz[r][m] = 0.f;
      }
    }
    __syncthreads();
    for (int r = 0; r < rows; ++r) {
      const float dt = sdt[r][c], x = sx[r][c], u = dt * x;
      float y = 0.f;
#pragma unroll
      for (int i = 0; i < kS; ++i) {
        h[i] = fmaf(ex2(dt * A2[i]), h[i], u * sB[r][n + i]);
        y = fmaf(sC[r][n + i], h[i], y);
      }
      y = lanes_sum<LPC>(y);
      if (q == 0 && own) {
        y = fmaf(D, x, y);
        if (zs) y *= seq::silu(sz[r][c]);
        ys[(t0 + r) * a.dim + d] = DT<T>::from_f(y);
      }
    }
  }
  if (a.final_state && own) store4(a.final_state + ((long long)p.s * a.dim + d) * a.state, h, n, a.state);
}

// Chunks of kChunk rows from the last to the first: the states of a chunk from its checkpoint, then its rows
// backwards. Sums over channels of a chunk's gB and gC go to part_bc[tile][row][2][group, NP] and are added over the tiles by
// scan_bc_reduce_kernel; sums over a sequence of gA, gD and gbias to part_a / part_d, added over the sequences.
template <typename T, int LPC>
__global__ void __launch_bounds__(kThreads) scan_bwd_kernel(ScanArgs a) {
  constexpr int CH = kThreads / LPC, NP = LPC * kS, CW = 32 / LPC, WARPS = kThreads / 32;
  __shared__ float sB[kChunk][NP], sC[kChunk][NP];
  __shared__ float sx[kChunk][CH], sdt[kChunk][CH], sz[kChunk][CH], sg[kChunk][CH], sraw[kChunk][CH];
  __shared__ float sgbc[WARPS][2][NP];
  const int per = a.dim / a.groups, tiles = (per + CH - 1) / CH;
  const int g = blockIdx.x / tiles, tile = blockIdx.x % tiles, d0 = g * per + tile * CH, dend = (g + 1) * per;
  const Span p = seq::seq_span(a.rows, blockIdx.y, kChunk);
  const int q = threadIdx.x % LPC, c = threadIdx.x / LPC, d = d0 + c, n = q * kS;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool own = d < dend;
  const T* xs = at<T>(a.x, a, p, a.x_batch, a.x_row);
  const T* dts = at<T>(a.dt, a, p, a.dt_batch, a.dt_row);
  const T* zs = a.z ? at<T>(a.z, a, p, a.z_batch, a.z_row) : nullptr;
  const T* Bs = at<T>(a.B, a, p, a.b_batch, a.b_row) + (long long)g * a.state;
  const T* Cs = at<T>(a.C, a, p, a.c_batch, a.c_row) + (long long)g * a.state;
  const long long r00 = row0(a, p);
  const T* dys = static_cast<const T*>(a.dy) + r00 * a.dim;
  T* dxs = static_cast<T*>(a.dx) + r00 * a.dim;
  T* ddts = static_cast<T*>(a.ddt) + r00 * a.dim;
  T* dzs = a.dz ? static_cast<T*>(a.dz) + r00 * a.dim : nullptr;
  const long long total_rows = a.rows.offsets ? a.rows.length : a.rows.length * a.rows.n_seq;

  float A[kS] = {}, gh[kS] = {}, gA[kS] = {};
  float D = 0.f, gD = 0.f, gbias = 0.f;
  if (own) {
    load4(A, a.A + (long long)d * a.state, n, a.state);
    if (a.dfinal) load4(gh, a.dfinal + ((long long)p.s * a.dim + d) * a.state, n, a.state);
    if (a.D) D = a.D[d];
  }
  const long long chunks = (p.len + kChunk - 1) / kChunk;
  for (long long ch = chunks - 1; ch >= 0; --ch) {
    const long long t0 = ch * kChunk;
    const int rows = (int)min((long long)kChunk, p.len - t0);
    __syncthreads();
    for (int i = threadIdx.x; i < kChunk * NP; i += kThreads) {
      const int r = i / NP, m = i % NP;
      const bool in = r < rows && m < a.state;
      sB[r][m] = in ? DT<T>::to_f(Bs[(t0 + r) * a.b_row + m]) : 0.f;
      sC[r][m] = in ? DT<T>::to_f(Cs[(t0 + r) * a.c_row + m]) : 0.f;
    }
    // Rows past the end have dt = x = dy = 0: they change nothing.
    for (int i = threadIdx.x; i < kChunk * CH; i += kThreads) {
      const int r = i / CH, m = i % CH;
      float x = 0.f, dt = 0.f, raw = 0.f, z = 0.f, gy = 0.f;
      if (r < rows && d0 + m < dend) {
        x = DT<T>::to_f(xs[(t0 + r) * a.x_row + d0 + m]);
        raw = DT<T>::to_f(dts[(t0 + r) * a.dt_row + d0 + m]);
        if (a.dt_bias) raw += a.dt_bias[d0 + m];
        dt = a.softplus ? seq::softplus(raw) : raw;
        if (zs) z = DT<T>::to_f(zs[(t0 + r) * a.z_row + d0 + m]);
        gy = DT<T>::to_f(dys[(t0 + r) * a.dim + d0 + m]);
      }
      sx[r][m] = x;
      sdt[r][m] = dt;
      sraw[r][m] = raw;
      sz[r][m] = z;
      sg[r][m] = gy;
    }
    __syncthreads();
    float hs[kChunk + 1][kS] = {};
    if (own) load4(hs[0], a.ck + ((p.slot0 + ch) * a.dim + d) * a.state, n, a.state);
#pragma unroll
    for (int r = 0; r < kChunk; ++r) {
      const float dt = sdt[r][c], u = dt * sx[r][c];
#pragma unroll
      for (int i = 0; i < kS; ++i) hs[r + 1][i] = fmaf(ex2(dt * (A[i] * kLog2e)), hs[r][i], u * sB[r][n + i]);
    }
#pragma unroll
    for (int r = kChunk - 1; r >= 0; --r) {
      if (r >= rows) continue;
      const float dt = sdt[r][c], x = sx[r][c], u = dt * x, gy = sg[r][c];
      float pre = 0.f;
#pragma unroll
      for (int i = 0; i < kS; ++i) pre = fmaf(sC[r][n + i], hs[r + 1][i], pre);
      pre = fmaf(D, x, lanes_sum<LPC>(pre));
      float gp = gy, gz = 0.f;
      if (zs) {
        gp *= seq::silu(sz[r][c]);
        gz = gy * pre * seq::dsilu(sz[r][c]);
      }
      float S = 0.f, qa = 0.f, vb[kS], vc[kS];
#pragma unroll
      for (int i = 0; i < kS; ++i) {
        gh[i] = fmaf(gp, sC[r][n + i], gh[i]);
        vc[i] = gp * hs[r + 1][i];
        vb[i] = gh[i] * u;
        S = fmaf(gh[i], sB[r][n + i], S);
        gh[i] *= ex2(dt * (A[i] * kLog2e));
        const float k = gh[i] * hs[r][i];
        qa = fmaf(k, A[i], qa);
        gA[i] = fmaf(k, dt, gA[i]);
      }
      S = lanes_sum<LPC>(S);
      qa = lanes_sum<LPC>(qa);
      float gdt = fmaf(x, S, qa);
      if (a.softplus) gdt *= seq::sigmoid(sraw[r][c]);
      gD = fmaf(gp, x, gD);
      gbias += gdt;
      if (q == 0 && own) {
        const long long o = (t0 + r) * a.dim + d;
        dxs[o] = DT<T>::from_f(fmaf(dt, S, D * gp));
        ddts[o] = DT<T>::from_f(gdt);
        if (dzs) dzs[o] = DT<T>::from_f(gz);
      }
#pragma unroll
      for (int i = 0; i < kS; ++i)
#pragma unroll
        for (int o = 16; o >= LPC; o >>= 1) {
          vb[i] += __shfl_xor_sync(0xffffffffu, vb[i], o);
          vc[i] += __shfl_xor_sync(0xffffffffu, vc[i], o);
        }
      __syncthreads();
      if (lane < LPC)
#pragma unroll
        for (int i = 0; i < kS; ++i) {
          sgbc[warp][0][n + i] = vb[i];
          sgbc[warp][1][n + i] = vc[i];
        }
      __syncthreads();
      for (int i = threadIdx.x; i < 2 * NP; i += kThreads) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) s += sgbc[w][i / NP][i % NP];
        a.part_bc[(((long long)tile * total_rows + r00 + t0 + r) * 2 * a.groups + (i / NP) * a.groups + g) * NP + i % NP] = s;
      }
    }
  }
  if (!own) return;
  const long long sd = (long long)p.s * a.dim + d;
  if (a.dinit) store4(a.dinit + sd * a.state, gh, n, a.state);
  store4(a.part_a + sd * a.state, gA, n, a.state);
  if (q == 0) {
    a.part_d[sd] = gD;
    a.part_d[(long long)a.rows.n_seq * a.dim + sd] = gbias;
  }
  (void)CW;
}

// dB, dC [rows, groups, state] from part_bc[tiles][rows][2][groups][NP].
template <typename T>
__global__ void scan_bc_reduce_kernel(const float* part, long long rows, int tiles, int groups, int NP, int state,
                                      T* dB, T* dC) {
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const long long per_row = 2ll * groups * NP;
  if (i >= rows * per_row) return;
  float s = 0.f;
  for (int j = 0; j < tiles; ++j) s += part[j * rows * per_row + i];
  const int m = (int)(i % NP), which = (int)(i / ((long long)groups * NP) % 2), g = (int)(i / NP % groups);
  if (m < state) (which ? dC : dB)[(i / per_row * groups + g) * state + m] = DT<T>::from_f(s);
}

// out[i] = sum over j < count of part[j * n + i], in order.
__global__ void scan_sum_kernel(const float* part, int count, long long n, float* out) {
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  float s = 0.f;
  for (int j = 0; j < count; ++j) s += part[j * n + i];
  out[i] = s;
}

template <typename T, int LPC>
__global__ void __launch_bounds__(kThreads) scan_update_kernel(ScanArgs a, float* pool, const int32_t* idx,
                                                               int n_slots) {
  constexpr int CH = kThreads / LPC;
  const int row = blockIdx.x, q = threadIdx.x % LPC, n = q * kS;
  const int d = blockIdx.y * CH + threadIdx.x / LPC;
  const int slot = idx ? idx[row] : row;
  const bool own = d < a.dim, live = own && slot >= 0 && slot < n_slots;
  float y = 0.f;
  if (live) {
    const int g = d / (a.dim / a.groups);
    float dt = DT<T>::to_f(static_cast<const T*>(a.dt)[(long long)row * a.dt_row + d]);
    if (a.dt_bias) dt += a.dt_bias[d];
    if (a.softplus) dt = seq::softplus(dt);
    const float x = DT<T>::to_f(static_cast<const T*>(a.x)[(long long)row * a.x_row + d]);
    const T* Bp = static_cast<const T*>(a.B) + (long long)row * a.b_row + (long long)g * a.state;
    const T* Cp = static_cast<const T*>(a.C) + (long long)row * a.c_row + (long long)g * a.state;
    float A[kS], h[kS];
    float* hp = pool + ((long long)slot * a.dim + d) * a.state;
    load4(A, a.A + (long long)d * a.state, n, a.state);
    load4(h, hp, n, a.state);
#pragma unroll
    for (int i = 0; i < kS; ++i)
      if (n + i < a.state) {
        h[i] = fmaf(ex2(dt * (A[i] * kLog2e)), h[i], dt * x * DT<T>::to_f(Bp[n + i]));
        y = fmaf(DT<T>::to_f(Cp[n + i]), h[i], y);
      }
    store4(hp, h, n, a.state);
  }
  y = lanes_sum<LPC>(y);
  if (q == 0 && own) {
    if (live) {
      if (a.D) y = fmaf(a.D[d], DT<T>::to_f(static_cast<const T*>(a.x)[(long long)row * a.x_row + d]), y);
      if (a.z) y *= seq::silu(DT<T>::to_f(static_cast<const T*>(a.z)[(long long)row * a.z_row + d]));
    }
    static_cast<T*>(a.y)[(long long)row * a.dim + d] = DT<T>::from_f(y);
  }
}

bool valid(const sf_selective_scan_desc* d) {
  return d && d->length >= 0 && d->n_seq >= 0 && d->dim >= 0 && d->state >= 1 && d->groups >= 1 &&
         d->dim % d->groups == 0 && dtype_size(d->dtype) != 0;
}
int lanes(int state) {
  int l = 1;
  while (l * kS < state) l *= 2;
  return l;
}
int tiles_of(const sf_selective_scan_desc* d) {
  const int ch = kThreads / lanes(d->state), per = d->dim / d->groups;
  return (per + ch - 1) / ch;
}
long long rows_of(const sf_selective_scan_desc* d) {
  return d->n_seq == 0 ? 0 : (d->packed ? d->length : d->length * d->n_seq);
}

ScanArgs base_args(const void* x, const void* dt, const float* A, const void* B, const void* C, const float* D,
                   const void* z, const float* dt_bias, const int32_t* offsets, const sf_selective_scan_desc* d) {
  ScanArgs a = {};
  a.x = x;
  a.dt = dt;
  a.A = A;
  a.B = B;
  a.C = C;
  a.D = D;
  a.z = z;
  a.dt_bias = dt_bias;
  a.rows = Rows{offsets, d->length, d->n_seq};
  a.x_batch = d->x_batch_stride;
  a.x_row = d->x_row_stride;
  a.dt_batch = d->dt_batch_stride;
  a.dt_row = d->dt_row_stride;
  a.z_batch = d->z_batch_stride;
  a.z_row = d->z_row_stride;
  a.b_batch = d->b_batch_stride;
  a.b_row = d->b_row_stride;
  a.c_batch = d->c_batch_stride;
  a.c_row = d->c_row_stride;
  a.dim = d->dim;
  a.state = d->state;
  a.groups = d->groups;
  a.softplus = d->dt_softplus;
  return a;
}

struct BwdLayout {  // floats
  long long bc, a, d, total;
};
BwdLayout bwd_layout(const sf_selective_scan_desc* d, long long rows) {
  BwdLayout l;
  const long long np = (long long)lanes(d->state) * kS;
  l.bc = 0;
  l.a = (tiles_of(d) * rows * 2 * d->groups * np + 3) / 4 * 4;
  l.d = l.a + (long long)d->n_seq * d->dim * d->state;
  l.total = l.d + 2ll * d->n_seq * d->dim;
  return l;
}

}  // namespace
}  // namespace sf

using namespace sf;

#define SF_SCAN_LANES(STATE, CALL)                        \
  switch (lanes(STATE)) {                                 \
    case 1: { constexpr int L = 1; CALL; break; }         \
    case 2: { constexpr int L = 2; CALL; break; }         \
    case 4: { constexpr int L = 4; CALL; break; }         \
    case 8: { constexpr int L = 8; CALL; break; }         \
    case 16: { constexpr int L = 16; CALL; break; }       \
    default: { constexpr int L = 32; CALL; break; }       \
  }
#define SF_SCAN_TYPES(DTYPE, CALL)                                  \
  switch (DTYPE) {                                                  \
    case SF_DTYPE_F32: { using T = float; CALL; break; }            \
    case SF_DTYPE_F16: { using T = __half; CALL; break; }           \
    default: { using T = __nv_bfloat16; CALL; break; }              \
  }

extern "C" size_t sf_selective_scan_checkpoint_bytes(const sf_selective_scan_desc* d) {
  if (!valid(d)) return 0;
  return (size_t)seq::total_slots(d->length, d->n_seq, d->packed, kChunk) * d->dim * d->state * sizeof(float);
}

extern "C" size_t sf_selective_scan_workspace_size(const sf_selective_scan_desc*) { return 0; }

extern "C" sf_status sf_selective_scan(const void* x, const void* dt, const float* A, const void* B, const void* C,
                                       const float* D, const void* z, const float* dt_bias,
                                       const float* initial_state, const int32_t* seq_offsets, void* y,
                                       float* final_state, void* checkpoints, const sf_selective_scan_desc* d,
                                       void* workspace, size_t workspace_bytes, void* stream) {
  (void)workspace;
  (void)workspace_bytes;
  if (!valid(d) || !A || (seq_offsets != nullptr) != (d->packed != 0)) return SF_ERR_INVALID_ARG;
  if (d->state > kMaxState || d->n_seq > 65535) return SF_ERR_UNSUPPORTED;
  if (d->n_seq == 0 || d->dim == 0) return SF_OK;
  if (d->length > 0 && (!x || !dt || !B || !C || !y)) return SF_ERR_INVALID_ARG;
  ScanArgs a = base_args(x, dt, A, B, C, D, z, dt_bias, seq_offsets, d);
  a.init = initial_state;
  a.y = y;
  a.final_state = final_state;
  a.ck_out = static_cast<float*>(checkpoints);
  const dim3 grid(tiles_of(d) * d->groups, d->n_seq);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  SF_SCAN_TYPES(d->dtype, SF_SCAN_LANES(d->state, (scan_fwd_kernel<T, L><<<grid, kThreads, 0, st>>>(a))))
  return cudaGetLastError() == cudaSuccess ? SF_OK : SF_ERR_CUDA;
}

extern "C" size_t sf_selective_scan_backward_workspace_size(const sf_selective_scan_desc* d) {
  if (!valid(d)) return 0;
  return (size_t)bwd_layout(d, rows_of(d)).total * sizeof(float);
}

extern "C" sf_status sf_selective_scan_backward(const void* x, const void* dt, const float* A, const void* B,
                                                const void* C, const float* D, const void* z, const float* dt_bias,
                                                const int32_t* seq_offsets, const void* checkpoints, const void* dy,
                                                const float* d_final_state, void* dx, void* ddt, float* dA, void* dB,
                                                void* dC, float* dD, void* dz, float* d_dt_bias,
                                                float* d_initial_state, const sf_selective_scan_desc* d,
                                                void* workspace, size_t workspace_bytes, void* stream) {
  if (!valid(d) || !A || !dA || (d->n_seq > 0 && (seq_offsets != nullptr) != (d->packed != 0)))
    return SF_ERR_INVALID_ARG;
  if (d->state > kMaxState || d->n_seq > 65535) return SF_ERR_UNSUPPORTED;
  if (d->dim == 0) return SF_OK;
  const bool some = d->n_seq > 0;
  const long long rows = rows_of(d);
  if (rows > 0 && (!x || !dt || !B || !C || !checkpoints || !dy || !dx || !ddt || !dB || !dC))
    return SF_ERR_INVALID_ARG;
  if ((z && rows > 0 && !dz) || (D && !dD) || (dt_bias && !d_dt_bias)) return SF_ERR_INVALID_ARG;
  const BwdLayout l = bwd_layout(d, rows);
  if (some && (!workspace || workspace_bytes < (size_t)l.total * sizeof(float))) return SF_ERR_WORKSPACE;
  if (some && !aligned16(workspace)) return SF_ERR_ALIGNMENT;
  float* ws = static_cast<float*>(workspace);
  ScanArgs a = base_args(x, dt, A, B, C, D, z, dt_bias, seq_offsets, d);
  a.ck = static_cast<const float*>(checkpoints);
  a.dy = dy;
  a.dfinal = d_final_state;
  a.dx = dx;
  a.ddt = ddt;
  a.dz = z ? dz : nullptr;
  a.dinit = d_initial_state;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (some) {
    a.part_bc = ws + l.bc;
    a.part_a = ws + l.a;
    a.part_d = ws + l.d;
    const dim3 grid(tiles_of(d) * d->groups, d->n_seq);
    SF_SCAN_TYPES(d->dtype, SF_SCAN_LANES(d->state, (scan_bwd_kernel<T, L><<<grid, kThreads, 0, st>>>(a))))
    if (rows > 0) {
      const int np = lanes(d->state) * kS;
      const long long n = rows * 2 * d->groups * np;
      SF_SCAN_TYPES(d->dtype, (scan_bc_reduce_kernel<T><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(
                                  a.part_bc, rows, tiles_of(d), d->groups, np, d->state, static_cast<T*>(dB),
                                  static_cast<T*>(dC))))
    }
  }
  const long long na = (long long)d->dim * d->state, nd = d->dim;
  scan_sum_kernel<<<(unsigned)((na + 255) / 256), 256, 0, st>>>(a.part_a, d->n_seq, na, dA);
  const unsigned gd = (unsigned)((nd + 255) / 256);
  if (dD) scan_sum_kernel<<<gd, 256, 0, st>>>(a.part_d, d->n_seq, nd, dD);
  if (d_dt_bias)
    scan_sum_kernel<<<gd, 256, 0, st>>>(some ? a.part_d + (long long)d->n_seq * nd : nullptr, d->n_seq, nd, d_dt_bias);
  return cudaGetLastError() == cudaSuccess ? SF_OK : SF_ERR_CUDA;
}

extern "C" sf_status sf_selective_scan_update(const void* x, const void* dt, const float* A, const void* B,
                                              const void* C, const float* D, const void* z, const float* dt_bias,
                                              float* state_pool, const int32_t* state_indices, void* y,
                                              int32_t n_slots, const sf_selective_scan_desc* d, void* stream) {
  if (!valid(d) || !A || n_slots < 0) return SF_ERR_INVALID_ARG;
  if (d->state > kMaxState) return SF_ERR_UNSUPPORTED;
  if (d->n_seq == 0 || d->dim == 0) return SF_OK;
  if (!x || !dt || !B || !C || !y || !state_pool) return SF_ERR_INVALID_ARG;
  ScanArgs a = base_args(x, dt, A, B, C, D, z, dt_bias, nullptr, d);
  a.y = y;
  const int ch = kThreads / lanes(d->state);
  const dim3 grid(d->n_seq, (d->dim + ch - 1) / ch);
  if (grid.y > 65535) return SF_ERR_UNSUPPORTED;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  SF_SCAN_TYPES(d->dtype, SF_SCAN_LANES(d->state, (scan_update_kernel<T, L><<<grid, kThreads, 0, st>>>(
                                                      a, state_pool, state_indices, n_slots))))
  return cudaGetLastError() == cudaSuccess ? SF_OK : SF_ERR_CUDA;
}
