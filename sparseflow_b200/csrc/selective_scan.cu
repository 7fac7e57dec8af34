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
// What bounds it: one exponential a state and row (16 a cycle and SM: 4.5e12/s) against 8 bytes a channel and row,
// so with 16 states the exponentials take three times as long as the bytes. Next come issue slots: fp32 pairs
// (mul/fma .f32x2) halve the multiply-adds, and everything that is per channel and row, not per state (softplus,
// the gate, D x), is done once, by the thread that loads the element, and handed on through shared memory.
//
// Layout: a lane owns 4 states of one channel; the LPC = ceil(state / 4) (a power of two) lanes of a channel lie
// next to each other. A block takes CH = 64 channels of one group (fewer above 16 states) through a segment of the
// rows, 16 rows a tile; tile t+1 is on its way to registers while tile t is worked on. Sums over the states end in
// a reduce-scatter over four rows and the lanes of a channel, so each lane finishes other rows.
// States past `state` have A = B = C = 0 and stay 0; rows past the end have dt = x = 0 and change nothing.
//
// Few channels and long sequences leave most of the GPU idle, so sequences are cut into segments: a first kernel
// finds what each segment adds to a state of 0 and how much it decays one (exp(A sum dt)), and the second starts
// each segment from the sum of those before it. The exponentials are then taken twice, so one segment is kept
// where the channels alone fill the GPU (segment_rows).
#include "sequence.cuh"

namespace sf {
namespace {

using seq::Rows;
using seq::Span;
typedef unsigned long long u64;

constexpr int kThreads = 128;  // of the single-token kernel
constexpr int kS = 4;          // states per lane
constexpr int kMaxState = 128;
constexpr int kRows = 16;      // rows per tile, and per checkpoint
constexpr int kHalf = 8;       // rows between two additions over the warps in the backward pass
constexpr int kPart = 4;       // rows whose states the backward pass keeps in registers
constexpr float kLog2e = 1.4426950408889634f;

struct ScanArgs {
  const void *x, *dt, *B, *C, *z, *dy;
  const float *A, *D, *dt_bias, *init, *dfinal, *ck;
  void *y, *dx, *ddt, *dz;
  float *final_state, *ck_out, *dinit;
  float *part_bc, *part_a, *part_d;  // backward partial sums
  float *seg_state, *seg_dt;         // what segments add to a state [slots][dim][state], and their sum of dt [slots][dim]
  Rows rows;
  long long seg_rows;                // rows per segment, a multiple of kRows
  long long x_batch, x_row, dt_batch, dt_row, z_batch, z_row, b_batch, b_row, c_batch, c_row;
  int dim, state, groups, softplus;
  int vec, words;  // four channels, 4 bytes of a row of B and C as one access: rows and pointers are aligned for it
};

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// Pairs of fp32: each half is rounded like the scalar operation.
__device__ __forceinline__ u64 pack2(float lo, float hi) {
  u64 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(float& lo, float& hi, u64 v) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ u64 mul2(u64 a, u64 b) {
  u64 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ u64 fma2(u64 a, u64 b, u64 c) {
  u64 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ u64 add2(u64 a, u64 b) {
  u64 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float sum2(u64 a) {
  float lo, hi;
  unpack2(lo, hi, a);
  return lo + hi;
}
__device__ __forceinline__ float rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ u64 ex2x2(u64 v) {
  float lo, hi;
  unpack2(lo, hi, v);
  return pack2(ex2(lo), ex2(hi));
}

// softplus(v) = max(v, 0) + log(1 + e) with e = exp(-|v|), which is returned too. log(1 + e) = 2 atanh(s), s = e / (2 + e)
// <= 1/3, is odd in s: s times a polynomial of degree 4 in s^2, fitted by weighted least squares to a relative error
// of 8e-9 (of fp32 coefficients) over [0, 1/9]. Small e keep all their digits (a time step of 1e-3 is e = 1e-3), which
// log(1 + e) from a logarithm would not. (Scalar: pairs would need a move for every coefficient.)
__device__ __forceinline__ float softplus(float v, float& e) {
  e = ex2(-kLog2e * fabsf(v));
  const float s = e * rcp(2.f + e), q = s * s;
  float c = 0.28178343176841736f;
  c = fmaf(c, q, 0.27960601449012756f);
  c = fmaf(c, q, 0.40024909377098083f);
  c = fmaf(c, q, 0.6666631698608398f);
  c = fmaf(c, q, 2.f);
  return fmaf(s, c, fmaxf(v, 0.f));
}
// 1 / (1 + exp(-v))
__device__ __forceinline__ float logistic(float v) { return rcp(1.f + ex2(-kLog2e * v)); }

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
  if ((state & 3) == 0) {
    if (n < state) {
      const float4 v = *reinterpret_cast<const float4*>(p + n);
      o[0] = v.x, o[1] = v.y, o[2] = v.z, o[3] = v.w;
    } else {
      o[0] = o[1] = o[2] = o[3] = 0.f;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < kS; ++i) o[i] = n + i < state ? p[n + i] : 0.f;
}
__device__ __forceinline__ void store4(float* p, const float (&v)[kS], int n, int state) {
  if ((state & 3) == 0) {
    if (n < state) *reinterpret_cast<float4*>(p + n) = make_float4(v[0], v[1], v[2], v[3]);
    return;
  }
#pragma unroll
  for (int i = 0; i < kS; ++i)
    if (n + i < state) p[n + i] = v[i];
}
__device__ __forceinline__ void load4(u64 (&o)[2], const float* p, int n, int state) {
  float v[kS];
  load4(v, p, n, state);
  o[0] = pack2(v[0], v[1]);
  o[1] = pack2(v[2], v[3]);
}
__device__ __forceinline__ void store4(float* p, const u64 (&v)[2], int n, int state) {
  float f[kS];
  unpack2(f[0], f[1], v[0]);
  unpack2(f[2], f[3], v[1]);
  store4(p, f, n, state);
}

template <int LPC>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = LPC / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sums of four rows' values over the lanes of a channel: lane q gets row q % 4 (two lanes: rows 2q and 2q + 1, one
// lane: all four). Three shuffles where four whole reductions would take eight.
template <int LPC>
constexpr int kRowsPerLane = LPC >= 4 ? 1 : 4 / LPC;
template <int LPC>
__device__ __forceinline__ void scatter4(float (&o)[kRowsPerLane<LPC>], const float (&v)[4], int q) {
  if constexpr (LPC == 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = v[i];
  } else if constexpr (LPC == 2) {
    const bool b = q & 1;
    o[0] = (b ? v[2] : v[0]) + __shfl_xor_sync(0xffffffffu, b ? v[0] : v[2], 1);
    o[1] = (b ? v[3] : v[1]) + __shfl_xor_sync(0xffffffffu, b ? v[1] : v[3], 1);
  } else {
    const bool b1 = q & 2, b0 = q & 1;
    const float k0 = (b1 ? v[2] : v[0]) + __shfl_xor_sync(0xffffffffu, b1 ? v[0] : v[2], 2);
    const float k1 = (b1 ? v[3] : v[1]) + __shfl_xor_sync(0xffffffffu, b1 ? v[1] : v[3], 2);
    o[0] = (b0 ? k1 : k0) + __shfl_xor_sync(0xffffffffu, b0 ? k0 : k1, 1);
#pragma unroll
    for (int s = 4; s < LPC; s <<= 1) o[0] += __shfl_xor_sync(0xffffffffu, o[0], s);
  }
}
template <int LPC>
__device__ __forceinline__ int scatter_row(int q) {  // the first row that lane q gets
  return LPC >= 4 ? (q & 3) : q * kRowsPerLane<LPC>;
}

template <int LPC>
struct Cfg {
  static constexpr int CH = LPC <= 4 ? 64 : 256 / LPC;  // channels per block
  static constexpr int NP = LPC * kS;
  static constexpr int THREADS = CH * LPC;
  static constexpr int WARPS = THREADS / 32;
  static constexpr int UNITS = kRows * CH / 4;  // four channels of a row each
  static constexpr int UPT = (UNITS + THREADS - 1) / THREADS;
  static constexpr int BPT = kRows * NP / THREADS;  // elements of B (and of C) per thread
  static constexpr int PAD = CH + 8;                // row pitch of arrays that are read four rows at a time
};

// Which 16-byte entry of a row holds channel c: threads write channels 4l + j (j fixed), lanes read eight
// neighbouring channels; with this exchange within groups of eight neither conflicts.
__device__ __forceinline__ int entry(int c) { return c ^ ((c >> 3) & 3); }

template <typename T>
__device__ __forceinline__ void load_unit(seq::Vec<T, 4>& o, const T* p, int valid, int vec) {
  if (vec && valid >= 4) {
    o = *reinterpret_cast<const seq::Vec<T, 4>*>(p);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) o.v[i] = i < valid ? p[i] : DT<T>::from_f(0.f);
}
template <typename T>
__device__ __forceinline__ void store_unit(T* p, const seq::Vec<T, 4>& v, int valid, int vec) {
  if (vec && valid >= 4) {
    *reinterpret_cast<seq::Vec<T, 4>*>(p) = v;
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < valid) p[i] = v.v[i];
}

// The block's place: its group and channels, its segment of a sequence.
template <int LPC>
struct Place {
  int g, tile, d0, ch;  // group, channel tile of the group, first channel, channels of the tile
  int c, q, n, d;       // this lane's channel (in the tile and in all), lane of the channel, first state
  bool own;
  __device__ __forceinline__ Place(const ScanArgs& a) {
    const int per = a.dim / a.groups, tiles = (per + Cfg<LPC>::CH - 1) / Cfg<LPC>::CH;
    g = blockIdx.x / tiles;
    tile = blockIdx.x % tiles;
    d0 = g * per + tile * Cfg<LPC>::CH;
    ch = min(Cfg<LPC>::CH, (g + 1) * per - d0);
    c = threadIdx.x / LPC;
    q = threadIdx.x % LPC;
    n = q * kS;
    d = d0 + c;
    own = c < ch;
  }
};

__device__ __forceinline__ void cp_async(void* dst, const void* src, int bytes, bool in) {
  const uint32_t d = smem_u32(dst);
  const int n = in ? bytes : 0;  // bytes past n are filled with 0
  if (bytes == 4) asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(d), "l"(src), "r"(n) : "memory");
  if (bytes == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(d), "l"(src), "r"(n) : "memory");
  if (bytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Tiles' elements on their way: x, dt, z and dy of four channels and one row, and words of B and C, copied
// asynchronously to a ring of STAGES tiles in shared memory. A thread copies what it will convert itself, so no barrier
// guards the ring, and it has the same channels in every tile. (In registers the tile ahead was spilled, which waits
// for the loads; one tile ahead is also less than the latency of memory.) Rows of 16-bit data that no word fits are
// loaded and stored by the thread, which waits for them.
template <typename T, int LPC, bool X, bool Z, bool GY, bool BB, bool CC, int STAGES>
struct Ring {
  using F = Cfg<LPC>;
  static constexpr int ARRAYS = X + 1 + Z + GY;
  static constexpr int EPW = 4 / (int)sizeof(T);  // elements per word of B and C
  static constexpr int WORDS = kRows * F::NP / EPW, WPT = (WORDS + F::THREADS - 1) / F::THREADS;
  seq::Vec<T, 4> v[STAGES][ARRAYS][F::UPT][F::THREADS];
  seq::Vec<T, EPW> bc[STAGES][BB + CC][WPT][F::THREADS];
  float bias[F::CH], D[F::CH];
};

template <typename T, int LPC, bool X, bool Z, bool GY, bool BB, bool CC, int STAGES>
struct Fetch {
  using F = Cfg<LPC>;
  using R = Ring<T, LPC, X, Z, GY, BB, CC, STAGES>;
  static constexpr int RSTEP = F::THREADS / (F::CH / 4);  // rows between a thread's units
  static constexpr int WROW = F::NP / R::EPW;             // words per row of B
  static constexpr int AX = 0, AT = X, AZ = X + 1, AG = X + 1 + Z;
  R& ring;
  const T *px, *pdt, *pz, *pgy, *pb, *pc;
  int r, m, valid;
  int put, get;  // stages

  // The first tile's rows start at t0 (of the sequence). Ends with the block's bias and D in shared memory, for the
  // barrier that follows.
  __device__ __forceinline__ Fetch(R& ring_, const ScanArgs& a, const Place<LPC>& k, const Span& p, long long t0)
      : ring(ring_) {
    r = threadIdx.x / (F::CH / 4);
    m = threadIdx.x % (F::CH / 4) * 4;
    valid = F::THREADS <= F::UNITS || threadIdx.x < F::UNITS ? max(0, min(4, k.ch - m)) : 0;
    put = get = 0;
    const long long t = t0 + r;
    const int wr = threadIdx.x / WROW, wm = threadIdx.x % WROW * R::EPW;
    if (X) px = at<T>(a.x, a, p, a.x_batch, a.x_row) + k.d0 + t * a.x_row + m;
    pdt = at<T>(a.dt, a, p, a.dt_batch, a.dt_row) + k.d0 + t * a.dt_row + m;
    if (Z) pz = a.z ? at<T>(a.z, a, p, a.z_batch, a.z_row) + k.d0 + t * a.z_row + m : nullptr;
    if (GY) pgy = static_cast<const T*>(a.dy) + (row0(a, p) + t) * a.dim + k.d0 + m;
    if (BB) pb = at<T>(a.B, a, p, a.b_batch, a.b_row) + (long long)k.g * a.state + (t0 + wr) * a.b_row + wm;
    if (CC) pc = at<T>(a.C, a, p, a.c_batch, a.c_row) + (long long)k.g * a.state + (t0 + wr) * a.c_row + wm;
    for (int i = threadIdx.x; i < F::CH; i += F::THREADS) {
      ring.bias[i] = a.dt_bias && i < k.ch ? a.dt_bias[k.d0 + i] : 0.f;
      ring.D[i] = a.D && i < k.ch ? a.D[k.d0 + i] : 0.f;
    }
  }
  __device__ __forceinline__ void unit_in(seq::Vec<T, 4>& dst, const T* src, int ok, int vec) {
    if (vec) {
      cp_async(&dst, src, 4 * sizeof(T), ok > 0);
    } else if (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) cp_async(&dst.v[i], src + (i < ok ? i : 0), 4, i < ok);
    } else {
      load_unit(dst, src, ok, 0);
    }
  }
  __device__ __forceinline__ void word_in(seq::Vec<T, R::EPW>& dst, const T* src, int ok, int words) {
    if (sizeof(T) == 4 || words) {
      cp_async(&dst, src, 4, ok > 0);
    } else {
#pragma unroll
      for (int i = 0; i < R::EPW; ++i) dst.v[i] = i < ok ? src[i] : DT<T>::from_f(0.f);
    }
  }
  // Starts a tile of `rows` rows at the pointers, which then move on by `next` rows. Rows below 1: nothing to copy.
  __device__ __forceinline__ void load(const ScanArgs& a, int rows, int next) {
    if (rows > 0) {
#pragma unroll
      for (int i = 0; i < F::UPT; ++i) {
        const int rr = i * RSTEP, ok = r + rr < rows ? valid : 0;
        if (X) unit_in(ring.v[put][AX][i][threadIdx.x], px + (ok ? rr * a.x_row : 0), ok, a.vec);
        unit_in(ring.v[put][AT][i][threadIdx.x], pdt + (ok ? rr * a.dt_row : 0), ok, a.vec);
        if (Z && a.z) unit_in(ring.v[put][AZ][i][threadIdx.x], pz + (ok ? rr * a.z_row : 0), ok, a.vec);
        if (GY) unit_in(ring.v[put][AG][i][threadIdx.x], pgy + (ok ? (long long)rr * a.dim : 0), ok, a.vec);
      }
      const int wr = threadIdx.x / WROW, wm = threadIdx.x % WROW * R::EPW;
#pragma unroll
      for (int i = 0; i < R::WPT; ++i) {
        const int rr = i * (F::THREADS / WROW), ok = wr + rr < rows ? a.state - wm : 0;
        if (R::WORDS % F::THREADS == 0 || threadIdx.x + i * F::THREADS < R::WORDS) {
          if (BB) word_in(ring.bc[put][0][i][threadIdx.x], pb + (ok > 0 ? rr * a.b_row : 0), ok, a.words);
          if (CC) word_in(ring.bc[put][BB][i][threadIdx.x], pc + (ok > 0 ? rr * a.c_row : 0), ok, a.words);
        }
      }
      if (X) px += next * a.x_row;
      pdt += next * a.dt_row;
      if (Z && a.z) pz += next * a.z_row;
      if (GY) pgy += (long long)next * a.dim;
      if (BB) pb += next * a.b_row;
      if (CC) pc += next * a.c_row;
    }
    cp_async_commit();
    put = put + 1 == STAGES ? 0 : put + 1;
  }
  // Waits for the oldest tile of STAGES - 1 in flight.
  __device__ __forceinline__ void wait() { cp_async_wait<STAGES - 2>(); }
  __device__ __forceinline__ void done() { get = get + 1 == STAGES ? 0 : get + 1; }
  __device__ __forceinline__ seq::Vec<T, 4> unit(int array, int i) const { return ring.v[get][array][i][threadIdx.x]; }
  __device__ __forceinline__ bool has_unit(int i) const {
    return F::UNITS % F::THREADS == 0 || threadIdx.x + i * F::THREADS < F::UNITS;
  }
  // B and C as floats, in [kRows][NP] arrays.
  __device__ __forceinline__ void convert_bc(float (*B)[F::NP], float (*C)[F::NP]) const {
    const int wr = threadIdx.x / WROW, wm = threadIdx.x % WROW * R::EPW;
#pragma unroll
    for (int i = 0; i < R::WPT; ++i)
      if (R::WORDS % F::THREADS == 0 || threadIdx.x + i * F::THREADS < R::WORDS) {
        const int rr = wr + i * (F::THREADS / WROW);
        float f[R::EPW];
        if (BB) {
          seq::load_vec<T, R::EPW>(f, ring.bc[get][0][i][threadIdx.x].v);
          *reinterpret_cast<seq::Vec<float, R::EPW>*>(&B[rr][wm]) = *reinterpret_cast<seq::Vec<float, R::EPW>*>(f);
        }
        if (CC) {
          seq::load_vec<T, R::EPW>(f, ring.bc[get][BB][i][threadIdx.x].v);
          *reinterpret_cast<seq::Vec<float, R::EPW>*>(&C[rr][wm]) = *reinterpret_cast<seq::Vec<float, R::EPW>*>(f);
        }
      }
  }
  // dt of element j of unit i as the recurrence uses it, 0 where there is no element (rows past the tile's, channels
  // past the block's); SLOPE: and its derivative by dt_raw.
  template <bool SLOPE>
  __device__ __forceinline__ float step(const ScanArgs& a, float raw, int i, int j, int rows, float& slope) const {
    float v = raw + ring.bias[m + j];
    slope = 1.f;
    if (a.softplus) {
      float e;
      const float u = v;
      v = softplus(u, e);
      if (SLOPE) slope = (u >= 0.f ? 1.f : e) * rcp(1.f + e);  // the logistic function of u
    }
    return r + i * RSTEP < rows && j < valid ? v : 0.f;
  }
};

// State at the start of segment j (of segment n_slots - 1 - j, going backwards): what the segments before it leave.
template <bool REV>
__device__ __forceinline__ void segment_start(u64 (&h)[2], const ScanArgs& a, const Span& p, const u64 (&A2)[2], int j,
                                              int d, int n) {
  for (int i = 0; i < j; ++i) {
    const long long slot = p.slot0 + (REV ? p.n_slots - 1 - i : i);
    u64 e[2];
    load4(e, a.seg_state + (slot * a.dim + d) * a.state, n, a.state);
    const float s = a.seg_dt[slot * a.dim + d];
    const u64 s2 = pack2(s, s);
    h[0] = fma2(ex2x2(mul2(s2, A2[0])), h[0], e[0]);
    h[1] = fma2(ex2x2(mul2(s2, A2[1])), h[1], e[1]);
  }
}

template <int LPC>
__device__ __forceinline__ void load_decay(u64 (&A2)[2], const ScanArgs& a, const Place<LPC>& k) {
  float v[kS] = {};
  if (k.own) load4(v, a.A + (long long)k.d * a.state, k.n, a.state);
  A2[0] = pack2(v[0] * kLog2e, v[1] * kLog2e);
  A2[1] = pack2(v[2] * kLog2e, v[3] * kLog2e);
}

// What a segment adds to a state of 0, forwards (h = a h + dt x B) or backwards (gh = a (gh + gp C)), and its sum of
// dt. The last segment's (backwards: the first's) is not needed.
template <typename T, int LPC, bool REV>
struct CarrySmem {
  using F = Cfg<LPC>;
  static constexpr int STAGES = sizeof(T) == 2 ? 4 : 3;
  float4 du[kRows][F::CH];  // dt, dt, dt x, dt x (backwards gp)
  float B[kRows][F::NP];
  Ring<T, LPC, !REV, REV, REV, !REV, REV, STAGES> ring;
};
template <typename T, int LPC, bool REV>
__global__ void __launch_bounds__(Cfg<LPC>::THREADS, 3) scan_carry_kernel(ScanArgs a) {
  using F = Cfg<LPC>;
  using S = CarrySmem<T, LPC, REV>;
  extern __shared__ __align__(16) char smem[];
  S& sm = *reinterpret_cast<S*>(smem);
  const Place<LPC> k(a);
  const Span p = seq::slot_span(a.rows, blockIdx.y, a.seg_rows);
  if (p.len < 0) return;
  const int seg = (int)(blockIdx.y - p.slot0);
  if (REV ? seg == 0 : seg == p.n_slots - 1) return;
  const long long r1 = min(p.r0 + a.seg_rows, p.len);
  const int tiles = (int)((r1 - p.r0 + kRows - 1) / kRows);
  Fetch<T, LPC, !REV, REV, REV, !REV, REV, S::STAGES> f(sm.ring, a, k, p, p.r0 + (REV ? (tiles - 1ll) * kRows : 0));
  auto tile_rows = [&](int i) {
    return i < tiles ? (int)min((long long)kRows, r1 - p.r0 - (long long)(REV ? tiles - 1 - i : i) * kRows) : 0;
  };
  for (int i = 0; i < S::STAGES - 1; ++i) f.load(a, tile_rows(i), REV ? -kRows : kRows);
  u64 A2[2], h[2] = {0, 0};
  load_decay(A2, a, k);
  float sum = 0.f;
  for (int i = 0; i < tiles; ++i) {
    const int rows = tile_rows(i);
    f.wait();
    __syncthreads();
#pragma unroll
    for (int v = 0; v < F::UPT; ++v)
      if (f.has_unit(v)) {
        const auto tdt = f.unit(f.AT, v), tx = f.unit(REV ? f.AG : f.AX, v);
        seq::Vec<T, 4> tz;
        if (REV && a.z) tz = f.unit(f.AZ, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float slope;
          const float dt = f.template step<false>(a, DT<T>::to_f(tdt.v[j]), v, j, rows, slope);
          float w = DT<T>::to_f(tx.v[j]);
          if (!REV) {
            w *= dt;
          } else if (a.z) {
            const float z = DT<T>::to_f(tz.v[j]);
            w *= z * logistic(z);
          }
          sm.du[f.r + v * f.RSTEP][entry(f.m + j)] = make_float4(dt, dt, w, w);
        }
      }
    f.convert_bc(sm.B, sm.B);
    f.done();
    f.load(a, tile_rows(i + S::STAGES - 1), REV ? -kRows : kRows);
    __syncthreads();
    const int e = entry(k.c);
#pragma unroll
    for (int rr = 0; rr < kRows; ++rr) {
      const int r = REV ? kRows - 1 - rr : rr;
      const ulonglong2 du = *reinterpret_cast<const ulonglong2*>(&sm.du[r][e]);
      const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(&sm.B[r][k.n]);
      const u64 a0 = ex2x2(mul2(du.x, A2[0])), a1 = ex2x2(mul2(du.x, A2[1]));
      if (REV) {
        h[0] = mul2(a0, fma2(du.y, b.x, h[0]));
        h[1] = mul2(a1, fma2(du.y, b.y, h[1]));
      } else {
        h[0] = fma2(a0, h[0], mul2(du.y, b.x));
        h[1] = fma2(a1, h[1], mul2(du.y, b.y));
      }
      sum += __uint_as_float((unsigned)du.x);
    }
  }
  if (!k.own) return;
  const long long o = (long long)blockIdx.y * a.dim + k.d;
  store4(a.seg_state + o * a.state, h, k.n, a.state);
  if (k.q == 0) a.seg_dt[o] = sum;
}

template <typename T, int LPC>
struct FwdSmem {
  using F = Cfg<LPC>;
  static constexpr int STAGES = sizeof(T) == 2 ? 4 : 3;
  float4 du[kRows][F::CH];  // dt, dt, dt x, dt x
  float2 gx[kRows][F::PAD]; // D x, gate
  float B[kRows][F::NP], C[kRows][F::NP];
  T out[kRows][F::PAD];
  Ring<T, LPC, true, true, false, true, true, STAGES> ring;
};

// One block: one segment of a sequence and CH channels of one group.
template <typename T, int LPC>
__global__ void __launch_bounds__(Cfg<LPC>::THREADS, 3) scan_fwd_kernel(ScanArgs a) {
  using F = Cfg<LPC>;
  extern __shared__ __align__(16) char smem[];
  FwdSmem<T, LPC>& s = *reinterpret_cast<FwdSmem<T, LPC>*>(smem);
  const Place<LPC> k(a);
  const Span p = seq::slot_span(a.rows, blockIdx.y, a.seg_rows);
  if (p.len < 0) return;
  const int seg = (int)(blockIdx.y - p.slot0);
  const long long r1 = min(p.r0 + a.seg_rows, p.len);
  const int tiles = (int)((r1 - p.r0 + kRows - 1) / kRows);
  constexpr int STAGES = FwdSmem<T, LPC>::STAGES;
  Fetch<T, LPC, true, true, false, true, true, STAGES> f(s.ring, a, k, p, p.r0);
  T* py = static_cast<T*>(a.y) + (row0(a, p) + p.r0 + f.r) * a.dim + k.d0 + f.m;
  auto tile_rows = [&](int i) {
    return i < tiles ? (int)min((long long)kRows, r1 - (p.r0 + (long long)i * kRows)) : 0;
  };
  auto put = [&](int rows) {  // a tile's results, four channels of a row together
#pragma unroll
    for (int v = 0; v < F::UPT; ++v) {
      const int r = f.r + v * f.RSTEP;
      if (f.has_unit(v) && r < rows)
        store_unit(py + (long long)v * f.RSTEP * a.dim, *reinterpret_cast<const seq::Vec<T, 4>*>(&s.out[r][f.m]),
                   f.valid, a.vec);
    }
    py += (long long)kRows * a.dim;
  };
  for (int i = 0; i < STAGES - 1; ++i) f.load(a, tile_rows(i), kRows);
  u64 A2[2], h[2] = {0, 0};
  load_decay(A2, a, k);
  if (k.own) {
    if (a.init) load4(h, a.init + ((long long)p.s * a.dim + k.d) * a.state, k.n, a.state);
    if (seg > 0) segment_start<false>(h, a, p, A2, seg, k.d, k.n);
  }
  float* ck = nullptr;
  if (a.ck_out && k.own)
    ck = a.ck_out + ((seq::seq_slot0(a.rows, p.s, kRows) + p.r0 / kRows) * a.dim + k.d) * a.state;
  const int e = entry(k.c);
  for (int i = 0; i < tiles; ++i) {
    const int rows = tile_rows(i);
    if (ck) {
      store4(ck, h, k.n, a.state);
      ck += (long long)a.dim * a.state;
    }
    f.wait();
    __syncthreads();
    if (i > 0) put(kRows);
#pragma unroll
    for (int v = 0; v < F::UPT; ++v)
      if (f.has_unit(v)) {
        const auto tdt = f.unit(f.AT, v), tx = f.unit(f.AX, v);
        seq::Vec<T, 4> tz;
        if (a.z) tz = f.unit(f.AZ, v);
        const int r = f.r + v * f.RSTEP;
        float px[4], g[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float slope;
          const float dt = f.template step<false>(a, DT<T>::to_f(tdt.v[j]), v, j, rows, slope);
          const float x = DT<T>::to_f(tx.v[j]), w = dt * x;
          px[j] = s.ring.D[f.m + j] * x;
          g[j] = 1.f;
          if (a.z) {
            g[j] = DT<T>::to_f(tz.v[j]);
            g[j] *= logistic(g[j]);
          }
          s.du[r][entry(f.m + j)] = make_float4(dt, dt, w, w);
        }
        *reinterpret_cast<float4*>(&s.gx[r][f.m]) = make_float4(px[0], g[0], px[1], g[1]);
        *reinterpret_cast<float4*>(&s.gx[r][f.m + 2]) = make_float4(px[2], g[2], px[3], g[3]);
      }
    f.convert_bc(s.B, s.C);
    f.done();
    f.load(a, tile_rows(i + STAGES - 1), kRows);
    __syncthreads();
#pragma unroll
    for (int r0 = 0; r0 < kRows; r0 += 4) {
      float y[4], o[kRowsPerLane<LPC>];
#pragma unroll
      for (int rr = 0; rr < 4; ++rr) {
        const int r = r0 + rr;
        const ulonglong2 du = *reinterpret_cast<const ulonglong2*>(&s.du[r][e]);
        const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(&s.B[r][k.n]);
        const ulonglong2 c = *reinterpret_cast<const ulonglong2*>(&s.C[r][k.n]);
        h[0] = fma2(ex2x2(mul2(du.x, A2[0])), h[0], mul2(du.y, b.x));
        h[1] = fma2(ex2x2(mul2(du.x, A2[1])), h[1], mul2(du.y, b.y));
        y[rr] = sum2(fma2(c.x, h[0], mul2(c.y, h[1])));
      }
      scatter4<LPC>(o, y, k.q);
      if (LPC <= 4 || k.q < 4)
#pragma unroll
        for (int j = 0; j < kRowsPerLane<LPC>; ++j) {
          const int r = r0 + scatter_row<LPC>(k.q) + j;
          const float2 g = s.gx[r][k.c];
          s.out[r][k.c] = DT<T>::from_f((o[j] + g.x) * g.y);
        }
    }
  }
  if (tiles > 0) {
    __syncthreads();
    put(tile_rows(tiles - 1));
  }
  if (a.final_state && k.own && seg == p.n_slots - 1)
    store4(a.final_state + ((long long)p.s * a.dim + k.d) * a.state, h, k.n, a.state);
}

template <typename T, int LPC>
struct BwdSmem {
  using F = Cfg<LPC>;
  static constexpr int STAGES = sizeof(T) == 2 ? 3 : 2;
  float4 du[kRows][F::CH];   // dt, dt, dt x, dt x
  float4 gp[kRows][F::CH];   // gp, gp, D gp, x
  float2 sg[kRows][F::PAD];  // softplus'(raw), dy silu'(z)
  float px[kRows][F::PAD];   // D x
  float B[kRows][F::NP], C[kRows][F::NP];
  float bc[2][F::WARPS][kHalf][2 * F::NP];  // sums over a warp's channels, one half tile after the other
  T dx[kRows][F::PAD], ddt[kRows][F::PAD], dz[kRows][F::PAD];
  Ring<T, LPC, true, true, true, true, true, STAGES> ring;
};

// Sums of 8 values over the channels of a warp: scattered over the lanes as far as they go. Returns how many values
// this lane has in v[0..], the first of them number `first`.
template <int LPC>
__device__ __forceinline__ void channels_sum(float (&v)[8], int lane) {
  int cnt = 8;
#pragma unroll
  for (int o = 16; o >= LPC; o >>= 1) {
    if (cnt > 1) {
      cnt >>= 1;
      const bool up = lane & o;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < cnt) {
          const float keep = up ? v[cnt + i] : v[i], send = up ? v[i] : v[cnt + i];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    }
  }
}
template <int LPC>
constexpr int kSumsPerLane = LPC <= 4 ? 1 : LPC / 4;
template <int LPC>
__device__ __forceinline__ int sums_first(int lane) {
  int cnt = 8, first = 0;
#pragma unroll
  for (int o = 16; o >= LPC; o >>= 1)
    if (cnt > 1) {
      cnt >>= 1;
      if (lane & o) first += cnt;
    }
  return first;
}

// Tiles from the last to the first: a tile's states again from its checkpoint, half a tile at a time in registers,
// then its rows backwards. Sums over a block's channels of gB and gC go to part_bc[tile][row][group][2][NP], added
// over the tiles by scan_bc_reduce_kernel; sums over a segment of gA, gD and gbias to part_a / part_d, added over
// the segments by scan_sum_kernel. No atomics: the order of every sum is fixed.
template <typename T, int LPC>
__global__ void __launch_bounds__(Cfg<LPC>::THREADS, 2) scan_bwd_kernel(ScanArgs a) {
  using F = Cfg<LPC>;
  extern __shared__ __align__(16) char smem[];
  BwdSmem<T, LPC>& s = *reinterpret_cast<BwdSmem<T, LPC>*>(smem);
  const Place<LPC> k(a);
  const Span p = seq::slot_span(a.rows, blockIdx.y, a.seg_rows);
  const long long sd = (long long)blockIdx.y * a.dim + k.d;
  if (p.len < 0) {  // a slot of no sequence still has a place in the sums
    if (k.own) {
      const u64 zero[2] = {0, 0};
      store4(a.part_a + sd * a.state, zero, k.n, a.state);
      if (k.q == 0) a.part_d[sd] = a.part_d[(long long)gridDim.y * a.dim + sd] = 0.f;
    }
    return;
  }
  const int seg = (int)(blockIdx.y - p.slot0), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long r00 = row0(a, p);
  const long long total_rows = a.rows.offsets ? a.rows.length : a.rows.length * a.rows.n_seq;
  const long long r1 = min(p.r0 + a.seg_rows, p.len);
  const int tiles = (int)((r1 - p.r0 + kRows - 1) / kRows);
  const long long last = p.r0 + (tiles - 1ll) * kRows;  // first row of the last tile
  float* bc_out = a.part_bc + ((k.tile * total_rows + r00 + last) * a.groups + k.g) * 2 * F::NP;
  const float* ck = a.ck + ((seq::seq_slot0(a.rows, p.s, kRows) + last / kRows) * a.dim + k.d) * a.state;

  constexpr int STAGES = BwdSmem<T, LPC>::STAGES;
  Fetch<T, LPC, true, true, true, true, true, STAGES> f(s.ring, a, k, p, last);
  long long po = (r00 + last + f.r) * a.dim + k.d0 + f.m;  // where a tile's results go
  auto put = [&](int rows) {
#pragma unroll
    for (int v = 0; v < F::UPT; ++v) {
      const int r = f.r + v * f.RSTEP;
      if (f.has_unit(v) && r < rows) {
        const long long o = po + (long long)v * f.RSTEP * a.dim;
        using V4 = seq::Vec<T, 4>;
        store_unit(static_cast<T*>(a.dx) + o, *reinterpret_cast<const V4*>(&s.dx[r][f.m]), f.valid, a.vec);
        store_unit(static_cast<T*>(a.ddt) + o, *reinterpret_cast<const V4*>(&s.ddt[r][f.m]), f.valid, a.vec);
        if (a.dz) store_unit(static_cast<T*>(a.dz) + o, *reinterpret_cast<const V4*>(&s.dz[r][f.m]), f.valid, a.vec);
      }
    }
    po -= (long long)kRows * a.dim;
  };
  const int last_rows = (int)(r1 - last);
  auto tile_rows = [&](int i) { return i < 0 ? 0 : i == tiles - 1 ? last_rows : kRows; };
  for (int i = 0; i < STAGES - 1; ++i) f.load(a, tile_rows(tiles - 1 - i), -kRows);
  u64 A2[2], gh[2] = {0, 0}, gA[2] = {0, 0};
  load_decay(A2, a, k);
  if (k.own) {
    if (a.dfinal) load4(gh, a.dfinal + ((long long)p.s * a.dim + k.d) * a.state, k.n, a.state);
    if (seg < p.n_slots - 1) segment_start<true>(gh, a, p, A2, p.n_slots - 1 - seg, k.d, k.n);
  }
  float gD = 0.f, gbias = 0.f;
  const int e = entry(k.c), first = sums_first<LPC>(lane);
  for (int i = tiles - 1; i >= 0; --i) {
    const int rows = tile_rows(i);
    u64 h0[2] = {0, 0};  // the states before the tile
    if (k.own) load4(h0, ck, k.n, a.state);
    ck -= (long long)a.dim * a.state;
    f.wait();
    __syncthreads();
    if (i + 1 < tiles) put(tile_rows(i + 1));
#pragma unroll
    for (int v = 0; v < F::UPT; ++v)
      if (f.has_unit(v)) {
        const auto tdt = f.unit(f.AT, v), tx = f.unit(f.AX, v), tg = f.unit(f.AG, v);
        seq::Vec<T, 4> tz;
        if (a.z) tz = f.unit(f.AZ, v);
        const int r = f.r + v * f.RSTEP;
        float slope[4], gz[4], px[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float dt = f.template step<true>(a, DT<T>::to_f(tdt.v[j]), v, j, rows, slope[j]);
          const float x = DT<T>::to_f(tx.v[j]), w = dt * x, D = s.ring.D[f.m + j];
          float g = DT<T>::to_f(tg.v[j]);
          gz[j] = 0.f;
          if (a.z) {
            const float z = DT<T>::to_f(tz.v[j]), sig = logistic(z);
            gz[j] = g * (sig * fmaf(z, 1.f - sig, 1.f));
            g *= z * sig;
          }
          px[j] = D * x;
          s.du[r][entry(f.m + j)] = make_float4(dt, dt, w, w);
          s.gp[r][entry(f.m + j)] = make_float4(g, g, D * g, x);
        }
        *reinterpret_cast<float4*>(&s.sg[r][f.m]) = make_float4(slope[0], gz[0], slope[1], gz[1]);
        *reinterpret_cast<float4*>(&s.sg[r][f.m + 2]) = make_float4(slope[2], gz[2], slope[3], gz[3]);
        *reinterpret_cast<float4*>(&s.px[r][f.m]) = make_float4(px[0], px[1], px[2], px[3]);
      }
    f.convert_bc(s.B, s.C);
    f.done();
    f.load(a, tile_rows(i - (STAGES - 1)), -kRows);
    __syncthreads();
    // The states before each part of kPart rows, then the parts from the last to the first.
    u64 hb[kRows / kPart][2] = {{h0[0], h0[1]}};
#pragma unroll
    for (int r = 0; r < kRows - kPart; ++r) {
      if (r % kPart == 0 && r + kPart >= rows) break;
      const ulonglong2 du = *reinterpret_cast<const ulonglong2*>(&s.du[r][e]);
      const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(&s.B[r][k.n]);
      h0[0] = fma2(ex2x2(mul2(du.x, A2[0])), h0[0], mul2(du.y, b.x));
      h0[1] = fma2(ex2x2(mul2(du.x, A2[1])), h0[1], mul2(du.y, b.y));
      if (r % kPart == kPart - 1) hb[r / kPart + 1][0] = h0[0], hb[r / kPart + 1][1] = h0[1];
    }
    u64 tA[2] = {0, 0};  // this tile's share of gA: sums of sums keep more digits than one long one
#pragma unroll
    for (int part = kRows / kPart - 1; part >= 0; --part) {
      const int t = part * kPart;
      if (t >= rows) continue;
      u64 hs[kPart + 1][2], as[kPart][2];
      hs[0][0] = hb[part][0];
      hs[0][1] = hb[part][1];
#pragma unroll
      for (int r = 0; r < kPart; ++r) {
        const ulonglong2 du = *reinterpret_cast<const ulonglong2*>(&s.du[t + r][e]);
        const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(&s.B[t + r][k.n]);
        as[r][0] = ex2x2(mul2(du.x, A2[0]));
        as[r][1] = ex2x2(mul2(du.x, A2[1]));
        hs[r + 1][0] = fma2(as[r][0], hs[r][0], mul2(du.y, b.x));
        hs[r + 1][1] = fma2(as[r][1], hs[r][1], mul2(du.y, b.y));
      }
      float pre[4], S[4], qa[4];
#pragma unroll
      for (int r = kPart - 1; r >= 0; --r) {
        const ulonglong2 du = *reinterpret_cast<const ulonglong2*>(&s.du[t + r][e]);
        const u64 gp = *reinterpret_cast<const u64*>(&s.gp[t + r][e]);
        const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(&s.B[t + r][k.n]);
        const ulonglong2 c = *reinterpret_cast<const ulonglong2*>(&s.C[t + r][k.n]);
        pre[r] = sum2(fma2(c.x, hs[r + 1][0], mul2(c.y, hs[r + 1][1])));
        gh[0] = fma2(gp, c.x, gh[0]);
        gh[1] = fma2(gp, c.y, gh[1]);
        S[r] = sum2(fma2(gh[0], b.x, mul2(gh[1], b.y)));
        float v[8];
        unpack2(v[0], v[1], mul2(gh[0], du.y));
        unpack2(v[2], v[3], mul2(gh[1], du.y));
        unpack2(v[4], v[5], mul2(gp, hs[r + 1][0]));
        unpack2(v[6], v[7], mul2(gp, hs[r + 1][1]));
        gh[0] = mul2(gh[0], as[r][0]);
        gh[1] = mul2(gh[1], as[r][1]);
        const u64 q0 = mul2(gh[0], hs[r][0]), q1 = mul2(gh[1], hs[r][1]);
        qa[r] = sum2(fma2(q0, A2[0], mul2(q1, A2[1])));
        tA[0] = fma2(q0, du.x, tA[0]);
        tA[1] = fma2(q1, du.x, tA[1]);
        channels_sum<LPC>(v, lane);
        // value i < 4: state n + i of gB, else of gC
        if (LPC >= 4 || (lane & 3 & ~(LPC - 1)) == 0)
#pragma unroll
          for (int j = 0; j < kSumsPerLane<LPC>; ++j)
            s.bc[part / 2 % 2][warp][t % kHalf + r][((first + j) >> 2) * F::NP + k.n + ((first + j) & 3)] = v[j];
      }
      float po4[kRowsPerLane<LPC>], So[kRowsPerLane<LPC>], qo[kRowsPerLane<LPC>];
      scatter4<LPC>(po4, pre, k.q);
      scatter4<LPC>(So, S, k.q);
      scatter4<LPC>(qo, qa, k.q);
      if (LPC <= 4 || k.q < 4)
#pragma unroll
        for (int j = 0; j < kRowsPerLane<LPC>; ++j) {
          const int r = t + scatter_row<LPC>(k.q) + j;
          const float4 g = s.gp[r][e];
          const float2 sg = s.sg[r][k.c];
          const float dt = s.du[r][e].x;
          const float gdt = fmaf(g.w, So[j], qo[j] * (1.f / kLog2e)) * sg.x;
          s.dx[r][k.c] = DT<T>::from_f(fmaf(dt, So[j], g.z));
          s.ddt[r][k.c] = DT<T>::from_f(gdt);
          s.dz[r][k.c] = DT<T>::from_f((po4[j] + s.px[r][k.c]) * sg.y);
          gD = fmaf(g.x, g.w, gD);
          gbias += r < rows ? gdt : 0.f;
        }
      if (t % kHalf == 0) {  // both parts of a half are done
        __syncthreads();
        for (int u = threadIdx.x; u < kHalf * 2 * F::NP; u += F::THREADS) {
          const int r = u / (2 * F::NP), m = u % (2 * F::NP);
          float v = 0.f;
#pragma unroll
          for (int w = 0; w < F::WARPS; ++w) v += s.bc[part / 2 % 2][w][r][m];
          if (t + r < rows) bc_out[(long long)(t + r) * a.groups * 2 * F::NP + m] = v;
        }
      }
    }
    gA[0] = add2(gA[0], tA[0]);
    gA[1] = add2(gA[1], tA[1]);
    bc_out -= (long long)kRows * a.groups * 2 * F::NP;
  }
  if (tiles > 0) {
    __syncthreads();
    put(tile_rows(0));
  }
  gD = lanes_sum<(LPC < 4 ? LPC : 4)>(gD);
  gbias = lanes_sum<(LPC < 4 ? LPC : 4)>(gbias);
  if (!k.own) return;
  if (a.dinit && seg == 0) store4(a.dinit + ((long long)p.s * a.dim + k.d) * a.state, gh, k.n, a.state);
  store4(a.part_a + sd * a.state, gA, k.n, a.state);
  if (k.q == 0) {
    a.part_d[sd] = gD;
    a.part_d[(long long)gridDim.y * a.dim + sd] = gbias;
  }
}

// dB, dC [rows, groups, state] from part_bc[tiles][rows][groups][2][NP].
template <typename T>
__global__ void scan_bc_reduce_kernel(const float* part, long long rows, int tiles, int groups, int NP, int state,
                                      T* dB, T* dC) {
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x, n = rows * groups * 2 * NP;
  if (i >= n) return;
  float v = 0.f;
#pragma unroll 8
  for (int j = 0; j < tiles; ++j) v += part[j * n + i];
  const int m = (int)(i % NP);
  if (m < state) (i / NP % 2 ? dC : dB)[i / (2 * NP) * state + m] = DT<T>::from_f(v);
}

// out[i] = sum over j < count of part[j * n + i], in order.
__global__ void scan_sum_kernel(const float* part, long long count, long long n, float* out) {
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  float v = 0.f;
#pragma unroll 8
  for (long long j = 0; j < count; ++j) v += part[j * n + i];
  out[i] = v;
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
int channels_per_block(int state) { return lanes(state) <= 4 ? 64 : 256 / lanes(state); }
int tiles_of(const sf_selective_scan_desc* d) {  // blocks for the channels of a group
  const int ch = channels_per_block(d->state), per = d->dim / d->groups;
  return (per + ch - 1) / ch;
}
constexpr long long kWhole = 1ll << 40;  // rows of a segment that takes any sequence whole

// Rows per segment: sequences whole where their channels alone give `want` blocks; else cut so that they do, but
// not below 128 rows, nor into more than 32 segments.
long long segment_rows(const sf_selective_scan_desc* d, long long want) {
  const long long blocks = (long long)tiles_of(d) * d->groups * d->n_seq;
  if (blocks >= want || d->length <= 256) return kWhole;
  const long long total = d->packed ? d->length : d->length * d->n_seq;
  const long long cuts = (want + (long long)tiles_of(d) * d->groups - 1) / ((long long)tiles_of(d) * d->groups);
  long long rows = (total + cuts - 1) / cuts;
  if (rows < 128) rows = 128;
  if (rows < (d->length + 31) / 32) rows = (d->length + 31) / 32;
  rows = (rows + kRows - 1) / kRows * kRows;
  return rows >= d->length ? kWhole : rows;
}
constexpr long long kFwdBlocks = 444, kBwdBlocks = 296;  // three, two blocks for each SM
long long slots_of(const sf_selective_scan_desc* d, long long seg) {
  return seq::total_slots(d->length, d->n_seq, d->packed, seg);
}
// Floats of seg_state and seg_dt.
long long carry_floats(const sf_selective_scan_desc* d, long long seg) {
  return seg == kWhole ? 0 : (slots_of(d, seg) * d->dim * (d->state + 1ll) + 3) / 4 * 4;
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

struct BwdLayout {  // floats from the start of the workspace
  long long carry, bc, a, d, total;
};
BwdLayout bwd_layout(const sf_selective_scan_desc* d, long long seg) {
  BwdLayout l;
  const long long np = (long long)lanes(d->state) * kS, slots = slots_of(d, seg);
  l.carry = 0;
  l.bc = carry_floats(d, seg);
  l.a = l.bc + (tiles_of(d) * rows_of(d) * 2 * d->groups * np + 3) / 4 * 4;
  l.d = l.a + (slots * d->dim * d->state + 3) / 4 * 4;
  l.total = l.d + 2 * slots * d->dim;
  return l;
}

// Whether four channels can be read and written as one word: every row of every group begins at a multiple.
bool vectors_fit(const sf_selective_scan_desc* d, std::initializer_list<const void*> ptrs) {
  if ((d->dim / d->groups) % 4) return false;
  for (long long v : {d->x_row_stride, d->dt_row_stride, d->z_row_stride})
    if (v % 4) return false;
  if (!d->packed && d->n_seq > 1)
    for (long long v : {d->x_batch_stride, d->dt_batch_stride, d->z_batch_stride})
      if (v % 4) return false;
  for (const void* p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) % (4 * dtype_size(d->dtype))) return false;
  return true;
}

// Whether 4 bytes of a row of B and C can be read as one word.
bool words_fit(const sf_selective_scan_desc* d, std::initializer_list<const void*> ptrs) {
  if (d->state % 2 || d->b_row_stride % 2 || d->c_row_stride % 2) return false;
  if (!d->packed && d->n_seq > 1 && (d->b_batch_stride % 2 || d->c_batch_stride % 2)) return false;
  for (const void* p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) % 4) return false;
  return true;
}

template <typename K>
bool prepare_smem(K kernel, size_t bytes) {
  return bytes <= 48 * 1024 || allow_max_smem(reinterpret_cast<const void*>(kernel));
}

template <typename T, int LPC>
sf_status run_fwd(const ScanArgs& a, dim3 grid, cudaStream_t st) {
  constexpr int threads = Cfg<LPC>::THREADS;
  if (a.seg_rows != kWhole) {
    constexpr size_t bytes = sizeof(CarrySmem<T, LPC, false>);
    if (!prepare_smem(scan_carry_kernel<T, LPC, false>, bytes)) return SF_ERR_CUDA;
    scan_carry_kernel<T, LPC, false><<<grid, threads, bytes, st>>>(a);
  }
  constexpr size_t smem = sizeof(FwdSmem<T, LPC>);
  if (!prepare_smem(scan_fwd_kernel<T, LPC>, smem)) return SF_ERR_CUDA;
  scan_fwd_kernel<T, LPC><<<grid, threads, smem, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? SF_OK : SF_ERR_CUDA;
}
template <typename T, int LPC>
sf_status run_bwd(const ScanArgs& a, dim3 grid, cudaStream_t st) {
  constexpr int threads = Cfg<LPC>::THREADS;
  if (a.seg_rows != kWhole) {
    constexpr size_t bytes = sizeof(CarrySmem<T, LPC, true>);
    if (!prepare_smem(scan_carry_kernel<T, LPC, true>, bytes)) return SF_ERR_CUDA;
    scan_carry_kernel<T, LPC, true><<<grid, threads, bytes, st>>>(a);
  }
  constexpr size_t smem = sizeof(BwdSmem<T, LPC>);
  if (!prepare_smem(scan_bwd_kernel<T, LPC>, smem)) return SF_ERR_CUDA;
  scan_bwd_kernel<T, LPC><<<grid, threads, smem, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? SF_OK : SF_ERR_CUDA;
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
  return (size_t)seq::total_slots(d->length, d->n_seq, d->packed, kRows) * d->dim * d->state * sizeof(float);
}

extern "C" size_t sf_selective_scan_workspace_size(const sf_selective_scan_desc* d) {
  if (!valid(d) || d->n_seq == 0) return 0;
  return (size_t)carry_floats(d, segment_rows(d, kFwdBlocks)) * sizeof(float);
}

extern "C" sf_status sf_selective_scan(const void* x, const void* dt, const float* A, const void* B, const void* C,
                                       const float* D, const void* z, const float* dt_bias,
                                       const float* initial_state, const int32_t* seq_offsets, void* y,
                                       float* final_state, void* checkpoints, const sf_selective_scan_desc* d,
                                       void* workspace, size_t workspace_bytes, void* stream) {
  if (!valid(d) || !A || (seq_offsets != nullptr) != (d->packed != 0)) return SF_ERR_INVALID_ARG;
  if (d->state > kMaxState || d->n_seq > 65535) return SF_ERR_UNSUPPORTED;
  if (d->n_seq == 0 || d->dim == 0) return SF_OK;
  if (d->length > 0 && (!x || !dt || !B || !C || !y)) return SF_ERR_INVALID_ARG;
  ScanArgs a = base_args(x, dt, A, B, C, D, z, dt_bias, seq_offsets, d);
  a.init = initial_state;
  a.y = y;
  a.final_state = final_state;
  a.ck_out = static_cast<float*>(checkpoints);
  a.vec = vectors_fit(d, {x, dt, z, y});
  a.words = words_fit(d, {B, C});
  a.seg_rows = segment_rows(d, kFwdBlocks);
  const long long carry = carry_floats(d, a.seg_rows), slots = slots_of(d, a.seg_rows);
  if (carry && (!workspace || workspace_bytes < (size_t)carry * sizeof(float))) return SF_ERR_WORKSPACE;
  for (const void* p : {static_cast<const void*>(A), static_cast<const void*>(initial_state),
                        static_cast<const void*>(final_state), static_cast<const void*>(checkpoints),
                        static_cast<const void*>(carry ? workspace : nullptr)})
    if (!aligned16(p)) return SF_ERR_ALIGNMENT;
  if (slots > 65535) return SF_ERR_UNSUPPORTED;
  a.seg_state = static_cast<float*>(workspace);
  a.seg_dt = a.seg_state + slots * d->dim * d->state;
  const dim3 grid(tiles_of(d) * d->groups, (unsigned)slots);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  sf_status status = SF_OK;
  SF_SCAN_TYPES(d->dtype, SF_SCAN_LANES(d->state, status = (run_fwd<T, L>(a, grid, st))))
  return status;
}

extern "C" size_t sf_selective_scan_backward_workspace_size(const sf_selective_scan_desc* d) {
  if (!valid(d)) return 0;
  return (size_t)bwd_layout(d, segment_rows(d, kBwdBlocks)).total * sizeof(float);
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
  const long long seg = segment_rows(d, kBwdBlocks), slots = slots_of(d, seg);
  const BwdLayout l = bwd_layout(d, seg);
  if (some && (!workspace || workspace_bytes < (size_t)l.total * sizeof(float))) return SF_ERR_WORKSPACE;
  if (some && !aligned16(workspace)) return SF_ERR_ALIGNMENT;
  for (const void* p : {static_cast<const void*>(A), checkpoints, static_cast<const void*>(d_final_state),
                        static_cast<const void*>(d_initial_state)})
    if (!aligned16(p)) return SF_ERR_ALIGNMENT;
  if (slots > 65535) return SF_ERR_UNSUPPORTED;
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
    a.seg_rows = seg;
    a.seg_state = ws + l.carry;
    a.seg_dt = a.seg_state + slots * d->dim * d->state;
    a.vec = vectors_fit(d, {x, dt, z, dy, dx, ddt, dz});
    a.words = words_fit(d, {B, C});
    const dim3 grid(tiles_of(d) * d->groups, (unsigned)slots);
    sf_status status = SF_OK;
    SF_SCAN_TYPES(d->dtype, SF_SCAN_LANES(d->state, status = (run_bwd<T, L>(a, grid, st))))
    if (status != SF_OK) return status;
    if (rows > 0) {
      const int np = lanes(d->state) * kS;
      const long long n = rows * 2 * d->groups * np;
      SF_SCAN_TYPES(d->dtype, (scan_bc_reduce_kernel<T><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(
                                  a.part_bc, rows, tiles_of(d), d->groups, np, d->state, static_cast<T*>(dB),
                                  static_cast<T*>(dC))))
    }
  }
  const long long na = (long long)d->dim * d->state, nd = d->dim, count = some ? slots : 0;
  scan_sum_kernel<<<(unsigned)((na + 127) / 128), 128, 0, st>>>(a.part_a, count, na, dA);
  const unsigned gd = (unsigned)((nd + 127) / 128);
  if (dD) scan_sum_kernel<<<gd, 128, 0, st>>>(a.part_d, count, nd, dD);
  if (d_dt_bias) scan_sum_kernel<<<gd, 128, 0, st>>>(some ? a.part_d + slots * nd : nullptr, count, nd, d_dt_bias);
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
  if (!aligned16(A) || !aligned16(state_pool)) return SF_ERR_ALIGNMENT;
  const int ch = kThreads / lanes(d->state);
  const dim3 grid(d->n_seq, (d->dim + ch - 1) / ch);
  if (grid.y > 65535) return SF_ERR_UNSUPPORTED;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  SF_SCAN_TYPES(d->dtype, SF_SCAN_LANES(d->state, (scan_update_kernel<T, L><<<grid, kThreads, 0, st>>>(
                                                      a, state_pool, state_indices, n_slots))))
  return cudaGetLastError() == cudaSuccess ? SF_OK : SF_ERR_CUDA;
}
