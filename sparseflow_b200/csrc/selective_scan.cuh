// The kernels of the selective state space scan: a learned linear recurrence along a sequence,
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
// Layout: a lane owns 4 states of each of two channels; the LPC = ceil(state / 4) (a power of two) lanes of a channel lie
// next to each other. B and C, read once for both channels, and the sums over channels that gB and gC need are then half
// as dear; with one channel a lane shared memory was the bound (14 wavefronts a row of 8 channels). A block takes CH =
// 64 channels of one group (fewer above 16 states) through a segment of the rows, 16 rows a tile, while the tiles ahead
// are copied to a ring. Sums over the states end in a reduce-scatter over four rows and the lanes of a channel, so
// each lane finishes other rows. States past `state` have A = B = C = 0 and stay 0; rows past the end have dt = x = 0
// and change nothing.
//
// Measured (bf16, 16 states, 8192 rows of 4096 channels as 4 sequences, 537 M state steps; the exponentials alone take
// 119 us): forward 0.33 ms, backward 0.97 ms. Forward 38 instructions a warp and row of 8 channels and 5.3 exponentials
// or reciprocals (8 cycles each) at 0.52 instructions a cycle; backward 109 at 0.56: bound by the latency of each
// warp's chain, of which registers allow 12 an SM.
//
// Few channels and long sequences leave most of the GPU idle, so sequences are cut into segments: a first kernel
// finds what each segment adds to a state of 0 and how much it decays one (exp(A sum dt)), and the second starts
// each segment from the sum of those before it. The exponentials are then taken twice, so one segment is kept
// where the channels alone fill the GPU (segment_rows).
#pragma once
#include <cstring>
#include <type_traits>
#include "sequence.cuh"

namespace sf {

using seq::Rows;
using seq::Span;
using seq::u64;

constexpr int kThreads = 128;  // of the single-token kernel
constexpr int kS = 4;          // states per lane
constexpr int kMaxState = 128;
constexpr int kRows = 16;      // rows per tile, and per checkpoint
constexpr int kHalf = 8;       // rows between two additions over the warps in the backward pass
constexpr int kCpt = 2;        // channels per lane
constexpr int kPart = 4;       // rows whose states the backward pass keeps in registers
using seq::kLog2e;

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
  int wide;  // whether rows of states (A, states, their gradients) begin at 16 bytes, four of them a word
};

constexpr long long kWhole = 1ll << 40;  // seg_rows of segments that take any sequence whole

// Launches the forward or backward kernels for `lanes` lanes a channel (instantiated in a file for each type). `vec`:
// whether rows and pointers are aligned for words of four channels, and of 4 bytes of B and C.
template <typename T>
sf_status scan_forward(const ScanArgs& a, int lanes, bool vec, dim3 grid, cudaStream_t st);
template <typename T>
sf_status scan_backward(const ScanArgs& a, int lanes, bool vec, dim3 grid, cudaStream_t st);

namespace {

using namespace seq;

__device__ __forceinline__ u64 ex2x2(u64 v) {
  float lo, hi;
  unpack2(lo, hi, v);
  return pack2(ex2(lo), ex2(hi));
}

template <typename T>
__device__ __forceinline__ const T* at(const void* p, const ScanArgs& a, const Span& s, long long batch,
                                       long long row) {
  return static_cast<const T*>(p) + (a.rows.offsets ? s.begin * row : (long long)s.s * batch);
}
__device__ __forceinline__ long long row0(const ScanArgs& a, const Span& s) {
  return a.rows.offsets ? s.begin : (long long)s.s * a.rows.length;
}

// Four values of a [.., state] row of floats from state n on, 0 past the end. WIDE: as one word without asking.
template <bool WIDE = false>
__device__ __forceinline__ void load4(float (&o)[kS], const float* p, int n, const ScanArgs& a) {
  if (WIDE || a.wide) {
    if (n < a.state) {
      const float4 v = *reinterpret_cast<const float4*>(p + n);
      o[0] = v.x, o[1] = v.y, o[2] = v.z, o[3] = v.w;
    } else {
      o[0] = o[1] = o[2] = o[3] = 0.f;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < kS; ++i) o[i] = n + i < a.state ? p[n + i] : 0.f;
}
template <bool WIDE = false>
__device__ __forceinline__ void store4(float* p, const float (&v)[kS], int n, const ScanArgs& a) {
  if (WIDE || a.wide) {
    if (n < a.state) *reinterpret_cast<float4*>(p + n) = make_float4(v[0], v[1], v[2], v[3]);
    return;
  }
#pragma unroll
  for (int i = 0; i < kS; ++i)
    if (n + i < a.state) p[n + i] = v[i];
}
__device__ __forceinline__ void load4(u64 (&o)[2], const float* p, int n, const ScanArgs& a) {
  float v[kS];
  load4(v, p, n, a);
  o[0] = pack2(v[0], v[1]);
  o[1] = pack2(v[2], v[3]);
}
__device__ __forceinline__ void store4(float* p, const u64 (&v)[2], int n, const ScanArgs& a) {
  float f[kS];
  unpack2(f[0], f[1], v[0]);
  unpack2(f[2], f[3], v[1]);
  store4(p, f, n, a);
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
    if constexpr (LPC > 4) {
#pragma unroll
      for (int s = 4; s < LPC; s <<= 1) o[0] += __shfl_xor_sync(0xffffffffu, o[0], s);
    }
  }
}
template <int LPC>
__device__ __forceinline__ int scatter_row(int q) {  // the first row that lane q gets
  return LPC >= 4 ? (q & 3) : q * kRowsPerLane<LPC>;
}

template <int LPC, int CPT>
struct Cfg {
  static constexpr int CH = LPC <= 4 ? 64 : 256 / LPC;  // channels per block
  static constexpr int NP = LPC * kS;
  static constexpr int THREADS = CH * LPC / CPT;
  static constexpr int WARPS = THREADS / 32;
  static constexpr int UNITS = kRows * CH / 4;  // four channels of a row each
  static constexpr int UPT = (UNITS + THREADS - 1) / THREADS;
  static constexpr int PAD = CH + 8;            // row pitch of arrays that are read four rows at a time
};

// Where channel c lies in a row of pairs: threads write two channels (16 bytes) at a time, 32 bytes apart, and lanes
// read eight neighbouring channels; with this exchange neither conflicts.
__device__ __forceinline__ int entry(int c) { return c ^ ((c >> 3) & 2); }

template <bool VEC, typename T>
__device__ __forceinline__ void store_unit(T* p, const seq::Vec<T, 4>& v, int valid) {
  if constexpr (VEC) {
    if (valid > 0) *reinterpret_cast<seq::Vec<T, 4>*>(p) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < valid) p[i] = v.v[i];
  }
}

// The block's place: its group and channels; the lane's CPT channels, CH / CPT apart.
template <int LPC, int CPT>
struct Place {
  int g, tile, d0, ch;  // group, channel tile of the group, first channel, channels of the tile
  int c, q, n;          // this lane's first channel of the tile, lane of the channel, first state
  __device__ __forceinline__ Place(const ScanArgs& a) {
    constexpr int CH = Cfg<LPC, CPT>::CH;
    const int per = a.dim / a.groups, tiles = (per + CH - 1) / CH;
    g = blockIdx.x / tiles;
    tile = blockIdx.x % tiles;
    d0 = g * per + tile * CH;
    ch = min(CH, (g + 1) * per - d0);
    c = threadIdx.x / LPC;
    q = threadIdx.x % LPC;
    n = q * kS;
  }
  __device__ __forceinline__ int chan(int j) const { return c + j * (Cfg<LPC, CPT>::CH / CPT); }
  __device__ __forceinline__ int d(int j) const { return d0 + chan(j); }
  __device__ __forceinline__ bool own(int j) const { return chan(j) < ch; }
};

// Tiles' elements on their way: x, dt, z and dy of four channels and one row, and words of B and C, copied
// asynchronously to a ring of STAGES tiles in shared memory. A thread copies what it will convert itself, so no barrier
// guards the ring, and it has the same channels in every tile. (In registers the tile ahead was spilled, which waits
// for the loads; one tile ahead is also less than the latency of memory in the forward pass.)
// VEC: all rows begin where four channels, and 4 bytes of B and C, can be copied as one word. Otherwise 32-bit
// elements are copied one by one, and of 16-bit ones the aligned words that hold them, with a note of where they begin
// (an aligned word that holds a valid element lies in the tensor's memory).
struct Shifted4 {
  uint32_t w[3], odd;
};
struct Shifted1 {
  uint32_t w, odd;
};
template <typename T, int LPC, int CPT, bool VEC, bool X, bool Z, bool GY, bool BB, bool CC, int STAGES>
struct Ring {
  using F = Cfg<LPC, CPT>;
  static constexpr bool WHOLE = VEC || sizeof(T) == 4;
  static constexpr int ARRAYS = X + 1 + Z + GY;
  static constexpr int EPW = VEC ? 4 / (int)sizeof(T) : 1;  // elements of B and C copied together
  static constexpr int WORDS = kRows * F::NP / EPW, WPT = (WORDS + F::THREADS - 1) / F::THREADS;
  using Unit = typename std::conditional<WHOLE, seq::Vec<T, 4>, Shifted4>::type;
  using Word = typename std::conditional<WHOLE, seq::Vec<T, EPW>, Shifted1>::type;
  Unit v[STAGES][ARRAYS][F::UPT][F::THREADS];
  Word bc[STAGES][BB + CC][WPT][F::THREADS];
  float bias[F::CH], D[F::CH];
};

template <typename T, int LPC, int CPT, bool VEC, bool X, bool Z, bool GY, bool BB, bool CC, int STAGES>
struct Fetch {
  using F = Cfg<LPC, CPT>;
  using R = Ring<T, LPC, CPT, VEC, X, Z, GY, BB, CC, STAGES>;
  static constexpr int RSTEP = F::THREADS / (F::CH / 4);  // rows between a thread's units
  static constexpr int WROW = F::NP / R::EPW;             // words per row of B
  static constexpr int AX = 0, AT = X, AZ = X + 1, AG = X + 1 + Z;
  R& ring;
  const T *px, *pdt, *pz, *pgy, *pb, *pc;
  int r, m, valid;
  int put, get;  // stages

  // The first tile's rows start at t0 (of the sequence). Ends with the block's bias and D in shared memory, for the
  // barrier that follows.
  __device__ __forceinline__ Fetch(R& ring_, const ScanArgs& a, const Place<LPC, CPT>& k, const Span& p, long long t0)
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
  __device__ __forceinline__ void unit_in(typename R::Unit& dst, const T* src, int ok) {
    if constexpr (VEC) {
      cp_async(&dst, src, 4 * sizeof(T), ok > 0);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) cp_async(&dst.v[i], src + (i < ok ? i : 0), 4, i < ok);
    } else {
      const uintptr_t at = reinterpret_cast<uintptr_t>(src);
      const int odd = (int)(at >> 1) & 1;
      const uint32_t* w = reinterpret_cast<const uint32_t*>(at & ~(uintptr_t)3);
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        const bool in = ok > 0 && 2 * i - odd < ok;
        cp_async(&dst.w[i], w + (in ? i : 0), 4, in);
      }
      dst.odd = odd;
    }
  }
  __device__ __forceinline__ void word_in(typename R::Word& dst, const T* src, bool in) {
    if constexpr (R::WHOLE) {
      cp_async(&dst, src, 4, in);
    } else {
      const uintptr_t at = reinterpret_cast<uintptr_t>(src);
      cp_async(&dst.w, reinterpret_cast<const void*>(at & ~(uintptr_t)3), 4, in);
      dst.odd = (uint32_t)(at >> 1) & 1;
    }
  }
  // Starts a tile of `rows` rows at the pointers, which then move on by `next` rows. Rows below 1: nothing to copy.
  __device__ __forceinline__ void load(const ScanArgs& a, int rows, int next) {
    if (rows > 0) {
#pragma unroll
      for (int i = 0; i < F::UPT; ++i) {
        const int rr = i * RSTEP, ok = r + rr < rows ? valid : 0;
        if (X) unit_in(ring.v[put][AX][i][threadIdx.x], px + (ok ? rr * a.x_row : 0), ok);
        unit_in(ring.v[put][AT][i][threadIdx.x], pdt + (ok ? rr * a.dt_row : 0), ok);
        if (Z && a.z) unit_in(ring.v[put][AZ][i][threadIdx.x], pz + (ok ? rr * a.z_row : 0), ok);
        if (GY) unit_in(ring.v[put][AG][i][threadIdx.x], pgy + (ok ? (long long)rr * a.dim : 0), ok);
      }
      const int wr = threadIdx.x / WROW, wm = threadIdx.x % WROW * R::EPW;
#pragma unroll
      for (int i = 0; i < R::WPT; ++i) {
        const int rr = i * (F::THREADS / WROW), ok = wr + rr < rows ? a.state - wm : 0;
        if (R::WORDS % F::THREADS == 0 || threadIdx.x + i * F::THREADS < R::WORDS) {
          if (BB) word_in(ring.bc[put][0][i][threadIdx.x], pb + (ok > 0 ? rr * a.b_row : 0), ok > 0);
          if (CC) word_in(ring.bc[put][BB][i][threadIdx.x], pc + (ok > 0 ? rr * a.c_row : 0), ok > 0);
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
  // Four channels' elements; 0 past the block's channels.
  __device__ __forceinline__ seq::Vec<T, 4> unit(int array, int i) const {
    if constexpr (R::WHOLE) {
      return ring.v[get][array][i][threadIdx.x];
    } else {
      const Shifted4 w = ring.v[get][array][i][threadIdx.x];
      uint32_t p[2];
      p[0] = w.odd ? __funnelshift_r(w.w[0], w.w[1], 16) : w.w[0];
      p[1] = w.odd ? __funnelshift_r(w.w[1], w.w[2], 16) : w.w[1];
      if (valid < 4) p[1] = valid < 3 ? 0u : p[1] & 0xffffu;
      if (valid < 2) p[0] = valid < 1 ? 0u : p[0] & 0xffffu;
      seq::Vec<T, 4> v;
      memcpy(&v, p, 8);
      return v;
    }
  }
  __device__ __forceinline__ void word_out(float (&f)[R::EPW], const typename R::Word& w) const {
    if constexpr (R::WHOLE) {
      seq::load_vec<T, R::EPW>(f, w.v);
    } else {
      const uint16_t h = (uint16_t)(w.odd ? w.w >> 16 : w.w);
      T t;
      memcpy(&t, &h, 2);
      f[0] = DT<T>::to_f(t);
    }
  }
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
          word_out(f, ring.bc[get][0][i][threadIdx.x]);
          *reinterpret_cast<seq::Vec<float, R::EPW>*>(&B[rr][wm]) = *reinterpret_cast<seq::Vec<float, R::EPW>*>(f);
        }
        if (CC) {
          word_out(f, ring.bc[get][BB][i][threadIdx.x]);
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

// Whether states of these decays can grow: A > 0, or dt < 0, which softplus rules out.
__device__ __forceinline__ bool can_grow(const ScanArgs& a, const u64 (&A2)[2]) {
  float v[kS];
  unpack2(v[0], v[1], A2[0]);
  unpack2(v[2], v[3], A2[1]);
  return !a.softplus || fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])) > 0.f;
}
// 2^v h for any exponent: in two steps of half of v each, whose exponentials end at the largest number, where 2^v is past
// fp32. A state of 0 stays 0, and the product is infinite only where it is past fp32 itself.
__device__ __forceinline__ float grown(float v, float h) {
  if (v < 128.f) return ex2(v) * h;
  const float e = fminf(ex2(0.5f * v), 3.402823466e38f);
  return e * (e * h);
}
// h <- exp(A dt) h + what a tile (or segment) with that sum of dt adds to a state of 0. A long chain of states goes from
// tile to tile by this rather than row by row: a state that remembers a thousand rows is then rounded once a tile, not a
// thousand times (errors of the final states and of dA against 64 bits 1.4e-6 and 1.1e-6 row by row). Where states can
// grow, the exponential of a tile can be infinite although those of its rows are not, and times a state of 0 not a number.
__device__ __forceinline__ void add_tile(u64 (&h)[2], const u64 (&tile)[2], float dt, const u64 (&A2)[2], bool grow) {
  const u64 s = pack2(dt, dt);
  if (!grow) {
    h[0] = fma2(ex2x2(mul2(s, A2[0])), h[0], tile[0]);
    h[1] = fma2(ex2x2(mul2(s, A2[1])), h[1], tile[1]);
    return;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float v0, v1, h0, h1;
    unpack2(v0, v1, mul2(s, A2[i]));
    unpack2(h0, h1, h[i]);
    h[i] = add2(pack2(grown(v0, h0), grown(v1, h1)), tile[i]);
  }
}

// State at the start of segment j (of segment n_slots - 1 - j, going backwards): what the segments before it leave. The
// loop without a branch loads several segments at a time (with one, a prompt of 16384 rows took 499 us instead of 478).
template <bool REV, bool GROW>
__device__ __forceinline__ void add_segments(u64 (&h)[2], const ScanArgs& a, const Span& p, const u64 (&A2)[2], int j,
                                             int d, int n) {
  for (int i = 0; i < j; ++i) {
    const long long slot = p.slot0 + (REV ? p.n_slots - 1 - i : i);
    u64 e[2];
    load4(e, a.seg_state + (slot * a.dim + d) * a.state, n, a);
    add_tile(h, e, a.seg_dt[slot * a.dim + d], A2, GROW);
  }
}
template <bool REV>
__device__ __forceinline__ void segment_start(u64 (&h)[2], const ScanArgs& a, const Span& p, const u64 (&A2)[2], int j,
                                              int d, int n) {
  if (can_grow(a, A2)) add_segments<REV, true>(h, a, p, A2, j, d, n);
  else add_segments<REV, false>(h, a, p, A2, j, d, n);
}

// A log2(e) of channel j of the lane, so that exp(dt A) = 2^(dt A2).
template <int LPC, int CPT>
__device__ __forceinline__ void load_decay(u64 (&A2)[2], const ScanArgs& a, const Place<LPC, CPT>& k, int j) {
  float v[kS] = {};
  if (k.own(j)) load4(v, a.A + (long long)k.d(j) * a.state, k.n, a);
  A2[0] = pack2(v[0] * kLog2e, v[1] * kLog2e);
  A2[1] = pack2(v[2] * kLog2e, v[3] * kLog2e);
}
// (dt, dt x) of a channel and row as pairs.
__device__ __forceinline__ void load_du(u64& dt, u64& u, const float2* p) {
  const float2 v = *p;
  dt = pack2(v.x, v.x);
  u = pack2(v.y, v.y);
}

// What a segment adds to a state of 0, forwards (h = a h + dt x B) or backwards (gh = a (gh + gp C)), and its sum of
// dt. The last segment's (backwards: the first's) is not needed.
template <typename T, int LPC, int CPT, bool VEC, bool REV>
struct CarrySmem {
  using F = Cfg<LPC, CPT>;
  static constexpr int STAGES = sizeof(T) == 2 ? 4 : 3;
  float2 du[kRows][F::CH];  // dt, dt x (backwards gp)
  float B[kRows][F::NP];
  Ring<T, LPC, CPT, VEC, !REV, REV, REV, !REV, REV, STAGES> ring;
};
template <typename T, int LPC, int CPT, bool VEC, bool REV>
__global__ void __launch_bounds__(Cfg<LPC, CPT>::THREADS) scan_carry_kernel(ScanArgs a) {
  using F = Cfg<LPC, CPT>;
  using S = CarrySmem<T, LPC, CPT, VEC, REV>;
  extern __shared__ __align__(16) char smem[];
  S& sm = *reinterpret_cast<S*>(smem);
  const Place<LPC, CPT> k(a);
  const Span p = seq::slot_span(a.rows, blockIdx.y, a.seg_rows);
  if (p.len < 0) return;
  const int seg = (int)(blockIdx.y - p.slot0);
  if (REV ? seg == 0 : seg == p.n_slots - 1) return;
  const long long r1 = min(p.r0 + a.seg_rows, p.len);
  const int tiles = (int)((r1 - p.r0 + kRows - 1) / kRows);
  Fetch<T, LPC, CPT, VEC, !REV, REV, REV, !REV, REV, S::STAGES> f(sm.ring, a, k, p,
                                                            p.r0 + (REV ? (tiles - 1ll) * kRows : 0));
  auto tile_rows = [&](int i) {
    return i < tiles ? (int)min((long long)kRows, r1 - p.r0 - (long long)(REV ? tiles - 1 - i : i) * kRows) : 0;
  };
  for (int i = 0; i < S::STAGES - 1; ++i) f.load(a, tile_rows(i), REV ? -kRows : kRows);
  u64 A2[CPT][2], E[CPT][2] = {};
  float sum[CPT] = {};
  bool grow = false;
#pragma unroll
  for (int j = 0; j < CPT; ++j) {
    load_decay(A2[j], a, k, j);
    grow |= can_grow(a, A2[j]);
  }
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
        float dt[4], w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float slope;
          dt[j] = f.template step<false>(a, DT<T>::to_f(tdt.v[j]), v, j, rows, slope);
          w[j] = DT<T>::to_f(tx.v[j]);
          if (!REV) {
            w[j] *= dt[j];
          } else if (a.z) {
            const float z = DT<T>::to_f(tz.v[j]);
            w[j] *= z * logistic(z);
          }
        }
        float2* o = sm.du[f.r + v * f.RSTEP];
        *reinterpret_cast<float4*>(o + entry(f.m)) = make_float4(dt[0], w[0], dt[1], w[1]);
        *reinterpret_cast<float4*>(o + entry(f.m + 2)) = make_float4(dt[2], w[2], dt[3], w[3]);
      }
    f.convert_bc(sm.B, sm.B);
    f.done();
    f.load(a, tile_rows(i + S::STAGES - 1), REV ? -kRows : kRows);
    __syncthreads();
    u64 h[CPT][2] = {};
    float tsum[CPT] = {};
#pragma unroll
    for (int rr = 0; rr < kRows; ++rr) {
      const int r = REV ? kRows - 1 - rr : rr;
      const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(&sm.B[r][k.n]);
#pragma unroll
      for (int j = 0; j < CPT; ++j) {
        u64 dt, u;
        load_du(dt, u, &sm.du[r][entry(k.chan(j))]);
        const u64 a0 = ex2x2(mul2(dt, A2[j][0])), a1 = ex2x2(mul2(dt, A2[j][1]));
        if (REV) {
          h[j][0] = mul2(a0, fma2(u, b.x, h[j][0]));
          h[j][1] = mul2(a1, fma2(u, b.y, h[j][1]));
        } else {
          h[j][0] = fma2(a0, h[j][0], mul2(u, b.x));
          h[j][1] = fma2(a1, h[j][1], mul2(u, b.y));
        }
        tsum[j] += __uint_as_float((unsigned)dt);
      }
    }
#pragma unroll
    for (int j = 0; j < CPT; ++j) {
      sum[j] += tsum[j];
      add_tile(E[j], h[j], tsum[j], A2[j], grow);
    }
  }
#pragma unroll
  for (int j = 0; j < CPT; ++j)
    if (k.own(j)) {
      const long long o = (long long)blockIdx.y * a.dim + k.d(j);
      store4(a.seg_state + o * a.state, E[j], k.n, a);
      if (k.q == 0) a.seg_dt[o] = sum[j];
    }
}

template <typename T, int LPC, int CPT, bool VEC>
struct FwdSmem {
  using F = Cfg<LPC, CPT>;
  static constexpr int STAGES = sizeof(T) == 2 ? 4 : 3;
  float2 du[kRows][F::CH];   // dt, dt x
  float2 gx[kRows][F::PAD]; // D x, gate
  float B[kRows][F::NP], C[kRows][F::NP];
  T out[kRows][F::PAD];
  Ring<T, LPC, CPT, VEC, true, true, false, true, true, STAGES> ring;
};

// One block: one segment of a sequence and CH channels of one group. BLOCKS on an SM: three have the registers to load
// ahead over a whole tile, four hide more latency where there are as many (2048 rows, 256 blocks 0.33 / 0.38 ms, 384
// 0.43 / 0.48, 512 0.61 / 0.58).
template <typename T, int LPC, int CPT, bool VEC, int BLOCKS>
__global__ void __launch_bounds__(Cfg<LPC, CPT>::THREADS, BLOCKS) scan_fwd_kernel(ScanArgs a) {
  using F = Cfg<LPC, CPT>;
  extern __shared__ __align__(16) char smem[];
  FwdSmem<T, LPC, CPT, VEC>& s = *reinterpret_cast<FwdSmem<T, LPC, CPT, VEC>*>(smem);
  const Place<LPC, CPT> k(a);
  const Span p = seq::slot_span(a.rows, blockIdx.y, a.seg_rows);
  if (p.len < 0) return;
  const int seg = (int)(blockIdx.y - p.slot0);
  const long long r1 = min(p.r0 + a.seg_rows, p.len);
  const int tiles = (int)((r1 - p.r0 + kRows - 1) / kRows);
  constexpr int STAGES = FwdSmem<T, LPC, CPT, VEC>::STAGES;
  Fetch<T, LPC, CPT, VEC, true, true, false, true, true, STAGES> f(s.ring, a, k, p, p.r0);
  T* py = static_cast<T*>(a.y) + (row0(a, p) + p.r0 + f.r) * a.dim + k.d0 + f.m;
  auto tile_rows = [&](int i) {
    return i < tiles ? (int)min((long long)kRows, r1 - (p.r0 + (long long)i * kRows)) : 0;
  };
  auto put = [&](int rows) {  // a tile's results, four channels of a row together
#pragma unroll
    for (int v = 0; v < F::UPT; ++v) {
      const int r = f.r + v * f.RSTEP;
      if (f.has_unit(v) && r < rows)
        store_unit<VEC>(py + (long long)v * f.RSTEP * a.dim, *reinterpret_cast<const seq::Vec<T, 4>*>(&s.out[r][f.m]),
                   f.valid);
    }
    py += (long long)kRows * a.dim;
  };
  for (int i = 0; i < STAGES - 1; ++i) f.load(a, tile_rows(i), kRows);
  u64 A2[CPT][2], h[CPT][2] = {};
  float* ck[CPT] = {};
  bool grow = false;
#pragma unroll
  for (int j = 0; j < CPT; ++j) {
    load_decay(A2[j], a, k, j);
    grow |= can_grow(a, A2[j]);
    if (!k.own(j)) continue;
    if (a.init) load4(h[j], a.init + ((long long)p.s * a.dim + k.d(j)) * a.state, k.n, a);
    if (seg > 0) segment_start<false>(h[j], a, p, A2[j], seg, k.d(j), k.n);
    if (a.ck_out)
      ck[j] = a.ck_out + ((seq::seq_slot0(a.rows, p.s, kRows) + p.r0 / kRows) * a.dim + k.d(j)) * a.state;
  }
  for (int i = 0; i < tiles; ++i) {
    const int rows = tile_rows(i);
#pragma unroll
    for (int j = 0; j < CPT; ++j)
      if (ck[j]) {
        store4(ck[j], h[j], k.n, a);
        ck[j] += (long long)a.dim * a.state;
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
        float dt[4], w[4], px[4], g[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float slope;
          const float x = DT<T>::to_f(tx.v[j]);
          dt[j] = f.template step<false>(a, DT<T>::to_f(tdt.v[j]), v, j, rows, slope);
          w[j] = dt[j] * x;
          px[j] = s.ring.D[f.m + j] * x;
          g[j] = 1.f;
          if (a.z) {
            g[j] = DT<T>::to_f(tz.v[j]);
            g[j] *= logistic(g[j]);
          }
        }
        *reinterpret_cast<float4*>(&s.du[r][entry(f.m)]) = make_float4(dt[0], w[0], dt[1], w[1]);
        *reinterpret_cast<float4*>(&s.du[r][entry(f.m + 2)]) = make_float4(dt[2], w[2], dt[3], w[3]);
        *reinterpret_cast<float4*>(&s.gx[r][f.m]) = make_float4(px[0], g[0], px[1], g[1]);
        *reinterpret_cast<float4*>(&s.gx[r][f.m + 2]) = make_float4(px[2], g[2], px[3], g[3]);
      }
    f.convert_bc(s.B, s.C);
    f.done();
    f.load(a, tile_rows(i + STAGES - 1), kRows);
    __syncthreads();
    u64 start[CPT][2], tile[CPT][2] = {};  // the states before the tile, and what it adds to a state of 0
    float sum[CPT] = {};
#pragma unroll
    for (int j = 0; j < CPT; ++j) start[j][0] = h[j][0], start[j][1] = h[j][1];
#pragma unroll
    for (int r0 = 0; r0 < kRows; r0 += 4) {
      float y[CPT][4];
#pragma unroll
      for (int rr = 0; rr < 4; ++rr) {
        const int r = r0 + rr;
        const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(&s.B[r][k.n]);
        const ulonglong2 c = *reinterpret_cast<const ulonglong2*>(&s.C[r][k.n]);
#pragma unroll
        for (int j = 0; j < CPT; ++j) {
          u64 dt, u;
          load_du(dt, u, &s.du[r][entry(k.chan(j))]);
          const u64 a0 = ex2x2(mul2(dt, A2[j][0])), a1 = ex2x2(mul2(dt, A2[j][1]));
          const u64 w0 = mul2(u, b.x), w1 = mul2(u, b.y);
          h[j][0] = fma2(a0, h[j][0], w0);
          h[j][1] = fma2(a1, h[j][1], w1);
          tile[j][0] = fma2(a0, tile[j][0], w0);
          tile[j][1] = fma2(a1, tile[j][1], w1);
          sum[j] += __uint_as_float((unsigned)dt);
          y[j][rr] = sum2(fma2(c.x, h[j][0], mul2(c.y, h[j][1])));
        }
      }
#pragma unroll
      for (int j = 0; j < CPT; ++j) {
        float o[kRowsPerLane<LPC>];
        scatter4<LPC>(o, y[j], k.q);
        if (LPC <= 4 || k.q < 4)
#pragma unroll
          for (int l = 0; l < kRowsPerLane<LPC>; ++l) {
            const int r = r0 + scatter_row<LPC>(k.q) + l;
            const float2 g = s.gx[r][k.chan(j)];
            s.out[r][k.chan(j)] = DT<T>::from_f((o[l] + g.x) * g.y);
          }
      }
    }
#pragma unroll
    for (int j = 0; j < CPT; ++j) {
      add_tile(start[j], tile[j], sum[j], A2[j], grow);
      h[j][0] = start[j][0], h[j][1] = start[j][1];
    }
  }
  if (tiles > 0) {
    __syncthreads();
    put(tile_rows(tiles - 1));
  }
  if (a.final_state && seg == p.n_slots - 1)
#pragma unroll
    for (int j = 0; j < CPT; ++j)
      if (k.own(j)) store4(a.final_state + ((long long)p.s * a.dim + k.d(j)) * a.state, h[j], k.n, a);
}

template <typename T, int LPC, int CPT, bool VEC>
struct BwdSmem {
  using F = Cfg<LPC, CPT>;
  static constexpr int STAGES = 2;  // a tile takes longer than the latency of memory
  float2 du[kRows][F::CH];   // dt, dt x
  float2 gx[kRows][F::CH];   // gp, x; when a part is done: dx, -
  float2 sg[kRows][F::PAD];  // softplus'(raw), dy silu'(z); when a part is done: ddt, dz
  float B[kRows][F::NP], C[kRows][F::NP];
  float bc[2][F::WARPS][kHalf][2 * F::NP];  // sums over a warp's channels, one half tile after the other
  float4 ck[2][CPT][F::THREADS];                      // each thread's states before a tile, and before the next
  ulonglong2 hb[kRows / kPart - 1][CPT][F::THREADS];  // and before its parts but the first
  Ring<T, LPC, CPT, VEC, true, true, true, true, true, STAGES> ring;
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

// Tiles from the last to the first: a tile's states again from its checkpoint, a quarter (kPart rows) at a time in registers,
// then its rows backwards. Sums over a block's channels of gB and gC go to part_bc[tile][row][group][2][NP], added
// over the tiles by scan_bc_reduce_kernel; sums over a segment of gA, gD and gbias to part_a / part_d, added over
// the segments by scan_sum_kernel. No atomics: the order of every sum is fixed.
template <typename T, int LPC, int CPT, bool VEC>
__global__ void __launch_bounds__(Cfg<LPC, CPT>::THREADS, 3) scan_bwd_kernel(ScanArgs a) {
  using F = Cfg<LPC, CPT>;
  extern __shared__ __align__(16) char smem[];
  BwdSmem<T, LPC, CPT, VEC>& s = *reinterpret_cast<BwdSmem<T, LPC, CPT, VEC>*>(smem);
  const Place<LPC, CPT> k(a);
  const Span p = seq::slot_span(a.rows, blockIdx.y, a.seg_rows);
  const long long sd0 = (long long)blockIdx.y * a.dim;
  if (p.len < 0) {  // a slot of no sequence still has a place in the sums
    const u64 zero[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < CPT; ++j)
      if (k.own(j)) {
        const long long sd = sd0 + k.d(j);
        store4(a.part_a + sd * a.state, zero, k.n, a);
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
  const float* ck = a.ck + ((seq::seq_slot0(a.rows, p.s, kRows) + last / kRows) * a.dim + k.d0) * a.state;

  constexpr int STAGES = BwdSmem<T, LPC, CPT, VEC>::STAGES;
  Fetch<T, LPC, CPT, VEC, true, true, true, true, true, STAGES> f(s.ring, a, k, p, last);
  long long po = (r00 + last + f.r) * a.dim + k.d0 + f.m;  // where a tile's results go
  auto put = [&](int rows) {
#pragma unroll
    for (int v = 0; v < F::UPT; ++v) {
      const int r = f.r + v * f.RSTEP;
      if (f.has_unit(v) && r < rows) {
        const long long o = po + (long long)v * f.RSTEP * a.dim;
        seq::Vec<T, 4> dx, ddt, dz;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          dx.v[j] = DT<T>::from_f(s.gx[r][entry(f.m + j)].x);
          ddt.v[j] = DT<T>::from_f(s.sg[r][f.m + j].x);
          dz.v[j] = DT<T>::from_f(s.sg[r][f.m + j].y);
        }
        store_unit<VEC>(static_cast<T*>(a.dx) + o, dx, f.valid);
        store_unit<VEC>(static_cast<T*>(a.ddt) + o, ddt, f.valid);
        if (a.dz) store_unit<VEC>(static_cast<T*>(a.dz) + o, dz, f.valid);
      }
    }
    po -= (long long)kRows * a.dim;
  };
  // The checkpoint of a tile into this thread's place of it, in the copies' group of the tile above.
  auto load_ck = [&](int i) {
#pragma unroll
    for (int j = 0; j < CPT; ++j) {
      float4* dst = &s.ck[i & 1][j][threadIdx.x];
      const float* src = ck + (long long)k.chan(j) * a.state;
      if (a.wide) {
        cp_async(dst, k.own(j) && k.n < a.state ? src + k.n : a.ck, 16, k.own(j) && k.n < a.state);
      } else {
        float v[kS] = {};
        if (k.own(j)) load4(v, src, k.n, a);
        *dst = make_float4(v[0], v[1], v[2], v[3]);
      }
    }
    ck -= (long long)a.dim * a.state;
  };
  const int last_rows = (int)(r1 - last);
  auto tile_rows = [&](int i) { return i < 0 ? 0 : i == tiles - 1 ? last_rows : kRows; };
  if (tiles > 0) load_ck(tiles - 1);
  for (int i = 0; i < STAGES - 1; ++i) f.load(a, tile_rows(tiles - 1 - i), -kRows);
  u64 A2[CPT][2], gh[CPT][2] = {}, gA[CPT][2] = {};
  float D[CPT], gD[CPT] = {}, gbias[CPT] = {};
#pragma unroll
  for (int j = 0; j < CPT; ++j) {
    load_decay(A2[j], a, k, j);
    D[j] = a.D && k.own(j) ? a.D[k.d(j)] : 0.f;
    if (!k.own(j)) continue;
    if (a.dfinal) load4(gh[j], a.dfinal + ((long long)p.s * a.dim + k.d(j)) * a.state, k.n, a);
    if (seg < p.n_slots - 1) segment_start<true>(gh[j], a, p, A2[j], p.n_slots - 1 - seg, k.d(j), k.n);
  }
  const int first = sums_first<LPC>(lane);
  for (int i = tiles - 1; i >= 0; --i) {
    const int rows = tile_rows(i);
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
        float slope[4], gz[4], dt[4], x[4], g[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          dt[j] = f.template step<true>(a, DT<T>::to_f(tdt.v[j]), v, j, rows, slope[j]);
          x[j] = DT<T>::to_f(tx.v[j]);
          g[j] = DT<T>::to_f(tg.v[j]);
          gz[j] = 0.f;
          if (a.z) {
            const float z = DT<T>::to_f(tz.v[j]), sig = logistic(z);
            gz[j] = g[j] * (sig * fmaf(z, 1.f - sig, 1.f));
            g[j] *= z * sig;
          }
        }
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          const int m = f.m + j, en = entry(m);
          *reinterpret_cast<float4*>(&s.du[r][en]) = make_float4(dt[j], dt[j] * x[j], dt[j + 1], dt[j + 1] * x[j + 1]);
          *reinterpret_cast<float4*>(&s.gx[r][en]) = make_float4(g[j], x[j], g[j + 1], x[j + 1]);
          *reinterpret_cast<float4*>(&s.sg[r][m]) = make_float4(slope[j], gz[j], slope[j + 1], gz[j + 1]);
        }
      }
    f.convert_bc(s.B, s.C);
    f.done();
    if (i > 0) load_ck(i - 1);
    f.load(a, tile_rows(i - (STAGES - 1)), -kRows);
    __syncthreads();
    const int parts = (rows + kPart - 1) / kPart;
    {
      u64 h[CPT][2];
#pragma unroll
      for (int j = 0; j < CPT; ++j) {
        const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&s.ck[i & 1][j][threadIdx.x]);
        h[j][0] = v.x, h[j][1] = v.y;
      }
#pragma unroll 1
      for (int part = 0; part < parts - 1; ++part) {
#pragma unroll
        for (int r = 0; r < kPart; ++r) {
          const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(&s.B[part * kPart + r][k.n]);
#pragma unroll
          for (int j = 0; j < CPT; ++j) {
            u64 dt, u;
            load_du(dt, u, &s.du[part * kPart + r][entry(k.chan(j))]);
            h[j][0] = fma2(ex2x2(mul2(dt, A2[j][0])), h[j][0], mul2(u, b.x));
            h[j][1] = fma2(ex2x2(mul2(dt, A2[j][1])), h[j][1], mul2(u, b.y));
          }
        }
#pragma unroll
        for (int j = 0; j < CPT; ++j) s.hb[part][j][threadIdx.x] = make_ulonglong2(h[j][0], h[j][1]);
      }
    }
    u64 tA[CPT][2] = {};  // this tile's share of gA: sums of sums keep more digits than one long one
#pragma unroll 1
    for (int part = parts - 1; part >= 0; --part) {
      const int t = part * kPart;
      u64 hs[CPT][kPart + 1][2], as[CPT][kPart][2];
#pragma unroll
      for (int j = 0; j < CPT; ++j) {
        const ulonglong2 v = part > 0 ? s.hb[part - 1][j][threadIdx.x]
                                      : *reinterpret_cast<const ulonglong2*>(&s.ck[i & 1][j][threadIdx.x]);
        hs[j][0][0] = v.x, hs[j][0][1] = v.y;
      }
#pragma unroll
      for (int r = 0; r < kPart; ++r) {
        const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(&s.B[t + r][k.n]);
#pragma unroll
        for (int j = 0; j < CPT; ++j) {
          u64 dt, u;
          load_du(dt, u, &s.du[t + r][entry(k.chan(j))]);
          as[j][r][0] = ex2x2(mul2(dt, A2[j][0]));
          as[j][r][1] = ex2x2(mul2(dt, A2[j][1]));
          hs[j][r + 1][0] = fma2(as[j][r][0], hs[j][r][0], mul2(u, b.x));
          hs[j][r + 1][1] = fma2(as[j][r][1], hs[j][r][1], mul2(u, b.y));
        }
      }
      float pre[CPT][4], S[CPT][4], qa[CPT][4];
#pragma unroll
      for (int r = kPart - 1; r >= 0; --r) {
        const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(&s.B[t + r][k.n]);
        const ulonglong2 c = *reinterpret_cast<const ulonglong2*>(&s.C[t + r][k.n]);
        u64 vb[2], vc[2];
#pragma unroll
        for (int j = 0; j < CPT; ++j) {
          u64 dt, u;
          load_du(dt, u, &s.du[t + r][entry(k.chan(j))]);
          const float g1 = s.gx[t + r][entry(k.chan(j))].x;
          const u64 gp = pack2(g1, g1);
          pre[j][r] = sum2(fma2(c.x, hs[j][r + 1][0], mul2(c.y, hs[j][r + 1][1])));
          gh[j][0] = fma2(gp, c.x, gh[j][0]);
          gh[j][1] = fma2(gp, c.y, gh[j][1]);
          S[j][r] = sum2(fma2(gh[j][0], b.x, mul2(gh[j][1], b.y)));
          vb[0] = j ? fma2(gh[j][0], u, vb[0]) : mul2(gh[j][0], u);
          vb[1] = j ? fma2(gh[j][1], u, vb[1]) : mul2(gh[j][1], u);
          vc[0] = j ? fma2(gp, hs[j][r + 1][0], vc[0]) : mul2(gp, hs[j][r + 1][0]);
          vc[1] = j ? fma2(gp, hs[j][r + 1][1], vc[1]) : mul2(gp, hs[j][r + 1][1]);
          gh[j][0] = mul2(gh[j][0], as[j][r][0]);
          gh[j][1] = mul2(gh[j][1], as[j][r][1]);
          const u64 q0 = mul2(gh[j][0], hs[j][r][0]), q1 = mul2(gh[j][1], hs[j][r][1]);
          qa[j][r] = sum2(fma2(q0, A2[j][0], mul2(q1, A2[j][1])));
          tA[j][0] = fma2(q0, dt, tA[j][0]);
          tA[j][1] = fma2(q1, dt, tA[j][1]);
        }
        float v[8];
        unpack2(v[0], v[1], vb[0]);
        unpack2(v[2], v[3], vb[1]);
        unpack2(v[4], v[5], vc[0]);
        unpack2(v[6], v[7], vc[1]);
        channels_sum<LPC>(v, lane);
        // value i < 4: state n + i of gB, else of gC
        if (LPC >= 4 || (lane & 3 & ~(LPC - 1)) == 0)
#pragma unroll
          for (int j = 0; j < kSumsPerLane<LPC>; ++j)
            s.bc[part >> 1 & 1][warp][t % kHalf + r][((first + j) >> 2) * F::NP + k.n + ((first + j) & 3)] = v[j];
      }
#pragma unroll
      for (int j = 0; j < CPT; ++j) {
        float po4[kRowsPerLane<LPC>], So[kRowsPerLane<LPC>], qo[kRowsPerLane<LPC>];
        scatter4<LPC>(po4, pre[j], k.q);
        scatter4<LPC>(So, S[j], k.q);
        scatter4<LPC>(qo, qa[j], k.q);
        if (LPC <= 4 || k.q < 4)
#pragma unroll
          for (int l = 0; l < kRowsPerLane<LPC>; ++l) {
            const int r = t + scatter_row<LPC>(k.q) + l, c = k.chan(j);
            const float2 g = s.gx[r][entry(c)], sg = s.sg[r][c];
            const float dt = s.du[r][entry(c)].x;
            const float gdt = fmaf(g.y, So[l], qo[l] * (1.f / kLog2e)) * sg.x;
            s.gx[r][entry(c)].x = fmaf(dt, So[l], D[j] * g.x);
            s.sg[r][c] = make_float2(gdt, fmaf(D[j], g.y, po4[l]) * sg.y);
            gD[j] = fmaf(g.x, g.y, gD[j]);
            gbias[j] += r < rows ? gdt : 0.f;
          }
      }
      if (t % kHalf == 0) {  // both parts of a half are done
        __syncthreads();
        for (int u = threadIdx.x; u < kHalf * 2 * F::NP; u += F::THREADS) {
          const int r = u / (2 * F::NP), m = u % (2 * F::NP);
          float v = 0.f;
#pragma unroll
          for (int w = 0; w < F::WARPS; ++w) v += s.bc[part >> 1 & 1][w][r][m];
          if (t + r < rows) bc_out[(long long)(t + r) * a.groups * 2 * F::NP + m] = v;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < CPT; ++j) {
      gA[j][0] = add2(gA[j][0], tA[j][0]);
      gA[j][1] = add2(gA[j][1], tA[j][1]);
    }
    bc_out -= (long long)kRows * a.groups * 2 * F::NP;
  }
  if (tiles > 0) {
    __syncthreads();
    put(tile_rows(0));
  }
#pragma unroll
  for (int j = 0; j < CPT; ++j) {
    const float d = lanes_sum<(LPC < 4 ? LPC : 4)>(gD[j]), bias = lanes_sum<(LPC < 4 ? LPC : 4)>(gbias[j]);
    if (!k.own(j)) continue;
    const long long sd = sd0 + k.d(j);
    if (a.dinit && seg == 0) store4(a.dinit + ((long long)p.s * a.dim + k.d(j)) * a.state, gh[j], k.n, a);
    store4(a.part_a + sd * a.state, gA[j], k.n, a);
    if (k.q == 0) {
      a.part_d[sd] = d;
      a.part_d[(long long)gridDim.y * a.dim + sd] = bias;
    }
  }
}

template <typename K>
bool prepare_smem(K kernel, size_t bytes) {
  return bytes <= 48 * 1024 || allow_max_smem(reinterpret_cast<const void*>(kernel));
}

template <typename T, int LPC, int CPT, bool VEC>
sf_status run_fwd(const ScanArgs& a, dim3 grid, cudaStream_t st) {
  constexpr int threads = Cfg<LPC, CPT>::THREADS;
  if (a.seg_rows != kWhole) {
    constexpr size_t bytes = sizeof(CarrySmem<T, LPC, CPT, VEC, false>);
    if (!prepare_smem(scan_carry_kernel<T, LPC, CPT, VEC, false>, bytes)) return SF_ERR_CUDA;
    scan_carry_kernel<T, LPC, CPT, VEC, false><<<grid, threads, bytes, st>>>(a);
  }
  constexpr size_t smem = sizeof(FwdSmem<T, LPC, CPT, VEC>);
  auto kernel = (long long)grid.x * grid.y > 3 * kSms ? scan_fwd_kernel<T, LPC, CPT, VEC, 4>
                                                     : scan_fwd_kernel<T, LPC, CPT, VEC, 3>;
  if (!prepare_smem(kernel, smem)) return SF_ERR_CUDA;
  kernel<<<grid, threads, smem, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? SF_OK : SF_ERR_CUDA;
}
template <typename T, int LPC, int CPT, bool VEC>
sf_status run_bwd(const ScanArgs& a, dim3 grid, cudaStream_t st) {
  constexpr int threads = Cfg<LPC, CPT>::THREADS;
  if (a.seg_rows != kWhole) {
    constexpr size_t bytes = sizeof(CarrySmem<T, LPC, CPT, VEC, true>);
    if (!prepare_smem(scan_carry_kernel<T, LPC, CPT, VEC, true>, bytes)) return SF_ERR_CUDA;
    scan_carry_kernel<T, LPC, CPT, VEC, true><<<grid, threads, bytes, st>>>(a);
  }
  constexpr size_t smem = sizeof(BwdSmem<T, LPC, CPT, VEC>);
  if (!prepare_smem(scan_bwd_kernel<T, LPC, CPT, VEC>, smem)) return SF_ERR_CUDA;
  scan_bwd_kernel<T, LPC, CPT, VEC><<<grid, threads, smem, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? SF_OK : SF_ERR_CUDA;
}

template <typename T, bool VEC, bool BWD>
sf_status run_lanes(const ScanArgs& a, int lanes, dim3 grid, cudaStream_t st) {
  auto run = [&](auto l) {
    constexpr int LPC = decltype(l)::value;
    return BWD ? run_bwd<T, LPC, kCpt, VEC>(a, grid, st) : run_fwd<T, LPC, kCpt, VEC>(a, grid, st);
  };
  switch (lanes) {
    case 1: return run(std::integral_constant<int, 1>());
    case 2: return run(std::integral_constant<int, 2>());
    case 4: return run(std::integral_constant<int, 4>());
    case 8: return run(std::integral_constant<int, 8>());
    case 16: return run(std::integral_constant<int, 16>());
    default: return run(std::integral_constant<int, 32>());
  }
}

}  // namespace

template <typename T>
sf_status scan_forward(const ScanArgs& a, int lanes, bool vec, dim3 grid, cudaStream_t st) {
  return vec ? run_lanes<T, true, false>(a, lanes, grid, st) : run_lanes<T, false, false>(a, lanes, grid, st);
}
template <typename T>
sf_status scan_backward(const ScanArgs& a, int lanes, bool vec, dim3 grid, cudaStream_t st) {
  return vec ? run_lanes<T, true, true>(a, lanes, grid, st) : run_lanes<T, false, true>(a, lanes, grid, st);
}

}  // namespace sf
