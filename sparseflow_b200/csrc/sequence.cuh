// Shared helpers of the sequence operators: rows of packed or batched
// sequences, vectors of any data type as floats, the activations.
#pragma once
#include "common.cuh"

namespace sf {
namespace seq {

typedef unsigned long long u64;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kSms = 148;  // of a B200

// 2^v and 1 / v in one instruction each, good to about two units of the last place; results below 2^-126 are 0. Every
// decay, gate and softplus takes one or two, and their pipe is what the scan runs against; a full exponential and division
// would take several instructions more. The scan in fp32 is 7e-7 off the 64-bit result, plain 32-bit operations 4e-7.
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
// Asynchronous copy of 4, 8 or 16 bytes to shared memory, zeros where `in` is false (then nothing is read).
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

// V consecutive elements of T, loaded and stored as one word where V > 1.
template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ void load_vec(float (&out)[V], const T* p) {
  const Vec<T, V> r = *reinterpret_cast<const Vec<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = DT<T>::to_f(r.v[i]);
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&in)[V]) {
  Vec<T, V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = DT<T>::from_f(in[i]);
  *reinterpret_cast<Vec<T, V>*>(p) = r;
}

// Parameters (weights, biases) come in a type of their own; they are read once
// per thread, so the type is a uniform branch rather than a template argument.
__device__ __forceinline__ float load_param(const void* p, long long i, int dtype) {
  if (dtype == SF_DTYPE_F32) return static_cast<const float*>(p)[i];
  if (dtype == SF_DTYPE_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_param(void* p, long long i, int dtype, float v) {
  if (dtype == SF_DTYPE_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == SF_DTYPE_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
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
// v / (1 + exp(-v)); where exp overflows the quotient is 0, its limit.
__device__ __forceinline__ float silu(float v) { return v * logistic(v); }
// d silu(v) / dv
__device__ __forceinline__ float dsilu(float v) {
  const float s = logistic(v);
  return s * fmaf(v, 1.f - s, 1.f);
}

// Where the rows of a sequence lie. Work on long sequences is cut into slots of `rows` rows.
struct Rows {
  const int32_t* offsets;  // packed sequences, or null
  long long length;        // rows per sequence, packed: rows in all
  int n_seq;
};
struct Span {
  int s;            // sequence
  long long begin;  // first row (packed: in the packed rows, batched: 0)
  long long len;    // rows of the sequence
  long long r0;     // first row of this slot, relative to begin
  int n_slots;      // slots of this sequence
  long long slot0;  // its first slot
};

// Slots of all sequences. Packed sequence s has its slots from off[s] / rows + s on: enough for its
// rows wherever it begins, at least one even if it is empty, and no two sequences share one.
__host__ __device__ inline long long total_slots(long long length, int n_seq, bool packed, long long rows) {
  if (packed) return length / rows + n_seq;
  return (length > 0 ? (length + rows - 1) / rows : 1) * n_seq;
}

__device__ __forceinline__ long long packed_offset(const Rows& q, int s) {
  const long long v = q.offsets[s];
  return v < 0 ? 0 : (v > q.length ? q.length : v);
}

__device__ __forceinline__ long long seq_slot0(const Rows& q, int s, long long rows) {
  return q.offsets ? packed_offset(q, s) / rows + s : s * total_slots(q.length, 1, false, rows);
}

__device__ __forceinline__ Span seq_span(const Rows& q, int s, long long rows) {
  Span p;
  p.s = s;
  p.begin = 0;
  p.len = q.length;
  p.r0 = 0;
  if (q.offsets) {
    p.begin = packed_offset(q, s);
    const long long end = packed_offset(q, s + 1);
    p.len = end > p.begin ? end - p.begin : 0;
  }
  p.slot0 = seq_slot0(q, s, rows);
  p.n_slots = p.len > 0 ? (int)((p.len + rows - 1) / rows) : 1;
  return p;
}

// The rows of a slot; len < 0 where the slot is of no sequence.
__device__ __forceinline__ Span slot_span(const Rows& q, long long slot, long long rows) {
  int s;
  if (q.offsets) {
    int lo = 0, hi = q.n_seq - 1;  // the last sequence whose first slot is at most `slot`
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (packed_offset(q, mid) / rows + mid <= slot) lo = mid;
      else hi = mid - 1;
    }
    s = lo;
  } else {
    s = (int)(slot / total_slots(q.length, 1, false, rows));
  }
  Span p = seq_span(q, s, rows);
  const long long j = slot - p.slot0;
  p.r0 = j * rows;
  if (j < 0 || j >= p.n_slots) p.len = -1;
  return p;
}

}  // namespace seq
}  // namespace sf
