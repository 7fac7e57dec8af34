// Shared helpers of the sequence operators: rows of packed or batched
// sequences, vectors of any data type as floats, the activations.
#pragma once
#include "common.cuh"

namespace sf {
namespace seq {

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

__device__ __forceinline__ float sigmoid(float v) { return __fdividef(1.f, 1.f + __expf(-v)); }
// v / (1 + e^-v). __fdividef gives 0 for a divisor above 2^126, the limit of v / (1 + e^-v) for v -> -inf.
__device__ __forceinline__ float silu(float v) { return __fdividef(v, 1.f + __expf(-v)); }
// d silu(v) / dv
__device__ __forceinline__ float dsilu(float v) {
  const float s = sigmoid(v);
  return s * (1.f + v * (1.f - s));
}
// log(1 + e^v) without overflow, and exact to a few ulp for very negative v too
// (a time step of 1e-3 comes from v = -7).
__device__ __forceinline__ float softplus(float v) { return fmaxf(v, 0.f) + log1pf(__expf(-fabsf(v))); }

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
