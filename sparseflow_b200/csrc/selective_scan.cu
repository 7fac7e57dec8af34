// Selective state space scan: the C entries, the sums over blocks that end the backward pass, and the single-token
// form (one launch: the states of a channel are read, moved one step and written once; HBM-bound).
#include "selective_scan.cuh"

namespace sf {
extern template sf_status scan_forward<float>(const ScanArgs&, int, bool, dim3, cudaStream_t);
extern template sf_status scan_forward<__half>(const ScanArgs&, int, bool, dim3, cudaStream_t);
extern template sf_status scan_forward<__nv_bfloat16>(const ScanArgs&, int, bool, dim3, cudaStream_t);
extern template sf_status scan_backward<float>(const ScanArgs&, int, bool, dim3, cudaStream_t);
extern template sf_status scan_backward<__half>(const ScanArgs&, int, bool, dim3, cudaStream_t);
extern template sf_status scan_backward<__nv_bfloat16>(const ScanArgs&, int, bool, dim3, cudaStream_t);

namespace {

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

// dA [na], dD and dbias [nd] (each may be null): sums over `count` segments of part_a [count][na] and part_d [2][count][nd],
// in order.
__global__ void scan_sum_kernel(const float* part_a, const float* part_d, long long count, long long na, long long nd,
                                float* dA, float* dD, float* dbias) {
  long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const float* p = part_a;
  float* out = dA;
  long long n = na;
  if (i >= na) {
    i -= na;
    n = nd;
    p = part_d;
    out = dD;
    if (i >= nd) {
      i -= nd;
      p += count * nd;
      out = dbias;
    }
    if (i >= nd) return;
  }
  if (!out) return;
  float v = 0.f;
#pragma unroll 8
  for (long long j = 0; j < count; ++j) v += p[j * n + i];
  out[i] = v;
}

// Single tokens. Memory-bound: 32 bytes of states moved for 4 exponentials a lane. A lane has 4 states of one channel
// for 4 rows, so that A (a third of the bytes of one row) is read once for all of them; what is per channel and row
// (softplus, the gate) is done by one lane for each row and handed on by shuffles. All loads come before the first use
// and without branches: rows of padding and channels past the end read a valid place and write nothing.
// VEC: rows of A, the states, B and C can be moved four elements at a time, which is not asked again where they are: the
// branches cost registers (256 rows of 5120 channels of 16 states: 40.8 us with them, 34.6 without, 5.2 TB/s).
template <typename T, int LPC, bool VEC>
__global__ void __launch_bounds__(kThreads, 8) scan_update_kernel(ScanArgs a, float* pool, const int32_t* idx,
                                                               int n_slots) {
  constexpr int CH = kThreads / LPC, RPL = kRowsPerLane<LPC>;
  const int lane = threadIdx.x & 31, q = threadIdx.x % LPC, n = q * kS;
  const int c = blockIdx.x * CH + threadIdx.x / LPC, d = min(c, a.dim - 1);
  const int row0 = blockIdx.y * 4, rows = a.rows.n_seq, g = d / (a.dim / a.groups);
  const int mine = scatter_row<LPC>(q);  // the first of this lane's RPL rows
  int slot[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int row = min(row0 + r, rows - 1);
    slot[r] = idx ? idx[row] : row;
    if (slot[r] >= n_slots || c >= a.dim || row0 + r >= rows) slot[r] = -1;
  }
  float h[4][kS], Bv[4][kS], Cv[4][kS], A[kS], x[RPL], dt[RPL], z[RPL];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const long long row = min(row0 + r, rows - 1);
    const T* Bp = static_cast<const T*>(a.B) + row * a.b_row + (long long)g * a.state;
    const T* Cp = static_cast<const T*>(a.C) + row * a.c_row + (long long)g * a.state;
    if (VEC) {  // the state is a multiple of 4; lanes past it have h = 0
      const int m = min(n, a.state - kS);
      seq::load_vec<T, kS>(Bv[r], Bp + m);
      seq::load_vec<T, kS>(Cv[r], Cp + m);
    } else {
#pragma unroll
      for (int i = 0; i < kS; ++i) {
        Bv[r][i] = n + i < a.state ? DT<T>::to_f(Bp[n + i]) : 0.f;
        Cv[r][i] = n + i < a.state ? DT<T>::to_f(Cp[n + i]) : 0.f;
      }
    }
  }
#pragma unroll
  for (int l = 0; l < RPL; ++l) {
    const long long row = min(row0 + mine + l, rows - 1);
    dt[l] = DT<T>::to_f(static_cast<const T*>(a.dt)[row * a.dt_row + d]);
    x[l] = DT<T>::to_f(static_cast<const T*>(a.x)[row * a.x_row + d]);
    z[l] = a.z ? DT<T>::to_f(static_cast<const T*>(a.z)[row * a.z_row + d]) : 0.f;
  }
  load4<VEC>(A, a.A + (long long)d * a.state, n, a);
  const float bias = a.dt_bias ? a.dt_bias[d] : 0.f, D = a.D ? a.D[d] : 0.f;
  // The states last: their addresses wait for the slots.
#pragma unroll
  for (int r = 0; r < 4; ++r)
    load4<VEC>(h[r], pool + ((long long)max(slot[r], 0) * a.dim + d) * a.state, n, a);
#pragma unroll
  for (int i = 0; i < kS; ++i) A[i] *= kLog2e;
  float u[RPL], y[4];
#pragma unroll
  for (int l = 0; l < RPL; ++l) {
    float e;
    dt[l] += bias;
    if (a.softplus) dt[l] = softplus(dt[l], e);
    u[l] = dt[l] * x[l];
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    float step, w;
    if constexpr (LPC == 1) {
      step = dt[r];
      w = u[r];
    } else {
      const int from = (lane & ~(LPC - 1)) | r / RPL;
      step = __shfl_sync(0xffffffffu, dt[r % RPL], from);
      w = __shfl_sync(0xffffffffu, u[r % RPL], from);
    }
    y[r] = 0.f;
#pragma unroll
    for (int i = 0; i < kS; ++i) {
      // A lane past the state (VEC) has read other states' B and C: its own stay 0.
      const float b = VEC && LPC > 1 && n >= a.state ? 0.f : Bv[r][i];
      h[r][i] = fmaf(ex2(step * A[i]), h[r][i], w * b);
      y[r] = fmaf(Cv[r][i], h[r][i], y[r]);
    }
    if (slot[r] >= 0) store4<VEC>(pool + ((long long)slot[r] * a.dim + d) * a.state, h[r], n, a);
  }
  float o[RPL];
  scatter4<LPC>(o, y, q);
  if ((LPC > 4 && q >= 4) || c >= a.dim) return;
#pragma unroll
  for (int l = 0; l < RPL; ++l) {
    const int r = mine + l;
    if (row0 + r >= rows) continue;
    float v = fmaf(D, x[l], o[l]);
    if (a.z) v *= seq::silu(z[l]);
    const int s = idx ? idx[row0 + r] : row0 + r;
    static_cast<T*>(a.y)[(long long)(row0 + r) * a.dim + d] = DT<T>::from_f(s >= 0 && s < n_slots ? v : 0.f);
  }
}

template <typename T, int LPC, bool VEC>
void run_update(const ScanArgs& a, float* pool, const int32_t* idx, int n_slots, cudaStream_t st) {
  constexpr int CH = kThreads / LPC;
  const unsigned tiles = (a.dim + CH - 1) / CH;
  scan_update_kernel<T, LPC, VEC>
      <<<dim3(tiles, (a.rows.n_seq + 3) / 4), kThreads, 0, st>>>(a, pool, idx, n_slots);
}

bool valid(const sf_selective_scan_desc* d) {
  return d && d->length >= 0 && d->n_seq >= 0 && d->dim >= 0 && d->state >= 1 && d->groups >= 1 &&
         d->dim % d->groups == 0 && dtype_size(d->dtype) != 0;
}
// Whether buffers can be sized: blocks have channels up to kMaxState states.
bool sized(const sf_selective_scan_desc* d) { return valid(d) && d->state <= kMaxState; }
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

// Rows per segment. Measured on a B200 (bf16, 16 states, sequences of 2048 rows, times in ms): whole, a block takes as
// long alone on its SM as t[0], two or more together as t[1], t[2] ..; cut into about 1400 blocks in all, so that the
// last round of them is short beside the rest, the time goes with the work, `cut` a block's sequence (the kernel that
// finds the segments' shares included). Whole against cut, forward: 64 blocks 0.25 / 0.14, 128: 0.25 / 0.24, 192:
// 0.33 / 0.36, 256: 0.33 / 0.48, 512: 0.58 / 0.95; backward: 128 blocks 0.76 / 0.52, 256: 1.02 / 0.96, 320: 1.29 / 1.16,
// 384: 1.29 / 1.39, 512: 1.97 / 1.86. The cheaper is taken; 0.01 ms stands for the launch that cutting adds. Packed
// sequences count as of equal length (the host does not know theirs). The costs of 16 states in bf16 stand for all: of 4
// to 128 states in bf16 and fp32, 512 to 8192 rows and 64 to 512 blocks, the choice was within 8 % of the better one, but
// for 128 blocks of 512 rows of up to 8 states, kept whole (0.14 ms, cut 0.07), 256 of 4 states (0.14, cut 0.12) and, cut,
// the backward pass of 512 blocks of up to 8 states in bf16 (2.05 ms with the forward pass, whole 1.80), of 256 blocks in
// fp32 (1.48 / 1.35) and of 64 or more states (1.57 / 1.46).
struct SegmentCosts {
  int resident;  // blocks on an SM
  double t[4], cut;
};
constexpr SegmentCosts kFwdCosts = {4, {0.250, 0.327, 0.430, 0.580}, 1.86e-3};
constexpr SegmentCosts kBwdCosts = {3, {0.750, 1.000, 1.290, 0.}, 3.62e-3};

long long segment_rows(const sf_selective_scan_desc* d, const SegmentCosts& k) {
  if (d->n_seq == 0 || d->length == 0) return kWhole;
  const long long across = (long long)tiles_of(d) * d->groups, blocks = across * d->n_seq;
  const long long total = d->packed ? d->length : d->length * d->n_seq;
  const double length = (double)total / d->n_seq / 2048.;
  const long long w = (blocks + seq::kSms - 1) / seq::kSms;
  double whole = (double)(w / k.resident) * k.t[k.resident - 1];
  if (w % k.resident) whole += k.t[w % k.resident - 1];
  if (whole * length <= k.cut * blocks * length + 0.01) return kWhole;
  long long rows = (total * across + 1399) / 1400;
  if (rows < 64) rows = 64;
  if (rows < (d->length + 63) / 64) rows = (d->length + 63) / 64;
  rows = (rows + kRows - 1) / kRows * kRows;
  return rows >= d->length ? kWhole : rows;
}
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

// Whether rows of states can be read and written as words of four, in every tensor that has them.
bool states_fit(const sf_selective_scan_desc* d, std::initializer_list<const void*> ptrs) {
  if (d->state % kS) return false;
  for (const void* p : ptrs)
    if (!aligned16(p)) return false;
  return true;
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
  if (d->dtype == SF_DTYPE_F32) return true;
  if (d->state % 2 || d->b_row_stride % 2 || d->c_row_stride % 2) return false;
  if (!d->packed && d->n_seq > 1 && (d->b_batch_stride % 2 || d->c_batch_stride % 2)) return false;
  for (const void* p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) % 4) return false;
  return true;
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
  if (!sized(d)) return 0;
  return (size_t)seq::total_slots(d->length, d->n_seq, d->packed, kRows) * d->dim * d->state * sizeof(float);
}

extern "C" size_t sf_selective_scan_workspace_size(const sf_selective_scan_desc* d) {
  if (!sized(d) || d->n_seq == 0) return 0;
  return (size_t)carry_floats(d, segment_rows(d, kFwdCosts)) * sizeof(float);
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
  const bool vec = vectors_fit(d, {x, dt, z, y}) && words_fit(d, {B, C});
  a.seg_rows = segment_rows(d, kFwdCosts);
  const long long carry = carry_floats(d, a.seg_rows), slots = slots_of(d, a.seg_rows);
  if (carry && (!workspace || workspace_bytes < (size_t)carry * sizeof(float))) return SF_ERR_WORKSPACE;
  if (!aligned16(checkpoints) || (carry && !aligned16(workspace))) return SF_ERR_ALIGNMENT;
  a.wide = states_fit(d, {A, initial_state, final_state});
  if (slots > 65535) return SF_ERR_UNSUPPORTED;
  a.seg_state = static_cast<float*>(workspace);
  a.seg_dt = a.seg_state + slots * d->dim * d->state;
  const dim3 grid(tiles_of(d) * d->groups, (unsigned)slots);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  sf_status status = SF_OK;
  SF_SCAN_TYPES(d->dtype, status = scan_forward<T>(a, lanes(d->state), vec, grid, st))
  return status;
}

extern "C" size_t sf_selective_scan_backward_workspace_size(const sf_selective_scan_desc* d) {
  if (!sized(d)) return 0;
  return (size_t)bwd_layout(d, segment_rows(d, kBwdCosts)).total * sizeof(float);
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
  const long long seg = segment_rows(d, kBwdCosts), slots = slots_of(d, seg);
  const BwdLayout l = bwd_layout(d, seg);
  if (some && (!workspace || workspace_bytes < (size_t)l.total * sizeof(float))) return SF_ERR_WORKSPACE;
  if (some && (!aligned16(workspace) || !aligned16(checkpoints))) return SF_ERR_ALIGNMENT;
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
  a.wide = states_fit(d, {A, d_final_state, d_initial_state});
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (some) {
    a.part_bc = ws + l.bc;
    a.part_a = ws + l.a;
    a.part_d = ws + l.d;
    a.seg_rows = seg;
    a.seg_state = ws + l.carry;
    a.seg_dt = a.seg_state + slots * d->dim * d->state;
    const bool vec = vectors_fit(d, {x, dt, z, dy, dx, ddt, dz}) && words_fit(d, {B, C});
    const dim3 grid(tiles_of(d) * d->groups, (unsigned)slots);
    sf_status status = SF_OK;
    SF_SCAN_TYPES(d->dtype, status = scan_backward<T>(a, lanes(d->state), vec, grid, st))
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
  scan_sum_kernel<<<(unsigned)((na + 2 * nd + 127) / 128), 128, 0, st>>>(a.part_a, a.part_d, count, na, nd, dA, dD,
                                                                         d_dt_bias);
  return cudaGetLastError() == cudaSuccess ? SF_OK : SF_ERR_CUDA;
}

extern "C" sf_status sf_selective_scan_update(const void* x, const void* dt, const float* A, const void* B,
                                              const void* C, const float* D, const void* z, const float* dt_bias,
                                              float* state_pool, const int32_t* state_indices, void* y,
                                              int32_t n_slots, const sf_selective_scan_desc* d, void* stream) {
  if (!valid(d) || !A || n_slots < 0) return SF_ERR_INVALID_ARG;
  if (d->state > kMaxState) return SF_ERR_UNSUPPORTED;
  if (d->n_seq == 0 || d->dim == 0) return SF_OK;
  if (!x || !dt || !B || !C || !y || (!state_pool && n_slots > 0)) return SF_ERR_INVALID_ARG;
  if (n_slots == 0)  // every row is padding
    return cudaMemsetAsync(y, 0, (size_t)d->n_seq * d->dim * dtype_size(d->dtype), static_cast<cudaStream_t>(stream)) ==
                   cudaSuccess
               ? SF_OK
               : SF_ERR_CUDA;
  if (d->n_seq > 4 * 65535) return SF_ERR_UNSUPPORTED;  // a block has four rows
  ScanArgs a = base_args(x, dt, A, B, C, D, z, dt_bias, nullptr, d);
  a.y = y;
  a.wide = states_fit(d, {A, state_pool});
  const bool vec = a.wide && d->b_row_stride % 4 == 0 && d->c_row_stride % 4 == 0 &&
                   reinterpret_cast<uintptr_t>(B) % (4 * dtype_size(d->dtype)) == 0 &&
                   reinterpret_cast<uintptr_t>(C) % (4 * dtype_size(d->dtype)) == 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  SF_SCAN_TYPES(d->dtype,
                SF_SCAN_LANES(d->state, (vec ? run_update<T, L, true>(a, state_pool, state_indices, n_slots, st)
                                             : run_update<T, L, false>(a, state_pool, state_indices, n_slots, st))))
  return cudaGetLastError() == cudaSuccess ? SF_OK : SF_ERR_CUDA;
}
