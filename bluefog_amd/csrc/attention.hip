// Copyright 2026. Licensed under the Apache License, Version 2.0.
//
// Attention over packed sequences, forward and backward:
//   S = scale q k^T (within a sequence, j <= i if causal), P = softmax(S),
//   O = (P keep) v;   delta = rowsum(dO O), dP = keep (dO v^T),
//   dS = P (dP - delta), dq = scale dS k, dk = scale dS^T q, dv = (P keep)^T dO
// with dk and dv summed over the query heads that share a key/value head.

#include <hip/hip_runtime.h>

#include "convert.h"
#include "transformer_kernels.h"

namespace {

constexpr int kWaves = 4;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
  return x;
}

// the sequence that holds a row: [begin, end), empty if none does. Bounds that
// are not ordered or leave [0, rows] are cut to it, so no access leaves the
// tensors.
__device__ __forceinline__ int2 sequence_of(const BfAttnArgs& a, int row) {
  int lo = 0, hi = a.seqs;  // last b with cu[b] <= row
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.cu[mid] <= row) lo = mid; else hi = mid - 1;
  }
  if (lo >= a.seqs) return make_int2(0, 0);
  const int begin = max(a.cu[lo], 0), end = min(a.cu[lo + 1], a.rows);
  return row >= begin && row < end ? make_int2(begin, end) : make_int2(0, 0);
}

// One wave to a row and head; lane l holds columns l and l + 64.
template <typename T>
struct Row {
  float x[2];
  __device__ Row() : x{0.f, 0.f} {}
  __device__ void load(const void* base, long at, int dim, int lane) {
    const T* p = static_cast<const T*>(base) + at;
    x[0] = lane < dim ? bf_to_float(p[lane]) : 0.f;
    x[1] = lane + 64 < dim ? bf_to_float(p[lane + 64]) : 0.f;
  }
  __device__ void store(void* base, long at, int dim, int lane, float f) const {
    T* p = static_cast<T*>(base) + at;
    if (lane < dim) p[lane] = static_cast<T>(x[0] * f);
    if (lane + 64 < dim) p[lane + 64] = static_cast<T>(x[1] * f);
  }
  __device__ float dot(const Row& o) const {
    return wave_sum(x[0] * o.x[0] + x[1] * o.x[1]);
  }
  __device__ void add(const Row& o, float f) {
    x[0] += f * o.x[0];
    x[1] += f * o.x[1];
  }
};

template <typename T>
__global__ __launch_bounds__(kWaves * 64) void attn_fwd_k(BfAttnArgs a) {
  const long unit = static_cast<long>(blockIdx.x) * kWaves + threadIdx.x / 64;
  if (unit >= static_cast<long>(a.rows) * a.heads) return;
  const int lane = threadIdx.x & 63;
  const int row = static_cast<int>(unit / a.heads), h = static_cast<int>(unit % a.heads);
  const int g = h / (a.heads / a.kv_heads);
  const int2 seq = sequence_of(a, row);
  const BfKey key = a.drop.threshold ? bf_key(a.drop) : BfKey{0, 0};
  Row<T> q, o, k, v;
  q.load(a.q, row * a.q_row + h * a.q_head, a.dim, lane);
  float m = -INFINITY, l = 0.f;
  const int stop = a.causal ? min(seq.y, row + 1) : seq.y;
  for (int j = seq.x; j < stop; ++j) {
    k.load(a.k, j * a.k_row + g * a.k_head, a.dim, lane);
    v.load(a.v, j * a.v_row + g * a.v_head, a.dim, lane);
    const float s = q.dot(k) * a.scale * kLog2e;
    const float top = fmaxf(m, s), base = top == -INFINITY ? 0.f : top;
    const float shrink = exp2f(m - base), p = exp2f(s - base);
    l = l * shrink + p;
    o.x[0] *= shrink;
    o.x[1] *= shrink;
    m = top;
    const float keep = a.drop.threshold ? bf_attn_keep(h, row, j - seq.x, a.drop, key) : 1.f;
    if (keep != 0.f) o.add(v, p * keep);
  }
  o.store(a.o, unit * a.dim, a.dim, lane, stop > seq.x ? 1.f / l : 0.f);
  if (a.lse && lane == 0) a.lse[static_cast<long>(h) * a.rows + row] = m + log2f(l);
}

template <typename T>
__global__ __launch_bounds__(kWaves * 64) void attn_dq_k(BfAttnArgs a) {
  const long unit = static_cast<long>(blockIdx.x) * kWaves + threadIdx.x / 64;
  if (unit >= static_cast<long>(a.rows) * a.heads) return;
  const int lane = threadIdx.x & 63;
  const int row = static_cast<int>(unit / a.heads), h = static_cast<int>(unit % a.heads);
  const int g = h / (a.heads / a.kv_heads);
  const int2 seq = sequence_of(a, row);
  const BfKey key = a.drop.threshold ? bf_key(a.drop) : BfKey{0, 0};
  const long at = static_cast<long>(h) * a.rows + row;
  Row<T> q, o, go, k, v, dq;
  q.load(a.q, row * a.q_row + h * a.q_head, a.dim, lane);
  go.load(a.dout, row * a.do_row + h * a.do_head, a.dim, lane);
  o.load(a.out, unit * a.dim, a.dim, lane);
  const float delta = go.dot(o), lse = a.lse[at];
  if (lane == 0) a.delta[at] = delta;
  const int stop = a.causal ? min(seq.y, row + 1) : seq.y;
  // a row that sees one key has P = 1 whatever its score: dS is 0, not the
  // rounding of dP - delta
  for (int j = seq.x; j < stop && stop - seq.x > 1; ++j) {
    k.load(a.k, j * a.k_row + g * a.k_head, a.dim, lane);
    v.load(a.v, j * a.v_row + g * a.v_head, a.dim, lane);
    const float p = exp2f(q.dot(k) * a.scale * kLog2e - lse);
    const float keep = a.drop.threshold ? bf_attn_keep(h, row, j - seq.x, a.drop, key) : 1.f;
    const float dp = keep != 0.f ? keep * go.dot(v) : 0.f;
    dq.add(k, p * (dp - delta));
  }
  dq.store(a.dq, unit * a.dim, a.dim, lane, a.scale);
}

template <typename T>
__global__ __launch_bounds__(kWaves * 64) void attn_dkv_k(BfAttnArgs a) {
  const long unit = static_cast<long>(blockIdx.x) * kWaves + threadIdx.x / 64;
  if (unit >= static_cast<long>(a.rows) * a.kv_heads) return;
  const int lane = threadIdx.x & 63;
  const int j = static_cast<int>(unit / a.kv_heads), g = static_cast<int>(unit % a.kv_heads);
  const int group = a.heads / a.kv_heads;
  const int2 seq = sequence_of(a, j);
  const BfKey key = a.drop.threshold ? bf_key(a.drop) : BfKey{0, 0};
  Row<T> q, go, k, v, dk, dv;
  k.load(a.k, j * a.k_row + g * a.k_head, a.dim, lane);
  v.load(a.v, j * a.v_row + g * a.v_head, a.dim, lane);
  for (int h = g * group; h < (g + 1) * group; ++h)
    for (int row = a.causal ? max(j, seq.x) : seq.x; row < seq.y; ++row) {
      const long at = static_cast<long>(h) * a.rows + row;
      q.load(a.q, row * a.q_row + h * a.q_head, a.dim, lane);
      go.load(a.dout, row * a.do_row + h * a.do_head, a.dim, lane);
      const float p = exp2f(q.dot(k) * a.scale * kLog2e - a.lse[at]);
      const float keep = a.drop.threshold ? bf_attn_keep(h, row, j - seq.x, a.drop, key) : 1.f;
      if (keep != 0.f) dv.add(go, p * keep);
      const int sees = a.causal ? row + 1 - seq.x : seq.y - seq.x;
      if (sees > 1) {
        const float dp = keep != 0.f ? keep * go.dot(v) : 0.f;
        dk.add(q, p * (dp - a.delta[at]));
      }
    }
  dk.store(a.dk, unit * a.dim, a.dim, lane, a.scale);
  dv.store(a.dv, unit * a.dim, a.dim, lane, 1.f);
}

template <typename T>
hipError_t fwd(const BfAttnArgs& a, hipStream_t stream) {
  const long units = static_cast<long>(a.rows) * a.heads;
  hipLaunchKernelGGL(attn_fwd_k<T>, dim3((units + kWaves - 1) / kWaves), dim3(kWaves * 64), 0, stream, a);
  return hipGetLastError();
}

template <typename T>
hipError_t bwd(const BfAttnArgs& a, bool need_dkv, hipStream_t stream) {
  const long units = static_cast<long>(a.rows) * a.heads, shared = static_cast<long>(a.rows) * a.kv_heads;
  hipLaunchKernelGGL(attn_dq_k<T>, dim3((units + kWaves - 1) / kWaves), dim3(kWaves * 64), 0, stream, a);
  if (hipError_t e = hipGetLastError()) return e;
  if (!need_dkv) return hipSuccess;
  hipLaunchKernelGGL(attn_dkv_k<T>, dim3((shared + kWaves - 1) / kWaves), dim3(kWaves * 64), 0, stream, a);
  return hipGetLastError();
}

}  // namespace

extern "C" {

hipError_t bf_attn_fwd(const BfAttnArgs* a, int dtype, hipStream_t stream) {
  switch (dtype) {
    case 0: return fwd<float>(*a, stream);
    case 2: return fwd<_Float16>(*a, stream);
    case 3: return fwd<__bf16>(*a, stream);
  }
  return hipErrorInvalidValue;
}

hipError_t bf_attn_bwd(const BfAttnArgs* a, int dtype, int need_dq, int need_dkv, hipStream_t stream) {
  (void)need_dq;  // delta comes with dq
  switch (dtype) {
    case 0: return bwd<float>(*a, need_dkv, stream);
    case 2: return bwd<_Float16>(*a, need_dkv, stream);
    case 3: return bwd<__bf16>(*a, need_dkv, stream);
  }
  return hipErrorInvalidValue;
}

}  // extern "C"
