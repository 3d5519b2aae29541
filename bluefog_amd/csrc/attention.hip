// Copyright 2026. Licensed under the Apache License, Version 2.0.
//
// Attention over packed sequences, forward and backward:
//   S = scale q k^T (within a sequence, j <= i if causal), P = softmax(S),
//   O = (P keep) v;   delta = rowsum(dO O), dP = keep (dO v^T),
//   dS = P (dP - delta), dq = scale dS k, dk = scale dS^T q, dv = (P keep)^T dO
// with dk and dv summed over the query heads that share a key/value head.

#include <hip/hip_runtime.h>

#include "attention_tile.h"
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

using namespace bf_attn;

// ---------------------------------------------------------------------------
// forward. A wave has 32 query rows, one to a lane of each half, and computes
// S^T = k q^T, so that a row's scores lie in the registers of its lane pair: the
// running maximum and sum cost one exchange of halves, and P^T is the operand
// of O^T = v^T P^T as it stands. The tiles of k and v go to LDS while the
// last ones are used.
// ---------------------------------------------------------------------------

template <typename T>
constexpr int kKeys = sizeof(T) == 2 ? 64 : 32;  // keys of a tile

// The accumulators are scaled down only where a maximum has grown by more than
// this (in powers of two): until then P is at most 2^8, in range of every type.
constexpr float kSlack = 8.f;

template <typename T, int DP, bool VEC, bool DROP>
__global__ __launch_bounds__(256, 2) void attn_fwd_k(BfAttnArgs a) {
  constexpr int kQ = 128, BN = kKeys<T>, kSub = BN / 32, kSteps = DP / 16, kDT = DP / 32;
  typedef Tile<T, BN, DP, 256, VEC> KV;
  __shared__ __align__(1024) char lds[2][2][KV::kBytes];
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x >> 6;
  const int h = blockIdx.x % a.heads, g = h / (a.heads / a.kv_heads);
  Work w = find_tile(a, blockIdx.x / a.heads, kQ);
  if (!w.any) return;
  if (a.causal) w.tile = w.tiles - 1 - w.tile;  // the long ones first
  const int q0 = w.tile * kQ, qw = q0 + wave * 32, qi = qw + (lane & 31);
  const bool inside = qi < w.len;
  const long row = w.begin + qi;
  T* out = static_cast<T*>(a.o) + (row * a.heads + h) * a.dim;
  Acc o[kDT];
#pragma unroll
  for (int i = 0; i < kDT; ++i) o[i] = Acc{};
  if (w.seq == a.seqs) {  // behind the last sequence
    store_row<VEC>(out, o, 0.f, half, a.dim, inside);
    if (a.lse && inside && half == 0) a.lse[static_cast<long>(h) * a.rows + row] = 0.f;
    return;
  }
  const T* q = static_cast<const T*>(a.q) + static_cast<long>(w.begin + min(qi, w.len - 1)) * a.q_row + h * a.q_head;
  const T* k = static_cast<const T*>(a.k) + static_cast<long>(w.begin) * a.k_row + g * a.k_head;
  const T* v = static_cast<const T*>(a.v) + static_cast<long>(w.begin) * a.v_row + g * a.v_head;
  const int last = w.len - 1, keys = a.causal ? min(w.len, q0 + kQ) : w.len;
  if (a.dim < DP) {
    KV::clear(&lds[0][0][0], sizeof(lds));
    __syncthreads();
  }
  KV::load(lds[0][0], k, a.k_row, 0, last, a.dim);
  KV::load(lds[0][1], v, a.v_row, 0, last, a.dim);
  Frag<T> qf[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) qf[s] = load_row<VEC>(q, s, half, a.dim);
  const BfKey key = DROP ? bf_key(a.drop) : BfKey{0, 0};
  const float c = a.scale * kLog2e;
  float m = -INFINITY, l = 0.f;  // of scores without c
  loads_done();
  for (int k0 = 0, buf = 0; k0 < keys; k0 += BN, buf ^= 1) {
    if (k0 + BN < keys) {
      KV::load(lds[buf ^ 1][0], k, a.k_row, k0 + BN, last, a.dim);
      KV::load(lds[buf ^ 1][1], v, a.v_row, k0 + BN, last, a.dim);
    }
    if (qw < w.len && !(a.causal && k0 > qw + 31)) {
      Acc s[kSub];
#pragma unroll
      for (int u = 0; u < kSub; ++u) {
        s[u] = Acc{};
#pragma unroll
        for (int i = 0; i < kSteps; ++i) s[u] = mma(KV::read_row(lds[buf][0], u * 32 + (lane & 31), i, half), qf[i], s[u]);
      }
      const bool masked = k0 + BN > w.len || (a.causal && k0 + BN - 1 > qw);
      if (masked) {
#pragma unroll
        for (int u = 0; u < kSub; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int j = k0 + u * 32 + row_of(r, half);
            if (j >= w.len || (a.causal && j > qi)) s[u][r] = -INFINITY;
          }
      }
      float top = s[0][0];
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[u][r]);
      top = fmaxf(top, swap_halves(top));
      const bool grow = (top - m) * c > kSlack || m == -INFINITY;
      if (__any(grow)) {
        const float grown = grow ? fmaxf(m, top) : m;  // a row's roundings do not depend on other rows
        const float shrink = m == -INFINITY ? 0.f : exp2f((m - grown) * c);
        l *= shrink;
#pragma unroll
        for (int i = 0; i < kDT; ++i) o[i] *= shrink;
        m = grown;
      }
      const float base = m == -INFINITY ? 0.f : m * c;  // all scores so far -inf: P = 0
      Frag<T> p[BN / 16];
#pragma unroll
      for (int u = 0; u < BN / 16; ++u) {
        uint4 bits;
        if (DROP) bits = bf_philox((k0 / 16 + u) * 2 + half, static_cast<uint32_t>(row), h, a.drop.offset, key);
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          float x = __builtin_amdgcn_exp2f(s[u / 2][(u & 1) * 8 + r] * c - base);
          l += x;
          if (DROP) x = bf_half(bits, r) >= a.drop.threshold ? x : 0.f;
          p[u][r] = static_cast<T>(x);
        }
      }
      // A masked P is 0, and 0 times a value that is no number is none: where a
      // later key's v holds one, it leaves the product and its column is set
      // for the rows that see the key.
      bool spoilt = false;
      if (masked && a.causal) {
        int found = 0;
#pragma unroll
        for (int u = 0; u < BN / 16; ++u)
#pragma unroll
          for (int i = 0; i < kDT; ++i) found |= not_finite(KV::read_columns(lds[buf][1], u * 16, i, lane));
        spoilt = __any(found);
      }
      if (!spoilt) {
#pragma unroll
        for (int u = 0; u < BN / 16; ++u)
#pragma unroll
          for (int i = 0; i < kDT; ++i) o[i] = mma(KV::read_columns(lds[buf][1], u * 16, i, lane), p[u], o[i]);
      } else {
#pragma unroll
        for (int i = 0; i < kDT; ++i) {
          Acc count{};
#pragma unroll
          for (int u = 0; u < BN / 16; ++u) {
            Frag<T> f = KV::read_columns(lds[buf][1], u * 16, i, lane), bad, seen;
#pragma unroll
            for (int r = 0; r < 8; ++r) {
              const int j = k0 + u * 16 + row_of(r, half);
              const bool fine = fabsf(static_cast<float>(f[r])) < INFINITY;
              bad[r] = static_cast<T>(fine ? 0.f : 1.f);
              f[r] = fine ? f[r] : static_cast<T>(0.f);
              seen[r] = static_cast<T>(j < w.len && j <= qi ? 1.f : 0.f);
            }
            o[i] = mma(f, p[u], o[i]);
            count = mma(bad, seen, count);
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) o[i][r] = count[r] > 0.f ? NAN : o[i][r];
        }
      }
    }
    loads_done();
  }
  l += swap_halves(l);
  store_row<VEC>(out, o, (DROP ? a.drop.scale : 1.f) / l, half, a.dim, inside);
  if (a.lse && inside && half == 0) a.lse[static_cast<long>(h) * a.rows + row] = m * c + log2f(l);
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

template <typename T, int DP, bool VEC>
hipError_t fwd(const BfAttnArgs& a, hipStream_t stream) {
  const long groups = most_tiles(a, 128) * a.heads;
  if (groups > 0x7FFFFFFF) return hipErrorInvalidValue;
  if (a.drop.threshold) hipLaunchKernelGGL((attn_fwd_k<T, DP, VEC, true>), dim3(groups), dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((attn_fwd_k<T, DP, VEC, false>), dim3(groups), dim3(256), 0, stream, a);
  return hipGetLastError();
}

template <typename T>
hipError_t fwd(const BfAttnArgs& a, hipStream_t stream) {
  if (!a.vec) return a.dim <= 64 ? fwd<T, 64, false>(a, stream) : fwd<T, 128, false>(a, stream);
  return a.dim <= 64 ? fwd<T, 64, true>(a, stream) : fwd<T, 128, true>(a, stream);
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
