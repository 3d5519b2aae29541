// Copyright 2026. Licensed under the Apache License, Version 2.0.
//
// Layer norm over rows, forward and backward, and dropout:
//   z = r + keep x,  y = (z - mean) rstd w + b
//   g = dy w,  dz = rstd (g - mean(g) - xhat mean(g xhat)),
//   dr = dz,  dx = keep dz,  dw = sum_rows dy xhat,  db = sum_rows dy
//
// All of it is bound by memory: each pass reads its inputs once and writes its
// outputs once. A row stays in registers between the statistics and the
// result, eight neighbouring columns to a lane, so the deviations are summed
// (not the squares, which lose a row whose mean is large), and a lane's columns
// are the same in every row, so the backward pass sums the weight's gradient in
// registers. Odd widths keep that layout: their 16-byte accesses are unaligned,
// which gfx950 allows.

#include <hip/hip_runtime.h>

#include "convert.h"
#include "counter_rng.h"
#include "transformer_kernels.h"

namespace {

constexpr int kVec = 8;  // columns of a lane's piece; also the values of a Philox call

// ---------------------------------------------------------------------------
// pieces of eight columns
// ---------------------------------------------------------------------------

template <typename T>
struct Piece {
  T v[kVec];
};

// n: columns that are left; those behind the row's end read as 0. The values
// stay as they are stored: a conversion here would wait for the load.
template <typename T>
__device__ __forceinline__ void load8(const T* p, int n, Piece<T>& out) {
  if (n >= kVec) {
    __builtin_memcpy(&out, p, sizeof(out));
  } else {
#pragma unroll
    for (int u = 0; u < kVec; ++u) out.v[u] = u < n ? p[u] : static_cast<T>(0.f);
  }
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, int n, float* out) {
  Piece<T> t;
  load8(p, n, t);
#pragma unroll
  for (int u = 0; u < kVec; ++u) out[u] = bf_to_float(t.v[u]);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, int n, const float* in) {
  T t[kVec];
#pragma unroll
  for (int u = 0; u < kVec; ++u) t[u] = static_cast<T>(in[u]);
  if (n >= kVec) {
    __builtin_memcpy(p, t, sizeof(t));
  } else {
#pragma unroll
    for (int u = 0; u < kVec; ++u)
      if (u < n) p[u] = t[u];
  }
}

template <typename T>
__device__ __forceinline__ void load8_param(const void* p, int c, int n, int f32, float other, float* out) {
  if (!p) {
#pragma unroll
    for (int u = 0; u < kVec; ++u) out[u] = other;
  } else if (f32) {
    load8(static_cast<const float*>(p) + c, n, out);
  } else {
    load8(static_cast<const T*>(p) + c, n, out);
  }
}

// which of the elements i .. i + 7 are kept. A row whose start is no multiple
// of eight takes its pieces from two calls.
__device__ __forceinline__ void keep8(uint64_t i, const BfDropout& d, BfKey key, bool* kept) {
  const int s = static_cast<int>(i & 7);
  const uint4 w = bf_flat_bits(i >> 3, d, key);
  if (s == 0) {
#pragma unroll
    for (int u = 0; u < kVec; ++u) kept[u] = bf_half(w, u) >= d.threshold;
    return;
  }
  const uint4 w2 = bf_flat_bits((i >> 3) + 1, d, key);
  uint32_t m = 0;
#pragma unroll
  for (int u = 0; u < kVec; ++u)
    m |= (bf_half(w, u) >= d.threshold ? 1u << u : 0u) | (bf_half(w2, u) >= d.threshold ? 256u << u : 0u);
#pragma unroll
  for (int u = 0; u < kVec; ++u) kept[u] = (m >> (s + u)) & 1;
}

// ---------------------------------------------------------------------------
// sums over a row of WAVES waves
// ---------------------------------------------------------------------------

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
  return x;
}

template <int WAVES>
__device__ __forceinline__ float row_sum(float x, float* lds) {
  x = wave_sum(x);
  if (WAVES == 1) return x;
  __syncthreads();  // lds is free
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) s += lds[w];
  return s;
}

template <int WAVES>
__device__ __forceinline__ float2 row_sum2(float x, float y, float2* lds) {
  x = wave_sum(x);
  y = wave_sum(y);
  if (WAVES == 1) return make_float2(x, y);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = make_float2(x, y);
  __syncthreads();
  float2 s = make_float2(0.f, 0.f);
#pragma unroll
  for (int w = 0; w < WAVES; ++w) s.x += lds[w].x, s.y += lds[w].y;
  return s;
}

// z of a lane's piece from x, r; kept is written where there is dropout
template <bool DROP, typename TX, typename TR>
__device__ __forceinline__ void join8(const BfNormArgs& a, long row, int c, BfKey key, const Piece<TX>& x,
                                      const Piece<TR>& r, float* z, bool* kept) {
#pragma unroll
  for (int u = 0; u < kVec; ++u) z[u] = bf_to_float(x.v[u]);
  if (DROP) {
    keep8(static_cast<uint64_t>(row) * a.width + c, a.drop, key, kept);
    // a dropped element counts as 0 whatever it holds
#pragma unroll
    for (int u = 0; u < kVec; ++u) z[u] = kept[u] ? z[u] * a.drop.scale : 0.f;
  }
  if (a.r) {
#pragma unroll
    for (int u = 0; u < kVec; ++u) z[u] += bf_to_float(r.v[u]);
  }
}

// ---------------------------------------------------------------------------
// a row in registers: WAVES waves of NIT pieces a lane hold widths from 8 to
// 512 * WAVES * NIT. A workgroup of one-wave rows has four of them. The next
// row's loads are under way while a row is summed.
//
// No access is guarded by column: the last piece of a width that is no
// multiple of eight is moved back to end with the row (what it repeats is left
// out of the sums and stored twice, with the same value), and the lanes behind
// the row read the last piece and leave it alone. Guards cost more than the
// arithmetic: with them the forward pass of 8192 rows of 8192 bf16 took 129 us.
// ---------------------------------------------------------------------------

constexpr int threads_of(int waves) { return waves == 1 ? 256 : waves * 64; }
constexpr int rows_of(int waves) { return waves == 1 ? 4 : 1; }

// a lane's piece `it` of a row
template <int WAVES, bool EVEN>
struct Place {
  int c;     // first column
  int skip;  // columns that the piece in front has; 8 and more: not in the row
  __device__ __forceinline__ Place(int lane, int it, int width) {
    const int at = (it * WAVES * 64 + lane) * kVec;
    c = min(at, width - kVec);
    skip = at - c;
  }
  __device__ __forceinline__ bool inside() const { return EVEN ? skip == 0 : skip < kVec; }
  __device__ __forceinline__ bool counts(int u) const { return EVEN ? skip == 0 : u >= skip; }
};

template <typename TX, typename TR, int WAVES, int NIT, bool EVEN, bool DROP>
__global__ __launch_bounds__(threads_of(WAVES)) void norm_fwd_k(BfNormArgs a) {
  __shared__ float lds[WAVES];
  constexpr int kLanes = WAVES * 64;
  const int lane = threadIdx.x % kLanes;
  const BfKey key = DROP ? bf_key(a.drop) : BfKey{0, 0};
  const float width = static_cast<float>(a.width);  // divided by: a constant row has exactly its mean
  const long step = static_cast<long>(gridDim.x) * rows_of(WAVES);
  long row = static_cast<long>(blockIdx.x) * rows_of(WAVES) + threadIdx.x / kLanes;
  Piece<TX> x[NIT];
  Piece<TR> r[NIT];
  float w[NIT][kVec], b[NIT][kVec];
  const auto fetch = [&](long at) {
    at = at < a.rows ? at : a.rows - 1;
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      const Place<WAVES, EVEN> p(lane, it, a.width);
      load8(static_cast<const TX*>(a.x) + at * a.x_row + p.c, kVec, x[it]);
      if (a.r) load8(static_cast<const TR*>(a.r) + at * a.r_row + p.c, kVec, r[it]);
    }
  };
  fetch(row);
#pragma unroll
  for (int it = 0; it < NIT; ++it) {
    const Place<WAVES, EVEN> p(lane, it, a.width);
    load8_param<TX>(a.weight, p.c, kVec, a.weight_f32, 1.f, w[it]);
    load8_param<TX>(a.bias, p.c, kVec, a.weight_f32, 0.f, b[it]);
  }
  for (; row < a.rows; row += step) {
    float z[NIT][kVec];
    float s = 0.f, q = 0.f;
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      const Place<WAVES, EVEN> p(lane, it, a.width);
      bool kept[kVec];
      join8<DROP>(a, row, p.c, key, x[it], r[it], z[it], kept);
#pragma unroll
      for (int u = 0; u < kVec; ++u) s += p.counts(u) ? z[it][u] : 0.f;
    }
    fetch(row + step);
    const float mean = row_sum<WAVES>(s, lds) / width;
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      const Place<WAVES, EVEN> p(lane, it, a.width);
#pragma unroll
      for (int u = 0; u < kVec; ++u) {
        z[it][u] -= mean;
        q += p.counts(u) ? z[it][u] * z[it][u] : 0.f;
      }
    }
    const float rstd = 1.f / sqrtf(row_sum<WAVES>(q, lds) / width + a.eps);
    if (a.mean && lane == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      const Place<WAVES, EVEN> p(lane, it, a.width);
      float y[kVec];
#pragma unroll
      for (int u = 0; u < kVec; ++u) y[u] = z[it][u] * rstd * w[it][u] + b[it][u];
      if (p.inside()) store8(static_cast<TR*>(a.y) + row * a.width + p.c, kVec, y);
    }
  }
}

template <typename TX, typename TR, int WAVES, int NIT, bool EVEN, bool DROP>
__global__ __launch_bounds__(threads_of(WAVES)) void norm_bwd_k(BfNormArgs a) {
  constexpr int kLanes = WAVES * 64;
  __shared__ float2 lds[WAVES];
  __shared__ float fold[WAVES == 1 ? 3 * kLanes * kVec : 1];
  const int lane = threadIdx.x % kLanes;
  const BfKey key = DROP ? bf_key(a.drop) : BfKey{0, 0};
  const float width = static_cast<float>(a.width);
  const long step = static_cast<long>(gridDim.x) * rows_of(WAVES);
  long row = static_cast<long>(blockIdx.x) * rows_of(WAVES) + threadIdx.x / kLanes;
  Piece<TX> x[NIT];
  Piece<TR> r[NIT], dy[NIT];
  float next_mean = 0.f, next_rstd = 0.f;
  const auto fetch = [&](long at) {
    at = at < a.rows ? at : a.rows - 1;
    next_mean = a.mean[at];
    next_rstd = a.rstd[at];
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      const Place<WAVES, EVEN> p(lane, it, a.width);
      load8(static_cast<const TX*>(a.x) + at * a.x_row + p.c, kVec, x[it]);
      if (a.r) load8(static_cast<const TR*>(a.r) + at * a.r_row + p.c, kVec, r[it]);
      load8(static_cast<const TR*>(a.dy) + at * a.dy_row + p.c, kVec, dy[it]);
    }
  };
  fetch(row);
  float w[NIT][kVec], dw[NIT][kVec], db[NIT][kVec];
#pragma unroll
  for (int it = 0; it < NIT; ++it) {
    const Place<WAVES, EVEN> p(lane, it, a.width);
    load8_param<TX>(a.weight, p.c, kVec, a.weight_f32, 1.f, w[it]);
#pragma unroll
    for (int u = 0; u < kVec; ++u) dw[it][u] = db[it][u] = 0.f;
  }
  for (; row < a.rows; row += step) {
    const float mean = next_mean, rstd = next_rstd;
    float xhat[NIT][kVec], g[NIT][kVec];
    bool kept[NIT][kVec];
    float s = 0.f, q = 0.f;
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      const Place<WAVES, EVEN> p(lane, it, a.width);
      join8<DROP>(a, row, p.c, key, x[it], r[it], xhat[it], kept[it]);
#pragma unroll
      for (int u = 0; u < kVec; ++u) {
        const float up = bf_to_float(dy[it].v[u]), h = (xhat[it][u] - mean) * rstd;
        dw[it][u] += up * h;
        db[it][u] += up;
        xhat[it][u] = h;
        g[it][u] = up * w[it][u];
        s += p.counts(u) ? g[it][u] : 0.f;
        q += p.counts(u) ? g[it][u] * h : 0.f;
      }
    }
    fetch(row + step);
    if (!a.dx && !a.dr) continue;
    const float2 sums = row_sum2<WAVES>(s, q, lds);
    const float m1 = sums.x / width, m2 = sums.y / width;
#pragma unroll
    for (int it = 0; it < NIT; ++it) {
      const Place<WAVES, EVEN> p(lane, it, a.width);
#pragma unroll
      for (int u = 0; u < kVec; ++u) g[it][u] = rstd * (g[it][u] - m1 - xhat[it][u] * m2);
      if (!p.inside()) continue;
      if (a.dr) store8(static_cast<TR*>(a.dr) + row * a.width + p.c, kVec, g[it]);
      if (!a.dx) continue;
      if (DROP) {
#pragma unroll
        for (int u = 0; u < kVec; ++u) g[it][u] = kept[it][u] ? g[it][u] * a.drop.scale : 0.f;
      }
      store8(static_cast<TX*>(a.dx) + row * a.width + p.c, kVec, g[it]);
    }
  }
  if (!a.partial) return;
  // one partial sum for each column of a workgroup, in a slot of its own: the
  // order of all sums is fixed
  float* out = a.partial + static_cast<long>(blockIdx.x) * 2 * a.width;
#pragma unroll
  for (int it = 0; it < NIT; ++it) {
    const Place<WAVES, EVEN> p(lane, it, a.width);
#pragma unroll
    for (int both = 0; both < 2; ++both) {
      float* mine = both ? db[it] : dw[it];
      if (WAVES == 1) {  // four rows' waves into one
        const int wave = threadIdx.x / kLanes;
        __syncthreads();
        if (wave)
#pragma unroll
          for (int u = 0; u < kVec; ++u) fold[((wave - 1) * kVec + u) * kLanes + lane] = mine[u];
        __syncthreads();
        if (wave) continue;
#pragma unroll
        for (int k = 0; k < 3; ++k)
#pragma unroll
          for (int u = 0; u < kVec; ++u) mine[u] += fold[(k * kVec + u) * kLanes + lane];
      }
      if (p.inside()) store8(out + both * a.width + p.c, kVec, mine);
    }
  }
}

// ---------------------------------------------------------------------------
// wider rows, and those of less than one piece: the row is read again for each
// of its passes (the cache holds it), and the weight's gradient has a pass of
// its own
// ---------------------------------------------------------------------------

template <typename TX, typename TR>
__device__ __forceinline__ void join8(const BfNormArgs& a, long row, int c, BfKey key, float* z, bool* kept) {
  const int n = a.width - c;
  Piece<TX> x;
  Piece<TR> r;
  load8(static_cast<const TX*>(a.x) + row * a.x_row + c, n, x);
  if (a.r) load8(static_cast<const TR*>(a.r) + row * a.r_row + c, n, r);
  if (a.drop.threshold) join8<true>(a, row, c, key, x, r, z, kept);
  else join8<false>(a, row, c, key, x, r, z, kept);
}

template <typename TX, typename TR, int WAVES>
__global__ __launch_bounds__(threads_of(WAVES)) void norm_fwd_wide_k(BfNormArgs a) {
  __shared__ float lds[WAVES];
  constexpr int kLanes = WAVES * 64, kStep = kLanes * kVec;
  const BfKey key = a.drop.threshold ? bf_key(a.drop) : BfKey{0, 0};
  const float width = static_cast<float>(a.width);
  const int first = threadIdx.x % kLanes * kVec;
  const long step = static_cast<long>(gridDim.x) * rows_of(WAVES);
  for (long row = static_cast<long>(blockIdx.x) * rows_of(WAVES) + threadIdx.x / kLanes; row < a.rows; row += step) {
    float s = 0.f, q = 0.f, z[kVec];
    bool kept[kVec];
    for (int c = first; c < a.width; c += kStep) {
      join8<TX, TR>(a, row, c, key, z, kept);
#pragma unroll
      for (int u = 0; u < kVec; ++u) s += c + u < a.width ? z[u] : 0.f;
    }
    const float mean = row_sum<WAVES>(s, lds) / width;
    for (int c = first; c < a.width; c += kStep) {
      join8<TX, TR>(a, row, c, key, z, kept);
#pragma unroll
      for (int u = 0; u < kVec; ++u) q += c + u < a.width ? (z[u] - mean) * (z[u] - mean) : 0.f;
    }
    const float rstd = 1.f / sqrtf(row_sum<WAVES>(q, lds) / width + a.eps);
    if (a.mean && threadIdx.x % kLanes == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
    for (int c = first; c < a.width; c += kStep) {
      const int n = a.width - c;
      float w[kVec], b[kVec];
      join8<TX, TR>(a, row, c, key, z, kept);
      load8_param<TX>(a.weight, c, n, a.weight_f32, 1.f, w);
      load8_param<TX>(a.bias, c, n, a.weight_f32, 0.f, b);
#pragma unroll
      for (int u = 0; u < kVec; ++u) b[u] += (z[u] - mean) * rstd * w[u];
      store8(static_cast<TR*>(a.y) + row * a.width + c, n, b);
    }
  }
}

template <typename TX, typename TR, int WAVES>
__global__ __launch_bounds__(threads_of(WAVES)) void norm_bwd_wide_k(BfNormArgs a) {
  __shared__ float2 lds[WAVES];
  constexpr int kLanes = WAVES * 64, kStep = kLanes * kVec;
  const BfKey key = a.drop.threshold ? bf_key(a.drop) : BfKey{0, 0};
  const float width = static_cast<float>(a.width);
  const int first = threadIdx.x % kLanes * kVec;
  const long step = static_cast<long>(gridDim.x) * rows_of(WAVES);
  for (long row = static_cast<long>(blockIdx.x) * rows_of(WAVES) + threadIdx.x / kLanes; row < a.rows; row += step) {
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s = 0.f, q = 0.f, z[kVec], g[kVec], w[kVec];
    bool kept[kVec];
    for (int c = first; c < a.width; c += kStep) {
      const int n = a.width - c;
      join8<TX, TR>(a, row, c, key, z, kept);
      load8(static_cast<const TR*>(a.dy) + row * a.dy_row + c, n, g);
      load8_param<TX>(a.weight, c, n, a.weight_f32, 1.f, w);
#pragma unroll
      for (int u = 0; u < kVec; ++u) {
        const float t = u < n ? g[u] * w[u] : 0.f;
        s += t;
        q += u < n ? t * (z[u] - mean) * rstd : 0.f;
      }
    }
    const float2 sums = row_sum2<WAVES>(s, q, lds);
    const float m1 = sums.x / width, m2 = sums.y / width;
    for (int c = first; c < a.width; c += kStep) {
      const int n = a.width - c;
      join8<TX, TR>(a, row, c, key, z, kept);
      load8(static_cast<const TR*>(a.dy) + row * a.dy_row + c, n, g);
      load8_param<TX>(a.weight, c, n, a.weight_f32, 1.f, w);
#pragma unroll
      for (int u = 0; u < kVec; ++u) g[u] = rstd * (g[u] * w[u] - m1 - (z[u] - mean) * rstd * m2);
      if (a.dr) store8(static_cast<TR*>(a.dr) + row * a.width + c, n, g);
      if (!a.dx) continue;
      if (a.drop.threshold) {
#pragma unroll
        for (int u = 0; u < kVec; ++u) g[u] = kept[u] ? g[u] * a.drop.scale : 0.f;
      }
      store8(static_cast<TX*>(a.dx) + row * a.width + c, n, g);
    }
  }
}

template <typename TX, typename TR>
__global__ __launch_bounds__(256) void norm_param_wide_k(BfNormArgs a) {
  const int c = (blockIdx.x * 256 + threadIdx.x) * kVec, n = a.width - c;
  if (n <= 0) return;
  const BfKey key = a.drop.threshold ? bf_key(a.drop) : BfKey{0, 0};
  float z[kVec], g[kVec], dw[kVec] = {}, db[kVec] = {};
  bool kept[kVec];
  for (long row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float mean = a.mean[row], rstd = a.rstd[row];
    join8<TX, TR>(a, row, c, key, z, kept);
    load8(static_cast<const TR*>(a.dy) + row * a.dy_row + c, n, g);
#pragma unroll
    for (int u = 0; u < kVec; ++u) {
      dw[u] += g[u] * ((z[u] - mean) * rstd);
      db[u] += g[u];
    }
  }
  float* out = a.partial + static_cast<long>(blockIdx.y) * 2 * a.width + c;
  store8(out, n, dw);
  store8(out + a.width, n, db);
}

// the partial sums [slots][2][width] into dw and db: COLUMNS of them to a
// workgroup, the slots over its other lanes; every sum has a fixed order.
// Narrow rows take 16 columns, so that there are workgroups enough (768 columns
// of 1024 slots: 4.7 us, with 64 columns 7.4), wide ones 64, whole lines of
// 256 bytes (8192 of 512: 7.7 us, with 16 columns 14.1).
template <typename TX, int COLUMNS>
__global__ __launch_bounds__(1024) void norm_fold_k(BfNormArgs a, int slots) {
  constexpr int kParts = 1024 / COLUMNS;
  __shared__ float lds[kParts][COLUMNS];
  const int column = threadIdx.x % COLUMNS, part = threadIdx.x / COLUMNS;
  const long i = static_cast<long>(blockIdx.x) * COLUMNS + column, n = 2L * a.width;
  float s = 0.f;
  if (i < n) {
#pragma unroll 8
    for (int k = part; k < slots; k += kParts) s += a.partial[k * n + i];
  }
  lds[part][column] = s;
  for (int half = kParts / 2; half > 0; half /= 2) {
    __syncthreads();
    if (part < half) lds[part][column] += lds[part + half][column];
  }
  if (part || i >= n) return;
  s = lds[0][column];
  void* to = i < a.width ? a.dweight : a.dbias;
  const long c = i < a.width ? i : i - a.width;
  if (!to) return;
  if (a.weight_f32) static_cast<float*>(to)[c] = s;
  else static_cast<TX*>(to)[c] = static_cast<TX>(s);
}

// ---------------------------------------------------------------------------
// dropout: 16 bytes a lane (32 of f32), one Philox call to eight elements
// ---------------------------------------------------------------------------

template <typename T>
__global__ __launch_bounds__(256) void dropout_k(T* __restrict__ y, const T* __restrict__ x, long n, BfDropout d) {
  const BfKey key = bf_key(d);
  const long i = (static_cast<long>(blockIdx.x) * 256 + threadIdx.x) * kVec;
  if (i >= n) return;
  const int left = n - i < kVec ? static_cast<int>(n - i) : kVec;
  float v[kVec];
  load8(x + i, left, v);
  const uint4 w = bf_flat_bits(i >> 3, d, key);
#pragma unroll
  for (int u = 0; u < kVec; ++u) v[u] = bf_half(w, u) >= d.threshold ? v[u] * d.scale : 0.f;
  store8(y + i, left, v);
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------

constexpr int kWidest = 16384;

bool in_registers(int width) { return width >= kVec && width <= kWidest; }

int waves_of(int width) { return width <= 1024 ? 1 : width <= 4096 ? 4 : width <= 8192 ? 8 : 16; }

// workgroups of `waves` waves that fill the card's 256 CUs with `deep` waves
// to a SIMD
long filling(int waves, int deep) { return 256L * 4 * deep / (threads_of(waves) / 64); }

// workgroups of the backward pass: each leaves 8 * width bytes of partial sums
int slots_of(long rows, int width) {
  if (!in_registers(width)) {
    const long most = width < kVec ? 1024 : 64;  // a slot of few columns is a small thing
    return static_cast<int>(rows < most ? rows : most);
  }
  const int waves = waves_of(width);
  const long groups = (rows + rows_of(waves) - 1) / rows_of(waves), most = filling(waves, 4);
  return static_cast<int>(groups < most ? groups : most);
}

template <typename TX, typename TR, int WAVES, int NIT, bool EVEN, bool DROP>
void launch(bool backward, const BfNormArgs& a, long grid, hipStream_t stream) {
  if (backward)
    hipLaunchKernelGGL((norm_bwd_k<TX, TR, WAVES, NIT, EVEN, DROP>), dim3(grid), dim3(threads_of(WAVES)), 0, stream, a);
  else
    hipLaunchKernelGGL((norm_fwd_k<TX, TR, WAVES, NIT, EVEN, DROP>), dim3(grid), dim3(threads_of(WAVES)), 0, stream, a);
}

template <typename TX, typename TR, int WAVES, int NIT>
void launch(bool backward, const BfNormArgs& a, long grid, hipStream_t stream) {
  const bool even = a.width % kVec == 0, drop = a.drop.threshold != 0;
  if (even && drop) launch<TX, TR, WAVES, NIT, true, true>(backward, a, grid, stream);
  else if (even) launch<TX, TR, WAVES, NIT, true, false>(backward, a, grid, stream);
  else if (drop) launch<TX, TR, WAVES, NIT, false, true>(backward, a, grid, stream);
  else launch<TX, TR, WAVES, NIT, false, false>(backward, a, grid, stream);
}

template <typename TX, typename TR>
void launch(bool backward, const BfNormArgs& a, long grid, hipStream_t stream) {
  const int waves = waves_of(a.width);
  const bool two = a.width > waves * 512;
  if (waves == 1 && !two) launch<TX, TR, 1, 1>(backward, a, grid, stream);
  else if (waves == 1) launch<TX, TR, 1, 2>(backward, a, grid, stream);
  else if (waves == 4 && !two) launch<TX, TR, 4, 1>(backward, a, grid, stream);
  else if (waves == 4) launch<TX, TR, 4, 2>(backward, a, grid, stream);
  else if (waves == 8) launch<TX, TR, 8, 2>(backward, a, grid, stream);
  else launch<TX, TR, 16, 2>(backward, a, grid, stream);
}

struct Fwd {
  template <typename TX, typename TR>
  static hipError_t run(const BfNormArgs& a, hipStream_t stream) {
    const int waves = waves_of(a.width);
    const long groups = (a.rows + rows_of(waves) - 1) / rows_of(waves), most = filling(waves, 8);
    const long grid = groups < most ? groups : most;
    if (in_registers(a.width)) launch<TX, TR>(false, a, grid, stream);
    else if (waves == 1) hipLaunchKernelGGL((norm_fwd_wide_k<TX, TR, 1>), dim3(grid), dim3(threads_of(1)), 0, stream, a);
    else hipLaunchKernelGGL((norm_fwd_wide_k<TX, TR, 16>), dim3(grid), dim3(threads_of(16)), 0, stream, a);
    return hipGetLastError();
  }
};

struct Bwd {
  template <typename TX, typename TR>
  static hipError_t run(const BfNormArgs& a, hipStream_t stream) {
    const int slots = slots_of(a.rows, a.width), waves = waves_of(a.width);
    if (!in_registers(a.width)) {
      if (a.dx || a.dr) {
        const long groups = (a.rows + rows_of(waves) - 1) / rows_of(waves), most = filling(waves, 8);
        const long grid = groups < most ? groups : most;
        if (waves == 1) hipLaunchKernelGGL((norm_bwd_wide_k<TX, TR, 1>), dim3(grid), dim3(threads_of(1)), 0, stream, a);
        else hipLaunchKernelGGL((norm_bwd_wide_k<TX, TR, 16>), dim3(grid), dim3(threads_of(16)), 0, stream, a);
        if (hipError_t e = hipGetLastError()) return e;
      }
      if (a.partial)
        hipLaunchKernelGGL((norm_param_wide_k<TX, TR>), dim3((a.width + 2047) / 2048, slots), dim3(256), 0, stream, a);
    } else {
      launch<TX, TR>(true, a, slots, stream);
    }
    if (hipError_t e = hipGetLastError()) return e;
    if (!a.partial) return hipSuccess;
    if (a.width < 4096)
      hipLaunchKernelGGL((norm_fold_k<TX, 16>), dim3((2L * a.width + 15) / 16), dim3(1024), 0, stream, a, slots);
    else
      hipLaunchKernelGGL((norm_fold_k<TX, 64>), dim3((2L * a.width + 63) / 64), dim3(1024), 0, stream, a, slots);
    return hipGetLastError();
  }
};

template <typename Op>
hipError_t dispatch(const BfNormArgs& a, int x_dtype, int r_dtype, hipStream_t stream) {
  if (x_dtype == 0 && r_dtype == 0) return Op::template run<float, float>(a, stream);
  if (x_dtype == 2 && r_dtype == 2) return Op::template run<_Float16, _Float16>(a, stream);
  if (x_dtype == 3 && r_dtype == 3) return Op::template run<__bf16, __bf16>(a, stream);
  if (x_dtype == 2 && r_dtype == 0) return Op::template run<_Float16, float>(a, stream);
  if (x_dtype == 3 && r_dtype == 0) return Op::template run<__bf16, float>(a, stream);
  return hipErrorInvalidValue;
}

template <typename T>
hipError_t drop(void* y, const void* x, long n, const BfDropout& d, hipStream_t stream) {
  const long blocks = (n + 256 * kVec - 1) / (256 * kVec);
  if (n > bf_dropout_most()) return hipErrorInvalidValue;
  hipLaunchKernelGGL(dropout_k<T>, dim3(blocks), dim3(256), 0, stream, static_cast<T*>(y), static_cast<const T*>(x), n,
                     d);
  return hipGetLastError();
}

}  // namespace

extern "C" {

hipError_t bf_norm_fwd(const BfNormArgs* a, int x_dtype, int r_dtype, hipStream_t stream) {
  return dispatch<Fwd>(*a, x_dtype, r_dtype, stream);
}

hipError_t bf_norm_bwd(const BfNormArgs* a, int x_dtype, int r_dtype, hipStream_t stream) {
  return dispatch<Bwd>(*a, x_dtype, r_dtype, stream);
}

long bf_norm_partial_floats(long rows, int width) { return 2L * width * slots_of(rows, width); }

long bf_dropout_most() { return 0xFFFFFFL * 256 * kVec; }  // a launch has less than 2^32 threads

hipError_t bf_dropout(void* y, const void* x, long n, int dtype, const BfDropout* d, hipStream_t stream) {
  switch (dtype) {
    case 0: return drop<float>(y, x, n, *d, stream);
    case 2: return drop<_Float16>(y, x, n, *d, stream);
    case 3: return drop<__bf16>(y, x, n, *d, stream);
  }
  return hipErrorInvalidValue;
}

}  // extern "C"
