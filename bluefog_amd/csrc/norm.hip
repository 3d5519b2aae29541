// Copyright 2026. Licensed under the Apache License, Version 2.0.
//
// Layer norm over rows, forward and backward, and dropout:
//   z = r + keep x,  y = (z - mean) rstd w + b
//   g = dy w,  dz = rstd (g - mean(g) - xhat mean(g xhat)),
//   dr = dz,  dx = keep dz,  dw = sum_rows dy xhat,  db = sum_rows dy

#include <hip/hip_runtime.h>

#include "convert.h"
#include "transformer_kernels.h"

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float block_sum(float x, float* lds) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  return lds[0] + lds[1] + lds[2] + lds[3];
}

template <typename T>
__device__ __forceinline__ float param(const void* p, int c, int f32) {
  return f32 ? static_cast<const float*>(p)[c] : bf_to_float(static_cast<const T*>(p)[c]);
}

template <typename T>
__device__ __forceinline__ void put_param(void* p, int c, int f32, float x) {
  if (f32) static_cast<float*>(p)[c] = x;
  else static_cast<T*>(p)[c] = static_cast<T>(x);
}

template <typename TX, typename TR>
__device__ __forceinline__ float joined(const BfNormArgs& a, long row, int c, float keep) {
  // a dropped element counts as 0 whatever it holds
  float z = keep != 0.f ? bf_to_float(static_cast<const TX*>(a.x)[row * a.x_row + c]) * keep : 0.f;
  if (a.r) z += bf_to_float(static_cast<const TR*>(a.r)[row * a.r_row + c]);
  return z;
}

__device__ __forceinline__ float keep_of(const BfNormArgs& a, long row, int c, BfKey key) {
  return a.drop.threshold ? bf_flat_keep(static_cast<uint64_t>(row) * a.width + c, a.drop, key) : 1.f;
}

template <typename TX, typename TR>
__global__ __launch_bounds__(kThreads) void norm_fwd_k(BfNormArgs a) {
  __shared__ float lds[4];
  const BfKey key = a.drop.threshold ? bf_key(a.drop) : BfKey{0, 0};
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    float s = 0.f, q = 0.f;
    for (int c = threadIdx.x; c < a.width; c += kThreads) s += joined<TX, TR>(a, row, c, keep_of(a, row, c, key));
    const float mean = block_sum(s, lds) / a.width;
    for (int c = threadIdx.x; c < a.width; c += kThreads) {
      const float d = joined<TX, TR>(a, row, c, keep_of(a, row, c, key)) - mean;
      q += d * d;
    }
    const float rstd = 1.f / sqrtf(block_sum(q, lds) / a.width + a.eps);
    if (a.mean && threadIdx.x == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
    for (int c = threadIdx.x; c < a.width; c += kThreads) {
      float y = (joined<TX, TR>(a, row, c, keep_of(a, row, c, key)) - mean) * rstd;
      if (a.weight) y *= param<TX>(a.weight, c, a.weight_f32);
      if (a.bias) y += param<TX>(a.bias, c, a.weight_f32);
      static_cast<TR*>(a.y)[row * a.width + c] = static_cast<TR>(y);
    }
  }
}

template <typename TX, typename TR>
__global__ __launch_bounds__(kThreads) void norm_bwd_k(BfNormArgs a) {
  __shared__ float lds[4];
  const BfKey key = a.drop.threshold ? bf_key(a.drop) : BfKey{0, 0};
  for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s = 0.f, q = 0.f;
    for (int c = threadIdx.x; c < a.width; c += kThreads) {
      const float xhat = (joined<TX, TR>(a, row, c, keep_of(a, row, c, key)) - mean) * rstd;
      float g = bf_to_float(static_cast<const TR*>(a.dy)[row * a.dy_row + c]);
      if (a.weight) g *= param<TX>(a.weight, c, a.weight_f32);
      s += g;
      q += g * xhat;
    }
    const float m1 = block_sum(s, lds) / a.width, m2 = block_sum(q, lds) / a.width;
    for (int c = threadIdx.x; c < a.width; c += kThreads) {
      const float keep = keep_of(a, row, c, key);
      const float xhat = (joined<TX, TR>(a, row, c, keep) - mean) * rstd;
      float g = bf_to_float(static_cast<const TR*>(a.dy)[row * a.dy_row + c]);
      if (a.weight) g *= param<TX>(a.weight, c, a.weight_f32);
      const float dz = rstd * (g - m1 - xhat * m2);
      if (a.dx) static_cast<TX*>(a.dx)[row * a.width + c] = static_cast<TX>(keep != 0.f ? dz * keep : 0.f);
      if (a.dr) static_cast<TR*>(a.dr)[row * a.width + c] = static_cast<TR>(dz);
    }
  }
}

template <typename TX, typename TR>
__global__ __launch_bounds__(kThreads) void norm_param_k(BfNormArgs a) {
  __shared__ float lds[4];
  const BfKey key = a.drop.threshold ? bf_key(a.drop) : BfKey{0, 0};
  const int c = blockIdx.x;
  float dw = 0.f, db = 0.f;
  for (long row = threadIdx.x; row < a.rows; row += kThreads) {
    const float xhat = (joined<TX, TR>(a, row, c, keep_of(a, row, c, key)) - a.mean[row]) * a.rstd[row];
    const float g = bf_to_float(static_cast<const TR*>(a.dy)[row * a.dy_row + c]);
    dw += g * xhat;
    db += g;
  }
  dw = block_sum(dw, lds);
  db = block_sum(db, lds);
  if (threadIdx.x) return;
  if (a.dweight) put_param<TX>(a.dweight, c, a.weight_f32, dw);
  if (a.dbias) put_param<TX>(a.dbias, c, a.weight_f32, db);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void dropout_k(T* y, const T* x, long n, BfDropout d) {
  const BfKey key = bf_key(d);
  const long stride = static_cast<long>(gridDim.x) * kThreads;
  for (long i = static_cast<long>(blockIdx.x) * kThreads + threadIdx.x; i < n; i += stride) {
    const float keep = bf_flat_keep(i, d, key);
    y[i] = static_cast<T>(keep != 0.f ? bf_to_float(x[i]) * keep : 0.f);
  }
}

struct Fwd {
  template <typename TX, typename TR>
  static hipError_t run(const BfNormArgs& a, hipStream_t stream) {
    const int grid = static_cast<int>(a.rows < 65536 ? a.rows : 65536);
    hipLaunchKernelGGL((norm_fwd_k<TX, TR>), dim3(grid), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
  }
};

struct Bwd {
  template <typename TX, typename TR>
  static hipError_t run(const BfNormArgs& a, hipStream_t stream) {
    const int grid = static_cast<int>(a.rows < 65536 ? a.rows : 65536);
    if (a.dx || a.dr) {
      hipLaunchKernelGGL((norm_bwd_k<TX, TR>), dim3(grid), dim3(kThreads), 0, stream, a);
      if (hipError_t e = hipGetLastError()) return e;
    }
    if (!a.dweight && !a.dbias) return hipSuccess;
    hipLaunchKernelGGL((norm_param_k<TX, TR>), dim3(a.width), dim3(kThreads), 0, stream, a);
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
  const long blocks = (n + kThreads - 1) / kThreads;
  hipLaunchKernelGGL(dropout_k<T>, dim3(blocks < 65536 ? blocks : 65536), dim3(kThreads), 0, stream,
                     static_cast<T*>(y), static_cast<const T*>(x), n, d);
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

long bf_norm_partial_floats(long, int, int, int) { return 0; }

hipError_t bf_dropout(void* y, const void* x, long n, int dtype, const BfDropout* d, hipStream_t stream) {
  switch (dtype) {
    case 0: return drop<float>(y, x, n, *d, stream);
    case 2: return drop<_Float16>(y, x, n, *d, stream);
    case 3: return drop<__bf16>(y, x, n, *d, stream);
  }
  return hipErrorInvalidValue;
}

}  // extern "C"
