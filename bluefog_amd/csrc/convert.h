// Copyright 2026. Licensed under the Apache License, Version 2.0.
//
// Conversions between storage types and the 32-bit arithmetic of the
// transformer kernels (round to nearest even).
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

template <typename T>
__device__ __forceinline__ float bf_to_float(T x);
template <>
__device__ __forceinline__ float bf_to_float(float x) { return x; }
template <>
__device__ __forceinline__ float bf_to_float(_Float16 x) { return static_cast<float>(x); }
template <>
__device__ __forceinline__ float bf_to_float(__bf16 x) { return static_cast<float>(x); }
