// Copyright 2026. Licensed under the Apache License, Version 2.0.
//
// C entries of the transformer training operators (packed attention, layer
// norm, counter-based dropout). dtype codes: 0 f32, 2 f16, 3 bf16. Every
// entry returns an error code instead of throwing.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

struct BfDropout {
  const int64_t* seed_ptr;  // seed on the device, or null: `seed` holds
  uint64_t seed;
  uint32_t offset;
  uint32_t threshold;  // 0: no dropout
  float scale;
};

struct BfAttnArgs {
  const void *q, *k, *v, *dout;
  const void* out;  // backward: the forward's output
  void *o, *dq, *dk, *dv;  // written; contiguous [rows, heads, dim]
  void* rest;    // what rounding took from o, [rows, heads, dim]; may be null
  float* lse;    // [heads, rows]; forward: written unless null
  float* delta;  // [heads, rows]; backward: written by dq, read by dk/dv
  float* partial;  // bf_attn_partial_floats() of them
  int key_slices, query_slices;  // of the axes that workgroups go along
  const int* cu;  // seqs + 1 ends of the sequences
  const int* table;  // bf_attn_table_ints() of them, by bf_attn_table
  int seqs, rows, heads, kv_heads, dim;
  // element strides of a row and a head; the last dimension is dense
  long q_row, q_head, k_row, k_head, v_row, v_head, do_row, do_head;
  float scale;
  int causal;
  int vec;  // 16-byte accesses are allowed in all tensors
  BfDropout drop;
};

struct BfNormArgs {
  const void *x, *r, *dy;   // r may be null
  const void *weight, *bias;  // each may be null
  int weight_f32;           // weight and bias are f32 (else the type of x)
  void *y, *dx, *dr;        // y, dr: the type of r
  void *dweight, *dbias;    // type of weight; may be null
  float *mean, *rstd;       // forward: written unless null
  float* partial;           // backward: bf_norm_partial_floats() of them
  long rows, x_row, r_row, dy_row;
  int width;
  float eps;
  BfDropout drop;
};

extern "C" {
int bf_attn_fits(const BfAttnArgs* a, int dtype, int backward);
int bf_attn_table_ints(const BfAttnArgs* a);
hipError_t bf_attn_table(const BfAttnArgs* a, int* table, hipStream_t stream);
hipError_t bf_attn_fwd(const BfAttnArgs* a, int dtype, hipStream_t stream);
int bf_attn_key_slices(const BfAttnArgs* a, int dtype);
int bf_attn_query_slices(const BfAttnArgs* a, int dtype);
long bf_attn_partial_floats(const BfAttnArgs* a);
// dq always: delta, which dk and dv need, comes with it
hipError_t bf_attn_bwd(const BfAttnArgs* a, int dtype, int need_dkv, hipStream_t stream);
hipError_t bf_norm_fwd(const BfNormArgs* a, int x_dtype, int r_dtype,
                       hipStream_t stream);
hipError_t bf_norm_bwd(const BfNormArgs* a, int x_dtype, int r_dtype,
                       hipStream_t stream);
long bf_norm_partial_floats(long rows, int width);
long bf_dropout_most();  // values of a call
hipError_t bf_dropout(void* y, const void* x, long n, int dtype,
                      const BfDropout* d, hipStream_t stream);
}
