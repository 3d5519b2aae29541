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

constexpr float kLog2e = 1.4426950408889634f;

using namespace bf_attn;

// ---------------------------------------------------------------------------
// forward. A wave has 32 query rows, one to a lane of each half, and computes
// S^T = k q^T, so that a row's scores lie in the registers of its lane pair: the
// running maximum and sum cost one exchange of halves, and P^T is the operand
// of O^T = v^T P^T as it stands. The tiles of k and v go to LDS while the
// last ones are used.
//
// P is rounded to the type in front of the product. The sum of its roundings is
// about as large as the output's own, so that out (and dv, below) is 1.4 times as
// far off as that: 2.3e-3 of its size in bf16, 2.9e-4 in f16, where P in 32 bits gives
// 1.7e-3 and 2.1e-4. What the rounding took could go through the matrix units too,
// as for dS, and does give those. It is left out for its time: with it (in out
// and dv) two causal prompts to 8192 (32/8 heads of 128, forward) took 789 us, 600
// without; training on 6 causal sequences to 4096 (16/4 heads of 128) 1193 and 1074, on 64
// to 512 (12 heads of 64, dropout) 239 and 222.
// ---------------------------------------------------------------------------

constexpr int kRows = 128;  // queries, or keys of dk and dv, of a workgroup

template <typename T>
constexpr int kKeys = sizeof(T) == 2 ? 64 : 32;  // keys of a tile

// waves of a SIMD whose registers the kernels are held to
template <typename T, int DP>
constexpr int kFwdWaves = sizeof(T) == 2 && DP == 64 ? 3 : 2;
// f32 under two waves of heads of 128 spills: 3.9 ms where it takes 1.8 (8192 tokens, 16 heads)
template <typename T, int DP>
constexpr int kDqWaves = sizeof(T) == 4 && DP == 128 ? 1 : kFwdWaves<T, DP>;

// a slice's keys of `keys`, whole tiles
__device__ __forceinline__ int2 keys_of(int keys, int tile, int slice, int slices) {
  const int tiles = (keys + tile - 1) / tile;
  return make_int2(tiles * slice / slices * tile, min(keys, tiles * (slice + 1) / slices * tile));
}

template <int N>
struct Mode {
  static constexpr int value = N;
};

// The accumulators are scaled down only where a maximum has grown by more than
// this (in powers of two): until then P is at most 2^8, in range of every type.
constexpr float kSlack = 8.f;

template <typename T, int DP, bool VEC, bool DROP>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(kFwdWaves<T, DP>, kFwdWaves<T, DP>))) void attn_fwd_k(BfAttnArgs a) {
  constexpr int kQ = kRows, BN = kKeys<T>, kSub = BN / 32, kSteps = DP / 16, kDT = DP / 32;
  typedef Tile<T, BN, DP, 256, VEC> KV;
  __shared__ __align__(1024) char lds[2][2][KV::kBytes];
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x >> 6;
  const Unit unit = unit_of(blockIdx.x, a.heads);
  const int h = unit.head, g = h / (a.heads / a.kv_heads);
  const int slice = unit.number % a.key_slices;  // of the keys
  const Work w = find_tile(a, unit.number / a.key_slices, kQ, a.causal);
  if (!w.any) return;
  const int q0 = w.tile * kQ, qw = q0 + wave * 32, qi = qw + (lane & 31);
  const bool inside = qi < w.len;
  const long row = w.begin + qi;
  Acc o[kDT];
#pragma unroll
  for (int i = 0; i < kDT; ++i) o[i] = Acc{};
  // o times f, and the logarithm of its sum to base 2
  const auto finish = [&](float f, float lse) __attribute__((always_inline)) {
    const long at = (row * a.heads + h) * a.dim, all = static_cast<long>(a.rows) * a.heads;
    if (a.key_slices == 1) {
      store_row<VEC>(static_cast<T*>(a.o) + at, o, f, half, a.dim, inside, a.rest ? static_cast<T*>(a.rest) + at : nullptr);
      if (a.lse && inside && half == 0) a.lse[static_cast<long>(h) * a.rows + row] = lse;
    } else {
      store_row<VEC>(a.partial + slice * all * a.dim + at, o, f, half, a.dim, inside);
      float* sums = a.partial + a.key_slices * all * a.dim;
      if (inside && half == 0) sums[slice * all + static_cast<long>(h) * a.rows + row] = lse;
    }
  };
  if (w.seq == a.seqs) {  // behind the last sequence
    finish(0.f, 0.f);
    return;
  }
  const T* q = static_cast<const T*>(a.q) + static_cast<long>(w.begin + min(qi, w.len - 1)) * a.q_row + h * a.q_head;
  typedef Loader<T, BN, DP, 256, VEC> Load;
  const Load k(static_cast<const T*>(a.k) + w.begin * a.k_row + g * a.k_head, a.k_row, a.dim);
  const Load v(static_cast<const T*>(a.v) + w.begin * a.v_row + g * a.v_head, a.v_row, a.dim);
  const int last = w.len - 1;
  const int seen = a.causal ? min(w.len, qi + 1) : w.len;  // keys of the lane's row
  const int2 range = keys_of(a.causal ? min(w.len, q0 + kQ) : w.len, BN, slice, a.key_slices);
  if (range.x >= range.y) {
    finish(0.f, -INFINITY);
    return;
  }
  if (a.dim < DP) {
    KV::clear(&lds[0][0][0], sizeof(lds));
    __syncthreads();
  }
  k.load(lds[0][0], range.x, last);
  v.load(lds[0][1], range.x, last);
  Frag<T> qf[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) qf[s] = load_row<VEC>(q, s, half, a.dim);
  const BfKey key = DROP ? bf_key(a.drop) : BfKey{0, 0};
  const float c = a.scale * kLog2e;
  float m = -INFINITY, l = 0.f;  // of scores without c
  // One tile of keys, the first 32 * SUBS of them. MASKED: some of them are not
  // seen by some of the workgroup's rows. CLEAN: v that is no number or infinite
  // is left out.
  const auto attend = [&](auto mode, auto subs, int k0, int buf) __attribute__((always_inline)) {
    constexpr bool MASKED = decltype(mode)::value > 0, CLEAN = decltype(mode)::value > 1;
    constexpr int SUBS = decltype(subs)::value;
    const int rows = KV::row_place(lane & 31, half), columns = KV::columns_place(lane);
    Acc s[SUBS];
#pragma unroll
    for (int u = 0; u < SUBS; ++u) {
      s[u] = Acc{};
#pragma unroll
      for (int i = 0; i < kSteps; ++i) s[u] = mma(KV::read_row(lds[buf][0], rows, u * 32, i, half), qf[i], s[u]);
    }
    if (sizeof(T) == 2) feed<4, SUBS * kSteps, 1>();
    if (MASKED) {
#pragma unroll
      for (int u = 0; u < SUBS; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[u][r] = k0 + u * 32 + row_of(r, half) < seen ? s[u][r] : -INFINITY;
    }
    float top = s[0][0];
#pragma unroll
    for (int u = 0; u < SUBS; ++u)
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
    Frag<T> p[2 * SUBS];
#pragma unroll
    for (int u = 0; u < 2 * SUBS; ++u) {
      uint4 bits;
      if (DROP) bits = bf_philox((k0 / 16 + u) * 2 + half, static_cast<uint32_t>(row), h, a.drop.offset, key);
      float x[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        x[r] = __builtin_amdgcn_exp2f(s[u / 2][(u & 1) * 8 + r] * c - base);
        l += x[r];
        if (DROP) x[r] = bf_half(bits, r) >= a.drop.threshold ? x[r] : 0.f;
      }
      p[u] = rounded<T>(x);
    }
    if (!CLEAN) {
#pragma unroll
      for (int u = 0; u < 2 * SUBS; ++u)
#pragma unroll
        for (int i = 0; i < kDT; ++i) o[i] = mma(KV::read_columns(lds[buf][1], columns, u * 16, i), p[u], o[i]);
    } else {
#pragma unroll
      for (int u = 0; u < 2 * SUBS; ++u)
#pragma unroll
        for (int i = 0; i < kDT; ++i) {
          Frag<T> f = KV::read_columns(lds[buf][1], columns, u * 16, i);
#pragma unroll
          for (int r = 0; r < 8; ++r) f[r] = finite(f[r]) ? f[r] : static_cast<T>(0.f);
          o[i] = mma(f, p[u], o[i]);
        }
    }
  };
  // all tiles, from the one whose load is under way into buffer 0; those that
  // no row has to mask have a loop of their own
  const auto all_tiles = [&](auto masked) __attribute__((always_inline)) {
    constexpr bool kClean = decltype(masked)::value > 1;
    const int whole = kClean ? range.x : min(range.y, (a.causal ? q0 + 1 : w.len) / BN * BN);
    loads_done();
    int k0 = range.x, buf = 0;
    const auto next = [&]() __attribute__((always_inline)) {
      if (k0 + BN >= range.y) return;
      k.load(lds[buf ^ 1][0], k0 + BN, last);
      v.load(lds[buf ^ 1][1], k0 + BN, last);
    };
    for (; k0 < whole; k0 += BN, buf ^= 1) {
      next();
      if (qw < w.len) attend(Mode<0>(), Mode<kSub>(), k0, buf);
      loads_done();
    }
    for (; k0 < range.y; k0 += BN, buf ^= 1) {
      next();
      const int seen_here = min(range.y, a.causal ? qw + 32 : w.len) - k0;  // keys that some row of the wave sees
      if (qw < w.len && seen_here > 0) {
        if (kSub == 1 || seen_here > 32) attend(masked, Mode<kSub>(), k0, buf);
        else attend(masked, Mode<1>(), k0, buf);
      }
      loads_done();
    }
  };
  all_tiles(Mode<1>());
  // A P of 0 times a v that is no number or infinite is no number. That P may be
  // masked, or of a row behind the sequence (which repeats the last), or have been
  // rounded to 0 where the sum has an infinity. So if a sum is lost, once more
  // without such v, which are then added where the row sees the key: as they are with
  // a P, and no number with a P of 0 (a score of -inf, or dropped).
  bool lost = false;
#pragma unroll
  for (int i = 0; i < kDT; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) lost |= !finite(o[i][r]);
  if (__syncthreads_or(lost)) {
    m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < kDT; ++i) o[i] = Acc{};
    k.load(lds[0][0], range.x, last);
    v.load(lds[0][1], range.x, last);
    all_tiles(Mode<2>());
    for (int k0 = range.x; k0 < range.y; k0 += 32) {  // half a tile's rows, in buffer 0
      const int at = (k0 - range.x) % BN;
      if (at == 0) {
        k.load(lds[0][0], k0, last);
        v.load(lds[0][1], k0, last);
        loads_done();
      }
      bool bad = false;  // the lane's key has such a v
      if (lane < 32)
        for (int d = 0; d < DP; ++d) bad |= !finite(KV::value(lds[0][1], at + lane, d));
      uint32_t left = static_cast<uint32_t>(__ballot(bad));
      if (left) {
        const int rows = KV::row_place(lane & 31, half);
        Acc s{};
#pragma unroll
        for (int i = 0; i < kSteps; ++i) s = mma(KV::read_row(lds[0][0], rows, at, i, half), qf[i], s);
        uint32_t with = 0, without = 0;  // keys that the row sees, by their P
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          uint4 bits;
          if (DROP) bits = bf_philox((k0 / 16 + t) * 2 + half, static_cast<uint32_t>(row), h, a.drop.offset, key);
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            const int j = t * 16 + row_of(r, half);
            const bool keep = !DROP || bf_half(bits, r) >= a.drop.threshold;
            if (k0 + j < seen) (keep && s[t * 8 + r] > -INFINITY ? with : without) |= 1u << j;
          }
        }
        with |= __float_as_uint(swap_halves(__uint_as_float(with)));
        without |= __float_as_uint(swap_halves(__uint_as_float(without)));
        for (; left; left &= left - 1) {
          const int j = __builtin_ctz(left), h2 = here<true>(half);
#pragma unroll
          for (int i = 0; i < kDT; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const T x = KV::value(lds[0][1], at + j, i * 32 + row_of(r, h2));
              if (!finite(x)) o[i][r] += with >> j & 1 ? static_cast<float>(x) : without >> j & 1 ? NAN : 0.f;
            }
        }
      }
      if (at + 32 == BN) __syncthreads();  // the buffer is free
    }
  }
  l += swap_halves(l);
  // a slice may have no key that the row sees; a row whose scores are all -inf
  // has no softmax
  const bool none = a.key_slices > 1 && l == 0.f;
  finish(none ? 0.f : (DROP ? a.drop.scale : 1.f) / l, none ? -INFINITY : m * c + log2f(l));
}

// the slices' rows into one, each by its share of the sum: four columns a lane
template <typename T>
__global__ __launch_bounds__(256) void attn_join_k(BfAttnArgs a) {
  const long all = static_cast<long>(a.rows) * a.heads;
  const int each = (a.dim + 3) / 4;
  const long i = static_cast<long>(blockIdx.x) * 256 + threadIdx.x;
  const long at = i / each;  // row and head
  const int c = static_cast<int>(i % each) * 4, n = min(4, a.dim - c);
  if (at >= all) return;
  const float* sums = a.partial + a.key_slices * all * a.dim + at % a.heads * a.rows + at / a.heads;
  float top = -INFINITY, total = 0.f, out[4] = {};
  for (int s = 0; s < a.key_slices; ++s) top = fmaxf(top, sums[s * all]);
  for (int s = 0; s < a.key_slices; ++s) {
    const float share = exp2f(sums[s * all] - top);
    const float* part = a.partial + (s * all + at) * a.dim + c;
    float x[4];
    if (n == 4) __builtin_memcpy(x, part, sizeof(x));
    else
      for (int u = 0; u < 4; ++u) x[u] = u < n ? part[u] : 0.f;
    total += share;
#pragma unroll
    for (int u = 0; u < 4; ++u) out[u] += fabsf(x[u]) < INFINITY ? share * x[u] : x[u];  // a share may round to 0
  }
  T* o = static_cast<T*>(a.o) + at * a.dim + c;
  T* rest = a.rest ? static_cast<T*>(a.rest) + at * a.dim + c : nullptr;
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (u < n) {
      out[u] /= total;
      o[u] = static_cast<T>(out[u]);
      if (rest) rest[u] = static_cast<T>(out[u] - static_cast<float>(o[u]));
    }
  if (a.lse && c == 0) a.lse[at % a.heads * a.rows + at / a.heads] = top + log2f(total);
}

// ---------------------------------------------------------------------------
// backward, dq: the same loop as forward, with dP^T = v dO^T beside S^T, and
// dq^T = k^T dS^T. Its first act is delta, which the other kernel reads: from O
// as it was before it was rounded (the forward pass keeps the rest, in the same
// type), since delta's error goes into all dS of a row at once. With the rounded
// O, dq and dk were 1.6 times as far off as the rounding of P and dS makes them.
//
// A row's dS sum to 0, but their roundings do not, and softmax has picked keys
// that lie along q: the roundings' sum moves dq by their mean. So what dS
// lost goes through the matrix units too, on the fragments that are there: dq is
// 1.05 to 1.15 times as far off as its own rounding, 1.45 to 1.6 times without
// (13195 tokens, 16 heads of 128, causal: 0.38 ms, and 0.31 without).
//
// f16 would lose small dS and overflow with large ones, whatever dO's size.
// Its dS is held times a power of two of its own for each lane's row (or key),
// lowered with the accumulators when a tile brings a larger value.
// ---------------------------------------------------------------------------

template <typename T>
constexpr bool kScaled = false;
template <>
constexpr bool kScaled<_Float16> = true;
// power of two that P is held times in the backward pass
template <typename T>
constexpr float kPower = kScaled<T> ? 12.f : 0.f;

template <int TILES>
__device__ __forceinline__ void rescale(Acc (&acc)[TILES], float& factor, const float* x) {
  float top = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(x[r]));
  top = fmaxf(top, swap_halves(top));
  const bool lower = top < INFINITY && top > 0.f && (factor == 0.f || top * factor > 32768.f);
  if (!__any(lower)) return;
  if (lower) {
    int e;
    frexpf(top, &e);
    const float next = ldexpf(1.f, min(14 - e, 100));
    const float by = factor == 0.f ? 1.f : next / factor;
    factor = next;
#pragma unroll
    for (int i = 0; i < TILES; ++i) acc[i] *= by;
  }
}

template <typename T, int DP, bool VEC, bool DROP>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(kDqWaves<T, DP>, kDqWaves<T, DP>))) void attn_dq_k(BfAttnArgs a) {
  constexpr int kQ = kRows, BN = kKeys<T>, kSub = BN / 32, kSteps = DP / 16, kDT = DP / 32;
  typedef Tile<T, BN, DP, 256, VEC> KV;
  __shared__ __align__(1024) char lds[2][2][KV::kBytes];
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x >> 6;
  const Unit unit = unit_of(blockIdx.x, a.heads);
  const int h = unit.head, g = h / (a.heads / a.kv_heads);
  const int slice = unit.number % a.key_slices;
  const Work w = find_tile(a, unit.number / a.key_slices, kQ, a.causal);
  if (!w.any) return;
  const int q0 = w.tile * kQ, qw = q0 + wave * 32, qi = qw + (lane & 31);
  const bool inside = qi < w.len;
  const long row = w.begin + min(qi, w.len - 1), at = static_cast<long>(h) * a.rows + row;
  Acc dq[kDT];
#pragma unroll
  for (int i = 0; i < kDT; ++i) dq[i] = Acc{};
  const auto finish = [&](float f) __attribute__((always_inline)) {
    const long out = (row * a.heads + h) * a.dim;
    if (a.key_slices == 1) store_row<VEC>(static_cast<T*>(a.dq) + out, dq, f, half, a.dim, inside);
    else
      store_row<VEC>(a.partial + slice * static_cast<long>(a.rows) * a.heads * a.dim + out, dq, f, half, a.dim, inside);
  };
  if (w.seq == a.seqs) {  // behind the last sequence
    finish(0.f);
    return;
  }
  typedef Loader<T, BN, DP, 256, VEC> Load;
  const Load k(static_cast<const T*>(a.k) + w.begin * a.k_row + g * a.k_head, a.k_row, a.dim);
  const Load v(static_cast<const T*>(a.v) + w.begin * a.v_row + g * a.v_head, a.v_row, a.dim);
  const int last = w.len - 1;
  const int2 range = keys_of(a.causal ? min(w.len, q0 + kQ) : w.len, BN, slice, a.key_slices);
  if (range.x >= range.y && slice) {  // slice 0 has delta to write
    finish(0.f);
    return;
  }
  if (a.dim < DP) {
    KV::clear(&lds[0][0][0], sizeof(lds));
    __syncthreads();
  }
  k.load(lds[0][0], range.x, last);
  v.load(lds[0][1], range.x, last);
  Frag<T> qf[kSteps], gf[kSteps];
  float delta = 0.f;
  {
    const T* q = static_cast<const T*>(a.q) + row * a.q_row + h * a.q_head;
    const T* go = static_cast<const T*>(a.dout) + row * a.do_row + h * a.do_head;
    const T* o = static_cast<const T*>(a.out) + (row * a.heads + h) * a.dim;
    const T* rest = a.rest ? static_cast<const T*>(a.rest) + (row * a.heads + h) * a.dim : nullptr;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      qf[s] = load_row<VEC>(q, s, half, a.dim);
      gf[s] = load_row<VEC>(go, s, half, a.dim);
      const Frag<T> of = load_row<VEC>(o, s, half, a.dim);
#pragma unroll
      for (int i = 0; i < 8; ++i) delta += static_cast<float>(gf[s][i]) * static_cast<float>(of[i]);
      if (rest) {
        const Frag<T> rf = load_row<VEC>(rest, s, half, a.dim);
#pragma unroll
        for (int i = 0; i < 8; ++i) delta += static_cast<float>(gf[s][i]) * static_cast<float>(rf[i]);
      }
    }
    delta += swap_halves(delta);
  }
  if (inside && half == 0 && slice == 0) a.delta[at] = delta;
  const BfKey key = DROP ? bf_key(a.drop) : BfKey{0, 0};
  const float c = a.scale * kLog2e, lse = a.lse[at] - kPower<T>;
  // keys of the lane's row that have a dS: a row that sees one key has P = 1
  // whatever its score, and dS is 0, not the rounding of dP - delta
  int seen = a.causal ? min(w.len, qi + 1) : w.len;
  seen = seen == 1 ? 0 : seen;
  float factor = 0.f;  // f16: what dS is held times
  loads_done();
  for (int k0 = range.x, buf = 0; k0 < range.y; k0 += BN, buf ^= 1) {
    if (k0 + BN < range.y) {
      k.load(lds[buf ^ 1][0], k0 + BN, last);
      v.load(lds[buf ^ 1][1], k0 + BN, last);
    }
    if (qw < w.len && !(a.causal && k0 > qw + 31)) {
      const bool masked = k0 + BN > w.len || (a.causal && (k0 + BN - 1 > qw || qw == 0));
      const int rows = KV::row_place(lane & 31, half), columns = KV::columns_place(lane);
#pragma unroll
      for (int u = 0; u < kSub; ++u) {
        if (u && masked && k0 + u * 32 >= (a.causal ? min(w.len, qw + 32) : w.len)) continue;  // none sees them
        Acc s{}, dp{};
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          s = mma(KV::read_row(lds[buf][0], rows, u * 32, i, half), qf[i], s);
          dp = mma(KV::read_row(lds[buf][1], rows, u * 32, i, half), gf[i], dp);
        }
        if (sizeof(T) == 2) feed<8, 2 * kSteps, 1>();
        float ds[16];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          uint4 bits;
          if (DROP)
            bits = bf_philox((k0 / 16 + u * 2 + t) * 2 + half, static_cast<uint32_t>(row), h, a.drop.offset, key);
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            float x = dp[t * 8 + r];
            if (DROP) x = bf_half(bits, r) >= a.drop.threshold ? x * a.drop.scale : 0.f;
            ds[t * 8 + r] = __builtin_amdgcn_exp2f(s[t * 8 + r] * c - lse) * (x - delta);
          }
        }
        if (masked) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int j = k0 + u * 32 + row_of(r, half);
            ds[r] = j < seen ? ds[r] : 0.f;
          }
        }
        if constexpr (kScaled<T>) {
          rescale(dq, factor, ds);
#pragma unroll
          for (int r = 0; r < 16; ++r) ds[r] *= factor;
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const Frag<T> f = rounded<T>(ds + t * 8), less = rest_of<T>(ds + t * 8, f);
#pragma unroll
          for (int i = 0; i < kDT; ++i) {
            const Frag<T> kt = KV::read_columns(lds[buf][0], columns, u * 32 + t * 16, i);
            dq[i] = mma(kt, f, dq[i]);
            if (sizeof(T) == 2) dq[i] = mma(kt, less, dq[i]);
          }
        }
        if (sizeof(T) == 2) feed<8, 4 * kDT, 1>();
      }
    }
    loads_done();
  }
  const float f = kScaled<T> ? (factor == 0.f ? 1.f : exp2f(-kPower<T>) / factor) : 1.f;
  finish(a.scale * f);
}

// ---------------------------------------------------------------------------
// backward, dk and dv: a wave has 32 keys, one to a lane of each half, and goes
// over the queries that see them, head by head of the group. S = q k^T and dP
// lie with a key's queries in the registers of its lane pair, so that P and dS
// are the operands of dv^T = dO^T P and dk^T = q^T dS as they stand.
//
// What dS lost to rounding is multiplied too, as for dq: dk is 1.02 to 1.24 times
// as far off as its own rounding, 1.41 to 1.51 times without (13195 tokens, 16
// heads of 128, causal: 0.55 ms, and 0.47 without). P's rounding stays in dv, which
// is 1.2 to 1.42 times as far off.
// ---------------------------------------------------------------------------

// A workgroup has 128 keys, four waves of 32, and a step is some queries of
// one head. What a workgroup does in a step:
//   SUBS  tiles of 32 queries that a wave takes
//   SPLIT 2: four more waves have the same keys and take other queries; their
//         sums meet in LDS at the end
//   V_IN_LDS: v's fragments are read again rather than kept in registers
//   WAVES of a SIMD whose registers it is held to
//
// Heads of 128: the sums take 128 registers. Eight waves, two to a SIMD, reached
// 735 TFLOP/s (16384 tokens, 16 heads, bf16, dS rounded once); four with all registers 630.
template <typename T, int DP>
struct DkvShape {
  static constexpr bool kHalf = sizeof(T) == 2, kWide = DP == 128;
  static constexpr int kSplit = kHalf && kWide ? 2 : 1;
  static constexpr int kSubs = kHalf && !kWide ? 2 : 1;  // f32: LDS holds 32 queries a step
  static constexpr int kWaves = kWide && !kHalf ? 1 : 2;
  static constexpr bool kVInLds = kWide;
};

// the sums of the second four waves to those of the first, through LDS
template <int TILES>
__device__ __forceinline__ void join(Acc (&acc)[TILES], void* lds, int part) {
  Acc* place = static_cast<Acc*>(lds) + ((threadIdx.x >> 6) & 3) * TILES * 64 + (threadIdx.x & 63);
  if (part) {
#pragma unroll
    for (int i = 0; i < TILES; ++i) place[i * 64] = acc[i];
  }
  __syncthreads();
  if (!part) {
#pragma unroll
    for (int i = 0; i < TILES; ++i) acc[i] += place[i * 64];
  }
}

template <typename T, int DP, bool VEC, bool DROP>
__global__ __launch_bounds__((256 * DkvShape<T, DP>::kSplit))
__attribute__((amdgpu_waves_per_eu(DkvShape<T, DP>::kWaves, DkvShape<T, DP>::kWaves))) void attn_dkv_k(BfAttnArgs a) {
  typedef DkvShape<T, DP> Shape;
  constexpr int kK = kRows, SPLIT = Shape::kSplit, SUBS = Shape::kSubs, THREADS = 256 * SPLIT;
  constexpr int BM = 32 * SPLIT * SUBS;  // queries of a step
  constexpr int kSteps = DP / 16, kDT = DP / 32;
  constexpr bool V_IN_LDS = Shape::kVInLds;
  constexpr bool kHide = sizeof(T) == 2 && DP == 128;  // 670 TFLOP/s without, 710 with (dS rounded once)
  typedef Tile<T, BM, DP, THREADS, VEC> QG;
  typedef Tile<T, kK, DP, THREADS, VEC> Values;
  __shared__ __align__(1024) char lds[2][2][QG::kBytes];
  __shared__ __align__(1024) char v_lds[V_IN_LDS ? Values::kBytes : 16];
  __shared__ __align__(16) float stat[2][2][64];  // lse and delta of the tile's queries
  __shared__ __align__(16) uint32_t kept[4 * SPLIT][DROP ? 32 : 4];  // a wave's mask: a query's 32 keys to a word
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x >> 6, part = wave >> 2;
  const Unit unit = unit_of(blockIdx.x, a.kv_heads);
  const int g = unit.head, group = a.heads / a.kv_heads;
  const int slice = unit.number % a.query_slices;  // of the steps
  Work w = find_tile(a, unit.number / a.query_slices, kK, a.causal);
  if (!w.any) return;
  if (a.causal) w.tile = (w.len - 1) / kK - w.tile;  // the first keys have most queries
  const int j0 = w.tile * kK, jl = (wave & 3) * 32 + (lane & 31), jw = j0 + (wave & 3) * 32, ji = j0 + jl;
  const bool inside = ji < w.len && part == 0;
  const long row = w.begin + min(ji, w.len - 1), out = (row * a.kv_heads + g) * a.dim;
  Acc dk[kDT], dv[kDT];
#pragma unroll
  for (int i = 0; i < kDT; ++i) dk[i] = dv[i] = Acc{};
  const auto finish = [&]() __attribute__((always_inline)) {
    if (a.query_slices == 1) {
      store_row<VEC>(static_cast<T*>(a.dk) + out, dk, 1.f, half, a.dim, inside);
      store_row<VEC>(static_cast<T*>(a.dv) + out, dv, 1.f, half, a.dim, inside);
    } else {
      const long all = static_cast<long>(a.rows) * a.kv_heads * a.dim;
      store_row<VEC>(a.partial + 2 * slice * all + out, dk, 1.f, half, a.dim, inside);
      store_row<VEC>(a.partial + (2 * slice + 1) * all + out, dv, 1.f, half, a.dim, inside);
    }
  };
  if (w.seq == a.seqs) {  // behind the last sequence
    finish();
    return;
  }
  const int last = w.len - 1;
  if (a.dim < DP) {
    QG::clear(&lds[0][0][0], sizeof(lds));
    if (V_IN_LDS) Values::clear(v_lds, sizeof(v_lds));
    __syncthreads();
  }
  Frag<T> kf[kSteps], vf[V_IN_LDS ? 1 : kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    kf[s] = load_row<VEC>(static_cast<const T*>(a.k) + row * a.k_row + g * a.k_head, s, half, a.dim);
    if (!V_IN_LDS) vf[s] = load_row<VEC>(static_cast<const T*>(a.v) + row * a.v_row + g * a.v_head, s, half, a.dim);
  }
  if (V_IN_LDS)
    Loader<T, kK, DP, THREADS, VEC>(static_cast<const T*>(a.v) + w.begin * a.v_row + g * a.v_head, a.v_row, a.dim)
        .load(v_lds, j0, last);
  const int first = a.causal ? j0 / BM * BM : 0;  // queries in front of the keys see none of them
  const int from = a.causal ? ji : 0;  // first query that sees the lane's key
  const int from_ds = a.causal ? max(ji, 1) : w.len == 1 ? 1 : 0;  // and has another: with one key dS is 0
  const int steps = (w.len - first + BM - 1) / BM, total = steps * group;
  const int begin = static_cast<int>(static_cast<long>(total) * slice / a.query_slices);
  const int end = static_cast<int>(static_cast<long>(total) * (slice + 1) / a.query_slices);
  typedef Loader<T, BM, DP, THREADS, VEC> Load;
  Load q(nullptr, a.q_row, a.dim), go(nullptr, a.do_row, a.dim);
  const auto fetch = [&](int h, int i0, int buf) __attribute__((always_inline)) {
    q.base = reinterpret_cast<const char*>(static_cast<const T*>(a.q) + w.begin * a.q_row + h * a.q_head);
    go.base = reinterpret_cast<const char*>(static_cast<const T*>(a.dout) + w.begin * a.do_row + h * a.do_head);
    q.load(lds[buf][0], i0, last);
    go.load(lds[buf][1], i0, last);
    if (wave < 2 && lane < BM) {
      const float* from = (wave ? a.delta : a.lse) + static_cast<long>(h) * a.rows + w.begin + min(i0 + lane, last);
      load_to_lds<4>(from, stat[buf][wave]);
    }
  };
  const BfKey key = DROP ? bf_key(a.drop) : BfKey{0, 0};
  const float c = a.scale * kLog2e;
  float factor = 0.f;
  int h = g * group + begin / steps, i0 = first + begin % steps * BM;  // head and queries of a step, and of the next
  if (begin < end) fetch(h, i0, 0);
  loads_done();
  for (int n = begin, buf = 0, next_h, next_i0; n < end; ++n, buf ^= 1, h = next_h, i0 = next_i0) {
    next_h = h, next_i0 = i0 + BM;
    if (next_i0 >= w.len) ++next_h, next_i0 = first;
    if (n + 1 < end) fetch(next_h, next_i0, buf ^ 1);
#pragma unroll
    for (int n32 = 0; n32 < SUBS; ++n32) {
      const int sub = (part * SUBS + n32) * 32, iw = i0 + sub;  // the wave's queries
      if (jw < w.len && iw < w.len && !(a.causal && iw + 31 < jw)) {
        const bool masked = iw + 32 > w.len || (a.causal && (iw < jw + 31 || iw == 0)) || w.len == 1;
        const int rows = here<kHide>(QG::row_place(lane & 31, half)), columns = here<kHide>(QG::columns_place(lane));
        const int own = here<kHide>(Values::row_place(jl, half));
        Acc s{}, dp{};
#pragma unroll
        for (int i = 0; i < kSteps; ++i) s = mma(QG::read_row(lds[buf][0], rows, sub, i, half), kf[i], s);
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
          dp = mma(QG::read_row(lds[buf][1], rows, sub, i, half),
                   V_IN_LDS ? Values::read_row(v_lds, own, 0, i, half) : vf[V_IN_LDS ? 0 : i], dp);
        if (sizeof(T) == 2) feed<6, 2 * kSteps, 2>();
        if (DROP) {
          // the lane's share of a query's mask, as the forward pass has it
          uint32_t bits = 0;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const uint4 x = bf_philox((jw / 16 + t) * 2 + half, static_cast<uint32_t>(w.begin + iw + (lane & 31)), h,
                                      a.drop.offset, key);
#pragma unroll
            for (int r = 0; r < 8; ++r)
              bits |= (bf_half(x, r) >= a.drop.threshold ? 1u : 0u) << (t * 16 + 8 * (r >> 2) + (r & 3));
          }
          bits <<= 4 * half;
          bits |= __float_as_uint(swap_halves(__uint_as_float(bits)));
          wave_exchange();  // the last mask is read
          if (half == 0) kept[wave][lane] = bits;
          wave_exchange();
        }
        float p[16], ds[16];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const float4 lse = *reinterpret_cast<const float4*>(&stat[buf][0][sub + t * 8 + half * 4]);
          const float4 delta = *reinterpret_cast<const float4*>(&stat[buf][1][sub + t * 8 + half * 4]);
          uint4 m = uint4{0, 0, 0, 0};
          if (DROP) m = *reinterpret_cast<const uint4*>(&kept[wave][t * 8 + half * 4]);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float l = r == 0 ? lse.x : r == 1 ? lse.y : r == 2 ? lse.z : lse.w;
            const float d = r == 0 ? delta.x : r == 1 ? delta.y : r == 2 ? delta.z : delta.w;
            const uint32_t word = r == 0 ? m.x : r == 1 ? m.y : r == 2 ? m.z : m.w;
            const float x = __builtin_amdgcn_exp2f(s[t * 4 + r] * c - (l - kPower<T>));
            const bool keep = !DROP || (word >> (lane & 31)) & 1;
            const float y = keep ? (DROP ? dp[t * 4 + r] * a.drop.scale : dp[t * 4 + r]) : 0.f;
            p[t * 4 + r] = keep ? x : 0.f;
            ds[t * 4 + r] = x * (y - d);
          }
        }
        if (masked) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int i = iw + row_of(r, half);
            p[r] = i >= from && i < w.len ? p[r] : 0.f;
            ds[r] = i >= from_ds && i < w.len ? ds[r] : 0.f;
          }
        }
        if constexpr (kScaled<T>) {
          rescale(dk, factor, ds);
#pragma unroll
          for (int r = 0; r < 16; ++r) ds[r] *= factor;
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const Frag<T> pf = rounded<T>(p + t * 8), df = rounded<T>(ds + t * 8), less = rest_of<T>(ds + t * 8, df);
#pragma unroll
          for (int i = 0; i < kDT; ++i) {
            dv[i] = mma(QG::read_columns(lds[buf][1], columns, sub + t * 16, i), pf, dv[i]);
            const Frag<T> qt = QG::read_columns(lds[buf][0], columns, sub + t * 16, i);
            dk[i] = mma(qt, df, dk[i]);
            if (sizeof(T) == 2) dk[i] = mma(qt, less, dk[i]);
          }
        }
        if (sizeof(T) == 2) feed<8, 6 * kDT, 1>();
      }
    }
    loads_done();
  }
  const float power = exp2f(-kPower<T>), f = kScaled<T> ? (factor == 0.f ? 1.f : power / factor) : 1.f;
#pragma unroll
  for (int i = 0; i < kDT; ++i) {
    dk[i] *= a.scale * f;
    dv[i] *= power * (DROP ? a.drop.scale : 1.f);
  }
  if constexpr (SPLIT == 2) {
    join(dk, &lds[0][0][0], part);
    __syncthreads();
    join(dv, &lds[0][0][0], part);
  }
  finish();
}

// the slices' gradients into one, in a fixed order: dq, or dk and dv, which lie
// side by side in a slice
template <typename T>
__global__ __launch_bounds__(256) void attn_fold_k(T* first, T* second, const float* partial, long all, int slices) {
  const long i = (static_cast<long>(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (i >= all) return;
  const int n = all - i < 4 ? static_cast<int>(all - i) : 4;
  const long next = all * gridDim.y;
  partial += blockIdx.y * all + i;
  float sum[4] = {};
  for (int s = 0; s < slices; ++s) {
    float x[4];
    if (n == 4) __builtin_memcpy(x, partial + s * next, sizeof(x));
    else
      for (int u = 0; u < 4; ++u) x[u] = u < n ? partial[s * next + u] : 0.f;
#pragma unroll
    for (int u = 0; u < 4; ++u) sum[u] += x[u];
  }
  T* out = (blockIdx.y ? second : first) + i;
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (u < n) out[u] = static_cast<T>(sum[u]);
}

__global__ __launch_bounds__(1024) void attn_table_k(BfAttnArgs a, int* table) { make_table(a, table, kRows); }

constexpr long kMostThreads = 0xFFFFFFFF;  // of a launch

template <typename T>
hipError_t fold(void* first, void* second, const float* partial, long all, int slices, hipStream_t stream) {
  const long blocks = (all + 1023) / 1024;  // slices have few rows: far from kMostThreads
  hipLaunchKernelGGL(attn_fold_k<T>, dim3(blocks, second ? 2 : 1), dim3(256), 0, stream, static_cast<T*>(first),
                     static_cast<T*>(second), partial, all, slices);
  return hipGetLastError();
}

template <typename T, int DP, bool VEC>
hipError_t fwd(const BfAttnArgs& a, hipStream_t stream) {
  const long groups = units(most_tiles(a, kRows) * a.key_slices, a.heads);
  if (groups * 256 > kMostThreads) return hipErrorInvalidValue;
  if (a.drop.threshold) hipLaunchKernelGGL((attn_fwd_k<T, DP, VEC, true>), dim3(groups), dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((attn_fwd_k<T, DP, VEC, false>), dim3(groups), dim3(256), 0, stream, a);
  if (hipError_t e = hipGetLastError()) return e;
  if (a.key_slices == 1) return hipSuccess;
  const long blocks = (static_cast<long>(a.rows) * a.heads * ((a.dim + 3) / 4) + 255) / 256;
  hipLaunchKernelGGL(attn_join_k<T>, dim3(blocks), dim3(256), 0, stream, a);
  return hipGetLastError();
}

template <typename T>
hipError_t fwd(const BfAttnArgs& a, hipStream_t stream) {
  if (!a.vec) return a.dim <= 64 ? fwd<T, 64, false>(a, stream) : fwd<T, 128, false>(a, stream);
  return a.dim <= 64 ? fwd<T, 64, true>(a, stream) : fwd<T, 128, true>(a, stream);
}

template <typename T, int DP, bool VEC, bool DROP>
hipError_t bwd(const BfAttnArgs& a, bool need_dkv, hipStream_t stream) {
  constexpr int kThreads = 256 * DkvShape<T, DP>::kSplit;
  const long groups = units(most_tiles(a, kRows) * a.key_slices, a.heads);
  const long shared = units(most_tiles(a, kRows) * a.query_slices, a.kv_heads);
  if (groups * 256 > kMostThreads || shared * kThreads > kMostThreads) return hipErrorInvalidValue;
  hipLaunchKernelGGL((attn_dq_k<T, DP, VEC, DROP>), dim3(groups), dim3(256), 0, stream, a);
  if (hipError_t e = hipGetLastError()) return e;
  if (a.key_slices > 1)
    if (hipError_t e = fold<T>(a.dq, nullptr, a.partial, static_cast<long>(a.rows) * a.heads * a.dim, a.key_slices, stream))
      return e;
  if (!need_dkv) return hipSuccess;
  hipLaunchKernelGGL((attn_dkv_k<T, DP, VEC, DROP>), dim3(shared), dim3(kThreads), 0, stream, a);
  if (hipError_t e = hipGetLastError()) return e;
  if (a.query_slices == 1) return hipSuccess;
  return fold<T>(a.dk, a.dv, a.partial, static_cast<long>(a.rows) * a.kv_heads * a.dim, a.query_slices, stream);
}

template <typename T, int DP, bool VEC>
hipError_t bwd(const BfAttnArgs& a, bool need_dkv, hipStream_t stream) {
  return a.drop.threshold ? bwd<T, DP, VEC, true>(a, need_dkv, stream) : bwd<T, DP, VEC, false>(a, need_dkv, stream);
}

template <typename T>
hipError_t bwd(const BfAttnArgs& a, bool need_dkv, hipStream_t stream) {
  if (!a.vec) return a.dim <= 64 ? bwd<T, 64, false>(a, need_dkv, stream) : bwd<T, 128, false>(a, need_dkv, stream);
  return a.dim <= 64 ? bwd<T, 64, true>(a, need_dkv, stream) : bwd<T, 128, true>(a, need_dkv, stream);
}

int slices(long wanted, long most) {
  const long n = wanted < most ? wanted : most;
  return static_cast<int>(n < 1 ? 1 : n > 16 ? 16 : n);
}

}  // namespace

extern "C" {

// Slices of the long axis: a workgroup goes over all keys of its rows, or (dk
// and dv) over all queries of its keys and head group. Few tokens or few key
// heads leave few workgroups, which then take a share of that axis each; a second
// kernel joins the shares, from 32-bit sums in memory. That pays up to about two
// workgroups of a CU. With dS rounded once, forward and backward of 1689 tokens
// (10/2 heads of 80) took 137 us with slices and 417 without, but those of 4 K
// tokens under 8 heads of 128 took 469 us with a target of 512 workgroups, 576 with 1024.
constexpr long kWanted = 512;

int bf_attn_key_slices(const BfAttnArgs* a, int dtype) {
  const long groups = (a->rows + 127L) / 128 * a->heads;
  const long length = a->rows / (a->seqs > 0 ? a->seqs : 1);
  return slices((kWanted + groups - 1) / groups, (length + 63) / 64 * (dtype == 0 ? 2 : 1) / 2);
}

int bf_attn_query_slices(const BfAttnArgs* a, int dtype) {
  const long groups = (a->rows + 127L) / 128 * a->kv_heads;
  const long length = a->rows / (a->seqs > 0 ? a->seqs : 1);
  const long steps = (length + 63) / 64 * (a->heads / a->kv_heads) * (dtype == 0 ? 2 : 1);
  return slices((kWanted + groups - 1) / groups, steps / 2);
}

long bf_attn_partial_floats(const BfAttnArgs* a) {
  const long wide = static_cast<long>(a->rows) * a->heads, narrow = static_cast<long>(a->rows) * a->kv_heads;
  const long keys = a->key_slices > 1 ? a->key_slices * wide * (a->dim + 1) : 0;
  const long queries = a->query_slices > 1 ? a->query_slices * narrow * a->dim * 2 : 0;
  return keys > queries ? keys : queries;
}

// Whether the launches have room for the workgroups of any bounds: fewer than
// 2^24 tiles and heads together, or 2^23 for dk and dv of wide half-type heads,
// whose workgroups are twice as large.
int bf_attn_fits(const BfAttnArgs* a, int dtype, int backward) {
  if (a->rows == 0) return 1;  // nothing is launched
  const long tiles = most_tiles(*a, kRows);
  if (units(tiles * bf_attn_key_slices(a, dtype), a->heads) * 256 > kMostThreads) return 0;
  const int threads = dtype != 0 && a->dim > 64 ? 512 : 256;
  return !backward || units(tiles * bf_attn_query_slices(a, dtype), a->kv_heads) * threads <= kMostThreads;
}

int bf_attn_table_ints(const BfAttnArgs* a) { return a->seqs > kLanes ? a->seqs + 1 : 0; }

hipError_t bf_attn_table(const BfAttnArgs* a, int* table, hipStream_t stream) {
  hipLaunchKernelGGL(attn_table_k, dim3(1), dim3(1024), 0, stream, *a, table);
  return hipGetLastError();
}

hipError_t bf_attn_fwd(const BfAttnArgs* a, int dtype, hipStream_t stream) {
  switch (dtype) {
    case 0: return fwd<float>(*a, stream);
    case 2: return fwd<_Float16>(*a, stream);
    case 3: return fwd<__bf16>(*a, stream);
  }
  return hipErrorInvalidValue;
}

hipError_t bf_attn_bwd(const BfAttnArgs* a, int dtype, int need_dkv, hipStream_t stream) {
  switch (dtype) {
    case 0: return bwd<float>(*a, need_dkv, stream);
    case 2: return bwd<_Float16>(*a, need_dkv, stream);
    case 3: return bwd<__bf16>(*a, need_dkv, stream);
  }
  return hipErrorInvalidValue;
}

}  // extern "C"
