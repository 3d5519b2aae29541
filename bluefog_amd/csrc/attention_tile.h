// Copyright 2026. Licensed under the Apache License, Version 2.0.
//
// What the attention kernels share: matrix fragments, LDS tiles, the search
// for a workgroup's rows.
//
// All products run on 32x32 matrix tiles. A fragment is 8 values of a lane: of
// row (or column) lane & 31, at the inner positions 8 * (lane >> 5) ... + 7 of
// a step of 16. Half-precision types have one instruction for a step
// (32x32x16); f32 takes eight 32x32x2, of which number i multiplies value i of
// both halves, which is the same sum in another order. The accumulator holds
// column lane & 31 and, in register r, row 8 * (r >> 2) + 4 * (lane >> 5) +
// (r & 3).
//
// That accumulator is the next product's operand as it stands: eight of its
// registers are the inner positions {4 half ... + 3, 8 + 4 half ... + 3} of a
// step of 16, and the other operand is read in the same order (read_columns).
#pragma once

#include <hip/hip_runtime.h>

#include "convert.h"
#include "counter_rng.h"
#include "transformer_kernels.h"

namespace bf_attn {

typedef float Acc __attribute__((ext_vector_type(16)));

template <typename T>
struct FragOf {
  typedef T type __attribute__((ext_vector_type(8)));
};
template <typename T>
using Frag = typename FragOf<T>::type;

// eight values rounded at once: two to an instruction
template <typename T>
__device__ __forceinline__ Frag<T> rounded(const float* x) {
  typedef float F8 __attribute__((ext_vector_type(8)));
  F8 f;
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = x[i];
  return __builtin_convertvector(f, Frag<T>);
}

// and what that took from them
template <typename T>
__device__ __forceinline__ Frag<T> rest_of(const float* x, Frag<T> of) {
  float less[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) less[i] = x[i] - static_cast<float>(of[i]);
  return rounded<T>(less);
}

template <typename T>
__device__ __forceinline__ bool finite(T x) { return fabsf(static_cast<float>(x)) < INFINITY; }

__device__ __forceinline__ Acc mma(Frag<__bf16> a, Frag<__bf16> b, Acc c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ Acc mma(Frag<_Float16> a, Frag<_Float16> b, Acc c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ Acc mma(Frag<float> a, Frag<float> b, Acc c) {
#pragma unroll
  for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
  return c;
}

// inner position of accumulator register r
__device__ __forceinline__ int row_of(int r, int half) { return 8 * (r >> 2) + 4 * half + (r & 3); }

// BYTES of each active lane's memory to lds + BYTES * lane, without a register
template <int BYTES>
__device__ __forceinline__ void load_to_lds(const void* from, void* lds) {
  const auto* g = (const __attribute__((address_space(1))) void*)from;
  auto* l = (__attribute__((address_space(3))) void*)lds;
  static_assert(BYTES == 4 || BYTES == 16, "a load's size");
  if constexpr (BYTES == 16) __builtin_amdgcn_global_load_lds(g, l, 16, 0, 0);
  else __builtin_amdgcn_global_load_lds(g, l, 4, 0, 0);
}

// ---------------------------------------------------------------------------
// LDS tiles: ROWS rows of DP columns, 16-byte chunks, chunk c of row r at
// c ^ swizzle(r). Eight neighbouring rows' chunks lie in different banks (a
// fragment of rows), and so do the chunk pairs of four (a fragment of columns).
// ---------------------------------------------------------------------------

template <typename T, int ROWS, int DP, int THREADS, bool VEC>
struct Tile {
  static constexpr int kEach = 16 / sizeof(T);  // values of a chunk
  static constexpr int kChunks = DP / kEach;
  static constexpr int kRowBytes = DP * sizeof(T);
  static constexpr int kBytes = ROWS * kRowBytes;

  static __device__ __forceinline__ int swizzle(int r) {
    return kChunks == 8 ? (((r >> 1) & 3) << 1) | ((r >> 3) & 1) : ((r & 7) << 1) | ((r >> 3) & 1);
  }
  static __device__ __forceinline__ int at(int row, int chunk) {
    return row * kRowBytes + ((chunk ^ swizzle(row)) << 4);
  }

  static __device__ __forceinline__ void clear(char* lds, int bytes) {
    for (int i = threadIdx.x * 16; i < bytes; i += THREADS * 16) *reinterpret_cast<uint4*>(lds + i) = uint4{0, 0, 0, 0};
  }

  static __device__ __forceinline__ T value(const char* lds, int row, int column) {
    return *reinterpret_cast<const T*>(lds + at(row, column / kEach) + column % kEach * sizeof(T));
  }

  // Places of a lane in a tile, from which those of its fragments differ in bits
  // of the chunk: row_place for row `row` (columns of step 0), columns_place for
  // column `lane & 31` (rows 0 and on). For f32 they are row and lane themselves.
  static __device__ __forceinline__ int row_place(int row, int half) {
    return sizeof(T) == 2 ? at(row, half) : row;
  }
  static __device__ __forceinline__ int columns_place(int lane) {
    if (sizeof(T) == 4) return lane;
    // sixteen lanes give the addresses of 4 rows of 16 values, four to a lane
    return at(4 * (lane >> 5) + ((lane & 15) >> 2), ((lane & 16) >> 3) + ((lane & 3) >> 1)) + (lane & 1) * 8;
  }

  // fragment of the place's row, `down` (a multiple of 16) rows on, inner
  // positions = columns of step `step`
  static __device__ __forceinline__ Frag<T> read_row(const char* lds, int place, int down, int step, int half) {
    Frag<T> f;
    if constexpr (sizeof(T) == 2) {
      f = *reinterpret_cast<const Frag<T>*>(lds + (place ^ (step << 5)) + down * kRowBytes);
    } else {
      typedef float F4 __attribute__((ext_vector_type(4)));
      const F4 x = *reinterpret_cast<const F4*>(lds + at(place + down, step * 4 + half * 2));
      const F4 y = *reinterpret_cast<const F4*>(lds + at(place + down, step * 4 + half * 2 + 1));
      f = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    }
    return f;
  }

  // fragment of the place's column, 32 * dt columns on, inner positions = rows
  // base (a multiple of 16) + {4 half .. + 3, 8 + 4 half .. + 3}
  static __device__ __forceinline__ Frag<T> read_columns(const char* lds, int place, int base, int dt) {
    Frag<T> f;
    if constexpr (sizeof(T) == 2) {
      // the transposing read: lane i of sixteen gets column i of the four rows
      typedef short S4 __attribute__((ext_vector_type(4)));
      S4 part[2];
#pragma unroll
      for (int k = 0; k < 2; ++k)
        part[k] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) S4*)(lds + (place ^ (dt << 6) ^ (k << 4)) + (base + 8 * k) * kRowBytes));
      __builtin_memcpy(&f, part, sizeof(f));
    } else {
      const int c = dt * 32 + (place & 31), half = place >> 5;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        f[j] = *reinterpret_cast<const T*>(lds + at(base + row_of(j, half), c / kEach) + (c % kEach) * sizeof(T));
    }
    return f;
  }
};

// Brings rows of a matrix into a tile, without a register: a wave's load fills
// 1024 bytes, and each lane picks the chunk that belongs there. Rows behind
// `last` repeat it (they are masked where they would count, and hold nothing
// that their sequence does not). Columns behind dim stay as they are: cleared
// once. A row is `stride` values wide, at most 2^22, so that places in a tile
// fit 32 bits. All but one register of the addresses are scalar; worked out
// load by load they were a third of the forward pass's vector instructions.
template <typename T, int ROWS, int DP, int THREADS, bool VEC>
struct Loader {
  typedef Tile<T, ROWS, DP, THREADS, VEC> Of;
  static constexpr int kLoads = Of::kBytes / (THREADS * 16);
  static constexpr int kRound = THREADS * 16 / Of::kRowBytes;  // rows of the workgroup's loads number n
  static constexpr bool kSame = kRound % 16 == 0;              // they have the same chunks for all n

  const char* base;
  uint32_t step;      // bytes of a row
  int wave, dim;
  uint32_t at;        // the lane's place in load 0
  bool ok;            // its chunk has columns

  __device__ __forceinline__ Loader(const T* first_row, long stride, int dim_)
      : base(reinterpret_cast<const char*>(first_row)), step(static_cast<uint32_t>(stride) * sizeof(T)),
        wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), dim(dim_) {
    const uint32_t off = threadIdx.x * 16;
    const int row = off / Of::kRowBytes, chunk = ((off % Of::kRowBytes) >> 4) ^ Of::swizzle(row);
    at = row * step + chunk * 16;
    ok = chunk * Of::kEach < dim;
  }

  __device__ __forceinline__ void load(char* lds, int first, int last) const {
    const char* from = base + static_cast<uint64_t>(step) * static_cast<uint32_t>(first);
    if constexpr (VEC) {
      if (kSame && last - first >= ROWS - 1) {
        if (ok)
#pragma unroll
          for (int n = 0; n < kLoads; ++n)
            load_to_lds<16>(from + static_cast<uint64_t>(step) * (n * kRound) + at, lds + n * THREADS * 16 + wave * 1024);
      } else {
        const uint32_t most = min(last - first, ROWS - 1) * step;
        uint32_t off = threadIdx.x * 16;
        asm volatile("" : "+v"(off));  // worked out here: kept over the loop, it would cost the loop registers
#pragma unroll
        for (int n = 0; n < kLoads; ++n) {
          const int r = off / Of::kRowBytes + n * kRound, c = ((off % Of::kRowBytes) >> 4) ^ Of::swizzle(r);
          if (c * Of::kEach < dim)
            load_to_lds<16>(from + min(r * step, most) + c * 16, lds + n * THREADS * 16 + wave * 1024);
        }
      }
    } else {
      // rows that do not start on 16 bytes: through registers, unaligned
      const uint32_t most = min(last - first, ROWS - 1) * step;
#pragma unroll 4
      for (uint32_t off = threadIdx.x * 16; off < Of::kBytes; off += THREADS * 16) {
        const int r = off / Of::kRowBytes, c = (off % Of::kRowBytes >> 4) * Of::kEach;
        const T* values = reinterpret_cast<const T*>(from + min(r * step, most)) + c;
        T got[Of::kEach];
        if (c + Of::kEach <= dim) __builtin_memcpy(got, values, 16);
        else
#pragma unroll
          for (int u = 0; u < Of::kEach; ++u) got[u] = c + u < dim ? values[u] : static_cast<T>(0.f);
        __builtin_memcpy(__builtin_assume_aligned(lds + Of::at(r, c / Of::kEach), 16), got, 16);
      }
    }
  }
};

// all of a wave's loads into LDS have landed, and everybody's
__device__ __forceinline__ void loads_done() {
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  __syncthreads();
}

// LDS that the lanes of one wave exchange: what stands in front is done before
// what follows. The hardware keeps a wave's LDS accesses in order; this tells the
// compiler, at no instruction.
__device__ __forceinline__ void wave_exchange() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The order of a stretch of matrix products and the LDS reads that feed them:
// AHEAD reads first, then a product and EACH reads in turn. Left to itself the
// compiler reads one fragment at a time and waits for it, four times as long as
// the product takes.
template <int AHEAD, int PRODUCTS, int EACH>
__device__ __forceinline__ void feed() {
  __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
  for (int i = 0; i < PRODUCTS; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, EACH, 0);
  }
}

// A place as something that the compiler cannot work out ahead: the fragments'
// addresses are then made where they are used, one instruction each, in place of
// a register each over the whole loop.
template <bool HIDE>
__device__ __forceinline__ int here(int place) {
  if (HIDE) asm volatile("" : "+v"(place));
  return place;
}

// fragment of a row in memory, columns of step `step`; 0 behind dim
template <bool VEC, typename T>
__device__ __forceinline__ Frag<T> load_row(const T* row, int step, int half, int dim) {
  Frag<T> f;
  const int c = step * 16 + half * 8;
  if (c + 8 <= dim) {
    __builtin_memcpy(&f, row + c, sizeof(f));
  } else {
    // whole 16 bytes of halves; of f32, four of eight
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (!VEC || (sizeof(T) == 4 && i < 4)) && c + i < dim ? row[c + i] : static_cast<T>(0.f);
  }
  return f;
}

// accumulators [columns of the row on 32 * tiles][one row a lane] times f into
// memory: 16 bytes a lane. The halves hold quads of columns; a swap gives each
// eight in a row. What the rounding took goes to `rest` unless that is null.
template <bool VEC, typename T, int TILES>
__device__ __forceinline__ void store_row(T* row, Acc (&acc)[TILES], float f, int half, int dim, bool inside,
                                          T* rest = nullptr) {
#pragma unroll
  for (int dt = 0; dt < TILES; ++dt)
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // lower half keeps its first quad and takes the upper's, the upper
        // half keeps its second and takes the lower's
        const float a = acc[dt][s * 8 + i] * f, b = acc[dt][s * 8 + 4 + i] * f;
        const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
        x[i] = __uint_as_float(both[0]);
        x[4 + i] = __uint_as_float(both[1]);
      }
      const int c = dt * 32 + s * 16 + half * 8;
      if (!inside) continue;
      const Frag<T> t = rounded<T>(x), less = rest_of<T>(x, t);
      if (c + 8 <= dim) {
        __builtin_memcpy(row + c, &t, sizeof(t));
        if (rest) __builtin_memcpy(rest + c, &less, sizeof(less));
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c + i < dim) {
            row[c + i] = t[i];
            if (rest) rest[c + i] = less[i];
          }
      }
    }
}

__device__ __forceinline__ float swap_halves(float x) {
  const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return (threadIdx.x & 32) ? __uint_as_float(both[0]) : __uint_as_float(both[1]);
}

// ---------------------------------------------------------------------------
// Which rows a workgroup has.
//
// Workgroups go to the eight XCDs in turn, and each XCD has an L2 of its own. So
// the heads are dealt out in runs, gcd(heads, 8) of them, and a run's tiles to
// the XCDs that share it: what an XCD reads of k and v are few heads, and those
// of a group together.
//
// The sequences' tiles of `size` rows are numbered through, and so are those
// of the rows behind the last sequence (`seq` == seqs then). Bounds that are
// not ordered or leave [0, rows] are cut to it, so that no access leaves the
// tensors. Every wave searches by itself: up to kLanes sequences with a lane to
// each, more in a table of the call's.
// ---------------------------------------------------------------------------

struct Unit {
  int head, number;
};

inline __host__ __device__ int runs_of(int heads) { return heads % 8 == 0 ? 8 : heads % 4 == 0 ? 4 : heads % 2 == 0 ? 2 : 1; }

__device__ __forceinline__ Unit unit_of(int block, int heads) {
  const int runs = runs_of(heads), each = heads / runs, share = 8 / runs;
  const int xcd = block % 8, i = block / 8;
  return {xcd % runs * each + i % each, i / each * share + xcd / runs};
}

// workgroups for `tiles` tiles of each head
inline long units(long tiles, int heads) {
  const int share = 8 / runs_of(heads);
  return (tiles + share - 1) / share * share * heads;
}

// A launch has fewer tiles. Sequences that overlap can count more, and a sum of
// the lanes' counts must not leave 32 bits.
constexpr int kMostTiles = 1 << 24;

struct Work {
  int begin, len;  // rows of the sequence
  int seq, tile;   // tile inside it
  bool any;
};

__device__ __forceinline__ int2 bounds_of(const BfAttnArgs& a, int seq) {
  const int begin = min(max(a.cu[seq], 0), a.rows), next = a.cu[min(seq + 1, a.seqs)];
  return make_int2(begin, seq < a.seqs ? min(max(next, begin), a.rows) : a.rows);
}

__device__ __forceinline__ int wave_sum(int x) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
  return x;
}

__device__ __forceinline__ int sum_up_to(int x) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(x, off, 64);
    if ((threadIdx.x & 63) >= off) x += y;
  }
  return x;
}

// The table of more than kLanes sequences: tiles in front of each, and of all.
// Every workgroup would read all bounds otherwise, so that the time grew with the
// square of their number: 3000 sequences of 0 to 3 tokens (12 heads of 64, bf16,
// forward and backward) took 1643 us that way and take 658 with the table, 80 of 64
// tokens 79 and 82.
constexpr int kLanes = 64;

// x + y; sums of tiles stay at kMostTiles once they reach it
__device__ __forceinline__ int add_tiles(int x, int y) { return min(x + y, kMostTiles); }

__device__ __forceinline__ int tiles_of(const BfAttnArgs& a, int seq, int size) {
  const int2 b = bounds_of(a, seq);
  return min((b.y - b.x + size - 1) / size, kMostTiles);
}

// table[i] for i in 0 .. seqs, by one workgroup of 16 waves
__device__ __forceinline__ void make_table(const BfAttnArgs& a, int* table, int size) {
  __shared__ int sums[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int before = 0;
  if (threadIdx.x == 0) table[0] = 0;
  for (int first = 0; first < a.seqs; first += 1024) {
    const int seq = first + threadIdx.x;
    int upto = seq < a.seqs ? tiles_of(a, seq, size) : 0;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int y = __shfl_up(upto, off, 64);
      if (lane >= off) upto = add_tiles(upto, y);
    }
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    int all = before;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (i == wave) upto = add_tiles(upto, all);
      all = add_tiles(all, sums[i]);
    }
    if (seq < a.seqs) table[seq + 1] = upto;
    before = all;
    __syncthreads();  // sums are free
  }
}

// Tile `number`. Causal tiles cost the more the later they are, and an expensive
// one that starts last keeps the card waiting: up to kLanes sequences' tiles are
// numbered by their cost, the most expensive first, as their number from the
// sequence's start (dk and dv: from its end). Other tiles, which cost as their
// sequence is long, are numbered in order; sorted they took as long.
__device__ __forceinline__ Work find_tile(const BfAttnArgs& a, int number, int size, bool causal) {
  const int lane = threadIdx.x & 63;
  Work w{};
  int mine = 0, upto = 0, all;
  if (a.seqs > kLanes) {
    all = a.table[a.seqs];
  } else {
    mine = lane < a.seqs ? tiles_of(a, lane, size) : 0;
    upto = sum_up_to(mine);
    all = __builtin_amdgcn_readlane(upto, 63);
  }
  if (number >= all) {  // behind the last sequence
    const int2 rest = bounds_of(a, a.seqs);
    w.seq = a.seqs;
    w.tile = number - all;
    if (w.tile * size >= rest.y - rest.x) return w;
  } else if (a.seqs > kLanes) {
    // the last sequence with no more than `number` tiles in front: table[first]
    // <= number < table[first + count]
    int first = 0, count = a.seqs;
    while (count > 1) {
      const int chunk = (count + 63) / 64, at = lane * chunk;
      const int pick = __popcll(__ballot(at < count && a.table[first + min(at, count)] <= number)) - 1;
      first += pick * chunk;
      count = min(chunk, count - pick * chunk);
    }
    w.seq = first;
    w.tile = number - a.table[first];
  } else if (causal) {
    int low = 0, high = a.rows / size + 1;  // more tiles than `number` cost `low` or more, and not `high`
    while (high - low > 1) {
      const int mid = (low + high) / 2;
      if (wave_sum(max(mine - mid, 0)) > number) low = mid;
      else high = mid;
    }
    number -= wave_sum(max(mine - low - 1, 0));
    w.seq = __ffsll(__ballot(sum_up_to(mine > low ? 1 : 0) > number)) - 1;
    w.tile = low;
  } else {
    w.seq = __ffsll(__ballot(upto > number)) - 1;
    w.tile = number - __builtin_amdgcn_readlane(upto - mine, w.seq);
  }
  w.seq = __builtin_amdgcn_readfirstlane(w.seq);
  w.tile = __builtin_amdgcn_readfirstlane(w.tile);
  const int2 b = bounds_of(a, w.seq);
  w.begin = b.x;
  w.len = b.y - b.x;
  w.any = true;
  return w;
}

// tiles of `size` rows that any bounds can have, the rows behind included
inline long most_tiles(const BfAttnArgs& a, int size) { return a.rows / size + static_cast<long>(a.seqs) + 1; }

}  // namespace bf_attn
