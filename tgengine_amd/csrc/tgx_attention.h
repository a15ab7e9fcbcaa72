// Shared by the attention kernels (tgx_attention.hip, tgx_att_fwd.hip, tgx_att_bwd.hip):
// arguments, matrix instructions, tiles and the walk over the keys that a mask keeps.
//
// The query heads of one key/value head and the tokens of one batch row meet the same
// keys under the same mask, so a "problem" is (batch row, key/value head) and its rows
// are r = token * group + head of the group.
#pragma once

#include "tgx_ops.h"

namespace tgx {

struct AttArgs {
  const void *q, *k, *v, *out, *dout;
  const uint8_t* mask;
  void *o, *dq, *dk, *dv;
  float* lse;
  int64_t batch, lq, lk, mask_stride;
  int64_t qs[3], ks[3], vs[3], os[3];  // os: of out, dout and dq
  int32_t heads, kv_heads, group, dim;
  float scale;
};

// Problems of at most kMostRows rows go to tgx_att_rows.hip, the others to
// tgx_att_fwd.hip and tgx_att_bwd.hip
constexpr int kMostRows = 4;
size_t att_rows_forward_workspace(const AttArgs& a);
int att_rows_forward(const AttArgs& a, int dtype, void* ws, hipStream_t s);
size_t att_rows_backward_workspace(const AttArgs& a);
int att_rows_backward(const AttArgs& a, int dtype, void* ws, hipStream_t s);
// joins the key ranges' parts, per row and range: maximum, sum, dim outputs
int att_join_forward(const AttArgs& a, int dtype, int splits, const float* part, hipStream_t s);
size_t att_mma_forward_workspace(const AttArgs& a, int dtype);
int att_mma_forward(const AttArgs& a, int dtype, void* ws, hipStream_t s);
size_t att_mma_backward_workspace(const AttArgs& a, int dtype);
int att_mma_backward(const AttArgs& a, int dtype, void* ws, hipStream_t s);

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));

// A fragment is 16 bytes a lane of a 32-row operand of the 32 x 32 matrix instructions:
// lane l holds row l % 32, and its half h = l / 32 the values [h V, h V + V) of a step
// of kStep = 2 V values along the summed axis.  For f32 that is four instructions of two
// values each (the halves' values stand in for two neighbours: the order of a sum's
// terms is free as long as both operands agree on it).
template <typename T>
constexpr int kStep = 2 * kWide<T>;

template <typename T>
__device__ __forceinline__ f32x16 mma(f32x16 c, u32x4 a, u32x4 b) {
  if constexpr (sizeof(T) == 2) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[e]), __uint_as_float(b[e]), c, 0, 0,
                                               0);
    return c;
  }
}

// A product's 16 values a lane belong to column l % 32 and rows 8 (i / 4) + 4 h + i % 4.
__device__ __forceinline__ constexpr int mma_row(int i, int h) { return 8 * (i / 4) + 4 * h + i % 4; }

// Fragment f (of 16 / V) of such values as the second operand of a product that sums
// over their rows: no lane gives a value to another.
template <typename T>
__device__ __forceinline__ u32x4 to_frag(const f32x16& x, int f) {
  u32x4 y;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    if constexpr (sizeof(T) == 2)  // two values at a time: one conversion
      y[u] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{x[f * 8 + 2 * u], x[f * 8 + 2 * u + 1]}), bf16x2));
    else
      y[u] = __float_as_uint(x[f * 4 + u]);
  }
  return y;
}

// The first operand that goes with it: 32 columns from `col` on of rows of an LDS tile,
// transposed, in the rows' order of to_frag.  In bf16 by the transposing LDS read: a
// group of 16 lanes reads 4 rows of 16 values and each lane gets a column of 4.
template <typename T>
__device__ __forceinline__ u32x4 transposed(const T* tile, int stride, int row0, int f, int col) {
  const int lane = threadIdx.x & (kWave - 1), h = lane / 32;
  if constexpr (sizeof(T) == 2) {
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const int i = lane & 15;
    const T* p = tile + (row0 + 16 * f + 4 * h + i / 4) * stride + col + (lane & 16) + (i & 3) * 4;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 8 * stride));
    return __builtin_bit_cast(u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  } else {
    u32x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      x[e] = __builtin_bit_cast(uint32_t, tile[(row0 + 8 * f + 4 * h + e) * stride + col + (lane & 31)]);
    return x;
  }
}

template <typename T>
__device__ __forceinline__ u32x4 load16(const T* p) {
  return *reinterpret_cast<const u32x4_any*>(p);
}

// V values of a row of `dim` from column c on as they are in memory: the row's last V
// values where fewer than V are left (finish() moves them).  TINY: rows of fewer than V
// values, read one by one.
template <typename T, bool TINY>
__device__ __forceinline__ u32x4 row_part(const T* row, int c, int dim) {
  constexpr int V = kWide<T>;
  if constexpr (TINY) {
    Pack<T, V> p = {};
    for (int u = 0; u < V; ++u)
      if (c + u < dim) p.v[u] = row[c + u];
    return __builtin_bit_cast(u32x4, p);
  } else {
    return load16(row + min(c, dim - V));
  }
}
template <typename T>
__device__ __forceinline__ u32x4 row_part(const T* row, int c, int dim) {
  return dim < kWide<T> ? row_part<T, true>(row, c, dim) : row_part<T, false>(row, c, dim);
}

// row_part's values in their places, zeros after the row's end (rows of at least V values)
template <typename T>
__device__ __forceinline__ u32x4 finish(u32x4 x, int c, int dim) {
  constexpr int V = kWide<T>;
  const int over = c + V - dim;
  if (over <= 0 || over >= V) return x;  // whole, or zeros already
  const unsigned __int128 w = __builtin_bit_cast(unsigned __int128, x) >> (over * 8 * static_cast<int>(sizeof(T)));
  return __builtin_bit_cast(u32x4, w);
}

// both at once
template <typename T>
__device__ __forceinline__ u32x4 row_values(const T* row, int c, int dim) {
  return dim < kWide<T> ? row_part<T, true>(row, c, dim) : finish<T>(row_part<T, false>(row, c, dim), c, dim);
}

constexpr int pow2_at_least(int x) {
  int p = 1;
  while (p < x) p *= 2;
  return p;
}

// NT threads move ROWS rows of up to DP values into an LDS tile of rows STRIDE apart:
// load() issues the reads, store() waits for them and writes.  A thread keeps one column
// of all its rows, so that a row costs it one address step; lanes past the last column
// stay idle.
template <typename T, bool TINY, int ROWS, int DP, int NT, int STRIDE>
struct Stage {
  static constexpr int V = kWide<T>, LANES = pow2_at_least(DP / V), STEP = NT / LANES,
                       N = (ROWS + STEP - 1) / STEP;
  static_assert(N * STEP == ROWS || N == 1, "whole steps");
  u32x4 x[N];
  int col, row0;
  bool in;
  __device__ explicit Stage(int dim) : col(threadIdx.x % LANES * V), row0(threadIdx.x / LANES) {
    in = col < dim && row0 < ROWS;
  }
  // rows base, base + stride, ...: those whose bit is set, zeros for the others
  __device__ __forceinline__ void load(const T* base, int64_t stride, uint64_t bits, int dim) {
    const T* p = base + row0 * stride;
    const uint64_t mine = in ? bits >> row0 : 0;
#pragma unroll
    for (int n = 0; n < N; ++n, p += STEP * stride) {
      x[n] = u32x4{0, 0, 0, 0};
      if (mine >> (n * STEP) & 1) x[n] = row_part<T, TINY>(p, col, dim);
    }
  }
  // the rows that p(n) gives the addresses of, nullptr for zeros
  template <typename At>
  __device__ __forceinline__ void load(int dim, At&& p) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      x[n] = u32x4{0, 0, 0, 0};
      const T* row = p(n);
      if (in && row != nullptr) x[n] = row_part<T, TINY>(row, col, dim);
    }
  }
  __device__ __forceinline__ void store(T* tile, int dim) const {
    if (LANES * V > DP && col >= DP) return;
    if (STEP > ROWS && row0 >= ROWS) return;
    T* p = tile + row0 * STRIDE + col;
    if (TINY || dim % V == 0) {
#pragma unroll
      for (int n = 0; n < N; ++n) *reinterpret_cast<u32x4*>(p + n * STEP * STRIDE) = x[n];
    } else {
#pragma unroll
      for (int n = 0; n < N; ++n) *reinterpret_cast<u32x4*>(p + n * STEP * STRIDE) = finish<T>(x[n], col, dim);
    }
  }
};

// The fragments of one row a lane (row l % 32), from global memory; nullptr gives zeros
template <typename T, bool TINY, int DP>
__device__ __forceinline__ void row_frags(u32x4 (&x)[DP / kStep<T>], const T* row, int dim) {
  const int h = (threadIdx.x & (kWave - 1)) / 32;
#pragma unroll
  for (int s = 0; s < DP / kStep<T>; ++s) {
    const int c = s * kStep<T> + h * kWide<T>;
    x[s] = u32x4{0, 0, 0, 0};
    if (row != nullptr && c < dim) x[s] = row_part<T, TINY>(row, c, dim);
  }
  if (!TINY && dim % kWide<T> != 0)
#pragma unroll
    for (int s = 0; s < DP / kStep<T>; ++s) x[s] = finish<T>(x[s], s * kStep<T> + h * kWide<T>, dim);
}

// bit j: byte j of x is not zero
__device__ __forceinline__ uint32_t nonzero4(uint32_t x) {
  const uint32_t y = ((((x & 0x7f7f7f7fu) + 0x7f7f7f7fu) | x) >> 7) & 0x01010101u;
  return (y | y >> 7 | y >> 14 | y >> 21) & 15u;
}

// Walks over the tiles of KT (32 or 64) keys of [lo, hi) that keep any key; every wave
// walks for itself and all come to the same.  A lane reads the mask of 64 keys at a
// time, so that 4,096 keys are looked through at once and empty ones cost nothing more.
template <int KT>
struct Keys {
  const uint8_t* mask;
  int64_t base, hi;
  uint64_t word = 0, active = 0;
  uint32_t later = 0;  // KT = 32: the upper half of the word at hand
  int64_t later_at = 0;

  __device__ Keys(const uint8_t* mask_, int64_t lo, int64_t hi_) : mask(mask_), base(lo - 64 * kWave), hi(hi_) {}

  __device__ __forceinline__ uint64_t read(int64_t at) const {
    const int64_t left = hi - at;
    if (left <= 0) return 0;
    if (mask == nullptr) return left >= 64 ? ~uint64_t(0) : (uint64_t(1) << left) - 1;
    uint64_t w = 0;
    if (left >= 64) {
      u32x4 x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = load16(mask + at + 16 * j);
#pragma unroll
      for (int j = 0; j < 16; ++j) w |= static_cast<uint64_t>(nonzero4(x[j / 4][j % 4])) << (4 * j);
    } else {
      for (int j = 0; j < static_cast<int>(left); ++j) w |= static_cast<uint64_t>(mask[at + j] != 0) << j;
    }
    return w;
  }

  // the next tile's first key and kept keys; false after the last
  __device__ __forceinline__ bool next(int64_t& key, uint64_t& bits) {
    if (KT == 32 && later != 0) {
      key = later_at;
      bits = later;
      later = 0;
      return true;
    }
    while (active == 0) {
      base += 64 * kWave;
      if (base >= hi) return false;
      word = read(base + static_cast<int64_t>(threadIdx.x & (kWave - 1)) * 64);
      active = __ballot(word != 0);
    }
    const int at = __builtin_ctzll(active);
    active &= active - 1;
    const uint32_t w0 = __builtin_amdgcn_readlane(static_cast<uint32_t>(word), at);
    const uint32_t w1 = __builtin_amdgcn_readlane(static_cast<uint32_t>(word >> 32), at);
    key = base + at * 64;
    if (KT == 64) {
      bits = static_cast<uint64_t>(w1) << 32 | w0;
      return true;
    }
    if (w0 == 0) {
      key += 32;
      bits = w1;
      return true;
    }
    later = w1;
    later_at = key + 32;
    bits = w0;
    return true;
  }
};

// Workgroups go to the eight dies in turn, each with an L2 of its own: those of one
// problem, which read the same keys and values, are put on one die.
__device__ __forceinline__ int64_t by_die(int64_t id, int64_t total) {
  const int64_t q = total / 8, r = total % 8, die = id % 8;
  return die * q + min(die, r) + id / 8;
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// Calls f(T{}, DP, TINY) with the head size padded to whole 32-column tiles
template <typename F>
int by_head(int dtype, int dim, F&& f) {
  return by_type(dtype, [&](auto t) {
    constexpr std::false_type no{};
    if (dim < kWide<decltype(t)>) return f(t, std::integral_constant<int, 32>{}, std::true_type{});
    if (dim <= 32) return f(t, std::integral_constant<int, 32>{}, no);
    if (dim <= 64) return f(t, std::integral_constant<int, 64>{}, no);
    if (dim <= 96) return f(t, std::integral_constant<int, 96>{}, no);
    if (dim <= 128) return f(t, std::integral_constant<int, 128>{}, no);
    if (dim <= 192) return f(t, std::integral_constant<int, 192>{}, no);
    return f(t, std::integral_constant<int, 256>{}, no);
  });
}

}  // namespace
}  // namespace tgx
