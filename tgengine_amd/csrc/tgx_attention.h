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
  Pack<T, kWide<T>> p;
#pragma unroll
  for (int u = 0; u < kWide<T>; ++u) p.v[u] = from_f<T>(x[f * kWide<T> + u]);
  return __builtin_bit_cast(u32x4, p);
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
// values where fewer than V are left (finish() moves them), one by one where the row has
// fewer than V
template <typename T>
__device__ __forceinline__ u32x4 row_part(const T* row, int c, int dim) {
  constexpr int V = kWide<T>;
  u32x4 x = {0, 0, 0, 0};
  if (dim >= V) {
    x = load16(row + min(c, dim - V));
  } else {
    Pack<T, V> p = __builtin_bit_cast(Pack<T, V>, x);
    for (int u = 0; u < V; ++u)
      if (c + u < dim) p.v[u] = row[c + u];
    x = __builtin_bit_cast(u32x4, p);
  }
  return x;
}

// row_part's values in their places, zeros after the row's end
template <typename T>
__device__ __forceinline__ u32x4 finish(u32x4 x, int c, int dim) {
  constexpr int V = kWide<T>;
  const int over = c + V - dim;
  if (over <= 0 || dim < V) return x;
  if (over >= V) return u32x4{0, 0, 0, 0};
  const unsigned __int128 w = __builtin_bit_cast(unsigned __int128, x) >> (over * 8 * static_cast<int>(sizeof(T)));
  return __builtin_bit_cast(u32x4, w);
}

// NT threads move ROWS rows of up to DP values into an LDS tile of rows STRIDE apart:
// load() issues the reads, store() waits for them and writes.  at(row) gives a row's
// address, or nullptr for zeros.
template <typename T, int ROWS, int DP, int NT, int STRIDE>
struct Stage {
  static constexpr int V = kWide<T>, PER = DP / V, N = (ROWS * PER + NT - 1) / NT;
  u32x4 x[N];
  template <typename At>
  __device__ __forceinline__ void load(int dim, At&& at) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int e = threadIdx.x + n * NT, row = e / PER, c = e % PER * V;
      x[n] = u32x4{0, 0, 0, 0};
      if (ROWS * PER % NT != 0 && e >= ROWS * PER) continue;
      const T* p = at(row);
      if (p != nullptr && c < dim) x[n] = row_part(p, c, dim);
    }
  }
  __device__ __forceinline__ void store(T* tile, int dim) const {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int e = threadIdx.x + n * NT, row = e / PER, c = e % PER * V;
      if (ROWS * PER % NT != 0 && e >= ROWS * PER) continue;
      *reinterpret_cast<u32x4*>(tile + row * STRIDE + c) = finish<T>(x[n], c, dim);
    }
  }
};

// The fragments of one row a lane (row l % 32), from global memory; nullptr gives zeros
template <typename T, int DP>
__device__ __forceinline__ void row_frags(u32x4 (&x)[DP / kStep<T>], const T* row, int dim) {
  const int h = (threadIdx.x & (kWave - 1)) / 32;
#pragma unroll
  for (int s = 0; s < DP / kStep<T>; ++s) {
    const int c = s * kStep<T> + h * kWide<T>;
    x[s] = u32x4{0, 0, 0, 0};
    if (row != nullptr && c < dim) x[s] = finish<T>(row_part(row, c, dim), c, dim);
  }
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

// Calls f(T{}, DP) with the head size padded to whole 32-column tiles
template <typename F>
int by_head(int dtype, int dim, F&& f) {
  return by_type(dtype, [&](auto t) {
    if (dim <= 32) return f(t, std::integral_constant<int, 32>{});
    if (dim <= 64) return f(t, std::integral_constant<int, 64>{});
    if (dim <= 96) return f(t, std::integral_constant<int, 96>{});
    if (dim <= 128) return f(t, std::integral_constant<int, 128>{});
    if (dim <= 192) return f(t, std::integral_constant<int, 192>{});
    return f(t, std::integral_constant<int, 256>{});
  });
}

}  // namespace
}  // namespace tgx
