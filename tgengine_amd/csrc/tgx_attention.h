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
  void *o, *rest, *dq, *dk, *dv;  // rest: what rounding took from o (bf16), or nullptr
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
// Parts of key ranges: per row and range, its maximum and sum in ml, its outputs in o.
// att_join_forward joins them into a.o and a.lse, att_join_sums adds up the ranges' o.
struct AttParts {
  float2* ml;
  float* o;
  AttParts(void* ws, int64_t rows, int splits)
      : ml(static_cast<float2*>(ws)), o(reinterpret_cast<float*>(ml + (rows * splits + 1) / 2 * 2)) {}
  static size_t bytes(int64_t rows, int splits, int dim) {
    return splits > 1 ? static_cast<size_t>((rows * splits + 1) / 2 * 2) * 8 + static_cast<size_t>(rows) * splits * dim * 4
                      : 0;
  }
};
int att_join_forward(const AttArgs& a, int dtype, int splits, const AttParts& part, hipStream_t s);
int att_join_sums(void* out, int64_t rows, int dim, int dtype, float by, int splits, const float* part, hipStream_t s);
size_t att_mma_forward_workspace(const AttArgs& a, int dtype);
int att_mma_forward(const AttArgs& a, int dtype, void* ws, hipStream_t s);
size_t att_mma_backward_workspace(const AttArgs& a, int dtype);
int att_mma_backward(const AttArgs& a, int dtype, void* ws, hipStream_t s);

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));

// The matrix instructions: bf16 takes the 32 x 32 tile, whose operands cost half the LDS
// reads of the 16 x 16 one; f32, eight times slower for the same bytes, the 16 x 16 one,
// which pads sequences of 1 + 32 or 1 + 64 tokens less.
//   kTile  : rows and columns of a tile
//   kRegs  : a lane's values of a product
//   kFrags : fragments that the kTile rows of a product make as the next one's operand
template <typename T>
constexpr int kTile = sizeof(T) == 2 ? 32 : 16;
template <typename T>
constexpr int kRegs = kTile<T> * kTile<T> / kWave;
template <typename T>
constexpr int kFrags = kRegs<T> / kWide<T>;
template <typename T>
using Acc = std::conditional_t<sizeof(T) == 2, f32x16, f32x4>;

// A fragment is 16 bytes a lane of a kTile-row operand: lane l holds row l % kTile, and
// its group l / kTile the values [group V, group V + V) of a step of 16 along the summed
// axis.  For f32 that is four instructions, each with one value of every group (they
// stand in for four neighbours: the order of a sum's terms is free as long as both
// operands agree on it).
constexpr int kStep = 16;

template <typename T>
__device__ __forceinline__ int lane_row() { return threadIdx.x & (kTile<T> - 1); }
template <typename T>
__device__ __forceinline__ int lane_group() { return (threadIdx.x & (kWave - 1)) / kTile<T>; }

template <typename T>
__device__ __forceinline__ Acc<T> mma(Acc<T> c, u32x4 a, u32x4 b) {
  if constexpr (sizeof(T) == 2) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[e]), __uint_as_float(b[e]), c, 0, 0, 0);
    return c;
  }
}

// Value i of a lane of a product belongs to column lane_row and to this row
template <typename T>
__device__ __forceinline__ constexpr int mma_row(int i, int group) {
  return sizeof(T) == 2 ? 8 * (i / 4) + 4 * group + i % 4 : 4 * group + i;
}

// What rounding to T takes from x; nothing from an infinity, nor from a value that becomes one
template <typename T>
__device__ __forceinline__ float lost(float x) {
  const float y = to_f(from_f<T>(x));
  return fabsf(y) == INFINITY ? 0.f : x - y;
}

// What cutting x to bf16 leaves, with x's sign and never 0 unless x is, nor NaN for an infinity:
// an infinite factor, or an infinite x, then gives the same infinity with both parts.  (The
// median of numbers one of which is NaN is the least of the others.)
template <bool SIGNED>
__device__ __forceinline__ float left(float x) {
  const float cut = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
  if constexpr (!SIGNED) return __builtin_amdgcn_fmed3f(x - cut, 0x1p-126f, x);
  return copysignf(__builtin_amdgcn_fmed3f(fabsf(x) - fabsf(cut), 0x1p-126f, fabsf(x)), x);
}

// Fragment f (of kFrags) of such values as the second operand of a product that sums
// over their rows: no lane gives a value to another.  bf16 comes in two parts, for a product
// each: the values cut to bf16, and what that left (rest_frag), which is below 2^-7 of a value,
// so that its own rounding takes at most 2^-16 of it.
template <typename T>
__device__ __forceinline__ u32x4 to_frag(const Acc<T>& x, int f) {
  u32x4 y;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    if constexpr (sizeof(T) == 2)  // the upper halves of two values
      y[u] = __builtin_amdgcn_perm(__float_as_uint(x[f * 8 + 2 * u + 1]), __float_as_uint(x[f * 8 + 2 * u]), 0x07060302);
    else
      y[u] = __float_as_uint(x[u]);
  }
  return y;
}
template <bool SIGNED>  // whether values below 0 are among them
__device__ __forceinline__ u32x4 rest_frag(const f32x16& x, int f) {
  u32x4 y;
#pragma unroll
  for (int u = 0; u < 4; ++u)
    y[u] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{left<SIGNED>(x[f * 8 + 2 * u]),
                                                                       left<SIGNED>(x[f * 8 + 2 * u + 1])}), bf16x2));
  return y;
}

// An LDS tile of rows of DP values, longer by what keeps its reads off each other's banks
// (64 of 4 bytes).  A fragment reads 16 bytes of each of 16 rows at a time: rows an odd
// multiple of 16 bytes apart are free of conflicts.  The transposed reads of bf16 take 64
// bytes of each of 4 rows at a time: rows 64 bytes apart (mod 256).  A tile read both ways
// takes rows 80 bytes apart, or 176: fragments are free, a transposed read meets one
// conflict.  (Chunks that trade places by row would meet none, but their addresses cost the
// backward pass more registers and instructions than the conflicts: 633 us for dk and dv of
// 1,000 x 8,000 tokens against 470 with rows of 16 bytes more.)  f32 rows 16 bytes longer
// serve both.
enum class Reads { kRows, kColumns, kBoth };

template <typename T, int DP, Reads HOW>
struct LdsTile {
  static constexpr int next(int bytes, int x, int y) {  // the next length that is x or y mod 256
    while (bytes % 256 != x && bytes % 256 != y) bytes += 16;
    return bytes;
  }
  static constexpr int ROW =  // values
      sizeof(T) == 4            ? DP + 4
      : HOW == Reads::kRows     ? DP + (DP / 8 % 2 == 0 ? 8 : 0)
      : HOW == Reads::kColumns  ? next(DP * 2, 64, 192) / 2
                                : next(DP * 2, 80, 176) / 2;
  // fragment e of rows row0 .. (a multiple of kTile): a lane's 16 bytes
  __device__ static __forceinline__ u32x4 frag(const T* tile, int row0, int e) {
    return *reinterpret_cast<const u32x4*>(tile + (row0 + lane_row<T>()) * ROW + e * kStep +
                                           lane_group<T>() * kWide<T>);
  }
  // The first operand that goes with to_frag's: kTile columns from kTile t on of rows
  // row0 .., transposed, in the rows' order of to_frag.  In bf16 by the transposing LDS
  // read: 16 lanes read 4 rows of 16 values and each lane gets a column of 4.
  __device__ static __forceinline__ u32x4 transposed(const T* tile, int row0, int f, int t) {
    const int lane = threadIdx.x & (kWave - 1), group = lane_group<T>();
    if constexpr (sizeof(T) == 2) {
      typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
      const int i = lane & 15;
      const T* p = tile + (row0 + 16 * f + 4 * group + i / 4) * ROW + t * 32 + (lane & 16) + (i & 3) * 4;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 8 * ROW));
      return __builtin_bit_cast(u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      u32x4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = __float_as_uint(tile[(row0 + 4 * group + e) * ROW + t * 16 + lane_row<T>()]);
      return x;
    }
  }
};

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

// The workgroup's waves, MINW of them (or more, if not FIXED), move ROWS rows of up to DP
// values into an LDS tile: load() issues the reads, store() waits for them and writes.  A thread keeps
// one column of all its rows, so that a row costs it one address step; lanes past the last
// column stay idle.
template <typename T, bool TINY, int ROWS, int DP, int MINW, bool FIXED>
struct Stage {
  static constexpr int V = kWide<T>, LANES = pow2_at_least(DP / V), N = (ROWS * LANES + 64 * MINW - 1) / (64 * MINW);
  u32x4 x[N];
  int col, row0, steps;
  bool in;
  __device__ explicit Stage(int dim)
      : col(threadIdx.x % LANES * V), row0(threadIdx.x / LANES), steps(blockDim.x / LANES), in(col < dim) {}
  __device__ __forceinline__ int step() const { return FIXED ? 64 * MINW / LANES : steps; }
  __device__ __forceinline__ int row(int n) const { return row0 + n * step(); }
  __device__ __forceinline__ bool whole(int n) const {  // row n of every thread is a row of the tile
    return FIXED && (n + 1) * (64 * MINW / LANES) <= ROWS;
  }
  // rows base, base + stride, ...: those whose bit is set, zeros for the others
  __device__ __forceinline__ void load(const T* base, int64_t stride, uint64_t bits, int dim) {
    const T* p = base + row0 * stride;
    const int64_t by = step() * stride;
    const uint64_t mine = in && row0 < ROWS ? bits >> row0 : 0;
#pragma unroll
    for (int n = 0; n < N; ++n, p += by) {
      x[n] = u32x4{0, 0, 0, 0};
      if ((whole(n) || row(n) < ROWS) && (mine >> (n * step()) & 1)) x[n] = row_part<T, TINY>(p, col, dim);
    }
  }
  // the rows that p(n) gives the addresses of, nullptr for zeros
  template <typename At>
  __device__ __forceinline__ void load(int dim, At&& p) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      x[n] = u32x4{0, 0, 0, 0};
      const T* at = p(n);
      if (in && at != nullptr) x[n] = row_part<T, TINY>(at, col, dim);
    }
  }
  template <int ROW>  // values from row to row of the tile
  __device__ __forceinline__ void store(T* tile, int dim) const {
    if (LANES * V > DP && col >= DP) return;
    const bool asis = TINY || dim % V == 0;
#pragma unroll
    for (int n = 0; n < N; ++n)
      if (whole(n) || row(n) < ROWS)
        *reinterpret_cast<u32x4*>(tile + row(n) * ROW + col) = asis ? x[n] : finish<T>(x[n], col, dim);
  }
};

// The fragments of one row a lane (lane_row), from global memory; nullptr gives zeros
template <typename T, bool TINY, int DP>
__device__ __forceinline__ void row_frags(u32x4 (&x)[DP / kStep], const T* row, int dim) {
  const int at = lane_group<T>() * kWide<T>;
#pragma unroll
  for (int s = 0; s < DP / kStep; ++s) {
    x[s] = u32x4{0, 0, 0, 0};
    if (row != nullptr && s * kStep + at < dim) x[s] = row_part<T, TINY>(row, s * kStep + at, dim);
  }
  if (!TINY && dim % kWide<T> != 0)
#pragma unroll
    for (int s = 0; s < DP / kStep; ++s) x[s] = finish<T>(x[s], s * kStep + at, dim);
}

// A product with the head's columns down a lane's registers and one row a lane, to rows
// of `dim` values: 4 neighbours at a time
template <typename T, int DP>
__device__ __forceinline__ void store_columns(T* row, const Acc<T> (&x)[DP / kTile<T>], float by, int dim) {
#pragma unroll
  for (int t = 0; t < DP / kTile<T>; ++t)
#pragma unroll
    for (int j = 0; j < kRegs<T> / 4; ++j) {
      const int d = t * kTile<T> + mma_row<T>(4 * j, lane_group<T>());
      Pack<T, 4> y;
#pragma unroll
      for (int u = 0; u < 4; ++u) y.v[u] = from_f<T>(x[t][4 * j + u] * by);
      if (d + 4 <= dim) {
        store_pack<T, 4>(row + d, y);
      } else {
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (d + u < dim) row[d + u] = y.v[u];
      }
    }
}

// the same in 32 bits, for the parts of ranges
template <typename T, int DP>
__device__ __forceinline__ void store_parts(float* row, const Acc<T> (&x)[DP / kTile<T>], int dim) {
#pragma unroll
  for (int t = 0; t < DP / kTile<T>; ++t)
#pragma unroll
    for (int j = 0; j < kRegs<T> / 4; ++j) {
      const int d = t * kTile<T> + mma_row<T>(4 * j, lane_group<T>());
      Pack<float, 4> y;
#pragma unroll
      for (int u = 0; u < 4; ++u) y.v[u] = x[t][4 * j + u];
      if (d + 4 <= dim) {
        store_pack<float, 4>(row + d, y);
      } else {
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (d + u < dim) row[d + u] = y.v[u];
      }
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

// Waves of a workgroup for n tiles of rows (or keys): as few workgroups as `most` waves
// each allow, and then as few waves, but `least`
inline int waves_for(int64_t n, int least, int most) {
  const int64_t groups = std::max<int64_t>(ops_cdiv(n, most), 1);
  return static_cast<int>(std::max<int64_t>(ops_cdiv(n, groups), least));
}

constexpr int kNoLoads = 0x0f70;  // s_waitcnt: no vector load outstanding

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// A row's log sum from its maximum, in units of log 2, and its sum.  -inf stands for a row
// without keys (a sum of 0) alone: a score of NaN or +inf makes the sum NaN, and the log sum
// has to say so, or the gradient would take the row for one without keys.
__device__ __forceinline__ float log_sum(float m, float l) { return l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2; }

// Calls f(T{}, DP, TINY) with the head size padded to one of six or seven widths, each a set of
// kernels.  f32, bound by its matrix units, has two more between the widths of bf16: with 112
// and 176 the forward pass, dk and dv and dq of 400 x (65 x 65), 2 heads, take 55, 109 and 31 us
// for 100 values and 94, 199 and 52 for 172; padded to 128 and 256 they take 73, 118 and 33, and
// 121, 254 and 67.  Heads of 177 to 192 values, which pad to 256, would win as much by one more.
template <typename F>
int by_head(int dtype, int dim, F&& f) {
#define TGX_HEAD(DP) f(t, std::integral_constant<int, DP>{}, std::false_type{})
  return by_type(dtype, [&](auto t) {
    constexpr bool F32 = sizeof(t) == 4;
    if (dim < kWide<decltype(t)>) return f(t, std::integral_constant<int, 32>{}, std::true_type{});
    if (dim <= 32) return TGX_HEAD(32);
    if (dim <= 64) return TGX_HEAD(64);
    if (dim <= 96) return TGX_HEAD(96);
    if constexpr (F32)
      if (dim <= 112) return TGX_HEAD(112);
    if (dim <= 128) return TGX_HEAD(128);
    if constexpr (F32)
      if (dim <= 176) return TGX_HEAD(176);
    if constexpr (!F32)
      if (dim <= 192) return TGX_HEAD(192);
    return TGX_HEAD(256);
  });
#undef TGX_HEAD
}

}  // namespace
}  // namespace tgx
