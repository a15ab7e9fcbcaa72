// Element types and wide accesses shared by the model-side operators
// (tgx_embed.hip, tgx_norm.hip, tgx_attention.hip, tgx_clip.hip).
#pragma once

#include "tgx_internal.h"

#include <algorithm>
#include <type_traits>

namespace tgx {
namespace {

using bf16 = __bf16;

// V consecutive values, moved as one access of V * sizeof(T) <= 16 bytes.  gfx950
// takes global accesses at any address, so that a row of odd length, or one that
// starts between two 16-byte steps, still moves 16 bytes a lane: its last pack
// starts V values before its end and overlaps the one before.
template <typename T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) Pack {
  T v[V];
};
// values that one lane moves at once
template <typename T>
constexpr int kWide = 16 / sizeof(T);

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(bf16 x) { return static_cast<float>(x); }
// round to nearest even; NaN stays NaN
template <typename T>
__device__ __forceinline__ T from_f(float x) {
  return static_cast<T>(x);
}

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
  return *reinterpret_cast<const Pack<T, V>*>(p);
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& x) {
  *reinterpret_cast<Pack<T, V>*>(p) = x;
}

inline int64_t ops_cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline size_t ops_align(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

inline uint64_t addr(const void* p) { return reinterpret_cast<uint64_t>(p); }
inline int elem_bytes(int dtype) { return feat_elem_bytes(dtype); }

template <int L>
__device__ __forceinline__ float group_sum(float x) {  // over groups of L <= 64 neighbouring lanes
#pragma unroll
  for (int off = L / 2; off > 0; off >>= 1) x += __shfl_xor(x, off, kWave);
  return x;
}

// calls f(T{}) for the dtype
template <typename F>
int by_type(int dtype, F&& f) {
  return dtype == TGX_F32 ? f(float{}) : f(bf16{});
}

}  // namespace
}  // namespace tgx
