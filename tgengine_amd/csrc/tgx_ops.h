// Element types and wide accesses shared by the model-side operators
// (tgx_embed.hip, tgx_norm.hip, tgx_attention.hip, tgx_clip.hip, tgx_scan.hip,
// tgx_resnorm.hip, tgx_adamw.hip).
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

// The smaller of sigmoid(g) and 1 - sigmoid(g), sigmoid(g) itself where g < 0, and the larger one
// as a reciprocal.  u = 2^-24.  The power's argument is off by 1.3 u |g| (its constant and a
// product), the power and the reciprocal by 2 u each, their sum and product by u: small is off by
// (1.3 |g| + 6) u relatively, the larger by 5 u, and 1 - small by 7 u.  Where |g| is above 87.3 the
// power's instruction, and small with it, is 0.  A step of Newton's at the reciprocal takes the root
// mean square of small's errors from 0.98 u to 0.94 u, for |g| about 2, and the scan of 600 rows of
// 512 tokens and 100 bf16 channels from 67 us to 72.
__device__ __forceinline__ float sigmoid_small(float g, float& larger) {
  const float e = __builtin_amdgcn_exp2f(-1.44269504f * __builtin_fabsf(g));
  larger = __builtin_amdgcn_rcpf(1.f + e);
  return e * larger;
}
// a = sigmoid(g) and 1 - a: neither is a difference
__device__ __forceinline__ void sigmoids(float g, float& a, float& rest) {
  float r;
  const float small = sigmoid_small(g, r);
  a = g < 0.f ? small : r;  // NaN: r, which is NaN
  rest = g < 0.f ? r : small;
}

template <int L>
__device__ __forceinline__ float group_sum(float x) {  // over groups of L <= 64 neighbouring lanes
#pragma unroll
  for (int off = L / 2; off > 0; off >>= 1) x += __shfl_xor(x, off, kWave);
  return x;
}

// thread t of `step` writes its share of an array's zeros: 16 bytes at a time, the bytes
// before and after the 16-byte steps one by one
__device__ __forceinline__ void zero_bytes(uint8_t* __restrict__ p, int head, int64_t n16, int tail, int64_t t,
                                           int64_t step) {
  uint4* body = reinterpret_cast<uint4*>(p + head);
  for (int64_t i = t; i < n16; i += step) body[i] = make_uint4(0, 0, 0, 0);
  if (t < head) p[t] = 0;
  if (t < tail) p[head + n16 * 16 + t] = 0;
}

struct ZeroSpan {
  uint8_t* p;
  size_t bytes;
  int head, tail;
  int64_t n16;
  ZeroSpan(void* to, size_t n) : p(static_cast<uint8_t*>(to)), bytes(n) {
    head = static_cast<int>(std::min(bytes, static_cast<size_t>(-addr(p) & 15)));
    n16 = static_cast<int64_t>((bytes - head) / 16);
    tail = static_cast<int>((bytes - head) % 16);
  }
};

__global__ __launch_bounds__(256) void zero_kernel(uint8_t* __restrict__ p, int head, int64_t n16, int tail) {
  zero_bytes(p, head, n16, tail, static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x,
             static_cast<int64_t>(gridDim.x) * 256);
}

// a kernel, not a memset: callers may capture the call in a graph
inline int fill_zero(void* p, size_t bytes, hipStream_t s) {
  if (bytes == 0) return TGX_OK;
  const ZeroSpan z(p, bytes);
  const int64_t blocks = std::clamp<int64_t>(ops_cdiv(z.n16, 256), 1, 8192);
  hipLaunchKernelGGL(zero_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, s, z.p, z.head, z.n16, z.tail);
  return check_launch("zero_kernel");
}

// a grid's threads are counted in 32 bits
inline int check_grid(const char* what, int64_t blocks, int64_t threads) {
  if (blocks > ((int64_t(1) << 32) - 1) / threads)
    return fail(TGX_ERR_LIMIT, "%s: %lld workgroups of %lld threads: more than one launch takes", what,
                static_cast<long long>(blocks), static_cast<long long>(threads));
  return TGX_OK;
}

// calls f(T{}) for the dtype
template <typename F>
int by_type(int dtype, F&& f) {
  return dtype == TGX_F32 ? f(float{}) : f(bf16{});
}

}  // namespace
}  // namespace tgx
