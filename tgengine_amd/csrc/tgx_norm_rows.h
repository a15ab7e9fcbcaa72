// Rows that lanes share, as the norms read them (tgx_norm.hip, tgx_resnorm.h).
#pragma once

#include "tgx_ops.h"

namespace tgx {
namespace {

constexpr int kNormThreads = 256;

// the sum over the L lanes of a row; L > 64: the whole workgroup, through `lds` [L / 64]
template <int L>
__device__ __forceinline__ float row_sum(float x, float* lds) {
  if constexpr (L <= kWave) {
    return group_sum<L>(x);
  } else {
    x = group_sum<kWave>(x);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) lds[threadIdx.x / kWave] = x;
    __syncthreads();
    if constexpr (L == 256) {
      return (lds[0] + lds[1]) + (lds[2] + lds[3]);
    } else {
      x = lds[threadIdx.x & (L / kWave - 1)];
      return group_sum<L / kWave>(x);
    }
  }
}

// the lane's C packs of a row of `dim` values: pack j starts at at(j); its values below
// skip(j) belong to the pack before (the last pack of a row overlaps it), and a pack
// past the row has none
template <int V, int L>
struct Place {
  int lane, dim, packs;
  __device__ Place(int dim_) : lane(threadIdx.x & (L - 1)), dim(dim_), packs((dim_ + V - 1) / V) {}
  __device__ int at(int j) const { return min((j * L + lane) * V, dim - V); }
  __device__ int skip(int j) const {
    const int p = j * L + lane;
    return p < packs ? max(p * V - (dim - V), 0) : V;
  }
};

}  // namespace
}  // namespace tgx
