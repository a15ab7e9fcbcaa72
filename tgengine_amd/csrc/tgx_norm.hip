// Layer norm over the last dimension, forward and backward.
//
//   m = mean x,  r = 1 / sqrt(mean (x - m)^2 + eps),  h = (x - m) r,  y = h w + b
//   dx = r (g - mean g - h mean (g h)),  g = dy w
//   dw = sum over rows of dy h,  db = sum over rows of dy
//
// L lanes share a row and keep it in registers as C packs each, so that x is read
// once and its variance is the mean of squares about the mean, not a difference of
// sums.  Statistics and sums are held in 32 bits; y and dx are rounded once, dw and
// db once after the last sum.
#include "tgx_ops.h"

namespace tgx {
namespace {

constexpr int kNormThreads = 256;

// the sum over the L lanes of a row; L = 256: the whole workgroup, through `lds` [4]
template <int L>
__device__ __forceinline__ float row_sum(float x, float* lds) {
  if constexpr (L <= kWave) {
    return group_sum<L>(x);
  } else {
    x = group_sum<kWave>(x);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) lds[threadIdx.x / kWave] = x;
    __syncthreads();
    return (lds[0] + lds[1]) + (lds[2] + lds[3]);
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

// Rows that a group of lanes takes at a time: with one pack a lane, several rows are in
// flight, share the weights and hide each other's sums.  Lanes that take a whole row side
// by side touch fewer cache lines than few lanes with more packs each where rows do not
// begin on a line (786,432 x 172 bf16 rows, forward: 8 lanes of 3 packs 141 us, 32 lanes of
// one 163, and with four rows 135; backward 209, 192, and with two rows 176).  Not every call
// is faster so: with 136 and 192 values the forward pass takes 118 and 128 us, and 94 and 111
// with 8 lanes of 3 packs; with 172, where a backward pass runs between the calls, 131 to 154
// and 109 to 114.
//
// HBM bounds it: those 541 MB take the forward pass 135 us, 4.0 TB/s where a copy without
// gaps in its lines reaches 6.2; 240 x 172 f32 rows take 4.4 us, a chain of one read, two
// sums over the lanes and one write.
constexpr int fwd_rows(int c) { return c == 1 ? 4 : c == 2 ? 2 : 1; }
constexpr int bwd_rows(int c) { return c == 1 ? 2 : 1; }

template <typename T, typename W, int V, int L, int C>
__global__ __launch_bounds__(kNormThreads) void norm_fwd(const T* __restrict__ x, int64_t rows, int dim, int64_t stride,
                                                         const W* __restrict__ weight, const W* __restrict__ bias,
                                                         float eps, T* __restrict__ out, float* __restrict__ mean,
                                                         float* __restrict__ rstd) {
  constexpr int U = fwd_rows(C), G = kNormThreads / L;
  __shared__ float lds[kNormThreads / kWave];
  const Place<V, L> at(dim);
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * (G * U) + threadIdx.x / L;
  Pack<T, V> p[U][C];
#pragma unroll
  for (int a = 0; a < U; ++a)
#pragma unroll
    for (int j = 0; j < C; ++j) p[a][j] = load_pack<T, V>(x + min(row0 + a * G, rows - 1) * stride + at.at(j));
  float m[U], r[U];
#pragma unroll
  for (int a = 0; a < U; ++a) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int skip = at.skip(j);
#pragma unroll
      for (int u = 0; u < V; ++u) s += u >= skip ? to_f(p[a][j].v[u]) : 0.f;
    }
    m[a] = s;
  }
#pragma unroll
  for (int a = 0; a < U; ++a) m[a] = row_sum<L>(m[a], lds) / static_cast<float>(dim);
#pragma unroll
  for (int a = 0; a < U; ++a) {
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int skip = at.skip(j);
#pragma unroll
      for (int u = 0; u < V; ++u) {
        const float f = to_f(p[a][j].v[u]) - m[a];
        q += u >= skip ? f * f : 0.f;
      }
    }
    r[a] = q;
  }
#pragma unroll
  for (int a = 0; a < U; ++a) r[a] = 1.f / sqrtf(row_sum<L>(r[a], lds) / static_cast<float>(dim) + eps);
#pragma unroll
  for (int j = 0; j < C; ++j) {
    if (at.skip(j) == V) continue;
    const int c = at.at(j);
    Pack<W, V> w, b;
    if (weight != nullptr) w = load_pack<W, V>(weight + c);
    if (bias != nullptr) b = load_pack<W, V>(bias + c);
#pragma unroll
    for (int a = 0; a < U; ++a) {
      if (row0 + a * G >= rows) break;
      Pack<T, V> o;
#pragma unroll
      for (int u = 0; u < V; ++u) {
        float y = (to_f(p[a][j].v[u]) - m[a]) * r[a];
        if (weight != nullptr) y *= to_f(w.v[u]);
        if (bias != nullptr) y += to_f(b.v[u]);
        o.v[u] = from_f<T>(y);
      }
      store_pack<T, V>(out + (row0 + a * G) * dim + c, o);
    }
  }
  if (at.lane == 0 && mean != nullptr)
#pragma unroll
    for (int a = 0; a < U; ++a) {
      if (row0 + a * G >= rows) break;
      mean[row0 + a * G] = m[a];
      rstd[row0 + a * G] = r[a];
    }
}

// A workgroup takes every gridDim.x-th group of rows.  Its lanes own fixed columns, so
// the sums over rows for dw and db stay in registers until the end, are joined over the
// workgroup's rows in LDS in a fixed order and left in part[block][2][dim].
// HBM bounds it: 786,432 x 172 bf16 rows (818 MB) 171 us, 4.8 TB/s, and norm_join 7.5 us.
template <typename T, typename W, int V, int L, int C>
__global__ __launch_bounds__(kNormThreads) void norm_bwd(const T* __restrict__ x, const T* __restrict__ dy, int64_t rows,
                                                         int dim, int64_t stride, const W* __restrict__ weight,
                                                         const float* __restrict__ mean, const float* __restrict__ rstd,
                                                         T* __restrict__ dx, float* __restrict__ part) {
  constexpr int R = kNormThreads / L;  // rows a workgroup takes at a time
  __shared__ float lds[kNormThreads / kWave];
  __shared__ float join[R > 1 ? kNormThreads * V : 1];
  const Place<V, L> at(dim);
  float aw[C][V], ab[C][V];
#pragma unroll
  for (int j = 0; j < C; ++j)
#pragma unroll
    for (int u = 0; u < V; ++u) aw[j][u] = ab[j][u] = 0.f;
  constexpr int U = bwd_rows(C);
  const int64_t step = static_cast<int64_t>(gridDim.x) * R * U;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * R * U; base < rows; base += step) {  // workgroup-uniform
    const int64_t row0 = base + threadIdx.x / L;
    Pack<T, V> px[U][C], pg[U][C];
    float m[U], r[U], s1[U], s2[U];
#pragma unroll
    for (int a = 0; a < U; ++a) {
      const int64_t row = min(row0 + a * R, rows - 1);
      m[a] = mean[row];
      r[a] = rstd[row];
#pragma unroll
      for (int j = 0; j < C; ++j) {
        px[a][j] = load_pack<T, V>(x + row * stride + at.at(j));
        pg[a][j] = load_pack<T, V>(dy + row * dim + at.at(j));
      }
    }
    Pack<W, V> w[C];
#pragma unroll
    for (int j = 0; j < C; ++j)
      if (weight != nullptr) w[j] = load_pack<W, V>(weight + at.at(j));
#pragma unroll
    for (int a = 0; a < U; ++a) {
      s1[a] = s2[a] = 0.f;
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const int skip = row0 + a * R < rows ? at.skip(j) : V;
#pragma unroll
        for (int u = 0; u < V; ++u) {
          const float h = (to_f(px[a][j].v[u]) - m[a]) * r[a], d = to_f(pg[a][j].v[u]);
          const float g = weight != nullptr ? d * to_f(w[j].v[u]) : d;
          if (u >= skip) {
            s1[a] += g;
            s2[a] = fmaf(g, h, s2[a]);
            aw[j][u] = fmaf(d, h, aw[j][u]);
            ab[j][u] += d;
          }
        }
      }
    }
#pragma unroll
    for (int a = 0; a < U; ++a) {
      s1[a] = row_sum<L>(s1[a], lds) / static_cast<float>(dim);
      s2[a] = row_sum<L>(s2[a], lds) / static_cast<float>(dim);
    }
    if (dx == nullptr) continue;
#pragma unroll
    for (int a = 0; a < U; ++a) {
      const int64_t row = row0 + a * R;
      if (row >= rows) break;
#pragma unroll
      for (int j = 0; j < C; ++j) {
        if (at.skip(j) == V) continue;
        Pack<T, V> o;
#pragma unroll
        for (int u = 0; u < V; ++u) {
          const float h = (to_f(px[a][j].v[u]) - m[a]) * r[a], d = to_f(pg[a][j].v[u]);
          const float g = weight != nullptr ? d * to_f(w[j].v[u]) : d;
          o.v[u] = from_f<T>(r[a] * (g - s1[a] - h * s2[a]));
        }
        store_pack<T, V>(dx + row * dim + at.at(j), o);
      }
    }
  }
  if (part == nullptr) return;
  float* pw = part + static_cast<int64_t>(blockIdx.x) * 2 * dim;
#pragma unroll
  for (int j = 0; j < C; ++j) {
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      float t[V];
#pragma unroll
      for (int u = 0; u < V; ++u) t[u] = which ? ab[j][u] : aw[j][u];
      if constexpr (R > 1) {
        __syncthreads();
#pragma unroll
        for (int u = 0; u < V; ++u) join[threadIdx.x * V + u] = t[u];
        __syncthreads();
        if (threadIdx.x < L) {
#pragma unroll 4
          for (int w = 1; w < R; ++w)
#pragma unroll
            for (int u = 0; u < V; ++u) t[u] += join[(w * L + threadIdx.x) * V + u];
        }
      }
      if (threadIdx.x < L) {
        const int skip = at.skip(j);
#pragma unroll
        for (int u = 0; u < V; ++u)
          if (u >= skip) pw[which * dim + at.at(j) + u] = t[u];
      }
    }
  }
}

// dw and db: column sums of part [blocks][2 dim], kCols columns per workgroup
constexpr int kCols = 16;
constexpr int kJoinThreads = 1024;

template <typename W>
__global__ __launch_bounds__(kJoinThreads) void norm_join(const float* __restrict__ part, int blocks, int dim,
                                                          W* __restrict__ dw, W* __restrict__ db) {
  constexpr int G = kJoinThreads / kCols;
  __shared__ float lds[kJoinThreads];
  const int col = blockIdx.x * kCols + threadIdx.x % kCols;
  float s = 0.f;
  if (col < 2 * dim) {
#pragma unroll 8
    for (int b = threadIdx.x / kCols; b < blocks; b += G) s += part[static_cast<int64_t>(b) * 2 * dim + col];
  }
  lds[threadIdx.x] = s;
  __syncthreads();
  for (int half = kJoinThreads / 2; half >= kCols; half /= 2) {
    if (threadIdx.x < half) lds[threadIdx.x] += lds[threadIdx.x + half];
    __syncthreads();
  }
  if (threadIdx.x < kCols && col < 2 * dim) {
    const W v = from_f<W>(lds[threadIdx.x]);
    if (col < dim) {
      if (dw != nullptr) dw[col] = v;
    } else if (db != nullptr) {
      db[col - dim] = v;
    }
  }
}

// Calls f(V, L, C) with the lanes and packs a row of `dim` values takes: one pack a lane up
// to 64 lanes, then more, then the whole workgroup.
// The backward pass of f32 rows of 33 to 64 packs takes 16 lanes of 3 or 4: 264,192 x 256
// take 163 us so and 169 with 64 lanes, 393,216 x 172 189 and 193 (bf16 rows of 512, whose
// sums take twice the registers, 206 and 165).
template <typename T, bool GRAD, typename F>
int by_shape(int64_t dim, F&& f) {
#define TGX_SHAPE(V, L, C) \
  f(std::integral_constant<int, V>{}, std::integral_constant<int, L>{}, std::integral_constant<int, C>{})
  constexpr int V = kWide<T>;
  if (dim < V) return TGX_SHAPE(1, 8, 1);
  const int64_t packs = ops_cdiv(dim, V);
  if (packs <= 8) return TGX_SHAPE(V, 8, 1);
  if (packs <= 16) return TGX_SHAPE(V, 16, 1);
  if (packs <= 32) return TGX_SHAPE(V, 32, 1);
  if constexpr (GRAD && sizeof(T) == 4) {
    if (packs <= 48) return TGX_SHAPE(V, 16, 3);
    if (packs <= 64) return TGX_SHAPE(V, 16, 4);
  } else {
    if (packs <= 64) return TGX_SHAPE(V, 64, 1);
  }
  if (packs <= 128) return TGX_SHAPE(V, 64, 2);
  if (packs <= 256) return TGX_SHAPE(V, 64, 4);
  if (packs <= 512) return TGX_SHAPE(V, 256, 2);
  if (packs <= 1024) return TGX_SHAPE(V, 256, 4);
  if constexpr (V == 8) {
    return TGX_SHAPE(V, 256, 8);
  } else {
    if (packs <= 2048) return TGX_SHAPE(V, 256, 8);
    return TGX_SHAPE(V, 256, 16);
  }
#undef TGX_SHAPE
}
static_assert(TGX_MAX_NORM_DIM <= 256 * 8 * 8 && TGX_MAX_NORM_DIM <= 256 * 16 * 4, "a row fits its workgroup");

// workgroups of the backward pass: enough to fill the device, and rows enough for each
// that its part of dw and db (8 dim bytes) stays small beside the rows it reads
int64_t norm_blocks(int64_t rows, int64_t dim) {
  const int64_t per = std::max<int64_t>(1, 2048 / std::max<int64_t>(dim, 1)) * 4;
  return std::clamp<int64_t>(ops_cdiv(rows, per), 1, 2048);
}

int check_norm(const char* what, const void* x, const void* y, int64_t rows, int64_t dim, int64_t stride,
               int32_t dtype, int32_t wdtype) {
  if (rows < 0 || dim < 1 || (rows > 1 && stride < 0))
    return fail(TGX_ERR_ARG, "%s: rows=%lld dim=%lld stride=%lld", what, static_cast<long long>(rows),
                static_cast<long long>(dim), static_cast<long long>(stride));
  if (elem_bytes(dtype) == 0 || elem_bytes(wdtype) == 0)
    return fail(TGX_ERR_DTYPE, "%s: dtypes %d and %d", what, dtype, wdtype);
  if (dim > TGX_MAX_NORM_DIM || rows >= (int64_t(1) << 31))
    return fail(TGX_ERR_LIMIT, "%s: dim=%lld (at most %d), rows=%lld (below 2^31)", what, static_cast<long long>(dim),
                TGX_MAX_NORM_DIM, static_cast<long long>(rows));
  if (rows > 0 && (x == nullptr || y == nullptr)) return fail(TGX_ERR_ARG, "%s: x and y must not be NULL", what);
  return TGX_OK;
}

}  // namespace
}  // namespace tgx

using namespace tgx;

extern "C" int tgx_layer_norm(const void* x, int64_t rows, int64_t dim, int64_t stride, int32_t dtype,
                              const void* weight, const void* bias, int32_t wdtype, float eps, void* out, float* mean,
                              float* rstd, void* stream) {
  const int rc = check_norm("tgx_layer_norm", x, out, rows, dim, stride, dtype, wdtype);
  if (rc) return rc;
  if ((mean == nullptr) != (rstd == nullptr)) return fail(TGX_ERR_ARG, "tgx_layer_norm: mean and rstd come together");
  if (rows == 0) return TGX_OK;
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    return by_type(wdtype, [&](auto wt) {
      using W = decltype(wt);
      return by_shape<T, false>(dim, [&](auto v, auto l, auto c) {
        constexpr int V = decltype(v)::value, L = decltype(l)::value, C = decltype(c)::value;
        const int64_t blocks = ops_cdiv(rows, kNormThreads / L * fwd_rows(C));
        if (const int e = check_grid("tgx_layer_norm", blocks, kNormThreads)) return e;
        hipLaunchKernelGGL((norm_fwd<T, W, V, L, C>), dim3(static_cast<unsigned>(blocks)), dim3(kNormThreads), 0,
                           static_cast<hipStream_t>(stream), static_cast<const T*>(x), rows, static_cast<int>(dim),
                           stride, static_cast<const W*>(weight), static_cast<const W*>(bias), eps,
                           static_cast<T*>(out), mean, rstd);
        return check_launch("norm_fwd");
      });
    });
  });
}

extern "C" size_t tgx_layer_norm_grad_workspace_size(int64_t rows, int64_t dim) {
  if (rows <= 0 || dim <= 0) return 0;
  return static_cast<size_t>(norm_blocks(rows, dim)) * 2 * static_cast<size_t>(dim) * 4;
}

extern "C" int tgx_layer_norm_grad(const void* x, const void* dy, int64_t rows, int64_t dim, int64_t stride,
                                   int32_t dtype, const void* weight, int32_t wdtype, const float* mean,
                                   const float* rstd, void* dx, void* dw, void* db, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  int rc = check_norm("tgx_layer_norm_grad", x, dy, rows, dim, stride, dtype, wdtype);
  if (rc) return rc;
  const bool sums = dw != nullptr || db != nullptr;
  if (rows > 0 && (mean == nullptr || rstd == nullptr))
    return fail(TGX_ERR_ARG, "tgx_layer_norm_grad: mean and rstd must not be NULL");
  const size_t need = tgx_layer_norm_grad_workspace_size(rows, dim);
  if (sums && rows > 0 && (workspace == nullptr || workspace_bytes < need || !aligned16(workspace)))
    return fail(TGX_ERR_ARG, "tgx_layer_norm_grad: workspace of %zu bytes, 16-byte aligned, needed", need);
  hipStream_t s = static_cast<hipStream_t>(stream);
  float* part = sums ? static_cast<float*>(workspace) : nullptr;
  const int64_t blocks = rows > 0 ? norm_blocks(rows, dim) : 0;
  if (rows > 0 && (sums || dx != nullptr)) {
    rc = by_type(dtype, [&](auto t) {
      using T = decltype(t);
      return by_type(wdtype, [&](auto wt) {
        using W = decltype(wt);
        return by_shape<T, true>(dim, [&](auto v, auto l, auto c) {
          constexpr int V = decltype(v)::value, L = decltype(l)::value, C = decltype(c)::value;
          hipLaunchKernelGGL((norm_bwd<T, W, V, L, C>), dim3(static_cast<unsigned>(blocks)), dim3(kNormThreads), 0, s,
                             static_cast<const T*>(x), static_cast<const T*>(dy), rows, static_cast<int>(dim), stride,
                             static_cast<const W*>(weight), mean, rstd, static_cast<T*>(dx), part);
          return check_launch("norm_bwd");
        });
      });
    });
    if (rc) return rc;
  }
  if (!sums) return TGX_OK;
  return by_type(wdtype, [&](auto wt) {
    using W = decltype(wt);
    hipLaunchKernelGGL(norm_join<W>, dim3(static_cast<unsigned>(ops_cdiv(2 * dim, kCols))), dim3(kJoinThreads), 0, s,
                       part, static_cast<int>(blocks), static_cast<int>(dim), static_cast<W*>(dw),
                       static_cast<W*>(db));
    return check_launch("norm_join");
  });
}
