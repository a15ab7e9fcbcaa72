// The residual norm's gradients (the formulas of the forward pass stand in tgx_resnorm.hip).
//
//   h = (s - m) r,  g = dy weight,  d = ds + r (g - [mean g] - h mean(g h))      ([.]: centred rows)
//   dresidual = d,  dn = d scale sigmoid(gate),  dgate = dn n (1 - sigmoid(gate))
//   dx = dn, or through the block's norm: hx = (x - mx) rx, q = dn post,
//        rx (q - [mean q] - hx mean(q hx))
//   dweight = sum dy h,  dbias = sum dy,  dscale = sum d sigmoid(gate) n,  dpost = sum dn hx
//
// The sum is formed again from x, residual and gate, as the forward pass formed it, so that
// no rounded sum enters a gradient.  A workgroup takes every gridDim.x-th group of rows; its
// lanes own fixed columns, whose sums over rows stay in registers until the end, are joined
// over the workgroup's rows in LDS in a fixed order and left in part[block][.][dim].
#include "tgx_resnorm.h"

namespace tgx {
namespace {

template <typename T, typename W, int V, int L, int C, bool PARTS>
__global__ __launch_bounds__(res_threads(L)) void resnorm_bwd(const ResArgs a) {
  constexpr int N = res_threads(L), R = N / L, S = sums_of(PARTS);
  __shared__ float lds[N / kWave];
  __shared__ float join[R > 1 ? N * V : 1];
  const Place<V, L> at(a.dim);
  const float inv = 1.f / static_cast<float>(a.dim);
  float acc[S][C][V];
#pragma unroll
  for (int k = 0; k < S; ++k)
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int u = 0; u < V; ++u) acc[k][j][u] = 0.f;
  const int64_t step = static_cast<int64_t>(gridDim.x) * R;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * R; base < a.rows; base += step) {  // workgroup-uniform
    const int64_t mine = base + threadIdx.x / L, row = min(mine, a.rows - 1);
    const bool live = mine < a.rows;
    Pack<T, V> px[C], pr[C], pg[C], py[C], ps[C];
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int c = at.at(j);
      px[j] = load_pack<T, V>(static_cast<const T*>(a.x) + row * a.x_stride + c);
      if (a.residual != nullptr) pr[j] = load_pack<T, V>(static_cast<const T*>(a.residual) + row * a.residual_stride + c);
      if (PARTS && a.gate != nullptr) pg[j] = load_pack<T, V>(static_cast<const T*>(a.gate) + row * a.gate_stride + c);
      if (a.dout != nullptr) py[j] = load_pack<T, V>(static_cast<const T*>(a.dout) + row * a.dim + c);
      if (a.dsum != nullptr) ps[j] = load_pack<T, V>(static_cast<const T*>(a.dsum) + row * a.dim + c);
    }
    const float m = a.stats[row], r = a.stats[a.rows + row];
    float mx = 0.f, rx = 1.f;
    if (PARTS && a.post != nullptr) mx = a.stats[2 * a.rows + row], rx = a.stats[3 * a.rows + row];
    // h; n, hx, and the two factors of n
    float h[C][V], n[C][V], hx[C][V], sig[C][V], rest[C][V], by[C][V];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < C; ++j) {
      Pack<W, V> w, wp, wc;
      if (a.weight != nullptr) w = load_pack<W, V>(static_cast<const W*>(a.weight) + at.at(j));
      if (PARTS && a.post != nullptr) wp = load_pack<W, V>(static_cast<const W*>(a.post) + at.at(j));
      if (PARTS && a.scale != nullptr) wc = load_pack<W, V>(static_cast<const W*>(a.scale) + at.at(j));
      const int skip = live ? at.skip(j) : V;
#pragma unroll
      for (int u = 0; u < V; ++u) {
        float s = to_f(px[j].v[u]);
        if constexpr (PARTS) {
          hx[j][u] = (s - mx) * rx;
          if (a.post != nullptr) s = hx[j][u] * to_f(wp.v[u]);
          n[j][u] = s;
          by[j][u] = a.scale != nullptr ? to_f(wc.v[u]) : 1.f;
          sig[j][u] = rest[j][u] = 1.f;
          if (a.gate != nullptr) {
            sigmoids(to_f(pg[j].v[u]), sig[j][u], rest[j][u]);
            by[j][u] *= sig[j][u];
          }
          s = fmaf(by[j][u], s, to_f(pr[j].v[u]));
        } else if (a.residual != nullptr) {
          s += to_f(pr[j].v[u]);
        }
        h[j][u] = (s - m) * r;
        const float d = a.dout != nullptr ? to_f(py[j].v[u]) : 0.f;
        const float g = a.weight != nullptr ? d * to_f(w.v[u]) : d;
        if (u >= skip) {
          s1 += g;
          s2 = fmaf(g, h[j][u], s2);
          acc[0][j][u] = fmaf(d, h[j][u], acc[0][j][u]);
          acc[1][j][u] += d;
        }
      }
    }
    if (a.dout != nullptr) {
      s1 = a.center ? row_sum<L>(s1, lds) * inv : 0.f;
      s2 = row_sum<L>(s2, lds) * inv;
    }
    float t1 = 0.f, t2 = 0.f;
#pragma unroll
    for (int j = 0; j < C; ++j) {
      Pack<W, V> w, wp;
      if (a.weight != nullptr) w = load_pack<W, V>(static_cast<const W*>(a.weight) + at.at(j));
      if (PARTS && a.post != nullptr) wp = load_pack<W, V>(static_cast<const W*>(a.post) + at.at(j));
      const int skip = live ? at.skip(j) : V;
      Pack<T, V> od, og, ox;
#pragma unroll
      for (int u = 0; u < V; ++u) {
        float d = 0.f;
        if (a.dout != nullptr) {
          const float e = to_f(py[j].v[u]);
          const float g = a.weight != nullptr ? e * to_f(w.v[u]) : e;
          d = r * (g - s1 - h[j][u] * s2);
        }
        if (a.dsum != nullptr) d += to_f(ps[j].v[u]);
        od.v[u] = from_f<T>(d);
        if constexpr (PARTS) {
          const float dn = d * by[j][u];
          og.v[u] = from_f<T>(dn * n[j][u] * rest[j][u]);
          const float q = a.post != nullptr ? dn * to_f(wp.v[u]) : dn;
          if (u >= skip) {
            acc[2][j][u] = fmaf(d * sig[j][u], n[j][u], acc[2][j][u]);
            acc[3][j][u] = fmaf(dn, hx[j][u], acc[3][j][u]);
            t1 += q;
            t2 = fmaf(q, hx[j][u], t2);
          }
          ox.v[u] = from_f<T>(q);
          n[j][u] = q;
        }
      }
      if (skip == V) continue;
      const int64_t to = row * a.dim + at.at(j);
      if (a.dres != nullptr) store_pack<T, V>(static_cast<T*>(a.dres) + to, od);
      if constexpr (PARTS) {
        if (a.dgate != nullptr) store_pack<T, V>(static_cast<T*>(a.dgate) + to, og);
        if (a.dx != nullptr && a.post == nullptr) store_pack<T, V>(static_cast<T*>(a.dx) + to, ox);
      }
    }
    if constexpr (PARTS) {
      if (a.post == nullptr || a.dx == nullptr) continue;
      t1 = a.center ? row_sum<L>(t1, lds) * inv : 0.f;
      t2 = row_sum<L>(t2, lds) * inv;
#pragma unroll
      for (int j = 0; j < C; ++j) {
        if (!live || at.skip(j) == V) continue;
        Pack<T, V> ox;
#pragma unroll
        for (int u = 0; u < V; ++u) ox.v[u] = from_f<T>(rx * (n[j][u] - t1 - hx[j][u] * t2));
        store_pack<T, V>(static_cast<T*>(a.dx) + row * a.dim + at.at(j), ox);
      }
    }
  }
  if (a.part == nullptr) return;
  float* part = a.part + static_cast<int64_t>(blockIdx.x) * S * a.dim;
#pragma unroll
  for (int k = 0; k < S; ++k)
#pragma unroll
    for (int j = 0; j < C; ++j) {
      float t[V];
#pragma unroll
      for (int u = 0; u < V; ++u) t[u] = acc[k][j][u];
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
          if (u >= skip) part[static_cast<int64_t>(k) * a.dim + at.at(j) + u] = t[u];
      }
    }
}

// the sums over the workgroups' parts [blocks][sums][dim], kCols columns per workgroup
constexpr int kCols = 16;
constexpr int kJoinThreads = 1024;

struct SumOuts {
  void* to[kSums];
};

template <typename W>
__global__ __launch_bounds__(kJoinThreads) void resnorm_join(const float* __restrict__ part, int blocks, int dim, int sums,
                                                             const SumOuts outs) {
  constexpr int G = kJoinThreads / kCols;
  __shared__ float lds[kJoinThreads];
  const int all = sums * dim, col = blockIdx.x * kCols + threadIdx.x % kCols;
  float s = 0.f;
  if (col < all) {
#pragma unroll 8
    for (int b = threadIdx.x / kCols; b < blocks; b += G) s += part[static_cast<int64_t>(b) * all + col];
  }
  lds[threadIdx.x] = s;
  __syncthreads();
  for (int half = kJoinThreads / 2; half >= kCols; half /= 2) {
    if (threadIdx.x < half) lds[threadIdx.x] += lds[threadIdx.x + half];
    __syncthreads();
  }
  if (threadIdx.x < kCols && col < all) {
    W* to = static_cast<W*>(outs.to[col / dim]);
    if (to != nullptr) to[col % dim] = from_f<W>(lds[threadIdx.x]);
  }
}

// workgroups: enough to fill the device, and rows enough for each that its sums stay small
// beside the rows it reads
int64_t res_blocks(int64_t rows, int64_t dim) {
  const int64_t per = std::max<int64_t>(1, 2048 / std::max<int64_t>(dim, 1)) * 4;
  return std::clamp<int64_t>(ops_cdiv(rows, per), 1, 2048);
}

}  // namespace
}  // namespace tgx

using namespace tgx;

extern "C" size_t tgx_residual_norm_grad_workspace_size(const tgx_residual_norm_args* args) {
  if (check_resnorm("tgx_residual_norm_grad", args, true) || args->rows == 0) return 0;
  return static_cast<size_t>(res_blocks(args->rows, args->dim)) * sums_of(has_parts(args)) * args->dim * 4;
}

extern "C" int tgx_residual_norm_grad(const tgx_residual_norm_args* args, void* stream) {
  if (const int rc = check_resnorm("tgx_residual_norm_grad", args, true)) return rc;
  const bool parts = has_parts(args);
  const SumOuts outs{{args->grad_weight, args->grad_bias, parts ? args->grad_scale : nullptr,
                      parts ? args->grad_post_weight : nullptr}};
  const bool sums = std::any_of(outs.to, outs.to + kSums, [](void* p) { return p != nullptr; });
  if (!parts && args->grad_x != nullptr)
    return fail(TGX_ERR_ARG, "tgx_residual_norm_grad: grad_x is grad_residual where nothing scales x");
  if (args->rows > 0 && args->stats == nullptr)
    return fail(TGX_ERR_ARG, "tgx_residual_norm_grad: stats must not be NULL");
  const size_t need = tgx_residual_norm_grad_workspace_size(args);
  if (sums && need > 0 && (args->workspace == nullptr || args->workspace_bytes < need || !aligned16(args->workspace)))
    return fail(TGX_ERR_ARG, "tgx_residual_norm_grad: workspace of %zu bytes, 16-byte aligned, needed", need);
  hipStream_t s = static_cast<hipStream_t>(stream);
  ResArgs a = res_args(args);
  a.part = sums ? static_cast<float*>(args->workspace) : nullptr;
  const int64_t blocks = args->rows > 0 ? res_blocks(args->rows, args->dim) : 0;
  if (blocks > 0 && (sums || a.dx != nullptr || a.dres != nullptr || a.dgate != nullptr)) {
    const int rc = by_type(args->dtype, [&](auto t) {
      using T = decltype(t);
      return by_type(args->wdtype, [&](auto wt) {
        using W = decltype(wt);
        return res_shape<T>(args->dim, [&](auto v, auto l, auto c) {
          constexpr int V = decltype(v)::value, L = decltype(l)::value, C = decltype(c)::value;
          const dim3 grid(static_cast<unsigned>(blocks)), block(res_threads(L));
          if (parts) hipLaunchKernelGGL((resnorm_bwd<T, W, V, L, C, true>), grid, block, 0, s, a);
          else hipLaunchKernelGGL((resnorm_bwd<T, W, V, L, C, false>), grid, block, 0, s, a);
          return check_launch("resnorm_bwd");
        });
      });
    });
    if (rc) return rc;
  }
  if (!sums) return TGX_OK;
  return by_type(args->wdtype, [&](auto wt) {
    using W = decltype(wt);
    const int n = sums_of(parts);
    hipLaunchKernelGGL(resnorm_join<W>, dim3(static_cast<unsigned>(ops_cdiv(n * args->dim, kCols))), dim3(kJoinThreads), 0,
                       s, a.part, static_cast<int>(blocks), static_cast<int>(args->dim), n, outs);
    return check_launch("resnorm_join");
  });
}
