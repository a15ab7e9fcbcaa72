// The residual sum after a block and the norm before the next one, forward.
//
//   n = x, or with post the block's own norm: (x - mx) rx post
//   s = residual + scale sigmoid(gate) n          (a factor that is left out is 1)
//   y = (s - m) r weight + bias
//
// m is the mean of a row and r = 1 / sqrt(mean (s - m)^2 + eps); rows that are not centred
// take m = 0.  L lanes share a row and hold it in registers as C packs each, so that x,
// residual and gate are read once and the norm works on the sum before it is rounded: s and
// y are rounded once each.  Statistics and sums are of 32 bits.
//
// HBM bounds it, and vector instructions are close: 786,432 x 172 bf16 rows (1.08 GB, rows that
// begin inside a line) take 179 us at best, 6.0 TB/s, and 198 in the median between backward
// passes; their 106M instructions keep the vector units busy all the time, so that the time goes
// with the clock, which falls in long runs.  8,001 x 4,096 gated bf16 rows (0.33 GB) 63 us (61 at
// best), 5.2 TB/s, units busy 77%; 240 x 172 f32 rows 3.6 us, a chain of one read, two sums and one
// write.
#include "tgx_resnorm.h"

namespace tgx {
namespace {

// Rows that a group of lanes takes at a time: with one pack a lane and nothing that scales x,
// two are in flight and hide each other's sums.  786,432 x 172 bf16 rows, forward and backward:
// 489 us with two or four, 510 with one; 240 x 172 f32 rows: 3.4 us with one, 3.7 with two, 5.1
// with four.
constexpr int res_rows(int lanes, int packs, bool parts) { return packs == 1 && lanes <= kWave && !parts ? 2 : 1; }

template <typename T, typename W, int V, int L, int C, bool PARTS>
__global__ __launch_bounds__(res_threads(L)) void resnorm_fwd(const ResArgs a) {
  constexpr int N = res_threads(L), G = N / L, U = res_rows(L, C, PARTS);
  __shared__ float lds[N / kWave];
  const Place<V, L> at(a.dim);
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (G * U) + threadIdx.x / L;
  Pack<T, V> px[U][C], pr[U][C], pg[C];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int64_t row = min(first + i * G, a.rows - 1);
#pragma unroll
    for (int j = 0; j < C; ++j) {
      px[i][j] = load_pack<T, V>(static_cast<const T*>(a.x) + row * a.x_stride + at.at(j));
      pr[i][j] = load_pack<T, V>(static_cast<const T*>(a.residual) + row * a.residual_stride + at.at(j));
      if constexpr (PARTS)
        if (a.gate != nullptr) pg[j] = load_pack<T, V>(static_cast<const T*>(a.gate) + row * a.gate_stride + at.at(j));
    }
  }
  float s[U][C][V], m[U], r[U], mx = 0.f, rx = 0.f;
#pragma unroll
  for (int i = 0; i < U; ++i) {
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int u = 0; u < V; ++u) s[i][j][u] = to_f(px[i][j].v[u]);
    if constexpr (PARTS) {
      if (a.post != nullptr) {
        row_stats<V, L, C>(s[i], at, a, lds, mx, rx);
#pragma unroll
        for (int j = 0; j < C; ++j) {
          const Pack<W, V> w = load_pack<W, V>(static_cast<const W*>(a.post) + at.at(j));
#pragma unroll
          for (int u = 0; u < V; ++u) s[i][j][u] = (s[i][j][u] - mx) * rx * to_f(w.v[u]);
        }
      }
#pragma unroll
      for (int j = 0; j < C; ++j) {
        Pack<W, V> w;
        if (a.scale != nullptr) w = load_pack<W, V>(static_cast<const W*>(a.scale) + at.at(j));
#pragma unroll
        for (int u = 0; u < V; ++u) {
          float by = a.scale != nullptr ? to_f(w.v[u]) : 1.f;
          if (a.gate != nullptr) {
            // 1 less the smaller one, as the backward pass, which keeps only that, forms it again
            const float g = to_f(pg[j].v[u]);
            float larger;
            const float small = sigmoid_small(g, larger);
            by *= g < 0.f ? small : 1.f - small;
          }
          s[i][j][u] = fmaf(by, s[i][j][u], to_f(pr[i][j].v[u]));
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < C; ++j)
#pragma unroll
        for (int u = 0; u < V; ++u) s[i][j][u] += to_f(pr[i][j].v[u]);
    }
  }
#pragma unroll
  for (int i = 0; i < U; ++i) row_stats<V, L, C>(s[i], at, a, lds, m[i], r[i]);
#pragma unroll
  for (int j = 0; j < C; ++j) {
    if (at.skip(j) == V) continue;
    const int c = at.at(j);
    Pack<W, V> w, b;
    if (a.weight != nullptr) w = load_pack<W, V>(static_cast<const W*>(a.weight) + c);
    if (a.bias != nullptr) b = load_pack<W, V>(static_cast<const W*>(a.bias) + c);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t row = first + i * G;
      if (row >= a.rows) break;
      Pack<T, V> o, t;
#pragma unroll
      for (int u = 0; u < V; ++u) {
        float y = (s[i][j][u] - m[i]) * r[i];
        if (a.weight != nullptr) y *= to_f(w.v[u]);
        if (a.bias != nullptr) y += to_f(b.v[u]);
        o.v[u] = from_f<T>(y);
        t.v[u] = from_f<T>(s[i][j][u]);
      }
      store_pack<T, V>(static_cast<T*>(a.out) + row * a.dim + c, o);
      store_pack<T, V>(static_cast<T*>(a.sum) + row * a.dim + c, t);
    }
  }
  if (at.lane == 0 && a.stats != nullptr)
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t row = first + i * G;
      if (row >= a.rows) break;
      a.stats[row] = m[i];
      a.stats[a.rows + row] = r[i];
      if (PARTS && a.post != nullptr) {
        a.stats[2 * a.rows + row] = mx;
        a.stats[3 * a.rows + row] = rx;
      }
    }
}

}  // namespace
}  // namespace tgx

using namespace tgx;

extern "C" int tgx_residual_norm(const tgx_residual_norm_args* args, void* stream) {
  if (const int rc = check_resnorm("tgx_residual_norm", args, false)) return rc;
  if (args->rows == 0) return TGX_OK;
  if (args->out == nullptr || args->sum == nullptr)
    return fail(TGX_ERR_ARG, "tgx_residual_norm: out and sum must not be NULL");
  return by_type(args->dtype, [&](auto t) {
    using T = decltype(t);
    return by_type(args->wdtype, [&](auto wt) {
      using W = decltype(wt);
      return res_shape<T>(args->dim, [&](auto v, auto l, auto c) {
        constexpr int V = decltype(v)::value, L = decltype(l)::value, C = decltype(c)::value, N = res_threads(L);
        auto launch = [&](auto parts) {
          constexpr bool PARTS = decltype(parts)::value;
          const int64_t blocks = ops_cdiv(args->rows, N / L * res_rows(L, C, PARTS));
          if (const int e = check_grid("tgx_residual_norm", blocks, N)) return e;
          hipLaunchKernelGGL((resnorm_fwd<T, W, V, L, C, PARTS>), dim3(static_cast<unsigned>(blocks)), dim3(N), 0,
                             static_cast<hipStream_t>(stream), res_args(args));
          return check_launch("resnorm_fwd");
        };
        return has_parts(args) ? launch(std::true_type{}) : launch(std::false_type{});
      });
    });
  });
}
