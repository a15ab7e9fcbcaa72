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
//
// The sum alone is bound by vector instructions beside HBM: 786,432 x 172 bf16 rows (five
// tensors, 1.35 GB) take 288 us at best, 4.7 TB/s, and 306 in the median, with the vector units
// busy 86% (128M instructions; 22 of the 32 lanes of a row hold values).  With a gate and a scale
// 176 registers allow two wavefronts a SIMD, one workgroup of 8,001 x 4,096 bf16 rows (seven tensors,
// 0.46 GB) on a compute unit: 121 us (118 at best) and 9 for the join, 3.8 TB/s, units busy 52%,
// so that neither is full: each row's barrier is waited for with nothing beside it.
#include "tgx_resnorm.h"

namespace tgx {
namespace {

// Bits of a kernel's kind: what the call's sums have.  Without kScaled, x joins the sum as it is.
constexpr int kScaled = 1, kGate = 2, kPost = 4;

template <size_t N>
struct __attribute__((packed, aligned(2))) Regs {
  uint32_t v[N];
};

// What a second pass over a row needs of a value it forms again from what was read, rather
// than have six values more a value leave the device half empty.  `again` makes the compiler
// do so.
template <typename T, int V>
__device__ __forceinline__ void again(Pack<T, V>& p) {
  if constexpr (sizeof(p) % 4 == 0) {
    auto w = __builtin_bit_cast(Regs<sizeof(p) / 4>, p);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(p) / 4); ++i) asm volatile("" : "+v"(w.v[i]));
    p = __builtin_bit_cast(Pack<T, V>, w);
  }
}

// both sums over the L lanes of a row; `lds` [2][2][L / 64], whose halves take turns, so that
// one barrier a call is enough
template <int L>
__device__ __forceinline__ void row_sums(float& x, float& y, float* lds, int turn) {
  if constexpr (L <= kWave) {
    x = group_sum<L>(x);
    y = group_sum<L>(y);
  } else {
    constexpr int N = L / kWave;
    x = group_sum<kWave>(x);
    y = group_sum<kWave>(y);
    float* at = lds + (turn & 1) * 2 * N;
    if ((threadIdx.x & (kWave - 1)) == 0) {
      at[threadIdx.x / kWave] = x;
      at[N + threadIdx.x / kWave] = y;
    }
    __syncthreads();
    x = group_sum<N>(at[threadIdx.x & (N - 1)]);
    y = group_sum<N>(at[N + (threadIdx.x & (N - 1))]);
  }
}

template <typename T, typename W, int V, int L, int C, int KIND>
__global__ __launch_bounds__(res_threads(L)) void resnorm_bwd(const ResArgs a) {
  constexpr bool SCALED = KIND & kScaled, GATE = KIND & kGate, POST = KIND & kPost;
  constexpr int N = res_threads(L), R = N / L, S = sums_of(SCALED);
  __shared__ float lds[L > kWave ? 4 * L / kWave : 1];
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
  Pack<W, V> w[C], wp[C], wc[C];
#pragma unroll
  for (int j = 0; j < C; ++j) {
#pragma unroll
    for (int u = 0; u < V; ++u) w[j].v[u] = wc[j].v[u] = from_f<W>(1.f);
    if (a.weight != nullptr) w[j] = load_pack<W, V>(static_cast<const W*>(a.weight) + at.at(j));
    if (POST) wp[j] = load_pack<W, V>(static_cast<const W*>(a.post) + at.at(j));
    if (SCALED && a.scale != nullptr) wc[j] = load_pack<W, V>(static_cast<const W*>(a.scale) + at.at(j));
  }
  struct Row {
    Pack<T, V> x[C], r[C], g[C], y[C], s[C];
    float m, rstd, mx, rx;
  };
  // from the last row: what the forward pass read last is still in the caches
  auto row_of = [&](int64_t mine) { return a.rows - 1 - mine; };
  // gradients that are not given are zeros, and so are those of rows past the last: they add
  // nothing to a sum
  auto read = [&](Row& o, int64_t mine) {
    const int64_t row = row_of(min(mine, a.rows - 1));
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int c = at.at(j);
      o.x[j] = load_pack<T, V>(static_cast<const T*>(a.x) + row * a.x_stride + c);
      if (SCALED || a.residual != nullptr) o.r[j] = load_pack<T, V>(static_cast<const T*>(a.residual) + row * a.residual_stride + c);
      if (GATE) o.g[j] = load_pack<T, V>(static_cast<const T*>(a.gate) + row * a.gate_stride + c);
      if (a.dout != nullptr) o.y[j] = load_pack<T, V>(static_cast<const T*>(a.dout) + row * a.dim + c);
      if (a.dsum != nullptr) o.s[j] = load_pack<T, V>(static_cast<const T*>(a.dsum) + row * a.dim + c);
    }
    o.m = a.stats[row];
    o.rstd = a.stats[a.rows + row];
    if (POST) o.mx = a.stats[2 * a.rows + row], o.rx = a.stats[3 * a.rows + row];
  };
  auto clear = [](Pack<T, V>& p, int n) {
#pragma unroll
    for (int u = 0; u < V; ++u) p.v[u] = u < n ? from_f<T>(0.f) : p.v[u];
  };
  const int64_t step = static_cast<int64_t>(gridDim.x) * R;
  Row now, next;
  read(next, static_cast<int64_t>(blockIdx.x) * R + threadIdx.x / L);
  int turn = 0;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * R; base < a.rows; base += step) {  // workgroup-uniform
    const int64_t mine = base + threadIdx.x / L;
    now = next;
    read(next, mine + step);  // on its way while this row is worked on
#pragma unroll
    for (int j = 0; j < C; ++j) {
      again(w[j]);
      if constexpr (POST) again(wp[j]);
      if constexpr (SCALED) again(wc[j]);
      if (a.dout == nullptr || mine >= a.rows) clear(now.y[j], V);
      if (a.dsum == nullptr || mine >= a.rows) clear(now.s[j], V);
    }
    const float m = now.m, r = now.rstd, mx = POST ? now.mx : 0.f, rx = POST ? now.rx : 1.f;
    // the smaller of sigmoid(gate) and 1 - sigmoid(gate): the other is 1 less it
    float small[C][V];
    struct Value {
      float h, hx, n, sig, rest, by;
    };
    auto value = [&](int j, int u) {
      Value v{0.f, 0.f, to_f(now.x[j].v[u]), 1.f, 1.f, 1.f};
      if constexpr (SCALED) {
        if constexpr (POST) {
          v.hx = (v.n - mx) * rx;
          v.n = v.hx * to_f(wp[j].v[u]);
        }
        v.by = to_f(wc[j].v[u]);
        if constexpr (GATE) {
          const bool neg = to_f(now.g[j].v[u]) < 0.f;
          const float big = 1.f - small[j][u];
          v.sig = neg ? small[j][u] : big;
          v.rest = neg ? big : small[j][u];
          v.by *= v.sig;
        }
        v.h = (fmaf(v.by, v.n, to_f(now.r[j].v[u])) - m) * r;
      } else {
        v.h = ((a.residual != nullptr ? v.n + to_f(now.r[j].v[u]) : v.n) - m) * r;
      }
      return v;
    };
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < C; ++j) {
      Pack<T, V> y = now.y[j];
      if (at.skip(j) > 0) clear(y, at.skip(j));  // values of the pack before
#pragma unroll
      for (int u = 0; u < V; ++u) {
        if constexpr (GATE) {
          float larger;
          small[j][u] = sigmoid_small(to_f(now.g[j].v[u]), larger);
        }
        const float h = value(j, u).h, dy = to_f(y.v[u]), g = dy * to_f(w[j].v[u]);
        s1 += g;
        s2 = fmaf(g, h, s2);
        acc[0][j][u] = fmaf(dy, h, acc[0][j][u]);
        acc[1][j][u] += dy;
      }
      again(now.x[j]);
    }
    row_sums<L>(s1, s2, lds, turn++);
    s1 = a.center ? s1 * inv : 0.f;
    s2 *= inv;
    float t1 = 0.f, t2 = 0.f, q[C][V];
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int skip = mine < a.rows ? at.skip(j) : V;
      Pack<T, V> od, og, ox;
#pragma unroll
      for (int u = 0; u < V; ++u) {
        const Value v = value(j, u);
        const float g = to_f(now.y[j].v[u]) * to_f(w[j].v[u]);
        const float d = fmaf(r, fmaf(-v.h, s2, g - s1), to_f(now.s[j].v[u]));
        od.v[u] = from_f<T>(d);
        if constexpr (SCALED) {
          const float dn = d * v.by;
          acc[2][j][u] = fmaf(d * v.sig, v.n, acc[2][j][u]);
          if constexpr (GATE) og.v[u] = from_f<T>(dn * v.n * v.rest);
          if constexpr (POST) {
            acc[3][j][u] = fmaf(dn, v.hx, acc[3][j][u]);
            q[j][u] = dn * to_f(wp[j].v[u]);
            const float own = u >= skip ? q[j][u] : 0.f;
            t1 += own;
            t2 = fmaf(own, v.hx, t2);
          } else {
            ox.v[u] = from_f<T>(dn);
          }
        }
      }
      again(now.x[j]);
      if (skip == V) continue;
      const int64_t to = row_of(mine) * a.dim + at.at(j);
      if (a.dres != nullptr) store_pack<T, V>(static_cast<T*>(a.dres) + to, od);
      if constexpr (GATE)
        if (a.dgate != nullptr) store_pack<T, V>(static_cast<T*>(a.dgate) + to, og);
      if constexpr (SCALED && !POST)
        if (a.dx != nullptr) store_pack<T, V>(static_cast<T*>(a.dx) + to, ox);
    }
    if constexpr (POST) {
      if (a.dx == nullptr) continue;
      row_sums<L>(t1, t2, lds, turn++);
      t1 = a.center ? t1 * inv : 0.f;
      t2 *= inv;
#pragma unroll
      for (int j = 0; j < C; ++j) {
        if (mine >= a.rows || at.skip(j) == V) continue;
        Pack<T, V> ox;
#pragma unroll
        for (int u = 0; u < V; ++u) {
          const float hx = (to_f(now.x[j].v[u]) - mx) * rx;
          ox.v[u] = from_f<T>(rx * fmaf(-hx, t2, q[j][u] - t1));
        }
        store_pack<T, V>(static_cast<T*>(a.dx) + row_of(mine) * a.dim + at.at(j), ox);
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
constexpr int kCols = 32;
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

// workgroups: about what the device holds, because each leaves its sums (16 dim bytes with all
// parts), and rows enough for each that they stay small beside the rows it reads.  8,001 x
// 4,096 gated bf16 rows: 125 us and 9 for the join with 512 workgroups, 146 and 17 with 1,024;
// 786,432 x 172: 311 and 6 with 1,024, 315 and 10 with 2,048, with 512 twice the time.
int64_t res_blocks(int64_t rows, int64_t dim, int dtype) {
  const int64_t per = std::max<int64_t>(1, 2048 / std::max<int64_t>(dim, 1)) * 4;
  const int64_t lanes = ops_cdiv(dim * elem_bytes(dtype), 16);
  const int64_t most = lanes <= 256 ? 1024 : lanes <= 512 ? 512 : 256;
  return std::clamp<int64_t>(ops_cdiv(rows, per), 1, most);
}

}  // namespace
}  // namespace tgx

using namespace tgx;

extern "C" size_t tgx_residual_norm_grad_workspace_size(const tgx_residual_norm_args* args) {
  if (check_resnorm("tgx_residual_norm_grad", args, true) || args->rows == 0) return 0;
  return static_cast<size_t>(res_blocks(args->rows, args->dim, args->dtype)) * sums_of(has_parts(args)) * args->dim * 4;
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
  const int64_t blocks = args->rows > 0 ? res_blocks(args->rows, args->dim, args->dtype) : 0;
  if (blocks > 0 && (sums || a.dx != nullptr || a.dres != nullptr || a.dgate != nullptr)) {
    const int rc = by_type(args->dtype, [&](auto t) {
      using T = decltype(t);
      return by_type(args->wdtype, [&](auto wt) {
        using W = decltype(wt);
        return res_shape<T>(args->dim, [&](auto v, auto l, auto c) {
          constexpr int V = decltype(v)::value, L = decltype(l)::value, C = decltype(c)::value;
          const dim3 grid(static_cast<unsigned>(blocks)), block(res_threads(L));
          auto launch = [&](auto kind) {
            hipLaunchKernelGGL((resnorm_bwd<T, W, V, L, C, decltype(kind)::value>), grid, block, 0, s, a);
            return check_launch("resnorm_bwd");
          };
          if (!parts) return launch(std::integral_constant<int, 0>{});
          if (a.post == nullptr)
            return a.gate == nullptr ? launch(std::integral_constant<int, kScaled>{})
                                     : launch(std::integral_constant<int, kScaled | kGate>{});
          return a.gate == nullptr ? launch(std::integral_constant<int, kScaled | kPost>{})
                                   : launch(std::integral_constant<int, kScaled | kGate | kPost>{});
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
