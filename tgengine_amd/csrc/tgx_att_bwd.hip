// Attention backward on the matrix units.
//
// Three launches: delta_i = do_i . o_i and the log sum of every row; dk and dv, where a wave owns 32
// keys and walks over the problem's rows; dq, where a wave owns 32 rows and walks over
// the keys.  Scores are computed anew in both from the saved log sums (7 products of
// M x Lk x D, the sums of each output in one place and in one order, no atomics).
//
// As in the forward pass every score tile stays in the registers it was computed in: a
// wave's columns are what it owns (keys for dk and dv, rows for dq), a lane's 16 values
// run along the axis that the next product sums over, and that product's first operand
// comes transposed out of LDS.  p and ds are rounded to the inputs' type for those
// products, sums stay in 32 bits.
#include "tgx_attention.h"

namespace tgx {
namespace {

constexpr int kDeltaLanes = 16;

// Per row, in the order of problems and their rows: its log sum in units of log 2 (+inf
// for a row that keeps no key: its probabilities are then zeros) and delta
template <typename T>
__global__ __launch_bounds__(256) void att_stats(const T* __restrict__ out, const T* __restrict__ dout,
                                                 const float* __restrict__ lse, int64_t rows, int64_t lq, int heads,
                                                 int group, int dim, float2* __restrict__ stats) {
  constexpr int V = kWide<T>;
  const int lane = threadIdx.x % kDeltaLanes;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (256 / kDeltaLanes) + threadIdx.x / kDeltaLanes;
  const int64_t at = (row < rows ? row : 0) * dim;
  float s = 0.f;
  for (int c = lane * V; c < dim; c += kDeltaLanes * V) {
    const Pack<T, V> x = __builtin_bit_cast(Pack<T, V>, row_values(out + at, c, dim));
    const Pack<T, V> y = __builtin_bit_cast(Pack<T, V>, row_values(dout + at, c, dim));
#pragma unroll
    for (int u = 0; u < V; ++u) s += to_f(x.v[u]) * to_f(y.v[u]);
  }
  s = group_sum<kDeltaLanes>(s);
  if (lane != 0 || row >= rows) return;
  const int head = static_cast<int>(row % heads);
  const int64_t tok = row / heads % lq, b = row / heads / lq;
  const int64_t to = ((b * (heads / group) + head / group) * lq + tok) * group + head % group;
  const float x = lse[row];
  stats[to] = make_float2(x == -INFINITY ? INFINITY : x * kLog2e, s);
}

// 32 columns of a product with 4 values of a row in a lane, to rows of `dim` values
template <typename T, int DP>
__device__ __forceinline__ void store_columns(T* row, const f32x16 (&x)[DP / 32], float by, int dim) {
  const int h = (threadIdx.x & (kWave - 1)) / 32;
#pragma unroll
  for (int t = 0; t < DP / 32; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = t * 32 + mma_row(4 * j, h);
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

// dk and dv (WHAT: 1 = dv, 2 = dk, 3 = both) of 32 W keys.  S = Q K^T and dP = dO V^T
// have the rows down a lane's registers and one key a lane; dV^T += dO^T P and
// dK^T += Q^T dS follow.
template <typename T, bool TINY, int DP, int W, int WHAT>
__global__ __launch_bounds__(64 * W, DP > 64 ? 1 : 2) void att_mma_kv(const AttArgs a, int ktiles,
                                                                      const float2* __restrict__ stats) {
  constexpr int NT = 64 * W, V = kWide<T>, ST = DP + 16 / static_cast<int>(sizeof(T)), R = 32;
  constexpr bool DV = (WHAT & 1) != 0, DK = (WHAT & 2) != 0;
  __shared__ __align__(16) T sq[R * ST], sg[R * ST];
  __shared__ __align__(16) float slse[R], sdelta[R];
  const int lane = threadIdx.x & (kWave - 1), h = lane / 32, wave = threadIdx.x / kWave;
  const int64_t w = by_die(blockIdx.x, gridDim.x);
  const int64_t j = w % ktiles * (32 * W) + wave * 32 + (lane & 31);
  const int64_t p = w / ktiles;
  const int hk = static_cast<int>(p % a.kv_heads);
  const int64_t b = p / a.kv_heads;
  const bool kept = j < a.lk && (a.mask == nullptr || a.mask[b * a.mask_stride + j] != 0);
  const int64_t at = (b * a.lk + j) * a.kv_heads + hk;
  f32x16 dk[DK ? DP / 32 : 1], dv[DV ? DP / 32 : 1];
#pragma unroll
  for (int t = 0; t < DP / 32; ++t) {
    if constexpr (DK) dk[t] = f32x16{};
    if constexpr (DV) dv[t] = f32x16{};
  }
  if (__syncthreads_or(kept)) {
    const bool all = __all(kept);
    u32x4 kf[DP / kStep<T>], vf[DK ? DP / kStep<T> : 1];
    row_frags<T, TINY, DP>(kf, kept ? static_cast<const T*>(a.k) + b * a.ks[0] + j * a.ks[1] + hk * a.ks[2] : nullptr, a.dim);
    if constexpr (DK)
      row_frags<T, TINY, DP>(vf, kept ? static_cast<const T*>(a.v) + b * a.vs[0] + j * a.vs[1] + hk * a.vs[2] : nullptr,
                       a.dim);
    const float c = a.scale * kLog2e;
    const int64_t rows = a.lq * a.group;
    const T* qp = static_cast<const T*>(a.q) + b * a.qs[0] + static_cast<int64_t>(hk) * a.group * a.qs[2];
    const T* gp = static_cast<const T*>(a.dout) + b * a.os[0] + static_cast<int64_t>(hk) * a.group * a.os[2];
    stats += p * rows;
    Stage<T, TINY, R, DP, NT, ST> q(a.dim), g(a.dim);
    constexpr int N = Stage<T, TINY, R, DP, NT, ST>::N, STEP = Stage<T, TINY, R, DP, NT, ST>::STEP;
    // each of the thread's rows: its head of the group and its offsets, moved on by R rows
    // a tile without a division
    int hg[N];
    int64_t qo[N], go[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int row = q.row0 + n * STEP, tok = row / a.group;
      hg[n] = row - tok * a.group;
      qo[n] = tok * a.qs[1] + hg[n] * a.qs[2];
      go[n] = tok * a.os[1] + hg[n] * a.os[2];
    }
    const int dt = R / a.group, dh = R % a.group;
    float2 st = make_float2(INFINITY, 0.f);
    auto fetch = [&](int64_t first) {
      q.load(a.dim, [&](int n) { return first + q.row0 + n * STEP < rows ? qp + qo[n] : nullptr; });
      g.load(a.dim, [&](int n) { return first + q.row0 + n * STEP < rows ? gp + go[n] : nullptr; });
      if (threadIdx.x < R) st = first + threadIdx.x < rows ? stats[first + threadIdx.x] : make_float2(INFINITY, 0.f);
#pragma unroll
      for (int n = 0; n < N; ++n) {
        hg[n] += dh;
        qo[n] += dt * a.qs[1] + dh * a.qs[2];
        go[n] += dt * a.os[1] + dh * a.os[2];
        if (hg[n] >= a.group) {
          hg[n] -= a.group;
          qo[n] += a.qs[1] - a.group * a.qs[2];
          go[n] += a.os[1] - a.group * a.os[2];
        }
      }
    };
    fetch(0);
    for (int64_t first = 0; first < rows; first += R) {
      __syncthreads();
      q.store(sq, a.dim);
      g.store(sg, a.dim);
      if (threadIdx.x < R) {
        slse[threadIdx.x] = st.x;
        sdelta[threadIdx.x] = st.y;
      }
      __syncthreads();
      if (first + R < rows) fetch(first + R);
      f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
      for (int e = 0; e < DP / kStep<T>; ++e) {
        s = mma<T>(s, *reinterpret_cast<const u32x4*>(sq + (lane & 31) * ST + e * kStep<T> + h * V), kf[e]);
        if constexpr (DK)
          dp = mma<T>(dp, *reinterpret_cast<const u32x4*>(sg + (lane & 31) * ST + e * kStep<T> + h * V), vf[e]);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = mma_row(i, h);
        s[i] = exp2_(fmaf(s[i], c, -slse[r]));
        if (!all) s[i] = kept ? s[i] : 0.f;
        if constexpr (DK) dp[i] = s[i] * (dp[i] - sdelta[r]);
      }
#pragma unroll
      for (int f = 0; f < 16 / V; ++f) {
        const u32x4 pf = to_frag<T>(s, f);
        u32x4 df;
        if constexpr (DK) df = to_frag<T>(dp, f);
#pragma unroll
        for (int t = 0; t < DP / 32; ++t) {
          if constexpr (DV) dv[t] = mma<T>(dv[t], transposed(sg, ST, 0, f, t * 32), pf);
          if constexpr (DK) dk[t] = mma<T>(dk[t], transposed(sq, ST, 0, f, t * 32), df);
        }
      }
    }
  }
  if (j >= a.lk) return;
  if constexpr (DK)
    if (a.dk != nullptr) store_columns<T, DP>(static_cast<T*>(a.dk) + at * a.dim, dk, a.scale, a.dim);
  if constexpr (DV)
    if (a.dv != nullptr) store_columns<T, DP>(static_cast<T*>(a.dv) + at * a.dim, dv, 1.f, a.dim);
}

// dq of 32 W rows.  S^T = K Q^T and dP^T = V dO^T have the keys down a lane's registers
// and one row a lane; dQ^T += K^T dS^T follows.
template <typename T, bool TINY, int DP, int W>
__global__ __launch_bounds__(64 * W, DP > 128 ? 1 : 2) void att_mma_q(const AttArgs a, int mtiles,
                                                                     const float2* __restrict__ stats) {
  constexpr int NT = 64 * W, V = kWide<T>, ST = DP + 16 / static_cast<int>(sizeof(T)), KT = 32;
  __shared__ __align__(16) T sk[KT * ST], sv[KT * ST];
  const int lane = threadIdx.x & (kWave - 1), h = lane / 32, wave = threadIdx.x / kWave;
  const int64_t w = by_die(blockIdx.x, gridDim.x);
  const int64_t r = w % mtiles * (32 * W) + wave * 32 + (lane & 31);
  const int64_t p = w / mtiles;
  const int hk = static_cast<int>(p % a.kv_heads);
  const int64_t b = p / a.kv_heads;
  const int64_t rows = a.lq * a.group, tok = r < rows ? r / a.group : 0;
  const int head = hk * a.group + static_cast<int>(r - tok * a.group);
  const int64_t row = (b * a.lq + tok) * a.heads + head;
  const T* kp = static_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[2];
  const T* vp = static_cast<const T*>(a.v) + b * a.vs[0] + hk * a.vs[2];
  u32x4 qf[DP / kStep<T>], gf[DP / kStep<T>];
  row_frags<T, TINY, DP>(qf, r < rows ? static_cast<const T*>(a.q) + b * a.qs[0] + tok * a.qs[1] + head * a.qs[2] : nullptr,
                   a.dim);
  row_frags<T, TINY, DP>(gf, r < rows ? static_cast<const T*>(a.dout) + row * a.dim : nullptr, a.dim);
  const float2 st = r < rows ? stats[p * rows + r] : make_float2(INFINITY, 0.f);
  const float c = a.scale * kLog2e;
  f32x16 dq[DP / 32];
#pragma unroll
  for (int t = 0; t < DP / 32; ++t) dq[t] = f32x16{};

  Keys<KT> keys(a.mask == nullptr ? nullptr : a.mask + b * a.mask_stride, 0, a.lk);
  int64_t key;
  uint64_t bits;
  bool more = keys.next(key, bits);
  Stage<T, TINY, KT, DP, NT, ST> k(a.dim), v(a.dim);
  auto fetch = [&]() {
    k.load(kp + key * a.ks[1], a.ks[1], bits, a.dim);
    v.load(vp + key * a.vs[1], a.vs[1], bits, a.dim);
  };
  if (more) fetch();
  while (more) {  // workgroup-uniform
    __syncthreads();
    k.store(sk, a.dim);
    v.store(sv, a.dim);
    __syncthreads();
    const uint32_t now = static_cast<uint32_t>(bits), kept = now >> (4 * h);
    more = keys.next(key, bits);
    if (more) fetch();
    f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
    for (int e = 0; e < DP / kStep<T>; ++e) {
      s = mma<T>(s, *reinterpret_cast<const u32x4*>(sk + (lane & 31) * ST + e * kStep<T> + h * V), qf[e]);
      dp = mma<T>(dp, *reinterpret_cast<const u32x4*>(sv + (lane & 31) * ST + e * kStep<T> + h * V), gf[e]);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      dp[i] = exp2_(fmaf(s[i], c, -st.x)) * (dp[i] - st.y);
      if (now != ~0u) dp[i] = kept >> mma_row(i, 0) & 1 ? dp[i] : 0.f;
    }
#pragma unroll
    for (int f = 0; f < 16 / V; ++f) {
      const u32x4 df = to_frag<T>(dp, f);
#pragma unroll
      for (int t = 0; t < DP / 32; ++t) {
        dq[t] = mma<T>(dq[t], transposed(sk, ST, 0, f, t * 32), df);
      }
    }
  }
  if (r >= rows) return;
  store_columns<T, DP>(static_cast<T*>(a.dq) + row * a.dim, dq, a.scale, a.dim);
}

int waves_for(int64_t n) { return n <= 64 ? 2 : 4; }

}  // namespace

size_t att_mma_backward_workspace(const AttArgs& a, int dtype) {
  (void)dtype;
  return ops_align(static_cast<size_t>(a.batch * a.lq * a.heads) * sizeof(float2));
}

int att_mma_backward(const AttArgs& a, int dtype, void* ws, hipStream_t s) {
  const int64_t rows = a.batch * a.lq * a.heads;
  float2* stats = static_cast<float2*>(ws);
  return by_head(dtype, a.dim, [&](auto t, auto dp, auto tiny) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value;
    constexpr bool TINY = decltype(tiny)::value;
    hipLaunchKernelGGL(att_stats<T>, dim3(static_cast<unsigned>(ops_cdiv(rows, 256 / kDeltaLanes))), dim3(256), 0, s,
                       static_cast<const T*>(a.out), static_cast<const T*>(a.dout), a.lse, rows, a.lq, a.heads, a.group,
                       a.dim, stats);
    int rc = check_launch("att_stats");
    if (rc) return rc;
    if (a.lk > 0 && (a.dk != nullptr || a.dv != nullptr)) {
      auto go = [&](auto w, auto what) {
        constexpr int W = decltype(w)::value, WHAT = decltype(what)::value;
        const int ktiles = static_cast<int>(ops_cdiv(a.lk, 32 * W));
        hipLaunchKernelGGL((att_mma_kv<T, TINY, DP, W, WHAT>), dim3(static_cast<unsigned>(a.batch * a.kv_heads * ktiles)),
                           dim3(64 * W), 0, s, a, ktiles, stats);
        return check_launch("att_mma_kv");
      };
      auto by_waves = [&](auto what) {
        if (waves_for(a.lk) == 2) return go(std::integral_constant<int, 2>{}, what);
        return go(std::integral_constant<int, 4>{}, what);
      };
      // both sums and both operands of one wave exceed the registers for wide f32 heads
      if constexpr (sizeof(T) == 2 || DP <= 128) {
        rc = by_waves(std::integral_constant<int, 3>{});
      } else {
        if (a.dv != nullptr) rc = by_waves(std::integral_constant<int, 1>{});
        if (rc == TGX_OK && a.dk != nullptr) rc = by_waves(std::integral_constant<int, 2>{});
      }
      if (rc) return rc;
    }
    if (a.dq != nullptr) {
      auto go = [&](auto w) {
        constexpr int W = decltype(w)::value;
        const int mtiles = static_cast<int>(ops_cdiv(a.lq * a.group, 32 * W));
        hipLaunchKernelGGL((att_mma_q<T, TINY, DP, W>), dim3(static_cast<unsigned>(a.batch * a.kv_heads * mtiles)),
                           dim3(64 * W), 0, s, a, mtiles, stats);
        return check_launch("att_mma_q");
      };
      if (waves_for(a.lq * a.group) == 2) return go(std::integral_constant<int, 2>{});
      return go(std::integral_constant<int, 4>{});
    }
    return TGX_OK;
  });
}

}  // namespace tgx
