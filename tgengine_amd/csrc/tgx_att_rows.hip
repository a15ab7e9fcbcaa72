// Attention of a few rows a problem (at most 4: one or two query tokens, or the heads
// that share a key/value head), forward and backward, without matrix units: every key
// and value is used for 2 or 4 products a row only, and the reads decide.
//
// LP lanes share a key, each holding C packs of its row, so that a wave works on 64 / LP
// keys at a time and U of them deep: all their reads are in flight together.  Each group
// of LP lanes keeps a running maximum, sum and output of its own; groups, then the
// `wpp` waves of a problem, are joined once at the end.  The backward pass reads the
// keys once too: dk and dv of a key are complete as soon as its scores are.
//
// HBM bounds both: 24,576 rows with 32 keys, 2 f32 heads of 86, 80% kept: forward 198 us for
// 0.90 GB, 4.5 TB/s; backward 388 us for 2.0 GB, 5.2 TB/s.
#include "tgx_attention.h"

namespace tgx {
namespace {

constexpr int kRowThreads = 256;
constexpr int kRowWaves = kRowThreads / kWave;

// A lane's C packs of rows of `dim` values, the j-th from column col(j) on.  The row's last
// pack, which is some lane's last, ends with the row and may overlap the one before: both
// lanes then come to the same values there, and a dot product takes them from one (own()).
// TINY: rows of fewer than V values, read and written one by one.
template <typename T, bool TINY, int LP, int C>
struct Lanes {
  static constexpr int V = kWide<T>, N = C * V;
  int gl, dim, last;  // last: column of the last pack
  bool on;            // the last pack is within the row
  __device__ explicit Lanes(int dim_) : gl(threadIdx.x & (LP - 1)), dim(dim_) {
    last = ((C - 1) * LP + gl) * V;
    on = last < dim;
    if (!TINY) last = min(last, dim - V);
  }
  __device__ __forceinline__ int col(int j) const { return j == C - 1 ? last : (j * LP + gl) * V; }
  __device__ __forceinline__ bool has(int j) const { return j < C - 1 || on; }
  __device__ __forceinline__ void read(u32x4 (&x)[C], const T* row) const {
#pragma unroll
    for (int j = 0; j < C; ++j) {
      x[j] = u32x4{0, 0, 0, 0};
      if (row == nullptr || !has(j)) continue;
      if constexpr (TINY) x[j] = row_part<T, true>(row, col(j), dim);
      else x[j] = load16(row + col(j));
    }
  }
  __device__ __forceinline__ static void values(float (&f)[N], const u32x4 (&x)[C]) {
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const Pack<T, V> p = __builtin_bit_cast(Pack<T, V>, x[j]);
#pragma unroll
      for (int u = 0; u < V; ++u) f[j * V + u] = to_f(p.v[u]);
    }
  }
  __device__ __forceinline__ void load(float (&f)[N], const T* row) const {
    u32x4 x[C];
    read(x, row);
    values(f, x);
  }
  // the last pack without what the lane before has too
  __device__ __forceinline__ void own(float (&z)[V], const float (&f)[N]) const {
    const int twice = TINY ? 0 : ((C - 1) * LP + gl) * V - last;
#pragma unroll
    for (int u = 0; u < V; ++u) z[u] = u >= twice ? f[(C - 1) * V + u] : 0.f;
  }
  __device__ __forceinline__ static float dot(const float (&q)[N], const float (&z)[V], const float (&f)[N]) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N - V; ++i) s = fmaf(q[i], f[i], s);
#pragma unroll
    for (int u = 0; u < V; ++u) s = fmaf(z[u], f[N - V + u], s);
    return group_sum<LP>(s);
  }
  // kept: ~0, or 0 to store zeros in the values' place
  template <typename U>
  __device__ __forceinline__ void store(U* row, const float (&f)[N], uint32_t kept = ~0u) const {
#pragma unroll
    for (int j = 0; j < C; ++j) {
      if (!has(j)) continue;
      Pack<U, V> p;
#pragma unroll
      for (int u = 0; u < V; ++u) p.v[u] = from_f<U>(f[j * V + u]);
      if constexpr (sizeof(p) == 16) p = __builtin_bit_cast(decltype(p), __builtin_bit_cast(u32x4, p) & kept);
      if constexpr (!TINY) {
        store_pack<U, V>(row + col(j), p);
      } else {
#pragma unroll
        for (int u = 0; u < V; ++u)
          if (col(j) + u < dim) row[col(j) + u] = p.v[u];
      }
    }
  }
};

// What a wave works on: problem (b, hk), keys [lo, hi) in tiles of 64 from lo + 64 part on,
// every wpp-th
struct RowUnit {
  int64_t b, lo, hi;
  int hk, sp, part;
  bool live;
  __device__ RowUnit(const AttArgs& a, int wpp, int splits, int64_t span) {
    const int wave = threadIdx.x / kWave;
    int64_t unit = static_cast<int64_t>(blockIdx.x) * (kRowWaves / wpp) + wave / wpp;
    part = wave % wpp;
    live = unit < a.batch * a.kv_heads * splits;
    if (!live) unit = 0;
    sp = static_cast<int>(unit % splits);
    unit /= splits;
    hk = static_cast<int>(unit % a.kv_heads);
    b = unit / a.kv_heads;
    lo = sp * span;
    hi = lo + span < a.lk ? lo + span : a.lk;
  }
  __device__ uint64_t kept(const AttArgs& a, int64_t at) const {
    const int64_t j = at + (threadIdx.x & (kWave - 1));
    return __ballot(j < hi && (a.mask == nullptr || a.mask[b * a.mask_stride + j] != 0));
  }
};

template <typename T, bool TINY, int LP, int C, int M>
__global__ __launch_bounds__(kRowThreads, M == 1 && C < 4 ? 3 : 2) void att_rows_fwd(const AttArgs a, int wpp, int splits, int64_t span,
                                                            const AttParts part) {
  constexpr int V = kWide<T>, N = C * V, G = kWave / LP, U = M == 1 ? 4 : 2;
  __shared__ float join[kRowWaves][M][LP * N + 2];
  const int lane = threadIdx.x & (kWave - 1), grp = lane / LP, wave = threadIdx.x / kWave;
  const RowUnit w(a, wpp, splits, span);
  if (!w.live) return;  // wpp = 1 only: no barrier follows
  const Lanes<T, TINY, LP, C> at(a.dim);
  const int rows = static_cast<int>(a.lq) * a.group;
  const T* kp = static_cast<const T*>(a.k) + w.b * a.ks[0] + w.hk * a.ks[2];
  const T* vp = static_cast<const T*>(a.v) + w.b * a.vs[0] + w.hk * a.vs[2];
  float q[M][N], qo[M][V], acc[M][N], m[M], l[M];
#pragma unroll
  for (int r = 0; r < M; ++r) {
    const int i = r / a.group, head = w.hk * a.group + r % a.group;
    at.load(q[r], r < rows ? static_cast<const T*>(a.q) + w.b * a.qs[0] + i * a.qs[1] + head * a.qs[2] : nullptr);
    at.own(qo[r], q[r]);
#pragma unroll
    for (int x = 0; x < N; ++x) acc[r][x] = 0.f;
    m[r] = -INFINITY;
    l[r] = 0.f;
  }
  const float c = a.scale * kLog2e;
  for (int64_t t = w.lo + w.part * 64; t < w.hi; t += wpp * 64) {  // wave-uniform
    const uint64_t bits = w.kept(a, t);
#pragma unroll 1
    for (int k0 = 0; k0 < 64; k0 += G * U) {
      const uint64_t here = G * U == 64 ? bits : bits >> k0 & ((uint64_t(1) << (G * U % 64)) - 1);
      if (here == 0) continue;
      u32x4 kx[U][C], vx[U][C];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = u * G + grp;
        at.read(kx[u], here >> j & 1 ? kp + (t + k0 + j) * a.ks[1] : nullptr);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = u * G + grp;
        at.read(vx[u], here >> j & 1 ? vp + (t + k0 + j) * a.vs[1] : nullptr);
      }
      float s[M][U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f[N];
        at.values(f, kx[u]);
#pragma unroll
        for (int r = 0; r < M; ++r) {
          const float x = at.dot(q[r], qo[r], f) * c;
          s[r][u] = here >> (u * G + grp) & 1 ? x : -INFINITY;
        }
      }
#pragma unroll
      for (int r = 0; r < M; ++r) {
        float top = m[r];
#pragma unroll
        for (int u = 0; u < U; ++u) top = fmaxf(top, s[r][u]);
        const float from = top == -INFINITY ? 0.f : top, old = exp2_(m[r] - from);
        m[r] = top;
        l[r] *= old;
#pragma unroll
        for (int x = 0; x < N; ++x) acc[r][x] *= old;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          s[r][u] = exp2_(s[r][u] - from);
          l[r] += s[r][u];
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f[N];
        at.values(f, vx[u]);
#pragma unroll
        for (int r = 0; r < M; ++r)
#pragma unroll
          for (int x = 0; x < N; ++x) acc[r][x] = fmaf(s[r][u], f[x], acc[r][x]);
      }
    }
  }
  // the groups' parts, then the waves'
#pragma unroll
  for (int r = 0; r < M; ++r) {
    float top = m[r];
#pragma unroll
    for (int off = LP; off < kWave; off <<= 1) top = fmaxf(top, __shfl_xor(top, off, kWave));
    const float old = exp2_(m[r] - (top == -INFINITY ? 0.f : top));
    m[r] = top;
    l[r] *= old;
#pragma unroll
    for (int x = 0; x < N; ++x) acc[r][x] *= old;
#pragma unroll
    for (int off = LP; off < kWave; off <<= 1) {
      l[r] += __shfl_xor(l[r], off, kWave);
#pragma unroll
      for (int x = 0; x < N; ++x) acc[r][x] += __shfl_xor(acc[r][x], off, kWave);
    }
  }
  if (wpp > 1) {
    if (grp == 0) {
#pragma unroll
      for (int r = 0; r < M; ++r) {
#pragma unroll
        for (int x = 0; x < N; ++x) join[wave][r][x * LP + at.gl] = acc[r][x];
        if (at.gl == 0) {
          join[wave][r][LP * N] = m[r];
          join[wave][r][LP * N + 1] = l[r];
        }
      }
    }
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int r = 0; r < M; ++r) {
      float top = m[r];
      for (int y = 1; y < wpp; ++y) top = fmaxf(top, join[y][r][LP * N]);
      const float from = top == -INFINITY ? 0.f : top, old = exp2_(m[r] - from);
      l[r] *= old;
#pragma unroll
      for (int x = 0; x < N; ++x) acc[r][x] *= old;
      for (int y = 1; y < wpp; ++y) {
        const float by = exp2_(join[y][r][LP * N] - from);
        l[r] += join[y][r][LP * N + 1] * by;
#pragma unroll
        for (int x = 0; x < N; ++x) acc[r][x] += join[y][r][x * LP + at.gl] * by;
      }
      m[r] = top;
    }
  }
#pragma unroll
  for (int r = 0; r < M; ++r) {
    if (r >= rows || grp != r % G) continue;
    const int i = r / a.group, head = w.hk * a.group + r % a.group;
    const int64_t row = (w.b * a.lq + i) * a.heads + head;
    if (splits > 1) {
      float* out = part.o + (row * splits + w.sp) * a.dim;
      if (at.gl == 0) part.ml[row * splits + w.sp] = make_float2(m[r], l[r]);
      at.store(out, acc[r]);
      continue;
    }
    const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];
#pragma unroll
    for (int x = 0; x < N; ++x) acc[r][x] *= inv;
    at.store(static_cast<T*>(a.o) + row * a.dim, acc[r]);
    if (sizeof(T) == 2 && a.rest != nullptr) {
      float z[N];
#pragma unroll
      for (int x = 0; x < N; ++x) z[x] = lost<T>(acc[r][x]);
      at.store(static_cast<T*>(a.rest) + row * a.dim, z);
    }
    if (at.gl == 0 && a.lse != nullptr) a.lse[row] = log_sum(m[r], l[r]);
  }
}

template <typename T, bool TINY, int LP, int C, int M>
__global__ __launch_bounds__(kRowThreads, M == 1 ? (C < 4 ? 3 : 2) : (C < 4 ? 2 : 1)) void att_rows_bwd(const AttArgs a, int wpp, int splits, int64_t span,
                                                            float* __restrict__ part) {
  constexpr int V = kWide<T>, N = C * V, G = kWave / LP, U = M == 1 ? 2 : 1;
  __shared__ float join[kRowWaves][M][LP * N];
  const int lane = threadIdx.x & (kWave - 1), grp = lane / LP, wave = threadIdx.x / kWave;
  const RowUnit w(a, wpp, splits, span);
  if (!w.live) return;  // wpp = 1 only: no barrier follows
  const Lanes<T, TINY, LP, C> at(a.dim);
  const int rows = static_cast<int>(a.lq) * a.group;
  const T* kp = static_cast<const T*>(a.k) + w.b * a.ks[0] + w.hk * a.ks[2];
  const T* vp = static_cast<const T*>(a.v) + w.b * a.vs[0] + w.hk * a.vs[2];
  const int64_t key0 = w.b * a.lk * a.kv_heads + w.hk;
  float q[M][N], g[M][N], qo[M][V], go[M][V], dq[M][N], lse[M], delta[M];
#pragma unroll
  for (int r = 0; r < M; ++r) {
    const bool in = r < rows;
    const int i = r / a.group, head = w.hk * a.group + r % a.group;
    const int64_t row = (w.b * a.lq + i) * a.heads + head;
    float o[N];
    at.load(q[r], in ? static_cast<const T*>(a.q) + w.b * a.qs[0] + i * a.qs[1] + head * a.qs[2] : nullptr);
    at.load(g[r], in ? static_cast<const T*>(a.dout) + row * a.dim : nullptr);
    at.load(o, in ? static_cast<const T*>(a.out) + row * a.dim : nullptr);
    at.own(qo[r], q[r]);
    at.own(go[r], g[r]);
    delta[r] = at.dot(g[r], go[r], o);
    if (sizeof(T) == 2 && a.rest != nullptr) {
      at.load(o, in ? static_cast<const T*>(a.rest) + row * a.dim : nullptr);
      delta[r] += at.dot(g[r], go[r], o);
    }
    lse[r] = in ? a.lse[row] * kLog2e : INFINITY;
    if (lse[r] == -INFINITY) lse[r] = INFINITY;  // no key kept: p = 0
#pragma unroll
    for (int x = 0; x < N; ++x) dq[r][x] = 0.f;
  }
  const float c = a.scale * kLog2e;
  for (int64_t t = w.lo + w.part * 64; t < w.hi; t += wpp * 64) {  // wave-uniform
    const uint64_t bits = w.kept(a, t);
#pragma unroll 1
    for (int k0 = 0; k0 < 64 && t + k0 < w.hi; k0 += G * U) {
      u32x4 kx[U][C], vx[U][C];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = k0 + u * G + grp;
        at.read(kx[u], bits >> j & 1 ? kp + (t + j) * a.ks[1] : nullptr);
        at.read(vx[u], bits >> j & 1 ? vp + (t + j) * a.vs[1] : nullptr);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = k0 + u * G + grp;
        const bool on = bits >> j & 1;
        float f[N], y[N], dk[N], dv[N];
        at.values(f, kx[u]);
        at.values(y, vx[u]);
#pragma unroll
        for (int x = 0; x < N; ++x) dk[x] = dv[x] = 0.f;
#pragma unroll
        for (int r = 0; r < M; ++r) {
          const float s = at.dot(q[r], qo[r], f) * c, dp = at.dot(g[r], go[r], y);
          const float p = exp2_(s - lse[r]);
          const float ds = on ? p * (dp - delta[r]) * a.scale : 0.f;
#pragma unroll
          for (int x = 0; x < N; ++x) {
            dq[r][x] = fmaf(ds, f[x], dq[r][x]);
            dk[x] = fmaf(ds, q[r][x], dk[x]);
            dv[x] = fmaf(p, g[r][x], dv[x]);
          }
        }
        if (t + j < w.hi) {
          // whatever the rows hold (a gradient of NaN, say), a masked key takes none of it
          const uint32_t bits_kept = on ? ~0u : 0u;
          const int64_t to = (key0 + (t + j) * a.kv_heads) * a.dim;
          if (a.dk != nullptr) at.store(static_cast<T*>(a.dk) + to, dk, bits_kept);
          if (a.dv != nullptr) at.store(static_cast<T*>(a.dv) + to, dv, bits_kept);
        }
      }
    }
  }
  if (a.dq == nullptr) return;
#pragma unroll
  for (int r = 0; r < M; ++r)
#pragma unroll
    for (int off = LP; off < kWave; off <<= 1)
#pragma unroll
      for (int x = 0; x < N; ++x) dq[r][x] += __shfl_xor(dq[r][x], off, kWave);
  if (wpp > 1) {
    if (grp == 0) {
#pragma unroll
      for (int r = 0; r < M; ++r)
#pragma unroll
        for (int x = 0; x < N; ++x) join[wave][r][x * LP + at.gl] = dq[r][x];
    }
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int r = 0; r < M; ++r)
      for (int y = 1; y < wpp; ++y)
#pragma unroll
        for (int x = 0; x < N; ++x) dq[r][x] += join[y][r][x * LP + at.gl];
  }
#pragma unroll
  for (int r = 0; r < M; ++r) {
    if (r >= rows || grp != r % G) continue;
    const int64_t row = (w.b * a.lq + r / a.group) * a.heads + w.hk * a.group + r % a.group;
    if (splits == 1) {
      at.store(static_cast<T*>(a.dq) + row * a.dim, dq[r]);
      continue;
    }
    at.store(part + (row * splits + w.sp) * a.dim, dq[r]);
  }
}

// Waves per problem and key ranges: one wave a problem where the problems fill the
// device, four where they do not, and then ranges of at least 512 keys (f32, 2 heads of 64:
// 300 rows with 200 keys forward 13 us, 16 with one wave each, backward 23 and 26; from
// 1,000 rows on the two are even.  bf16, 4 rows with 4,000 keys forward 14 us, 39 in one
// range, backward 21 and 66).
struct RowShape {
  int wpp, splits;
  int64_t span, blocks;
  explicit RowShape(const AttArgs& a) {
    const int64_t problems = a.batch * a.kv_heads, tiles = ops_cdiv(std::max<int64_t>(a.lk, 1), 64);
    wpp = problems >= 4096 || tiles == 1 ? 1 : kRowWaves;
    const int64_t want = problems >= 512 ? 1 : ops_cdiv(1024, std::max<int64_t>(problems, 1));
    const int64_t per = ops_cdiv(tiles, std::clamp<int64_t>(std::min(want, tiles / 8), 1, 256));
    span = per * 64;
    splits = static_cast<int>(ops_cdiv(tiles, per));
    blocks = ops_cdiv(problems * splits, kRowWaves / wpp);
  }
};

// calls f(T{}, TINY, LP, C, M) with the lanes and packs that a head of `dim` values takes
template <typename F>
int by_lanes(int dtype, int dim, int64_t rows, F&& f) {
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto with = [&](auto lp, auto c, auto tiny) {
      if (rows == 1) return f(t, tiny, lp, c, std::integral_constant<int, 1>{});
      return f(t, tiny, lp, c, std::integral_constant<int, kMostRows>{});
    };
    const int packs = static_cast<int>(ops_cdiv(dim, kWide<T>));
#define TGX_LANES(LP, C) with(std::integral_constant<int, LP>{}, std::integral_constant<int, C>{}, std::false_type{})
    if (dim < kWide<T>) return with(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{}, std::true_type{});
    if (packs <= 8) return TGX_LANES(8, 1);
    if constexpr (sizeof(T) == 4) {
      if (packs <= 16) return TGX_LANES(8, 2);
      if (packs <= 24) return TGX_LANES(8, 3);
      if (packs <= 32) return TGX_LANES(8, 4);
      if (packs <= 48) return TGX_LANES(16, 3);
      return TGX_LANES(16, 4);
    } else {  // a pack is eight values: more lanes with fewer of them
      if (packs <= 16) return rows == 1 ? TGX_LANES(8, 2) : TGX_LANES(16, 1);
      return TGX_LANES(16, 2);
    }
#undef TGX_LANES
  });
}

}  // namespace

size_t att_rows_forward_workspace(const AttArgs& a) {
  return AttParts::bytes(a.batch * a.lq * a.heads, RowShape(a).splits, a.dim);
}

int att_rows_forward(const AttArgs& a, int dtype, void* ws, hipStream_t s) {
  const RowShape f(a);
  const AttParts part(ws, a.batch * a.lq * a.heads, f.splits);
  int rc = check_grid("tgx_attention", f.blocks, kRowThreads);
  if (rc) return rc;
  rc = by_lanes(dtype, a.dim, a.lq * a.group, [&](auto t, auto tiny, auto lp, auto c, auto m) {
    hipLaunchKernelGGL((att_rows_fwd<decltype(t), decltype(tiny)::value, decltype(lp)::value, decltype(c)::value,
                                     decltype(m)::value>),
                       dim3(static_cast<unsigned>(f.blocks)), dim3(kRowThreads), 0, s, a, f.wpp, f.splits, f.span, part);
    return check_launch("att_rows_fwd");
  });
  return rc || f.splits == 1 ? rc : att_join_forward(a, dtype, f.splits, part, s);
}

size_t att_rows_backward_workspace(const AttArgs& a) {
  const RowShape f(a);
  return f.splits > 1 ? static_cast<size_t>(a.batch * a.lq * a.heads) * f.splits * a.dim * 4 : 0;
}

int att_rows_backward(const AttArgs& a, int dtype, void* ws, hipStream_t s) {
  const RowShape f(a);
  float* part = static_cast<float*>(ws);
  int rc = check_grid("tgx_attention_grad", f.blocks, kRowThreads);
  if (rc) return rc;
  rc = by_lanes(dtype, a.dim, a.lq * a.group, [&](auto t, auto tiny, auto lp, auto c, auto m) {
    hipLaunchKernelGGL((att_rows_bwd<decltype(t), decltype(tiny)::value, decltype(lp)::value, decltype(c)::value,
                                     decltype(m)::value>),
                       dim3(static_cast<unsigned>(f.blocks)), dim3(kRowThreads), 0, s, a, f.wpp, f.splits, f.span, part);
    return check_launch("att_rows_bwd");
  });
  if (rc || f.splits == 1 || a.dq == nullptr) return rc;
  return att_join_sums(a.dq, a.batch * a.lq * a.heads, a.dim, dtype, 1.f, f.splits, part, s);
}

}  // namespace tgx
