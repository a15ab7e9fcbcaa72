// Attention forward on the matrix units, one pass over the keys.
//
// A wave owns 32 rows of a problem and keeps their queries as fragments.  A tile of
// keys gives S^T = K Q^T (keys down a lane's registers, one row a lane), so that the
// running maximum and sum of the softmax are a lane's own but for one exchange between
// the wave's halves now and then, and P^T, still in the same registers, is the second operand of
// O^T += V^T P^T.  Scores are in units of log 2.  Probabilities are rounded to the
// inputs' type for that product, as the matrix units take them; sums stay in 32 bits.
#include "tgx_attention.h"

namespace tgx {
namespace {

// Keys of a tile: K and V tiles take 2 KT (DP + pad) values of LDS
template <typename T, int WK>
constexpr int kKeys = (sizeof(T) == 2 || WK == 2) ? 64 : 32;

// WQ waves share the rows of a workgroup, 32 each; WK = 2: two waves take the same rows
// over half of each tile's keys and are joined at the end.  With splits > 1 the keys are
// cut in as many ranges of `span` keys and each leaves its maximum, sum and unscaled
// output in `part` for att_join.
template <typename T, bool TINY, int DP, int WQ, int WK>
__global__ __launch_bounds__(64 * WQ * WK, DP > 128 ? 1 : 2) void att_mma_fwd(const AttArgs a, int mtiles, int splits,
                                                                             int64_t span, float* __restrict__ part) {
  constexpr int NT = 64 * WQ * WK, KT = kKeys<T, WK>, SUB = KT / 32 / WK, V = kWide<T>;
  constexpr int KS = DP + 16 / static_cast<int>(sizeof(T)), VS = DP + (sizeof(T) == 2 ? 16 : 4);
  __shared__ __align__(16) T smem[KT * (KS + VS)];
  T* sk = smem;
  T* sv = smem + KT * KS;
  const int lane = threadIdx.x & (kWave - 1), h = lane / 32, wave = threadIdx.x / kWave;
  const int wq = wave / WK, wk = wave % WK;
  int64_t w = by_die(blockIdx.x, gridDim.x);
  const int sp = static_cast<int>(w % splits);
  w /= splits;
  const int64_t r0 = w % mtiles * (32 * WQ) + wq * 32;
  const int64_t p = w / mtiles;
  const int hk = static_cast<int>(p % a.kv_heads);
  const int64_t b = p / a.kv_heads;
  const int64_t rows = a.lq * a.group, r = r0 + (lane & 31);
  const int64_t tok = r < rows ? r / a.group : 0;
  const int head = hk * a.group + static_cast<int>(r - tok * a.group);
  const T* kp = static_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[2];
  const T* vp = static_cast<const T*>(a.v) + b * a.vs[0] + hk * a.vs[2];
  u32x4 qf[DP / kStep<T>];
  row_frags<T, TINY, DP>(qf, r < rows ? static_cast<const T*>(a.q) + b * a.qs[0] + tok * a.qs[1] + head * a.qs[2] : nullptr,
                   a.dim);
  // Scores are in units of 1 / c: the sign of the scale goes to the queries, so that the
  // largest score is the largest product, and a scale of zero makes them zero.
  const float c = a.scale == 0.f ? 1.f : fabsf(a.scale) * kLog2e;
  if (!(a.scale > 0.f))
#pragma unroll
    for (int e = 0; e < DP / kStep<T>; ++e)
#pragma unroll
      for (int u = 0; u < 4; ++u)
        qf[e][u] = a.scale == 0.f ? 0u : qf[e][u] ^ (sizeof(T) == 2 ? 0x80008000u : 0x80000000u);
  f32x16 o[DP / 32];
#pragma unroll
  for (int t = 0; t < DP / 32; ++t) o[t] = f32x16{};
  float m = -INFINITY, from = 0.f, l = 0.f;  // from: m, or 0 as long as no key was kept

  const int64_t lo = sp * span, hi = lo + span < a.lk ? lo + span : a.lk;
  Keys<KT> keys(a.mask == nullptr ? nullptr : a.mask + b * a.mask_stride, lo, hi);
  int64_t key;
  uint64_t bits;
  bool more = keys.next(key, bits);
  Stage<T, TINY, KT, DP, NT, KS> sk_(a.dim);
  Stage<T, TINY, KT, DP, NT, VS> sv_(a.dim);
  if (more) {
    sk_.load(kp + key * a.ks[1], a.ks[1], bits, a.dim);
    sk_.store(sk, a.dim);
  }
  __syncthreads();
  while (more) {  // workgroup-uniform
    sv_.load(vp + key * a.vs[1], a.vs[1], bits, a.dim);
    f32x16 s[SUB];
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      const int row0 = (wk * SUB + u) * 32;
      s[u] = f32x16{};
#pragma unroll
      for (int e = 0; e < DP / kStep<T>; ++e)
        s[u] = mma<T>(s[u], *reinterpret_cast<const u32x4*>(sk + (row0 + (lane & 31)) * KS + e * kStep<T> + h * V),
                      qf[e]);
      if (static_cast<uint32_t>(bits >> row0) != ~0u) {
        const uint32_t kept = static_cast<uint32_t>(bits >> row0) >> (4 * h);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[u][i] = kept >> mma_row(i, 0) & 1 ? s[u][i] : -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[u][i]);
    }
    // The running maximum moves only when it is passed by more than 8: probabilities of up
    // to 2^8 cost no accuracy, and most tiles neither exchange maxima nor scale the sums.
    if (__any(top * c > m + 8.f)) {
      const float now = fmaxf(m, fmaxf(top, __shfl_xor(top, 32, kWave)) * c);
      const float old = now == -INFINITY ? 1.f : exp2_(m - now);
      l *= old;
#pragma unroll
      for (int t = 0; t < DP / 32; ++t) o[t] *= old;
      m = now;
      from = now == -INFINITY ? 0.f : now;
    }
    u32x4 pf[SUB][16 / V];
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[u][i] = exp2_(fmaf(s[u][i], c, -from));
        l += s[u][i];
      }
#pragma unroll
      for (int f = 0; f < 16 / V; ++f) pf[u][f] = to_frag<T>(s[u], f);
    }
    sv_.store(sv, a.dim);
    more = keys.next(key, bits);
    if (more) sk_.load(kp + key * a.ks[1], a.ks[1], bits, a.dim);
    __syncthreads();
#pragma unroll
    for (int t = 0; t < DP / 32; ++t) {
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int f = 0; f < 16 / V; ++f)
          o[t] = mma<T>(o[t], transposed(sv, VS, (wk * SUB + u) * 32, f, t * 32), pf[u][f]);
    }
    if (more) {
      sk_.store(sk, a.dim);
      __syncthreads();
    }
  }

  if constexpr (WK == 2) {
    static_assert(WQ == 1 && sizeof(smem) >= 64 * 4 * (DP / 2 + 2), "the second wave's sums fit the tiles");
    float* join = reinterpret_cast<float*>(smem);
    __syncthreads();
    if (wk == 1) {
#pragma unroll
      for (int t = 0; t < DP / 32; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) join[(t * 16 + i) * 64 + lane] = o[t][i];
      join[DP / 2 * 64 + lane] = m;
      join[(DP / 2 + 1) * 64 + lane] = l;
    }
    __syncthreads();
    if (wk == 1) return;
    const float m1 = join[DP / 2 * 64 + lane], top = fmaxf(m, m1);
    const float at = top == -INFINITY ? 0.f : top, x0 = exp2_(m - at), x1 = exp2_(m1 - at);
    l = l * x0 + join[(DP / 2 + 1) * 64 + lane] * x1;
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[t][i] = o[t][i] * x0 + join[(t * 16 + i) * 64 + lane] * x1;
    m = top;
  }
  l += __shfl_xor(l, 32, kWave);
  if (r >= rows) return;
  const int64_t row = (b * a.lq + tok) * a.heads + head;
  if (splits > 1) {
    float* out = part + (row * splits + sp) * (a.dim + 2);
    if (h == 0) {
      out[0] = m;
      out[1] = l;
    }
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (t * 32 + mma_row(i, h) < a.dim) out[2 + t * 32 + mma_row(i, h)] = o[t][i];
    return;
  }
  if (h == 0 && a.lse != nullptr) a.lse[row] = l > 0.f ? (m + log2f(l)) * kLn2 : -INFINITY;
  const float inv = l > 0.f ? 1.f / l : 0.f;
  T* out = static_cast<T*>(a.o) + row * a.dim;
#pragma unroll
  for (int t = 0; t < DP / 32; ++t)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = t * 32 + mma_row(4 * j, h);
      Pack<T, 4> x;
#pragma unroll
      for (int u = 0; u < 4; ++u) x.v[u] = from_f<T>(o[t][4 * j + u] * inv);
      if (d + 4 <= a.dim) {
        store_pack<T, 4>(out + d, x);
      } else {
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (d + u < a.dim) out[d + u] = x.v[u];
      }
    }
}

// one wave per row: the ranges' outputs, weighed by exp(their maximum - the largest)
template <typename T>
__global__ __launch_bounds__(256) void att_join(const AttArgs a, int splits, const float* __restrict__ part) {
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / kWave;
  if (row >= a.batch * a.lq * a.heads) return;
  const int64_t step = a.dim + 2;
  const float* p = part + row * splits * step;
  float m = -INFINITY;
  for (int s = lane; s < splits; s += kWave) m = fmaxf(m, p[s * step]);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, kWave));
  const float at = m == -INFINITY ? 0.f : m;
  float l = 0.f, acc[TGX_MAX_HEAD_DIM / kWave] = {};
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float x = exp2_(p[s * step] - at);
    l += p[s * step + 1] * x;
#pragma unroll
    for (int u = 0; u < TGX_MAX_HEAD_DIM / kWave; ++u)
      if (lane + u * kWave < a.dim) acc[u] += p[s * step + 2 + lane + u * kWave] * x;
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int u = 0; u < TGX_MAX_HEAD_DIM / kWave; ++u)
    if (lane + u * kWave < a.dim)
      static_cast<T*>(a.o)[row * a.dim + lane + u * kWave] = from_f<T>(acc[u] * inv);
  if (lane == 0 && a.lse != nullptr) a.lse[row] = l > 0.f ? (m + log2f(l)) * kLn2 : -INFINITY;
}

// Row tiles, and the ranges the keys are cut in where the row tiles alone would leave
// most of the 256 compute units without work
struct FwdShape {
  int wq, wk, mtiles, splits;
  int64_t span;
  FwdShape(const AttArgs& a, int dtype) {
    const int64_t rows = a.lq * a.group;
    const bool small = rows <= 32 && (dtype == TGX_BF16 || a.dim <= 128);
    wq = small ? 1 : rows <= 64 ? 2 : 4;
    wk = small ? 2 : 1;
    mtiles = static_cast<int>(ops_cdiv(rows, 32 * wq));
    const int64_t blocks = a.batch * a.kv_heads * mtiles;
    const int64_t tiles = ops_cdiv(std::max<int64_t>(a.lk, 1), 64);
    const int64_t want = blocks >= 512 ? 1 : ops_cdiv(1024, blocks);
    const int64_t per = ops_cdiv(tiles, std::min(std::min(want, ops_cdiv(tiles, 4)), int64_t(256)));
    span = per * 64;
    splits = static_cast<int>(ops_cdiv(tiles, per));
  }
};

}  // namespace

size_t att_mma_forward_workspace(const AttArgs& a, int dtype) {
  const FwdShape f(a, dtype);
  return f.splits > 1 ? static_cast<size_t>(a.batch * a.lq * a.heads) * f.splits * (a.dim + 2) * 4 : 0;
}

int att_mma_forward(const AttArgs& a, int dtype, void* ws, hipStream_t s) {
  const FwdShape f(a, dtype);
  float* part = static_cast<float*>(ws);
  const int64_t blocks = a.batch * a.kv_heads * f.mtiles * f.splits;
  int rc = by_head(dtype, a.dim, [&](auto t, auto dp, auto tiny) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value;
    constexpr bool TINY = decltype(tiny)::value;
    const dim3 grid(static_cast<unsigned>(blocks));
    if (f.wk == 2) {
      if constexpr (sizeof(T) == 2 || DP <= 128)
        hipLaunchKernelGGL((att_mma_fwd<T, TINY, DP, 1, 2>), grid, dim3(128), 0, s, a, f.mtiles, f.splits, f.span, part);
    } else if (f.wq == 2) {
      hipLaunchKernelGGL((att_mma_fwd<T, TINY, DP, 2, 1>), grid, dim3(128), 0, s, a, f.mtiles, f.splits, f.span, part);
    } else {
      hipLaunchKernelGGL((att_mma_fwd<T, TINY, DP, 4, 1>), grid, dim3(256), 0, s, a, f.mtiles, f.splits, f.span, part);
    }
    return check_launch("att_mma_fwd");
  });
  return rc || f.splits == 1 ? rc : att_join_forward(a, dtype, f.splits, part, s);
}

int att_join_forward(const AttArgs& a, int dtype, int splits, const float* part, hipStream_t s) {
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL(att_join<T>, dim3(static_cast<unsigned>(ops_cdiv(a.batch * a.lq * a.heads, 4))), dim3(256), 0, s,
                       a, splits, part);
    return check_launch("att_join");
  });
}

}  // namespace tgx
