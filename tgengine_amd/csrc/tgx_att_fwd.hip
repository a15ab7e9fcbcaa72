// Attention forward on the matrix units, one pass over the keys.
//
// A wave owns a tile of rows of a problem and keeps their queries as fragments.  A tile of
// keys gives S^T = K Q^T (keys down a lane's registers, one row a lane), so that the
// running maximum and sum of the softmax are a lane's own but for an exchange between
// the lanes of a row now and then, and P^T, still in the same registers, is the second operand of
// O^T += V^T P^T.  Scores are in units of log 2.  bf16's matrix units take probabilities of
// bf16: a second product adds what cutting them to that left (to_frag), so that an output is
// off by its own rounding only.  Without it the two roundings' errors together were 1.41 times
// the output's own, however many keys there were.  It uses the same reads of V: 2 x (1,000 x
// 8,000 tokens), 16/4 heads of 128, take 224 us with it and 180 without, 200 x (200 x 200), 4
// heads of 64, 61 and 55, single tokens to 30,001 keys 96 either way.
//
// What bounds it: for bf16 the softmax between the products and the LDS reads that feed
// them (that first call, 92% kept: 538 TFLOP/s of the 1,225 that a matrix product of 8,192
// reaches, 807 with the second product counted); for f32 the matrix units, eight times slower
// (400 x (65 x 65), 2 heads of 100: 51 us for 75 MB and 1.4 GFLOP, whose 16-row tiles pad
// 65 to 80 and 100 to 112); for single tokens the reads of keys and values (5 x 30,001 keys
// of 8 heads of 128, bf16, 73% kept: 97 us for 447 MB, 4.6 TB/s).
#include "tgx_attention.h"

namespace tgx {
namespace {

// The waves of a workgroup take kTile rows each: WQ of them, or 4 to 8 for WQ = 0 (f32,
// whose 16-row tiles fit odd lengths better); WK > 1: WK waves take the same rows, one tile
// of each KT = 64 keys each, and are joined at the end.  With splits > 1 the keys are cut in
// as many ranges of `span` keys and each leaves its maximum, sum and unscaled output in
// `part` for att_join.
template <typename T, bool TINY, int DP, int WQ, int WK>
__global__ __launch_bounds__(WQ == 0 ? 512 : 64 * WQ * WK, DP > 128 ? 1 : WQ == 0 && DP <= 112 ? 4 : 2) void att_mma_fwd(const AttArgs a, int mtiles, int splits,
                                                                             int64_t span, const AttParts part) {
  using KTile = LdsTile<T, DP, Reads::kRows>;
  using VTile = LdsTile<T, DP, Reads::kColumns>;
  constexpr int TS = kTile<T>, KT = sizeof(T) == 2 || WK > 1 ? 64 : 32, SUB = KT / TS / WK,
                OT = DP / TS, ST = DP / kStep;
  static_assert(WK == 1 || SUB == 1, "one tile of keys a wave");
  __shared__ __align__(16) T smem[KT * (KTile::ROW + VTile::ROW)];
  T* sk = smem;
  T* sv = smem + KT * KTile::ROW;
  const int lane = threadIdx.x & (kWave - 1), group = lane_group<T>(), wave = threadIdx.x / kWave;
  const int wq = WK > 1 ? 0 : wave, wk = WK > 1 ? wave : 0, waves = WQ == 0 ? blockDim.x / kWave : WQ;
  int64_t w = by_die(blockIdx.x, gridDim.x);
  const int sp = static_cast<int>(w % splits);
  w /= splits;
  const int64_t r0 = w % mtiles * (TS * waves) + wq * TS;
  const int64_t p = w / mtiles;
  const int hk = static_cast<int>(p % a.kv_heads);
  const int64_t b = p / a.kv_heads;
  const int64_t rows = a.lq * a.group, r = r0 + lane_row<T>();
  const bool busy = r0 < rows;  // a wave past the last row only helps to move keys and values
  const int64_t tok = r < rows ? r / a.group : 0;
  const int head = hk * a.group + static_cast<int>(r - tok * a.group);
  const T* kp = static_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[2];
  const T* vp = static_cast<const T*>(a.v) + b * a.vs[0] + hk * a.vs[2];
  u32x4 qf[ST];
  row_frags<T, TINY, DP>(
      qf, r < rows ? static_cast<const T*>(a.q) + b * a.qs[0] + tok * a.qs[1] + head * a.qs[2] : nullptr, a.dim);
  // Scores are in units of 1 / c: the sign of the scale goes to the queries, so that the
  // largest score is the largest product, and a scale of zero makes them zero.
  const float c = a.scale == 0.f ? 1.f : fabsf(a.scale) * kLog2e;
  if (!(a.scale > 0.f))
#pragma unroll
    for (int e = 0; e < ST; ++e)
#pragma unroll
      for (int u = 0; u < 4; ++u)
        qf[e][u] = a.scale == 0.f ? 0u : qf[e][u] ^ (sizeof(T) == 2 ? 0x80008000u : 0x80000000u);
  Acc<T> o[OT];
#pragma unroll
  for (int t = 0; t < OT; ++t) o[t] = Acc<T>{};
  float m = -INFINITY, from = 0.f, l = 0.f;  // from: m, or 0 as long as no key was kept

  const int64_t lo = sp * span, hi = lo + span < a.lk ? lo + span : a.lk;
  Keys<KT> keys(a.mask == nullptr ? nullptr : a.mask + b * a.mask_stride, lo, hi);
  int64_t key;
  uint64_t bits;
  bool more = keys.next(key, bits);
  Stage<T, TINY, KT, DP, (WQ == 0 ? 4 : WQ * WK), (WQ > 0)> st(a.dim);
  if (more) {
    st.load(kp + key * a.ks[1], a.ks[1], bits, a.dim);
    st.template store<KTile::ROW>(sk, a.dim);
  }
  __syncthreads();
  while (more) {  // workgroup-uniform
    st.load(vp + key * a.vs[1], a.vs[1], bits, a.dim);
    u32x4 pf[SUB][kFrags<T>], rest[SUB][kFrags<T>];
    const uint64_t now = bits;
    constexpr uint32_t ALL = TS == 32 ? ~0u : 0xffffu;
    if (busy) {
      Acc<T> s[SUB];
      float top = -INFINITY;
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        const int row0 = (wk * SUB + u) * TS;
        const uint32_t here = static_cast<uint32_t>(now >> row0) & ALL;
        s[u] = Acc<T>{};
        if (here != 0)
#pragma unroll
          for (int e = 0; e < ST; ++e) s[u] = mma<T>(s[u], KTile::frag(sk, row0, e), qf[e]);
        if (here != ALL)
#pragma unroll
          for (int i = 0; i < kRegs<T>; ++i)
            s[u][i] = here >> (4 * group) >> mma_row<T>(i, 0) & 1 ? s[u][i] : -INFINITY;
#pragma unroll
        for (int i = 0; i < kRegs<T>; ++i) top = fmaxf(top, s[u][i]);
      }
      // The running maximum moves only when it is passed by more than 8: probabilities of
      // up to 2^8 cost no accuracy, and most tiles neither exchange maxima nor scale the
      // sums.
      if (__any(top * c > m + 8.f)) {
#pragma unroll
        for (int off = TS; off < kWave; off <<= 1) top = fmaxf(top, __shfl_xor(top, off, kWave));
        const float next = fmaxf(m, top * c);
        const float old = next == -INFINITY ? 1.f : exp2_(m - next);
        l *= old;
#pragma unroll
        for (int t = 0; t < OT; ++t) o[t] *= old;
        m = next;
        from = next == -INFINITY ? 0.f : next;
      }
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
#pragma unroll
        for (int i = 0; i < kRegs<T>; ++i) {
          s[u][i] = exp2_(fmaf(s[u][i], c, -from));
          l += s[u][i];
        }
#pragma unroll
        for (int f = 0; f < kFrags<T>; ++f) pf[u][f] = to_frag<T>(s[u], f);
        if constexpr (sizeof(T) == 2)
#pragma unroll
          for (int f = 0; f < kFrags<T>; ++f) rest[u][f] = rest_frag<false>(s[u], f);
      }
    }
    st.template store<VTile::ROW>(sv, a.dim);
    more = keys.next(key, bits);
    if (more) st.load(kp + key * a.ks[1], a.ks[1], bits, a.dim);
    __syncthreads();
    if (busy) {
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        const int row0 = (wk * SUB + u) * TS;
        if ((static_cast<uint32_t>(now >> row0) & ALL) == 0) continue;
#pragma unroll
        for (int t = 0; t < OT; ++t)
#pragma unroll
          for (int f = 0; f < kFrags<T>; ++f) {
            const u32x4 vf = VTile::transposed(sv, row0, f, t);
            o[t] = mma<T>(o[t], vf, pf[u][f]);
            if constexpr (sizeof(T) == 2) o[t] = mma<T>(o[t], vf, rest[u][f]);
          }
      }
    }
    if (more) {
      st.template store<KTile::ROW>(sk, a.dim);
      __syncthreads();
    }
  }

  if constexpr (WK > 1) {
    constexpr int OR = OT * kRegs<T>;
    static_assert(sizeof(smem) >= (WK - 1) * 64 * 4 * (OR + 2), "the other waves' sums fit the tiles");
    float* join = reinterpret_cast<float*>(smem);
    __syncthreads();
    if (wk > 0) {
      float* mine = join + (wk - 1) * 64 * (OR + 2) + lane;
#pragma unroll
      for (int x = 0; x < OR; ++x) mine[x * 64] = o[x / kRegs<T>][x % kRegs<T>];
      mine[OR * 64] = m;
      mine[(OR + 1) * 64] = l;
    }
    __syncthreads();
    if (wk > 0) return;
#pragma unroll
    for (int y = 0; y < WK - 1; ++y) {
      const float* other = join + y * 64 * (OR + 2) + lane;
      const float m1 = other[OR * 64], top = fmaxf(m, m1);
      const float at = top == -INFINITY ? 0.f : top, x0 = exp2_(m - at), x1 = exp2_(m1 - at);
      l = l * x0 + other[(OR + 1) * 64] * x1;
#pragma unroll
      for (int x = 0; x < OR; ++x)
        o[x / kRegs<T>][x % kRegs<T>] = o[x / kRegs<T>][x % kRegs<T>] * x0 + other[x * 64] * x1;
      m = top;
    }
  }
#pragma unroll
  for (int off = TS; off < kWave; off <<= 1) l += __shfl_xor(l, off, kWave);
  if (r >= rows) return;
  const int64_t row = (b * a.lq + tok) * a.heads + head;
  if (splits > 1) {
    if (group == 0) part.ml[row * splits + sp] = make_float2(m, l);
    store_parts<T, DP>(part.o + (row * splits + sp) * a.dim, o, a.dim);
    return;
  }
  if (group == 0 && a.lse != nullptr) a.lse[row] = log_sum(m, l);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  store_columns<T, DP>(static_cast<T*>(a.o) + row * a.dim, o, inv, a.dim);
  if (sizeof(T) == 2 && a.rest != nullptr) {
#pragma unroll
    for (int t = 0; t < OT; ++t)
#pragma unroll
      for (int i = 0; i < kRegs<T>; ++i) o[t][i] = lost<T>(o[t][i] * inv);
    store_columns<T, DP>(static_cast<T*>(a.rest) + row * a.dim, o, 1.f, a.dim);
  }
}

// One wave per row, LT lanes per range of 4 values each and 64 / LT ranges at a time.
// SUMS: the ranges' outputs added up; else each weighed by exp(its maximum - the largest)
// and divided by the sum.  Reads bound it: 160 rows of 128 in 26 ranges 9 us, 32,000 rows in
// 2 ranges 16 us.
template <typename T, int LT, bool SUMS>
__global__ __launch_bounds__(256) void att_join(T* __restrict__ out, T* __restrict__ rest, float* __restrict__ lse, int64_t rows, int dim,
                                                float by, int splits, const AttParts part) {
  constexpr int G = kWave / LT;
  const int lane = threadIdx.x & (kWave - 1), grp = lane / LT;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / kWave;
  if (row >= rows) return;
  const float2* ml = part.ml + row * splits;
  float m = -INFINITY, l = 0.f;
  if constexpr (!SUMS) {
    for (int y = lane; y < splits; y += kWave) m = fmaxf(m, ml[y].x);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, kWave));
    if (m == -INFINITY) m = 0.f;  // no range kept a key: all sums are 0
    for (int y = lane; y < splits; y += kWave) l += ml[y].y * exp2_(ml[y].x - m);
    l = group_sum<kWave>(l);
    by = l == 0.f ? 0.f : 1.f / l;
    if (lane == 0 && lse != nullptr) lse[row] = log_sum(m, l);
  }
  const float* o = part.o + row * splits * dim;
  for (int c = (lane % LT) * 4; c < dim; c += LT * 4) {
    const int n = min(4, dim - c);
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    if (n == 4) {
#pragma unroll 8
      for (int y = grp; y < splits; y += G) {
        const Pack<float, 4> x = load_pack<float, 4>(o + static_cast<int64_t>(y) * dim + c);
        const float w = SUMS ? 1.f : exp2_(ml[y].x - m);
#pragma unroll
        for (int u = 0; u < 4; ++u) acc[u] = fmaf(x.v[u], w, acc[u]);
      }
    } else {
      for (int y = grp; y < splits; y += G) {
        const float w = SUMS ? 1.f : exp2_(ml[y].x - m);
        for (int u = 0; u < 3; ++u)
          if (u < n) acc[u] = fmaf(o[static_cast<int64_t>(y) * dim + c + u], w, acc[u]);
      }
    }
#pragma unroll
    for (int off = LT; off < kWave; off <<= 1)
#pragma unroll
      for (int u = 0; u < 4; ++u) acc[u] += __shfl_xor(acc[u], off, kWave);
    if (grp == 0)
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (u < n) {
          out[row * dim + c + u] = from_f<T>(acc[u] * by);
          if (!SUMS && rest != nullptr) rest[row * dim + c + u] = from_f<T>(lost<T>(acc[u] * by));
        }
  }
}

template <bool SUMS>
int join_launch(void* out, void* rest, float* lse, int64_t rows, int dim, int dtype, float by, int splits, const AttParts& part,
                hipStream_t s) {
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    const dim3 grid(static_cast<unsigned>(ops_cdiv(rows, 4)));
    T *o = static_cast<T*>(out), *r = static_cast<T*>(rest);
    if (dim <= 64) hipLaunchKernelGGL((att_join<T, 16, SUMS>), grid, dim3(256), 0, s, o, r, lse, rows, dim, by, splits, part);
    else if (dim <= 128)
      hipLaunchKernelGGL((att_join<T, 32, SUMS>), grid, dim3(256), 0, s, o, r, lse, rows, dim, by, splits, part);
    else hipLaunchKernelGGL((att_join<T, 64, SUMS>), grid, dim3(256), 0, s, o, r, lse, rows, dim, by, splits, part);
    return check_launch("att_join");
  });
}

// Row tiles, and the ranges the keys are cut in where the row tiles alone would leave most
// of the 256 compute units without work: 512 workgroups, the most that the registers let run
// at a time (2 x (300 x 6,000 tokens), 8/4 heads of 128, bf16: 43 us, 54 with 1,024 and 206
// uncut; f32 192, 210 and 977), or 1,024 of the smaller ones that share a row tile (5 x
// 30,001 keys, 32/8 heads of 128, bf16, all kept: 118 us, 124 with 512, 135 with 2,048).
//
// A problem of one row tile gives every tile of keys to WK waves (f32, 4 x 10,000 keys,
// 32/8 heads of 128: 68 us, 94 with a tile of rows each; bf16 38 and 39 there, 27 and 34 for
// 2,000 x 70 keys, 8/2 heads of 64).
struct FwdShape {
  int wq, wk, mtiles, splits;
  int64_t span;
  FwdShape(const AttArgs& a, int dtype) {
    const int64_t rows = a.lq * a.group;
    const int tile = dtype == TGX_BF16 ? 32 : 16;
    wk = rows <= tile ? 64 / tile : 1;
    wq = wk > 1 ? 1 : tile == 32 ? (rows <= 64 ? 2 : 4) : waves_for(ops_cdiv(rows, tile), 4, 8);
    mtiles = static_cast<int>(ops_cdiv(rows, tile * wq));
    const int64_t blocks = a.batch * a.kv_heads * mtiles;
    const int64_t tiles = ops_cdiv(std::max<int64_t>(a.lk, 1), 64);
    const int64_t want = blocks >= 512 ? 1 : ops_cdiv(wk > 1 ? 1024 : 512, blocks);
    const int64_t per = ops_cdiv(tiles, std::min(std::min(want, ops_cdiv(tiles, 4)), int64_t(256)));
    span = per * 64;
    splits = static_cast<int>(ops_cdiv(tiles, per));
  }
};

}  // namespace

size_t att_mma_forward_workspace(const AttArgs& a, int dtype) {
  return AttParts::bytes(a.batch * a.lq * a.heads, FwdShape(a, dtype).splits, a.dim);
}

int att_mma_forward(const AttArgs& a, int dtype, void* ws, hipStream_t s) {
  const FwdShape f(a, dtype);
  const AttParts part(ws, a.batch * a.lq * a.heads, f.splits);
  const int64_t blocks = a.batch * a.kv_heads * f.mtiles * f.splits;
  int rc = check_grid("tgx_attention", blocks, 64 * f.wq * f.wk);
  if (rc) return rc;
  rc = by_head(dtype, a.dim, [&](auto t, auto dp, auto tiny) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value, TS = kTile<T>;
    constexpr bool TINY = decltype(tiny)::value;
    const dim3 grid(static_cast<unsigned>(blocks)), block(64 * f.wq * f.wk);
    auto go = [&](auto wq, auto wk) {
      hipLaunchKernelGGL((att_mma_fwd<T, TINY, DP, decltype(wq)::value, decltype(wk)::value>), grid, block, 0, s, a, f.mtiles,
                         f.splits, f.span, part);
    };
    constexpr std::integral_constant<int, 1> one{};
    if (f.wk > 1) go(one, std::integral_constant<int, 64 / TS>{});
    else if constexpr (sizeof(T) == 4) go(std::integral_constant<int, 0>{}, one);
    else if (f.wq == 2) go(std::integral_constant<int, 2>{}, one);
    else go(std::integral_constant<int, 4>{}, one);
    return check_launch("att_mma_fwd");
  });
  return rc || f.splits == 1 ? rc : att_join_forward(a, dtype, f.splits, part, s);
}

int att_join_forward(const AttArgs& a, int dtype, int splits, const AttParts& part, hipStream_t s) {
  return join_launch<false>(a.o, a.rest, a.lse, a.batch * a.lq * a.heads, a.dim, dtype, 1.f, splits, part, s);
}

int att_join_sums(void* out, int64_t rows, int dim, int dtype, float by, int splits, const float* part, hipStream_t s) {
  AttParts p(nullptr, 0, 1);
  p.o = const_cast<float*>(part);
  return join_launch<true>(out, nullptr, nullptr, rows, dim, dtype, by, splits, p, s);
}

}  // namespace tgx
