// Attention backward on the matrix units.
//
// Three launches: delta_i = do_i . o_i and the log sum of every row; dk and dv, where a wave
// owns a tile of keys and walks over the problem's rows; dq, where a wave owns a tile of rows
// and walks over the keys.  Scores are computed anew in both from the saved log sums (7
// products of M x Lk x D, the sums of each output in one place and in one order, no atomics).
//
// As in the forward pass every score tile stays in the registers it was computed in: a
// wave's columns are what it owns (keys for dk and dv, rows for dq), a lane's 16 values
// run along the axis that the next product sums over, and that product's first operand
// comes transposed out of LDS.  Sums stay in 32 bits, and bf16's products take p and ds in two
// parts, so that a gradient is off by its own rounding only (mma_fine).
#include "tgx_attention.h"

namespace tgx {
namespace {

constexpr int kDeltaLanes = 16;

// keys of a row of kept scores: whole 16-byte pieces
__host__ __device__ __forceinline__ int64_t scores_row(int64_t lk) { return (lk + 3) / 4 * 4; }

// Per row, in the order of problems and their rows: its log sum in units of log 2 (+inf
// for a row that keeps no key: its probabilities are then zeros) and delta, from the output
// as it was before rounding where its rest was kept: delta's error reaches every score of
// the row alike.
// kDeltaLanes lanes a row; HBM bounds it (52,000 f32 rows of 100: 42 MB in 11 us, 3.7 TB/s)
template <typename T>
__global__ __launch_bounds__(256) void att_stats(const T* __restrict__ out, const T* __restrict__ rest,
                                                 const T* __restrict__ dout,
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
    if (sizeof(T) == 2 && rest != nullptr) {
      const Pack<T, V> z = __builtin_bit_cast(Pack<T, V>, row_values(rest + at, c, dim));
#pragma unroll
      for (int u = 0; u < V; ++u) s += to_f(z.v[u]) * to_f(y.v[u]);
    }
  }
  s = group_sum<kDeltaLanes>(s);
  if (lane != 0 || row >= rows) return;
  const int head = static_cast<int>(row % heads);
  const int64_t tok = row / heads % lq, b = row / heads / lq;
  const int64_t to = ((b * (heads / group) + head / group) * lq + tok) * group + head % group;
  const float x = lse[row];
  stats[to] = make_float2(x == -INFINITY ? INFINITY : x * kLog2e, s);
}

// sums += fragment f of x times the tile's rows from row0 on.  bf16 takes what cutting x to
// bf16 leaves through a second product with the same operand out of LDS: without it dq, dk and
// dv were 1.41 to 1.45 times as far off as one rounding of them.  2 x (1,000 x 8,000 tokens),
// 16/4 heads of 128, 92% kept: dk and dv 488 us with it and 402 without, dq 308 and 252; 400 x
// (65 x 65), 2 heads of 100: 72 and 64, 28 and 27.
template <typename T, int DP, typename TILE, bool SIGNED>
__device__ __forceinline__ void mma_fine(Acc<T> (&sums)[DP / kTile<T>], const T* tile, int row0, const Acc<T>& x, int f) {
  const u32x4 xf = to_frag<T>(x, f);
  u32x4 rest;
  if constexpr (sizeof(T) == 2) rest = rest_frag<SIGNED>(x, f);
#pragma unroll
  for (int t = 0; t < DP / kTile<T>; ++t) {
    const u32x4 y = TILE::transposed(tile, row0, f, t);
    sums[t] = mma<T>(sums[t], y, xf);
    if constexpr (sizeof(T) == 2) sums[t] = mma<T>(sums[t], y, rest);
  }
}

// Keeps the steps of bf16's dk and dv apart: left to itself the compiler reads all operands
// ahead and runs out of registers (605 us for 1,000 x 8,000 tokens, 422 so, both with one
// product each; the other wave of the SIMD fills the gaps).  f32 has the registers.
template <typename T>
__device__ __forceinline__ void one_by_one() {
  if constexpr (sizeof(T) == 2) __builtin_amdgcn_sched_barrier(0);
}

// dk and dv, kTile keys a wave.  S = Q K^T and dP = dO V^T have the rows down a lane's
// registers and one key a lane; dV^T += dO^T P and dK^T += Q^T dS follow.
//
// The rows' tiles stand in LDS twice, so that one is filled while the other is read and a
// tile takes one barrier.
//
// With splits > 1 the rows are cut in ranges of `span` and each leaves its sums in `part`,
// dk's before dv's.
// KEEP (f32): ds goes to `scores`, rows of scores_row() keys, for att_scores_q.
//
// Bounded by the matrix units and the LDS reads that feed them, behind the steps that registers
// keep apart, for bf16: 2 x (1,000 x 8,000 tokens), 16/4 heads of 128, 92% kept, 488 us, 493
// TFLOP/s of four products and 740 of the six;
// by the matrix units for f32: 400 x (65 x 65), 2 heads of 100, 95 us, 48 TFLOP/s with the
// padding to 80 x 80 x 112 and 29 without.
//
// LEAST to kv_most() waves a workgroup.  bf16 heads of 65 to 128 values come two ways: 8
// waves, which leaves each the registers for one row of staging and two waves a SIMD, or 2
// to 4 with all registers for up to 64 keys, which 8 waves would mostly idle through (200 x
// 100 rows, 4/2 heads: of 128 with 64 keys 62 us by 8 waves and 36 so, with 100 66 and 64,
// with 144 72 and 120; of 80 with 64 42 and 27, with 90 43 and 48).
template <typename T, int DP>
constexpr bool kTwoWays = sizeof(T) == 2 && DP > 64 && DP <= 128;
template <typename T, int DP>
constexpr int kKvLeast = sizeof(T) == 2 ? 2 : 4;
template <typename T>
constexpr int kv_most(int dp, int least) {
  if (dp > 128) return sizeof(T) == 2 ? 2 : 4;  // wide heads: as many registers as there are
  return sizeof(T) == 2 && dp > 64 && least < 8 ? 4 : 8;
}

template <typename T, bool TINY, int DP, int LEAST, bool KEEP>
__global__ __launch_bounds__(64 * kv_most<T>(DP, LEAST), DP > 128 || (sizeof(T) == 2 && DP > 64 && LEAST < 8) ? 1 : 2)
void att_mma_kv(const AttArgs a, int ktiles, int splits, int64_t span, const float2* __restrict__ stats,
                float* __restrict__ scores, float* __restrict__ part) {
  using Tile = LdsTile<T, DP, Reads::kBoth>;
  using Own = LdsTile<T, DP, Reads::kRows>;
  constexpr int TS = kTile<T>, R = TS, OT = DP / TS, ST = DP / kStep, W = LEAST;
  constexpr bool FIXED = LEAST == kv_most<T>(DP, LEAST);
  // a wave holds its keys and values as fragments; wide bf16 heads, whose sums alone take
  // 256 registers, leave them in LDS
  constexpr bool HELD = sizeof(T) == 4 || DP <= 128;
  __shared__ __align__(16) T sq[2][R * Tile::ROW], sg[2][R * Tile::ROW];
  __shared__ __align__(16) T sk[HELD ? 8 : TS * W * Own::ROW], sv[HELD ? 8 : TS * W * Own::ROW];
  __shared__ __align__(16) float slse[2][R], sdelta[2][R];
  const int group = lane_group<T>(), wave = threadIdx.x / kWave;
  int64_t w = by_die(blockIdx.x, gridDim.x);
  const int sp = static_cast<int>(w % splits);
  w /= splits;
  const int64_t j = w % ktiles * (TS * (blockDim.x / kWave)) + wave * TS + lane_row<T>();
  const int64_t p = w / ktiles;
  const int hk = static_cast<int>(p % a.kv_heads);
  const int64_t b = p / a.kv_heads;
  const bool kept = j < a.lk && (a.mask == nullptr || a.mask[b * a.mask_stride + j] != 0);
  const int64_t at = (b * a.lk + j) * a.kv_heads + hk;
  Acc<T> dk[OT], dv[OT];
#pragma unroll
  for (int t = 0; t < OT; ++t) dk[t] = dv[t] = Acc<T>{};
  if (__syncthreads_or(kept)) {
    const bool busy = __any(kept);
    const T* kp = static_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[2];
    const T* vp = static_cast<const T*>(a.v) + b * a.vs[0] + hk * a.vs[2];
    u32x4 kf[HELD ? ST : 1], vf[HELD ? ST : 1];
    if constexpr (HELD) {
      row_frags<T, TINY, DP>(kf, kept ? kp + j * a.ks[1] : nullptr, a.dim);
      row_frags<T, TINY, DP>(vf, kept ? vp + j * a.vs[1] : nullptr, a.dim);
    } else {
      static_assert(HELD || TS * W == 64, "a bit of a word for each key");
      // every wave's lanes hold the same 32 keys twice: a wave's ballot has its keys' bits
      __shared__ uint32_t bits[W];
      const uint64_t mine = __ballot(kept);
      if ((threadIdx.x & (kWave - 1)) == 0) bits[wave] = static_cast<uint32_t>(mine);
      __syncthreads();
      const uint64_t both = static_cast<uint64_t>(bits[1]) << 32 | bits[0];
      const int64_t first = j - (wave * TS + lane_row<T>());
      Stage<T, TINY, TS * W, DP, W, true> kv(a.dim);
      kv.load(kp + first * a.ks[1], a.ks[1], both, a.dim);
      kv.template store<Own::ROW>(sk, a.dim);
      kv.load(vp + first * a.vs[1], a.vs[1], both, a.dim);
      kv.template store<Own::ROW>(sv, a.dim);
    }
    const float c = a.scale * kLog2e;
    const int64_t all_rows = a.lq * a.group, lo = sp * span, rows = lo + span < all_rows ? lo + span : all_rows;
    const T* qp = static_cast<const T*>(a.q) + b * a.qs[0] + static_cast<int64_t>(hk) * a.group * a.qs[2];
    const T* gp = static_cast<const T*>(a.dout) + b * a.os[0] + static_cast<int64_t>(hk) * a.group * a.os[2];
    stats += p * all_rows;
    Stage<T, TINY, R, DP, W, FIXED> q(a.dim), g(a.dim);
    constexpr int N = Stage<T, TINY, R, DP, W, FIXED>::N;
    // each of the thread's rows: its head of the group and its offsets, moved on by R rows
    // a tile without a division
    int hg[N];
    int64_t qo[N], go[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int64_t row = lo + q.row(n), tok = row / a.group;
      hg[n] = static_cast<int>(row - tok * a.group);
      qo[n] = tok * a.qs[1] + hg[n] * a.qs[2];
      go[n] = tok * a.os[1] + hg[n] * a.os[2];
    }
    const int dt = R / a.group, dh = R % a.group;
    float2 st = make_float2(INFINITY, 0.f);
    auto fetch = [&](int64_t first) {
      q.load(a.dim, [&](int n) { return (q.whole(n) || q.row(n) < R) && first + q.row(n) < rows ? qp + qo[n] : nullptr; });
      g.load(a.dim, [&](int n) { return (q.whole(n) || q.row(n) < R) && first + q.row(n) < rows ? gp + go[n] : nullptr; });
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
    __builtin_amdgcn_s_waitcnt(kNoLoads);  // the fragments are here: the loop does not wait for them again
    auto put = [&](int to) {
      q.template store<Tile::ROW>(sq[to], a.dim);
      g.template store<Tile::ROW>(sg[to], a.dim);
      if (threadIdx.x < R) {
        slse[to][threadIdx.x] = st.x;
        sdelta[to][threadIdx.x] = st.y;
      }
    };
    fetch(lo);
    put(0);
    if (lo + R < rows) fetch(lo + R);
    int cur = 0;
    for (int64_t first = lo; first < rows; first += R, cur ^= 1) {
      __syncthreads();
      if (sizeof(T) == 2 || busy) {
        Acc<T> s = Acc<T>{}, dp = Acc<T>{};
#pragma unroll
        for (int e = 0; e < ST; ++e) {
          s = mma<T>(s, Tile::frag(sq[cur], 0, e), HELD ? kf[HELD ? e : 0] : Own::frag(sk, wave * TS, e));
          if (e % 4 == 3) one_by_one<T>();
        }
        one_by_one<T>();
#pragma unroll
        for (int i = 0; i < kRegs<T>; ++i) s[i] = exp2_(fmaf(s[i], c, -slse[cur][mma_row<T>(i, group)]));
        one_by_one<T>();
#pragma unroll
        for (int f = 0; f < kFrags<T>; ++f) {
          mma_fine<T, DP, Tile, false>(dv, sg[cur], 0, s, f);
          one_by_one<T>();
        }
#pragma unroll
        for (int e = 0; e < ST; ++e) {
          dp = mma<T>(dp, Tile::frag(sg[cur], 0, e), HELD ? vf[HELD ? e : 0] : Own::frag(sv, wave * TS, e));
          if (e % 4 == 3) one_by_one<T>();
        }
        one_by_one<T>();
#pragma unroll
        for (int i = 0; i < kRegs<T>; ++i) dp[i] = s[i] * (dp[i] - sdelta[cur][mma_row<T>(i, group)]);
        if constexpr (KEEP) {
          float* to = scores + (p * all_rows + first) * scores_row(a.lk) + j;
          if (j < scores_row(a.lk))
#pragma unroll
            for (int i = 0; i < kRegs<T>; ++i)
              if (first + mma_row<T>(i, group) < rows)
                to[mma_row<T>(i, group) * scores_row(a.lk)] = kept ? dp[i] : 0.f;
        }
        one_by_one<T>();
#pragma unroll
        for (int f = 0; f < kFrags<T>; ++f) {
          mma_fine<T, DP, Tile, true>(dk, sq[cur], 0, dp, f);
          one_by_one<T>();
        }
      }
      if (first + R < rows) {
        put(cur ^ 1);
        if (first + 2 * R < rows) fetch(first + 2 * R);
      }
    }
  }
  if (j >= a.lk) return;
  // A masked key's sums were taken along: a product's columns are its lanes' own, and what
  // the rows hold (a gradient of NaN, say) must not reach it
  if (!kept)
#pragma unroll
    for (int t = 0; t < OT; ++t) dk[t] = dv[t] = Acc<T>{};
  if (splits > 1) {
    float* to = part + (at * splits + sp) * a.dim;
    if (a.dk != nullptr) store_parts<T, DP>(to, dk, a.dim);
    if (a.dv != nullptr) store_parts<T, DP>(to + a.batch * a.lk * a.kv_heads * splits * a.dim, dv, a.dim);
    return;
  }
  if (a.dk != nullptr) store_columns<T, DP>(static_cast<T*>(a.dk) + at * a.dim, dk, a.scale, a.dim);
  if (a.dv != nullptr) store_columns<T, DP>(static_cast<T*>(a.dv) + at * a.dim, dv, 1.f, a.dim);
}

// f32's dq from the ds that att_mma_kv kept: one product where att_mma_q takes three, for
// the writing and reading of the scores.  16 rows a wave, 4 to 8 waves; a wave reads its
// rows' scores as fragments.  400 x (65 x 65) tokens, 2 heads of 100: 29 us; by three
// products 74.
template <bool TINY, int DP>
__global__ __launch_bounds__(512, 2) void att_scores_q(const AttArgs a, int mtiles, const float* __restrict__ scores) {
  using T = float;
  using KTile = LdsTile<T, DP, Reads::kColumns>;
  constexpr int TS = kTile<T>, KT = 32, OT = DP / TS;
  __shared__ __align__(16) T sk[2][KT * KTile::ROW];
  const int group = lane_group<T>(), wave = threadIdx.x / kWave;
  const int64_t w = by_die(blockIdx.x, gridDim.x);
  const int64_t r0 = w % mtiles * (TS * (blockDim.x / kWave)) + wave * TS, r = r0 + lane_row<T>();
  const int64_t p = w / mtiles;
  const int hk = static_cast<int>(p % a.kv_heads);
  const int64_t b = p / a.kv_heads;
  const int64_t rows = a.lq * a.group, ks = scores_row(a.lk);
  const bool busy = r0 < rows;  // a wave past the last row only helps to move keys
  const T* kp = static_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[2];
  scores += (p * rows + (r < rows ? r : 0)) * ks + 4 * group;
  Acc<T> dq[OT];
#pragma unroll
  for (int t = 0; t < OT; ++t) dq[t] = Acc<T>{};
  Keys<KT> keys(a.mask == nullptr ? nullptr : a.mask + b * a.mask_stride, 0, a.lk);
  int64_t key;
  uint64_t bits;
  bool more = keys.next(key, bits);
  Stage<T, TINY, KT, DP, 4, false> k(a.dim);
  u32x4 next[KT / TS] = {};
  auto fetch = [&]() {
    k.load(kp + key * a.ks[1], a.ks[1], bits, a.dim);
#pragma unroll
    for (int u = 0; u < KT / TS; ++u) {
      next[u] = u32x4{0, 0, 0, 0};
      // tiles that keep no key were not written
      if (r < rows && (bits >> (u * TS) & 0xffff) != 0 && key + u * TS + 4 * group < ks)
        next[u] = load16(scores + key + u * TS);
    }
  };
  if (more) {
    fetch();
    k.template store<KTile::ROW>(sk[0], a.dim);
  }
  for (int cur = 0; more; cur ^= 1) {  // workgroup-uniform
    u32x4 ds[KT / TS];
#pragma unroll
    for (int u = 0; u < KT / TS; ++u) ds[u] = next[u];
    const uint32_t now = static_cast<uint32_t>(bits);
    __syncthreads();
    more = keys.next(key, bits);
    if (more) fetch();
    if (busy) {
#pragma unroll
      for (int u = 0; u < KT / TS; ++u)
        if ((now >> (u * TS) & 0xffff) != 0)
#pragma unroll
          for (int t = 0; t < OT; ++t) dq[t] = mma<T>(dq[t], KTile::transposed(sk[cur], u * TS, 0, t), ds[u]);
    }
    if (more) k.template store<KTile::ROW>(sk[cur ^ 1], a.dim);
  }
  if (r >= rows) return;
  const int64_t tok = r / a.group;
  const int head = hk * a.group + static_cast<int>(r - tok * a.group);
  store_columns<T, DP>(static_cast<T*>(a.dq) + ((b * a.lq + tok) * a.heads + head) * a.dim, dq, a.scale, a.dim);
}

// dq, kTile rows a wave.  S^T = K Q^T and dP^T = V dO^T have the keys down a lane's registers
// and one row a lane; dQ^T += K^T dS^T follows.  With splits > 1 each range of `span` keys
// leaves its sum in `part`.  W waves, or 4 to 8 for W = 0.  Bounded as att_mma_kv is: 2 x
// (1,000 x 8,000 tokens), 16/4 heads of 128, bf16, 92% kept, 308 us, 585 TFLOP/s of three
// products and 780 of the four.
template <typename T, bool TINY, int DP, int W>
__global__ __launch_bounds__(W == 0 ? 512 : 64 * W, DP > 128 ? 1 : 2) void att_mma_q(const AttArgs a, int mtiles, int splits,
                                                                     int64_t span, const float2* __restrict__ stats,
                                                                     float* __restrict__ part) {
  using KTile = LdsTile<T, DP, Reads::kBoth>;
  using VTile = LdsTile<T, DP, Reads::kRows>;
  constexpr int TS = kTile<T>, KT = 32, OT = DP / TS, ST = DP / kStep;
  __shared__ __align__(16) T sk[KT * KTile::ROW], sv[KT * VTile::ROW];
  const int group = lane_group<T>(), wave = threadIdx.x / kWave;
  int64_t w = by_die(blockIdx.x, gridDim.x);
  const int sp = static_cast<int>(w % splits);
  w /= splits;
  const int64_t r0 = w % mtiles * (TS * (W == 0 ? blockDim.x / kWave : W)) + wave * TS, r = r0 + lane_row<T>();
  const int64_t p = w / mtiles;
  const int hk = static_cast<int>(p % a.kv_heads);
  const int64_t b = p / a.kv_heads;
  const int64_t rows = a.lq * a.group, tok = r < rows ? r / a.group : 0;
  const bool busy = r0 < rows;  // a wave past the last row only helps to move keys and values
  const int head = hk * a.group + static_cast<int>(r - tok * a.group);
  const int64_t row = (b * a.lq + tok) * a.heads + head;
  const T* kp = static_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[2];
  const T* vp = static_cast<const T*>(a.v) + b * a.vs[0] + hk * a.vs[2];
  u32x4 qf[ST], gf[ST];
  row_frags<T, TINY, DP>(
      qf, r < rows ? static_cast<const T*>(a.q) + b * a.qs[0] + tok * a.qs[1] + head * a.qs[2] : nullptr, a.dim);
  row_frags<T, TINY, DP>(gf, r < rows ? static_cast<const T*>(a.dout) + row * a.dim : nullptr, a.dim);
  const float2 st = r < rows ? stats[p * rows + r] : make_float2(INFINITY, 0.f);
  const float c = a.scale * kLog2e;
  Acc<T> dq[OT];
#pragma unroll
  for (int t = 0; t < OT; ++t) dq[t] = Acc<T>{};

  const int64_t lo = sp * span, hi = lo + span < a.lk ? lo + span : a.lk;
  Keys<KT> keys(a.mask == nullptr ? nullptr : a.mask + b * a.mask_stride, lo, hi);
  int64_t key;
  uint64_t bits;
  bool more = keys.next(key, bits);
  Stage<T, TINY, KT, DP, (W == 0 ? 4 : W), (W > 0)> k(a.dim), v(a.dim);
  auto fetch = [&]() {
    k.load(kp + key * a.ks[1], a.ks[1], bits, a.dim);
    v.load(vp + key * a.vs[1], a.vs[1], bits, a.dim);
  };
  __builtin_amdgcn_s_waitcnt(kNoLoads);  // the fragments are here: the loop does not wait for them again
  if (more) fetch();
  while (more) {  // workgroup-uniform
    __syncthreads();
    k.template store<KTile::ROW>(sk, a.dim);
    v.template store<VTile::ROW>(sv, a.dim);
    __syncthreads();
    const uint32_t now = static_cast<uint32_t>(bits);
    more = keys.next(key, bits);
    if (more) fetch();
    if (!busy) continue;
    constexpr uint32_t ALL = TS == 32 ? ~0u : 0xffffu;
#pragma unroll
    for (int u = 0; u < KT / TS; ++u) {
      const uint32_t here = now >> (u * TS) & ALL;
      if (here == 0) continue;
      Acc<T> s = Acc<T>{}, dp = Acc<T>{};
#pragma unroll
      for (int e = 0; e < ST; ++e) {
        s = mma<T>(s, KTile::frag(sk, u * TS, e), qf[e]);
        dp = mma<T>(dp, VTile::frag(sv, u * TS, e), gf[e]);
      }
#pragma unroll
      for (int i = 0; i < kRegs<T>; ++i) {
        dp[i] = exp2_(fmaf(s[i], c, -st.x)) * (dp[i] - st.y);
        if (here != ALL) dp[i] = here >> (4 * group) >> mma_row<T>(i, 0) & 1 ? dp[i] : 0.f;
      }
#pragma unroll
      for (int f = 0; f < kFrags<T>; ++f) mma_fine<T, DP, KTile, true>(dq, sk, u * TS, dp, f);
    }
  }
  if (r >= rows) return;
  if (splits > 1) store_parts<T, DP>(part + (row * splits + sp) * a.dim, dq, a.dim);
  else store_columns<T, DP>(static_cast<T*>(a.dq) + row * a.dim, dq, a.scale, a.dim);
}

// dq's row tiles, and the ranges the keys are cut in where those alone leave compute units
// without work: 1,024 workgroups (2 x (300 x 6,000 tokens), 8/4 heads of 128, bf16, with dk
// and dv: 136 us, 151 with 256 workgroups and 342 uncut), of 4 waves where heads of more than
// 128 values take all registers
struct QShape {
  int w, mtiles, splits;
  int64_t span, blocks;  // blocks: of one range
  QShape(const AttArgs& a, int dtype) {
    const int64_t rows = a.lq * a.group;
    const int tile = dtype == TGX_BF16 ? 32 : 16;
    w = a.dim > 128 ? 4 : tile == 32 ? (rows <= 64 ? 2 : 4) : waves_for(ops_cdiv(rows, tile), 4, 8);
    mtiles = static_cast<int>(ops_cdiv(rows, tile * w));
    blocks = a.batch * a.kv_heads * mtiles;
    const int64_t tiles = ops_cdiv(std::max<int64_t>(a.lk, 1), 64);
    const int64_t want = blocks >= 512 ? 1 : ops_cdiv(1024, blocks);
    const int64_t per = ops_cdiv(tiles, std::min(std::min(want, ops_cdiv(tiles, 8)), int64_t(256)));
    span = per * 64;
    splits = a.dq != nullptr ? static_cast<int>(ops_cdiv(tiles, per)) : 1;
  }
};

// att_scores_q's row tiles
struct ScoresShape {
  int w, mtiles;
  explicit ScoresShape(const AttArgs& a) {
    const int64_t tiles = ops_cdiv(a.lq * a.group, kTile<float>);
    w = waves_for(tiles, 4, 8);
    mtiles = static_cast<int>(ops_cdiv(tiles, w));
  }
};

// dk's and dv's key tiles, and the ranges the rows are cut in where those alone leave half
// of the compute units without work: at most 256 workgroups, since every range writes
// its sums of all keys (1 x (2,000 x 2,000 tokens), 2/1 heads of 128, bf16: 91 us, 436 uncut;
// 2 x (300 x 6,000), 8/4 heads of 128: 136 us, 175 in three ranges)
struct KvShape {
  int least, w, ktiles, splits;
  int64_t span, sums;  // sums: values of dk's parts, and of dv's
  KvShape(const AttArgs& a, int dtype) {
    const bool bf = dtype == TGX_BF16;
    least = !bf ? 4 : a.dim > 64 && a.dim <= 128 && a.lk > 64 ? 8 : 2;
    w = waves_for(ops_cdiv(a.lk, bf ? 32 : 16), least, bf ? kv_most<bf16>(a.dim, least) : kv_most<float>(a.dim, least));
    ktiles = static_cast<int>(ops_cdiv(a.lk, (bf ? 32 : 16) * w));
    const int64_t blocks = std::max<int64_t>(a.batch * a.kv_heads * ktiles, 1), tiles = ops_cdiv(a.lq * a.group, 32);
    const int64_t want = std::max<int64_t>(256 / blocks, 1);
    const int64_t per = ops_cdiv(tiles, std::min(std::min(want, ops_cdiv(tiles, 8)), int64_t(64)));
    span = per * 32;
    splits = a.dk != nullptr || a.dv != nullptr ? static_cast<int>(ops_cdiv(tiles, per)) : 1;
    sums = splits > 1 ? a.batch * a.lk * a.kv_heads * splits * a.dim : 0;
  }
};

size_t stats_bytes(const AttArgs& a) { return ops_align(static_cast<size_t>(a.batch * a.lq * a.heads) * sizeof(float2)); }

// f32 keeps ds for dq where that is at most this much, because its matrix units, not HBM,
// bound the backward pass (400 x (65 x 65) tokens, 2 heads of 100: 142 us, 189 with three
// products for dq; 8 x (1,000 x 2,000), 4 heads of 100: 743 and 929).  att_scores_q walks over
// all keys in one workgroup, so few rows with long keys do without (1 x (300 x 6,000), 8/4
// heads of 128: 308 us, 630 with kept scores).
constexpr int64_t kMostScores = int64_t(1) << 29;

size_t scores_bytes(const AttArgs& a, int dtype) {
  if (dtype != TGX_F32 || a.dq == nullptr || (a.dk == nullptr && a.dv == nullptr) || a.lk == 0) return 0;
  if (a.lk > 1024 && QShape(a, dtype).blocks < 128) return 0;
  const int64_t rows = a.batch * a.lq * a.heads;
  return rows <= kMostScores / 4 / scores_row(a.lk) ? static_cast<size_t>(rows * scores_row(a.lk)) * 4 : 0;
}

// what dq's kernel leaves between its launches: kept scores, or the parts of its ranges
size_t q_bytes(const AttArgs& a, int dtype) {
  if (const size_t kept = scores_bytes(a, dtype)) return ops_align(kept);
  const QShape f(a, dtype);
  return f.splits > 1 ? ops_align(static_cast<size_t>(a.batch * a.lq * a.heads) * f.splits * a.dim * 4) : 0;
}

}  // namespace

size_t att_mma_backward_workspace(const AttArgs& a, int dtype) {
  return stats_bytes(a) + q_bytes(a, dtype) + static_cast<size_t>(KvShape(a, dtype).sums) * 8;
}

int att_mma_backward(const AttArgs& a, int dtype, void* ws, hipStream_t s) {
  const int64_t rows = a.batch * a.lq * a.heads;
  float2* stats = static_cast<float2*>(ws);
  float* part = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + stats_bytes(a));
  float* kv_part = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + stats_bytes(a) + q_bytes(a, dtype));
  const bool keep = scores_bytes(a, dtype) > 0;  // the same workspace holds them in the parts' place
  const KvShape kv(a, dtype);
  const QShape q(a, dtype);
  const ScoresShape sc(a);
  const int64_t problems = a.batch * a.kv_heads, kv_blocks = problems * kv.ktiles * kv.splits;
  const int64_t q_blocks = problems * (keep ? sc.mtiles : q.mtiles * q.splits);
  int fits = check_grid("tgx_attention_grad", ops_cdiv(rows, 256 / kDeltaLanes), 256);
  if (!fits && (a.dk != nullptr || a.dv != nullptr)) fits = check_grid("tgx_attention_grad", kv_blocks, 64 * kv.w);
  if (!fits && a.dq != nullptr) fits = check_grid("tgx_attention_grad", q_blocks, 64 * (keep ? sc.w : q.w));
  if (fits) return fits;
  return by_head(dtype, a.dim, [&](auto t, auto dp, auto tiny) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value, TS = kTile<T>;
    constexpr bool TINY = decltype(tiny)::value;
    hipLaunchKernelGGL(att_stats<T>, dim3(static_cast<unsigned>(ops_cdiv(rows, 256 / kDeltaLanes))), dim3(256), 0, s,
                       static_cast<const T*>(a.out), static_cast<const T*>(a.rest), static_cast<const T*>(a.dout), a.lse, rows,
                       a.lq, a.heads, a.group, a.dim, stats);
    int rc = check_launch("att_stats");
    if (rc) return rc;
    if (a.lk > 0 && (a.dk != nullptr || a.dv != nullptr)) {
      auto go = [&](auto least) {
        constexpr int LEAST = decltype(least)::value;
        const dim3 grid(static_cast<unsigned>(kv_blocks));
        if (sizeof(T) == 4 && keep)
          hipLaunchKernelGGL((att_mma_kv<T, TINY, DP, LEAST, sizeof(T) == 4>), grid, dim3(64 * kv.w), 0, s, a, kv.ktiles,
                             kv.splits, kv.span, stats, part, kv_part);
        else
          hipLaunchKernelGGL((att_mma_kv<T, TINY, DP, LEAST, false>), grid, dim3(64 * kv.w), 0, s, a, kv.ktiles, kv.splits,
                             kv.span, stats, part, kv_part);
        return check_launch("att_mma_kv");
      };
      if constexpr (kTwoWays<T, DP>)
        rc = kv.least == 8 ? go(std::integral_constant<int, 8>{}) : go(std::integral_constant<int, 2>{});
      else
        rc = go(std::integral_constant<int, kKvLeast<T, DP>>{});
      const int64_t keys = a.batch * a.lk * a.kv_heads;
      if (!rc && kv.splits > 1 && a.dk != nullptr)
        rc = att_join_sums(a.dk, keys, a.dim, dtype, a.scale, kv.splits, kv_part, s);
      if (!rc && kv.splits > 1 && a.dv != nullptr)
        rc = att_join_sums(a.dv, keys, a.dim, dtype, 1.f, kv.splits, kv_part + kv.sums, s);
      if (rc) return rc;
    }
    if (a.dq == nullptr) return TGX_OK;
    if constexpr (sizeof(T) == 4) {
      if (keep) {
        hipLaunchKernelGGL((att_scores_q<TINY, DP>), dim3(static_cast<unsigned>(q_blocks)), dim3(64 * sc.w), 0, s, a,
                           sc.mtiles, part);
        return check_launch("att_scores_q");
      }
    }
    auto go = [&](auto w) {
      hipLaunchKernelGGL((att_mma_q<T, TINY, DP, decltype(w)::value>), dim3(static_cast<unsigned>(q_blocks)),
                         dim3(64 * q.w), 0, s, a, q.mtiles, q.splits, q.span, stats, part);
      return check_launch("att_mma_q");
    };
    if constexpr (DP > 128) rc = go(std::integral_constant<int, 4>{});
    else if constexpr (sizeof(T) == 4) rc = go(std::integral_constant<int, 0>{});
    else rc = q.w == 2 ? go(std::integral_constant<int, 2>{}) : go(std::integral_constant<int, 4>{});
    return rc || q.splits == 1 ? rc : att_join_sums(a.dq, rows, a.dim, dtype, a.scale, q.splits, part, s);
  });
}

}  // namespace tgx
