// Embedding lookup with scaling, and the table's gradient by sorted ids.
//
//   out[i, :]  = scale * table[id_i, :]            (0 where id_i is outside [0, N))
//   grad[n, :] = scale * sum over {i : id_i = n} of dout[i, :]
//
// The gradient sorts (id, token) stably, so that a row's tokens lie beside each
// other in token order, and sums every row in 32 bits in an order that depends on
// the ids alone: no atomics, the same bits on every call.
#include "tgx_ops.h"
#include "tgx_radix.h"

namespace tgx {
namespace {

constexpr int kEmbThreads = 256;

template <typename I>
__device__ __forceinline__ int64_t row_of(const I* __restrict__ ids, int64_t i, int64_t rows) {
  const int64_t r = static_cast<int64_t>(ids[i]);
  return r >= 0 && r < rows ? r : -1;
}

// LT lanes take a token's row, a pack of V values each (further packs in turns), and
// kRowsAhead tokens at a time: their ids, then their rows, are in flight together.  What
// bounds it is writing the rows, behind two dependent reads: 240,000 x 100 bf16 (48 MB
// written) 16 us, 3.0 TB/s; 19,200 x 172 f32 (13 MB) 5.9 us; 120 x 32 f32 2.0 us.
constexpr int kRowsAhead = 4;

template <typename T, int V, int LT, typename I>
__global__ __launch_bounds__(kEmbThreads) void embed_rows(const T* __restrict__ table, int64_t rows, int64_t stride,
                                                          const I* __restrict__ ids, int64_t n, int dim, float scale,
                                                          T* __restrict__ out) {
  constexpr int GROUPS = kEmbThreads / LT;
  const int64_t step = static_cast<int64_t>(gridDim.x) * GROUPS * kRowsAhead;
  for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * GROUPS * kRowsAhead + threadIdx.x / LT; i0 < n; i0 += step) {
    int64_t r[kRowsAhead];
#pragma unroll
    for (int a = 0; a < kRowsAhead; ++a) r[a] = i0 + a * GROUPS < n ? row_of(ids, i0 + a * GROUPS, rows) : -1;
    for (int c = (threadIdx.x % LT) * V; c < dim; c += LT * V) {
      const int col = min(c, dim - V);
      Pack<T, V> x[kRowsAhead];
#pragma unroll
      for (int a = 0; a < kRowsAhead; ++a) {
#pragma unroll
        for (int u = 0; u < V; ++u) x[a].v[u] = from_f<T>(0.f);
        if (r[a] >= 0) x[a] = load_pack<T, V>(table + r[a] * stride + col);
      }
#pragma unroll
      for (int a = 0; a < kRowsAhead; ++a) {
        if (i0 + a * GROUPS >= n) break;
        if (r[a] >= 0)
#pragma unroll
          for (int u = 0; u < V; ++u) x[a].v[u] = from_f<T>(to_f(x[a].v[u]) * scale);
        store_pack<T, V>(out + (i0 + a * GROUPS) * dim + col, x[a]);
      }
    }
  }
}

// calls f(V, LT) with the pack and the lanes that rows of `dim` values take: 16 bytes a
// lane, as many lanes as the row has packs, up to a wave; rows shorter than a pack one value
// a lane
template <typename T, typename F>
int by_row(int64_t dim, F&& f) {
#define TGX_LANES(V, LT) f(std::integral_constant<int, V>{}, std::integral_constant<int, LT>{})
  constexpr int W = kWide<T>;
  if (dim < W) return TGX_LANES(1, 8);
  if (dim <= 8 * W) return TGX_LANES(W, 8);
  if (dim <= 16 * W) return TGX_LANES(W, 16);
  if (dim <= 32 * W) return TGX_LANES(W, 32);
  return TGX_LANES(W, 64);
#undef TGX_LANES
}

// The sort's keys are the rows, and `rows` for an id outside the table.

// Up to kSmallTokens tokens: workgroup 0 sorts them alone, each thread holding ITEMS keys
// (a wave's lie beside each other) and LDS one array of them; the other workgroups write
// the gradient's zeros meanwhile.  A pass ranks the keys of each wave by ballots, counts
// digits per wave, and moves keys, then tokens, through the LDS array: one launch in
// place of four.  Latency bounds it.  The whole gradient of 9,000 x 172 f32 rows takes 17 us
// for 2,000 tokens and 27 for 8,000; with the launches of more tokens 28 and 30.
constexpr int kSmallThreads = 1024;
constexpr int kSmallWaves = kSmallThreads / kWave;
constexpr int kSmallItems = 8;  // 24 keys a thread do not fit the registers: 19,200 tokens took 601 us
constexpr int kSmallBits = 9;  // of a pass
constexpr int64_t kSmallTokens = int64_t(kSmallThreads) * kSmallItems;

constexpr size_t small_lds(int items) {
  return static_cast<size_t>(kSmallThreads) * items * 4 + kSmallWaves * (size_t(2) << kSmallBits);
}
static_assert(small_lds(kSmallItems) <= 48 * 1024, "what any launch may have without asking");

template <int ITEMS, typename I>
__global__ __launch_bounds__(kSmallThreads) void embed_small_sort(const I* __restrict__ ids, int n, int64_t rows,
                                                                  int bits, uint32_t* __restrict__ keys,
                                                                  uint32_t* __restrict__ tokens,
                                                                  uint8_t* __restrict__ zero, int head, int64_t n16,
                                                                  int tail) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ uint32_t wsum[kSmallWaves];
  if (blockIdx.x > 0) {
    const int64_t t = static_cast<int64_t>(blockIdx.x - 1) * kSmallThreads + threadIdx.x;
    zero_bytes(zero, head, n16, tail, t, static_cast<int64_t>(gridDim.x - 1) * kSmallThreads);
    return;
  }
  uint32_t* buf = reinterpret_cast<uint32_t*>(smem);
  uint16_t* count = reinterpret_cast<uint16_t*>(smem + static_cast<size_t>(kSmallThreads) * ITEMS * 4);
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const uint64_t below_mask = (uint64_t(1) << lane) - 1;
  const int i0 = wave * (kWave * ITEMS) + lane;
  uint32_t k[ITEMS], v[ITEMS], rank[ITEMS];
#pragma unroll
  for (int r = 0; r < ITEMS; ++r) {
    const int i = i0 + r * kWave;
    const int64_t row = i < n ? row_of(ids, i, rows) : -1;
    k[r] = static_cast<uint32_t>(row < 0 ? rows : row);
    v[r] = static_cast<uint32_t>(i);
  }
  int passes = (bits + kSmallBits - 1) / kSmallBits;
  for (int shift = 0; shift < bits; --passes) {  // workgroup-uniform
    const int dbits = (bits - shift + passes - 1) / passes, bins = 1 << dbits;
    uint16_t* mine = count + (wave << dbits);
    for (int d = lane; d < bins; d += kWave) mine[d] = 0;
    sort_wave_sync();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r) {
      const bool valid = i0 + r * kWave < n;
      const int d = digit_of(k[r], shift, bins);
      uint64_t peers = __ballot(valid);
      for (int bit = 0; bit < dbits; ++bit) {
        const bool on = d >> bit & 1;
        const uint64_t m = __ballot(on);
        peers &= on ? m : ~m;
      }
      const uint32_t before = valid ? mine[d] : 0u;
      sort_wave_sync();  // every lane has read its counter
      const uint32_t below = static_cast<uint32_t>(__popcll(peers & below_mask));
      if (valid && below == 0) mine[d] = static_cast<uint16_t>(before + __popcll(peers));
      sort_wave_sync();
      rank[r] = before + below;
    }
    __syncthreads();
    uint32_t sum = 0, all;
    if (static_cast<int>(threadIdx.x) < bins)
      for (int w = 0; w < kSmallWaves; ++w) sum += count[(w << dbits) + threadIdx.x];
    uint32_t at = block_exclusive<kSmallThreads>(sum, wsum, all);
    if (static_cast<int>(threadIdx.x) < bins)
      for (int w = 0; w < kSmallWaves; ++w) {
        const uint32_t c = count[(w << dbits) + threadIdx.x];
        count[(w << dbits) + threadIdx.x] = static_cast<uint16_t>(at);
        at += c;
      }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r)
      if (i0 + r * kWave < n) {
        rank[r] += mine[digit_of(k[r], shift, bins)];
        buf[rank[r]] = k[r];
      }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r)
      if (i0 + r * kWave < n) k[r] = buf[i0 + r * kWave];
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r)
      if (i0 + r * kWave < n) buf[rank[r]] = v[r];
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ITEMS; ++r)
      if (i0 + r * kWave < n) v[r] = buf[i0 + r * kWave];
    __syncthreads();
    shift += dbits;
  }
#pragma unroll
  for (int r = 0; r < ITEMS; ++r)
    if (i0 + r * kWave < n) {
      keys[i0 + r * kWave] = k[r];
      tokens[i0 + r * kWave] = v[r];
    }
}

// More tokens: the first `ranges` workgroups write the keys and count the first pass's
// digits as radix_hist does, the others write the gradient's zeros, whose bytes bound it
// where the table is large: 1,000,000 x 100 bf16 rows (200 MB) 31 us, 6.5 TB/s.
template <typename I>
__global__ __launch_bounds__(kSortThreads) void embed_keys(const I* __restrict__ ids, int64_t n, int64_t range,
                                                           int64_t rows, int bins, int ranges,
                                                           uint32_t* __restrict__ keys, uint32_t* __restrict__ count,
                                                           uint8_t* __restrict__ zero, int head, int64_t n16,
                                                           int tail) {
  __shared__ uint32_t h[kMaxBins * kHistCopies];
  if (static_cast<int>(blockIdx.x) >= ranges) {
    const int64_t t = static_cast<int64_t>(blockIdx.x - ranges) * kSortThreads + threadIdx.x;
    zero_bytes(zero, head, n16, tail, t, static_cast<int64_t>(gridDim.x - ranges) * kSortThreads);
    return;
  }
  for (int i = threadIdx.x; i < bins * kHistCopies; i += kSortThreads) h[i] = 0;
  __syncthreads();
  const int64_t lo = blockIdx.x * range, hi = lo + range < n ? lo + range : n;
  uint32_t* mine = h + (threadIdx.x & (kHistCopies - 1));
#pragma unroll 4
  for (int64_t i = lo + threadIdx.x; i < hi; i += kSortThreads) {
    const int64_t r = row_of(ids, i, rows);
    const uint32_t k = static_cast<uint32_t>(r < 0 ? rows : r);
    keys[i] = k;
    atomicAdd(&mine[digit_of(k, 0, bins) * kHistCopies], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < bins; d += kSortThreads) {
    uint32_t c = 0;
#pragma unroll
    for (int u = 0; u < kHistCopies; ++u) c += h[d * kHistCopies + u];
    count[static_cast<int64_t>(d) * ranges + blockIdx.x] = c;
  }
}

// A tile is `tile` consecutive sorted tokens, taken by LT lanes (one pack of V columns
// each, further columns in turns); the workgroup's tiles lie beside each other.  A run
// of equal keys inside one tile is summed and written out; of a run that reaches into
// other tiles each tile leaves its part in 32 bits: part[2 t] for a run that the tile
// did not begin, part[2 t + 1] for one that begins in it and goes on after it.  A row's
// last pack overlaps the one before: both lanes come to the same sums there.
// Bounded by the reads of rows in the ids' order: 167,644 rows of 200 bytes (34 MB) in 22 us.
constexpr int kMostTile = 64;
constexpr int kAhead = 16;  // rows of one lane that are read at a time

template <typename T, int V, int LT>
__global__ __launch_bounds__(kEmbThreads) void embed_sum(const uint32_t* __restrict__ keys,
                                                         const uint32_t* __restrict__ tokens, int64_t n, int64_t rows,
                                                         int tile, int dim, const T* __restrict__ dout, float scale,
                                                         T* __restrict__ grad, float* __restrict__ part) {
  constexpr int TILES = kEmbThreads / LT;
  __shared__ uint32_t skey[TILES * kMostTile + 2], stok[TILES * kMostTile];
  const int64_t first = static_cast<int64_t>(blockIdx.x) * TILES * tile;
  // skey[i + 1]: key of the block's token i; 0xffffffff before the first and after the last
  for (int i = threadIdx.x; i < TILES * tile + 2; i += kEmbThreads) {
    const int64_t j = first + i - 1;
    skey[i] = j >= 0 && j < n ? keys[j] : 0xffffffffu;
    if (i < TILES * tile) stok[i] = j + 1 < n ? tokens[j + 1] : 0u;
  }
  __syncthreads();
  const int64_t t = static_cast<int64_t>(blockIdx.x) * TILES + threadIdx.x / LT;
  const uint32_t* key = skey + 1 + threadIdx.x / LT * tile;
  const uint32_t* tok = stok + threadIdx.x / LT * tile;
  // ids outside the table come last
  int count = 0;
  for (int step = kMostTile; step > 0; step >>= 1)
    if (count + step <= tile && key[count + step - 1] < rows) count += step;
  const bool from_before = count > 0 && key[0] == key[-1];
  for (int c = (threadIdx.x % LT) * V; c < dim; c += LT * V) {
    const int col = min(c, dim - V);
    float acc[V];
#pragma unroll
    for (int u = 0; u < V; ++u) acc[u] = 0.f;
    bool head = from_before;
    for (int i0 = 0; i0 < count; i0 += kAhead) {
      Pack<T, V> x[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        x[i] = load_pack<T, V>(dout + static_cast<int64_t>(tok[min(i0 + i, count - 1)]) * dim + col);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (i0 + i >= count) break;
#pragma unroll
        for (int u = 0; u < V; ++u) acc[u] += to_f(x[i].v[u]);
        const uint32_t k = key[i0 + i];
        const bool last = i0 + i + 1 == tile;
        if (key[i0 + i + 1] == k && !last) continue;
        // the run's end, or the tile's
        if (head || (last && key[i0 + i + 1] == k)) {
          Pack<float, V> y;
#pragma unroll
          for (int u = 0; u < V; ++u) y.v[u] = acc[u];
          store_pack<float, V>(part + (2 * t + (head ? 0 : 1)) * dim + col, y);
        } else {
          Pack<T, V> y;
#pragma unroll
          for (int u = 0; u < V; ++u) y.v[u] = from_f<T>(acc[u] * scale);
          store_pack<T, V>(grad + static_cast<int64_t>(k) * dim + col, y);
        }
        head = false;
#pragma unroll
        for (int u = 0; u < V; ++u) acc[u] = 0.f;
      }
    }
  }
}

// One workgroup per tile in which a run begins that later tiles go on with: its parts,
// every TILES-th of them summed by one group of lanes, then the groups' sums in order.
// A hub's run crosses thousands of tiles; its end is searched 64 tiles a step.  The largest
// run bounds it: 17 us where one row has over a third of 167,644 tokens.
constexpr int kJoinThreads = 512;

template <typename T, int V, int LT>
__global__ __launch_bounds__(kJoinThreads) void embed_join(const uint32_t* __restrict__ keys, int64_t n, int64_t rows,
                                                          int tile, int dim, const float* __restrict__ part,
                                                          float scale, T* __restrict__ grad) {
  constexpr int TILES = kJoinThreads / LT;
  __shared__ float lds[TILES > 1 ? kJoinThreads * V : 1];
  const int64_t t = blockIdx.x;
  const int64_t hi = (t + 1) * tile;
  if (hi >= n) return;
  const uint32_t key = keys[hi - 1];
  if (key >= rows || keys[hi] != key) return;
  if (t > 0 && keys[t * tile] == key && keys[t * tile - 1] == key) return;  // begun before this tile
  // tiles t + 1 .. end - 1 begin with the key
  int64_t lo = t + 1, end = (n + tile - 1) / tile;  // lo does, end does not
  while (end - lo > 1) {
    const int64_t step = (end - lo + kWave - 1) / kWave;
    const int64_t at = lo + (threadIdx.x & (kWave - 1)) * step;
    const uint64_t with = __ballot(at < end && keys[min(at, end - 1) * tile] == key);
    const int last = 63 - __builtin_clzll(with);  // lane 0's is
    end = min(end, lo + (last + 1) * step);
    lo += last * step;
  }
  const int group = threadIdx.x / LT;
  for (int c0 = 0; c0 < dim; c0 += LT * V) {  // workgroup-uniform
    const int c = c0 + (threadIdx.x % LT) * V, col = min(c, dim - V);
    float acc[V];
#pragma unroll
    for (int u = 0; u < V; ++u) acc[u] = 0.f;
    if (c < dim) {
      if (group == 0) {
        const Pack<float, V> x = load_pack<float, V>(part + (2 * t + 1) * dim + col);
#pragma unroll
        for (int u = 0; u < V; ++u) acc[u] = x.v[u];
      }
#pragma unroll 8
      for (int64_t y = t + 1 + group; y < end; y += TILES) {
        const Pack<float, V> x = load_pack<float, V>(part + 2 * y * dim + col);
#pragma unroll
        for (int u = 0; u < V; ++u) acc[u] += x.v[u];
      }
    }
    if constexpr (TILES > 1) {
      __syncthreads();
#pragma unroll
      for (int u = 0; u < V; ++u) lds[u * kJoinThreads + threadIdx.x] = acc[u];
      __syncthreads();
      if (group == 0)
#pragma unroll
        for (int u = 0; u < V; ++u)
          for (int g = 1; g < TILES; ++g) acc[u] += lds[u * kJoinThreads + g * LT + threadIdx.x];
    }
    if (group == 0 && c < dim) {
      Pack<T, V> y;
#pragma unroll
      for (int u = 0; u < V; ++u) y.v[u] = from_f<T>(acc[u] * scale);
      store_pack<T, V>(grad + static_cast<int64_t>(key) * dim + col, y);
    }
  }
}

// tokens per tile: short ones spread few tokens over the device, long ones leave fewer parts
// (the gradient by 16, 32 and 64: 19,200 tokens x 172 f32 34, 34 and 39 us; 100,000 x 100
// bf16 85, 83 and 84; 1,000,000 462, 339 and 274)
int tile_of(int64_t n) { return n <= (1 << 15) ? 16 : n <= (1 << 17) ? 32 : kMostTile; }

// embed_join takes kJoinThreads threads for every tile, and a grid fewer than 2^32
constexpr int64_t kMostGradTokens = ((int64_t(1) << 32) / kJoinThreads - 1) * kMostTile;

int check_embed(const char* what, const void* a, const void* b, int64_t rows, int64_t dim, int32_t dtype,
                const void* ids, int64_t n) {
  if (rows < 0 || dim < 1 || n < 0) return fail(TGX_ERR_ARG, "%s: rows=%lld dim=%lld n=%lld", what,
                                                static_cast<long long>(rows), static_cast<long long>(dim),
                                                static_cast<long long>(n));
  if (elem_bytes(dtype) == 0) return fail(TGX_ERR_DTYPE, "%s: dtype %d", what, dtype);
  if (dim > TGX_MAX_EMBED_DIM || rows >= (int64_t(1) << 31) || n >= (int64_t(1) << 31))
    return fail(TGX_ERR_LIMIT, "%s: dim=%lld (at most %d), rows=%lld, n=%lld (below 2^31)", what,
                static_cast<long long>(dim), TGX_MAX_EMBED_DIM, static_cast<long long>(rows),
                static_cast<long long>(n));
  if (n > 0 && (ids == nullptr || b == nullptr || (rows > 0 && a == nullptr)))
    return fail(TGX_ERR_ARG, "%s: table, ids and rows must not be NULL", what);
  return TGX_OK;
}

int key_bits(int64_t rows) {  // the keys are 0 .. rows
  int bits = 1;
  while ((int64_t(1) << bits) <= rows) ++bits;
  return bits;
}

// workspace: two key and two token buffers, the sort's counts, the tiles' parts
struct EmbedWs {
  size_t keys[2], tokens[2], count, sums, part, bytes;
  RadixScratch radix;
  EmbedWs(int64_t n, int64_t dim) : radix(radix_scratch(n)) {
    size_t o = 0;
    for (int j = 0; j < 2; ++j) {
      keys[j] = o;
      o += ops_align(static_cast<size_t>(n) * 4);
      tokens[j] = o;
      o += ops_align(static_cast<size_t>(n) * 4);
    }
    count = o;
    o += radix.count_bytes;
    sums = o;
    o += radix.sums_bytes;
    part = o;
    o += ops_align(static_cast<size_t>(ops_cdiv(n, tile_of(n))) * 2 * static_cast<size_t>(dim) * 4);
    bytes = o;
  }
};

// Ranges whose counts each workgroup of the sort's scatter adds up itself: a launch less
// for every pass (the gradient of 19,200 tokens: 33 us, 41 with it; 40,000: 39 and 45)
constexpr int kRawRanges = 32;

// the tokens of `ids` in the stable order of their rows: keys in k[cur], tokens in
// v[cur]; the gradient's zeros are written on the way
template <typename I>
int sort_tokens(const I* ids, int64_t n, int64_t rows, const EmbedWs& w, const ZeroSpan& z, uint8_t* ws,
                uint32_t* k[2], uint32_t* v[2], int& cur, hipStream_t s) {
  const int bits = key_bits(rows);
  if (n <= kSmallTokens) {
    const unsigned blocks = 1 + static_cast<unsigned>(std::clamp<int64_t>(ops_cdiv(z.n16, 4 * kSmallThreads), 1, 512));
    auto go = [&](auto items) {
      constexpr int ITEMS = decltype(items)::value;
      hipLaunchKernelGGL((embed_small_sort<ITEMS, I>), dim3(blocks), dim3(kSmallThreads), small_lds(ITEMS), s, ids,
                         static_cast<int>(n), rows, bits, k[0], v[0], z.p, z.head, z.n16, z.tail);
      return check_launch("embed_small_sort");
    };
    cur = 0;
    if (n <= 2 * kSmallThreads) return go(std::integral_constant<int, 2>{});
    return go(std::integral_constant<int, kSmallItems>{});
  }
  uint32_t* count = reinterpret_cast<uint32_t*>(ws + w.count);
  uint32_t* sums = reinterpret_cast<uint32_t*>(ws + w.sums);
  const int passes = static_cast<int>(cdiv(bits, kMaxDigitBits)), dbits = static_cast<int>(cdiv(bits, passes));
  const int ranges = static_cast<int>(w.radix.nblocks);
  const unsigned blocks = static_cast<unsigned>(ranges + std::clamp<int64_t>(ops_cdiv(z.n16, 4 * kSortThreads), 1, 2048));
  hipLaunchKernelGGL(embed_keys<I>, dim3(blocks), dim3(kSortThreads), 0, s, ids, n, w.radix.range, rows, 1 << dbits,
                     ranges, k[0], count, z.p, z.head, z.n16, z.tail);
  int rc = check_launch("embed_keys");
  if (rc) return rc;
  cur = 0;
  for (int shift = 0, left = passes; rc == TGX_OK && shift < bits; --left) {
    const int d = static_cast<int>(cdiv(bits - shift, left));
    const uint32_t* vin = shift == 0 ? nullptr : v[cur];  // the tokens in order at first
    if (shift > 0 || ranges > kRawRanges) {
      if (shift == 0) {
        hipLaunchKernelGGL(radix_rows, dim3(1u << d), dim3(kThreads), 0, s, count, ranges, sums);
        if ((rc = check_launch("radix_rows"))) return rc;
        rc = w.radix.items == 4
                 ? radix_scatter_launch<uint32_t, 4>(k[0], vin, k[1], v[1], n, 0, d, w.radix, count, sums, s)
                 : radix_scatter_launch<uint32_t, 8>(k[0], vin, k[1], v[1], n, 0, d, w.radix, count, sums, s);
      } else if (ranges > kRawRanges) {
        rc = radix_pass<uint32_t>(k[cur], vin, k[1 - cur], v[1 - cur], n, shift, d, w.radix, count, sums, s);
      } else {
        hipLaunchKernelGGL(radix_hist<uint32_t>, dim3(ranges), dim3(kSortThreads), (size_t(4) << d) * kHistCopies, s,
                           k[cur], n, w.radix.range, shift, 1 << d, count);
        if ((rc = check_launch("radix_hist"))) return rc;
      }
    }
    if (ranges <= kRawRanges)
      rc = radix_scatter_launch<uint32_t, 4, true>(k[cur], vin, k[1 - cur], v[1 - cur], n, shift, d, w.radix, count,
                                                   sums, s);
    cur = 1 - cur;
    shift += d;
  }
  return rc;
}

}  // namespace
}  // namespace tgx

using namespace tgx;

extern "C" int tgx_embed(const void* table, int64_t rows, int64_t dim, int64_t stride, int32_t dtype, const void* ids,
                         int32_t ids_i32, int64_t n, float scale, void* out, void* stream) {
  int rc = check_embed("tgx_embed", table, out, rows, dim, dtype, ids, n);
  if (rc) return rc;
  if (stride < dim && stride != 0 && rows > 1) return fail(TGX_ERR_ARG, "tgx_embed: row stride %lld below dim %lld",
                                            static_cast<long long>(stride), static_cast<long long>(dim));
  if (n == 0) return TGX_OK;
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    return by_row<T>(dim, [&](auto v, auto lt) {
      constexpr int V = decltype(v)::value, LT = decltype(lt)::value;
      const int64_t blocks = std::min<int64_t>(ops_cdiv(n, kEmbThreads / LT * kRowsAhead), 1 << 20);
      auto launch = [&](auto i) {
        using I = decltype(i);
        hipLaunchKernelGGL((embed_rows<T, V, LT, I>), dim3(static_cast<unsigned>(blocks)), dim3(kEmbThreads), 0,
                           static_cast<hipStream_t>(stream), static_cast<const T*>(table), rows, stride,
                           static_cast<const I*>(ids), n, static_cast<int>(dim), scale, static_cast<T*>(out));
        return check_launch("embed_rows");
      };
      return ids_i32 ? launch(int32_t{}) : launch(int64_t{});
    });
  });
}

extern "C" size_t tgx_embed_grad_workspace_size(int64_t n, int64_t dim) {
  if (n <= 0 || dim <= 0) return 0;
  return EmbedWs(n, dim).bytes;
}

extern "C" int tgx_embed_grad(const void* dout, const void* ids, int32_t ids_i32, int64_t n, int64_t rows, int64_t dim,
                              int32_t dtype, float scale, void* grad, void* workspace, size_t workspace_bytes,
                              void* stream) {
  int rc = check_embed("tgx_embed_grad", grad, dout, rows, dim, dtype, ids, n);
  if (rc) return rc;
  if (n > kMostGradTokens)
    return fail(TGX_ERR_LIMIT, "tgx_embed_grad: n=%lld (at most 2^29 - 64)", static_cast<long long>(n));
  if (rows == 0) return TGX_OK;
  if (grad == nullptr) return fail(TGX_ERR_ARG, "tgx_embed_grad: grad must not be NULL");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const EmbedWs w(n, dim);
  if (n > 0 && (workspace == nullptr || workspace_bytes < w.bytes || !aligned16(workspace)))
    return fail(TGX_ERR_ARG, "tgx_embed_grad: workspace of %zu bytes, 16-byte aligned, needed", w.bytes);
  const ZeroSpan z(grad, static_cast<size_t>(rows) * dim * elem_bytes(dtype));
  if (n == 0) return fill_zero(grad, z.bytes, s);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  uint32_t* k[2];
  uint32_t* v_[2];
  for (int j = 0; j < 2; ++j) {
    k[j] = reinterpret_cast<uint32_t*>(ws + w.keys[j]);
    v_[j] = reinterpret_cast<uint32_t*>(ws + w.tokens[j]);
  }
  int cur = 0;
  rc = ids_i32 ? sort_tokens(static_cast<const int32_t*>(ids), n, rows, w, z, ws, k, v_, cur, s)
               : sort_tokens(static_cast<const int64_t*>(ids), n, rows, w, z, ws, k, v_, cur, s);
  if (rc) return rc;
  float* part = reinterpret_cast<float*>(ws + w.part);
  const int tile = tile_of(n);
  const int64_t tiles = ops_cdiv(n, tile);
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto launch = [&](auto v, auto lt) {
      constexpr int V = decltype(v)::value, LT = decltype(lt)::value;
      hipLaunchKernelGGL((embed_sum<T, V, LT>), dim3(static_cast<unsigned>(ops_cdiv(tiles, kEmbThreads / LT))),
                         dim3(kEmbThreads), 0, s, k[cur], v_[cur], n, rows, tile, static_cast<int>(dim),
                         static_cast<const T*>(dout), scale, static_cast<T*>(grad), part);
      const int e = check_launch("embed_sum");
      if (e) return e;
      hipLaunchKernelGGL((embed_join<T, V, LT>), dim3(static_cast<unsigned>(tiles)), dim3(kJoinThreads), 0, s, k[cur], n,
                         rows, tile, static_cast<int>(dim), part, scale, static_cast<T*>(grad));
      return check_launch("embed_join");
    };
    return by_row<T>(dim, launch);
  });
}
