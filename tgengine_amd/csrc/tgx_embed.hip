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

// one thread per pack of V values, token-major
template <typename T, int V, typename I>
__global__ __launch_bounds__(kEmbThreads) void embed_rows(const T* __restrict__ table, int64_t rows, int64_t stride,
                                                          const I* __restrict__ ids, int64_t n, int dim, int packs,
                                                          float scale, T* __restrict__ out) {
  const int64_t total = n * packs;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kEmbThreads;
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * kEmbThreads + threadIdx.x; e < total; e += step) {
    const int64_t i = e / packs;
    const int c = min(static_cast<int>(e - i * packs) * V, dim - V);
    const int64_t r = row_of(ids, i, rows);
    Pack<T, V> x;
#pragma unroll
    for (int u = 0; u < V; ++u) x.v[u] = from_f<T>(0.f);
    if (r >= 0) {
      x = load_pack<T, V>(table + r * stride + c);
#pragma unroll
      for (int u = 0; u < V; ++u) x.v[u] = from_f<T>(to_f(x.v[u]) * scale);
    }
    store_pack<T, V>(out + i * dim + c, x);
  }
}

// sort keys: the row, or `rows` for an id outside the table
template <typename I>
__global__ __launch_bounds__(kEmbThreads) void embed_keys(const I* __restrict__ ids, int64_t n, int64_t rows,
                                                          uint32_t* __restrict__ keys) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kEmbThreads + threadIdx.x;
  if (i >= n) return;
  const int64_t r = row_of(ids, i, rows);
  keys[i] = static_cast<uint32_t>(r < 0 ? rows : r);
}

// A tile is `tile` consecutive sorted tokens, taken by LT lanes (one pack of V columns
// each, further columns in turns); the workgroup's tiles lie beside each other.  A run
// of equal keys inside one tile is summed and written out; of a run that reaches into
// other tiles each tile leaves its part in 32 bits: part[2 t] for a run that the tile
// did not begin, part[2 t + 1] for one that begins in it and goes on after it.  A row's
// last pack overlaps the one before: both lanes come to the same sums there.
constexpr int kMostTile = 64;
constexpr int kAhead = 8;  // rows of one lane that are read at a time

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
// A hub's run crosses thousands of tiles; its end is searched 64 tiles a step.
template <typename T, int V, int LT>
__global__ __launch_bounds__(kEmbThreads) void embed_join(const uint32_t* __restrict__ keys, int64_t n, int64_t rows,
                                                          int tile, int dim, const float* __restrict__ part,
                                                          float scale, T* __restrict__ grad) {
  constexpr int TILES = kEmbThreads / LT;
  __shared__ float lds[TILES > 1 ? kEmbThreads * V : 1];
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
      for (int u = 0; u < V; ++u) lds[u * kEmbThreads + threadIdx.x] = acc[u];
      __syncthreads();
      if (group == 0)
#pragma unroll
        for (int u = 0; u < V; ++u)
          for (int g = 1; g < TILES; ++g) acc[u] += lds[u * kEmbThreads + g * LT + threadIdx.x];
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
int tile_of(int64_t n) { return n <= (1 << 15) ? 16 : n <= (1 << 17) ? 32 : kMostTile; }

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

}  // namespace
}  // namespace tgx

using namespace tgx;

extern "C" int tgx_embed(const void* table, int64_t rows, int64_t dim, int64_t stride, int32_t dtype, const void* ids,
                         int32_t ids_i32, int64_t n, float scale, void* out, void* stream) {
  int rc = check_embed("tgx_embed", table, out, rows, dim, dtype, ids, n);
  if (rc) return rc;
  if (stride < dim && rows > 1) return fail(TGX_ERR_ARG, "tgx_embed: row stride %lld below dim %lld",
                                            static_cast<long long>(stride), static_cast<long long>(dim));
  if (n == 0) return TGX_OK;
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto launch = [&](auto i, auto v) {
      using I = decltype(i);
      constexpr int V = decltype(v)::value;
      const int packs = static_cast<int>(ops_cdiv(dim, V));
      const int64_t blocks = std::min<int64_t>(ops_cdiv(n * packs, kEmbThreads), 1 << 20);
      hipLaunchKernelGGL((embed_rows<T, V, I>), dim3(static_cast<unsigned>(blocks)), dim3(kEmbThreads), 0,
                         static_cast<hipStream_t>(stream), static_cast<const T*>(table), rows, stride,
                         static_cast<const I*>(ids), n, static_cast<int>(dim), packs, scale, static_cast<T*>(out));
      return check_launch("embed_rows");
    };
    auto wide = [&](auto i) {
      if (dim >= kWide<T>) return launch(i, std::integral_constant<int, kWide<T>>{});
      return launch(i, std::integral_constant<int, 1>{});
    };
    return ids_i32 ? wide(int32_t{}) : wide(int64_t{});
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
  if (rows == 0) return TGX_OK;
  if (grad == nullptr) return fail(TGX_ERR_ARG, "tgx_embed_grad: grad must not be NULL");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const EmbedWs w(n, dim);
  if (n > 0 && (workspace == nullptr || workspace_bytes < w.bytes || !aligned16(workspace)))
    return fail(TGX_ERR_ARG, "tgx_embed_grad: workspace of %zu bytes, 16-byte aligned, needed", w.bytes);
  if ((rc = fill_zero(grad, static_cast<size_t>(rows) * dim * elem_bytes(dtype), s))) return rc;
  if (n == 0) return TGX_OK;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  uint32_t* k[2];
  uint32_t* v_[2];
  for (int j = 0; j < 2; ++j) {
    k[j] = reinterpret_cast<uint32_t*>(ws + w.keys[j]);
    v_[j] = reinterpret_cast<uint32_t*>(ws + w.tokens[j]);
  }
  const unsigned blocks = static_cast<unsigned>(ops_cdiv(n, kEmbThreads));
  if (ids_i32)
    hipLaunchKernelGGL(embed_keys<int32_t>, dim3(blocks), dim3(kEmbThreads), 0, s, static_cast<const int32_t*>(ids), n,
                       rows, k[0]);
  else
    hipLaunchKernelGGL(embed_keys<int64_t>, dim3(blocks), dim3(kEmbThreads), 0, s, static_cast<const int64_t*>(ids), n,
                       rows, k[0]);
  if ((rc = check_launch("embed_keys"))) return rc;
  int cur = 0;
  if ((rc = radix_sort<uint32_t>(k, v_, cur, n, key_bits(rows), w.radix, reinterpret_cast<uint32_t*>(ws + w.count),
                                 reinterpret_cast<uint32_t*>(ws + w.sums), s, true)))
    return rc;
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
      hipLaunchKernelGGL((embed_join<T, V, LT>), dim3(static_cast<unsigned>(tiles)), dim3(kEmbThreads), 0, s, k[cur], n,
                         rows, tile, static_cast<int>(dim), part, scale, static_cast<T*>(grad));
      return check_launch("embed_join");
    };
#define TGX_LANES(V, LT) launch(std::integral_constant<int, V>{}, std::integral_constant<int, LT>{})
    constexpr int W = kWide<T>;
    if (dim < W) return TGX_LANES(1, 8);
    if (dim <= 8 * W) return TGX_LANES(W, 8);
    if (dim <= 16 * W) return TGX_LANES(W, 16);
    if (dim <= 32 * W) return TGX_LANES(W, 32);
    return TGX_LANES(W, 64);
#undef TGX_LANES
  });
}
