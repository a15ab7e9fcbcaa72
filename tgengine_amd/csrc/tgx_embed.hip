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

// A tile is kTile consecutive sorted tokens.  A run of equal keys inside one tile is
// summed and written out; of a run that reaches into other tiles each tile leaves its
// part in 32 bits: part[2 t] for a run that the tile did not begin, part[2 t + 1] for
// one that begins in it and goes on after it.
constexpr int kTile = 64;

template <typename T>
__global__ __launch_bounds__(kEmbThreads) void embed_sum(const uint32_t* __restrict__ keys,
                                                         const uint32_t* __restrict__ tokens, int64_t n, int64_t rows,
                                                         int dim, const T* __restrict__ dout, float scale,
                                                         T* __restrict__ grad, float* __restrict__ part) {
  const int64_t lo = static_cast<int64_t>(blockIdx.x) * kTile;
  const int64_t hi = lo + kTile < n ? lo + kTile : n;
  const uint32_t prev = lo > 0 ? keys[lo - 1] : 0xffffffffu;
  const uint32_t next = hi < n ? keys[hi] : 0xffffffffu;
  for (int c = threadIdx.x; c < dim; c += kEmbThreads) {
    float acc = 0.f;
    for (int64_t i = lo; i < hi; ++i) {
      const uint32_t key = keys[i];
      if (key >= rows) break;  // ids outside the table come last
      acc += to_f(dout[static_cast<int64_t>(tokens[i]) * dim + c]);
      const uint32_t after = i + 1 < hi ? keys[i + 1] : next;
      if (i + 1 < hi && after == key) continue;
      // the run's end, or the tile's
      const bool from_before = key == prev && keys[lo] == key;
      const bool goes_on = i + 1 == hi && after == key;
      if (from_before) part[(2 * static_cast<int64_t>(blockIdx.x)) * dim + c] = acc;
      else if (goes_on) part[(2 * static_cast<int64_t>(blockIdx.x) + 1) * dim + c] = acc;
      else grad[static_cast<int64_t>(key) * dim + c] = from_f<T>(acc * scale);
      acc = 0.f;
    }
  }
}

// one workgroup per tile in which a run begins that later tiles go on with: its parts in tile order
template <typename T>
__global__ __launch_bounds__(kEmbThreads) void embed_join(const uint32_t* __restrict__ keys, int64_t n, int64_t rows,
                                                          int dim, const float* __restrict__ part, float scale,
                                                          T* __restrict__ grad) {
  const int64_t t = blockIdx.x;
  const int64_t hi = (t + 1) * kTile;
  if (hi >= n) return;
  const uint32_t key = keys[hi - 1];
  if (key >= rows || keys[hi] != key) return;
  if (t > 0 && keys[t * kTile] == key && keys[t * kTile - 1] == key) return;  // begun before this tile
  for (int c = threadIdx.x; c < dim; c += kEmbThreads) {
    float acc = part[(2 * t + 1) * dim + c];
    for (int64_t u = t + 1; u * kTile < n && keys[u * kTile] == key; ++u) acc += part[2 * u * dim + c];
    grad[static_cast<int64_t>(key) * dim + c] = from_f<T>(acc * scale);
  }
}

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
    o += ops_align(static_cast<size_t>(ops_cdiv(n, kTile)) * 2 * static_cast<size_t>(dim) * 4);
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
  uint32_t* v[2];
  for (int j = 0; j < 2; ++j) {
    k[j] = reinterpret_cast<uint32_t*>(ws + w.keys[j]);
    v[j] = reinterpret_cast<uint32_t*>(ws + w.tokens[j]);
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
  if ((rc = radix_sort<uint32_t>(k, v, cur, n, key_bits(rows), w.radix, reinterpret_cast<uint32_t*>(ws + w.count),
                                 reinterpret_cast<uint32_t*>(ws + w.sums), s, true)))
    return rc;
  float* part = reinterpret_cast<float*>(ws + w.part);
  const unsigned tiles = static_cast<unsigned>(ops_cdiv(n, kTile));
  return by_type(dtype, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL(embed_sum<T>, dim3(tiles), dim3(kEmbThreads), 0, s, k[cur], v[cur], n, rows,
                       static_cast<int>(dim), static_cast<const T*>(dout), scale, static_cast<T*>(grad), part);
    int e = check_launch("embed_sum");
    if (e) return e;
    hipLaunchKernelGGL(embed_join<T>, dim3(tiles), dim3(kEmbThreads), 0, s, k[cur], n, rows, static_cast<int>(dim),
                       part, scale, static_cast<T*>(grad));
    return check_launch("embed_join");
  });
}
