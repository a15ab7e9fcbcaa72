// The global norm of many gradients, and the gradients clipped by it.
//
//   norm = sqrt(sum over all tensors of g^2),  c = min(1, max_norm / (norm + 1e-6)),  out = c g
//
// Two launches over all tensors together: each workgroup leaves the norm of its part in
// part[block], and in the second launch every workgroup adds up their squares in the same
// order and scales its part.  Squares and sums are of 64 bits: in 32 those of values above
// 2^64, as a run that diverges has them, are infinite, and clipping would make zeros of the
// gradients.  The tensors' addresses travel in the kernels' arguments, kList tensors a
// launch.  HBM bounds large lists: 100,000,000 bf16 values (200 MB) and 25 small tensors
// take the squares 38 us, 5.4 TB/s, and the scaling 73 us, 5.6 TB/s; 48 layers of up to
// 20,000 f32 values take 4.4 and 6.2 us, mostly the launches.  2,048 parts fill the 256
// compute units with eight workgroups each, and a part is long enough to hide its sum.
#include "tgx_ops.h"

#include <memory>
#include <new>

namespace tgx {
namespace {

constexpr int kClipThreads = 256;
constexpr int kClipWaves = kClipThreads / kWave;
constexpr int kList = 112;          // tensors per launch: their table stays below the 4 KB of kernel arguments
constexpr int64_t kMostParts = 2048;  // parts of all tensors together, about
constexpr int64_t kLeastPart = 8192;  // values

struct ClipList {
  const void* in[kList];
  void* out[kList];
  int64_t size[kList];
  uint32_t first[kList + 1];  // first part of each tensor among this launch's
  uint8_t in_bf16[kList], out_bf16[kList];
  int32_t count;
};
static_assert(sizeof(ClipList) <= 3800, "kernel arguments");

// the tensor that this workgroup's part belongs to
__device__ __forceinline__ int tensor_of(const ClipList& l, uint32_t block) {
  int lo = 0, hi = l.count;  // first[lo] <= block < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (l.first[mid] <= block) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <typename T>
__device__ __forceinline__ double squares(const T* __restrict__ p, int64_t lo, int64_t hi) {
  constexpr int V = kWide<T>;
  double s[V];
#pragma unroll
  for (int u = 0; u < V; ++u) s[u] = 0.0;
  const int64_t full = lo + (hi - lo) / V * V;
#pragma unroll 4
  for (int64_t i = lo + static_cast<int64_t>(threadIdx.x) * V; i < full; i += kClipThreads * V) {
    const Pack<T, V> x = load_pack<T, V>(p + i);
#pragma unroll
    for (int u = 0; u < V; ++u) {
      const double f = to_f(x.v[u]);
      s[u] = fma(f, f, s[u]);
    }
  }
  if (full + threadIdx.x < hi) {
    const double x = to_f(p[full + threadIdx.x]);
    s[0] = fma(x, x, s[0]);
  }
#pragma unroll
  for (int w = V / 2; w > 0; w /= 2)
#pragma unroll
    for (int u = 0; u < w; ++u) s[u] += s[u + w];
  return s[0];
}

__global__ __launch_bounds__(kClipThreads) void clip_squares(const ClipList l, int64_t per, float* __restrict__ part) {
  __shared__ double lds[kClipWaves];
  const int t = tensor_of(l, blockIdx.x);
  const int64_t lo = (blockIdx.x - l.first[t]) * per;
  const int64_t hi = lo + per < l.size[t] ? lo + per : l.size[t];
  double s = l.in_bf16[t] ? squares(static_cast<const bf16*>(l.in[t]), lo, hi)
                          : squares(static_cast<const float*>(l.in[t]), lo, hi);
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) s += __shfl_xor(s, off, kWave);
  if ((threadIdx.x & (kWave - 1)) == 0) lds[threadIdx.x / kWave] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x] = static_cast<float>(sqrt((lds[0] + lds[1]) + (lds[2] + lds[3])));
}

template <typename T, typename U>
__device__ __forceinline__ void scaled(const T* p, U* q, int64_t lo, int64_t hi, float by) {
  constexpr int V = kWide<T>;
  const int64_t full = lo + (hi - lo) / V * V;
#pragma unroll 4
  for (int64_t i = lo + static_cast<int64_t>(threadIdx.x) * V; i < full; i += kClipThreads * V) {
    const Pack<T, V> x = load_pack<T, V>(p + i);
    Pack<U, V> y;
#pragma unroll
    for (int u = 0; u < V; ++u) y.v[u] = from_f<U>(to_f(x.v[u]) * by);
    store_pack<U, V>(q + i, y);
  }
  if (full + threadIdx.x < hi) q[full + threadIdx.x] = from_f<U>(to_f(p[full + threadIdx.x]) * by);
}

__global__ __launch_bounds__(kClipThreads) void clip_scale(const ClipList l, int64_t per, const float* __restrict__ part,
                                                           int parts, float max_norm, float* __restrict__ norm,
                                                           bool first) {
  __shared__ double lds[kClipWaves];
  double s = 0.0;
  for (int i = threadIdx.x; i < parts; i += kClipThreads) s = fma(static_cast<double>(part[i]), static_cast<double>(part[i]), s);
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) s += __shfl_xor(s, off, kWave);
  if ((threadIdx.x & (kWave - 1)) == 0) lds[threadIdx.x / kWave] = s;
  __syncthreads();
  const float total = static_cast<float>(sqrt((lds[0] + lds[1]) + (lds[2] + lds[3])));
  if (first && blockIdx.x == 0 && threadIdx.x == 0) *norm = total;
  if (blockIdx.x >= l.first[l.count]) return;  // a launch of no parts still writes the norm
  float by = max_norm / (total + 1e-6f);
  by = by > 1.f ? 1.f : by;  // NaN stays
  // from the last part to the first: what the sums read last is still in the caches
  const uint32_t at = l.first[l.count] - 1 - blockIdx.x;
  const int t = tensor_of(l, at);
  if (by == 1.f && l.in[t] == l.out[t]) return;  // nothing changes
  const int64_t lo = (at - l.first[t]) * per;
  const int64_t hi = lo + per < l.size[t] ? lo + per : l.size[t];
  if (l.in_bf16[t]) {
    if (l.out_bf16[t]) scaled(static_cast<const bf16*>(l.in[t]), static_cast<bf16*>(l.out[t]), lo, hi, by);
    else scaled(static_cast<const bf16*>(l.in[t]), static_cast<float*>(l.out[t]), lo, hi, by);
  } else {
    if (l.out_bf16[t]) scaled(static_cast<const float*>(l.in[t]), static_cast<bf16*>(l.out[t]), lo, hi, by);
    else scaled(static_cast<const float*>(l.in[t]), static_cast<float*>(l.out[t]), lo, hi, by);
  }
}

// values per part: at least kLeastPart, and as many as keep the parts near kMostParts
int64_t part_values(const int64_t* sizes, int64_t count) {
  int64_t all = 0;
  for (int64_t i = 0; i < count; ++i) all += sizes[i];
  const int64_t per = std::max(kLeastPart, ops_cdiv(all, kMostParts));
  return ops_cdiv(per, kClipThreads * 8) * (kClipThreads * 8);
}

int64_t part_count(const int64_t* sizes, int64_t count, int64_t per) {
  int64_t parts = 0;
  for (int64_t i = 0; i < count; ++i) parts += ops_cdiv(sizes[i], per);
  return parts;
}

// Workgroups write all outputs at once, in no order: bytes that are written may not be
// written or read for another tensor.  A tensor that is its own output counts as one.
int check_apart(const void* const* grads, const int32_t* dtypes, void* const* outs, const int32_t* out_dtypes,
                const int64_t* sizes, int64_t count) {
  struct Range {
    uint64_t lo, hi;
    int64_t tensor;
    bool out;
  };
  const std::unique_ptr<Range[]> r(new (std::nothrow) Range[static_cast<size_t>(count) * 2]);
  if (r == nullptr) return fail(TGX_ERR_LIMIT, "tgx_clip_grad_norm: no memory to check %lld tensors", static_cast<long long>(count));
  int64_t n = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (sizes[i] == 0) continue;
    r[n++] = {addr(outs[i]), addr(outs[i]) + static_cast<uint64_t>(sizes[i]) * elem_bytes(out_dtypes[i]), i, true};
    if (grads[i] != outs[i])
      r[n++] = {addr(grads[i]), addr(grads[i]) + static_cast<uint64_t>(sizes[i]) * elem_bytes(dtypes[i]), i, false};
  }
  std::sort(r.get(), r.get() + n, [](const Range& x, const Range& y) { return x.lo < y.lo; });
  const Range *any = nullptr, *out = nullptr;  // of those before, the one that reaches farthest
  for (int64_t i = 0; i < n; ++i) {
    const Range* before = r[i].out ? any : out;
    if (before != nullptr && before->hi > r[i].lo)
      return fail(TGX_ERR_ARG, "tgx_clip_grad_norm: tensors %lld and %lld overlap (an output may be its own gradient only)",
                  static_cast<long long>(std::min(before->tensor, r[i].tensor)),
                  static_cast<long long>(std::max(before->tensor, r[i].tensor)));
    if (any == nullptr || r[i].hi > any->hi) any = &r[i];
    if (r[i].out && (out == nullptr || r[i].hi > out->hi)) out = &r[i];
  }
  return TGX_OK;
}

}  // namespace
}  // namespace tgx

using namespace tgx;

extern "C" size_t tgx_clip_grad_norm_workspace_size(const int64_t* sizes, int64_t count) {
  if (sizes == nullptr || count <= 0) return 0;
  for (int64_t i = 0; i < count; ++i)
    if (sizes[i] < 0) return 0;
  return static_cast<size_t>(part_count(sizes, count, part_values(sizes, count))) * 4;
}

extern "C" int tgx_clip_grad_norm(const void* const* grads, const int32_t* dtypes, void* const* outs,
                                  const int32_t* out_dtypes, const int64_t* sizes, int64_t count, float max_norm,
                                  float* norm, void* workspace, size_t workspace_bytes, void* stream) {
  if (count < 0 || norm == nullptr || (count > 0 && (grads == nullptr || dtypes == nullptr || outs == nullptr ||
                                                     out_dtypes == nullptr || sizes == nullptr)))
    return fail(TGX_ERR_ARG, "tgx_clip_grad_norm: count=%lld, and no array and not norm may be NULL",
                static_cast<long long>(count));
  for (int64_t i = 0; i < count; ++i) {
    if (sizes[i] < 0 || (sizes[i] > 0 && (grads[i] == nullptr || outs[i] == nullptr)))
      return fail(TGX_ERR_ARG, "tgx_clip_grad_norm: tensor %lld of %lld values must not be NULL",
                  static_cast<long long>(i), static_cast<long long>(sizes[i]));
    if (elem_bytes(dtypes[i]) == 0 || elem_bytes(out_dtypes[i]) == 0)
      return fail(TGX_ERR_DTYPE, "tgx_clip_grad_norm: tensor %lld has dtypes %d and %d", static_cast<long long>(i),
                  dtypes[i], out_dtypes[i]);
    if (sizes[i] > 0 && grads[i] == outs[i] && dtypes[i] != out_dtypes[i])
      return fail(TGX_ERR_ARG, "tgx_clip_grad_norm: tensor %lld is its own output in another dtype",
                  static_cast<long long>(i));
  }
  if (const int rc = check_apart(grads, dtypes, outs, out_dtypes, sizes, count)) return rc;
  const int64_t per = part_values(sizes, count);
  const int64_t parts = part_count(sizes, count, per);
  if (parts >= (int64_t(1) << 24)) return fail(TGX_ERR_LIMIT, "tgx_clip_grad_norm: %lld parts", static_cast<long long>(parts));
  if (parts > 0 && (workspace == nullptr || workspace_bytes < static_cast<size_t>(parts) * 4))
    return fail(TGX_ERR_ARG, "tgx_clip_grad_norm: workspace of %zu bytes needed", static_cast<size_t>(parts) * 4);
  hipStream_t s = static_cast<hipStream_t>(stream);
  float* part = static_cast<float*>(workspace);
  for (int pass = 0; pass < 2; ++pass) {
    int64_t at = 0;
    bool first = true;
    for (int64_t i = 0; i < count || (pass == 1 && first);) {
      ClipList l{};
      uint32_t n = 0;
      for (; i < count && l.count < kList; ++i) {
        if (sizes[i] == 0) continue;
        l.in[l.count] = grads[i];
        l.out[l.count] = outs[i];
        l.size[l.count] = sizes[i];
        l.in_bf16[l.count] = dtypes[i] == TGX_BF16;
        l.out_bf16[l.count] = out_dtypes[i] == TGX_BF16;
        l.first[l.count++] = n;
        n += static_cast<uint32_t>(ops_cdiv(sizes[i], per));
      }
      l.first[l.count] = n;
      if (pass == 0 && n > 0) {
        hipLaunchKernelGGL(clip_squares, dim3(n), dim3(kClipThreads), 0, s, l, per, part + at);
        const int rc = check_launch("clip_squares");
        if (rc) return rc;
      }
      if (pass == 1 && (n > 0 || first)) {
        hipLaunchKernelGGL(clip_scale, dim3(std::max(n, 1u)), dim3(kClipThreads), 0, s, l, per, part,
                           static_cast<int>(parts), max_norm, norm, first);
        const int rc = check_launch("clip_scale");
        if (rc) return rc;
      }
      at += n;
      first = false;
    }
  }
  return TGX_OK;
}
