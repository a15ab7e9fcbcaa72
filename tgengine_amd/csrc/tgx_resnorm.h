// What the residual norm's passes share (tgx_resnorm.hip, tgx_resnorm_bwd.hip).
#pragma once

#include "tgx_norm_rows.h"

namespace tgx {
namespace {

struct ResArgs {
  const void* x;
  const void* residual;  // NULL (without PARTS): x is the sum
  const void* gate;
  const void* weight;
  const void* bias;
  const void* scale;
  const void* post;
  int64_t x_stride, residual_stride, gate_stride, rows;
  int32_t dim;
  int32_t center;
  float eps;
  void* out;
  void* sum;
  float* stats;  // [2][rows] mean and 1 / deviation of the sum; [4][rows]: and of x
  const void* dout;
  const void* dsum;
  void* dx;
  void* dres;
  void* dgate;
  float* part;  // [blocks][sums_of][dim]
};

// column sums of the backward pass: weight, bias, scale, post
constexpr int kSums = 4;
constexpr int sums_of(bool parts) { return parts ? kSums : 2; }

// Calls f(V, L, C): a row of `dim` values on L lanes, C packs of V values each.  One pack a
// lane up to a whole workgroup, because the backward pass keeps up to four sums for each
// value of its packs.  1,024 lanes have 128 registers each, which the backward pass exceeds: it
// spills 24 to 264 bytes a lane for bf16 rows of more than 4,096 values (none for the sum alone)
// and 264 to 924 above 8,192; 20 to 24 for f32 rows of 2,049 to 4,096 values with all parts, 52 to 408 up to
// 8,192 and 584 to 1,428 above.  Trained, 8,001 gated bf16 rows of 4,096 values take 188 us, 4,000 of
// 8,192 321 and 2,000 of 16,384 800, for the same bytes; the sum alone of the last two 116 and
// 303; f32 rows with all parts, of twice the bytes, 805 and 1,700.
template <typename T, typename F>
int res_shape(int64_t dim, F&& f) {
#define TGX_SHAPE(V, L, C) \
  f(std::integral_constant<int, V>{}, std::integral_constant<int, L>{}, std::integral_constant<int, C>{})
  constexpr int V = kWide<T>;
  if (dim < V) return TGX_SHAPE(1, 8, 1);
  const int64_t packs = ops_cdiv(dim, V);
  if (packs <= 8) return TGX_SHAPE(V, 8, 1);
  if (packs <= 16) return TGX_SHAPE(V, 16, 1);
  if (packs <= 32) return TGX_SHAPE(V, 32, 1);
  if (packs <= 64) return TGX_SHAPE(V, 64, 1);
  if (packs <= 128) return TGX_SHAPE(V, 128, 1);
  if (packs <= 256) return TGX_SHAPE(V, 256, 1);
  if (packs <= 512) return TGX_SHAPE(V, 512, 1);
  if (packs <= 1024) return TGX_SHAPE(V, 1024, 1);
  if constexpr (V == 8) {
    return TGX_SHAPE(V, 1024, 2);
  } else {
    if (packs <= 2048) return TGX_SHAPE(V, 1024, 2);
    return TGX_SHAPE(V, 1024, 4);
  }
#undef TGX_SHAPE
}
static_assert(TGX_MAX_NORM_DIM <= 1024 * 2 * 8 && TGX_MAX_NORM_DIM <= 1024 * 4 * 4, "a row fits its workgroup");

// a workgroup: several rows of up to a wavefront each, or one
constexpr int res_threads(int lanes) { return lanes > kWave ? lanes : kNormThreads; }

// the mean of a row's values (0 where rows are not centred) and 1 / sqrt(their mean square
// about it + eps)
template <int V, int L, int C>
__device__ __forceinline__ void row_stats(const float (&v)[C][V], const Place<V, L>& at, const ResArgs& a, float* lds,
                                          float& m, float& r) {
  m = 0.f;
  if (a.center) {
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int u = 0; u < V; ++u) m += u >= at.skip(j) ? v[j][u] : 0.f;
    m = row_sum<L>(m, lds) / static_cast<float>(at.dim);
  }
  float q = 0.f;
#pragma unroll
  for (int j = 0; j < C; ++j)
#pragma unroll
    for (int u = 0; u < V; ++u) {
      const float f = v[j][u] - m;
      q += u >= at.skip(j) ? f * f : 0.f;
    }
  r = 1.f / sqrtf(row_sum<L>(q, lds) / static_cast<float>(at.dim) + a.eps);
}

bool has_parts(const tgx_residual_norm_args* a) {
  return a->gate != nullptr || a->scale != nullptr || a->post_weight != nullptr;
}

int check_resnorm(const char* what, const tgx_residual_norm_args* a, bool grad) {
  if (a == nullptr) return fail(TGX_ERR_ARG, "%s: args is NULL", what);
  const long long rows = a->rows, dim = a->dim;
  if (rows < 0 || dim < 1 || (rows > 1 && (a->x_stride < 0 || a->residual_stride < 0 || a->gate_stride < 0)))
    return fail(TGX_ERR_ARG, "%s: rows=%lld dim=%lld, and strides of %lld, %lld and %lld", what, rows, dim,
                static_cast<long long>(a->x_stride), static_cast<long long>(a->residual_stride),
                static_cast<long long>(a->gate_stride));
  if (elem_bytes(a->dtype) == 0 || elem_bytes(a->wdtype) == 0)
    return fail(TGX_ERR_DTYPE, "%s: dtypes %d and %d", what, a->dtype, a->wdtype);
  if (dim > TGX_MAX_NORM_DIM || rows >= (int64_t(1) << 31))
    return fail(TGX_ERR_LIMIT, "%s: dim=%lld (at most %d), rows=%lld (below 2^31)", what, dim, TGX_MAX_NORM_DIM, rows);
  if (rows == 0) return TGX_OK;
  if (a->x == nullptr) return fail(TGX_ERR_ARG, "%s: x must not be NULL", what);
  if (a->residual == nullptr && (!grad || has_parts(a)))
    return fail(TGX_ERR_ARG, "%s: residual must not be NULL", what);
  return TGX_OK;
}

ResArgs res_args(const tgx_residual_norm_args* p) {
  ResArgs a{};
  a.x = p->x;
  a.residual = p->residual;
  a.gate = p->gate;
  a.weight = p->weight;
  a.bias = p->bias;
  a.scale = p->scale;
  a.post = p->post_weight;
  a.x_stride = p->x_stride;
  a.residual_stride = p->residual_stride;
  a.gate_stride = p->gate_stride;
  a.rows = p->rows;
  a.dim = static_cast<int32_t>(p->dim);
  a.center = p->center;
  a.eps = p->eps;
  a.out = p->out;
  a.sum = p->sum;
  a.stats = p->stats;
  a.dout = p->grad_out;
  a.dsum = p->grad_sum;
  a.dx = p->grad_x;
  a.dres = p->grad_residual;
  a.dgate = p->grad_gate;
  return a;
}

}  // namespace
}  // namespace tgx
