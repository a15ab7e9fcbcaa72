// Attention of query tokens to the states of another sequence, forward and backward.
//
// For a batch row b and a query head h, with k and v of its key/value head (heads /
// kv_heads query heads share one) and the keys that mask[b] keeps:
//
//   s_ij = scale q_i . k_j,  p_ij = exp(s_ij - lse_i),  lse_i = log sum_j exp(s_ij)
//   o_i  = sum_j p_ij v_j                      (0 where no key is kept; lse_i = -inf)
//   dv_j = sum_i p_ij do_i,  dp_ij = do_i . v_j,  ds_ij = p_ij (dp_ij - do_i . o_i) scale
//   dq_i = sum_j ds_ij k_j,  dk_j = sum_i ds_ij q_i      (i over the group's heads too)
//
// A masked key's k and v are never used, whatever they hold.
#include "tgx_attention.h"

namespace tgx {
namespace {

constexpr int kAttThreads = 256;
constexpr int kAttWaves = kAttThreads / kWave;
constexpr int kPer = TGX_MAX_HEAD_DIM / kWave;  // values of a head per lane

// one wave per query token and head
template <typename T>
__global__ __launch_bounds__(kAttThreads) void att_fwd(const AttArgs a) {
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kAttWaves + threadIdx.x / kWave;
  if (row >= a.batch * a.lq * a.heads) return;
  const int h = static_cast<int>(row % a.heads);
  const int64_t i = row / a.heads % a.lq, b = row / a.heads / a.lq;
  const int hk = h / (a.heads / a.kv_heads);
  const T* q = static_cast<const T*>(a.q) + b * a.qs[0] + i * a.qs[1] + h * a.qs[2];
  const T* k = static_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[2];
  const T* v = static_cast<const T*>(a.v) + b * a.vs[0] + hk * a.vs[2];
  float x[kPer], acc[kPer];
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    x[u] = lane + u * kWave < a.dim ? to_f(q[lane + u * kWave]) : 0.f;
    acc[u] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int64_t j = 0; j < a.lk; ++j) {
    if (a.mask != nullptr && !a.mask[b * a.mask_stride + j]) continue;
    float s = 0.f;
#pragma unroll
    for (int u = 0; u < kPer; ++u)
      if (lane + u * kWave < a.dim) s += x[u] * to_f(k[j * a.ks[1] + lane + u * kWave]);
    s = group_sum<kWave>(s) * a.scale;
    const float top = fmaxf(m, s);
    const float old = top == -INFINITY ? 1.f : expf(m - top), p = top == -INFINITY ? 0.f : expf(s - top);
    l = l * old + p;
    m = top;
#pragma unroll
    for (int u = 0; u < kPer; ++u)
      if (lane + u * kWave < a.dim) acc[u] = acc[u] * old + p * to_f(v[j * a.vs[1] + lane + u * kWave]);
  }
  T* o = static_cast<T*>(a.o) + row * a.dim;
#pragma unroll
  for (int u = 0; u < kPer; ++u)
    if (lane + u * kWave < a.dim) o[lane + u * kWave] = from_f<T>(l > 0.f ? acc[u] / l : 0.f);
  if (lane == 0 && a.lse != nullptr) a.lse[row] = l > 0.f ? m + logf(l) : -INFINITY;
}

// one wave per query token and head: dq
template <typename T>
__global__ __launch_bounds__(kAttThreads) void att_bwd_q(const AttArgs a) {
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kAttWaves + threadIdx.x / kWave;
  if (row >= a.batch * a.lq * a.heads) return;
  const int h = static_cast<int>(row % a.heads);
  const int64_t i = row / a.heads % a.lq, b = row / a.heads / a.lq;
  const int hk = h / (a.heads / a.kv_heads);
  const T* q = static_cast<const T*>(a.q) + b * a.qs[0] + i * a.qs[1] + h * a.qs[2];
  const T* k = static_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[2];
  const T* v = static_cast<const T*>(a.v) + b * a.vs[0] + hk * a.vs[2];
  float x[kPer], g[kPer], acc[kPer], delta = 0.f;
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    const bool in = lane + u * kWave < a.dim;
    x[u] = in ? to_f(q[lane + u * kWave]) : 0.f;
    g[u] = in ? to_f(static_cast<const T*>(a.dout)[row * a.dim + lane + u * kWave]) : 0.f;
    if (in) delta += g[u] * to_f(static_cast<const T*>(a.out)[row * a.dim + lane + u * kWave]);
    acc[u] = 0.f;
  }
  delta = group_sum<kWave>(delta);
  const float lse = a.lse[row];
  for (int64_t j = 0; j < a.lk && lse > -INFINITY; ++j) {
    if (a.mask != nullptr && !a.mask[b * a.mask_stride + j]) continue;
    float s = 0.f, dp = 0.f, kv[kPer];
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const bool in = lane + u * kWave < a.dim;
      kv[u] = in ? to_f(k[j * a.ks[1] + lane + u * kWave]) : 0.f;
      s += x[u] * kv[u];
      if (in) dp += g[u] * to_f(v[j * a.vs[1] + lane + u * kWave]);
    }
    s = group_sum<kWave>(s) * a.scale;
    dp = group_sum<kWave>(dp);
    const float ds = expf(s - lse) * (dp - delta) * a.scale;
#pragma unroll
    for (int u = 0; u < kPer; ++u) acc[u] += ds * kv[u];
  }
  T* o = static_cast<T*>(a.dq) + row * a.dim;
#pragma unroll
  for (int u = 0; u < kPer; ++u)
    if (lane + u * kWave < a.dim) o[lane + u * kWave] = from_f<T>(acc[u]);
}

// one wave per key and key/value head: dk and dv
template <typename T>
__global__ __launch_bounds__(kAttThreads) void att_bwd_kv(const AttArgs a) {
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kAttWaves + threadIdx.x / kWave;
  if (row >= a.batch * a.lk * a.kv_heads) return;
  const int hk = static_cast<int>(row % a.kv_heads);
  const int64_t j = row / a.kv_heads % a.lk, b = row / a.kv_heads / a.lk;
  const int group = a.heads / a.kv_heads;
  float x[kPer], y[kPer], ak[kPer], av[kPer];
  const bool kept = a.mask == nullptr || a.mask[b * a.mask_stride + j];
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    const bool in = kept && lane + u * kWave < a.dim;
    x[u] = in ? to_f(static_cast<const T*>(a.k)[b * a.ks[0] + j * a.ks[1] + hk * a.ks[2] + lane + u * kWave]) : 0.f;
    y[u] = in ? to_f(static_cast<const T*>(a.v)[b * a.vs[0] + j * a.vs[1] + hk * a.vs[2] + lane + u * kWave]) : 0.f;
    ak[u] = av[u] = 0.f;
  }
  for (int64_t r = 0; kept && r < a.lq * group; ++r) {
    const int64_t i = r / group;
    const int h = hk * group + static_cast<int>(r % group);
    const int64_t at = (b * a.lq + i) * a.heads + h;
    const float lse = a.lse[at];
    float qv[kPer], g[kPer], s = 0.f, dp = 0.f, delta = 0.f;
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const bool in = lane + u * kWave < a.dim;
      qv[u] = in ? to_f(static_cast<const T*>(a.q)[b * a.qs[0] + i * a.qs[1] + h * a.qs[2] + lane + u * kWave]) : 0.f;
      g[u] = in ? to_f(static_cast<const T*>(a.dout)[at * a.dim + lane + u * kWave]) : 0.f;
      if (in) delta += g[u] * to_f(static_cast<const T*>(a.out)[at * a.dim + lane + u * kWave]);
      s += qv[u] * x[u];
      dp += g[u] * y[u];
    }
    s = group_sum<kWave>(s) * a.scale;
    dp = group_sum<kWave>(dp);
    delta = group_sum<kWave>(delta);
    const float p = expf(s - lse), ds = p * (dp - delta) * a.scale;
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      av[u] += p * g[u];
      ak[u] += ds * qv[u];
    }
  }
#pragma unroll
  for (int u = 0; u < kPer; ++u) {
    if (lane + u * kWave >= a.dim) continue;
    if (a.dk != nullptr) static_cast<T*>(a.dk)[row * a.dim + lane + u * kWave] = from_f<T>(ak[u]);
    if (a.dv != nullptr) static_cast<T*>(a.dv)[row * a.dim + lane + u * kWave] = from_f<T>(av[u]);
  }
}

int check_attention(const char* what, const tgx_attention_args* a, bool grad) {
  if (a == nullptr) return fail(TGX_ERR_ARG, "%s: args is NULL", what);
  if (a->batch < 0 || a->lq < 0 || a->lk < 0 || a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads != 0 ||
      a->dim < 1)
    return fail(TGX_ERR_ARG, "%s: batch=%lld lq=%lld lk=%lld heads=%d kv_heads=%d dim=%d", what,
                static_cast<long long>(a->batch), static_cast<long long>(a->lq), static_cast<long long>(a->lk),
                a->heads, a->kv_heads, a->dim);
  if (elem_bytes(a->dtype) == 0) return fail(TGX_ERR_DTYPE, "%s: dtype %d", what, a->dtype);
  if (a->dim > TGX_MAX_HEAD_DIM) return fail(TGX_ERR_LIMIT, "%s: dim=%d above %d", what, a->dim, TGX_MAX_HEAD_DIM);
  const int64_t most = int64_t(1) << 31;
  if (a->lq >= most || a->lk >= most || a->heads > 65535 || a->batch >= most ||
      a->batch * a->heads >= most || (a->lq > 0 && a->batch * a->heads > (int64_t(1) << 40) / a->lq) ||
      (a->lk > 0 && a->batch * a->kv_heads > (int64_t(1) << 40) / a->lk))
    return fail(TGX_ERR_LIMIT, "%s: batch=%lld lq=%lld lk=%lld heads=%d: more rows than one launch takes", what,
                static_cast<long long>(a->batch), static_cast<long long>(a->lq), static_cast<long long>(a->lk),
                a->heads);
  const bool queries = a->batch > 0 && a->lq > 0, keys = a->batch > 0 && a->lk > 0;
  if (queries && (a->q == nullptr || a->out == nullptr)) return fail(TGX_ERR_ARG, "%s: q and out must not be NULL", what);
  if (keys && queries && (a->k == nullptr || a->v == nullptr)) return fail(TGX_ERR_ARG, "%s: k and v must not be NULL", what);
  if (grad && queries && (a->grad_out == nullptr || a->lse == nullptr))
    return fail(TGX_ERR_ARG, "%s: grad_out and lse must not be NULL", what);
  return TGX_OK;
}

AttArgs att_args(const tgx_attention_args* p) {
  AttArgs a{};
  a.q = p->q;
  a.k = p->k;
  a.v = p->v;
  a.mask = p->mask;
  a.out = p->out;
  a.o = p->out;
  a.dout = p->grad_out;
  a.dq = p->grad_q;
  a.dk = p->grad_k;
  a.dv = p->grad_v;
  a.lse = p->lse;
  a.batch = p->batch;
  a.lq = p->lq;
  a.lk = p->lk;
  a.mask_stride = p->mask_stride;
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = p->q_stride[i];
    a.ks[i] = p->k_stride[i];
    a.vs[i] = p->v_stride[i];
  }
  a.os[0] = p->lq * p->heads * p->dim;
  a.os[1] = static_cast<int64_t>(p->heads) * p->dim;
  a.os[2] = p->dim;
  a.heads = p->heads;
  a.kv_heads = p->kv_heads;
  a.group = p->heads / p->kv_heads;
  a.dim = p->dim;
  a.scale = p->scale;
  return a;
}

// few rows to few keys: a row's work is too small for a matrix tile
bool by_rows(const AttArgs& a) { return a.lq * a.group <= 4 && a.lk <= 512; }

}  // namespace
}  // namespace tgx

using namespace tgx;

extern "C" size_t tgx_attention_workspace_size(const tgx_attention_args* args) {
  if (check_attention("tgx_attention", args, false)) return 0;
  const AttArgs a = att_args(args);
  return by_rows(a) || a.batch * a.lq == 0 ? 0 : att_mma_forward_workspace(a, args->dtype);
}

extern "C" int tgx_attention(const tgx_attention_args* args, void* stream) {
  const int rc = check_attention("tgx_attention", args, false);
  if (rc) return rc;
  const AttArgs a = att_args(args);
  const int64_t rows = a.batch * a.lq * a.heads;
  if (rows == 0) return TGX_OK;
  if (!by_rows(a)) {
    const size_t need = att_mma_forward_workspace(a, args->dtype);
    if (need > args->workspace_bytes || (need > 0 && !aligned16(args->workspace)))
      return fail(TGX_ERR_ARG, "tgx_attention: workspace of %zu bytes, 16-byte aligned, needed", need);
    return att_mma_forward(a, args->dtype, args->workspace, static_cast<hipStream_t>(stream));
  }
  return by_type(args->dtype, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL(att_fwd<T>, dim3(static_cast<unsigned>(ops_cdiv(rows, kAttWaves))), dim3(kAttThreads), 0,
                       static_cast<hipStream_t>(stream), a);
    return check_launch("att_fwd");
  });
}

extern "C" size_t tgx_attention_grad_workspace_size(const tgx_attention_args* args) {
  if (check_attention("tgx_attention_grad", args, false)) return 0;
  const AttArgs a = att_args(args);
  return by_rows(a) || a.batch * a.lq == 0 ? 0 : att_mma_backward_workspace(a, args->dtype);
}

extern "C" int tgx_attention_grad(const tgx_attention_args* args, void* stream) {
  const int rc = check_attention("tgx_attention_grad", args, true);
  if (rc) return rc;
  const AttArgs a = att_args(args);
  const int64_t rows = a.batch * a.lq * a.heads, keys = a.batch * a.lk * a.kv_heads;
  if (!by_rows(a) && rows > 0) {
    const size_t need = att_mma_backward_workspace(a, args->dtype);
    if (need > args->workspace_bytes || !aligned16(args->workspace))
      return fail(TGX_ERR_ARG, "tgx_attention_grad: workspace of %zu bytes, 16-byte aligned, needed", need);
    return att_mma_backward(a, args->dtype, args->workspace, static_cast<hipStream_t>(stream));
  }
  return by_type(args->dtype, [&](auto t) {
    using T = decltype(t);
    if (rows > 0 && a.dq != nullptr) {
      hipLaunchKernelGGL(att_bwd_q<T>, dim3(static_cast<unsigned>(ops_cdiv(rows, kAttWaves))), dim3(kAttThreads), 0,
                         static_cast<hipStream_t>(stream), a);
      const int e = check_launch("att_bwd_q");
      if (e) return e;
    }
    if (keys > 0 && (a.dk != nullptr || a.dv != nullptr)) {
      hipLaunchKernelGGL(att_bwd_kv<T>, dim3(static_cast<unsigned>(ops_cdiv(keys, kAttWaves))), dim3(kAttThreads), 0,
                         static_cast<hipStream_t>(stream), a);
      return check_launch("att_bwd_kv");
    }
    return TGX_OK;
  });
}
