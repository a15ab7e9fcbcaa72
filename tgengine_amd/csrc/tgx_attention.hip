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

int check_attention(const char* what, const tgx_attention_args* a, bool grad) {
  if (a == nullptr) return fail(TGX_ERR_ARG, "%s: args is NULL", what);
  if (a->batch < 0 || a->lq < 0 || a->lk < 0 || a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads != 0 ||
      a->dim < 1)
    return fail(TGX_ERR_ARG, "%s: batch=%lld lq=%lld lk=%lld heads=%d kv_heads=%d dim=%d", what,
                static_cast<long long>(a->batch), static_cast<long long>(a->lq), static_cast<long long>(a->lk),
                a->heads, a->kv_heads, a->dim);
  if (elem_bytes(a->dtype) == 0) return fail(TGX_ERR_DTYPE, "%s: dtype %d", what, a->dtype);
  if (a->dim > TGX_MAX_HEAD_DIM) return fail(TGX_ERR_LIMIT, "%s: dim=%d above %d", what, a->dim, TGX_MAX_HEAD_DIM);
  // No kernel takes 2^31 rows or more in one grid; up to 2^32 here, so that tiles of 16 rows
  // are counted in an int wherever the grids' own checks have not been yet
  const int64_t most = int64_t(1) << 31;
  if (a->lq >= most || a->lk >= most || a->heads > 65535 || a->batch >= most ||
      a->batch * a->heads >= most || (a->lq > 0 && a->batch * a->heads > (int64_t(1) << 32) / a->lq) ||
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
  a.rest = p->dtype == TGX_BF16 ? p->out_rest : nullptr;
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

// Whether a call takes the kernels of tgx_att_rows.hip.  A backward pass of at most 4 rows
// a problem does (2,000 x 2 problems of 4 rows and 64 keys, dim 128: 84 us in bf16 and 133
// in f32, against 174 and 249 of the matrix units), and a forward pass of one row (f32, 64
// keys: 42 us against 71; 10,000 keys, 8 x 2 problems: 37 against 50).  More rows take a
// vector kernel several times as many instructions and the matrix units none: above 64 keys
// they go there (500 x 2 problems of 4 rows and 256 keys, bf16: 39 us here, 28 there; at 20
// keys, 2,000 x 2 problems: 21 here, 42 there).
bool by_rows(const AttArgs& a, bool grad) {
  const int64_t rows = a.lq * a.group;
  return rows <= kMostRows && (grad || rows == 1 || a.lk <= 64);
}

}  // namespace
}  // namespace tgx

using namespace tgx;

extern "C" size_t tgx_attention_workspace_size(const tgx_attention_args* args) {
  if (check_attention("tgx_attention", args, false)) return 0;
  const AttArgs a = att_args(args);
  if (a.batch * a.lq == 0) return 0;
  return by_rows(a, false) ? att_rows_forward_workspace(a) : att_mma_forward_workspace(a, args->dtype);
}

extern "C" int tgx_attention(const tgx_attention_args* args, void* stream) {
  const int rc = check_attention("tgx_attention", args, false);
  if (rc) return rc;
  const AttArgs a = att_args(args);
  if (a.batch * a.lq == 0) return TGX_OK;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const size_t need = by_rows(a, false) ? att_rows_forward_workspace(a) : att_mma_forward_workspace(a, args->dtype);
  if (need > args->workspace_bytes || (need > 0 && !aligned16(args->workspace)))
    return fail(TGX_ERR_ARG, "tgx_attention: workspace of %zu bytes, 16-byte aligned, needed", need);
  return by_rows(a, false) ? att_rows_forward(a, args->dtype, args->workspace, s)
                    : att_mma_forward(a, args->dtype, args->workspace, s);
}

extern "C" size_t tgx_attention_grad_workspace_size(const tgx_attention_args* args) {
  if (check_attention("tgx_attention_grad", args, false)) return 0;
  const AttArgs a = att_args(args);
  if (a.batch * a.lq == 0) return 0;
  return by_rows(a, true) ? att_rows_backward_workspace(a) : att_mma_backward_workspace(a, args->dtype);
}

extern "C" int tgx_attention_grad(const tgx_attention_args* args, void* stream) {
  const int rc = check_attention("tgx_attention_grad", args, true);
  if (rc) return rc;
  const AttArgs a = att_args(args);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a.batch * a.lq == 0) {  // no query: the keys' gradients are zeros
    const size_t bytes = static_cast<size_t>(a.batch * a.lk * a.kv_heads * a.dim) * elem_bytes(args->dtype);
    for (void* p : {a.dk, a.dv})
      if (const int e = fill_zero(p, p != nullptr ? bytes : 0, s)) return e;
    return TGX_OK;
  }
  const size_t need = by_rows(a, true) ? att_rows_backward_workspace(a) : att_mma_backward_workspace(a, args->dtype);
  if (need > args->workspace_bytes || (need > 0 && !aligned16(args->workspace)))
    return fail(TGX_ERR_ARG, "tgx_attention_grad: workspace of %zu bytes, 16-byte aligned, needed", need);
  return by_rows(a, true) ? att_rows_backward(a, args->dtype, args->workspace, s)
                    : att_mma_backward(a, args->dtype, args->workspace, s);
}
