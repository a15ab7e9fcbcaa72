// One AdamW step over many tensors.
//
//   t = step + 1,  g = grad min(1, max_norm / (norm + 1e-6))
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr decay) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// A first launch counts the steps and leaves each tensor's factors, computed in 64 bits; the
// second takes all tensors together, whose addresses travel in its arguments, kList a
// launch.  The averages are f32, or 8 bits a value: m and sqrt(v) as e4m3 times a power of
// two that kBlock values share, the largest of them in [128, 256).  The root, because its
// range is half of v's, in octaves.  Which of the two neighbours of the format a value becomes is
// decided by a dither u in [0, 1), floor(x / spacing + u): rounded to the nearest, a root
// that shrinks by 0.05% a step would stay where it is for ever.  u is the fraction of
// i / p + t / p^2 (+ 1/2 for the root), i the value's place and p^3 = p + 1, a sequence
// that is even over neighbouring values and steps alike, and needs no state.  In a
// simulation of 8,192 roots whose gradients fall to a tenth after 3,000 steps, they stand at
// 0.93 of the exact ones after 3,000 more (deviation 0.13); with independent dithers at 1.02
// (deviation 0.35), rounded to the nearest at 4.1.  A root
// above zero is stored above zero, since the next step divides by it.  The 8-bit averages
// are updated in 64 bits, so that what is stored is what the formulas say and not
// what an intermediate rounding makes of a value next to a border; this step's update uses
// the averages before they are rounded.
#include "tgx_ops.h"
#include "tgx_ranges.h"

#include <memory>
#include <new>

namespace tgx {
namespace {

constexpr int kAdamThreads = 256;
constexpr int kBlock = TGX_ADAMW_BLOCK;
constexpr int kVals = 4;            // a lane's share of a block
constexpr int kList = 56;           // tensors per launch: their table stays below the 4 KB of kernel arguments
constexpr int64_t kMostParts = 2048;  // parts of all tensors together, about
static_assert(kBlock == kWave * kVals, "a wavefront takes a block");

struct AdamList {
  void* p[kList];
  const void* g[kList];
  void* m[kList];
  void* v[kList];
  float* scales[kList];
  int64_t size[kList];
  uint32_t first[kList + 1];  // first part of each tensor among this launch's
  uint16_t at[kList];         // its factors
  uint8_t p_bf16[kList], g_bf16[kList];
  int32_t count;
};
static_assert(sizeof(AdamList) <= 3800, "kernel arguments");

struct Factors {
  double clip;
  float clip_f, keep, by, even;  // keep = 1 - lr decay, by = lr / (1 - b1^t), even = 1 / sqrt(1 - b2^t)
  uint32_t t, reserved;
};

struct Constants {
  double b1, b2, c1, c2;  // c = 1 - b
  float eps;
};

constexpr int kSteps = 256;
struct StepList {
  int64_t* step[kSteps];
  int32_t count, first;
};

__global__ __launch_bounds__(kSteps) void adamw_begin(const StepList l, double lr, const float* __restrict__ lr_device,
                                                      double b1, double b2, double decay,
                                                      const float* __restrict__ norm, double max_norm,
                                                      Factors* __restrict__ to) {
  if (threadIdx.x >= l.count) return;
  int64_t* step = l.step[threadIdx.x];
  const int64_t t = *step + 1;
  *step = t;
  if (lr_device != nullptr) lr = *lr_device;
  Factors f{};
  f.clip = 1.0;
  if (norm != nullptr) {
    f.clip = max_norm / (static_cast<double>(*norm) + 1e-6);
    f.clip = f.clip > 1.0 ? 1.0 : f.clip;  // NaN stays
  }
  f.clip_f = static_cast<float>(f.clip);
  f.keep = static_cast<float>(1.0 - lr * decay);
  f.by = static_cast<float>(lr / (1.0 - pow(b1, static_cast<double>(t))));
  f.even = static_cast<float>(1.0 / sqrt(1.0 - pow(b2, static_cast<double>(t))));
  f.t = static_cast<uint32_t>(t);
  to[l.first + threadIdx.x] = f;
}

__device__ __forceinline__ int adam_tensor(const AdamList& l, uint32_t block) {
  int lo = 0, hi = l.count;  // first[lo] <= block < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (l.first[mid] <= block) lo = mid;
    else hi = mid;
  }
  return lo;
}

// n <= kVals values from p on, the others 0
template <typename T>
__device__ __forceinline__ Pack<T, kVals> load_some(const T* p, int n) {
  if (n == kVals) return load_pack<T, kVals>(p);
  Pack<T, kVals> x;
#pragma unroll
  for (int u = 0; u < kVals; ++u) x.v[u] = u < n ? p[u] : static_cast<T>(0.f);
  return x;
}
template <typename T>
__device__ __forceinline__ void store_some(T* p, const Pack<T, kVals>& x, int n) {
  if (n == kVals) return store_pack<T, kVals>(p, x);
#pragma unroll
  for (int u = 0; u < kVals; ++u)
    if (u < n) p[u] = x.v[u];
}

__device__ __forceinline__ float stepped(float p, float m, float root, const Factors& f, float eps) {
  return p * f.keep - f.by * m / (root * f.even + eps);
}

template <typename P, typename G>
__device__ __forceinline__ void adam_wide(P* __restrict__ p, const G* __restrict__ g, float* __restrict__ m,
                                          float* __restrict__ v, int64_t lo, int64_t hi, const Factors& f,
                                          const Constants& c) {
  const float b1 = static_cast<float>(c.b1), b2 = static_cast<float>(c.b2);
  const float c1 = static_cast<float>(c.c1), c2 = static_cast<float>(c.c2);
  for (int64_t i = lo + static_cast<int64_t>(threadIdx.x) * kVals; i < hi; i += kAdamThreads * kVals) {
    const int n = static_cast<int>(min(hi - i, static_cast<int64_t>(kVals)));
    Pack<P, kVals> pp = load_some(p + i, n);
    const Pack<G, kVals> pg = load_some(g + i, n);
    Pack<float, kVals> pm = load_some(m + i, n), pv = load_some(v + i, n);
#pragma unroll
    for (int u = 0; u < kVals; ++u) {
      const float d = to_f(pg.v[u]) * f.clip_f;
      pm.v[u] = b1 * pm.v[u] + c1 * d;
      pv.v[u] = b2 * pv.v[u] + c2 * d * d;
      pp.v[u] = from_f<P>(stepped(to_f(pp.v[u]), pm.v[u], sqrtf(pv.v[u]), f, c.eps));
    }
    store_some(p + i, pp, n);
    store_some(m + i, pm, n);
    store_some(v + i, pv, n);
  }
}

__device__ __forceinline__ int exponent(double x) {  // of a value that is not 0: floor(log2 |x|)
  return static_cast<int>((__double_as_longlong(x) >> 52) & 0x7ff) - 1023;
}
__device__ __forceinline__ double power(int k) { return __longlong_as_double(static_cast<int64_t>(k + 1023) << 52); }
constexpr int kNotFinite = 1024;  // the exponent of infinities and NaN

// the exponent of a block's power of two; e: of the lane's largest finite value
__device__ __forceinline__ int block_power(int e) {
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) e = max(e, __shfl_xor(e, off, kWave));
  return max(e - 7, -126);
}

// the e4m3 code of |x| / 2^k, below 256, by the dither w / 2^32
__device__ __forceinline__ uint32_t code(double x, int k, uint32_t w, bool above) {
  const int e = exponent(x);
  if (e == kNotFinite) return 0x7f;
  const int top = max(e - k, -6);  // the binade; its spacing is 2^(top - 3)
  const double y = fabs(x) * power(3 - top - k) + static_cast<double>(w) * 0x1p-32;
  uint32_t n = static_cast<uint32_t>(y);
  if (above) n = max(n, 1u);
  return x == 0.0 ? 0u : static_cast<uint32_t>((top + 6) << 3) + n;
}

constexpr uint32_t kPlace = 0xC13FA9A9u, kTurn = 0x91E10DA5u;  // 2^32 / p, 2^32 / p^2

template <typename P, typename G>
__device__ __forceinline__ void adam_held(P* __restrict__ p, const G* __restrict__ g, uint8_t* __restrict__ m,
                                          uint8_t* __restrict__ v, float* __restrict__ scales, int64_t blocks, int64_t lo,
                                          int64_t hi, const Factors& f, const Constants& c) {
  const int lane = threadIdx.x & (kWave - 1);
  for (int64_t b = lo / kBlock + threadIdx.x / kWave; b * kBlock < hi; b += kAdamThreads / kWave) {  // wave-uniform
    const int64_t i = b * kBlock + lane * kVals;
    const int n = static_cast<int>(max(static_cast<int64_t>(0), min(hi - i, static_cast<int64_t>(kVals))));
    Pack<P, kVals> pp = load_some(p + i, n);
    const Pack<G, kVals> pg = load_some(g + i, n);
    const Pack<uint8_t, kVals> pm = load_some(m + i, n), pv = load_some(v + i, n);
    const double sm = scales[b], sv = scales[blocks + b];
    double first[kVals], root[kVals];
    int em = -2000, ev = -2000;
#pragma unroll
    for (int u = 0; u < kVals; ++u) {
      const double d = static_cast<double>(to_f(pg.v[u])) * f.clip;
      const double r = static_cast<double>(__builtin_amdgcn_cvt_f32_fp8(pv.v[u], 0)) * sv;
      first[u] = c.b1 * (static_cast<double>(__builtin_amdgcn_cvt_f32_fp8(pm.v[u], 0)) * sm) + c.c1 * d;
      root[u] = sqrt(c.b2 * (r * r) + c.c2 * (d * d));
      const int e1 = exponent(first[u]), e2 = exponent(root[u]);
      if (e1 != kNotFinite && first[u] != 0.0) em = max(em, e1);
      if (e2 != kNotFinite && root[u] != 0.0) ev = max(ev, e2);
      pp.v[u] = from_f<P>(stepped(to_f(pp.v[u]), static_cast<float>(first[u]), static_cast<float>(root[u]), f, c.eps));
    }
    const int km = block_power(em), kv = block_power(ev);
    Pack<uint8_t, kVals> om, ov;
#pragma unroll
    for (int u = 0; u < kVals; ++u) {
      const uint32_t w = (static_cast<uint32_t>(i) + u) * kPlace + f.t * kTurn;
      om.v[u] = static_cast<uint8_t>(code(first[u], km, w, false) | (first[u] < 0.0 ? 0x80u : 0u));
      ov.v[u] = static_cast<uint8_t>(code(root[u], kv, w + 0x80000000u, true));
    }
    store_some(p + i, pp, n);
    store_some(m + i, om, n);
    store_some(v + i, ov, n);
    if (lane == 0) {
      scales[b] = static_cast<float>(power(km));
      scales[blocks + b] = static_cast<float>(power(kv));
    }
  }
}

template <bool HELD>
__global__ __launch_bounds__(kAdamThreads) void adamw_step(const AdamList l, int64_t per, const Constants c,
                                                           const Factors* __restrict__ factors) {
  const int t = adam_tensor(l, blockIdx.x);
  const int64_t lo = (blockIdx.x - l.first[t]) * per, size = l.size[t];
  const int64_t hi = lo + per < size ? lo + per : size;
  const Factors f = factors[l.at[t]];
  auto with = [&](auto* p, auto* g) {
    if constexpr (HELD)
      adam_held(p, g, static_cast<uint8_t*>(l.m[t]), static_cast<uint8_t*>(l.v[t]), l.scales[t], (size + kBlock - 1) / kBlock,
                lo, hi, f, c);
    else
      adam_wide(p, g, static_cast<float*>(l.m[t]), static_cast<float*>(l.v[t]), lo, hi, f, c);
  };
  if (l.p_bf16[t]) {
    if (l.g_bf16[t]) with(static_cast<bf16*>(l.p[t]), static_cast<const bf16*>(l.g[t]));
    else with(static_cast<bf16*>(l.p[t]), static_cast<const float*>(l.g[t]));
  } else {
    if (l.g_bf16[t]) with(static_cast<float*>(l.p[t]), static_cast<const bf16*>(l.g[t]));
    else with(static_cast<float*>(l.p[t]), static_cast<const float*>(l.g[t]));
  }
}

// values per part: one round of a workgroup or more, and as many as keep the parts near
// kMostParts; whole blocks
int64_t adam_part(const tgx_adamw_tensor* t, int64_t count) {
  int64_t all = 0;
  for (int64_t i = 0; i < count; ++i) all += t[i].size;
  constexpr int64_t round = kAdamThreads * kVals;
  return std::max<int64_t>(1, ops_cdiv(ops_cdiv(all, kMostParts), round)) * round;
}

int check_adamw(const tgx_adamw_args* a) {
  const char* what = "tgx_adamw";
  if (a == nullptr) return fail(TGX_ERR_ARG, "%s: args is NULL", what);
  if (a->count < 0 || (a->count > 0 && a->tensors == nullptr))
    return fail(TGX_ERR_ARG, "%s: count=%lld, and tensors must not be NULL", what, static_cast<long long>(a->count));
  if (!(a->beta1 >= 0.0 && a->beta1 < 1.0 && a->beta2 >= 0.0 && a->beta2 < 1.0 && a->eps >= 0.0 && a->weight_decay >= 0.0) ||
      (a->lr_device == nullptr && !(a->lr >= 0.0)))
    return fail(TGX_ERR_ARG, "%s: lr=%g beta1=%g beta2=%g eps=%g weight_decay=%g", what, a->lr, a->beta1, a->beta2, a->eps,
                a->weight_decay);
  if (a->grad_norm != nullptr && !(a->max_norm >= 0.0)) return fail(TGX_ERR_ARG, "%s: max_norm=%g", what, a->max_norm);
  if (a->count > 65535) return fail(TGX_ERR_LIMIT, "%s: %lld tensors (at most 65535)", what, static_cast<long long>(a->count));
  for (int64_t i = 0; i < a->count; ++i) {
    const tgx_adamw_tensor& t = a->tensors[i];
    const long long at = i;
    if (t.size < 0 || t.step == nullptr ||
        (t.size > 0 && (t.param == nullptr || t.grad == nullptr || t.exp_avg == nullptr || t.exp_avg_sq == nullptr)))
      return fail(TGX_ERR_ARG, "%s: tensor %lld of %lld values: no pointer may be NULL", what, at, static_cast<long long>(t.size));
    if (elem_bytes(t.dtype) == 0 || elem_bytes(t.grad_dtype) == 0)
      return fail(TGX_ERR_DTYPE, "%s: tensor %lld has dtypes %d and %d", what, at, t.dtype, t.grad_dtype);
    if ((t.bits != 8 && t.bits != 32) || (t.bits == 8 && t.size > 0 && t.scales == nullptr))
      return fail(TGX_ERR_ARG, "%s: tensor %lld has averages of %d bits (8, with scales, or 32)", what, at, t.bits);
    if (t.size >= (int64_t(1) << 40)) return fail(TGX_ERR_LIMIT, "%s: tensor %lld has %lld values", what, at, static_cast<long long>(t.size));
  }
  // workgroups write all outputs at once, in no order
  const std::unique_ptr<Range[]> r(new (std::nothrow) Range[static_cast<size_t>(a->count) * 6 + 2]);
  if (r == nullptr) return fail(TGX_ERR_LIMIT, "%s: no memory to check %lld tensors", what, static_cast<long long>(a->count));
  int64_t n = 0;
  auto add = [&](const void* p, int64_t bytes, int64_t i, bool out) {
    r[n++] = {addr(p), addr(p) + static_cast<uint64_t>(bytes), i, out};
  };
  for (int64_t i = 0; i < a->count; ++i) {
    const tgx_adamw_tensor& t = a->tensors[i];
    add(t.step, 8, i, true);
    if (t.size == 0) continue;
    add(t.param, t.size * elem_bytes(t.dtype), i, true);
    add(t.grad, t.size * elem_bytes(t.grad_dtype), i, false);
    add(t.exp_avg, t.size * (t.bits / 8), i, true);
    add(t.exp_avg_sq, t.size * (t.bits / 8), i, true);
    if (t.bits == 8) add(t.scales, ops_cdiv(t.size, kBlock) * 8, i, true);
  }
  if (a->lr_device != nullptr) add(a->lr_device, 4, a->count, false);
  if (a->grad_norm != nullptr) add(a->grad_norm, 4, a->count, false);
  int64_t one, other;
  if (overlap(r.get(), n, one, other))
    return fail(TGX_ERR_ARG, "%s: memory of tensors %lld and %lld overlaps", what, static_cast<long long>(one),
                static_cast<long long>(other));
  return TGX_OK;
}

}  // namespace
}  // namespace tgx

using namespace tgx;

extern "C" size_t tgx_adamw_workspace_size(int64_t count) {
  return count > 0 ? static_cast<size_t>(count) * sizeof(Factors) : 0;
}

extern "C" int tgx_adamw(const tgx_adamw_args* args, void* stream) {
  if (const int rc = check_adamw(args)) return rc;
  const tgx_adamw_args& a = *args;
  if (a.count == 0) return TGX_OK;
  const size_t need = tgx_adamw_workspace_size(a.count);
  if (a.workspace == nullptr || a.workspace_bytes < need || !aligned16(a.workspace))
    return fail(TGX_ERR_ARG, "tgx_adamw: workspace of %zu bytes, 16-byte aligned, needed", need);
  const int64_t per = adam_part(a.tensors, a.count);
  hipStream_t s = static_cast<hipStream_t>(stream);
  Factors* factors = static_cast<Factors*>(a.workspace);
  const Constants c{a.beta1, a.beta2, 1.0 - a.beta1, 1.0 - a.beta2, static_cast<float>(a.eps)};
  for (int64_t i = 0; i < a.count; i += kSteps) {
    StepList l{};
    l.first = static_cast<int32_t>(i);
    for (; l.count < kSteps && i + l.count < a.count; ++l.count) l.step[l.count] = a.tensors[i + l.count].step;
    hipLaunchKernelGGL(adamw_begin, dim3(1), dim3(kSteps), 0, s, l, a.lr, a.lr_device, a.beta1, a.beta2, a.weight_decay,
                       a.grad_norm, a.max_norm, factors);
    if (const int rc = check_launch("adamw_begin")) return rc;
  }
  for (const int bits : {32, 8}) {
    for (int64_t i = 0; i < a.count;) {
      AdamList l{};
      uint32_t n = 0;
      for (; i < a.count && l.count < kList; ++i) {
        const tgx_adamw_tensor& t = a.tensors[i];
        if (t.size == 0 || t.bits != bits) continue;
        l.p[l.count] = t.param;
        l.g[l.count] = t.grad;
        l.m[l.count] = t.exp_avg;
        l.v[l.count] = t.exp_avg_sq;
        l.scales[l.count] = t.scales;
        l.size[l.count] = t.size;
        l.at[l.count] = static_cast<uint16_t>(i);
        l.p_bf16[l.count] = t.dtype == TGX_BF16;
        l.g_bf16[l.count] = t.grad_dtype == TGX_BF16;
        l.first[l.count++] = n;
        n += static_cast<uint32_t>(ops_cdiv(t.size, per));
      }
      l.first[l.count] = n;
      if (n == 0) continue;
      if (bits == 8) hipLaunchKernelGGL(adamw_step<true>, dim3(n), dim3(kAdamThreads), 0, s, l, per, c, factors);
      else hipLaunchKernelGGL(adamw_step<false>, dim3(n), dim3(kAdamThreads), 0, s, l, per, c, factors);
      if (const int rc = check_launch("adamw_step")) return rc;
    }
  }
  return TGX_OK;
}
