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
// simulation of 8,192 roots that begin at their exact values and whose gradients fall to a tenth
// after 3,000 steps, they stand at 0.94 of the exact ones after 3,000 more (deviation 0.13); with
// independent dithers at 1.02 (deviation 0.35), rounded to the nearest at 4.1.  Roots that begin at
// zero end alike but for the nearest: 0.4 before the gradients fall, 1.6 at the end.  A root
// above zero is stored above zero, since the next step divides by it.  The 8-bit averages
// are updated in 64 bits, so that what is stored is what the formulas say and not
// what an intermediate rounding makes of a value next to a border; this step's update uses
// the averages before they are rounded.
//
// HBM bounds the 32-bit step of a large table: 100,000,000 bf16 values (2.2 GB) 369 to 382 us
// (medians of three runs), 5.9 TB/s, as a large copy.  The 8-bit one has as much to compute as to
// move: 172,000,000 f32 values (2.77 GB) 496 us a call, 5.6 TB/s, 85 vector instructions a value
// keep the units busy nearly all of it.  Their clock decides: 478 us for the launches after a
// pause, up to 734 after some in a row, and 530 to 590 from then on.  16 tensors of up to 20,001 values
// take 3.0 and 4.0 us, mostly the launches, behind a host call of 12.
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
// Parts of all tensors together, about.  Short parts keep the bytes that are in flight beside
// each other: a table of 100,000,000 bf16 values with 32-bit averages takes 403 us in 131,072
// parts, 424 in 16,384 and 597 in 2,048; one of 172,000,000 f32 values with 8-bit ones 536 in
// 65,536, 555 in 16,384 and 580 in 262,144, where no wavefront has a next block to load.
constexpr int64_t kMostParts[2] = {131072, 65536};  // 32 bits, 8
static_assert(kBlock == kWave * kVals, "a wavefront takes a block");

struct AdamList {
  void* p[kList];
  const void* g[kList];
  void* m[kList];
  void* v[kList];
  float* scales[kList];
  int64_t size[kList];
  uint32_t first[kList + 1];  // first part of each tensor among this launch's
  // In words, as everything here: scalar loads drop the two lowest bits of a base and of an offset
  // apart, and the compiler may add the 7 t between a byte's and an address's place to either.
  uint32_t kind[kList];       // 4 * the number of its factors + kParamBf16 + kGradBf16
  int32_t count;
};
constexpr uint32_t kParamBf16 = 1, kGradBf16 = 2;
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

// the tensor that this workgroup's part belongs to: lane i knows whether it lies behind the
// first part of tensor i
static_assert(kList <= kWave, "a lane for each tensor");
__device__ __forceinline__ int adam_tensor(const AdamList& l, uint32_t block) {
  const int lane = threadIdx.x & (kWave - 1);
  return __popcll(__ballot(lane < l.count && l.first[min(lane, kList)] <= block)) - 1;
}

// the first n of kVals values from p on, the others 0
template <typename T>
__device__ __forceinline__ Pack<std::remove_const_t<T>, kVals> load_some(T* p, int n) {
  Pack<std::remove_const_t<T>, kVals> x;
#pragma unroll
  for (int u = 0; u < kVals; ++u) x.v[u] = u < n ? p[u] : static_cast<std::remove_const_t<T>>(0.f);
  return x;
}
template <typename T>
__device__ __forceinline__ void store_some(T* p, const Pack<T, kVals>& x, int n) {
#pragma unroll
  for (int u = 0; u < kVals; ++u)
    if (u < n) p[u] = x.v[u];
}

// kVals values that nothing reads again before the caches have forgotten them.  Loads and
// stores that both say so take the step of a table with 32-bit averages from 409 us to 373
// (stores alone 410, loads alone 420), with 8-bit ones from 539 to 537.
template <typename T>
using Words = uint32_t __attribute__((ext_vector_type(sizeof(T) * kVals / 4), aligned(sizeof(T))));
template <typename T>
__device__ __forceinline__ Pack<std::remove_const_t<T>, kVals> load_once(T* p) {
  const Words<T> w = __builtin_nontemporal_load(reinterpret_cast<const Words<T>*>(p));
  return __builtin_bit_cast(Pack<std::remove_const_t<T>, kVals>, w);
}
template <typename T>
__device__ __forceinline__ void store_once(T* p, const Pack<T, kVals>& x) {
  __builtin_nontemporal_store(__builtin_bit_cast(Words<T>, x), reinterpret_cast<Words<T>*>(p));
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
  auto one = [&](P& p, G g, float& m, float& v) {
    const float d = to_f(g) * f.clip_f;
    m = b1 * m + c1 * d;
    v = b2 * v + c2 * d * d;
    p = from_f<P>(stepped(to_f(p), m, sqrtf(v), f, c.eps));
  };
  const int64_t full = lo + (hi - lo) / kVals * kVals;
  for (int64_t i = lo + static_cast<int64_t>(threadIdx.x) * kVals; i < full; i += kAdamThreads * kVals) {
    Pack<P, kVals> pp = load_once(p + i);
    const Pack<G, kVals> pg = load_once(g + i);
    Pack<float, kVals> pm = load_once(m + i), pv = load_once(v + i);
#pragma unroll
    for (int u = 0; u < kVals; ++u) one(pp.v[u], pg.v[u], pm.v[u], pv.v[u]);
    store_once(p + i, pp);
    store_once(m + i, pm);
    store_once(v + i, pv);
  }
  const int64_t i = full + threadIdx.x;
  if (i < hi) one(p[i], g[i], m[i], v[i]);
}

__device__ __forceinline__ double power(int k) { return __longlong_as_double(static_cast<int64_t>(k + 1023) << 52); }
__device__ __forceinline__ uint32_t high(double x) { return static_cast<uint32_t>(__double_as_longlong(x) >> 32) & 0x7fffffffu; }
constexpr uint32_t kNotFinite = 0x7ff00000u;  // the high word of infinity

// the largest x of the wavefront, the same in every lane
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
#define TGX_MAX(ctrl, rows) \
  x = max(x, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), ctrl, rows, 0xf, false)))
  TGX_MAX(0x111, 0xf);  // lanes 1, 2, 4 and 8 before, in rows of 16
  TGX_MAX(0x112, 0xf);
  TGX_MAX(0x114, 0xf);
  TGX_MAX(0x118, 0xf);
  TGX_MAX(0x142, 0xa);  // the last lane of a row to the next one
  TGX_MAX(0x143, 0xc);  // and of the first half to the second
#undef TGX_MAX
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x), kWave - 1));
}

// the exponent of a block's power of two, from the high word of its largest finite value
// (0: a block of zeros)
__device__ __forceinline__ int block_power(uint32_t top) {
  return max(static_cast<int>(top >> 20) - 1023 - 7, -126);
}

// the e4m3 code of |x| / 2^k, below 256, by the dither w / 2^32: a value's place between
// its two neighbours is what stands behind the three leading bits of its mantissa, where w is
// added, and a carry makes it the upper one.  Below 2^(k - 6) the spacing stays that of the
// binade above: the values, zero among them, are lifted into it.
__device__ __forceinline__ uint32_t code(double x, int k, uint32_t w) {
  const bool low = high(x) < static_cast<uint32_t>(k - 6 + 1023) << 20;
  const double z = fabs(x) + (low ? power(k - 6) : 0.0);
  const uint64_t bits = static_cast<uint64_t>(__double_as_longlong(z)) + (static_cast<uint64_t>(w) << 17);
  const uint32_t base = static_cast<uint32_t>(k - 7 + 1023) << 3;
  return static_cast<uint32_t>(bits >> 49) - (low ? base + 8 : base);
}
constexpr uint32_t kNan = 0x7f;

constexpr uint32_t kPlace = 0xC13FA9A9u, kTurn = 0x91E10DA5u;  // 2^32 / p, 2^32 / p^2

// sqrt(v): an estimate to 2^-24 and two steps of Newton's, the second for the last bit, so
// that the root of a square is that number.
__device__ __forceinline__ double root_of(double v) {
  const double y = fmin(__builtin_amdgcn_rsq(v), 1e150), half = 0.5 * y;  // finite, for v = 0
  const double r = fma(half, fma(-(v * y), v * y, v), v * y);
  return fma(half, fma(-r, r, v), r);
}

// kVals values of a block, n of them real: the averages' new ones in 64 bits, the parameters
// stepped, and the high words of the largest finite averages
template <typename P, typename G>
struct Held {
  Pack<P, kVals> p;
  Pack<G, kVals> g;
  Pack<uint8_t, kVals> m, v;
  float sm, sv;
  double first[kVals], root[kVals];

  __device__ __forceinline__ void step(const Factors& f, const Constants& c, uint32_t& em, uint32_t& ev) {
    const double bm = c.b1 * sm, bv = c.b2 * (static_cast<double>(sv) * sv);
    float least = 1e30f, most = 0.f, den[kVals];
#pragma unroll
    for (int u = 0; u < kVals; ++u) {
      const double d = static_cast<double>(to_f(g.v[u])) * f.clip;
      // powers of two and squares of 4-bit mantissas: b sm, b sv sv and r r are exact.  Each
      // product and sum rounds by itself, in the formulas' order: where an average equals its
      // gradient, a power of two say, a fused one would end below it, in another block scale.
      const float r = __builtin_amdgcn_cvt_f32_fp8(v.v[u], 0);
      first[u] = bm * static_cast<double>(__builtin_amdgcn_cvt_f32_fp8(m.v[u], 0)) + c.c1 * d;
      root[u] = root_of(bv * static_cast<double>(r * r) + c.c2 * (d * d));
      em = max(em, high(first[u]));
      ev = max(ev, high(root[u]));
      den[u] = static_cast<float>(root[u]) * f.even + c.eps;
      least = fminf(least, den[u]);
      most = fmaxf(most, den[u]);
    }
    // the reciprocal's instruction ends where its result or its argument is no normal number
    const bool usual = least > 1e-30f && most < 1e30f;
#pragma unroll
    for (int u = 0; u < kVals; ++u) {
      const float up = f.by * static_cast<float>(first[u]);
      const float q = usual ? up * __builtin_amdgcn_rcpf(den[u]) : up / den[u];
      p.v[u] = from_f<P>(to_f(p.v[u]) * f.keep - q);
    }
  }

  __device__ __forceinline__ void hold(uint32_t i, uint32_t turn, int km, int kv) {
#pragma unroll
    for (int u = 0; u < kVals; ++u) {
      const uint32_t w = (i + u) * kPlace + turn;
      const uint32_t sign = static_cast<uint32_t>(__double_as_longlong(first[u]) >> 56) & 0x80u;
      m.v[u] = static_cast<uint8_t>(code(first[u], km, w) | sign);
      const uint32_t r = code(root[u], kv, w + 0x80000000u);
      v.v[u] = static_cast<uint8_t>(root[u] > 0.0 ? max(r, 1u) : 0u);
    }
  }

  // the largest finite averages of a block that holds others
  __device__ __forceinline__ void finite(uint32_t& em, uint32_t& ev) const {
    em = ev = 0;
#pragma unroll
    for (int u = 0; u < kVals; ++u) {
      em = max(em, high(first[u]) < kNotFinite ? high(first[u]) : 0u);
      ev = max(ev, high(root[u]) < kNotFinite ? high(root[u]) : 0u);
    }
  }
  __device__ __forceinline__ void not_finite() {
#pragma unroll
    for (int u = 0; u < kVals; ++u) {
      if (high(first[u]) >= kNotFinite) m.v[u] = kNan;
      if (high(root[u]) >= kNotFinite) v.v[u] = kNan;
    }
  }
};

template <typename P, typename G>
__device__ __forceinline__ void adam_held(P* __restrict__ p, const G* __restrict__ g, uint8_t* __restrict__ m,
                                          uint8_t* __restrict__ v, float* __restrict__ scales, int64_t blocks, int64_t lo,
                                          int64_t hi, const Factors& f, const Constants& c) {
  const int lane = threadIdx.x & (kWave - 1);
  const uint32_t turn = f.t * kTurn;
  auto read = [&](Held<P, G>& x, int64_t b, auto load) {
    const int64_t i = b * kBlock + lane * kVals;
    x.p = load(p + i);
    x.g = load(g + i);
    x.m = load(m + i);
    x.v = load(v + i);
    x.sm = scales[b];
    x.sv = scales[blocks + b];
  };
  auto write = [&](Held<P, G>& x, int64_t b, auto store) {
    const int64_t i = b * kBlock + lane * kVals;
    uint32_t em = 0, ev = 0;
    x.step(f, c, em, ev);
    em = wave_max(em);
    ev = wave_max(ev);
    const bool others = max(em, ev) >= kNotFinite;  // wave-uniform, as em and ev
    if (others) {
      x.finite(em, ev);
      em = wave_max(em);
      ev = wave_max(ev);
    }
    const int km = block_power(em), kv = block_power(ev);
    x.hold(static_cast<uint32_t>(i), turn, km, kv);
    if (others) x.not_finite();
    store(p + i, x.p);
    store(m + i, x.m);
    store(v + i, x.v);
    if (lane == 0) {
      scales[b] = static_cast<float>(power(km));
      scales[blocks + b] = static_cast<float>(power(kv));
    }
  };
  auto all = [](auto* q) { return load_once(q); };
  // wave-uniform: a wavefront takes whole blocks, the next one's values on their way while it
  // steps one, and one wavefront the rest
  constexpr int kWaves = kAdamThreads / kWave;
  const int64_t whole = hi / kBlock, first = lo / kBlock + threadIdx.x / kWave;
  Held<P, G> x, next;
  if (first < whole) read(next, first, all);
  for (int64_t b = first; b < whole; b += kWaves) {
    x = next;
    read(next, min(b + kWaves, whole - 1), all);
    write(x, b, [](auto* q, const auto& y) { store_once(q, y); });
  }
  if (whole * kBlock < hi && (whole - first) % kWaves == 0) {
    const int n = static_cast<int>(hi - whole * kBlock) - lane * kVals;  // of this lane's, none where it is negative
    read(x, whole, [n](auto* q) { return load_some(q, n); });
    write(x, whole, [n](auto* q, const auto& y) { store_some(q, y, n); });
  }
}

template <bool HELD>
__global__ __launch_bounds__(kAdamThreads) void adamw_step(const AdamList l, int64_t per, const Constants c,
                                                           const Factors* __restrict__ factors) {
  const int t = adam_tensor(l, blockIdx.x);
  const int64_t lo = (blockIdx.x - l.first[t]) * per, size = l.size[t];
  const int64_t hi = lo + per < size ? lo + per : size;
  const uint32_t kind = l.kind[t];
  const Factors f = factors[kind / 4];
  auto with = [&](auto* p, auto* g) {
    if constexpr (HELD)
      adam_held(p, g, static_cast<uint8_t*>(l.m[t]), static_cast<uint8_t*>(l.v[t]), l.scales[t], (size + kBlock - 1) / kBlock,
                lo, hi, f, c);
    else
      adam_wide(p, g, static_cast<float*>(l.m[t]), static_cast<float*>(l.v[t]), lo, hi, f, c);
  };
  if (kind & kParamBf16) {
    if (kind & kGradBf16) with(static_cast<bf16*>(l.p[t]), static_cast<const bf16*>(l.g[t]));
    else with(static_cast<bf16*>(l.p[t]), static_cast<const float*>(l.g[t]));
  } else {
    if (kind & kGradBf16) with(static_cast<float*>(l.p[t]), static_cast<const bf16*>(l.g[t]));
    else with(static_cast<float*>(l.p[t]), static_cast<const float*>(l.g[t]));
  }
}

// values per part: one round of a workgroup or more, and as many as keep the parts near
// kMostParts; whole blocks
int64_t adam_part(const tgx_adamw_tensor* t, int64_t count, int bits) {
  int64_t all = 0;
  for (int64_t i = 0; i < count; ++i) all += t[i].bits == bits ? t[i].size : 0;
  constexpr int64_t round = kAdamThreads * kVals;
  return std::max<int64_t>(1, ops_cdiv(ops_cdiv(all, kMostParts[bits == 8]), round)) * round;
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
    const int64_t per = adam_part(a.tensors, a.count, bits);
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
        l.kind[l.count] = static_cast<uint32_t>(i) * 4 + (t.dtype == TGX_BF16 ? kParamBf16 : 0u) +
                          (t.grad_dtype == TGX_BF16 ? kGradBf16 : 0u);
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
