// A gated recurrence along the tokens of every batch row, forward and backward.
//
//   a_t = sigmoid(gate_t),  h_t = a_t h_{t-1} + (1 - a_t) x_t     (a masked token: h_t = h_{t-1})
//   dh_t = dout_t + a_{t+1} dh_{t+1}                              (dlast joins the last one)
//   dx_t = (1 - a_t) dh_t,  dgate_t = a_t (1 - a_t) (h_{t-1} - x_t) dh_t,  dstate = a_1 dh_1
//
// A thread keeps the state of V neighbouring channels of one row in 32 bits and walks the
// row's tokens kSpan at a time.  Channels are independent, so that nothing is exchanged
// between threads.  The forward pass leaves the state before every span but the first where
// a gradient will be taken; the backward pass walks the spans from the last, computes the
// states within one again from there, and so reads no rounded output.
//
// Where rows and channels are too few to fill the device, the tokens of a row are cut in
// pieces of whole spans.  A piece takes the state before it, h, to A h + E with A the product
// of its a_t and E its last state from zero: a first launch leaves (A, E) of every piece, and
// each piece of the second composes those before it, in their order.  Backward alike, from
// the right.
//
// A masked token's x and gate are not used: its loads go to the span's first token, whose
// line is read anyway.
#include "tgx_ops.h"

namespace tgx {
namespace {

constexpr int kScanThreads = 256;
constexpr int kSpan = 16;

struct ScanArgs {
  const void* x;
  const void* gate;
  const uint8_t* mask;
  const float* state;
  const void* dout;
  const float* dlast;
  void* out;
  float* last;
  float* starts;  // [batch, spans - 1, dim]
  float* ends;    // [2, batch, pieces, dim]
  void* dx;
  void* dgate;
  float* dstate;
  int64_t x_stride[2], gate_stride[2], mask_stride;
  int64_t length, batch;
  uint32_t items, packs, pieces;
  int32_t dim, per;  // per: tokens a piece, whole spans
};

// which thread does what
template <int V>
struct Part {
  int64_t row;
  uint32_t piece;
  int c, begin, end;  // channel, tokens
  __device__ Part(const ScanArgs& a, uint32_t id) {
    const uint32_t pack = id % a.packs, r = id / a.packs;
    piece = r % a.pieces;
    row = r / a.pieces;
    c = min(static_cast<int>(pack) * V, a.dim - V);
    begin = static_cast<int>(piece) * a.per;
    end = static_cast<int>(min(static_cast<int64_t>(begin) + a.per, a.length));
  }
};

// bit i: token t + i is kept; the bits from n on are 0
__device__ __forceinline__ uint32_t kept(const ScanArgs& a, int64_t row, int t, int n) {
  if (a.mask == nullptr) return (1u << n) - 1;
  const uint8_t* m = a.mask + row * a.mask_stride + t;
  uint32_t bits = 0;
  if (n == kSpan) {
    const Pack<uint8_t, kSpan> p = load_pack<uint8_t, kSpan>(m);
#pragma unroll
    for (int i = 0; i < kSpan; ++i) bits |= (p.v[i] != 0 ? 1u : 0u) << i;
  } else {
    for (int i = 0; i < n; ++i) bits |= (m[i] != 0 ? 1u : 0u) << i;
  }
  return bits;
}

// the tokens of a span that `bits` names; the others' places hold the first token
template <typename T, int V>
__device__ __forceinline__ void load_span(Pack<T, V> (&p)[kSpan], const T* first, int64_t stride, uint32_t bits) {
#pragma unroll
  for (int i = 0; i < kSpan; ++i) p[i] = load_pack<T, V>(first + ((bits >> i) & 1 ? i * stride : 0));
}

template <typename T, int V>
__device__ __forceinline__ const T* token(const void* p, const int64_t (&stride)[2], int64_t row, int t, int c) {
  return static_cast<const T*>(p) + row * stride[0] + t * stride[1] + c;
}

template <typename T, int V>
__global__ __launch_bounds__(kScanThreads) void scan_fwd(const ScanArgs a) {
  const uint32_t id = blockIdx.x * kScanThreads + threadIdx.x;
  if (id >= a.items) return;
  const Part<V> at(a, id);
  float h[V];
#pragma unroll
  for (int u = 0; u < V; ++u) h[u] = a.state != nullptr ? a.state[at.row * a.dim + at.c + u] : 0.f;
  if (at.piece > 0) {
    const float* before = a.ends + at.row * a.pieces * a.dim + at.c;
    const int64_t plane = a.batch * a.pieces * a.dim;
#pragma unroll 4
    for (uint32_t p = 0; p < at.piece; ++p)
#pragma unroll
      for (int u = 0; u < V; ++u) {
        const float* e = before + static_cast<int64_t>(p) * a.dim + u;
        h[u] = fmaf(e[0], h[u], e[plane]);
      }
  }
  const int64_t spans = (a.length + kSpan - 1) / kSpan;
  T* out = static_cast<T*>(a.out) + at.row * a.length * a.dim + at.c;
  for (int t = at.begin; t < at.end; t += kSpan) {
    const int n = min(kSpan, at.end - t);
    const uint32_t bits = kept(a, at.row, t, n);
    Pack<T, V> x[kSpan], g[kSpan];
    load_span<T, V>(x, token<T, V>(a.x, a.x_stride, at.row, t, at.c), a.x_stride[1], bits);
    load_span<T, V>(g, token<T, V>(a.gate, a.gate_stride, at.row, t, at.c), a.gate_stride[1], bits);
    if (a.starts != nullptr && t > 0) {
      Pack<float, V> p;
#pragma unroll
      for (int u = 0; u < V; ++u) p.v[u] = h[u];
      store_pack<float, V>(a.starts + (at.row * (spans - 1) + t / kSpan - 1) * a.dim + at.c, p);
    }
#pragma unroll
    for (int i = 0; i < kSpan; ++i) {
      if (i >= n) break;
      Pack<T, V> o;
#pragma unroll
      for (int u = 0; u < V; ++u) {
        float f, rest;
        sigmoids(to_f(g[i].v[u]), f, rest);
        const float next = fmaf(f, h[u], rest * to_f(x[i].v[u]));
        h[u] = (bits >> i) & 1 ? next : h[u];
        o.v[u] = from_f<T>(h[u]);
      }
      store_pack<T, V>(out + static_cast<int64_t>(t + i) * a.dim, o);
    }
  }
  if (at.piece == a.pieces - 1)
#pragma unroll
    for (int u = 0; u < V; ++u) a.last[at.row * a.dim + at.c + u] = h[u];
}

// (A, E) of every piece but the last; BACK: (A, R) of every piece but the first, where the
// gradient c that reaches the piece from the right leaves it as A c + R
template <typename T, int V, bool BACK>
__global__ __launch_bounds__(kScanThreads) void scan_ends(const ScanArgs a) {
  const uint32_t id = blockIdx.x * kScanThreads + threadIdx.x;
  if (id >= a.items) return;
  const Part<V> at(a, id);
  if (at.piece == (BACK ? 0 : a.pieces - 1)) return;
  float all[V], end[V];
#pragma unroll
  for (int u = 0; u < V; ++u) all[u] = 1.f, end[u] = 0.f;
  const int spans = (at.end - at.begin + kSpan - 1) / kSpan;
  for (int s = 0; s < spans; ++s) {
    const int t = at.begin + (BACK ? spans - 1 - s : s) * kSpan;
    const int n = min(kSpan, at.end - t);
    const uint32_t bits = kept(a, at.row, t, n);
    Pack<T, V> x[kSpan], g[kSpan];
    load_span<T, V>(g, token<T, V>(a.gate, a.gate_stride, at.row, t, at.c), a.gate_stride[1], bits);
    if constexpr (BACK) {
      if (a.dout != nullptr)
        load_span<T, V>(x, static_cast<const T*>(a.dout) + (at.row * a.length + t) * a.dim + at.c, a.dim, (1u << n) - 1);
    } else {
      load_span<T, V>(x, token<T, V>(a.x, a.x_stride, at.row, t, at.c), a.x_stride[1], bits);
    }
#pragma unroll
    for (int j = 0; j < kSpan; ++j) {
      const int i = BACK ? kSpan - 1 - j : j;
      const bool keep = (bits >> i) & 1;
#pragma unroll
      for (int u = 0; u < V; ++u) {
        float f, rest;
        sigmoids(to_f(g[i].v[u]), f, rest);
        f = keep ? f : 1.f;
        if constexpr (BACK) end[u] = f * (end[u] + (a.dout != nullptr && i < n ? to_f(x[i].v[u]) : 0.f));
        else end[u] = keep ? fmaf(f, end[u], rest * to_f(x[i].v[u])) : end[u];
        all[u] *= f;
      }
    }
  }
  float* to = a.ends + (at.row * a.pieces + at.piece) * a.dim + at.c;
  const int64_t plane = a.batch * a.pieces * a.dim;
#pragma unroll
  for (int u = 0; u < V; ++u) {
    to[u] = all[u];
    to[plane + u] = end[u];
  }
}

template <typename T, int V>
__global__ __launch_bounds__(kScanThreads) void scan_bwd(const ScanArgs a) {
  const uint32_t id = blockIdx.x * kScanThreads + threadIdx.x;
  if (id >= a.items) return;
  const Part<V> at(a, id);
  float c[V];
#pragma unroll
  for (int u = 0; u < V; ++u) c[u] = a.dlast != nullptr ? a.dlast[at.row * a.dim + at.c + u] : 0.f;
  const float* ends = a.ends + at.row * a.pieces * a.dim + at.c;
  const int64_t plane = a.batch * a.pieces * a.dim;
#pragma unroll 4
  for (uint32_t p = a.pieces - 1; p > at.piece; --p)
#pragma unroll
    for (int u = 0; u < V; ++u) {
      const float* e = ends + static_cast<int64_t>(p) * a.dim + u;
      c[u] = fmaf(e[0], c[u], e[plane]);
    }
  const int64_t spans = (a.length + kSpan - 1) / kSpan, first = at.row * a.length * a.dim + at.c;
  for (int t = at.begin + (at.end - at.begin - 1) / kSpan * kSpan; t >= at.begin && at.end > at.begin; t -= kSpan) {
    const int n = min(kSpan, at.end - t);
    const uint32_t bits = kept(a, at.row, t, n);
    Pack<T, V> x[kSpan], g[kSpan], d[kSpan];
    load_span<T, V>(x, token<T, V>(a.x, a.x_stride, at.row, t, at.c), a.x_stride[1], bits);
    load_span<T, V>(g, token<T, V>(a.gate, a.gate_stride, at.row, t, at.c), a.gate_stride[1], bits);
    if (a.dout != nullptr)
      load_span<T, V>(d, static_cast<const T*>(a.dout) + first + static_cast<int64_t>(t) * a.dim, a.dim, (1u << n) - 1);
    float h[V], f[kSpan][V], rest[kSpan][V], off[kSpan][V];
#pragma unroll
    for (int u = 0; u < V; ++u)
      h[u] = t > 0 ? a.starts[(at.row * (spans - 1) + t / kSpan - 1) * a.dim + at.c + u]
                   : a.state != nullptr ? a.state[at.row * a.dim + at.c + u] : 0.f;
#pragma unroll
    for (int i = 0; i < kSpan; ++i)
#pragma unroll
      for (int u = 0; u < V; ++u) {
        const float v = to_f(x[i].v[u]);
        sigmoids(to_f(g[i].v[u]), f[i][u], rest[i][u]);
        off[i][u] = h[u] - v;
        h[u] = (bits >> i) & 1 ? fmaf(f[i][u], h[u], rest[i][u] * v) : h[u];
      }
#pragma unroll
    for (int i = kSpan - 1; i >= 0; --i) {
      if (i >= n) continue;
      const bool keep = (bits >> i) & 1;
      Pack<T, V> px, pg;
#pragma unroll
      for (int u = 0; u < V; ++u) {
        const float dh = (a.dout != nullptr ? to_f(d[i].v[u]) : 0.f) + c[u];
        const float dx = dh * rest[i][u], back = dh * f[i][u];
        px.v[u] = from_f<T>(keep ? dx : 0.f);
        pg.v[u] = from_f<T>(keep ? dx * f[i][u] * off[i][u] : 0.f);
        c[u] = keep ? back : dh;
      }
      const int64_t to = first + static_cast<int64_t>(t + i) * a.dim;
      if (a.dx != nullptr) store_pack<T, V>(static_cast<T*>(a.dx) + to, px);
      if (a.dgate != nullptr) store_pack<T, V>(static_cast<T*>(a.dgate) + to, pg);
    }
  }
  if (at.piece == 0 && a.dstate != nullptr)
#pragma unroll
    for (int u = 0; u < V; ++u) a.dstate[at.row * a.dim + at.c + u] = c[u];
}

// channels a thread takes: 4 bytes of them
template <typename T>
constexpr int kChannels = 4 / sizeof(T);

struct Pieces {
  int64_t packs, per, pieces;
};

// the tokens a piece: as many pieces as bring about kFill threads, of 64 tokens or more
constexpr int64_t kFill = 131072;
Pieces cut(const tgx_scan_args* a) {
  const int64_t v = a->dtype == TGX_BF16 && a->dim >= kChannels<bf16> ? kChannels<bf16> : 1;
  Pieces p{ops_cdiv(a->dim, v), 0, 1};
  const int64_t threads = std::max<int64_t>(1, a->batch * p.packs);
  const int64_t most = std::clamp<int64_t>(kFill / threads, 1, std::max<int64_t>(1, a->length / 64));
  p.per = std::max<int64_t>(kSpan, ops_cdiv(ops_cdiv(a->length, most), kSpan) * kSpan);
  p.pieces = std::max<int64_t>(1, ops_cdiv(a->length, p.per));
  return p;
}

int check_scan(const char* what, const tgx_scan_args* a) {
  if (a == nullptr) return fail(TGX_ERR_ARG, "%s: args is NULL", what);
  if (a->batch < 0 || a->length < 0 || a->dim < 1)
    return fail(TGX_ERR_ARG, "%s: batch=%lld length=%lld dim=%lld", what, static_cast<long long>(a->batch),
                static_cast<long long>(a->length), static_cast<long long>(a->dim));
  if (elem_bytes(a->dtype) == 0) return fail(TGX_ERR_DTYPE, "%s: dtype %d", what, a->dtype);
  const int64_t most = int64_t(1) << 30;
  if (a->length > most || a->dim > most || a->batch > most || a->batch > (int64_t(1) << 32) / a->dim)
    return fail(TGX_ERR_LIMIT, "%s: batch=%lld length=%lld dim=%lld: more than one launch takes", what,
                static_cast<long long>(a->batch), static_cast<long long>(a->length), static_cast<long long>(a->dim));
  if (a->batch > 0 && a->length > 0 && (a->x == nullptr || a->gate == nullptr))
    return fail(TGX_ERR_ARG, "%s: x and gate must not be NULL", what);
  return TGX_OK;
}

size_t scan_ends_bytes(const tgx_scan_args* a) {
  const Pieces p = cut(a);
  return p.pieces > 1 ? static_cast<size_t>(2 * a->batch * p.pieces * a->dim) * 4 : 0;
}

// f<T, V>() launches
template <typename F>
int launch_scan(const char* what, const tgx_scan_args* p, F&& f) {
  ScanArgs a{};
  a.x = p->x;
  a.gate = p->gate;
  a.mask = p->mask;
  a.state = p->state;
  a.dout = p->grad_out;
  a.dlast = p->grad_last;
  a.out = p->out;
  a.last = p->last;
  a.starts = p->starts;
  a.ends = static_cast<float*>(p->workspace);
  a.dx = p->grad_x;
  a.dgate = p->grad_gate;
  a.dstate = p->grad_state;
  for (int i = 0; i < 2; ++i) a.x_stride[i] = p->x_stride[i], a.gate_stride[i] = p->gate_stride[i];
  a.mask_stride = p->mask_stride;
  a.length = p->length;
  a.batch = p->batch;
  a.dim = static_cast<int32_t>(p->dim);
  const Pieces c = cut(p);
  const size_t need = scan_ends_bytes(p);
  if (need > 0 && (p->workspace == nullptr || p->workspace_bytes < need || !aligned16(p->workspace)))
    return fail(TGX_ERR_ARG, "%s: workspace of %zu bytes, 16-byte aligned, needed", what, need);
  const int64_t items = p->batch * c.packs * c.pieces, blocks = ops_cdiv(items, kScanThreads);
  if (const int e = check_grid(what, blocks, kScanThreads)) return e;
  a.items = static_cast<uint32_t>(items);
  a.packs = static_cast<uint32_t>(c.packs);
  a.pieces = static_cast<uint32_t>(c.pieces);
  a.per = static_cast<int32_t>(c.per);
  return by_type(p->dtype, [&](auto t) {
    using T = decltype(t);
    if constexpr (kChannels<T> > 1) {
      if (p->dim < kChannels<T>) return f(t, std::integral_constant<int, 1>{}, a, dim3(static_cast<unsigned>(blocks)));
    }
    return f(t, std::integral_constant<int, kChannels<T>>{}, a, dim3(static_cast<unsigned>(blocks)));
  });
}

}  // namespace
}  // namespace tgx

using namespace tgx;

extern "C" int64_t tgx_scan_starts(int64_t length) { return length <= kSpan ? 0 : (length - 1) / kSpan; }

extern "C" size_t tgx_scan_workspace_size(const tgx_scan_args* args) {
  return check_scan("tgx_scan", args) ? 0 : scan_ends_bytes(args);
}

extern "C" int tgx_scan(const tgx_scan_args* args, void* stream) {
  if (const int rc = check_scan("tgx_scan", args)) return rc;
  if (args->batch == 0) return TGX_OK;
  if (args->last == nullptr || (args->length > 0 && args->out == nullptr))
    return fail(TGX_ERR_ARG, "tgx_scan: out and last must not be NULL");
  hipStream_t s = static_cast<hipStream_t>(stream);
  return launch_scan("tgx_scan", args, [&](auto t, auto v, const ScanArgs& a, dim3 grid) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value;
    if (a.pieces > 1) {
      hipLaunchKernelGGL((scan_ends<T, V, false>), grid, dim3(kScanThreads), 0, s, a);
      if (const int e = check_launch("scan_ends")) return e;
    }
    hipLaunchKernelGGL((scan_fwd<T, V>), grid, dim3(kScanThreads), 0, s, a);
    return check_launch("scan_fwd");
  });
}

extern "C" int tgx_scan_grad(const tgx_scan_args* args, void* stream) {
  if (const int rc = check_scan("tgx_scan_grad", args)) return rc;
  if (args->batch == 0 || (args->grad_x == nullptr && args->grad_gate == nullptr && args->grad_state == nullptr))
    return TGX_OK;
  if (tgx_scan_starts(args->length) > 0 && args->starts == nullptr)
    return fail(TGX_ERR_ARG, "tgx_scan_grad: starts must not be NULL");
  hipStream_t s = static_cast<hipStream_t>(stream);
  return launch_scan("tgx_scan_grad", args, [&](auto t, auto v, const ScanArgs& a, dim3 grid) {
    using T = decltype(t);
    constexpr int V = decltype(v)::value;
    if (a.pieces > 1) {
      hipLaunchKernelGGL((scan_ends<T, V, true>), grid, dim3(kScanThreads), 0, s, a);
      if (const int e = check_launch("scan_ends")) return e;
    }
    hipLaunchKernelGGL((scan_bwd<T, V>), grid, dim3(kScanThreads), 0, s, a);
    return check_launch("scan_bwd");
  });
}
