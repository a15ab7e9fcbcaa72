// A gated recurrence along the tokens of every batch row, forward and backward.
//
//   a_t = sigmoid(gate_t),  h_t = a_t h_{t-1} + (1 - a_t) x_t     (a masked token: h_t = h_{t-1})
//   dh_t = dout_t + a_{t+1} dh_{t+1}                              (dlast joins the last one)
//   dx_t = (1 - a_t) dh_t,  dgate_t = a_t (1 - a_t) (h_{t-1} - x_t) dh_t,  dstate = a_1 dh_1
//
// A thread keeps the state of V neighbouring channels of one row in 32 bits and walks the
// row's tokens kSpan at a time, the next span's on their way while it works on one.  Channels
// are independent, so that nothing is exchanged between threads.  The forward pass leaves the
// state before every span but the first where a gradient will be taken; the backward pass
// walks the spans from the last, computes the states within one again from there, and so
// reads no rounded output.
//
// Where rows and channels are too few to fill the device, the tokens of a row are cut in
// pieces of whole spans.  A piece takes the state before it, h, to A h + E with A the product
// of its a_t and E its last state from zero: a first launch leaves (A, E) of every piece, a
// second one turns them into the states between the pieces, in their order, and a third walks
// the pieces.  Backward alike, from the right.
//
// A masked token's x and gate are not used: its loads go to the span's first token, whose
// line is read anyway.
//
// Memory bounds it: 24,576 rows of 32 tokens and 172 bf16 channels take 175 us forward (0.75
// GB) and 282 backward (1.29 GB; medians), 4.3 and 4.6 TB/s; with the gates' arithmetic taken out they
// took the same.  4 bytes a lane and rows that end inside a line are what keeps it below a
// copy's 5 to 6.  2 rows of 30,001 tokens and 256 channels: 19 + 5 + 21 us forward and 24 + 5 + 31
// backward for the ends, what is between the pieces, and the pieces, which read x, gate and
// dout a second time.  A single token of 12 rows: 3 us.
#include "tgx_ops.h"

namespace tgx {
namespace {

// In one sweep 24,576 rows of 32 tokens and 172 bf16 channels take 175 us forward and 279 backward, with 128
// threads 188 and 292, with 512 184 and 318; 600 rows of 512 tokens and 100 f32 channels 89 and
// 141, 102 and 158, 136 and 223.
constexpr int kScanThreads = 256;
constexpr int kSpan = 8;

struct __attribute__((packed, aligned(1))) Words {
  uint32_t v[kSpan / 4];
};

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

// The workgroup's number, dealt out so that kNear of them that follow each other run on the same
// of the 8 dies, which the device gives workgroups in turn.  A row of odd length ends inside a
// cache line, and so does a workgroup's share of it at every token: neighbours that find those
// lines in one L2 write them once.  24,576 rows of 32 tokens and 172 bf16 channels, trained: 447
// us with 16, 466 with 4, 469 with an eighth of the grid, and 508 as they come.
__device__ __forceinline__ uint32_t block_number() {
  constexpr uint32_t kDies = 8, kNear = 16, kGroup = kDies * kNear;
  const uint32_t group = blockIdx.x / kGroup * kGroup, at = blockIdx.x % kGroup;
  const uint32_t size = min(gridDim.x - group, kGroup), die = at % kDies;
  return group + die * (size / kDies) + min(die, size % kDies) + at / kDies;
}

// which thread does what, and where its tensors' values begin
template <typename T, int V, typename O>
struct Part {
  O row, x, gate, dense, states, starts, ends;  // bytes to: its row's x, gate, [length, dim] values, [dim], ...
  O x_step, gate_step, dense_step, states_step;  // bytes a token, and a row of dim floats
  uint32_t piece;
  int begin, end;  // tokens
  __device__ Part(const ScanArgs& a, uint32_t id) {
    const uint32_t pack = id % a.packs, r = id / a.packs;
    piece = r % a.pieces;
    row = r / a.pieces;
    const O c = min(static_cast<int>(pack) * V, a.dim - V), dim = a.dim;
    begin = static_cast<int>(piece) * a.per;
    end = static_cast<int>(min(static_cast<int64_t>(begin) + a.per, a.length));
    x_step = static_cast<O>(a.x_stride[1]) * sizeof(T);
    gate_step = static_cast<O>(a.gate_stride[1]) * sizeof(T);
    dense_step = dim * sizeof(T);
    states_step = dim * 4;
    x = (row * static_cast<O>(a.x_stride[0]) + c) * sizeof(T);
    gate = (row * static_cast<O>(a.gate_stride[0]) + c) * sizeof(T);
    dense = (row * static_cast<O>(a.length) * dim + c) * sizeof(T);
    states = (row * dim + c) * 4;
    starts = (row * ((static_cast<O>(a.length) + kSpan - 1) / kSpan - 1) * dim + c) * 4;
    ends = ((row * a.pieces + piece) * dim + c) * 4;
  }
  // the state before the span that begins at token t > 0
  __device__ O start(int t) const { return starts + static_cast<O>(t / kSpan - 1) * states_step; }
};

// bit i: byte i of a span's is not 0
__device__ __forceinline__ uint32_t byte_bits(const Pack<uint8_t, kSpan>& p) {
  const Words w = __builtin_bit_cast(Words, p);
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < kSpan / 4; ++i) {
    const uint32_t high = (((w.v[i] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w.v[i]) & 0x80808080u;
    bits |= ((((high >> 7) * 0x00204081u) >> 21) & 0xfu) << (4 * i);
  }
  return bits;
}

// bit i: token t + i of a row's last n < kSpan tokens is kept
template <bool MASK>
__device__ __forceinline__ uint32_t kept_last(const ScanArgs& a, uint64_t row, int t, int n) {
  if (!MASK) return (1u << n) - 1;
  const uint8_t* m = a.mask + static_cast<int64_t>(row) * a.mask_stride + t;
  Pack<uint8_t, kSpan> p;
#pragma unroll
  for (int i = 0; i < kSpan; ++i) p.v[i] = i < n ? m[i] : 0;
  return byte_bits(p);
}

// Offsets are of bytes, in 32 bits (O) where every tensor ends within 4 GiB of its start: a
// quarter of the backward pass's instructions and half of its registers are addresses
// otherwise.
template <typename T, int V, typename O>
__device__ __forceinline__ Pack<T, V> load_at(const void* p, O off) {
  return load_pack<T, V>(reinterpret_cast<const T*>(static_cast<const char*>(p) + off));
}
template <typename T, int V, typename O>
__device__ __forceinline__ void store_at(void* p, O off, const Pack<T, V>& x) {
  store_pack<T, V>(reinterpret_cast<T*>(static_cast<char*>(p) + off), x);
}
template <int V, typename O>
__device__ __forceinline__ void load_floats(float (&to)[V], const float* from, O off) {
  const Pack<float, V> p = load_at<float, V>(from, off);
#pragma unroll
  for (int u = 0; u < V; ++u) to[u] = p.v[u];
}
template <int V, typename O>
__device__ __forceinline__ void store_floats(float* to, O off, const float (&from)[V]) {
  Pack<float, V> p;
#pragma unroll
  for (int u = 0; u < V; ++u) p.v[u] = from[u];
  store_at<float, V>(to, off, p);
}

constexpr uint32_t kAll = (1u << kSpan) - 1;

// a span's tokens from `first` on, `stride` apart, those that `bits` names; the others' places
// hold the first one
template <typename T, int V, typename O>
__device__ __forceinline__ void load_span(Pack<T, V> (&p)[kSpan], const void* from, O first, O stride, uint32_t bits) {
  O at = first;
#pragma unroll
  for (int i = 0; i < kSpan; ++i) {
    p[i] = load_at<T, V>(from, (bits >> i) & 1 ? at : first);
    at += stride;
  }
}

// what enters a piece: the state before it, or the gradient that reaches it from the right
template <typename T, int V, typename O>
__device__ __forceinline__ void enter(float (&h)[V], const ScanArgs& a, const Part<T, V, O>& at, const float* outer) {
#pragma unroll
  for (int u = 0; u < V; ++u) h[u] = 0.f;
  if (a.pieces > 1) load_floats(h, a.ends + a.batch * a.pieces * a.dim, at.ends);
  else if (outer != nullptr) load_floats(h, outer, at.states);
}

// Walks a piece's spans, from the first or from the last: load(span, t, bits) and then
// f(span, t, n) with n = kSpan, or fewer for a row's last tokens.  While one whole span is
// worked on, the next one's values and the mask after it are on their way: the loop's loads
// and stores are the same in every pass, so that the compiler's waits, which count them, reach
// no further than they have to.
template <bool BACK, bool MASK, typename S, typename L, typename F>
__device__ __forceinline__ void walk(const ScanArgs& a, uint64_t row, int begin, int end, L&& load, F&& f) {
  const int spans = (end - begin) / kSpan, rest = end - begin - spans * kSpan;
  S one, other;
  auto last = [&] {
    if (rest > 0) {
      const int t = begin + spans * kSpan;
      one.bits = kept_last<MASK>(a, row, t, rest);
      load(one, t, (1u << rest) - 1);
      f(one, t, rest);
    }
  };
  if (BACK) last();
  if (spans > 0) {
    auto at = [&](int k) { return begin + (BACK ? spans - 1 - k : k) * kSpan; };
    const uint8_t* m = MASK ? a.mask + static_cast<int64_t>(row) * a.mask_stride : nullptr;
    Pack<uint8_t, kSpan> raw;
    auto mask = [&](int k) {
      if constexpr (MASK) raw = load_pack<uint8_t, kSpan>(m + at(min(k, spans - 1)));
    };
    auto stage = [&](S& s, int k) {
      s.bits = kAll;
      if constexpr (MASK) s.bits = byte_bits(raw);
      mask(k + 1);
      load(s, at(k), kAll);
    };
    mask(0);
    stage(one, 0);
    for (int k = 0;;) {
      if (k + 1 == spans) {
        f(one, at(k), kSpan);
        break;
      }
      stage(other, k + 1);
      f(one, at(k), kSpan);
      if (++k + 1 == spans) {
        f(other, at(k), kSpan);
        break;
      }
      stage(one, k + 1);
      f(other, at(k), kSpan);
      ++k;
    }
  }
  if (!BACK) last();
}

template <typename T, int V>
struct Tokens {
  Pack<T, V> x[kSpan], g[kSpan];
  uint32_t bits;
};

template <typename T, int V, typename O, bool MASK>
__global__ __launch_bounds__(kScanThreads) void scan_fwd(const ScanArgs a) {
  const uint32_t id = block_number() * kScanThreads + threadIdx.x;
  if (id >= a.items) return;
  const Part<T, V, O> at(a, id);
  float h[V];
  enter(h, a, at, a.state);
  walk<false, MASK, Tokens<T, V>>(
      a, at.row, at.begin, at.end,
      [&](Tokens<T, V>& s, int t, uint32_t) {
        load_span<T, V, O>(s.x, a.x, at.x + t * at.x_step, at.x_step, s.bits);
        load_span<T, V, O>(s.g, a.gate, at.gate + t * at.gate_step, at.gate_step, s.bits);
      },
      [&](const Tokens<T, V>& s, int t, int n) {
        if (a.starts != nullptr && t > 0) store_floats(a.starts, at.start(t), h);
        O to = at.dense + t * at.dense_step;
#pragma unroll
        for (int i = 0; i < kSpan; ++i) {
          if (i >= n) break;
          Pack<T, V> o;
#pragma unroll
          for (int u = 0; u < V; ++u) {
            float f, rest;
            sigmoids(to_f(s.g[i].v[u]), f, rest);
            const float next = fmaf(f, h[u], rest * to_f(s.x[i].v[u]));
            h[u] = !MASK || ((s.bits >> i) & 1) ? next : h[u];
            o.v[u] = from_f<T>(h[u]);
          }
          store_at<T, V>(a.out, to, o);
          to += at.dense_step;
        }
      });
  if (at.piece == a.pieces - 1) store_floats(a.last, at.states, h);
}

// (A, E) of every piece but the last; BACK: (A, R) of every piece but the first, where the
// gradient c that reaches the piece from the right leaves it as A c + R
template <typename T, int V, typename O, bool MASK, bool BACK>
__global__ __launch_bounds__(kScanThreads) void scan_ends(const ScanArgs a) {
  const uint32_t id = block_number() * kScanThreads + threadIdx.x;
  if (id >= a.items) return;
  const Part<T, V, O> at(a, id);
  if (at.piece == (BACK ? 0 : a.pieces - 1)) return;
  float all[V], end[V];
#pragma unroll
  for (int u = 0; u < V; ++u) all[u] = 1.f, end[u] = 0.f;
  const bool given = !BACK || a.dout != nullptr;
  walk<BACK, MASK, Tokens<T, V>>(
      a, at.row, at.begin, at.end,
      [&](Tokens<T, V>& s, int t, uint32_t there) {
        if (!BACK) load_span<T, V, O>(s.x, a.x, at.x + t * at.x_step, at.x_step, s.bits);
        else if (given) load_span<T, V, O>(s.x, a.dout, at.dense + t * at.dense_step, at.dense_step, there);
        load_span<T, V, O>(s.g, a.gate, at.gate + t * at.gate_step, at.gate_step, s.bits);
      },
      [&](const Tokens<T, V>& s, int, int n) {
        float held[V];  // masked tokens' gradients, as in scan_bwd
#pragma unroll
        for (int u = 0; u < V; ++u) held[u] = 0.f;
#pragma unroll
        for (int j = 0; j < kSpan; ++j) {
          const int i = BACK ? kSpan - 1 - j : j;
          if (i >= n) continue;
          const bool keep = !MASK || ((s.bits >> i) & 1);
#pragma unroll
          for (int u = 0; u < V; ++u) {
            float f, rest;
            sigmoids(to_f(s.g[i].v[u]), f, rest);
            f = keep ? f : 1.f;
            if constexpr (BACK) {
              const float d = held[u] + (given ? to_f(s.x[i].v[u]) : 0.f);
              end[u] = keep ? f * (end[u] + d) : end[u];
              held[u] = keep ? 0.f : d;
            } else {
              end[u] = keep ? fmaf(f, end[u], rest * to_f(s.x[i].v[u])) : end[u];
            }
            all[u] *= f;
          }
        }
        if (BACK && MASK)
#pragma unroll
          for (int u = 0; u < V; ++u) end[u] += held[u];
      });
  store_floats(a.ends, at.ends, all);
  store_floats(a.ends + a.batch * a.pieces * a.dim, at.ends, end);
}

// Turns the (A, E) between the pieces into what enters each, in E's place.  kSegments threads
// share a channel's pieces: each composes its own, then takes what the segments before it
// make of the outer state through them.  Its pieces stay in registers on the way if they are
// no more than kOwn: 251 pieces of 2 rows of 256 channels take 4.5 us with 32 segments, 6.5
// with 16, which read their pieces twice, and 5.8 with 64, of 16-byte loads.
constexpr int kSegments = 32;
constexpr int kCarryChannels = kScanThreads / kSegments;
constexpr int kOwn = 8;

template <bool BACK>
__global__ __launch_bounds__(kScanThreads) void scan_carry(const ScanArgs a) {
  __shared__ float lds[2][kSegments][kCarryChannels];
  const int lane = threadIdx.x % kCarryChannels, seg = threadIdx.x / kCarryChannels;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kCarryChannels + lane;
  const bool live = id < a.batch * a.dim;
  const int64_t row = live ? id / a.dim : 0, c = live ? id % a.dim : 0;
  const int pieces = static_cast<int>(a.pieces), per = (pieces + kSegments - 1) / kSegments;
  const int lo = min(seg * per, pieces), hi = min(lo + per, pieces);
  const int64_t plane = a.batch * a.pieces * a.dim;
  float* ends = a.ends + row * a.pieces * a.dim + c;
  auto piece = [&](int p) { return ends + static_cast<int64_t>(BACK ? pieces - 1 - p : p) * a.dim; };
  const float* outer = BACK ? a.dlast : a.state;
  float h = live && outer != nullptr ? outer[row * a.dim + c] : 0.f;
  float all = 1.f, end = 0.f, f[kOwn], g[kOwn];
  const bool own = per <= kOwn;
  if (live && own) {
    // the last piece leads nowhere, and its place holds nothing
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const bool there = lo + i < min(hi, pieces - 1);
      const float* e = piece(min(lo + i, pieces - 1));
      f[i] = there ? e[0] : 1.f;
      g[i] = there ? e[plane] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      all *= f[i];
      end = fmaf(f[i], end, g[i]);
    }
  } else if (live) {
#pragma unroll 8
    for (int p = lo; p < min(hi, pieces - 1); ++p) {
      const float* e = piece(p);
      all *= e[0];
      end = fmaf(e[0], end, e[plane]);
    }
  }
  lds[0][seg][lane] = all;
  lds[1][seg][lane] = end;
  __syncthreads();
  if (!live) return;
  for (int s = 0; s < seg; ++s) h = fmaf(lds[0][s][lane], h, lds[1][s][lane]);
  if (own) {
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      if (lo + i < hi) piece(lo + i)[plane] = h;
      h = fmaf(f[i], h, g[i]);
    }
    return;
  }
#pragma unroll 8
  for (int p = lo; p < hi; ++p) {
    float* e = piece(p);
    const float f = e[0], g = e[plane];
    e[plane] = h;
    if (p < pieces - 1) h = fmaf(f, h, g);
  }
}

template <typename T, int V>
struct TokensBack {
  Pack<T, V> x[kSpan], g[kSpan], d[kSpan];
  float h[V];
  uint32_t bits;
};

// a pack, or zeros
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> kept_pack(const Pack<T, V>& p, bool keep) {
  Pack<T, V> o;
  if constexpr (sizeof(p) == 4) {
    o = __builtin_bit_cast(Pack<T, V>, keep ? __builtin_bit_cast(uint32_t, p) : 0u);
  } else {
#pragma unroll
    for (int u = 0; u < V; ++u) o.v[u] = keep ? p.v[u] : from_f<T>(0.f);
  }
  return o;
}

template <typename T, int V, typename O, bool MASK, bool DOUT>
__global__ __launch_bounds__(kScanThreads) void scan_bwd(const ScanArgs a) {
  // from the last rows: what the forward pass read last is still in the caches
  const uint32_t id = (gridDim.x - 1 - block_number()) * kScanThreads + threadIdx.x;
  if (id >= a.items) return;
  const Part<T, V, O> at(a, id);
  float c[V];
  enter(c, a, at, a.dlast);
  walk<true, MASK, TokensBack<T, V>>(
      a, at.row, at.begin, at.end,
      [&](TokensBack<T, V>& s, int t, uint32_t there) {
#pragma unroll
        for (int u = 0; u < V; ++u) s.h[u] = 0.f;
        if (t > 0) load_floats(s.h, a.starts, at.start(t));
        else if (a.state != nullptr) load_floats(s.h, a.state, at.states);
        load_span<T, V, O>(s.x, a.x, at.x + t * at.x_step, at.x_step, s.bits);
        load_span<T, V, O>(s.g, a.gate, at.gate + t * at.gate_step, at.gate_step, s.bits);
        if constexpr (DOUT) load_span<T, V, O>(s.d, a.dout, at.dense + t * at.dense_step, at.dense_step, there);
      },
      [&](const TokensBack<T, V>& s, int t, int n) {
        // dx = rest dh, dgate = grow dh, and f dh goes on to the token before.  Of f and rest the
        // smaller one is kept, and the gate's sign says which that is: 16 registers less, and a
        // third wavefront a SIMD.
        // Gradients of masked tokens that follow each other are added up for themselves, and a
        // span's sum to what came from the right: one by one, 500 of them would lose 500 roundings.
        // 600 rows of 512 tokens and 100 f32 channels, masked: the state's gradient is off by 1.3e-7
        // instead of 3.3e-7 (root mean squares), 210 us trained both ways; in bf16 214 instead of 211.
        float h[V], held[V], small[kSpan][V], grow[kSpan][V];
#pragma unroll
        for (int u = 0; u < V; ++u) h[u] = s.h[u], held[u] = 0.f;
#pragma unroll
        for (int i = 0; i < kSpan; ++i)
#pragma unroll
          for (int u = 0; u < V; ++u) {
            const bool keep = !MASK || ((s.bits >> i) & 1);
            const float x = to_f(s.x[i].v[u]), g = to_f(s.g[i].v[u]);
            float f, rest;
            sigmoids(g, f, rest);
            small[i][u] = g < 0.f ? f : rest;
            grow[i][u] = f * rest * (h[u] - x);
            h[u] = keep ? fmaf(f, h[u], rest * x) : h[u];
          }
        O to = at.dense + (t + kSpan) * at.dense_step;
#pragma unroll
        for (int i = kSpan - 1; i >= 0; --i) {
          to -= at.dense_step;
          if (i >= n) continue;
          const bool keep = !MASK || ((s.bits >> i) & 1);
          Pack<T, V> px, pg;
#pragma unroll
          for (int u = 0; u < V; ++u) {
            float d = DOUT ? to_f(s.d[i].v[u]) : 0.f;
            if constexpr (MASK) d += held[u];
            const float dh = d + c[u], big = 1.f - small[i][u];
            const bool neg = to_f(s.g[i].v[u]) < 0.f;
            px.v[u] = from_f<T>(dh * (neg ? big : small[i][u]));
            pg.v[u] = from_f<T>(dh * grow[i][u]);
            c[u] = keep ? dh * (neg ? small[i][u] : big) : c[u];
            held[u] = keep ? 0.f : d;
          }
          store_at<T, V>(a.dx, to, kept_pack(px, keep));
          store_at<T, V>(a.dgate, to, kept_pack(pg, keep));
        }
        if constexpr (MASK)
#pragma unroll
          for (int u = 0; u < V; ++u) c[u] += held[u];
      });
  if (at.piece == 0 && a.dstate != nullptr) store_floats(a.dstate, at.states, c);
}

// channels a thread takes: 4 bytes of them (8 are 2% faster in the forward pass and 40% slower
// backward, whose registers they fill)
template <typename T>
constexpr int kChannels = 4 / sizeof(T);

struct Pieces {
  int64_t per, pieces;
};

// The tokens a piece: as many pieces as bring about kFill threads, a wavefront a SIMD, of 64
// tokens or more.  Threads have enough loads under way that more of them win little: 600 rows
// of 512 tokens and 100 f32 channels (60,000 threads) take 95 us forward and 149 backward in
// one piece, in two 84 and 141, and 47 and 53 for what is between them; 2 rows of 30,001 tokens
// and 256 bf16 channels 47 and 61 with 65,536 threads, 47 and 59 with 131,072, 72 and 93 with
// 32,768.  What this rule costs where it makes few pieces, whole calls forward and trained: two
// lose (300 rows of 512 tokens and 100 f32 channels 53 and 170 us, in one piece 33 and 153; 600
// such rows in bf16 67 and 207, 50 and 173), three are even (200 x 1,024 x 100 f32 66 and 229,
// 59 and 284; 600 x 512 x 64 bf16 48 and 122, 49 and 131), and five or more win on long rows
// (120 x 1,024 x 100 f32 43 and 132, 58 and 211).
constexpr int64_t kFill = 65536;
Pieces cut(const tgx_scan_args* a) {
  const int64_t v = a->dtype == TGX_BF16 && a->dim >= kChannels<bf16> ? kChannels<bf16> : 1;
  const int64_t threads = std::max<int64_t>(1, a->batch * ops_cdiv(a->dim, v));
  const int64_t most = std::clamp<int64_t>(kFill / threads, 1, std::max<int64_t>(1, a->length / 64));
  Pieces p{};
  p.per = std::max<int64_t>(kSpan, ops_cdiv(ops_cdiv(a->length, most), kSpan) * kSpan);
  p.pieces = std::max<int64_t>(1, ops_cdiv(a->length, p.per));
  return p;
}

int check_scan(const char* what, const tgx_scan_args* a) {
  if (a == nullptr) return fail(TGX_ERR_ARG, "%s: args is NULL", what);
  if (a->batch < 0 || a->length < 0 || a->dim < 1)
    return fail(TGX_ERR_ARG, "%s: batch=%lld length=%lld dim=%lld", what, static_cast<long long>(a->batch),
                static_cast<long long>(a->length), static_cast<long long>(a->dim));
  for (int64_t s : {a->x_stride[0], a->x_stride[1], a->gate_stride[0], a->gate_stride[1], a->mask_stride})
    if (s < 0) return fail(TGX_ERR_ARG, "%s: a stride of %lld", what, static_cast<long long>(s));
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

// whether every tensor of the call ends within 4 GiB of its start
bool tensors_near(const tgx_scan_args* p) {
  const int64_t most = int64_t(1) << 32;
  const Pieces c = cut(p);
  const double rows = static_cast<double>(p->batch), n = static_cast<double>(p->length), dim = static_cast<double>(p->dim);
  const double size = elem_bytes(p->dtype);
  const double ends[] = {rows * (n + kSpan) * dim * size, rows * std::max(n / kSpan, static_cast<double>(c.pieces)) * dim * 4,
                         (rows * p->x_stride[0] + (n + kSpan) * p->x_stride[1] + dim) * size,
                         (rows * p->gate_stride[0] + (n + kSpan) * p->gate_stride[1] + dim) * size};
  return std::all_of(ends, ends + 4, [&](double x) { return x < static_cast<double>(most); });
}

ScanArgs scan_args(const tgx_scan_args* p) {
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
  a.pieces = static_cast<uint32_t>(c.pieces);
  a.per = static_cast<int32_t>(c.per);
  return a;
}

// the launches of one direction
template <bool BACK>
int launch_scan(const char* what, const tgx_scan_args* p, hipStream_t s) {
  ScanArgs a = scan_args(p);
  const size_t need = scan_ends_bytes(p);
  if (need > 0 && (p->workspace == nullptr || p->workspace_bytes < need || !aligned16(p->workspace)))
    return fail(TGX_ERR_ARG, "%s: workspace of %zu bytes, 16-byte aligned, needed", what, need);
  const bool near = tensors_near(p);
  return by_type(p->dtype, [&](auto t) {
    using T = decltype(t);
    auto run = [&](auto v) {
      constexpr int V = decltype(v)::value;
      const int64_t packs = ops_cdiv(p->dim, V), items = p->batch * packs * a.pieces;
      const int64_t blocks = ops_cdiv(items, kScanThreads);
      if (const int e = check_grid(what, blocks, kScanThreads)) return e;
      a.packs = static_cast<uint32_t>(packs);
      a.items = static_cast<uint32_t>(items);
      const dim3 grid(static_cast<unsigned>(blocks)), block(kScanThreads);
      // g(O{}, MASK) with the call's kinds
      auto kinds = [&](auto g) {
        auto masked = [&](auto o) { return p->mask != nullptr ? g(o, std::true_type{}) : g(o, std::false_type{}); };
        return near ? masked(uint32_t{}) : masked(uint64_t{});
      };
      if (a.pieces > 1) {
        const int rc = kinds([&](auto o, auto mask) {
          hipLaunchKernelGGL((scan_ends<T, V, decltype(o), decltype(mask)::value, BACK>), grid, block, 0, s, a);
          return check_launch("scan_ends");
        });
        if (rc) return rc;
        const int64_t carries = ops_cdiv(p->batch * p->dim, kCarryChannels);
        if (const int e = check_grid(what, carries, kScanThreads)) return e;
        hipLaunchKernelGGL(scan_carry<BACK>, dim3(static_cast<unsigned>(carries)), block, 0, s, a);
        if (const int e = check_launch("scan_carry")) return e;
      }
      return kinds([&](auto o, auto mask) {
        using O = decltype(o);
        constexpr bool MASK = decltype(mask)::value;
        if constexpr (!BACK) hipLaunchKernelGGL((scan_fwd<T, V, O, MASK>), grid, block, 0, s, a);
        else if (a.dout != nullptr) hipLaunchKernelGGL((scan_bwd<T, V, O, MASK, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((scan_bwd<T, V, O, MASK, false>), grid, block, 0, s, a);
        return check_launch(BACK ? "scan_bwd" : "scan_fwd");
      });
    };
    constexpr int V = kChannels<T>;
    return p->dim < V ? run(std::integral_constant<int, 1>{}) : run(std::integral_constant<int, V>{});
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
  return launch_scan<false>("tgx_scan", args, static_cast<hipStream_t>(stream));
}

extern "C" int tgx_scan_grad(const tgx_scan_args* args, void* stream) {
  if (const int rc = check_scan("tgx_scan_grad", args)) return rc;
  if (args->batch == 0) return TGX_OK;
  if (args->length > 0 && (args->grad_x == nullptr || args->grad_gate == nullptr))
    return fail(TGX_ERR_ARG, "tgx_scan_grad: grad_x and grad_gate must not be NULL");
  if (tgx_scan_starts(args->length) > 0 && args->starts == nullptr)
    return fail(TGX_ERR_ARG, "tgx_scan_grad: starts must not be NULL");
  return launch_scan<true>("tgx_scan_grad", args, static_cast<hipStream_t>(stream));
}
