// Gated linear recurrence over sequences of voxel rows, its backward pass, and its form for one row a sequence.
//   h[t] = f[t] h[t-1] + (1 - f[t]) x[t],  f = sigmoid(gate);  h in front of a sequence is initial[s] (zeros without)
//   delta[t] = grad[t] + f[t+1] delta[t+1]  (+ grad_final[s] at the last row),  dx = delta (1 - f),
//   dgate = delta (h[t-1] - x) f (1 - f),  dinitial[s] = f delta at the first row
// A row is the map c -> a c + b.  Maps compose: (a2, b2) after (a1, b1) is (a2 a1, a2 b1 + b2), so a tile of rows is one map per
// channel, and tiles can be worked on side by side: one kernel leaves the tiles' maps, one chains them, one goes over the rows
// again with what comes into each tile.  No kernel waits for another CTA, and every sum is made in one order.  A row that
// starts a sequence is the map c -> b whatever c is, also where c is not finite: its a is -0, and the sign says that what came
// before is not looked at (products keep it, f is never negative).
#include <type_traits>

#include "common.cuh"

namespace d3d {
namespace {

template <class T, int V> struct alignas(sizeof(T) * V) Pack { T v[V]; };

// The channels of a thread; two at a time are worked on by packed instructions.
template <int V> struct Vec { float v[V]; };
template <int V> __device__ __forceinline__ Vec<V> all(float x) {
  Vec<V> r;
#pragma unroll
  for (int e = 0; e < V; ++e) r.v[e] = x;
  return r;
}
template <int V> __device__ __forceinline__ float2 pair(const Vec<V>& a, int e) { return make_float2(a.v[e], a.v[e + 1]); }
template <int V> __device__ __forceinline__ Vec<V> fma(const Vec<V>& a, const Vec<V>& b, const Vec<V>& c) {
  Vec<V> r;
#pragma unroll
  for (int e = 0; e < V / 2 * 2; e += 2) {
    const float2 t = __ffma2_rn(pair(a, e), pair(b, e), pair(c, e));
    r.v[e] = t.x, r.v[e + 1] = t.y;
  }
  if constexpr (V % 2) r.v[V - 1] = fmaf(a.v[V - 1], b.v[V - 1], c.v[V - 1]);
  return r;
}
template <int V> __device__ __forceinline__ Vec<V> mul(const Vec<V>& a, const Vec<V>& b) {
  Vec<V> r;
#pragma unroll
  for (int e = 0; e < V / 2 * 2; e += 2) {
    const float2 t = __fmul2_rn(pair(a, e), pair(b, e));
    r.v[e] = t.x, r.v[e + 1] = t.y;
  }
  if constexpr (V % 2) r.v[V - 1] = a.v[V - 1] * b.v[V - 1];
  return r;
}
template <int V> __device__ __forceinline__ Vec<V> add(const Vec<V>& a, const Vec<V>& b) {
  Vec<V> r;
#pragma unroll
  for (int e = 0; e < V / 2 * 2; e += 2) {
    const float2 t = __fadd2_rn(pair(a, e), pair(b, e));
    r.v[e] = t.x, r.v[e + 1] = t.y;
  }
  if constexpr (V % 2) r.v[V - 1] = a.v[V - 1] + b.v[V - 1];
  return r;
}
template <class T, int V> __device__ __forceinline__ Vec<V> widen(const Pack<T, V>& p) {
  Vec<V> r;
  if constexpr (V == 2 && std::is_same<T, __nv_bfloat16>::value) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(&p);
    r.v[0] = __uint_as_float(w << 16), r.v[1] = __uint_as_float(w & 0xffff0000u);
    return r;
  }
  if constexpr (V == 2 && std::is_same<T, __half>::value) {
    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&p));
    r.v[0] = t.x, r.v[1] = t.y;
    return r;
  }
#pragma unroll
  for (int e = 0; e < V; ++e) r.v[e] = to_f32(p.v[e]);
  return r;
}
template <class T, int V> __device__ __forceinline__ Pack<T, V> narrow(const Vec<V>& x) {
  Pack<T, V> r;
  if constexpr (V == 2 && std::is_same<T, __nv_bfloat16>::value) {
    *reinterpret_cast<__nv_bfloat162*>(&r) = __float22bfloat162_rn(make_float2(x.v[0], x.v[1]));
    return r;
  }
  if constexpr (V == 2 && std::is_same<T, __half>::value) {
    *reinterpret_cast<__half2*>(&r) = __float22half2_rn(make_float2(x.v[0], x.v[1]));
    return r;
  }
#pragma unroll
  for (int e = 0; e < V; ++e) r.v[e] = from_f32<T>(x.v[e]);
  return r;
}

constexpr int kTile = 128;     // rows of a tile
constexpr int kThreads = 256;  // of a CTA
constexpr int kWarps = kThreads / 32;
constexpr int kTilesY = 32768;  // grid: slabs of channels, tiles, thousands of tiles

struct ScanArgs {
  const void *x, *gates;
  int64_t x_ld, gates_ld;
  const int32_t* offsets;
  int seqs;
  int64_t rows;
  int channels;
  int reverse;
  const float* initial;  // [seqs][channels] or null
  void* out;             // [rows][channels]
  float* final_state;    // [seqs][channels] or null
  // backward
  const void* grad;
  int64_t grad_ld;
  const float* grad_final;
  void *grad_x, *grad_gates;
  float* grad_initial;
  // between the passes
  float2* maps;   // [tiles][channels] the tile's map
  float* states;  // [tiles][channels] h in front of the tile's first row
  float* carry;   // [tiles][channels] backward: f delta of the row behind the tile
  int tiles;
};

__device__ __forceinline__ bool is_reset(float a) { return __float_as_int(a) < 0; }
__device__ __forceinline__ float reset_mark() { return __int_as_float((int)0x80000000u); }
// The map (a, b) at h.
__device__ __forceinline__ float apply(float a, float b, float h) { return is_reset(a) ? b : fmaf(a, h, b); }
// (a, b) after (pa, pb).
__device__ __forceinline__ void after(float& a, float& b, float pa, float pb) {
  if (!is_reset(a)) b = fmaf(a, pb, b), a *= pa;
}

// f = sigmoid(gate) and 1 - f: the smaller one is t / (1 + t), t = exp(-|gate|), the other one a difference that loses nothing.
// Neither has a sign, NaN included: the sign of a map means a reset.
// Features of 32 bits: exponential and quotient to two units of the last place.  Of 16 bits: the hardware's base-two exponential,
// whose argument is rounded to |gate| 2^-24 (so that 1 - f is off by that much, relatively; the gate itself came rounded to 2^-9
// or 2^-12 of it), a third of the instructions.
template <class T, int V> __device__ __forceinline__ Vec<V> small_of(const Vec<V>& g) {
  Vec<V> t, r;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < V; ++e) t.v[e] = expf(-fabsf(g.v[e]));
  } else {
    Vec<V> y;
#pragma unroll
    for (int e = 0; e < V; ++e) y.v[e] = fabsf(g.v[e]);
    y = mul(y, all<V>(-1.44269504f));
#pragma unroll
    for (int e = 0; e < V; ++e) asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t.v[e]) : "f"(y.v[e]));
  }
  const Vec<V> d = add(t, all<V>(1.f));
#pragma unroll
  for (int e = 0; e < V; ++e) {
    if constexpr (sizeof(T) == 4) r.v[e] = __fdividef(1.f, d.v[e]);
    else asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.v[e]) : "f"(d.v[e]));
  }
  return mul(t, r);
}
template <class T, int V> __device__ __forceinline__ void gate_of(const Vec<V>& g, Vec<V>& f, Vec<V>& rest) {
  const Vec<V> small = small_of<T, V>(g), large = fma(small, all<V>(-1.f), all<V>(1.f));
#pragma unroll
  for (int e = 0; e < V; ++e) f.v[e] = g.v[e] >= 0.f ? large.v[e] : small.v[e], rest.v[e] = g.v[e] >= 0.f ? small.v[e] : large.v[e];
}
// Both in one number: the smaller one, with a sign where that is f.
template <class T, int V> __device__ __forceinline__ Vec<V> folded_gate(const Vec<V>& g) {
  Vec<V> small = small_of<T, V>(g);
#pragma unroll
  for (int e = 0; e < V; ++e) small.v[e] = copysignf(small.v[e], g.v[e]);
  return small;
}
template <int V> __device__ __forceinline__ void open_gate(const Vec<V>& gate, Vec<V>& f, Vec<V>& rest) {
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const bool keeps = __float_as_int(gate.v[e]) >= 0;
    const float small = fabsf(gate.v[e]), large = 1.f - small;
    f.v[e] = keeps ? large : small, rest.v[e] = keeps ? small : large;
  }
}

// The rows the sequences cover, clamped to the tensor.
struct Span {
  int64_t begin, count;
};
__device__ __forceinline__ Span span_of(const ScanArgs& a) {
  int64_t b = __ldg(a.offsets), e = __ldg(a.offsets + a.seqs);
  b = b < 0 ? 0 : b < a.rows ? b : a.rows;
  e = e < b ? b : e < a.rows ? e : a.rows;
  return {b, a.seqs > 0 ? e - b : 0};
}
__device__ __forceinline__ int64_t row_at(const ScanArgs& a, const Span& s, int64_t p) {
  return a.reverse ? s.begin + s.count - 1 - p : s.begin + p;
}

// Where in a tile sequences start and end, in the order the rows are walked in: a bit per row, and whose row it is.
struct Marks {
  uint32_t first_bits[4], last_bits[4];
  int first[kTile], last[kTile];  // where the bit is set
  int range[2];                   // sequences of the tile's lowest and highest row
};

// The last sequence that starts at or before row t, by a whole warp: 32 probes a step.
__device__ __forceinline__ int sequence_of(const ScanArgs& a, int64_t t) {
  int lo = 0, n = a.seqs;
  while (n > 1) {
    const int step = (n + 31) / 32, at = lo + lane_id() * step;
    const unsigned before = __ballot_sync(0xffffffffu, at < lo + n && __ldg(a.offsets + at) <= t);
    const int k = before ? __popc(before) - 1 : 0, end = lo + n;
    lo += k * step;
    if (lo > end - 1) lo = end - 1;  // offsets out of order
    n = end - lo < step ? end - lo : step;
  }
  return lo;
}

// Fills `m` for the tile; the caller's barrier in front of its use of it.  Two barriers inside.
__device__ __forceinline__ void mark_ends(const ScanArgs& a, const Span& span, int tile, Marks* m) {
  const int64_t p0 = (int64_t)tile * kTile, n = span.count - p0 < kTile ? span.count - p0 : kTile;
  if (n <= 0) {
    if (threadIdx.x < 4) m->first_bits[threadIdx.x] = m->last_bits[threadIdx.x] = 0u;
    return;  // the whole CTA
  }
  const int64_t low = a.reverse ? row_at(a, span, p0 + n - 1) : row_at(a, span, p0);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x < 4) m->first_bits[threadIdx.x] = m->last_bits[threadIdx.x] = 0u;
  if (warp < 2) {
    const int s = sequence_of(a, warp ? low + n - 1 : low);
    if (lane_id() == 0) m->range[warp] = s;
  }
  __syncthreads();
  const int s1 = m->range[1];
  for (int s = m->range[0] + (int)threadIdx.x; s <= s1; s += kThreads) {
    const int64_t b = (int64_t)__ldg(a.offsets + s) - low, e = (int64_t)__ldg(a.offsets + s + 1) - 1 - low;
    if (e < b) continue;
    if (b >= 0 && b < n) {
      const int i = (int)(a.reverse ? n - 1 - b : b);
      (a.reverse ? m->last : m->first)[i] = s;
      atomicOr(&(a.reverse ? m->last_bits : m->first_bits)[i >> 5], 1u << (i & 31));
    }
    if (e >= 0 && e < n) {
      const int i = (int)(a.reverse ? n - 1 - e : e);
      (a.reverse ? m->first : m->last)[i] = s;
      atomicOr(&(a.reverse ? m->first_bits : m->last_bits)[i >> 5], 1u << (i & 31));
    }
  }
}

// A thread's place: kLanes threads stand side by side along the channels, V channels each; the groups of them follow the rows,
// kRows each.
template <int V, int kLanes> struct Place {
  static constexpr int kRows = kTile * kLanes / kThreads, kWidth = V * kLanes;
  int tile, slab, lane, group, c, rows;  // rows: of this thread that there are
  int64_t first;                         // row of the tensors that the tile's first one would be, walked upwards
  __device__ __forceinline__ Place(const ScanArgs& a, const Span& span) {
    slab = blockIdx.x, tile = blockIdx.z * kTilesY + blockIdx.y;
    lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes, c = slab * kWidth + lane * V;
    const int64_t p = (int64_t)tile * kTile, left = span.count - p - group * kRows;
    rows = c >= a.channels || left <= 0 ? 0 : left < kRows ? (int)left : kRows;
    first = a.reverse ? span.begin + span.count - p - kTile : span.begin + p;
  }
  // The thread's first row walked (of kRows) in rows `ld` elements apart, and the distance to the next one.
  template <class T> __device__ __forceinline__ T* start(T* base, int64_t ld, bool reverse) const {
    return base + (first + (reverse ? kTile - 1 - group * kRows : group * kRows)) * ld + c;
  }
  static __device__ __forceinline__ int64_t step(int64_t ld, bool reverse) { return reverse ? -ld : ld; }
  __device__ __forceinline__ uint32_t bits(const uint32_t* of_tile) const {
    const int at = group * kRows;
    return of_tile[at >> 5] >> (at & 31) & ((1u << kRows) - 1);
  }
};

template <class T, int V, int kLanes>
__device__ __forceinline__ void load_rows(Pack<T, V> (&to)[Place<V, kLanes>::kRows], const Place<V, kLanes>& at, const void* p, int64_t ld, bool reverse) {
  constexpr int kRows = Place<V, kLanes>::kRows;
  const T* src = at.start((const T*)p, ld, reverse);
  const int64_t step = at.step(ld, reverse);
  if (at.rows == kRows) {
#pragma unroll
    for (int r = 0; r < kRows; ++r, src += step) to[r] = *reinterpret_cast<const Pack<T, V>*>(src);
  } else {
#pragma unroll
    for (int r = 0; r < kRows; ++r, src += step)
      if (r < at.rows) to[r] = *reinterpret_cast<const Pack<T, V>*>(src);
  }
}
template <int V> __device__ __forceinline__ Vec<V> load_state(const float* p, int64_t s, int channels, int c) {
  Vec<V> r = all<V>(0.f);
  if (p)
#pragma unroll
    for (int e = 0; e < V; ++e) r.v[e] = __ldg(p + s * channels + c + e);
  return r;
}
template <int V> __device__ __forceinline__ void store_state(float* p, int64_t s, int channels, int c, const Vec<V>& h) {
  if (p)
#pragma unroll
    for (int e = 0; e < V; ++e) p[s * channels + c + e] = h.v[e];
}

// From the maps of the threads' rows to what comes in front of them (kUp) or behind them, in three steps with a barrier after
// each: every thread brings its map, the channels' chains over the warps are walked by a thread each (a product a warp), every
// thread takes what comes in.  Two of them side by side: the backward pass goes both ways.
template <int V, int kLanes, int kChains = 1> struct Chain {
  static constexpr int kWidth = V * kLanes;
  float2 totals[kChains][kWarps][kWidth];
  float into[kChains][kWarps][kWidth];

  // Afterwards the thread's map is that of its group and of those of its warp on the way to it.
  template <bool kUp> __device__ __forceinline__ void bring_unsynced(int i, Vec<V>& ma, Vec<V>& mb, const Place<V, kLanes>& at) {
    const int lane = lane_id(), warp = threadIdx.x >> 5, col = at.lane * V;
    if constexpr (kLanes < 32)
#pragma unroll
      for (int d = kLanes; d < 32; d <<= 1)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float pa = kUp ? __shfl_up_sync(0xffffffffu, ma.v[e], d) : __shfl_down_sync(0xffffffffu, ma.v[e], d);
          const float pb = kUp ? __shfl_up_sync(0xffffffffu, mb.v[e], d) : __shfl_down_sync(0xffffffffu, mb.v[e], d);
          if (kUp ? lane >= d : lane + d < 32) after(ma.v[e], mb.v[e], pa, pb);
        }
    if (kUp ? lane >= 32 - kLanes : lane < kLanes)
#pragma unroll
      for (int e = 0; e < V; ++e) totals[i][warp][col + e] = make_float2(ma.v[e], mb.v[e]);
  }
  template <bool kUp> __device__ __forceinline__ void bring(int i, Vec<V>& ma, Vec<V>& mb, const Place<V, kLanes>& at) {
    bring_unsynced<kUp>(i, ma, mb, at);
    __syncthreads();
  }
  // The tile's map.
  template <bool kUp> __device__ __forceinline__ void map(int i, float2* maps, const Place<V, kLanes>& at, int channels) const {
    const int t = threadIdx.x, c = at.slab * kWidth + t;
    if (t >= kWidth || c >= channels) return;
    float a = 1.f, b = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      float2 m = totals[i][kUp ? w : kWarps - 1 - w][t];
      after(m.x, m.y, a, b);
      a = m.x, b = m.y;
    }
    maps[(int64_t)at.tile * channels + c] = make_float2(a, b);
  }
  // carry: [tiles][channels] what comes into the tile, or null for zeros.  Chain i has the threads from i * kWidth on.
  template <bool kUp> __device__ __forceinline__ void walk(int i, const float* carry, const Place<V, kLanes>& at, int channels) {
    const int t = (int)threadIdx.x - i * kWidth, c = at.slab * kWidth + t;
    if (t < 0 || t >= kWidth || c >= channels) return;
    float h = carry ? __ldg(carry + (int64_t)at.tile * channels + c) : 0.f;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) {
      const int w = kUp ? k : kWarps - 1 - k;
      into[i][w][t] = h;
      const float2 m = totals[i][w][t];
      h = apply(m.x, m.y, h);
    }
  }
  template <bool kUp> __device__ __forceinline__ Vec<V> take(int i, const Vec<V>& ma, const Vec<V>& mb, const Place<V, kLanes>& at) const {
    const int lane = lane_id(), warp = threadIdx.x >> 5, col = at.lane * V;
    Vec<V> h;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      h.v[e] = into[i][warp][col + e];
      if constexpr (kLanes < 32) {
        const float pa = kUp ? __shfl_up_sync(0xffffffffu, ma.v[e], kLanes) : __shfl_down_sync(0xffffffffu, ma.v[e], kLanes);
        const float pb = kUp ? __shfl_up_sync(0xffffffffu, mb.v[e], kLanes) : __shfl_down_sync(0xffffffffu, mb.v[e], kLanes);
        if (kUp ? lane >= kLanes : lane + kLanes < 32) h.v[e] = apply(pa, pb, h.v[e]);
      }
    }
    return h;
  }
};

// Sequences without rows: their last state is the one they start with.
template <int V, int kLanes>
__device__ __forceinline__ void pass_empty(const ScanArgs& a, const Place<V, kLanes>& at, const float* from, float* to) {
  if (!to) return;
  const int tiles = a.tiles > 0 ? a.tiles : 1, low = at.slab * V * kLanes;
  const int high = low + V * kLanes < a.channels ? low + V * kLanes : a.channels;
  for (int64_t s = (int64_t)at.tile * kThreads + threadIdx.x; s < a.seqs; s += (int64_t)tiles * kThreads)
    if (__ldg(a.offsets + s + 1) <= __ldg(a.offsets + s))
      for (int c = low; c < high; ++c) to[s * a.channels + c] = from ? __ldg(from + s * a.channels + c) : 0.f;
}

// kMaps: the first pass, which leaves the tile's map.  Rows between two ends of sequences, all but a few, take a path without
// the tests.
template <class T, int V, int kLanes, bool kMaps>
__global__ void __launch_bounds__(kThreads, kMaps ? 3 : 2)
scan_kernel(const ScanArgs a) {
  constexpr int kRows = Place<V, kLanes>::kRows;
  using P = Pack<T, V>;
  __shared__ Marks marks;
  __shared__ Chain<V, kLanes> chain;
  const Span span = span_of(a);
  const Place<V, kLanes> at(a, span);
  const bool reverse = a.reverse != 0;
  if (at.tile >= a.tiles && at.tile > 0) return;  // the last thousands of tiles are not all there
  if (kMaps) pdl_release();
  P x[kRows], g[kRows];
  load_rows<T, V, kLanes>(x, at, a.x, a.x_ld, reverse);
  load_rows<T, V, kLanes>(g, at, a.gates, a.gates_ld, reverse);
  mark_ends(a, span, at.tile, &marks);
  __syncthreads();
  const uint32_t starts = at.bits(marks.first_bits), ends = at.bits(marks.last_bits);
  const int* first = marks.first + at.group * kRows;
  const int* last = marks.last + at.group * kRows;
  Vec<V> f[kRows], u[kRows], ma = all<V>(1.f), mb = all<V>(0.f);
  auto enter = [&](auto is_plain) {
    constexpr bool kPlain = decltype(is_plain)::value;
#pragma unroll
    for (int r = 0; r < kRows; ++r)
      if (kPlain || r < at.rows) {
        Vec<V> rest;
        gate_of<T, V>(widen<T, V>(g[r]), f[r], rest);
        u[r] = mul(rest, widen<T, V>(x[r]));
        if (!kPlain && (starts >> r & 1)) {
          u[r] = fma(f[r], load_state<V>(a.initial, first[r], a.channels, at.c), u[r]);
          f[r] = ma = all<V>(reset_mark()), mb = u[r];
        } else {
          mb = fma(f[r], mb, u[r]), ma = mul(ma, f[r]);
        }
      }
  };
  const bool plain = at.rows == kRows && starts == 0;
  if (plain) enter(std::true_type());
  else enter(std::false_type());
  if (!kMaps) pdl_wait();
  chain.template bring<true>(0, ma, mb, at);
  if (kMaps) {
    chain.template map<true>(0, a.maps, at, a.channels);
    return;
  }
  chain.template walk<true>(0, a.states, at, a.channels);
  __syncthreads();
  Vec<V> h = chain.template take<true>(0, ma, mb, at);
  T* out = at.start((T*)a.out, a.channels, reverse);
  const int64_t step = at.step(a.channels, reverse);
  auto leave = [&](auto is_plain) {
    constexpr bool kPlain = decltype(is_plain)::value;
#pragma unroll
    for (int r = 0; r < kRows; ++r, out += step)
      if (kPlain || r < at.rows) {
        h = !kPlain && (starts >> r & 1) ? u[r] : fma(f[r], h, u[r]);
        *reinterpret_cast<P*>(out) = narrow<T, V>(h);
        if (!kPlain && (ends >> r & 1)) store_state<V>(a.final_state, last[r], a.channels, at.c, h);
      }
  };
  if (plain && ends == 0) leave(std::true_type());
  else leave(std::false_type());
  pass_empty<V, kLanes>(a, at, a.initial, a.final_state);
}

// What comes into each tile: the tiles' maps one after the other, from the first (or, backwards, the last) on.  Eight channels to
// a CTA; 128 threads of each take kHeld tiles into registers, chain them, and are chained by shuffles and through shared memory.
constexpr int kHeld = 8, kCarryThreads = 1024, kCarryChannels = 8;
__global__ void __launch_bounds__(kCarryThreads)
carry_kernel(const float2* __restrict__ maps, float* __restrict__ into, int tiles, int channels, int backward) {
  __shared__ float2 totals[32][kCarryChannels];
  __shared__ float starts[32][kCarryChannels];
  const int lane = lane_id(), warp = threadIdx.x >> 5, ch = threadIdx.x % kCarryChannels, c = blockIdx.x * kCarryChannels + ch;
  const int segment = threadIdx.x / kCarryChannels;
  pdl_release();
  pdl_wait();
  float carry = 0.f;  // of channel `warp` of this CTA, in the warps that chain
  constexpr int kTurn = kCarryThreads / kCarryChannels * kHeld;
  for (int t0 = 0; t0 < tiles; t0 += kTurn) {
    float2 m[kHeld];
    float a = 1.f, b = 0.f;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int t = t0 + segment * kHeld + i;
      m[i] = make_float2(1.f, 0.f);
      if (t < tiles && c < channels) m[i] = __ldg(maps + (int64_t)(backward ? tiles - 1 - t : t) * channels + c);
    }
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      float na = m[i].x, nb = m[i].y;
      after(na, nb, a, b);
      a = na, b = nb;
    }
#pragma unroll
    for (int d = kCarryChannels; d < 32; d <<= 1) {
      const float pa = __shfl_up_sync(0xffffffffu, a, d), pb = __shfl_up_sync(0xffffffffu, b, d);
      if (lane >= d) after(a, b, pa, pb);
    }
    if (lane >= 32 - kCarryChannels) totals[warp][ch] = make_float2(a, b);
    __syncthreads();
    if (warp < kCarryChannels) {  // a warp per channel, a lane per warp's total
      float2 w = totals[lane][warp];
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const float pa = __shfl_up_sync(0xffffffffu, w.x, d), pb = __shfl_up_sync(0xffffffffu, w.y, d);
        if (lane >= d) after(w.x, w.y, pa, pb);
      }
      const float end = apply(w.x, w.y, carry), before = __shfl_up_sync(0xffffffffu, end, 1);
      starts[lane][warp] = lane ? before : carry;
      carry = __shfl_sync(0xffffffffu, end, 31);
    }
    __syncthreads();
    float h = starts[warp][ch];
    const float pa = __shfl_up_sync(0xffffffffu, a, kCarryChannels), pb = __shfl_up_sync(0xffffffffu, b, kCarryChannels);
    if (lane >= kCarryChannels) h = apply(pa, pb, h);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int t = t0 + segment * kHeld + i;
      if (t < tiles && c < channels) into[(int64_t)(backward ? tiles - 1 - t : t) * channels + c] = h;
      h = apply(m[i].x, m[i].y, h);
    }
  }
}

// Backward: the rows of a tile forward once more from the state in front of it, which gives h[t-1], and the gradients from its
// end.  The map of a row is c -> f (grad + c): c comes in from the row behind and goes out to the row in front.  Between the
// passes a thread holds its gates (the smaller halves), h[t-1] - x and the gradients as they came.
template <class T, int V, int kLanes, bool kMaps>
__global__ void __launch_bounds__(kThreads, kMaps ? 3 : 2)
scan_backward_kernel(const ScanArgs a) {
  constexpr int kRows = Place<V, kLanes>::kRows;
  using P = Pack<T, V>;
  __shared__ Marks marks;
  __shared__ Chain<V, kLanes, 2> chain;
  const Span span = span_of(a);
  const Place<V, kLanes> at(a, span);
  const bool reverse = a.reverse != 0;
  if (at.tile >= a.tiles && at.tile > 0) return;  // the last thousands of tiles are not all there
  if (kMaps) pdl_release();
  P x[kRows], g[kRows], d[kRows];
  if (!kMaps) load_rows<T, V, kLanes>(x, at, a.x, a.x_ld, reverse);
  load_rows<T, V, kLanes>(g, at, a.gates, a.gates_ld, reverse);
  load_rows<T, V, kLanes>(d, at, a.grad, a.grad_ld, reverse);
  mark_ends(a, span, at.tile, &marks);
  __syncthreads();
  const uint32_t starts = at.bits(marks.first_bits), ends = at.bits(marks.last_bits);
  const int* first = marks.first + at.group * kRows;
  const int* last = marks.last + at.group * kRows;
  const bool plain = at.rows == kRows && starts == 0 && ends == 0;
  Vec<V> gate[kRows], away[kRows];
  Vec<V> ma = all<V>(1.f), mb = all<V>(0.f), na = all<V>(1.f), nb = all<V>(0.f);  // forward; from the end
  auto enter = [&](auto is_plain) {
    constexpr bool kPlain = decltype(is_plain)::value;
#pragma unroll
    for (int r = 0; r < kRows; ++r)
      if (kPlain || r < at.rows) {
        gate[r] = folded_gate<T, V>(widen<T, V>(g[r]));
        Vec<V> f, rest;
        open_gate<V>(gate[r], f, rest);
        if (!kMaps) {
          const Vec<V> u = mul(rest, widen<T, V>(x[r]));
          if (!kPlain && (starts >> r & 1))
            ma = all<V>(reset_mark()), mb = fma(f, load_state<V>(a.initial, first[r], a.channels, at.c), u);
          else
            mb = fma(f, mb, u), ma = mul(ma, f);
        }
        // the rows so far after this one: its end is what comes in
        if (kPlain || !is_reset(na.v[0])) {
          Vec<V> dy = widen<T, V>(d[r]);
          const bool end = !kPlain && (ends >> r & 1);
          if (end) dy = add(dy, load_state<V>(a.grad_final, last[r], a.channels, at.c));
          nb = fma(mul(na, f), dy, nb);
          na = end ? all<V>(reset_mark()) : mul(na, f);
        }
      }
  };
  if (plain) enter(std::true_type());
  else enter(std::false_type());
  if (!kMaps) pdl_wait();
  if (!kMaps) chain.template bring_unsynced<true>(0, ma, mb, at);
  chain.template bring<false>(1, na, nb, at);
  if (kMaps) {
    chain.template map<false>(1, a.maps, at, a.channels);
    return;
  }
  chain.template walk<true>(0, a.states, at, a.channels);
  chain.template walk<false>(1, a.carry, at, a.channels);
  __syncthreads();
  Vec<V> h = chain.template take<true>(0, ma, mb, at), q = chain.template take<false>(1, na, nb, at);
  auto leave = [&](auto is_plain) {
    constexpr bool kPlain = decltype(is_plain)::value;
#pragma unroll
    for (int r = 0; r < kRows; ++r)
      if (kPlain || r < at.rows) {
        Vec<V> f, rest;
        open_gate<V>(gate[r], f, rest);
        if (!kPlain && (starts >> r & 1)) h = load_state<V>(a.initial, first[r], a.channels, at.c);
        const Vec<V> in = widen<T, V>(x[r]);
        away[r] = fma(in, all<V>(-1.f), h);
        h = fma(f, h, mul(rest, in));
      }
    const int64_t step = at.step(a.channels, reverse);
    T* dx_at = at.start((T*)a.grad_x, a.channels, reverse) + (kRows - 1) * step;
    T* dg_at = at.start((T*)a.grad_gates, a.channels, reverse) + (kRows - 1) * step;
#pragma unroll
    for (int r = kRows - 1; r >= 0; --r, dx_at -= step, dg_at -= step)
      if (kPlain || r < at.rows) {
        Vec<V> f, rest;
        open_gate<V>(gate[r], f, rest);
        if (!kPlain && (ends >> r & 1)) q = load_state<V>(a.grad_final, last[r], a.channels, at.c);
        const Vec<V> delta = add(widen<T, V>(d[r]), q), dx = mul(delta, rest);
        q = mul(f, delta);
        *reinterpret_cast<P*>(dx_at) = narrow<T, V>(dx);
        *reinterpret_cast<P*>(dg_at) = narrow<T, V>(mul(mul(q, rest), away[r]));
        if (!kPlain && (starts >> r & 1)) store_state<V>(a.grad_initial, first[r], a.channels, at.c, q);
      }
  };
  if (plain) leave(std::true_type());
  else leave(std::false_type());
  pass_empty<V, kLanes>(a, at, a.grad_final, a.grad_initial);
}

// One row a sequence: the state is read, moved on and written; state_out may be state.
template <class T, int V>
__global__ void __launch_bounds__(256)
step_kernel(const T* __restrict__ x, int64_t x_ld, const T* __restrict__ gates, int64_t gates_ld, const float* state,
            float* state_out, T* __restrict__ out, int64_t rows, int channels) {
  using P = Pack<T, V>;
  const int per_row = channels / V;
  const int64_t n = rows * per_row, nth = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += nth) {
    const int64_t row = i / per_row, at = i * V;
    const int c = (int)(i - row * per_row) * V;
    const P px = *reinterpret_cast<const P*>(x + row * x_ld + c), pg = *reinterpret_cast<const P*>(gates + row * gates_ld + c);
    Pack<float, V> h = *reinterpret_cast<const Pack<float, V>*>(state + at);
    Vec<V> f, rest, v;
#pragma unroll
    for (int e = 0; e < V; ++e) v.v[e] = h.v[e];
    gate_of<T, V>(widen<T, V>(pg), f, rest);
    v = fma(f, v, mul(rest, widen<T, V>(px)));
#pragma unroll
    for (int e = 0; e < V; ++e) h.v[e] = v.v[e];
    *reinterpret_cast<Pack<float, V>*>(state_out + at) = h;
    *reinterpret_cast<P*>(out + at) = narrow<T, V>(v);
  }
}

// f(V, lanes) for the tile shape of this many channels: two channels a thread where rows can be read so, and as few threads side
// by side as cover the channels.
template <class F> int by_shape(bool pairs, int channels, F f) {
#define D3D_SCAN_SHAPE(V, L) return f(std::integral_constant<int, V>(), std::integral_constant<int, L>())
  if (!pairs) D3D_SCAN_SHAPE(1, 32);
  if (channels <= 16) D3D_SCAN_SHAPE(2, 8);
  if (channels <= 32) D3D_SCAN_SHAPE(2, 16);
  D3D_SCAN_SHAPE(2, 32);
#undef D3D_SCAN_SHAPE
}
template <class F> int by_type(int dtype, F f) {
  switch (dtype) {
    case D3D_FLOAT: return f(float());
    case D3D_HALF: return f(__half());
    case D3D_BF16: return f(__nv_bfloat16());
    default: return D3D_ERR_UNSUPPORTED_DTYPE;
  }
}

dim3 grid_of(int tiles, int64_t slabs) {
  const int n = tiles > 0 ? tiles : 1;
  return dim3((unsigned)slabs, (unsigned)(n < kTilesY ? n : kTilesY), (unsigned)ceil_div(n, kTilesY));
}

// Whether rows of `ld` elements from `p` on can be read in pairs.
bool rows_paired(const void* p, int64_t ld, int esize) { return reinterpret_cast<uintptr_t>(p) % (2 * esize) == 0 && ld % 2 == 0; }

int check_scan(int dtype, const ScanArgs& a) {
  D3D_REQUIRE(dtype == D3D_FLOAT || dtype == D3D_HALF || dtype == D3D_BF16, D3D_ERR_UNSUPPORTED_DTYPE);
  D3D_REQUIRE(a.rows >= 0 && a.channels >= 1 && a.seqs >= 0 && a.x_ld >= a.channels && a.gates_ld >= a.channels && a.offsets,
              D3D_ERR_INVALID_ARGUMENT);
  D3D_REQUIRE(a.rows < (1ll << 31) && a.channels <= (1 << 16) &&
                  ceil_div(a.rows, kTile) * ceil_div(a.channels, 32) < (1ll << 30),
              D3D_ERR_TOO_LARGE);
  const int esize = (int)dtype_size(dtype);
  D3D_REQUIRE(reinterpret_cast<uintptr_t>(a.x) % esize == 0 && reinterpret_cast<uintptr_t>(a.gates) % esize == 0 &&
                  reinterpret_cast<uintptr_t>(a.grad) % esize == 0,
              D3D_ERR_INVALID_ARGUMENT);
  return D3D_OK;
}

}  // namespace
}  // namespace d3d

using namespace d3d;

extern "C" int64_t d3d_gated_recurrence_state_rows(int64_t rows) { return rows < 0 ? 0 : ceil_div(rows > 0 ? rows : 1, kTile); }

extern "C" size_t d3d_gated_recurrence_workspace(int64_t rows, int channels) {
  if (rows < 0 || channels < 1) return 0;
  const size_t n = (size_t)d3d_gated_recurrence_state_rows(rows) * channels;
  return align_up(n * sizeof(float2), 256) + align_up(n * sizeof(float), 256);
}

extern "C" int d3d_gated_recurrence(int dtype, const void* x, int64_t x_ld, const void* gates, int64_t gates_ld,
                                    const int32_t* offsets, int seqs, int64_t rows, int channels, int reverse,
                                    const float* initial, void* out, float* final_state, float* states, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  D3D_NVTX_RANGE("d3d_gated_recurrence");
  ScanArgs a = {};
  a.x = x, a.x_ld = x_ld, a.gates = gates, a.gates_ld = gates_ld, a.offsets = offsets, a.seqs = seqs, a.rows = rows;
  a.channels = channels, a.reverse = reverse != 0, a.initial = initial, a.out = out, a.final_state = final_state;
  const int rc = check_scan(dtype, a);
  D3D_REQUIRE(rc == D3D_OK, rc);
  D3D_REQUIRE(rows == 0 || (x && gates && out), D3D_ERR_INVALID_ARGUMENT);
  D3D_REQUIRE(workspace && reinterpret_cast<uintptr_t>(workspace) % 256 == 0, D3D_ERR_INVALID_ARGUMENT);
  D3D_REQUIRE(workspace_bytes >= d3d_gated_recurrence_workspace(rows, channels), D3D_ERR_WORKSPACE_TOO_SMALL);
  Carver w(workspace);
  a.maps = w.take<float2>((size_t)d3d_gated_recurrence_state_rows(rows) * channels);
  a.states = states ? states : w.take<float>((size_t)d3d_gated_recurrence_state_rows(rows) * channels);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int esize = (int)dtype_size(dtype);
  const bool pairs = channels % 2 == 0 && rows_paired(x, x_ld, esize) && rows_paired(gates, gates_ld, esize) && rows_paired(out, channels, esize);
  if (seqs == 0) return D3D_OK;
  return by_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    return by_shape(pairs, channels, [&](auto v, auto l) -> int {
      constexpr int V = decltype(v)::value, L = decltype(l)::value;
      a.tiles = (int)ceil_div(rows, kTile);
      const dim3 grid = grid_of(a.tiles, ceil_div(channels, V * L));
      if (a.tiles > 1) {
        scan_kernel<T, V, L, true><<<grid, kThreads, 0, st>>>(a);
        D3D_CHECK_LAUNCH();
        D3D_LAUNCH(true, carry_kernel, (unsigned)ceil_div(channels, kCarryChannels), kCarryThreads, 0, st, a.maps, a.states, a.tiles,
                   channels, 0);
      } else if (states) {  // nothing lies in front of the only tile
        if (cudaMemsetAsync(states, 0, channels * sizeof(float), st) != cudaSuccess) return D3D_ERR_CUDA;
      } else {
        a.states = nullptr;
      }
      D3D_LAUNCH(a.tiles > 1, (scan_kernel<T, V, L, false>), grid, kThreads, 0, st, a);
      D3D_CHECK_LAUNCH();
      return D3D_OK;
    });
  });
}

extern "C" int d3d_gated_recurrence_backward(int dtype, const void* grad, int64_t grad_ld, const void* x, int64_t x_ld,
                                             const void* gates, int64_t gates_ld, const int32_t* offsets, int seqs,
                                             int64_t rows, int channels, int reverse, const float* states,
                                             const float* initial, const float* grad_final, void* grad_x,
                                             void* grad_gates, float* grad_initial, void* workspace,
                                             size_t workspace_bytes, void* stream) {
  D3D_NVTX_RANGE("d3d_gated_recurrence_backward");
  ScanArgs a = {};
  a.x = x, a.x_ld = x_ld, a.gates = gates, a.gates_ld = gates_ld, a.offsets = offsets, a.seqs = seqs, a.rows = rows;
  a.channels = channels, a.reverse = reverse != 0, a.initial = initial, a.grad = grad, a.grad_ld = grad_ld;
  a.grad_final = grad_final, a.grad_x = grad_x, a.grad_gates = grad_gates, a.grad_initial = grad_initial;
  const int rc = check_scan(dtype, a);
  D3D_REQUIRE(rc == D3D_OK, rc);
  D3D_REQUIRE(grad_ld >= channels && (rows == 0 || (x && gates && grad && states && grad_x && grad_gates)),
              D3D_ERR_INVALID_ARGUMENT);
  D3D_REQUIRE(workspace && reinterpret_cast<uintptr_t>(workspace) % 256 == 0, D3D_ERR_INVALID_ARGUMENT);
  D3D_REQUIRE(workspace_bytes >= d3d_gated_recurrence_workspace(rows, channels), D3D_ERR_WORKSPACE_TOO_SMALL);
  Carver w(workspace);
  a.maps = w.take<float2>((size_t)d3d_gated_recurrence_state_rows(rows) * channels);
  a.carry = w.take<float>((size_t)d3d_gated_recurrence_state_rows(rows) * channels);
  a.states = const_cast<float*>(states);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int esize = (int)dtype_size(dtype);
  const bool pairs = channels % 2 == 0 && rows_paired(x, x_ld, esize) && rows_paired(gates, gates_ld, esize) &&
                     rows_paired(grad, grad_ld, esize) && rows_paired(grad_x, channels, esize) && rows_paired(grad_gates, channels, esize);
  if (seqs == 0) return D3D_OK;
  return by_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    return by_shape(pairs, channels, [&](auto v, auto l) -> int {
      constexpr int V = decltype(v)::value, L = decltype(l)::value;
      a.tiles = (int)ceil_div(rows, kTile);
      const dim3 grid = grid_of(a.tiles, ceil_div(channels, V * L));
      if (a.tiles > 1) {
        scan_backward_kernel<T, V, L, true><<<grid, kThreads, 0, st>>>(a);
        D3D_CHECK_LAUNCH();
        D3D_LAUNCH(true, carry_kernel, (unsigned)ceil_div(channels, kCarryChannels), kCarryThreads, 0, st, a.maps, a.carry, a.tiles,
                   channels, 1);
      } else {
        a.carry = nullptr;  // nothing lies behind the only tile
      }
      D3D_LAUNCH(a.tiles > 1, (scan_backward_kernel<T, V, L, false>), grid, kThreads, 0, st, a);
      D3D_CHECK_LAUNCH();
      return D3D_OK;
    });
  });
}

extern "C" int d3d_gated_recurrence_step(int dtype, const void* x, int64_t x_ld, const void* gates, int64_t gates_ld,
                                         const float* state, float* state_out, void* out, int64_t rows, int channels,
                                         void* stream) {
  D3D_NVTX_RANGE("d3d_gated_recurrence_step");
  D3D_REQUIRE(dtype == D3D_FLOAT || dtype == D3D_HALF || dtype == D3D_BF16, D3D_ERR_UNSUPPORTED_DTYPE);
  D3D_REQUIRE(rows >= 0 && channels >= 1 && x_ld >= channels && gates_ld >= channels, D3D_ERR_INVALID_ARGUMENT);
  if (rows == 0) return D3D_OK;
  const int esize = (int)dtype_size(dtype);
  D3D_REQUIRE(x && gates && state && state_out && out && reinterpret_cast<uintptr_t>(x) % esize == 0 &&
                  reinterpret_cast<uintptr_t>(gates) % esize == 0 && reinterpret_cast<uintptr_t>(out) % esize == 0,
              D3D_ERR_INVALID_ARGUMENT);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  auto wide_rows = [esize](const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * esize % 16 == 0; };
  const bool wide = channels * esize % 16 == 0 && wide_rows(x, x_ld) && wide_rows(gates, gates_ld) && wide_rows(out, channels) && reinterpret_cast<uintptr_t>(state) % 32 == 0 &&
                    reinterpret_cast<uintptr_t>(state_out) % 32 == 0;
  return by_type(dtype, [&](auto t) -> int {
    using T = decltype(t);
    constexpr int V = 16 / (int)sizeof(T);
    if (wide)
      step_kernel<T, V><<<stream_grid(rows * (channels / V), 256), 256, 0, st>>>((const T*)x, x_ld, (const T*)gates, gates_ld, state,
                                                                                state_out, (T*)out, rows, channels);
    else
      step_kernel<T, 1><<<stream_grid(rows * channels, 256), 256, 0, st>>>((const T*)x, x_ld, (const T*)gates, gates_ld, state,
                                                                          state_out, (T*)out, rows, channels);
    D3D_CHECK_LAUNCH();
    return D3D_OK;
  });
}
